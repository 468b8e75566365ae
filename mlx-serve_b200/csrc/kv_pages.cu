// The paged key-value cache: new rows into pages, and the bookkeeping of the pages themselves.
//
// A pool [pages, heads, page, cols] holds the rows of many sequences; table [sequences, M] names the pages of each (-1: none),
// lens the tokens, refs how many table entries name a page (0: free).  All three live on the device, so that a serving loop
// forks, grows and frees sequences without reading anything back.  Integer work throughout: results do not depend on the order
// in which blocks or atomics run.
#include <cstddef>
#include <cstring>
#include <mutex>

#include "kernels.h"
#include "quant_rows.cuh"
#include "stream_ptx.cuh"

namespace qb {
namespace {

// These kernels follow each other in a serving loop, each a few microseconds long: they are launched while the one before still runs
// and wait here for all that it writes.
__device__ __forceinline__ void grid_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// ---------------------------------------------------------------- new rows into pages
// Row (n, i) of head h goes to slot (pos % page) of page table[r, pos / page], pos = positions[n] + i.  16 values a thread: the four
// (head dim 64) or eight threads of a row are neighbours, rows of one head follow each other as tokens do, so that both sides are
// read and written in whole sectors.  A block has rows of one (sequence, K or V, head); the values are asked for before the table is
// looked up.  Bound by the launch at one token a sequence (13 sequences of 8 heads of 128: 5.5 to 6.1 us), by instructions at prompt lengths:
// a warp's 512 values take 388, most of them to divide as the quantiser defines it, and 68 % of the issue slots are used (8192 tokens
// of 8 heads at 8 bits, 45 MB in and out: 17.9 us, floor 6.9).
template <int BITS>
__global__ void __launch_bounds__(256) pages_append_kernel(const __grid_constant__ KvPagesAppendArgs a) {
  grid_wait();
  const uint32_t r2 = blockIdx.x / a.tiles, tile = blockIdx.x - r2 * a.tiles;
  const uint32_t r3 = r2 / a.H, h = r2 - r3 * a.H;
  const uint32_t kv = r3 & 1u, n = r3 >> 1;
  const uint32_t i = tile * blockDim.x + threadIdx.x, s0 = a.row_shift >= 0 ? i >> a.row_shift : i / a.per_row;
  const bool in = s0 < (uint32_t)a.S;
  const uint32_t s = in ? s0 : a.S - 1, c = i - s0 * a.per_row;
  const uint16_t* x = (kv ? a.dense[1] : a.dense[0]) + (int64_t)n * (kv ? a.dense_str[1][0] : a.dense_str[0][0]) + (int64_t)h * (kv ? a.dense_str[1][1] : a.dense_str[0][1]) +
                      (int64_t)s * (kv ? a.dense_str[1][2] : a.dense_str[0][2]) + c * kRowVals;
  uint4 raw[2];
  if (a.dense_vec) {
    raw[0] = ((const uint4*)x)[0]; raw[1] = ((const uint4*)x)[1];
  } else {
    uint32_t e[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) e[k] = (uint32_t)x[2 * k] | ((uint32_t)x[2 * k + 1] << 16);
    raw[0] = make_uint4(e[0], e[1], e[2], e[3]); raw[1] = make_uint4(e[4], e[5], e[6], e[7]);
  }
  const int64_t row = a.rows ? a.rows[n] : (int64_t)n;
  const int64_t first = a.positions[n], pos = first + s;
  // (below 0: an entry that reserve refused, none of whose rows has a place -- not even those whose own position would be 0 or above)
  bool live = in && row >= 0 && row < a.seqs && first >= 0 && (pos >> a.page_shift) < a.M && (!a.counts || (int64_t)s < a.counts[n]);
  const int64_t pid = live ? a.table[row * a.table_str + (pos >> a.page_shift)] : -1;
  live = live && pid >= 0 && pid < a.P;
  if (!__any_sync(0xffffffffu, live)) return;
  const KvPoolView& p = kv ? a.pool[1] : a.pool[0];
  const int64_t slot = pos & ((1 << a.page_shift) - 1);
  if constexpr (BITS == 16) {
    if (!live) return;
    uint4* o = (uint4*)((uint16_t*)p.q + pid * p.q_str[0] + h * p.q_str[1] + slot * p.q_str[2] + c * kRowVals);
    o[0] = raw[0]; o[1] = raw[1];
  } else {
    const uint32_t vals[8] = {raw[0].x, raw[0].y, raw[0].z, raw[0].w, raw[1].x, raw[1].y, raw[1].z, raw[1].w};
    float scale, bias;
    uint32_t w[BITS / 2];
    quantize16<BITS>(vals, 4, w, scale, bias);
    if (!live) return;
    uint32_t* o = (uint32_t*)p.q + pid * p.q_str[0] + h * p.q_str[1] + slot * p.q_str[2] + c * (BITS / 2);
    if constexpr (BITS == 4) *(uint2*)o = make_uint2(w[0], w[1]); else *(uint4*)o = make_uint4(w[0], w[1], w[BITS / 2 - 2], w[BITS / 2 - 1]);
    if ((c & 3u) == 0) {
      const int64_t g = pid * p.sb_str[0] + h * p.sb_str[1] + slot * p.sb_str[2] + (c >> 2);
      ((uint16_t*)p.s)[g] = f32_to_bf16_bits(scale);
      ((uint16_t*)p.b)[g] = f32_to_bf16_bits(bias);
    }
  }
}

// ---------------------------------------------------------------- freeing pages
// A block per listed sequence; the first of several entries that name the same sequence does the work.
__global__ void __launch_bounds__(256) pages_free_kernel(PageState st, const int32_t* rows, const int32_t* begin, const int32_t* end) {
  grid_wait();
  const int i = blockIdx.x, tid = threadIdx.x;
  const int r = rows[i];
  if (r < 0 || r >= st.S) return;
  bool again = false;
  for (int j = tid; j < i; j += 256) again |= rows[j] == r;
  if (__syncthreads_or(again)) return;
  const int64_t n = st.lens[r] > 0 ? st.lens[r] : 0;
  const int64_t b = begin ? (begin[i] > 0 ? begin[i] : 0) : 0;
  const int64_t e = end ? (end[i] < n ? (int64_t)end[i] : n) : n;
  const int64_t page = 1ll << st.page_shift;
  int64_t p1 = (n + page - 1) >> st.page_shift;
  p1 = p1 < st.M ? p1 : st.M;
  int32_t* row = st.table + (int64_t)r * st.table_str;
  for (int64_t p = ((b + page - 1) >> st.page_shift) + tid; p < p1; p += 256) {
    const int64_t stop = (p + 1) << st.page_shift;
    if ((stop < n ? stop : n) > e) break;
    const int32_t pid = row[p];
    if (pid < 0) continue;
    row[p] = -1;
    if (pid < st.P) atomicSub(st.refs + pid, 1);
  }
  __syncthreads();                       // (every thread has read the length)
  if (tid == 0 && e >= n && b < n) st.lens[r] = (int32_t)b;
}

// ---------------------------------------------------------------- one cluster for what has steps
// Forking, reserving and compacting each read the whole state before they change it.  One cluster of up to eight blocks does
// that in one launch with the hardware's barrier between the steps; a launch of one block is the same program.
constexpr int kPageThreads = 512;
constexpr int kStateBlocks = 8;      // one, two, four or eight blocks take the same for pools of 700 pages; 200,000 pages take 77, 49, 34, 26 us

__device__ __forceinline__ uint32_t ld_cluster_u32(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}
// Inclusive sum over the block of one value per thread; *total = the block's sum.
__device__ __forceinline__ int block_scan(int v, int* warp_sums, int* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += u;
  }
  if (lane == 31) warp_sums[warp] = v;
  __syncthreads();
  int before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kPageThreads / 32; ++w) {
    const int s = warp_sums[w];
    if (w < warp) before += s;
    all += s;
  }
  __syncthreads();
  *total = all;
  return v + before;
}

// The pages of this block's share of the pool as bits (bit set: refs == 0 where `free_bits`, else refs > 0), their exclusive
// counts per word within the share, and the counts of all blocks.  words: [w0, w1) of ceil(P / 32).
struct Share { int w0, w1, base, total; };
__device__ __forceinline__ Share page_bits(const PageState& st, bool free_bits, uint32_t* bits, int* pre, int* warp_sums, int* block_count) {
  const int nr = (int)cluster_size(), me = (int)cluster_rank();
  const int W = (st.P + 31) / 32, per = (W + nr - 1) / nr;
  Share sh;
  sh.w0 = per * me < W ? per * me : W;
  sh.w1 = sh.w0 + per < W ? sh.w0 + per : W;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, n = sh.w1 - sh.w0;
  constexpr int kWarpsHere = kPageThreads / 32, kBatch = 8;
  for (int w = warp * kBatch; w < n; w += kWarpsHere * kBatch) {
    int v[kBatch];
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      const int64_t page = (int64_t)(sh.w0 + w + k) * 32 + lane;
      v[k] = w + k < n && page < st.P ? st.refs[page] : (free_bits ? 1 : 0);
    }
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      const uint32_t m = __ballot_sync(0xffffffffu, free_bits ? v[k] == 0 : v[k] > 0);
      if (lane == 0 && w + k < n) bits[w + k] = m;
    }
  }
  __syncthreads();
  int run = 0;
  for (int w0 = 0; w0 < n; w0 += kPageThreads) {
    const int w = w0 + threadIdx.x, c = w < n ? __popc(bits[w]) : 0;
    int all;
    const int upto = block_scan(c, warp_sums, &all);
    if (w < n) pre[w] = run + upto - c;
    run += all;
  }
  if (threadIdx.x == 0) *block_count = run;
  cluster_sync_all();                    // counts are in place, and every block has read what it needs of refs
  const uint32_t addr = (uint32_t)__cvta_generic_to_shared(block_count);
  sh.base = 0; sh.total = 0;
  for (int r = 0; r < nr; ++r) {
    const int c = (int)ld_cluster_u32(map_to_rank(addr, (uint32_t)r));
    if (r < me) sh.base += c;
    sh.total += c;
  }
  return sh;
}

// ---- fork: sequence dst[i] begins with the first tokens[i] tokens (all, where null) of sequence src[i] ----
__global__ void __launch_bounds__(kPageThreads) pages_fork_kernel(PageState st, const int32_t* src, const int32_t* dst, const int32_t* tokens, int n, int32_t* shared) {
  extern __shared__ int sm[];
  int* s_dst = sm;          // [n]
  int* s_tok = sm + n;      // [n]: tokens shared, -1 = refused
  const int tid = threadIdx.x;
  grid_wait();
  for (int i = tid; i < n; i += kPageThreads) s_dst[i] = dst[i];
  __syncthreads();
  for (int i = tid; i < n; i += kPageThreads) {
    const int s = src[i], d = s_dst[i];
    int t = -1;
    if (s >= 0 && s < st.S && d >= 0 && d < st.S && s != d && st.lens[d] == 0) {
      t = st.lens[s] > 0 ? st.lens[s] : 0;
      if (tokens && tokens[i] < t) t = tokens[i] > 0 ? tokens[i] : 0;
      const int64_t cap = (int64_t)st.M << st.page_shift;
      if (t > cap) t = (int)cap;
      for (int j = 0; j < i; ++j)
        if (s_dst[j] == d) { t = -1; break; }
    }
    s_tok[i] = t;
  }
  cluster_sync_all();                    // every block has seen the state before the call
  // a warp takes up to 512 pages of an entry at a time
  constexpr int kChunk = 512;
  const int nw = (int)cluster_size() * (kPageThreads / 32), w = (int)cluster_rank() * (kPageThreads / 32) + (tid >> 5), lane = tid & 31;
  const int chunks = (st.M + kChunk - 1) / kChunk > 0 ? (st.M + kChunk - 1) / kChunk : 1;
  for (int item = w; item < n * chunks; item += nw) {
    const int i = item / chunks, c = item - i * chunks, t = s_tok[i];
    const int np = t > 0 ? (int)(((int64_t)t + (1 << st.page_shift) - 1) >> st.page_shift) : 0;
    const int stop = np < (c + 1) * kChunk ? np : (c + 1) * kChunk;
    if (c * kChunk < stop) {
      const int32_t* from = st.table + (int64_t)src[i] * st.table_str;
      int32_t* to = st.table + (int64_t)s_dst[i] * st.table_str;
#pragma unroll 4
      for (int p = c * kChunk + lane; p < stop; p += 32) {
        const int32_t pid = from[p];
        to[p] = pid;
        if (pid >= 0 && pid < st.P) atomicAdd(st.refs + pid, 1);
      }
    }
    if (c == 0 && lane == 0) {
      if (t > 0) st.lens[s_dst[i]] = t;
      shared[i] = t;
    }
  }
}

// ---- reserve: room for counts[i] more tokens in sequence rows[i] ----
// The k-th page that the list asks for is the k-th free page of the pool in ascending order: a prefix sum over the list, one over
// the free pages, and each free page finds by bisection whose it is.
__global__ void __launch_bounds__(kPageThreads) pages_reserve_kernel(PageState st, const int32_t* rows, const int32_t* counts, int n, int32_t* positions,
                                                                     int32_t* copies, int bit_words) {
  extern __shared__ int sm[];
  uint32_t* bits = (uint32_t*)sm;             // [bit_words]
  int* pre = sm + bit_words;                  // [bit_words]
  int* s_row = pre + bit_words;               // [n]
  int* s_len = s_row + n;                     // [n], -1: refused
  int* s_cnt = s_len + n;                     // [n]
  int* s_first = s_cnt + n;                   // [n]: rank of the entry's first fresh page
  int* s_col = s_first + n;                   // [n]: column of that page, negative (~column) where the page before is copied to it
  __shared__ int warp_sums[kPageThreads / 32];
  __shared__ int block_count;
  const int tid = threadIdx.x;
  const int64_t page = 1ll << st.page_shift;
  grid_wait();
  for (int i = tid; i < n; i += kPageThreads) s_row[i] = rows[i];
  __syncthreads();
  int run = 0;
  for (int i0 = 0; i0 < n; i0 += kPageThreads) {
    const int i = i0 + tid;
    int need = 0;
    if (i < n) {
      const int r = s_row[i], c = counts[i];
      int len = -1, col = 0;
      if (r >= 0 && r < st.S && c >= 0) {
        len = st.lens[r] > 0 ? st.lens[r] : 0;
        if ((int64_t)len + c > (int64_t)st.M * page || (int64_t)len + c > 0x7fffffff) len = -1;
        for (int j = 0; j < i && len >= 0; ++j)
          if (s_row[j] == r) len = -1;
      }
      if (len >= 0 && c > 0) {
        const int have = (int)(((int64_t)len + page - 1) >> st.page_shift), want = (int)(((int64_t)len + c + page - 1) >> st.page_shift);
        need = want - have;
        col = have;
        if (len & (page - 1)) {
          const int32_t last = st.table[(int64_t)r * st.table_str + have - 1];
          const bool none = last < 0 || last >= st.P;
          if (none || st.refs[last] > 1) {      // no page there, or one that others read: a fresh one takes its place
            ++need;
            col = none ? have - 1 : ~(have - 1);
          }
        }
        // (an entry that asks for more pages than there are is refused by one too many as well, and so 2048 of them stay below 2^31)
        need = need < st.P + 1 ? need : st.P + 1;
      }
      s_len[i] = len; s_cnt[i] = c; s_col[i] = col;
    }
    int all;
    const int upto = block_scan(need, warp_sums, &all);
    if (i < n) s_first[i] = run + upto - need;
    run += all;
  }
  const int total = run;
  const Share sh = page_bits(st, true, bits, pre, warp_sums, &block_count);   // (a barrier of the cluster inside: the state has been read)
  auto fresh_of = [&](int i) { return (i + 1 < n ? s_first[i + 1] : total) - s_first[i]; };
  auto served = [&](int i) { const int f = fresh_of(i); return s_len[i] >= 0 && (f == 0 || s_first[i] + f <= sh.total); };
  const int lane = tid & 31, warp = tid >> 5;
  for (int w = warp; w < sh.w1 - sh.w0; w += kPageThreads / 32) {
    const int rank0 = sh.base + pre[w];
    if (rank0 >= total) break;
    const uint32_t m = bits[w];
    const int rank = rank0 + __popc(m & ((1u << lane) - 1u));
    if (!((m >> lane) & 1u) || rank >= total) continue;
    int lo = 0, hi = n - 1;              // the last entry whose first rank is <= rank: it owns the page
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (s_first[mid] <= rank) lo = mid; else hi = mid - 1;
    }
    if (!served(lo)) continue;
    const int32_t pid = (sh.w0 + w) * 32 + lane;
    const bool copy = s_col[lo] < 0;
    const int k = rank - s_first[lo], col = (copy ? ~s_col[lo] : s_col[lo]) + k;
    int32_t* e = st.table + (int64_t)s_row[lo] * st.table_str + col;
    if (copy && k == 0) {
      const int32_t old = *e;
      copies[2 * lo] = old;
      copies[2 * lo + 1] = pid;
      atomicSub(st.refs + old, 1);
    }
    *e = pid;
    st.refs[pid] = 1;
  }
  if (cluster_rank() == 0)
    for (int i = tid; i < n; i += kPageThreads) {
      const bool ok = served(i);
      positions[i] = ok ? s_len[i] : -1;
      if (ok && s_cnt[i] > 0) st.lens[s_row[i]] = s_len[i] + s_cnt[i];
      if (!(ok && s_col[i] < 0)) { copies[2 * i] = -1; copies[2 * i + 1] = -1; }
    }
  cluster_sync_all();                    // (shared memory that others read stays until they have)
}

// ---- compact: the live pages behind the first `live` ones move into the holes before them, k-th into k-th ----
__global__ void __launch_bounds__(kPageThreads) pages_compact_kernel(PageState st, int32_t* remap, int32_t* moves, int64_t cap, int32_t* count, int bit_words) {
  extern __shared__ int sm[];
  uint32_t* bits = (uint32_t*)sm;
  int* pre = sm + bit_words;
  __shared__ int warp_sums[kPageThreads / 32];
  __shared__ int block_count, in_front;
  const int nr = (int)cluster_size(), me = (int)cluster_rank(), tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  grid_wait();
  const Share sh = page_bits(st, false, bits, pre, warp_sums, &block_count);
  const int live = sh.total;
  // how many of the first `live` pages are live: the block that holds page `live` knows, and tells the others
  const int wl = live >> 5;
  if (tid == 0 && ((wl >= sh.w0 && wl < sh.w1) || (me == 0 && wl >= (st.P + 31) / 32))) {
    const int v = wl >= (st.P + 31) / 32 ? live : sh.base + pre[wl - sh.w0] + __popc(bits[wl - sh.w0] & ((1u << (live & 31)) - 1u));
    for (int r = 0; r < nr; ++r)
      asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(map_to_rank((uint32_t)__cvta_generic_to_shared(&in_front), (uint32_t)r)), "r"(v) : "memory");
  }
  cluster_sync_all();
  const int front = in_front, num = live - front;
  for (int w = warp; w < sh.w1 - sh.w0; w += kPageThreads / 32) {
    const int id = (sh.w0 + w) * 32 + lane;
    if (id >= st.P) continue;
    const bool is_live = (bits[w] >> lane) & 1u;
    const int before = sh.base + pre[w] + __popc(bits[w] & ((1u << lane) - 1u));
    if (id < live && !is_live) moves[2 * (int64_t)(id - before) + 1] = id;
    if (id >= live && is_live) moves[2 * (int64_t)(before - front)] = id;
    else remap[id] = is_live ? id : -1;
  }
  for (int64_t k = num + (int64_t)me * kPageThreads + tid; k < cap; k += (int64_t)nr * kPageThreads) { moves[2 * k] = -1; moves[2 * k + 1] = -1; }
  if (me == 0 && tid == 0) *count = num;
  cluster_sync_all();
  for (int k = me * kPageThreads + tid; k < num; k += nr * kPageThreads) {
    const int2 mv = __ldcg((const int2*)moves + k);
    remap[mv.x] = mv.y;
    st.refs[mv.y] = st.refs[mv.x];
    st.refs[mv.x] = 0;
  }
}

// The table's entries become what remap says: a launch of its own over the whole device, a warp 512 entries of a sequence at a time, all
// asked for at once.  (By the cluster itself, behind its other steps, 1024 x 2048 entries took 104 us in all, so 55; 24 x 128 take 11 either way.)
constexpr int kRemapChunk = 512;
__global__ void __launch_bounds__(256) pages_remap_kernel(PageState st, const int32_t* remap, int chunks) {
  grid_wait();
  const int lane = threadIdx.x & 31;
  const int64_t items = (int64_t)st.S * chunks;
  for (int64_t item = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); item < items; item += (int64_t)gridDim.x * 8) {
    const int64_t s = item / chunks;
    const int p0 = (int)(item - s * chunks) * kRemapChunk + lane;
    int32_t* row = st.table + s * st.table_str;
    int32_t pid[kRemapChunk / 32], to[kRemapChunk / 32];
#pragma unroll
    for (int k = 0; k < kRemapChunk / 32; ++k) pid[k] = p0 + k * 32 < st.M ? row[p0 + k * 32] : -1;
#pragma unroll
    for (int k = 0; k < kRemapChunk / 32; ++k) to[k] = pid[k] < 0 ? pid[k] : (pid[k] < st.P ? remap[pid[k]] : -1);
#pragma unroll
    for (int k = 0; k < kRemapChunk / 32; ++k)
      if (to[k] != pid[k]) row[p0 + k * 32] = to[k];
  }
}

// ---------------------------------------------------------------- copying pages
// Pair by pair, pool by pool, in pieces that a warp copies with four vectors a lane: pages of codes have many, those of scales one or
// two, and no warp waits for another's.  Bound by HBM: 336 MB of moved pages, read and written, take 105 us, 6.4 TB/s (pieces of 1024, 8192
// and 16384 bytes: 158, 150, 160 us).
constexpr int kCopyPiece = 2048;

template <typename V, int N>
__global__ void __launch_bounds__(256) pages_copy_kernel(const __grid_constant__ PagesCopyList<N> a) {
  grid_wait();
  const int64_t n = a.count ? min((int64_t)(*a.count > 0 ? *a.count : 0), a.n) : a.n;
  const int64_t work = n * a.pieces;
  const int lane = threadIdx.x & 31;
  for (int64_t w = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); w < work; w += (int64_t)gridDim.x * 8) {
    const int64_t pair = work <= 0x7fffffff ? (int64_t)((uint32_t)w / (uint32_t)a.pieces) : w / a.pieces;
    const int piece = (int)(w - pair * a.pieces);
    const int64_t src = a.pairs[2 * pair], dst = a.pairs[2 * pair + 1];
    if (src < 0 || src >= a.P || dst < 0 || dst >= a.P || src == dst) continue;
    int lo = 0, hi = a.pools - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (a.pool[mid].first_piece <= piece) lo = mid; else hi = mid - 1;
    }
    const PagesCopyPool& p = a.pool[lo];
    const char* from = p.base + src * p.page_str;
    char* to = p.base + dst * p.page_str;
    const uint32_t at = (uint32_t)(piece - p.first_piece) * kCopyPiece, left = p.bytes - at;
    constexpr int kVecs = kCopyPiece / 32 / (int)sizeof(V);
    constexpr int kBatch = kVecs < 8 ? kVecs : 8;
#pragma unroll 1
    for (int k0 = 0; k0 < kVecs; k0 += kBatch) {
      V v[kBatch];
      int64_t off[kBatch];
#pragma unroll
      for (int k = 0; k < kBatch; ++k) {
        const uint32_t o = ((k0 + k) * 32 + lane) * (uint32_t)sizeof(V);
        off[k] = -1;
        if (o < left) {
          uint32_t e = at + o;
          if (p.run == p.bytes) off[k] = e;
          else {
            const uint32_t run = e / p.run, x = e - run * p.run, hh = run / p.inner;
            off[k] = (int64_t)hh * p.outer_str + (int64_t)(run - hh * p.inner) * p.inner_str + x;
          }
          v[k] = *(const V*)(from + off[k]);
        }
      }
#pragma unroll
      for (int k = 0; k < kBatch; ++k)
        if (off[k] >= 0) *(V*)(to + off[k]) = v[k];
    }
  }
}

// ---------------------------------------------------------------- the nodes of drafted trees that stay
// The walk: from node 0 to the first child that carries the token sampled behind it, and on from there.  A warp holds the tree, two nodes
// a lane, and finds a child with two ballots; every block walks again, so that one launch does it all.  A path's nodes ascend and stand
// at or behind the places they go to, path[i] >= i: taken in ascending order, no row is overwritten that is still to be read, and a
// thread's column of a row (16 bytes of one head in one pool) needs no other thread.  Eight rows are asked for at a time.
// Bound by the launch and two dependent reads: 4 trees of eight over two layers 10 us a call, 16 trees over more layers 15 (their rows alone 0.5).
template <typename V, int N>
__global__ void __launch_bounds__(256) pages_accept_kernel(const __grid_constant__ PagesAcceptList<N> a) {
  __shared__ int s_path[kMaxNodes], s_pid[kMaxNodes + 1][2], s_n;   // of a place: its page and the page of the node that goes there
  grid_wait();
  const int b = (int)(blockIdx.x / (unsigned)a.blocks), part = (int)(blockIdx.x - (unsigned)b * (unsigned)a.blocks), tid = threadIdx.x;
  const int64_t row = a.rows ? a.rows[b] : (int64_t)b;
  const bool known = row >= 0 && row < a.seqs;
  int64_t len = known ? a.lens[row] : 0;
  const int64_t cap = (int64_t)a.M << a.page_shift;
  len = len < 0 ? 0 : (len > cap ? cap : len);
  bool again = false;                                  // (a sequence listed before: its rows move once)
  if (a.rows)
    for (int j = tid; j < b; j += 256) again |= a.rows[j] == row;
  again = __syncthreads_or(again);
  int64_t n64 = a.counts ? a.counts[b] : a.T;
  n64 = n64 < 0 ? 0 : (n64 > a.T ? a.T : n64);
  const int n = again ? 0 : (int)(n64 > len ? len : n64);
  const int64_t base = len - n;
  if (tid < 32) {
    int parent[2], token[2], behind[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int i = tid + 32 * h;
      parent[h] = -1; token[h] = 0; behind[h] = 0;
      if (i < n) {
        parent[h] = a.lists[0][b * a.list_str[0] + i];
        token[h] = a.lists[1][b * a.list_str[1] + i];
        behind[h] = a.lists[2][b * a.list_str[2] + i];
      }
      if (parent[h] >= i) parent[h] = -1;              // (no parent stands at its node or behind it)
    }
    int at = 0, len_path = 0;
    while (len_path < n) {                             // (nodes ascend: at most n steps)
      const int want = __shfl_sync(0xffffffffu, at & 32 ? behind[1] : behind[0], at & 31);
      if (tid == 0) s_path[len_path] = at;
      if (part == 0 && a.path != nullptr && tid == 0) { a.path[(int64_t)b * a.T + len_path] = at; a.next[(int64_t)b * a.T + len_path] = want; }
      ++len_path;
      const uint32_t lo = __ballot_sync(0xffffffffu, parent[0] == at && token[0] == want), hi = __ballot_sync(0xffffffffu, parent[1] == at && token[1] == want);
      if ((lo | hi) == 0) break;
      at = lo ? __ffs(lo) - 1 : 31 + __ffs(hi);
    }
    if (part == 0 && a.path != nullptr) {
      for (int i = len_path + tid; i < a.T; i += 32) { a.path[(int64_t)b * a.T + i] = -1; a.next[(int64_t)b * a.T + i] = -1; }
      if (tid == 0) { a.accepted[b] = len_path; a.ends[b] = (int32_t)(base + len_path); }
    }
    __syncwarp();
    const int32_t* const tab = a.table + row * a.table_str;
    for (int i = tid; i < len_path; i += 32) {
      const int64_t to = base + i, from = base + s_path[i];
      int p0 = tab[to >> a.page_shift], p1 = tab[from >> a.page_shift];
      if (p0 >= a.P) p0 = -1;
      if (p1 >= a.P) p1 = -1;
      s_pid[i][0] = p0; s_pid[i][1] = from == to ? -1 : p1;
    }
    if (tid == 0) s_n = len_path;
  }
  __syncthreads();
  const int rows = s_n;
  const int mask = (1 << a.page_shift) - 1;
  for (int c = part * 256 + tid; c < a.cols; c += a.blocks * 256) {
    int lo = 0, hi = a.pools - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (a.pool[mid].first <= c) lo = mid; else hi = mid - 1;
    }
    const AcceptPool& p = a.pool[lo];
    const int in = c - p.first, head = in / p.vecs;
    char* const column = p.base + (int64_t)head * p.head_str + (int64_t)(in - head * p.vecs) * (int64_t)sizeof(V);
#pragma unroll 1
    for (int i0 = 0; i0 < rows; i0 += 8) {
      V v[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int i = i0 + k;
        if (i < rows && s_pid[i][0] >= 0 && s_pid[i][1] >= 0)
          v[k] = *(const V*)(column + (int64_t)s_pid[i][1] * p.page_str + ((base + s_path[i]) & mask) * p.tok_str);
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int i = i0 + k;
        if (i < rows && s_pid[i][0] >= 0 && s_pid[i][1] >= 0) *(V*)(column + (int64_t)s_pid[i][0] * p.page_str + ((base + i) & mask) * p.tok_str) = v[k];
      }
    }
  }
}

// The kernel may take kPageSmem bytes on the current device: set once for each, whatever the first call needs (without it a launch has
// 48 KB less what the kernel holds statically).
template <auto KERN>
cudaError_t allow_page_smem() {
  static bool done[64] = {};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  std::lock_guard<std::mutex> setup_lk(setup_mutex());       // first use on a device, from any thread
  if (dev >= 0 && dev < 64 && done[dev]) return cudaSuccess;
  e = cudaFuncSetAttribute(KERN, cudaFuncAttributeMaxDynamicSharedMemorySize, kPageSmem);
  if (e == cudaSuccess && dev >= 0 && dev < 64) done[dev] = true;
  return e;
}

template <auto KERN, typename... A>
cudaError_t launch_page_cluster(int want, size_t smem, cudaStream_t st, A... args) {
  constexpr auto kern = KERN;
  const cudaError_t ready = allow_page_smem<KERN>();
  if (ready != cudaSuccess) return ready;
  if (want > 1) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)want);
    cfg.blockDim = dim3(kPageThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)want; attr[1].val.clusterDim.y = 1; attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    const cudaError_t e = launch_clusters(cfg, kern, args...);
    if (e == cudaSuccess) return e;
    (void)cudaGetLastError();            // the device places no clusters: one block does it
  }
  return launch_behind(kern, dim3(1), dim3(kPageThreads), smem, st, args...);
}
int bit_words(int64_t P, int blocks) { return (int)(((P + 31) / 32 + blocks - 1) / blocks); }
}  // namespace

cudaError_t launch_pages_append(const KvPagesAppendArgs& a, cudaStream_t st) {
  const int64_t head = (int64_t)a.S * a.per_row;             // threads that the rows of a head take
  const int block = head >= 256 ? 256 : (int)((head + 31) / 32 * 32);
  KvPagesAppendArgs k = a;
  k.tiles = (int)((head + block - 1) / block);
  k.row_shift = -1;
  for (int i = 0; i < 16; ++i)
    if (a.per_row == 1 << i) k.row_shift = i;
  auto kern = a.bits == 4 ? pages_append_kernel<4> : (a.bits == 8 ? pages_append_kernel<8> : pages_append_kernel<16>);
  return launch_behind(kern, dim3((unsigned)((int64_t)k.tiles * a.N * 2 * a.H)), dim3((unsigned)block), 0, st, k);
}
cudaError_t launch_pages_free(const PageState& s, const int32_t* rows, const int32_t* begin, const int32_t* end, int n, cudaStream_t st) {
  return launch_behind(pages_free_kernel, dim3((unsigned)n), dim3(256), 0, st, s, rows, begin, end);
}
// One block's bits take 2 words per 32 pages and the list five: both fit where kMaxPages and kMaxPageList hold.
cudaError_t launch_pages_fork(const PageState& s, const int32_t* src, const int32_t* dst, const int32_t* tokens, int n, int32_t* shared, cudaStream_t st) {
  return launch_page_cluster<pages_fork_kernel>(kStateBlocks, (size_t)n * 8, st, s, src, dst, tokens, n, shared);
}
cudaError_t launch_pages_reserve(const PageState& s, const int32_t* rows, const int32_t* counts, int n, int32_t* positions, int32_t* copies, cudaStream_t st) {
  const int bw = bit_words(s.P, 1);
  return launch_page_cluster<pages_reserve_kernel>(kStateBlocks, (size_t)bw * 8 + (size_t)n * 20, st, s, rows, counts, n, positions, copies, bw);
}
cudaError_t launch_pages_compact(const PageState& s, int32_t* remap, int32_t* moves, int64_t cap, int32_t* count, cudaStream_t st) {
  const int bw = bit_words(s.P, 1);
  const cudaError_t e = launch_page_cluster<pages_compact_kernel>(kStateBlocks, (size_t)bw * 8, st, s, remap, moves, cap, count, bw);
  if (e != cudaSuccess || s.S == 0 || s.M == 0) return e;
  const int chunks = (s.M - 1) / kRemapChunk + 1;
  const int64_t blocks = ((int64_t)s.S * chunks + 7) / 8, most = (int64_t)sm_count() * 4;
  return launch_behind(pages_remap_kernel, dim3((unsigned)(blocks < most ? blocks : most)), dim3(256), 0, st, s, remap, chunks);
}
template <int N> cudaError_t launch_copy(const PagesCopyArgs& a, int vec, cudaStream_t st) {
  PagesCopyList<N> k;
  k.pairs = a.pairs; k.count = a.count; k.n = a.n; k.P = a.P; k.pools = a.pools; k.pieces = a.pieces;
  std::memcpy(k.pool, a.pool, sizeof(PagesCopyPool) * (size_t)a.pools);
  const int64_t work = (a.n * a.pieces + 7) / 8, most = (int64_t)sm_count() * 8;   // eight warps a block
  const dim3 grid((unsigned)(work < most ? work : most));
  switch (vec) {
    case 16: return launch_behind(pages_copy_kernel<uint4, N>, grid, dim3(256), 0, st, k);
    case 4: return launch_behind(pages_copy_kernel<uint32_t, N>, grid, dim3(256), 0, st, k);
    case 2: return launch_behind(pages_copy_kernel<uint16_t, N>, grid, dim3(256), 0, st, k);
    default: return launch_behind(pages_copy_kernel<uint8_t, N>, grid, dim3(256), 0, st, k);
  }
}
// (4.6 KB of arguments cost the host 3.5 us a launch, 0.6 KB 2.6.)
cudaError_t launch_pages_copy(const PagesCopyArgs& a, int vec, cudaStream_t st) {
  return a.pools <= 12 ? launch_copy<12>(a, vec, st) : launch_copy<kMaxCopyPools>(a, vec, st);
}
int pages_copy_piece() { return kCopyPiece; }

template <int N> cudaError_t launch_accept(const PagesAcceptArgs& a, int vec, cudaStream_t st) {
  PagesAcceptList<N> k;
  std::memcpy((void*)&k, (const void*)&a, offsetof(PagesAcceptArgs, pool));
  std::memcpy(k.pool, a.pool, sizeof(AcceptPool) * (size_t)a.pools);
  // blocks a sequence: a column a thread, as far as the device has room for at once
  const int64_t need = ((int64_t)a.cols + 255) / 256, most = (int64_t)sm_count() * 8 / a.B;
  k.blocks = (int)(need < 1 ? 1 : (need < most ? need : (most < 1 ? 1 : most)));
  const dim3 grid((unsigned)((int64_t)k.blocks * a.B));
  switch (vec) {
    case 16: return launch_behind(pages_accept_kernel<uint4, N>, grid, dim3(256), 0, st, k);
    case 4: return launch_behind(pages_accept_kernel<uint32_t, N>, grid, dim3(256), 0, st, k);
    case 2: return launch_behind(pages_accept_kernel<uint16_t, N>, grid, dim3(256), 0, st, k);
    default: return launch_behind(pages_accept_kernel<uint8_t, N>, grid, dim3(256), 0, st, k);
  }
}
cudaError_t launch_pages_accept(const PagesAcceptArgs& a, int vec, cudaStream_t st) {
  return a.pools <= 12 ? launch_accept<12>(a, vec, st) : launch_accept<kMaxCopyPools>(a, vec, st);
}

}  // namespace qb
