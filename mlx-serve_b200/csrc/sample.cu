// A token from every row of logits: temperature, top-k, top-p and min-p, with a random number given for the row.
//
// With m the row's largest logit, w_i = exp((l_i - m) / temperature) and the order "larger logit first, then lower index": the first k
// of the order stay; of these the shortest prefix whose weights reach p of their sum; of these those with w_i >= min_p; the token is the
// first one in index order at which the running sum of the weights that stay passes u times their sum.
//
//  * Weights are whole numbers, round(w_i * 2^44), of a 64-bit exponential: sums of them do not depend on the order in which threads
//    or atomics run, and borders (the nucleus, the token) are met as 64-bit sums meet them, but for the rounding: 2^-45 of the largest for each
//    weight.  2^19 of them fit 63 bits; a token below 2^-45 of the largest counts as 0.
//  * A row is a cluster of up to eight blocks, each with a share of the row in shared memory (read from memory again where it is too
//    large); sums and histograms meet through distributed shared memory.
//  * By temperature alone a row is read once, in parts of 512 elements that a warp weighs relative to its own largest logit in 32 bits, with a bound on how far
//    such a sum may be off; the part where the token lies, and the parts beside it that the bound leaves open, are summed exactly.  Where the bound
//    leaves too much open, all of the row is.
//  * The border of top-k and top-p in the order: a histogram of how far the logits lie below the largest, 4096 steps over 32 temperatures, says in which step it
//    lies (top-k exactly; top-p by the steps' mean weights, and the sums of the next pass say whether that was right).  The logits of
//    these steps go to a list in the first block, by 1024 slots along the order, and those of one slot look at one another.  Few that stay are drawn from that list alone.  Where the list
//    would be too long (equal logits, flat rows) the border is found by halving the range of the logits' patterns, a sum over the row each time.
//
// Measured: one row of 128256 with top-k 50 and top-p 0.95 18.6 us (meetings of its eight blocks and the work on a list, one after the other); 256 rows of
// 32001 (fp32) with filters of all kinds 70 us, where reading them once takes 5; 24 rows with a nucleus of flat logits 57, or 69 to 78 where one of them is left
// open by the fp32 weights; 256 rows of 262144 by temperature alone 111 us, 1.2 TB/s: instructions bound it (30 a warp for 32 logits), not the memory.  256 rows
// of 128256 in bf16, behind a write of 256 MB: 115 us with top-k 50 and top-p 0.95, 289 with top-p alone, 33 greedy.
// The 64 registers that two blocks an SM leave a thread do not hold everything: -Xptxas -v reports 128 to 144 bytes of spill stores, 128 to 140 of loads.
#include <cstddef>
#include <mutex>
#include <type_traits>

#include "kernels.h"
#include "stream_ptx.cuh"

namespace qb {
namespace {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kBins = 4096;
constexpr float kRange = 32.f;                 // temperatures below the largest that the bins cover: e^-32 < 2^-45
constexpr int kList = 2048;
constexpr int kSlots = 1024;                   // of a list's entries, by where they stand in an order
constexpr int kPairs = 128;                    // entries of a slot that are compared pair by pair
constexpr double kOne = 17592186044416.0;      // 2^44
constexpr int kMaxCtas = 8;
constexpr int kDeep = 2;                       // vectors of eight elements a lane has of a warp's part of a row
constexpr int kMaxParts = kMaxVocab / (32 * 8 * kDeep) + 2;

// larger patterns for larger floats (no NaN, no -0 comes here)
__device__ __forceinline__ uint32_t pattern(float x) {
  const uint32_t b = __float_as_uint(x);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }
__device__ __forceinline__ float clean(float x) { return x == x ? x + 0.f : -INFINITY; }   // (a NaN counts as masked; -0 as 0)

__device__ __forceinline__ uint64_t warp_sum(uint64_t v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ void put64(uint64_t* p, uint32_t rank, uint64_t v) {
  asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(map_to_rank(smem_u32(p), rank)), "l"(v) : "memory");
}
__device__ __forceinline__ void put32(void* p, uint32_t rank, uint32_t v) {
  asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(map_to_rank(smem_u32(p), rank)), "r"(v) : "memory");
}
__device__ __forceinline__ uint32_t get32(const void* p, uint32_t rank) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(map_to_rank(smem_u32(p), rank)) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t add32(void* p, uint32_t rank, uint32_t v) {
  uint32_t r;
  asm volatile("atom.shared::cluster.add.u32 %0, [%1], %2;" : "=r"(r) : "r"(map_to_rank(smem_u32(p), rank)), "r"(v) : "memory");
  return r;
}

// 2^(i / 32)
__constant__ double kRoots[32] = {
    1.0, 1.0218971486541166, 1.0442737824274138, 1.0671404006768237,
    1.0905077326652577, 1.1143867425958924, 1.1387886347566916, 1.1637248587775775,
    1.189207115002721, 1.215247359980469, 1.241857812073484, 1.2690509571917332,
    1.2968395546510096, 1.3252366431597413, 1.3542555469368927, 1.383909881963832,
    1.4142135623730951, 1.4451808069770467, 1.4768261459394993, 1.5091644275934228,
    1.5422108254079407, 1.5759808451078865, 1.6104903319492543, 1.645755478153965,
    1.681792830507429, 1.718619298122478, 1.7562521603732995, 1.7947090750031072,
    1.8340080864093424, 1.8741676341103, 1.9152065613971474, 1.9571441241754002};
// round(2^44 * 2^(d * c / 32)) for d <= 0, c > 0: d c = 32 n + i + f with |f| <= 1/2 (the nearest whole number by adding 1.5 * 2^52), 2^(f / 32)
// as its series to f^5 (the next term is below 2.3e-15), 2^(i / 32) from a table, 2^n into the exponent, the whole number out of the low bits of a
// sum with 2^52.  What lies below 2^-46.9, or is no number, counts as that, which rounds to 0.
__device__ __forceinline__ uint64_t weight64(double d, double c, const double* roots) {
  const double t = fmax(d * c, -46.9 * 32.0);
  const double shifted = t + 6755399441055744.0, f = t - (shifted - 6755399441055744.0);
  const int n = __double2loint(shifted);
  double y = fma(f, 3.973709984549416e-11, 9.172562701824643e-09);
  y = fma(y, f, 1.693850972437182e-06);
  y = fma(y, f, 0.0002345961982022468);
  y = fma(y, f, 0.02166084939249829);
  const double root = roots[n & 31];
  y = fma(y * f, root, root);
  const double w = __hiloint2double(__double2hiint(y) + (((n >> 5) + 44) << 20), __double2loint(y));
  return (uint64_t)__double_as_longlong(w + 4503599627370496.0) & 0xfffffffffffffull;
}

// What stays: everything in front of (key, index) in the order, and that itself.
struct Border { uint32_t key; int index; };

struct alignas(16) Shared {
  uint64_t gather[2][kMaxCtas];                // a value of every block; two, taken in turn
  uint64_t red[kWarps];
  double red_d[kWarps];
  double part[kMaxCtas], part_top[kMaxCtas];   // of the sum for the log-probability: a block's sum and its largest
  double once_sum[kMaxCtas];
  double far[kMaxCtas];                        // a block's sum of weights times how far their logits lie from the reference, or a bound of it
  double roots[32];
  union {                                      // (never of use at the same time)
    uint32_t hist[kBins];
    uint64_t list[kList];                      // pattern, then V - 1 - index: larger ones come first in the order
    uint64_t sums[kMaxParts];                  // of every warp's part
  };
  union {
    uint32_t merged[kBins];
    float refs[kMaxParts];                     // of the parts: what their sums are relative to
  };
  struct {
    uint64_t mass[kSlots], order[kPairs], weight[kPairs], before;
    uint32_t members;
    int slot, found;
  } slots;
  uint32_t scan[kWarps];
  uint32_t listed, staged, place;
  int answer[4], range[4];
};
static_assert(sizeof(Shared) % 16 == 0, "vectors behind it");

template <typename T> struct Row {
  static constexpr int W = (int)sizeof(T) / 2;   // 16-byte vectors of eight elements
  const T* x;                  // this block's share
  const unsigned char* held;   // the same in shared memory, cleaned, element e of it at place e + off; null: read from memory
  int begin, n, off, vecs;
  struct Raw { uint4 w[W]; };
  // eight elements from place 8 v on; -inf where the row has none
  __device__ __forceinline__ Raw load_raw(int v) const {
    const int i0 = 8 * v - off;
    Raw r;
    if (i0 >= 0 && i0 + 8 <= n) {
#pragma unroll
      for (int q = 0; q < W; ++q) r.w[q] = ((const uint4*)(x + i0))[q];
    } else {
      alignas(16) T e8[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) e8[e] = i0 + e >= 0 && i0 + e < n ? x[i0 + e] : (T)(-INFINITY);
#pragma unroll
      for (int q = 0; q < W; ++q) r.w[q] = ((const uint4*)e8)[q];
    }
    return r;
  }
  __device__ __forceinline__ static void unpack(const Raw& r, float (&f)[8]) {
#pragma unroll
    for (int q = 0; q < W; ++q) {
      const uint32_t w[4] = {r.w[q].x, r.w[q].y, r.w[q].z, r.w[q].w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if constexpr (sizeof(T) == 4) f[4 * q + k] = __uint_as_float(w[k]);
        else if constexpr (std::is_same<T, __half>::value) {
          const float2 h = __half22float2(*(const __half2*)&w[k]);
          f[2 * k] = h.x; f[2 * k + 1] = h.y;
        } else { f[2 * k] = bf16lo(w[k]); f[2 * k + 1] = bf16hi(w[k]); }
      }
    }
  }
  __device__ __forceinline__ void load8(int v, float (&f)[8]) const {
    Raw r;
    if (held) {
#pragma unroll
      for (int q = 0; q < W; ++q) r.w[q] = *(const uint4*)(held + v * (16 * W) + 16 * q);
      unpack(r, f);
    } else {
      unpack(load_raw(v), f);
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] = clean(f[e]);
    }
  }
  __device__ __forceinline__ int index(int v, int e) const { return begin + 8 * v + e - off; }
};

template <typename T>
__global__ void __launch_bounds__(kThreads, 2) sample_kernel(const __grid_constant__ SampleArgs a, int share, int held_bytes) {
  constexpr int DEEP = kDeep;
  constexpr float kLog2e = 1.4426950408889634f;
  extern __shared__ __align__(16) unsigned char raw[];
  Shared& sh = *(Shared*)raw;
  const uint32_t C = cluster_size(), me = cluster_rank();
  // A block's shared memory may be written by the others once it runs: all say so here, and wait for it before the first value that goes to another
  // block, behind the reading of the row (every block and thread does both, whatever its row asks for).
  cluster_arrive();
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int row_no = (int)(blockIdx.x / C), tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, V = a.V;
  const float temp = a.temperature ? a.temperature[row_no * a.str[1]] : 1.f, u = a.random[row_no * a.str[0]];
  const int k = a.top_k ? a.top_k[row_no * a.str[2]] : 0;
  const float p = a.top_p ? a.top_p[row_no * a.str[3]] : 1.f, least = a.min_p ? a.min_p[row_no * a.str[4]] : 0.f;

  Row<T> r;
  r.begin = (int)me * share < V ? (int)me * share : V;
  r.n = V - r.begin < share ? V - r.begin : share;
  r.x = (const T*)((const char*)a.logits + (int64_t)row_no * a.row_bytes) + r.begin;
  r.off = (int)((uintptr_t)r.x & (8 * sizeof(T) - 1)) / (int)sizeof(T);
  r.vecs = (r.n + r.off + 7) / 8;
  r.held = nullptr;
  const int parts = (r.vecs + 32 * DEEP - 1) / (32 * DEEP);
  unsigned char* const held = raw + sizeof(Shared);
  const bool greedy = !(temp > 0.f), by_k = k > 0 && k < V, by_p = p < 1.f;
  // by temperature alone the row is read once, its parts weighed relative to a largest of their own
  const bool once = !greedy && !by_k && !by_p && !(least > 0.f) && temp >= 1e-6f && temp <= 1e6f;
  const bool hold = !greedy && !once && r.vecs * 8 * (int)sizeof(T) <= held_bytes;
  if (tid == 0) sh.listed = sh.staged = 0;
  if (tid < 32) sh.roots[tid] = kRoots[tid];

  int turn = 0;
  // a value of every block, in all blocks
  auto gather = [&](uint64_t mine) {
    uint64_t* const g = sh.gather[turn];
    turn ^= 1;
    if (tid < (int)C) put64(&g[me], (uint32_t)tid, mine);
    cluster_sync_all();
    return g;
  };
  auto block_sum = [&](uint64_t v) {
    v = warp_sum(v);
    __syncthreads();
    if (lane == 0) sh.red[warp] = v;
    __syncthreads();
    return warp_sum(lane < kWarps ? sh.red[lane] : (uint64_t)0);
  };
  auto block_sum_d = [&](double v) {
    v = warp_sum(v);
    __syncthreads();
    if (lane == 0) sh.red_d[warp] = v;
    __syncthreads();
    return warp_sum(lane < kWarps ? sh.red_d[lane] : 0.0);
  };
  // of a sum, and of how far its terms may be off, for all blocks behind the next meeting
  auto block_sums_d = [&](double v, double off) {
    v = warp_sum(v);
    off = warp_sum(off);
    __syncthreads();
    if (lane == 0) { sh.red_d[warp] = v; sh.red[warp] = (uint64_t)__double_as_longlong(off); }
    __syncthreads();
    off = warp_sum(lane < kWarps ? __longlong_as_double((long long)sh.red[lane]) : 0.0);
    if (tid < (int)C) put64((uint64_t*)&sh.far[me], (uint32_t)tid, (uint64_t)__double_as_longlong(off));
    return warp_sum(lane < kWarps ? sh.red_d[lane] : 0.0);
  };
  auto total = [&](uint64_t v) {
    const uint64_t* const g = gather(block_sum(v));
    uint64_t s = 0;
    for (uint32_t c = 0; c < C; ++c) s += g[c];
    return s;
  };
  const double per_t = 1.0 / (double)temp, c64 = 32.0 * 1.4426950408889634 * per_t, c_all = 1.4426950408889634 * per_t;
  const float ch = (float)c_all, cl = (float)(c_all - (double)ch);
  // Weights in fp32, relative to `largest`, from the approximate exponential (relative error 2^-22), whose argument, difference times factor, is carried
  // in two parts, and which is rounded once more with the second.  `exact`: with the rounding of the difference to fp32 in the second part too.
  auto weights32 = [&](auto exact, const float (&f)[8], float largest, float (&w)[8]) {
    // what lies further down weighs 0, as this does (several steps of fp32 below the largest, so that it is below it, however large that is)
    const float floor_f = largest - (200.f / ch + fabsf(largest) * 4.76837158203125e-7f);
    const uint64_t ch2 = two(ch, ch), cl2 = two(cl, cl), top2 = two(-largest, -largest), ln2 = two(0.6931471805599453f, 0.6931471805599453f), minus = two(-1.f, -1.f);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      float y0, y1;
      const uint64_t x = two(fmaxf(f[2 * q], floor_f), fmaxf(f[2 * q + 1], floor_f)), d = add2(x, top2), y = mul2(d, ch2);
      uint64_t rest = fma2(d, cl2, fma2(d, ch2, mul2(y, minus)));
      if constexpr (decltype(exact)::value) {
        const uint64_t b = fma2(x, minus, d);    // (what the sum has of -largest; Knuth's exact sum of two)
        rest = fma2(add2(fma2(fma2(b, minus, d), minus, x), fma2(b, minus, top2)), ch2, rest);
      }
      untwo(y, y0, y1);
      const uint64_t e = two(ex2(y0), ex2(y1));
      untwo(fma2(e, mul2(rest, ln2), e), w[2 * q], w[2 * q + 1]);
    }
  };
  auto add8 = [](const float (&w)[8]) { return ((w[0] + w[1]) + (w[2] + w[3])) + ((w[4] + w[5]) + (w[6] + w[7])); };
  // How far a sum of such weights and u times their whole may lie from one another's true place: every weight is within e = 4.3e-7 (2^-22, and three
  // roundings of 2^-24: one of its own, two where four are added; the rest is added in 64 bits) of itself, those before the place count 1 - u times
  // and those behind it u times.
  const double u64 = u > 0.f ? (u < 1.f ? (double)u : 1.0) : 0.0;
  auto slack_of = [&](double all) { return all * (2.0 * u64 * (1.0 - u64) * 4.3e-7 + 1e-11); };
  auto place_of = [&](double all) { return u > 0.f ? (u < 1.f ? (double)u * all : all) : 0.0; };
  double* const sums_d = (double*)sh.sums;
  // The part at which the running sum of the parts' passes t, by a warp; *before = the sum before it; -1: none.
  auto part_of = [&](auto* sums, auto t, auto* before) -> int {
    auto b = *before;
    for (int q0 = 0; q0 < parts; q0 += 32) {
      auto upto = q0 + lane < parts ? sums[q0 + lane] : (decltype(b))0;
      const auto x = upto;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const auto n = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += n;
      }
      const uint32_t hit = __ballot_sync(0xffffffffu, b + upto > t);
      if (hit) {
        const int l = __ffs(hit) - 1;
        *before = b + __shfl_sync(0xffffffffu, upto - x, l);
        return q0 + l;
      }
      b += __shfl_sync(0xffffffffu, upto, 31);
    }
    return -1;
  };
  // The element of part q at which the running sum from `before` on passes t by more than `slack` and before which it stays as far below, by a warp;
  // -1: none.
  auto within = [&](int q, auto before, auto t, auto slack, auto weights) -> int {
    using S = decltype(before);
    S mine[DEEP];
#pragma unroll 2
    for (int s = 0; s < DEEP; ++s) {
      const int v = (q * DEEP + s) * 32 + lane;
      mine[s] = 0;
      if (v < r.vecs) {
        auto w = weights(v);
#pragma unroll
        for (int e = 0; e < 8; ++e) mine[s] += (S)w.w[e];
      }
    }
    int at = -1;
    S run = before;
#pragma unroll 1
    for (int s = 0; s < DEEP; ++s) {
      S m = 0;
#pragma unroll
      for (int x = 0; x < DEEP; ++x) m = x == s ? mine[x] : m;
      const S all = warp_sum(m);
      if (run + all > t || run + all + slack > t) {
        S upto = m;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const S n = __shfl_up_sync(0xffffffffu, upto, o);
          if (lane >= o) upto += n;
        }
        S b = run + upto - m;
        const int v = (q * DEEP + s) * 32 + lane;
        if (v < r.vecs && b <= t && b + m >= t) {
          auto w = weights(v);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            if (at < 0 && b + slack <= t && t + slack < b + (S)w.w[e]) at = r.index(v, e);
            b += (S)w.w[e];
          }
        }
        break;
      }
      run += all;
    }
    const uint32_t hit = __ballot_sync(0xffffffffu, at >= 0);
    return hit ? __shfl_sync(0xffffffffu, at, __ffs(hit) - 1) : -1;
  };
  struct W8 { float w[8]; };
  struct U8 { uint64_t w[8]; };

  // ---- the row's largest; sums for the log-probability; where the row is read once, of the weights too ----
  // Weights and the terms of the log-probability are relative to a reference of the warp's own: the largest of its parts so far, to a factor of
  // 2^(1/4) of a weight.  A part is asked for while the one before is worked on.
  float top;
  int token = -1;
  {
    uint64_t best = 0;                           // pattern, V - 1 - index (the index where the largest is all that is asked for)
    float ref = -INFINITY, mx = -INFINITY;
    const float steep = a.logprobs ? fmaxf(once ? ch : 0.f, kLog2e) : ch;
    double lp = 0.0;
    typename Row<T>::Raw next[DEEP];
    auto ask = [&](int q) {
#pragma unroll
      for (int s = 0; s < DEEP; ++s) {
        const int v = (q * DEEP + s) * 32 + lane;
        if (v < r.vecs) next[s] = r.load_raw(v);
        else {
          alignas(16) T none[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) none[e] = (T)(-INFINITY);
#pragma unroll
          for (int x = 0; x < Row<T>::W; ++x) next[s].w[x] = ((const uint4*)none)[x];
        }
      }
    };
    ask(warp);
#pragma unroll 1
    for (int q = warp; q < parts; q += kWarps) {
      float f[DEEP][8], m = -INFINITY;
#pragma unroll
      for (int s = 0; s < DEEP; ++s) {
        Row<T>::unpack(next[s], f[s]);
#pragma unroll
        for (int e = 0; e < 8; ++e) { f[s][e] = clean(f[s][e]); m = fmaxf(m, f[s][e]); }
      }
      ask(q + kWarps);
      if (hold) {
#pragma unroll
        for (int s = 0; s < DEEP; ++s) {
          const int v = (q * DEEP + s) * 32 + lane;
          alignas(16) T e8[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) e8[e] = (T)f[s][e];
          if (v < r.vecs)
#pragma unroll
            for (int x = 0; x < Row<T>::W; ++x) *(uint4*)(held + v * (16 * Row<T>::W) + 16 * x) = ((const uint4*)e8)[x];
        }
      }
      mx = fmaxf(mx, m);
      if (greedy) {
        if (pattern(m) > (uint32_t)(best >> 32)) {           // (parts ascend: an equal one further back does not count)
          int at = 0;
#pragma unroll
          for (int s = DEEP - 1; s >= 0; --s)
#pragma unroll
            for (int e = 7; e >= 0; --e) at = f[s][e] == m ? s * 256 + e : at;
          if (m > -INFINITY) best = (uint64_t)pattern(m) << 32 | (uint32_t)(V - 1 - r.index(q * DEEP * 32 + lane, at));
        }
      }
      if (!once && !a.logprobs) continue;
      if (__any_sync(0xffffffffu, m > ref && !((m - ref) * steep < 0.25f))) {
        const float up = value_of(__reduce_max_sync(0xffffffffu, pattern(m)));
        if (a.logprobs) lp = ref > -INFINITY ? lp * exp2((double)(ref - up) * 1.4426950408889634) : 0.0;
        ref = up;
      }
      if (once) {
        double t = 0.0;
        if (ref > -INFINITY && ref < INFINITY) {
#pragma unroll
          for (int s = 0; s < DEEP; ++s) {
            float w[8];
            weights32(std::false_type{}, f[s], ref, w);
            t += (double)((w[0] + w[1]) + (w[2] + w[3])) + (double)((w[4] + w[5]) + (w[6] + w[7]));
          }
          t = warp_sum(t);
        }
        if (lane == 0) { sums_d[q] = t; sh.refs[q] = ref; }
      }
      if (a.logprobs && ref > -INFINITY) {
#pragma unroll
        for (int s = 0; s < DEEP; ++s) {
          float w[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) w[e] = f[s][e] == ref ? 1.f : ex2((f[s][e] - ref) * kLog2e);
          lp += (double)add8(w);
        }
      }
    }
    if (!greedy && mx > -INFINITY) best = (uint64_t)pattern(mx) << 32;
    if (hold) r.held = held;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) best = max(best, (uint64_t)__shfl_xor_sync(0xffffffffu, best, o));
    __syncthreads();
    if (lane == 0) sh.red[warp] = best;
    __syncthreads();
    best = lane < kWarps ? sh.red[lane] : 0;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) best = max(best, (uint64_t)__shfl_xor_sync(0xffffffffu, best, o));
    const float mine_top = best ? value_of((uint32_t)(best >> 32)) : -INFINITY;
    cluster_wait();                              // all blocks of the cluster run
    double mine = 0.0;
    if (once) {
      // Parts relative to the block's largest (where that is infinite the row is not decided here).  The differences were rounded to fp32, which puts a
      // weight e^-x off by 2^-24 x of itself.  With x weighted by the weights, its mean over a part's n = 512 and ln(sum) make the weights' entropy,
      // at most ln(n): their x add up to no more than sum * ln(n / sum).  (A logit may lie above its reference, by a factor of 2^(1/4) of its
      // weight, which takes up to 0.18 of the sum from that and may be off by as much.)
      double far = 0.0;
      for (int q = tid; q < parts; q += kThreads) {
        const float at = sh.refs[q];
        double w = 0.0;
        if (at > -INFINITY && mine_top < INFINITY) {
          const double sum = sums_d[q], down = exp2(((double)at - (double)mine_top) * c_all);
          w = sum * down;
          far += w * (double)(0.37f + fmaxf(logf(32.f * 8.f * DEEP / fmaxf((float)sum, 1e-30f)), 0.f));
        }
        sums_d[q] = w;
        mine += w;
      }
      mine = block_sums_d(mine, far);
      if (tid < (int)C) put64((uint64_t*)&sh.once_sum[me], (uint32_t)tid, (uint64_t)__double_as_longlong(mine));
    }
    if (a.logprobs) {
      lp = block_sum_d(ref > -INFINITY ? (ref != mine_top ? lp * exp2((double)(ref - mine_top) * 1.4426950408889634) : lp) : 0.0);
      if (tid == 0) put64((uint64_t*)&sh.part[me], 0, (uint64_t)__double_as_longlong(lp));
      if (tid == 32) put64((uint64_t*)&sh.part_top[me], 0, (uint64_t)__double_as_longlong((double)mine_top));
    }
    const uint64_t* const g = gather(best);
    for (uint32_t c = 0; c < C; ++c) best = max(best, g[c]);
    top = best ? value_of((uint32_t)(best >> 32)) : -INFINITY;
    if (greedy && best) token = V - 1 - (int)(uint32_t)best;
    if (once && best && top < INFINITY) {
      double all = 0.0, far_all = 0.0, part[kMaxCtas], far_of[kMaxCtas];
#pragma unroll
      for (uint32_t c = 0; c < kMaxCtas; ++c) {
        const double down = c < C && g[c] ? exp2(((double)value_of((uint32_t)(g[c] >> 32)) - (double)top) * c_all) : 0.0;
        part[c] = down > 0.0 ? sh.once_sum[c] * down : 0.0;
        far_of[c] = down > 0.0 ? sh.far[c] * down : 0.0;
        far_all += far_of[c];
        all += part[c];
      }
      const double t = place_of(all);
      uint32_t who = C - 1;
      double before = 0.0, run = 0.0, far_run = 0.0, off = 0.0;
      bool found = false;
#pragma unroll
      for (uint32_t c = 0; c < kMaxCtas; ++c) {
        if (c < C && !found && t < run + part[c]) {
          who = c; before = run; found = true;
          // (2^-24 and 1 % for what it is made of in fp32)
          off = 6.02e-8 * ((1.0 - u64) * far_run + u64 * (far_all - far_run - far_of[c]) + fmax(u64, 1.0 - u64) * far_of[c]);
        }
        run += part[c];
        far_run += far_of[c];
      }
      const double slack = slack_of(all) + off;
      if (who == me && warp == 0) {
        // everything relative to this block's largest, then to the part's
        int at = -1;
        if (found) {
          const double up = exp2(((double)top - (double)mine_top) * c_all);
          double b = before * up;
          const int q = part_of(sums_d, t * up, &b);
          if (q >= 0) {
            const double there = exp2(((double)mine_top - (double)sh.refs[q]) * c_all);
            at = within(q, b * there, t * up * there, slack * up * there, [&](int v) {
              float f[8];
              W8 w;
              r.load8(v, f);
              weights32(std::false_type{}, f, sh.refs[q], w.w);
              return w;
            });
          }
        }
        if (lane < (int)C) put32(&sh.answer[0], (uint32_t)lane, (uint32_t)at);
      }
      cluster_sync_all();
      token = sh.answer[0];
    }
  }
  const bool nothing = top == -INFINITY;
  const double top64 = top;
  double log_whole = 0.0;
  if (a.logprobs && me == 0 && tid == kThreads - 1) {        // (while the others go on)
    double all = 0.0;
    for (uint32_t c = 0; c < C; ++c) {
      const double ref = sh.part_top[c];
      if (ref > -INFINITY) all += ref == top64 ? sh.part[c] : sh.part[c] * exp(ref - top64);
    }
    log_whole = log(all);
  }
  auto weigh = [&](float x) -> uint64_t { return weight64(x == top ? 0.0 : (double)x - top64, c64, sh.roots); };   // (of an infinite temperature: all alike)
  auto enough = [&](float x) { return !(least > 0.f) || x == top || exp(((double)x - (double)top) * per_t) >= (double)least; };

  auto stays = [&](const Border& b, float x, int i) { return pattern(x) > b.key || (pattern(x) == b.key && i <= b.index); };
  // What a logit counts: its weight, or 1; of those that stay at `b`, and with a key from `least_key` on, or that key alone.
  struct What { bool weight, all, min_p, alone; uint32_t least_key; Border b; };
  auto amount_of = [&](const What& h, float x, int i) -> uint64_t {
    const uint32_t key = pattern(x);
    const bool in = (h.all || stays(h.b, x, i)) && (h.alone ? key == h.least_key : key >= h.least_key) && (!h.min_p || enough(x));
    const uint64_t w = h.weight ? weigh(x) : 1;
    return in ? w : 0;
  };
  // The first index at which the sum passes a place (below 0: that of the random number), all blocks' answer.
  auto find = [&](auto plain, const What& h, int64_t at_count) -> int {
    auto amount = [&](float x, int i) -> uint64_t {
      if constexpr (decltype(plain)::value) return weigh(x); else return amount_of(h, x, i);
    };
    uint64_t mine = 0;
#pragma unroll 1
    for (int q = warp; q < parts; q += kWarps) {
      uint64_t t = 0;
#pragma unroll 1
      for (int s = 0; s < DEEP; ++s) {
        const int v = (q * DEEP + s) * 32 + lane;
        if (v >= r.vecs) continue;
        float f[8];
        r.load8(v, f);
#pragma unroll
        for (int e = 0; e < 8; ++e) t += amount(f[e], r.index(v, e));
      }
      t = warp_sum(t);
      if (lane == 0) { sh.sums[q] = t; mine += t; }
    }
    const uint64_t* const g = gather(block_sum(mine));
    uint64_t all = 0;
    for (uint32_t c = 0; c < C; ++c) all += g[c];
    uint64_t t = (uint64_t)at_count;
    if (at_count < 0) {
      t = u > 0.f ? (u < 1.f ? (uint64_t)((double)u * (double)all) : all) : 0;
      t = t < all ? t : all - 1;
    }
    uint64_t before = 0;
    uint32_t who = 0;
    for (; who + 1 < C && before + g[who] <= t; ++who) before += g[who];
    if (who == me && warp == 0) {
      const int q = part_of(sh.sums, t, &before);
      const int at = q < 0 ? V - 1 : within(q, before, t, (uint64_t)0, [&](int v) {
        float f[8];
        U8 w;
        r.load8(v, f);
#pragma unroll
        for (int e = 0; e < 8; ++e) w.w[e] = amount(f[e], r.index(v, e));
        return w;
      });
      if (lane < (int)C) put32(&sh.answer[0], (uint32_t)lane, (uint32_t)at);
    }
    cluster_sync_all();
    return sh.answer[0];
  };
  // The token among those of which `stay(x, i)` says so, by weights in fp32.  -1 where the place to find lies too near an element's border (or a weight
  // too near min_p): then the whole numbers decide.
  auto find_fast = [&](auto stay) -> int {
    auto weights = [&](int v) {
      float f[8];
      W8 w;
      r.load8(v, f);
      weights32(std::true_type{}, f, top, w.w);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if (least > 0.f) {
          const float off = w.w[e] - least;
          if (fabsf(off) <= least * 1.9073486328125e-6f && f[e] != top) w.w[e] = __uint_as_float(0x7fc00000u);    // 2^-19
          else if (off < 0.f && f[e] != top) w.w[e] = 0.f;
        }
        if (!stay(f[e], r.index(v, e))) w.w[e] = 0.f;
      }
      return w;
    };
    double mine = 0.0;
    for (int q = warp; q < parts; q += kWarps) {
      double t = 0.0;
#pragma unroll 2
      for (int s = 0; s < DEEP; ++s) {
        const int v = (q * DEEP + s) * 32 + lane;
        if (v < r.vecs) {
          const W8 w = weights(v);
          t += (double)((w.w[0] + w.w[1]) + (w.w[2] + w.w[3])) + (double)((w.w[4] + w.w[5]) + (w.w[6] + w.w[7]));
        }
      }
      t = warp_sum(t);
      if (lane == 0) { sums_d[q] = t; mine += t; }
    }
    const uint64_t* const g = gather((uint64_t)__double_as_longlong(block_sum_d(mine)));
    double all = 0.0;
    for (uint32_t c = 0; c < C; ++c) all += __longlong_as_double((long long)g[c]);
    const double t = place_of(all);
    uint32_t who = 0;
    double before = 0.0;
    for (; who + 1 < C; ++who) {
      const double n = __longlong_as_double((long long)g[who]);
      if (t < before + n) break;
      before += n;
    }
    if (who == me && warp == 0) {
      const int q = part_of(sums_d, t, &before);
      const int at = q >= 0 ? within(q, before, t, slack_of(all), weights) : -1;
      if (lane < (int)C) put32(&sh.answer[0], (uint32_t)lane, (uint32_t)at);
    }
    cluster_sync_all();
    return sh.answer[0];
  };
  // a look at every element of the share
  auto each = [&](auto look) {
    for (int v = tid; v < r.vecs; v += kThreads) {
      float f[8];
      r.load8(v, f);
#pragma unroll
      for (int e = 0; e < 8; ++e) look(f[e], r.index(v, e));
    }
  };
  auto sum_of = [&](const What& h) {
    uint64_t s = 0;
    each([&](float x, int i) { s += amount_of(h, x, i); });
    return total(s);
  };
  // The border at which the counts (or weights) of what stays before it reach `target`, of what stays at `from`: by halving.
  auto border = [&](bool weight, uint64_t target, const Border& from) {
    What h = {weight, false, false, false, 0u, from};
    uint32_t lo = 0, hi = pattern(top);          // the largest key whose sum from there up reaches the target
    uint64_t above = 0;                          // (of the smallest key that is known not to)
    while (lo < hi) {
      h.least_key = lo + (hi - lo) / 2 + 1;
      const uint64_t n = sum_of(h);
      if (n >= target) lo = h.least_key; else { hi = h.least_key - 1; above = n; }
    }
    Border b = {lo, V - 1};
    const uint64_t one = weight ? weigh(value_of(lo)) : 1;
    if (one > 0) {                               // among equal ones, the first so many by index
      h.weight = false; h.alone = true; h.least_key = lo;
      b.index = find(std::false_type{}, h, (int64_t)((target - above + one - 1) / one) - 1);
    }
    return b;
  };
  // how many steps below the largest; kBins: further than the bins go
  const float per_step = (float)kBins / (kRange * temp);
  auto bin_of = [&](float x) {
    if (x == top) return 0;
    const float d = (top - x) * per_step;
    return d < (float)kBins ? (int)d : kBins;
  };

  if (!greedy && !nothing && token < 0) {
    Border b = {0u, V - 1};
    if (by_k || by_p) {
      // ---- how many logits in which step ----
      for (int i = tid; i < kBins; i += kThreads) sh.hist[i] = 0;
      __syncthreads();
      each([&](float x, int) {
        const int bin = bin_of(x);
        if (bin < kBins) atomicAdd(&sh.hist[bin], 1u);
      });
      cluster_sync_all();
      const int bins = kBins / (int)C;           // every block adds its part of the bins, for all
      for (int i = tid; i < bins; i += kThreads) {
        const int bin = (int)me * bins + i;
        uint32_t n = 0;
        for (uint32_t c = 0; c < C; ++c) n += get32(&sh.hist[bin], c);
        for (uint32_t c = 0; c < C; ++c) put32(&sh.merged[bin], c, n);
      }
      cluster_sync_all();
      // ---- the steps that matter: a thread has eight neighbours ----
      constexpr int PER = kBins / kThreads;
      uint32_t cnt[PER], mine = 0;
#pragma unroll
      for (int i = 0; i < PER; ++i) { cnt[i] = sh.merged[tid * PER + i]; mine += cnt[i]; }
      uint32_t upto = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t n = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += n;
      }
      if (lane == 31) sh.scan[warp] = upto;
      __syncthreads();
      uint32_t before = upto - mine, in_range = 0;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) { if (w < warp) before += sh.scan[w]; in_range += sh.scan[w]; }
      const uint32_t want = by_k && (uint32_t)k < in_range ? (uint32_t)k : in_range;     // (what lies further has no weight)
      if (before < want && want <= before + mine) {
        uint32_t run = before;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
          if (run < want && want <= run + cnt[i]) { sh.answer[0] = tid * PER + i; sh.answer[1] = (int)(run + cnt[i]); sh.answer[2] = (int)run; }
          run += cnt[i];
        }
      }
      __syncthreads();
      const int k_bin = sh.answer[0], k_upto = sh.answer[1], k_before = sh.answer[2];
      const bool cut = want < in_range;          // top-k leaves something out
      const bool few = k_upto <= kList;          // all that may stay fits the list
      // Entries are gathered in a block's own list, then put into the first block's, behind its own and one another.
      auto enlist = [&](float x, int index) {
        const uint32_t at = atomicAdd(&sh.staged, 1u);
        if (at < kList) sh.list[at] = (uint64_t)pattern(x) << 32 | (uint32_t)(V - 1 - index);
      };
      auto deliver = [&]() {
        __syncthreads();
        const uint32_t n = min(sh.staged, (uint32_t)kList);
        if (me == 0 && tid == 0) sh.listed = n;
        cluster_sync_all();                      // (the first block's own entries are in place)
        if (me != 0) {
          if (tid == 0 && n > 0) sh.place = add32(&sh.listed, 0, n);
          __syncthreads();
          for (uint32_t i = tid; i < n; i += kThreads)
            if (sh.place + i < kList) put64(&sh.list[sh.place + i], 0, sh.list[i]);
        }
        if (C > 1) cluster_sync_all();
        if (tid == 0) sh.staged = 0;
        __syncthreads();
      };
      auto into_list = [&](int lo, int hi) {
        each([&](float x, int i) {
          const int bin = bin_of(x);
          if (bin >= lo && bin <= hi && bin < kBins) enlist(x, i);
        });
        deliver();
      };
      constexpr int LPT = kList / kThreads;      // neighbours of a thread
      // The first n entries of the list in descending order, by the first block: bitonic, an entry's partner in the same thread, in the same
      // warp, or through shared memory (ten of 55 steps for 1024).  What fills up the power of two is 0.
      auto sort_list = [&](int n) {
        int m = LPT * 32;
        while (m < n) m *= 2;
        const bool live = LPT * 32 * warp < m;
        uint64_t x[LPT];
        if (live)
#pragma unroll
          for (int q = 0; q < LPT; ++q) x[q] = LPT * tid + q < n ? sh.list[LPT * tid + q] : 0;
        for (int span = 2; span <= m; span *= 2)
          for (int d = span / 2; d > 0; d /= 2) {
            if (d >= LPT * 32) {
              __syncthreads();
              if (live)
#pragma unroll
                for (int q = 0; q < LPT; ++q) sh.list[LPT * tid + q] = x[q];
              __syncthreads();
            }
            if (!live) continue;
            if (d < LPT) {
#pragma unroll
              for (int dd = 1; dd < LPT; dd *= 2)
                if (dd == d)
#pragma unroll
                  for (int q = 0; q < LPT; ++q)
                    if ((q & dd) == 0) {
                      const bool down = ((LPT * tid + q) & span) == 0;
                      const uint64_t a0 = x[q], a1 = x[q + dd];
                      if ((a0 < a1) == down) { x[q] = a1; x[q + dd] = a0; }
                    }
            } else {
              const bool first = (LPT * tid & d) == 0;
#pragma unroll
              for (int q = 0; q < LPT; ++q) {
                const uint64_t y = d < LPT * 32 ? (uint64_t)__shfl_xor_sync(0xffffffffu, x[q], d / LPT) : sh.list[(LPT * tid + q) ^ d];
                const bool larger = (((LPT * tid + q) & span) == 0) == first;
                x[q] = (x[q] < y) == larger ? y : x[q];
              }
            }
          }
        __syncthreads();
        if (live)
#pragma unroll
          for (int q = 0; q < LPT; ++q) sh.list[LPT * tid + q] = x[q];
        __syncthreads();
      };
      // sums before each of a thread's entries, of amounts in order; *all = their sum
      auto list_sums = [&](const uint64_t (&w)[LPT], uint64_t (&before)[LPT], uint64_t* all) {
        uint64_t mine = 0;
#pragma unroll
        for (int q = 0; q < LPT; ++q) { before[q] = mine; mine += w[q]; }
        uint64_t upto = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const uint64_t x = __shfl_up_sync(0xffffffffu, upto, o);
          if (lane >= o) upto += x;
        }
        __syncthreads();
        if (lane == 31) sh.red[warp] = upto;
        __syncthreads();
        uint64_t base = upto - mine, sum = 0;
#pragma unroll
        for (int x = 0; x < kWarps; ++x) { if (x < warp) base += sh.red[x]; sum += sh.red[x]; }
#pragma unroll
        for (int q = 0; q < LPT; ++q) before[q] += base;
        *all = sum;
      };
      auto nucleus = [&](uint64_t Z) {           // the sum that the weights in front of an element that stays are below
        if (!by_p) return ~(uint64_t)0;
        const uint64_t t = p > 0.f ? (uint64_t)ceil((double)p * (double)Z) : 1ull;
        return t < 1 ? (uint64_t)1 : t;
      };
      auto place = [&](uint64_t Z) {
        const uint64_t t = u > 0.f ? (u < 1.f ? (uint64_t)((double)u * (double)Z) : Z) : 0;
        return t < Z ? t : Z - 1;
      };
      // Entry at which the amounts w of the entries [0, n) (LPT a thread, entry tid + q * kThreads), taken by descending `order`, reach `target`; by the first block.  An
      // entry's slot (ascending where `order` descends) says roughly where; 1024 slots are added up, and the entries of the one that matters compared
      // pair by pair.  -1: none, or too many in one slot.  (256 rows with top-k 500 and top-p 0.9: 88 us by
      // sorting, 62 by slots.)
      auto locate = [&](int n, const int (&slot)[LPT], const uint64_t (&order)[LPT], const uint64_t (&w)[LPT], uint64_t target) -> int {
        uint64_t* const mass = sh.slots.mass;
        for (int i = tid; i < kSlots; i += kThreads) mass[i] = 0;
        if (tid == 0) { sh.slots.members = 0; sh.slots.slot = -1; sh.slots.found = -1; }
        __syncthreads();
#pragma unroll
        for (int q = 0; q < LPT; ++q)
          if (w[q] > 0) atomicAdd((unsigned long long*)&mass[slot[q]], (unsigned long long)w[q]);
        __syncthreads();
        const uint64_t m0 = mass[2 * tid], m1 = mass[2 * tid + 1];
        static_assert(kSlots == 2 * kThreads, "two a thread");
        uint64_t upto = m0 + m1;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const uint64_t x = __shfl_up_sync(0xffffffffu, upto, o);
          if (lane >= o) upto += x;
        }
        if (lane == 31) sh.red[warp] = upto;
        __syncthreads();
        uint64_t before = upto - m0 - m1;
#pragma unroll
        for (int x = 0; x < kWarps; ++x) before += x < warp ? sh.red[x] : 0;
        if (before < target && target <= before + m0) { sh.slots.slot = 2 * tid; sh.slots.before = before; }
        else if (before + m0 < target && target <= before + m0 + m1) { sh.slots.slot = 2 * tid + 1; sh.slots.before = before + m0; }
        __syncthreads();
        const int in = sh.slots.slot;
        int at[LPT];
#pragma unroll
        for (int q = 0; q < LPT; ++q) {
          at[q] = -1;
          if (w[q] > 0 && slot[q] == in) {
            at[q] = (int)atomicAdd(&sh.slots.members, 1u);
            if (at[q] < kPairs) { sh.slots.order[at[q]] = order[q]; sh.slots.weight[at[q]] = w[q]; }
          }
        }
        __syncthreads();
        const int members = (int)sh.slots.members;
        if (in < 0 || members > kPairs) return -1;
        const uint64_t base = sh.slots.before;
#pragma unroll
        for (int q = 0; q < LPT; ++q)
          if (at[q] >= 0) {
            uint64_t sum = base;
            for (int i = 0; i < members; ++i) sum += sh.slots.order[i] > order[q] ? sh.slots.weight[i] : 0ull;
            if (sum < target && target <= sum + w[q]) sh.slots.found = tid + q * kThreads;
          }
        __syncthreads();
        return sh.slots.found;
      };
      // the same by sorting (ties may fill a slot); the entries are in descending order afterwards
      auto locate_sorted = [&](int n, bool weights, int limit, uint64_t target, bool by_index = false) -> int {
        sort_list(n);
        uint64_t w[LPT], before[LPT], all;
#pragma unroll
        for (int q = 0; q < LPT; ++q) {
          const uint64_t x = LPT * tid + q < n && LPT * tid + q < limit ? sh.list[LPT * tid + q] : 0;
          w[q] = x == 0 ? 0 : (weights ? weigh(value_of((uint32_t)(by_index ? x : x >> 32))) : 1);
        }
        list_sums(w, before, &all);
        if (tid == 0) sh.slots.found = -1;
        __syncthreads();
#pragma unroll
        for (int q = 0; q < LPT; ++q)
          if (before[q] < target && target <= before[q] + w[q]) sh.slots.found = LPT * tid + q;
        __syncthreads();
        return sh.slots.found;
      };
      auto slot_by_value = [&](float x, int lo, int hi) {    // of a logit in steps [lo, hi]
        const float d = x == top ? 0.f : (top - x) * per_step;
        const float sl = (d - (float)lo) * ((float)kSlots / (float)(hi + 1 - lo));
        return sl < 0.f ? 0 : (sl < (float)(kSlots - 1) ? (int)sl : kSlots - 1);
      };
      // the element at which the sum of the list's counts (or weights), in order, reaches `target`; by the first block, told to all
      auto in_list = [&](bool weights, int lo, int hi, uint64_t target) {
        if (me == 0) {
          const int n = (int)min(sh.listed, (uint32_t)kList);
          int slot[LPT];
          uint64_t order[LPT], w[LPT];
#pragma unroll
          for (int q = 0; q < LPT; ++q) {
            const int i = tid + q * kThreads;
            order[q] = i < n ? sh.list[i] : 0;
            const float x = value_of((uint32_t)(order[q] >> 32));
            w[q] = i < n ? (weights ? weigh(x) : 1) : 0;
            slot[q] = i < n ? slot_by_value(x, lo, hi) : 0;
          }
          int at = locate(n, slot, order, w, target);
          if (at < 0) at = locate_sorted(n, weights, n, target);
          if (tid < (int)C && at >= 0) {
            const uint64_t x = sh.list[at];
            put32(&sh.answer[2], (uint32_t)tid, (uint32_t)(x >> 32)); put32(&sh.answer[3], (uint32_t)tid, (uint32_t)(V - 1 - (int)(uint32_t)x));
          }
        }
        cluster_sync_all();
      };
      if (few) {
        // ---- all that may stay is in the list: the first block draws the token ----
        into_list(0, k_bin);
        if (me == 0 && k_upto <= kPairs) {
          // every entry looks at all others: its rank and the sum in front of it, then the sum up to it by index
          const int n = k_upto;
          uint64_t x = 0, w = 0, before_w = 0;
          uint32_t rank = 0;
          if (tid < n) {
            x = sh.list[tid];
            w = weigh(value_of((uint32_t)(x >> 32)));
            sh.slots.weight[tid] = w;
          }
          __syncthreads();
          if (tid < n)
#pragma unroll 4
            for (int i = 0; i < n; ++i)
              if (sh.list[i] > x) { ++rank; before_w += sh.slots.weight[i]; }
          const bool in_k = tid < n && rank < want;
          const uint64_t target = nucleus(block_sum(in_k ? w : 0));
          const bool stay = in_k && w > 0 && before_w < target && enough(value_of((uint32_t)(x >> 32)));
          if (tid < n) sh.slots.weight[tid] = stay ? w : 0;
          const uint64_t t = place(block_sum(stay ? w : 0));
          if (stay) {
            uint64_t run = 0;
#pragma unroll 4
            for (int i = 0; i < n; ++i) run += (uint32_t)sh.list[i] > (uint32_t)x ? sh.slots.weight[i] : 0ull;
            if (run <= t && t < run + w)
              for (uint32_t c = 0; c < C; ++c) put32(&sh.answer[0], c, (uint32_t)(V - 1 - (int)(uint32_t)x));
          }
        } else if (me == 0) {
          const int n = k_upto;
          int slot[LPT], at = 0;
          uint64_t order[LPT], w[LPT], zero[LPT], mine = 0;
          Border kb = {0u, V - 1};               // of top-k
          auto fill = [&]() {
#pragma unroll
            for (int q = 0; q < LPT; ++q) {
              const int i = tid + q * kThreads;
              order[q] = i < n ? sh.list[i] : 0;
              const float x = value_of((uint32_t)(order[q] >> 32));
              slot[q] = i < n ? slot_by_value(x, 0, k_bin) : 0;
              zero[q] = i < n;
              w[q] = i < n ? weigh(x) : 0;
            }
          };
          fill();
          // Where each border lies: the entry itself, so that an entry stays where its order is not below it.
          uint64_t last = 0;
          if (want < (uint32_t)n) {
            at = locate(n, slot, order, zero, (uint64_t)want);
            if (at < 0) { at = locate_sorted(n, false, n, (uint64_t)want); fill(); }
            last = sh.list[at];
          }
#pragma unroll
          for (int q = 0; q < LPT; ++q) { w[q] = order[q] >= last ? w[q] : 0; mine += w[q]; }
          if (by_p) {
            const uint64_t target = nucleus(block_sum(mine));
            __syncthreads();
            at = locate(n, slot, order, w, target);
            if (at < 0) {
              at = locate_sorted(n, true, (int)want, target);
              fill();
#pragma unroll
              for (int q = 0; q < LPT; ++q) w[q] = order[q] >= last ? w[q] : 0;
            }
            last = at >= 0 ? sh.list[at] : last;             // (what has no weight may lie behind)
          }
          mine = 0;
#pragma unroll
          for (int q = 0; q < LPT; ++q) {
            const int i = tid + q * kThreads;
            if (w[q] > 0 && (order[q] < last || !enough(value_of((uint32_t)(order[q] >> 32))))) w[q] = 0;
            slot[q] = i < n ? (int)((uint64_t)(uint32_t)(V - 1 - (int)(uint32_t)order[q]) * kSlots / (uint32_t)V) : 0;
            order[q] = (uint64_t)(uint32_t)order[q];         // by index from here on
            mine += w[q];
          }
          const uint64_t t = place(block_sum(mine));
          __syncthreads();
          at = locate(n, slot, order, w, t + 1);
          uint32_t back = at >= 0 ? (uint32_t)sh.list[at] : 0u;               // V - 1 - index
          if (at < 0) {                          // (too many neighbours in a 1024th of the row: sorted by index)
            __syncthreads();
            uint64_t turned[LPT];
#pragma unroll
            for (int q = 0; q < LPT; ++q) {
              const int i = tid + q * kThreads;
              turned[q] = i < n && w[q] > 0 ? sh.list[i] << 32 | sh.list[i] >> 32 : 0;
            }
            __syncthreads();
#pragma unroll
            for (int q = 0; q < LPT; ++q)
              if (tid + q * kThreads < n) sh.list[tid + q * kThreads] = turned[q];
            __syncthreads();
            at = locate_sorted(n, true, n, t + 1, true);
            back = at >= 0 ? (uint32_t)(sh.list[at] >> 32) : 0u;
          }
          if (tid < (int)C) put32(&sh.answer[0], (uint32_t)tid, (uint32_t)(V - 1 - (int)back));
        }
        cluster_sync_all();
        token = sh.answer[0];
      } else {
        if (cut) {
          if (k_upto - k_before <= kList) {
            into_list(k_bin, k_bin);
            in_list(false, k_bin, k_bin, (uint64_t)(want - (uint32_t)k_before));
            b = {(uint32_t)sh.answer[2], sh.answer[3]};
          } else b = border(false, (uint64_t)want, b);
        }
        if (by_p) {
          // Where it should lie by the steps' mean weights, as whole numbers like the weights: their sums are the same in whatever order they are added, so
          // that every place in (0, all] lies in one step of one thread, and in the same one in all blocks, which go on by it alike.
          uint64_t est[PER], sum = 0;
#pragma unroll
          for (int i = 0; i < PER; ++i) {
            const int bin = tid * PER + i;
            const uint32_t n = bin < k_bin ? cnt[i] : (bin == k_bin ? want - (uint32_t)k_before : 0u);
            est[i] = n * (uint64_t)(exp2f(-((float)bin + 0.5f) * (kRange / (float)kBins * kLog2e)) * (float)kOne);
            sum += est[i];
          }
          uint64_t upto_e = sum;
#pragma unroll
          for (int o = 1; o < 32; o <<= 1) {
            const uint64_t n = __shfl_up_sync(0xffffffffu, upto_e, o);
            if (lane >= o) upto_e += n;
          }
          __syncthreads();
          if (lane == 31) sh.red[warp] = upto_e;
          __syncthreads();
          uint64_t run = upto_e - sum, all = 0;
#pragma unroll
          for (int w = 0; w < kWarps; ++w) { if (w < warp) run += sh.red[w]; all += sh.red[w]; }
          // a step's weights are within 2^-8 of their middle: the border is sought as far on both sides, where the list has room for that (it has where
          // few heavy logits make the mean a poor one), else in three steps
          auto inside_of = [&](double x) {           // (the largest logit's step alone makes `all` more than 1)
            const uint64_t v = x > 1.0 ? (uint64_t)x : 1;
            return v < all ? v : all;
          };
          const double t = (double)p * (double)all;
          const uint64_t t_mid = inside_of(t), t_lo = inside_of(t * 0.995), t_hi = inside_of(t * 1.005);
#pragma unroll
          for (int i = 0; i < PER; ++i) {
            const uint32_t upto_n = before;
            before += cnt[i];
            if (run < t_mid && t_mid <= run + est[i]) sh.answer[0] = tid * PER + i;
            if (run < t_lo && t_lo <= run + est[i]) { sh.range[0] = tid * PER + i; sh.range[1] = (int)upto_n; }
            if (run < t_hi && t_hi <= run + est[i]) { sh.range[2] = tid * PER + i; sh.range[3] = (int)before; }
            run += est[i];
          }
          __syncthreads();
          const bool wide = sh.range[3] - sh.range[1] <= kList * 3 / 4;
          const int from_bin = wide ? sh.range[0] : sh.answer[0], to_bin = wide ? sh.range[2] : sh.answer[0];
          const int first_bin = from_bin > 0 ? from_bin - 1 : 0, last_bin = to_bin + 1 < kBins ? to_bin + 1 : kBins - 1;
          int list_n = wide ? sh.range[3] - sh.range[1] + (int)sh.merged[first_bin] + (int)sh.merged[last_bin] : 0;
          if (!wide)
            for (int i = first_bin; i <= last_bin; ++i) list_n += (int)sh.merged[i];
          // the sums above, in and below these steps, and the list, in one pass
          uint64_t s_above = 0, s_list = 0, s_rest = 0;
          bool by_list = list_n <= kList;
          each([&](float x, int i) {
            const int bin = bin_of(x);
            const uint64_t w = weigh(x);
            const bool in = !cut || stays(b, x, i), mine = in && bin >= first_bin && bin <= last_bin;
            s_above += in && bin < first_bin ? w : 0;
            s_list += mine ? w : 0;
            s_rest += in && bin > last_bin ? w : 0;
            if (mine && by_list) enlist(x, i);
          });
          if (by_list) deliver();
          const uint64_t above = total(s_above), inside = total(s_list), whole = above + inside + total(s_rest);
          uint64_t target = nucleus(whole);
          target = target > whole ? whole : target;
          by_list = by_list && above < target && target <= above + inside;
          if (by_list) {
            in_list(true, first_bin, last_bin, target - above);
            b = {(uint32_t)sh.answer[2], sh.answer[3]};
          } else b = border(true, target, b);
        }
      }
    }
    // (at temperatures like these -200 / c, which stands in for all that lies further down, weighs 0 and is itself exact enough)
    if (token < 0 && !once && top < INFINITY && temp >= 1e-6f && temp <= 1e6f) token = find_fast([&](float x, int i) { return !(by_k || by_p) || stays(b, x, i); });
    const What all = {true, !(by_k || by_p), least > 0.f, false, 0u, b};
    if (token < 0) token = once ? find(std::true_type{}, all, -1) : find(std::false_type{}, all, -1);
  }
  if (a.logprobs && me == 0 && tid == kThreads - 1) {
    float y = 0.f;
    if (!nothing) {
      const float x = clean(IO<T>::load((const char*)a.logits + (int64_t)row_no * a.row_bytes, token));
      y = (float)((x == top ? 0.0 : (double)x - top64) - log_whole);
    }
    a.logprobs[row_no] = y;
  }
  if (me == 0 && tid == 0) a.tokens[row_no] = token;
  cluster_sync_all();                            // (shared memory stays until all have read it)
}

template <typename T> cudaError_t launch_t(const SampleArgs& a, cudaStream_t st) {
  auto kern = sample_kernel<T>;
  static bool done[64] = {};
  constexpr int kHeld = 96 * 1024;               // of a row's share at most (beside 43 KB of Shared: two blocks an SM up to 70 KB of it, one above)
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  {
    std::lock_guard<std::mutex> setup_lk(setup_mutex());     // first use on a device, from any thread
    if (dev < 0 || dev >= 64 || !done[dev]) {
      e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(Shared) + kHeld);
      if (e != cudaSuccess) return e;
      if (dev >= 0 && dev < 64) done[dev] = true;
    }
  }
  // Blocks a row: enough that there is one for every SM (two a row up to two rows an SM), of at least 8192 and, up to eight blocks, at most 65536 elements
  // each.  A share of up to 96 KB stays in shared memory (49152 elements of 16 bits, 24576 of 32); a larger one is read again in every pass, as those of 74
  // and more rows of 128256 logits in bf16 are, or of 296 and more rows of 32001 in fp32.  (128256 logits, the 50 largest, by 1, 2, 4, 8 blocks a row: one row 68, 42, 24, 19 us;
  // 64 rows 74, 45, 32, 47; 128 rows -, 57, 62, 90.  256 rows of 32001 with filters of all kinds 78, 66, 87, 151.  A nucleus over flat rows pays for more: 48
  // rows by 4 blocks 120, by 8 102.  Not measured: more blocks where a share does not stay.)
  int ctas = 1;
  while (ctas < kMaxCtas && ((int64_t)a.N * ctas < (ctas == 1 ? 2 : 1) * sm_count() || a.V > ctas * 65536) && a.V > ctas * 8192) ctas *= 2;
  for (;; ctas = 1) {
    const int share = ((a.V + ctas - 1) / ctas + 7) / 8 * 8;
    const int need = (share + 16) * (int)sizeof(T);
    const int bytes = need <= kHeld ? (need + 15) / 16 * 16 : 0;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)a.N * (unsigned)ctas);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = sizeof(Shared) + (size_t)bytes;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)ctas; attr[1].val.clusterDim.y = 1; attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = ctas == 1 ? 1 : 2;
    if (ctas == 1) return cudaLaunchKernelEx(&cfg, kern, a, share, bytes);
    e = launch_clusters(cfg, kern, a, share, bytes);
    if (e == cudaSuccess) return e;
    (void)cudaGetLastError();                    // the device places no clusters: a block a row
  }
}
}  // namespace

cudaError_t launch_sample(const SampleArgs& a, cudaStream_t st) {
  return a.dtype == QB200_BFLOAT16 ? launch_t<__nv_bfloat16>(a, st) : (a.dtype == QB200_FLOAT16 ? launch_t<__half>(a, st) : launch_t<float>(a, st));
}

}  // namespace qb
