// A token from every row of logits: temperature, top-k, top-p and min-p, with a random number given for the row.
//
// With m the row's largest logit, w_i = exp((l_i - m) / temperature) and the order "larger logit first, then lower index": the first k
// of the order stay; of these the shortest prefix whose weights reach p of their sum; of these those with w_i >= min_p; the token is the
// first one in index order at which the running sum of the weights that stay passes u times their sum.
//
//  * Weights are whole numbers, round(w_i * 2^44), of a 64-bit exponential: sums of them do not depend on the order in which threads
//    or atomics run, and borders (the nucleus, the token) are met as 64-bit sums meet them.  2^19 of them fit 63 bits; a token below
//    2^-45 of the largest counts as 0.
//  * A row is a cluster of up to eight blocks, each with a share of the row in shared memory (read from memory again where it is too
//    large); sums and histograms meet through distributed shared memory.
//  * The border of top-k and top-p in the order: a histogram of how far the logits lie below the largest, in steps of 2^-7 of the temperature, says in which step it lies
//    (top-k exactly; top-p by the steps' mean weights, and the sums of the next pass say whether that was right).  The logits of
//    these steps go to a list in the first block, where each looks at all others.  Few that stay are drawn from that list alone.  Where the list
//    would be too long (equal logits, flat rows) the border is found by halving the range of the logits' patterns, a sum over the row each time.
#include <cstddef>
#include <mutex>
#include <type_traits>

#include "kernels.h"
#include "stream_ptx.cuh"

namespace qb {
namespace {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kStrip = kThreads * 8;           // elements that the block takes at a time, eight a thread
constexpr int kMaxStrips = kMaxVocab / kStrip + 2;
constexpr int kBins = 4096;
constexpr float kRange = 32.f;                 // temperatures below the largest that the bins cover: e^-32 < 2^-45
constexpr int kList = 2048;
constexpr double kOne = 17592186044416.0;      // 2^44
constexpr int kMaxCtas = 8;

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
// sum with 2^52.  0 where the exponent is below -46.
__device__ __forceinline__ uint64_t weight64(double d, double c, const double* roots) {
  const double t = d * c;
  if (!(t > -46.0 * 32.0)) return 0;
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
  double roots[32];
  uint64_t above, whole;
  union {                                      // (never of use at the same time)
    uint32_t hist[kBins];
    uint64_t list[kList];                      // pattern, then V - 1 - index: larger ones come first in the order
    uint64_t sums[kMaxStrips * kWarps];        // of every warp's part of every strip
  };
  union {
    uint32_t merged[kBins];
    float refs[kMaxStrips * kWarps];           // of the parts: what their sums are relative to
  };
  uint32_t scan[kWarps];
  uint32_t listed, staged, place;
  int answer[4];
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
  extern __shared__ __align__(16) unsigned char raw[];
  Shared& sh = *(Shared*)raw;
  const uint32_t C = cluster_size(), me = cluster_rank();
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int row_no = (int)(blockIdx.x / C), tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, V = a.V;
  const float temp = a.temperature ? a.temperature[row_no * a.str[1]] : 1.f, u = a.random[row_no * a.str[0]];
  const int k = a.top_k ? a.top_k[row_no * a.str[2]] : 0;
  const float p = a.top_p ? a.top_p[row_no * a.str[3]] : 1.f, least = a.min_p ? a.min_p[row_no * a.str[4]] : 0.f;

  // ---- this block's share, and the row's largest ----
  Row<T> r;
  r.begin = (int)me * share < V ? (int)me * share : V;
  r.n = V - r.begin < share ? V - r.begin : share;
  r.x = (const T*)((const char*)a.logits + (int64_t)row_no * a.row_bytes) + r.begin;
  r.off = (int)((uintptr_t)r.x & (8 * sizeof(T) - 1)) / (int)sizeof(T);
  r.vecs = (r.n + r.off + 7) / 8;
  unsigned char* const held = raw + sizeof(Shared);
  const bool greedy = !(temp > 0.f), by_k = k > 0 && k < V, by_p = p < 1.f;
  // by temperature alone the row is read once, each warp's 256 elements at a time with a largest of their own
  const bool once = !greedy && !by_k && !by_p && !(least > 0.f) && temp >= 1e-6f && temp <= 1e6f;
  if (tid == 0) sh.listed = sh.staged = 0;
  if (tid < 32) sh.roots[tid] = kRoots[tid];
  if (by_k || by_p)
    for (int i = tid; i < kBins; i += kThreads) sh.hist[i] = 0;
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
  auto total = [&](uint64_t v) {
    const uint64_t* const g = gather(block_sum(v));
    uint64_t s = 0;
    for (uint32_t c = 0; c < C; ++c) s += g[c];
    return s;
  };
  constexpr int kAhead = sizeof(T) == 4 ? 4 : 8;   // loads of a thread in flight
  constexpr float kLog2e = 1.4426950408889634f;
  const double per_t = 1.0 / (double)temp, c64 = 32.0 * 1.4426950408889634 * per_t, c_all = 1.4426950408889634 * per_t;
  const float ch = (float)c_all, cl = (float)(c_all - (double)ch);
  const int strips = (r.vecs + kThreads - 1) / kThreads;
  // Weights in fp32, relative to `largest`, from the approximate exponential (relative error 2^-22), whose argument is carried in two parts and
  // whose product with the rest rounds twice (2^-23).
  auto weights32 = [&](const float (&f)[8], float largest, float (&w)[8]) {
    const float floor_d = -200.f / ch;           // (what lies further down weighs 0, as this does)
    const uint64_t ch2 = two(ch, ch), cl2 = two(cl, cl), top2 = two(-largest, -largest), ln2 = two(0.6931471805599453f, 0.6931471805599453f), minus = two(-1.f, -1.f);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      float d0, d1, y0, y1;
      untwo(add2(two(f[2 * q], f[2 * q + 1]), top2), d0, d1);
      const uint64_t d = two(fmaxf(d0, floor_d), fmaxf(d1, floor_d)), y = mul2(d, ch2);
      const uint64_t rest = fma2(d, cl2, fma2(d, ch2, mul2(y, minus)));
      untwo(y, y0, y1);
      const uint64_t e = two(ex2(y0), ex2(y1));
      untwo(fma2(e, mul2(rest, ln2), e), w[2 * q], w[2 * q + 1]);
    }
  };
  auto add8 = [](const float (&w)[8]) { return ((w[0] + w[1]) + (w[2] + w[3])) + ((w[4] + w[5]) + (w[6] + w[7])); };
  // How far a sum of such weights and u times their whole may lie from one another's true place: every weight is within e = 2^-20.7 (2^-22, 2^-23,
  // three roundings of 2^-24 where eight are added) of itself, those before the place count 1 - u times and those behind it u times.
  auto slack_of = [&](double all) { const double v = u > 0.f ? (u < 1.f ? (double)u : 1.0) : 0.0; return all * (2.0 * v * (1.0 - v) * 5.9e-7 + 1e-11); };
  double lp_sum = 0.0;                           // of exp(x - this block's largest), for the log-probability
  float top, mine_top;
  int token = -1;
  double* const sums_d = (double*)sh.sums;
  // The element of a warp's part q of a strip at which the sum passes t (all given relative to `largest` of that part), by a warp; -1: too near a border.
  auto within = [&](int q, double before, double t, double slack, auto weights) -> int {
    const int v = q / kWarps * kThreads + q % kWarps * 32 + lane;
    float w[8];
    if (v < r.vecs) weights(v, w);
    else {
#pragma unroll
      for (int e = 0; e < 8; ++e) w[e] = 0.f;
    }
    double s = 0.0;
#pragma unroll
    for (int e = 0; e < 8; ++e) s += (double)w[e];
    double upto = s;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double n = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += n;
    }
    double run = before + upto - s;
    int at = -1;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if (at < 0 && run + slack < t && t < run + (double)w[e] - slack) at = r.index(v, e);
      run += (double)w[e];
    }
    const uint32_t hit = __ballot_sync(0xffffffffu, at >= 0);
    return hit ? __shfl_sync(0xffffffffu, at, __ffs(hit) - 1) : -1;
  };
  // The part at which the running sum of sums_d passes t, by a warp; *before = the sum before it; -1: none.
  auto part_of = [&](double t, double* before) -> int {
    double b = *before;
    for (int q0 = 0; q0 < strips * kWarps; q0 += 32) {
      const double x = q0 + lane < strips * kWarps ? sums_d[q0 + lane] : 0.0;
      double upto = x;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const double n = __shfl_up_sync(0xffffffffu, upto, o);
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
  auto block_sum_d = [&](double v) {
    v = warp_sum(v);
    __syncthreads();
    if (lane == 0) sh.red_d[warp] = v;
    __syncthreads();
    return warp_sum(lane < kWarps ? sh.red_d[lane] : 0.0);
  };
  {
    // ---- the row's largest; where the row is read once, sums of the weights too ----
    r.held = nullptr;
    const bool hold = !greedy && !once && r.vecs * 8 * (int)sizeof(T) <= held_bytes;
    uint64_t best = 0;                           // pattern, V - 1 - index
    for (int v0 = tid; v0 < strips * kThreads; v0 += kAhead * kThreads) {   // (by whole warps)
      typename Row<T>::Raw got[kAhead];
#pragma unroll
      for (int q = 0; q < kAhead; ++q)
        if (v0 + q * kThreads < r.vecs) got[q] = r.load_raw(v0 + q * kThreads);
#pragma unroll
      for (int q = 0; q < kAhead; ++q) {
        const int v = v0 + q * kThreads;
        if (v - lane >= r.vecs) continue;
        float f[8];
        if (v < r.vecs) {
          Row<T>::unpack(got[q], f);
#pragma unroll
          for (int e = 0; e < 8; ++e) f[e] = clean(f[e]);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) f[e] = -INFINITY;
        }
        float mx = f[0];
#pragma unroll
        for (int e = 1; e < 8; ++e) mx = fmaxf(mx, f[e]);
        if (hold && v < r.vecs) {
          alignas(16) T e8[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) e8[e] = (T)f[e];
#pragma unroll
          for (int x = 0; x < Row<T>::W; ++x) *(uint4*)(held + v * (16 * Row<T>::W) + 16 * x) = ((const uint4*)e8)[x];
        }
        if (once) {
          const uint32_t key = __reduce_max_sync(0xffffffffu, pattern(mx));
          const float largest = value_of(key);
          double t = 0.0;
          if (largest > -INFINITY && largest < INFINITY) {
            float w[8];
            weights32(f, largest, w);
            t = warp_sum((double)add8(w));
          }
          const int part = v / kThreads * kWarps + warp;
          if (lane == 0) { sums_d[part] = t; sh.refs[part] = largest; }
          best = max(best, (uint64_t)key << 32);
        } else {
          int at = 0;
#pragma unroll
          for (int e = 7; e >= 0; --e) at = f[e] == mx ? e : at;
          const int index = r.index(v, at);
          best = max(best, (uint64_t)pattern(mx) << 32 | (uint32_t)(index >= 0 && index < V ? V - 1 - index : 0));
        }
      }
    }
    if (hold) r.held = held;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) best = max(best, (uint64_t)__shfl_xor_sync(0xffffffffu, best, o));
    __syncthreads();
    if (lane == 0) sh.red[warp] = best;
    __syncthreads();
    best = lane < kWarps ? sh.red[lane] : 0;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) best = max(best, (uint64_t)__shfl_xor_sync(0xffffffffu, best, o));
    mine_top = r.vecs > 0 ? value_of((uint32_t)(best >> 32)) : -INFINITY;
    double mine = 0.0;
    if (once) {
      // parts relative to the block's largest (both below infinity, else the row is not decided here)
      for (int q = tid; q < strips * kWarps; q += kThreads) {
        const int v = q / kWarps * kThreads + q % kWarps * 32;
        const float ref = v < r.vecs ? sh.refs[q] : -INFINITY;
        const double w = ref > -INFINITY && mine_top < INFINITY ? sums_d[q] * exp2(((double)ref - (double)mine_top) * c_all) : 0.0;
        sums_d[q] = w;
        mine += w;
      }
      mine = block_sum_d(mine);
    }
    if (a.logprobs) {
      // (the row is in shared memory, or has just been read)
      for (int v = tid; v < r.vecs; v += kThreads) {
        float f[8], t = 0.f;
        r.load8(v, f);
#pragma unroll
        for (int e = 0; e < 8; ++e) t += f[e] == mine_top ? 1.f : ex2((f[e] - mine_top) * kLog2e);
        lp_sum += (double)t;
      }
      lp_sum = block_sum_d(lp_sum);
      if (tid == 0) put64((uint64_t*)&sh.part[me], 0, (uint64_t)__double_as_longlong(lp_sum));
      if (tid == 32) put64((uint64_t*)&sh.part_top[me], 0, (uint64_t)__double_as_longlong((double)mine_top));
    }
    if (once && tid < (int)C) put64((uint64_t*)&sh.once_sum[me], (uint32_t)tid, (uint64_t)__double_as_longlong(mine));
    const uint64_t* const g = gather(best);
    for (uint32_t c = 0; c < C; ++c) best = max(best, g[c]);
    top = value_of((uint32_t)(best >> 32));
    if (greedy && top > -INFINITY) token = V - 1 - (int)(uint32_t)best;
    if (once && top > -INFINITY && top < INFINITY) {
      double all = 0.0, part[kMaxCtas];
#pragma unroll
      for (uint32_t c = 0; c < kMaxCtas; ++c) {
        part[c] = 0.0;
        if (c < C) {
          const float ref = value_of((uint32_t)(g[c] >> 32));
          part[c] = g[c] && ref > -INFINITY ? sh.once_sum[c] * exp2(((double)ref - (double)top) * c_all) : 0.0;
          all += part[c];
        }
      }
      const double slack = slack_of(all), t = u > 0.f ? (u < 1.f ? (double)u * all : all) : 0.0;
      uint32_t who = C;
      double before = 0.0, run = 0.0;
#pragma unroll
      for (uint32_t c = 0; c < kMaxCtas; ++c) {
        if (c < C && who == C && t < run + part[c]) { who = c; before = run; }
        run += part[c];
      }
      if (who == C) who = C - 1;
      if (who == me && warp == 0) {
        // everything relative to this block's largest
        const double up = exp2(((double)top - (double)mine_top) * c_all);
        double b = before * up;
        const int q = mine_top > -INFINITY ? part_of(t * up, &b) : -1;
        int at = -1;
        if (q >= 0) {
          const double there = exp2(((double)mine_top - (double)sh.refs[q]) * c_all);
          at = within(q, b * there, t * up * there, slack * up * there, [&](int v, float (&w)[8]) {
            float f[8];
            r.load8(v, f);
            weights32(f, sh.refs[q], w);
          });
        }
        if (lane < (int)C) put32(&sh.answer[0], (uint32_t)lane, (uint32_t)at);
      }
      cluster_sync_all();
      token = sh.answer[0];
    }
  }
  const bool nothing = top == -INFINITY;
  const double top64 = top;
  auto weigh = [&](float x) -> uint64_t {        // (of an infinite temperature: all alike)
    if (x == top) return (uint64_t)kOne;
    if (x == -INFINITY || top == INFINITY) return 0;
    return weight64((double)x - top64, c64, sh.roots);
  };
  auto enough = [&](float x) { return !(least > 0.f) || x == top || exp(((double)x - (double)top) * per_t) >= (double)least; };

  // The first index at which the sum of `amount` passes `target(whole sum)`, all blocks' answer; *whole = the sum.
  auto find = [&](auto amount, auto target, uint64_t* whole) -> int {
    uint64_t mine = 0;
    for (int s = 0; s < strips; ++s) {
      const int v = s * kThreads + tid;
      uint64_t t = 0;
      if (v < r.vecs) {
        float f[8];
        r.load8(v, f);
#pragma unroll
        for (int e = 0; e < 8; ++e) t += amount(f[e], r.index(v, e));
      }
      t = warp_sum(t);
      if (lane == 0) sh.sums[s * kWarps + warp] = t;
      mine += t;
    }
    __syncthreads();
    if (lane == 0) sh.red[warp] = mine;
    __syncthreads();
    const uint64_t* const g = gather(warp_sum(lane < kWarps ? sh.red[lane] : (uint64_t)0));
    uint64_t all = 0;
    for (uint32_t c = 0; c < C; ++c) all += g[c];
    *whole = all;
    uint64_t t = target(all);
    uint32_t who = 0;
    while (who + 1 < C && t >= g[who]) t -= g[who++];
    if (who == me && warp == 0) {                            // the warp's part of a strip, the lane, the element
      int q = 0;
      uint64_t before = 0;
      for (int q0 = 0; q0 < strips * kWarps; q0 += 32) {
        const uint64_t x = q0 + lane < strips * kWarps ? sh.sums[q0 + lane] : 0;
        uint64_t upto = x;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const uint64_t n = __shfl_up_sync(0xffffffffu, upto, o);
          if (lane >= o) upto += n;
        }
        const uint32_t hit = __ballot_sync(0xffffffffu, before + upto > t);
        if (hit) {
          const int l = __ffs(hit) - 1;
          q = q0 + l;
          before += __shfl_sync(0xffffffffu, upto - x, l);
          break;
        }
        before += __shfl_sync(0xffffffffu, upto, 31);
        q = q0 + 31;
      }
      const int v = q / kWarps * kThreads + q % kWarps * 32 + lane;
      float f[8];
      uint64_t w[8], s = 0;
      if (v < r.vecs) r.load8(v, f);
#pragma unroll
      for (int e = 0; e < 8; ++e) { w[e] = v < r.vecs ? amount(f[e], r.index(v, e)) : 0; s += w[e]; }
      uint64_t upto = s;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint64_t n = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += n;
      }
      uint64_t run = before + upto - s;
      int at = -1;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if (at < 0 && run + w[e] > t) at = r.index(v, e);
        run += w[e];
      }
      const uint32_t hit = __ballot_sync(0xffffffffu, at >= 0);
      at = hit ? __shfl_sync(0xffffffffu, at, __ffs(hit) - 1) : V - 1;
      if (lane < (int)C) put32(&sh.answer[0], (uint32_t)lane, (uint32_t)at);
    }
    cluster_sync_all();
    return sh.answer[0];
  };
  // The token among those of which `stay(x, i)` says so, by weights in fp32.  -1 where the place to find lies too near an element's border (or a weight
  // too near min_p): then the whole numbers decide.
  auto find_fast = [&](auto stay) -> int {
    auto weights = [&](int v, float (&w)[8]) {
      float f[8];
      r.load8(v, f);
      weights32(f, top, w);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if (least > 0.f) {
          const float off = w[e] - least;
          if (fabsf(off) <= least * 1.9073486328125e-6f && f[e] != top) w[e] = __uint_as_float(0x7fc00000u);    // 2^-19
          else if (off < 0.f && f[e] != top) w[e] = 0.f;
        }
        if (!stay(f[e], r.index(v, e))) w[e] = 0.f;
      }
    };
    double mine = 0.0;
    for (int s = 0; s < strips; ++s) {
      const int v = s * kThreads + tid;
      double t = 0.0;
      if (v < r.vecs) {
        float w[8];
        weights(v, w);
        t = (double)add8(w);
      }
      t = warp_sum(t);
      if (lane == 0) sums_d[s * kWarps + warp] = t;
      mine += t;
    }
    __syncthreads();
    if (lane == 0) sh.red_d[warp] = mine;
    __syncthreads();
    mine = warp_sum(lane < kWarps ? sh.red_d[lane] : 0.0);
    const uint64_t* const g = gather((uint64_t)__double_as_longlong(mine));
    double all = 0.0;
    for (uint32_t c = 0; c < C; ++c) all += __longlong_as_double((long long)g[c]);
    const double t = u > 0.f ? (u < 1.f ? (double)u * all : all) : 0.0;
    uint32_t who = 0;
    double before = 0.0;
    for (; who + 1 < C; ++who) {
      const double n = __longlong_as_double((long long)g[who]);
      if (t < before + n) break;
      before += n;
    }
    if (who == me && warp == 0) {
      const int q = part_of(t, &before);
      const int at = q >= 0 ? within(q, before, t, slack_of(all), weights) : -1;
      if (lane < (int)C) put32(&sh.answer[0], (uint32_t)lane, (uint32_t)at);
    }
    cluster_sync_all();
    return sh.answer[0];
  };
  auto sum_of = [&](auto amount) {
    uint64_t s = 0;
    for (int v = tid; v < r.vecs; v += kThreads) {
      float f[8];
      r.load8(v, f);
#pragma unroll
      for (int e = 0; e < 8; ++e) s += amount(f[e], r.index(v, e));
    }
    return total(s);
  };
  auto stays = [&](const Border& b, float x, int i) { return pattern(x) > b.key || (pattern(x) == b.key && i <= b.index); };
  // The border at which the amounts of what stays before it reach `target`, of what stays at `from`: by halving.
  auto border = [&](auto amount, uint64_t target, const Border& from) {
    uint32_t lo = 0, hi = pattern(top);          // the largest key whose sum from there up reaches the target
    while (lo < hi) {
      const uint32_t mid = lo + (hi - lo) / 2 + 1;
      if (sum_of([&](float x, int i) { return pattern(x) >= mid && stays(from, x, i) ? amount(x) : 0ull; }) >= target) lo = mid; else hi = mid - 1;
    }
    const uint64_t above = sum_of([&](float x, int i) { return pattern(x) > lo && stays(from, x, i) ? amount(x) : 0ull; });
    const uint64_t each = amount(value_of(lo));
    Border b = {lo, V - 1};
    if (each > 0) {                              // among equal ones, the first so many by index
      const uint64_t n = (target - above + each - 1) / each;
      uint64_t all;
      b.index = find([&](float x, int i) { return (uint64_t)(pattern(x) == lo && stays(from, x, i)); }, [&](uint64_t) { return n - 1; }, &all);
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
      for (int v = tid; v < r.vecs; v += kThreads) {
        float f[8];
        r.load8(v, f);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int bin = bin_of(f[e]);
          if (bin < kBins) atomicAdd(&sh.hist[bin], 1u);
        }
      }
      cluster_sync_all();
      const int each = kBins / (int)C;           // every block adds its part of the bins, for all
      for (int i = tid; i < each; i += kThreads) {
        const int bin = (int)me * each + i;
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
      if (tid < 4) sh.answer[tid] = -1;
      __syncthreads();
      uint32_t before = upto - mine, in_range = 0;
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
      int last_bin = sh.answer[0], list_n = sh.answer[1], first_bin = 0;                  // of the list
      const int k_bin = last_bin, k_before = sh.answer[2];
      const bool cut = want < in_range;                      // top-k leaves something out
      bool few = list_n <= kList;                            // all that may stay fits the list
      bool by_list = few;
      uint64_t above = 0, whole = 0;
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
        cluster_sync_all();
        if (tid == 0) sh.staged = 0;
        __syncthreads();
      };
      auto into_list = [&](int lo, int hi) {
        for (int v = tid; v < r.vecs; v += kThreads) {
          float f[8];
          r.load8(v, f);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const int bin = bin_of(f[e]);
            if (bin >= lo && bin <= hi && bin < kBins) enlist(f[e], r.index(v, e));
          }
        }
        deliver();
      };
      constexpr int LPT = kList / kThreads;      // neighbours of a thread
      // The first n entries of the list in descending order, by the first block: bitonic, an entry's partner in the same thread, in the same
      // warp, or through shared memory (ten of 55 steps for 1024).  What fills up the power of two is 0.
      auto sort_list = [&](int n) {
        int m = LPT * 32;
        while (m < n) m *= 2;
        uint64_t x[LPT];
#pragma unroll
        for (int q = 0; q < LPT; ++q) x[q] = LPT * tid + q < n ? sh.list[LPT * tid + q] : 0;
        for (int span = 2; span <= m; span *= 2)
          for (int d = span / 2; d > 0; d /= 2) {
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
            } else if (d < LPT * 32) {
              const bool first = (lane & (d / LPT)) == 0;
#pragma unroll
              for (int q = 0; q < LPT; ++q) {
                const uint64_t y = __shfl_xor_sync(0xffffffffu, x[q], d / LPT);
                const bool larger = (((LPT * tid + q) & span) == 0) == first;
                x[q] = (x[q] < y) == larger ? y : x[q];
              }
            } else {
              __syncthreads();
#pragma unroll
              for (int q = 0; q < LPT; ++q) sh.list[LPT * tid + q] = x[q];
              __syncthreads();
              const bool first = (LPT * tid & d) == 0;
#pragma unroll
              for (int q = 0; q < LPT; ++q) {
                const uint64_t y = sh.list[(LPT * tid + q) ^ d];
                const bool larger = (((LPT * tid + q) & span) == 0) == first;
                x[q] = (x[q] < y) == larger ? y : x[q];
              }
            }
          }
        __syncthreads();
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
        for (int x = 0; x < kWarps; ++x) { if (x < warp) base += sh.red[x]; sum += sh.red[x]; }
#pragma unroll
        for (int q = 0; q < LPT; ++q) before[q] += base;
        *all = sum;
      };
      auto list_value = [&](int i) { return value_of((uint32_t)(sh.list[i] >> 32)); };
      auto list_index = [&](int i) { return V - 1 - (int)(uint32_t)sh.list[i]; };
      // the element at which the sum of the list's amounts, in order, reaches `target`; by the first block, told to all
      auto in_list = [&](auto amount, uint64_t target) {
        if (me == 0) {
          const int n = (int)min(sh.listed, (uint32_t)kList);
          sort_list(n);
          uint64_t w[LPT], before[LPT], all;
#pragma unroll
          for (int q = 0; q < LPT; ++q) w[q] = LPT * tid + q < n ? amount(list_value(LPT * tid + q)) : 0;
          list_sums(w, before, &all);
#pragma unroll
          for (int q = 0; q < LPT; ++q) {
            const int i = LPT * tid + q;
            if (i < n && before[q] < target && target <= before[q] + w[q])
              for (uint32_t c = 0; c < C; ++c) { put32(&sh.answer[2], c, (uint32_t)(sh.list[i] >> 32)); put32(&sh.answer[3], c, (uint32_t)list_index(i)); }
          }
        }
        cluster_sync_all();
      };
      if (few) {
        // ---- all that may stay is in the list: the first block draws the token ----
        into_list(0, last_bin);
        if (me == 0) {
          const int n = list_n;
          sort_list(n);
          uint64_t w[LPT], before[LPT], Z;
#pragma unroll
          for (int q = 0; q < LPT; ++q) w[q] = LPT * tid + q < n && (uint32_t)(LPT * tid + q) < want ? weigh(list_value(LPT * tid + q)) : 0;
          list_sums(w, before, &Z);
          uint64_t target = ~0ull;
          if (by_p) {
            target = p > 0.f ? (uint64_t)ceil((double)p * (double)Z) : 1ull;
            target = target < 1 ? 1 : target;
          }
          // what stays is a first part of the order: how long, and back by index
          int stay = 0;
#pragma unroll
          for (int q = 0; q < LPT; ++q) {
            const int i = LPT * tid + q;
            if (w[q] > 0 && before[q] < target && enough(list_value(i))) stay = i + 1;
          }
          stay = __reduce_max_sync(0xffffffffu, stay);
          __syncthreads();
          if (lane == 0) sh.red[warp] = (uint64_t)stay;
          __syncthreads();
          for (int x = 0; x < kWarps; ++x) stay = max(stay, (int)sh.red[x]);
          uint64_t turned[LPT];
#pragma unroll
          for (int q = 0; q < LPT; ++q) turned[q] = LPT * tid + q < stay ? sh.list[LPT * tid + q] : 0;
          __syncthreads();
#pragma unroll
          for (int q = 0; q < LPT; ++q)
            if (LPT * tid + q < stay) sh.list[LPT * tid + q] = turned[q] << 32 | turned[q] >> 32;      // V - 1 - index, pattern
          sort_list(stay);
#pragma unroll
          for (int q = 0; q < LPT; ++q) w[q] = LPT * tid + q < stay ? weigh(value_of((uint32_t)sh.list[LPT * tid + q])) : 0;
          list_sums(w, before, &Z);
          uint64_t t = u > 0.f ? (u < 1.f ? (uint64_t)((double)u * (double)Z) : Z) : 0;
          t = t < Z ? t : Z - 1;
#pragma unroll
          for (int q = 0; q < LPT; ++q)
            if (before[q] <= t && t < before[q] + w[q])
              for (uint32_t c = 0; c < C; ++c) put32(&sh.answer[0], c, (uint32_t)(V - 1 - (int)(uint32_t)(sh.list[LPT * tid + q] >> 32)));
        }
        cluster_sync_all();
        token = sh.answer[0];
      } else {
        if (cut) {
          if (list_n - k_before <= kList) {
            into_list(k_bin, k_bin);
            in_list([](float) { return 1ull; }, (uint64_t)(want - (uint32_t)k_before));
            b = {(uint32_t)sh.answer[2], sh.answer[3]};
          } else b = border([](float) { return 1ull; }, (uint64_t)want, b);
        }
        if (by_p) {
          // where it should lie by the steps' mean weights
          __syncthreads();
          double est[PER], sum = 0.0;
#pragma unroll
          for (int i = 0; i < PER; ++i) {
            const int bin = tid * PER + i;
            const uint32_t n = bin < k_bin ? cnt[i] : (bin == k_bin ? want - (uint32_t)k_before : 0u);
            est[i] = (double)n * (double)exp2f(-((float)bin + 0.5f) * (kRange / (float)kBins * 1.4426950408889634f));
            sum += est[i];
          }
          double upto_d = sum;
#pragma unroll
          for (int o = 1; o < 32; o <<= 1) {
            const double n = __shfl_up_sync(0xffffffffu, upto_d, o);
            if (lane >= o) upto_d += n;
          }
          if (lane == 31) sh.red_d[warp] = upto_d;
          if (tid == 0) sh.answer[0] = k_bin;
          __syncthreads();
          double run = upto_d - sum, all = 0.0;
          for (int w = 0; w < kWarps; ++w) { if (w < warp) run += sh.red_d[w]; all += sh.red_d[w]; }
          const double t = (double)p * all;
#pragma unroll
          for (int i = 0; i < PER; ++i) {
            if (run < t && t <= run + est[i]) sh.answer[0] = tid * PER + i;
            run += est[i];
          }
          __syncthreads();
          first_bin = sh.answer[0] > 0 ? sh.answer[0] - 1 : 0;
          last_bin = sh.answer[0] + 1 < kBins ? sh.answer[0] + 1 : kBins - 1;
          list_n = 0;
          for (int i = first_bin; i <= last_bin; ++i) list_n += (int)sh.merged[i];
          // (the three sums and the list in one pass)
          uint64_t s_above = 0, s_list = 0, s_rest = 0;
          by_list = list_n <= kList;
          for (int v = tid; v < r.vecs; v += kThreads) {
            float f[8];
            r.load8(v, f);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              if (!stays(b, f[e], r.index(v, e))) continue;
              const int bin = bin_of(f[e]);
              const uint64_t w = weigh(f[e]);
              if (bin < first_bin) s_above += w;
              else if (bin > last_bin) s_rest += w;
              else {
                s_list += w;
                if (by_list) enlist(f[e], r.index(v, e));
              }
            }
          }
          if (by_list) deliver();
          above = total(s_above);
          const uint64_t inside = total(s_list);
          whole = above + inside + total(s_rest);
          uint64_t target = p > 0.f ? (uint64_t)ceil((double)p * (double)whole) : 1;
          target = target < 1 ? 1 : (target > whole ? whole : target);
          by_list = by_list && above < target && target <= above + inside;
          if (by_list) {
            in_list(weigh, target - above);
            b = {(uint32_t)sh.answer[2], sh.answer[3]};
          } else b = border(weigh, target, b);
        }
      }
    }
    // (at temperatures like these -200 / c, which stands in for all that lies further down, weighs 0 and is itself exact enough)
    if (token < 0 && !once && top < INFINITY && temp >= 1e-6f && temp <= 1e6f) token = find_fast([&](float x, int i) { return !(by_k || by_p) || stays(b, x, i); });
    if (token < 0) {
      uint64_t Z;
      token = find([&](float x, int i) { return stays(b, x, i) && enough(x) ? weigh(x) : 0ull; },
                   [&](uint64_t whole) {
                     const uint64_t t = u > 0.f ? (u < 1.f ? (uint64_t)((double)u * (double)whole) : whole) : 0;
                     return t < whole ? t : whole - 1;
                   }, &Z);
    }
  }
  if (a.logprobs && me == 0 && tid == 0) {
    float y = 0.f;
    if (!nothing) {
      double all = 0.0;
      for (uint32_t c = 0; c < C; ++c) {
        const double ref = sh.part_top[c];
        if (ref > -INFINITY) all += ref == top64 ? sh.part[c] : sh.part[c] * exp(ref - top64);
      }
      const float x = clean(IO<T>::load((const char*)a.logits + (int64_t)row_no * a.row_bytes, token));
      y = (float)((x == top ? 0.0 : (double)x - top64) - log(all));
    }
    a.logprobs[row_no] = y;
  }
  if (me == 0 && tid == 0) a.tokens[row_no] = token;
  cluster_sync_all();                            // (shared memory stays until all have read it)
}

template <typename T> cudaError_t launch_t(const SampleArgs& a, cudaStream_t st) {
  auto kern = sample_kernel<T>;
  static bool done[64] = {};
  constexpr int kHeld = 96 * 1024;               // of a row's share at most: two blocks an SM
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
  // Blocks a row: enough that there are two for every SM, of at least 8192 elements each.  (What the blocks of a row say to one another takes 0.7 us
  // each time, so that many rows are better off with a block or two each; one row of 128256 takes 23 us by one, 13 by eight.)
  int ctas = 1;
  while (ctas < kMaxCtas && (int64_t)a.N * ctas < 2 * sm_count() && a.V > ctas * 2 * kStrip) ctas *= 2;
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
