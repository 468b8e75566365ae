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
  double part[kMaxCtas];                       // of the sum for the log-probability
  double roots[32];
  uint64_t above, whole;
  union {                                      // (never of use at the same time)
    uint64_t list[kList];                      // pattern, then V - 1 - index: larger ones come first in the order
    uint64_t sums[kMaxStrips * kWarps];        // of every warp's part of every strip
  };
  uint32_t hist[kBins], merged[kBins];
  uint32_t scan[kWarps];
  uint32_t listed;
  int answer[4];
};

static_assert(sizeof(Shared) % 16 == 0 && offsetof(Shared, hist) % 8 == 0, "vectors behind it, weights in it");

template <typename T> struct Row {
  const T* x;                  // this block's share
  const unsigned char* held;   // the same in shared memory, element e of it at place e + off; null: read from memory
  int begin, n, off, vecs;
  // eight elements from place 8 v on; -inf where the row has none
  __device__ __forceinline__ void load8(int v, float (&f)[8]) const {
    if (held) {
      if constexpr (sizeof(T) == 4) {
        const float4 a = *(const float4*)(held + v * 32), b = *(const float4*)(held + v * 32 + 16);
        f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w; f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
      } else {
        const uint4 a = *(const uint4*)(held + v * 16);
        const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          if constexpr (std::is_same<T, __half>::value) {
            const float2 h = __half22float2(*(const __half2*)&w[k]);
            f[2 * k] = h.x; f[2 * k + 1] = h.y;
          } else { f[2 * k] = bf16lo(w[k]); f[2 * k + 1] = bf16hi(w[k]); }
        }
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int i = 8 * v + e - off;
        f[e] = i >= 0 && i < n ? clean(IO<T>::load(x, i)) : -INFINITY;
      }
    }
  }
  __device__ __forceinline__ int index(int v, int e) const { return begin + 8 * v + e - off; }
};

template <typename T>
__global__ void __launch_bounds__(kThreads) sample_kernel(const __grid_constant__ SampleArgs a, int share, int held_bytes) {
  extern __shared__ __align__(16) unsigned char raw[];
  Shared& sh = *(Shared*)raw;
  const uint32_t C = cluster_size(), me = cluster_rank();
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
  r.held = r.vecs * 8 * (int)sizeof(T) <= held_bytes ? held : nullptr;
  float mx = -INFINITY;
  for (int v = tid; v < r.vecs; v += kThreads) {
    const int i0 = 8 * v - r.off;
    alignas(16) T raw8[8];
    if (i0 >= 0 && i0 + 8 <= r.n) {
#pragma unroll
      for (int q = 0; q < (int)sizeof(T) / 2; ++q) ((uint4*)raw8)[q] = ((const uint4*)(r.x + i0))[q];
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) raw8[e] = i0 + e >= 0 && i0 + e < r.n ? r.x[i0 + e] : (T)(-INFINITY);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float f = clean((float)raw8[e]);
      mx = fmaxf(mx, f);
      raw8[e] = (T)f;
    }
    if (r.held) {
#pragma unroll
      for (int q = 0; q < (int)sizeof(T) / 2; ++q) *(uint4*)(held + v * 8 * sizeof(T) + 16 * q) = ((const uint4*)raw8)[q];
    }
  }
  if (tid == 0) sh.listed = 0;
  if (tid < 32) sh.roots[tid] = kRoots[tid];
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
  float top;
  {
    const uint32_t w = __reduce_max_sync(0xffffffffu, pattern(mx));
    if (lane == 0) sh.red[warp] = w;
    __syncthreads();
    const uint32_t b = __reduce_max_sync(0xffffffffu, lane < kWarps ? (uint32_t)sh.red[lane] : 0u);
    const uint64_t* const g = gather(b);
    uint32_t key = 0;
    for (uint32_t c = 0; c < C; ++c) key = max(key, (uint32_t)g[c]);
    top = value_of(key);
  }
  const bool greedy = !(temp > 0.f), nothing = top == -INFINITY;
  const double per_t = 1.0 / (double)temp, c64 = 32.0 * 1.4426950408889634 * per_t, top64 = top;
  auto weigh = [&](float x) -> uint64_t {        // (of an infinite temperature: all alike)
    if (x == top) return (uint64_t)kOne;
    if (x == -INFINITY || top == INFINITY) return 0;
    return weight64((double)x - top64, c64, sh.roots);
  };
  auto enough = [&](float x) { return !(least > 0.f) || x == top || exp(((double)x - (double)top) * per_t) >= (double)least; };

  // The first index at which the sum of `amount` passes `target(whole sum)`, all blocks' answer; *whole = the sum.
  auto find = [&](auto amount, auto target, uint64_t* whole) -> int {
    const int strips = (r.vecs + kThreads - 1) / kThreads;
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
  // The token among those of which `stay(x, i)` says so, by weights in fp32 from the approximate exponential (relative error 2^-22), whose argument is
  // carried in two parts: eight of them are added in fp32 (three roundings of 2^-24), the rest in 64 bits, so that every sum is within
  // 2^-20 of itself.  -1 where the place to find lies within that of an element's border (or a weight that near min_p): then the whole numbers decide.
  auto find_fast = [&](auto stay) -> int {
    const double c = 1.4426950408889634 * per_t;
    const float ch = (float)c, cl = (float)(c - (double)ch), floor_d = fmaxf(-200.f / ch, -1e30f);
    const uint64_t ch2 = two(ch, ch), cl2 = two(cl, cl), top2 = two(-top, -top), ln2 = two(0.6931471805599453f, 0.6931471805599453f), minus = two(-1.f, -1.f);
    auto weights = [&](const float (&f)[8], int v, float (&w)[8]) {
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
    const int strips = (r.vecs + kThreads - 1) / kThreads;
    double* const sums = (double*)sh.sums;
    double mine = 0.0;
    for (int s = 0; s < strips; ++s) {
      const int v = s * kThreads + tid;
      double t = 0.0;
      if (v < r.vecs) {
        float f[8], w[8];
        r.load8(v, f);
        weights(f, v, w);
        t = (double)(((w[0] + w[1]) + (w[2] + w[3])) + ((w[4] + w[5]) + (w[6] + w[7])));
      }
      t = warp_sum(t);
      if (lane == 0) sums[s * kWarps + warp] = t;
      mine += t;
    }
    __syncthreads();
    if (lane == 0) sh.red_d[warp] = mine;
    __syncthreads();
    mine = warp_sum(lane < kWarps ? sh.red_d[lane] : 0.0);
    const uint64_t* const g = gather((uint64_t)__double_as_longlong(mine));
    double all = 0.0;
    for (uint32_t c1 = 0; c1 < C; ++c1) all += __longlong_as_double((long long)g[c1]);
    const double slack = all * 9.5367431640625e-7;           // 2^-20
    double t = u > 0.f ? (u < 1.f ? (double)u * all : all) : 0.0;
    uint32_t who = 0;
    double before = 0.0;
    for (; who + 1 < C; ++who) {
      const double n = __longlong_as_double((long long)g[who]);
      if (t < before + n) break;
      before += n;
    }
    if (who == me && warp == 0) {
      int q = 0;
      bool found = false;
      for (int q0 = 0; q0 < strips * kWarps && !found; q0 += 32) {
        const double x = q0 + lane < strips * kWarps ? sums[q0 + lane] : 0.0;
        double upto = x;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const double n = __shfl_up_sync(0xffffffffu, upto, o);
          if (lane >= o) upto += n;
        }
        const uint32_t hit = __ballot_sync(0xffffffffu, before + upto > t);
        if (hit) {
          const int l = __ffs(hit) - 1;
          q = q0 + l;
          before += __shfl_sync(0xffffffffu, upto - x, l);
          found = true;
        } else before += __shfl_sync(0xffffffffu, upto, 31);
      }
      const int v = q / kWarps * kThreads + q % kWarps * 32 + lane;
      float f[8], w[8];
      if (found && v < r.vecs) { r.load8(v, f); weights(f, v, w); }
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
      for (int e = 0; e < 8; ++e) {              // (the first element of the row begins at 0 exactly, the last one ends at the whole)
        if (at < 0 && run + slack < t && t < run + (double)w[e] - slack) at = r.index(v, e);
        run += (double)w[e];
      }
      const uint32_t hit = __ballot_sync(0xffffffffu, at >= 0);
      at = hit ? __shfl_sync(0xffffffffu, at, __ffs(hit) - 1) : -1;
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

  int token = -1;
  if (greedy && !nothing) {
    uint64_t all;
    token = find([&](float x, int) { return (uint64_t)(x == top); }, [](uint64_t) { return 0ull; }, &all);
  } else if (!nothing) {
    Border b = {0u, V - 1};
    const bool by_k = k > 0 && k < V, by_p = p < 1.f;
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
      auto into_list = [&](int lo, int hi, const Border* from) {
        for (int v = tid; v < r.vecs; v += kThreads) {
          float f[8];
          r.load8(v, f);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const int bin = bin_of(f[e]);
            if (bin >= lo && bin <= hi && bin < kBins && (from == nullptr || stays(*from, f[e], r.index(v, e)))) {
              const uint32_t at = add32(&sh.listed, 0, 1u);
              if (at < kList) put64(&sh.list[at], 0, (uint64_t)pattern(f[e]) << 32 | (uint32_t)(V - 1 - r.index(v, e)));   // (larger first: larger logit, then lower index)
            }
          }
        }
        cluster_sync_all();
      };
      // the element at which the sum of the list's amounts, in order, reaches `target`; by the first block, told to all
      auto in_list = [&](auto amount, uint64_t target) {
        if (me == 0) {
          const int n = (int)min(sh.listed, (uint32_t)kList);
          uint64_t* const weight = (uint64_t*)sh.hist;       // (the histogram has been added up)
          static_assert(kList * 8 <= sizeof(sh.hist), "weights");
          for (int i = tid; i < n; i += kThreads) weight[i] = amount(value_of((uint32_t)(sh.list[i] >> 32)));
          __syncthreads();
          for (int i = tid; i < n; i += kThreads) {
            const uint64_t x = sh.list[i], w = weight[i];
            uint64_t sum = 0;
#pragma unroll 4
            for (int j = 0; j < n; ++j) sum += sh.list[j] > x ? weight[j] : 0ull;
            if (sum < target && target <= sum + w)
              for (uint32_t c = 0; c < C; ++c) { put32(&sh.answer[2], c, (uint32_t)(x >> 32)); put32(&sh.answer[3], c, (uint32_t)(V - 1 - (int)(uint32_t)x)); }
          }
          __syncthreads();
          if (tid == 0) sh.listed = 0;
        }
        cluster_sync_all();
      };
      if (few) {
        // ---- all that may stay is in the list: the first block draws the token ----
        into_list(0, last_bin, nullptr);
        if (me == 0) {
          const int n = list_n;
          // ranks and sums in the order; the weights in place of the histogram
          uint64_t* const weight = (uint64_t*)sh.hist;
          for (int i = tid; i < n; i += kThreads) weight[i] = weigh(value_of((uint32_t)(sh.list[i] >> 32)));
          __syncthreads();
          uint64_t sum_k = 0;                                // of the first k
          uint64_t before_w[kList / kThreads];
          bool in_k[kList / kThreads];
#pragma unroll
          for (int q = 0; q < kList / kThreads; ++q) {
            const int i = tid + q * kThreads;
            before_w[q] = 0; in_k[q] = false;
            if (i < n) {
              const uint64_t x = sh.list[i];
              uint32_t rank = 0;
              uint64_t sum = 0;
              for (int j = 0; j < n; ++j)
                if (sh.list[j] > x) { ++rank; sum += weight[j]; }
              before_w[q] = sum;
              in_k[q] = rank < want;
              if (in_k[q]) sum_k += weight[i];
            }
          }
          const uint64_t Zk = block_sum(sum_k);
          uint64_t target = ~0ull;
          if (by_p) {
            const double t = ceil((double)p * (double)Zk);
            target = p > 0.f ? (uint64_t)t : 1ull;
            target = target < 1 ? 1 : target;
          }
          uint64_t sum_s = 0;
          __syncthreads();
#pragma unroll
          for (int q = 0; q < kList / kThreads; ++q) {
            const int i = tid + q * kThreads;
            if (i >= n) continue;
            const bool stay = in_k[q] && before_w[q] < target && enough(value_of((uint32_t)(sh.list[i] >> 32)));
            if (!stay) weight[i] = 0;
            else sum_s += weight[i];
          }
          const uint64_t Z = block_sum(sum_s);
          __syncthreads();
          uint64_t t = u > 0.f ? (u < 1.f ? (uint64_t)((double)u * (double)Z) : Z) : 0;
          t = t < Z ? t : Z - 1;
          for (int i = tid; i < n; i += kThreads) {
            if (weight[i] == 0) continue;
            const uint32_t x = (uint32_t)sh.list[i];         // V - 1 - index
            uint64_t sum = 0;
            for (int j = 0; j < n; ++j)
              if ((uint32_t)sh.list[j] > x) sum += weight[j];
            if (sum <= t && t < sum + weight[i])
              for (uint32_t c = 0; c < C; ++c) put32(&sh.answer[0], c, (uint32_t)(V - 1 - (int)x));
          }
        }
        cluster_sync_all();
        token = sh.answer[0];
      } else {
        if (cut) {
          if (list_n - k_before <= kList) {
            into_list(k_bin, k_bin, nullptr);
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
                if (by_list) {
                  const uint32_t at = add32(&sh.listed, 0, 1u);
                  if (at < kList) put64(&sh.list[at], 0, (uint64_t)pattern(f[e]) << 32 | (uint32_t)(V - 1 - r.index(v, e)));
                }
              }
            }
          }
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
    if (token < 0 && top < INFINITY && temp >= 1e-6f && temp <= 1e6f) token = find_fast([&](float x, int i) { return !(by_k || by_p) || stays(b, x, i); });
    if (token < 0) {
      uint64_t Z;
      token = find([&](float x, int i) { return stays(b, x, i) && enough(x) ? weigh(x) : 0ull; },
                   [&](uint64_t whole) {
                     const uint64_t t = u > 0.f ? (u < 1.f ? (uint64_t)((double)u * (double)whole) : whole) : 0;
                     return t < whole ? t : whole - 1;
                   }, &Z);
    }
  }
  if (a.logprobs && !nothing) {
    double s = 0.0;
    for (int v = tid; v < r.vecs; v += kThreads) {
      float f[8], t = 0.f;
      r.load8(v, f);
#pragma unroll
      for (int e = 0; e < 8; ++e) t += f[e] == top ? 1.f : ex2((f[e] - top) * 1.4426950408889634f);
      s += (double)t;
    }
    s = warp_sum(s);
    __syncthreads();
    if (lane == 0) sh.red_d[warp] = s;
    __syncthreads();
    if (tid == 0) {
      double all = 0.0;
      for (int w = 0; w < kWarps; ++w) all += sh.red_d[w];
      put64((uint64_t*)&sh.part[me], 0, (uint64_t)__double_as_longlong(all));
    }
    cluster_sync_all();
    if (me == 0 && tid == 0) {
      double all = 0.0;
      for (uint32_t c = 0; c < C; ++c) all += sh.part[c];
      const float x = clean(IO<T>::load((const char*)a.logits + (int64_t)row_no * a.row_bytes, token));
      a.logprobs[row_no] = (float)((x == top ? 0.0 : (double)x - (double)top) - log(all));
    }
  } else if (a.logprobs && me == 0 && tid == 0) a.logprobs[row_no] = 0.f;
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
  int ctas = 1;
  while (ctas < kMaxCtas && a.V > ctas * 2 * kStrip) ctas *= 2;
  for (;; ctas = 1) {
    const int share = ((a.V + ctas - 1) / ctas + 7) / 8 * 8;
    const int need = (share + 16) * (int)sizeof(T);
    const int bytes = need <= kHeld ? (need + 15) / 16 * 16 : 0;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)a.N * (unsigned)ctas);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = sizeof(Shared) + (size_t)bytes;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)ctas; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
    if (ctas == 1) return cudaLaunchKernelEx(&cfg, kern, a, share, bytes);
    cfg.attrs = attr;
    cfg.numAttrs = 1;
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
