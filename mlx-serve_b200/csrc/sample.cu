// A token from every row of logits: temperature, top-k, top-p and min-p, with a random number given for the row.
//
// With m the row's largest logit, w_i = exp((l_i - m) / temperature) and the order "larger logit first, then lower index": the first k
// of the order stay; of these the shortest prefix whose weights reach p of their sum; of these those with w_i >= min_p; the token is the
// first one in index order at which the running sum of the weights that stay passes u times their sum.
//
//  * Weights are whole numbers, round(w_i * 2^44), of a 64-bit exponential: sums of them do not depend on the order in which threads
//    or atomics run, and borders (the nucleus, the token) are met as 64-bit sums meet them.  2^19 of them fit 63 bits; a token below
//    2^-45 of the largest counts as 0.
//  * A border in the order is found by its value, eight bits of the logit's order-preserving pattern at a time, with a histogram of
//    counts or of weights; among equal logits by index.
#include "kernels.h"

namespace qb {
namespace {

constexpr int kThreads = 1024;
constexpr int kWarps = kThreads / 32;
constexpr double kOne = 17592186044416.0;      // 2^44

template <typename T> __device__ __forceinline__ float logit(const void* p, int64_t i) {
  const float x = IO<T>::load(p, i);
  return x == x ? x + 0.f : -INFINITY;         // (a NaN counts as masked; -0 as 0)
}
// larger patterns for larger floats
__device__ __forceinline__ uint32_t pattern(float x) {
  const uint32_t b = __float_as_uint(x);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }

struct Weigh {
  float top;
  double per_t, least;         // 1 / temperature, min_p
  __device__ __forceinline__ uint64_t operator()(float x) const {
    if (x == top) return (uint64_t)kOne;
    if (x == -INFINITY) return 0;
    return (uint64_t)__double2ll_rn(exp(((double)x - (double)top) * per_t) * kOne);
  }
};

__device__ __forceinline__ uint64_t warp_sum(uint64_t v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ uint64_t block_sum(uint64_t v, uint64_t* red) {
  v = warp_sum(v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  return warp_sum(red[threadIdx.x & 31]);
}
// sum of the values of the threads before this one; *all = the block's
__device__ __forceinline__ uint64_t block_before(uint64_t v, uint64_t* red, uint64_t* all) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint64_t upto = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint64_t n = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += n;
  }
  __syncthreads();
  if (lane == 31) red[warp] = upto;
  __syncthreads();
  const uint64_t w = red[lane];
  *all = warp_sum(w);
  return upto - v + warp_sum(lane < warp ? w : 0);
}

// What stays: everything in front of (key, index) in the order, and that itself.
struct Border { uint32_t key; int index; };
__device__ __forceinline__ bool stays(const Border& b, uint32_t key, int i) { return key > b.key || (key == b.key && i <= b.index); }

template <typename T>
__global__ void __launch_bounds__(kThreads) sample_kernel(const __grid_constant__ SampleArgs a) {
  __shared__ uint64_t hist[256], red[32];
  __shared__ uint64_t found_above;
  __shared__ int found;
  const int row = blockIdx.x, tid = threadIdx.x, V = a.V;
  const void* const x = (const char*)a.logits + (int64_t)row * a.row_bytes;

  uint32_t mx = 0;
  for (int i = tid; i < V; i += kThreads) mx = max(mx, pattern(logit<T>(x, i)));
  const uint32_t top_key = (uint32_t)[&] {
    const uint32_t w = __reduce_max_sync(0xffffffffu, mx);
    if ((tid & 31) == 0) red[tid >> 5] = w;
    __syncthreads();
    return __reduce_max_sync(0xffffffffu, (uint32_t)red[tid & 31]);
  }();
  Weigh weigh;
  weigh.top = value_of(top_key);
  const float temp = a.temperature ? a.temperature[row * a.str[1]] : 1.f, u = a.random[row * a.str[0]];
  const int k = a.top_k ? a.top_k[row * a.str[2]] : 0;
  const float p = a.top_p ? a.top_p[row * a.str[3]] : 1.f, least = a.min_p ? a.min_p[row * a.str[4]] : 0.f;
  weigh.per_t = 1.0 / (double)temp;
  weigh.least = least;
  if (weigh.top == -INFINITY) {
    if (tid == 0) {
      a.tokens[row] = -1;
      if (a.logprobs) a.logprobs[row] = 0.f;
    }
    return;
  }

  // The border at which the counts (or weights) of what stays before it reach `target`, of what stays at `from`.
  auto border = [&](auto amount, uint64_t target, const Border& from) {
    uint32_t prefix = 0, mask = 0;
    uint64_t above = 0;                        // of larger keys
    for (int shift = 24; shift >= 0; shift -= 8) {
      __syncthreads();
      for (int i = tid; i < 256; i += kThreads) hist[i] = 0;
      __syncthreads();
      for (int i = tid; i < V; i += kThreads) {
        const float v = logit<T>(x, i);
        const uint32_t key = pattern(v);
        if ((key & mask) == prefix && stays(from, key, i)) atomicAdd((unsigned long long*)&hist[(key >> shift) & 255], (unsigned long long)amount(v));
      }
      __syncthreads();
      if (tid == 0) {
        int bin = 255;
        for (; bin > 0 && above + hist[bin] < target; --bin) above += hist[bin];
        found = bin; found_above = above;
      }
      __syncthreads();
      above = found_above;
      prefix |= (uint32_t)found << shift;
      mask |= 255u << shift;
    }
    // among equal ones, the first so many by index
    const uint64_t each = amount(value_of(prefix));
    uint64_t left = each > 0 ? (target - above + each - 1) / each : (uint64_t)V;
    Border to = {prefix, V - 1};
    for (int i0 = 0; i0 < V; i0 += kThreads) {
      const int i = i0 + tid;
      const bool one = i < V && pattern(logit<T>(x, i)) == prefix;
      uint64_t n;
      const uint64_t before = block_before(one, red, &n);
      if (one && before + 1 == left) found = i;
      __syncthreads();
      if (n >= left) { to.index = found; break; }
      left -= n;
    }
    return to;
  };

  Border b = {0, V - 1};
  int token = 0;
  const bool greedy = !(temp > 0.f);
  if (greedy) b = border([](float) { return (uint64_t)1; }, 1, b);
  else {
    if (k > 0 && k < V) b = border([](float) { return (uint64_t)1; }, (uint64_t)k, b);
    if (p < 1.f) {
      uint64_t s = 0;
      for (int i = tid; i < V; i += kThreads) {
        const float v = logit<T>(x, i);
        if (stays(b, pattern(v), i)) s += weigh(v);
      }
      const uint64_t Z = block_sum(s, red);
      const uint64_t target = p > 0.f ? (uint64_t)ceil((double)p * (double)Z) : 1;
      b = border(weigh, target < 1 ? 1 : (target > Z ? Z : target), b);
    }
  }
  auto kept = [&](float v, int i) -> uint64_t {
    if (!stays(b, pattern(v), i)) return 0;
    if (greedy) return 1;
    return v == weigh.top || !(least > 0.f) || exp(((double)v - (double)weigh.top) * weigh.per_t) >= weigh.least ? weigh(v) : 0;
  };
  uint64_t s = 0;
  for (int i = tid; i < V; i += kThreads) { const float v = logit<T>(x, i); s += kept(v, i); }
  const uint64_t Z = block_sum(s, red);
  uint64_t t = u > 0.f ? (u < 1.f ? (uint64_t)((double)u * (double)Z) : Z) : 0;
  t = t < Z ? t : Z - 1;
  for (int i0 = 0; i0 < V; i0 += kThreads) {
    const int i = i0 + tid;
    const uint64_t w = i < V ? kept(logit<T>(x, i), i) : 0;
    uint64_t n;
    const uint64_t before = block_before(w, red, &n);
    if (before <= t && t < before + w) found = i;
    __syncthreads();
    if (t < n) { token = found; break; }
    t -= n;
  }
  if (a.logprobs) {
    double e = 0.0;
    for (int i = tid; i < V; i += kThreads) {
      const float v = logit<T>(x, i);
      e += v == weigh.top ? 1.0 : (v == -INFINITY ? 0.0 : exp((double)v - (double)weigh.top));
    }
    const uint64_t sum = block_sum((uint64_t)(e * kOne), red);
    if (tid == 0) {
      const float v = logit<T>(x, token);
      a.logprobs[row] = (float)((v == weigh.top ? 0.0 : (double)v - (double)weigh.top) - log((double)sum / kOne));
    }
  }
  if (tid == 0) a.tokens[row] = token;
}
}  // namespace

cudaError_t launch_sample(const SampleArgs& a, cudaStream_t st) {
  auto kern = a.dtype == QB200_BFLOAT16 ? sample_kernel<__nv_bfloat16> : (a.dtype == QB200_FLOAT16 ? sample_kernel<__half> : sample_kernel<float>);
  return launch_kernel(kern, dim3((unsigned)a.N), dim3(kThreads), 0, st, a);
}

}  // namespace qb
