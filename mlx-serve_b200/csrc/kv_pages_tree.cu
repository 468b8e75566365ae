// Attention of a tree of drafted tokens over a paged key-value cache: a warp a query row, one pass over the tokens that some node may see.
#include "kernels.h"
#include "stream_ptx.cuh"

namespace qb {
namespace {

constexpr float kLog2e = 1.4426950408889634f;

template <int BITS, int D>
__global__ void __launch_bounds__(256) tree_simple_kernel(const __grid_constant__ KvPagesTreeArgs t) {
  const KvPagesAttnArgs& a = t.a;
  constexpr int E = D / 32;
  const int64_t w = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (w >= (int64_t)a.B * a.Hq * t.T) return;
  const int node = (int)(w % t.T), h = (int)(w / t.T % a.Hq), b = (int)(w / t.T / a.Hq), hk = h / a.gqa;
  const int64_t row = a.rows ? a.rows[b] : b;
  int64_t len = row >= 0 && row < a.seqs ? a.lens[row] : 0;
  const int64_t cap = (int64_t)a.M << a.page_shift;
  len = len < 0 ? 0 : (len > cap ? cap : len);
  int64_t n = t.counts ? t.counts[b] : t.T;
  n = n < 0 ? 0 : (n > t.T ? t.T : n);
  n = n > len ? len : n;
  const int64_t base = len - n;
  uint16_t* out = (uint16_t*)a.out + (int64_t)b * a.o_str[0] + (int64_t)h * a.o_str[1] + (int64_t)node * t.o_tok;
  const uint16_t* q = (const uint16_t*)a.q + (int64_t)b * a.q_str[0] + (int64_t)h * a.q_str[1] + (int64_t)node * t.q_tok;
  const int32_t* par = t.parents + (int64_t)b * t.par_str;
  if (node >= n) {
    for (int e = 0; e < E; ++e) out[lane * E + e] = 0;
    return;
  }
  uint64_t line = 0;
  int depth[64];
  for (int i = 0; i < n; ++i) { const int p = par[i]; depth[i] = p >= 0 && p < i ? depth[p] + 1 : 0; }
  for (int i = node; ; ) { line |= 1ull << i; const int p = par[i]; if (p < 0 || p >= i) break; i = p; }
  const int64_t me = base + depth[node];
  float qv[E], o[E], m = -INFINITY, l = 0.f;
  for (int e = 0; e < E; ++e) { qv[e] = bf16_bits_to_f32(q[lane * E + e]) * a.scale * kLog2e; o[e] = 0.f; }
  for (int64_t j = 0; j < len; ++j) {
    int64_t at = j;
    if (j >= base) {
      if (!((line >> (j - base)) & 1)) continue;
      at = base + depth[j - base];
    }
    if (a.window > 0 && at >= a.sinks && at <= me - a.window) continue;
    const int64_t pid = a.table[row * a.table_str + (j >> a.page_shift)], slot = j & ((1 << a.page_shift) - 1);
    if (pid < 0 || pid >= a.P) continue;
    float kv[2][E];
    for (int s = 0; s < 2; ++s) {
      const KvPoolView& p = a.pool[s];
      const int64_t at_q = pid * p.q_str[0] + hk * p.q_str[1] + slot * p.q_str[2];
      for (int e = 0; e < E; ++e) {
        const int d = lane * E + e;
        if (BITS == 16) kv[s][e] = bf16_bits_to_f32(((const uint16_t*)p.q)[at_q + d]);
        else {
          const uint32_t word = ((const uint32_t*)p.q)[at_q + d * BITS / 32];
          const int64_t g = pid * p.sb_str[0] + hk * p.sb_str[1] + slot * p.sb_str[2] + d / 64;
          kv[s][e] = fmaf((float)((word >> (d % (32 / BITS) * BITS)) & ((1u << (BITS & 15)) - 1)), bf16_bits_to_f32(((const uint16_t*)p.s)[g]), bf16_bits_to_f32(((const uint16_t*)p.b)[g]));
        }
      }
    }
    float s = 0.f;
    for (int e = 0; e < E; ++e) s = fmaf(qv[e], kv[0][e], s);
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
    if (s == -INFINITY) continue;
    const float mn = fmaxf(m, s), f = m == mn ? 1.f : exp2f(m - mn), pr = exp2f(s - mn);
    l = l * f + pr;
    for (int e = 0; e < E; ++e) o[e] = fmaf(pr, kv[1][e], o[e] * f);
    m = mn;
  }
  const float inv = l > 0.f ? 1.f / l : (l == l ? 0.f : l);
  for (int e = 0; e < E; ++e) out[lane * E + e] = f32_to_bf16_bits(o[e] * inv);
}
}  // namespace

size_t kv_pages_tree_workspace_bytes(int64_t, int64_t, int64_t, int64_t, int64_t) { return 16; }

cudaError_t launch_kv_pages_tree(KvPagesTreeArgs t, int D, void*, cudaStream_t st) {
  const unsigned grid = (unsigned)(((int64_t)t.a.B * t.a.Hq * t.T + 7) / 8);
  switch (t.a.bits * 1000 + D) {
    case 4064: return launch_kernel(tree_simple_kernel<4, 64>, dim3(grid), dim3(256), 0, st, t);
    case 4128: return launch_kernel(tree_simple_kernel<4, 128>, dim3(grid), dim3(256), 0, st, t);
    case 8064: return launch_kernel(tree_simple_kernel<8, 64>, dim3(grid), dim3(256), 0, st, t);
    case 8128: return launch_kernel(tree_simple_kernel<8, 128>, dim3(grid), dim3(256), 0, st, t);
    case 16064: return launch_kernel(tree_simple_kernel<16, 64>, dim3(grid), dim3(256), 0, st, t);
    case 16128: return launch_kernel(tree_simple_kernel<16, 128>, dim3(grid), dim3(256), 0, st, t);
    default: return cudaErrorInvalidValue;
  }
}
}  // namespace qb
