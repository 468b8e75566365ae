// Causal attention of a prompt (or a chunk of one behind cached tokens) with an optional sliding window and a few first tokens that
// stay visible: bf16, head dim 64 or 128, on the tensor cores (tcgen05) with the scores and results in tensor memory.
//
// Query i stands at position p = kv_len - Tq + i and sees the keys j <= p with j > p - window or j < sinks.
//   o = sum_j P_j v_j / sum_j P_j,  P_j = 2^(c s_j - c r),  s = q . k, c = scale * log2(e), r a running reference of the row.
//
// One CTA of 12 warps takes two tiles of 128 queries that read the same keys: two heads of a group where the group is even, else
// two neighbouring tiles of one head (one tile where a launch has fewer tiles than the device has SMs).
//   warps 0-3, 4-7 : the softmax of a tile, a thread a row.  Scores come from tensor memory, the probabilities go back in their place as
//                    bf16, the A operand of the second product.  Blocks that all queries see whole are taken with the reference r as it
//                    is, without looking for their maximum first; only where a block's sum passes 2^24 (and in masked blocks, where
//                    the maximum is found anyway and r may lie 2^8 below it) r moves and the result is rescaled.
//   warp 8         : copies (TMA): both query tiles once, then keys and values of 128 tokens in a ring.
//   warp 9         : issues the matrix products, S = Q K^T of the next step behind P V of this one, the tiles in turn: while one
//                    tile's softmax runs, the tensor cores work for the other.
//   warps 10, 11   : make the values fit for a product with masked probabilities (0 * NaN is NaN): where a block is masked for
//                    some query, rows that no query of the CTA sees are zeroed, and rows with anything not finite are zeroed and
//                    noted; the queries that see such a row give NaN.
// Blocks of 128 keys that no query of a tile sees are left out; only those cut by a border of the mask are masked element by element.
// Where there are few tiles, a CTA takes one, whose scores are made two steps ahead in the place of the other tile's (the tensor cores then
// wait for the softmax alone: 1.03 us a step), or clusters share a tile's keys and join their sums through distributed shared memory.
//
// Floor: 4 D operations per visible pair on the tensor cores.  32 heads of 128, 16384 tokens, window 4096: 0.96 TFLOP, 589 us at 1634
// TFLOP/s, takes 955 us pass after pass, where the power cap holds the clock down (1.01 PFLOP/s, 0.62 of the measured burst peak), 820 with a
// pause before each (1.17 PFLOP/s, 0.72).  The variants below were timed with pauses, against 811.  A step of a tile is a chain: softmax of 128 keys 1400 cycles, P V and
// S 512 each, 450 of hand-over; the other tile fills part of it, and the tensor cores work for 2048 of every 3100 cycles.  Tried and
// not kept: 16 softmax warps (845 us), scores in halves of 64 keys made ahead (1040: a product of 64 columns takes as long as
// one of 128), an issuer for each tile (870: they fall into step and wait together), the first half of P handed over early (862).
#include <mutex>
#include <type_traits>

#include "tc_ptx.cuh"

namespace qb {
namespace {

__device__ int g_window_error = 0;   // 0 = ok; otherwise the code of the wait that expired

constexpr int kThreads = 384;
constexpr int kTile = 128;           // queries of a tile, keys of a block
constexpr uint32_t kPolls = 1u << 18, kSpins = 1u << 23;
constexpr int kPolyOf8 = 2;          // pairs of 8 whose exponentials the fp32 units work out (chosen at head dim 128)
constexpr float kMostSum = 16777216.f;   // of a block's probabilities, with the reference as it was
constexpr float kSlack = 8.f;        // exponents that the reference may lie below the maximum

template <int D> struct Shape {
  static constexpr int BYTES = kTile * D * 2;              // a tile of queries, keys or values
  static constexpr int STAGES = D == 128 ? 5 : 8;
  static constexpr int SMEM = (2 + STAGES) * BYTES + 1024;
  static constexpr int HALVES = D / 64;                    // blocks of 64 columns (128 bytes) side by side
};

struct WindowK {
  uint16_t* out; int64_t o_str[3];     // (sequence, head, token)
  const int32_t* kv_lens;
  int B, Hq, gqa, Tq, Tk, window, sinks;
  int qblocks, heads2;                 // 1: the two tiles are two heads; 0: two tiles of one head
  int split;                           // CTAs of a cluster that share the keys of the tiles (1, 2, 4, 8)
  int mul[3][2];                       // coordinates along (head, sequence) of q, k, v: 0 where the tensor is broadcast
  float c;
  int o_vec;                           // result rows can be stored 16 bytes at a time
};

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, uint64_t* bar, int x, int y, int z, int w) {
  asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];"
               ::"r"(dst), "l"(map), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}
__device__ __forceinline__ void umma_ss(uint32_t d, uint64_t ad, uint64_t bd, uint32_t idesc, uint32_t accum) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
               ::"r"(d), "l"(ad), "l"(bd), "r"(idesc), "r"(accum) : "memory");
}
__device__ __forceinline__ void umma_ts(uint32_t d, uint32_t a, uint64_t bd, uint32_t idesc, uint32_t accum) {   // A in tensor memory
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
               ::"r"(d), "r"(a), "l"(bd), "r"(idesc), "r"(accum) : "memory");
}
__device__ __forceinline__ void commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,"
      "%22,%23,%24,%25,%26,%27,%28,%29,%30,%31};"
      ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]),
      "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]),
      "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31]), "r"(taddr)
      : "memory");
}
__device__ __forceinline__ uint32_t cluster_addr(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ float ex2f(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ float max3_nan(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ float clamp126(float x) {
  asm("max.NaN.f32 %0, %0, %1;\n\tmin.NaN.f32 %0, %0, %2;" : "+f"(x) : "f"(-126.f), "f"(126.f));
  return x;
}
// 2^x for a pair without the special-function unit, which the softmax would otherwise wait for: x = n + f with n the nearest
// integer (from the low bits of x + 1.5 * 2^23), 2^f on [-1/2, 1/2] by the cubic of least relative error (7.5e-5, a fiftieth of what
// rounding to bf16 takes; Lawson's iteration), n added to the exponent.  x counts as -126 below that, as 126 above, a NaN gives
// 3.4e38: what the sum over the row then shows.
__device__ __forceinline__ uint64_t exp2_pair(uint64_t x) {
  const uint64_t magic = two(12582912.f, 12582912.f), unmagic = two(-12582912.f, -12582912.f), minus = two(-1.f, -1.f);
  float a, b, p, q, u, v;
  untwo(x, a, b);
  x = two(clamp126(a), clamp126(b));
  const uint64_t t = add2(x, magic), f = fma2(add2(t, unmagic), minus, x);
  uint64_t y = fma2(f, two(0.0551716685f, 0.0551716685f), two(0.2426111251f, 0.2426111251f));
  y = fma2(y, f, two(0.6932609677f, 0.6932609677f));
  y = fma2(y, f, two(0.9999280572f, 0.9999280572f));
  untwo(y, p, q);
  untwo(t, u, v);
  return two(__int_as_float(__float_as_int(p) + (__float_as_int(u) << 23)), __int_as_float(__float_as_int(q) + (__float_as_int(v) << 23)));
}

// A bounded wait that polls without sleeping.
__device__ __forceinline__ bool spin_cta(uint64_t* bar, uint32_t parity) {
  const uint32_t addr = smem_u32(bar);
  for (uint32_t it = 0; it < kSpins; ++it) {
    uint32_t done;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(done) : "r"(addr), "r"(parity) : "memory");
    if (done) return true;
  }
  return false;
}

// The key blocks of a CTA and what its tiles see of them; every role works this out for itself.
struct Plan {
  int p_lo[2], p_hi[2];     // positions of a tile's first and last query (p_lo may be below 0; p_hi < 0: it sees nothing)
  int lo, hi;               // keys [lo, hi] and the sinks are all that the CTA sees
  int window, sinks;
  int front, skip, blocks;  // blocks [0, front), then i + skip
  int from;                 // of these, the ones from here on are this CTA's (`blocks` of them)
  __device__ __forceinline__ int block(int i) const { return i + from < front ? i + from : i + from + skip; }
  __device__ __forceinline__ bool needs(int t, int blk) const {       // some query of tile t sees some key of the block
    const int k0 = blk * kTile, lo_t = t ? p_lo[1] : p_lo[0], hi_t = t ? p_hi[1] : p_hi[0];
    const int first = lo_t > 0 ? lo_t : 0;
    return k0 <= hi_t && (window == 0 || k0 + kTile - 1 > first - window || k0 < sinks);
  }
  __device__ __forceinline__ bool whole(int t, int blk) const {       // every query of tile t sees every key of the block
    const int k0 = blk * kTile, lo_t = t ? p_lo[1] : p_lo[0], hi_t = t ? p_hi[1] : p_hi[0];
    return k0 + kTile - 1 <= lo_t && (window == 0 || k0 > hi_t - window || k0 + kTile <= sinks);
  }
  __device__ __forceinline__ bool masked(int blk) const { return (needs(0, blk) && !whole(0, blk)) || (needs(1, blk) && !whole(1, blk)); }
};

template <bool SINGLE> __device__ __forceinline__ Plan make_plan(const WindowK& a, int b, int row0, int rank) {
  Plan p;
  int len = a.kv_lens ? a.kv_lens[b] : a.Tk;
  len = len < 0 ? 0 : (len > a.Tk ? a.Tk : len);
  const int base = len - a.Tq;
  const int r1 = a.heads2 ? row0 : (SINGLE ? a.Tq : row0 + kTile);
  const int rows[2] = {row0, r1};
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const int last = rows[t] + kTile - 1 < a.Tq - 1 ? rows[t] + kTile - 1 : a.Tq - 1;
    p.p_lo[t] = base + rows[t];
    p.p_hi[t] = rows[t] < a.Tq ? base + last : -1;
  }
  p.window = a.window;
  p.hi = p.p_hi[0] > p.p_hi[1] ? p.p_hi[0] : p.p_hi[1];
  const int first = p.p_lo[0] > 0 ? p.p_lo[0] : 0;
  p.lo = a.window > 0 && first - a.window + 1 > 0 ? first - a.window + 1 : 0;
  p.sinks = a.sinks < p.hi + 1 ? a.sinks : p.hi + 1;
  if (p.sinks < 0) p.sinks = 0;
  const int nb = p.hi >= 0 ? p.hi / kTile + 1 : 0;
  p.front = (p.sinks + kTile - 1) / kTile;
  p.skip = p.lo / kTile - p.front;
  if (p.skip < 0) p.skip = 0;
  const int all = nb - p.skip, each = all / a.split, rest = all - each * a.split;
  p.from = each * rank + (rank < rest ? rank : rest);
  p.blocks = each + (rank < rest ? 1 : 0);
  return p;
}

// V as the B operand with its columns contiguous (rows of 128 bytes, swizzled): atoms of 8 tokens 1024 bytes apart, blocks of 64
// columns a tile of 128 tokens apart.
__device__ __forceinline__ uint64_t make_desc_mn(uint32_t saddr) {
  uint64_t d = 0;
  d |= (uint64_t)((saddr & 0x3FFFF) >> 4);
  d |= (uint64_t)((kTile * 128) >> 4) << 16;     // from 64 columns to the next 64
  d |= (uint64_t)(1024 >> 4) << 32;              // from 8 tokens to the next 8
  d |= (uint64_t)1 << 46;
  d |= (uint64_t)2 << 61;
  return d;
}

constexpr int kNotes = 48;    // groups of 32 keys of masked blocks: at most 3 blocks at the diagonal, 3 at the window's start, 2 where the sinks end

// SINGLE: one tile (heads2 is 0; the second lies behind the last query), whose steps take the places and barriers of the two tiles in turn.
template <int D, bool SINGLE>
__global__ void __launch_bounds__(kThreads, 1) window_attn_kernel(const __grid_constant__ CUtensorMap mq, const __grid_constant__ CUtensorMap mk,
                                                                  const __grid_constant__ CUtensorMap mv, const __grid_constant__ WindowK a) {
  using SH = Shape<D>;
  constexpr int ST = SH::STAGES;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = (unsigned char*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  __shared__ uint64_t q_full, kv_full[ST], kv_empty[ST], s_full[2], p_ready[2], o_done[2];
  __shared__ uint32_t tmem_slot;
  __shared__ int s_fail, noted;
  __shared__ int note_key[kNotes];
  __shared__ uint32_t note_bits[kNotes];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  asm volatile("griddepcontrol.wait;" ::: "memory");         // (before tensor memory is taken, too: the kernel before may hold it)

  // ---- which tiles: the longest rows of the prompt first ----
  const int per_q = (a.heads2 ? a.Hq / 2 : a.Hq) * a.B;
  const int rank = a.split > 1 ? (int)cluster_rank_tc() : 0, unit = a.split > 1 ? (int)blockIdx.x / a.split : (int)blockIdx.x;
  const int qb = a.qblocks - 1 - unit / per_q;
  const int rem = unit % per_q;
  const int b = rem / (per_q / a.B), hu = rem % (per_q / a.B);
  const int head0 = a.heads2 ? 2 * hu : hu, head1 = a.heads2 ? head0 + 1 : head0, hk = head0 / a.gqa;
  const int row0 = qb * (a.heads2 || SINGLE ? kTile : 2 * kTile), row1 = a.heads2 ? row0 : (SINGLE ? a.Tq : row0 + kTile);
  const Plan plan = make_plan<SINGLE>(a, b, row0, rank);

  if (tid >= 32 && tid < 32 + kNotes) note_bits[tid - 32] = 0u;
  if (tid == 0) {
    s_fail = 0; noted = 0;
    mbar_init(&q_full, 1);
    for (int i = 0; i < ST; ++i) { mbar_init(&kv_full[i], 1); mbar_init(&kv_empty[i], 1); }
    for (int i = 0; i < 2; ++i) { mbar_init(&s_full[i], 1); mbar_init(&p_ready[i], 6); mbar_init(&o_done[i], 1); }
    asm volatile("fence.mbarrier_init.release.cluster;\n\tfence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == 9) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"(512u));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::);
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = tmem_slot;
  const uint32_t ring = smem_u32(smem) + 2 * SH::BYTES;
  auto failed = [&](int code) { s_fail = code; atomicCAS(&g_window_error, 0, code); };

  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
    if (warp == 8) {
      // ---- copies ----
      if (elect_one() && plan.blocks > 0) {
        constexpr int tiles = SINGLE ? 1 : 2;
        mbar_expect_tx(&q_full, tiles * SH::BYTES);
        for (int t = 0; t < tiles; ++t)
#pragma unroll
          for (int h = 0; h < SH::HALVES; ++h)
            tma_load_4d(smem_u32(smem) + t * SH::BYTES + h * kTile * 128, &mq, &q_full, 64 * h, t ? row1 : row0, (t ? head1 : head0) * a.mul[0][0], b * a.mul[0][1]);
        bool ok = true;
        for (int it = 0; it < 2 * plan.blocks; ++it) {
          const int st = it % ST, round = it / ST;
          if (round > 0 && !wait_cta(&kv_empty[st], (uint32_t)(round - 1) & 1, kPolls)) { failed(501); ok = false; break; }
          const int blk = plan.block(it >> 1), kv = 1 + (it & 1);
          mbar_expect_tx(&kv_full[st], SH::BYTES);
#pragma unroll
          for (int h = 0; h < SH::HALVES; ++h)
            tma_load_4d(ring + st * SH::BYTES + h * kTile * 128, kv == 1 ? &mk : &mv, &kv_full[st], 64 * h, blk * kTile, hk * a.mul[kv][0], b * a.mul[kv][1]);
        }
        if (!ok)
          for (int i = 0; i < 1000; ++i) __nanosleep(1000);    // (copies may still be on their way)
      }
    } else if (warp == 9) {
      // ---- products ----
      // What the instructions take is made uniform over the warp, and one lane is elected where the compiler sees that it is one: an
      // MMA issues in 9 - 16 cycles then, in about 73 otherwise, which is more than it takes.
      constexpr uint32_t idesc0 = (1u << 4) | (1u << 7) | (1u << 10) | ((128u >> 4) << 24);   // f32 += bf16 x bf16, M = 128
      constexpr uint32_t idesc_s = idesc0 | ((uint32_t)(kTile >> 3) << 17), idesc_o = idesc0 | ((uint32_t)(D >> 3) << 17) | (1u << 16);
      auto U = [](int v) { return __shfl_sync(0xffffffffu, v, 0); };
      Plan pl;
#pragma unroll
      for (int t = 0; t < 2; ++t) { pl.p_lo[t] = U(plan.p_lo[t]); pl.p_hi[t] = U(plan.p_hi[t]); }
      pl.window = U(plan.window); pl.sinks = U(plan.sinks); pl.front = U(plan.front); pl.skip = U(plan.skip); pl.from = U(plan.from); pl.blocks = U(plan.blocks);
      const uint32_t tm = (uint32_t)U((int)tmem), slot = SH::BYTES >> 4;
      const uint64_t hi_k = make_desc(0) & 0xFFFFFFFF00000000ull, hi_v = make_desc_mn(0) & 0xFFFFFFFF00000000ull;
      const uint32_t q_d = (uint32_t)U((int)(uint32_t)make_desc(smem_u32(smem))), k_d = (uint32_t)U((int)(uint32_t)make_desc(ring)),
                     v_d = (uint32_t)U((int)(uint32_t)make_desc_mn(ring));
      auto wait = [&](uint64_t* bar, uint32_t phase) { return __all_sync(0xffffffffu, spin_cta(bar, phase & 1)); };
      auto scores = [&](int t, uint32_t st) {                // S of tile t (or step t of one tile) with the keys in ring slot st (by the elected lane)
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          const uint32_t o = (k >> 2) * ((kTile * 128) >> 4) + (k & 3) * 2;
          umma_ss(tm + t * 128, hi_k | (q_d + (SINGLE ? 0 : t) * slot + o), hi_k | (k_d + st * slot + o), idesc_s, k > 0);
        }
        commit(&s_full[t]);
      };
      auto products = [&]() -> bool {
        if (!wait(&q_full, 0) || !wait(&kv_full[0], 0)) return false;
        uint32_t done[2] = {0, 0};
        bool now[2] = {pl.needs(0, pl.block(0)), pl.needs(1, pl.block(0))};
        if (elect_one()) {
#pragma unroll
          for (int t = 0; t < 2; ++t)
            if (now[t]) scores(t, 0);
          commit(&kv_empty[0]);
        }
        __syncwarp();
        // A wait takes the issuer some 160 cycles even where there is nothing to wait for, and the tensor cores take few products in
        // advance.  So it waits for p_ready alone: the warps that look after the values arrive there too, once this block's values
        // and the next one's keys are in place.
        uint32_t sv = 1, sk = 2, rk = 0;                     // slots of this block's values and of the next one's keys, the latter's round
        for (int n = 0; n < pl.blocks; ++n) {
          const bool more = n + 1 < pl.blocks;
          const int next = pl.block(n + 1);
          const bool then[2] = {more && pl.needs(0, next), more && pl.needs(1, next)};
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            if (now[t]) {
              if (!wait(&p_ready[t], done[t])) return false;
              fence_after();
            } else if (then[t] && !wait(&kv_full[sk], rk)) return false;
            if (elect_one()) {
              if (now[t]) {
#pragma unroll
                for (int k = 0; k < kTile / 16; ++k)
                  umma_ts(tm + 256 + t * D, tm + t * 128 + k * 8, hi_v | (v_d + sv * slot + k * (2048 >> 4)), idesc_o, k > 0 ? 1u : (done[t] > 0 ? 1u : 0u));
                commit(&o_done[t]);
              }
              if (t == 1) commit(&kv_empty[sv]);
              if (then[t]) scores(t, sk);
              if (t == 1 && more) commit(&kv_empty[sk]);
            }
            __syncwarp();
            if (now[t]) ++done[t];
          }
          now[0] = then[0]; now[1] = then[1];
          sv = sk + 1;
          if (sv == ST) { sv = 0; ++rk; }
          sk = sv + 1;
          if (sk == ST) { sk = 0; ++rk; }
        }
        // every product is complete before tensor memory and the ring go
#pragma unroll
        for (int t = 0; t < 2; ++t)
          if (done[t] > 0 && !wait(&o_done[t], done[t] - 1)) return false;
        return true;
      };
      // One tile: S of the step after the next follows P V of this one, in the place of its probabilities, so that the softmax finds the next
      // scores done.  Steps take turns with all barriers: two of them may be complete before a waiter looks.
      auto products_single = [&]() -> bool {
        if (!wait(&q_full, 0)) return false;
        uint32_t sv = 1, sk = 0, rk = 0;
        for (int n = -2; n < pl.blocks; ++n) {
          const int step = n & 1;
          if (n >= 0) {
            if (!wait(&p_ready[step], (uint32_t)(n >> 1))) return false;
            fence_after();
            if (elect_one()) {
#pragma unroll
              for (int k = 0; k < kTile / 16; ++k)
                umma_ts(tm + 256, tm + step * 128 + k * 8, hi_v | (v_d + sv * slot + k * (2048 >> 4)), idesc_o, k > 0 ? 1u : (n > 0 ? 1u : 0u));
              commit(&o_done[step]);
              commit(&kv_empty[sv]);
            }
            __syncwarp();
            sv = sv + 2 < ST ? sv + 2 : sv + 2 - ST;
          }
          if (n + 2 < pl.blocks) {
            if (!wait(&kv_full[sk], rk)) return false;
            if (elect_one()) {
              scores(step, sk);
              commit(&kv_empty[sk]);
            }
            __syncwarp();
            sk += 2;
            if (sk >= ST) { sk -= ST; ++rk; }
          }
        }
        return wait(&o_done[(pl.blocks - 1) & 1], (uint32_t)((pl.blocks - 1) >> 1));
      };
      if (pl.blocks > 0 && !(SINGLE ? products_single() : products())) {
        if (lane == 0 && !s_fail) failed(502);
        for (int i = 0; i < 1000; ++i) __nanosleep(1000);    // (products may still be on their way)
      }
    } else {
      // ---- values of masked blocks ----
      bool ok = true;
      const int me = tid - 320;
      int cnt[2] = {0, 0};
      for (int n = 0; n < plan.blocks && ok; ++n) {
        const int iv = 2 * n + 1, blk = plan.block(n);
        ok = __all_sync(0xffffffffu, wait_cta(&kv_full[iv % ST], (uint32_t)(iv / ST) & 1, kPolls));
        if (ok && plan.masked(blk)) {
          unsigned char* v = smem + (2 + iv % ST) * SH::BYTES;
#pragma unroll 1
          for (int half = 0; half < 2; ++half) {
            const int r = half * 64 + me, key = blk * kTile + r;
            const bool seen = key <= plan.hi && (key >= plan.lo || key < plan.sinks);
            bool bad = false;
            if (seen) {
              uint32_t acc = 0;
#pragma unroll
              for (int c = 0; c < D / 8; ++c) {
                const uint4 x = *(const uint4*)(v + (c >> 3) * kTile * 128 + r * 128 + (((c & 7) ^ (r & 7)) << 4));
                acc |= ((x.x & 0x7F807F80u) + 0x00800080u) | ((x.y & 0x7F807F80u) + 0x00800080u) | ((x.z & 0x7F807F80u) + 0x00800080u) | ((x.w & 0x7F807F80u) + 0x00800080u);
              }
              bad = (acc & 0x80008000u) != 0;      // an exponent of all ones
            }
            if (!seen || bad)
#pragma unroll
              for (int c = 0; c < D / 8; ++c) *(uint4*)(v + (c >> 3) * kTile * 128 + r * 128 + (((c & 7) ^ (r & 7)) << 4)) = make_uint4(0u, 0u, 0u, 0u);
            const uint32_t m = __ballot_sync(0xffffffffu, bad);
            if (m && lane == 0) {
              const int at = atomicAdd(&noted, 1);
              if (at < kNotes) {
                note_key[at] = blk * kTile + half * 64 + (warp - 10) * 32;
                __threadfence_block();           // (the bits, zero until now, make the note count)
                *(volatile uint32_t*)&note_bits[at] = m;
              }
            }
          }
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        }
        if (!SINGLE && ok && n + 1 < plan.blocks) ok = __all_sync(0xffffffffu, wait_cta(&kv_full[(iv + 1) % ST], (uint32_t)((iv + 1) / ST) & 1, kPolls));
#pragma unroll
        for (int t = 0; t < 2; ++t)
          if (SINGLE ? t == (n & 1) : plan.needs(t, blk)) {
            // (the phase before is complete, so that this arrival is not taken for one of its own)
            if (ok && cnt[t] > 0) ok = __all_sync(0xffffffffu, wait_cta(&p_ready[t], (uint32_t)(cnt[t] - 1) & 1, kPolls));
            __syncwarp();
            if (ok && lane == 0) mbar_arrive(&p_ready[t]);
            ++cnt[t];
          }
      }
      if (!ok && lane == 0 && !s_fail) failed(503);
    }
    __syncwarp();
    if (a.split > 1) { cluster_sync_tc(); cluster_sync_tc(); }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
    // ---- softmax: a thread a row ----
    const int t = warp >> 2, in_tile = tid & 127, row = (t ? row1 : row0) + in_tile, pos = (t ? plan.p_lo[1] : plan.p_lo[0]) + in_tile;
    const uint32_t lanes = tmem + ((uint32_t)(warp & 3) << 21), o_at = lanes + 256 + (uint32_t)t * D;
    float ref = -INFINITY, l = 0.f;
    int done = 0;
    bool ok = true;
    const uint64_t c2 = two(a.c, a.c);
    auto turn = [&](int n) { return SINGLE ? n & 1 : t; };                        // whose place and barriers step n of the tile takes
    auto phase = [&](int n) { return (uint32_t)(SINGLE ? n >> 1 : n) & 1u; };
    for (int n = 0; n < plan.blocks; ++n) {
      const int blk = plan.block(n);
      if (!plan.needs(t, blk)) continue;
      ok = __all_sync(0xffffffffu, wait_cta(&s_full[turn(done)], phase(done), kPolls));
      if (!ok) break;
      fence_after();
      const uint32_t s_at = lanes + (uint32_t)turn(done) * 128;
      // A block that all queries see whole is taken with the reference as it is, scores and all in one pass: the sum tells afterwards
      // whether that was right (a maximum of more than 2^24 would be among it, and what is not finite shows).
      uint32_t p[64];
      float sum = 0.f;
      bool again = true;
      const bool whole = plan.whole(t, blk);
      if (whole && __all_sync(0xffffffffu, ref > -INFINITY)) {
        const uint64_t r2 = two(-ref, -ref);
        uint64_t sums[2] = {0ull, 0ull};
        uint32_t s[2][32];
        tmem_ld32(s_at, s[0]);
        asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          if (q < 3) tmem_ld32(s_at + 32 * (q + 1), s[(q + 1) & 1]);
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const uint64_t x = fma2(two(__uint_as_float(s[q & 1][2 * i]), __uint_as_float(s[q & 1][2 * i + 1])), c2, r2);
            float x0, x1;
            if ((i & 7) < kPolyOf8) untwo(exp2_pair(x), x0, x1);
            else {
              untwo(x, x0, x1);
              x0 = ex2f(x0); x1 = ex2f(x1);
            }
            sums[i & 1] = add2(sums[i & 1], two(x0, x1));
            p[16 * q + i] = pack2(x0, x1);
          }
          if (q < 3) asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
        }
        float u, v;
        untwo(add2(sums[0], sums[1]), u, v);
        sum = u + v;
        again = __any_sync(0xffffffffu, !(sum <= kMostSum));
      }
      if (again) {
        uint32_t s[4][32];
#pragma unroll
        for (int q = 0; q < 4; ++q) tmem_ld32(s_at + 32 * q, s[q]);
        asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
        if (!whole) {
          // key k0 + i is seen where i <= hi and (i > lo or i < sk)
          const int k0 = blk * kTile, hi = pos - k0, lo = plan.window > 0 ? pos - plan.window - k0 : -1, sk = plan.sinks - k0;
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            auto below = [&](int x) { const int y = x - 32 * q; return y <= 0 ? 0u : (y >= 32 ? 0xffffffffu : (1u << y) - 1u); };   // keys < x
            const uint32_t m = below(hi + 1) & (~below(lo + 1) | below(sk));
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (!((m >> i) & 1u)) s[q][i] = 0xff800000u;
          }
        }
        // the row's maximum, NaN if anything is NaN or +inf: the whole row is then
        float mx;
        {
          float m8[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) m8[i] = __uint_as_float(s[0][i]);
#pragma unroll
          for (int q = 0; q < 4; ++q)
#pragma unroll
            for (int i = q ? 0 : 8; i < 32; i += 2) m8[(i >> 1) & 7] = max3_nan(m8[(i >> 1) & 7], __uint_as_float(s[q][i]), __uint_as_float(s[q][i + 1]));
          mx = max3_nan(max3_nan(m8[0], m8[1], m8[2]), max3_nan(m8[3], m8[4], m8[5]), max3_nan(m8[6], m8[6], m8[7]));
        }
        mx = mx < INFINITY ? mx * a.c : __uint_as_float(0x7fc00000u);
        const bool grow = !(mx <= ref + kSlack) && mx != -INFINITY;
        if (__any_sync(0xffffffffu, grow)) {
          const float f = grow ? ex2f(ref - mx) : 1.f;      // (0 for a row that saw nothing before)
          if (grow) ref = mx;
          l *= f;
          if (done > 0) {
            ok = __all_sync(0xffffffffu, wait_cta(&o_done[turn(done - 1)], phase(done - 1), kPolls));
            if (!ok) break;
            fence_after();
#pragma unroll 1
            for (int q = 0; q < D / 32; ++q) {
              uint32_t o[32];
              tmem_ld32(o_at + 32 * q, o);
              asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
              for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
              tmem_st32(o_at + 32 * q, o);
            }
          }
        }
        const float r = ref == -INFINITY ? 0.f : ref;
        float sums[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < 64; ++i) {                       // (scores of -inf give 0)
          const float x0 = ex2f(fmaf(__uint_as_float(s[i >> 4][2 * (i & 15)]), a.c, -r)), x1 = ex2f(fmaf(__uint_as_float(s[i >> 4][2 * (i & 15) + 1]), a.c, -r));
          sums[2 * (i & 1)] += x0;
          sums[2 * (i & 1) + 1] += x1;
          p[i] = pack2(x0, x1);
        }
        sum = (sums[0] + sums[1]) + (sums[2] + sums[3]);
      }
      tmem_st32(s_at, *(const uint32_t(*)[32])&p[0]);
      tmem_st32(s_at + 32, *(const uint32_t(*)[32])&p[32]);
      asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
      fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_ready[turn(done)]);
      l += sum;
      ++done;
    }
    if (ok && done > 0) ok = __all_sync(0xffffffffu, spin_cta(&o_done[turn(done - 1)], phase(done - 1)));
    fence_after();
    if (!ok && lane == 0 && !s_fail) failed(504);
    bool poisoned = false;
    const int notes = *(volatile int*)&noted;
    for (int i = 0; i < notes && i < kNotes; ++i)
      for (uint32_t m = *(volatile uint32_t*)&note_bits[i]; m; m &= m - 1) {
        const int key = *(volatile int*)&note_key[i] + __ffs(m) - 1;
        poisoned |= key <= pos && (plan.window == 0 || key > pos - plan.window || key < plan.sinks);
      }
    if (a.split > 1) {
      // Every CTA of the cluster takes 256 / split rows of the two tiles.  The sums are laid out in the CTA's own ring, and read by the others a row a warp (written to the others a row a thread, 16 bytes at a time, they took
      // 40 us).
      const int r_all = t * kTile + in_tile;
      if (poisoned) ref = __uint_as_float(0x7fc00000u);
      __syncwarp();
      unsigned char* const sums = smem + 2 * SH::BYTES;
      float2* const stats = (float2*)(sums + 2 * kTile * D * 4);
      asm volatile("bar.sync 1, 256;" ::: "memory");         // (the other tile is done with the ring, too)
#pragma unroll 1
      for (int q = 0; q < D / 32; ++q) {
        uint32_t o[32];
        if (done > 0) {
          tmem_ld32(o_at + 32 * q, o);
          asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = 0u;
        }
#pragma unroll
        for (int c = 0; c < 8; ++c)
          *(uint4*)(sums + r_all * (D * 4) + (((8 * q + c) ^ (r_all & 7)) << 4)) = make_uint4(o[4 * c], o[4 * c + 1], o[4 * c + 2], o[4 * c + 3]);
      }
      stats[r_all] = make_float2(ref, l);
      __syncwarp();
      cluster_sync_tc();
      // out = (sum o_s w_s) / (sum l_s w_s), w_s = 2^(r_s - max r): 4 values of a row a thread
      const uint32_t sums_a = smem_u32(sums), stats_a = smem_u32(stats);
      constexpr int CQ = D / 4;
      auto join = [&](auto split_c) {                        // 16 pieces asked for at a time
        constexpr int S = decltype(split_c)::value, kItems = 16 / S, kRows = 2 * kTile / S;
        float2* const got = stats + 2 * kTile;               // [rank][row] of this CTA's rows
        asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(got[tid].x), "=f"(got[tid].y)
                     : "r"(cluster_addr(stats_a + (uint32_t)(rank * kRows + tid % kRows) * 8u, (uint32_t)(tid / kRows))));
        asm volatile("bar.sync 1, 256;" ::: "memory");
#pragma unroll 1
        for (int i0 = tid; i0 < kRows * CQ; i0 += 2 * kTile * kItems) {
          float4 x[kItems][S];
#pragma unroll
          for (int j = 0; j < kItems; ++j) {
            const int i = i0 + j * 2 * kTile, mine = rank * kRows + (i < kRows * CQ ? i / CQ : 0), c = i % CQ;
#pragma unroll
            for (int k = 0; k < S; ++k) {
              asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(x[j][k].x), "=f"(x[j][k].y), "=f"(x[j][k].z), "=f"(x[j][k].w)
                           : "r"(cluster_addr(sums_a + (uint32_t)(mine * (D * 4) + ((c ^ (mine & 7)) << 4)), (uint32_t)k)));
            }
          }
#pragma unroll
          for (int j = 0; j < kItems; ++j) {
            const int i = i0 + j * 2 * kTile, r = i / CQ, c = i % CQ, mine = rank * kRows + r, tt = mine / kTile, rr = (tt ? row1 : row0) + mine - tt * kTile;
            if (i >= kRows * CQ || rr >= a.Tq) continue;
            float top = -INFINITY, L = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
            float2 rl[S];
#pragma unroll
            for (int k = 0; k < S; ++k) { rl[k] = got[k * kRows + r]; top = fmaxf(top, rl[k].x); }
#pragma unroll
            for (int k = 0; k < S; ++k)
              if (!(rl[k].x == -INFINITY)) {                 // (nothing was seen there)
                const float w = ex2f(rl[k].x - top);
                L = fmaf(rl[k].y, w, L);
                o[0] = fmaf(x[j][k].x, w, o[0]); o[1] = fmaf(x[j][k].y, w, o[1]); o[2] = fmaf(x[j][k].z, w, o[2]); o[3] = fmaf(x[j][k].w, w, o[3]);
              }
            const float inv = L > 0.f ? 1.f / L : (L == L ? 0.f : L);
            uint16_t* p = a.out + (int64_t)b * a.o_str[0] + (int64_t)(tt ? head1 : head0) * a.o_str[1] + (int64_t)rr * a.o_str[2] + 4 * c;
            const uint32_t w0 = pack2(o[0] * inv, o[1] * inv), w1 = pack2(o[2] * inv, o[3] * inv);
            if (a.o_vec) *(uint2*)p = make_uint2(w0, w1);
            else { p[0] = (uint16_t)w0; p[1] = (uint16_t)(w0 >> 16); p[2] = (uint16_t)w1; p[3] = (uint16_t)(w1 >> 16); }
          }
        }
      };
      if (a.split == 2) join(std::integral_constant<int, 2>{});
      else if (a.split == 4) join(std::integral_constant<int, 4>{});
      else join(std::integral_constant<int, 8>{});
      __syncwarp();
      cluster_sync_tc();                                     // (shared memory stays until all have read it)
    } else {
      const float inv = poisoned ? __uint_as_float(0x7fc00000u) : (l > 0.f ? 1.f / l : (l == l ? 0.f : l));
      // The results go through shared memory, in the place of the warp's own queries, so that a store covers whole rows (a thread a
      // row, 32 rows a store, took 5000 cycles); 16-byte chunks swizzled by the row.
      // (a tile that saw nothing has not waited for its queries, which must have arrived before anything is put in their place)
      if (plan.blocks > 0 && done == 0 && !__all_sync(0xffffffffu, wait_cta(&q_full, 0, kPolls)) && lane == 0 && !s_fail) failed(504);
      unsigned char* const stage = smem + t * SH::BYTES + (warp & 3) * (32 * D * 2);
      constexpr int CH = D / 8;
#pragma unroll 1
      for (int q = 0; q < D / 32; ++q) {
        uint32_t o[32];
        if (done > 0) {
          tmem_ld32(o_at + 32 * q, o);
          asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = 0u;
        }
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t w[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) w[i] = pack2(__uint_as_float(o[8 * c + 2 * i]) * inv, __uint_as_float(o[8 * c + 2 * i + 1]) * inv);
          *(uint4*)(stage + lane * (D * 2) + (((4 * q + c) ^ (lane & 7)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
        }
      }
      __syncwarp();
      uint16_t* out = a.out + (int64_t)b * a.o_str[0] + (int64_t)(t ? head1 : head0) * a.o_str[1];
      const int first = row - lane;
#pragma unroll 4
      for (int i = lane; i < 32 * CH; i += 32) {
        const int r = i / CH, c = i % CH;
        if (first + r >= a.Tq) break;
        const uint4 v = *(const uint4*)(stage + r * (D * 2) + ((c ^ (r & 7)) << 4));
        uint16_t* p = out + (int64_t)(first + r) * a.o_str[2] + 8 * c;
        if (a.o_vec) *(uint4*)p = v;
        else {
          const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
          for (int k = 0; k < 4; ++k) { p[2 * k] = (uint16_t)w[k]; p[2 * k + 1] = (uint16_t)(w[k] >> 16); }
        }
      }
    }
  }
  __syncwarp();
  fence_before();
  __syncthreads();
  if (warp == 9) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u));
}

// [T, H, B] rows of D values as boxes of 64 x 128; broadcast axes as one entry at coordinate 0.
bool rows_map(CUtensorMap* m, const void* base, int64_t D, const int64_t (&shape)[3], const int64_t (&str)[3], int* mul) {
  const EncodeFn enc = get_encode();
  cuuint64_t dims[4] = {(cuuint64_t)D, (cuuint64_t)shape[2], 1, 1}, strides[3] = {(cuuint64_t)str[2] * 2, (cuuint64_t)D * 2, (cuuint64_t)D * 2};
  if (shape[2] == 1) strides[0] = (cuuint64_t)D * 2;
  for (int d = 0; d < 2; ++d) {            // head, sequence
    mul[d] = shape[1 - d] > 1 && str[1 - d] > 0 ? 1 : 0;
    if (mul[d]) { dims[2 + d] = (cuuint64_t)shape[1 - d]; strides[1 + d] = (cuuint64_t)str[1 - d] * 2; }
  }
  const cuuint32_t box[4] = {64, kTile, 1, 1}, es[4] = {1, 1, 1, 1};
  return enc && enc(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, (void*)base, dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                    CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// How many CTAs, clusters of 2, 4 and 8 of the kernel the device holds at once.
template <int D> cudaError_t places(int (&fit)[4]) {
  auto kern = window_attn_kernel<D, false>;
  static int cached[64][4] = {};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  std::lock_guard<std::mutex> setup_lk(setup_mutex());       // first use on a device, from any thread
  if (dev < 0 || dev >= 64 || cached[dev][0] == 0) {
    e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape<D>::SMEM);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(window_attn_kernel<D, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape<D>::SMEM);
    if (e != cudaSuccess) return e;
    fit[0] = sm_count();
    for (int i = 1; i < 4; ++i) {
      cudaLaunchConfig_t cfg = {};
      cfg.gridDim = dim3(1u << i);
      cfg.blockDim = dim3(kThreads);
      cfg.dynamicSmemBytes = Shape<D>::SMEM;
      cudaLaunchAttribute attr[1];
      attr[0].id = cudaLaunchAttributeClusterDimension;
      attr[0].val.clusterDim.x = 1u << i; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
      cfg.attrs = attr;
      cfg.numAttrs = 1;
      if (cudaOccupancyMaxActiveClusters(&fit[i], kern, &cfg) != cudaSuccess) {
        (void)cudaGetLastError();
        fit[i] = 0;
      }
    }
    if (dev >= 0 && dev < 64)
      for (int i = 0; i < 4; ++i) cached[dev][i] = fit[i];
  } else
    for (int i = 0; i < 4; ++i) fit[i] = cached[dev][i];
  return cudaSuccess;
}

template <int D> cudaError_t launch_d(const WindowArgs& w, cudaStream_t st) {
  WindowK a;
  a.out = (uint16_t*)w.out; a.kv_lens = w.kv_lens;
  for (int i = 0; i < 3; ++i) a.o_str[i] = w.o_str[i];
  a.o_vec = w.o_vec;
  a.B = (int)w.B; a.Hq = (int)w.Hq; a.gqa = (int)(w.Hq / w.Hkv); a.Tq = (int)w.Tq; a.Tk = (int)w.Tk;
  a.window = w.window; a.sinks = w.sinks;
  a.c = w.scale * 1.4426950408889634f;
  CUtensorMap m[3];
  const int64_t qs[3] = {w.B, w.Hq, w.Tq}, ks[3] = {w.B, w.Hkv, w.Tk};
  if (!rows_map(&m[0], w.q, D, qs, w.str[0], a.mul[0]) || !rows_map(&m[1], w.k, D, ks, w.str[1], a.mul[1]) || !rows_map(&m[2], w.v, D, ks, w.str[2], a.mul[2]))
    return cudaErrorInvalidValue;
  auto kern = window_attn_kernel<D, false>;
  int fit[4];
  cudaError_t e = places<D>(fit);
  if (e != cudaSuccess) return e;
  // Two tiles a CTA, which fill the tensor cores between them, where there are enough for all SMs.  Where there are not: one tile a CTA,
  // whose step takes 1.03 us (two tiles' 1.75), or clusters that share a tile's keys, as many as the device places at once (of 8
  // CTAs it places fewer than 16), which takes 8 to 10 us for the join.  Of the forms that run in one wave the one that
  // should end first is taken.  (32 query heads of 128 on 8, two tiles by clusters / one tile: 512 queries, 4099 keys, a window of 1024 35 us
  // alone / 27 alone; without a window 51 by 2 / 48 alone; 512 on 16384 130 by 2 / 142 alone; 256 on 4096 34 by 4 / 36 by 2;
  // 64 on 8192 46 by 4 / 35 by 4; 128 on 32768 125 by 4 / 85 by 4.  All at head dim 128; at 64, where a step and a join move half as much,
  // the same constants choose, unmeasured.)
  auto shape = [&](bool single) {
    a.heads2 = !single && a.gqa % 2 == 0;
    const int rows = a.heads2 || single ? kTile : 2 * kTile;
    a.qblocks = (a.Tq + rows - 1) / rows;
    return (int64_t)a.qblocks * (a.heads2 ? a.Hq / 2 : a.Hq) * a.B;
  };
  const int64_t tiles[2] = {shape(false), shape(true)};
  int64_t most = (w.Tk + kTile - 1) / kTile;                 // steps of a tile
  if (w.window > 0) {
    const int64_t seen = (w.window + (int64_t)kTile + kTile - 2) / kTile + 1 + (w.sinks + kTile - 1) / kTile;
    most = most < seen ? most : seen;
  }
  bool single = false;
  float best = 1.7f * (float)most;
  a.split = 1;
  for (int one = 0; one < 2; ++one)
    for (int i = 0; i < 4; ++i) {
      if (tiles[one] > fit[i]) continue;
      const float steps = (one ? 1.f : 1.7f) * (float)((most + (1 << i) - 1) >> i) + (i ? 8.f : 0.f);
      if (steps < best) { best = steps; single = one; a.split = 1 << i; }
    }
  if (single) kern = window_attn_kernel<D, true>;
  const int64_t ctas = shape(single);
  if (a.split > 1) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(ctas * a.split));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = Shape<D>::SMEM;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)a.split; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    e = launch_clusters(cfg, kern, m[0], m[1], m[2], a);
    if (e == cudaSuccess) return e;
    (void)cudaGetLastError();            // the device places no clusters after all: every tile by itself
    a.split = 1;
  }
  return launch_behind(kern, dim3((unsigned)ctas), dim3(kThreads), Shape<D>::SMEM, st, m[0], m[1], m[2], a);
}
}  // namespace

cudaError_t launch_window_attn(const WindowArgs& w, cudaStream_t st) { return w.D == 64 ? launch_d<64>(w, st) : launch_d<128>(w, st); }

void window_attn_error_reset() {
  const int zero = 0;
  cudaMemcpyToSymbol(g_window_error, &zero, sizeof(int));
}
int window_attn_error_code() {
  int v = 0;
  cudaMemcpyFromSymbol(&v, g_window_error, sizeof(int));
  return v;
}

}  // namespace qb
