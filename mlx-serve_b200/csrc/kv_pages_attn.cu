// Attention of one new token over a paged key-value cache, 4- or 8-bit codes or bf16 rows, head dim 64 or 128, with an optional
// window and a few first tokens that stay visible.
//
// o = sum_j p_j v_j, p = softmax_j(scale * q . k_j) over the cached tokens j < len that the newest token sees: all of them, or
// j < sinks and j >= len - window.  The codes are read once, straight from their pages; with q*s + b the weight terms stay in
// fp32: s scales sums of codes, b meets the group sums of q (keys) or is summed with p (values).
//
//  * Work.  A unit is a block of 64 tokens of one (sequence, cache head, tile of 8 query heads).  The grid is what the device holds
//    at once; every CTA works out all lengths' units from `lens` and takes an even share of their total, so that ragged batches stay
//    balanced with lengths that only the device knows.  A share cuts at most two sequences; their parts go to the workspace and a
//    second kernel joins them, whole sequences are stored directly.
//  * A warp walks blocks of 64 tokens with its own softmax (running maximum and sum per query in fp32) and its own cp.async ring.
//    Page numbers are read a block ahead; rows that the query does not see are not read, their place is zeroed.
//  * Codes are the A operand of the fp16 tensor cores: 16 tokens x 16 dims for the scores, 16 dims x 16 tokens for the values, the
//    8 queries the B operand, so that a matrix instruction takes 256 codes (as the B operand it would take 128).  A code in the low
//    bits of a 16-bit word IS the fp16 subnormal c * 2^-24: one AND makes an operand register; the next nibble is 16 times that.
//    The value operand comes out of ldmatrix.m16n16.trans.b8, four tokens of a byte column a lane.
//  * Queries are scaled by a power of two into fp16's range: the row's largest lies in [2^14, 2^15), so that a bf16 is exact down to 2^-31
//    of it (2^-27 for the odd dims at 4 bits, whose operand is a sixteenth), with an error of half of fp16's smallest step, 2^-24, below.
//    The probabilities times the value scale are rounded once to fp16 (2^-11 relative, against 2^-8 of the bf16 result); the value
//    scales of a group are multiplied by a power of two of the group's own that keeps p * v_scale below 2^15, so that neither the other
//    group's size nor what is not finite there counts for it.  Tokens whose p * v_scale is so far below the largest that some query of
//    the tile meets (2^29) that it drops under fp16's normal range keep an error of 2^-25 in its place.  At 16 bits the probabilities
//    stay a sum of two bf16 (16 bits).  The score tile's layout becomes the B operand of the next product by movmatrix.
//
// Floor: the visible rows' bytes at the copy bandwidth (6.54 TB/s measured).  Sequences of 16k to 32k tokens, 16 of them, 32 query heads on 8 of
// 128, pages of 64: 4 bits 463 MB, floor 71 us, takes 104 to 112 on different GPUs (4.1 to 4.4 TB/s); 8 bits 874 MB, 134 and 156; bf16
// 1.64 GB, 251 and 258.  At 4 bits the issue slots bound it: 278 warp instructions per 16 tokens, 7 of them for the groups' units (406 before
// a token's four neighbours were placed for wide scale loads and the rescaling became lazy), 56 % of the slots used with the 12 warps
// an SM that 168 registers leave; 128 registers and 16 warps spill and take 126 to 137 us, 5 warps a CTA 127.  Short calls wait for
// dependent reads (lengths, table, rows) and the join: one sequence of 700 tokens takes 9.7 to 10.1 us, 12.3 before the kernels were launched
// behind one another.
#include <mutex>
#include <type_traits>

#include "kernels.h"
#include "stream_ptx.cuh"

namespace qb {
namespace {

constexpr int kWarps = 4;
constexpr int kBlk = 64;              // tokens per unit
constexpr int kRows = 8;              // queries per tile
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kNegBig = -1e30f;
constexpr int kMergeWarps = 16;
constexpr int kLowExp = 60;           // the exponent (biased by 127) that a group's value scales are taken to have at least: 2^-67
constexpr int kPiece = 3;             // what a piece of a sequence takes beside its blocks, in blocks of a warp

template <int BITS, int D> struct Geo {
  static constexpr int G = BITS == 16 ? 1 : D / 64;       // scale groups per token
  static constexpr int ROWB = D * BITS / 8;               // bytes per token
  static constexpr int CH = ROWB / 16;                    // 16-byte chunks per token
  static constexpr int TOK = ROWB >= 256 ? 16 : 32;       // tokens per ring stage
  static constexpr int STAGE = TOK * ROWB;
  static constexpr int STAGES = 4;
  static constexpr int ITEMS = 2 * kBlk / TOK;            // stages per block: K, then V
  static constexpr int SB = BITS == 16 ? 0 : kBlk * G * 2;    // bytes of one of {ks, kb, vs, vb} for a block
  static constexpr int RING = STAGES * STAGE;
  static constexpr int NT = D / 16;                       // 16-dim tiles of the output
  static constexpr int SMEM_MAIN = kWarps * (RING + 2 * 4 * SB);
  static constexpr int WROW = D + 4;                      // a query's row of a warp's result, padded against bank conflicts
  static constexpr int SMEM_MERGE = kWarps * kRows * (WROW + 2) * 4;
  static constexpr int SMEM = SMEM_MAIN > SMEM_MERGE ? SMEM_MAIN : SMEM_MERGE;
};

template <int BITS, int CH> __device__ __forceinline__ int swz(int row) {
  if (BITS == 16) return row & 7;
  int f = (row >> 3) & 1;
  if (CH >= 4) f |= ((row >> 1) & 1) << 1;
  if (CH >= 8) f |= (row & 1) << 2;
  return f;
}
// Where a stage's token lies in shared memory: at 4 and 8 bits the four tokens 4g .. 4g + 3 of its 32 are rows g, g + 8, g + 16, g + 24, so
// that the tokens whose scores a lane holds have their scales side by side.
template <int BITS> __device__ __forceinline__ int place(int tok) { return BITS == 16 ? tok : (tok & 3) * 8 + (tok >> 2); }
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
// D = A B (+ D unless the sum begins): no registers to clear first
__device__ __forceinline__ void mma_f16_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1, bool first) {
  if (first)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
  else mma_f16_16816(d, a0, a1, a2, a3, b0, b1);
}
__device__ __forceinline__ void mma_bf16_1688_z(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t b) {
  asm("mma.sync.aligned.m16n8k8.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5}, {%6}, {%7,%7,%7,%7};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3]) : "r"(a0), "r"(a1), "r"(b), "f"(0.f));
}
// bf16 pairs times bf16 pairs: exact for powers of two
__device__ __forceinline__ uint32_t mul_bf16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
// bf16 parameters of four consecutive tokens, G a token, each token's in one register (at G = 1 in its low half)
template <int G> __device__ __forceinline__ void load4(uint32_t (&r)[4], const unsigned char* p) {
  if constexpr (G == 2) {
    const uint4 v = *(const uint4*)p;
    r[0] = v.x; r[1] = v.y; r[2] = v.z; r[3] = v.w;
  } else {
    const uint2 v = *(const uint2*)p;
    r[0] = v.x & 0xFFFFu; r[1] = v.x >> 16; r[2] = v.y & 0xFFFFu; r[3] = v.y >> 16;
  }
}
template <bool TRANS> __device__ __forceinline__ void ldmatrix_b16_x4(uint32_t (&r)[4], uint32_t addr) {
  if constexpr (TRANS)
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
  else
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}

// What the newest token of a sequence sees, in blocks of 64 tokens.
struct Seen {
  int len, w0, sinks;       // tokens; start of the window
  int front, skip;          // blocks [0, front) and, from there on, block i + skip
  int blocks;
};
__device__ __forceinline__ Seen seen_of(const KvPagesAttnArgs& a, int64_t b) {
  Seen s;
  const int64_t row = a.rows ? a.rows[b] : b;
  int64_t len = row >= 0 && row < a.seqs ? a.lens[row] : 0;
  const int64_t cap = (int64_t)a.M << a.page_shift;
  len = len < 0 ? 0 : (len > cap ? cap : len);
  s.len = (int)len;
  const int nb = (int)((len + kBlk - 1) / kBlk);
  s.w0 = a.window > 0 && a.window < len ? (int)(len - a.window) : 0;
  s.sinks = a.sinks < s.len ? a.sinks : s.len;
  s.front = (int)(((int64_t)s.sinks + kBlk - 1) / kBlk);
  s.skip = s.w0 / kBlk - s.front;
  if (s.skip < 0) s.skip = 0;
  s.blocks = nb - s.skip;
  return s;
}

// All lengths, as every CTA reads them: the units before each sequence, and what the cut is decided by.  Up to 32 sequences a warp keeps
// them in registers, one a lane (no barrier, no second look at memory); above, they lie in shared memory.
struct Lengths {
  Seen mine; int before;      // of sequence `lane` (B <= 32)
  int all, longest;           // units; blocks of the longest sequence
};
__device__ __forceinline__ int warp_scan(int v) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += u;
  }
  return v;
}
__device__ __forceinline__ Lengths read_lengths(const KvPagesAttnArgs& a, int* units, int* warp_sums) {
  Lengths L;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (a.B <= 32) {
    if (lane < a.B) L.mine = seen_of(a, lane);
    else { L.mine.len = L.mine.w0 = L.mine.sinks = L.mine.front = L.mine.skip = L.mine.blocks = 0; }
    const int n = L.mine.blocks * a.tiles, upto = warp_scan(n);
    L.before = upto - n;
    L.all = __shfl_sync(0xffffffffu, upto, 31);
    L.longest = __reduce_max_sync(0xffffffffu, L.mine.blocks);
    return L;
  }
  const int each = (a.B + kWarps * 32 - 1) / (kWarps * 32), b0 = tid * each;
  int mine = 0, longest = 0;
  for (int i = 0; i < each && b0 + i < a.B; ++i) {
    const int n = seen_of(a, b0 + i).blocks;
    units[b0 + i] = mine;
    mine += n * a.tiles;
    longest = n > longest ? n : longest;
  }
  const int upto = warp_scan(mine);
  longest = __reduce_max_sync(0xffffffffu, longest);
  if (lane == 31) { warp_sums[warp] = upto; warp_sums[kWarps + warp] = longest; }
  __syncthreads();
  int before = upto - mine;
  L.all = 0; L.longest = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) before += warp_sums[w];
    L.all += warp_sums[w];
    L.longest = warp_sums[kWarps + w] > L.longest ? warp_sums[kWarps + w] : L.longest;
  }
  for (int i = 0; i < each && b0 + i < a.B; ++i) units[b0 + i] += before;
  if (tid == 0) units[a.B] = L.all;
  __syncthreads();
  return L;
}
__device__ __forceinline__ Seen seen_from(const Lengths& L, int b) {
  Seen s;
  s.len = __shfl_sync(0xffffffffu, L.mine.len, b); s.w0 = __shfl_sync(0xffffffffu, L.mine.w0, b); s.sinks = __shfl_sync(0xffffffffu, L.mine.sinks, b);
  s.front = __shfl_sync(0xffffffffu, L.mine.front, b); s.skip = __shfl_sync(0xffffffffu, L.mine.skip, b); s.blocks = __shfl_sync(0xffffffffu, L.mine.blocks, b);
  return s;
}

template <int BITS, int D>
__global__ void __launch_bounds__(kWarps * 32, 3) kv_pages_kernel(const __grid_constant__ KvPagesAttnArgs a) {
  using GE = Geo<BITS, D>;
  constexpr int G = GE::G, CH = GE::CH, TOK = GE::TOK, ITEMS = GE::ITEMS, STAGES = GE::STAGES;
  extern __shared__ __align__(128) unsigned char smem[];
  int* const units = (int*)(smem + GE::SMEM);      // [B + 1], above 32 sequences
  __shared__ int warp_sums[2 * kWarps];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;");
  const bool few = a.B <= 32;
  const Lengths L = read_lengths(a, units, warp_sums);
  // sequences that see nothing: zeros
  for (int b = blockIdx.x; b < a.B; b += gridDim.x)
    if ((few ? __shfl_sync(0xffffffffu, L.mine.blocks, b) : units[b + 1] - units[b]) == 0)
      for (int i = tid; i < a.Hq * D; i += kWarps * 32) ((uint16_t*)a.out)[(int64_t)b * a.o_str[0] + (int64_t)(i / D) * a.o_str[1] + i % D] = 0;

  // The cut: an even share of all units for every CTA, or every sequence in the same number of parts, whichever ends first by blocks a
  // warp walks and what a piece takes beside them (about kPiece blocks' time): even shares cut long ragged batches best, parts keep a
  // CTA from working on the ends of two short sequences.  (By even shares and in parts, us: 16 sequences of 16k to 32k tokens 110 and 122; 48
  // of 1k to 2k 41 and 31; 32 windows of 1024 tokens at 16 bits 24.4 and 18.3; 13 of 4k to 8k at 8 bits 32.1 and 28.6; one of 700 tokens 13.8
  // and 10.1; these go by the better one.  4 of 4k to 8k, 16.4 and 18.3, go in parts: the estimate is off there.)
  const int U = L.all, ctas = (int)gridDim.x, seqs = a.B * a.tiles;
  int per = (U + ctas - 1) / ctas;
  per = per < a.min_units ? a.min_units : per;
  int parts = ctas / seqs;                              // 0: even shares
  if (parts > 0) {
    const int most = (L.longest + a.min_units - 1) / a.min_units;
    parts = parts > most ? (most < 1 ? 1 : most) : parts;
    const int pieces = 1 + (int)ceilf(__fdividef((float)per * (float)seqs, (float)(U > 0 ? U : 1)));   // that an even share touches
    if ((L.longest + parts - 1) / parts + kPiece * kWarps > per + pieces * kPiece * kWarps) parts = 0;
  }
  int64_t u_from = (int64_t)blockIdx.x * per;
  int u_to = u_from + per < U ? (int)(u_from + per) : U;
  if (tid == 0) a.joins[blockIdx.x] = make_int4(-1, 0, 0, 0);

  const uint32_t my_ring = (uint32_t)__cvta_generic_to_shared(smem + (size_t)warp * GE::RING);
  const unsigned char* my_ring_p = smem + (size_t)warp * GE::RING;
  unsigned char* my_sb_p = smem + (size_t)kWarps * GE::RING + (size_t)warp * 2 * 4 * GE::SB;
  const uint32_t my_sb = (uint32_t)__cvta_generic_to_shared(my_sb_p);

  int b = 0;
  bool next = parts > 0 ? (int)blockIdx.x < seqs * parts : u_from < U;
  for (int u = (int)u_from; next;) {
    Seen sn;
    int tile, blk0, todo, more;                      // blocks [blk0, blk0 + todo) of the tile; how many CTAs behind this one share it
    if (parts > 0) {
      const int seq = (int)blockIdx.x / parts, part = (int)blockIdx.x - seq * parts;
      b = seq / a.tiles;
      tile = seq - b * a.tiles;
      sn = few ? seen_from(L, b) : seen_of(a, b);
      const int mine = parts < sn.blocks ? parts : sn.blocks;
      if (part >= mine) return;
      const int each = sn.blocks / mine, rest = sn.blocks - each * mine;
      blk0 = each * part + (part < rest ? part : rest);
      todo = each + (part < rest ? 1 : 0);
      more = mine - 1;
      next = false;
    } else {
      int before;
      if (few) {
        b = 31 - __clz(__ballot_sync(0xffffffffu, L.before <= u && L.mine.blocks > 0));
        before = __shfl_sync(0xffffffffu, L.before, b);
        sn = seen_from(L, b);
      } else {
        int hi = a.B - 1;                            // (the last one that begins at u or before: empty ones share their begin with the next)
        while (b < hi) {
          const int mid = (b + hi + 1) >> 1;
          if (units[mid] <= u) b = mid; else hi = mid - 1;
        }
        before = units[b];
        sn = seen_of(a, b);
      }
      tile = (u - before) / sn.blocks;
      blk0 = u - before - tile * sn.blocks;
      const int left = sn.blocks - blk0;
      todo = left < u_to - u ? left : u_to - u;
      more = (before + (tile + 1) * sn.blocks - 1) / per - (int)blockIdx.x;
      u += todo;
      next = u < u_to;
    }
    const int hk = tile / a.qtiles, qt = tile - hk * a.qtiles;
    const int row = a.rows ? a.rows[b] : b;
    const int32_t* tab = a.table + (int64_t)row * a.table_str;
    const int my_blocks = warp < todo ? (todo - warp + kWarps - 1) / kWarps : 0;
    const int pmask = (1 << a.page_shift) - 1;
    auto first_token = [&](int j) { const int i = blk0 + warp + j * kWarps; return (i < sn.front ? i : i + sn.skip) * kBlk; };
    auto visible = [&](int tok) { return tok < sn.len && (tok >= sn.w0 || tok < sn.sinks); };

    // ---- queries: row g of the tile, asked for before anything else ----
    const bool q_live = qt * kRows + g < a.gqa;
    const uint16_t* const qp = (const uint16_t*)a.q + (int64_t)b * a.q_str[0] + (int64_t)(hk * a.gqa + (q_live ? qt * kRows + g : 0)) * a.q_str[1];
    uint32_t qraw[D / 16][2];        // at 16 bits the operand, else dims 16 t .. 16 t + 15 of a group in eight registers
    if constexpr (BITS == 16) {
#pragma unroll
      for (int s = 0; s < D / 16; ++s)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint16_t* p = qp + 16 * s + 2 * t + 8 * h;
          qraw[s][h] = (uint32_t)p[0] | ((uint32_t)p[1] << 16);
        }
    } else {
#pragma unroll
      for (int grp = 0; grp < G; ++grp) {
        const uint16_t* p = qp + grp * 64 + 16 * t;
        if (a.q_vec) {
          const uint4 x = ((const uint4*)p)[0], y = ((const uint4*)p)[1];
          qraw[4 * grp][0] = x.x; qraw[4 * grp][1] = x.y; qraw[4 * grp + 1][0] = x.z; qraw[4 * grp + 1][1] = x.w;
          qraw[4 * grp + 2][0] = y.x; qraw[4 * grp + 2][1] = y.y; qraw[4 * grp + 3][0] = y.z; qraw[4 * grp + 3][1] = y.w;
        } else {
#pragma unroll
          for (int k = 0; k < 8; ++k) qraw[4 * grp + (k >> 1)][k & 1] = (uint32_t)p[2 * k] | ((uint32_t)p[2 * k + 1] << 16);
        }
      }
    }

    // ---- producer ----
    // lane l holds the page of the 16 tokens from 16 * (l & 3) on, -1 where there is none
    auto page_at = [&](int j) {
      int pid = -1;
      if (j < my_blocks) {
        const int tok = first_token(j) + 16 * (lane & 3);
        if (tok < sn.len) pid = tab[tok >> a.page_shift];
        if (pid >= a.P) pid = -1;
      }
      return pid;
    };
    constexpr int RPI = 32 / CH;                          // token rows of one copy instruction
    const int cc = lane % CH, r0 = lane / CH;
    const unsigned char* const base_k = (const unsigned char*)a.pool[0].q + (int64_t)hk * a.q_head[0] + (int64_t)r0 * a.tok_bytes[0] + cc * 16;
    const unsigned char* const base_v = (const unsigned char*)a.pool[1].q + (int64_t)hk * a.q_head[1] + (int64_t)r0 * a.tok_bytes[1] + cc * 16;
    // scales and biases of a block, [ks, kb, vs, vb][64 tokens][G]: 16-byte pieces, G of them a lane (ks or kb, then vs or vb; at G = 1 one of the four)
    constexpr int TP = 8 / G;                             // tokens per piece
    const int sb_tok = lane % (kBlk / TP) * TP;
    const uint16_t* sb_at[G];
    if constexpr (BITS != 16) {
#pragma unroll
      for (int k = 0; k < G; ++k) {
        const int arr = (lane + 32 * k) / (kBlk / TP), kv = arr >> 1;
        const uint16_t* const p = (const uint16_t*)(arr == 0 ? a.pool[0].s : (arr == 1 ? a.pool[0].b : (arr == 2 ? a.pool[1].s : a.pool[1].b)));
        sb_at[k] = p + (int64_t)hk * (kv ? a.pool[1].sb_str[1] : a.pool[0].sb_str[1]);
      }
    }
    // what the block whose copies are being issued is: its first token, its pages, which 16 tokens have one, whether the query sees it all
    int pid_next = page_at(0), pid_cur = -1, blk_tok = 0;
    uint32_t vm_next = 0;
    bool whole_next = false;
    // the copies of stage `part` of block j (a constant in the loop over the blocks; the first three stages go through one copy of the
    // code: a short sequence waits for instructions more than for data)
    auto issue = [&](const int part, int j) {
      const int stage = part % STAGES;
      if (part == 0) {
        pid_cur = pid_next;
        blk_tok = first_token(j);
        vm_next = __ballot_sync(0xffffffffu, pid_cur >= 0) & 15u;
        whole_next = vm_next == 15u && blk_tok + kBlk <= sn.len && (blk_tok >= sn.w0 || blk_tok + kBlk <= sn.sinks);
        pid_next = page_at(j + 1);
        if constexpr (BITS != 16) {
          const uint32_t dst0 = my_sb + (j & 1) * 4 * GE::SB;
          if (a.sb_vec) {
            const int pid = __shfl_sync(0xffffffffu, pid_cur, sb_tok >> 4);
            const bool ok = pid >= 0 && blk_tok + sb_tok < sn.len;
            const int slot = ((blk_tok + sb_tok) & pmask) * G;
#pragma unroll
            for (int k = 0; k < G; ++k) {
              const bool v = G == 2 ? k == 1 : lane >= 16;
              const uint16_t* src = sb_at[k] + (int64_t)(ok ? pid : 0) * (v ? a.pool[1].sb_str[0] : a.pool[0].sb_str[0]) + slot;
              cp_async16_z(dst0 + (lane + 32 * k) * 16, src, ok ? 16u : 0u);
            }
          } else {
            uint16_t* dst = (uint16_t*)(my_sb_p + (j & 1) * 4 * GE::SB);
#pragma unroll
            for (int arr = 0; arr < 4; ++arr) {
              const KvPoolView& pl = a.pool[arr >> 1];
              const uint16_t* src = (const uint16_t*)((arr & 1) ? pl.b : pl.s) + (int64_t)hk * pl.sb_str[1];
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const int tk = h * 32 + lane;
                const int pid = __shfl_sync(0xffffffffu, pid_cur, tk >> 4);
#pragma unroll
                for (int c = 0; c < G; ++c)
                  dst[arr * (GE::SB / 2) + tk * G + c] = pid >= 0 && blk_tok + tk < sn.len
                      ? src[(int64_t)pid * pl.sb_str[0] + (int64_t)((blk_tok + tk) & pmask) * pl.sb_str[2] + c] : (uint16_t)0;
              }
            }
          }
        }
      }
      const bool V = part >= ITEMS / 2;
      const int tk0 = (part % (ITEMS / 2)) * TOK;
      const uint32_t page_b = a.page_bytes[V], tok_b = a.tok_bytes[V], st = my_ring + stage * GE::STAGE;
      auto copy = [&](auto all_c) {
#pragma unroll
        for (int s16 = 0; s16 < TOK / 16; ++s16) {        // 16 tokens lie in one page
          const int pid = __shfl_sync(0xffffffffu, pid_cur, tk0 / 16 + s16);
          const int tok = blk_tok + tk0 + s16 * 16;
          const unsigned char* src = (V ? base_v : base_k) + (uint64_t)(uint32_t)(pid < 0 ? 0 : pid) * page_b + (uint64_t)(uint32_t)(tok & pmask) * tok_b;
#pragma unroll
          for (int r = 0; r < 16 / RPI; ++r) {
            const int in = s16 * 16 + r * RPI + r0, rw = place<BITS>(in);
            const uint32_t dst = st + rw * GE::ROWB + ((cc ^ swz<BITS, CH>(rw)) << 4);
            if (decltype(all_c)::value) cp_async16(dst, src);
            else cp_async16_z(dst, src, pid >= 0 && visible(tok + r * RPI + r0) ? 16u : 0u);
            src += (uint64_t)tok_b * RPI;
          }
        }
      };
      if (whole_next) copy(std::true_type{}); else copy(std::false_type{});
    };
#define QB_PART(n) std::integral_constant<int, (n)>{}
#pragma unroll 1
    for (int part = 0; part < STAGES - 1; ++part) {
      if (my_blocks > 0) issue(part, 0);
      cp_async_commit();
    }

    // ---- the queries as the B operand ----
    uint32_t qf[D / 16][2];
    uint32_t qb = 0;                 // bias product: this lane's part of the group sums of query g
    float C0, C1;                    // factor of the scores of queries 2t and 2t + 1
    {
      // (the sign of the scale goes to the queries, so that the largest score is the largest sum; a factor of 0 would meet scores of -inf)
      const float factor = fmaxf(fabsf(a.scale) * kLog2e, 1e-30f);
      if constexpr (BITS == 16) {
#pragma unroll
        for (int s = 0; s < D / 16; ++s)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            qf[s][h] = q_live ? qraw[s][h] ^ (a.scale < 0.f ? 0x80008000u : 0u) : 0u;
          }
        C0 = C1 = factor;
      } else {
        float f[G][16], sum[G], mx = 0.f;
#pragma unroll
        for (int grp = 0; grp < G; ++grp) {
          sum[grp] = 0.f;
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            f[grp][2 * k] = q_live ? bf16lo(qraw[4 * grp + (k >> 1)][k & 1]) : 0.f; f[grp][2 * k + 1] = q_live ? bf16hi(qraw[4 * grp + (k >> 1)][k & 1]) : 0.f;
            mx = fmax_nan(mx, fmax_nan(fabsf(f[grp][2 * k]), fabsf(f[grp][2 * k + 1])));
            sum[grp] += f[grp][2 * k] + f[grp][2 * k + 1];
          }
          sum[grp] += __shfl_xor_sync(0xffffffffu, sum[grp], 1);
          sum[grp] += __shfl_xor_sync(0xffffffffu, sum[grp], 2);
        }
        mx = fmax_nan(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmax_nan(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        int e = (int)((__float_as_uint(mx) >> 23) & 0xFF) - 127;    // mx < 2^(e + 1)
        e = e < -100 ? -100 : (e > 110 ? 110 : e);
        const float up = a.scale < 0.f ? -pow2i(14 - e) : pow2i(14 - e);
        const float least = 1e-37f, qf2 = pow2i(24 - 14 + e) * factor, qc = poison_if(nonfinite(mx), qf2 < least ? least : qf2);
        C0 = __shfl_sync(0xffffffffu, qc, 8 * t);
        C1 = __shfl_sync(0xffffffffu, qc, 8 * t + 4);
        // s = qc * (scale * sum q~ c 2^-24 + bias * sum q~ 2^-24): the sum in three bf16 parts, one a lane
#pragma unroll
        for (int grp = 0; grp < G; ++grp) {
          float v = sum[grp] * up * 5.9604644775390625e-8f;
          uint16_t part = 0;
#pragma unroll
          for (int i = 0; i < 3; ++i) {
            const uint16_t pi = f32_to_bf16_bits(v);
            v -= bf16_bits_to_f32(pi);
            part = t == i ? pi : part;
          }
          qb |= (uint32_t)part << (16 * grp);
#pragma unroll
          for (int s = 0; s < 4; ++s) {
            const float* x = BITS == 4 ? &f[grp][8 * (s >> 1) + 2 * (s & 1)] : &f[grp][4 * s];
            if constexpr (BITS == 4) {   // codes j and j + 4 of a word, then 16 times codes j + 1 and j + 5
              qf[grp * 4 + s][0] = pack_f16x2(x[0] * up, x[4] * up);
              qf[grp * 4 + s][1] = pack_f16x2(x[1] * up * 0.0625f, x[5] * up * 0.0625f);
            } else {                     // codes 0 and 2 of a word, then 1 and 3
              qf[grp * 4 + s][0] = pack_f16x2(x[0] * up, x[2] * up);
              qf[grp * 4 + s][1] = pack_f16x2(x[1] * up, x[3] * up);
            }
          }
        }
      }
    }

    // the next stage of block j: what it takes to stay three stages ahead is issued, and its own copies are complete
    auto acquire = [&](auto it_c, int j) -> const unsigned char* {
      constexpr int it = decltype(it_c)::value, ahead = it + STAGES - 1;
      if constexpr (ahead < ITEMS) issue(ahead, j);
      else if (j + 1 < my_blocks) issue(ahead - ITEMS, j + 1);
      cp_async_commit();
      cp_async_wait<STAGES - 1>();
      __syncwarp();
      return my_ring_p + (it % STAGES) * GE::STAGE;
    };

    float r_run[2] = {kNegBig, kNegBig}, l_part[2] = {0.f, 0.f};
    // A group's value scales are multiplied by 2^(141 - e), e the largest exponent (biased by 127) of p * v_scale so far: as a pair of bf16,
    // whose own biased exponents are 268 - e.
    uint32_t v_unit = (uint32_t)(268 - kLowExp) << 7 | (G == 2 ? (uint32_t)(268 - kLowExp) << 23 : 0u);
    auto v_exp = [&](int grp) { return 268 - (int)((v_unit >> (16 * grp + 7)) & 0xFFu); };
    float O[GE::NT][4];
    float ob[G][2];
#pragma unroll
    for (int i = 0; i < GE::NT; ++i) O[i][0] = O[i][1] = O[i][2] = O[i][3] = 0.f;
#pragma unroll
    for (int i = 0; i < G; ++i) ob[i][0] = ob[i][1] = 0.f;

    for (int j = 0; j < my_blocks; ++j) {
      const int tok_blk = first_token(j);
      unsigned char* sbb = my_sb_p + (j & 1) * 4 * GE::SB;
      float sc[4][4];     // [16 tokens][token g | g + 8][query 2t | 2t + 1]
      const bool whole = whole_next;
      const uint32_t vm = vm_next;
      // ---------------- scores ----------------
      auto score_stage = [&](auto it_c) {
        constexpr int it = decltype(it_c)::value;
        const unsigned char* st = acquire(it_c, j);
        if constexpr (it == 0) {
          if constexpr (BITS != 16) {
            if (!whole) {             // parameters of rows that were not read: zero, whatever lies there
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const int tk = h * 32 + lane;
                if (!(visible(tok_blk + tk) && ((vm >> (tk >> 4)) & 1u)))
#pragma unroll
                  for (int i = 0; i < 4 * G; ++i) ((uint16_t*)(sbb + (i / G) * GE::SB))[tk * G + i % G] = 0;
              }
              __syncwarp();
            }
          }
        }
        uint32_t ks[4], kb[4];            // of the lane's four tokens 4g + i: sub s2 has i = 2 s2 (row g of the tile) and 2 s2 + 1 (row g + 8)
        if constexpr (BITS != 16) {
          load4<G>(ks, sbb + (it * TOK + 4 * g) * G * 2);
          load4<G>(kb, sbb + GE::SB + (it * TOK + 4 * g) * G * 2);
        }
#pragma unroll
        for (int s2 = 0; s2 < TOK / 16; ++s2) {
          const int sub = it * (TOK / 16) + s2;
          if constexpr (BITS == 16) {
            float d[4] = {0.f, 0.f, 0.f, 0.f};
            const int rw = s2 * 16 + (lane & 15);
            const uint32_t addr = (uint32_t)__cvta_generic_to_shared(st) + rw * GE::ROWB;
#pragma unroll
            for (int s = 0; s < D / 16; ++s) {
              uint32_t k4[4];
              ldmatrix_b16_x4<false>(k4, addr + (((2 * s + (lane >> 4)) ^ swz<BITS, CH>(rw)) << 4));
              mma_bf16_16816(d, k4, qf[s][0], qf[s][1]);
            }
            sc[sub][0] = d[0]; sc[sub][1] = d[1]; sc[sub][2] = d[2]; sc[sub][3] = d[3];
          } else {
            float d[G][4];
            const int ra = s2 * 16 + g, rb = ra + 8;
#pragma unroll
            for (int grp = 0; grp < G; ++grp) {
              uint32_t wa[4], wb[4];
              if constexpr (BITS == 4) {
                const int c = 2 * grp + (t >> 1), o = (t & 1) * 8;
                const uint2 x = *(const uint2*)(st + ra * GE::ROWB + ((c ^ swz<BITS, CH>(ra)) << 4) + o);
                const uint2 y = *(const uint2*)(st + rb * GE::ROWB + ((c ^ swz<BITS, CH>(rb)) << 4) + o);
                wa[0] = x.x; wa[1] = x.y; wb[0] = y.x; wb[1] = y.y;
              } else {
                const int c = 4 * grp + t;
                const uint4 x = *(const uint4*)(st + ra * GE::ROWB + ((c ^ swz<BITS, CH>(ra)) << 4));
                const uint4 y = *(const uint4*)(st + rb * GE::ROWB + ((c ^ swz<BITS, CH>(rb)) << 4));
                wa[0] = x.x; wa[1] = x.y; wa[2] = x.z; wa[3] = x.w;
                wb[0] = y.x; wb[1] = y.y; wb[2] = y.z; wb[3] = y.w;
              }
#pragma unroll
              for (int s = 0; s < 4; ++s) {
                uint32_t a0, a1, a2, a3;
                if constexpr (BITS == 4) {
                  const uint32_t x = (s & 1) ? wa[s >> 1] >> 8 : wa[s >> 1], y = (s & 1) ? wb[s >> 1] >> 8 : wb[s >> 1];
                  a0 = x & 0x000F000Fu; a1 = y & 0x000F000Fu; a2 = x & 0x00F000F0u; a3 = y & 0x00F000F0u;
                } else {
                  a0 = wa[s] & 0x00FF00FFu; a1 = wb[s] & 0x00FF00FFu; a2 = (wa[s] >> 8) & 0x00FF00FFu; a3 = (wb[s] >> 8) & 0x00FF00FFu;
                }
                mma_f16_first(d[grp], a0, a1, a2, a3, qf[grp * 4 + s][0], qf[grp * 4 + s][1], s == 0);
              }
            }
            float e[4], s0[G], s1[G];
            mma_bf16_1688_z(e, kb[2 * s2], kb[2 * s2 + 1], qb);
            s0[0] = bf16lo(ks[2 * s2]); s1[0] = bf16lo(ks[2 * s2 + 1]);
            if constexpr (G == 2) { s0[G - 1] = bf16hi(ks[2 * s2]); s1[G - 1] = bf16hi(ks[2 * s2 + 1]); }
#pragma unroll
            for (int grp = 0; grp < G; ++grp) {
              e[0] = fmaf(s0[grp], d[grp][0], e[0]); e[1] = fmaf(s0[grp], d[grp][1], e[1]);
              e[2] = fmaf(s1[grp], d[grp][2], e[2]); e[3] = fmaf(s1[grp], d[grp][3], e[3]);
            }
            sc[sub][0] = e[0]; sc[sub][1] = e[1]; sc[sub][2] = e[2]; sc[sub][3] = e[3];
          }
        }
        __syncwarp();
      };
      score_stage(QB_PART(0)); score_stage(QB_PART(1));
      if constexpr (ITEMS == 8) { score_stage(QB_PART(2)); score_stage(QB_PART(3)); }
      if (!whole) {
#pragma unroll
        for (int sub = 0; sub < 4; ++sub)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int tk = BITS == 16 ? sub * 16 + h * 8 + g : (sub >> 1) * 32 + 4 * g + 2 * (sub & 1) + h;
            if (!(visible(tok_blk + tk) && ((vm >> (tk >> 4)) & 1u))) sc[sub][2 * h] = sc[sub][2 * h + 1] = -INFINITY;
          }
      }
      // ---------------- the block's softmax ----------------
      int ex[G];                         // exponents of the block's largest |v_scale| of a group
      bool larger = false;
      if constexpr (BITS != 16) {
        if constexpr (G == 2) {
          const uint2 v = *(const uint2*)(sbb + 2 * GE::SB + lane * 8);
          const uint32_t m = __vmaxu2(v.x & 0x7FFF7FFFu, v.y & 0x7FFF7FFFu);
          ex[0] = (int)(__reduce_max_sync(0xffffffffu, m & 0xFFFFu) >> 7);
          ex[G - 1] = (int)(__reduce_max_sync(0xffffffffu, m >> 16) >> 7);
        } else {
          const uint32_t m = *(const uint32_t*)(sbb + 2 * GE::SB + lane * 4) & 0x7FFF7FFFu;
          ex[0] = (int)(__reduce_max_sync(0xffffffffu, max(m >> 16, m & 0xFFFFu)) >> 7);
        }
#pragma unroll
        for (int i = 0; i < G; ++i) {
          ex[i] = ex[i] > 254 ? 254 : ex[i];
          larger |= ex[i] > v_exp(i);
        }
      }
      float mb[2];     // the least reference that this block allows: p = 2^(s - r) <= 1
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float m = fmaxf(sc[0][c], sc[0][2 + c]);
#pragma unroll
        for (int sub = 1; sub < 4; ++sub) m = fmaxf(m, fmaxf(sc[sub][c], sc[sub][2 + c]));
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 4));
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 8));
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 16));
        mb[c] = m * (c ? C1 : C0);
      }
      // a reference that has to move moves 6 further, an exponent 1, so that few blocks have to rescale (from 12 of 21 blocks of a warp to 2)
      if (larger || __any_sync(0xffffffffu, mb[0] > r_run[0] || mb[1] > r_run[1])) {
        const float n0 = mb[0] > r_run[0] ? mb[0] + 6.f : r_run[0], n1 = mb[1] > r_run[1] ? mb[1] + 6.f : r_run[1];
        const float al0 = ex2(r_run[0] - n0), al1 = ex2(r_run[1] - n1);
        float f[G];
        if constexpr (BITS != 16) {
          // A group's unit has to fit the largest p * v_scale.  No probability of this block is above 2^-gap, and those before shrink by
          // 2^-rise for every query, so that large values that no query looks at, or that are forgotten, do not cost the others' bits (up
          // to 100, so that v_scale times the unit is a bf16).  What the references' slack explains does not count, else most blocks
          // would move the unit: 110 us for 104.
          const int q0 = qt * kRows + 2 * t;
          int gap = __reduce_min_sync(0xffffffffu, (int)fminf(fminf(q0 < a.gqa ? n0 - mb[0] : 100.f, q0 + 1 < a.gqa ? n1 - mb[1] : 100.f), 100.f));
          int rise = __reduce_min_sync(0xffffffffu, (int)fminf(fminf(q0 < a.gqa ? n0 - r_run[0] : 100.f, q0 + 1 < a.gqa ? n1 - r_run[1] : 100.f), 100.f));
          gap = gap < 16 ? 0 : gap;
          rise = rise < 16 ? 0 : rise;
#pragma unroll
          for (int grp = 0; grp < G; ++grp) {
            const int was = v_exp(grp), before = max(was - rise, kLowExp), now = ex[grp] - gap > before ? min(ex[grp] - gap + 1, 254) : before;
            f[grp] = pow2i(max(was - now, -126));
            v_unit += (uint32_t)(was - now) << (16 * grp + 7);
          }
        } else f[0] = 1.f;
#pragma unroll
        for (int i = 0; i < GE::NT; ++i) {
          const float g0 = al0 * f[i / (GE::NT / G)], g1 = al1 * f[i / (GE::NT / G)];
          O[i][0] *= g0; O[i][1] *= g1; O[i][2] *= g0; O[i][3] *= g1;
        }
#pragma unroll
        for (int i = 0; i < G; ++i) { ob[i][0] *= al0; ob[i][1] *= al1; }
        l_part[0] *= al0; l_part[1] *= al1;
        r_run[0] = n0; r_run[1] = n1;
      }
#pragma unroll
      for (int sub = 0; sub < 4; ++sub)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float p = ex2(fmaf(sc[sub][i], (i & 1) ? C1 : C0, -r_run[i & 1]));   // (0 where the score is -inf: r is finite)
          l_part[i & 1] += p;
          sc[sub][i] = p;
        }
      // ---------------- values ----------------
      auto value_stage = [&](auto it_c) {
        constexpr int it = decltype(it_c)::value - ITEMS / 2;
        const uint32_t stv = (uint32_t)__cvta_generic_to_shared(acquire(it_c, j));
        uint32_t vs4[4], vb4[4];
        if constexpr (BITS != 16) {
          load4<G>(vs4, sbb + 2 * GE::SB + (it * TOK + 4 * g) * G * 2);
#pragma unroll
          for (int i = 0; i < 4; ++i) vs4[i] = mul_bf16x2(vs4[i], v_unit);
          load4<G>(vb4, sbb + 3 * GE::SB + (it * TOK + 4 * g) * G * 2);
        }
#pragma unroll
        for (int s2 = 0; s2 < TOK / 16; ++s2) {
          const int sub = it * (TOK / 16) + s2;
          if constexpr (BITS == 16) {
            uint32_t hi[2], lo[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const float p0 = sc[sub][2 * h], p1 = sc[sub][2 * h + 1];
              const uint32_t u = pack2(p0, p1);
              hi[h] = transpose8x8(u);
              lo[h] = transpose8x8(pack2(p0 - bf16lo(u), p1 - bf16hi(u)));
            }
            const int rw = s2 * 16 + (lane & 7) + ((lane >> 4) << 3);
#pragma unroll
            for (int n = 0; n < GE::NT; ++n) {
              uint32_t v4[4];
              ldmatrix_b16_x4<true>(v4, stv + rw * GE::ROWB + (((2 * n + ((lane >> 3) & 1)) ^ swz<BITS, CH>(rw)) << 4));
              mma_bf16_16816(O[n], v4, hi[0], hi[1]);
              mma_bf16_16816(O[n], v4, lo[0], lo[1]);
            }
          } else {
            uint32_t pb[G][2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const float p0 = sc[sub][2 * h], p1 = sc[sub][2 * h + 1];
              float vs[G], vb[G];
              vs[0] = bf16lo(vs4[2 * s2 + h]); vb[0] = bf16lo(vb4[2 * s2 + h]);
              if constexpr (G == 2) { vs[G - 1] = bf16hi(vs4[2 * s2 + h]); vb[G - 1] = bf16hi(vb4[2 * s2 + h]); }
#pragma unroll
              for (int grp = 0; grp < G; ++grp) {
                pb[grp][h] = transpose8x8(pack_f16x2(p0 * vs[grp], p1 * vs[grp]));
                ob[grp][0] = fmaf(p0, vb[grp], ob[grp][0]);
                ob[grp][1] = fmaf(p1, vb[grp], ob[grp][1]);
              }
            }
            // matrix row 4u + i of ldmatrix = row {2u, 8 + 2u, 2u + 1, 9 + 2u}[i] of the tile, which is row 16 s2 + that of the stage
            const int mr = lane & 15, half_m = lane >> 4;
            const int tokrow = s2 * 16 + 2 * (mr >> 2) + ((mr >> 1) & 1) + 8 * (mr & 1);
#pragma unroll
            for (int kb = 0; kb < CH; kb += 2) {
              uint32_t r[4];
              ldmatrix_b8_trans_x2(r, stv + tokrow * GE::ROWB + (((kb + half_m) ^ swz<BITS, CH>(tokrow)) << 4));
#pragma unroll
              for (int m = 0; m < 2; ++m) {   // chunk kb + m: byte columns g (row g of the tile) and g + 8
                const uint32_t x = r[2 * m], y = r[2 * m + 1], xh = x >> 8, yh = y >> 8;
                if constexpr (BITS == 4) {
                  const int grp = (kb + m) >> 1, n = 2 * (kb + m);
                  mma_f16_16816(O[n], x & 0x000F000Fu, y & 0x000F000Fu, xh & 0x000F000Fu, yh & 0x000F000Fu, pb[grp][0], pb[grp][1]);
                  mma_f16_16816(O[n + 1], x & 0x00F000F0u, y & 0x00F000F0u, xh & 0x00F000F0u, yh & 0x00F000F0u, pb[grp][0], pb[grp][1]);
                } else {
                  const int grp = (kb + m) >> 2, n = kb + m;
                  mma_f16_16816(O[n], x & 0x00FF00FFu, y & 0x00FF00FFu, xh & 0x00FF00FFu, yh & 0x00FF00FFu, pb[grp][0], pb[grp][1]);
                }
              }
            }
          }
        }
        __syncwarp();
      };
      if constexpr (ITEMS == 8) { value_stage(QB_PART(4)); value_stage(QB_PART(5)); value_stage(QB_PART(6)); value_stage(QB_PART(7)); }
      else { value_stage(QB_PART(2)); value_stage(QB_PART(3)); }
    }
    cp_async_wait<0>();

#undef QB_PART

    // ---- join the warps: sums are partial over the 8 lanes that share a query ----
#pragma unroll
    for (int c = 0; c < 2; ++c) {
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) {
        l_part[c] += __shfl_xor_sync(0xffffffffu, l_part[c], o);
#pragma unroll
        for (int grp = 0; grp < G; ++grp) ob[grp][c] += __shfl_xor_sync(0xffffffffu, ob[grp][c], o);
      }
    }
    float v_back[G];
#pragma unroll
    for (int i = 0; i < G; ++i) v_back[i] = pow2i(v_exp(i) - 141);
    __syncthreads();      // every warp is done with its ring
    float* wm = (float*)smem;                     // [warp][8]
    float* wl = wm + kWarps * kRows;
    float* wo = wl + kWarps * kRows;              // [warp][8][WROW]
    if (g == 0) {
#pragma unroll
      for (int c = 0; c < 2; ++c) { wm[warp * kRows + 2 * t + c] = r_run[c]; wl[warp * kRows + 2 * t + c] = l_part[c]; }
    }
#pragma unroll
    for (int n = 0; n < GE::NT; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int m = g + 8 * (i >> 1), c = i & 1;
        int dim; float v = O[n][i];
        if constexpr (BITS == 4) {      // codes came in as c * 2^-24 (even dims) or 16 c * 2^-24 (odd)
          dim = 32 * (n >> 1) + 2 * m + (n & 1);
          v = fmaf(v * ((n & 1) ? 1048576.f : 16777216.f), v_back[(n >> 2) % G], ob[(n >> 2) % G][c]);
        } else if constexpr (BITS == 8) {
          dim = 16 * n + m;
          v = fmaf(v * 16777216.f, v_back[(n >> 2) % G], ob[(n >> 2) % G][c]);
        } else dim = 16 * n + m;
        wo[(warp * kRows + 2 * t + c) * GE::WROW + dim] = v;
      }
    __syncthreads();
    const int rows = a.gqa - qt * kRows < kRows ? a.gqa - qt * kRows : kRows;
    const bool all = blk0 == 0 && todo == sn.blocks;
    const int slot = 2 * blockIdx.x + (blk0 == 0 ? 1 : 0);
    if (!all && blk0 == 0 && tid == 0) {          // the first of the blocks that share this sequence
      a.joins[blockIdx.x] = make_int4(b, hk * a.gqa + qt * kRows, rows, more);
    }
    for (int i = tid; i < rows * D; i += kWarps * 32) {
      const int h = i / D, e = i - h * D;
      float M = kNegBig;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) M = fmaxf(M, wm[w * kRows + h]);
      float L = 0.f, Ov = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float f = ex2(wm[w * kRows + h] - M);
        L += wl[w * kRows + h] * f;
        Ov += wo[(w * kRows + h) * GE::WROW + e] * f;
      }
      if (all) {
        const float v = Ov * (L > 0.f ? 1.f / L : (L == L ? 0.f : L));
        ((uint16_t*)a.out)[(int64_t)b * a.o_str[0] + (int64_t)(hk * a.gqa + qt * kRows + h) * a.o_str[1] + e] = f32_to_bf16_bits(v);
      } else {
        a.part_o[((int64_t)slot * kRows + h) * D + e] = Ov;
        if (e == 0) { a.part_ml[slot * kRows + h] = make_float2(M, L); }
      }
    }
    __syncthreads();      // the ring may be filled again
  }
}

// ---- the parts of a sequence that several blocks share: out = (sum_r o_r w_r) / (sum_r l_r w_r), w_r = 2^(m_r - max m) ----
// Block c joins the sequence that begins in block c's share and ends behind it: its own part (slot 2c + 1) and those of the next
// blocks (slots 2(c + k)).  A warp takes one query's every parts-th part.
template <int D>
__global__ void __launch_bounds__(kMergeWarps * 32) kv_pages_join_kernel(const __grid_constant__ KvPagesAttnArgs a) {
  __shared__ float red[kMergeWarps][D + 2];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int4 jn = a.joins[blockIdx.x];
  if (jn.x < 0) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, rows = jn.z, n = jn.w + 1;
  const int parts = kMergeWarps / rows, h = warp % rows, part = warp / rows;
  constexpr int V = D / 32;
  auto slot = [&](int k) { return k == 0 ? 2 * (int)blockIdx.x + 1 : 2 * ((int)blockIdx.x + k); };
  float M = kNegBig, L = 0.f, o[V];
#pragma unroll
  for (int i = 0; i < V; ++i) o[i] = 0.f;
  if (part < parts) {
    for (int k0 = part; k0 < n; k0 += parts * 32) {
      const int k = k0 + lane * parts;
      float2 ml = make_float2(kNegBig, 0.f);
      if (k < n) ml = __ldcg(a.part_ml + slot(k) * kRows + h);
      float m = ml.x;
#pragma unroll
      for (int x = 16; x > 0; x >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, x));
      const float Mn = fmaxf(M, m), f = ex2(M - Mn), w = ex2(ml.x - Mn);
      L = L * f + w * ml.y;          // a lane's own parts
#pragma unroll
      for (int i = 0; i < V; ++i) o[i] *= f;
      M = Mn;
      const int cnt = (n - k0 + parts - 1) / parts < 32 ? (n - k0 + parts - 1) / parts : 32;
#pragma unroll 8
      for (int q = 0; q < cnt; ++q) {
        const float wq = __shfl_sync(0xffffffffu, w, q);
        const float* src = a.part_o + ((int64_t)slot(k0 + q * parts) * kRows + h) * D + lane * V;
        if constexpr (V == 4) {
          const float4 x = __ldcg((const float4*)src);
          o[0] = fmaf(wq, x.x, o[0]); o[1] = fmaf(wq, x.y, o[1]); o[2] = fmaf(wq, x.z, o[2]); o[3] = fmaf(wq, x.w, o[3]);
        } else {
          const float2 x = __ldcg((const float2*)src);
          o[0] = fmaf(wq, x.x, o[0]); o[1] = fmaf(wq, x.y, o[1]);
        }
      }
    }
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) L += __shfl_xor_sync(0xffffffffu, L, x);
#pragma unroll
    for (int i = 0; i < V; ++i) red[warp][lane * V + i] = o[i];
    if (lane == 0) { red[warp][D] = M; red[warp][D + 1] = L; }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < rows * D; i += kMergeWarps * 32) {
    const int r = i / D, e = i - r * D;
    float Mx = kNegBig;
    for (int p = 0; p < parts; ++p) Mx = fmaxf(Mx, red[p * rows + r][D]);
    float Ls = 0.f, Os = 0.f;
    for (int p = 0; p < parts; ++p) {
      const float f = ex2(red[p * rows + r][D] - Mx);
      Ls += red[p * rows + r][D + 1] * f;
      Os += red[p * rows + r][e] * f;
    }
    const float v = Os * (Ls > 0.f ? 1.f / Ls : (Ls == Ls ? 0.f : Ls));
    ((uint16_t*)a.out)[(int64_t)jn.x * a.o_str[0] + (int64_t)(jn.y + r) * a.o_str[1] + e] = f32_to_bf16_bits(v);
  }
}

// CTAs of an instance that the device holds at once, with the lengths of up to 32, 512 or more sequences in shared memory.
constexpr int kSeqSteps[3] = {32, 512, kMaxPageSeqs};
template <int BITS, int D> constexpr int smem_of(int step) { return Geo<BITS, D>::SMEM + (step == 0 ? 0 : (kSeqSteps[step] + 1) * 4); }
template <int BITS, int D> cudaError_t resident(int step, int* n) {
  auto kern = kv_pages_kernel<BITS, D>;
  static int cached[64][3] = {};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  std::lock_guard<std::mutex> setup_lk(setup_mutex());   // first use on a device, from any thread
  if (dev >= 0 && dev < 64 && cached[dev][step] != 0) { *n = cached[dev][step]; return cudaSuccess; }
  e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem_of<BITS, D>(2));
  if (e != cudaSuccess) return e;
  int per = 0;
  e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per, kern, kWarps * 32, smem_of<BITS, D>(step));
  if (e != cudaSuccess) return e;
  *n = (per < 1 ? 1 : (per > kPagesCtas ? kPagesCtas : per)) * sm_count();
  if (dev >= 0 && dev < 64) cached[dev][step] = *n;
  return cudaSuccess;
}

template <int BITS, int D> cudaError_t launch_inst(KvPagesAttnArgs a, int64_t most_units, cudaStream_t st) {
  int n = 0;
  const int step = a.B <= kSeqSteps[0] ? 0 : (a.B <= kSeqSteps[1] ? 1 : 2);
  cudaError_t e = resident<BITS, D>(step, &n);
  if (e != cudaSuccess) return e;
  const unsigned grid = (unsigned)(most_units < n ? (most_units < 1 ? 1 : most_units) : n);
  e = launch_behind(kv_pages_kernel<BITS, D>, dim3(grid), dim3(kWarps * 32), smem_of<BITS, D>(step), st, a);
  if (e != cudaSuccess) return e;
  return launch_behind(kv_pages_join_kernel<D>, dim3(grid), dim3(kMergeWarps * 32), 0, st, a);
}
}  // namespace

// [joins: int4 per CTA][m, l: float2 per slot and row][o: D floats per slot and row], two slots a CTA
size_t kv_pages_workspace_bytes(int64_t D) {
  const size_t ctas = (size_t)kPagesCtas * sm_count();
  return ctas * 16 + ctas * 2 * kRows * 8 + ctas * 2 * kRows * (size_t)D * 4;
}

cudaError_t launch_kv_pages_attn(KvPagesAttnArgs a, int D, void* workspace, cudaStream_t st) {
  const size_t ctas = (size_t)kPagesCtas * sm_count();
  a.joins = (int4*)workspace;
  a.part_ml = (float2*)((char*)workspace + ctas * 16);
  a.part_o = (float*)((char*)workspace + ctas * 16 + ctas * 2 * kRows * 8);
  a.qtiles = (a.gqa + kRows - 1) / kRows;
  a.tiles = a.Hkv * a.qtiles;
  a.min_units = kWarps;
  // the most blocks that a sequence can see
  int64_t most = (((int64_t)a.M << a.page_shift) + kBlk - 1) / kBlk;
  if (a.window > 0) {
    const int64_t w = ((int64_t)a.window + kBlk - 1) / kBlk + 1 + ((int64_t)a.sinks + kBlk - 1) / kBlk;
    most = most < w ? most : w;
  }
  const int64_t units = most * a.tiles * a.B;
  switch (a.bits * 1000 + D) {
    case 4064: return launch_inst<4, 64>(a, units, st);
    case 4128: return launch_inst<4, 128>(a, units, st);
    case 8064: return launch_inst<8, 64>(a, units, st);
    case 8128: return launch_inst<8, 128>(a, units, st);
    case 16064: return launch_inst<16, 64>(a, units, st);
    case 16128: return launch_inst<16, 128>(a, units, st);
    default: return cudaErrorInvalidValue;
  }
}

}  // namespace qb
