// Attention of a tree of drafted tokens over a paged key-value cache, 4- or 8-bit codes or bf16 rows, head dim 64 or 128, with an
// optional window and a few first tokens that stay visible, on the tensor cores (tcgen05) with keys, scores and results in tensor memory.
//
// Node t of a sequence stands at position p(t) = base + depth(t) behind `base` cached tokens; it sees the cached tokens, itself and the
// nodes before it on its line (with a window those at positions > p(t) - window or < sinks).
//   o = sum_j p_j v_j / sum_j p_j,  p_j = 2^(c s_j - r),  s = q . k, c = scale * log2(e), r a running reference of the row.
//
// A tile is N (16, 32, 64 or 128) query rows of one cache head: nodes times the heads of its group, node after node, so that a tree with few nodes
// fills few tiles.  The products are transposed, S^T = K Q^T and O^T = V^T P^T: the 128 tokens of a block are the rows (lanes), the queries the
// columns, so that a product takes time in proportion to N, a thread of the softmax has one token, and what belongs to a token is a
// register of its thread:
//  * Codes are dequantised to fp16, rounded once, in a unit of the token's own (a power of two, its largest |q s + b| in [2^14, 2^15)), so that the
//    range of fp16 holds for each token by itself; a key's unit is a factor of its thread's scores, a value's goes to its probabilities: P' = p * unit, and the
//    row's sum takes P' / unit.  Tokens and groups 2^28 apart in size keep fp16's 11 bits.  At 16 bits the operands are the cache's bf16 and
//    P is a sum of two bf16 (16 bits, as where one token is decoded), each multiplied with the values: rounded to one its errors were as large as
//    the result's own rounding.
//  * r moves only where some P' would pass 2^15: then it is placed 2^8 below the block's maximum, and O is rescaled.
//  * Roles of a CTA's warps: four a 32 columns of the softmax; four read keys and dequantise them into tensor memory (the A operand of S^T); four
//    read values and dequantise them into shared memory; one issues the products, S^T two blocks ahead of O^T; two issue the copies: codes by
//    TMA in boxes of up to a page, scales and biases as bulk copies where a page's are one run, into rings of whole blocks.  At 16 bits the
//    rings' places are the operands themselves.
//  * The grid is one CTA an SM; every CTA works out all sequences' blocks from `lens` and takes an even share of them, or every tile is cut in the
//    same number of parts.  Parts of a tile go to the workspace and are joined by a second kernel.
//
// Measured: 16 sequences of 32k tokens, 4 bits, 32 query heads over 8, 518 us with 32 nodes (128 rows of a cache head; the products alone take 102 us at
// the rate of a library's, the codes 72 at that of a copy), 371 with 16, 324 with 8, 277 with 4; 4 sequences of 8k, 8 bits, 64 nodes 128 to 133 us; 32
// sequences of a window of 1024 over bf16 99 us; one of 700 tokens 22.  What bounds a long one is neither the bytes nor the products but the work a block of 128
// tokens takes, handed from warp to warp: 3.0 us a block with 128 rows, 1.5 of them copies, products and barriers alone (260 of 515 us; 177 of 277 with 16
// rows; without the readers' arithmetic 407 and 189, without the softmax's 347 and 231).  A short one is bound by what a call and a piece take beside their
// blocks: 2, 8, 32 and 128 blocks a CTA of 128 rows take 61, 78, 149 and 399 us behind a write of 256 MB, 16 rows 31, 39, 80 and 213, that is about 56 and 28 us
// and 2.7 and 1.4 for a block.  Rings by cp.async in every reader took 695 instead of 527 us; two groups of readers that
// take turns, a sleeping instead of a polling issuer, and operands made uniform for it changed nothing.
// With 128 columns the softmax's 88 registers (the readers' 56) do not hold everything: -Xptxas -v reports 272 to 324 bytes of spill stores and 392 to 456 of
// loads a thread for codes, 88 and 216 of stores for bf16 rows; narrower tiles have 64 and 132 at most.  What fewer registers' worth would give is not measured.
#include <mutex>
#include <type_traits>

#include "stream_ptx.cuh"
#include "tc_ptx.cuh"

namespace qb {
namespace {

__device__ int g_tree_error = 0;     // 0 = ok; otherwise the code of the wait that expired

constexpr int kBlk = 128;            // tokens of a block
constexpr uint32_t kPolls = 1u << 18, kSpins = 1u << 23;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kNegBig = -1e30f;
constexpr float kTop = 15.f, kAim = 8.f;   // exponents of P': the reference moves above the first, and then aims at the second
constexpr int kLowExp = -80, kHighExp = 113;   // of a token's largest value, beyond which its unit does not follow
constexpr int kNotes = 2 * kMaxNodes;       // the drafted tokens, and where a window begins the tokens that its deepest node sees no more
constexpr int kPiece = 5;            // what a piece of a tile takes beside its blocks, in blocks
constexpr int kJoinRows = 8, kJoinWarps = 16;

template <int BITS, int D, int N> struct Shape {
  static constexpr bool QUANT = BITS != 16;
  static constexpr int G = BITS == 16 ? 1 : D / 64;          // scale groups of a token
  static constexpr int HALVES = D / 64;                      // blocks of 64 columns (128 bytes) side by side
  static constexpr int ROWB = D * BITS / 8, CH = ROWB / 16;  // bytes of a token, 16-byte chunks of it
  static constexpr int NC = N < 32 ? N : 32;                 // columns of a softmax warp
  static constexpr int WGS = N / NC, SW = 4 * WGS;           // groups of four softmax warps
  static constexpr int KW = QUANT ? 4 : 0;                   // warps that read keys
  static constexpr int V_AT = SW + KW, MMA_AT = V_AT + 4, COPY_AT = MMA_AT + 1;   // first warp of the values, of the products, of the copies (keys, values)
  // registers dealt out by role, where the warps' even share is too little for the softmax; the warps fill up groups of four then
  static constexpr bool SPLIT = WGS == 4 || (QUANT && WGS == 2);
  static constexpr int THREADS = (SPLIT ? (COPY_AT + 5) / 4 * 4 : COPY_AT + 2) * 32;
  static constexpr int R_SOFT = WGS == 4 ? (QUANT ? 88 : 96) : 128, R_READ = WGS == 4 ? 56 : 80, R_MISC = WGS == 4 ? 40 : 64;
  static constexpr int TILE = kBlk * 128 * HALVES;           // a block's keys or values as an operand
  static constexpr int SB = kBlk * G * 2;                    // bytes of a block's scales (or biases)
  static constexpr int VT = 2;                               // places for values as operands
  static constexpr int PS = N == 128 || (D == 128 && (BITS == 8 || (BITS == 16 && N == 64))) ? 1 : 2;   // places for P
  // P of a block, 128 bytes of columns a token; at 16 bits what bf16 leaves of it stands behind it: in the other half of the 128 bytes, or in a tile of its own
  static constexpr int PP = QUANT ? 1 : 2, PCOLS = kBlk * 128 * (N > 64 ? 2 : 1), LOW = N <= 32 ? 64 : PCOLS, PTILE = PP == 2 && N > 32 ? 2 * PCOLS : PCOLS;
  // the rings: codes with scales and biases (the keys' with the values' too, for their units), or at 16 bits the operands themselves
  static constexpr int KS = BITS == 4 ? 4 : (BITS == 8 ? (N == 128 && D == 128 ? 2 : 3) : (D == 64 ? (N >= 64 ? 3 : 4) : (N == 128 ? 1 : 2))), VS = BITS == 4 ? 4 : (BITS == 8 ? (N == 128 && D == 128 ? 2 : 3) : (D == 64 ? (N >= 64 ? 3 : 4) : (N >= 64 ? 2 : 3)));
  static constexpr int K_STAGE = QUANT ? kBlk * ROWB + 4 * SB : TILE, V_STAGE = QUANT ? kBlk * ROWB + 2 * SB : TILE;
  static constexpr int V0 = 0, Q0 = QUANT ? VT * TILE : 0, P0 = Q0 + N * 128 * HALVES, KR = P0 + PS * PTILE, VR = KR + KS * K_STAGE;
  static constexpr int SMEM = VR + VS * V_STAGE + (QUANT || D == 128 ? 0 : TILE) + 1024;   // (a product of 128 rows reads a tile past the last one of 64)
  static constexpr int ATOM = QUANT && ROWB < 128 ? 512 : 1024;
  static_assert(KR % 1024 == 0 && K_STAGE % ATOM == 0 && V_STAGE % ATOM == 0, "places of boxes");
  static_assert(SMEM + 2 * (kMaxPageSeqs + 1) * 4 + 13 * 1024 <= 227 * 1024, "shared memory");
  static constexpr uint32_t SW_AT = N > 64 ? 128 : 64, S_AT = 0, O_AT = 2 * SW_AT, K_AT = 3 * SW_AT;   // columns of tensor memory: two of S, O, two of K
  static_assert(K_AT + (QUANT ? 128 : 0) <= 512, "tensor memory");
};

// A pool's codes (or rows) as boxes of up to 128 tokens of one head in one page, and what a box takes along head and page (0: broadcast).
struct TreeMaps {
  int mul[2][2];
  int piece;                 // tokens of a box
};

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
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
                 "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
               : "r"(taddr));
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};"
               ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]),
                 "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(taddr)
               : "memory");
}
template <int NC> __device__ __forceinline__ void tmem_get(uint32_t taddr, uint32_t (&r)[NC]) {
  if constexpr (NC == 32) tmem_ld32(taddr, r); else tmem_ld16(taddr, r);
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}
template <int NC> __device__ __forceinline__ void tmem_put(uint32_t taddr, const uint32_t (&r)[NC]) {
  if constexpr (NC == 32) tmem_st32(taddr, r); else tmem_st16(taddr, r);
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void bar_sync(int id, int n) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(n) : "memory"); }
__device__ __forceinline__ bool bar_any(int id, int n, bool v) {
  uint32_t r;
  asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %3, 0;\n\tbar.red.or.pred q, %1, %2, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
               : "=r"(r) : "r"(id), "r"(n), "r"((uint32_t)v) : "memory");
  return r != 0;
}
__device__ __forceinline__ float max3(float a, float b, float c) {   // (a NaN does not count)
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, uint64_t* bar, int x, int y, int z, int w) {
  asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];"
               ::"r"(dst), "l"(map), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
               ::"r"(dst), "l"(src), "r"(bytes), "r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ bool arrived(uint32_t bar, uint32_t parity) {
  uint32_t done;
  asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\tselp.u32 %0, 1, 0, p;\n\t}"
               : "=r"(done) : "r"(bar), "r"(parity), "r"(kNap) : "memory");
  return done != 0;
}
// The rest of a wait, for a warp whose barrier had not arrived at the first look: `most` looks, each held by the hardware for kNap ns at most.  A wait
// that runs out is noted once.  From then on nothing is copied any more and the issuer does not wait for what has not come; the readers and the softmax go
// on without waiting, on data that is not there and within their bounds, so that all warps meet at every barrier and the CTA ends; and its results are NaN.
__device__ __forceinline__ void wait_on(uint32_t bar, uint32_t parity, int code, int* fail, uint32_t most) {
  if (*(volatile int*)fail == 0) {
    for (uint32_t it = 0; it < most; ++it)
      if (arrived(bar, parity)) return;
    *(volatile int*)fail = code;
    atomicCAS(&g_tree_error, 0, code);
  }
}
// A bounded wait that polls without sleeping, and ends too where another has run out.
__device__ __forceinline__ bool spin_cta(uint64_t* bar, uint32_t parity, uint32_t most, const int* fail) {
  const uint32_t addr = smem_u32(bar);
  for (uint32_t it = 0; it < most && ((it & 15) != 8 || *(volatile const int*)fail == 0); ++it) {
    uint32_t done;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(done) : "r"(addr), "r"(parity) : "memory");
    if (done) return true;
  }
  return false;
}
// Rows of 128 bytes with their 64 columns contiguous, swizzled, as an operand whose columns are its M or N: 8 rows 1024 bytes apart, the next
// 64 columns a block of 128 rows further.
__device__ __forceinline__ uint64_t make_desc_mn(uint32_t saddr) {
  uint64_t d = 0;
  d |= (uint64_t)((saddr & 0x3FFFF) >> 4);
  d |= (uint64_t)((kBlk * 128) >> 4) << 16;
  d |= (uint64_t)(1024 >> 4) << 32;
  d |= (uint64_t)1 << 46;
  d |= (uint64_t)2 << 61;
  return d;
}

// The largest |code * s + b| of a group, and its unit: values times 2^(14 - e) lie below 2^15.  What is not finite does not count.
template <int BITS> __device__ __forceinline__ float group_top(float s, float b) { return fmaxf(fabsf(b), fabsf(fmaf(s, (float)((1 << (BITS & 15)) - 1), b))); }
__device__ __forceinline__ int unit_exp(float top) {
  const int e = (int)(__float_as_uint(top) >> 23) - 127;
  return e < kLowExp ? kLowExp : (e > kHighExp ? kHighExp : e);
}
// Codes of a packed word as fp16 values c * s + b, rounded once: a code in the low bits of 1024, or at 4 bits a nibble further up of 64, is exact,
// and so is taking that away.  Pairs come out of a word in the order its bits allow: dims 0 4, 1 5, 2 6, 3 7 at 4 bits, 0 2, 1 3 at 8.
template <int BITS> __device__ __forceinline__ void dequant_word(uint32_t w, __half2 s, __half2 b, uint32_t* o) {
  const __half2 c1024 = __float2half2_rn(1024.f), c64 = __float2half2_rn(64.f);
  auto out = [&](uint32_t bits, __half2 off) {
    const __half2 v = __hfma2(__hsub2(*(const __half2*)&bits, off), s, b);
    return *(const uint32_t*)&v;
  };
  if constexpr (BITS == 4) {
    const uint32_t w8 = w >> 8;
    o[0] = out(lop3_and_or(w, 0x000F000Fu, 0x64006400u), c1024);
    o[1] = out(lop3_and_or(w, 0x00F000F0u, 0x54005400u), c64);
    o[2] = out(lop3_and_or(w8, 0x000F000Fu, 0x64006400u), c1024);
    o[3] = out(lop3_and_or(w8, 0x00F000F0u, 0x54005400u), c64);
  } else {
    o[0] = out(lop3_and_or(w, 0x00FF00FFu, 0x64006400u), c1024);
    o[1] = out(lop3_and_or(w >> 8, 0x00FF00FFu, 0x64006400u), c1024);
  }
}
// the dim that stands at a place of the operands
template <int BITS> __device__ __forceinline__ int dim_at(int place) {
  if constexpr (BITS == 4) return (place & ~7) | ((place & 1) << 2) | ((place >> 1) & 3);
  else if constexpr (BITS == 8) return (place & ~3) | ((place & 1) << 1) | ((place >> 1) & 1);
  else return place;
}

// A sequence's tree, and the blocks that its nodes see: [0, front) and, from there on, block i + skip.
struct Seq {
  int row, base, n, len, w0, sinks, front, skip, blocks, tiles;
};
__device__ __forceinline__ Seq seq_of(const KvPagesTreeArgs& t, int b, int N) {
  const KvPagesAttnArgs& a = t.a;
  Seq s;
  const int64_t row = a.rows ? a.rows[b] : b;
  const bool known = row >= 0 && row < a.seqs;
  int64_t len = known ? a.lens[row] : 0, n = t.counts ? t.counts[b] : t.T;
  const int64_t cap = (int64_t)a.M << a.page_shift;
  len = len < 0 ? 0 : (len > cap ? cap : len);
  n = n < 0 ? 0 : (n > t.T ? t.T : n);
  n = n > len ? len : n;
  s.row = known ? (int)row : 0; s.len = (int)len; s.n = (int)n; s.base = (int)(len - n);
  s.w0 = a.window > 0 && s.base - a.window + 1 > 0 ? s.base - a.window + 1 : 0;
  s.sinks = a.sinks < s.len ? a.sinks : s.len;
  s.front = (int)(((int64_t)s.sinks + kBlk - 1) / kBlk);
  s.skip = s.w0 / kBlk - s.front;
  if (s.skip < 0) s.skip = 0;
  s.blocks = n > 0 ? (int)((len + kBlk - 1) / kBlk) - s.skip : 0;
  s.tiles = n > 0 ? a.Hkv * (int)(((int64_t)n * a.gqa + N - 1) / N) : 0;
  return s;
}

// What a CTA works on: blocks [blk0, blk0 + todo) of a tile, and how many CTAs behind this one share it.
struct Piece {
  Seq s;
  int b, hk, rt, blk0, todo, more;
  __device__ __forceinline__ int first_token(int j) const { const int i = blk0 + j; return (i < s.front ? i : i + s.skip) * kBlk; }
  __device__ __forceinline__ bool some_see(int tok) const { return tok < s.len && (tok >= s.w0 || tok < s.sinks); }
  __device__ __forceinline__ bool all_see(const KvPagesTreeArgs& t, int tok) const {    // (no node is deeper than n - 1)
    return tok < s.base && (t.a.window == 0 || tok < s.sinks || tok > s.base + s.n - 1 - t.a.window);
  }
  __device__ __forceinline__ bool whole(const KvPagesTreeArgs& t, int k0) const {
    return k0 + kBlk <= s.base && (t.a.window == 0 || k0 + kBlk <= s.sinks || k0 > s.base + s.n - 1 - t.a.window);
  }
};
// The pieces of a CTA, one after the other; every role goes through them by itself.
struct Pieces {
  const KvPagesTreeArgs& t;
  const int *units, *tiles;      // [B + 1]: blocks, tiles before each sequence
  int N, per, parts, u, u_to;
  bool more;
  __device__ __forceinline__ Pieces(const KvPagesTreeArgs& t_, const int* units_, const int* tiles_, int longest, int N_) : t(t_), units(units_), tiles(tiles_), N(N_) {
    const int U = units[t.a.B], all = tiles[t.a.B], ctas = (int)gridDim.x;
    per = (U + ctas - 1) / ctas;
    if (per < 1) per = 1;
    parts = all > 0 ? ctas / all : 0;
    if (parts > 0) {
      parts = parts > longest ? (longest < 1 ? 1 : longest) : parts;
      const int pieces = 1 + (int)ceilf(__fdividef((float)per * (float)all, (float)(U > 0 ? U : 1)));   // that an even share touches
      if ((longest + parts - 1) / parts + kPiece > per + pieces * kPiece) parts = 0;
    }
    const int64_t from = (int64_t)blockIdx.x * per;
    u = from < U ? (int)from : U;
    u_to = u + per < U ? u + per : U;
    more = parts > 0 ? (int)blockIdx.x < all * parts : u < U;
  }
  __device__ __forceinline__ int find(const int* before, int x) const {       // the last sequence that begins at x or before
    int lo = 0, hi = t.a.B - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (before[mid] <= x) lo = mid; else hi = mid - 1;
    }
    return lo;
  }
  __device__ __forceinline__ bool next(Piece& p) {
    if (!more) return false;
    int tile;
    if (parts > 0) {
      more = false;
      const int at = (int)blockIdx.x / parts, part = (int)blockIdx.x - at * parts;
      p.b = find(tiles, at);
      p.s = seq_of(t, p.b, N);
      tile = at - tiles[p.b];
      const int mine = parts < p.s.blocks ? parts : p.s.blocks;
      if (part >= mine) return false;
      const int each = p.s.blocks / mine, rest = p.s.blocks - each * mine;
      p.blk0 = each * part + (part < rest ? part : rest);
      p.todo = each + (part < rest ? 1 : 0);
      p.more = mine - 1;
    } else {
      p.b = find(units, u);
      p.s = seq_of(t, p.b, N);
      const int before = units[p.b];
      tile = (u - before) / p.s.blocks;
      p.blk0 = u - before - tile * p.s.blocks;
      const int left = p.s.blocks - p.blk0;
      p.todo = left < u_to - u ? left : u_to - u;
      p.more = (before + (tile + 1) * p.s.blocks - 1) / per - (int)blockIdx.x;
      u += p.todo;
      more = u < u_to;
    }
    const int rts = p.s.tiles / t.a.Hkv;
    p.hk = tile / rts;
    p.rt = tile - p.hk * rts;
    return true;
  }
};

template <int BITS, int D, int N>
__global__ void __launch_bounds__(Shape<BITS, D, N>::THREADS, 1) tree_kernel(const __grid_constant__ CUtensorMap mk, const __grid_constant__ CUtensorMap mv,
                                                                             const __grid_constant__ KvPagesTreeArgs t, const __grid_constant__ TreeMaps maps) {
  using SH = Shape<BITS, D, N>;
  constexpr int G = SH::G, CH = SH::CH, NC = SH::NC, SW = SH::SW, KS = SH::KS, VS = SH::VS, THREADS = SH::THREADS;
  constexpr bool QUANT = SH::QUANT;
  const KvPagesAttnArgs& a = t.a;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* const smem = (unsigned char*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  int* const units = (int*)(smem + SH::SMEM - 1024);          // [B + 1], [B + 1]
  int* const tiles = units + a.B + 1;
  __shared__ uint64_t q_ready, k_ready[2], v_ready[2], s_ready[2], p_ready[2], o_done[2], k_full[KS], k_empty[KS], v_full[VS], v_empty[VS];
  __shared__ uint32_t tmem_slot;
  __shared__ int s_fail, s_longest[32], warp_sums[2][32];
  __shared__ __align__(16) float s_nr[N], s_kunit[4][kBlk];     // -r of the columns; of a block's tokens
  __shared__ int s_vexp[4][kBlk];
  __shared__ uint32_t s_pages[2][16];    // of a block, from the keys' and from the values' copies: which of its 16 tokens have a page
  __shared__ float s_wmax[SH::WGS][4][NC];
  __shared__ int s_par[kMaxNodes], s_depth[kMaxNodes], s_clo[N], s_qe[N];
  __shared__ uint64_t s_line[kMaxNodes], s_cline[N];
  __shared__ int note_count[4], note_key[4][kNotes];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  asm volatile("griddepcontrol.wait;" ::: "memory");         // (before tensor memory is taken, too: the kernel before may hold it)
  asm volatile("griddepcontrol.launch_dependents;");

  // ---- all sequences' blocks and tiles ----
  {
    const int each = (a.B + THREADS - 1) / THREADS, b0 = tid * each;
    int mine = 0, mine_t = 0, longest = 0;
    for (int i = 0; i < each && b0 + i < a.B; ++i) {
      const Seq s = seq_of(t, b0 + i, N);
      units[b0 + i] = mine; tiles[b0 + i] = mine_t;
      mine += s.blocks * s.tiles;
      mine_t += s.tiles;
      longest = s.blocks > longest ? s.blocks : longest;
    }
    int upto = mine, upto_t = mine_t;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, upto, o), y = __shfl_up_sync(0xffffffffu, upto_t, o);
      if (lane >= o) { upto += x; upto_t += y; }
    }
    longest = __reduce_max_sync(0xffffffffu, longest);
    if (lane == 31) { warp_sums[0][warp] = upto; warp_sums[1][warp] = upto_t; s_longest[warp] = longest; }
    if (tid == 0) {
      s_fail = t.polls < 0 ? 600 : 0;
      if (t.polls < 0) atomicCAS(&g_tree_error, 0, 600);
      mbar_init(&q_ready, SW);
      for (int i = 0; i < 2; ++i) { mbar_init(&k_ready[i], 4); mbar_init(&v_ready[i], 4); mbar_init(&s_ready[i], 1); mbar_init(&p_ready[i], SW); mbar_init(&o_done[i], 1); }
      for (int i = 0; i < KS; ++i) { mbar_init(&k_full[i], 1); mbar_init(&k_empty[i], QUANT ? 4 : 1); }
      for (int i = 0; i < VS; ++i) { mbar_init(&v_full[i], 1); mbar_init(&v_empty[i], QUANT ? 4 : 1); }
      for (int i = 0; i < 4; ++i) note_count[i] = 0;
      a.joins[blockIdx.x] = make_int4(-1, 0, 0, 0);
      asm volatile("fence.mbarrier_init.release.cluster;\n\tfence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == SH::MMA_AT) {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"(512u));
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::);
    }
    __syncthreads();
    int before = upto - mine, before_t = upto_t - mine_t;
    for (int w = 0; w < warp; ++w) { before += warp_sums[0][w]; before_t += warp_sums[1][w]; }
    for (int i = 0; i < each && b0 + i < a.B; ++i) { units[b0 + i] += before; tiles[b0 + i] += before_t; }
    if (tid == THREADS - 1) { units[a.B] = before + mine; tiles[a.B] = before_t + mine_t; }
  }
  fence_before();
  __syncthreads();
  fence_after();
  int longest = 0;
#pragma unroll
  for (int w = 0; w < THREADS / 32; ++w) longest = s_longest[w] > longest ? s_longest[w] : longest;
  const uint32_t tmem = tmem_slot;
  Pieces pieces(t, units, tiles, longest, N);
  Piece pc;
  auto wait = [&](uint64_t* bar, uint32_t phase, int code) {
    if (__builtin_expect(!arrived(smem_u32(bar), phase & 1), 0)) wait_on(smem_u32(bar), phase & 1, code, &s_fail, t.polls > 0 ? (uint32_t)t.polls : kPolls);
    __syncwarp();
  };
  auto failed = [&]() { return __any_sync(0xffffffffu, *(volatile int*)&s_fail != 0); };   // (the same for the warp, whoever notes it when)
  const int pmask = (1 << a.page_shift) - 1;
  int J0 = 0;                        // blocks before this piece

  if (warp >= SW && warp < SH::MMA_AT) {
    // ---------------- keys, values ----------------
    if constexpr (SH::SPLIT) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(SH::R_READ));
    const bool V = warp >= SH::V_AT;
    const int wq = warp & 3, key = 32 * wq + lane;             // quarter of the block: 32 tokens, one a lane
    uint64_t* const full = V ? v_full : k_full;
    uint64_t* const empty = V ? v_empty : k_empty;
    const int stages = V ? VS : KS, stage_b = V ? SH::V_STAGE : SH::K_STAGE;
    unsigned char* const ring = smem + (V ? SH::VR : SH::KR);
    const int swz = CH >= 8 ? lane & 7 & (CH - 1) : (lane / (8 / CH)) % CH;       // (16-byte chunks of a row, as the copies place them)
    int piece_no = 0, st = 0;
    uint32_t round = 0;
    while (pieces.next(pc)) {
#pragma unroll 1
      for (int j = 0; j < pc.todo; ++j) {
        const int J = J0 + j, k0 = pc.first_token(j), tok = k0 + key;
        wait(&full[st], round, 605);
        // a value that some nodes see and others do not must not meet their 0 if it is not finite: it is zeroed and noted
        bool mine = true, partly = false, bad = false;
        const uint32_t have = s_pages[V][J & 15];              // (their own copies' word: the other's may be ahead or behind)
        if (!pc.whole(t, k0) || have != 0xffu) {
          mine = pc.some_see(tok) && ((have >> (key >> 4)) & 1u);
          partly = V && mine && !pc.all_see(t, tok);
        }
        if constexpr (QUANT) {
          const unsigned char* const codes = ring + st * stage_b;
          const unsigned char* const sb = codes + kBlk * SH::ROWB;
          float s[G], b[G];
          auto params = [&](int arr, float (&x)[G]) {
            uint32_t v = 0u;
            if (a.sb_vec) {
              if constexpr (G == 2) v = *(const uint32_t*)(sb + arr * SH::SB + key * 4);
              else v = *(const uint16_t*)(sb + arr * SH::SB + key * 2);
            } else if (mine) {
              const KvPoolView& pl = a.pool[V || arr >= 2];
              const int pid = a.table[(int64_t)pc.s.row * a.table_str + (tok >> a.page_shift)];
              const uint16_t* const src = (const uint16_t*)((arr & 1) ? pl.b : pl.s) + (int64_t)pid * pl.sb_str[0] + (int64_t)pc.hk * pl.sb_str[1] + (int64_t)(tok & pmask) * pl.sb_str[2];
              if (pid >= 0 && pid < a.P) {                     // (behind a wait that ran out `mine` may not be true)
                v = src[0];
                if constexpr (G == 2) v |= (uint32_t)src[1] << 16;
              }
            }
            v = mine ? v : 0u;
            x[0] = bf16lo(v);
            if constexpr (G == 2) x[G - 1] = bf16hi(v);
          };
          auto largest = [&]() {
            float m = 0.f;                                     // (what is not finite does not count)
#pragma unroll
            for (int g = 0; g < G; ++g) {
              const float x = group_top<BITS>(s[g], b[g]);
              m = x < INFINITY ? fmaxf(m, x) : m;
            }
            return m;
          };
          int ev = 0;
          if (!V) {
            params(2, s); params(3, b);
            ev = unit_exp(largest()) - 14;
          }
          params(0, s); params(1, b);
          const int e = unit_exp(largest());
          const float up = pow2i(14 - e);
          if (partly)
#pragma unroll
            for (int g = 0; g < G; ++g) bad |= !(fabsf(s[g]) < INFINITY) || !(group_top<BITS>(s[g], b[g]) < INFINITY);
          const bool drop = partly && bad;
          __half2 s2[G], b2[G];
#pragma unroll
          for (int g = 0; g < G; ++g) { s2[g] = __float2half2_rn(drop ? 0.f : s[g] * up); b2[g] = __float2half2_rn(drop ? 0.f : b[g] * up); }
          if (J >= 2) wait((V ? o_done : s_ready) + (J & 1), (uint32_t)((J >> 1) - 1), V ? 602 : 601);
          if (!V) {                                            // (S two blocks back is complete, so the softmax has left the block four back: its place is free)
            s_kunit[J & 3][key] = pow2i(e - 14);
            s_vexp[J & 3][key] = ev;
          }
          unsigned char* const vrow = smem + SH::V0 + (J & 1) * SH::TILE + key * 128;
          constexpr int CG = CH / G;                           // chunks of a group
          // (Rolled, the code is shorter: 16 sequences of 32k tokens, 64 rows 424 -> 382 us, 16 rows 302 -> 274.  With 128 rows the readers' registers
          // are fewer and it takes longer, 515 -> 549.)
#pragma unroll (N < 128 ? 1 : G)
          for (int g = 0; g < G; ++g) {
            const __half2 sg = g ? s2[G - 1] : s2[0], bg = g ? b2[G - 1] : b2[0];
            uint32_t o[32];
#pragma unroll
            for (int c = 0; c < CG; ++c) {
              // (a token that is not seen: 0 * 0 + 0 whatever the codes are)
              const uint4 x = *(const uint4*)(codes + key * SH::ROWB + (((g * CG + c) ^ swz) << 4));
              constexpr int W = 32 / BITS / 2;                 // registers of a word
              dequant_word<BITS>(x.x, sg, bg, &o[(4 * c + 0) * W]); dequant_word<BITS>(x.y, sg, bg, &o[(4 * c + 1) * W]);
              dequant_word<BITS>(x.z, sg, bg, &o[(4 * c + 2) * W]); dequant_word<BITS>(x.w, sg, bg, &o[(4 * c + 3) * W]);
            }
            if (!V) tmem_st32(tmem + SH::K_AT + (J & 1) * 64 + g * 32 + ((uint32_t)wq << 21), o);
            else {
#pragma unroll
              for (int c = 0; c < 8; ++c)
                *(uint4*)(vrow + g * (kBlk * 128) + ((c ^ (key & 7)) << 4)) = make_uint4(o[4 * c], o[4 * c + 1], o[4 * c + 2], o[4 * c + 3]);
            }
          }
          if (!V) {
            asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
            fence_before();
          } else fence_async();
        } else {
          // (the products two blocks back are done, so that this arrival is not taken for one of theirs)
          if (J >= 2) wait(&o_done[J & 1], (uint32_t)((J >> 1) - 1), 602);
          if (__any_sync(0xffffffffu, partly || !mine)) {
            unsigned char* const vrow = ring + st * stage_b + key * 128;
            if (partly) {
              uint32_t acc = 0;
#pragma unroll
              for (int c = 0; c < D / 8; ++c) {
                const uint4 x = *(const uint4*)(vrow + (c >> 3) * (kBlk * 128) + (((c & 7) ^ (key & 7)) << 4));
                acc |= ((x.x & 0x7F807F80u) + 0x00800080u) | ((x.y & 0x7F807F80u) + 0x00800080u) | ((x.z & 0x7F807F80u) + 0x00800080u) | ((x.w & 0x7F807F80u) + 0x00800080u);
              }
              bad = (acc & 0x80008000u) != 0;                  // an exponent of all ones
            }
            if (bad || !mine)
#pragma unroll
              for (int c = 0; c < D / 8; ++c) *(uint4*)(vrow + (c >> 3) * (kBlk * 128) + (((c & 7) ^ (key & 7)) << 4)) = make_uint4(0u, 0u, 0u, 0u);
            fence_async();
          }
        }
        if (partly && bad) {
          const int at = atomicAdd(&note_count[piece_no & 3], 1);
          if (at < kNotes) note_key[piece_no & 3][at] = tok;
        }
        __syncwarp();
        if (lane == 0) {
          mbar_arrive((V ? v_ready : k_ready) + (J & 1));
          if (QUANT) mbar_arrive(&empty[st]);
        }
        if (++st == stages) { st = 0; ++round; }
      }
      J0 += pc.todo;
      ++piece_no;
    }
  } else if (warp == SH::COPY_AT || warp == SH::COPY_AT + 1) {
    // ---------------- copies: keys, values ----------------
    // (one elected lane issues them all; a lane of its own for every piece was no faster)
    if constexpr (SH::SPLIT) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(SH::R_MISC));
    const bool V = warp != SH::COPY_AT;
    const int pieces_of = kBlk / maps.piece, groups = maps.piece / 16, stages = V ? VS : KS;
    uint64_t* const full = V ? v_full : k_full;
    uint64_t* const empty = V ? v_empty : k_empty;
    const uint32_t ring = smem_u32(smem + (V ? SH::VR : SH::KR)), stage_b = V ? SH::V_STAGE : SH::K_STAGE;
    const uint32_t codes_b = (uint32_t)maps.piece * SH::ROWB, box_b = QUANT ? codes_b : (uint32_t)maps.piece * 128u, sb_b = (uint32_t)maps.piece * G * 2;
    const bool vec = QUANT && a.sb_vec;
    const uint32_t piece_b = codes_b + (vec ? (V ? 2u : 4u) * sb_b : 0u);
    int st = 0;
    uint32_t round = 0;
    bool stop = false;
    while (!stop && pieces.next(pc)) {
      const int32_t* const tab = a.table + (int64_t)pc.s.row * a.table_str;
      auto page_at = [&](int j) {
        int pid = -1;
        if (j < pc.todo && lane < pieces_of) {
          const int tok = pc.first_token(j) + lane * maps.piece;
          if (tok < pc.s.len) pid = tab[tok >> a.page_shift];
          if (pid >= a.P) pid = -1;
        }
        return pid;
      };
      int pid_next = page_at(0);
#pragma unroll 1
      for (int j = 0; j < pc.todo; ++j) {
        const int pid = pid_next, row0 = pc.first_token(j) & pmask;      // (pieces of one page follow each other; else each begins its page)
        pid_next = page_at(j + 1);
        const uint32_t have = __ballot_sync(0xffffffffu, pid >= 0);
        if (round > 0) wait(&empty[st], round - 1, V ? 614 : 613);
        stop = failed();                                       // (a place whose copies may not have come is not armed again)
        if (stop) break;
        const uint32_t to = ring + st * stage_b;
        if (lane == 0) {
          uint32_t bits = 0xffu;                               // of 16 tokens each
          if (have != (1u << pieces_of) - 1u) {
            bits = 0;
            for (int i = 0; i < pieces_of; ++i)
              if ((have >> i) & 1u) bits |= ((1u << groups) - 1u) << (i * groups);
          }
          s_pages[V][(J0 + j) & 15] = bits;
          mbar_expect_tx(&full[st], (uint32_t)__popc(have) * piece_b);
        }
        __syncwarp();
        for (int i = 0; i < pieces_of; ++i) {
          const int page = __shfl_sync(0xffffffffu, pid, i);
          if (page < 0) continue;
          const int row = (row0 + i * maps.piece) & pmask;
          if (elect_one()) {
#pragma unroll
            for (int h = 0; h < (QUANT ? 1 : SH::HALVES); ++h)
              tma_load_4d(to + h * kBlk * 128 + i * box_b, V ? &mv : &mk, &full[st], 64 * h, row, pc.hk * maps.mul[V][0], page * maps.mul[V][1]);
            if (vec) {
              const uint32_t sb = to + kBlk * SH::ROWB + i * sb_b;
              const int64_t at_v = (int64_t)page * a.pool[1].sb_str[0] + (int64_t)pc.hk * a.pool[1].sb_str[1] + (int64_t)row * G;
              if (V) {
                bulk_load(sb, (const uint16_t*)a.pool[1].s + at_v, sb_b, &full[st]);
                bulk_load(sb + SH::SB, (const uint16_t*)a.pool[1].b + at_v, sb_b, &full[st]);
              } else {
                const int64_t at_k = (int64_t)page * a.pool[0].sb_str[0] + (int64_t)pc.hk * a.pool[0].sb_str[1] + (int64_t)row * G;
                bulk_load(sb, (const uint16_t*)a.pool[0].s + at_k, sb_b, &full[st]);
                bulk_load(sb + SH::SB, (const uint16_t*)a.pool[0].b + at_k, sb_b, &full[st]);
                bulk_load(sb + 2 * SH::SB, (const uint16_t*)a.pool[1].s + at_v, sb_b, &full[st]);
                bulk_load(sb + 3 * SH::SB, (const uint16_t*)a.pool[1].b + at_v, sb_b, &full[st]);
              }
            }
          }
          __syncwarp();
        }
        if (++st == stages) { st = 0; ++round; }
      }
      J0 += pc.todo;
    }
  } else if (warp == SH::MMA_AT) {
    // ---------------- products ----------------
    if constexpr (SH::SPLIT) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(SH::R_MISC));
    constexpr uint32_t type = QUANT ? 0u : 1u;                 // fp16, bf16
    constexpr uint32_t idesc0 = (1u << 4) | (type << 7) | (type << 10) | ((uint32_t)(N >> 3) << 17) | ((128u >> 4) << 24);
    constexpr uint32_t idesc_s = idesc0, idesc_o = idesc0 | (1u << 15) | (1u << 16);   // the values and P: columns contiguous
    auto U = [](int v) { return __shfl_sync(0xffffffffu, v, 0); };
    const uint32_t tm = (uint32_t)U((int)tmem), sm = (uint32_t)U((int)smem_u32(smem));
    const uint64_t hi_k = make_desc(0) & 0xFFFFFFFF00000000ull, hi_v = make_desc_mn(0) & 0xFFFFFFFF00000000ull;
    const uint32_t q_d = (uint32_t)make_desc(sm + SH::Q0), k_d = (uint32_t)make_desc(sm + SH::KR), v_d = (uint32_t)make_desc_mn(sm + (QUANT ? SH::V0 : SH::VR)), p_d = (uint32_t)make_desc_mn(sm + SH::P0);
    const uint32_t most = t.polls > 0 ? (uint32_t)t.polls : kSpins;
    auto spin = [&](uint64_t* bar, uint32_t phase, int code) {
      const bool ok = __all_sync(0xffffffffu, spin_cta(bar, phase & 1, most, &s_fail));
      if (!ok && lane == 0) { *(volatile int*)&s_fail = code; atomicCAS(&g_tree_error, 0, code); }
      __syncwarp();
      return ok;
    };
    int piece_no = 0, ks = 0, vs = 0;                          // (at 16 bits the operands are the rings' places)
    uint32_t kr = 0;
    auto scores = [&](int J) {
      bool ok;
      if constexpr (QUANT) ok = spin(&k_ready[J & 1], (uint32_t)(J >> 1), 603);
      else ok = spin(&k_full[ks], kr, 603);
      fence_after();
      if (ok && elect_one()) {
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          const uint64_t q = hi_k | (q_d + (k >> 2) * ((N * 128) >> 4) + (k & 3) * 2);
          if constexpr (QUANT) umma_ts(tm + SH::S_AT + (J & 1) * SH::SW_AT, tm + SH::K_AT + (J & 1) * 64 + k * 8, q, idesc_s, k > 0);
          else umma_ss(tm + SH::S_AT + (J & 1) * SH::SW_AT, hi_k | (k_d + ks * (SH::TILE >> 4) + (k >> 2) * ((kBlk * 128) >> 4) + (k & 3) * 2), q, idesc_s, k > 0);
        }
        commit(&s_ready[J & 1]);
        if (!QUANT) commit(&k_empty[ks]);
      }
      __syncwarp();
      if (!QUANT && ++ks == KS) { ks = 0; ++kr; }
    };
    while (pieces.next(pc)) {
      const int todo = U(pc.todo);
      spin(&q_ready, (uint32_t)piece_no, 604);
      for (int j = -2; j < todo; ++j) {
        if (j >= 0) {
          const int J = J0 + j;
          const bool ok = spin(&v_ready[J & 1], (uint32_t)(J >> 1), 606) && spin(&p_ready[J & 1], (uint32_t)(J >> 1), 607);
          fence_after();
          if (ok && elect_one()) {
#pragma unroll
            for (int part = 0; part < SH::PP; ++part)
#pragma unroll
              for (int k = 0; k < kBlk / 16; ++k)
                umma_ss(tm + SH::O_AT, hi_v | (v_d + (QUANT ? J & 1 : vs) * (SH::TILE >> 4) + k * (2048 >> 4)),
                        hi_v | (p_d + (J % SH::PS) * (SH::PTILE >> 4) + part * (SH::LOW >> 4) + k * (2048 >> 4)), idesc_o, part + k > 0 ? 1u : (j > 0 ? 1u : 0u));
            commit(&o_done[J & 1]);
            if (!QUANT) commit(&v_empty[vs]);
          }
          __syncwarp();
          if (!QUANT && ++vs == VS) vs = 0;
        }
        if (j + 2 < todo) scores(J0 + j + 2);
      }
      J0 += todo;
      ++piece_no;
    }
    // every product is complete before tensor memory and shared memory go
    if (J0 > 0) spin(&o_done[(J0 - 1) & 1], (uint32_t)((J0 - 1) >> 1), 608);
  } else if (warp < SW) {
    // ---------------- softmax: a thread a token ----------------
    if constexpr (SH::SPLIT) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(SH::R_SOFT));
    const int wg = warp >> 2, wq = warp & 3, key = tid & 127, col0 = wg * NC;
    const uint32_t lanes = tmem + ((uint32_t)wq << 21);
    constexpr int ALL = SW * 32;
    const float factor = fmaxf(fabsf(a.scale) * kLog2e, 1e-30f);   // (a factor of 0 would meet scores of -inf)
    int piece_no = 0;
    while (pieces.next(pc)) {
      const Seq& s = pc.s;
      // ---- the tree, the queries ----
      constexpr int LPR = D / 4, RPW = 32 / LPR, IT = N / (SW * RPW);    // lanes of a row, rows of a warp at a time
      uint32_t raw[IT][2];
      const int live = s.n * a.gqa;
#pragma unroll
      for (int i = 0; i < IT; ++i) {
        const int n = (i * SW + warp) * RPW + lane / LPR, R = pc.rt * N + n;
        raw[i][0] = raw[i][1] = 0u;
        if (R < live) {
          const int node = R / a.gqa, h = R - node * a.gqa;
          const uint16_t* const p = (const uint16_t*)a.q + (int64_t)pc.b * a.q_str[0] + (int64_t)(pc.hk * a.gqa + h) * a.q_str[1] + (int64_t)node * t.q_tok + (lane % LPR) * 4;
          if (a.q_vec) { const uint2 x = *(const uint2*)p; raw[i][0] = x.x; raw[i][1] = x.y; }
          else { raw[i][0] = (uint32_t)p[0] | ((uint32_t)p[1] << 16); raw[i][1] = (uint32_t)p[2] | ((uint32_t)p[3] << 16); }
        }
        if (a.scale < 0.f) { raw[i][0] ^= 0x80008000u; raw[i][1] ^= 0x80008000u; }   // so that the largest score is the largest sum
      }
      if (piece_no > 0) bar_sync(1 + 2 * SH::WGS, ALL);                      // (all are done with the last tile's lists)
      if (tid < kMaxNodes && tid < s.n) {
        const int p = t.parents[(int64_t)pc.b * t.par_str + tid];
        s_par[tid] = p >= 0 && p < tid ? p : -1;
      }
      if (tid < N) s_nr[tid] = -kNegBig;
      if constexpr (QUANT) {
#pragma unroll
        for (int i = 0; i < IT; ++i) {
          float mx = 0.f;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const float x = fabsf((k & 1) ? bf16hi(raw[i][k >> 1]) : bf16lo(raw[i][k >> 1]));
            mx = x < INFINITY ? fmaxf(mx, x) : mx;
          }
#pragma unroll
          for (int o = LPR / 2; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
          const int e = (int)(__float_as_uint(mx) >> 23) - 127;
          if (lane % LPR == 0) s_qe[(i * SW + warp) * RPW + lane / LPR] = mx > 0.f ? (e < -100 ? -100 : (e > 110 ? 110 : e)) : -1000;
        }
      }
      bar_sync(1 + 2 * SH::WGS, ALL);
      if (tid < s.n && tid < kMaxNodes) {
        uint64_t line = 0;
        int depth = -1;
        for (int i = tid; i >= 0; i = s_par[i]) { line |= 1ull << i; ++depth; }
        s_line[tid] = line; s_depth[tid] = depth;
      }
      // queries in fp16: all in the unit of the largest, where their sizes are near one another, else each in its own
      int emax = 0;
      bool alike = true;
      if constexpr (QUANT) {
        int hi = -1000, lo = 1000;
        for (int i = lane; i < N; i += 32) { const int e = s_qe[i]; if (e > -1000) { hi = e > hi ? e : hi; lo = e < lo ? e : lo; } }
        hi = __reduce_max_sync(0xffffffffu, hi); lo = __reduce_min_sync(0xffffffffu, lo);
        emax = hi > -1000 ? hi : 0;
        alike = hi - lo <= 12;
      }
#pragma unroll
      for (int i = 0; i < IT; ++i) {
        const int n = (i * SW + warp) * RPW + lane / LPR, l = lane % LPR;
        uint32_t w0 = raw[i][0], w1 = raw[i][1];
        if constexpr (QUANT) {
          const int e = alike || s_qe[n] == -1000 ? emax : s_qe[n];
          const float up = pow2i(14 - e);
          const uint32_t h0 = pack_f16x2(bf16lo(raw[i][0]) * up, bf16hi(raw[i][0]) * up), h1 = pack_f16x2(bf16lo(raw[i][1]) * up, bf16hi(raw[i][1]) * up);
          if constexpr (BITS == 4) {       // eight dims of two lanes: 0 4 1 5 in the first, 2 6 3 7 in the second
            const uint32_t got = __shfl_xor_sync(0xffffffffu, l & 1 ? h0 : h1, 1);
            const uint32_t x = l & 1 ? got : h0, y = l & 1 ? h1 : got;
            w0 = __byte_perm(x, y, 0x5410); w1 = __byte_perm(x, y, 0x7632);
          } else { w0 = __byte_perm(h0, h1, 0x5410); w1 = __byte_perm(h0, h1, 0x7632); }
        }
        const int d = 4 * l, c = (d & 63) >> 3;
        *(uint2*)(smem + SH::Q0 + (d >> 6) * (N * 128) + n * 128 + ((c ^ (n & 7)) << 4) + (l & 1) * 8) = make_uint2(w0, w1);
      }
      fence_async();
      bar_sync(1 + 2 * SH::WGS, ALL);
      if (lane == 0) mbar_arrive(&q_ready);
      if (tid < N) {
        const int R = pc.rt * N + tid, node = R < live ? R / a.gqa : -1;
        s_cline[tid] = node >= 0 ? s_line[node] : 0ull;
        s_clo[tid] = node >= 0 ? s.base + s_depth[node] - a.window : 0;
      }
      if (tid == 0) note_count[(piece_no + 3) & 3] = 0;        // (read before, and not yet used again: the other roles are two blocks ahead at most)
      bar_sync(1 + 2 * SH::WGS, ALL);
      const float Cq = QUANT ? factor * pow2i(emax - 14) : factor;

      uint64_t l2[NC / 2];
#pragma unroll
      for (int i = 0; i < NC / 2; ++i) l2[i] = 0ull;
#pragma unroll 1
      for (int j = 0; j < pc.todo; ++j) {
        const int J = J0 + j, k0 = pc.first_token(j), tok = k0 + key;
        wait(&s_ready[J & 1], (uint32_t)(J >> 1), 609);
        fence_after();
        float ck = Cq, w = 1.f, ev = 0.f;
        if constexpr (QUANT) {
          const int e = s_vexp[J & 3][key];
          ck *= s_kunit[J & 3][key];
          ev = (float)e;
          w = pow2i(-e);
        }
        const bool masked = s_pages[0][J & 15] != 0xffu || !pc.whole(t, k0);
        const uint32_t s_at = lanes + SH::S_AT + (J & 1) * SH::SW_AT + col0;
        uint32_t z[NC];
        auto exponents = [&](bool with_reference) {            // of P' (or, without the reference, of P' 2^r)
          tmem_get<NC>(s_at, z);
          if (QUANT && !alike)
#pragma unroll
            for (int i = 0; i < NC; ++i) {
              const int e = s_qe[col0 + i];
              z[i] = __float_as_uint(__uint_as_float(z[i]) * (e == -1000 ? 1.f : pow2i(e - emax < -126 ? -126 : e - emax)));
            }
          const uint64_t ck2 = two(ck, ck), ev2 = two(ev, ev);
#pragma unroll
          for (int i = 0; i < NC / 4; ++i) {
            uint64_t r0 = ev2, r1 = ev2;
            if (with_reference) {
              const ulonglong2 nr = *(const ulonglong2*)&s_nr[col0 + 4 * i];
              if constexpr (QUANT) { r0 = add2(nr.x, ev2); r1 = add2(nr.y, ev2); } else { r0 = nr.x; r1 = nr.y; }
            }
            const uint64_t x = fma2(two(__uint_as_float(z[4 * i]), __uint_as_float(z[4 * i + 1])), ck2, r0), y = fma2(two(__uint_as_float(z[4 * i + 2]), __uint_as_float(z[4 * i + 3])), ck2, r1);
            float f0, f1, f2, f3;
            untwo(x, f0, f1); untwo(y, f2, f3);
            z[4 * i] = __float_as_uint(f0); z[4 * i + 1] = __float_as_uint(f1); z[4 * i + 2] = __float_as_uint(f2); z[4 * i + 3] = __float_as_uint(f3);
          }
          if (masked) {
            const bool mine = pc.some_see(tok) && ((s_pages[0][J & 15] >> (key >> 4)) & 1u), drafted = tok >= s.base;
            const int m = drafted ? tok - s.base : 0, at = drafted ? s.base + (mine ? s_depth[m] : 0) : tok;
            const bool inside = a.window == 0 || at < a.sinks;
#pragma unroll
            for (int i = 0; i < NC; ++i) {
              const bool sees = mine && (!drafted || ((s_cline[col0 + i] >> m) & 1ull)) && (inside || at > s_clo[col0 + i]);
              if (!sees) z[i] = 0xff800000u;
            }
          }
        };
        exponents(true);
        float mx = -INFINITY;
#pragma unroll
        for (int i = 0; i < NC; i += 2) mx = max3(mx, __uint_as_float(z[i]), __uint_as_float(z[i + 1]));
        if (bar_any(1 + wg, 128, mx > kTop)) {
          exponents(false);
          // the columns' maxima over the warp's tokens: lane n ends with that of column n
          float v[NC];
#pragma unroll
          for (int i = 0; i < NC; ++i) v[i] = __uint_as_float(z[i]);
#pragma unroll
          for (int o = NC / 2; o > 0; o >>= 1)
#pragma unroll
            for (int i = 0; i < o; ++i) {
              const bool up = (lane & o) != 0;
              const float keep = up ? v[i + o] : v[i], give = up ? v[i] : v[i + o];
              v[i] = fmaxf(fmaxf(keep, -INFINITY), __shfl_xor_sync(0xffffffffu, give, o));
            }
          if constexpr (NC == 16) v[0] = fmaxf(v[0], __shfl_xor_sync(0xffffffffu, v[0], 16));
          if (lane < NC) s_wmax[wg][wq][lane] = v[0];
          bar_sync(1 + SH::WGS + wg, 128);
          float f = 1.f, nr = 0.f;
          if (lane < NC) {
            nr = s_nr[col0 + lane];
            const float top = fmaxf(fmaxf(s_wmax[wg][0][lane], s_wmax[wg][1][lane]), fmaxf(s_wmax[wg][2][lane], s_wmax[wg][3][lane]));
            if (top + nr > kTop) {
              f = ex2(kAim - top - nr);
              nr = kAim - top;
            }
          }
          bar_sync(1 + SH::WGS + wg, 128);                               // (all have read the old ones)
          if (wq == 0 && lane < NC) s_nr[col0 + lane] = nr;
          if (j > 0) {
            wait(&o_done[(J - 1) & 1], (uint32_t)((J - 1) >> 1), 610);
            fence_after();
            uint32_t o[NC];
            tmem_get<NC>(lanes + SH::O_AT + col0, o);
#pragma unroll
            for (int i = 0; i < NC; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * __shfl_sync(0xffffffffu, f, i));
            tmem_put<NC>(lanes + SH::O_AT + col0, o);
#pragma unroll
            for (int i = 0; i < NC / 2; ++i) l2[i] = mul2(l2[i], two(__shfl_sync(0xffffffffu, f, 2 * i), __shfl_sync(0xffffffffu, f, 2 * i + 1)));
          }
          bar_sync(1 + SH::WGS + wg, 128);
          exponents(true);
        }
        uint32_t p[NC / 2];
        const uint64_t w2 = two(w, w);
#pragma unroll
        for (int i = 0; i < NC / 2; ++i) {
          const float x0 = ex2(__uint_as_float(z[2 * i])), x1 = ex2(__uint_as_float(z[2 * i + 1]));
          if constexpr (QUANT) { l2[i] = fma2(two(x0, x1), w2, l2[i]); p[i] = pack_f16x2(x0, x1); }
          else {
            l2[i] = add2(l2[i], two(x0, x1));
            p[i] = pack2(x0, x1);
            z[i] = pack2(x0 - bf16lo(p[i]), x1 - bf16hi(p[i]));
          }
        }
        if (J >= SH::PS) wait(&o_done[(J - SH::PS) & 1], (uint32_t)((J - SH::PS) >> 1), 611);
        unsigned char* const prow = smem + SH::P0 + (J % SH::PS) * SH::PTILE + (col0 >> 6) * (kBlk * 128) + key * 128;
#pragma unroll
        for (int c = 0; c < NC / 8; ++c)
          *(uint4*)(prow + ((((col0 & 63) / 8 + c) ^ (key & 7)) << 4)) = make_uint4(p[4 * c], p[4 * c + 1], p[4 * c + 2], p[4 * c + 3]);
        if constexpr (SH::PP == 2)
#pragma unroll
          for (int c = 0; c < NC / 8; ++c)
            *(uint4*)(prow + (N > 32 ? SH::LOW : 0) + ((((col0 & 63) / 8 + c + (N > 32 ? 0 : 4)) ^ (key & 7)) << 4)) = make_uint4(z[4 * c], z[4 * c + 1], z[4 * c + 2], z[4 * c + 3]);
        fence_async();
        fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_ready[J & 1]);
      }
      // ---- the tile's results, a thread a dim ----
      const int last = J0 + pc.todo - 1;
      float l[NC];
#pragma unroll
      for (int i = 0; i < NC / 2; ++i) untwo(l2[i], l[2 * i], l[2 * i + 1]);
#pragma unroll
      for (int o = NC / 2; o > 0; o >>= 1)
#pragma unroll
        for (int i = 0; i < o; ++i) {
          const bool up = (lane & o) != 0;
          const float keep = up ? l[i + o] : l[i], give = up ? l[i] : l[i + o];
          l[i] = keep + __shfl_xor_sync(0xffffffffu, give, o);
        }
      if constexpr (NC == 16) l[0] += __shfl_xor_sync(0xffffffffu, l[0], 16);
      if (lane < NC) s_wmax[wg][wq][lane] = l[0];
      wait(&o_done[last & 1], (uint32_t)(last >> 1), 612);
      fence_after();
      uint32_t o[NC];
      tmem_get<NC>(lanes + SH::O_AT + col0, o);
      fence_before();
      bar_sync(1 + SH::WGS + wg, 128);
      float L = 0.f, r = 0.f;
      if (lane < NC) {
        L = (s_wmax[wg][0][lane] + s_wmax[wg][1][lane]) + (s_wmax[wg][2][lane] + s_wmax[wg][3][lane]);
        r = -s_nr[col0 + lane];
        if (*(volatile int*)&s_fail) L = __uint_as_float(0x7fc00000u);
        const int notes = note_count[piece_no & 3];
        for (int i = 0; i < notes && i < kNotes; ++i) {
          const int k = note_key[piece_no & 3][i];
          const bool drafted = k >= s.base;
          const int m = drafted ? (k - s.base) & (kMaxNodes - 1) : 0;        // (behind a wait that ran out, k may be anything)
          const int at = drafted ? s.base + s_depth[m] : k;
          if ((!drafted || ((s_cline[col0 + lane] >> m) & 1ull)) && (a.window == 0 || at < a.sinks || at > s_clo[col0 + lane])) L = __uint_as_float(0x7fc00000u);
        }
      }
      const bool all = pc.blk0 == 0 && pc.todo == s.blocks;
      const int rows = live - pc.rt * N < N ? live - pc.rt * N : N;
      if (all) {
        const float inv = L > 0.f ? 1.f / L : (L == L ? 0.f : L);
        const int dim = dim_at<BITS>(key);
#pragma unroll
        for (int i = 0; i < NC; ++i) {
          const float v = __uint_as_float(o[i]) * __shfl_sync(0xffffffffu, inv, i);
          if (col0 + i < rows && key < D) {
            const int R = pc.rt * N + col0 + i, node = R / a.gqa, h = R - node * a.gqa;
            ((uint16_t*)a.out)[(int64_t)pc.b * a.o_str[0] + (int64_t)(pc.hk * a.gqa + h) * a.o_str[1] + (int64_t)node * t.o_tok + dim] = f32_to_bf16_bits(v);
          }
        }
      } else {
        const int64_t slot = 2 * (int64_t)blockIdx.x + (pc.blk0 == 0 ? 1 : 0);
        if (pc.blk0 == 0 && tid == 0) a.joins[blockIdx.x] = make_int4(pc.b, pc.hk, pc.rt, pc.more);
        if (wq == 0 && lane < NC) a.part_ml[slot * N + col0 + lane] = make_float2(r, L);
#pragma unroll
        for (int i = 0; i < NC; ++i)
          if (col0 + i < rows && key < D) a.part_o[(slot * N + col0 + i) * D + key] = __uint_as_float(o[i]);
      }
      J0 += pc.todo;
      ++piece_no;
    }
    // nodes that are not there: zeros
    for (int b = blockIdx.x; b < a.B; b += gridDim.x) {
      const int n = seq_of(t, b, N).n;
      for (int64_t i = tid; i < (int64_t)(t.T - n) * a.Hq * D; i += ALL) {
        const int e = (int)(i % D), h = (int)(i / D % a.Hq), node = n + (int)(i / D / a.Hq);
        ((uint16_t*)a.out)[(int64_t)b * a.o_str[0] + (int64_t)h * a.o_str[1] + (int64_t)node * t.o_tok + e] = 0;
      }
    }
  }
  else if constexpr (SH::SPLIT) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(SH::R_MISC));   // (two warps without a role complete the group of four)
  __syncwarp();
  fence_before();
  __syncthreads();
  if (*(volatile int*)&s_fail)
    for (int i = 0; i < 1000; ++i) __nanosleep(1000);          // (copies and products may still be on their way: a millisecond for them)
  if (warp == SH::MMA_AT) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u));
}

// ---- the parts of a tile that several CTAs share: out = (sum_i o_i w_i) / (sum_i l_i w_i), w_i = 2^(r_i - max r) ----
// CTA (c, y) joins 8 rows of the tile that begins in CTA c's share and ends behind it: its own part (slot 2c + 1) and those of the next
// CTAs (slots 2(c + k)).  A warp takes one row's every second part.
template <int BITS, int D>
__global__ void __launch_bounds__(kJoinWarps * 32) tree_join_kernel(const __grid_constant__ KvPagesTreeArgs t, int N) {
  __shared__ float red[kJoinWarps][D + 2];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const KvPagesAttnArgs& a = t.a;
  const int4 jn = a.joins[blockIdx.x];
  if (jn.x < 0) return;
  const Seq s = seq_of(t, jn.x, N);
  const int row0 = (int)blockIdx.y * kJoinRows, left = s.n * a.gqa - jn.z * N - row0;
  if (left <= 0) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, n = jn.w + 1;
  constexpr int parts = kJoinWarps / kJoinRows;
  const int rows = left < kJoinRows ? left : kJoinRows, h = warp % kJoinRows, part = warp / kJoinRows;
  constexpr int E = D / 32;
  auto slot = [&](int k) { return (int64_t)(k == 0 ? 2 * (int)blockIdx.x + 1 : 2 * ((int)blockIdx.x + k)); };
  float M = kNegBig, L = 0.f, o[E];
#pragma unroll
  for (int i = 0; i < E; ++i) o[i] = 0.f;
  if (h < rows) {
    for (int k0 = part; k0 < n; k0 += parts * 32) {
      const int k = k0 + lane * parts;
      float2 ml = make_float2(kNegBig, 0.f);
      if (k < n) ml = __ldcg(a.part_ml + slot(k) * N + row0 + h);
      float m = ml.x;
#pragma unroll
      for (int x = 16; x > 0; x >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, x));
      const float Mn = fmaxf(M, m), f = ex2(M - Mn), w = ex2(ml.x - Mn);
      L = L * f + w * ml.y;          // a lane's own parts
#pragma unroll
      for (int i = 0; i < E; ++i) o[i] *= f;
      M = Mn;
      const int cnt = (n - k0 + parts - 1) / parts < 32 ? (n - k0 + parts - 1) / parts : 32;
#pragma unroll 8
      for (int q = 0; q < cnt; ++q) {
        const float wq = __shfl_sync(0xffffffffu, w, q);
        const float* src = a.part_o + (slot(k0 + q * parts) * N + row0 + h) * D + lane * E;
        if constexpr (E == 4) {
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
    for (int i = 0; i < E; ++i) red[warp][lane * E + i] = o[i];
    if (lane == 0) { red[warp][D] = M; red[warp][D + 1] = L; }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < rows * D; i += kJoinWarps * 32) {
    const int r = i / D, e = i - r * D;
    float Mx = kNegBig;
#pragma unroll
    for (int p = 0; p < parts; ++p) Mx = fmaxf(Mx, red[p * kJoinRows + r][D]);
    float Ls = 0.f, Os = 0.f;
#pragma unroll
    for (int p = 0; p < parts; ++p) {
      const float f = ex2(red[p * kJoinRows + r][D] - Mx);
      Ls += red[p * kJoinRows + r][D + 1] * f;
      Os += red[p * kJoinRows + r][e] * f;
    }
    const float v = Os * (Ls > 0.f ? 1.f / Ls : (Ls == Ls ? 0.f : Ls));
    const int R = jn.z * N + row0 + r, node = R / a.gqa, hh = R - node * a.gqa;
    ((uint16_t*)a.out)[(int64_t)jn.x * a.o_str[0] + (int64_t)(jn.y * a.gqa + hh) * a.o_str[1] + (int64_t)node * t.o_tok + dim_at<BITS>(e)] = f32_to_bf16_bits(v);
  }
}

// Columns of a tile: as many as the widest tree has rows of a cache head, up to 128.  More than 64 rows take 128 columns where there is much to
// read (128 rows over 16 sequences of 32k tokens 515 us, as two tiles of 64 723), but 64 where the tables hold at most four blocks an SM, since
// the wide tile takes longer to begin and to end (135 rows over 3 sequences of 2k tokens 31.9 us, 37.5 with 128; one of 2k with 128 rows 30.9 and 36.5;
// with seven blocks an SM 36.0 and 34.9).
int columns(int64_t T, int64_t gqa) { return T * gqa <= 16 ? 16 : (T * gqa <= 32 ? 32 : (T * gqa <= 64 ? 64 : 128)); }
int columns_of(const KvPagesTreeArgs& t) {
  const int n = columns(t.T, t.a.gqa);
  if (n < 128) return n;
  const int64_t blocks = (((int64_t)t.a.M << t.a.page_shift) + kBlk - 1) / kBlk, tiles = (int64_t)t.a.B * t.a.Hkv * (((int64_t)t.T * t.a.gqa + 63) / 64);
  return blocks * tiles <= 4 * (int64_t)sm_count() ? 64 : 128;
}

// [pages, heads, page, cols] as boxes of `piece` tokens; axes that repeat one entry as one entry at coordinate 0.
template <int BITS, int D> bool pool_map(CUtensorMap* m, const KvPagesAttnArgs& a, int side, int piece, int* mul) {
  const EncodeFn enc = get_encode();
  constexpr int ROWB = D * BITS / 8, COLS = BITS == 16 ? D : ROWB / 4, BOX = BITS == 16 ? 64 : COLS;
  const cuuint64_t page = (cuuint64_t)1 << a.page_shift;
  cuuint64_t dims[4] = {(cuuint64_t)COLS, page, 1, 1}, strides[3] = {(cuuint64_t)a.tok_bytes[side], (cuuint64_t)ROWB, (cuuint64_t)ROWB};
  const int64_t shape[2] = {a.Hkv, a.P}, str[2] = {a.q_head[side], (int64_t)a.page_bytes[side]};
  for (int d = 0; d < 2; ++d) {
    mul[d] = shape[d] > 1 && str[d] > 0 ? 1 : 0;
    if (mul[d]) { dims[2 + d] = (cuuint64_t)shape[d]; strides[1 + d] = (cuuint64_t)str[d]; }
  }
  const cuuint32_t box[4] = {(cuuint32_t)BOX, (cuuint32_t)piece, 1, 1}, es[4] = {1, 1, 1, 1};
  constexpr CUtensorMapSwizzle swizzle = BITS == 16 || ROWB == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : (ROWB == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_32B);
  return enc && enc(m, BITS == 16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_UINT32, 4, (void*)a.pool[side].q, dims, strides, box, es,
                    CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int BITS, int D, int N> cudaError_t launch_n(const KvPagesTreeArgs& t, cudaStream_t st) {
  auto kern = tree_kernel<BITS, D, N>;
  static bool done[64] = {};
  const size_t most = Shape<BITS, D, N>::SMEM + 2 * (kMaxPageSeqs + 1) * 4, smem = Shape<BITS, D, N>::SMEM + 2 * (size_t)(t.a.B + 1) * 4;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  {
    std::lock_guard<std::mutex> setup_lk(setup_mutex());     // first use on a device, from any thread
    if (dev < 0 || dev >= 64 || !done[dev]) {
      e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most);
      if (e != cudaSuccess) return e;
      if (dev >= 0 && dev < 64) done[dev] = true;
    }
  }
  CUtensorMap mk, mv;
  TreeMaps maps;
  maps.piece = t.a.page_shift >= 7 ? kBlk : 1 << t.a.page_shift;
  if (!pool_map<BITS, D>(&mk, t.a, 0, maps.piece, maps.mul[0]) || !pool_map<BITS, D>(&mv, t.a, 1, maps.piece, maps.mul[1])) return cudaErrorInvalidValue;
  const unsigned grid = (unsigned)sm_count();
  e = launch_behind(kern, dim3(grid), dim3(Shape<BITS, D, N>::THREADS), smem, st, mk, mv, t, maps);
  if (e != cudaSuccess) return e;
  return launch_behind(tree_join_kernel<BITS, D>, dim3(grid, (N + kJoinRows - 1) / kJoinRows), dim3(kJoinWarps * 32), 0, st, t, N);
}
template <int BITS, int D> cudaError_t launch_d(const KvPagesTreeArgs& t, cudaStream_t st) {
  switch (columns_of(t)) {
    case 16: return launch_n<BITS, D, 16>(t, st);
    case 32: return launch_n<BITS, D, 32>(t, st);
    case 64: return launch_n<BITS, D, 64>(t, st);
    default: return launch_n<BITS, D, 128>(t, st);
  }
}
}  // namespace

// [joins: int4 per CTA][r, l: float2 per slot and row][o: D floats per slot and row], two slots a CTA
size_t kv_pages_tree_workspace_bytes(int64_t, int64_t Hq, int64_t Hkv, int64_t T, int64_t D) {
  const size_t ctas = (size_t)sm_count(), rows = (size_t)columns(T, Hq / Hkv);
  return ctas * 16 + ctas * 2 * rows * (8 + (size_t)D * 4);
}

cudaError_t launch_kv_pages_tree(KvPagesTreeArgs t, int D, void* workspace, cudaStream_t st) {
  const size_t ctas = (size_t)sm_count(), rows = (size_t)columns_of(t);
  t.polls = wait_polls();
  t.a.joins = (int4*)workspace;
  t.a.part_ml = (float2*)((char*)workspace + ctas * 16);
  t.a.part_o = (float*)((char*)workspace + ctas * 16 + ctas * 2 * rows * 8);
  switch (t.a.bits * 1000 + D) {
    case 4064: return launch_d<4, 64>(t, st);
    case 4128: return launch_d<4, 128>(t, st);
    case 8064: return launch_d<8, 64>(t, st);
    case 8128: return launch_d<8, 128>(t, st);
    case 16064: return launch_d<16, 64>(t, st);
    case 16128: return launch_d<16, 128>(t, st);
    default: return cudaErrorInvalidValue;
  }
}

void tree_attn_error_reset() {
  const int zero = 0;
  cudaMemcpyToSymbol(g_tree_error, &zero, sizeof(int));
}
int tree_attn_error_code() {
  int v = 0;
  cudaMemcpyFromSymbol(&v, g_tree_error, sizeof(int));
  return v;
}

}  // namespace qb
