// C ABI of the paged key-value cache and of windowed prompt attention: argument validation and dispatch (include/qb200.h).
// As in the other entries everything is checked on the host before any CUDA call; what only the device knows (page numbers,
// lengths, listed sequences) is checked by the kernels, which skip what lies outside the tensors.
#include <cstdarg>
#include <cstdio>
#include <cstring>

#include "kernels.h"

using namespace qb;

namespace {

int pg_fail(int status, const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  return report_error(status, buf);
}
int pg_cuda(cudaError_t e, const char* who) {
  (void)cudaGetLastError();              // (reported here, so that no later entry takes it for its own)
  return pg_fail(QB200_ERR_CUDA, "%s: CUDA error %d (%s)", who, (int)e, cudaGetErrorString(e));
}
bool empty(const qb200_tensor* t) { return t == nullptr || (t->data == nullptr && t->ndim == 0); }

int elem_size(int dtype) {
  switch (dtype) {
    case QB200_UINT8: case QB200_INT8: return 1;
    case QB200_UINT16: case QB200_INT16: case QB200_FLOAT16: case QB200_BFLOAT16: return 2;
    case QB200_UINT32: case QB200_INT32: case QB200_FLOAT32: return 4;
    default: return 0;
  }
}
// A tensor of a given rank and dtype, aligned to its elements, whose last axis is contiguous.
int expect(const qb200_tensor* t, const char* who, const char* name, int ndim, int dtype) {
  if (t == nullptr) return pg_fail(QB200_ERR_BAD_ARG, "%s: %s: null tensor", who, name);
  if (t->ndim != ndim) return pg_fail(QB200_ERR_BAD_SHAPE, "%s: %s must have %d dimensions, not %d", who, name, ndim, t->ndim);
  if (ndim > QB200_MAX_DIMS) return pg_fail(QB200_ERR_BAD_SHAPE, "%s: %s has %d dimensions", who, name, ndim);
  if (t->dtype != dtype) return pg_fail(QB200_ERR_BAD_DTYPE, "%s: %s has dtype %d, expected %d", who, name, t->dtype, dtype);
  const int esz = elem_size(dtype);
  if (esz > 1 && (uintptr_t)t->data % esz) return pg_fail(QB200_ERR_BAD_STRIDE, "%s: %s does not start on its elements' size", who, name);
  int64_t n = 1;
  for (int d = 0; d < ndim; ++d) {
    if (t->shape[d] < 0) return pg_fail(QB200_ERR_BAD_SHAPE, "%s: %s: negative extent in dim %d", who, name, d);
    if (t->stride[d] < 0) return pg_fail(QB200_ERR_BAD_STRIDE, "%s: %s: negative stride in dim %d", who, name, d);
    n = t->shape[d] > 0 && n > INT64_MAX / t->shape[d] ? INT64_MAX : n * t->shape[d];
  }
  if (n > 0 && t->data == nullptr) return pg_fail(QB200_ERR_BAD_ARG, "%s: %s: null data pointer", who, name);
  if (ndim > 0 && t->shape[ndim - 1] > 1 && t->stride[ndim - 1] != 1)
    return pg_fail(QB200_ERR_BAD_STRIDE, "%s: %s: last axis must be contiguous (stride %lld)", who, name, (long long)t->stride[ndim - 1]);
  return 0;
}
int expect_list(const qb200_tensor* t, const char* who, const char* name, int64_t n) {
  if (int st = expect(t, who, name, 1, QB200_INT32)) return st;
  if (t->shape[0] != n) return pg_fail(QB200_ERR_BAD_SHAPE, "%s: %s has %lld entries, expected %lld", who, name, (long long)t->shape[0], (long long)n);
  return 0;
}
// What a kernel writes: no two elements may be the same memory.  Axes by growing stride, each has to reach over all that the smaller
// ones span (so layouts in which the axes are nested in any order pass, and those that are not are refused).
bool distinct(const qb200_tensor* t) {
  int order[QB200_MAX_DIMS], n = 0;
  for (int d = 0; d < t->ndim; ++d) {
    if (t->shape[d] == 0) return true;
    if (t->shape[d] == 1) continue;
    int at = n++;
    for (; at > 0 && t->stride[order[at - 1]] > t->stride[d]; --at) order[at] = order[at - 1];
    order[at] = d;
  }
  int64_t span = 1;
  for (int i = 0; i < n; ++i) {
    const int64_t str = t->stride[order[i]], ext = t->shape[order[i]] - 1;
    if (str < span || str > (INT64_MAX - span) / ext) return false;
    span += str * ext;
  }
  return true;
}
int page_shift_of(int64_t page) {
  for (int k = 4; k <= 16; ++k)
    if (page == (int64_t)1 << k) return k;
  return -1;
}

// table [S, M], lens [S], refs [P]; lens and refs may be left out (null) where an operator has none.
int parse_state(PageState* s, const char* who, const qb200_tensor* table, const qb200_tensor* lens, const qb200_tensor* refs, int page) {
  int st;
  if ((st = expect(table, who, "table", 2, QB200_INT32))) return st;
  s->page_shift = page_shift_of(page);
  if (s->page_shift < 0) return pg_fail(QB200_ERR_UNSUPPORTED, "%s: pages of %d tokens are not served (a power of two from 16 to 65536)", who, page);
  if (table->shape[0] > INT32_MAX || table->shape[1] > INT32_MAX || ((table->shape[1] << s->page_shift) >> s->page_shift) != table->shape[1] ||
      (table->shape[1] << s->page_shift) > INT32_MAX)
    return pg_fail(QB200_ERR_UNSUPPORTED, "%s: a table of %lld sequences of %lld pages is not served (at most 2^31 - 1 tokens each)", who,
                   (long long)table->shape[0], (long long)table->shape[1]);
  if (table->shape[0] > 1 && table->stride[0] < table->shape[1]) return pg_fail(QB200_ERR_BAD_STRIDE, "%s: the table's rows overlap", who);
  s->table = (int32_t*)table->data; s->table_str = table->stride[0];
  s->S = (int)table->shape[0]; s->M = (int)table->shape[1];
  s->lens = nullptr; s->refs = nullptr; s->P = 0;
  if (lens) {
    if ((st = expect_list(lens, who, "lens", s->S))) return st;
    s->lens = (int32_t*)lens->data;
  }
  if (refs) {
    if ((st = expect(refs, who, "refs", 1, QB200_INT32))) return st;
    if (refs->shape[0] > kMaxPages)
      return pg_fail(QB200_ERR_UNSUPPORTED, "%s: a pool of %lld pages is not served (at most %d)", who, (long long)refs->shape[0], kMaxPages);
    s->refs = (int32_t*)refs->data; s->P = (int)refs->shape[0];
  }
  return 0;
}

// One side of a pool.  *vec: the scale rows of a page follow each other and start on 16 bytes.
int parse_pool(KvPoolView* v, bool* vec, const char* who, const char* side, const qb200_tensor* q, const qb200_tensor* s, const qb200_tensor* b, int bits,
               int64_t P, int64_t H, int64_t page, int64_t D) {
  int st;
  char name[32];
  snprintf(name, sizeof(name), "%s codes", side);
  const qb200_tensor* const ts[3] = {q, s, b};
  if ((st = expect(q, who, name, 4, bits == 16 ? QB200_BFLOAT16 : QB200_UINT32))) return st;
  const int n = bits == 16 ? 1 : 3;
  for (int i = 1; i < 3; ++i) {
    snprintf(name, sizeof(name), "%s %s", side, i == 1 ? "scales" : "biases");
    if (bits == 16) {
      if (!empty(ts[i])) return pg_fail(QB200_ERR_BAD_ARG, "%s: %s given for pages of 16 bits", who, name);
    } else if ((st = expect(ts[i], who, name, 4, QB200_BFLOAT16))) return st;
  }
  for (int i = 0; i < n; ++i) {
    const int64_t want[4] = {P, H, page, i ? D / 64 : (bits == 16 ? D : D * bits / 32)};
    for (int d = 0; d < 4; ++d)
      if (ts[i]->shape[d] != want[d])
        return pg_fail(QB200_ERR_BAD_SHAPE, "%s: dim %d of the %s %s is %lld, expected %lld", who, d, side, i ? "scales or biases" : "codes",
                       (long long)ts[i]->shape[d], (long long)want[d]);
  }
  const int64_t per16 = bits == 16 ? 8 : 4;
  bool ok = ((uintptr_t)q->data & 15) == 0;
  for (int d = 0; d < 3; ++d) ok = ok && (q->shape[d] <= 1 || q->stride[d] % per16 == 0);
  if (!ok) return pg_fail(QB200_ERR_UNSUPPORTED, "%s: the %s codes' rows must start on 16 bytes", who, side);
  std::memset(v, 0, sizeof(*v));
  v->q = q->data;
  for (int d = 0; d < 3; ++d) v->q_str[d] = q->stride[d];
  *vec = true;
  if (bits != 16) {
    for (int d = 0; d < 3; ++d)
      if (s->shape[d] > 1 && s->stride[d] != b->stride[d]) return pg_fail(QB200_ERR_BAD_STRIDE, "%s: %s scales and biases must have identical strides", who, side);
    v->s = s->data; v->b = b->data;
    for (int d = 0; d < 3; ++d) v->sb_str[d] = s->stride[d];
    *vec = s->stride[2] == D / 64 && (((uintptr_t)s->data | (uintptr_t)b->data) & 15) == 0 && (s->shape[0] <= 1 || s->stride[0] % 8 == 0) &&
           (s->shape[1] <= 1 || s->stride[1] % 8 == 0);
  }
  return 0;
}
int check_format(const char* who, int bits, int group_size, int64_t D) {
  if (bits != 4 && bits != 8 && bits != 16) return pg_fail(QB200_ERR_UNSUPPORTED, "%s: bits=%d is not served (4, 8, 16)", who, bits);
  if (bits != 16 && group_size != 64) return pg_fail(QB200_ERR_UNSUPPORTED, "%s: group_size=%d is not served (64)", who, group_size);
  if (D < 64 || D % 64 != 0 || D > 1024) return pg_fail(QB200_ERR_UNSUPPORTED, "%s: head dim %lld is not served (a multiple of 64 up to 1024)", who, (long long)D);
  return 0;
}

}  // namespace

extern "C" {

QB200_API int qb200_kv_pages_append(qb200_tensor* k_q, qb200_tensor* k_scales, qb200_tensor* k_biases, qb200_tensor* v_q, qb200_tensor* v_scales,
                                    qb200_tensor* v_biases, const qb200_tensor* dense_k, const qb200_tensor* dense_v, const qb200_tensor* table,
                                    const qb200_tensor* rows, const qb200_tensor* positions, const qb200_tensor* counts, int bits, int group_size,
                                    qb200_stream s) {
  const char* who = "kv_pages_append";
  int st;
  if ((st = expect(dense_k, who, "dense_k", 4, QB200_BFLOAT16)) || (st = expect(dense_v, who, "dense_v", 4, QB200_BFLOAT16))) return st;
  const int64_t N = dense_k->shape[0], H = dense_k->shape[1], S = dense_k->shape[2], D = dense_k->shape[3];
  if ((st = check_format(who, bits, group_size, D))) return st;
  for (int d = 0; d < 4; ++d)
    if (dense_v->shape[d] != dense_k->shape[d])
      return pg_fail(QB200_ERR_BAD_SHAPE, "%s: dense_k and dense_v differ in dim %d (%lld, %lld)", who, d, (long long)dense_k->shape[d], (long long)dense_v->shape[d]);
  if (k_q == nullptr || k_q->ndim != 4) return pg_fail(QB200_ERR_BAD_SHAPE, "%s: K codes must be [pages, heads, page, cols]", who);
  const int64_t P = k_q->shape[0], page = k_q->shape[2];
  PageState ps;
  if (page > 65536) return pg_fail(QB200_ERR_UNSUPPORTED, "%s: pages of %lld tokens are not served (a power of two from 16 to 65536)", who, (long long)page);
  if ((st = parse_state(&ps, who, table, nullptr, nullptr, (int)page))) return st;
  KvPagesAppendArgs a;
  std::memset(&a, 0, sizeof(a));
  bool vec;
  if ((st = parse_pool(&a.pool[0], &vec, who, "K", k_q, k_scales, k_biases, bits, P, H, page, D)) ||
      (st = parse_pool(&a.pool[1], &vec, who, "V", v_q, v_scales, v_biases, bits, P, H, page, D)))
    return st;
  const qb200_tensor* const written[6] = {k_q, k_scales, k_biases, v_q, v_scales, v_biases};
  for (int i = 0; i < 6; ++i)
    if (!empty(written[i]) && !distinct(written[i])) return pg_fail(QB200_ERR_BAD_STRIDE, "%s: rows of a pool overlap", who);
  if ((st = expect_list(positions, who, "positions", N))) return st;
  if (!empty(rows)) {
    if ((st = expect_list(rows, who, "rows", N))) return st;
    a.rows = (const int32_t*)rows->data;
  } else if (ps.S != N) return pg_fail(QB200_ERR_BAD_SHAPE, "%s: %lld sequences of new rows for a table of %d (pass rows)", who, (long long)N, ps.S);
  if (!empty(counts)) {
    if ((st = expect_list(counts, who, "counts", N))) return st;
    a.counts = (const int32_t*)counts->data;
  }
  if (N == 0 || H == 0 || S == 0 || P == 0 || ps.M == 0 || ps.S == 0) return QB200_OK;
  const qb200_tensor* const dense[2] = {dense_k, dense_v};
  a.dense_vec = 1;
  for (int i = 0; i < 2; ++i) {
    a.dense[i] = (const uint16_t*)dense[i]->data;
    if ((uintptr_t)dense[i]->data & 15) a.dense_vec = 0;
    for (int d = 0; d < 3; ++d) {
      a.dense_str[i][d] = dense[i]->stride[d];
      if (dense[i]->shape[d] > 1 && dense[i]->stride[d] % 8 != 0) a.dense_vec = 0;
    }
  }
  a.table = ps.table; a.table_str = ps.table_str;
  a.positions = (const int32_t*)positions->data;
  a.M = ps.M; a.seqs = ps.S; a.P = P; a.page_shift = ps.page_shift;
  const int64_t lim = (int64_t)1 << 31, per_row = D / 16;
  if (N >= lim || H >= lim || S >= lim || N * H >= lim || N * H * S >= lim || N * H * S * 2 * per_row >= lim)
    return pg_fail(QB200_ERR_UNSUPPORTED, "%s: %lld x %lld x %lld new rows are too many for one call", who, (long long)N, (long long)H, (long long)S);
  a.N = (int)N; a.H = (int)H; a.S = (int)S; a.per_row = (int)per_row; a.bits = bits;
  const cudaError_t e = launch_pages_append(a, (cudaStream_t)s);
  return e == cudaSuccess ? QB200_OK : pg_cuda(e, who);
}

QB200_API int qb200_kv_pages_free(qb200_tensor* table, qb200_tensor* lens, qb200_tensor* refs, int page, const qb200_tensor* rows, const qb200_tensor* begin,
                                  const qb200_tensor* end, qb200_stream s) {
  const char* who = "kv_pages_free";
  int st;
  PageState ps;
  if (lens == nullptr || refs == nullptr) return pg_fail(QB200_ERR_BAD_ARG, "%s: lens and refs are needed", who);
  if ((st = parse_state(&ps, who, table, lens, refs, page)) || (st = expect(rows, who, "rows", 1, QB200_INT32))) return st;
  const int64_t n = rows->shape[0];
  if (!empty(begin) && (st = expect_list(begin, who, "begin", n))) return st;
  if (!empty(end) && (st = expect_list(end, who, "end", n))) return st;
  if (n > 65535) return pg_fail(QB200_ERR_UNSUPPORTED, "%s: %lld sequences in one list are not served (at most 65535)", who, (long long)n);
  if (n == 0 || ps.S == 0) return QB200_OK;
  const cudaError_t e = launch_pages_free(ps, (const int32_t*)rows->data, empty(begin) ? nullptr : (const int32_t*)begin->data,
                                          empty(end) ? nullptr : (const int32_t*)end->data, (int)n, (cudaStream_t)s);
  return e == cudaSuccess ? QB200_OK : pg_cuda(e, who);
}

QB200_API int qb200_kv_pages_fork(qb200_tensor* shared, qb200_tensor* table, qb200_tensor* lens, qb200_tensor* refs, int page, const qb200_tensor* src,
                                  const qb200_tensor* dst, const qb200_tensor* tokens, qb200_stream s) {
  const char* who = "kv_pages_fork";
  int st;
  PageState ps;
  if (lens == nullptr || refs == nullptr) return pg_fail(QB200_ERR_BAD_ARG, "%s: lens and refs are needed", who);
  if ((st = parse_state(&ps, who, table, lens, refs, page)) || (st = expect(src, who, "src", 1, QB200_INT32))) return st;
  const int64_t n = src->shape[0];
  if ((st = expect_list(dst, who, "dst", n)) || (st = expect_list(shared, who, "shared", n))) return st;
  if (!empty(tokens) && (st = expect_list(tokens, who, "tokens", n))) return st;
  if (n > kMaxPageList) return pg_fail(QB200_ERR_UNSUPPORTED, "%s: %lld sequences in one list are not served (at most %d)", who, (long long)n, kMaxPageList);
  if (n == 0) return QB200_OK;
  const cudaError_t e = launch_pages_fork(ps, (const int32_t*)src->data, (const int32_t*)dst->data, empty(tokens) ? nullptr : (const int32_t*)tokens->data, (int)n,
                                          (int32_t*)shared->data, (cudaStream_t)s);
  return e == cudaSuccess ? QB200_OK : pg_cuda(e, who);
}

QB200_API int qb200_kv_pages_reserve(qb200_tensor* positions, qb200_tensor* copies, qb200_tensor* table, qb200_tensor* lens, qb200_tensor* refs, int page,
                                     const qb200_tensor* rows, const qb200_tensor* counts, qb200_stream s) {
  const char* who = "kv_pages_reserve";
  int st;
  PageState ps;
  if (lens == nullptr || refs == nullptr) return pg_fail(QB200_ERR_BAD_ARG, "%s: lens and refs are needed", who);
  if ((st = parse_state(&ps, who, table, lens, refs, page)) || (st = expect(rows, who, "rows", 1, QB200_INT32))) return st;
  const int64_t n = rows->shape[0];
  if ((st = expect_list(counts, who, "counts", n)) || (st = expect_list(positions, who, "positions", n)) || (st = expect(copies, who, "copies", 2, QB200_INT32))) return st;
  if (copies->shape[0] != n || copies->shape[1] != 2 || (n > 1 && copies->stride[0] != 2))
    return pg_fail(QB200_ERR_BAD_SHAPE, "%s: copies must be a contiguous [%lld, 2]", who, (long long)n);
  if (n > kMaxPageList) return pg_fail(QB200_ERR_UNSUPPORTED, "%s: %lld sequences in one list are not served (at most %d)", who, (long long)n, kMaxPageList);
  if (n == 0) return QB200_OK;
  const cudaError_t e = launch_pages_reserve(ps, (const int32_t*)rows->data, (const int32_t*)counts->data, (int)n, (int32_t*)positions->data, (int32_t*)copies->data,
                                             (cudaStream_t)s);
  return e == cudaSuccess ? QB200_OK : pg_cuda(e, who);
}

QB200_API int qb200_kv_pages_compact(qb200_tensor* remap, qb200_tensor* moves, qb200_tensor* count, qb200_tensor* table, qb200_tensor* refs, qb200_stream s) {
  const char* who = "kv_pages_compact";
  int st;
  PageState ps;
  if (refs == nullptr) return pg_fail(QB200_ERR_BAD_ARG, "%s: refs are needed", who);
  if ((st = parse_state(&ps, who, table, nullptr, refs, 16))) return st;
  if ((st = expect_list(remap, who, "remap", ps.P)) || (st = expect(moves, who, "moves", 2, QB200_INT32)) || (st = expect_list(count, who, "count", 1))) return st;
  if (moves->shape[0] < ps.P / 2 || moves->shape[1] != 2 || (moves->shape[0] > 1 && moves->stride[0] != 2))
    return pg_fail(QB200_ERR_BAD_SHAPE, "%s: moves must be a contiguous [at least %d, 2]", who, ps.P / 2);
  if (moves->data && ((uintptr_t)moves->data & 7)) return pg_fail(QB200_ERR_BAD_STRIDE, "%s: moves must start on 8 bytes", who);
  const cudaError_t e = launch_pages_compact(ps, (int32_t*)remap->data, (int32_t*)moves->data, moves->shape[0], (int32_t*)count->data, (cudaStream_t)s);
  return e == cudaSuccess ? QB200_OK : pg_cuda(e, who);
}

QB200_API int qb200_kv_pages_copy(qb200_tensor* const* pools, int num_pools, const qb200_tensor* pairs, const qb200_tensor* count, qb200_stream s) {
  const char* who = "kv_pages_copy";
  int st;
  if (num_pools < 0 || (num_pools > 0 && pools == nullptr)) return pg_fail(QB200_ERR_BAD_ARG, "%s: null pool list", who);
  if ((st = expect(pairs, who, "pairs", 2, QB200_INT32))) return st;
  if (pairs->shape[1] != 2 || (pairs->shape[0] > 1 && pairs->stride[0] != 2)) return pg_fail(QB200_ERR_BAD_SHAPE, "%s: pairs must be a contiguous [n, 2]", who);
  if (!empty(count) && (st = expect_list(count, who, "count", 1))) return st;
  const int piece = pages_copy_piece();
  const int launches = (num_pools + kMaxCopyPools - 1) / kMaxCopyPools;
  for (int pass = launches > 1 ? 0 : 1; pass < 2; ++pass) {    // every pool is checked before the first launch
    for (int p0 = 0; p0 < num_pools; p0 += kMaxCopyPools) {
      PagesCopyArgs a;
      a.pools = 0;
      uint64_t bits = 0;                       // every address, stride and run, or-ed: what they are all multiples of
      int64_t pieces = 0;
      for (int i = p0; i < num_pools && i < p0 + kMaxCopyPools; ++i) {
        const qb200_tensor* t = pools[i];
        if (t == nullptr || t->ndim < 1) return pg_fail(QB200_ERR_BAD_ARG, "%s: pool %d is no tensor of pages", who, i);
        const int esz = elem_size(t->dtype);
        if (esz == 0) return pg_fail(QB200_ERR_BAD_DTYPE, "%s: pool %d has dtype %d", who, i, t->dtype);
        if ((st = expect(t, who, "pool", t->ndim, t->dtype))) return st;
        if (t->shape[0] != pools[0]->shape[0])
          return pg_fail(QB200_ERR_BAD_SHAPE, "%s: pool %d holds %lld pages, pool 0 %lld", who, i, (long long)t->shape[0], (long long)pools[0]->shape[0]);
        // the page's axes from the innermost stride out, neighbours that follow each other taken as one
        int64_t ext[QB200_MAX_DIMS], str[QB200_MAX_DIMS];
        int nd = 0;
        bool none = false;
        for (int d = 1; d < t->ndim; ++d) {
          none = none || t->shape[d] == 0;
          if (t->shape[d] == 1) continue;
          int at = nd++;
          while (at > 0 && str[at - 1] > t->stride[d]) { str[at] = str[at - 1]; ext[at] = ext[at - 1]; --at; }
          str[at] = t->stride[d]; ext[at] = t->shape[d];
        }
        int64_t run = 1;
        int k = 0;
        while (k < nd && str[k] == run) run *= ext[k++];
        int64_t inner = 1, inner_str = 0, outer = 1, outer_str = 0;
        if (k < nd) {
          inner = ext[k]; inner_str = str[k]; ++k;
          while (k < nd && str[k] == inner * inner_str) inner *= ext[k++];
        }
        if (k < nd) {
          outer = ext[k]; outer_str = str[k]; ++k;
          while (k < nd && str[k] == outer * outer_str) outer *= ext[k++];
        }
        if (k < nd) return pg_fail(QB200_ERR_UNSUPPORTED, "%s: the pages of pool %d lie in more than two levels of strides", who, i);
        if (!distinct(t)) return pg_fail(QB200_ERR_BAD_STRIDE, "%s: pages or rows of pool %d overlap", who, i);
        const int64_t bytes = none ? 0 : run * inner * outer * esz;
        if (bytes > (1ll << 31)) return pg_fail(QB200_ERR_UNSUPPORTED, "%s: pages of %lld bytes are not served", who, (long long)bytes);
        if (bytes == 0) continue;
        PagesCopyPool& p = a.pool[a.pools++];
        p.base = (char*)t->data;
        p.page_str = t->stride[0] * esz; p.outer_str = outer_str * esz; p.inner_str = inner_str * esz;
        p.bytes = (uint32_t)bytes; p.run = (uint32_t)(run * esz); p.inner = (uint32_t)inner;
        p.first_piece = (int)pieces;
        pieces += (bytes + piece - 1) / piece;
        bits |= (uint64_t)(uintptr_t)t->data | (t->shape[0] > 1 ? (uint64_t)p.page_str : 0) | (uint64_t)p.outer_str | (uint64_t)p.inner_str | p.run;
      }
      a.pairs = (const int32_t*)pairs->data;
      a.count = empty(count) ? nullptr : (const int32_t*)count->data;
      a.n = pairs->shape[0]; a.P = num_pools ? pools[0]->shape[0] : 0; a.pieces = (int)pieces;
      if (pass == 0 || a.pools == 0 || a.n == 0 || a.P == 0) continue;
      const int vec = bits % 16 == 0 ? 16 : (bits % 4 == 0 ? 4 : (bits % 2 == 0 ? 2 : 1));
      const cudaError_t e = launch_pages_copy(a, vec, (cudaStream_t)s);
      if (e != cudaSuccess) return pg_cuda(e, who);
    }
  }
  return QB200_OK;
}

QB200_API size_t qb200_kv_pages_decode_attention_workspace_size(int64_t B, int64_t Hq, int64_t Hkv, int64_t D) {
  if (B <= 0 || Hq <= 0 || Hkv <= 0 || (D != 64 && D != 128)) return 0;
  return kv_pages_workspace_bytes(D);
}

QB200_API int qb200_kv_pages_decode_attention(qb200_tensor* res, const qb200_tensor* q, const qb200_tensor* k_q, const qb200_tensor* k_scales,
                                              const qb200_tensor* k_biases, const qb200_tensor* v_q, const qb200_tensor* v_scales, const qb200_tensor* v_biases,
                                              const qb200_tensor* table, const qb200_tensor* rows, const qb200_tensor* lens, int bits, int group_size, float scale,
                                              int64_t window, int64_t sinks, void* workspace, size_t workspace_bytes, qb200_stream s) {
  const char* who = "kv_pages_decode_attention";
  int st;
  if (q == nullptr || q->ndim != 4) return pg_fail(QB200_ERR_BAD_SHAPE, "%s: q must be [B, Hq, 1, D]", who);
  if (q->dtype != QB200_BFLOAT16) return pg_fail(QB200_ERR_UNSUPPORTED, "%s: q must be bf16", who);
  if ((st = expect(q, who, "q", 4, QB200_BFLOAT16)) || (st = expect(res, who, "res", 4, QB200_BFLOAT16))) return st;
  const int64_t B = q->shape[0], Hq = q->shape[1], D = q->shape[3];
  if (q->shape[2] != 1) return pg_fail(QB200_ERR_UNSUPPORTED, "%s: T_q=%lld (only one new token is served)", who, (long long)q->shape[2]);
  for (int d = 0; d < 4; ++d)
    if (res->shape[d] != q->shape[d]) return pg_fail(QB200_ERR_BAD_SHAPE, "%s: res must have q's shape", who);
  if ((st = check_format(who, bits, group_size, D))) return st;
  if (D != 64 && D != 128) return pg_fail(QB200_ERR_UNSUPPORTED, "%s: head dim %lld is not served (64, 128)", who, (long long)D);
  if (k_q == nullptr || k_q->ndim != 4) return pg_fail(QB200_ERR_BAD_SHAPE, "%s: K codes must be [pages, heads, page, cols]", who);
  const int64_t P = k_q->shape[0], Hkv = k_q->shape[1], page = k_q->shape[2];
  if (Hkv <= 0 || Hq % Hkv != 0) return pg_fail(QB200_ERR_BAD_SHAPE, "%s: Hq %lld not a multiple of Hkv %lld", who, (long long)Hq, (long long)Hkv);
  if (page > 65536) return pg_fail(QB200_ERR_UNSUPPORTED, "%s: pages of %lld tokens are not served (a power of two from 16 to 65536)", who, (long long)page);
  PageState ps;
  if ((st = parse_state(&ps, who, table, nullptr, nullptr, (int)page))) return st;
  KvPagesAttnArgs a;
  std::memset(&a, 0, sizeof(a));
  bool vec[2];
  if ((st = parse_pool(&a.pool[0], &vec[0], who, "K", k_q, k_scales, k_biases, bits, P, Hkv, page, D)) ||
      (st = parse_pool(&a.pool[1], &vec[1], who, "V", v_q, v_scales, v_biases, bits, P, Hkv, page, D)))
    return st;
  if ((st = expect_list(lens, who, "lens", ps.S))) return st;
  if (!empty(rows)) {
    if ((st = expect_list(rows, who, "rows", B))) return st;
    a.rows = (const int32_t*)rows->data;
  } else if (ps.S != B) return pg_fail(QB200_ERR_BAD_SHAPE, "%s: %lld queries for a table of %d sequences (pass rows)", who, (long long)B, ps.S);
  if (!(scale >= -3.0e38f && scale <= 3.0e38f)) return pg_fail(QB200_ERR_BAD_ARG, "%s: scale must be finite", who);
  if (window < 0 || sinks < 0) return pg_fail(QB200_ERR_BAD_ARG, "%s: window and sinks must not be negative", who);
  if (!distinct(res)) return pg_fail(QB200_ERR_BAD_STRIDE, "%s: rows of res overlap", who);
  if (B == 0 || Hq == 0) return QB200_OK;
  if (P < 1) return pg_fail(QB200_ERR_BAD_SHAPE, "%s: the pool holds no pages", who);
  if (P > INT32_MAX || B > kMaxPageSeqs) return pg_fail(QB200_ERR_UNSUPPORTED, "%s: %lld sequences are not served (at most %d)", who, (long long)B, kMaxPageSeqs);
  const int64_t gqa = Hq / Hkv, tiles = Hkv * ((gqa + 7) / 8), most = (((int64_t)ps.M << ps.page_shift) + 63) / 64;
  if (Hq > 65536 || B * tiles * most > INT32_MAX)
    return pg_fail(QB200_ERR_UNSUPPORTED, "%s: %lld sequences of %lld heads and up to %lld tokens are too many for one call", who, (long long)B, (long long)Hq,
                   (long long)ps.M << ps.page_shift);
  const size_t need = kv_pages_workspace_bytes(D);
  if (workspace == nullptr || workspace_bytes < need)
    return pg_fail(QB200_ERR_WORKSPACE, "%s: workspace of %zu bytes needed, %zu given", who, need, workspace_bytes);
  if ((uintptr_t)workspace & 15) return pg_fail(QB200_ERR_WORKSPACE, "%s: the workspace must start on 16 bytes", who);
  a.q = q->data; a.out = res->data;
  a.q_vec = ((uintptr_t)q->data & 15) == 0;
  for (int d = 0; d < 2; ++d) {
    a.q_str[d] = q->stride[d]; a.o_str[d] = res->stride[d];
    if (q->shape[d] > 1 && q->stride[d] % 8 != 0) a.q_vec = 0;
  }
  const int64_t esz = bits == 16 ? 2 : 4;
  for (int i = 0; i < 2; ++i) {
    const int64_t pb = a.pool[i].q_str[0] * esz, tb = a.pool[i].q_str[2] * esz;
    if ((P > 1 && pb > UINT32_MAX) || tb > UINT32_MAX) return pg_fail(QB200_ERR_UNSUPPORTED, "%s: pages more than 4 GB apart are not served", who);
    a.page_bytes[i] = (uint32_t)pb; a.tok_bytes[i] = (uint32_t)tb; a.q_head[i] = a.pool[i].q_str[1] * esz;
  }
  a.table = ps.table; a.table_str = ps.table_str;
  a.lens = (const int32_t*)lens->data; a.seqs = ps.S;
  a.B = (int)B; a.Hq = (int)Hq; a.Hkv = (int)Hkv; a.gqa = (int)gqa; a.M = ps.M; a.P = (int)P; a.page_shift = ps.page_shift;
  a.window = (int)(window < INT32_MAX ? window : 0);      // (no sequence is longer: everything is inside)
  a.sinks = (int)(sinks < INT32_MAX ? sinks : INT32_MAX);
  a.bits = bits; a.scale = scale; a.sb_vec = vec[0] && vec[1];
  const cudaError_t e = launch_kv_pages_attn(a, (int)D, workspace, (cudaStream_t)s);
  return e == cudaSuccess ? QB200_OK : pg_cuda(e, who);
}

QB200_API int qb200_window_attention(qb200_tensor* res, const qb200_tensor* q, const qb200_tensor* k, const qb200_tensor* v, float scale, int64_t window,
                                     int64_t sinks, const qb200_tensor* kv_lens, qb200_stream s) {
  const char* who = "window_attention";
  int st;
  const qb200_tensor* const ts[4] = {q, k, v, res};
  const char* const names[4] = {"q", "k", "v", "res"};
  for (int i = 0; i < 4; ++i) {
    if (ts[i] != nullptr && ts[i]->dtype != QB200_BFLOAT16) return pg_fail(QB200_ERR_UNSUPPORTED, "%s: %s must be bf16", who, names[i]);
    if ((st = expect(ts[i], who, names[i], 4, QB200_BFLOAT16))) return st;
  }
  const int64_t B = q->shape[0], Hq = q->shape[1], Tq = q->shape[2], D = q->shape[3], Hkv = k->shape[1], Tk = k->shape[2];
  if (k->shape[0] != B || k->shape[3] != D) return pg_fail(QB200_ERR_BAD_SHAPE, "%s: k must be [B, Hkv, Tk, D] with q's B and D", who);
  for (int d = 0; d < 4; ++d) {
    if (v->shape[d] != k->shape[d]) return pg_fail(QB200_ERR_BAD_SHAPE, "%s: v must have k's shape", who);
    if (res->shape[d] != q->shape[d]) return pg_fail(QB200_ERR_BAD_SHAPE, "%s: res must have q's shape", who);
  }
  if (Hkv <= 0 || Hq % Hkv != 0) return pg_fail(QB200_ERR_BAD_SHAPE, "%s: Hq %lld not a multiple of Hkv %lld", who, (long long)Hq, (long long)Hkv);
  if (D != 64 && D != 128) return pg_fail(QB200_ERR_UNSUPPORTED, "%s: head dim %lld is not served (64, 128)", who, (long long)D);
  if (window < 0 || sinks < 0) return pg_fail(QB200_ERR_BAD_ARG, "%s: window and sinks must not be negative", who);
  if (!(scale > 0.f) || !(scale <= 1.0e38f)) return pg_fail(QB200_ERR_UNSUPPORTED, "%s: scale must be positive and finite", who);
  if (!empty(kv_lens)) {
    if ((st = expect_list(kv_lens, who, "kv_lens", B))) return st;
  } else if (Tk < Tq) return pg_fail(QB200_ERR_BAD_SHAPE, "%s: %lld queries need as many keys (%lld given)", who, (long long)Tq, (long long)Tk);
  if (!distinct(res)) return pg_fail(QB200_ERR_BAD_STRIDE, "%s: rows of res overlap", who);
  if (B == 0 || Hq == 0 || Tq == 0) return QB200_OK;
  if (Tk == 0) return pg_fail(QB200_ERR_BAD_SHAPE, "%s: no keys", who);
  const int64_t lim = (int64_t)1 << 30;
  if (Tq > lim || Tk > lim || B > lim || Hq > lim || B * Hq > lim || ((Tq + 127) / 128) * B * Hq > INT32_MAX)
    return pg_fail(QB200_ERR_UNSUPPORTED, "%s: %lld x %lld heads of %lld queries are too many for one call", who, (long long)B, (long long)Hq, (long long)Tq);
  WindowArgs a;
  std::memset(&a, 0, sizeof(a));
  for (int i = 0; i < 3; ++i) {
    bool ok = ((uintptr_t)ts[i]->data & 15) == 0;
    for (int d = 0; d < 3; ++d) {
      a.str[i][d] = ts[i]->stride[d];
      if (ts[i]->shape[d] > 1) ok = ok && ts[i]->stride[d] % 8 == 0 && ts[i]->stride[d] < ((int64_t)1 << 38);
    }
    if (!ok) return pg_fail(QB200_ERR_UNSUPPORTED, "%s: the rows of %s must start on 16 bytes", who, names[i]);
    if (ts[i]->shape[2] > 1 && ts[i]->stride[2] == 0) return pg_fail(QB200_ERR_UNSUPPORTED, "%s: %s repeats one token", who, names[i]);
  }
  a.o_vec = ((uintptr_t)res->data & 15) == 0;
  for (int d = 0; d < 3; ++d) {
    a.o_str[d] = res->stride[d];
    if (res->shape[d] > 1 && res->stride[d] % 8 != 0) a.o_vec = 0;
  }
  a.q = q->data; a.k = k->data; a.v = v->data; a.out = res->data;
  a.kv_lens = empty(kv_lens) ? nullptr : (const int32_t*)kv_lens->data;
  a.B = B; a.Hq = Hq; a.Hkv = Hkv; a.Tq = Tq; a.Tk = Tk; a.D = D;
  a.window = window >= Tk ? 0 : (int)window;            // (no query has that many keys before it)
  a.sinks = (int)(sinks < Tk ? sinks : Tk);
  a.scale = scale;
  const cudaError_t e = launch_window_attn(a, (cudaStream_t)s);
  return e == cudaSuccess ? QB200_OK : pg_cuda(e, who);
}

}  // extern "C"
