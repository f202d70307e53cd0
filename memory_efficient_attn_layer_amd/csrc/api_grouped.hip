// C ABI of the grouped attention, the paged cache and the attention over it:
// argument checks, workspaces and launch sequences. Contracts: include/mea.h.
#include <math.h>
#include <stdint.h>

#include <initializer_list>

#include "../../include/mea.h"
#include "grouped.h"
#include "launch.h"

namespace {

using namespace mea::kernel_ids;
using mea::bits16;
using mea::timed;

#define MEA_TRY(expr)                                  \
  do {                                                 \
    if ((expr) != hipSuccess) return MEA_ERR_LAUNCH;   \
  } while (0)

size_t align_up(size_t v) { return (v + 255) / 256 * 256; }
bool misaligned(const void* p, size_t a) { return ((uintptr_t)p & (a - 1)) != 0; }

int check16(std::initializer_list<const void*> ps) {
  for (const void* p : ps) {
    if (p == nullptr) return MEA_ERR_NULL;
    if (misaligned(p, 16)) return MEA_ERR_ALIGN;
  }
  return MEA_OK;
}
int check4(std::initializer_list<const void*> ps) {
  for (const void* p : ps) {
    if (p == nullptr) return MEA_ERR_NULL;
    if (misaligned(p, 4)) return MEA_ERR_ALIGN;
  }
  return MEA_OK;
}

bool width_ok(int64_t N) { return N == 32 || N == 64 || N == 128 || N == 256; }
bool dtype_ok(int32_t t) { return t == MEA_BF16 || t == MEA_FP16; }
// (The kernels take log2(e) times it, and its inverse.)
bool scale_ok(float s) { return s >= 0x1p-100f && s <= 0x1p100f; }
// A row stride: a tile's rows are addressed with 32-bit byte offsets.
bool row_stride_ok(int64_t s) { return s % 8 == 0 && s >= 0 && s <= (INT64_C(1) << 24); }
bool stride_ok(int64_t s) { return s % 8 == 0 && s >= 0; }

constexpr int64_t kInt31 = INT64_C(1) << 31;

int check_grouped(const mea_grouped* d) {
  if (d == nullptr) return MEA_ERR_NULL;
  if (!width_ok(d->N)) return MEA_ERR_HEAD_DIM;
  if (d->total < 1 || d->nseq < 1 || d->Hq < 1 || d->Hkv < 1) return MEA_ERR_SHAPE;
  if (d->Hq % d->Hkv != 0) return MEA_ERR_HEADS;
  // Virtual blocks (at most total / 32 + nseq + 2 of them) times heads are the grid.
  if (d->total >= (INT64_C(1) << 30) || d->nseq >= (INT64_C(1) << 24) || d->Hq >= 65536 ||
      (d->total / 32 + d->nseq + 2) * d->Hq >= kInt31)
    return MEA_ERR_SHAPE;
  if (!dtype_ok(d->dtype)) return MEA_ERR_DTYPE;
  if (!scale_ok(d->scale)) return MEA_ERR_SCALE;
  if (!row_stride_ok(d->q_tok) || !row_stride_ok(d->k_tok) || !row_stride_ok(d->v_tok) || !stride_ok(d->q_head) ||
      !stride_ok(d->k_head) || !stride_ok(d->v_head) || d->Hq * d->N > (INT64_C(1) << 24))
    return MEA_ERR_STRIDE;
  return MEA_OK;
}

mea::GroupedParams grouped_params(const mea_grouped* d, const void* q, const void* k, const void* v, const int32_t* cu) {
  mea::GroupedParams p = {};
  p.q = static_cast<const bits16*>(q);
  p.k = static_cast<const bits16*>(k);
  p.v = static_cast<const bits16*>(v);
  p.q_tok = d->q_tok;
  p.q_head = d->q_head;
  p.k_tok = d->k_tok;
  p.k_head = d->k_head;
  p.v_tok = d->v_tok;
  p.v_head = d->v_head;
  p.cu = cu;
  p.nseq = (int)d->nseq;
  p.total = (int)d->total;
  p.Hq = (int)d->Hq;
  p.Hkv = (int)d->Hkv;
  p.scale = d->scale;
  p.sl2e = d->scale * 1.4426950408889634f;
  return p;
}

size_t grouped_delta_bytes(const mea_grouped* d) { return align_up((size_t)(d->total * d->Hq) * sizeof(float)); }

int check_cache(const mea_paged* c) {
  if (c == nullptr) return MEA_ERR_NULL;
  if (!width_ok(c->N)) return MEA_ERR_HEAD_DIM;
  if (c->page < 16 || c->page > 256 || (c->page & (c->page - 1)) != 0) return MEA_ERR_PAGE;
  if (c->seqs < 1 || c->pages < 1 || c->Hkv < 1 || c->max_pages < 1 || c->seqs >= (INT64_C(1) << 20) ||
      c->pages >= (INT64_C(1) << 30) || c->Hkv >= 65536 || c->seqs * c->Hkv >= kInt31 / 256 ||
      c->max_pages * c->page >= (INT64_C(1) << 30))
    return MEA_ERR_SHAPE;
  if (!dtype_ok(c->dtype)) return MEA_ERR_DTYPE;
  const int rc = check16({c->k, c->v});
  return rc != MEA_OK ? rc : check4({c->table, c->lengths, c->refs, c->status});
}

mea::PagedCache cache_of(const mea_paged* c) {
  mea::PagedCache r;
  r.k = static_cast<bits16*>(c->k);
  r.v = static_cast<bits16*>(c->v);
  r.table = c->table;
  r.lengths = c->lengths;
  r.refs = c->refs;
  r.status = c->status;
  r.seqs = (int)c->seqs;
  r.pages = (int)c->pages;
  r.Hkv = (int)c->Hkv;
  r.page = (int)c->page;
  r.lg_page = __builtin_ctz((unsigned)c->page);
  r.N = (int)c->N;
  r.max_pages = (int)c->max_pages;
  return r;
}

// Workspace of the largest of the cache's own calls.
size_t paged_ws(const mea_paged* c) {
  const int S = (int)c->seqs, P = (int)c->pages;
  size_t n = mea::append_ws_ints(S, P);
  const size_t others[3] = {mea::accept_ws_ints(S, P, (int)c->page, mea::kMaxTree),
                            mea::fork_ws_ints(S, (int)c->max_pages), mea::compact_ws_ints(P)};
  for (size_t o : others) n = o > n ? o : n;
  return align_up(n * sizeof(int));
}

mea::TreeGrid tree_grid_of(const mea_paged* c, int64_t n, int64_t Hq) {
  return mea::tree_grid((int)c->seqs, (int)c->Hkv, (int)(n * (Hq / c->Hkv)), (int)(c->max_pages * c->page), (int)c->N);
}

int check_tree(const mea_paged* c, int64_t n, int64_t Hq) {
  const int rc = check_cache(c);
  if (rc != MEA_OK) return rc;
  if (n < 1 || n > mea::kMaxTree || Hq < 1 || Hq >= 65536) return MEA_ERR_SHAPE;
  if (Hq % c->Hkv != 0) return MEA_ERR_HEADS;
  // Grid: items * Hkv by row groups; query rows in the y dimension of the second launch.
  const mea::TreeGrid g = tree_grid_of(c, n, Hq);
  if (n * Hq >= 65536 || g.items * g.row_groups * c->Hkv >= kInt31) return MEA_ERR_SHAPE;
  return MEA_OK;
}

size_t tree_ws(const mea_paged* c, int64_t n, int64_t Hq) {
  const mea::TreeGrid g = tree_grid_of(c, n, Hq);
  return g.split ? align_up((mea::tree_head_floats((int)c->seqs) + (size_t)g.items * n * Hq * (c->N + 4)) * sizeof(float)) : 0;
}

// Checks of a call on the cache with a workspace.
int check_paged_call(const mea_paged* c, const void* ws, size_t ws_bytes) {
  int rc = check_cache(c);
  if (rc != MEA_OK) return rc;
  rc = check16({ws});
  if (rc != MEA_OK) return rc;
  return ws_bytes < paged_ws(c) ? MEA_ERR_WORKSPACE : MEA_OK;
}

}  // namespace

extern "C" {

int mea_grouped_fwd(const mea_grouped* d, const int32_t* cu_seqlens, const void* q, const void* k, const void* v, void* o,
                    void* o_rest, float* lse, void* stream) {
  int rc = check_grouped(d);
  if (rc == MEA_OK) rc = check16({q, k, v, o});
  if (rc == MEA_OK) rc = check4({cu_seqlens});
  if (rc == MEA_OK && (o_rest == nullptr) != (lse == nullptr)) rc = MEA_ERR_NULL;
  if (rc == MEA_OK && lse != nullptr && d->dtype != MEA_BF16) rc = MEA_ERR_DTYPE;
  if (rc == MEA_OK && (misaligned(o_rest, 16) || misaligned(lse, 4))) rc = MEA_ERR_ALIGN;
  if (rc != MEA_OK) return rc;
  mea::GroupedParams p = grouped_params(d, q, k, v, cu_seqlens);
  p.o = static_cast<bits16*>(o);
  p.o_rest = static_cast<bits16*>(o_rest);
  p.lse = lse;
  hipStream_t s = static_cast<hipStream_t>(stream);
  MEA_TRY(timed(K_GROUPED_FWD, s, [&] { return mea::launch_grouped_fwd(p, (int)d->N, d->dtype == MEA_FP16, s); }));
  return MEA_OK;
}

size_t mea_grouped_workspace_bytes(const mea_grouped* d) {
  if (check_grouped(d) != MEA_OK) return 0;
  const size_t parts = (size_t)mea::dkdv_parts((int)d->total, (int)d->nseq, (int)d->Hq, (int)d->Hkv, (int)d->N);
  return grouped_delta_bytes(d) + (parts > 1 ? align_up(parts * 2 * (size_t)(d->total * d->Hkv * d->N) * sizeof(float)) : 0);
}

int mea_grouped_bwd(const mea_grouped* d, const int32_t* cu_seqlens, const void* dout, const void* q, const void* k,
                    const void* v, const void* o, const void* o_rest, const float* lse, void* dq, void* dk, void* dv, void* ws, size_t ws_bytes,
                    void* stream) {
  int rc = check_grouped(d);
  if (rc == MEA_OK && d->dtype != MEA_BF16) rc = MEA_ERR_DTYPE;
  if (rc == MEA_OK) rc = check16({dout, q, k, v, o, o_rest, dq, dk, dv, ws});
  if (rc == MEA_OK) rc = check4({cu_seqlens, lse});
  if (rc != MEA_OK) return rc;
  if (ws_bytes < mea_grouped_workspace_bytes(d)) return MEA_ERR_WORKSPACE;
  mea::GroupedParams p = grouped_params(d, q, k, v, cu_seqlens);
  p.o = const_cast<bits16*>(static_cast<const bits16*>(o));
  p.o_rest = const_cast<bits16*>(static_cast<const bits16*>(o_rest));
  p.dO = static_cast<const bits16*>(dout);
  p.lse_in = lse;
  p.delta = static_cast<float*>(ws);
  p.parts = mea::dkdv_parts(p.total, p.nseq, p.Hq, p.Hkv, (int)d->N);
  p.sums = reinterpret_cast<float*>(static_cast<unsigned char*>(ws) + grouped_delta_bytes(d));
  p.dq = static_cast<bits16*>(dq);
  p.dk = static_cast<bits16*>(dk);
  p.dv = static_cast<bits16*>(dv);
  hipStream_t s = static_cast<hipStream_t>(stream);
  const int N = (int)d->N;
  MEA_TRY(timed(K_GROUPED_DQ, s, [&] { return mea::launch_grouped_dq(p, N, s); }));
  MEA_TRY(timed(K_GROUPED_DKDV, s, [&] { return mea::launch_grouped_dkdv(p, N, s); }));
  if (p.parts > 1) MEA_TRY(timed(K_GROUPED_JOIN, s, [&] { return mea::launch_grouped_join(p, N, s); }));
  return MEA_OK;
}

size_t mea_paged_workspace_bytes(const mea_paged* c) { return check_cache(c) != MEA_OK ? 0 : paged_ws(c); }

int mea_paged_append(const mea_paged* c, const void* k, const void* v, const int64_t* strides, const int32_t* cu_seqlens,
                     int64_t n, int64_t total, void* ws, size_t ws_bytes, void* stream) {
  int rc = check_paged_call(c, ws, ws_bytes);
  if (rc == MEA_OK) rc = check16({k, v});
  if (rc == MEA_OK && strides == nullptr) rc = MEA_ERR_NULL;
  if (rc == MEA_OK && misaligned(cu_seqlens, 4)) rc = MEA_ERR_ALIGN;
  if (rc != MEA_OK) return rc;
  const int64_t rows = cu_seqlens == nullptr ? c->seqs * n : total;
  if (rows < 1 || n < 0 || rows >= (INT64_C(1) << 30) || rows * c->Hkv * (c->N / 8) / 256 + c->seqs * c->Hkv + 1 >= kInt31)
    return MEA_ERR_SHAPE;
  for (int i = 0; i < 6; ++i)
    if (!stride_ok(strides[i])) return MEA_ERR_STRIDE;
  mea::AppendParams p;
  p.c = cache_of(c);
  p.k = static_cast<const bits16*>(k);
  p.v = static_cast<const bits16*>(v);
  p.k_seq = strides[0];
  p.k_tok = strides[1];
  p.k_head = strides[2];
  p.v_seq = strides[3];
  p.v_tok = strides[4];
  p.v_head = strides[5];
  p.cu = cu_seqlens;
  p.n = (int)n;
  p.total = (int)total;
  p.ws = static_cast<int*>(ws);
  hipStream_t s = static_cast<hipStream_t>(stream);
  MEA_TRY(timed(K_APPEND_PLAN, s, [&] { return mea::launch_paged_append_plan(p, s); }));
  MEA_TRY(timed(K_APPEND_ROWS, s, [&] { return mea::launch_paged_append_rows(p, s); }));
  return MEA_OK;
}

int mea_paged_accept(const mea_paged* c, int64_t n, const int32_t* path, int64_t most, const int32_t* counts, void* ws,
                     size_t ws_bytes, void* stream) {
  int rc = check_paged_call(c, ws, ws_bytes);
  if (rc == MEA_OK) rc = check4({path, counts});
  if (rc != MEA_OK) return rc;
  if (n < 1 || n > mea::kMaxTree || most < 1 || most > n) return MEA_ERR_SHAPE;
  mea::AcceptParams p;
  p.c = cache_of(c);
  p.path = path;
  p.counts = counts;
  p.n = (int)n;
  p.most = (int)most;
  p.ws = static_cast<int*>(ws);
  hipStream_t s = static_cast<hipStream_t>(stream);
  MEA_TRY(timed(K_ACCEPT_PLAN, s, [&] { return mea::launch_paged_accept_plan(p, s); }));
  MEA_TRY(timed(K_ACCEPT_ROWS, s, [&] { return mea::launch_paged_accept_rows(p, s); }));
  return MEA_OK;
}

int mea_paged_truncate(const mea_paged* c, const int32_t* lengths, void* stream) {
  int rc = check_cache(c);
  if (rc == MEA_OK) rc = check4({lengths});
  if (rc != MEA_OK) return rc;
  const mea::PagedCache p = cache_of(c);
  hipStream_t s = static_cast<hipStream_t>(stream);
  MEA_TRY(timed(K_TRUNCATE, s, [&] { return mea::launch_paged_truncate(p, lengths, s); }));
  return MEA_OK;
}

int mea_paged_fork(const mea_paged* c, const int32_t* parents, void* ws, size_t ws_bytes, void* stream) {
  int rc = check_paged_call(c, ws, ws_bytes);
  if (rc == MEA_OK) rc = check4({parents});
  if (rc != MEA_OK) return rc;
  const mea::PagedCache p = cache_of(c);
  hipStream_t s = static_cast<hipStream_t>(stream);
  int* w = static_cast<int*>(ws);
  if (mea::paged_fork_small(p)) {
    MEA_TRY(timed(K_FORK, s, [&] { return mea::launch_paged_fork(p, parents, s); }));
    return MEA_OK;
  }
  MEA_TRY(timed(K_FORK_READ, s, [&] { return mea::launch_paged_fork_read(p, parents, w, s); }));
  MEA_TRY(timed(K_FORK_WRITE, s, [&] { return mea::launch_paged_fork_write(p, parents, w, s); }));
  return MEA_OK;
}

int mea_paged_compact(const mea_paged* c, void* ws, size_t ws_bytes, void* stream) {
  const int rc = check_paged_call(c, ws, ws_bytes);
  if (rc != MEA_OK) return rc;
  const mea::PagedCache p = cache_of(c);
  hipStream_t s = static_cast<hipStream_t>(stream);
  int* w = static_cast<int*>(ws);
  MEA_TRY(timed(K_COMPACT_PLAN, s, [&] { return mea::launch_paged_compact_plan(p, w, s); }));
  MEA_TRY(timed(K_COMPACT_MOVE, s, [&] { return mea::launch_paged_compact_move(p, w, s); }));
  return MEA_OK;
}

size_t mea_tree_workspace_bytes(const mea_paged* c, int64_t n, int64_t Hq) {
  return check_tree(c, n, Hq) != MEA_OK ? 0 : tree_ws(c, n, Hq);
}

int mea_tree_attn(const mea_paged* c, int64_t n, int64_t Hq, float scale, const void* q, const int64_t* q_strides,
                  const void* mask, int64_t mask_seq, void* o, void* ws, size_t ws_bytes, void* stream) {
  int rc = check_tree(c, n, Hq);
  if (rc == MEA_OK) rc = check16({q, o});
  if (rc == MEA_OK && q_strides == nullptr) rc = MEA_ERR_NULL;
  if (rc != MEA_OK) return rc;
  if (!scale_ok(scale)) return MEA_ERR_SCALE;
  if (!stride_ok(q_strides[0]) || !stride_ok(q_strides[1]) || !stride_ok(q_strides[2]) || mask_seq < 0) return MEA_ERR_STRIDE;
  const size_t need = tree_ws(c, n, Hq);
  if (need > 0) {
    rc = check16({ws});
    if (rc != MEA_OK) return rc;
    if (ws_bytes < need) return MEA_ERR_WORKSPACE;
  }
  mea::TreeParams p;
  p.c = cache_of(c);
  p.q = static_cast<const bits16*>(q);
  p.q_seq = q_strides[0];
  p.q_tok = q_strides[1];
  p.q_head = q_strides[2];
  p.mask = static_cast<const unsigned char*>(mask);
  p.mask_seq = mask_seq;
  p.n = (int)n;
  p.Hq = (int)Hq;
  const mea::TreeGrid g = tree_grid_of(c, n, Hq);
  p.want = g.want;
  p.least = g.least;
  p.full = g.full;
  p.row_groups = g.row_groups;
  p.sl2e = scale * 1.4426950408889634f;
  p.o = static_cast<bits16*>(o);
  p.part = g.split ? static_cast<float*>(ws) : nullptr;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const bool fp16 = c->dtype == MEA_FP16;
  MEA_TRY(timed(K_TREE_ATTN, s, [&] { return mea::launch_tree_attn(p, fp16, s); }));
  if (g.split) MEA_TRY(timed(K_TREE_COMBINE, s, [&] { return mea::launch_tree_combine(p, fp16, s); }));
  return MEA_OK;
}

}  // extern "C"
