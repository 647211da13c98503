// nq8_decode_api.cu -- the decoding operators of libnq8 (C ABI in
// include/nq8.h): window attention, the paged cache, beam search.
#include <cuda_runtime.h>

#include <cfloat>
#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <string>

#include "../../include/nq8.h"
#include "nq8_cache.h"
#include "nq8_host.h"
#include "nq8_overlap.h"
#include "nq8_window_attention.h"

namespace nq {
// nq8_api.cu, for the current device: its SMs and control block; a tensor map
// of bf16 elements with the 128-byte swizzle (strides in bytes, innermost 1).
int device_info(int *sm_count, DevCtl *ctl);
int tensor_map(CUtensorMap *map, const void *ptr, int rank, const uint64_t *dims, const uint64_t *strides, const uint32_t *box);
}

namespace {

constexpr int kSmCountB200 = 148;

int bad(int code, const char *fmt, ...) {
  char buf[256];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  return nq::api_fail(code, buf);
}
int done(cudaError_t e, const char *what) {
  return e == cudaSuccess ? NQ_OK : bad(NQ_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
}
int elem(int dtype) { return dtype == NQ_F32 ? 4 : 2; }
bool aligned(const void *p, int to) { return reinterpret_cast<uintptr_t>(p) % to == 0; }

struct Heads {
  int q, kv, dim;
};
int check_attention(const char *who, int dtype, int seqs, int64_t q_rows, const Heads &h, int sinks, bool uniform) {
  if (dtype != NQ_F32 && dtype != NQ_BF16) return bad(NQ_ERR_DTYPE, "%s: dtype %d unsupported", who, dtype);
  if (seqs < 0 || q_rows < 0 || sinks < 0) return bad(NQ_ERR_ARG, "%s: negative count", who);
  if (h.q < 1 || h.kv < 1 || h.q % h.kv || h.kv > 65535)
    return bad(NQ_ERR_SHAPE, "%s: %d query heads over %d kv heads", who, h.q, h.kv);
  if (h.dim < 1 || h.dim > nq::kWinMaxDim) return bad(NQ_ERR_SHAPE, "%s: head dim %d (1 to %d)", who, h.dim, nq::kWinMaxDim);
  if (q_rows * (h.q / h.kv) > (1 << 30) || seqs > (1 << 24)) return bad(NQ_ERR_SHAPE, "%s: too many rows", who);
  if (uniform && seqs > 0 && q_rows % seqs)
    return bad(NQ_ERR_SHAPE, "%s: %lld rows are not the same number for each of %d sequences", who, (long long)q_rows, seqs);
  return NQ_OK;
}
int limit(int w) { return w < 0 || w > nq::kWinUnlimited ? nq::kWinUnlimited : w; }
int sms() {
  int n = 0;
  return nq::device_info(&n, nullptr) == NQ_OK ? n : kSmCountB200;
}

int check_cache(const char *who, const nq_cache *c) {
  if (!c || !c->k || !c->v || !c->table || !c->lens || !c->refs || !c->state) return bad(NQ_ERR_ARG, "%s: null argument", who);
  if (c->dtype != NQ_F32 && c->dtype != NQ_BF16) return bad(NQ_ERR_DTYPE, "%s: dtype %d unsupported", who, c->dtype);
  if (c->page_tokens < 8 || c->page_tokens > 1024 || (c->page_tokens & (c->page_tokens - 1)))
    return bad(NQ_ERR_SHAPE, "%s: %d tokens a page (a power of two, 8 to 1024)", who, c->page_tokens);
  if (c->layers < 1 || c->layers > 32767 || c->kv_heads < 1 || c->kv_heads > 65535 || c->head_dim < 1 || c->head_dim > nq::kWinMaxDim)
    return bad(NQ_ERR_SHAPE, "%s: %d layers, %d kv heads of %d", who, c->layers, c->kv_heads, c->head_dim);
  if (c->pages < 1 || c->pages > nq::kCacheMaxPages || c->slots < 1 || c->slots > (1 << 24) || c->max_pages < 1 ||
      static_cast<int64_t>(c->max_pages) * c->page_tokens > (1 << 30))
    return bad(NQ_ERR_SHAPE, "%s: %d pages, %d slots of up to %d pages", who, c->pages, c->slots, c->max_pages);
  if (static_cast<int64_t>(c->page_tokens) * c->kv_heads * c->head_dim > nq::kCacheMaxPageElems)
    return bad(NQ_ERR_SHAPE, "%s: pages of %d tokens, %d kv heads of %d", who, c->page_tokens, c->kv_heads, c->head_dim);
  if (!aligned(c->k, 16) || !aligned(c->v, 16)) return bad(NQ_ERR_ALIGN, "%s: the pages must be 16-byte aligned", who);
  return NQ_OK;
}
int check_slots(const char *who, const nq_cache *c, int first, int n) {
  if (first < 0 || n < 0 || static_cast<int64_t>(first) + n > c->slots)
    return bad(NQ_ERR_SHAPE, "%s: slots [%d, %lld) of %d", who, first, static_cast<long long>(first) + n, c->slots);
  if (n > nq::kCacheMaxCall) return bad(NQ_ERR_SHAPE, "%s: %d slots, at most %d a call", who, n, nq::kCacheMaxCall);
  return NQ_OK;
}
int shift_of(int page_tokens) {
  int s = 0;
  while ((1 << s) < page_tokens) ++s;
  return s;
}
nq::CacheView view(const nq_cache *c) {
  nq::CacheView v;
  v.k = c->k;
  v.v = c->v;
  v.table = c->table;
  v.lens = c->lens;
  v.refs = c->refs;
  v.state = c->state;
  v.size = elem(c->dtype);
  v.layers = c->layers;
  v.pages = c->pages;
  v.page_shift = shift_of(c->page_tokens);
  v.kv_heads = c->kv_heads;
  v.dim = c->head_dim;
  v.slots = c->slots;
  v.max_pages = c->max_pages;
  return v;
}

// Rows that a tensor map takes: 16-byte aligned address and strides (a single
// head or row needs no stride).
struct MapRows {
  const void *ptr;
  int64_t ts, hs;
  int rows, heads;
  bool fits() const {
    return aligned(ptr, 16) && rows > 0 && (heads == 1 || (hs > 0 && hs % 8 == 0)) && (rows == 1 || (ts > 0 && ts % 8 == 0));
  }
  int make(CUtensorMap *m, int dim, int box_heads, int box_rows) const {
    const uint64_t dims[3] = {static_cast<uint64_t>(dim), static_cast<uint64_t>(heads), static_cast<uint64_t>(rows)};
    const uint64_t any = static_cast<uint64_t>(dim) * 2;
    const uint64_t strides[2] = {heads == 1 ? any : static_cast<uint64_t>(hs) * 2, rows == 1 ? any : static_cast<uint64_t>(ts) * 2};
    const uint32_t box[3] = {64, static_cast<uint32_t>(box_heads), static_cast<uint32_t>(box_rows)};
    return nq::tensor_map(m, ptr, 3, dims, strides, box);
  }
};

// The tensor maps of the tensor-core form; *fits: whether the call is one that
// it takes (its sizes, 16-byte alignment, a positive scale: masked scores are
// -inf before the scaling, which must neither turn nor lose them).
int tensor_maps(const nq::WinAttnParams &p, int dtype, CUtensorMap *tq, CUtensorMap *tk, CUtensorMap *tv, bool *fits) {
  *fits = false;
  const int heads = p.kv_heads * p.group;
  const MapRows q{p.q, p.q_ts, p.q_hs, p.q_rows, heads}, out{p.out, p.o_ts, p.o_hs, p.q_rows, heads};
  if (p.dim % 8 || !(p.sl2 >= FLT_MIN) || !nq::win_attn_tc_fits(dtype == NQ_F32, p.seqs, p.q_rows, p.group) || !q.fits() || !out.fits())
    return NQ_OK;
  int rc;
  if (p.table) {
    const int64_t rows = (static_cast<int64_t>(p.pages) * p.kv_heads) << p.page_shift;
    if (rows > INT32_MAX) return NQ_OK;
    const uint64_t dims[2] = {static_cast<uint64_t>(p.dim), static_cast<uint64_t>(rows)}, stride[1] = {static_cast<uint64_t>(p.dim) * 2};
    const uint32_t box[2] = {64, static_cast<uint32_t>(1 << p.page_shift < nq::kWinTcKeys ? 1 << p.page_shift : nq::kWinTcKeys)};
    if ((rc = nq::tensor_map(tk, p.k, 2, dims, stride, box)) || (rc = nq::tensor_map(tv, p.v, 2, dims, stride, box))) return rc;
  } else {
    const MapRows k{p.k, p.k_ts, p.k_hs, p.k_rows, p.kv_heads}, v{p.v, p.v_ts, p.v_hs, p.k_rows, p.kv_heads};
    if (!k.fits() || !v.fits()) return NQ_OK;
    if ((rc = k.make(tk, p.dim, 1, nq::kWinTcKeys)) || (rc = v.make(tv, p.dim, 1, nq::kWinTcKeys))) return rc;
  }
  if ((rc = q.make(tq, p.dim, p.group, 128 / p.group))) return rc;
  *fits = true;
  return NQ_OK;
}

int run_attention(const char *who, nq::WinAttnParams &p, int dtype, int64_t key_bound, void *workspace, int64_t workspace_bytes,
                  void *stream) {
  int sm = 0;
  int rc = nq::device_info(&sm, &p.ctl);
  if (rc) return rc;
  CUtensorMap tq, tk, tv;
  bool tensor = false;
  if ((rc = tensor_maps(p, dtype, &tq, &tk, &tv, &tensor))) return rc;
  const nq::WinAttnPlan pl = nq::win_attn_plan(sm, dtype == NQ_F32, tensor, !p.q_off && !p.q_len, p.seqs, p.q_rows, key_bound,
                                               p.kv_heads, p.group, p.dim, p.left, p.right, p.sinks);
  p.splits = workspace ? pl.splits : 1;
  p.split_keys = pl.split_keys;
  p.pair = pl.pair;
  if (p.splits > 1) {
    if (static_cast<size_t>(workspace_bytes < 0 ? 0 : workspace_bytes) < pl.workspace)
      return bad(NQ_ERR_SHAPE, "%s: a workspace of %lld bytes, %zu are needed", who, (long long)workspace_bytes, pl.workspace);
    if (!aligned(workspace, 16)) return bad(NQ_ERR_ALIGN, "%s: the workspace must be 16-byte aligned", who);
    const int64_t rows = static_cast<int64_t>(pl.splits) * p.q_rows * p.kv_heads * p.group;
    p.part_o = static_cast<float *>(workspace);
    p.part_ml = reinterpret_cast<float2 *>(p.part_o + rows * (p.dim <= 64 ? 64 : 128));
  }
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  return done(tensor ? nq::launch_win_attn_tc(tq, tk, tv, p, pl, s) : nq::launch_win_attn(p, dtype == NQ_F32, pl, s), who);
}

// The larger of the two forms' workspaces: which one runs depends on addresses.
int64_t attention_workspace(int dtype, int seqs, int64_t q_rows, int64_t key_bound, const Heads &h, int left, int right, int sinks) {
  if (seqs == 0 || q_rows == 0) return 0;
  const int sm = sms(), group = h.q / h.kv, n = static_cast<int>(q_rows);
  size_t most = 0;
  for (const bool tensor : {false, true})
    if (!tensor || nq::win_attn_tc_fits(dtype == NQ_F32, seqs, n, group)) {
      const size_t w = nq::win_attn_plan(sm, dtype == NQ_F32, tensor, false, seqs, n, key_bound, h.kv, group, h.dim, limit(left),
                                         limit(right), sinks).workspace;
      most = w > most ? w : most;
    }
  return static_cast<int64_t>(most);
}

}  // namespace

extern "C" {

int64_t nq_window_attention_workspace(int dtype, int seqs, int64_t q_rows, int64_t k_rows, int q_heads, int kv_heads, int head_dim,
                                      int left, int right, int sinks) {
  const Heads h{q_heads, kv_heads, head_dim};
  const int rc = check_attention("nq_window_attention_workspace", dtype, seqs, q_rows, h, sinks, false);
  if (rc) return rc;
  return attention_workspace(dtype, seqs, q_rows, seqs ? k_rows / seqs : 0, h, left, right, sinks);
}

int nq_window_attention(const nq_rows *q, const nq_rows *k, const nq_rows *v, const nq_rows *out, int dtype, int seqs, int64_t q_rows,
                        int64_t k_rows, const int32_t *q_offsets, const int32_t *k_offsets, const int32_t *q_lens,
                        const int32_t *k_lens, int q_heads, int kv_heads, int head_dim, int left, int right, int sinks, float scale,
                        void *workspace, int64_t workspace_bytes, void *stream) {
  const char *who = "nq_window_attention";
  if (!q || !k || !v || !out) return bad(NQ_ERR_ARG, "%s: null argument", who);
  const Heads h{q_heads, kv_heads, head_dim};
  int rc = check_attention(who, dtype, seqs, q_rows, h, sinks, !q_offsets);
  if (rc) return rc;
  if (k_rows < 0 || k_rows > (1 << 30)) return bad(NQ_ERR_SHAPE, "%s: %lld key rows", who, (long long)k_rows);
  if (seqs == 0 || q_rows == 0) return NQ_OK;
  if (!k_offsets && k_rows % seqs)
    return bad(NQ_ERR_SHAPE, "%s: %lld key rows are not the same number for each of %d sequences", who, (long long)k_rows, seqs);
  if (!q->ptr || !out->ptr || (k_rows > 0 && (!k->ptr || !v->ptr))) return bad(NQ_ERR_ARG, "%s: null rows", who);
  for (const nq_rows *r : {q, k, v, out}) {
    if (r->token_stride < 0 || r->head_stride < 0) return bad(NQ_ERR_SHAPE, "%s: negative stride", who);
    if (!aligned(r->ptr, elem(dtype))) return bad(NQ_ERR_ALIGN, "%s: rows must be aligned to their elements", who);
  }
  nq::WinAttnParams p = {};
  p.q = q->ptr;
  p.k = k->ptr;
  p.v = v->ptr;
  p.out = out->ptr;
  p.q_ts = q->token_stride;
  p.q_hs = q->head_stride;
  p.k_ts = k->token_stride;
  p.k_hs = k->head_stride;
  p.v_ts = v->token_stride;
  p.v_hs = v->head_stride;
  p.o_ts = out->token_stride;
  p.o_hs = out->head_stride;
  p.seqs = seqs;
  p.q_rows = static_cast<int>(q_rows);
  p.k_rows = static_cast<int>(k_rows);
  p.q_off = q_offsets;
  p.k_off = k_offsets;
  p.q_len = q_lens;
  p.k_len = k_lens;
  p.kv_heads = kv_heads;
  p.group = q_heads / kv_heads;
  p.dim = head_dim;
  p.left = limit(left);
  p.right = limit(right);
  p.sinks = sinks < nq::kWinUnlimited ? sinks : nq::kWinUnlimited;
  p.sl2 = static_cast<float>(scale * 1.4426950408889634);
  return run_attention(who, p, dtype, k_rows / seqs, workspace, workspace_bytes, stream);
}

int64_t nq_cache_state_ints(int slots, int pages) {
  if (slots < 1 || pages < 1 || pages > nq::kCacheMaxPages) return bad(NQ_ERR_SHAPE, "nq_cache_state_ints: %d slots, %d pages", slots, pages);
  return nq::cache_state_ints(slots, pages);
}

int64_t nq_cache_attention_workspace(const nq_cache *c, int seqs, int64_t q_rows, int q_heads, int left, int right, int sinks) {
  const char *who = "nq_cache_attention_workspace";
  int rc = check_cache(who, c);
  if (rc) return rc;
  const Heads h{q_heads, c->kv_heads, c->head_dim};
  rc = check_attention(who, c->dtype, seqs, q_rows, h, sinks, false);
  if (rc) return rc;
  return attention_workspace(c->dtype, seqs, q_rows, static_cast<int64_t>(c->max_pages) * c->page_tokens, h, left, right, sinks);
}

int nq_cache_attention(const nq_cache *c, int layer, const nq_rows *q, const nq_rows *out, int first, int n, int64_t q_rows,
                       const int32_t *offsets, int q_heads, int left, int right, int sinks, float scale, void *workspace,
                       int64_t workspace_bytes, void *stream) {
  const char *who = "nq_cache_attention";
  int rc = check_cache(who, c);
  if (rc) return rc;
  if (!q || !out) return bad(NQ_ERR_ARG, "%s: null argument", who);
  if (first < 0 || n < 0 || static_cast<int64_t>(first) + n > c->slots)
    return bad(NQ_ERR_SHAPE, "%s: slots [%d, %lld) of %d", who, first, static_cast<long long>(first) + n, c->slots);
  if (layer < 0 || layer >= c->layers) return bad(NQ_ERR_SHAPE, "%s: layer %d of %d", who, layer, c->layers);
  const Heads h{q_heads, c->kv_heads, c->head_dim};
  rc = check_attention(who, c->dtype, n, q_rows, h, sinks, !offsets);
  if (rc) return rc;
  if (n == 0 || q_rows == 0) return NQ_OK;
  if (!q->ptr || !out->ptr) return bad(NQ_ERR_ARG, "%s: null rows", who);
  for (const nq_rows *r : {q, out}) {
    if (r->token_stride < 0 || r->head_stride < 0) return bad(NQ_ERR_SHAPE, "%s: negative stride", who);
    if (!aligned(r->ptr, elem(c->dtype))) return bad(NQ_ERR_ALIGN, "%s: rows must be aligned to their elements", who);
  }
  const int64_t layer_bytes = static_cast<int64_t>(layer) * c->pages * c->page_tokens * c->kv_heads * c->head_dim * elem(c->dtype);
  nq::WinAttnParams p = {};
  p.q = q->ptr;
  p.k = static_cast<const char *>(c->k) + layer_bytes;
  p.v = static_cast<const char *>(c->v) + layer_bytes;
  p.out = out->ptr;
  p.q_ts = q->token_stride;
  p.q_hs = q->head_stride;
  p.o_ts = out->token_stride;
  p.o_hs = out->head_stride;
  p.seqs = n;
  p.q_rows = static_cast<int>(q_rows);
  p.q_off = offsets;
  p.k_len = c->lens + first;
  p.kv_heads = c->kv_heads;
  p.group = q_heads / c->kv_heads;
  p.dim = c->head_dim;
  p.left = limit(left);
  p.right = limit(right);
  p.sinks = sinks < nq::kWinUnlimited ? sinks : nq::kWinUnlimited;
  p.sl2 = static_cast<float>(scale * 1.4426950408889634);
  p.table = c->table + static_cast<int64_t>(first) * c->max_pages;
  p.table_ld = c->max_pages;
  p.pages = c->pages;
  p.page_shift = shift_of(c->page_tokens);
  p.max_pages = c->max_pages;
  return run_attention(who, p, c->dtype, static_cast<int64_t>(c->max_pages) * c->page_tokens, workspace, workspace_bytes, stream);
}

int nq_cache_reserve(const nq_cache *c, int first, int n, const int32_t *offsets, int tokens, void *stream) {
  const char *who = "nq_cache_reserve";
  int rc = check_cache(who, c);
  if (rc || (rc = check_slots(who, c, first, n))) return rc;
  if (!offsets && (tokens < 0 || tokens > (1 << 30))) return bad(NQ_ERR_ARG, "%s: %d tokens", who, tokens);
  int sm = 0;
  if ((rc = nq::device_info(&sm, nullptr)) || n == 0) return rc;
  return done(nq::launch_cache_reserve(view(c), offsets, tokens, first, n, static_cast<cudaStream_t>(stream)), who);
}

int nq_cache_write(const nq_cache *c, const nq_rows *k, const nq_rows *v, int64_t k_layer_stride, int64_t v_layer_stride, int layer,
                   int layers, int64_t rows, int first, int n, const int32_t *offsets, int tokens, void *stream) {
  const char *who = "nq_cache_write";
  int rc = check_cache(who, c);
  if (rc || (rc = check_slots(who, c, first, n))) return rc;
  if (!k || !v) return bad(NQ_ERR_ARG, "%s: null argument", who);
  if (layer < 0 || layers < 0 || static_cast<int64_t>(layer) + layers > c->layers)
    return bad(NQ_ERR_SHAPE, "%s: layers [%d, %lld) of %d", who, layer, static_cast<long long>(layer) + layers, c->layers);
  if (rows < 0 || rows > (1 << 30)) return bad(NQ_ERR_SHAPE, "%s: %lld rows", who, (long long)rows);
  if (!offsets && (tokens < 0 || static_cast<int64_t>(tokens) * n != rows))
    return bad(NQ_ERR_SHAPE, "%s: %lld rows for %d slots of %d tokens", who, (long long)rows, n, tokens);
  int sm = 0;
  if ((rc = nq::device_info(&sm, nullptr)) || n == 0 || rows == 0 || layers == 0) return rc;
  if (!k->ptr || !v->ptr) return bad(NQ_ERR_ARG, "%s: null rows", who);
  const int64_t ls[2] = {k_layer_stride, v_layer_stride};
  const nq_rows *side[2] = {k, v};
  for (int i = 0; i < 2; ++i) {
    if (side[i]->token_stride < 0 || side[i]->head_stride < 0 || ls[i] < 0) return bad(NQ_ERR_SHAPE, "%s: negative stride", who);
    if (!aligned(side[i]->ptr, elem(c->dtype))) return bad(NQ_ERR_ALIGN, "%s: rows must be aligned to their elements", who);
  }
  return done(nq::launch_cache_write(view(c), k->ptr, v->ptr, k->token_stride, k->head_stride, k_layer_stride, v->token_stride,
                                     v->head_stride, v_layer_stride, layer, layers, static_cast<int>(rows), offsets, tokens, first, n,
                                     static_cast<cudaStream_t>(stream)),
              who);
}

int nq_cache_fork(const nq_cache *c, int first, int n, const int32_t *src, void *stream) {
  const char *who = "nq_cache_fork";
  int rc = check_cache(who, c);
  if (rc || (rc = check_slots(who, c, first, n))) return rc;
  int sm = 0;
  if ((rc = nq::device_info(&sm, nullptr)) || n == 0) return rc;
  return done(nq::launch_cache_fork(view(c), src, first, n, static_cast<cudaStream_t>(stream)), who);
}

int nq_cache_trim(const nq_cache *c, int first, int n, int sinks, int window, void *stream) {
  const char *who = "nq_cache_trim";
  int rc = check_cache(who, c);
  if (rc || (rc = check_slots(who, c, first, n))) return rc;
  if (sinks < 0 || window < 0) return bad(NQ_ERR_ARG, "%s: %d sinks, a window of %d", who, sinks, window);
  int sm = 0;
  if ((rc = nq::device_info(&sm, nullptr)) || n == 0) return rc;
  return done(nq::launch_cache_trim(view(c), first, n, sinks, window, static_cast<cudaStream_t>(stream)), who);
}

int nq_cache_compact(const nq_cache *c, void *stream) {
  const char *who = "nq_cache_compact";
  int rc = check_cache(who, c);
  if (rc) return rc;
  int sm = 0;
  if ((rc = nq::device_info(&sm, nullptr))) return rc;
  return done(nq::launch_cache_compact(view(c), sm, static_cast<cudaStream_t>(stream)), who);
}

int nq_cache_status(const nq_cache *c, int *bits, void *stream) {
  const char *who = "nq_cache_status";
  int rc = check_cache(who, c);
  if (rc) return rc;
  int sm = 0, v = 0;
  if ((rc = nq::device_info(&sm, nullptr))) return rc;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaError_t e = cudaMemcpyAsync(&v, c->state, sizeof(int), cudaMemcpyDeviceToHost, s);
  if (e == cudaSuccess) e = cudaStreamSynchronize(s);
  if (e == cudaSuccess && v) e = cudaMemsetAsync(c->state, 0, sizeof(int), s);
  if (e != cudaSuccess) return done(e, who);
  if (bits) *bits = v;
  if (!v) return NQ_OK;
  return bad(NQ_ERR_CACHE, "cache status 0x%x:%s%s%s%s", v, v & NQ_CACHE_OUT_OF_PAGES ? " no free pages left" : "",
             v & NQ_CACHE_SLOT_FULL ? " a slot has no room for its tokens" : "", v & NQ_CACHE_BAD_INDEX ? " a slot or a page that is not there" : "",
             v & NQ_CACHE_SHARED_PAGE ? " a write to a page that other slots hold" : "");
}

int64_t nq_beam_workspace(int items, int beams, int64_t vocab) {
  if (items < 0 || beams < 1 || beams > nq::kBeamMax || vocab < 1 || vocab > (1 << 30) || static_cast<int64_t>(items) * beams > 65535)
    return bad(NQ_ERR_SHAPE, "nq_beam_workspace: %d items of %d beams over %lld tokens", items, beams, (long long)vocab);
  const int rows = items * beams;
  return static_cast<int64_t>(nq::beam_workspace(rows, beams, nq::beam_splits(sms(), rows, static_cast<int>(vocab))));
}

int nq_beam_select(const void *logits, int dtype, int64_t ld, int items, int beams, int64_t vocab, const float *scores,
                   const uint8_t *finished, int eos, float *out_scores, int32_t *out_parents, int32_t *out_tokens,
                   uint8_t *out_finished, void *workspace, int64_t workspace_bytes, void *stream) {
  const char *who = "nq_beam_select";
  if (dtype != NQ_F32 && dtype != NQ_BF16) return bad(NQ_ERR_DTYPE, "%s: dtype %d unsupported", who, dtype);
  const int64_t need = nq_beam_workspace(items, beams, vocab);
  if (need < 0) return static_cast<int>(need);
  if (ld < vocab) return bad(NQ_ERR_SHAPE, "%s: rows of %lld logits, %lld apart", who, (long long)vocab, (long long)ld);
  int sm = 0;
  const int rc = nq::device_info(&sm, nullptr);
  if (rc || items == 0) return rc;
  if (!logits || !scores || !out_scores || !out_parents || !out_tokens || !workspace) return bad(NQ_ERR_ARG, "%s: null argument", who);
  if (workspace_bytes < need) return bad(NQ_ERR_SHAPE, "%s: a workspace of %lld bytes, %lld are needed", who, (long long)workspace_bytes, (long long)need);
  if (!aligned(workspace, 8) || !aligned(logits, elem(dtype))) return bad(NQ_ERR_ALIGN, "%s: misaligned logits or workspace", who);
  nq::BeamParams p = {};
  const int rows = items * beams;
  p.logits = logits;
  p.ld = ld;
  p.bf16 = dtype == NQ_BF16;
  p.items = items;
  p.beams = beams;
  p.vocab = static_cast<int>(vocab);
  p.scores = scores;
  p.finished = finished;
  p.eos = eos;
  p.out_scores = out_scores;
  p.out_parents = out_parents;
  p.out_tokens = out_tokens;
  p.out_finished = out_finished;
  p.splits = nq::beam_splits(sm, rows, static_cast<int>(vocab));
  const int64_t parts = static_cast<int64_t>(rows) * p.splits;
  p.part_keys = static_cast<unsigned long long *>(workspace);
  p.part_sum = reinterpret_cast<double *>(p.part_keys + parts * beams);
  p.part_max = reinterpret_cast<float *>(p.part_sum + parts);
  return done(nq::launch_beam_select(p, static_cast<cudaStream_t>(stream)), who);
}

int nq_beam_reorder(const void *const *src, void *const *dst, const int64_t *row_bytes, const int64_t *src_stride,
                    const int64_t *dst_stride, int count, int rows, const int32_t *parents, void *stream) {
  const char *who = "nq_beam_reorder";
  if (count < 0 || count > nq::kReorderMax) return bad(NQ_ERR_SHAPE, "%s: %d states, at most %d a call", who, count, nq::kReorderMax);
  if (rows < 0 || rows > nq::kReorderMaxRows) return bad(NQ_ERR_SHAPE, "%s: %d rows, at most %d", who, rows, nq::kReorderMaxRows);
  if (count == 0 || rows == 0) return NQ_OK;
  if (!src || !dst || !row_bytes || !src_stride || !dst_stride || !parents) return bad(NQ_ERR_ARG, "%s: null argument", who);
  nq::ReorderParams p = {};
  int64_t strips = 0;
  for (int i = 0; i < count; ++i) {
    if (row_bytes[i] < 1) return bad(NQ_ERR_SHAPE, "%s: rows of %lld bytes", who, (long long)row_bytes[i]);
    if (!src[i] || !dst[i]) return bad(NQ_ERR_ARG, "%s: null state", who);
    if (rows > 1 && (src_stride[i] < row_bytes[i] || dst_stride[i] < row_bytes[i]))
      return bad(NQ_ERR_SHAPE, "%s: rows of %lld bytes overlap", who, (long long)row_bytes[i]);
    strips += row_bytes[i] / 16 + 1;
    p.src[i] = src[i];
    p.dst[i] = dst[i];
    p.row_bytes[i] = row_bytes[i];
    p.src_ld[i] = src_stride[i];
    p.dst_ld[i] = dst_stride[i];
  }
  if (strips > (1LL << 30)) return bad(NQ_ERR_SHAPE, "%s: rows too long", who);
  if (nq::reorder_overlaps(src, dst, row_bytes, src_stride, dst_stride, count, rows))
    return bad(NQ_ERR_ARG, "%s: an output overlaps another state", who);
  int sm = 0;
  const int rc = nq::device_info(&sm, nullptr);
  if (rc) return rc;
  p.count = count;
  p.rows = rows;
  p.parents = parents;
  return done(nq::launch_beam_reorder(p, static_cast<cudaStream_t>(stream)), who);
}

}  // extern "C"
