// nq8_cache.h -- launch interfaces of the paged cache and of beam search
// (internal).
#pragma once

#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "nq8_common.cuh"

namespace nq {

// A cache's device state (nq_cache of include/nq8.h).  `state` holds the
// status bits, counts and lists below; its size is cache_state_ints().
struct CacheView {
  void *k, *v;     // [layers][pages][kv_heads][page_tokens][dim]
  int *table;      // [slots][max_pages], -1: no page
  int *lens;       // [slots]
  int *refs;       // [pages] slots that hold the page; 0: free
  int *state;
  int size;        // bytes of an element
  int layers, pages, page_shift, kv_heads, dim, slots, max_pages;
};
constexpr int kCacheOutOfPages = 1, kCacheSlotFull = 2, kCacheBadIndex = 4, kCacheSharedPage = 8;
constexpr int kCacheMaxCall = 4096;       // slots of one call
constexpr int kCacheMaxPages = 1 << 20;
constexpr int kCacheMaxPageElems = 1 << 28;  // of a page in one layer: a copy's units are counted in 32 bits
// state[0] status bits, [1] live pages after a compaction, [2] entries of the
// copy list; then the copy list (page from, page to, rows) per slot, and three
// lists of `pages` entries.
constexpr int kStateStatus = 0, kStateLive = 1, kStateCopies = 2, kStateLists = 16;
__host__ __device__ inline int64_t cache_state_ints(int slots, int pages) {
  return kStateLists + 3 * static_cast<int64_t>(slots) + 3 * static_cast<int64_t>(pages);
}

cudaError_t launch_cache_reserve(const CacheView &c, const int *offsets, int uniform, int first, int n, cudaStream_t s);
cudaError_t launch_cache_write(const CacheView &c, const void *k, const void *v, int64_t ts, int64_t hs, int64_t ls, int64_t v_ts,
                               int64_t v_hs, int64_t v_ls, int layer, int layers, int rows, const int *offsets, int uniform,
                               int first, int n, cudaStream_t s);
cudaError_t launch_cache_fork(const CacheView &c, const int *src, int first, int n, cudaStream_t s);
cudaError_t launch_cache_trim(const CacheView &c, int first, int n, int sinks, int window, cudaStream_t s);
cudaError_t launch_cache_compact(const CacheView &c, int sm_count, cudaStream_t s);

// ---- beam search (nq8_beam.cu)
constexpr int kBeamMax = 32;
struct BeamParams {
  const void *logits;      // [items * beams] rows of ld elements
  int64_t ld;
  int bf16;
  int items, beams;
  int vocab;
  const float *scores;     // [items * beams]
  const uint8_t *finished; // [items * beams] or null
  int eos;
  float *out_scores;       // [items * beams]
  int *out_parents, *out_tokens;
  uint8_t *out_finished;   // or null
  int splits;              // CTAs of a row
  unsigned long long *part_keys;  // [rows][splits][beams]
  double *part_sum;        // [rows][splits]
  float *part_max;         // [rows][splits]
};
int beam_splits(int sm_count, int rows, int vocab);
size_t beam_workspace(int rows, int beams, int splits);
cudaError_t launch_beam_select(const BeamParams &p, cudaStream_t s);

constexpr int kReorderMax = 16;  // states of one call
struct ReorderParams {
  const void *src[kReorderMax];
  void *dst[kReorderMax];
  int64_t row_bytes[kReorderMax];
  int64_t src_ld[kReorderMax], dst_ld[kReorderMax];  // bytes
  int strip0[kReorderMax + 1];  // first strip of each state
  int count, rows, strip_bytes;
  const int *parents;
};
constexpr int kReorderMaxRows = 12288;
cudaError_t launch_beam_reorder(ReorderParams &p, cudaStream_t s);

}  // namespace nq
