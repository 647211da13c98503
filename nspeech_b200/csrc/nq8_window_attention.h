// nq8_window_attention.h -- launch interface of the sliding-window attention
// kernels (internal): plain rows and the paged cache share them.
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "nq8_common.cuh"

namespace nq {

constexpr int kWinMaxDim = 128;      // largest head dimension
constexpr int kWinUnlimited = 1 << 30;  // left / right without a limit

// o_i = sum_j softmax_j(scale q_i . k_j) v_j over the keys that query i sees.
// Query i of a sequence (of n_q queries and n_k keys) stands at position
// p = n_k - n_q + i and sees key j when 0 <= j < n_k, j <= p + right,
// (j >= p - left or j < sinks), and, in a paged cache, its page exists.
// Without a visible key o_i = 0.
struct WinAttnParams {
  const void *q, *k, *v;
  void *out;
  int64_t q_ts, q_hs, k_ts, k_hs, v_ts, v_hs, o_ts, o_hs;  // token and head strides in elements (k_*, v_*: plain rows only)
  int seqs;
  int q_rows, k_rows;      // rows of q / out and of k, v: offsets are clamped to them
  const int *q_off;        // [seqs + 1], or null: q_rows / seqs rows each
  const int *k_off;        // plain rows: [seqs + 1], or null: k_rows / seqs rows each
  const int *q_len;        // [seqs] or null: only the first q_len[b] rows of a sequence's span
  const int *k_len;        // plain rows: the same for keys; paged: [seqs] tokens in the cache
  int kv_heads, group;     // query heads = kv_heads * group; query head h reads kv head h / group
  int dim;
  int left, right, sinks;  // kWinUnlimited: no limit
  float sl2;               // scale * log2(e)
  // Paged cache (table non-null): k, v point at the layer's pages, each
  // [kv_heads][page_tokens][dim].
  const int *table;        // [seqs][table_ld]
  int table_ld, pages, page_shift, max_pages;
  // Split of a row tile's keys over gridDim.z CTAs: unnormalised outputs,
  // row maxima (log2 units) and sums, joined by a second kernel.
  int splits, split_keys;  // CTAs of a tile's keys, and the keys that each takes at least
  int pair;                // as in WinAttnPlan
  float *part_o;           // [splits][q_rows * query heads][dim padded to 64 or 128]
  float2 *part_ml;         // [splits][q_rows * query heads]
  DevCtl ctl;
};

// What a call runs as; a function of its sizes alone.
struct WinAttnPlan {
  int rows;    // query rows (token, head of a group) of a CTA
  int splits, split_keys;
  int pair;    // tensor-core form: 128-row tiles of a CTA, 1 or 2
  int tiles;   // CTAs along x: an upper bound of the row tiles of all sequences
  size_t workspace;
};
// tensor: the tensor-core form (nq8_window_attention_tc.cu) instead of the
// warp-level ones; win_attn_tc_fits says whether a call's sizes are for it.
// key_bound: keys of a sequence, about.  uniform: every sequence has q_rows / seqs rows.
bool win_attn_tc_fits(int f32, int seqs, int q_rows, int group);
WinAttnPlan win_attn_plan(int sm_count, int f32, bool tensor, bool uniform, int seqs, int q_rows, int64_t key_bound, int kv_heads,
                          int group, int dim, int left, int right, int sinks);
constexpr int kWinTcKeys = 128;  // keys (rows of a box of tm_k, tm_v over plain rows)
// tm_q: box {64, group, 128 / group} over {dim, heads, rows}; tm_k, tm_v: box
// {64, 1, 128} over {dim, kv heads, rows}, or over a layer's pages box
// {64, min(128, page tokens)} over {dim, rows of all pages}; 128-byte swizzle.
cudaError_t launch_win_attn_tc(const CUtensorMap &tm_q, const CUtensorMap &tm_k, const CUtensorMap &tm_v, const WinAttnParams &p,
                               const WinAttnPlan &plan, cudaStream_t stream);
// The splits' join (p.splits > 1), run by both launchers.
cudaError_t launch_win_attn_join(const WinAttnParams &p, int f32, const WinAttnPlan &plan, cudaStream_t stream);
cudaError_t launch_win_attn(const WinAttnParams &p, int f32, const WinAttnPlan &plan, cudaStream_t stream);

}  // namespace nq
