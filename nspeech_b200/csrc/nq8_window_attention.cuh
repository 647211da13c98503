// nq8_window_attention.cuh -- what the window attention kernels share: a
// sequence's rows, the row tile of a CTA, and the keys that a tile sees.
// The kernels start before the one ahead of them has ended, so what it may
// write (rows, lengths, offsets, page tables) is read by plain loads, not by
// the read-only path.
#pragma once

#include "nq8_window_attention.h"

namespace nq {
namespace win {

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// One sequence: its first query row, its queries, first key row (plain rows)
// and keys.
struct Seq {
  int q0, nq, k0, nk;
};
__device__ __forceinline__ void span(const int *off, const int *len, int rows, int seqs, int b, int &begin, int &n) {
  int e;
  if (off) {
    begin = min(max(off[b], 0), rows);
    e = min(max(off[b + 1], begin), rows);
  } else {
    const int each = rows / seqs;
    begin = b * each;
    e = begin + each;
  }
  n = e - begin;
  if (len) n = min(n, max(len[b], 0));
}
__device__ __forceinline__ Seq seq_of(const WinAttnParams &p, int b) {
  Seq s;
  span(p.q_off, p.q_len, p.q_rows, p.seqs, b, s.q0, s.nq);
  if (p.table) {
    s.k0 = 0;
    s.nk = static_cast<int>(min(static_cast<long long>(max(p.k_len[b], 0)),
                                static_cast<long long>(p.max_pages) << p.page_shift));
  } else {
    span(p.k_off, p.k_len, p.k_rows, p.seqs, b, s.k0, s.nk);
  }
  return s;
}
// The row tile `tile` of all sequences' tiles of `rows` rows: sequence and
// first row in it.  Every warp finds it by itself, 32 sequences at a time.
__device__ __forceinline__ bool find_tile(const WinAttnParams &p, int tile, int rows, int &b, int &row0) {
  if (!p.q_off && !p.q_len) {
    const int per = ((p.q_rows / p.seqs) * p.group + rows - 1) / rows;
    b = per ? tile / per : p.seqs;
    row0 = per ? (tile - b * per) * rows : 0;
    return b < p.seqs;
  }
  const int lane = threadIdx.x & 31;
  int done = 0;
  for (int base = 0; base < p.seqs; base += 32) {
    int n = 0;
    if (base + lane < p.seqs) {
      int q0, nq;
      span(p.q_off, p.q_len, p.q_rows, p.seqs, base + lane, q0, nq);
      n = (nq * p.group + rows - 1) / rows;
    }
    int upto = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += x;
    }
    const int all = __shfl_sync(0xffffffffu, upto, 31);
    if (tile < done + all) {
      const unsigned m = __ballot_sync(0xffffffffu, tile < done + upto);
      const int w = __ffs(m) - 1;
      b = base + w;
      row0 = (tile - done - __shfl_sync(0xffffffffu, upto - n, w)) * rows;
      return true;
    }
    done += all;
  }
  return false;
}

// The keys of a row tile: the sinks [0, s_end) and the window [lo, hi].
struct Keys {
  int lo, hi, s_end;  // s_end = 0 where the window's tiles hold the sinks too
  int gap_lo, gap_hi; // then [lo, hi] begins at 0, and no row sees its keys [gap_lo, gap_hi)
  int sink_tiles;
};
template <int KT>
__device__ __forceinline__ Keys keys_of(const WinAttnParams &p, const Seq &s, int i_first, int i_last) {
  Keys k;
  const int p_lo = s.nk - s.nq + i_first, p_hi = s.nk - s.nq + i_last;
  k.hi = p.right >= kWinUnlimited ? s.nk - 1 : min(s.nk - 1, p_hi + p.right);
  k.lo = p.left >= kWinUnlimited ? 0 : max(0, p_lo - p.left);
  k.s_end = max(0, min(min(p.sinks, k.lo), k.hi + 1));
  k.sink_tiles = (k.s_end + KT - 1) / KT;
  k.gap_lo = k.gap_hi = 0;
  if (k.lo <= k.sink_tiles * KT) {  // the two parts touch: one run of tiles
    if (k.s_end > 0) {
      k.gap_lo = k.s_end;
      k.gap_hi = k.lo;
      k.lo = 0;
    }
    k.s_end = 0;
    k.sink_tiles = 0;
  }
  return k;
}
}  // namespace win
}  // namespace nq
