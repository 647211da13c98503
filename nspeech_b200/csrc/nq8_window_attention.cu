// nq8_window_attention.cu -- softmax attention through a sliding window whose
// first tokens ("sinks") stay visible, over plain rows or a paged cache.
//
// Work item: a tile of R query rows of one kv head.  The rows of a tile are
// (token, head of the group) pairs, token-major, so the heads that share keys
// read them once, and a tile spans few positions, hence few keys outside the
// window.  The tile's keys are the sinks [0, s) and the window [lo, hi] of all
// its rows; they are walked in 64-key (bf16) or 32-key (f32) tiles with the
// running maximum and sum of the softmax (f32, log2 units), one pass.
//
// bf16: scores and P V by warp-level MMA (m16n8k16, f32 accumulators), P
// rounded to bf16 as the MMA's operand.  Few rows (a decoder's token): the
// four warps take different keys of each tile and join at the end, so a step
// streams K and V at the rate of memory instead of idling three warps.
// f32: products as three tf32 products, or by FMA for single tokens.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include "nq8_window_attention.cuh"

namespace nq {
namespace {

using namespace win;

constexpr int kThreads = 128;

// 16-byte copy global -> shared; zeros where !there (src is not read).
__device__ __forceinline__ void cp16(uint32_t dst, const void *src, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t a) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(a)
               : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t a) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(a)
               : "memory");
}

// The keys that a row tile sees, one after the other: the sinks [0, s_end),
// then the window from lo on.  Tiles are cut from this list, so a few sinks
// cost no tile of their own.
struct KeyList {
  int lo, s_end, n;
  int tiles;
  __device__ __forceinline__ int key(int u) const { return u < s_end ? u : u - s_end + lo; }
};
template <int KT>
__device__ __forceinline__ KeyList list_of(const WinAttnParams &p, const Seq &s, int i_first, int i_last) {
  const Keys k = keys_of<1>(p, s, i_first, i_last);
  KeyList l{k.lo, k.s_end, k.s_end + max(0, k.hi - k.lo + 1), 0};
  l.tiles = (l.n + KT - 1) / KT;
  return l;
}
// Tiles of a list that one of its `splits` CTAs takes: an equal share, but not
// less than split_keys, so that short sequences take fewer CTAs.
template <int KT>
__device__ __forceinline__ int share_of(const WinAttnParams &p, int tiles) {
  return max((tiles + p.splits - 1) / p.splits, p.split_keys / KT);
}
// Whether every row between positions pos_lo and pos_hi sees all of the list's
// entries [u, u + KT).
template <int KT>
__device__ __forceinline__ bool all_see(const WinAttnParams &p, const Seq &s, const KeyList &k, int u, int pos_lo, int pos_hi) {
  const int j = k.key(u);
  return u >= k.s_end && u + KT <= k.n && j + KT - 1 <= (p.right >= kWinUnlimited ? s.nk - 1 : min(s.nk - 1, pos_lo + p.right)) &&
         (p.left >= kWinUnlimited || j >= pos_hi - p.left);
}
// Whether a row at position `at` sees the list's entry u.
__device__ __forceinline__ bool sees(const WinAttnParams &p, const KeyList &k, int u, int at) {
  const int j = k.key(u);
  return u < k.n && (p.right >= kWinUnlimited || j <= at + p.right) && (p.left >= kWinUnlimited || j >= at - p.left || j < p.sinks);
}

// The same for the list's entries [u, u + 32) as bits.
__device__ __forceinline__ uint32_t bits_between(int lo, int hi) {  // bits lo..hi, any integers
  lo = max(lo, 0);
  hi = min(hi, 31);
  return hi < lo ? 0u : (0xffffffffu >> (31 - hi)) & (0xffffffffu << lo);
}
__device__ __forceinline__ uint32_t row_bits(const WinAttnParams &p, const KeyList &k, int u, int at) {
  const int shift = k.s_end - k.lo - u;  // of a window key's bit
  const int last = k.n - 1 - u;
  const int hi = p.right >= kWinUnlimited ? last : min(last, max(at + p.right, -1) + shift);
  const int lo = p.left >= kWinUnlimited ? k.s_end - u : max(at - p.left, k.lo) + shift;
  // first keys: entries of their own, or the window's first where it begins at key 0
  const int first = k.s_end ? k.s_end : k.lo ? 0 : p.sinks;
  const int first_hi = min(p.right >= kWinUnlimited ? first - 1 : min(first - 1, at + p.right), k.n - 1) - u;
  return bits_between(lo, hi) | bits_between(-u, first_hi);
}

// Element offset of the row of entry u for kv head h; -1 past the list's end
// and where the key's page is missing (the row reads as zeros).
template <bool PAGED>
__device__ __forceinline__ int64_t key_row(const WinAttnParams &p, const KeyList &k, const Seq &s, const int *table, int h, int u, bool v) {
  if (u >= k.n) return -1;
  const int j = k.key(u);
  if constexpr (PAGED) {
    const int pg = table[j >> p.page_shift];
    if (pg < 0 || pg >= p.pages) return -1;
    const int r = j & ((1 << p.page_shift) - 1);
    return (((static_cast<int64_t>(pg) * p.kv_heads + h) << p.page_shift) + r) * p.dim;
  } else {
    return v ? (s.k0 + static_cast<int64_t>(j)) * p.v_ts + h * p.v_hs : (s.k0 + static_cast<int64_t>(j)) * p.k_ts + h * p.k_hs;
  }
}

// Joins the splits' partial results of one row tile, in split order.
template <typename T, int DP>
__global__ void __launch_bounds__(kThreads) win_attn_join(const __grid_constant__ WinAttnParams p, int rows) {
  pdl_wait();
  pdl_trigger();
  int b, row0;
  if (!find_tile(p, blockIdx.x, rows, b, row0)) return;
  const Seq s = seq_of(p, b);
  const int h = blockIdx.y, heads = p.kv_heads * p.group;
  const int64_t all = static_cast<int64_t>(p.q_rows) * heads;
  constexpr int kLanes = DP / 4, kRowsAtOnce = kThreads / kLanes;
  const int c = (threadIdx.x % kLanes) * 4;
  for (int r = row0 + threadIdx.x / kLanes; r < min(row0 + rows, s.nq * p.group); r += kRowsAtOnce) {
    const int i = r / p.group, hq = h * p.group + r % p.group;
    const int64_t row = static_cast<int64_t>(s.q0 + i) * heads + hq;
    float m = -INFINITY;
    for (int z = 0; z < p.splits; ++z) m = fmaxf(m, p.part_ml[z * all + row].x);
    float l = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int z = 0; z < p.splits; ++z) {
      const float2 ml = p.part_ml[z * all + row];
      if (ml.x == -INFINITY) {
        l += ml.y;  // 0, or NaN where the scores are
        continue;
      }
      const float f = ex2(ml.x - m);
      const float4 x = *reinterpret_cast<const float4 *>(p.part_o + (z * all + row) * DP + c);
      l += ml.y * f;
      o.x += x.x * f;
      o.y += x.y * f;
      o.z += x.z * f;
      o.w += x.w * f;
    }
    const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
    T *out = static_cast<T *>(p.out) + (s.q0 + static_cast<int64_t>(i)) * p.o_ts + hq * p.o_hs;
    const float e[4] = {o.x * inv, o.y * inv, o.z * inv, o.w * inv};
#pragma unroll
    for (int x = 0; x < 4; ++x)
      if (c + x < p.dim) out[c + x] = T(e[x]);
  }
}

// ---------------------------------------------------------------------- bf16
// WR warps along the rows (16 each), WK = 4 / WR along the keys of a tile.
template <int DP, int R, int STAGES>
struct MmaSmem {
  static constexpr int kKT = 64;
  static constexpr int kTileBytes = kKT * DP * 2;
  static constexpr int kRing = STAGES + 1;  // row offsets and holes are made one tile ahead of the copies
  static constexpr int kOffK = 0;
  static constexpr int kOffV = STAGES * kTileBytes;
  static constexpr int kOffQ = 2 * STAGES * kTileBytes;
  static constexpr int kOffRow = kOffQ + (R * DP * 2 > 512 ? R * DP * 2 : 512);  // the join's 64 maxima and sums lie there too
  static constexpr int kOffHole = kOffRow + kRing * kKT * 8;
  static constexpr int kBytes = kOffHole + kRing * 8;
};

template <int DP, int WR, int STAGES, bool PAGED, bool VEC>
__global__ void __launch_bounds__(kThreads) win_attn_mma(const __grid_constant__ WinAttnParams p) {
  using L = MmaSmem<DP, 16 * WR, STAGES>;
  constexpr int KT = L::kKT, WK = 4 / WR, KW = KT / WK, R = 16 * WR, CH = DP / 8;
  static_assert(4 * 16 * (DP + 4) * 4 <= 2 * STAGES * L::kTileBytes, "the warps' join fits the key tiles");
  extern __shared__ __align__(128) uint8_t smem[];
  const uint32_t sb = smem_u32(smem);
  int64_t *row_off = reinterpret_cast<int64_t *>(smem + L::kOffRow);
  uint32_t *holes = reinterpret_cast<uint32_t *>(smem + L::kOffHole);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  pdl_wait();
  pdl_trigger();
  int b, row0;
  // later tiles of a causal sequence see more keys: they go first
  if (!find_tile(p, gridDim.x - 1 - blockIdx.x, R, b, row0)) return;
  const Seq s = seq_of(p, b);
  const int h = blockIdx.y, G = p.group;
  const int n_rows = s.nq * G;
  const int r_last = min(row0 + R, n_rows) - 1;
  const KeyList k = list_of<KT>(p, s, row0 / G, r_last / G);
  const int share = share_of<KT>(p, k.tiles), t0 = min(static_cast<int>(blockIdx.z) * share, k.tiles), t1 = min(t0 + share, k.tiles);
  const int nt = t1 - t0;
  const int *table = PAGED ? p.table + static_cast<int64_t>(b) * p.table_ld : nullptr;
  const __nv_bfloat16 *kp = static_cast<const __nv_bfloat16 *>(p.k), *vp = static_cast<const __nv_bfloat16 *>(p.v);

  // Row offsets of tile t (and its holes: keys whose page is missing).
  auto rows_of_tile = [&](int t) {
    if constexpr (PAGED) {
      if (warp < 2 && t < nt) {
        const int slot = t % L::kRing;
        const int j = (t0 + t) * KT + tid;
        const int64_t o = key_row<true>(p, k, s, table, h, j, false);
        row_off[slot * KT + tid] = o;
        const unsigned m = __ballot_sync(0xffffffffu, o < 0);
        if (lane == 0) holes[slot * 2 + warp] = m;
      }
    }
  };
  auto copy_row = [&](uint32_t dst, const __nv_bfloat16 *src, bool there, int c) {
    if constexpr (VEC) {
      cp16(dst, src + 8 * c, there && 8 * c < p.dim);
    } else {
      uint32_t w[4];
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const int e = 8 * c + 2 * x;
        const __nv_bfloat16 z = __float2bfloat16_rn(0.f);
        const __nv_bfloat16 a = there && e < p.dim ? src[e] : z, d = there && e + 1 < p.dim ? src[e + 1] : z;
        __nv_bfloat162 y(a, d);
        w[x] = *reinterpret_cast<uint32_t *>(&y);
      }
      asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(dst), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]) : "memory");
    }
  };
  auto sw = [](int row, int c) { return static_cast<uint32_t>(row * (DP * 2) + ((c ^ (row & 7)) << 4)); };
  auto load_tile = [&](int t) {
    if (t < nt) {
      const int st = t % STAGES, slot = t % L::kRing, base = (t0 + t) * KT;
      const uint32_t ks = sb + L::kOffK + st * L::kTileBytes, vs = sb + L::kOffV + st * L::kTileBytes;
      const int c = tid % CH;
#pragma unroll
      for (int r = tid / CH; r < KT; r += kThreads / CH) {
        int64_t ok, ov;
        if constexpr (PAGED) {
          ok = ov = row_off[slot * KT + r];
        } else {
          ok = key_row<false>(p, k, s, nullptr, h, base + r, false);
          ov = ok < 0 ? -1 : key_row<false>(p, k, s, nullptr, h, base + r, true);
        }
        copy_row(ks + sw(r, c), kp + (ok < 0 ? 0 : ok), ok >= 0, c);
        copy_row(vs + sw(r, c), vp + (ov < 0 ? 0 : ov), ov >= 0, c);
      }
    }
    cp_commit();
  };

  // Q tile.
  const __nv_bfloat16 *qp = static_cast<const __nv_bfloat16 *>(p.q);
  for (int x = tid; x < R * CH; x += kThreads) {
    const int r = x / CH, c = x % CH, rr = row0 + r;
    const bool there = rr < n_rows;
    const int i = there ? rr / G : 0, g = there ? rr - i * G : 0;
    copy_row(sb + L::kOffQ + sw(r, c), qp + (there ? (s.q0 + static_cast<int64_t>(i)) * p.q_ts + (h * G + g) * p.q_hs : 0), there, c);
  }
#pragma unroll
  for (int t = 0; t < STAGES; ++t) rows_of_tile(t);
  __syncthreads();
#pragma unroll
  for (int t = 0; t < STAGES - 1; ++t) load_tile(t);  // the first group holds Q too

  const int wr = warp % WR, wk = warp / WR;
  const int qr = lane >> 2;  // this thread's rows of the warp's 16: qr and qr + 8
  int pos[2];                // their positions
#pragma unroll
  for (int x = 0; x < 2; ++x) pos[x] = s.nk - s.nq + min(row0 + 16 * wr + qr + 8 * x, n_rows - 1) / G;
  const int pos_lo = s.nk - s.nq + row0 / G, pos_hi = s.nk - s.nq + r_last / G;
  uint32_t qf[DP / 16][4];
  float o[DP / 8][4];
#pragma unroll
  for (int d = 0; d < DP / 8; ++d)
#pragma unroll
    for (int e = 0; e < 4; ++e) o[d][e] = 0.f;
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};

  for (int t = 0; t < nt; ++t) {
    cp_wait<STAGES - 2>();
    if constexpr (!VEC) asm volatile("" ::: "memory");
    __syncthreads();
    if (t == 0) {
      const int r = 16 * wr + (lane & 7) + ((lane >> 3) & 1) * 8;
#pragma unroll
      for (int kk = 0; kk < DP / 16; ++kk) ldsm4(qf[kk], sb + L::kOffQ + sw(r, 2 * kk + (lane >> 4)));
    }
    load_tile(t + STAGES - 1);
    rows_of_tile(t + STAGES);
    const int st = t % STAGES, slot = t % L::kRing, base = (t0 + t) * KT;
    const uint32_t ks = sb + L::kOffK + st * L::kTileBytes, vs = sb + L::kOffV + st * L::kTileBytes;
    float sc[KW / 8][4];
#pragma unroll
    for (int n = 0; n < KW / 8; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) sc[n][e] = 0.f;
    {
      const int r = wk * KW + (lane & 7) + ((lane >> 4) << 3), c = (lane >> 3) & 1;
#pragma unroll
      for (int kk = 0; kk < DP / 16; ++kk)
#pragma unroll
        for (int n = 0; n < KW / 16; ++n) {
          uint32_t f[4];
          ldsm4(f, ks + sw(r + 16 * n, 2 * kk + c));
          mma_16816_bf16(sc[2 * n], qf[kk], f[0], f[1]);
          mma_16816_bf16(sc[2 * n + 1], qf[kk], f[2], f[3]);
        }
    }
    uint32_t hole[2] = {0u, 0u};
    if constexpr (PAGED) {
      hole[0] = holes[slot * 2];
      hole[1] = holes[slot * 2 + 1];
    }
    const bool inside = all_see<KT>(p, s, k, base, pos_lo, pos_hi) && !(hole[0] | hole[1]);
    float top[2] = {-INFINITY, -INFINITY};
    if (inside) {
#pragma unroll
      for (int n = 0; n < KW / 8; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          sc[n][e] *= p.sl2;
          top[e >> 1] = fmaxf(top[e >> 1], sc[n][e]);
        }
    } else {
      constexpr int kWords = (KW + 31) / 32;  // of this warp's keys
      uint32_t see[2][kWords];
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int w = 0; w < kWords; ++w) {
          const int u = wk * KW + 32 * w;
          see[x][w] = row_bits(p, k, base + u, pos[x]) & ~(hole[u >> 5] >> (u & 31));
        }
#pragma unroll
      for (int n = 0; n < KW / 8; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const bool on = see[e >> 1][8 * n / 32] >> (8 * n % 32 + 2 * (lane & 3) + (e & 1)) & 1u;
          sc[n][e] = on ? sc[n][e] * p.sl2 : -INFINITY;
          top[e >> 1] = fmaxf(top[e >> 1], sc[n][e]);
        }
    }
    float ref[2];
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      top[x] = fmaxf(top[x], __shfl_xor_sync(0xffffffffu, top[x], 1));
      top[x] = fmaxf(top[x], __shfl_xor_sync(0xffffffffu, top[x], 2));
      top[x] = fmaxf(top[x], m[x]);
      ref[x] = top[x] == -INFINITY ? 0.f : top[x];
      const float f = ex2(m[x] - ref[x]);
      l[x] *= f;
      m[x] = top[x];
#pragma unroll
      for (int d = 0; d < DP / 8; ++d) {
        o[d][2 * x] *= f;
        o[d][2 * x + 1] *= f;
      }
    }
    uint32_t pf[KW / 8][2];
#pragma unroll
    for (int n = 0; n < KW / 8; ++n)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const float a = ex2(sc[n][2 * x] - ref[x]), c = ex2(sc[n][2 * x + 1] - ref[x]);
        l[x] += a + c;
        pf[n][x] = pack_bf16x2(a, c);
      }
    {
      const int r = wk * KW + (lane & 7) + ((lane >> 3) & 1) * 8, c = lane >> 4;
#pragma unroll
      for (int n = 0; n < KW / 16; ++n) {
        const uint32_t a[4] = {pf[2 * n][0], pf[2 * n][1], pf[2 * n + 1][0], pf[2 * n + 1][1]};
#pragma unroll
        for (int d = 0; d < DP / 16; ++d) {
          uint32_t f[4];
          ldsm4t(f, vs + sw(r + 16 * n, 2 * d + c));
          mma_16816_bf16(o[2 * d], a, f[0], f[1]);
          mma_16816_bf16(o[2 * d + 1], a, f[2], f[3]);
        }
      }
    }
  }
  cp_wait<0>();
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    l[x] += __shfl_xor_sync(0xffffffffu, l[x], 1);
    l[x] += __shfl_xor_sync(0xffffffffu, l[x], 2);
  }
  const int heads = p.kv_heads * G;
  const int64_t all = static_cast<int64_t>(p.q_rows) * heads;
  __nv_bfloat16 *outp = static_cast<__nv_bfloat16 *>(p.out);
  if constexpr (WK == 1) {
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const int r = row0 + 16 * wr + qr + 8 * x;
      if (r >= n_rows) continue;
      const int i = r / G, hq = h * G + r % G;
      if (p.splits > 1) {
        const int64_t row = blockIdx.z * all + static_cast<int64_t>(s.q0 + i) * heads + hq;
        if ((lane & 3) == 0) p.part_ml[row] = make_float2(m[x], l[x]);
#pragma unroll
        for (int d = 0; d < DP / 8; ++d)
          *reinterpret_cast<float2 *>(p.part_o + row * DP + 8 * d + 2 * (lane & 3)) = make_float2(o[d][2 * x], o[d][2 * x + 1]);
      } else {
        const float inv = l[x] > 0.f ? 1.f / l[x] : (l[x] == 0.f ? 0.f : l[x]);
        __nv_bfloat16 *out = outp + (s.q0 + static_cast<int64_t>(i)) * p.o_ts + hq * p.o_hs;
#pragma unroll
        for (int d = 0; d < DP / 8; ++d) {
          const int c = 8 * d + 2 * (lane & 3);
          if constexpr (VEC) {
            if (c < p.dim) *reinterpret_cast<uint32_t *>(out + c) = pack_bf16x2(o[d][2 * x] * inv, o[d][2 * x + 1] * inv);
          } else {
            if (c < p.dim) out[c] = __float2bfloat16_rn(o[d][2 * x] * inv);
            if (c + 1 < p.dim) out[c + 1] = __float2bfloat16_rn(o[d][2 * x + 1] * inv);
          }
        }
      }
    }
  } else {
    // Join the WK warps of each 16 rows through shared memory.
    constexpr int P = DP + 4;
    __syncthreads();
    float *jo = reinterpret_cast<float *>(smem);                        // [4 warps][16][P]
    float2 *jml = reinterpret_cast<float2 *>(smem + L::kOffQ);          // [4 warps][16]
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const int r = 16 * warp + qr + 8 * x;
      if ((lane & 3) == 0) jml[r] = make_float2(m[x], l[x]);
#pragma unroll
      for (int d = 0; d < DP / 8; ++d)
        *reinterpret_cast<float2 *>(jo + r * P + 8 * d + 2 * (lane & 3)) = make_float2(o[d][2 * x], o[d][2 * x + 1]);
    }
    __syncthreads();
    constexpr int kPer = kThreads / R;        // threads of a row
    const int r = tid / kPer, rr = row0 + r;  // r < R
    if (rr < n_rows) {
      const int w0 = r / 16;                  // warp w0 + WR x holds the row's part x
      float mm = -INFINITY, ll = 0.f, f[WK];
#pragma unroll
      for (int x = 0; x < WK; ++x) mm = fmaxf(mm, jml[16 * (w0 + WR * x) + r % 16].x);
#pragma unroll
      for (int x = 0; x < WK; ++x) {
        const float2 ml = jml[16 * (w0 + WR * x) + r % 16];
        f[x] = ml.x == -INFINITY ? 0.f : ex2(ml.x - mm);
        ll += ml.y * f[x];
      }
      const int i = rr / G, hq = h * G + rr % G;
      const float inv = ll > 0.f ? 1.f / ll : (ll == 0.f ? 0.f : ll);
      const int64_t row = blockIdx.z * all + static_cast<int64_t>(s.q0 + i) * heads + hq;
      __nv_bfloat16 *out = outp + (s.q0 + static_cast<int64_t>(i)) * p.o_ts + hq * p.o_hs;
      if (p.splits > 1 && tid % kPer == 0) p.part_ml[row] = make_float2(mm, ll);
#pragma unroll
      for (int c = (tid % kPer) * 4; c < DP; c += kPer * 4) {
        float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int x = 0; x < WK; ++x) {
          if (f[x] == 0.f) continue;  // a part without a visible key
          const float4 y = *reinterpret_cast<const float4 *>(jo + (16 * (w0 + WR * x) + r % 16) * P + c);
          v[0] += y.x * f[x];
          v[1] += y.y * f[x];
          v[2] += y.z * f[x];
          v[3] += y.w * f[x];
        }
        if (p.splits > 1) {
          *reinterpret_cast<float4 *>(p.part_o + row * DP + c) = make_float4(v[0], v[1], v[2], v[3]);
        } else if constexpr (VEC) {
          if (c < p.dim)
            *reinterpret_cast<uint2 *>(out + c) = make_uint2(pack_bf16x2(v[0] * inv, v[1] * inv), pack_bf16x2(v[2] * inv, v[3] * inv));
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (c + e < p.dim) out[c + e] = __float2bfloat16_rn(v[e] * inv);
        }
      }
    }
  }
}

// ----------------------------------------------------------------------- f32
// Tile form, on the tensor cores: a product of two f32 as three tf32 products,
// x y = xh yh + xh yl + xl yh with xh = x rounded to tf32 (11 bits) and xl =
// x - xh (exact, taken at 11 bits): 2^-20 of |x y| at most is lost, 2^-22 on
// the mean.  The tensor cores add with truncation, so their sums are kept
// short: the large and the small products apart, and an output's sum over the
// 32 keys of a tile is added to the running one in f32.  Bound by issue slots:
// the parts' splitting (three instructions an element, in every warp) and the
// warp-level MMAs (0.27 PFLOP/s of tf32, a third of it for f32 products).  32
// segments of up to 1501 tokens, 10 heads of 64, window 64 + 16: 307 us; the
// same tiles by FMA 544 us, bound by shared memory (128-bit loads of operands
// that 16 products each use); two row tiles a warp, which share the parts of
// keys and values but leave two CTAs an SM, 400 us.  NARROW: heads of at most
// DP - 8 skip the columns of zeros (4 x 1000 tokens, 10 heads of 40, causal: 158 -> 116
// us); the test costs full ones 3 to 8 %, so they go without it.
template <int DP>
struct F32Smem {
  static constexpr int kKT = 32, kP = DP + 4;  // pitch: rows 16 bytes apart in the banks
  static constexpr int kTileBytes = kKT * kP * 4;
  static constexpr int kOffK = 0;
  static constexpr int kOffV = 2 * kTileBytes;
  static constexpr int kOffQ = 4 * kTileBytes;
  static constexpr int kOffRow = kOffQ + 64 * kP * 4;
  static constexpr int kBytes = kOffRow + 3 * kKT * 8;
};

template <bool VEC>
__device__ __forceinline__ void copy4(float *dst, const float *src, bool there, int c, int dim) {
  if constexpr (VEC) {
    cp16(smem_u32(dst), src + c, there && c < dim);
  } else {
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
    if (there) {
      if (c < dim) x.x = src[c];
      if (c + 1 < dim) x.y = src[c + 1];
      if (c + 2 < dim) x.z = src[c + 2];
      if (c + 3 < dim) x.w = src[c + 3];
    }
    *reinterpret_cast<float4 *>(dst) = x;
  }
}
__device__ __forceinline__ void mma_tf32(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void split_tf32(uint32_t x, uint32_t &hi, uint32_t &lo) {
  hi = (x + 0x1000u) & 0xffffe000u;  // to nearest
  lo = __float_as_uint(__uint_as_float(x) - __uint_as_float(hi));
}

template <int DP, int WR, bool PAGED, bool VEC, bool NARROW>
__global__ void __launch_bounds__(kThreads) win_attn_tf32(const __grid_constant__ WinAttnParams p) {
  using L = F32Smem<DP>;
  constexpr int KT = L::kKT, WK = 4 / WR, KW = KT / WK, R = 16 * WR, P = L::kP, CH = DP / 4;
  extern __shared__ __align__(128) uint8_t smem[];
  const uint32_t sb = smem_u32(smem);
  int64_t *row_off = reinterpret_cast<int64_t *>(smem + L::kOffRow);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  pdl_wait();
  pdl_trigger();
  int b, row0;
  if (!find_tile(p, gridDim.x - 1 - blockIdx.x, R, b, row0)) return;
  const Seq s = seq_of(p, b);
  const int h = blockIdx.y, G = p.group, n_rows = s.nq * G, r_last = min(row0 + R, n_rows) - 1;
  const KeyList k = list_of<KT>(p, s, row0 / G, r_last / G);
  const int share = share_of<KT>(p, k.tiles), t0 = min(static_cast<int>(blockIdx.z) * share, k.tiles), nt = min(share, k.tiles - t0);
  const int *table = PAGED ? p.table + static_cast<int64_t>(b) * p.table_ld : nullptr;
  const float *kp = static_cast<const float *>(p.k), *vp = static_cast<const float *>(p.v), *qp = static_cast<const float *>(p.q);
  auto rows_of_tile = [&](int t) {
    if (PAGED && tid < KT && t < nt) row_off[(t % 3) * KT + tid] = key_row<true>(p, k, s, table, h, (t0 + t) * KT + tid, false);
  };
  auto load_tile = [&](int t) {
    if (t < nt) {
      float *ks = reinterpret_cast<float *>(smem + L::kOffK) + (t & 1) * KT * P;
      float *vs = reinterpret_cast<float *>(smem + L::kOffV) + (t & 1) * KT * P;
      const int c = (tid % CH) * 4, base = (t0 + t) * KT;
#pragma unroll
      for (int r = tid / CH; r < KT; r += kThreads / CH) {
        int64_t ok, ov;
        if constexpr (PAGED) {
          ok = ov = row_off[(t % 3) * KT + r];
        } else {
          ok = key_row<false>(p, k, s, nullptr, h, base + r, false);
          ov = ok < 0 ? -1 : key_row<false>(p, k, s, nullptr, h, base + r, true);
        }
        copy4<VEC>(ks + r * P + c, kp + (ok < 0 ? 0 : ok), ok >= 0, c, p.dim);
        copy4<VEC>(vs + r * P + c, vp + (ov < 0 ? 0 : ov), ov >= 0, c, p.dim);
      }
    }
    cp_commit();
  };
  float *qs = reinterpret_cast<float *>(smem + L::kOffQ);
  for (int x = tid; x < R * CH; x += kThreads) {
    const int r = x / CH, c = (x % CH) * 4, rr = row0 + r;
    const bool there = rr < n_rows;
    const int i = there ? rr / G : 0, g = there ? rr - i * G : 0;
    copy4<VEC>(qs + r * P + c, qp + (there ? (s.q0 + static_cast<int64_t>(i)) * p.q_ts + (h * G + g) * p.q_hs : 0), there, c, p.dim);
  }
  rows_of_tile(0);
  rows_of_tile(1);
  __syncthreads();
  load_tile(0);
  const int wr = warp % WR, wk = warp / WR;
  const int qr = lane >> 2, qc = lane & 3;  // this thread's rows qr, qr + 8 of the warp's 16
  int pos[2];
#pragma unroll
  for (int x = 0; x < 2; ++x) pos[x] = s.nk - s.nq + min(row0 + 16 * wr + qr + 8 * x, n_rows - 1) / G;
  const int pos_lo = s.nk - s.nq + row0 / G, pos_hi = s.nk - s.nq + r_last / G;
  float o[DP / 8][4];
#pragma unroll
  for (int d = 0; d < DP / 8; ++d)
#pragma unroll
    for (int e = 0; e < 4; ++e) o[d][e] = 0.f;
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
  const uint32_t q_at = sb + L::kOffQ + ((16 * wr + (lane & 7) + ((lane >> 3) & 1) * 8) * P + (lane >> 4) * 4) * 4;
  for (int t = 0; t < nt; ++t) {
    load_tile(t + 1);
    cp_wait<1>();
    __syncthreads();
    rows_of_tile(t + 2);
    const uint32_t ks = sb + L::kOffK + (t & 1) * L::kTileBytes;
    const float *vs = reinterpret_cast<const float *>(smem + L::kOffV) + (t & 1) * KT * P;
    const int base = (t0 + t) * KT;
    // Scores: KW / 8 tiles of 8 keys.
    constexpr int N = KW / 8;
    float hi[N][4], lo[N][4];
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) hi[n][e] = lo[n][e] = 0.f;
    auto products = [&](int n, const uint32_t (&ah)[4], const uint32_t (&al)[4], uint32_t x0, uint32_t x1) {
      uint32_t h0, l0, h1, l1;
      split_tf32(x0, h0, l0);
      split_tf32(x1, h1, l1);
      mma_tf32(hi[n], ah, h0, h1);
      mma_tf32(lo[n], ah, l0, l1);
      mma_tf32(lo[n], al, h0, h1);
    };
    if constexpr (N >= 2) {
      const uint32_t k_at = ks + ((wk * KW + (lane & 7) + ((lane >> 4) << 3)) * P + ((lane >> 3) & 1) * 4) * 4;
#pragma unroll
      for (int kk = 0; kk < DP / 8; ++kk) {
        if (NARROW && 8 * kk >= p.dim) break;
        uint32_t a[4], ah[4], al[4];
        ldsm4(a, q_at + kk * 32);
#pragma unroll
        for (int e = 0; e < 4; ++e) split_tf32(a[e], ah[e], al[e]);
#pragma unroll
        for (int n = 0; n < N; n += 2) {
          uint32_t f[4];
          ldsm4(f, k_at + n * 8 * P * 4 + kk * 32);
          products(n, ah, al, f[0], f[1]);
          products(n + 1, ah, al, f[2], f[3]);
        }
      }
    } else {
      const uint32_t k_at = ks + ((wk * KW + (lane & 7)) * P + (lane >> 3) * 4) * 4;
#pragma unroll
      for (int kk = 0; kk < DP / 8; kk += 2) {
        if (NARROW && 8 * kk >= p.dim) break;
        uint32_t f[4];
        ldsm4(f, k_at + kk * 32);
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          uint32_t a[4], ah[4], al[4];
          ldsm4(a, q_at + (kk + x) * 32);
#pragma unroll
          for (int e = 0; e < 4; ++e) split_tf32(a[e], ah[e], al[e]);
          products(0, ah, al, f[2 * x], f[2 * x + 1]);
        }
      }
    }
    const bool inside = all_see<KT>(p, s, k, base, pos_lo, pos_hi);
    uint32_t see[2] = {0xffffffffu, 0xffffffffu}, gone = 0;  // gone: entries whose page is missing
    if constexpr (PAGED) gone = __ballot_sync(0xffffffffu, row_off[(t % 3) * KT + lane] < 0);
    if (!inside || gone) {
#pragma unroll
      for (int x = 0; x < 2; ++x) see[x] = row_bits(p, k, base, pos[x]) & ~gone;
    }
    float top[2] = {m[0], m[1]};
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float x = (hi[n][e] + lo[n][e]) * p.sl2;
        hi[n][e] = see[e >> 1] >> (wk * KW + 8 * n + 2 * qc + (e & 1)) & 1u ? x : -INFINITY;
        top[e >> 1] = fmaxf(top[e >> 1], hi[n][e]);
      }
    float ref[2], f[2];
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      top[x] = fmaxf(top[x], __shfl_xor_sync(0xffffffffu, top[x], 1));
      top[x] = fmaxf(top[x], __shfl_xor_sync(0xffffffffu, top[x], 2));
      ref[x] = top[x] == -INFINITY ? 0.f : top[x];
      f[x] = ex2(m[x] - ref[x]);
      l[x] *= f[x];
      m[x] = top[x];
    }
    // Weights as the A operand: this thread's keys 2 qc and 2 qc + 1 stand in
    // columns qc and qc + 4, for V alike.
    uint32_t ah[N][4], al[N][4];
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float w = ex2(hi[n][e] - ref[e >> 1]);
        l[e >> 1] += w;
        constexpr int to[4] = {0, 2, 1, 3};
        split_tf32(__float_as_uint(w), ah[n][to[e]], al[n][to[e]]);
      }
#pragma unroll
    for (int d = 0; d < DP / 8; ++d) {
      if (NARROW && 8 * d >= p.dim) break;
      float big[4] = {0.f, 0.f, 0.f, 0.f}, small[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int n = 0; n < N; ++n) {
        const float *v = vs + (wk * KW + 8 * n + 2 * qc) * P + 8 * d + qr;
        uint32_t h0, l0, h1, l1;
        split_tf32(__float_as_uint(v[0]), h0, l0);
        split_tf32(__float_as_uint(v[P]), h1, l1);
        mma_tf32(big, ah[n], h0, h1);
        mma_tf32(small, ah[n], l0, l1);
        mma_tf32(small, al[n], h0, h1);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) o[d][e] = fmaf(o[d][e], f[e >> 1], big[e] + small[e]);
    }
    __syncthreads();
  }
  cp_wait<0>();
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    l[x] += __shfl_xor_sync(0xffffffffu, l[x], 1);
    l[x] += __shfl_xor_sync(0xffffffffu, l[x], 2);
  }
  const int heads = p.kv_heads * G;
  const int64_t all = static_cast<int64_t>(p.q_rows) * heads;
  float *outp = static_cast<float *>(p.out);
  if constexpr (WK == 1) {
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const int r = row0 + 16 * wr + qr + 8 * x;
      if (r >= n_rows) continue;
      const int i = r / G, hq = h * G + r % G;
      const int64_t row = blockIdx.z * all + static_cast<int64_t>(s.q0 + i) * heads + hq;
      if (p.splits > 1 && qc == 0) p.part_ml[row] = make_float2(m[x], l[x]);
      const float inv = p.splits > 1 ? 1.f : l[x] > 0.f ? 1.f / l[x] : (l[x] == 0.f ? 0.f : l[x]);
      float *out = p.splits > 1 ? p.part_o + row * DP : outp + (s.q0 + static_cast<int64_t>(i)) * p.o_ts + hq * p.o_hs;
      const int width = p.splits > 1 ? DP : p.dim;
#pragma unroll
      for (int d = 0; d < DP / 8; ++d) {
        const int c = 8 * d + 2 * qc;
        if constexpr (VEC) {
          if (c < width) *reinterpret_cast<float2 *>(out + c) = make_float2(o[d][2 * x] * inv, o[d][2 * x + 1] * inv);
        } else {
          if (c < width) out[c] = o[d][2 * x] * inv;
          if (c + 1 < width) out[c + 1] = o[d][2 * x + 1] * inv;
        }
      }
    }
  } else {
    // Join the WK warps of each 16 rows through shared memory.
    float *jo = reinterpret_cast<float *>(smem);                // [4 warps][16][P]
    float2 *jml = reinterpret_cast<float2 *>(smem + L::kOffQ);  // [4 warps][16]
    static_assert(64 * P * 4 <= L::kOffQ, "the warps' join fits the key tiles");
    __syncthreads();
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const int r = 16 * warp + qr + 8 * x;
      if (qc == 0) jml[r] = make_float2(m[x], l[x]);
#pragma unroll
      for (int d = 0; d < DP / 8; ++d) *reinterpret_cast<float2 *>(jo + r * P + 8 * d + 2 * qc) = make_float2(o[d][2 * x], o[d][2 * x + 1]);
    }
    __syncthreads();
    constexpr int kPer = kThreads / R;
    const int r = tid / kPer, rr = row0 + r;
    if (rr < n_rows) {
      const int w0 = r / 16;
      float mm = -INFINITY, ll = 0.f, f[WK];
#pragma unroll
      for (int x = 0; x < WK; ++x) mm = fmaxf(mm, jml[16 * (w0 + WR * x) + r % 16].x);
#pragma unroll
      for (int x = 0; x < WK; ++x) {
        const float2 ml = jml[16 * (w0 + WR * x) + r % 16];
        f[x] = ml.x == -INFINITY ? 0.f : ex2(ml.x - mm);
        ll += ml.y * f[x];
      }
      const int i = rr / G, hq = h * G + rr % G;
      const int64_t row = blockIdx.z * all + static_cast<int64_t>(s.q0 + i) * heads + hq;
      if (p.splits > 1 && tid % kPer == 0) p.part_ml[row] = make_float2(mm, ll);
      const float inv = p.splits > 1 ? 1.f : ll > 0.f ? 1.f / ll : (ll == 0.f ? 0.f : ll);
      float *out = p.splits > 1 ? p.part_o + row * DP : outp + (s.q0 + static_cast<int64_t>(i)) * p.o_ts + hq * p.o_hs;
      const int width = p.splits > 1 ? DP : p.dim;
      for (int c = tid % kPer; c < width; c += kPer) {
        float v = 0.f;
#pragma unroll
        for (int x = 0; x < WK; ++x)
          if (f[x] != 0.f) v = fmaf(jo[(16 * (w0 + WR * x) + r % 16) * P + c], f[x], v);  // 0: a part without a visible key
        out[c] = v * inv;
      }
    }
  }
}

// Row form, for a decoder's single tokens: at most R (1, 2, 4) rows share a
// key, and a warp takes 8 loads of 32 / (DP / 4) keys at a time straight from
// memory (lane: four columns), K and V together, so that 32 KB of a CTA are in
// flight; the four warps and the keys' lane groups join at the end.  Bound by
// latency: a few rounds of dependent loads (length, page, key) a piece, then the
// join.  16 sequences of up to 5000 tokens, 10 heads of 64, window 1023: 27 us,
// 3.1 TB/s of the keys and values read.
template <int DP, int R, bool PAGED, bool VEC>
__global__ void __launch_bounds__(kThreads) win_attn_f32_rows(const __grid_constant__ WinAttnParams p) {
  constexpr int LPK = DP / 4, KPL = 32 / LPK, U = 8, KT = U * KPL;
  __shared__ float4 jo[4][R][32];
  __shared__ float2 jml[4][R][KPL];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, sub = lane / LPK, c = (lane % LPK) * 4;
  pdl_wait();
  pdl_trigger();
  int b, row0;
  if (!find_tile(p, gridDim.x - 1 - blockIdx.x, R, b, row0)) return;
  const Seq s = seq_of(p, b);
  const int h = blockIdx.y, G = p.group, n_rows = s.nq * G, r_last = min(row0 + R, n_rows) - 1;
  const KeyList k = list_of<KT>(p, s, row0 / G, r_last / G);
  const int share = share_of<KT>(p, k.tiles), t0 = min(static_cast<int>(blockIdx.z) * share, k.tiles), t1 = min(t0 + share, k.tiles);
  const int *table = PAGED ? p.table + static_cast<int64_t>(b) * p.table_ld : nullptr;
  const float *kp = static_cast<const float *>(p.k), *vp = static_cast<const float *>(p.v), *qp = static_cast<const float *>(p.q);
  auto fetch = [&](const float *src, bool there) {
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
    if constexpr (VEC) {
      if (there && c < p.dim) x = *reinterpret_cast<const float4 *>(src + c);
    } else if (there) {
      if (c < p.dim) x.x = src[c];
      if (c + 1 < p.dim) x.y = src[c + 1];
      if (c + 2 < p.dim) x.z = src[c + 2];
      if (c + 3 < p.dim) x.w = src[c + 3];
    }
    return x;
  };
  float4 q[R], o[R];
  int pos[R];
  float m[R], l[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int rr = min(row0 + r, n_rows - 1), i = rr / G;
    q[r] = fetch(qp + (s.q0 + static_cast<int64_t>(i)) * p.q_ts + (h * G + rr - i * G) * p.q_hs, true);
    pos[r] = s.nk - s.nq + i;
    o[r] = make_float4(0.f, 0.f, 0.f, 0.f);
    m[r] = -INFINITY;
    l[r] = 0.f;
  }
  // A lane for each of a tile's keys: where its rows are (-1: nowhere), handed
  // to the lanes that load them.
  auto row_of = [&](int t, bool v) -> int64_t {
    return lane < KT && t < t1 ? key_row<PAGED>(p, k, s, table, h, t * KT + lane, v) : -1;
  };
  int64_t mine = row_of(t0 + warp, false);
  for (int t = t0 + warp; t < t1; t += 4) {
    const int64_t mine_v = PAGED || mine < 0 ? mine : row_of(t, true);
    float4 kk[U], vv[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t ok = __shfl_sync(0xffffffffu, mine, u * KPL + sub), ov = PAGED ? ok : __shfl_sync(0xffffffffu, mine_v, u * KPL + sub);
      kk[u] = fetch(kp + (ok < 0 ? 0 : ok), ok >= 0);
      vv[u] = fetch(vp + (ok < 0 ? 0 : ov), ok >= 0);
    }
    unsigned see[R];
#pragma unroll
    for (int r = 0; r < R; ++r) see[r] = __ballot_sync(0xffffffffu, mine >= 0 && sees(p, k, t * KT + lane, pos[r])) >> sub;
    mine = row_of(t + 4, false);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      float sc[U], top = -INFINITY;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float x = q[r].x * kk[u].x;
        x = fmaf(q[r].y, kk[u].y, x);
        x = fmaf(q[r].z, kk[u].z, x);
        x = fmaf(q[r].w, kk[u].w, x);
#pragma unroll
        for (int y = LPK / 2; y > 0; y >>= 1) x += __shfl_xor_sync(0xffffffffu, x, y);
        sc[u] = see[r] >> (u * KPL) & 1u ? x * p.sl2 : -INFINITY;
        top = fmaxf(top, sc[u]);
      }
      top = fmaxf(top, m[r]);  // each lane group keeps its own keys' maximum
      const float ref = top == -INFINITY ? 0.f : top, f = exp2f(m[r] - ref);
      m[r] = top;
      l[r] *= f;
      o[r].x *= f;
      o[r].y *= f;
      o[r].z *= f;
      o[r].w *= f;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const float e = exp2f(sc[u] - ref);
        l[r] += e;
        o[r].x = fmaf(e, vv[u].x, o[r].x);
        o[r].y = fmaf(e, vv[u].y, o[r].y);
        o[r].z = fmaf(e, vv[u].z, o[r].z);
        o[r].w = fmaf(e, vv[u].w, o[r].w);
      }
    }
  }
#pragma unroll
  for (int r = 0; r < R; ++r) {
    jo[warp][r][lane] = o[r];
    if (lane % LPK == 0) jml[warp][r][sub] = make_float2(m[r], l[r]);
  }
  __syncthreads();
  const int heads = p.kv_heads * G;
  const int64_t all = static_cast<int64_t>(p.q_rows) * heads;
  for (int x = tid; x < R * LPK; x += kThreads) {
    const int r = x / LPK, cc = x % LPK, rr = row0 + r;
    if (rr >= n_rows) continue;
    float mm = -INFINITY, ll = 0.f;
    float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < 4 * KPL; ++w) mm = fmaxf(mm, jml[w / KPL][r][w % KPL].x);
#pragma unroll
    for (int w = 0; w < 4 * KPL; ++w) {
      const float2 ml = jml[w / KPL][r][w % KPL];
      if (ml.x == -INFINITY) {
        ll += ml.y;  // 0, or NaN where the scores are
        continue;
      }
      const float f = exp2f(ml.x - mm);
      const float4 z = jo[w / KPL][r][(w % KPL) * LPK + cc];
      ll += ml.y * f;
      y.x += z.x * f;
      y.y += z.y * f;
      y.z += z.z * f;
      y.w += z.w * f;
    }
    const int i = rr / G, hq = h * G + rr % G;
    if (p.splits > 1) {
      const int64_t row = blockIdx.z * all + static_cast<int64_t>(s.q0 + i) * heads + hq;
      if (cc == 0) p.part_ml[row] = make_float2(mm, ll);
      *reinterpret_cast<float4 *>(p.part_o + row * DP + 4 * cc) = y;
    } else {
      const float inv = ll > 0.f ? 1.f / ll : (ll == 0.f ? 0.f : ll);
      float *out = static_cast<float *>(p.out) + (s.q0 + static_cast<int64_t>(i)) * p.o_ts + hq * p.o_hs;
      const float e[4] = {y.x * inv, y.y * inv, y.z * inv, y.w * inv};
#pragma unroll
      for (int z = 0; z < 4; ++z)
        if (4 * cc + z < p.dim) out[4 * cc + z] = e[z];
    }
  }
}

template <auto KERN>
cudaError_t launch_smem(dim3 grid, size_t smem, cudaStream_t stream, const WinAttnParams &p) {
  static bool done[64] = {false};  // per device
  int dev = 0;
  cudaGetDevice(&dev);
  if (smem > 48 * 1024 && !(dev < 64 && done[dev])) {
    const cudaError_t e = cudaFuncSetAttribute(KERN, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
    if (e != cudaSuccess) return e;
    if (dev < 64) done[dev] = true;
  }
  return launch_pdl(KERN, grid, dim3(kThreads), smem, stream, 1, p);
}

template <int DP, int WR, bool PAGED, bool VEC>
cudaError_t launch_tf32(dim3 grid, cudaStream_t stream, const WinAttnParams &p) {
  return p.dim <= DP - 8 ? launch_smem<win_attn_tf32<DP, WR, PAGED, VEC, true>>(grid, F32Smem<DP>::kBytes, stream, p)
                         : launch_smem<win_attn_tf32<DP, WR, PAGED, VEC, false>>(grid, F32Smem<DP>::kBytes, stream, p);
}

template <int DP, bool PAGED, bool VEC>
cudaError_t launch_form(const WinAttnParams &p, int f32, const WinAttnPlan &pl, cudaStream_t stream) {
  const dim3 grid(pl.tiles, p.kv_heads, p.splits);
  constexpr int kDeep = DP == 64 ? 3 : 2;  // three CTAs an SM and more (with one stage more, two CTAs: 311 for 258 us at 64 x 8192 tokens, 32/8 heads of 128)
  if (f32) {
    if (pl.rows == 1) return launch_smem<win_attn_f32_rows<DP, 1, PAGED, VEC>>(grid, 0, stream, p);
    if (pl.rows == 2) return launch_smem<win_attn_f32_rows<DP, 2, PAGED, VEC>>(grid, 0, stream, p);
    if (pl.rows == 4) return launch_smem<win_attn_f32_rows<DP, 4, PAGED, VEC>>(grid, 0, stream, p);
    if (pl.rows == 16) return launch_tf32<DP, 1, PAGED, VEC>(grid, stream, p);
    if (pl.rows == 32) return launch_tf32<DP, 2, PAGED, VEC>(grid, stream, p);
    return launch_tf32<DP, 4, PAGED, VEC>(grid, stream, p);
  }
  if (pl.rows == 16) return launch_smem<win_attn_mma<DP, 1, kDeep, PAGED, VEC>>(grid, MmaSmem<DP, 16, kDeep>::kBytes, stream, p);
  if (pl.rows == 32) return launch_smem<win_attn_mma<DP, 2, kDeep, PAGED, VEC>>(grid, MmaSmem<DP, 32, kDeep>::kBytes, stream, p);
  return launch_smem<win_attn_mma<DP, 4, 2, PAGED, VEC>>(grid, MmaSmem<DP, 64, 2>::kBytes, stream, p);
}

bool aligned16(const void *x, int64_t a, int64_t b, int size) {
  return reinterpret_cast<uintptr_t>(x) % 16 == 0 && (a * size) % 16 == 0 && (b * size) % 16 == 0;
}

}  // namespace

// The tensor-core form takes 256 rows a CTA and wins from about 32 rows of a
// sequence and kv head on (B200, 10 heads of 64: 40 rows 6.1 against 7.1 us,
// 16 rows 5.9 against 4.9; 24 sequences of 20 rows 13.1 against 7.1, of 70
// rows 13.9 against 17.4; long prompts 2.5 to 4.7 times faster).
bool win_attn_tc_fits(int f32, int seqs, int q_rows, int group) {
  return !f32 && group <= 128 && static_cast<int64_t>(q_rows) * group > 32 * static_cast<int64_t>(seqs);
}

WinAttnPlan win_attn_plan(int sm_count, int f32, bool tensor, bool uniform, int seqs, int q_rows, int64_t key_bound, int kv_heads,
                          int group, int dim, int left, int right, int sinks) {
  WinAttnPlan pl = {};
  const int64_t rows = static_cast<int64_t>(q_rows) * group;
  const int64_t mean = (rows + seqs - 1) / seqs;  // rows of a sequence and kv head
  if (tensor) {
    // Two tiles keep the tensor cores busy during one's exponentials; where even
    // single ones leave SMs idle, they end sooner.
    const int64_t one = 128 / group * group, items = (rows + one - 1) / one;
    pl.pair = (items > seqs ? items : seqs) * kv_heads <= sm_count ? 1 : 2;
    pl.rows = pl.pair * static_cast<int>(one);
  } else if (f32) {
    pl.rows = mean <= 1 ? 1 : mean <= 2 ? 2 : mean <= 4 ? 4 : mean <= 16 ? 16 : mean <= 32 ? 32 : 64;
    // Where 64-row tiles leave SMs idle, 32-row ones end sooner (501 tokens, 10
    // heads of 64, window 16 + 4: 12.3 -> 9.4 us; 8 x 100 tokens, 8 heads of 64:
    // 14.8 -> 12.1); with more of them the keys' splitting twice costs more (4000
    // tokens, 4 heads of 128, window 500, 252 tiles: 119 us, 32-row tiles 164).
    const int64_t each = (rows + 63) / 64;
    if (pl.rows == 64 && (each > seqs ? each : seqs) * kv_heads <= sm_count) pl.rows = 32;
  } else {
    pl.rows = mean <= 16 ? 16 : mean <= 32 ? 32 : 64;
  }
  // every sequence's last tile may hold as little as one row
  const int64_t bound = (rows + static_cast<int64_t>(seqs) * (pl.rows - 1)) / pl.rows;
  pl.tiles = static_cast<int>(uniform ? seqs * ((mean + pl.rows - 1) / pl.rows) : bound < rows ? bound : rows);
  // Keys of a tile at most, and the CTAs that the call has without a split.
  int64_t keys = key_bound;
  if (left < kWinUnlimited && right < kWinUnlimited)
    keys = keys < static_cast<int64_t>(left) + right + sinks + pl.rows ? keys : static_cast<int64_t>(left) + right + sinks + pl.rows;
  const int64_t each = (rows + pl.rows - 1) / pl.rows;
  const int64_t have = (each > seqs ? each : seqs) * kv_heads;
  // CTAs an SM that a split aims at, and the keys that each takes at least: the
  // f32 row form (little shared memory, loads straight to registers, four CTAs
  // an SM at 110 registers) four of 64, the other warp-level forms two of 256,
  // the tensor-core form one of 1024 (it fills and drains in the time of 256).
  // Measured for the row form, 16 sequences, 10 heads of 64, window 1023: four
  // an SM 26.9 us, six 32.3 (a second wave); one sequence of 700 keys: 64 keys
  // 8.4 us, 128 9.6, 256 12.4.
  const bool rows_form = f32 && pl.rows <= 4;
  const int64_t want = static_cast<int64_t>(tensor ? 1 : rows_form ? 4 : 2) * sm_count;
  int64_t z = have > 0 ? want / have : 1;
  pl.split_keys = tensor ? 1024 : rows_form ? 64 : 256;
  const int64_t most = keys / pl.split_keys;
  z = z < most ? z : most;
  // The keys are what a sequence may have, not what it has (that is on the device):
  // over a cache, what a slot has room for.  One token over 201 cached ones, 10
  // heads of 64: room for 240 tokens 5.1 us, 1024 7.3 (two launches), 8192 9.8,
  // 65536 12.9; of 64 sequences 11.9, 11.8, 25.7, 141.
  // Few rows over long contexts: pieces of 1024 keys (f32: 384), so that
  // sequences of unlike lengths keep all SMs busy to the end (64 sequences of
  // 2048 to 8192 tokens, 32/8 heads of 128: 258 us, pieces of 512 keys 281; f32,
  // 32 sequences of up to 4000 tokens, 8 heads of 128: 131 us, of 1024 160).
  const int64_t piece = f32 ? 384 : 1024;
  if (!tensor && mean <= 32 && keys >= 2 * piece && z < (keys + piece - 1) / piece) {
    z = (keys + piece - 1) / piece;
    pl.split_keys = static_cast<int>(piece);
  }
  pl.splits = static_cast<int>(z < 1 ? 1 : z > 64 ? 64 : z);
  const int dp = dim <= 64 ? 64 : 128;
  pl.workspace = pl.splits > 1 ? static_cast<size_t>(pl.splits) * q_rows * kv_heads * group * (dp * 4 + 8) : 0;
  return pl;
}

cudaError_t launch_win_attn_join(const WinAttnParams &p, int f32, const WinAttnPlan &pl, cudaStream_t stream) {
  const dim3 grid(pl.tiles, p.kv_heads);
  if (f32)
    return p.dim <= 64 ? launch_pdl(win_attn_join<float, 64>, grid, dim3(kThreads), 0, stream, 1, p, pl.rows)
                       : launch_pdl(win_attn_join<float, 128>, grid, dim3(kThreads), 0, stream, 1, p, pl.rows);
  return p.dim <= 64 ? launch_pdl(win_attn_join<__nv_bfloat16, 64>, grid, dim3(kThreads), 0, stream, 1, p, pl.rows)
                     : launch_pdl(win_attn_join<__nv_bfloat16, 128>, grid, dim3(kThreads), 0, stream, 1, p, pl.rows);
}

cudaError_t launch_win_attn(const WinAttnParams &p, int f32, const WinAttnPlan &pl, cudaStream_t stream) {
  const int size = f32 ? 4 : 2;
  const bool vec = (p.dim * size) % 16 == 0 && aligned16(p.q, p.q_ts, p.q_hs, size) && aligned16(p.out, p.o_ts, p.o_hs, size) &&
                   (p.table ? aligned16(p.k, 0, 0, size) && aligned16(p.v, 0, 0, size)
                            : aligned16(p.k, p.k_ts, p.k_hs, size) && aligned16(p.v, p.v_ts, p.v_hs, size));
  const bool paged = p.table != nullptr;
  cudaError_t e;
  if (p.dim <= 64) {
    e = paged ? vec ? launch_form<64, true, true>(p, f32, pl, stream) : launch_form<64, true, false>(p, f32, pl, stream)
              : vec ? launch_form<64, false, true>(p, f32, pl, stream) : launch_form<64, false, false>(p, f32, pl, stream);
  } else {
    e = paged ? vec ? launch_form<128, true, true>(p, f32, pl, stream) : launch_form<128, true, false>(p, f32, pl, stream)
              : vec ? launch_form<128, false, true>(p, f32, pl, stream) : launch_form<128, false, false>(p, f32, pl, stream);
  }
  return e != cudaSuccess || p.splits == 1 ? e : launch_win_attn_join(p, f32, pl, stream);
}

}  // namespace nq
