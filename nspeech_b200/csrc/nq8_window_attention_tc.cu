// nq8_window_attention_tc.cu -- window attention of many bf16 query rows on
// the 5th-generation tensor cores (tcgen05 + TMEM).
//
// Work item: two tiles (A, B) of 128 query rows of one kv head (one where that
// many items leave SMs idle); a row is a
// (token, head of the group) pair, token-major, which is the order in which
// one TMA box {64 columns, group heads, tokens} arrives.  The item's keys (the
// sinks, then the window of all its rows) are walked in tiles of 128; a tile
// that none of A's (B's) rows sees is skipped for A (B).
//
// Roles (384 threads, one CTA an SM; a twelfth warp idles):
//   warps 0-3   softmax of tile A: thread = query row = TMEM lane
//   warps 4-7   softmax of tile B
//   warp 8      K loads (one lane); owns the TMEM
//   warp 9      V loads
//   warp 10     MMA issue
// TMEM (512 columns, f32): S_A, S_B 128 columns each, O_A, O_B DP columns
// each.  P (bf16, two a column) overwrites the first half of its S and is the
// PV MMA's A operand straight from TMEM; V is an MN-major B operand from its
// TMA tile.  Per key tile and X the issuing thread runs PV_X(t - 1), then
// QK_X(t), in order, so S_X(t) full means that PV_X(t - 1) is done too.  While
// A's threads are in their exponentials, the tensor cores work for B.
//
// Bound: per pair of tiles and 128 keys the MMAs take 2 x 2 x 128 x 128 x DP x 2
// flops (2048 clocks at DP = 128), the exponentials 2 x 128 x 128 at 16 a clock
// (2048 clocks), and shared memory moves about as long (operands of QK^T 1024,
// of PV 512, TMA 512).  Such a step takes about 3300 clocks.  16384 tokens, 16
// query heads over 4 kv heads of 128, window 4096 and 4 sinks: 430 us in bursts
// of 20 calls at 1965 MHz, 0.67 of the time of its flops at the measured burst
// rate of 1666 TFLOP/s; call after call, where the power cap holds the clock at
// 1710 MHz, 497 us (0.58); the warp-level form takes 2460 us.  On the way, in
// bursts: registers limited for all code by a setmaxnreg ahead of
// the branches 661 us, MMAs issued by one lane of a divergent warp 471 us, a
// quarter to three quarters of the exponentials on the FMA pipe 501 to 514 us.
//
// O is rescaled only when a row's maximum grows by more than 2^8 (exponentials
// stay <= 256; the final O / l does not depend on the reference maximum).
//
// Rows of V that no query of the item sees may hold anything: a weight of 0
// times NaN would be NaN, so a tile's PV runs only the 16-key steps that hold
// seen keys, and the other rows of those steps are zeroed in shared memory.
//
// Every wait is bounded (DevCtl); a role that gives up raises the CTA's abort
// flag, all roles leave their loops, copies and MMAs in flight are waited for,
// and TMEM is freed.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include <type_traits>

#include "nq8_window_attention.cuh"

namespace nq {
namespace {

using namespace win;

constexpr int kKT = 128;  // keys of a tile
constexpr int kWarpK = 8, kWarpV = 9, kWarpMma = 10;  // after the eight softmax warps
constexpr int kTcThreads = 32 * 12;  // one warp idles: registers are split by groups of four warps

template <int DP>
struct TcSmem {
  static constexpr int kStages = DP == 64 ? 4 : 2;
  static constexpr uint32_t kBox = 128 * 64 * 2;           // 128 rows x 64 columns, 128-byte swizzle
  static constexpr uint32_t kTile = kBox * (DP / 64);
  static constexpr uint32_t kOffQ = 0;                     // A, B
  static constexpr uint32_t kOffK = 2 * kTile;
  static constexpr uint32_t kOffV = kOffK + kStages * kTile;
  static constexpr uint32_t kOffBar = kOffV + kStages * kTile;
  static constexpr uint32_t kOffHole = kOffBar + 256;      // [8 tiles][4 words] keys whose page is missing
  static constexpr uint32_t kBytes = kOffHole + 8 * 16 + 1024;  // 1024: alignment
  // barriers
  static constexpr int kKFull = 0, kKEmpty = kStages, kVFull = 2 * kStages, kVEmpty = 3 * kStages, kQFull = 4 * kStages,
                       kSFull = kQFull + 1, kPReady = kSFull + 2, kOFull = kPReady + 4, kDone = kOFull + 2, kBars = kDone + 1;
};
static_assert(TcSmem<64>::kBars * 8 + 8 <= 256, "barrier block");

__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap *map, uint32_t bar, int x, int y, int z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
      "[%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y), "r"(z)
      : "memory");
}
// MN-major operand of 128-byte swizzle atoms (64 MN elements by 8 k rows,
// 1024 bytes): `mn` bytes between atoms along MN, 1024 along k.
__device__ __forceinline__ uint64_t mn_desc(uint32_t saddr, uint32_t mn) {
  uint64_t d = 0;
  d |= static_cast<uint64_t>((saddr >> 4) & 0x3FFFu);
  d |= static_cast<uint64_t>((mn >> 4) & 0x3FFFu) << 16;
  d |= static_cast<uint64_t>(1024u >> 4) << 32;
  d |= static_cast<uint64_t>(1u) << 46;
  d |= static_cast<uint64_t>(2u) << 61;
  return d;
}
// D[tmem] (+)= A[tmem] . B[smem]
__device__ __forceinline__ void umma_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t *r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
      "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]),
      "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]),
      "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred q;\n\telect.sync _|q, 0xffffffff;\n\tselp.u32 %0, 1, 0, q;\n\t}" : "=r"(p));
  return p != 0;
}

// Two f32 at a time.
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.ftz.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.ftz.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ void unpack2(uint64_t v, float &a, float &b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }

// Bits lo..hi (any integers) of a 32-bit word.
__device__ __forceinline__ uint32_t bit_range(int lo, int hi) {
  lo = max(lo, 0);
  hi = min(hi, 31);
  return hi < lo ? 0u : (0xffffffffu >> (31 - hi)) & (0xffffffffu << lo);
}

// The key tiles of an item: the sinks' from key 0, then the window's.  A CTA
// walks n of them, from tile `off` on (a split of the keys).
struct Tiles {
  int sink_tiles, lo, off, n;  // lo: first key of the window's tiles
  __device__ __forceinline__ bool in_sinks(int t) const { return t + off < sink_tiles; }
  __device__ __forceinline__ int base(int t) const { return in_sinks(t) ? (t + off) * kKT : lo + (t + off - sink_tiles) * kKT; }
};
// The part of them that one of the two row tiles sees: tiles [0, head) for the
// sinks, [first, last] for its window (none: last < first, head = 0).
struct Part {
  int head, first, last;
  __device__ __forceinline__ bool sees(int t) const { return t < head || (t >= first && t <= last); }
};
__device__ __forceinline__ Part part_of(const WinAttnParams &p, const Tiles &k, const Seq &s, int G, int r0, int rows, int n_rows) {
  Part x{0, 0, -1};
  if (r0 >= n_rows) return x;
  const int i0 = r0 / G, i1 = (min(r0 + rows, n_rows) - 1) / G;
  const int hi = p.right >= kWinUnlimited ? s.nk - 1 : min(s.nk - 1, s.nk - s.nq + i1 + p.right);
  if (hi < 0) return x;
  const int lo = p.left >= kWinUnlimited ? 0 : max(0, s.nk - s.nq + i0 - p.left);
  const int sinks = min(p.sinks, hi + 1);
  // tiles with base < sinks (bases grow with t), and those that meet [lo, hi]
  x.head = min((sinks + kKT - 1) / kKT, k.sink_tiles);
  if (k.sink_tiles == 0 && sinks > k.lo) x.head = (sinks - k.lo + kKT - 1) / kKT;
  x.first = k.sink_tiles + max(0, lo - k.lo) / kKT;
  x.last = k.sink_tiles + (hi - k.lo) / kKT;
  // the CTA's own tiles
  x.head = min(max(x.head - k.off, 0), k.n);
  x.first = max(x.first - k.off, 0);
  x.last = hi < k.lo ? -1 : min(x.last - k.off, k.n - 1);
  if (x.last < x.first) x.last = -1;
  return x;
}

template <int DP, bool PAGED>
__global__ void __launch_bounds__(kTcThreads, 1)
    win_attn_tc(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ WinAttnParams p) {
  using L = TcSmem<DP>;
  constexpr int S = L::kStages;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  const uint32_t raw_u32 = smem_u32(smem_raw);
  uint8_t *smem = smem_raw + (((raw_u32 + 1023u) & ~1023u) - raw_u32);
  const uint32_t sbase = smem_u32(smem);
  uint64_t *bars = reinterpret_cast<uint64_t *>(smem + L::kOffBar);
  auto bar = [&](int i) { return smem_u32(&bars[i]); };
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(&bars[L::kBars]);
  volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);
  uint32_t *holes = reinterpret_cast<uint32_t *>(smem + L::kOffHole);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long lim = p.ctl.wait_limit;

  if (threadIdx.x == 0) {
    for (int i = 0; i < L::kBars; ++i) mbar_init(bar(i), i >= L::kPReady && i < L::kPReady + 4 ? 128 : 1);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == kWarpK) {
    tmem_alloc(smem_u32(tmem_slot), 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_wait();
  pdl_trigger();

  const int G = p.group, h = blockIdx.y;
  const int rows = 128 / G * G;  // query rows of a tile
  int b = 0, row0 = 0, n_rows = 0;
  Seq sq = {};
  Keys ks = {};
  Tiles tl = {};
  if (find_tile(p, gridDim.x - 1 - blockIdx.x, p.pair * rows, b, row0)) {
    sq = seq_of(p, b);
    n_rows = sq.nq * G;
    ks = keys_of<kKT>(p, sq, row0 / G, (min(row0 + p.pair * rows, n_rows) - 1) / G);
    tl.sink_tiles = ks.sink_tiles;
    tl.lo = ks.lo;
    if (PAGED) tl.lo &= ~(min(kKT, 1 << p.page_shift) - 1);  // the window's tiles begin with a box
    const int all = ks.sink_tiles + (ks.hi >= ks.lo ? (ks.hi - tl.lo + kKT) / kKT : 0);
    tl.off = static_cast<int>(static_cast<int64_t>(all) * blockIdx.z / p.splits);
    tl.n = static_cast<int>(static_cast<int64_t>(all) * (blockIdx.z + 1) / p.splits) - tl.off;
  }
  const int nt = tl.n;
  // Rows of tile t that some query of the item may see, [v0, v1) without [g0, g1)
  // (between the sinks and the window): the others hold anything.
  auto seen_rows = [&](int t, int &v0, int &v1, int &g0, int &g1) {
    const int base = tl.base(t);
    v0 = tl.in_sinks(t) ? 0 : max(0, ks.lo - base);
    v1 = min(kKT, (tl.in_sinks(t) ? ks.s_end : ks.hi + 1) - base);
    g0 = max(0, ks.gap_lo - base);
    g1 = min(kKT, ks.gap_hi - base);
  };

  // Registers: 384 threads launch with 168 each; 256 x 208 + 128 x 80 is less.
  // One branch for each of the two shares, or the lower limit would hold for all code.
  if (warp >= kWarpK) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 80;");
    if (warp == kWarpK || warp == kWarpV) {
      if ((PAGED || lane == 0) && nt > 0) {
        // ------------------------------------------------------------- loads
        // Plain rows: one lane, a box a tile.  Pages: a lane for each box of a
        // tile (at most 16), whose page is looked up a tile ahead.
        const bool is_v = warp == kWarpV;
        const CUtensorMap *map = is_v ? &tm_v : &tm_k;
        const int full0 = is_v ? L::kVFull : L::kKFull, empty0 = is_v ? L::kVEmpty : L::kKEmpty;
        const uint32_t slot0 = is_v ? L::kOffV : L::kOffK;
        bool q_issued = false;
        if (lane == 0) {
          prefetch_tmap(map);
          if (!is_v) {
            prefetch_tmap(&tm_q);
            const int toks = 128 / G;
            mbar_arrive_expect_tx(bar(L::kQFull), p.pair * (DP / 64) * static_cast<uint32_t>(toks * G * 128));
            for (int x = 0; x < p.pair; ++x)
  #pragma unroll
              for (int c = 0; c < DP / 64; ++c)
                tma_load_3d(sbase + L::kOffQ + x * L::kTile + c * L::kBox, &tm_q, bar(L::kQFull), 64 * c, h * G,
                            sq.q0 + (row0 + x * rows) / G);
            q_issued = true;
          }
        }
        const int box = PAGED ? min(kKT, 1 << p.page_shift) : kKT;  // rows of a box
        const int *table = PAGED ? p.table + static_cast<int64_t>(b) * p.table_ld : nullptr;
        auto page_of = [&](int t) {  // of this lane's box; -1: none, or no key of the list
          const int key = t < nt ? tl.base(t) + lane * box : 0;
          if (t >= nt || lane * box >= kKT || key > ks.hi || (tl.in_sinks(t) && key >= ks.s_end)) return -1;
          const int pg = table[key >> p.page_shift];
          return pg < p.pages ? pg : -1;
        };
        int pg = PAGED ? page_of(0) : 0;
        int n = 0;
        for (int t = 0; t < nt; ++t) {
          const int s = t % S, use = t / S;
          const int pg_next = PAGED ? page_of(t + 1) : 0;
          bool ok = use == 0 || mbar_wait(bar(empty0 + s), (use - 1) & 1, lim, abort_flag);
          if (PAGED) ok = __all_sync(0xffffffffu, ok);
          if (!ok) {
            if (lane == 0 && !*abort_flag) report(p.ctl, abort_flag, kDevTimeoutProducer);
            break;
          }
          if (PAGED ? __any_sync(0xffffffffu, *abort_flag) : *abort_flag) break;
          const uint32_t full = bar(full0 + s), dst = sbase + slot0 + s * L::kTile;
          const int base = tl.base(t);
          if constexpr (!PAGED) {
            mbar_arrive_expect_tx(full, L::kTile);
  #pragma unroll
            for (int c = 0; c < DP / 64; ++c) tma_load_3d(dst + c * L::kBox, map, full, 64 * c, h, sq.k0 + base);
          } else {
            const int boxes = kKT / box;
            const unsigned have = __ballot_sync(0xffffffffu, pg >= 0);  // boxes whose page exists
            if (!is_v) {
              // the softmax's view of missing pages (keys past the end are masked anyway)
              if (lane < 4) {
                uint32_t m = 0;
                for (int j = 0; j < boxes; ++j)
                  if (!(have >> j & 1)) m |= bit_range(j * box - 32 * lane, (j + 1) * box - 1 - 32 * lane);
                holes[(t & 7) * 4 + lane] = m;
              }
            } else if (have != (boxes == 32 ? 0xffffffffu : (1u << boxes) - 1u)) {
              // missing pages' values: zeros (their weights are zero)
              for (int j = 0; j < boxes; ++j)
                if (!(have >> j & 1))
                  for (int c = 0; c < DP / 64; ++c)
                    for (int x = lane; x < box * 8; x += 32)
                      asm volatile("st.shared.v4.b32 [%0], {%1,%1,%1,%1};" ::"r"(dst + c * L::kBox + j * box * 128 + x * 16), "r"(0) : "memory");
              fence_proxy_async_smem();
            }
            __syncwarp();
            const uint32_t box_bytes = static_cast<uint32_t>(box) * 128u;
            if (lane == 0) mbar_arrive_expect_tx(full, __popc(have) * box_bytes * (DP / 64));
            __syncwarp();
            if (pg >= 0) {
              const int row = ((pg * p.kv_heads + h) << p.page_shift) + ((base + lane * box) & ((1 << p.page_shift) - 1));
  #pragma unroll
              for (int c = 0; c < DP / 64; ++c) tma_load_2d(dst + c * L::kBox + lane * box_bytes, map, full, 64 * c, row);
            }
            pg = pg_next;
          }
          ++n;
        }
        // Every copy issued into shared memory has landed.
        volatile int no_abort = 0;
        if (lane == 0) {
          for (int s = 0; s < S; ++s) {
            const int uses = n > s ? (n - 1 - s) / S + 1 : 0;
            if (uses > 0 && !mbar_wait(bar(full0 + s), (uses - 1) & 1, lim, &no_abort)) atomicOr(p.ctl.status, kDevTimeoutDrain);
          }
          if (q_issued && !mbar_wait(bar(L::kQFull), 0, lim, &no_abort)) atomicOr(p.ctl.status, kDevTimeoutDrain);
        }
        __syncwarp(PAGED ? 0xffffffffu : 1u);
      }
    } else if (warp == kWarpMma && nt > 0) {
      // ----------------------------------------------------------------- MMA
      // The whole warp walks the loop, so that addresses and descriptors live in
      // uniform registers; one elected lane issues.
      constexpr uint32_t kIdescS = idesc_bf16_f32(128, kKT);
      constexpr uint32_t kIdescPV = idesc_bf16_f32(128, DP) | (1u << 16);  // B (V) MN-major
      const bool leader = elect_one();
      auto uniform = [](int v) { return __shfl_sync(0xffffffffu, v, 0); };
      auto wait = [&](int i, int parity) -> bool {
        if (__all_sync(0xffffffffu, mbar_try_wait(bar(i), parity))) return true;
        const bool ok = __all_sync(0xffffffffu, mbar_wait(bar(i), parity, lim, abort_flag));
        if (!ok && lane == 0 && !*abort_flag) report(p.ctl, abort_flag, kDevTimeoutMma);
        return ok;
      };
      Part part[2];
      int final_t[2];
  #pragma unroll
      for (int x = 0; x < 2; ++x) {
        const Part y = part_of(p, tl, sq, G, row0 + x * rows, rows, x < p.pair ? n_rows : 0);
        part[x] = Part{uniform(y.head), uniform(y.first), uniform(y.last)};
        final_t[x] = max(part[x].head - 1, part[x].last);
      }
      const int n_tiles = uniform(nt);
      const uint32_t tm = uniform(tmem);
      int done_p[2] = {0, 0};  // P tiles consumed
      bool ok = wait(L::kQFull, 0);
      int slot = 0, phase = 0, v_slot = 0, v_phase = 0;  // of K tile t, of V tile t - 1
      for (int t = 0; t <= n_tiles && ok; ++t) {
        if (t < n_tiles && !(ok = wait(L::kKFull + slot, phase))) break;
        const uint32_t va = sbase + L::kOffV + v_slot * L::kTile;
        // Descriptors differ in the address field alone.
        const uint64_t vd = mn_desc(va, L::kBox), kd = sw128_kmajor_desc(sbase + L::kOffK + slot * L::kTile);
        bool v_ready = false;
        int k0 = 0, k1 = kKT / 16;
  #pragma unroll
        for (int x = 0; x < 2; ++x) {
          if (!ok) break;
          if (t > 0 && part[x].sees(t - 1)) {
            if (!v_ready) {
              if (!(ok = wait(L::kVFull + v_slot, v_phase))) break;
              v_ready = true;
              int v0, v1, g0, g1;
              seen_rows(t - 1, v0, v1, g0, g1);
              if (v0 > 0 || v1 < kKT || g0 < g1) {
                k0 = uniform(v0 / 16);
                k1 = uniform((v1 + 15) / 16);
                for (int r = 16 * k0 + lane / 8; r < 16 * k1; r += 4)
                  if (r < v0 || r >= v1 || (r >= g0 && r < g1))
                    for (int c = 0; c < DP / 64; ++c)
                      asm volatile("st.shared.v4.b32 [%0], {%1,%1,%1,%1};" ::"r"(va + c * L::kBox + r * 128 + (lane & 7) * 16), "r"(0) : "memory");
                fence_proxy_async_smem();
                __syncwarp();
              }
            }
            const uint32_t first = done_p[x] == 0;
            if (!(ok = wait(L::kPReady + x, done_p[x] & 1))) break;
            tc_fence_after();
            const uint32_t d = tm + 256 + x * DP, a = tm + x * 128;
            const bool whole = k0 == 0 && k1 == kKT / 16;
            if (whole && leader) {
  #pragma unroll
              for (int kk = 0; kk < kKT / 32; ++kk) umma_ts(d, a + kk * 8, vd + kk * (2048 >> 4), kIdescPV, kk > 0 ? 1u : 1u - first);
            }
            if (!(ok = wait(L::kPReady + 2 + x, done_p[x] & 1))) break;
            ++done_p[x];
            tc_fence_after();
            if (leader) {
              if (whole) {
  #pragma unroll
                for (int kk = kKT / 32; kk < kKT / 16; ++kk) umma_ts(d, a + kk * 8, vd + kk * (2048 >> 4), kIdescPV, 1u);
              } else {
                for (int kk = k0; kk < k1; ++kk) umma_ts(d, a + kk * 8, vd + kk * (2048 >> 4), kIdescPV, kk > k0 ? 1u : 1u - first);
              }
              if (t - 1 == final_t[x]) umma_commit(bar(L::kOFull + x));
            }
          }
          if (t < n_tiles && part[x].sees(t)) {
            tc_fence_after();
            const uint64_t qd = sw128_kmajor_desc(sbase + L::kOffQ + x * L::kTile);
            if (leader) {
  #pragma unroll
              for (int kk = 0; kk < DP / 16; ++kk) {
                const uint32_t o = ((kk >> 2) * L::kBox + (kk & 3) * 32) >> 4;
                umma_bf16(tm + x * 128, qd + o, kd + o, kIdescS, kk > 0 ? 1u : 0u);
              }
              umma_commit(bar(L::kSFull + x));
            }
          }
        }
        if (!ok) break;
        if (t > 0) {
          // a tile's values are waited for even where no row sees them, so that the ring goes on
          if (!v_ready && !(ok = wait(L::kVFull + v_slot, v_phase))) break;
          if (leader) umma_commit(bar(L::kVEmpty + v_slot));
          if (++v_slot == S) v_slot = 0, v_phase ^= 1;
        }
        if (t < n_tiles) {
          if (leader) umma_commit(bar(L::kKEmpty + slot));
          if (++slot == S) slot = 0, phase ^= 1;
        }
      }
      // Every MMA issued completes before TMEM is freed.
      volatile int no_abort = 0;
      if (leader) {
        umma_commit(bar(L::kDone));
        if (!mbar_wait(bar(L::kDone), 0, lim, &no_abort)) atomicOr(p.ctl.status, kDevTimeoutDrain);
      }
      __syncwarp();
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
    // ------------------------------------------------------------- softmax
    const int x = warp >> 2;
    const int r = 32 * (warp & 3) + lane;        // TMEM lane, row of the tile
    const int row = row0 + x * rows + r;         // row of the sequence
    const bool there = r < rows && row < n_rows && x < p.pair;
    const uint32_t lanes = tmem + (static_cast<uint32_t>(32 * (warp & 3)) << 16);
    const uint32_t ts = lanes + x * 128, to = lanes + 256 + x * DP;
    const int pos = there ? sq.nk - sq.nq + row / G : 0;
    const Part part = part_of(p, tl, sq, G, row0 + x * rows, rows, x < p.pair ? n_rows : 0);
    // keys that every row of the tile sees: [all_lo, all_hi], sinks apart
    const int pos_lo = sq.nk - sq.nq + (row0 + x * rows) / G, pos_hi = sq.nk - sq.nq + (min(row0 + (x + 1) * rows, n_rows) - 1) / G;
    const int all_hi = p.right >= kWinUnlimited ? sq.nk - 1 : min(sq.nk - 1, pos_lo + p.right);
    const int all_lo = p.left >= kWinUnlimited ? 0 : pos_hi - p.left;
    float m_use = -INFINITY, l = 0.f;
    int n = 0;
    bool dead = false;
    auto wait_all = [&](int i, int parity, int bit) -> bool {
      bool ok = mbar_wait(bar(i), parity, lim, abort_flag) && !*abort_flag;
      ok = __all_sync(0xffffffffu, ok);
      if (!ok && lane == 0 && !*abort_flag) report(p.ctl, abort_flag, bit);
      return ok;
    };
    const int jmax_row = p.right >= kWinUnlimited ? sq.nk - 1 : min(sq.nk - 1, pos + p.right);
    const int jmin_row = p.left >= kWinUnlimited ? 0 : max(0, pos - p.left);
    for (int t = 0; t < nt; ++t) {
      if (!part.sees(t)) continue;
      if (!wait_all(L::kSFull + x, n & 1, kDevTimeoutConsumer)) {
        dead = true;
        break;
      }
      tc_fence_after();
      uint32_t sr[128];
#pragma unroll
      for (int c = 0; c < 4; ++c) tmem_ld32(ts + 32 * c, *reinterpret_cast<uint32_t(*)[32]>(sr + 32 * c));
      tmem_ld_wait();
      const int base = tl.base(t);
      uint32_t hole[4] = {0u, 0u, 0u, 0u};
      if constexpr (PAGED) {
#pragma unroll
        for (int c = 0; c < 4; ++c) hole[c] = *reinterpret_cast<volatile uint32_t *>(holes + (t & 7) * 4 + c);
      }
      const bool inside = base + kKT - 1 <= all_hi && (base >= all_lo || base + kKT <= p.sinks) && !(hole[0] | hole[1] | hole[2] | hole[3]);
      unsigned live = 15;  // quarters of the tile that a row of the warp sees a key of
      if (!inside) {
        live = 0;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const int o = base + 32 * c;
          const uint32_t see = (bit_range(jmin_row - o, jmax_row - o) | bit_range(0, min(p.sinks - 1, jmax_row) - o)) & ~hole[c];
          live |= __any_sync(0xffffffffu, see != 0u) ? 1u << c : 0u;
#pragma unroll
          for (int e = 0; e < 32; ++e) sr[32 * c + e] = see >> e & 1u ? sr[32 * c + e] : __float_as_uint(-INFINITY);
        }
      }
      float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int e = 0; e < 128; e += 2) top[(e >> 1) & 3] = fmaxf(fmaxf(top[(e >> 1) & 3], __uint_as_float(sr[e])), __uint_as_float(sr[e + 1]));
      const float tmax = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) * p.sl2;  // log2 units; the scale is positive
      bool resc = false;
      float factor = 1.f;
      if (tmax > m_use + 8.f || (m_use == -INFINITY && tmax > -INFINITY)) {
        resc = n > 0 && m_use > -INFINITY;
        factor = resc ? ex2(m_use - tmax) : 1.f;
        m_use = tmax;
      }
      if (__any_sync(0xffffffffu, resc)) {
        // PV of this X's previous tile is done: it was issued before this S
#pragma unroll 1
        for (int c = 0; c < DP / 32; ++c) {
          uint32_t o[32];
          tmem_ld32(to + 32 * c, o);
          tmem_ld_wait();
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * factor);
          tmem_st32(to + 32 * c, o);
        }
      }
      l *= factor;
      const float ref = m_use == -INFINITY ? 0.f : m_use;
      const uint64_t scale2 = f2(p.sl2, p.sl2), nref2 = f2(-ref, -ref);
      uint64_t sum2 = f2(0.f, 0.f);
      // P in two halves, so that PV begins with the first.  In a masked tile the
      // quarters that nobody sees are zeros.
      auto weights = [&](auto masked) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          uint32_t pk[32];
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            if (!decltype(masked)::value || (live >> (2 * c + q) & 1u)) {
#pragma unroll
              for (int e = 16 * q; e < 16 * q + 16; ++e) {
                float pa, pb;
                unpack2(fma2(f2(__uint_as_float(sr[64 * c + 2 * e]), __uint_as_float(sr[64 * c + 2 * e + 1])), scale2, nref2), pa, pb);
                pa = ex2(pa);
                pb = ex2(pb);
                sum2 = add2(sum2, f2(pa, pb));
                pk[e] = pack_bf16x2(pa, pb);
              }
            } else {
#pragma unroll
              for (int e = 16 * q; e < 16 * q + 16; ++e) pk[e] = 0u;
            }
          }
          tmem_st32(ts + 32 * c, pk);
          tmem_st_wait();
          tc_fence_before();
          mbar_arrive(bar(L::kPReady + 2 * c + x));
        }
      };
      if (inside)
        weights(std::false_type());
      else
        weights(std::true_type());
      float la, lb;
      unpack2(sum2, la, lb);
      l += la + lb;
      ++n;
    }
    // ---- output
    if (n > 0 && !dead && !wait_all(L::kOFull + x, 0, kDevTimeoutEpilogue)) dead = true;
    if (!dead) {
      tc_fence_after();
      const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
      const int i = there ? row / G : 0, hq = h * G + (there ? row - i * G : 0);
      const int64_t heads = static_cast<int64_t>(p.kv_heads) * G;
      const int64_t part_row = (blockIdx.z * static_cast<int64_t>(p.q_rows) + sq.q0 + i) * heads + hq;
      if (p.splits > 1 && there) p.part_ml[part_row] = make_float2(m_use, l);
      __nv_bfloat16 *out = static_cast<__nv_bfloat16 *>(p.out) + (there ? (sq.q0 + static_cast<int64_t>(i)) * p.o_ts + hq * p.o_hs : 0);
#pragma unroll
      for (int c = 0; c < DP / 32; ++c) {
        uint32_t o[32];
        if (n > 0) {
          tmem_ld32(to + 32 * c, o);
          tmem_ld_wait();
        } else {
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = 0u;
        }
        if (there && inv == 0.f) {
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = 0u;
        }
        if (p.splits > 1) {
          if (there) {
#pragma unroll
            for (int e = 0; e < 8; ++e)
              *reinterpret_cast<uint4 *>(p.part_o + part_row * DP + 32 * c + 4 * e) = make_uint4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
          }
        } else if (there) {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (32 * c + 8 * e < p.dim) {
              auto v = [&](int y) { return __uint_as_float(o[8 * e + y]) * inv; };
              *reinterpret_cast<uint4 *>(out + 32 * c + 8 * e) =
                  make_uint4(pack_bf16x2(v(0), v(1)), pack_bf16x2(v(2), v(3)), pack_bf16x2(v(4), v(5)), pack_bf16x2(v(6), v(7)));
            }
        }
      }
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == kWarpK) {
    tc_fence_after();
    __syncwarp();
    tmem_dealloc(tmem, 512);
  }
}

template <int DP, bool PAGED>
cudaError_t launch_tc(const CUtensorMap &q, const CUtensorMap &k, const CUtensorMap &v, const WinAttnParams &p, int tiles,
                      cudaStream_t stream) {
  static bool done[64] = {false};  // per device
  int dev = 0;
  cudaGetDevice(&dev);
  if (!(dev < 64 && done[dev])) {
    const cudaError_t e = cudaFuncSetAttribute(win_attn_tc<DP, PAGED>, cudaFuncAttributeMaxDynamicSharedMemorySize, TcSmem<DP>::kBytes);
    if (e != cudaSuccess) return e;
    if (dev < 64) done[dev] = true;
  }
  return launch_pdl(win_attn_tc<DP, PAGED>, dim3(tiles, p.kv_heads, p.splits), dim3(kTcThreads), TcSmem<DP>::kBytes, stream, 1, q, k, v, p);
}

}  // namespace

cudaError_t launch_win_attn_tc(const CUtensorMap &q, const CUtensorMap &k, const CUtensorMap &v, const WinAttnParams &p,
                               const WinAttnPlan &pl, cudaStream_t stream) {
  cudaError_t e;
  if (p.dim <= 64)
    e = p.table ? launch_tc<64, true>(q, k, v, p, pl.tiles, stream) : launch_tc<64, false>(q, k, v, p, pl.tiles, stream);
  else
    e = p.table ? launch_tc<128, true>(q, k, v, p, pl.tiles, stream) : launch_tc<128, false>(q, k, v, p, pl.tiles, stream);
  return e != cudaSuccess || p.splits == 1 ? e : launch_win_attn_join(p, 0, pl, stream);
}

}  // namespace nq
