// nq8_beam.cu -- beam search: the best continuations of an utterance's beams
// by log probability, and the reordering of what each beam carries.
//
// score(b, k, t) = scores[b][k] + x[t] - log sum_u exp(x[u]) over the row x of
// logits; of all beams and tokens the `beams` best, equal scores by beam, then
// token.  The sum of a row does not change the order within it, so one pass
// over the logits makes, per part of a row, its maximum, its sum of
// exponentials and its `beams` best values (beam_part_kernel); a second, small
// launch joins the parts and compares across beams in f64 (beam_join_kernel):
// the terms of a sum are f32 and added up in f64 from one thread's round on, so
// that candidates of two beams compare as their exact scores do up to about
// 2e-7 (the exponential's 2^-22; up to 1.5e-6 where the row's maximum lies up to
// 40 above its first round's, to which the terms then refer).
//
// Selection of the W best of a round of logits without sorting it: the W-th
// largest of the maxima of 32 thread groups is no larger than the W-th largest
// value, so only values from it on are looked at (about W ln of them for
// unordered logits), and they are ranked by sorting networks.  Where more than a list
// holds lie above it (many equal values), the same is done with keys (value
// and inverted index, all different) and a second bound from the thread maxima
// leaves W threads' values at most.
//
// The kernels start before the one ahead of them has ended, so the logits and
// parents that it may write are read by plain loads, not by the read-only path.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include "nq8_cache.h"

namespace nq {
namespace {

using Key = unsigned long long;
constexpr int kPartThreads = 256;
constexpr int kPerThread = 32;
constexpr int kPartElems = kPartThreads * kPerThread;  // logits of one round of a CTA
constexpr int kBeamSplitsMax = 16;
constexpr int kList = kBeamMax * kPerThread;           // the most that the exact bound leaves

// An f32 as an unsigned integer of the same order.
__device__ __forceinline__ uint32_t ordered(float x) {
  const uint32_t u = __float_as_uint(x);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float unordered(uint32_t u) {
  return __uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~u);
}
__device__ __forceinline__ Key make_key(float x, uint32_t index) {  // -0 as +0
  return static_cast<Key>(ordered(x + 0.f)) << 32 | static_cast<uint32_t>(~index);
}
__device__ __forceinline__ Key shfl_xor_key(Key v, int o) { return __shfl_xor_sync(0xffffffffu, v, o); }

// NaN and +inf count as -inf.
__device__ __forceinline__ float clean(float x) { return x < INFINITY ? x : -INFINITY; }

// Two at a time: 2^(x log2e - m'), with m' the rounded multiple of the
// round's maximum; the one factor that its rounding makes is put right in f64.
constexpr float kLog2e = 1.4426950408889634f;
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
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float halves(uint64_t v) {  // their sum
  float a, b;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
  return a + b;
}
__device__ __forceinline__ uint64_t ex2_2(uint64_t v) {
  float a, b;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
  return f2(ex2(a), ex2(b));
}

// Sorting networks of a warp, a key a lane, largest in lane 0.
__device__ __forceinline__ Key sort32(Key v, int lane) {
#pragma unroll
  for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
    for (int o = size / 2; o > 0; o >>= 1) {
      const Key y = shfl_xor_key(v, o);
      v = ((lane & o) == 0) == ((lane & size) == 0) ? (y > v ? y : v) : (y < v ? y : v);
    }
  return v;
}
// The 32 largest of two sorted runs, sorted.
__device__ __forceinline__ Key merge32(Key a, Key b, int lane) {
  const Key r = __shfl_sync(0xffffffffu, b, 31 - lane);
  Key v = r > a ? r : a;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const Key y = shfl_xor_key(v, o);
    v = (lane & o) == 0 ? (y > v ? y : v) : (y < v ? y : v);
  }
  return v;
}

// One part of one row: CTA (blockIdx.x of `splits`, row blockIdx.y).  Values
// that may be among the W best are listed as the rounds go by; the list is
// ranked at the end, or when it is half full.  A round is one pass over 8192
// logits with one synchronisation; its exponentials, the pass through shared
// memory and the wait for the next round's loads follow one another, so four
// CTAs an SM share the units.  512 rows of 32768 f32, 8 beams: 22.5 us,
// 3.0 TB/s; 4 rows of bf16: 6.9 us, latency.
template <bool BF16, bool VEC>
__global__ void __launch_bounds__(kPartThreads, 4) beam_part_kernel(const __grid_constant__ BeamParams p) {
  __shared__ float group_max[2][32];
  __shared__ Key key_max[32];
  __shared__ Key list[kList];
  __shared__ Key best[kBeamMax];  // of the rounds ranked so far, best first, 0: none
  __shared__ Key runs[kPartThreads / 32][32];
  __shared__ int added[2];  // entries listed in rounds of either parity, ever
  __shared__ int listed, ties;
  __shared__ double sums[kPartThreads / 32];
  extern __shared__ __align__(16) float4 xs[];  // [kPerThread / 4][kPartThreads]
  pdl_wait();
  pdl_trigger();
  const int row = blockIdx.y, tid = threadIdx.x, lane = tid & 31;
  const int W = p.beams;
  if (p.finished && p.finished[row]) return;
  const int rounds = (p.vocab + kPartElems - 1) / kPartElems;
  const int c0 = static_cast<int>(static_cast<int64_t>(rounds) * blockIdx.x / p.splits);
  const int c1 = static_cast<int>(static_cast<int64_t>(rounds) * (blockIdx.x + 1) / p.splits);
  const char *src = static_cast<const char *>(p.logits) + row * p.ld * (BF16 ? 2 : 4);
  constexpr int kVec = VEC ? BF16 ? 8 : 4 : 1;  // logits of a load
  auto index = [&](int base, int e) { return base + (e / kVec * kPartThreads + tid) * kVec + e % kVec; };
  // The thread's logits of a round lie in shared memory, in a place of its own that
  // its warp's lanes read when they list candidates; those of the next round are on
  // their way in registers.
  constexpr int kRaw = VEC ? kPerThread / kVec * 4 : kPerThread;
  uint32_t raw[kRaw];
  auto fetch = [&](int c) {  // -inf past the end
    if constexpr (VEC) {
#pragma unroll
      for (int u = 0; u < kPerThread / kVec; ++u) {
        const int i = index(c * kPartElems, u * kVec);
        constexpr uint32_t none = BF16 ? 0xff80ff80u : 0xff800000u;
        uint4 v = make_uint4(none, none, none, none);
        if (i < p.vocab) v = *reinterpret_cast<const uint4 *>(src + static_cast<int64_t>(i) * (BF16 ? 2 : 4));
        raw[4 * u] = v.x, raw[4 * u + 1] = v.y, raw[4 * u + 2] = v.z, raw[4 * u + 3] = v.w;
      }
    } else {
#pragma unroll
      for (int e = 0; e < kPerThread; ++e) {
        const int i = index(c * kPartElems, e);
        raw[e] = BF16 ? 0xff80u : 0xff800000u;
        if (i < p.vocab) {
          if constexpr (BF16)
            raw[e] = reinterpret_cast<const uint16_t *>(src)[i];
          else
            raw[e] = reinterpret_cast<const uint32_t *>(src)[i];
        }
      }
    }
  };
  auto place = [&](int q) { return xs + (q * kPartThreads + tid); };  // elements 4 q .. 4 q + 3
  // Puts the fetched logits in place, f(values) on the way.
  auto keep = [&](auto f) {
#pragma unroll
    for (int q = 0; q < kPerThread / 4; ++q) {
      float4 v;
      if constexpr (VEC && BF16)
        v = make_float4(bf16_bits_to_f32(raw[2 * q] & 0xffffu), __uint_as_float(raw[2 * q] & 0xffff0000u),
                        bf16_bits_to_f32(raw[2 * q + 1] & 0xffffu), __uint_as_float(raw[2 * q + 1] & 0xffff0000u));
      else if constexpr (BF16)
        v = make_float4(bf16_bits_to_f32(raw[4 * q]), bf16_bits_to_f32(raw[4 * q + 1]), bf16_bits_to_f32(raw[4 * q + 2]),
                        bf16_bits_to_f32(raw[4 * q + 3]));
      else
        v = make_float4(__uint_as_float(raw[4 * q]), __uint_as_float(raw[4 * q + 1]), __uint_as_float(raw[4 * q + 2]),
                        __uint_as_float(raw[4 * q + 3]));
      *place(q) = v;
      f(v);
    }
  };
  auto each = [&](auto f) {  // f(e, value) for the thread's elements
#pragma unroll
    for (int q = 0; q < kPerThread / 4; ++q) {
      const float4 v = *place(q);
      f(4 * q, v.x);
      f(4 * q + 1, v.y);
      f(4 * q + 2, v.z);
      f(4 * q + 3, v.w);
    }
  };
  auto clean_all = [&]() {
#pragma unroll 1
    for (int q = 0; q < kPerThread / 4; ++q) {
      const float4 v = *place(q);
      *place(q) = make_float4(clean(v.x), clean(v.y), clean(v.z), clean(v.w));
    }
  };
  if (tid < kBeamMax) best[tid] = 0;
  if (tid == 0) added[0] = added[1] = 0;
  float ref = -INFINITY;  // the sum's reference: the first rounds' maximum
  double sum = 0.0;       // this thread's part of the sum of exp(x - ref)
  // At least W values of earlier rounds are `floor` or more; -inf counts with floored.
  float floor = -INFINITY;
  bool floored = false;

  // The list's n entries and the earlier best are ranked together (all threads):
  // every warp sorts 32 at a time and keeps its 32 best, one warp joins them.
  auto rank_list = [&](int n) {
    const int warp = tid >> 5;
    Key v = warp == 0 ? best[lane] : 0;
    for (int at = 32 * warp; at < n; at += kPartThreads) v = merge32(v, sort32(at + lane < n ? list[at + lane] : 0, lane), lane);
    runs[warp][lane] = v;
    __syncthreads();
    if (warp == 0) {
      for (int w = 1; w < min((n + 31) / 32, kPartThreads / 32); ++w) v = merge32(v, runs[w][lane], lane);
      best[lane] = v;
    }
    __syncthreads();
  };
  // Round c had more values at its bound than the list holds (many equal ones):
  // the same with keys, which are all different.  `before`: entries of earlier rounds.
  auto exact_round = [&](int c, int before) {
    rank_list(before);
    const Key worst = best[W - 1];
    const int base = c * kPartElems;
    fetch(c);
    keep([](const float4 &) {});
    Key km = 0;
    each([&](int e, float v) {
      const int i = index(base, e);
      const Key k = i < p.vocab ? make_key(clean(v), static_cast<uint32_t>(i)) : 0;
      km = k > km ? k : km;
    });
    Key kg = km;
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) {
      const Key y = shfl_xor_key(kg, o);
      kg = y > kg ? y : kg;
    }
    if ((tid & 7) == 0) key_max[tid >> 3] = kg;
    if (tid == 0) ties = listed = 0;
    __syncthreads();
    const Key mykey = key_max[lane];
    int above = 0;
    for (int o = 0; o < 32; ++o) above += key_max[o] > mykey || (key_max[o] == mykey && o < lane);
    const Key bound1 = __shfl_sync(0xffffffffu, mykey, __ffs(__ballot_sync(0xffffffffu, above == W - 1)) - 1);
    if (km && km >= bound1) list[atomicAdd(&ties, 1)] = km;
    __syncthreads();
    const int n1 = ties;
    if (tid == 0 && n1 < W) key_max[0] = 0;  // fewer threads than W: all their keys
    for (int a = tid; a < n1; a += kPartThreads) {
      const Key k = list[a];
      int over = 0;
      for (int z = 0; z < n1; ++z) over += list[z] > k;
      if (over == W - 1) key_max[0] = k;
    }
    __syncthreads();
    const Key bound2 = key_max[0];  // W threads' keys at most lie above it
    each([&](int e, float v) {
      const int i = index(base, e);
      const Key k = make_key(clean(v), static_cast<uint32_t>(i));
      if (i < p.vocab && k >= bound2 && k > worst) list[atomicAdd(&listed, 1)] = k;
    });
    __syncthreads();
    rank_list(listed);
  };
  // Entries, those before the latest round, and what `added` was: every thread
  // keeps the same.  A round's entries are counted by its parity, so that the
  // count can be read while the next round's are being added.
  int n_list = 0, n_before = 0, seen[2] = {0, 0};
  auto count_round = [&](int c) {
    const int now = added[c & 1];
    n_before = n_list;
    n_list += now - (c & 1 ? seen[1] : seen[0]);
    if (c & 1)
      seen[1] = now;
    else
      seen[0] = now;
  };
  fetch(c0);
  for (int c = c0;; ++c) {
    const int base = c * kPartElems;
    float mine = -INFINITY, part = NAN;  // part: the thread's terms of the sum, NaN: not yet
    if (c < c1) {
      // The largest (fmaxf passes over NaN) and, where there is a reference for
      // it, the sum, straight from the registers.
      uint64_t a = f2(0.f, 0.f), b = a;
      const bool known = fabsf(ref) < 64.f;
      if (known) {
        const uint64_t l2 = f2(kLog2e, kLog2e), m2 = f2(-(ref * kLog2e), -(ref * kLog2e));
        keep([&](const float4 &v) {
          mine = fmaxf(fmaxf(fmaxf(mine, v.x), fmaxf(v.y, v.z)), v.w);
          a = add2(a, ex2_2(fma2(f2(v.x, v.y), l2, m2)));
          b = add2(b, ex2_2(fma2(f2(v.z, v.w), l2, m2)));
        });
      } else {
        keep([&](const float4 &v) { mine = fmaxf(fmaxf(fmaxf(mine, v.x), fmaxf(v.y, v.z)), v.w); });
      }
      part = known ? halves(add2(a, b)) : NAN;
      if (c + 1 < c1) fetch(c + 1);
      // +inf is taken out here, NaN where the sum shows it
      auto largest = [&]() {
        float v = -INFINITY;
        each([&](int, float y) { v = fmaxf(v, y); });
        return v;
      };
      if (!(mine < INFINITY)) {
        clean_all();
        mine = largest();
        part = NAN;
      }
      float g = mine;
#pragma unroll
      for (int o = 1; o < 8; o <<= 1) g = fmaxf(g, __shfl_xor_sync(0xffffffffu, g, o));
      if ((tid & 7) == 0) group_max[c & 1][tid >> 3] = g;
    }
    __syncthreads();
    if (c > c0) {
      count_round(c - 1);
      if (n_list > kList / 2 || c == c1) {
        if (n_list > kList) {
          exact_round(c - 1, n_before);
          if (c < c1) {  // the round at hand again
            fetch(c);
            keep([](const float4 &) {});
            clean_all();
            if (c + 1 < c1) fetch(c + 1);
          }
        } else
          rank_list(n_list);
        n_list = 0;
      }
    }
    if (c == c1) break;
    // Every warp for itself: the round's maximum and the W-th largest group maximum.
    const float gm = group_max[c & 1][lane];
    const float top = unordered(__reduce_max_sync(0xffffffffu, ordered(gm)));
    // Where the floor leaves more than a few groups, the round's own bound: its
    // W-th largest group maximum.
    float bound = floor;
    const int over = __popc(__ballot_sync(0xffffffffu, !floored || gm > floor));
    if (!floored || over > W) {
      int rank = 0;
#pragma unroll
      for (int o = 0; o < 32; ++o) {
        const float y = group_max[c & 1][o];
        rank += y > gm || (y == gm && o < lane);
      }
      bound = __shfl_sync(0xffffffffu, gm, __ffs(__ballot_sync(0xffffffffu, rank == W - 1)) - 1);
    }
    // The sum, against a reference that moves only where a term could overflow.
    if (top > -INFINITY && !(top < ref + 40.f)) {
      if (ref > -INFINITY) sum *= exp(static_cast<double>(ref) - top);
      ref = top;
      part = NAN;
    }
    if (ref > -INFINITY) {
      const bool near = fabsf(ref) < 64.f;
      auto terms = [&]() {  // 0 where x is -inf
        if (!near) {  // far from 0: the difference first
          float d = 0.f;
          each([&](int, float y) { d += ex2((y - ref) * kLog2e); });
          return d;
        }
        const uint64_t l2 = f2(kLog2e, kLog2e), m2 = f2(-(ref * kLog2e), -(ref * kLog2e));
        uint64_t a = f2(0.f, 0.f), b = a;
#pragma unroll
        for (int q = 0; q < kPerThread / 4; ++q) {
          const float4 v = *place(q);
          a = add2(a, ex2_2(fma2(f2(v.x, v.y), l2, m2)));
          b = add2(b, ex2_2(fma2(f2(v.z, v.w), l2, m2)));
        }
        return halves(add2(a, b));
      };
      if (isnan(part)) part = terms();
      if (isnan(part)) {
        clean_all();
        part = terms();
      }
      // 2^(m' - m log2e') to first order: the difference is below 2^-18
      const double fix = near ? 1.0 + (static_cast<double>(ref * kLog2e) - static_cast<double>(ref) * static_cast<double>(kLog2e)) * 0.6931471805599453 : 1.0;
      sum += static_cast<double>(part) * fix;
    }
    // Values below this round's bound are out, and those not above the floor:
    // W earlier ones go before them.
    // The threads that hold one, one after the other: a lane for each of the
    // thread's elements, which the thread itself may have put in place after the
    // round's synchronisation.
    __syncwarp();
    const float *xf = reinterpret_cast<const float *>(xs);
    for (unsigned who = __ballot_sync(0xffffffffu, mine >= bound && (!floored || mine > floor) && index(base, 0) < p.vocab); who; who &= who - 1) {
      const int t = (tid & ~31) + __ffs(who) - 1;
      const int i = base + (lane / kVec * kPartThreads + t) * kVec + lane % kVec;
      const float v = clean(xf[(lane / 4 * kPartThreads + t) * 4 + lane % 4]);
      if (v >= bound && (!floored || v > floor) && i < p.vocab) {
        const int at = n_list + atomicAdd(&added[c & 1], 1) - (c & 1 ? seen[1] : seen[0]);
        if (at < kList) list[at] = make_key(v, static_cast<uint32_t>(i));
      }
    }
    __syncwarp();
    const bool full = base + kPartThreads * kVec <= p.vocab;  // every group has a value of the row
    if ((full && !floored) || bound > floor) floor = bound, floored = true;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (lane == 0) sums[tid >> 5] = sum;
  __syncthreads();
  const int64_t at = static_cast<int64_t>(row) * p.splits + blockIdx.x;
  if (tid < W) p.part_keys[at * W + tid] = best[tid];
  if (tid == 0) {
    double s = 0.0;
#pragma unroll
    for (int w = 0; w < kPartThreads / 32; ++w) s += sums[w];
    p.part_max[at] = ref;
    p.part_sum[at] = s;
  }
}

__device__ __forceinline__ Key ordered64(double x) {  // never 0; -0 as +0
  const Key u = static_cast<Key>(__double_as_longlong(x + 0.0));
  return u >> 63 ? ~u : u | Key{1} << 63;
}
__device__ __forceinline__ double unordered64(Key u) { return __longlong_as_double(static_cast<long long>(u >> 63 ? u & ~(Key{1} << 63) : ~u)); }

// One utterance, a warp a beam: the beam's log sum exp and its W best from its
// parts' sorted lists, merged.  Then one warp takes the best head of the beams'
// lists (a lane each) W times.  Better scores go first, then lower beams; within
// a beam the keys' order is that of the scores.  Latency: one utterance of 4
// beams 4.8 us, 64 of 8 beams 5.8, 8 of 32 beams 8.9; with one warp over all parts'
// lists 32 beams over 200000 tokens took 250 us a step, this way 37.
__global__ void __launch_bounds__(32 * kBeamMax) beam_join_kernel(const __grid_constant__ BeamParams p) {
  __shared__ ulonglong2 lists[kBeamMax][kBeamMax];  // [beam][rank]: score (0: none), key
  __shared__ bool over[kBeamMax];  // out_finished may be finished: it is read before any is written
  pdl_wait();
  pdl_trigger();
  const int W = p.beams, S = p.splits, b = blockIdx.x, k = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int row = b * W + k;
  const bool fin = p.finished && p.finished[row];
  const float given = p.scores[row];
  const double base = isnan(given) ? -INFINITY : static_cast<double>(given);
  Key key = 0;
  double lse = 0.0;
  if (fin) {  // its row was not read
    if (lane == 0) key = static_cast<Key>(~static_cast<uint32_t>(p.eos)) | Key{1} << 63;
  } else {
    const Key *keys = p.part_keys + static_cast<int64_t>(row) * S * W;
    double sum = 0.0;
    float m = -INFINITY;
    if (lane < S) {
      m = p.part_max[static_cast<int64_t>(row) * S + lane];
      sum = p.part_sum[static_cast<int64_t>(row) * S + lane];
    }
    // Short lists are taken together, 32 keys at a time (a sort and a join for
    // them all), long ones one by one (a join each).
    const int step = W <= 8 ? 32 : W, runs = W <= 8 ? (S * W + 31) / 32 : S;
    constexpr int kAhead = 4;
    for (int run = 0; run < runs; run += kAhead) {
      Key y[kAhead];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) y[i] = lane < step && (run + i) * step + lane < S * W ? keys[(run + i) * step + lane] : 0;
#pragma unroll
      for (int i = 0; i < kAhead; ++i)
        if (run + i < runs) {
          const Key z = W <= 8 ? sort32(y[i], lane) : y[i];
          key = run + i ? merge32(key, z, lane) : z;
        }
    }
    float top = m;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    sum = m > -INFINITY ? (m == top ? sum : sum * exp(static_cast<double>(m) - top)) : 0.0;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    lse = static_cast<double>(top) + log(sum);
  }
  const float x = unordered(static_cast<uint32_t>(key >> 32));
  // every logit -inf: there is no sum, and the candidates count as -inf
  const double s = fin ? base : x > -INFINITY ? base + (static_cast<double>(x) - lse) : -INFINITY;
  if (lane == 0) over[k] = fin;
  lists[k][lane] = make_ulonglong2(key ? ordered64(isnan(s) ? -INFINITY : s) : 0, key);
  __syncthreads();
  if (k) return;
  // The lane's beam: its best candidate that is left, and that one's rank.
  ulonglong2 head = lane < W ? lists[lane][0] : make_ulonglong2(0, 0);
  int rank = 0, parent = 0;
  ulonglong2 mine = make_ulonglong2(0, 0);  // the lane-th of the chosen
  for (int r = 0; r < W; ++r) {
    const uint32_t hi = __reduce_max_sync(0xffffffffu, static_cast<uint32_t>(head.x >> 32));
    const bool most = static_cast<uint32_t>(head.x >> 32) == hi;
    const uint32_t lo = __reduce_max_sync(0xffffffffu, most ? static_cast<uint32_t>(head.x) : 0u);
    const int who = __ffs(__ballot_sync(0xffffffffu, most && static_cast<uint32_t>(head.x) == lo)) - 1;
    const Key chosen = __shfl_sync(0xffffffffu, head.y, who);
    if (lane == r) parent = who, mine = make_ulonglong2(static_cast<Key>(hi) << 32 | lo, chosen);
    if (lane == who) head = ++rank < W ? lists[lane][rank] : make_ulonglong2(0, 0);
  }
  if (lane < W) {
    const int out = b * W + lane, t = static_cast<int>(~static_cast<uint32_t>(mine.y));
    p.out_scores[out] = static_cast<float>(unordered64(mine.x));
    p.out_parents[out] = b * W + parent;
    p.out_tokens[out] = t;
    if (p.out_finished) p.out_finished[out] = over[parent] || t == p.eos;
  }
}

// dst[r] = src[parents[r]] into other memory: a warp a row and 2 KB of it, all of
// it under way before any is stored.  Latency at a step's sizes:
// 512 rows of four states 4.5 us.
constexpr int kCopyBytes = 2048;
template <typename T>
__global__ void __launch_bounds__(256) beam_gather_kernel(const __grid_constant__ ReorderParams p) {
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x & 31;
  const int64_t unit = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  const int r = static_cast<int>(unit % p.rows);
  const int strip = static_cast<int>(unit / p.rows);
  if (strip >= p.strip0[p.count]) return;
  int i = 0;
  while (i + 1 < p.count && strip >= p.strip0[i + 1]) ++i;
  const int64_t lo = static_cast<int64_t>(strip - p.strip0[i]) * kCopyBytes;
  const int64_t left = p.row_bytes[i] - lo;
  const int n = static_cast<int>((left < kCopyBytes ? left : kCopyBytes) / static_cast<int>(sizeof(T)));
  int from = p.parents[r];
  if (from < 0 || from >= p.rows) from = r;  // out of range: the row's own
  const T *src = reinterpret_cast<const T *>(static_cast<const char *>(p.src[i]) + from * p.src_ld[i] + lo);
  T *dst = reinterpret_cast<T *>(static_cast<char *>(p.dst[i]) + r * p.dst_ld[i] + lo);
  if constexpr (sizeof(T) == 16) {
    T v[kCopyBytes / 512];
#pragma unroll
    for (int u = 0; u < kCopyBytes / 512; ++u)
      if (lane + 32 * u < n) v[u] = src[lane + 32 * u];
#pragma unroll
    for (int u = 0; u < kCopyBytes / 512; ++u)
      if (lane + 32 * u < n) dst[lane + 32 * u] = v[u];
  } else {
    for (int x = lane; x < n; x += 32) dst[x] = src[x];
  }
}

// The same in place (or between any two): a CTA holds one strip of every row of one
// state, and reads all rows before it writes any.  512 rows of four states of 640
// f32: 4.8 us in a stream (into other memory 2.9).
template <typename T>
__global__ void __launch_bounds__(256) beam_reorder_kernel(const __grid_constant__ ReorderParams p) {
  extern __shared__ __align__(16) uint8_t strip_raw[];
  T *strip = reinterpret_cast<T *>(strip_raw);
  pdl_wait();
  pdl_trigger();
  int i = 0;
  while (i + 1 < p.count && static_cast<int>(blockIdx.x) >= p.strip0[i + 1]) ++i;
  const int64_t lo = static_cast<int64_t>(blockIdx.x - p.strip0[i]) * p.strip_bytes;
  const int64_t left = p.row_bytes[i] - lo;
  const int n = static_cast<int>((left < p.strip_bytes ? left : p.strip_bytes) / static_cast<int>(sizeof(T)));
  const char *src = static_cast<const char *>(p.src[i]) + lo;
  char *dst = static_cast<char *>(p.dst[i]) + lo;
  for (int x = threadIdx.x; x < n * p.rows; x += blockDim.x) {
    const int r = x / n, c = x - r * n;
    int from = p.parents[r];
    if (from < 0 || from >= p.rows) from = r;  // out of range: the row stays
    strip[x] = reinterpret_cast<const T *>(src + from * p.src_ld[i])[c];
  }
  __syncthreads();
  for (int x = threadIdx.x; x < n * p.rows; x += blockDim.x) {
    const int r = x / n, c = x - r * n;
    reinterpret_cast<T *>(dst + r * p.dst_ld[i])[c] = strip[x];
  }
}

}  // namespace

// CTAs of a row: one wave of four CTAs an SM, each with at least one round of logits.
int beam_splits(int sm_count, int rows, int vocab) {
  const int rounds = (vocab + kPartElems - 1) / kPartElems;
  int s = 4 * sm_count / (rows > 0 ? rows : 1);
  s = s < rounds ? s : rounds;
  return s < 1 ? 1 : s > kBeamSplitsMax ? kBeamSplitsMax : s;
}
size_t beam_workspace(int rows, int beams, int splits) {
  return static_cast<size_t>(rows) * splits * (static_cast<size_t>(beams) * 8 + 8 + 4);
}

cudaError_t launch_beam_select(const BeamParams &p, cudaStream_t s) {
  const int rows = p.items * p.beams;
  const bool vec = (reinterpret_cast<uintptr_t>(p.logits) | static_cast<uintptr_t>(p.ld * (p.bf16 ? 2 : 4))) % 16 == 0 &&
                   p.vocab % (p.bf16 ? 8 : 4) == 0;
  const dim3 grid(p.splits, rows);
  constexpr size_t smem = kPartElems * 4;
  static_assert(smem + 16 * 1024 <= 48 * 1024, "no attribute is needed");
  cudaError_t e = p.bf16 ? vec ? launch_pdl(beam_part_kernel<true, true>, grid, dim3(kPartThreads), smem, s, 1, p)
                               : launch_pdl(beam_part_kernel<true, false>, grid, dim3(kPartThreads), smem, s, 1, p)
                  : vec ? launch_pdl(beam_part_kernel<false, true>, grid, dim3(kPartThreads), smem, s, 1, p)
                        : launch_pdl(beam_part_kernel<false, false>, grid, dim3(kPartThreads), smem, s, 1, p);
  if (e != cudaSuccess) return e;
  return launch_pdl(beam_join_kernel, dim3(p.items), dim3(32 * p.beams), 0, s, 1, p);
}

cudaError_t launch_beam_reorder(ReorderParams &p, cudaStream_t s) {
  uint64_t bits = 0;
  for (int i = 0; i < p.count; ++i)
    bits |= reinterpret_cast<uintptr_t>(p.src[i]) | reinterpret_cast<uintptr_t>(p.dst[i]) | static_cast<uint64_t>(p.row_bytes[i]) |
            static_cast<uint64_t>(p.src_ld[i]) | static_cast<uint64_t>(p.dst_ld[i]);
  bool in_place = false;
  for (int i = 0; i < p.count; ++i) in_place |= p.src[i] == p.dst[i];
  if (!in_place) {
    int n = 0;
    for (int i = 0; i < p.count; ++i) {
      p.strip0[i] = n;
      n += static_cast<int>((p.row_bytes[i] + kCopyBytes - 1) / kCopyBytes);
    }
    p.strip0[p.count] = n;
    const int64_t blocks = (static_cast<int64_t>(n) * p.rows + 7) / 8;
    if (blocks <= INT32_MAX) {
      auto go = [&](auto kern) { return launch_pdl(kern, dim3(static_cast<unsigned>(blocks)), dim3(256), 0, s, 1, static_cast<const ReorderParams &>(p)); };
      return bits % 16 == 0 ? go(beam_gather_kernel<uint4>) : bits % 4 == 0 ? go(beam_gather_kernel<uint32_t>) : bits % 2 == 0 ? go(beam_gather_kernel<uint16_t>) : go(beam_gather_kernel<uint8_t>);
    }
  }
  // strips of about 16 KB over all rows, of 16 bytes of a row at least
  int strip = 16384 / p.rows / 16 * 16;
  p.strip_bytes = strip < 16 ? 16 : strip;
  int n = 0;
  for (int i = 0; i < p.count; ++i) {
    p.strip0[i] = n;
    n += static_cast<int>((p.row_bytes[i] + p.strip_bytes - 1) / p.strip_bytes);
  }
  p.strip0[p.count] = n;
  const size_t smem = static_cast<size_t>(p.rows) * p.strip_bytes;
  auto go = [&](auto kern) {
    if (smem > 48 * 1024) {
      const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kReorderMaxRows * 16);
      if (e != cudaSuccess) return e;
    }
    return launch_pdl(kern, dim3(n), dim3(256), smem, s, 1, static_cast<const ReorderParams &>(p));
  };
  return bits % 16 == 0 ? go(beam_reorder_kernel<uint4>) : bits % 4 == 0 ? go(beam_reorder_kernel<uint32_t>) : bits % 2 == 0 ? go(beam_reorder_kernel<uint16_t>) : go(beam_reorder_kernel<uint8_t>);
}

}  // namespace nq
