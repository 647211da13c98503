// nq8_beam.cu -- beam search: the best continuations of an utterance's beams
// by log probability, and the reordering of what each beam carries.
//
// score(b, k, t) = scores[b][k] + x[t] - log sum_u exp(x[u]) over the row x of
// logits; of all beams and tokens the `beams` best, equal scores by beam, then
// token.  The sum of a row does not change the order within it, so one pass
// over the logits makes, per part of a row, its maximum, its sum of
// exponentials and its `beams` best values (beam_part_kernel); a second, small
// launch joins the parts and compares across beams in f64 (beam_join_kernel):
// the terms of a sum are f32, everything added up is f64, so that candidates
// of two beams compare as their exact scores do up to about 1e-8.
//
// Selection of the W best of a part without sorting it: the values are kept as
// keys (ordered value, inverted index), all different.  The W-th largest of
// the maxima of 32 thread groups bounds the W-th largest key from below, the
// W-th largest of the thread maxima above that bound does so more closely, and
// only W threads hold keys above the second bound: at most 16 W keys, ranked
// by counting.  Nothing depends on the values' distribution but the count.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include "nq8_cache.h"

namespace nq {
namespace {

using Key = unsigned long long;
constexpr int kPartThreads = 256;
constexpr int kPerThread = 16;
constexpr int kPartElems = kPartThreads * kPerThread;  // logits of one round of a CTA
constexpr int kBeamSplitsMax = 16;

// An f32 as an unsigned integer of the same order.
__device__ __forceinline__ uint32_t ordered(float x) {
  const uint32_t u = __float_as_uint(x);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float unordered(uint32_t u) {
  return __uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~u);
}
__device__ __forceinline__ Key make_key(float x, uint32_t index) {
  return static_cast<Key>(ordered(x)) << 32 | static_cast<uint32_t>(~index);
}
__device__ __forceinline__ Key shfl_xor_key(Key v, int o) { return __shfl_xor_sync(0xffffffffu, v, o); }

// NaN and +inf count as -inf; -0 as +0.
__device__ __forceinline__ float clean(float x) { return x < INFINITY ? x + 0.f : -INFINITY; }

// One part of one row: CTA (blockIdx.x of `splits`, row blockIdx.y).
template <bool BF16, bool VEC>
__global__ void __launch_bounds__(kPartThreads) beam_part_kernel(const __grid_constant__ BeamParams p) {
  __shared__ Key group_max[32];
  __shared__ Key list[kBeamMax * kPerThread > kPartThreads ? kBeamMax * kPerThread : kPartThreads];
  __shared__ Key best[2][kBeamMax];
  __shared__ int counts[4];
  __shared__ double sums[kPartThreads / 32];
  pdl_wait();
  pdl_trigger();
  const int row = blockIdx.y, tid = threadIdx.x, lane = tid & 31;
  const int W = p.beams;
  if (p.finished && p.finished[row]) return;
  const int rounds = (p.vocab + kPartElems - 1) / kPartElems;
  const int c0 = static_cast<int>(static_cast<int64_t>(rounds) * blockIdx.x / p.splits);
  const int c1 = static_cast<int>(static_cast<int64_t>(rounds) * (blockIdx.x + 1) / p.splits);
  const char *src = static_cast<const char *>(p.logits) + row * p.ld * (BF16 ? 2 : 4);
  constexpr int kVec = BF16 ? 8 : 4;

  float run_max = -INFINITY;
  double run_sum = 0.0;  // of exp(x - run_max), over the CTA's rounds (thread 0)
  if (tid < kBeamMax) best[0][tid] = 0;
  int cur = 0;
  for (int c = c0; c < c1; ++c) {
    const int base = c * kPartElems;
    float x[kPerThread];
    auto index = [&](int e) { return base + (e / kVec * kPartThreads + tid) * kVec + e % kVec; };
#pragma unroll
    for (int u = 0; u < kPerThread / kVec; ++u) {
      const int i = index(u * kVec);
      if (VEC && i + kVec <= p.vocab) {
        const uint4 w = __ldg(reinterpret_cast<const uint4 *>(src + static_cast<int64_t>(i) * (BF16 ? 2 : 4)));
        const uint32_t r[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if constexpr (BF16) {
            x[u * kVec + 2 * e] = bf16_bits_to_f32(r[e] & 0xffffu);
            x[u * kVec + 2 * e + 1] = __uint_as_float(r[e] & 0xffff0000u);
          } else {
            x[u * kVec + e] = __uint_as_float(r[e]);
          }
        }
      } else {
#pragma unroll
        for (int e = 0; e < kVec; ++e) {
          float y = -INFINITY;
          if (i + e < p.vocab) {
            if constexpr (BF16)
              y = __bfloat162float(reinterpret_cast<const __nv_bfloat16 *>(src)[i + e]);
            else
              y = reinterpret_cast<const float *>(src)[i + e];
          }
          x[u * kVec + e] = y;
        }
      }
    }
    // The thread's largest key: larger value first, then lower index.
    Key mine = 0;
#pragma unroll
    for (int e = 0; e < kPerThread; ++e) {
      x[e] = clean(x[e]);
      const int i = index(e);
      if (i < p.vocab) {
        const Key k = make_key(x[e], static_cast<uint32_t>(i));
        mine = k > mine ? k : mine;
      }
    }
    Key g = mine;
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) {
      const Key y = shfl_xor_key(g, o);
      g = y > g ? y : g;
    }
    if ((tid & 7) == 0) group_max[tid >> 3] = g;
    if (tid < 2) counts[tid] = 0;
    __syncthreads();
    // Every warp for itself: the round's maximum, and the W-th largest group maximum.
    const Key gm = group_max[lane];
    int rank = 0;
    Key top = gm;
#pragma unroll
    for (int o = 0; o < 32; ++o) rank += group_max[o] > gm || (group_max[o] == gm && o < lane);
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const Key y = shfl_xor_key(top, o);
      top = y > top ? y : top;
    }
    const Key bound1 = __shfl_sync(0xffffffffu, gm, __ffs(__ballot_sync(0xffffffffu, rank == W - 1)) - 1);
    const float new_max = fmaxf(run_max, unordered(static_cast<uint32_t>(top >> 32)));
    // Sum of exponentials.
    float part = 0.f;
    if (new_max > -INFINITY) {
#pragma unroll
      for (int e = 0; e < kPerThread; ++e) part += expf(x[e] - new_max);  // 0 where x is -inf
    }
    double d = part;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) d += __shfl_xor_sync(0xffffffffu, d, o);
    if (lane == 0) sums[tid >> 5] = d;
    const Key floor_key = best[cur][W - 1];  // the W-th best of earlier rounds
    const bool select = top > floor_key;
    if (select && mine >= bound1 && mine) list[atomicAdd(&counts[0], 1)] = mine;
    __syncthreads();
    if (tid == 0 && new_max > -INFINITY) {
      double s = 0.0;
#pragma unroll
      for (int w = 0; w < kPartThreads / 32; ++w) s += sums[w];
      run_sum = (run_max > -INFINITY ? run_sum * exp(static_cast<double>(run_max) - new_max) : 0.0) + s;
    }
    run_max = new_max;
    if (select) {
      // W-th largest of the listed thread maxima (all different), 0 if fewer
      const int n1 = counts[0];
      if (tid == 0 && n1 < W) group_max[0] = 0;  // group_max is free now: it carries the second bound
      for (int a = tid; a < n1; a += kPartThreads) {
        const Key k = list[a];
        int above = 0;
        for (int z = 0; z < n1; ++z) above += list[z] > k;
        if (above == W - 1) group_max[0] = k;
      }
      __syncthreads();
      const Key bound2 = group_max[0] > floor_key ? group_max[0] : floor_key;
#pragma unroll
      for (int e = 0; e < kPerThread; ++e) {
        const int i = index(e);
        if (i >= p.vocab) continue;
        const Key k = make_key(x[e], static_cast<uint32_t>(i));
        if (k >= bound2 && k > floor_key) list[atomicAdd(&counts[1], 1)] = k;
      }
      if (tid < kBeamMax) best[cur ^ 1][tid] = 0;
      __syncthreads();
      const int n2 = counts[1];
      // Rank among this round's keys and the earlier best.
      for (int a = tid; a < n2 + W; a += kPartThreads) {
        const Key k = a < n2 ? list[a] : best[cur][a - n2];
        if (k == 0) continue;
        int above = 0;
        for (int z = 0; z < n2; ++z) above += list[z] > k;
        for (int z = 0; z < W; ++z) above += best[cur][z] > k;
        if (above < W) best[cur ^ 1][above] = k;
      }
      cur ^= 1;
    }
    __syncthreads();
  }
  const int64_t at = static_cast<int64_t>(row) * p.splits + blockIdx.x;
  if (tid < W) p.part_keys[at * W + tid] = best[cur][tid];
  if (tid == 0) {
    p.part_max[at] = run_max;
    p.part_sum[at] = run_sum;
  }
}

// One utterance: warp k joins beam k's parts, warp 0 the beams.
__global__ void __launch_bounds__(32 * kBeamMax) beam_join_kernel(const __grid_constant__ BeamParams p) {
  extern __shared__ __align__(8) Key parts[];  // [beams][splits][beams]
  __shared__ double score[kBeamMax][kBeamMax];
  __shared__ int token[kBeamMax][kBeamMax];
  __shared__ int have[kBeamMax];
  pdl_wait();
  pdl_trigger();
  const int W = p.beams, S = p.splits, b = blockIdx.x, k = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int row = b * W + k;
  const bool done = p.finished && p.finished[row];
  const float base = p.scores[row];
  Key *mine = parts + static_cast<int64_t>(k) * S * W;
  if (done) {
    if (lane == 0) {
      score[k][0] = isnan(base) ? -INFINITY : static_cast<double>(base);
      token[k][0] = p.eos;
      have[k] = 1;
    }
  } else {
    for (int x = lane; x < S * W; x += 32) mine[x] = p.part_keys[static_cast<int64_t>(row) * S * W + x];
    // log sum exp of the row
    const float m = lane < S ? p.part_max[static_cast<int64_t>(row) * S + lane] : -INFINITY;
    float top = m;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    double sum = 0.0;
    if (m > -INFINITY) sum = p.part_sum[static_cast<int64_t>(row) * S + lane] * exp(static_cast<double>(m) - top);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    const double lse = static_cast<double>(top) + log(sum);
    __syncwarp();
    // W times the largest head of the parts' lists (lane: a part)
    int at = 0, found = 0;
    for (int r = 0; r < W; ++r) {
      const Key head = lane < S && at < W ? mine[lane * W + at] : 0;
      Key best = head;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        const Key y = shfl_xor_key(best, o);
        best = y > best ? y : best;
      }
      if (best == 0) break;  // fewer tokens than beams
      if (head == best) ++at;
      if (lane == 0) {
        const float x = unordered(static_cast<uint32_t>(best >> 32));
        // every logit -inf: the sum is none, and the candidates count as -inf
        const double s = x > -INFINITY ? static_cast<double>(base) + (static_cast<double>(x) - lse) : -INFINITY;
        score[k][r] = isnan(s) || isnan(base) ? -INFINITY : s;
        token[k][r] = static_cast<int>(~static_cast<uint32_t>(best));
      }
      ++found;
    }
    if (lane == 0) have[k] = found;
  }
  __syncthreads();
  if (k) return;
  int at = 0;
  const int n = lane < W ? have[lane] : 0;
  const bool was = lane < W && p.finished && p.finished[b * W + lane];  // before the outputs, which may lie there
  for (int r = 0; r < W; ++r) {
    double s = at < n ? score[lane][at] : -INFINITY;
    int who = at < n ? lane : 64;  // past every beam
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const double y = __shfl_xor_sync(0xffffffffu, s, o);
      const int z = __shfl_xor_sync(0xffffffffu, who, o);
      if (y > s || (y == s && z < who)) {
        s = y;
        who = z;
      }
    }
    if (lane == who) {
      const int t = token[lane][at];
      const int out = b * W + r;
      p.out_scores[out] = static_cast<float>(s);
      p.out_parents[out] = b * W + lane;
      p.out_tokens[out] = t;
      if (p.out_finished) p.out_finished[out] = was || t == p.eos;
      ++at;
    }
  }
}

// dst[r] = src[parents[r]]: a CTA holds one strip of every row of one state,
// and reads all rows before it writes any, so dst may be src.
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
    int from = __ldg(p.parents + r);
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

// CTAs of a row: enough that all rows' CTAs fill the GPU four times over, each
// with at least one round of logits.
int beam_splits(int sm_count, int rows, int vocab) {
  const int rounds = (vocab + kPartElems - 1) / kPartElems;
  int s = (4 * sm_count + rows - 1) / (rows > 0 ? rows : 1);
  s = s < rounds ? s : rounds;
  return s < 1 ? 1 : s > kBeamSplitsMax ? kBeamSplitsMax : s;
}
size_t beam_workspace(int rows, int beams, int splits) {
  return static_cast<size_t>(rows) * splits * (static_cast<size_t>(beams) * 8 + 8 + 4);
}

cudaError_t launch_beam_select(const BeamParams &p, cudaStream_t s) {
  const int rows = p.items * p.beams;
  const bool vec = (reinterpret_cast<uintptr_t>(p.logits) | static_cast<uintptr_t>(p.ld * (p.bf16 ? 2 : 4))) % 16 == 0;
  const dim3 grid(p.splits, rows);
  cudaError_t e = p.bf16 ? vec ? launch_pdl(beam_part_kernel<true, true>, grid, dim3(kPartThreads), 0, s, 1, p)
                               : launch_pdl(beam_part_kernel<true, false>, grid, dim3(kPartThreads), 0, s, 1, p)
                  : vec ? launch_pdl(beam_part_kernel<false, true>, grid, dim3(kPartThreads), 0, s, 1, p)
                        : launch_pdl(beam_part_kernel<false, false>, grid, dim3(kPartThreads), 0, s, 1, p);
  if (e != cudaSuccess) return e;
  const size_t smem = static_cast<size_t>(p.beams) * p.splits * p.beams * 8;
  if (smem > 32 * 1024) {  // next to the kernel's static arrays
    e = cudaFuncSetAttribute(beam_join_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kBeamMax * kBeamSplitsMax * kBeamMax * 8);
    if (e != cudaSuccess) return e;
  }
  return launch_pdl(beam_join_kernel, dim3(p.items), dim3(32 * p.beams), smem, s, 1, p);
}

cudaError_t launch_beam_reorder(ReorderParams &p, cudaStream_t s) {
  uint64_t bits = 0;
  for (int i = 0; i < p.count; ++i)
    bits |= reinterpret_cast<uintptr_t>(p.src[i]) | reinterpret_cast<uintptr_t>(p.dst[i]) | static_cast<uint64_t>(p.row_bytes[i]) |
            static_cast<uint64_t>(p.src_ld[i]) | static_cast<uint64_t>(p.dst_ld[i]);
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
