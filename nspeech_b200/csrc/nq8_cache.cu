// nq8_cache.cu -- the pages of a key / value cache: room for new tokens,
// forking, copying on write, freeing, compacting, and the tokens' entry.
//
// A slot's sequence is a row of page numbers and a length; pages carry a count
// of the slots that hold them.  All of it lives on the device and every call
// is a fixed number of launches, so a decoding step can be captured into a
// graph.  Results depend on the order of slots alone: pages are given out
// lowest number first, and counts are integers, so atomics' order is not seen.
// A call that cannot be done changes nothing and sets a status bit; later
// calls then do nothing until the host has read the status.
// Kernels start before the one ahead of them has ended and wait for it, so
// what that one may write (keys and values, offsets, sources) is read by plain
// loads: the read-only path holds for data that stays as it is for a kernel's
// whole life.
#include <cuda_runtime.h>
#include <stdint.h>

#include "nq8_cache.h"

namespace nq {
namespace {

constexpr int kBlock = 1024;

__device__ __forceinline__ int *copies_of(const CacheView &c) { return c.state + kStateLists; }
__device__ __forceinline__ int *list_of(const CacheView &c, int i) {
  return c.state + kStateLists + 3 * static_cast<int64_t>(c.slots) + i * static_cast<int64_t>(c.pages);
}

// Exclusive prefix sum over the block (kBlock threads); all: the total.
__device__ __forceinline__ int block_scan(int x, int *warp_sums, int &all) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int upto = x;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += y;
  }
  __syncthreads();  // the previous scan's sums are read
  if (lane == 31) warp_sums[warp] = upto;
  __syncthreads();
  int w = warp_sums[lane];
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, w, o);
    if (lane >= o) w += y;
  }
  all = __shfl_sync(0xffffffffu, w, 31);
  const int before = __shfl_sync(0xffffffffu, w, warp > 0 ? warp - 1 : 0);
  return upto - x + (warp > 0 ? before : 0);
}

// Tokens that slot i of a call gets: offsets[i + 1] - offsets[i], or `uniform`.
__device__ __forceinline__ int count_of(const int *offsets, int uniform, int i) {
  return offsets ? max(0, offsets[i + 1] - offsets[i]) : uniform;
}

// One bit per page, set where refs > 0, by whole warps.
__device__ __forceinline__ void held_bits(const CacheView &c, uint32_t *bits) {
  const int lane = threadIdx.x & 31;
  const int words = (c.pages + 31) / 32;
  constexpr int U = 8;  // loads in flight a thread
  for (int w = (threadIdx.x >> 5) * U; w < words; w += kBlock / 32 * U) {
    int r[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int page = (w + u) * 32 + lane;
      r[u] = page < c.pages ? c.refs[page] : 1;  // past the end: not free
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint32_t m = __ballot_sync(0xffffffffu, r[u] > 0);
      if (lane == 0 && w + u < words) bits[w + u] = m;
    }
  }
}

// Room for the new tokens of slots [first, first + n): one CTA.
// Shared: held bits of all pages, and per slot its shared last page (-1: none,
// or it may keep it) and the rank of its first new page.  One CTA, because
// "lowest free page first, in slot order" is one scan over all of them; bound by
// latency (counts, lengths and tables, three scans, the rows' new entries): 64
// slots 7.6 to 9 us by itself, of which its neighbours in the stream cover some.
// Holders of a shared last page are counted by looking at all slots of the call
// for each: where every slot shares one, 64 slots 9 us, 512 26, 4096 664 (with
// the copies' launch).
__global__ void __launch_bounds__(kBlock) cache_reserve_kernel(const CacheView c, const int *offsets, int uniform, int first, int n) {
  extern __shared__ uint32_t sh[];
  __shared__ int sums[32];
  __shared__ int bad, copies;
  const int words = (c.pages + 31) / 32;
  uint32_t *bits = sh;
  int *tail = reinterpret_cast<int *>(sh + words), *start = tail + n;
  pdl_wait();
  pdl_trigger();
  const int status = c.state[kStateStatus];
  const int P = 1 << c.page_shift;
  const int64_t room = static_cast<int64_t>(c.max_pages) << c.page_shift;
  if (threadIdx.x == 0) copies = 0, bad = status;
  held_bits(c, bits);
  for (int i = threadIdx.x; i < n; i += kBlock) {
    const int old = c.lens[first + i], add = count_of(offsets, uniform, i);
    int t = -1;
    if (add > 0 && (old & (P - 1)) && old > 0 && old <= room) {
      t = c.table[static_cast<int64_t>(first + i) * c.max_pages + (old >> c.page_shift)];
      if (t < 0 || t >= c.pages || c.refs[t] <= 1) t = -1;  // a page of its own
    }
    tail[i] = t;
  }
  __syncthreads();
  // The pages that each slot takes, in the slots' order.
  int total = 0;
  for (int base = 0; base < n; base += kBlock) {
    const int i = base + threadIdx.x;
    int need = 0, copy = 0;
    if (i < n) {
      const int old = c.lens[first + i], add = count_of(offsets, uniform, i), t = tail[i];
      if (t >= 0) {
        // the last holder keeps the page where every holder of it appends
        int same = 0, later = 0;
        for (int j = 0; j < n; ++j) {
          const int e = tail[j] == t;
          same += e;
          later |= e && j > i;
        }
        copy = c.refs[t] != same || later;
      }
      if (old < 0 || old + static_cast<int64_t>(add) > room) {
        bad = kCacheSlotFull;
      } else {
        need = ((old + add + P - 1) >> c.page_shift) - ((old + P - 1) >> c.page_shift) + copy;
        need = min(need, c.pages + 1);  // more than there are: the block's sum stays in range
      }
    }
    int all;
    const int at = block_scan(need, sums, all);
    if (i < n) start[i] = ((total + at) << 1) | copy;
    total += all;
    if (total > c.pages) total = c.pages + 1;  // cannot be met; keeps the sum in range
  }
  int free_pages = 0;
  {
    int mine = 0, all;
    for (int w = threadIdx.x; w < words; w += kBlock) mine += __popc(~bits[w]);
    block_scan(mine, sums, all);
    free_pages = all;
  }
  __syncthreads();
  if (bad || total > free_pages) {
    if (threadIdx.x == 0) {
      if (!status) c.state[kStateStatus] = bad ? bad : kCacheOutOfPages;
      c.state[kStateCopies] = 0;
    }
    return;
  }
  // The `total` lowest free pages in order.
  int *list = list_of(c, 0);
  for (int base = 0, done = 0; base < words && done < total; base += kBlock) {
    const int w = base + threadIdx.x;
    uint32_t m = w < words ? ~bits[w] : 0u;
    int all;
    int at = done + block_scan(__popc(m), sums, all);
    for (; m && at < total; m &= m - 1) list[at++] = w * 32 + __ffs(m) - 1;
    done += all;
  }
  __syncthreads();
  int *cp = copies_of(c);
  const int lane = threadIdx.x & 31;
  for (int i = threadIdx.x >> 5; i < n; i += kBlock / 32) {
    const int old = c.lens[first + i], add = count_of(offsets, uniform, i), copy = start[i] & 1, at = start[i] >> 1;
    const int have = (old + P - 1) >> c.page_shift, want = (old + add + P - 1) >> c.page_shift;
    int *row = c.table + static_cast<int64_t>(first + i) * c.max_pages;
    for (int x = lane; x < want - have + copy; x += 32) {
      const int page = list[at + x];
      c.refs[page] = 1;
      if (copy && x == 0) {
        const int e = atomicAdd(&copies, 1);
        cp[3 * e] = tail[i];
        cp[3 * e + 1] = page;
        cp[3 * e + 2] = old & (P - 1);
        atomicSub(c.refs + tail[i], 1);
        row[old >> c.page_shift] = page;
      } else {
        row[have + x - copy] = page;
      }
    }
    __syncwarp();
    if (lane == 0) c.lens[first + i] = old + add;
  }
  __syncthreads();
  if (threadIdx.x == 0) c.state[kStateCopies] = copies;
}

// The copied last pages: entry blockIdx.x of the list, layer and side of
// blockIdx.y, the first rows of each head's part of the page.  Bound by latency
// where few are copied (a step of 8 x 8 beams, 14 layers: 7.5 us by itself).
template <typename T>
__global__ void __launch_bounds__(128) cache_copy_kernel(const CacheView c) {
  pdl_wait();
  pdl_trigger();
  if (c.state[kStateStatus]) return;
  const int n = c.state[kStateCopies];
  const int layer = blockIdx.y >> 1;
  char *pool = static_cast<char *>(blockIdx.y & 1 ? c.v : c.k);
  const int64_t head_bytes = (static_cast<int64_t>(c.dim) << c.page_shift) * c.size;
  const int64_t page_bytes = head_bytes * c.kv_heads;
  for (int e = blockIdx.x; e < n; e += gridDim.x) {
    const int *cp = copies_of(c) + 3 * e;
    const int units = cp[2] * c.dim * c.size / static_cast<int>(sizeof(T));  // of one head
    const char *src = pool + (static_cast<int64_t>(layer) * c.pages + cp[0]) * page_bytes;
    char *dst = pool + (static_cast<int64_t>(layer) * c.pages + cp[1]) * page_bytes;
    for (int x = threadIdx.x; x < units * c.kv_heads; x += blockDim.x) {
      const int h = x / units;
      const int64_t o = h * head_bytes + static_cast<int64_t>(x - h * units) * sizeof(T);
      *reinterpret_cast<T *>(dst + o) = *reinterpret_cast<const T *>(src + o);
    }
  }
}

// The last i in [0, n) with offsets[i] <= r, by a whole warp: 32 probes a step.
__device__ __forceinline__ int slot_of(const int *offsets, int n, int r) {
  const int lane = threadIdx.x & 31;
  int lo = 0, len = n;
  while (len > 1) {
    const int step = (len + 31) / 32;
    const int i = lane * step;
    const unsigned m = __ballot_sync(0xffffffffu, i < len && offsets[lo + i] <= r);
    const int at = max(__popc(m) - 1, 0) * step;  // the probes that hold come first
    lo += at;
    len = min(step, len - at);
  }
  return lo;
}

// New tokens into their places: ROWS rows of one layer a CTA.  Within a head a
// page's rows are adjacent, so the threads go along rows first; their first
// loads are under way while the rows' places are looked up.  Bound by memory:
// 32 prompts of up to 1001 tokens, 14 layers, 10 heads of 64: 240 us, 0.95 of
// the measured rate; a step's single tokens of 64 slots 5.5 us, by latency (one
// layer's, in a stream, 2.6).
template <typename T, int ROWS>
__global__ void __launch_bounds__(256) cache_write_kernel(const CacheView c, const char *k, const char *v, int64_t k_ts,
                                                          int64_t k_hs, int64_t k_ls, int64_t v_ts, int64_t v_hs, int64_t v_ls,
                                                          int layer0, int rows, const int *offsets, int uniform, int first, int n) {
  __shared__ int64_t place[ROWS];  // page row of head 0 (in rows of `dim`), -1: none
  pdl_wait();
  pdl_trigger();
  const int row0 = blockIdx.x * ROWS, layer = blockIdx.y;
  const int units = c.dim * c.size / static_cast<int>(sizeof(T));  // of a row of one head
  const int row_bytes = c.dim * c.size;
  const int all = units * ROWS * c.kv_heads;
  auto source = [&](const char *base, int64_t ts, int64_t hs, int64_t ls, int x) {
    const int u = x % units, r = x / units % ROWS, h = x / (units * ROWS);
    return reinterpret_cast<const T *>(base + (layer * ls + (row0 + r) * ts + h * hs) * c.size + u * sizeof(T));
  };
  constexpr int U = 2;
  T kk[U], vv[U];
#pragma unroll
  for (int i = 0; i < U; ++i) {
    const int x = threadIdx.x + 256 * i;
    if (x < all && row0 + x / units % ROWS < rows) {
      kk[i] = *source(k, k_ts, k_hs, k_ls, x);
      vv[i] = *source(v, v_ts, v_hs, v_ls, x);
    }
  }
  const int status = c.state[kStateStatus];
  for (int j = threadIdx.x >> 5; j < ROWS; j += 8) {
    const int r = row0 + j;
    int64_t at = -1;
    int fault = 0;
    if (r < rows) {
      int i, begin, end;
      if (offsets) {
        i = slot_of(offsets, n, r);
        begin = offsets[i];
        end = offsets[i + 1];
      } else {
        i = uniform > 0 ? r / uniform : n;
        begin = i * uniform;
        end = begin + uniform;
      }
      if (i < n && r >= begin && r < end) {
        const int64_t pos = c.lens[first + i] - static_cast<int64_t>(end - r);
        fault = kCacheBadIndex;
        if (pos >= 0 && pos < static_cast<int64_t>(c.max_pages) << c.page_shift) {
          const int page = c.table[static_cast<int64_t>(first + i) * c.max_pages + (pos >> c.page_shift)];
          if (page >= 0 && page < c.pages) {
            fault = c.refs[page] == 1 ? 0 : kCacheSharedPage;
            if (!fault) at = (static_cast<int64_t>(page) * c.kv_heads << c.page_shift) + (pos & ((1 << c.page_shift) - 1));
          }
        }
      }
    }
    if ((threadIdx.x & 31) == 0) {
      place[j] = status ? -1 : at;
      if (fault && !status) atomicOr(c.state + kStateStatus, fault);
    }
  }
  __syncthreads();
  const int64_t base = static_cast<int64_t>(layer0 + layer) * c.pages * c.kv_heads << c.page_shift;
  auto put = [&](int x, const T &a, const T &b) {
    const int u = x % units, r = x / units % ROWS, h = x / (units * ROWS);
    const int64_t to = (base + place[r] + (static_cast<int64_t>(h) << c.page_shift)) * row_bytes + u * sizeof(T);
    *reinterpret_cast<T *>(static_cast<char *>(c.k) + to) = a;
    *reinterpret_cast<T *>(static_cast<char *>(c.v) + to) = b;
  };
#pragma unroll
  for (int i = 0; i < U; ++i) {
    const int x = threadIdx.x + 256 * i;
    if (x < all && place[x / units % ROWS] >= 0) put(x, kk[i], vv[i]);
  }
#pragma unroll 1  // the other warps hide the loads; two units at a time took 276 us for 260 (the prompts above, whole passes)
  for (int x = threadIdx.x + 256 * U; x < all; x += 256)
    if (place[x / units % ROWS] >= 0) {
      const T a = *source(k, k_ts, k_hs, k_ls, x), b = *source(v, v_ts, v_hs, v_ls, x);
      put(x, a, b);
    }
}

// Slots [first, first + n) become what the slots src[i] were.  A CTA owns a
// few columns of the table for all n rows and reads them before it writes
// any, so sources may be among the rows written and repeat.  Bound by latency
// (status, source, entry, count): 64 slots of up to 16 pages 5.4 us.
__global__ void __launch_bounds__(256) cache_fork_kernel(const CacheView c, const int *src, int first, int n, int cols) {
  extern __shared__ int fork_sh[];  // sources [n], new entries [n][cols]
  int *from = fork_sh, *entry = fork_sh + n;
  pdl_wait();
  pdl_trigger();
  const int status = c.state[kStateStatus];
  const int col0 = blockIdx.x * cols;
  const int width = min(cols, c.max_pages - col0);
  const bool lens_too = blockIdx.x == gridDim.x - 1;  // one more CTA moves the lengths
  // Every CTA looks at all sources, so that a bad one leaves all columns alone.
  int wrong = status;
  for (int i = threadIdx.x; i < n; i += blockDim.x) {
    const int f = src ? src[i] : -1;
    from[i] = f;
    wrong |= f < -1 || f >= c.slots;
  }
  if (__syncthreads_or(wrong)) {
    if (lens_too && threadIdx.x == 0 && !status) atomicOr(c.state + kStateStatus, kCacheBadIndex);
    return;
  }
  if (lens_too) {
    for (int i = threadIdx.x; i < n; i += blockDim.x) entry[i] = from[i] < 0 ? 0 : c.lens[from[i]];
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += blockDim.x) c.lens[first + i] = entry[i];
    return;
  }
  int *rows = c.table + static_cast<int64_t>(first) * c.max_pages + col0;
#pragma unroll 4
  for (int x = threadIdx.x; x < n * cols; x += blockDim.x) {
    const int i = x / cols, col = x % cols, f = from[i];
    entry[x] = f < 0 || col >= width ? -1 : c.table[static_cast<int64_t>(f) * c.max_pages + col0 + col];
  }
  __syncthreads();
#pragma unroll 4
  for (int x = threadIdx.x; x < n * cols; x += blockDim.x) {
    const int i = x / cols, col = x % cols;
    if (col >= width) continue;
    int *e = rows + static_cast<int64_t>(i) * c.max_pages + col;
    const int was = *e, is = entry[x];
    if (was == is) continue;
    if (is >= 0 && is < c.pages) atomicAdd(c.refs + is, 1);
    if (was >= 0 && was < c.pages) atomicSub(c.refs + was, 1);
    *e = is;
  }
}

// Pages that hold neither one of the first `sinks` tokens nor one of the last
// `window` of their slot are given back.  A CTA a slot; latency: 64 slots of 5000
// tokens 2.0 us in a stream.
__global__ void __launch_bounds__(128) cache_trim_kernel(const CacheView c, int first, int sinks, int window) {
  pdl_wait();
  pdl_trigger();
  if (c.state[kStateStatus]) return;
  const int slot = first + blockIdx.x, P = 1 << c.page_shift;
  const int len = c.lens[slot];
  const int lo = (sinks + static_cast<int64_t>(P) - 1) >> c.page_shift;
  const int hi = len > window ? min((len - window) >> c.page_shift, c.max_pages) : 0;  // pages [lo, hi) lie between
  for (int col = lo + threadIdx.x; col < hi; col += blockDim.x) {
    int *e = c.table + static_cast<int64_t>(slot) * c.max_pages + col;
    const int was = *e;
    if (was >= 0 && was < c.pages) atomicSub(c.refs + was, 1);
    *e = -1;
  }
}

// Which pages move: the live ones at or above their count, in order, into the
// free ones below it.  list 0: moved pages, list 1: their places, list 2: the
// place of each moved page.  One CTA, like a reservation; latency: 3001 pages 7 us.
__global__ void __launch_bounds__(kBlock) cache_plan_kernel(const CacheView c) {
  extern __shared__ uint32_t bits[];
  __shared__ int sums[32];
  pdl_wait();
  pdl_trigger();
  if (c.state[kStateStatus]) {
    if (threadIdx.x == 0) c.state[kStateCopies] = 0;
    return;
  }
  const int words = (c.pages + 31) / 32;
  held_bits(c, bits);
  __syncthreads();
  auto held = [&](int w) {  // without the bits past the last page
    const uint32_t m = bits[w];
    return w == words - 1 && (c.pages & 31) ? m & ((1u << (c.pages & 31)) - 1u) : m;
  };
  int mine = 0, live;
  for (int w = threadIdx.x; w < words; w += kBlock) mine += __popc(held(w));
  block_scan(mine, sums, live);
  int *from = list_of(c, 0), *to = list_of(c, 1), *place = list_of(c, 2);
  int moves = 0, holes = 0;
  for (int base = 0; base < words; base += kBlock) {
    const int w = base + threadIdx.x;
    uint32_t up = 0, down = 0;
    if (w < words) {
      const int page = w * 32;
      const uint32_t low = page + 32 <= live ? 0xffffffffu : page >= live ? 0u : (1u << (live - page)) - 1u;  // pages below the count
      up = held(w) & ~low;
      down = ~bits[w] & low;
    }
    int all;
    int at = moves + block_scan(__popc(up), sums, all);
    moves += all;
    for (; up; up &= up - 1) from[at++] = w * 32 + __ffs(up) - 1;
    at = holes + block_scan(__popc(down), sums, all);
    holes += all;
    for (; down; down &= down - 1) to[at++] = w * 32 + __ffs(down) - 1;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < moves; i += kBlock) {
    place[from[i]] = to[i];
    c.refs[to[i]] = c.refs[from[i]];
    c.refs[from[i]] = 0;
  }
  if (threadIdx.x == 0) {
    c.state[kStateCopies] = moves;
    c.state[kStateLive] = live;
  }
}

// The moves' data and the table's new page numbers.  Bound by memory: equal pieces
// of at most 24 KB, read whole into registers before they are written, eight CTAs
// an SM.  750 pages of 20 KB in 14 layers, keys and values: 140 us, 6.2 TB/s.
constexpr int kMoveBytes = 24576;  // at most, of a CTA's turn
__global__ void __launch_bounds__(256) cache_move_kernel(const CacheView c) {
  pdl_wait();
  pdl_trigger();
  if (c.state[kStateStatus]) return;
  const int moves = c.state[kStateCopies], live = c.state[kStateLive];
  const int *from = list_of(c, 0), *to = list_of(c, 1), *place = list_of(c, 2);
  if (moves == 0) return;
  const int64_t entries = static_cast<int64_t>(c.slots) * c.max_pages;
  for (int64_t x = blockIdx.x * static_cast<int64_t>(blockDim.x) + threadIdx.x; x < entries; x += static_cast<int64_t>(gridDim.x) * blockDim.x) {
    const int page = c.table[x];
    if (page >= live && page < c.pages) c.table[x] = place[page];
  }
  const int64_t page_bytes = (static_cast<int64_t>(c.dim) * c.kv_heads << c.page_shift) * c.size;  // a multiple of 16
  const int pieces = static_cast<int>((page_bytes + kMoveBytes - 1) / kMoveBytes);
  const int64_t piece_bytes = ((page_bytes + pieces - 1) / pieces + 15) / 16 * 16;  // equal ones
  const int64_t units = static_cast<int64_t>(moves) * c.layers * 2 * pieces;
  for (int64_t x = blockIdx.x; x < units; x += gridDim.x) {
    const int piece = static_cast<int>(x % pieces);
    const int64_t y = x / pieces;
    const int side = static_cast<int>(y & 1), layer = static_cast<int>((y >> 1) % c.layers), i = static_cast<int>((y >> 1) / c.layers);
    char *pool = static_cast<char *>(side ? c.v : c.k);
    const int64_t lo = piece * piece_bytes;
    const uint4 *src = reinterpret_cast<const uint4 *>(pool + (static_cast<int64_t>(layer) * c.pages + from[i]) * page_bytes + lo);
    uint4 *dst = reinterpret_cast<uint4 *>(pool + (static_cast<int64_t>(layer) * c.pages + to[i]) * page_bytes + lo);
    const int n = static_cast<int>((page_bytes - lo < piece_bytes ? page_bytes - lo : piece_bytes) / 16);
    constexpr int U = kMoveBytes / 16 / 256;
    uint4 r[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (static_cast<int>(threadIdx.x) + 256 * u < n) r[u] = src[threadIdx.x + 256 * u];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (static_cast<int>(threadIdx.x) + 256 * u < n) dst[threadIdx.x + 256 * u] = r[u];
  }
}

// The largest dynamic shared memory of each: with the kernels' static part it
// stays below the 227 KB of a block.
constexpr int kReserveSmem = kCacheMaxPages / 8 + kCacheMaxCall * 8;
constexpr int kPlanSmem = kCacheMaxPages / 8;
constexpr int fork_cols(int n) { return n <= 16 ? 32 : n <= 32 ? 16 : 8; }
constexpr int kForkSmem = kCacheMaxCall * (fork_cols(kCacheMaxCall) + 1) * 4;
static_assert(kReserveSmem <= 226 * 1024 && kForkSmem <= 226 * 1024, "1 KB for static shared memory");

template <auto KERN, int MOST>
cudaError_t set_smem(size_t bytes) {
  static bool done[64] = {false};
  int dev = 0;
  cudaGetDevice(&dev);
  if (bytes <= 48 * 1024 - 1024 || (dev < 64 && done[dev])) return cudaSuccess;  // 1 KB: the static part
  const cudaError_t e = cudaFuncSetAttribute(KERN, cudaFuncAttributeMaxDynamicSharedMemorySize, MOST);
  if (e == cudaSuccess && dev < 64) done[dev] = true;
  return e;
}

}  // namespace

cudaError_t launch_cache_reserve(const CacheView &c, const int *offsets, int uniform, int first, int n, cudaStream_t s) {
  const size_t smem = (static_cast<size_t>(c.pages) + 31) / 32 * 4 + static_cast<size_t>(n) * 8;
  cudaError_t e = set_smem<cache_reserve_kernel, kReserveSmem>(smem);
  if (e != cudaSuccess) return e;
  e = launch_pdl(cache_reserve_kernel, dim3(1), dim3(kBlock), smem, s, 1, c, offsets, uniform, first, n);
  if (e != cudaSuccess) return e;
  const dim3 grid(n < 512 ? n : 512, c.layers * 2);
  return c.dim * c.size % 16 == 0 ? launch_pdl(cache_copy_kernel<uint4>, grid, dim3(128), 0, s, 1, c)
         : c.dim * c.size % 4 == 0 ? launch_pdl(cache_copy_kernel<uint32_t>, grid, dim3(128), 0, s, 1, c)
                                   : launch_pdl(cache_copy_kernel<uint16_t>, grid, dim3(128), 0, s, 1, c);
}

cudaError_t launch_cache_write(const CacheView &c, const void *k, const void *v, int64_t ts, int64_t hs, int64_t ls, int64_t v_ts,
                               int64_t v_hs, int64_t v_ls, int layer, int layers, int rows, const int *offsets, int uniform,
                               int first, int n, cudaStream_t s) {
  auto fits = [&](int unit) {
    const int64_t x = reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) | (ts * c.size) | (hs * c.size) | (ls * c.size) |
                      (v_ts * c.size) | (v_hs * c.size) | (v_ls * c.size) | (static_cast<int64_t>(c.dim) * c.size);
    return x % unit == 0;
  };
  auto go = [&](auto kern, int each) {
    return launch_pdl(kern, dim3((rows + each - 1) / each, layers), dim3(256), 0, s, 1, c, static_cast<const char *>(k),
                      static_cast<const char *>(v), ts, hs, ls, v_ts, v_hs, v_ls, layer, rows, offsets, uniform, first, n);
  };
  // A step's few tokens are spread over more CTAs.
  const bool few = static_cast<int64_t>(rows) * layers < 16 * 1024;
  if (fits(16)) return few ? go(cache_write_kernel<uint4, 4>, 4) : go(cache_write_kernel<uint4, 16>, 16);
  return fits(4) ? go(cache_write_kernel<uint32_t, 16>, 16) : go(cache_write_kernel<uint16_t, 16>, 16);
}

cudaError_t launch_cache_fork(const CacheView &c, const int *src, int first, int n, cudaStream_t s) {
  // Few columns a CTA: two entries a thread, and whole 32-byte sectors; at most 144 KB of shared memory.
  const int cols = fork_cols(n);
  const size_t smem = static_cast<size_t>(n) * (cols + 1) * 4;
  const cudaError_t e = set_smem<cache_fork_kernel, kForkSmem>(smem);
  if (e != cudaSuccess) return e;
  return launch_pdl(cache_fork_kernel, dim3((c.max_pages + cols - 1) / cols + 1), dim3(256), smem, s, 1, c, src, first, n, cols);
}

cudaError_t launch_cache_trim(const CacheView &c, int first, int n, int sinks, int window, cudaStream_t s) {
  return launch_pdl(cache_trim_kernel, dim3(n), dim3(128), 0, s, 1, c, first, sinks, window);
}

cudaError_t launch_cache_compact(const CacheView &c, int sm_count, cudaStream_t s) {
  const size_t smem = (static_cast<size_t>(c.pages) + 31) / 32 * 4;
  cudaError_t e = set_smem<cache_plan_kernel, kPlanSmem>(smem);
  if (e != cudaSuccess) return e;
  e = launch_pdl(cache_plan_kernel, dim3(1), dim3(kBlock), smem, s, 1, c);
  if (e != cudaSuccess) return e;
  return launch_pdl(cache_move_kernel, dim3(sm_count * 8), dim3(256), 0, s, 1, c);
}

}  // namespace nq
