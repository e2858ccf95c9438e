// Grouping of positions by cluster id: order[b] lists the positions of every
// cluster in ascending order, cluster after cluster, and offsets[b, k] is the
// first slot of cluster k. An id outside [0, K) belongs to no cluster: its
// slot comes after offsets[b, K] and holds -1.
//
// A stable least-significant-digit radix sort of (id, position), in digits of
// at most 11 bits: one pass up to K = 2047, two up to 4 M. Per pass
//   hist     (group_hist_kernel)    digit counts of chunks of R positions;
//   prefix   (group_prefix_kernel)  exclusive sums over the chunks per digit, and
//            the digit totals of the row (where there are few, the scatter does it);
//   scatter  (group_scatter_kernel) scan of the totals; every warp ranks its own
//            positions in order with its own row of 16-bit counters (match_any
//            ranks the 32 positions of a step), so equal ids keep their order.
// Rows of at most one chunk need the scatter kernel alone. No atomic decides a
// place, so the result depends on the ids only. Every pass reads and writes 8
// bytes per position; the counters (16 warps x 2^bits x 2 bytes) set the digit
// width: 11 bits take 64 KB, one more would halve the resident CTAs.
//
// Bound by latency, not bytes: 8 x 32768 ids, 512 clusters take 14 us where their 2 MB of traffic
// need 0.3 us: three launches (4, 5 and 7 us alone, overlapped by programmatic launch), each a
// chain of loads, ranks and scans. One chunk (4 x 1000 ids): one launch, 6.2 us.
#include <algorithm>

#include "fkc_internal.h"
#include "fkc_launch.cuh"

namespace fkc {
namespace {

constexpr int kWarps = 16;
constexpr int kThreads = 32 * kWarps;
constexpr int kMaxBits = 11;
constexpr int kPer = (1 << kMaxBits) / kThreads;  // digits per thread
constexpr int kBatch = 8;        // 32-position steps whose keys are loaded together
constexpr int kOneChunk = 4096;  // rows up to here are one chunk
constexpr int kMinChunk = 1024;  // positions per chunk of longer rows: a multiple of kThreads ...
constexpr int kMaxChunk = 16384; // ... and below 65536: ranks fit 16 bits

struct GroupGeom {
  int passes, bits, R, C;
};

GroupGeom group_geom(int64_t B, int64_t N, int64_t K) {
  int total = 1;
  while ((K >> total) != 0) ++total;  // the keys 0 .. K
  GroupGeom g;
  g.passes = (total + kMaxBits - 1) / kMaxBits;
  g.bits = (total + g.passes - 1) / g.passes;
  // about two chunks per SM where the rows are long enough (a chunk's warps walk their
  // positions one 32-wide step after another: 1024 positions are two steps)
  int64_t r = (B * N + 2 * 148 - 1) / (2 * 148);
  r = (r + kThreads - 1) / kThreads * kThreads;
  g.R = N <= kOneChunk ? kOneChunk
                       : static_cast<int>(std::min<int64_t>(std::max<int64_t>(r, kMinChunk), kMaxChunk));
  g.C = static_cast<int>((N + g.R - 1) / g.R);
  return g;
}

__device__ __forceinline__ uint32_t lanes_below() {
  uint32_t m;
  asm volatile("mov.u32 %0, %%lanemask_lt;" : "=r"(m));
  return m;
}

// The sort key of an id: itself, or K for one that names no cluster.
template <typename Id>
__device__ __forceinline__ int key_of(Id v, int K) {
  return (v >= 0 && v < static_cast<Id>(K)) ? static_cast<int>(v) : K;
}

template <typename Id>
__global__ void __launch_bounds__(kThreads) group_hist_kernel(const Id* __restrict__ ids,
                                                              int64_t stride, int N, int K, int R,
                                                              int C, int shift, int bits,
                                                              int32_t* __restrict__ hist) {
  extern __shared__ int32_t cnt32[];
  const int bins = 1 << bits;
  for (int i = threadIdx.x; i < bins; i += kThreads) cnt32[i] = 0;
  __syncthreads();
  pdl_wait();
  const int b = blockIdx.x / C, c = blockIdx.x - b * C;
  const int64_t rb = static_cast<int64_t>(b) * stride;
  const int r1 = static_cast<int>(min(static_cast<int64_t>(c + 1) * R, static_cast<int64_t>(N)));
  for (int r = c * R + threadIdx.x; r < r1; r += kThreads)
    atomicAdd(&cnt32[(key_of<Id>(ids[rb + r], K) >> shift) & (bins - 1)], 1);
  __syncthreads();
  int32_t* h = hist + static_cast<int64_t>(blockIdx.x) * bins;
  for (int i = threadIdx.x; i < bins; i += kThreads) h[i] = cnt32[i];
}

// 32 digits per CTA; 32 groups of lanes split the chunks.
__global__ void __launch_bounds__(1024) group_prefix_kernel(int32_t* __restrict__ hist,
                                                            int32_t* __restrict__ total, int bins,
                                                            int C, int ctas_per_row) {
  __shared__ int part[32][32];
  pdl_wait();
  const int b = blockIdx.x / ctas_per_row;
  const int lane = threadIdx.x & 31, grp = threadIdx.x >> 5;
  const int d = (blockIdx.x - b * ctas_per_row) * 32 + lane;
  int32_t* hb = hist + static_cast<int64_t>(b) * C * bins + d;
  const int per = (C + 31) / 32;
  const int c0 = min(C, grp * per), c1 = min(C, c0 + per);
  int sum = 0;
  if (d < bins)
    for (int c = c0; c < c1; ++c) sum += hb[static_cast<int64_t>(c) * bins];
  part[grp][lane] = sum;
  __syncthreads();
  int run = 0;
  for (int g = 0; g < grp; ++g) run += part[g][lane];
  if (d < bins) {
    for (int c = c0; c < c1; ++c) {
      int32_t* p = hb + static_cast<int64_t>(c) * bins;
      const int v = *p;
      *p = run;
      run += v;
    }
    if (grp == 31) total[static_cast<int64_t>(b) * bins + d] = run;
  }
}

// The same for few chunks: a thread per digit.
__global__ void __launch_bounds__(256) group_prefix_few_kernel(int32_t* __restrict__ hist,
                                                               int32_t* __restrict__ total, int bins,
                                                               int C, int64_t digits) {
  pdl_wait();
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i >= digits) return;
  const int64_t b = i / bins;
  int32_t* h = hist + b * C * bins + (i - b * bins);
  int run = 0;
  for (int c0 = 0; c0 < C; c0 += 8) {
    int v[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) v[u] = c0 + u < C ? h[static_cast<int64_t>(c0 + u) * bins] : 0;
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      if (c0 + u < C) h[static_cast<int64_t>(c0 + u) * bins] = run;
      run += v[u];
    }
  }
  total[i] = run;
}

// Positions (and, before the last pass, their keys) of a chunk to their slots.
// total null: hist holds the chunks' counts, else their prefixes; hist null: one chunk.
// vals_in null: the value is the position itself. offsets non-null (one-pass
// sorts): the first slot of every cluster.
template <typename Id>
__global__ void __launch_bounds__(kThreads) group_scatter_kernel(
    const Id* __restrict__ keys_in, int64_t stride, const int32_t* __restrict__ vals_in,
    const int32_t* __restrict__ hist, const int32_t* __restrict__ total,
    int32_t* __restrict__ keys_out, int32_t* __restrict__ vals_out,
    int32_t* __restrict__ offsets, bool last, int N, int K, int R, int C, int shift, int bits) {
  extern __shared__ int32_t sm[];  // base[bins], then 16-bit counters [kWarps][bins]
  __shared__ int warp_sum[kWarps];
  const int bins = 1 << bits;
  int32_t* base = sm;
  uint16_t* cnt = reinterpret_cast<uint16_t*>(sm + bins);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int i = threadIdx.x; i < bins * kWarps / 2; i += kThreads)
    reinterpret_cast<uint32_t*>(cnt)[i] = 0;
  __syncthreads();
  pdl_wait();
  const int b = blockIdx.x / C, c = blockIdx.x - b * C;
  const int64_t rb = static_cast<int64_t>(b) * N;
  const Id* keys = keys_in + b * stride;
  const int RW = R / kWarps;
  // 64-bit: the last chunk may end past 2^31
  const int64_t q0 = static_cast<int64_t>(c) * R + warp * RW;
  const int r0 = static_cast<int>(min(q0, static_cast<int64_t>(N)));
  const int r1 = static_cast<int>(min(q0 + RW, static_cast<int64_t>(N)));
  uint16_t* my = cnt + warp * bins;
  const uint32_t lt = lanes_below();

  // Walks the warp's positions in order; visit(position, key, slot in digit) per position.
  auto walk = [&](auto&& visit) {
    for (int at = r0; at < r1; at += 32 * kBatch) {
      int key[kBatch];
#pragma unroll
      for (int u = 0; u < kBatch; ++u)
        key[u] = at + u * 32 + lane < r1 ? key_of<Id>(keys[at + u * 32 + lane], K) : -1;
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        if (at + u * 32 >= r1) break;  // warp-uniform
        const int d = key[u] < 0 ? -1 : (key[u] >> shift) & (bins - 1);
        const uint32_t peers = __match_any_sync(0xFFFFFFFFu, d);
        int old = 0;
        if (d >= 0) old = my[d];
        __syncwarp();
        if (d >= 0 && lane == __ffs(peers) - 1)
          my[d] = static_cast<uint16_t>(old + __popc(peers));
        __syncwarp();
        if (d >= 0) visit(at + u * 32 + lane, key[u], d, old + __popc(peers & lt));
      }
    }
  };
  // each thread takes `per` neighbouring digits: their totals in the row, and before this chunk
  const int per = (bins + kThreads - 1) / kThreads;
  const int d0 = min(bins, static_cast<int>(threadIdx.x) * per), d1 = min(bins, d0 + per);
  int all[kPer], before[kPer];
#pragma unroll
  for (int x = 0; x < kPer; ++x) {
    all[x] = before[x] = 0;
    const int d = d0 + x;
    if (hist == nullptr || d >= d1) continue;
    if (total != nullptr) {
      all[x] = total[static_cast<int64_t>(b) * bins + d];
      before[x] = hist[static_cast<int64_t>(blockIdx.x) * bins + d];
    } else {
      const int32_t* h = hist + static_cast<int64_t>(b) * C * bins + d;
      for (int c1 = 0; c1 < C; c1 += 16) {
        int v[16];
#pragma unroll
        for (int u = 0; u < 16; ++u) v[u] = c1 + u < C ? h[(c1 + u) * bins] : 0;
#pragma unroll
        for (int u = 0; u < 16; ++u) {
          all[x] += v[u];
          if (c1 + u < c) before[x] += v[u];
        }
      }
    }
  }
  walk([](int, int, int, int) {});
  __syncthreads();
  // counters -> exclusive prefixes over the warps; the chunk's totals where it is the only one
  int sum = 0;
#pragma unroll
  for (int x = 0; x < kPer; ++x) {
    const int d = d0 + x;
    if (d >= d1) continue;
    int run = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const int v = cnt[w * bins + d];
      cnt[w * bins + d] = static_cast<uint16_t>(run);
      run += v;
    }
    if (hist == nullptr) all[x] = run;
    sum += all[x];
  }
  // exclusive scan of the row's digit totals
  int inc = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xFFFFFFFFu, inc, o);
    if (lane >= o) inc += u;
  }
  if (lane == 31) warp_sum[warp] = inc;
  __syncthreads();
  int run = inc - sum;
  for (int w = 0; w < warp; ++w) run += warp_sum[w];
#pragma unroll
  for (int x = 0; x < kPer; ++x) {
    const int d = d0 + x;
    if (d >= d1) continue;
    if (offsets != nullptr && c == 0 && d <= K) offsets[static_cast<int64_t>(b) * (K + 1) + d] = run;
    base[d] = run + before[x];
    run += all[x];
  }
  __syncthreads();
  walk([&](int r, int key, int d, int slot) {
    const int64_t to = rb + base[d] + slot;
    const int val = vals_in != nullptr ? vals_in[rb + r] : r;
    vals_out[to] = last && key == K ? -1 : val;
    if (keys_out != nullptr) keys_out[to] = key;
  });
}

// offsets[b, k] = number of sorted keys below k (sorts of several passes): a search among
// every step-th key in shared memory, then among the keys of one step.
constexpr int kSamples = 1024;
__global__ void __launch_bounds__(256) group_offsets_kernel(const int32_t* __restrict__ keys,
                                                            int32_t* __restrict__ offsets, int N,
                                                            int K, int per_row) {
  __shared__ int32_t sample[kSamples];
  pdl_wait();
  const int b = blockIdx.x / per_row;
  const int32_t* kb = keys + static_cast<int64_t>(b) * N;
  const int step = (N + kSamples - 1) / kSamples, n = (N + step - 1) / step;
  for (int i = threadIdx.x; i < n; i += 256) sample[i] = kb[static_cast<int64_t>(i) * step];
  __syncthreads();
  for (int k = (blockIdx.x - b * per_row) * 256 + threadIdx.x; k <= K; k += per_row * 256) {
    int lo = 0, hi = n;  // the first sample that is not below k
    while (lo < hi) {
      const int mid = (lo + hi) / 2;
      if (sample[mid] < k)
        lo = mid + 1;
      else
        hi = mid;
    }
    int64_t from = lo == 0 ? 0 : static_cast<int64_t>(lo - 1) * step + 1;
    int64_t to = lo == n ? N : static_cast<int64_t>(lo) * step;
    while (from < to) {
      const int64_t mid = (from + to) / 2;
      if (kb[mid] < k)
        from = mid + 1;
      else
        to = mid;
    }
    offsets[static_cast<int64_t>(b) * (K + 1) + k] = static_cast<int32_t>(from);
  }
}

struct GroupBuffers {
  int32_t *hist, *total, *keys[2], *vals[2];
};

size_t carve_group(const GroupGeom& g, int64_t B, int64_t N, void* ws, GroupBuffers* out) {
  GroupBuffers w{};
  uint8_t* p = static_cast<uint8_t*>(ws);
  size_t used = 0;
  auto take = [&](int64_t elems) {
    int32_t* r = ws != nullptr ? reinterpret_cast<int32_t*>(p + used) : nullptr;
    used += align_up(static_cast<size_t>(elems) * 4, 256);
    return r;
  };
  if (g.C > 1) {
    w.hist = take(B * g.C << g.bits);
    w.total = take(B << g.bits);
  }
  if (g.passes > 1) {
    w.keys[0] = take(B * N);
    w.keys[1] = take(B * N);
    w.vals[0] = take(B * N);
  }
  if (g.passes > 2) w.vals[1] = take(B * N);
  if (out != nullptr) *out = w;
  return used;
}

// One pass: src keys (and values) -> dst.
template <typename Id>
int group_pass(const GroupGeom& g, const GroupBuffers& w, const Id* keys_in, int64_t stride,
               const int32_t* vals_in, int32_t* keys_out, int32_t* vals_out, int32_t* offsets,
               int pass, int64_t B, int64_t N, int64_t K, cudaStream_t stream) {
  const int bins = 1 << g.bits, shift = pass * g.bits;
  const int n = static_cast<int>(N), k = static_cast<int>(K);
  const dim3 grid(static_cast<unsigned>(B * g.C));
  // few counts are summed by every CTA of the scatter, which saves a launch. Measured, with the launch
  // and without: 16 chunks of 512 digits 9.5, 8.7 us; 32 of 512 18.2, 18.5; 64 of 512 11.9, 11.6; 5 of
  // 2048 11.1, 13.0; 256 of 32 11.5, 19.5
  const bool sums = bins <= 512 && g.C <= 64;
  if (g.C > 1) {
    FKC_TRY(launch_pdl(group_hist_kernel<Id>, grid, dim3(kThreads), bins * 4, stream, keys_in,
                       stride, n, k, g.R, g.C, shift, g.bits, w.hist));
    const int per_row = (bins + 31) / 32;
    if (!sums && g.C <= 64)  // eight loads in flight a thread; more chunks are split over warps
      FKC_TRY(launch_pdl(group_prefix_few_kernel, dim3(static_cast<unsigned>((B * bins + 255) / 256)),
                         dim3(256), 0, stream, w.hist, w.total, bins, g.C, B * bins));
    else if (!sums)
      FKC_TRY(launch_pdl(group_prefix_kernel, dim3(static_cast<unsigned>(B * per_row)), dim3(1024), 0,
                         stream, w.hist, w.total, bins, g.C, per_row));
  }
  const size_t smem = static_cast<size_t>(bins) * (4 + 2 * kWarps);
  if (smem > 48 * 1024)
    FKC_CUDA_TRY(cudaFuncSetAttribute(group_scatter_kernel<Id>,
                                      cudaFuncAttributeMaxDynamicSharedMemorySize,
                                      static_cast<int>(smem)));
  return launch_pdl(group_scatter_kernel<Id>, grid, dim3(kThreads), smem, stream, keys_in, stride, vals_in,
                    static_cast<const int32_t*>(w.hist), static_cast<const int32_t*>(sums ? nullptr : w.total),
                    keys_out, vals_out, offsets, pass == g.passes - 1, n, k, g.R, g.C, shift,
                    g.bits);
}

template <typename Id>
int launch_group_typed(const Id* ids, int64_t stride, int32_t* order, int32_t* offsets, int64_t B, int64_t N,
                       int64_t K, void* ws, cudaStream_t stream) {
  const GroupGeom g = group_geom(B, N, K);
  GroupBuffers w;
  carve_group(g, B, N, ws, &w);
  if (g.passes == 1)
    return group_pass<Id>(g, w, ids, stride, nullptr, nullptr, order, offsets, 0, B, N, K, stream);
  FKC_TRY(group_pass<Id>(g, w, ids, stride, nullptr, w.keys[0], w.vals[0], nullptr, 0, B, N, K, stream));
  int cur = 0;
  for (int p = 1; p < g.passes; ++p, cur ^= 1) {
    const bool last = p == g.passes - 1;
    FKC_TRY(group_pass<int32_t>(g, w, w.keys[cur], N, w.vals[cur], w.keys[cur ^ 1],
                                last ? order : w.vals[cur ^ 1], nullptr, p, B, N, K, stream));
  }
  const int per_row = static_cast<int>(std::min<int64_t>((K + 256) / 256, 148));
  return launch_pdl(group_offsets_kernel, dim3(static_cast<unsigned>(B * per_row)), dim3(256), 0, stream,
                    static_cast<const int32_t*>(w.keys[cur]), offsets, static_cast<int>(N),
                    static_cast<int>(K), per_row);
}

}  // namespace

size_t group_workspace_bytes(int64_t B, int64_t N, int64_t K) {
  return carve_group(group_geom(B, N, K), B, N, nullptr, nullptr);
}

int launch_group(const void* ids, bool ids_64, int64_t stride, int32_t* order, int32_t* offsets,
                 int64_t B, int64_t N, int64_t K, void* ws, cudaStream_t stream) {
  if (ids_64)
    return launch_group_typed(static_cast<const int64_t*>(ids), stride, order, offsets, B, N, K, ws,
                              stream);
  return launch_group_typed(static_cast<const int32_t*>(ids), stride, order, offsets, B, N, K, ws,
                            stream);
}

}  // namespace fkc
