// Rows of a table by id, scaled, and the gradient of the table.
//
//   y[b, n]  = scale * table[b, ids[b, n]]            (0 for an id outside [0, K))
//   dT[b, k] = scale * sum over {n : ids[b, n] = k} of dy[b, n]
//
// The lookup is a copy: bound by the rows it writes (and the distinct rows it
// reads). A group of lanes owns a row, 16 bytes a lane, four rows in flight.
//
// The gradient is the centroid update without the division: positions grouped
// by id (cluster_group.cu), rows summed in fp32 in ascending position, one
// rounding at the end. It is bound by reading dy once and writing every row of
// dT once. No float is added by an atomic, so two runs give the same bits:
//   * a cluster of at most 2 * Lb positions is summed and stored by one group of
//     lanes (an empty one stores zeros);
//   * of a larger cluster every aligned block of Lb sorted positions leaves a
//     partial row. A block of Lb meets at most two clusters of more than 2 * Lb,
//     one that reaches over its start (slot 0) and one that begins in it (slot 1);
//   * grad_join_kernel adds a large cluster's partial rows in block order.
//
// 16384 ids of skewed frequency, table 50000 x 1024 bf16, forward and gradient: 100 us (lookup
// 13 us, gradient 60 us: 34 MB read, 102 MB written, of which 42 MB reach DRAM within the kernel);
// 32 x 16384 ids, tables 1024 x 64 fp32: 104 us (lookup 36 us: 268 MB through L2; gradient 43 us
// for 134 MB of dy, 3 TB/s: a cluster's 16 rows are two dependent flights of loads after their
// positions). Between lookup and gradient lies the grouping, some 15 us of launches. A few hundred ids take
// 18 us of launches, and 56 to 58 us with the host's side of a backward pass (a copy's takes 44).
#include <algorithm>

#include "fkc_common.cuh"
#include "fkc_internal.h"
#include "fkc_launch.cuh"

namespace fkc {
namespace {

constexpr int kThreads = 256;
constexpr int kRows = 4;   // rows in flight per group, lookup
constexpr int kFlight = 8; // vectors in flight per lane, gradient

// A vector of VEC elements of T: 16 bytes, or one element where rows are not
// whole 16-byte vectors in 16-byte aligned memory.
template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) Vec {
  T v[VEC];
};

template <typename Id>
__device__ __forceinline__ int64_t row_of(Id v, int64_t K) {
  return (v >= 0 && static_cast<int64_t>(v) < K) ? static_cast<int64_t>(v) : -1;
}

// L lanes (a power of two) per row.
template <typename T, int VEC, typename Id>
__global__ void __launch_bounds__(kThreads) lookup_kernel(const T* __restrict__ table,
                                                          const Id* __restrict__ ids,
                                                          T* __restrict__ y, int64_t total, int N,
                                                          int K, int nvec, int log_l, float scale) {
  using V = Vec<T, VEC>;
  const int L = 1 << log_l;
  const int lane = threadIdx.x & (L - 1), grp = threadIdx.x >> log_l;
  const int groups = kThreads >> log_l;
  const V* tab = reinterpret_cast<const V*>(table);
  V* out = reinterpret_cast<V*>(y);
  pdl_wait();
  const int64_t step = static_cast<int64_t>(gridDim.x) * groups * kRows;
  for (int64_t r0 = (static_cast<int64_t>(blockIdx.x) * groups + grp) * kRows; r0 < total;
       r0 += step) {
    int64_t src[kRows];
#pragma unroll
    for (int u = 0; u < kRows; ++u) {
      const int64_t r = r0 + u;
      src[u] = -1;
      if (r < total) {
        const int64_t k = row_of<Id>(ids[r], K);
        if (k >= 0) src[u] = (total == N ? 0 : r / N * K) + k;
      }
    }
    for (int c = lane; c < nvec; c += L) {
      V v[kRows];
#pragma unroll
      for (int u = 0; u < kRows; ++u) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[u].v[e] = from_f32<T>(0.f);
        if (src[u] >= 0) v[u] = tab[src[u] * nvec + c];
      }
#pragma unroll
      for (int u = 0; u < kRows; ++u) {
        if (r0 + u >= total) break;
        const float f = src[u] >= 0 ? scale : 0.f;  // zeros whatever the scale is
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[u].v[e] = from_f32<T>(to_f32<T>(v[u].v[e]) * f);
        out[(r0 + u) * nvec + c] = v[u];
      }
    }
  }
}

template <typename T, int VEC>
__device__ __forceinline__ void add_vec(float (&acc)[VEC], const Vec<T, VEC>& v) {
#pragma unroll
  for (int e = 0; e < VEC; ++e) acc[e] += to_f32<T>(v.v[e]);
}

// The next F rows: acc[w] += vector c + w * L of each, in order.
template <int F, typename T, int VEC, int WIDE>
__device__ __forceinline__ void sum_some(float (&acc)[WIDE][VEC], const Vec<T, VEC>* __restrict__ dy,
                                         const int32_t* __restrict__ order, int nvec, int c, int L) {
  Vec<T, VEC> v[F][WIDE];
#pragma unroll
  for (int u = 0; u < F; ++u) {
    const Vec<T, VEC>* row = dy + static_cast<int64_t>(order[u]) * nvec;
#pragma unroll
    for (int w = 0; w < WIDE; ++w)
      if (w == 0 || c + w * L < nvec) v[u][w] = row[c + w * L];
  }
#pragma unroll
  for (int u = 0; u < F; ++u)
#pragma unroll
    for (int w = 0; w < WIDE; ++w)
      if (w == 0 || c + w * L < nvec) add_vec<T, VEC>(acc[w], v[u][w]);
}

// acc[w] += vector c + w * L of dy at the sorted positions [p0, p1), in order. The next
// flight's row numbers are fetched with this one's rows.
template <typename T, int VEC, int WIDE>
__device__ __forceinline__ void sum_rows(float (&acc)[WIDE][VEC], const Vec<T, VEC>* __restrict__ dy,
                                         const int32_t* __restrict__ order, int p0, int p1,
                                         int nvec, int c, int L) {
  constexpr int F = kFlight / WIDE;
  int p = p0;
  if (p + F <= p1) {
    int idx[F];
#pragma unroll
    for (int u = 0; u < F; ++u) idx[u] = order[p + u];
    while (p + F <= p1) {
      int now[F];
#pragma unroll
      for (int u = 0; u < F; ++u) now[u] = idx[u];
      p += F;
      const int q = min(p, p1 - F);  // in range; what is not a whole flight is not used
#pragma unroll
      for (int u = 0; u < F; ++u) idx[u] = order[q + u];
      sum_some<F, T, VEC, WIDE>(acc, dy, now, nvec, c, L);
    }
  }
  if constexpr (F > 4)
    if (p + 4 <= p1) {
      sum_some<4, T, VEC, WIDE>(acc, dy, order + p, nvec, c, L);
      p += 4;
    }
  if (p + 2 <= p1) {
    sum_some<2, T, VEC, WIDE>(acc, dy, order + p, nvec, c, L);
    p += 2;
  }
  if (p < p1) sum_some<1, T, VEC, WIDE>(acc, dy, order + p, nvec, c, L);
}

template <typename T, int VEC, int WIDE>
__device__ __forceinline__ void store_scaled(Vec<T, VEC>* dst, const float (&acc)[WIDE][VEC], int nvec,
                                             int c, int L, float scale) {
#pragma unroll
  for (int w = 0; w < WIDE; ++w) {
    if (c + w * L >= nvec) break;
    Vec<T, VEC> o;
#pragma unroll
    for (int x = 0; x < VEC; ++x) o.v[x] = from_f32<T>(acc[w][x] * scale);
    dst[c + w * L] = o;
  }
}

// CTAs 0 .. block_ctas - 1: blocks of Lb sorted positions, groups of 2^log_b lanes (partial rows
// of the large clusters). The other CTAs: groups of 2^log_l lanes over the clusters that
// are not large.
template <typename T, int VEC, int WIDE, typename Id>
__global__ void __launch_bounds__(kThreads) lookup_grad_kernel(
    const T* __restrict__ dy, const Id* __restrict__ ids, const int32_t* __restrict__ order,
    const int32_t* __restrict__ offsets, T* __restrict__ dt, float* __restrict__ part, int N, int K,
    int nvec, int log_l, int log_b, int Lb, int J, int64_t blocks_total, int block_ctas,
    int64_t clusters, float scale) {
  using V = Vec<T, VEC>;
  pdl_wait();
  if (static_cast<int>(blockIdx.x) < block_ctas) {
    const int L = 1 << log_b;
    const int lane = threadIdx.x & (L - 1);
    const int64_t u = (static_cast<int64_t>(blockIdx.x) << (8 - log_b)) + (threadIdx.x >> log_b);
    if (u >= blocks_total) return;
    const int64_t b = u / J;
    const int32_t* of = offsets + b * (K + 1);
    const int32_t* ord = order + b * N;
    const V* rows = reinterpret_cast<const V*>(dy) + b * N * nvec;
    const int used = of[K];
    const int p0 = static_cast<int>(u - b * J) * Lb;
    if (p0 >= used) return;
    const int p1 = min(p0 + Lb, used);
#pragma unroll
    for (int slot = 0; slot < 2; ++slot) {
      const int64_t k = row_of<Id>(ids[b * N + ord[slot == 0 ? p0 : p1 - 1]], K);
      if (k < 0) continue;  // order does not group these ids
      const int s = of[k], e = of[k + 1];
      if (e - s <= 2 * Lb || (slot == 1 && s <= p0)) continue;
      float* dst = part + (u * 2 + slot) * nvec * VEC;
      for (int c = lane; c < nvec; c += L) {
        float acc[1][VEC] = {};
        sum_rows<T, VEC, 1>(acc, rows, ord, max(s, p0), min(e, p1), nvec, c, L);
#pragma unroll
        for (int x = 0; x < VEC; ++x) dst[c * VEC + x] = acc[0][x];
      }
    }
    return;
  }
  const int L = 1 << log_l;
  const int lane = threadIdx.x & (L - 1);
  const int64_t step = static_cast<int64_t>(gridDim.x - block_ctas) << (8 - log_l);
  for (int64_t row = (static_cast<int64_t>(blockIdx.x - block_ctas) << (8 - log_l)) + (threadIdx.x >> log_l);
       row < clusters; row += step) {  // b * K + k
    const int64_t b = row / K;
    const int32_t* of = offsets + b * (K + 1) + (row - b * K);
    const int s = of[0], e = of[1];
    if (e - s > 2 * Lb) continue;
    const V* rows = reinterpret_cast<const V*>(dy) + b * N * nvec;
    V* dst = reinterpret_cast<V*>(dt) + row * nvec;
    for (int c = lane; c < nvec; c += L * WIDE) {
      float acc[WIDE][VEC] = {};
      sum_rows<T, VEC, WIDE>(acc, rows, order + b * N, s, e, nvec, c, L);
      store_scaled<T, VEC, WIDE>(dst, acc, nvec, c, L, scale);
    }
  }
}

// The large clusters, by the block in which each begins: their partial rows in block order.
template <typename T, int VEC, typename Id>
__global__ void __launch_bounds__(kThreads) grad_join_kernel(
    const Id* __restrict__ ids, const int32_t* __restrict__ order,
    const int32_t* __restrict__ offsets, const float* __restrict__ part, T* __restrict__ dt, int N,
    int K, int nvec, int log_l, int Lb, int J, int64_t blocks_total, float scale) {
  using V = Vec<T, VEC>;
  constexpr int kAhead = 8;  // partial rows in flight
  const int L = 1 << log_l;
  const int lane = threadIdx.x & (L - 1), grp = threadIdx.x >> log_l;
  const int64_t u = static_cast<int64_t>(blockIdx.x) * (kThreads >> log_l) + grp;
  pdl_wait();
  if (u >= blocks_total) return;
  const int64_t b = u / J;
  const int32_t* of = offsets + b * (K + 1);
  const int p0 = static_cast<int>(u - b * J) * Lb, used = of[K];
  if (p0 >= used) return;
  // the last cluster of the block: a large one that begins here reaches over its end
  const int64_t k = row_of<Id>(ids[b * N + order[b * N + min(p0 + Lb, used) - 1]], K);
  if (k < 0) return;
  const int s = of[k], e = of[k + 1];
  if (e - s <= 2 * Lb || s < p0) return;
  const int j0 = s / Lb, j1 = (e - 1) / Lb;
  V* dst = reinterpret_cast<V*>(dt) + (b * K + k) * nvec;
  for (int c = lane; c < nvec; c += L) {
    float acc[VEC] = {};
    int j = j0;
    auto some = [&](auto count) {
      constexpr int F = decltype(count)::value;
      Vec<float, VEC> v[F];
#pragma unroll
      for (int q = 0; q < F; ++q) {
        const int slot = j + q == j0 && s % Lb != 0 ? 1 : 0;
        const float* src = part + ((b * J + j + q) * 2 + slot) * nvec * VEC + c * VEC;
#pragma unroll
        for (int x = 0; x < VEC; ++x) v[q].v[x] = src[x];
      }
#pragma unroll
      for (int q = 0; q < F; ++q)
#pragma unroll
        for (int x = 0; x < VEC; ++x) acc[x] += v[q].v[x];
      j += F;
    };
    while (j + kAhead - 1 <= j1) some(std::integral_constant<int, kAhead>{});
    while (j + 1 <= j1) some(std::integral_constant<int, 2>{});
    if (j <= j1) some(std::integral_constant<int, 1>{});
    V o;
#pragma unroll
    for (int x = 0; x < VEC; ++x) o.v[x] = from_f32<T>(acc[x] * scale);
    dst[c] = o;
  }
}

// Lanes per row: the vectors of a row rounded up to a power of two, `most` at most.
int lanes_log2(int64_t nvec, int most) {
  int l = 0;
  while ((1 << l) < nvec && (1 << l) < most) ++l;
  return l;
}

// Positions per block: longer blocks for longer rows of ids, so that neither a block's sum (Lb rows) nor a
// cluster's join (N / Lb partial rows) becomes a long chain. Forward and gradient in us with 16, 32, 64 and
// 128, over tables of 8, 500 and 50000 rows: 4096 ids, rows of 2 KB: 31 31 76, 25 32 83, 23 44 108, -;
// 8192: 45 35 84, 34 35 79, 29 43 99, -; 16385, 128 bytes: 49 30 42, 33 27 40, 31 30 42, 38 38 49;
// 32768, 128 bytes: 79 41 48, 50 32 43, 38 32 47, 41 39 52; 65536, 512 bytes: -, 103 55 85, 62 46 93, 51 51 117.
int block_len(int64_t N) {
  int lb = 16;
  while (lb < 512 && static_cast<int64_t>(lb) * lb * 24 < N) lb *= 2;
  return lb;
}

unsigned grid_for(int64_t groups_needed, int log_l) {
  const int64_t ctas = (groups_needed + (kThreads >> log_l) - 1) / (kThreads >> log_l);
  return static_cast<unsigned>(std::max<int64_t>(1, std::min<int64_t>(ctas, 148 * 32)));
}

struct GradLayout {
  size_t order, offsets, part, group, total;
  int Lb;
  int64_t J;
};

GradLayout grad_layout(int64_t B, int64_t N, int64_t K, int64_t D) {
  GradLayout l{};
  l.Lb = block_len(N);
  l.J = (N + l.Lb - 1) / l.Lb;
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t r = at;
    at += align_up(bytes, 256);
    return r;
  };
  l.order = take(static_cast<size_t>(B * N) * 4);
  l.offsets = take(static_cast<size_t>(B * (K + 1)) * 4);
  // no cluster is large below 2 * Lb + 1 positions
  l.part = take(N > 2 * l.Lb ? static_cast<size_t>(B * l.J) * 2 * D * 4 : 0);
  l.group = take(group_workspace_bytes(B, N, K));
  l.total = at;
  return l;
}

bool vec_ok(const void* p, const void* q, int64_t D, size_t elem) {
  return (reinterpret_cast<uintptr_t>(p) | reinterpret_cast<uintptr_t>(q)) % 16 == 0 &&
         D * static_cast<int64_t>(elem) % 16 == 0;
}

template <typename T, int VEC>
int lookup_typed(const void* table, const void* ids, bool ids_64, void* y, int64_t B, int64_t N,
                 int64_t K, int64_t D, float scale, cudaStream_t stream) {
  const int nvec = static_cast<int>(D / VEC);
  const int log_l = lanes_log2(nvec, kThreads);
  const int64_t total = B * N;
  const dim3 grid(grid_for((total + kRows - 1) / kRows, log_l));
  const T* t = static_cast<const T*>(table);
  T* o = static_cast<T*>(y);
  const int n = static_cast<int>(N), k = static_cast<int>(K);
  if (ids_64)
    return launch_pdl(lookup_kernel<T, VEC, int64_t>, grid, dim3(kThreads), 0, stream, t,
                      static_cast<const int64_t*>(ids), o, total, n, k, nvec, log_l, scale);
  return launch_pdl(lookup_kernel<T, VEC, int32_t>, grid, dim3(kThreads), 0, stream, t,
                    static_cast<const int32_t*>(ids), o, total, n, k, nvec, log_l, scale);
}

template <typename T, int VEC>
int grad_typed(const void* dy, const void* ids, bool ids_64, void* dt, int64_t B, int64_t N,
               int64_t K, int64_t D, float scale, uint8_t* ws, cudaStream_t stream) {
  const GradLayout l = grad_layout(B, N, K, D);
  int32_t* order = reinterpret_cast<int32_t*>(ws + l.order);
  int32_t* offsets = reinterpret_cast<int32_t*>(ws + l.offsets);
  float* part = reinterpret_cast<float*>(ws + l.part);
  FKC_TRY(launch_group(ids, ids_64, N, order, offsets, B, N, K, ws + l.group, stream));
  const int nvec = static_cast<int>(D / VEC);
  // a warp at most: most clusters of a large table have no row or one, and what counts is how
  // many are in flight
  const int log_l = lanes_log2(nvec, 32), log_b = lanes_log2(nvec, kThreads);
  const bool large = N > 2 * l.Lb;
  const int64_t blocks = large ? B * l.J : 0;
  const int64_t block_ctas = (blocks + (kThreads >> log_b) - 1) / (kThreads >> log_b);
  const int64_t clusters = B * K;
  // CTAs that the GPU holds at once: each warp goes on to its next cluster by itself, while a CTA
  // of few clusters would keep its place until the largest is done
  const int64_t ctas = block_ctas + std::min<int64_t>(grid_for(clusters, log_l), 148 * 5);
  FKC_REQUIRE(ctas <= 2147483647ll, "lookup gradient: too many clusters");
  const dim3 grid(static_cast<unsigned>(ctas));
  const int n = static_cast<int>(N), k = static_cast<int>(K), j = static_cast<int>(l.J);
  const T* g = static_cast<const T*>(dy);
  T* o = static_cast<T*>(dt);
  auto run = [&](auto id) {
    using Id = decltype(id);
    const Id* in = static_cast<const Id*>(ids);
    // rows wider than a warp: two vectors of a row at once
    auto kern = nvec > 32 ? lookup_grad_kernel<T, VEC, 2, Id> : lookup_grad_kernel<T, VEC, 1, Id>;
    FKC_TRY(launch_pdl(kern, grid, dim3(kThreads), 0, stream, g, in, static_cast<const int32_t*>(order),
                       static_cast<const int32_t*>(offsets), o, part, n, k, nvec, log_l, log_b, l.Lb, j,
                       blocks, static_cast<int>(block_ctas), clusters, scale));
    if (!large) return static_cast<int>(FKC_OK);
    return launch_pdl(grad_join_kernel<T, VEC, Id>, dim3(static_cast<unsigned>(block_ctas)),
                      dim3(kThreads), 0, stream, in, static_cast<const int32_t*>(order),
                      static_cast<const int32_t*>(offsets), static_cast<const float*>(part), o, n, k,
                      nvec, log_b, l.Lb, j, blocks, scale);
  };
  return ids_64 ? run(int64_t{}) : run(int32_t{});
}

}  // namespace

int launch_lookup(const void* table, const void* ids, bool ids_64, void* y, int64_t B, int64_t N,
                  int64_t K, int64_t D, int dtype, float scale, cudaStream_t stream) {
  const bool v = vec_ok(table, y, D, dtype_size(dtype));
  switch (dtype) {
    case FKC_DTYPE_F16:
      return v ? lookup_typed<__half, 8>(table, ids, ids_64, y, B, N, K, D, scale, stream)
               : lookup_typed<__half, 1>(table, ids, ids_64, y, B, N, K, D, scale, stream);
    case FKC_DTYPE_BF16:
      return v ? lookup_typed<__nv_bfloat16, 8>(table, ids, ids_64, y, B, N, K, D, scale, stream)
               : lookup_typed<__nv_bfloat16, 1>(table, ids, ids_64, y, B, N, K, D, scale, stream);
    default:
      return v ? lookup_typed<float, 4>(table, ids, ids_64, y, B, N, K, D, scale, stream)
               : lookup_typed<float, 1>(table, ids, ids_64, y, B, N, K, D, scale, stream);
  }
}

size_t lookup_grad_workspace_bytes(int64_t B, int64_t N, int64_t K, int64_t D) {
  return grad_layout(B, N, K, D).total;
}

int launch_lookup_grad(const void* dy, const void* ids, bool ids_64, void* dt, int64_t B,
                       int64_t N, int64_t K, int64_t D, int dtype, float scale, void* ws,
                       cudaStream_t stream) {
  uint8_t* w = static_cast<uint8_t*>(ws);
  const bool v = vec_ok(dy, dt, D, dtype_size(dtype));
  switch (dtype) {
    case FKC_DTYPE_F16:
      return v ? grad_typed<__half, 8>(dy, ids, ids_64, dt, B, N, K, D, scale, w, stream)
               : grad_typed<__half, 1>(dy, ids, ids_64, dt, B, N, K, D, scale, w, stream);
    case FKC_DTYPE_BF16:
      return v ? grad_typed<__nv_bfloat16, 8>(dy, ids, ids_64, dt, B, N, K, D, scale, w, stream)
               : grad_typed<__nv_bfloat16, 1>(dy, ids, ids_64, dt, B, N, K, D, scale, w, stream);
    default:
      return v ? grad_typed<float, 4>(dy, ids, ids_64, dt, B, N, K, D, scale, w, stream)
               : grad_typed<float, 1>(dy, ids, ids_64, dt, B, N, K, D, scale, w, stream);
  }
}

}  // namespace fkc
