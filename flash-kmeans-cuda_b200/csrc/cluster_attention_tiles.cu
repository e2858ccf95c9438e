// Attention over selected clusters, cluster by cluster: the form for many queries.
//
// The walk of cluster_attention.cu reads every selected key once per query: 4 * D bytes
// a key for 4 * D * G flops, from L2. Here the queries that selected a cluster are brought
// together instead: sel is grouped by cluster (cluster_group.cu: entry e is query
// e / top), the heads of its queries become the rows of tiles of 128, and a tile reads the
// cluster's keys once for all of them. A tile leaves, for every (query, slot of sel, head),
// the normalised output over that cluster in fp32 and its log-sum-exp, and tiles_join_kernel
// joins a query's top parts. So the traffic is D * (2 + 4 + 4) bytes per (query, slot,
// head) instead of 4 * D per (query, key): at G = 4 and 64 keys a cluster a sixth.
//
// A tile's CTA: four warps of 32 rows; Q gathered once; keys and values in tiles of 64,
// gathered into a double buffer; online softmax over the cluster's tiles in registers
// (m16n8k16: S = Q K^T, then P straight from the score registers as the A operand).
// P is rounded to the 16-bit input type for the second product, as its operand type
// demands.
#include <algorithm>

#include "cluster_attention.cuh"

namespace fkc {
namespace attn {
namespace {

constexpr int kRows = 128;  // rows (query, head) per tile
constexpr int kKeys = 64;   // keys per step

// units[r, j] = (cluster, first row of the tile among the cluster's rows); count[r] of them.
__global__ void __launch_bounds__(1024) tile_units_kernel(const int32_t* __restrict__ inv_offsets,
                                                          int2* __restrict__ units,
                                                          int32_t* __restrict__ count, int K, int G,
                                                          int rows, int units_max) {
  __shared__ int warp_total[32];
  pdl_wait();
  const int r = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int32_t* of = inv_offsets + static_cast<int64_t>(r) * (K + 1);
  int2* out = units + static_cast<int64_t>(r) * units_max;
  int carry = 0;
  for (int c0 = 0; c0 < K; c0 += 1024) {
    const int c = c0 + threadIdx.x;
    int n = 0;
    if (c < K) n = static_cast<int>((static_cast<int64_t>(of[c + 1] - of[c]) * G + rows - 1) / rows);
    int inc = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xFFFFFFFFu, inc, o);
      if (lane >= o) inc += u;
    }
    __syncthreads();
    if (lane == 31) warp_total[warp] = inc;
    __syncthreads();
    int at = carry + inc - n;
    for (int w = 0; w < 32; ++w) {
      if (w < warp) at += warp_total[w];
      carry += warp_total[w];
    }
    for (int t = 0; t < n; ++t)
      if (at + t < units_max) out[at + t] = make_int2(c, t * rows);
  }
  if (threadIdx.x == 0) count[r] = min(carry, units_max);
}

// What a tile of `kRows` rows knows about them.
struct RowData {
  int64_t q[kRows];   // element offset of the query row
  int32_t slot[kRows];  // (query, slot, head) of its part; -1: no row
  int32_t pos[kRows];   // last position it sees; -1: none
};

template <int DP>
struct FwdSmem {
  static constexpr int kQ = 0;
  static constexpr int kTile = kKeys * DP * 2;
  static constexpr int kK = kRows * DP * 2;      // two buffers
  static constexpr int kV = kK + 2 * kTile;      // two buffers
  static constexpr int kBytes = kV + 2 * kTile;
};

template <typename T, int DP>
__global__ void __launch_bounds__(128, 2) tiles_fwd_kernel(
    Args a, int i0, int nq, const int32_t* __restrict__ inv_order,
    const int32_t* __restrict__ inv_offsets, const int2* __restrict__ units,
    const int32_t* __restrict__ count, float* __restrict__ part_o, float* __restrict__ part_lse,
    int units_max) {
  constexpr int KS = DP / 16, CH = DP / 8;
  using S = FwdSmem<DP>;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ RowData rows;
  __shared__ int s_key[2][kKeys];  // positions of a step's keys; INT_MAX behind the last
  __shared__ int s_high;           // the largest of the rows' positions
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int g = lane >> 2, t4 = lane & 3;
  const uint32_t base = static_cast<uint32_t>(__cvta_generic_to_shared(smem));
  if (a.D < DP)
    for (int o = tid * 16; o < S::kBytes; o += 2048)
      *reinterpret_cast<uint4*>(smem + o) = make_uint4(0, 0, 0, 0);
  if (tid == 0) s_high = -1;
  __syncthreads();
  pdl_wait();
  const int r = blockIdx.x / units_max, unit = blockIdx.x - r * units_max;
  if (unit >= count[r]) return;
  const int2 un = units[static_cast<int64_t>(r) * units_max + unit];
  const int c = un.x, b = r / a.Hkv, hk = r - b * a.Hkv;
  const int32_t* iof = inv_offsets + static_cast<int64_t>(r) * (a.K + 1);
  const int e0 = iof[c];
  const int64_t rows_all = static_cast<int64_t>(iof[c + 1] - e0) * a.G;
  int s0, s1;
  cluster_span(a, r, c, s0, s1);
  const int steps = (s1 - s0 + kKeys - 1) / kKeys;
  const int32_t* order = a.order + static_cast<int64_t>(r) * a.N;
  {
    const int64_t row = un.y + static_cast<int64_t>(tid);
    int64_t q = 0;
    int slot = -1, pos = -1;
    if (row < rows_all) {
      const int e = static_cast<int>(row / a.G), h = static_cast<int>(row - static_cast<int64_t>(e) * a.G);
      const int p = inv_order[static_cast<int64_t>(r) * nq * a.top + e0 + e];
      const int i = i0 + p / a.top;
      slot = p * a.G + h;
      pos = min(a.q_pos != nullptr ? a.q_pos[static_cast<int64_t>(b) * a.Nq + i] : a.N, a.N);
      q = b * a.qs.b + (static_cast<int64_t>(hk) * a.G + h) * a.qs.h + i * a.qs.n;
      atomicMax(&s_high, pos);
    }
    rows.q[tid] = q;
    rows.slot[tid] = slot;
    rows.pos[tid] = pos;
  }
  auto key_at = [&](int step) {  // threads 0 .. kKeys - 1
    const int s = s0 + step * kKeys + tid;
    if (s >= s1) return INT_MAX;
    const int row = order[s];
    return row >= 0 && row < a.N ? row : INT_MAX;
  };
  if (tid < kKeys) {
    s_key[0][tid] = steps > 0 ? key_at(0) : INT_MAX;
    s_key[1][tid] = steps > 1 ? key_at(1) : INT_MAX;
  }
  __syncthreads();
  const int high = s_high;
  const T* q = static_cast<const T*>(a.q);
  const T* kb = static_cast<const T*>(a.k) + b * a.ks.b + hk * a.ks.h;
  const T* vb = static_cast<const T*>(a.v) + b * a.vs.b + hk * a.vs.h;
  const int dchunks = a.D / 8;
  auto copy_keys = [&](int step) {
    const int u = step & 1;
#pragma unroll
    for (int it = 0; it < kKeys * CH / 128; ++it) {
      const int e = it * 128 + tid, key = e / CH, ch = e % CH;
      if (ch >= dchunks) continue;
      const int row = s_key[u][key];
      const bool on = row <= high;  // a key that no row sees is not read
      const int64_t at = on ? row : 0;
      mma::cp_async16(base + S::kK + u * S::kTile + tile_at<DP>(key, ch), kb + at * a.ks.n + ch * 8, on);
      mma::cp_async16(base + S::kV + u * S::kTile + tile_at<DP>(key, ch), vb + at * a.vs.n + ch * 8, on);
    }
  };
#pragma unroll
  for (int it = 0; it < kRows * CH / 128; ++it) {
    const int e = it * 128 + tid, row = e / CH, ch = e % CH;
    if (ch >= dchunks) continue;
    const bool on = rows.pos[row] >= 0;
    mma::cp_async16(base + S::kQ + tile_at<DP>(row, ch), q + (on ? rows.q[row] + ch * 8 : 0), on);
  }
  if (steps > 0) copy_keys(0);
  mma::cp_async_commit();

  const int row0 = warp * 32;
  int pos[2][2];
  float m[2][2], l[2][2];
  float o[2][DP / 8][4];
#pragma unroll
  for (int x = 0; x < 2; ++x) {
#pragma unroll
    for (int y = 0; y < 2; ++y) {
      pos[x][y] = rows.pos[row0 + x * 16 + y * 8 + g];
      m[x][y] = -INFINITY;
      l[x][y] = 0.f;
    }
#pragma unroll
    for (int n = 0; n < DP / 8; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[x][n][e] = 0.f;
  }
  const bool idle = un.y + row0 >= rows_all;  // no row for this warp
  const float sc = a.scale * kLog2e;
  for (int step = 0; step < steps; ++step) {
    mma::cp_async_wait<0>();
    __syncthreads();  // this step's tiles; the other buffers are free
    if (step + 1 < steps) copy_keys(step + 1);
    mma::cp_async_commit();
    int later = INT_MAX;
    if (tid < kKeys && step + 2 < steps) later = key_at(step + 2);
    const int u = step & 1;
    const int keys = min(kKeys, s1 - s0 - step * kKeys);
    if (!idle) {
      const uint32_t kt = base + S::kK + u * S::kTile, vt = base + S::kV + u * S::kTile;
      float s[2][kKeys / 8][4];
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int n = 0; n < kKeys / 8; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[x][n][e] = 0.f;
#pragma unroll
      for (int kk = 0; kk < KS; ++kk) {
        uint32_t fa[2][4];
        load_a<DP>(fa[0], base + S::kQ, row0, kk);
        load_a<DP>(fa[1], base + S::kQ, row0 + 16, kk);
#pragma unroll
        for (int n = 0; n < kKeys / 8; n += 2) {
          if (n * 8 >= keys) break;
          uint32_t f[4];
          load_b<DP>(f, kt, n * 8, kk);
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            mma::m16n8k16<T>(s[x][n], fa[x], f[0], f[1]);
            mma::m16n8k16<T>(s[x][n + 1], fa[x], f[2], f[3]);
          }
        }
      }
      float top[2][2] = {{-INFINITY, -INFINITY}, {-INFINITY, -INFINITY}};
#pragma unroll
      for (int n = 0; n < kKeys / 8; ++n) {
        const int2 key = *reinterpret_cast<const int2*>(&s_key[u][n * 8 + t4 * 2]);
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            float& a0 = s[x][n][y * 2];
            float& a1 = s[x][n][y * 2 + 1];
            a0 = key.x <= pos[x][y] ? a0 * sc : -INFINITY;
            a1 = key.y <= pos[x][y] ? a1 * sc : -INFINITY;
            top[x][y] = fmaxf(top[x][y], fmaxf(a0, a1));
          }
      }
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          float v = top[x][y];
          v = fmaxf(v, __shfl_xor_sync(0xFFFFFFFFu, v, 1));
          v = fmaxf(v, __shfl_xor_sync(0xFFFFFFFFu, v, 2));
          const float mn = fmaxf(m[x][y], v);
          const float from = mn == -INFINITY ? 0.f : mn;
          const float alpha = exp2f(m[x][y] - from);
          m[x][y] = mn;
          float sum = 0.f;
#pragma unroll
          for (int n = 0; n < kKeys / 8; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              s[x][n][y * 2 + e] = exp2f(s[x][n][y * 2 + e] - from);
              sum += s[x][n][y * 2 + e];
            }
          l[x][y] = l[x][y] * alpha + sum;
          if (step > 0)
#pragma unroll
            for (int n = 0; n < DP / 8; ++n) o[x][n][y * 2] *= alpha, o[x][n][y * 2 + 1] *= alpha;
        }
#pragma unroll
      for (int j = 0; j < kKeys / 16; ++j) {
        if (j * 16 >= keys) break;
        uint32_t p[2][4];
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          p[x][0] = mma::pack2<T>(s[x][2 * j][0], s[x][2 * j][1]);
          p[x][1] = mma::pack2<T>(s[x][2 * j][2], s[x][2 * j][3]);
          p[x][2] = mma::pack2<T>(s[x][2 * j + 1][0], s[x][2 * j + 1][1]);
          p[x][3] = mma::pack2<T>(s[x][2 * j + 1][2], s[x][2 * j + 1][3]);
        }
#pragma unroll
        for (int nd = 0; nd < KS; ++nd) {
          uint32_t f[4];
          load_b_trans<DP>(f, vt, j * 16, nd);
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            mma::m16n8k16<T>(o[x][2 * nd], p[x], f[0], f[1]);
            mma::m16n8k16<T>(o[x][2 * nd + 1], p[x], f[2], f[3]);
          }
        }
      }
    }
    __syncthreads();  // all reads of this step's tiles and positions
    if (tid < kKeys) s_key[u][tid] = later;
  }
  mma::cp_async_wait<0>();
  if (idle) return;
#pragma unroll
  for (int x = 0; x < 2; ++x)
#pragma unroll
    for (int y = 0; y < 2; ++y) {
      float sum = l[x][y];
      sum += __shfl_xor_sync(0xFFFFFFFFu, sum, 1);
      sum += __shfl_xor_sync(0xFFFFFFFFu, sum, 2);
      const int slot = rows.slot[row0 + x * 16 + y * 8 + g];
      if (slot < 0) continue;
      const float inv = sum == 0.f ? 0.f : 1.f / sum;
      const int64_t at = static_cast<int64_t>(r) * nq * a.top * a.G + slot;
      if (t4 == 0) part_lse[at] = sum == 0.f ? -INFINITY : m[x][y] + log2f(sum);
      float* row = part_o + at * a.D;
#pragma unroll
      for (int n = 0; n < DP / 8; ++n) {
        const int d = n * 8 + t4 * 2;
        if (d < a.D)
          *reinterpret_cast<float2*>(row + d) =
              make_float2(o[x][n][y * 2] * inv, o[x][n][y * 2 + 1] * inv);
      }
    }
}

// One warp per (query, head): joins the parts of its clusters, whose log-sum-exps are to base 2.
template <typename T>
__global__ void __launch_bounds__(256) tiles_join_kernel(Args a, int i0, int nq,
                                                         const float* __restrict__ part_o,
                                                         const float* __restrict__ part_lse,
                                                         T* __restrict__ out,
                                                         float* __restrict__ lse, int64_t rows) {
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);  // (r, i - i0, h)
  if (row >= rows) return;
  const int h = static_cast<int>(row % a.G);
  const int64_t qi = row / a.G;
  const int r = static_cast<int>(qi / nq), i = i0 + static_cast<int>(qi % nq);
  const int b = r / a.Hkv, hq = (r - b * a.Hkv) * a.G + h;
  const int32_t* sel = a.sel + (static_cast<int64_t>(r) * a.Nq + i) * a.top;
  const float* pl = part_lse + qi * a.top * a.G + h;  // slot s: + s * G
  const float* po = part_o + (qi * a.top * a.G + h) * a.D;
  float top = -INFINITY;
  for (int s = lane; s < a.top; s += 32)
    if (sel[s] >= 0 && sel[s] < a.K) top = fmaxf(top, pl[static_cast<int64_t>(s) * a.G]);
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
  const float from = top == -INFINITY ? 0.f : top;
  float acc[4] = {0.f, 0.f, 0.f, 0.f}, sum = 0.f;
  const bool on = lane * 4 < a.D;
#pragma unroll 4
  for (int s = 0; s < a.top; ++s) {
    const bool has = sel[s] >= 0 && sel[s] < a.K;
    const float ls = has ? pl[static_cast<int64_t>(s) * a.G] : -INFINITY;
    const float w = ls == -INFINITY ? 0.f : exp2f(ls - from);
    if (ls == -INFINITY) continue;
    sum += w;
    if (on) {
      const float4 v = *reinterpret_cast<const float4*>(po + static_cast<int64_t>(s) * a.G * a.D + lane * 4);
      acc[0] += w * v.x;
      acc[1] += w * v.y;
      acc[2] += w * v.z;
      acc[3] += w * v.w;
    }
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  const int64_t at = (static_cast<int64_t>(b) * a.Hq + hq) * a.Nq + i;
  if (on) {
    uint2 v;
    v.x = mma::pack2<T>(acc[0] * inv, acc[1] * inv);
    v.y = mma::pack2<T>(acc[2] * inv, acc[3] * inv);
    *reinterpret_cast<uint2*>(out + at * a.D + lane * 4) = v;
  }
  if (lane == 0) lse[at] = sum == 0.f ? -INFINITY : (from + log2f(sum)) * kLn2;
}

// Queries that one round takes: rounds of equal size whose parts stay below 2^31 bytes (a
// round has its own grouping, so short ones cost launches), 64 queries at least.
int64_t queries_per_round(const Args& a) {
  const int64_t R = static_cast<int64_t>(a.batch) * a.Hkv;
  const int64_t per = R * a.top * a.G * (a.D + 1) * 4;
  const int64_t most = std::max<int64_t>(64, (1ll << 31) / per);
  const int64_t rounds = (a.Nq + most - 1) / most;
  return (a.Nq + rounds - 1) / rounds;
}

struct Layout {
  size_t inv_order, inv_offsets, units, count, part_lse, part_o, group, total;
  int64_t nq, units_max;
};

Layout fwd_layout(const Args& a) {
  Layout l{};
  const int64_t R = static_cast<int64_t>(a.batch) * a.Hkv;
  l.nq = queries_per_round(a);
  const int64_t entries = l.nq * a.top;
  l.units_max = entries * a.G / kRows + std::min<int64_t>(a.K, entries);
  size_t at = 0;
  auto take = [&](int64_t bytes) {
    const size_t p = at;
    at += align_up(static_cast<size_t>(bytes), 256);
    return p;
  };
  l.inv_order = take(R * entries * 4);
  l.inv_offsets = take(R * (a.K + 1) * 4);
  l.units = take(R * l.units_max * 8);
  l.count = take(R * 4);
  l.part_lse = take(R * entries * a.G * 4);
  l.part_o = take(R * entries * a.G * a.D * 4);
  l.group = take(static_cast<int64_t>(group_workspace_bytes(R, entries, a.K)));
  l.total = at;
  return l;
}

template <typename T, int DP>
int fwd_typed(const Args& a, T* out, float* lse, uint8_t* ws, cudaStream_t stream) {
  const Layout l = fwd_layout(a);
  const int64_t R = static_cast<int64_t>(a.batch) * a.Hkv;
  int32_t* inv_order = reinterpret_cast<int32_t*>(ws + l.inv_order);
  int32_t* inv_offsets = reinterpret_cast<int32_t*>(ws + l.inv_offsets);
  int2* units = reinterpret_cast<int2*>(ws + l.units);
  int32_t* count = reinterpret_cast<int32_t*>(ws + l.count);
  float* part_lse = reinterpret_cast<float*>(ws + l.part_lse);
  float* part_o = reinterpret_cast<float*>(ws + l.part_o);
  auto kern = tiles_fwd_kernel<T, DP>;
  const int smem = FwdSmem<DP>::kBytes;
  FKC_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  for (int64_t i0 = 0; i0 < a.Nq; i0 += l.nq) {
    const int nq = static_cast<int>(std::min<int64_t>(l.nq, a.Nq - i0));
    FKC_TRY(launch_group(a.sel + i0 * a.top, false, static_cast<int64_t>(a.Nq) * a.top, inv_order,
                         inv_offsets, R, static_cast<int64_t>(nq) * a.top, a.K, ws + l.group, stream));
    FKC_TRY(launch_pdl(tile_units_kernel, dim3(static_cast<unsigned>(R)), dim3(1024), 0, stream,
                       static_cast<const int32_t*>(inv_offsets), units, count, a.K, a.G, kRows,
                       static_cast<int>(l.units_max)));
    FKC_TRY(launch_pdl(kern, dim3(static_cast<unsigned>(R * l.units_max)), dim3(128), smem, stream, a,
                       static_cast<int>(i0), nq, static_cast<const int32_t*>(inv_order),
                       static_cast<const int32_t*>(inv_offsets), static_cast<const int2*>(units),
                       static_cast<const int32_t*>(count), part_o, part_lse,
                       static_cast<int>(l.units_max)));
    const int64_t rows = R * nq * a.G;
    FKC_TRY(launch_pdl(tiles_join_kernel<T>, dim3(static_cast<unsigned>((rows + 7) / 8)), dim3(256), 0,
                       stream, a, static_cast<int>(i0), nq, static_cast<const float*>(part_o),
                       static_cast<const float*>(part_lse), out, lse, rows));
  }
  return FKC_OK;
}

template <typename T>
int fwd_dtype(const Args& a, void* out, float* lse, void* ws, cudaStream_t stream) {
  T* o = static_cast<T*>(out);
  uint8_t* w = static_cast<uint8_t*>(ws);
  return a.D <= 64 ? fwd_typed<T, 64>(a, o, lse, w, stream) : fwd_typed<T, 128>(a, o, lse, w, stream);
}

}  // namespace

bool use_tiles(const Args& a) {
  const int64_t R = static_cast<int64_t>(a.batch) * a.Hkv;
  const int64_t per_round = queries_per_round(a) * a.top;
  // rows of a cluster fill half a tile, keys of a cluster repay its parts, and there are
  // enough tiles for the GPU
  return per_round * a.G >= 64ll * a.K && a.N / a.K >= 4 * a.G + 8 &&
         R * a.Nq * a.top * a.G >= 148ll * kRows;
}

size_t tiles_forward_workspace_bytes(const Args& a) { return fwd_layout(a).total; }

int launch_tiles_forward(const Args& a, int dtype, void* out, float* lse, void* ws,
                         cudaStream_t stream) {
  return dtype == FKC_DTYPE_F16 ? fwd_dtype<__half>(a, out, lse, ws, stream)
                                : fwd_dtype<__nv_bfloat16>(a, out, lse, ws, stream);
}

}  // namespace attn
}  // namespace fkc
