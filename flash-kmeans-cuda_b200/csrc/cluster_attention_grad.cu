// Gradients of attention over selected clusters. With P = exp(scale S - lse) and
// delta = rowsum(dout * out) = rowsum(P dP) per query and head,
//
//   dV = P^T dout,  dP = dout V^T,  dS = scale P (dP - delta),  dQ = dS K,  dK = dS^T Q.
//
//   dQ     (attn_dq_kernel)     the forward's walk: one warp per query and group, keys and
//          values gathered in tiles of 16, S^T and dP^T formed transposed, dQ^T += K^T dS^T.
//          It walks twice, first for delta = sum of P dP (all that is done where dQ is not wanted): keys
//          lie close to one another within a cluster, and a cache's have offsets in common, so that
//          what a rounded delta is off by adds up over them (dS no longer sums to zero). With delta
//          from the 16-bit out, dQ of one cluster of 30 keys was off by 0.0051 of its norm, of 8
//          clusters of 64 keys with a common offset ten times their spread by 0.019; its own rounding
//          is 0.0017, and that is what is left.
//   dK, dV (attn_dkv_kernel)    one CTA per 64 keys of a cluster, whose keys and values stay in
//          shared memory. The queries that selected the cluster come from the same grouping
//          that orders the keys (sel as ids: entry e is query e / top), their heads side by
//          side as columns; tiles of 32 columns of Q and dout are gathered in a double buffer.
//          The four warps take 16 keys each; the sums over all queries and heads of the group
//          stay in fp32 registers, in ascending query order, so two runs give the same bits.
//
// P and dS enter the second products as two terms of the 16-bit input type, which their operands have:
// the gradients are off by their own last rounding (0.0017 of the norm with bf16; with one term each
// 0.0024). Sums are fp32 and rounded once on the way out. Keys in no cluster get zeros.
//
// Bound by the products and the gathers that feed them: 24 * D flops per (query head, key) pair, of which
// the formulas need 10: S and dP are formed three times and the other three products have two terms. 256
// queries x 8 rows of 1 head, 16 of 512 clusters of 24 keys: 296 us (by clusters 330); 2048 queries: 1186 us
// (by clusters 368).
#include <algorithm>

#include "cluster_attention.cuh"
#include "fkc_common.cuh"

namespace fkc {
namespace attn {
namespace {

constexpr int kWarps = 4;
constexpr int kTile = 16;  // keys per tile of the dQ walk
constexpr int kKeys = 64;  // keys per CTA of the dK, dV walk
constexpr int kCols = 32;  // (query, head) columns per step of it

template <int DP, int STAGES>
constexpr int ring_bytes() {
  return STAGES * 2 * kTile * DP * 2;
}
template <int DP, int STAGES>
__host__ __device__ constexpr int warp_smem(int top) {
  return ring_bytes<DP, STAGES>() + ((STAGES * 4 + (2 * top + 1) * 4 + 15) / 16) * 16;
}

// dq may be null: delta alone. largest, with dK: the largest A of each row of clusters.
template <typename T, int DP, int NT, int STAGES>
__global__ void __launch_bounds__(32 * kWarps) attn_dq_kernel(Args a, const T* __restrict__ dout,
                                                              const float* __restrict__ lse,
                                                              float* __restrict__ delta,
                                                              T* __restrict__ dq, float* __restrict__ largest, int chunks,
                                                              int64_t units) {
  constexpr int KS = DP / 16;
  extern __shared__ __align__(16) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t4 = lane & 3;
  uint8_t* mine = smem + static_cast<size_t>(warp) * warp_smem<DP, STAGES>(a.top);
  const uint32_t ring = static_cast<uint32_t>(__cvta_generic_to_shared(mine));
  uint32_t* masks = reinterpret_cast<uint32_t*>(mine + ring_bytes<DP, STAGES>());
  if (a.D < DP)
    for (int o = lane * 16; o < ring_bytes<DP, STAGES>(); o += 512)
      *reinterpret_cast<uint4*>(mine + o) = make_uint4(0, 0, 0, 0);
  __syncwarp();
  pdl_wait();
  const int64_t unit = static_cast<int64_t>(blockIdx.x) * kWarps + warp;
  if (unit >= units) return;
  const int hc = static_cast<int>(unit % chunks);
  const int64_t qi = unit / chunks;
  const int r = static_cast<int>(qi / a.Nq), i = static_cast<int>(qi % a.Nq);
  const int b = r / a.Hkv, hk = r - b * a.Hkv;
  const int h0 = hk * a.G + hc * 8 * NT;
  const int heads = min(8 * NT, a.G - hc * 8 * NT);
  const int pos = a.q_pos != nullptr ? a.q_pos[static_cast<int64_t>(b) * a.Nq + i] : a.N;
  auto flat = [&](int h) { return (static_cast<int64_t>(b) * a.Hq + h0 + h) * a.Nq + i; };

  uint32_t qf[NT][KS][2], df[NT][KS][2];
  float ls[NT][2], dl[NT][2], pw[NT][2];  // pw: the power of two of dS (1 in the first pass)
  const T* qb = static_cast<const T*>(a.q) + b * a.qs.b + i * a.qs.n;
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const bool on = n * 8 + g < heads;
    const T* row = qb + static_cast<int64_t>(h0 + (on ? n * 8 + g : 0)) * a.qs.h;
    const T* drow = dout + flat(on ? n * 8 + g : 0) * a.D;
#pragma unroll
    for (int kk = 0; kk < KS; ++kk)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int d = kk * 16 + e * 8 + t4 * 2;
        const bool in = on && d < a.D;
        qf[n][kk][e] = in ? *reinterpret_cast<const uint32_t*>(row + d) : 0u;
        df[n][kk][e] = in ? *reinterpret_cast<const uint32_t*>(drow + d) : 0u;
      }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int h = n * 8 + t4 * 2 + e;
      ls[n][e] = h < heads ? lse[flat(h)] * kLog2e : 0.f;
      dl[n][e] = 0.f, pw[n][e] = 1.f;
    }
  }
  KeyList list;
  list.build(a, r, i, reinterpret_cast<int*>(masks + STAGES));
  const int tiles = (list.total + kTile - 1) / kTile;
  const int32_t* order = a.order + static_cast<int64_t>(r) * a.N;
  const T* kb = static_cast<const T*>(a.k) + b * a.ks.b + hk * a.ks.h;
  const T* vb = static_cast<const T*>(a.v) + b * a.vs.b + hk * a.vs.h;
  const int dchunks = a.D / 8;
  int cur = 0, idx = -1, idx_next = -1;
  auto issue = [&](int t) {
    const int half = t & 1;
    if (half == 0) {
      idx = KeyList::visible(a, idx_next, pos);
      idx_next = list.key(a, order, (t + 2) * kTile + lane, cur);
    }
    const int stage = t % STAGES;
    const uint32_t kt = ring + stage * (2 * kTile * DP * 2), vt = kt + kTile * DP * 2;
    const uint32_t live = __ballot_sync(0xFFFFFFFFu, idx >= 0) >> (half * 16) & 0xFFFFu;
    if (lane == 0) masks[stage] = live;
    constexpr int CH = DP / 8;
#pragma unroll
    for (int it = 0; it < kTile * CH / 32; ++it) {
      const int key = (it * 32 + lane) / CH, c = (it * 32 + lane) % CH;
      const int row = __shfl_sync(0xFFFFFFFFu, idx, half * 16 + key);
      if (c < dchunks) {
        const int64_t at = row < 0 ? 0 : row;
        mma::cp_async16(kt + tile_at<DP>(key, c), kb + at * a.ks.n + c * 8, row >= 0);
        mma::cp_async16(vt + tile_at<DP>(key, c), vb + at * a.vs.n + c * 8, row >= 0);
      }
    }
  };
  float o[NT][KS][4];
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int kk = 0; kk < KS; ++kk)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[n][kk][e] = 0.f;
  const float sc = a.scale * kLog2e;
  // pass 0: delta = sum of P dP; pass 1: dQ
#pragma unroll 1
  for (int pass = 0; pass < 2; ++pass) {
  cur = 0;
  idx_next = list.key(a, order, lane, cur);
#pragma unroll
  for (int s = 0; s < STAGES - 1; ++s) {
    if (s < tiles) issue(s);
    mma::cp_async_commit();
  }
  float sum[NT][2], mag[NT][2];
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int e = 0; e < 2; ++e) sum[n][e] = mag[n][e] = 0.f;
  for (int t = 0; t < tiles; ++t) {
    mma::cp_async_wait<STAGES - 2>();
    __syncwarp();
    if (t + STAGES - 1 < tiles) issue(t + STAGES - 1);
    mma::cp_async_commit();
    const int stage = t % STAGES;
    const uint32_t live = masks[stage];
    if (live == 0) continue;
    const uint32_t kt = ring + stage * (2 * kTile * DP * 2), vt = kt + kTile * DP * 2;
    float s[NT][4], dp[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[n][e] = 0.f, dp[n][e] = 0.f;
#pragma unroll
    for (int kk = 0; kk < KS; ++kk) {
      uint32_t f[4], fv[4];
      load_a<DP>(f, kt, 0, kk);
      load_a<DP>(fv, vt, 0, kk);
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        mma::m16n8k16<T>(s[n], f, qf[n][kk][0], qf[n][kk][1]);
        mma::m16n8k16<T>(dp[n], fv, df[n][kk][0], df[n][kk][1]);
      }
    }
    const bool on0 = live >> g & 1, on1 = live >> (g + 8) & 1;
    uint32_t hi[NT][2], lo[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        s[n][e] = on0 ? exp2f(s[n][e] * sc - ls[n][e]) * ((dp[n][e] - dl[n][e]) * pw[n][e]) : 0.f;
        s[n][2 + e] = on1 ? exp2f(s[n][2 + e] * sc - ls[n][e]) * ((dp[n][2 + e] - dl[n][e]) * pw[n][e]) : 0.f;
        sum[n][e] += s[n][e] + s[n][2 + e];
        if (Range<T>::kNarrow) mag[n][e] += fabsf(s[n][e]) + fabsf(s[n][2 + e]);
      }
    }
    if (pass == 0) continue;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        uint32_t first, second;
        mma::split2<T>(s[n][2 * e], s[n][2 * e + 1], first, second);
        hi[n][e] = mma::movmatrix_trans(first);
        lo[n][e] = mma::movmatrix_trans(second);
      }
    }
#pragma unroll
    for (int md = 0; md < KS; ++md) {
      uint32_t f[4];
      load_a_trans<DP>(f, kt, 0, md);
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        mma::m16n8k16<T>(o[n][md], f, hi[n][0], hi[n][1]);
        mma::m16n8k16<T>(o[n][md], f, lo[n][0], lo[n][1]);
      }
    }
  }
  mma::cp_async_wait<0>();
  __syncwarp();
  if (pass == 0) {
    float most = 0.f;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float d = sum[n][e], A = mag[n][e];
#pragma unroll
        for (int o = 4; o <= 16; o <<= 1) {
          d += __shfl_xor_sync(0xFFFFFFFFu, d, o);
          if (Range<T>::kNarrow) A += __shfl_xor_sync(0xFFFFFFFFu, A, o);
        }
        dl[n][e] = d;
        if (Range<T>::kNarrow) {
          pw[n][e] = power(A);
          if (A < INFINITY) most = fmaxf(most, A);
        }
        const int h = n * 8 + t4 * 2 + e;
        if (g == 0 && h < heads) delta[flat(h)] = d;
      }
    if (Range<T>::kNarrow && largest != nullptr) {
      most = fmaxf(most, __shfl_xor_sync(0xFFFFFFFFu, most, 1));
      most = fmaxf(most, __shfl_xor_sync(0xFFFFFFFFu, most, 2));
      if (lane == 0) note_largest(largest + r, most);
    }
    if (dq == nullptr) return;
  }
  }
  float out[NT][2];  // what the sums are multiplied by
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int e = 0; e < 2; ++e) out[n][e] = a.scale * inverse_power(pw[n][e]);
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int md = 0; md < KS; ++md) {
      const uint32_t lo =
          mma::movmatrix_trans(mma::pack2<T>(o[n][md][0] * out[n][0], o[n][md][1] * out[n][1]));
      const uint32_t hi =
          mma::movmatrix_trans(mma::pack2<T>(o[n][md][2] * out[n][0], o[n][md][3] * out[n][1]));
      const int h = n * 8 + g, d = md * 16 + t4 * 2;
      if (h < heads) {
        T* row = dq + flat(h) * a.D;
        if (d < a.D) *reinterpret_cast<uint32_t*>(row + d) = lo;
        if (d + 8 < a.D) *reinterpret_cast<uint32_t*>(row + d + 8) = hi;
      }
    }
}

// tile_off[r, c]: first key tile of cluster c among the row's; tile_off[r, K]: their number.
__global__ void __launch_bounds__(1024) key_tiles_kernel(Args a, int32_t* __restrict__ tile_off,
                                                         int32_t* odd, float* __restrict__ largest) {
  __shared__ int warp_total[32];
  pdl_wait();
  if (blockIdx.x == 0 && threadIdx.x == 0) *odd = 0;
  if (threadIdx.x == 0) largest[blockIdx.x] = 0.f;
  const int r = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int32_t* out = tile_off + static_cast<int64_t>(r) * (a.K + 1);
  int carry = 0;
  for (int c0 = 0; c0 < a.K; c0 += 1024) {
    const int c = c0 + threadIdx.x;
    int s, e;
    cluster_span(a, r, c, s, e);
    const int n = (e - s + kKeys - 1) / kKeys;
    int inc = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xFFFFFFFFu, inc, o);
      if (lane >= o) inc += u;
    }
    __syncthreads();
    if (lane == 31) warp_total[warp] = inc;
    __syncthreads();
    int before = carry;
    for (int w = 0; w < 32; ++w) {
      if (w < warp) before += warp_total[w];
      carry += warp_total[w];
    }
    if (c < a.K) out[c] = before + inc - n;
  }
  if (threadIdx.x == 0) out[a.K] = carry;
}

template <int DP>
struct DkvSmem {
  static constexpr int kTileBytes = kKeys * DP * 2;
  static constexpr int kColBytes = kCols * DP * 2;
  static constexpr int kK = 0, kV = kTileBytes;
  static constexpr int kQ = 2 * kTileBytes;               // two buffers of Q, then of dout
  static constexpr int kDo = kQ + 2 * kColBytes;
  static constexpr int kBytes = kDo + 2 * kColBytes;
};

template <typename T, int DP>
__global__ void __launch_bounds__(128) attn_dkv_kernel(
    Args a, const T* __restrict__ dout, const float* __restrict__ lse,
    const float* __restrict__ delta, const int32_t* __restrict__ inv_order,
    const int32_t* __restrict__ inv_offsets, const int32_t* __restrict__ tile_off,
    const float* __restrict__ largest, T* __restrict__ dk, T* __restrict__ dv,
    int32_t* __restrict__ odd, int tiles_max) {
  constexpr int KS = DP / 16, CH = DP / 8;
  using S = DkvSmem<DP>;
  extern __shared__ __align__(16) uint8_t smem[];
  // of two column tiles: lse * log2(e) less P's shift, delta, the query's position (-1: reads nothing)
  __shared__ float c_lse[2][kCols], c_delta[2][kCols];
  __shared__ int c_pos[2][kCols];
  __shared__ int64_t c_q[2][kCols], c_do[2][kCols];  // row offsets
  __shared__ int s_row[kKeys];                       // the keys' positions, -1 behind the last
  __shared__ int s_min;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int g = lane >> 2, t4 = lane & 3;
  const uint32_t base = static_cast<uint32_t>(__cvta_generic_to_shared(smem));
  if (a.D < DP)
    for (int o = tid * 16; o < S::kBytes; o += 2048)
      *reinterpret_cast<uint4*>(smem + o) = make_uint4(0, 0, 0, 0);
  if (tid == 0) s_min = INT_MAX;
  __syncthreads();
  pdl_wait();
  const int r = blockIdx.x / tiles_max, tile = blockIdx.x - r * tiles_max;
  const int b = r / a.Hkv, hk = r - b * a.Hkv;
  const int32_t* off = tile_off + static_cast<int64_t>(r) * (a.K + 1);
  if (tile >= off[a.K]) return;
  int c = 0;  // the last cluster whose first tile is not behind this one
  for (int lo = 0, hi = a.K - 1; lo <= hi;) {
    const int mid = (lo + hi) / 2;
    if (off[mid] <= tile)
      c = mid, lo = mid + 1;
    else
      hi = mid - 1;
  }
  int s0, s1;
  cluster_span(a, r, c, s0, s1);
  s0 += (tile - off[c]) * kKeys;
  const int keys = min(kKeys, s1 - s0);
  if (tid < kKeys) {
    int row = -1;
    if (tid < keys) {
      row = a.order[static_cast<int64_t>(r) * a.N + s0 + tid];
      if (row < 0 || row >= a.N) row = -1;
    }
    s_row[tid] = row;
    if (row >= 0) atomicMin(&s_min, row);
  }
  __syncthreads();
  const int first = s_min;  // a query before it sees none of these keys
  const T* kb = static_cast<const T*>(a.k) + b * a.ks.b + hk * a.ks.h;
  const T* vb = static_cast<const T*>(a.v) + b * a.vs.b + hk * a.vs.h;
  const int dchunks = a.D / 8;
  for (int e = tid; e < kKeys * CH; e += 128) {
    const int key = e / CH, ch = e % CH;
    if (ch >= dchunks) continue;
    const int row = s_row[key];
    const int64_t at = row < 0 ? 0 : row;
    mma::cp_async16(base + S::kK + tile_at<DP>(key, ch), kb + at * a.ks.n + ch * 8, row >= 0);
    mma::cp_async16(base + S::kV + tile_at<DP>(key, ch), vb + at * a.vs.n + ch * 8, row >= 0);
  }
  const int32_t* iof = inv_offsets + static_cast<int64_t>(r) * (a.K + 1);
  const int e0 = iof[c];
  const int64_t cols = static_cast<int64_t>(iof[c + 1] - e0) * a.G;
  const int32_t* entries = inv_order + static_cast<int64_t>(r) * a.Nq * a.top + e0;
  const int steps = static_cast<int>((cols + kCols - 1) / kCols);

  // Column data of step s: loaded by the first 32 threads one step before its copies start.
  struct Col {
    float lse, delta;
    int pos;
    int64_t q, d;
  };
  auto column = [&](int s) {
    Col x{0.f, 0.f, -1, 0, 0};
    const int64_t col = static_cast<int64_t>(s) * kCols + lane;
    if (col >= cols) return x;
    const int64_t e = col / a.G;
    const int h = hk * a.G + static_cast<int>(col - e * a.G);
    const int i = entries[e] / a.top;
    const int p = a.q_pos != nullptr ? a.q_pos[static_cast<int64_t>(b) * a.Nq + i] : a.N;
    if (p < first) return x;
    const int64_t at = (static_cast<int64_t>(b) * a.Hq + h) * a.Nq + i;
    x.pos = p;
    x.lse = lse[at] * kLog2e - Range<T>::kShift;
    x.delta = delta[at];
    x.q = b * a.qs.b + h * a.qs.h + i * a.qs.n;
    x.d = at * a.D;
    return x;
  };
  auto publish = [&](int s, const Col& x) {
    const int u = s & 1;
    c_lse[u][lane] = x.lse;
    c_delta[u][lane] = x.delta;
    c_pos[u][lane] = x.pos;
    c_q[u][lane] = x.q;
    c_do[u][lane] = x.d;
  };
  auto copy = [&](int s) {
    const int u = s & 1;
    const T* q = static_cast<const T*>(a.q);
#pragma unroll
    for (int it = 0; it < kCols * CH / 128; ++it) {
      const int e = it * 128 + tid, col = e / CH, ch = e % CH;
      if (ch >= dchunks) continue;
      const bool on = c_pos[u][col] >= 0;
      mma::cp_async16(base + S::kQ + u * S::kColBytes + tile_at<DP>(col, ch),
                      q + (on ? c_q[u][col] + ch * 8 : 0), on);
      mma::cp_async16(base + S::kDo + u * S::kColBytes + tile_at<DP>(col, ch),
                      dout + (on ? c_do[u][col] + ch * 8 : 0), on);
    }
  };
  float ak[DP / 8][4], av[DP / 8][4];
#pragma unroll
  for (int n = 0; n < DP / 8; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) ak[n][e] = 0.f, av[n][e] = 0.f;
  Col next{};
  if (warp == 0) {
    if (steps > 0) publish(0, column(0));
    next = column(1);
  }
  __syncthreads();
  if (steps > 0) copy(0);
  mma::cp_async_commit();
  const int row0 = s_row[warp * 16 + g], row1 = s_row[warp * 16 + 8 + g];
  const float sc = a.scale * kLog2e;
  const float pw = Range<T>::kNarrow ? power(largest[r]) : 1.f, ds_power = pw * Range<T>::unshift();
  const bool idle = warp * 16 >= keys;  // no key for this warp
  for (int s = 0; s < steps; ++s) {
    // the other buffer was read in step s - 1, which the barrier below ended
    if (warp == 0 && s + 1 < steps) publish(s + 1, next);
    mma::cp_async_wait<0>();
    __syncthreads();
    if (s + 1 < steps) copy(s + 1);
    mma::cp_async_commit();
    if (warp == 0) next = column(s + 2);
    const int u = s & 1;
    const uint32_t qt = base + S::kQ + u * S::kColBytes, dt = base + S::kDo + u * S::kColBytes;
    if (!idle) {
      float ss[4][4], dp[4][4];
#pragma unroll
      for (int n = 0; n < 4; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) ss[n][e] = 0.f, dp[n][e] = 0.f;
#pragma unroll
      for (int kk = 0; kk < KS; ++kk) {
        uint32_t fk[4], fv[4];
        load_a<DP>(fk, base + S::kK, warp * 16, kk);
        load_a<DP>(fv, base + S::kV, warp * 16, kk);
#pragma unroll
        for (int n = 0; n < 4; n += 2) {
          uint32_t f[4];
          load_b<DP>(f, qt, n * 8, kk);
          mma::m16n8k16<T>(ss[n], fk, f[0], f[1]);
          mma::m16n8k16<T>(ss[n + 1], fk, f[2], f[3]);
          load_b<DP>(f, dt, n * 8, kk);
          mma::m16n8k16<T>(dp[n], fv, f[0], f[1]);
          mma::m16n8k16<T>(dp[n + 1], fv, f[2], f[3]);
        }
      }
      // in two terms, (key g, columns) and (key g + 8, columns)
      uint32_t pp[4][2], pl[4][2], ds[4][2], dl2[4][2];
#pragma unroll
      for (int n = 0; n < 4; ++n) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int col = n * 8 + t4 * 2 + e;
          const float ls = c_lse[u][col], dl = c_delta[u][col];
          const int pos = c_pos[u][col];
          const bool on0 = row0 >= 0 && row0 <= pos, on1 = row1 >= 0 && row1 <= pos;
          const float p0 = on0 ? exp2f(ss[n][e] * sc - ls) : 0.f;
          const float p1 = on1 ? exp2f(ss[n][2 + e] * sc - ls) : 0.f;
          ss[n][e] = p0;
          ss[n][2 + e] = p1;
          dp[n][e] = on0 ? p0 * ((dp[n][e] - dl) * ds_power) : 0.f;
          dp[n][2 + e] = on1 ? p1 * ((dp[n][2 + e] - dl) * ds_power) : 0.f;
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          mma::split2_weights<T>(ss[n][2 * e], ss[n][2 * e + 1], pp[n][e], pl[n][e]);
          mma::split2<T>(dp[n][2 * e], dp[n][2 * e + 1], ds[n][e], dl2[n][e]);
        }
      }
#pragma unroll
      for (int cc = 0; cc < 2; ++cc) {  // 16 columns as depth
        const uint32_t fp[4] = {pp[2 * cc][0], pp[2 * cc][1], pp[2 * cc + 1][0], pp[2 * cc + 1][1]};
        const uint32_t fd[4] = {ds[2 * cc][0], ds[2 * cc][1], ds[2 * cc + 1][0], ds[2 * cc + 1][1]};
        const uint32_t fq[4] = {pl[2 * cc][0], pl[2 * cc][1], pl[2 * cc + 1][0], pl[2 * cc + 1][1]};
        const uint32_t fl[4] = {dl2[2 * cc][0], dl2[2 * cc][1], dl2[2 * cc + 1][0], dl2[2 * cc + 1][1]};
#pragma unroll
        for (int nd = 0; nd < KS; ++nd) {
          uint32_t f[4];
          load_b_trans<DP>(f, dt, cc * 16, nd);
          mma::m16n8k16<T>(av[2 * nd], fp, f[0], f[1]);
          mma::m16n8k16<T>(av[2 * nd + 1], fp, f[2], f[3]);
          mma::m16n8k16<T>(av[2 * nd], fq, f[0], f[1]);
          mma::m16n8k16<T>(av[2 * nd + 1], fq, f[2], f[3]);
          load_b_trans<DP>(f, qt, cc * 16, nd);
          mma::m16n8k16<T>(ak[2 * nd], fd, f[0], f[1]);
          mma::m16n8k16<T>(ak[2 * nd + 1], fd, f[2], f[3]);
          mma::m16n8k16<T>(ak[2 * nd], fl, f[0], f[1]);
          mma::m16n8k16<T>(ak[2 * nd + 1], fl, f[2], f[3]);
        }
      }
    }
    __syncthreads();  // all reads of this step's buffers and column data
  }
  mma::cp_async_wait<0>();
  const int64_t kv = (static_cast<int64_t>(b) * a.Hkv + hk) * a.N;
  const float k_out = a.scale * inverse_power(pw), v_out = Range<T>::unshift();
  float bad = 0.f;
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const int row = half == 0 ? row0 : row1;
    if (row < 0) continue;
#pragma unroll
    for (int n = 0; n < DP / 8; ++n) {
#pragma unroll
      for (int e = 0; e < 2; ++e) bad = not_finite(ak[n][half * 2 + e], not_finite(av[n][half * 2 + e], bad));
      const int d = n * 8 + t4 * 2;
      if (d >= a.D) continue;
      const int64_t at = (kv + row) * a.D + d;
      *reinterpret_cast<uint32_t*>(dk + at) =
          mma::pack2<T>(ak[n][half * 2] * k_out, ak[n][half * 2 + 1] * k_out);
      *reinterpret_cast<uint32_t*>(dv + at) =
          mma::pack2<T>(av[n][half * 2] * v_out, av[n][half * 2 + 1] * v_out);
    }
  }
  if (bad != 0.f) *odd = 1;
}

struct GradLayout {
  size_t delta, odd, largest, inv_order, inv_offsets, tile_off, group, tiles, total;
};

GradLayout grad_layout(const Args& a) {
  GradLayout l{};
  const int64_t R = static_cast<int64_t>(a.batch) * a.Hkv;
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t p = at;
    at += align_up(bytes, 256);
    return p;
  };
  l.delta = take(static_cast<size_t>(a.batch) * a.Hq * a.Nq * 4);
  if (use_tiles_grad(a)) {
    l.tiles = take(tiles_backward_workspace_bytes(a));
    l.total = at;
    return l;
  }
  l.odd = take(4);
  l.largest = take(static_cast<size_t>(R) * 4);
  l.inv_order = take(static_cast<size_t>(R) * a.Nq * a.top * 4);
  l.inv_offsets = take(static_cast<size_t>(R) * (a.K + 1) * 4);
  l.tile_off = take(static_cast<size_t>(R) * (a.K + 1) * 4);
  l.group = take(group_workspace_bytes(R, static_cast<int64_t>(a.Nq) * a.top, a.K));
  l.total = at;
  return l;
}

template <typename T, int DP, int NT>
int dq_typed(const Args& a, const T* dout, const float* lse, float* delta, T* dq, float* largest,
             cudaStream_t stream) {
  constexpr int STAGES = 3;
  const int chunks = (a.G + 8 * NT - 1) / (8 * NT);
  const int64_t units = static_cast<int64_t>(a.batch) * a.Hkv * a.Nq * chunks;
  const int smem = kWarps * warp_smem<DP, STAGES>(a.top);
  auto kern = attn_dq_kernel<T, DP, NT, STAGES>;
  FKC_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  return launch_pdl(kern, dim3(static_cast<unsigned>((units + kWarps - 1) / kWarps)),
                    dim3(32 * kWarps), smem, stream, a, dout, lse, delta, dq, largest, chunks, units);
}

template <typename T, int DP>
int grad_typed(const Args& a, int dtype, const float* lse, const T* dout, T* dq, T* dk, T* dv,
               uint8_t* ws, cudaStream_t stream) {
  const GradLayout l = grad_layout(a);
  float* delta = reinterpret_cast<float*>(ws + l.delta);
  int32_t* odd = reinterpret_cast<int32_t*>(ws + l.odd);
  int32_t* inv_order = reinterpret_cast<int32_t*>(ws + l.inv_order);
  int32_t* inv_offsets = reinterpret_cast<int32_t*>(ws + l.inv_offsets);
  int32_t* tile_off = reinterpret_cast<int32_t*>(ws + l.tile_off);
  const int64_t R = static_cast<int64_t>(a.batch) * a.Hkv;
  if (use_tiles_grad(a))
    return launch_tiles_backward(a, dtype, lse, delta, dout, dq, dk, dv, ws + l.tiles, stream);
  float* largest = dk != nullptr ? reinterpret_cast<float*>(ws + l.largest) : nullptr;
  if (dk != nullptr) {
    FKC_TRY(launch_group(a.sel, false, static_cast<int64_t>(a.Nq) * a.top, inv_order, inv_offsets, R,
                         static_cast<int64_t>(a.Nq) * a.top, a.K, ws + l.group, stream));
    FKC_TRY(launch_pdl(key_tiles_kernel, dim3(static_cast<unsigned>(R)), dim3(1024), 0, stream, a,
                       tile_off, odd, largest));
  }
  if (a.G <= 8)
    FKC_TRY((dq_typed<T, DP, 1>(a, dout, lse, delta, dq, largest, stream)));
  else
    FKC_TRY((dq_typed<T, DP, 2>(a, dout, lse, delta, dq, largest, stream)));
  if (dk == nullptr) return FKC_OK;
  const size_t kv_bytes = static_cast<size_t>(R) * a.N * a.D * sizeof(T);
  FKC_TRY(launch_zero_fill(dk, kv_bytes, stream));
  FKC_TRY(launch_zero_fill(dv, kv_bytes, stream));
  const int64_t tiles_max = std::min<int64_t>(a.K, a.N) + a.N / kKeys;
  FKC_REQUIRE(R * tiles_max <= 2147483647ll, "attention: too many key tiles");
  auto kern = attn_dkv_kernel<T, DP>;
  const int smem = DkvSmem<DP>::kBytes;
  FKC_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  FKC_TRY(launch_pdl(kern, dim3(static_cast<unsigned>(R * tiles_max)), dim3(128), smem, stream, a,
                     dout, lse, static_cast<const float*>(delta),
                     static_cast<const int32_t*>(inv_order),
                     static_cast<const int32_t*>(inv_offsets),
                     static_cast<const int32_t*>(tile_off), static_cast<const float*>(largest), dk, dv,
                     odd, static_cast<int>(tiles_max)));
  // dq's walk takes one query's keys at a time: none that the query does not see
  return launch_again(a, dtype, odd, lse, delta, dout, nullptr, inv_order, inv_offsets, dk, dv, stream);
}

template <typename T>
int grad_dtype(const Args& a, int dtype, const float* lse, const void* dout, void* dq, void* dk, void* dv,
               void* ws, cudaStream_t stream) {
  const T* d = static_cast<const T*>(dout);
  T *q = static_cast<T*>(dq), *k = static_cast<T*>(dk), *v = static_cast<T*>(dv);
  uint8_t* w = static_cast<uint8_t*>(ws);
  return a.D <= 64 ? grad_typed<T, 64>(a, dtype, lse, d, q, k, v, w, stream)
                   : grad_typed<T, 128>(a, dtype, lse, d, q, k, v, w, stream);
}

}  // namespace

size_t backward_workspace_bytes(const Args& a) { return grad_layout(a).total; }

int launch_backward(const Args& a, int dtype, const float* lse, const void* dout, void* dq, void* dk,
                    void* dv, void* ws, cudaStream_t stream) {
  return dtype == FKC_DTYPE_F16
             ? grad_dtype<__half>(a, dtype, lse, dout, dq, dk, dv, ws, stream)
             : grad_dtype<__nv_bfloat16>(a, dtype, lse, dout, dq, dk, dv, ws, stream);
}

}  // namespace attn
}  // namespace fkc
