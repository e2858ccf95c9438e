// Attention of queries over the keys of the clusters that each of them selected.
//
//   out[b, h, i] = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale * q . k_j - max)
//   lse[b, h, i] = max + log(sum_j p_j)
//
// over the positions j of the clusters sel[r, i, :] (r = b * Hkv + h / G; a cluster
// listed twice counts twice) with j <= q_pos[b, i]; a query that sees nothing gets
// zeros and -inf.
//
// One warp takes one (row r, query i), all G heads of the group, and walks the keys
// of its clusters in tiles of 16: the keys and values of a tile are gathered through
// order with 16-byte asynchronous copies into the warp's own ring in shared memory,
// scores are formed transposed, S^T = K Q^T (keys x heads, m16n8k16: 8 heads fill
// the instruction's narrow side, which a tile of queries could not since every query
// has its own keys), the running maximum and sum stay in fp32 registers, and O^T +=
// V^T P^T takes P^T straight from the score registers (transposed in the register
// file by movmatrix). Warps never wait for one another.
//
// P enters the second product as two terms of the 16-bit input type, which its operands have (2^-16 of it
// is lost with bf16), so that out is off by its own last rounding alone: 0.0017 of its norm with bf16, 0.0022
// with one term, for 1 us of one query's 11 and of a batch's 52. The sum of a row uses the values themselves.
//
// Bound by the gather: 4 * D bytes per key and query row from L2 or HBM against
// 4 * D * G flops. Where there are few queries the keys of one are split over
// several warps (at least four tiles each, about 8 per SM in all), and attn_join_kernel joins the
// parts by their log-sum-exp.
//
// 16 sequences x 8 rows, one query each, 64 of 1024 clusters, D = 128: on average 3425 keys a query,
// 224 MB, in 52 us, 4.3 TB/s (the join 5 us, with eight parts' loads in flight; one after another
// they took 8). While its SMs are busy the walk moves some 6 TB/s; it loses a fifth to the
// largest queries, whose warps end last (twice as many, shorter parts: 64 us, since each warp
// builds its list). One query of 512 keys: 11 us, a chain of list, gather, products and join.
#include <algorithm>

#include "cluster_attention.cuh"

namespace fkc {
namespace attn {
namespace {

constexpr int kWarps = 4;
constexpr int kTile = 16;

template <int DP, int STAGES>
constexpr int ring_bytes() {
  return STAGES * 2 * kTile * DP * 2;
}

// Per-warp shared memory: the ring, the tiles' validity masks, the key list.
template <int DP, int STAGES>
__host__ __device__ constexpr int warp_smem(int top) {
  return ring_bytes<DP, STAGES>() + ((STAGES * 4 + (2 * top + 1) * 4 + 15) / 16) * 16;
}

template <typename T, int DP, int NT, int STAGES>
__global__ void __launch_bounds__(32 * kWarps) attn_fwd_kernel(Args a, T* __restrict__ out,
                                                               float* __restrict__ lse,
                                                               float* __restrict__ part_o,
                                                               float* __restrict__ part_lse,
                                                               int chunks, int nsplit,
                                                               int64_t units) {
  constexpr int KS = DP / 16;
  extern __shared__ __align__(16) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t4 = lane & 3;
  uint8_t* mine = smem + static_cast<size_t>(warp) * warp_smem<DP, STAGES>(a.top);
  const uint32_t ring = static_cast<uint32_t>(__cvta_generic_to_shared(mine));
  uint32_t* masks = reinterpret_cast<uint32_t*>(mine + ring_bytes<DP, STAGES>());
  if (a.D < DP)  // columns past D are never copied: they stay zero
    for (int o = lane * 16; o < ring_bytes<DP, STAGES>(); o += 512)
      *reinterpret_cast<uint4*>(mine + o) = make_uint4(0, 0, 0, 0);
  __syncwarp();
  pdl_wait();
  const int64_t unit = static_cast<int64_t>(blockIdx.x) * kWarps + warp;
  if (unit >= units) return;
  const int split = static_cast<int>(unit % nsplit);
  const int64_t u1 = unit / nsplit;
  const int hc = static_cast<int>(u1 % chunks);
  const int64_t qi = u1 / chunks;  // r * Nq + i
  const int r = static_cast<int>(qi / a.Nq), i = static_cast<int>(qi % a.Nq);
  const int b = r / a.Hkv, hk = r - b * a.Hkv;
  const int h0 = hk * a.G + hc * 8 * NT;        // first query head of this unit
  const int heads = min(8 * NT, a.G - hc * 8 * NT);
  const int pos = a.q_pos != nullptr ? a.q_pos[static_cast<int64_t>(b) * a.Nq + i] : a.N;

  // Q^T as B fragments: head g (of each n tile), elements 16 kk + 2 t4 (+ 8)
  uint32_t qf[NT][KS][2];
  const T* qb = static_cast<const T*>(a.q) + b * a.qs.b + i * a.qs.n;
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const bool on = n * 8 + g < heads;
    const T* row = qb + static_cast<int64_t>(h0 + (on ? n * 8 + g : 0)) * a.qs.h;
#pragma unroll
    for (int kk = 0; kk < KS; ++kk)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int d = kk * 16 + e * 8 + t4 * 2;
        qf[n][kk][e] = on && d < a.D ? *reinterpret_cast<const uint32_t*>(row + d) : 0u;
      }
  }

  KeyList list;
  list.build(a, r, i, reinterpret_cast<int*>(masks + STAGES));
  const int tiles = (list.total + kTile - 1) / kTile;
  const int per = (tiles + nsplit - 1) / nsplit;
  const int t_end = min(tiles, (split + 1) * per);
  const int t_beg = min(split * per, t_end);
  const int32_t* order = a.order + static_cast<int64_t>(r) * a.N;
  const T* kb = static_cast<const T*>(a.k) + b * a.ks.b + hk * a.ks.h;
  const T* vb = static_cast<const T*>(a.v) + b * a.vs.b + hk * a.vs.h;
  const int dchunks = a.D / 8;

  // keys of the next 32 places (two tiles), fetched one round ahead of their copies
  int cur = 0;
  int idx = -1, idx_next = list.key(a, order, t_beg * kTile + lane, cur);
  auto issue = [&](int t) {  // tiles are issued in order from t_beg
    const int half = (t - t_beg) & 1;
    if (half == 0) {
      idx = KeyList::visible(a, idx_next, pos);
      idx_next = list.key(a, order, (t + 2) * kTile + lane, cur);
    }
    const int stage = (t - t_beg) % STAGES;
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
  float m[NT][2], l[NT][2];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
#pragma unroll
    for (int e = 0; e < 2; ++e) m[n][e] = -INFINITY, l[n][e] = 0.f;
#pragma unroll
    for (int kk = 0; kk < KS; ++kk)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[n][kk][e] = 0.f;
  }
#pragma unroll
  for (int s = 0; s < STAGES - 1; ++s) {
    if (t_beg + s < t_end) issue(t_beg + s);
    mma::cp_async_commit();
  }
  const float sc = a.scale * kLog2e;
  for (int t = t_beg; t < t_end; ++t) {
    mma::cp_async_wait<STAGES - 2>();
    __syncwarp();  // the tile's copies of all lanes, and all reads of the stage refilled next
    if (t + STAGES - 1 < t_end) issue(t + STAGES - 1);
    mma::cp_async_commit();
    const int stage = (t - t_beg) % STAGES;
    const uint32_t live = masks[stage];
    if (live == 0) continue;
    const uint32_t kt = ring + stage * (2 * kTile * DP * 2), vt = kt + kTile * DP * 2;
    float s[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[n][e] = 0.f;
#pragma unroll
    for (int kk = 0; kk < KS; ++kk) {
      uint32_t f[4];
      load_a<DP>(f, kt, 0, kk);
#pragma unroll
      for (int n = 0; n < NT; ++n) mma::m16n8k16<T>(s[n], f, qf[n][kk][0], qf[n][kk][1]);
    }
    const bool on0 = live >> g & 1, on1 = live >> (g + 8) & 1;
    uint32_t pf[NT][2], pl[NT][2];  // P and what its rounding left
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        s[n][e] = on0 ? s[n][e] * sc : -INFINITY;
        s[n][2 + e] = on1 ? s[n][2 + e] * sc : -INFINITY;
        float top = fmaxf(s[n][e], s[n][2 + e]);
        top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 4));
        top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 8));
        top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 16));
        const float mn = fmaxf(m[n][e], top);
        const float base = mn == -INFINITY ? 0.f : mn;  // nothing finite so far
        const float alpha = exp2f(m[n][e] - base);
        m[n][e] = mn;
        s[n][e] = exp2f(s[n][e] - (base - Range<T>::kShift));
        s[n][2 + e] = exp2f(s[n][2 + e] - (base - Range<T>::kShift));
        l[n][e] = l[n][e] * alpha + (s[n][e] + s[n][2 + e]);
#pragma unroll
        for (int kk = 0; kk < KS; ++kk) o[n][kk][e] *= alpha, o[n][kk][2 + e] *= alpha;
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        uint32_t hi, lo;
        mma::split2_weights<T>(s[n][2 * e], s[n][2 * e + 1], hi, lo);
        pf[n][e] = mma::movmatrix_trans(hi);
        pl[n][e] = mma::movmatrix_trans(lo);
      }
    }
#pragma unroll
    for (int md = 0; md < KS; ++md) {
      uint32_t f[4];
      load_a_trans<DP>(f, vt, 0, md);
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        mma::m16n8k16<T>(o[n][md], f, pf[n][0], pf[n][1]);
        mma::m16n8k16<T>(o[n][md], f, pl[n][0], pl[n][1]);
      }
    }
  }
  mma::cp_async_wait<0>();

#pragma unroll
  for (int n = 0; n < NT; ++n) {
    float inv[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float sum = l[n][e];
      sum += __shfl_xor_sync(0xFFFFFFFFu, sum, 4);
      sum += __shfl_xor_sync(0xFFFFFFFFu, sum, 8);
      sum += __shfl_xor_sync(0xFFFFFFFFu, sum, 16);
      inv[e] = sum == 0.f ? 0.f : 1.f / sum;
      const float ls = sum == 0.f ? -INFINITY : (m[n][e] - Range<T>::kShift + log2f(sum)) * kLn2;
      const int h = n * 8 + t4 * 2 + e;
      if (g == 0 && h < heads) {
        const int64_t at = (static_cast<int64_t>(b) * a.Hq + h0 + h) * a.Nq + i;
        if (nsplit == 1)
          lse[at] = ls;
        else
          part_lse[at * nsplit + split] = ls;
      }
    }
#pragma unroll
    for (int md = 0; md < KS; ++md) {
      if (nsplit > 1) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int h = n * 8 + t4 * 2 + (e & 1), d = md * 16 + g + (e >> 1) * 8;
          const int64_t at = (static_cast<int64_t>(b) * a.Hq + h0 + h) * a.Nq + i;
          if (h < heads && d < a.D)
            part_o[(at * nsplit + split) * a.D + d] = o[n][md][e] * inv[e & 1];
        }
      } else {
        // to (head g, elements 2 t4, 2 t4 + 1)
        const uint32_t lo =
            mma::movmatrix_trans(mma::pack2<T>(o[n][md][0] * inv[0], o[n][md][1] * inv[1]));
        const uint32_t hi =
            mma::movmatrix_trans(mma::pack2<T>(o[n][md][2] * inv[0], o[n][md][3] * inv[1]));
        const int h = n * 8 + g, d = md * 16 + t4 * 2;
        if (h < heads) {
          T* row = out + ((static_cast<int64_t>(b) * a.Hq + h0 + h) * a.Nq + i) * a.D;
          if (d < a.D) *reinterpret_cast<uint32_t*>(row + d) = lo;
          if (d + 8 < a.D) *reinterpret_cast<uint32_t*>(row + d + 8) = hi;
        }
      }
    }
  }
}

// out = sum_s w_s part_s / sum_s w_s, w_s = exp(lse_s - max): one warp per (b, h, i).
template <typename T>
__global__ void __launch_bounds__(128) attn_join_kernel(const float* __restrict__ part_o,
                                                        const float* __restrict__ part_lse,
                                                        T* __restrict__ out,
                                                        float* __restrict__ lse, int nsplit, int D,
                                                        int64_t rows) {
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 5);
  if (row >= rows) return;
  // lane l takes columns 4 l ..; of up to 64 parts, it holds the weights of l and l + 32
  const float* po = part_o + row * nsplit * D + lane * 4;
  const bool on = lane * 4 < D;
  float w[2];
#pragma unroll
  for (int x = 0; x < 2; ++x)
    w[x] = x * 32 + lane < nsplit ? part_lse[row * nsplit + x * 32 + lane] : -INFINITY;
  float4 v[8];
  auto fetch = [&](int s0) {
#pragma unroll
    for (int u = 0; u < 8; ++u)
      v[u] = on && s0 + u < nsplit ? *reinterpret_cast<const float4*>(po + static_cast<int64_t>(s0 + u) * D)
                                   : make_float4(0.f, 0.f, 0.f, 0.f);
  };
  fetch(0);  // on its way with the weights
  float top = fmaxf(w[0], w[1]);
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
  const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
  for (int x = 0; x < 2; ++x) w[x] = exp2f((w[x] - base) * kLog2e);
  float acc[4] = {0.f, 0.f, 0.f, 0.f}, sum = 0.f;
  for (int s0 = 0; s0 < nsplit; s0 += 8) {
    if (s0 > 0) fetch(s0);
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int s = s0 + u;  // weights behind the last part are 0
      const float f = __shfl_sync(0xFFFFFFFFu, s < 32 ? w[0] : w[1], s & 31);
      sum += f;
      acc[0] += f * v[u].x, acc[1] += f * v[u].y, acc[2] += f * v[u].z, acc[3] += f * v[u].w;
    }
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  if (on)
    *reinterpret_cast<uint2*>(out + row * D + lane * 4) =
        make_uint2(mma::pack2<T>(acc[0] * inv, acc[1] * inv), mma::pack2<T>(acc[2] * inv, acc[3] * inv));
  if (lane == 0) lse[row] = sum == 0.f ? -INFINITY : base + log2f(sum) * kLn2;
}

template <typename T, int DP, int NT>
int fwd_typed(const Args& a, void* out, float* lse, float* ws, cudaStream_t stream) {
  constexpr int STAGES = 3;
  const int chunks = (a.G + 8 * NT - 1) / (8 * NT);
  const int nsplit = split_count(a);
  const int64_t rows = static_cast<int64_t>(a.batch) * a.Hq * a.Nq;
  const int64_t units = static_cast<int64_t>(a.batch) * a.Hkv * a.Nq * chunks * nsplit;
  const int smem = kWarps * warp_smem<DP, STAGES>(a.top);
  auto kern = attn_fwd_kernel<T, DP, NT, STAGES>;
  FKC_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  float* part_lse = nsplit > 1 ? ws : nullptr;
  float* part_o = nsplit > 1 ? ws + align_up(static_cast<size_t>(rows * nsplit), 64) : nullptr;
  FKC_TRY(launch_pdl(kern, dim3(static_cast<unsigned>((units + kWarps - 1) / kWarps)),
                     dim3(32 * kWarps), smem, stream, a, static_cast<T*>(out), lse, part_o, part_lse,
                     chunks, nsplit, units));
  if (nsplit == 1) return FKC_OK;
  return launch_pdl(attn_join_kernel<T>, dim3(static_cast<unsigned>((rows + 3) / 4)), dim3(128), 0,
                    stream, static_cast<const float*>(part_o), static_cast<const float*>(part_lse),
                    static_cast<T*>(out), lse, nsplit, a.D, rows);
}

template <typename T>
int fwd_dtype(const Args& a, void* out, float* lse, float* ws, cudaStream_t stream) {
  if (a.D <= 64)
    return a.G <= 8 ? fwd_typed<T, 64, 1>(a, out, lse, ws, stream)
                    : fwd_typed<T, 64, 2>(a, out, lse, ws, stream);
  return a.G <= 8 ? fwd_typed<T, 128, 1>(a, out, lse, ws, stream)
                  : fwd_typed<T, 128, 2>(a, out, lse, ws, stream);
}

}  // namespace

// Warps per query row: the keys of one are split while there are fewer warps than
// the GPU holds at once (148 SMs x 8; one more would start a second wave), a part taking
// at least 4 tiles of the average selection (top * N / K keys).
int split_count(const Args& a) {
  const int64_t chunks = (a.G + 15) / 16;
  const int64_t rows = static_cast<int64_t>(a.batch) * a.Hkv * a.Nq * chunks;
  const int64_t keys = std::min<int64_t>(static_cast<int64_t>(a.top) * ((a.N + a.K - 1) / a.K), a.N);
  const int64_t most = std::max<int64_t>(1, keys / (4 * kTile));
  return static_cast<int>(std::min<int64_t>({most, std::max<int64_t>(1, 148 * 8 / rows), 64}));
}

size_t forward_workspace_bytes(const Args& a) {
  if (use_tiles(a)) return tiles_forward_workspace_bytes(a);
  const int nsplit = split_count(a);
  if (nsplit == 1) return 0;
  const int64_t rows = static_cast<int64_t>(a.batch) * a.Hq * a.Nq;
  return (align_up(static_cast<size_t>(rows * nsplit), 64) + static_cast<size_t>(rows * nsplit) * a.D) * 4;
}

int launch_forward(const Args& a, int dtype, void* out, float* lse, void* ws,
                   cudaStream_t stream) {
  if (use_tiles(a)) return launch_tiles_forward(a, dtype, out, lse, ws, stream);
  return dtype == FKC_DTYPE_F16
             ? fwd_dtype<__half>(a, out, lse, static_cast<float*>(ws), stream)
             : fwd_dtype<__nv_bfloat16>(a, out, lse, static_cast<float*>(ws), stream);
}

}  // namespace attn
}  // namespace fkc
