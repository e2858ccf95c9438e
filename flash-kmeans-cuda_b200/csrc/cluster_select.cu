// Selection of clusters for a query by a cheap score:
//
//   score[r, i, c] = scale * max over the heads h of the group of q[b, h, i] . centroid[r, c]
//                    + bias[r, c]
//
// Clusters without positions, and (with q_pos) those whose first position lies
// behind the query, cannot be selected, nor can one whose score is NaN or -inf. The
// top best of the rest, ties to the lowest index, are written in ascending order; -1
// fills what is left.
//
//   score  (score_kernel)  128 clusters x 16 or 64 queries per CTA; the heads are
//          walked one by one and the running maximum stays in the accumulator layout,
//          so any group size fills the instruction (m16n8k16, fp32 accumulation). Also
//          the largest norms of a query's heads and of a tile's centroids.
//   choose (choose_warp_kernel, one warp per query up to 1024 clusters, and for few queries or
//          more clusters choose_cta_kernel)  the top-th largest fp32 score t by bisection over its
//          bits. What lies above t by more than the scores can be off is in, what lies
//          below by more is out; where that leaves more candidates than places, theirs
//          are computed again in 64 bits and ranked. So the selection is that of exact
//          arithmetic, whatever order the products were added in.
//
// How far an fp32 score can be off: a product of two 16-bit values is exact in fp32;
// adding D of them with truncation to 2^-22 of the largest magnitude so far, none of
// which exceeds |q||c|, is off by at most D * 2^-22 |q||c|; the two roundings of scale
// and the rounding of the sum with bias add 2^-22 (scale |q||c| + |score|) at most. Squares and
// products that underflow are covered by the least norm that counts, 2^-50: its square is more than
// 128 squares below 2^-126 can lose, and D * 2^-22 of two such norms more than D products can.
//
// The scores go through L2, in rounds of 64 MB at most. 4096 queries x 256
// clusters x 8 rows of 4 heads, D = 128: 8.6 GFLOP and 34 MB of scores, score 58 us (three CTAs an SM; it was 70 with
// two and with norms read again from shared memory by half of the warps), choose 43 us
// (two thirds of the issue slots, some 890 instructions a query: bisection 6 to 8 steps, a border of
// 64-bit scores for 6% of them; 59 us with bisection bit by bit and one query a warp, 53 us
// with as many CTAs as the SMs hold, which the queries with a border leave at different times).
// 128 queries of 1024 clusters, 4 heads: 32 us in all, most of it latency (51 us before the heads
// shared a tile, thresholds started from the scores' common leading bits and borders went
// four at a time).
#include <algorithm>
#include <cmath>

#include "cluster_attention.cuh"
#include "fkc_common.cuh"

namespace fkc {
namespace attn {
namespace {

constexpr int kClusters = 128;  // clusters per tile
constexpr uint32_t kNever = 0xFFC0DEADu;  // score bits of a cluster that cannot be selected

struct SelectArgs {
  const void *q, *centroids;
  Strides qs;
  const int32_t* offsets;
  const int32_t* order;  // with q_pos
  const int32_t* q_pos;
  const float* bias;  // (R, K) or null
  int32_t* sel;
  int Hkv, G, Nq, N, K, top, D;
  int r0, all;  // the round's first row of clusters; queries of the call, of which a round takes Nq from q on
  double scale;
  double unsure;  // how far a score can be off, of |q||c|
};

constexpr float kLeastNorm2 = 0x1p-100f;  // squares of smaller values underflow (see the top)

__device__ __forceinline__ float fold_max(float a, float b) {
  return (isnan(a) || isnan(b)) ? INFINITY : fmaxf(a, b);  // a NaN norm counts as unbounded
}

// QW warps along the queries, 4 / QW along the clusters. PACK (QW = 1): at most 16 rows (query,
// head) in all, side by side in one tile; the maximum over a query's heads is taken in
// shared memory.
template <typename T, int DP, int QW, bool PACK>
__global__ void __launch_bounds__(128, 3) score_kernel(SelectArgs a, float* __restrict__ scores,
                                                    float* __restrict__ q_norm,
                                                    float* __restrict__ c_norm, int ctiles,
                                                    int qtiles) {
  constexpr int CW = 4 / QW, KS = DP / 16, CH = DP / 8;
  constexpr int NW = kClusters / CW / 8;  // 8-cluster groups per warp
  constexpr int MQ = 16 * QW;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ __align__(8) float s_bias[kClusters];
  __shared__ __align__(8) int s_first[kClusters];  // first position; INT_MAX: never selected
  __shared__ float s_red[4];
  __shared__ float s_pack[PACK ? 16 * (kClusters + 4) : 1];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int g = lane >> 2, t4 = lane & 3;
  const uint32_t ct = static_cast<uint32_t>(__cvta_generic_to_shared(smem));
  const uint32_t qt0 = ct + kClusters * DP * 2;
  pdl_wait();
  const int tile = blockIdx.x % ctiles, rest = blockIdx.x / ctiles;
  const int qtile = rest % qtiles, lr = rest / qtiles, r = a.r0 + lr;  // lr: the scratch's row
  const int b = r / a.Hkv, hk = r - b * a.Hkv;
  const int c0 = tile * kClusters, i0 = qtile * MQ;
  const T* cen = static_cast<const T*>(a.centroids) + (static_cast<int64_t>(r) * a.K + c0) * a.D;
  const T* q = static_cast<const T*>(a.q) + b * a.qs.b + static_cast<int64_t>(hk) * a.G * a.qs.h;
  const int dchunks = a.D / 8;
  for (int e = tid; e < kClusters * CH; e += 128) {
    const int row = e / CH, c = e % CH;
    const bool ok = c0 + row < a.K && c < dchunks;
    mma::cp_async16(ct + tile_at<DP>(row, c), cen + (ok ? static_cast<int64_t>(row) * a.D + c * 8 : 0),
                    ok);
  }
  auto load_q = [&](int h, int buf) {
    const uint32_t qt = qt0 + buf * (MQ * DP * 2);
    for (int e = tid; e < MQ * CH; e += 128) {
      const int row = e / CH, c = e % CH;
      const int i = PACK ? row / a.G : i0 + row, hh = PACK ? row - i * a.G : h;
      const bool ok = i < a.Nq && c < dchunks;
      mma::cp_async16(qt + tile_at<DP>(row, c), q + (ok ? hh * a.qs.h + i * a.qs.n + c * 8 : 0), ok);
    }
  };
  load_q(0, 0);
  mma::cp_async_commit();
  {
    const int c = c0 + tid;
    int first = INT_MAX;
    float bias = 0.f;
    if (c < a.K) {
      const int32_t* of = a.offsets + static_cast<int64_t>(r) * (a.K + 1) + c;
      const int s = of[0], e = of[1];
      if (e > s && s >= 0 && s < a.N)
        first = a.q_pos != nullptr ? a.order[static_cast<int64_t>(r) * a.N + s] : 0;
      if (first < 0) first = INT_MAX;
      if (a.bias != nullptr) bias = a.bias[static_cast<int64_t>(r) * a.K + c];
      if (isnan(bias) || bias == -INFINITY) first = INT_MAX;
    }
    s_first[tid] = first;
    s_bias[tid] = bias;
  }
  const int wq = warp % QW, wc = warp / QW;
  float best[NW][4];
#pragma unroll
  for (int n = 0; n < NW; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) best[n][e] = -INFINITY;
  float qn[2] = {0.f, 0.f};  // largest norm^2 of the heads: the warp's rows g and g + 8
  const bool norms = tile == 0 && wc == 0;
  const int passes = PACK ? 1 : a.G;
#pragma unroll 1
  for (int h = 0; h < passes; ++h) {
    mma::cp_async_wait<0>();
    __syncthreads();
    if (h + 1 < passes) load_q(h + 1, (h + 1) & 1);
    mma::cp_async_commit();
    const uint32_t qt = qt0 + (h & 1) * (MQ * DP * 2);
    float acc[NW][4], sq[2] = {0.f, 0.f};
#pragma unroll
    for (int n = 0; n < NW; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[n][e] = 0.f;
#pragma unroll
    for (int kk = 0; kk < KS; ++kk) {
      uint32_t fa[4];
      load_a<DP>(fa, qt, wq * 16, kk);
      if (norms) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 f = mma::unpack2<T>(fa[e]);
          sq[e & 1] = fmaf(f.x, f.x, fmaf(f.y, f.y, sq[e & 1]));
        }
      }
#pragma unroll
      for (int n = 0; n < NW; n += 2) {
        uint32_t fb[4];
        load_b<DP>(fb, ct, (wc * NW + n) * 8, kk);
        mma::m16n8k16<T>(acc[n], fa, fb[0], fb[1]);
        mma::m16n8k16<T>(acc[n + 1], fa, fb[2], fb[3]);
      }
    }
#pragma unroll
    for (int n = 0; n < NW; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) best[n][e] = fmaxf(best[n][e], acc[n][e]);
    if (norms) {
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        sq[x] += __shfl_xor_sync(0xFFFFFFFFu, sq[x], 1);
        sq[x] += __shfl_xor_sync(0xFFFFFFFFu, sq[x], 2);
        qn[x] = fold_max(qn[x], sq[x]);
      }
    }
  }
  if (!PACK && norms && t4 < 2) {
    const int i = i0 + wq * 16 + t4 * 8 + g;
    if (i < a.Nq) q_norm[static_cast<int64_t>(lr) * a.Nq + i] = sqrtf(fmaxf(t4 == 0 ? qn[0] : qn[1], kLeastNorm2));
  }
  if constexpr (PACK) {
    __syncthreads();
    if (norms && t4 < 2) s_pack[t4 * 8 + g] = t4 == 0 ? qn[0] : qn[1];
    __syncthreads();
    if (tile == 0 && tid < a.Nq) {
      float m = 0.f;
      for (int h = 0; h < a.G; ++h) m = fold_max(m, s_pack[tid * a.G + h]);
      q_norm[static_cast<int64_t>(lr) * a.Nq + tid] = sqrtf(fmaxf(m, kLeastNorm2));
    }
    __syncthreads();
#pragma unroll
    for (int n = 0; n < NW; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        s_pack[(g + (e >> 1) * 8) * (kClusters + 4) + (wc * NW + n) * 8 + t4 * 2 + (e & 1)] = best[n][e];
    __syncthreads();
  }
  if (qtile == 0) {  // the tile's largest centroid norm, of the clusters that can be selected
    float s = 0.f;
    for (int c = 0; c < CH; ++c) {
      const uint4 u = *reinterpret_cast<const uint4*>(smem + tile_at<DP>(tid, c));
      const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float2 f = mma::unpack2<T>(w[k]);
        s += f.x * f.x + f.y * f.y;
      }
    }
    if (s_first[tid] == INT_MAX) s = 0.f;
    s = fold_max(s, 0.f);
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) s = fmaxf(s, __shfl_xor_sync(0xFFFFFFFFu, s, o));
    if (lane == 0) s_red[warp] = s;
    __syncthreads();
    if (tid == 0)
      c_norm[static_cast<int64_t>(lr) * ctiles + tile] =
          sqrtf(fmaxf(fmaxf(fmaxf(s_red[0], s_red[1]), fmaxf(s_red[2], s_red[3])), kLeastNorm2));
  }
  const float scale = static_cast<float>(a.scale);
  if constexpr (PACK) {
    for (int i = 0; i < a.Nq && c0 + tid < a.K; ++i) {
      const int pos =
          a.q_pos != nullptr ? min(a.q_pos[static_cast<int64_t>(b) * a.all + i], a.N) : a.N;
      float m = -INFINITY;
      for (int h = 0; h < a.G; ++h) m = fmaxf(m, s_pack[(i * a.G + h) * (kClusters + 4) + tid]);
      scores[(static_cast<int64_t>(lr) * a.Nq + i) * a.K + c0 + tid] =
          s_first[tid] > pos ? __uint_as_float(kNever) : m * scale + s_bias[tid];
    }
  } else {
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const int i = i0 + wq * 16 + half * 8 + g;
    if (i >= a.Nq) continue;
    const int pos =
        a.q_pos != nullptr ? min(a.q_pos[static_cast<int64_t>(b) * a.all + i], a.N) : a.N;
    float* row = scores + (static_cast<int64_t>(lr) * a.Nq + i) * a.K + c0;
#pragma unroll
    for (int n = 0; n < NW; ++n) {
      const int cl = (wc * NW + n) * 8 + t4 * 2;
      const float2 bias = *reinterpret_cast<const float2*>(s_bias + cl);
      const int2 first = *reinterpret_cast<const int2*>(s_first + cl);
      const float x = first.x > pos ? __uint_as_float(kNever) : best[n][half * 2] * scale + bias.x;
      const float y = first.y > pos ? __uint_as_float(kNever) : best[n][half * 2 + 1] * scale + bias.y;
      if (c0 + cl + 1 < a.K && a.K % 2 == 0) {
        *reinterpret_cast<float2*>(row + cl) = make_float2(x, y);
      } else {
        if (c0 + cl < a.K) row[cl] = x;
        if (c0 + cl + 1 < a.K) row[cl + 1] = y;
      }
    }
  }
  }
}

// fp32 scores as integers that compare the same way; 0: cannot be selected.
__device__ __forceinline__ uint32_t sort_key(float s) {
  const uint32_t u = __float_as_uint(s);
  if (u == kNever) return 0u;
  if (isnan(s)) return 1u;  // undecided: only 64 bits can tell
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float key_score(uint32_t k) {
  return __uint_as_float((k & 0x80000000u) ? (k & 0x7FFFFFFFu) : ~k);
}

// The score of cluster c for query i in 64 bits, by eight lanes (the same in each); c < 0: none.
template <typename T>
__device__ double exact_score(const SelectArgs& a, int r, int i, int c) {
  const int l8 = threadIdx.x & 7;
  const int b = r / a.Hkv, hk = r - b * a.Hkv;
  const T* cen = static_cast<const T*>(a.centroids) +
                 (static_cast<int64_t>(r) * a.K + (c < 0 ? 0 : c)) * a.D;
  const T* q = static_cast<const T*>(a.q) + b * a.qs.b + static_cast<int64_t>(hk) * a.G * a.qs.h +
               i * a.qs.n;
  double best = -INFINITY;
  bool nan = false;
  for (int h = 0; h < a.G; ++h) {
    double s = 0.0;
    for (int d = l8 * 8; d < a.D; d += 64) {
      const uint4 x = *reinterpret_cast<const uint4*>(q + h * a.qs.h + d);
      const uint4 y = *reinterpret_cast<const uint4*>(cen + d);
      const uint32_t u[4] = {x.x, x.y, x.z, x.w}, v[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float2 f = mma::unpack2<T>(u[k]), g = mma::unpack2<T>(v[k]);
        s += static_cast<double>(f.x) * static_cast<double>(g.x);
        s += static_cast<double>(f.y) * static_cast<double>(g.y);
      }
    }
#pragma unroll
    for (int o = 4; o >= 1; o >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, o);
    nan |= isnan(s);
    best = fmax(best, s);
  }
  double s = best * a.scale;
  if (a.bias != nullptr && c >= 0) s += static_cast<double>(a.bias[static_cast<int64_t>(r) * a.K + c]);
  return nan || isnan(s) || c < 0 ? -INFINITY : s;
}

// The band around the top-th score t in which fp32 cannot tell; infinite where a
// norm or the score is not finite.
__device__ __forceinline__ float band_of(const SelectArgs& a, float t, float qn, float cn) {
  const float eps = static_cast<float>(a.unsure * qn * cn) + fabsf(t) * 0x1p-22f;
  return eps < INFINITY ? 2.f * (eps + 0x1p-126f) : INFINITY;  // the least: scores that underflow
}

__device__ __forceinline__ float largest_norm(const float* c_norm, int64_t r, int ctiles) {
  float m = 0.f;
  for (int i = threadIdx.x & 31; i < ctiles; i += 32) m = fmaxf(m, c_norm[r * ctiles + i]);
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
  return m;
}

// One warp per query at a time, whose next query's scores are on their way meanwhile; KPL scores a
// lane, cluster j * 32 + lane.
template <typename T, int KPL>
__global__ void __launch_bounds__(128, KPL <= 8 ? 10 : 4) choose_warp_kernel(
    SelectArgs a, const float* __restrict__ scores, const float* __restrict__ q_norm,
    const float* __restrict__ c_norm, int ctiles, int64_t queries) {
  __shared__ double s_exact[4][KPL * 32];
  __shared__ uint16_t s_list[4][KPL * 32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t below = (1u << lane) - 1u;
  pdl_wait();
  const int64_t step = static_cast<int64_t>(gridDim.x) * 4;
  float ahead[KPL];
  auto fetch = [&](int64_t qi) {
#pragma unroll
    for (int j = 0; j < KPL; ++j)
      ahead[j] = j * 32 + lane < a.K ? scores[qi * a.K + j * 32 + lane] : __uint_as_float(kNever);
  };
  int64_t qi = static_cast<int64_t>(blockIdx.x) * 4 + warp;
  if (qi < queries) fetch(qi);
  for (; qi < queries; qi += step) {
    // (a 64-bit division costs as much as four bisections)
    const int r = queries <= 0xFFFFFFFFll
                      ? static_cast<int>(static_cast<uint32_t>(qi) / static_cast<uint32_t>(a.Nq))
                      : static_cast<int>(qi / a.Nq);
    const int i = static_cast<int>(qi - static_cast<int64_t>(r) * a.Nq);
    const float qn = q_norm[qi];
    uint32_t key[KPL];
    int have = 0;
#pragma unroll
    for (int j = 0; j < KPL; ++j) {
      key[j] = sort_key(ahead[j]);
      have += key[j] != 0u;
    }
    if (qi + step < queries) fetch(qi + step);
    have = __reduce_add_sync(0xFFFFFFFFu, have);
    // t: the want-th largest key, by bisection between a key that at least `want` reach and one past
    // the largest; where a count meets it, the smallest key counted
    const int want = min(a.top, have);
    uint32_t t = 0;
    if (have > 0) {
      uint32_t low = 0xFFFFFFFFu, high = 0;
#pragma unroll
      for (int j = 0; j < KPL; ++j) low = min(low, key[j] - 1u), high = max(high, key[j]);
      // of up to 32 places: each lane's largest key is one of `want` at least
      const uint32_t tops = __reduce_min_sync(0xFFFFFFFFu, high);
      low = __reduce_min_sync(0xFFFFFFFFu, low) + 1u;  // keys of 0 were the largest there
      high = __reduce_max_sync(0xFFFFFFFFu, high) + 1u;  // no key is the largest integer
      t = want < have && want <= 32 && tops != 0u ? tops : low;
      while (want < have && high - t > 1u) {
        // scores on both sides of zero first part there: the keys between are many
        const uint32_t cand = t < 0x80000000u && high > 0x80000000u ? 0x80000000u : t + (high - t) / 2;
        int n = 0;
#pragma unroll
        for (int j = 0; j < KPL; ++j) n += key[j] >= cand;
        n = __reduce_add_sync(0xFFFFFFFFu, n);
        if (n < want) {
          high = cand;
          continue;
        }
        t = cand;
        if (n == want) {
          uint32_t least = 0xFFFFFFFFu;
#pragma unroll
          for (int j = 0; j < KPL; ++j)
            if (key[j] >= cand) least = min(least, key[j]);
          t = __reduce_min_sync(0xFFFFFFFFu, least);
          break;
        }
      }
    }
    const float cn = largest_norm(c_norm, r, ctiles);
    const float ts = key_score(t);
    const float band = t <= 1u ? INFINITY : band_of(a, ts, qn, cn);
    const bool open = !(band < INFINITY) || isinf(ts);  // fp32 says nothing: all in 64 bits
    // in: above the band; undecided: inside (a step wider, for the two zeros' sake)
    const uint32_t over = open ? 0xFFFFFFFFu : sort_key(ts + band) + 1u;
    uint32_t from = open ? 1u : max(sort_key(ts - band), 2u) - 1u;
    int sure = 0, undecided = 0;
#pragma unroll
    for (int j = 0; j < KPL; ++j) {
      sure += key[j] > over;
      undecided += key[j] >= from;
    }
    sure = __reduce_add_sync(0xFFFFFFFFu, sure);
    undecided = __reduce_add_sync(0xFFFFFFFFu, undecided) - sure;
    const int places = want - sure;
    if ((undecided != places || open) && undecided > 0) {
      double* ex = s_exact[warp];
      uint16_t* list = s_list[warp];
      uint32_t mid = 0;
      int listed = 0;
      __syncwarp();  // the last such query's reads
#pragma unroll
      for (int j = 0; j < KPL; ++j) {
        const bool on = key[j] >= from && key[j] <= over;
        const uint32_t who = __ballot_sync(0xFFFFFFFFu, on);
        if (on) mid |= 1u << j, list[listed + __popc(who & below)] = static_cast<uint16_t>(j * 32 + lane);
        listed += __popc(who);
      }
      __syncwarp();
      for (int k = 0; k < listed; k += 4) {  // four at a time, eight lanes each
        const int at = k + (lane >> 3);
        const int c = at < listed ? list[at] : -1;
        const double s = exact_score<T>(a, a.r0 + r, i, c);
        if (c >= 0 && (lane & 7) == 0) ex[c] = s;
      }
      __syncwarp();
      // the places best of them, largest score, then lowest index, get the largest keys
      uint32_t in = 0;
      for (int n = 0; n < places; ++n) {
        double best = -INFINITY;
        int at = INT_MAX;
#pragma unroll 1
        for (int j = 0; j < KPL; ++j)
          if (mid >> j & 1u) {
            const double s = ex[j * 32 + lane];
            if (s > best) best = s, at = j * 32 + lane;
          }
#pragma unroll
        for (int o = 16; o >= 1; o >>= 1) {
          const double s = __shfl_xor_sync(0xFFFFFFFFu, best, o);
          const int x = __shfl_xor_sync(0xFFFFFFFFu, at, o);
          if (s > best || (s == best && x < at)) best = s, at = x;
        }
        if (at == INT_MAX) break;  // nothing above -inf is left
        if ((at & 31) == lane) {
          mid &= ~(1u << (at >> 5));
          in |= 1u << (at >> 5);
        }
      }
#pragma unroll
      for (int j = 0; j < KPL; ++j)
        if (in >> j & 1u) key[j] = 0xFFFFFFFFu;
      from = over == 0xFFFFFFFFu ? over : over + 1u;
    }
    int32_t* out = a.sel + (static_cast<int64_t>(a.r0 + r) * a.all + i) * a.top;
    int done = 0;
#pragma unroll
    for (int j = 0; j < KPL; ++j) {
      const bool on = key[j] >= from;
      const uint32_t who = __ballot_sync(0xFFFFFFFFu, on);
      const int at = done + __popc(who & below);
      if (on && at < a.top) out[at] = j * 32 + lane;
      done += __popc(who);
    }
    for (int j = done + lane; j < a.top; j += 32) out[j] = -1;
  }
}

constexpr int kCtaThreads = 512;

// Sum over the CTA (every thread gets it). red: two rows used in turn, so that one barrier is
// enough.
struct CtaSum {
  int (*red)[kCtaThreads / 32];
  int turn = 0;
  __device__ __forceinline__ int operator()(int v) {
    v = __reduce_add_sync(0xFFFFFFFFu, v);
    int* r = red[turn];
    turn ^= 1;
    if ((threadIdx.x & 31) == 0) r[threadIdx.x >> 5] = v;
    __syncthreads();
    int s = 0;
#pragma unroll
    for (int w = 0; w < kCtaThreads / 32; ++w) s += r[w];
    return s;
  }
};
__device__ __forceinline__ uint32_t cta_max(uint32_t v, uint32_t* red) {
  v = __reduce_max_sync(0xFFFFFFFFu, v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  uint32_t m = 0;
#pragma unroll
  for (int w = 0; w < kCtaThreads / 32; ++w) m = max(m, red[w]);
  return m;
}

// One CTA per query, for few queries or many clusters, up to 16384: keys, states and 64-bit scores in shared memory.
template <typename T>
__global__ void __launch_bounds__(kCtaThreads) choose_cta_kernel(
    SelectArgs a, const float* __restrict__ scores, const float* __restrict__ q_norm,
    const float* __restrict__ c_norm, int ctiles) {
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ int sums[2][kCtaThreads / 32], red[kCtaThreads / 32];
  __shared__ uint32_t maxima[kCtaThreads / 32];
  __shared__ double s_best[kCtaThreads / 32];
  __shared__ int s_at[kCtaThreads / 32];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  double* ex = reinterpret_cast<double*>(smem);
  uint32_t* key = reinterpret_cast<uint32_t*>(smem + static_cast<size_t>(a.K) * 8);
  uint8_t* state = smem + static_cast<size_t>(a.K) * 12;  // 0 out, 1 in, 2 undecided
  pdl_wait();
  const int64_t qi = blockIdx.x;
  const int r = static_cast<int>(qi / a.Nq), i = static_cast<int>(qi % a.Nq);
  const float* row = scores + qi * a.K;
  CtaSum cta_sum{sums};
  int have = 0;
  uint32_t low = 0, high = 0;  // low: the complement of the smallest
  for (int c = tid; c < a.K; c += kCtaThreads) {
    const uint32_t k = sort_key(row[c]);
    key[c] = k;
    if (k == 0u) continue;
    ++have;
    low = max(low, ~k), high = max(high, k);
  }
  have = cta_sum(have);
  low = ~cta_max(low, maxima);
  high = cta_max(high, maxima);
  const int want = min(a.top, have);
  uint32_t t = 0;  // as in choose_warp_kernel
  if (have > 0) {
    const int open_bits = 32 - __clz(low ^ high);
    t = want == have ? low : open_bits == 32 ? 0u : high >> open_bits << open_bits;
    for (int bit = want == have ? -1 : open_bits - 1; bit >= 0; --bit) {
      const uint32_t cand = t | (1u << bit);
      int n = 0;
      for (int c = tid; c < a.K; c += kCtaThreads) n += key[c] >= cand;
      n = cta_sum(n);
      if (n >= want) t = cand;
      if (n == want) {
        uint32_t least = 0;
        for (int c = tid; c < a.K; c += kCtaThreads)
          if (key[c] >= cand) least = max(least, ~key[c]);
        t = ~cta_max(least, maxima);
        break;
      }
    }
  }
  const float cn = largest_norm(c_norm, r, ctiles);
  const float ts = key_score(t);
  const float band = t <= 1u ? INFINITY : band_of(a, ts, q_norm[qi], cn);
  const bool open = !(band < INFINITY) || isinf(ts);
  int sure = 0, undecided = 0;
  for (int c = tid; c < a.K; c += kCtaThreads) {
    uint8_t st = 0;
    if (key[c] != 0u) {
      const float s = key_score(key[c]);
      if (!open && s > ts + band)
        st = 1, ++sure;
      else if (open || s >= ts - band)
        st = 2, ++undecided;
    }
    state[c] = st;
  }
  sure = cta_sum(sure);
  undecided = cta_sum(undecided);
  const int places = want - sure;
  const bool all = undecided == places && !open;
  if (!all && undecided > 0) {
    __syncthreads();
    for (int c0 = warp * 4; c0 < a.K; c0 += kCtaThreads / 8) {  // four at a time, eight lanes each
      const int c = c0 + (lane >> 3);
      const bool mine = c < a.K && state[c] == 2;
      if (!__any_sync(0xFFFFFFFFu, mine)) continue;
      const double s = exact_score<T>(a, a.r0 + r, i, mine ? c : -1);
      if (mine && (lane & 7) == 0) ex[c] = s;
    }
    __syncthreads();
    for (int n = 0; n < places; ++n) {
      double best = -INFINITY;
      int at = INT_MAX;
      for (int c = tid; c < a.K; c += kCtaThreads)
        if (state[c] == 2 && ex[c] > best) best = ex[c], at = c;
#pragma unroll
      for (int o = 16; o >= 1; o >>= 1) {
        const double s = __shfl_xor_sync(0xFFFFFFFFu, best, o);
        const int x = __shfl_xor_sync(0xFFFFFFFFu, at, o);
        if (s > best || (s == best && x < at)) best = s, at = x;
      }
      if (lane == 0) s_best[warp] = best, s_at[warp] = at;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < kCtaThreads / 32; ++w)
        if (s_best[w] > best || (s_best[w] == best && s_at[w] < at)) best = s_best[w], at = s_at[w];
      if (at == INT_MAX) break;  // the same in every thread
      if (tid == 0) state[at] = 1;
      __syncthreads();
    }
  }
  __syncthreads();
  int32_t* out = a.sel + (static_cast<int64_t>(a.r0 + r) * a.all + i) * a.top;
  int done = 0;
  for (int c0 = 0; c0 < a.K; c0 += kCtaThreads) {
    const int c = c0 + tid;
    const bool on = c < a.K && (state[c] == 1 || (all && state[c] == 2));
    const uint32_t who = __ballot_sync(0xFFFFFFFFu, on);
    __syncthreads();
    if (lane == 0) red[warp] = __popc(who);
    __syncthreads();
    int before = done, total = 0;
#pragma unroll
    for (int w = 0; w < kCtaThreads / 32; ++w) {
      if (w < warp) before += red[w];
      total += red[w];
    }
    const int at = before + __popc(who & ((1u << lane) - 1u));
    if (on && at < a.top) out[at] = c;
    done += total;
  }
  for (int j = done + tid; j < a.top; j += kCtaThreads) out[j] = -1;
}

size_t cta_smem(int K) { return align_up(static_cast<size_t>(K) * 13, 16); }

// Rounds of rows, or of one row's queries, whose scores stay below 2^24 (64 MB): the scratch does not
// grow with the prompt, and the scores are still in L2 when the choice reads them.
struct SelectLayout {
  size_t scores, q_norm, c_norm, total;
  int64_t rows, queries;  // of a round, at most
  int ctiles;
};

SelectLayout select_layout(int64_t R, int64_t Nq, int64_t K) {
  SelectLayout l{};
  auto even = [](int64_t all, int64_t most) {  // rounds of equal size
    const int64_t rounds = (all + most - 1) / most;
    return (all + rounds - 1) / rounds;
  };
  constexpr int64_t kScores = 1 << 24;
  l.queries = even(Nq, std::max<int64_t>(1, kScores / K));
  l.rows = l.queries < Nq ? 1 : even(R, std::max<int64_t>(1, kScores / (Nq * K)));
  R = l.rows, Nq = l.queries;
  l.ctiles = static_cast<int>((K + kClusters - 1) / kClusters);
  l.scores = 0;
  l.q_norm = align_up(static_cast<size_t>(R * Nq * K) * 4, 256);
  l.c_norm = l.q_norm + align_up(static_cast<size_t>(R * Nq) * 4, 256);
  l.total = l.c_norm + align_up(static_cast<size_t>(R * l.ctiles) * 4, 256);
  return l;
}

template <typename T, int DP, int QW, bool PACK = false>
int score_typed(const SelectArgs& a, int64_t R, float* scores, float* qn, float* cn, int ctiles,
                cudaStream_t stream) {
  const int qtiles = (a.Nq + 16 * QW - 1) / (16 * QW);
  const int smem = (kClusters + 2 * 16 * QW) * DP * 2;
  auto kern = score_kernel<T, DP, QW, PACK>;
  FKC_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  const int64_t blocks = R * qtiles * ctiles;
  FKC_REQUIRE(blocks <= 2147483647ll, "select: too many tiles");
  return launch_pdl(kern, dim3(static_cast<unsigned>(blocks)), dim3(128), smem, stream, a, scores,
                    qn, cn, ctiles, qtiles);
}

template <typename T>
int select_round(const SelectArgs& a, int64_t R, const SelectLayout& l, uint8_t* ws, cudaStream_t stream) {
  float* scores = reinterpret_cast<float*>(ws + l.scores);
  float* qn = reinterpret_cast<float*>(ws + l.q_norm);
  float* cn = reinterpret_cast<float*>(ws + l.c_norm);
  // a few queries: one warp's rows (of all heads at once where they fit), the other warps
  // take clusters
  const bool pack = static_cast<int64_t>(a.Nq) * a.G <= 16, few = a.Nq <= 16;
  auto score = a.D <= 64 ? (pack  ? score_typed<T, 64, 1, true>
                            : few ? score_typed<T, 64, 1>
                                  : score_typed<T, 64, 4>)
                         : (pack  ? score_typed<T, 128, 1, true>
                            : few ? score_typed<T, 128, 1>
                                  : score_typed<T, 128, 4>);
  FKC_TRY(score(a, R, scores, qn, cn, l.ctiles, stream));
  const int64_t queries = R * a.Nq;
  // a warp's registers hold the scores of 1024 clusters; where there are fewer warps than
  // schedulers (148 x 4), a CTA per query is faster (128 queries of 1024 clusters: 21 us, a warp
  // per query 33 us; 32768 queries of 256: a warp 42 us, and a CTA's barriers would come 32768
  // times)
  if (a.K <= 1024 && queries > 592) {
    auto kern = a.K <= 128   ? choose_warp_kernel<T, 4>
                : a.K <= 256 ? choose_warp_kernel<T, 8>
                : a.K <= 512 ? choose_warp_kernel<T, 16>
                             : choose_warp_kernel<T, 32>;
    // three times what the SMs hold: a warp has a few queries to prefetch over, and their uneven
    // work evens out
    const int64_t ctas = std::min<int64_t>((queries + 3) / 4, 148 * (a.K <= 256 ? 30 : 12));
    return launch_pdl(kern, dim3(static_cast<unsigned>(ctas)), dim3(128), 0, stream, a,
                      static_cast<const float*>(scores), static_cast<const float*>(qn),
                      static_cast<const float*>(cn), l.ctiles, queries);
  }
  const size_t smem = cta_smem(a.K);
  FKC_CUDA_TRY(cudaFuncSetAttribute(choose_cta_kernel<T>,
                                    cudaFuncAttributeMaxDynamicSharedMemorySize,
                                    static_cast<int>(smem)));
  return launch_pdl(choose_cta_kernel<T>, dim3(static_cast<unsigned>(queries)), dim3(kCtaThreads),
                    smem, stream, a, static_cast<const float*>(scores),
                    static_cast<const float*>(qn), static_cast<const float*>(cn), l.ctiles);
}

template <typename T>
int select_dtype(SelectArgs a, int64_t R, uint8_t* ws, cudaStream_t stream) {
  const SelectLayout l = select_layout(R, a.all, a.K);
  const T* q = static_cast<const T*>(a.q);
  const int32_t* q_pos = a.q_pos;
  int32_t* sel = a.sel;
  for (int64_t r0 = 0; r0 < R; r0 += l.rows)
    for (int64_t i0 = 0; i0 < a.all; i0 += l.queries) {
      a.r0 = static_cast<int>(r0);
      a.Nq = static_cast<int>(std::min(l.queries, a.all - i0));
      a.q = q + i0 * a.qs.n;
      a.q_pos = q_pos != nullptr ? q_pos + i0 : nullptr;
      a.sel = sel + i0 * a.top;
      FKC_TRY(select_round<T>(a, std::min(l.rows, R - r0), l, ws, stream));
    }
  return FKC_OK;
}

}  // namespace

size_t select_workspace_bytes(int64_t R, int64_t Nq, int64_t K) {
  return select_layout(R, Nq, K).total;
}

int launch_select(const Args& f, const void* centroids, const float* bias, double scale, int dtype,
                  int32_t* sel, void* ws, cudaStream_t stream) {
  SelectArgs a{};
  a.q = f.q;
  a.centroids = centroids;
  a.qs = f.qs;
  a.offsets = f.offsets;
  a.order = f.order;
  a.q_pos = f.q_pos;
  a.bias = bias;
  a.Hkv = f.Hkv;
  a.G = f.G;
  a.all = f.Nq;
  a.sel = sel;
  a.N = f.N;
  a.K = f.K;
  a.top = f.top;
  a.D = f.D;
  a.scale = scale;
  // (a scale below fp32's least normal number is off by 2^-150 itself)
  a.unsure = std::max(std::fabs(scale), 0x1p-126) * (f.D * 0x1p-22 + 0x1p-21);
  const int64_t R = static_cast<int64_t>(f.batch) * f.Hkv;
  uint8_t* w = static_cast<uint8_t*>(ws);
  return dtype == FKC_DTYPE_F16 ? select_dtype<__half>(a, R, w, stream)
                                : select_dtype<__nv_bfloat16>(a, R, w, stream);
}

}  // namespace attn
}  // namespace fkc
