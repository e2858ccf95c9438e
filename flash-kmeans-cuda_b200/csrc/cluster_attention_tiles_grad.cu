// Gradients of attention over selected clusters, cluster by cluster (see
// cluster_attention_tiles.cu for units and rows, cluster_attention_grad.cu for the formulas).
//
//   delta   (tiles_dq_kernel)   the sum of P dP over each row's keys, cluster by cluster, and
//           tiles_delta_join_kernel adds a query's top sums (why not from out: cluster_attention_grad.cu).
//   dQ      (tiles_dq_kernel)   a unit's 128 rows against the cluster's keys in steps of 128:
//           S = Q K^T and dP = dO V^T into TMEM, dS in place, dQ += dS K. A row leaves its
//           gradient over that cluster as the forward leaves its output, and
//           tiles_dq_join_kernel adds a query's top parts.
//   dK, dV  (tiles_dkv_kernel)  128 keys of a cluster against the cluster's rows in steps of
//           128: S^T = K Q^T and dP^T = V dO^T, P^T and dS^T in place, dV += P^T dO and
//           dK += dS^T Q. All steps of all key tiles are one sequence, cut into equal shares, so
//           that a cluster that many queries read occupies many CTAs; a key tile cut by a
//           border leaves fp32 sums of each side, and tiles_dkv_join_kernel adds them in order.
//           The sequence is fixed by the inputs, so two runs give the same bits.
//
// The 128 columns of a step are two halves of 64, a warpgroup each (a thread a row of TMEM), whose
// products start as each is done. (S and dP of 64 columns at a time, so that one half's
// products would run beside the other's scores, took twice as long: an MMA of N = 64 costs
// about as much as one of 128.) P and dS enter
// their products as two terms each (cluster_attention_grad.cu).
//
// 4096 queries x 4 rows of G = 4, 8 of 64 clusters of 64 keys, D = 128: delta 108 us and its join 6, dQ 155
// and its join 36, dK and dV 173 and their join 14, rows and tiles listed in 55 (forward and backward
// together 680 us; with delta from out, one term of P and of dK's dS and parts of two bytes 494). The
// three large kernels are bound by the chain of one 128-row step: gathered rows (twice the warps
// gathering them took 4% off delta's), two score products, the warpgroups' turn (a thread a row, 64
// columns), two or four products; the tensor pipe is busy for 16%, 22% and 37%. The walk took 2200 us for
// the gradients, warp-level matrix instructions as little; scores of 64 columns at a time 630 us, joins of
// single heads 560.
#include <algorithm>

#include "cluster_tiles.cuh"
#include "fkc_common.cuh"

namespace fkc {
namespace attn {
namespace {

enum : int { kErrDqLoad = 161, kErrDqMma = 162, kErrDq = 163, kErrDkvLoad = 171, kErrDkvMma = 172, kErrDkv = 173 };

// ---------------------------------------------------------------------------- dQ
// The 128-row halves of a CTA's units in turn, as UnitIter.
struct SubIter {
  const Unit* units;
  int n, total, x;
  uint32_t load;
  bool again, keep, follows;  // follows: another unit of the cluster, in this CTA
  Unit un, next;

  __device__ __forceinline__ SubIter(const Unit* u, const int32_t* start)
      : units(u), n(__ldg(start + blockIdx.x)), total(__ldg(start + blockIdx.x + 1)), x(0), load(0),
        again(false), keep(false), follows(false) {
    if (n < total) next = load_unit(units + n);
    open();
  }
  __device__ __forceinline__ void open() {
    if (n >= total) return;
    un = next;
    if (n + 1 < total) next = load_unit(units + n + 1);
    follows = (un.nrows & Unit::kMore) != 0 && n + 1 < total;
    un.nrows &= Unit::kMore - 1;
    keep = un.steps() <= 2 && (more() || follows);
  }
  __device__ __forceinline__ bool more() const { return x == 0 && un.nrows > kSub; }
  __device__ __forceinline__ bool valid() const { return n < total; }
  // unit row of the half's first row, and of the next half's (-1: none)
  __device__ __forceinline__ int64_t row() const { return static_cast<int64_t>(n) * kUnitRows + x * kSub; }
  __device__ __forceinline__ int64_t next_row() const {
    return more() ? row() + kSub : n + 1 < total ? static_cast<int64_t>(n + 1) * kUnitRows : -1;
  }
  __device__ __forceinline__ void advance() {
    if (!keep) load += un.steps();
    again = keep;
    if (more()) {
      x = 1;
      keep = un.steps() <= 2 && follows;
    } else {
      x = 0;
      ++n;
      keep = false;
      open();
    }
  }
};

template <int DP>
struct DqSmem {
  static constexpr uint32_t kTile = tc_tile_bytes<DP>();
  static constexpr uint32_t kQ = 0, kDo = kTile;
  static constexpr uint32_t kK = 2 * kTile;  // two stages
  static constexpr uint32_t kV = 4 * kTile;  // two stages
  static constexpr uint32_t kOut = 6 * kTile;
  static constexpr uint32_t kMeta = kOut + 8 * 4096;
  struct Meta {
    int32_t key[2][kKeysStep];
    uint64_t k_full[2], v_full[2], kv_free[2], q_full, q_free, sp_full[2], sp_free[2], ds_full[2], dq_full, dq_free;
    uint64_t drain;
    uint32_t tmem;
    int abort;
  };
  static constexpr uint32_t kBytes = kMeta + sizeof(Meta) + 1024;
};

// Warps 0-3, 4-7: keys 0-63 and 64-127 of a step; 8: the MMAs; 9, 10: gathers of keys and
// values; 11, 12: of Q; 13, 14: of dout.
constexpr int kGradThreads = 32 * 15;

// kDelta: the sums of P dP over each row's keys instead, two floats a row (one per half of a step's
// keys), and behind those of all units' rows the same of P |dP| for fp16 (see Range); with two S and dP in
// TMEM in turn, since nothing follows them.
template <typename T, int DP, bool kDelta>
__global__ void __launch_bounds__(kGradThreads, 1) tiles_dq_kernel(
    const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
    const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ CUtensorMap tm_do, RowMap rk,
    RowMap rv, Args a, const int32_t* __restrict__ q_row, const int32_t* __restrict__ do_row,
    const int32_t* __restrict__ row_pos, const float* __restrict__ row_lse,
    const float* __restrict__ row_delta, const float* __restrict__ row_power,
    const Unit* __restrict__ units, const int32_t* __restrict__ start, uint8_t* __restrict__ part,
    int64_t units_max, int* err) {
  using namespace ptx;
  using S = DqSmem<DP>;
  constexpr uint32_t kBf16 = std::is_same<T, __half>::value ? 0u : 1u;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  const uint32_t sb = smem_u32(smem);
  typename S::Meta& mt = *reinterpret_cast<typename S::Meta*>(smem + S::kMeta);
  volatile int* abort = &mt.abort;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int x = 0; x < 2; ++x) {
      mbar_init(smem_u32(&mt.k_full[x]), 32);  // the gathering lanes (their keys), and the bytes
      mbar_init(smem_u32(&mt.v_full[x]), 1);
      mbar_init(smem_u32(&mt.kv_free[x]), kDelta ? 9 : 1);  // kDelta: the warps that read the keys, too
      mbar_init(smem_u32(&mt.ds_full[x]), 128);
      mbar_init(smem_u32(&mt.sp_full[x]), 1);
      mbar_init(smem_u32(&mt.sp_free[x]), 256);
    }
    mbar_init(smem_u32(&mt.q_full), 4);
    mbar_init(smem_u32(&mt.q_free), 1);
    mbar_init(smem_u32(&mt.dq_full), 1);
    mbar_init(smem_u32(&mt.dq_free), 256);
    mbar_init(smem_u32(&mt.drain), 1);
    mt.abort = 0;
    fence_mbar_init();
  }
  if (warp == 8) {
    tmem_alloc(smem_u32(&mt.tmem), 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = mt.tmem;  // S at 0, dP at 128, dQ at 256 (kDelta: the second S and dP)
  pdl_wait();

  if (warp < 8) {
    // ------------------------------------------------------------ dS, output
    const int half = warp >> 2, row = (warp & 3) * 32 + lane;
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t t_s = tmem + lanes + half * 64, t_p = t_s + 128, t_q = tmem + lanes + 256;
    const float sc = a.scale * kLog2e;
    uint32_t uses = 0, s_uses = 0;
    bool ok = true;
    SubIter it(units, start);
    int pos_next = -1;
    float lse_next = 0.f, delta_next = 0.f, power_next = 1.f;
    auto fetch = [&](int64_t first) {
      if (first < 0) return;
      pos_next = __ldg(row_pos + first + row);
      lse_next = __ldg(row_lse + first + row);
      if (!kDelta) delta_next = __ldg(row_delta + first + row);
      if (!kDelta && Range<T>::kNarrow) power_next = __ldg(row_power + first + row);
    };
    if (it.valid()) fetch(it.row());
    if constexpr (kDelta) {
      for (; ok && it.valid(); it.advance()) {
        const int pos = pos_next;
        const float lse = lse_next;
        fetch(it.next_row());
        const int steps = it.un.steps();
        float sum[4] = {0.f, 0.f, 0.f, 0.f}, mag[4] = {0.f, 0.f, 0.f, 0.f};
        for (int step = 0; step < steps; ++step, ++s_uses) {
          const int keys = it.un.keys(step) - half * 64;  // may be none, but every phase is waited for
          const uint32_t load = it.load + step, buf = s_uses & 1;
          const int st = load & 1;
          ok = warp_mbar_wait(&mt.k_full[st], (load >> 1) & 1, abort) &&
               warp_mbar_wait(&mt.sp_full[buf], (s_uses >> 1) & 1, abort);
          if (!ok) break;
          tc_fence_after();
          const int32_t* key = mt.key[st] + half * 64;
#pragma unroll 1
          for (int c = 0; c < 2; ++c) {
            if (c * 32 >= keys) break;
            float s[32], dp[32];
            tmem_ld_f32_x32(t_s + buf * 256 + c * 32, s);
            tmem_ld_f32_x32(t_p + buf * 256 + c * 32, dp);
            tmem_wait_ld();
#pragma unroll
            for (int j = 0; j < 32; j += 4) {
              const int4 k4 = *reinterpret_cast<const int4*>(key + c * 32 + j);
              const int k[4] = {k4.x, k4.y, k4.z, k4.w};
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const float x = ex2(fmaf(s[j + e], sc, -lse)) * dp[j + e];
                sum[e] += k[e] <= pos ? x : 0.f;
                if (Range<T>::kNarrow) mag[e] += k[e] <= pos ? fabsf(x) : 0.f;
              }
            }
          }
          tc_fence_before();
          mbar_arrive(smem_u32(&mt.sp_free[buf]));
          __syncwarp();
          if (lane == 0 && !it.keep) mbar_arrive(smem_u32(&mt.kv_free[st]));
        }
        if (!ok) break;
        float* to = reinterpret_cast<float*>(part) + (it.row() + row) * 2 + half;
        *to = (sum[0] + sum[1]) + (sum[2] + sum[3]);
        if (Range<T>::kNarrow) to[units_max * kUnitRows * 2] = (mag[0] + mag[1]) + (mag[2] + mag[3]);
      }
      if (!ok) give_up(abort, err, kErrDq);
    } else {
      for (; ok && it.valid(); it.advance(), ++uses) {
        const int pos = pos_next;
        const float lse = lse_next, pw = power_next, delta = delta_next * pw;
        fetch(it.next_row());
        const int steps = it.un.steps();
        for (int step = 0; step < steps; ++step, ++s_uses) {
          const int keys = it.un.keys(step) - half * 64;
          if (keys <= 0) continue;
          const uint32_t load = it.load + step;
          const int st = load & 1;
          ok = warp_mbar_wait(&mt.k_full[st], (load >> 1) & 1, abort) &&
               warp_mbar_wait(&mt.sp_full[0], s_uses & 1, abort);
          if (!ok) break;
          tc_fence_after();
          const int32_t* key = mt.key[st] + half * 64;
#pragma unroll 1
          for (int c = 0; c < 2; ++c) {
            if (c * 32 >= keys) break;
            float s[32], dp[32];
            tmem_ld_f32_x32(t_s + c * 32, s);
            tmem_ld_f32_x32(t_p + c * 32, dp);
            tmem_wait_ld();
#pragma unroll
            for (int j = 0; j < 32; j += 4) {
              const int4 k4 = *reinterpret_cast<const int4*>(key + c * 32 + j);
              const int k[4] = {k4.x, k4.y, k4.z, k4.w};
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const float p = ex2(fmaf(s[j + e], sc, -lse)) * fmaf(dp[j + e], pw, -delta);
                s[j + e] = k[e] <= pos ? p : 0.f;
              }
            }
            split32<T, false>(t_s + c * 32, s);
          }
          tmem_wait_st();
          tc_fence_before();
          mbar_arrive(smem_u32(&mt.ds_full[half]));
        }
        if (ok) ok = warp_mbar_wait(&mt.dq_full, uses & 1, abort);
        if (!ok) break;
        tc_fence_after();
        const int64_t urow = it.row() + row;
        const uint32_t buf = sb + S::kOut + warp * 4096;
        uint8_t* dst = part + (urow - lane) * (DP * kPartBytes);
#pragma unroll 1
        for (int c = half * (DP / 64); c < (half + 1) * (DP / 64); ++c) {  // the segments are shared out
          uint32_t o[32];
          tmem_ld_32x32b_x32(t_q + c * 32, o);
          tmem_wait_ld();
          if (Range<T>::kNarrow) {
            const float back = inverse_power(pw);
#pragma unroll
            for (int j = 0; j < 32; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * back);
          }
          put_segment(buf, o, dst + c * kSegment);
        }
        tc_fence_before();
        mbar_arrive(smem_u32(&mt.dq_free));
      }
      if (!ok) give_up(abort, err, kErrDq);
      if (lane == 0) bulk_wait_all();
    }
  } else if (warp == 8) {
    // ------------------------------------------------------------ MMAs (one thread)
    if (lane == 0) {
      const int dsteps = (a.D + 15) / 16;
      constexpr uint32_t idesc_o = umma_idesc_f16(kBf16, kSub, DP) | kIdescMnB;
      uint32_t uses = 0, ds_uses[2] = {0, 0};
      struct Pending {
        bool has, first, last;
        int stage, ksteps;
        uint32_t use;
      } pend[2] = {};
      int to_free = -1;
      bool ok = true;
      auto product = [&](int half) {  // dQ (+)= dS K over the half's keys
        Pending& p = pend[half];
        if (!p.has) return;
        p.has = false;
        ok = ok && mbar_wait(smem_u32(&mt.ds_full[half]), ds_uses[half] & 1, abort);
        ++ds_uses[half];
        if (ok && p.first) ok = mbar_wait(smem_u32(&mt.dq_free), (p.use & 1) ^ 1, abort);
        if (!ok) return;
        tc_fence_after();
        const uint32_t kt = sb + S::kK + p.stage * S::kTile + half * 64 * 128;
        mma_tmem_rows<4>(tmem + 256, tmem + half * 64, kt, idesc_o, p.ksteps, p.first);
        if (p.last) umma_commit(smem_u32(&mt.dq_full));
      };
      uint32_t n = 0;  // steps
      for (SubIter it(units, start); ok && it.valid(); it.advance(), ++uses) {
        const int steps = it.un.steps();
        for (int step = 0; ok && step < steps; ++step, ++n) {
          const uint32_t load = it.load + step, buf = kDelta ? n & 1 : 0;
          const int st = load & 1;
          const int keys = it.un.keys(step);
          if constexpr (kDelta) {
            ok = mbar_wait(smem_u32(&mt.sp_free[buf]), ((n >> 1) & 1) ^ 1, abort);
          } else {
            product(0);
            product(1);
          }
          ok = ok && mbar_wait(smem_u32(&mt.k_full[st]), (load >> 1) & 1, abort) &&
               mbar_wait(smem_u32(&mt.v_full[st]), (load >> 1) & 1, abort) &&
               mbar_wait(smem_u32(&mt.q_full), uses & 1, abort);
          if (!ok) break;
          const uint32_t idesc = umma_idesc_f16(kBf16, kSub, (keys + 15) / 16 * 16);
          tc_fence_after();
          mma_kmajor<DP>(tmem + buf * 256, sb + S::kQ, sb + S::kK + st * S::kTile, idesc, dsteps);
          mma_kmajor<DP>(tmem + buf * 256 + 128, sb + S::kDo, sb + S::kV + st * S::kTile, idesc, dsteps);
          umma_commit(smem_u32(&mt.sp_full[buf]));
          const bool end = step == steps - 1, two = keys > 64;
          if (end) umma_commit(smem_u32(&mt.q_free));
          if constexpr (kDelta) {
            if (!it.keep) umma_commit(smem_u32(&mt.kv_free[st]));
            continue;
          }
          pend[0] = {true, step == 0, end && !two, st, (min(keys, 64) + 15) / 16, uses};
          if (two) pend[1] = {true, false, end, st, (keys - 64 + 15) / 16, uses};
          if (ok && to_free >= 0) umma_commit(smem_u32(&mt.kv_free[to_free]));
          to_free = it.keep ? -1 : st;
        }
      }
      for (int half = 0; half < 2; ++half)
        if (ok) product(half);
      if (!ok) give_up(abort, err, kErrDqMma);
      umma_commit(smem_u32(&mt.drain));  // nothing is in flight when TMEM is freed
      const int never = 0;
      mbar_wait(smem_u32(&mt.drain), 0, &never);
    }
  } else {
    // ------------------------------------------------------------ gathers
    bool ok = true;
    SubIter it(units, start);
    if (warp <= 10) {
      const bool values = warp == 10;
      const CUtensorMap* tm = values ? &tm_v : &tm_k;
      const RowMap rm = values ? rv : rk;
      const uint32_t tiles = sb + (values ? S::kV : S::kK);
      int step = 0, idx[4];
      auto fetch = [&] {  // positions of keys 4 lane .. of the step
        const int32_t* order = a.order + static_cast<int64_t>(it.un.r) * a.N;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int s = it.un.s0 + step * kKeysStep + lane * 4 + j;
          const int row = s < it.un.s1 ? __ldg(order + s) : -1;
          idx[j] = row >= 0 && row < a.N ? row : INT_MAX;
        }
      };
      if (it.valid()) fetch();
      while (it.valid()) {
        const uint32_t load = it.load + step;
        const int st = load & 1;
        const int b = it.un.r / a.Hkv, hk = it.un.r - b * a.Hkv;
        const int quads = (it.un.keys(step) + 15) / 16 * 4;
        int rows[4];
#pragma unroll
        for (int j = 0; j < 4; ++j)  // a key that no query sees is not read
          rows[j] = idx[j] <= it.un.high ? rm.at(b, hk, idx[j]) : rm.rows;
        const int4 key = make_int4(idx[0], idx[1], idx[2], idx[3]);
        if (++step == it.un.steps()) {
          step = 0;
          do {
            it.advance();
          } while (it.valid() && it.again);
        }
        if (it.valid()) fetch();
        ok = warp_mbar_wait(&mt.kv_free[st], ((load >> 1) & 1) ^ 1, abort);
        if (!ok) break;
        uint64_t* full = values ? &mt.v_full[st] : &mt.k_full[st];
        if (!values) *reinterpret_cast<int4*>(&mt.key[st][lane * 4]) = key;
        if (lane == 0)
          mbar_arrive_expect_tx(smem_u32(full), quads * 4 * DP * 2);
        else if (!values)
          mbar_arrive(smem_u32(full));
        if (lane < quads)
          gather_rows4<DP>(tiles + st * S::kTile, tm, full, lane * 4, rows[0], rows[1], rows[2], rows[3]);
        __syncwarp();
      }
    } else {
      const bool grads = warp >= 13;
      const CUtensorMap* tm = grads ? &tm_do : &tm_q;
      const int row0 = ((warp - 11) & 1) * 64 + (lane & 15) * 4, blk = lane >> 4;
      const int32_t* src = (grads ? do_row : q_row) + row0;
      const uint32_t dst = sb + (grads ? S::kDo : S::kQ) + blk * (128 * kSub) + row0 * 128;
      auto fetch = [&](int64_t first) {
        return first < 0 ? make_int4(0, 0, 0, 0) : __ldg(reinterpret_cast<const int4*>(src + first));
      };
      int4 ahead = it.valid() ? fetch(it.row()) : make_int4(0, 0, 0, 0);
      for (uint32_t uses = 0; it.valid(); it.advance(), ++uses) {
        const int4 rows = ahead;
        ahead = fetch(it.next_row());
        ok = warp_mbar_wait(&mt.q_free, (uses & 1) ^ 1, abort);
        if (!ok) break;
        if (lane == 0) mbar_arrive_expect_tx(smem_u32(&mt.q_full), S::kTile / 2);
        if (blk < DP / 64)  // a block of 64 elements by each half of the warp
          tma_gather4(dst, tm, smem_u32(&mt.q_full), blk * 64, rows.x, rows.y, rows.z, rows.w);
        __syncwarp();
      }
    }
    if (!ok) give_up(abort, err, kErrDqLoad);
    if (!ok || *abort) {  // copies in flight end before the CTA does
      const uint64_t t0 = globaltimer_ns();
      while (globaltimer_ns() - t0 < 1000000ull) {
      }
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == 8) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// One thread per (query, head): delta and the power of two of dS from its clusters' sums, to their units'
// rows, and the largest A of each row of clusters.
template <typename T>
__global__ void __launch_bounds__(256) tiles_delta_join_kernel(Args a, const int32_t* __restrict__ pair_row,
                                                               const float2* __restrict__ part,
                                                               int64_t units_max,
                                                               float* __restrict__ delta,
                                                               float* __restrict__ row_delta,
                                                               float* __restrict__ row_power,
                                                               float* __restrict__ largest, int64_t rows) {
  pdl_wait();
  const int64_t t = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;  // (r, i, head)
  if (t >= rows) return;
  const int64_t qi = t / a.G;
  const int h = static_cast<int>(t - qi * a.G), r = static_cast<int>(qi / a.Nq), i = static_cast<int>(qi - static_cast<int64_t>(r) * a.Nq);
  const int32_t* pairs = pair_row + qi * a.top;
  auto total = [&](const float2* x) {
    float sum = 0.f;
    for (int s0 = 0; s0 < a.top; s0 += 8) {
      float2 v[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const int n = s0 + u < a.top ? pairs[s0 + u] : -1;
        v[u] = n >= 0 ? x[static_cast<int64_t>(n) + h] : make_float2(0.f, 0.f);
      }
#pragma unroll
      for (int u = 0; u < 8; ++u) sum += v[u].x + v[u].y;
    }
    return sum;
  };
  const float sum = total(part), A = Range<T>::kNarrow ? total(part + units_max * kUnitRows) : 0.f;
  const int b = r / a.Hkv;
  delta[(static_cast<int64_t>(b) * a.Hq + (r - b * a.Hkv) * a.G + h) * a.Nq + i] = sum;
  for (int s = 0; s < a.top; ++s) {
    const int n = pairs[s];
    if (n < 0) continue;
    row_delta[static_cast<int64_t>(n) + h] = sum;
    if (Range<T>::kNarrow) row_power[static_cast<int64_t>(n) + h] = power(A);
  }
  if (Range<T>::kNarrow && A < INFINITY) note_largest(largest + r, A);
}

// One warp per (query, GP heads): dq = scale * the sum of its clusters' parts.
template <typename T, int DP>
__global__ void __launch_bounds__(256, 3) tiles_dq_join_kernel(Args a, int gp, int chunks,
                                                            const int32_t* __restrict__ pair_row,
                                                            const uint8_t* __restrict__ part,
                                                            T* __restrict__ dq, int32_t* __restrict__ odd,
                                                            int64_t warps) {
  constexpr int E = 8, SEGS = DP / 64;
  constexpr int kAhead = 8 / SEGS;  // slots in flight per lane
  pdl_wait();
  const int64_t w0 = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);  // (r, i, heads)
  if (w0 >= warps) return;
  const JoinLane me(gp);
  const int h = static_cast<int>(w0 % chunks) * gp + me.head;
  const int64_t qi = w0 / chunks;
  const int r = static_cast<int>(qi / a.Nq), i = static_cast<int>(qi % a.Nq);
  const int b = r / a.Hkv, per = 4 / gp;
  const int32_t* pairs = pair_row + qi * a.top;
  float acc[SEGS][E];
#pragma unroll
  for (int g = 0; g < SEGS; ++g)
#pragma unroll
    for (int e = 0; e < E; ++e) acc[g][e] = 0.f;
  for (int s0 = 0; s0 < a.top; s0 += kAhead * per) {
    Part8 v[kAhead][SEGS];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int s = s0 + u * per + me.slot;
      const int64_t n = s < a.top && h < a.G ? pairs[s] : -1;
#pragma unroll
      for (int g = 0; g < SEGS; ++g) {
        v[u][g] = Part8{};
        if (n >= 0) v[u][g] = load_part<DP>(part, n + h, g * 8 + me.piece);
      }
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
#pragma unroll
      for (int g = 0; g < SEGS; ++g) add_part(acc[g], v[u][g], 1.f);
  }
  for (int o = 8 * gp; o < 32; o <<= 1)  // the slots' lanes
#pragma unroll
    for (int g = 0; g < SEGS; ++g)
#pragma unroll
      for (int e = 0; e < E; ++e) acc[g][e] += __shfl_xor_sync(0xFFFFFFFFu, acc[g][e], o);
  if (me.slot != 0 || h >= a.G) return;
  T* out = dq + ((static_cast<int64_t>(b) * a.Hq + (r - b * a.Hkv) * a.G + h) * a.Nq + i) * a.D;
#pragma unroll
  for (int g = 0; g < SEGS; ++g) {
    const int d = (g * 8 + me.piece) * E;
    if (d < a.D) store_out<T>(out + d, acc[g], a.scale);
  }
  float bad = 0.f;
#pragma unroll
  for (int g = 0; g < SEGS; ++g)
#pragma unroll
    for (int e = 0; e < E; ++e) bad = not_finite(acc[g][e], bad);
  if (bad != 0.f) *odd = 1;
}

// ---------------------------------------------------------------------------- dK, dV
// 128 keys of a cluster: slots [s0, s0 + keys) of row r, and the cluster's `nrows` rows from unit
// row row0 on, in steps of 128; base: steps of the tiles before.
struct __align__(16) KeyTile {
  int r, s0, keys, high;
  int row0, nrows;
  int64_t base;
  __device__ __forceinline__ int steps() const { return (nrows + kSub - 1) / kSub; }
};
__device__ __forceinline__ KeyTile load_tile(const KeyTile* t) {
  KeyTile x;
  const int4 lo = __ldg(reinterpret_cast<const int4*>(t)), hi = __ldg(reinterpret_cast<const int4*>(t) + 1);
  x.r = lo.x, x.s0 = lo.y, x.keys = lo.z, x.high = lo.w;
  x.row0 = hi.x, x.nrows = hi.y;
  x.base = (static_cast<int64_t>(hi.w) << 32) | static_cast<uint32_t>(hi.z);
  return x;
}

// Key tiles of one row at most: of n keys a cluster has one for every kSub and one for the rest.
__host__ __device__ __forceinline__ int64_t row_tiles_max(int64_t K, int64_t N) { return (K < N ? K : N) + N / kSub; }

// Key tiles and steps of every row r: first[2 r], first[2 r + 1] before the scan over rows. A row whose
// offsets no grouping gives (clusters that overlap) may have more tiles than row_tiles_max: it has none
// at all then, and no gradient of its keys, since the list has no room for them.
__device__ __forceinline__ void tiles_of(const Args& a, const int32_t* inv_offsets, int r, int c, int& s0,
                                         int& s1, int& nrows) {
  nrows = 0;
  s0 = s1 = 0;
  if (c >= a.K) return;
  const int32_t* of = inv_offsets + static_cast<int64_t>(r) * (a.K + 1) + c;
  cluster_span(a, r, c, s0, s1);
  nrows = (of[1] - of[0]) * a.G;
}

__global__ void __launch_bounds__(1024) key_count_kernel(Args a, const int32_t* __restrict__ inv_offsets,
                                                         int64_t* __restrict__ first) {
  __shared__ int64_t sums[2][32];
  pdl_wait();
  const int r = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int64_t tiles = 0, steps = 0;
  for (int c = threadIdx.x; c < a.K; c += 1024) {
    int s0, s1, nrows;
    tiles_of(a, inv_offsets, r, c, s0, s1, nrows);
    if (nrows == 0) continue;
    const int n = (s1 - s0 + kSub - 1) / kSub;
    tiles += n;
    steps += static_cast<int64_t>(n) * ((nrows + kSub - 1) / kSub);
  }
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) {
    tiles += __shfl_xor_sync(0xFFFFFFFFu, tiles, o);
    steps += __shfl_xor_sync(0xFFFFFFFFu, steps, o);
  }
  if (lane == 0) sums[0][warp] = tiles, sums[1][warp] = steps;
  __syncthreads();
  if (threadIdx.x < 2) {
    int64_t n = 0, s = 0;
    for (int w = 0; w < 32; ++w) n += sums[0][w], s += sums[threadIdx.x][w];
    first[2 * r + threadIdx.x] = n <= row_tiles_max(a.K, a.N) ? s : 0;
  }
}

// The key tiles in the order of rows and clusters, each CTA's share of the steps, [share[j],
// share[j + 1]) with share[j] = j total / ctas, and the tile in which it begins.
__global__ void __launch_bounds__(1024) key_tiles_kernel(Args a, const int32_t* __restrict__ inv_offsets,
                                                         const int32_t* __restrict__ first_unit,
                                                         const int64_t* __restrict__ first,
                                                         KeyTile* __restrict__ tiles,
                                                         int64_t* __restrict__ share,
                                                         int32_t* __restrict__ start, int ctas, int R) {
  __shared__ int64_t sums[3][32];
  __shared__ int highs[32];
  pdl_wait();
  const int r = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int64_t tile0 = 0, step0 = 0, total = 0;
  for (int q = threadIdx.x; q < R; q += 1024) {
    const int64_t t = first[2 * q], s = first[2 * q + 1];
    if (q < r) tile0 += t, step0 += s;
    total += s;
  }
  int high = a.q_pos != nullptr ? -1 : a.N;
  if (a.q_pos != nullptr)
    for (int i = threadIdx.x; i < a.Nq; i += 1024)
      high = max(high, min(a.q_pos[static_cast<int64_t>(r / a.Hkv) * a.Nq + i], a.N));
  high = __reduce_max_sync(0xFFFFFFFFu, high);
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) {
    tile0 += __shfl_xor_sync(0xFFFFFFFFu, tile0, o);
    step0 += __shfl_xor_sync(0xFFFFFFFFu, step0, o);
    total += __shfl_xor_sync(0xFFFFFFFFu, total, o);
  }
  if (lane == 0) sums[0][warp] = tile0, sums[1][warp] = step0, sums[2][warp] = total, highs[warp] = high;
  __syncthreads();
  tile0 = step0 = total = 0;
  for (int w = 0; w < 32; ++w) {
    tile0 += sums[0][w], step0 += sums[1][w], total += sums[2][w];
    high = max(high, highs[w]);
  }
  if (r == 0)
    for (int j = threadIdx.x; j <= ctas; j += 1024) {
      share[j] = j * total / ctas;
      if (total == 0 && j < ctas) start[j] = 0;
    }
  if (first[2 * r] == 0) return;
  for (int c0 = 0; c0 < a.K; c0 += 1024) {
    const int c = c0 + threadIdx.x;
    int s0, s1, nrows;
    tiles_of(a, inv_offsets, r, c, s0, s1, nrows);
    const int n = nrows > 0 ? (s1 - s0 + kSub - 1) / kSub : 0;
    const int per = (nrows + kSub - 1) / kSub;
    int64_t ti = n, si = static_cast<int64_t>(n) * per;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t t = __shfl_up_sync(0xFFFFFFFFu, ti, o), s = __shfl_up_sync(0xFFFFFFFFu, si, o);
      if (lane >= o) ti += t, si += s;
    }
    __syncthreads();
    if (lane == 31) sums[0][warp] = ti, sums[1][warp] = si;
    __syncthreads();
    int64_t t_at = tile0 + ti - n, s_at = step0 + si - static_cast<int64_t>(n) * per;
    for (int w = 0; w < 32; ++w) {
      if (w < warp) t_at += sums[0][w], s_at += sums[1][w];
      tile0 += sums[0][w], step0 += sums[1][w];
    }
    for (int k = 0; k < n; ++k, ++t_at, s_at += per) {
      KeyTile t;
      t.r = r, t.s0 = s0 + k * kSub, t.keys = min(kSub, s1 - s0 - k * kSub), t.high = high;
      t.row0 = first_unit[static_cast<int64_t>(r) * a.K + c] * kUnitRows;
      t.nrows = nrows, t.base = s_at;
      tiles[t_at] = t;
      // the shares that begin inside: j total / ctas in [s_at, s_at + per)
      for (int64_t j = (s_at * ctas + total - 1) / total; j < ctas && j * total < (s_at + per) * ctas; ++j)
        start[j] = static_cast<int32_t>(t_at);
    }
  }
}

// A CTA's share as segments: steps [step, end) of the 128-row steps of a key tile.
struct SegIter {
  const KeyTile* tiles;
  int64_t at, to;  // in the sequence of all steps
  int n, step, end, seg;
  KeyTile tile;
  __device__ __forceinline__ SegIter(const KeyTile* t, const int32_t* start, const int64_t* share)
      : tiles(t), at(__ldg(share + blockIdx.x)), to(__ldg(share + blockIdx.x + 1)),
        n(__ldg(start + blockIdx.x)), seg(0) {
    if (at < to) open();
  }
  __device__ __forceinline__ void open() {
    tile = load_tile(tiles + n);
    step = static_cast<int>(at - tile.base);
    end = static_cast<int>(min(static_cast<int64_t>(tile.steps()), to - tile.base));
  }
  __device__ __forceinline__ bool valid() const { return at < to; }
  __device__ __forceinline__ void advance() {
    at += end - step;
    ++n;
    ++seg;
    if (at < to) open();
  }
};

template <int DP>
struct DkvSmem {
  static constexpr uint32_t kTile = tc_tile_bytes<DP>();
  static constexpr uint32_t kK = 0, kV = kTile;
  static constexpr uint32_t kQ = 2 * kTile;   // two stages
  static constexpr uint32_t kDo = 4 * kTile;  // two stages
  static constexpr uint32_t kMeta = 6 * kTile;
  struct Meta {
    float lse[2][kSub], delta[2][kSub];  // of a stage's rows; lse less P's shift
    int32_t pos[2][kSub];
    uint64_t kv_full, kv_free, q_full[2], q_free[2], sp_full, ds_full[2], acc_full, acc_free;
    uint64_t drain;
    uint32_t tmem;
    int abort;
  };
  static constexpr uint32_t kBytes = kMeta + sizeof(Meta) + 1024;
};

// Warps 0-3, 4-7: rows 0-63 and 64-127 of a step (a thread a key); 8: the MMAs; 9, 10: gathers
// of the tile's keys and values; 11, 12: of Q; 13, 14: of dout. part: two fp32 (dV, dK) tiles per
// CTA, for a first segment that began in another CTA and a last one that goes on in the next.
template <typename T, int DP>
__global__ void __launch_bounds__(kGradThreads, 1) tiles_dkv_kernel(
    const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
    const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ CUtensorMap tm_do, RowMap rk,
    RowMap rv, Args a, const int32_t* __restrict__ q_row, const int32_t* __restrict__ do_row,
    const int32_t* __restrict__ row_pos, const float* __restrict__ row_lse,
    const float* __restrict__ row_delta, const KeyTile* __restrict__ tiles,
    const int64_t* __restrict__ share, const int32_t* __restrict__ start,
    const float* __restrict__ largest, T* __restrict__ dk, T* __restrict__ dv, float* __restrict__ part,
    int32_t* __restrict__ odd, int* err) {
  using namespace ptx;
  using S = DkvSmem<DP>;
  constexpr uint32_t kBf16 = std::is_same<T, __half>::value ? 0u : 1u;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  const uint32_t sb = smem_u32(smem);
  typename S::Meta& mt = *reinterpret_cast<typename S::Meta*>(smem + S::kMeta);
  volatile int* abort = &mt.abort;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int x = 0; x < 2; ++x) {
      mbar_init(smem_u32(&mt.q_full[x]), 66);  // two warps' lanes (their rows' data), two warps' bytes
      mbar_init(smem_u32(&mt.q_free[x]), 1);
      mbar_init(smem_u32(&mt.ds_full[x]), 128);
    }
    mbar_init(smem_u32(&mt.kv_full), 2);
    mbar_init(smem_u32(&mt.kv_free), 1);
    mbar_init(smem_u32(&mt.sp_full), 1);
    mbar_init(smem_u32(&mt.acc_full), 1);
    mbar_init(smem_u32(&mt.acc_free), 256);
    mbar_init(smem_u32(&mt.drain), 1);
    mt.abort = 0;
    fence_mbar_init();
  }
  if (warp == 8) {
    tmem_alloc(smem_u32(&mt.tmem), 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = mt.tmem;  // S^T at 0, dP^T at 128, dV at 256, dK at 384
  pdl_wait();

  if (warp < 8) {
    // ------------------------------------------------------------ P^T and dS^T, output
    const int half = warp >> 2, row = (warp & 3) * 32 + lane;  // a key
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t t_s = tmem + lanes + half * 64, t_p = t_s + 128;
    const uint32_t t_acc = tmem + lanes + 256 + half * 128;  // warps 0-3 write dV, 4-7 dK
    const float sc = a.scale * kLog2e;
    uint32_t item = 0;
    bool ok = true;
    for (SegIter it(tiles, start, share); ok && it.valid(); it.advance()) {
      int key = INT_MAX;
      if (row < it.tile.keys) {
        const int k = __ldg(a.order + static_cast<int64_t>(it.tile.r) * a.N + it.tile.s0 + row);
        if (k >= 0 && k < a.N) key = k;
      }
      const float pw = Range<T>::kNarrow ? power(__ldg(largest + it.tile.r)) : 1.f, ds_power = pw * Range<T>::unshift();
      for (int step = it.step; step < it.end; ++step, ++item) {
        const int rows = it.tile.nrows - step * kSub - half * 64;
        if (rows <= 0) continue;
        const int st = item & 1;
        ok = warp_mbar_wait(&mt.q_full[st], (item >> 1) & 1, abort) &&
             warp_mbar_wait(&mt.sp_full, item & 1, abort);
        if (!ok) break;
        tc_fence_after();
#pragma unroll 1
        for (int c = 0; c < 2; ++c) {
          if (c * 32 >= rows) break;
          float s[32], dp[32];
          tmem_ld_f32_x32(t_s + c * 32, s);
          tmem_ld_f32_x32(t_p + c * 32, dp);
          tmem_wait_ld();
          const int j0 = half * 64 + c * 32;
#pragma unroll
          for (int j = 0; j < 32; j += 4) {
            const int4 p4 = *reinterpret_cast<const int4*>(&mt.pos[st][j0 + j]);
            const float4 l4 = *reinterpret_cast<const float4*>(&mt.lse[st][j0 + j]);
            const float4 d4 = *reinterpret_cast<const float4*>(&mt.delta[st][j0 + j]);
            const int pos[4] = {p4.x, p4.y, p4.z, p4.w};
            const float lse[4] = {l4.x, l4.y, l4.z, l4.w}, delta[4] = {d4.x, d4.y, d4.z, d4.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const bool on = key <= pos[e];
              const float p = ex2(fmaf(s[j + e], sc, -lse[e]));
              const float ds = p * ((dp[j + e] - delta[e]) * ds_power);
              s[j + e] = on ? p : 0.f;
              dp[j + e] = on ? ds : 0.f;
            }
          }
          split32<T, true>(t_s + c * 32, s);
          split32<T, false>(t_p + c * 32, dp);
        }
        tmem_wait_st();
        tc_fence_before();
        mbar_arrive(smem_u32(&mt.ds_full[half]));
      }
      if (ok) ok = warp_mbar_wait(&mt.acc_full, it.seg & 1, abort);
      if (!ok) break;
      tc_fence_after();
      const bool whole = it.step == 0 && it.end == it.tile.steps();
      const float scale = half == 0 ? Range<T>::unshift() : a.scale * inverse_power(pw);
      const int b = it.tile.r / a.Hkv, hk = it.tile.r - b * a.Hkv;
      T* out = (half == 0 ? dv : dk) + ((static_cast<int64_t>(b) * a.Hkv + hk) * a.N + (key == INT_MAX ? 0 : key)) * a.D;
      // a segment that does not begin its tile is the CTA's first
      float* sums = part + ((static_cast<int64_t>(blockIdx.x) * 2 + (it.step == 0)) * 2 + half) * (kSub * DP) + row * DP;
      float bad = 0.f;
#pragma unroll 1
      for (int c = 0; c < DP / 32; ++c) {
        float o[32];
        tmem_ld_f32_x32(t_acc + c * 32, o);
        tmem_wait_ld();
#pragma unroll
        for (int j = 0; j < 32; ++j) bad = not_finite(o[j], bad);
        if (whole) {
#pragma unroll
          for (int j = 0; j < 32; j += 8) {
            const uint4 v = make_uint4(mma::pack2<T>(o[j] * scale, o[j + 1] * scale), mma::pack2<T>(o[j + 2] * scale, o[j + 3] * scale),
                                       mma::pack2<T>(o[j + 4] * scale, o[j + 5] * scale), mma::pack2<T>(o[j + 6] * scale, o[j + 7] * scale));
            if (key != INT_MAX && c * 32 + j < a.D) *reinterpret_cast<uint4*>(out + c * 32 + j) = v;
          }
        } else {
#pragma unroll
          for (int j = 0; j < 32; j += 4)
            *reinterpret_cast<float4*>(sums + c * 32 + j) = make_float4(o[j], o[j + 1], o[j + 2], o[j + 3]);
        }
        __syncwarp();
      }
      if (bad != 0.f && key != INT_MAX) *odd = 1;
      tc_fence_before();
      mbar_arrive(smem_u32(&mt.acc_free));
    }
    if (!ok) give_up(abort, err, kErrDkv);
  } else if (warp == 8) {
    // ------------------------------------------------------------ MMAs (one thread)
    if (lane == 0) {
      const int dsteps = (a.D + 15) / 16;
      constexpr uint32_t idesc_o = umma_idesc_f16(kBf16, kSub, DP) | kIdescMnB;
      uint32_t item = 0, ds_uses[2] = {0, 0};
      struct Pending {
        bool has, first, last;
        int stage, ksteps, seg;
      } pend[2] = {};
      int to_free = -1;
      bool ok = true;
      auto product = [&](int half) {  // dV (+)= P^T dO, dK (+)= dS^T Q over the half's rows
        Pending& p = pend[half];
        if (!p.has) return;
        p.has = false;
        ok = ok && mbar_wait(smem_u32(&mt.ds_full[half]), ds_uses[half] & 1, abort);
        ++ds_uses[half];
        if (ok && p.first) ok = mbar_wait(smem_u32(&mt.acc_free), (p.seg & 1) ^ 1, abort);
        if (!ok) return;
        tc_fence_after();
        const uint32_t o = p.stage * S::kTile + half * 64 * 128;
        mma_tmem_rows<4>(tmem + 256, tmem + half * 64, sb + S::kDo + o, idesc_o, p.ksteps, p.first);
        mma_tmem_rows<4>(tmem + 384, tmem + 128 + half * 64, sb + S::kQ + o, idesc_o, p.ksteps, p.first);
        if (p.last) umma_commit(smem_u32(&mt.acc_full));
      };
      for (SegIter it(tiles, start, share); ok && it.valid(); it.advance()) {
        for (int step = it.step; ok && step < it.end; ++step, ++item) {
          const int st = item & 1;
          const int rows = it.tile.nrows - step * kSub;
          product(0);
          product(1);
          ok = ok && mbar_wait(smem_u32(&mt.kv_full), it.seg & 1, abort) &&
               mbar_wait(smem_u32(&mt.q_full[st]), (item >> 1) & 1, abort);
          if (!ok) break;
          const int mine = min(kSub, rows);
          const uint32_t idesc = umma_idesc_f16(kBf16, kSub, (mine + 15) / 16 * 16);
          mma_kmajor<DP>(tmem, sb + S::kK, sb + S::kQ + st * S::kTile, idesc, dsteps);
          mma_kmajor<DP>(tmem + 128, sb + S::kV, sb + S::kDo + st * S::kTile, idesc, dsteps);
          umma_commit(smem_u32(&mt.sp_full));
          const bool end = step == it.end - 1, two = mine > 64;
          if (end) umma_commit(smem_u32(&mt.kv_free));
          pend[0] = {true, step == it.step, end && !two, st, (min(mine, 64) + 15) / 16, it.seg};
          if (two) pend[1] = {true, false, end, st, (mine - 64 + 15) / 16, it.seg};
          if (ok && to_free >= 0) umma_commit(smem_u32(&mt.q_free[to_free]));
          to_free = st;
        }
      }
      for (int half = 0; half < 2; ++half)
        if (ok) product(half);
      if (!ok) give_up(abort, err, kErrDkvMma);
      umma_commit(smem_u32(&mt.drain));  // nothing is in flight when TMEM is freed
      const int never = 0;
      mbar_wait(smem_u32(&mt.drain), 0, &never);
    }
  } else {
    // ------------------------------------------------------------ gathers
    bool ok = true;
    SegIter it(tiles, start, share);
    if (warp <= 10) {
      const bool values = warp == 10;
      const CUtensorMap* tm = values ? &tm_v : &tm_k;
      const RowMap rm = values ? rv : rk;
      for (; it.valid(); it.advance()) {
        const int32_t* order = a.order + static_cast<int64_t>(it.tile.r) * a.N + it.tile.s0;
        const int b = it.tile.r / a.Hkv, hk = it.tile.r - b * a.Hkv;
        int rows[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {  // a key that no query sees is not read
          const int k = lane * 4 + j < it.tile.keys ? __ldg(order + lane * 4 + j) : -1;
          rows[j] = k >= 0 && k < a.N && k <= it.tile.high ? rm.at(b, hk, k) : rm.rows;
        }
        ok = warp_mbar_wait(&mt.kv_free, (it.seg & 1) ^ 1, abort);
        if (!ok) break;
        if (lane == 0) mbar_arrive_expect_tx(smem_u32(&mt.kv_full), S::kTile);
        gather_rows4<DP>(sb + (values ? S::kV : S::kK), tm, &mt.kv_full, lane * 4, rows[0], rows[1],
                         rows[2], rows[3]);
        __syncwarp();
      }
    } else {
      const bool grads = warp >= 13;
      const CUtensorMap* tm = grads ? &tm_do : &tm_q;
      const int mine = ((warp - 11) & 1) * 64, row0 = mine + (lane & 15) * 4, blk = lane >> 4;
      const int32_t* src = (grads ? do_row : q_row) + row0;
      const uint32_t dst = sb + (grads ? S::kDo : S::kQ) + blk * (128 * kSub) + row0 * 128;
      uint32_t item = 0;
      int4 ahead;
      float lse[2], delta[2];
      int pos[2];
      auto fetch = [&](const SegIter& s, int step) {
        const int64_t first = static_cast<int64_t>(s.tile.row0) + static_cast<int64_t>(step) * kSub;
        ahead = __ldg(reinterpret_cast<const int4*>(src + first));
        if (grads) return;
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const int64_t at = first + mine + x * 32 + lane;
          lse[x] = __ldg(row_lse + at) - Range<T>::kShift, delta[x] = __ldg(row_delta + at), pos[x] = __ldg(row_pos + at);
        }
      };
      if (it.valid()) fetch(it, it.step);
      int step = it.valid() ? it.step : 0;
      while (it.valid()) {
        const int4 rows = ahead;
        const float l[2] = {lse[0], lse[1]}, d[2] = {delta[0], delta[1]};
        const int p[2] = {pos[0], pos[1]};
        if (++step == it.end) {
          it.advance();
          if (it.valid()) step = it.step;
        }
        if (it.valid()) fetch(it, step);
        const int st = item & 1;
        ok = warp_mbar_wait(&mt.q_free[st], ((item >> 1) & 1) ^ 1, abort);
        if (!ok) break;
        if (!grads) {
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const int at = mine + x * 32 + lane;
            mt.lse[st][at] = l[x], mt.delta[st][at] = d[x], mt.pos[st][at] = p[x];
          }
        }
        if (lane == 0)
          mbar_arrive_expect_tx(smem_u32(&mt.q_full[st]), S::kTile / 2);
        else if (!grads)
          mbar_arrive(smem_u32(&mt.q_full[st]));
        if (blk < DP / 64)
          tma_gather4(dst + st * S::kTile, tm, smem_u32(&mt.q_full[st]), blk * 64, rows.x, rows.y, rows.z,
                      rows.w);
        __syncwarp();
        ++item;
      }
    }
    if (!ok) give_up(abort, err, kErrDkvLoad);
    if (!ok || *abort) {  // copies in flight end before the CTA does
      const uint64_t t0 = globaltimer_ns();
      while (globaltimer_ns() - t0 < 1000000ull) {
      }
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == 8) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// The key tiles that shares cut: the CTA whose share holds a tile's first step, but not its
// last, adds the sums of the CTAs that hold the others, in their order. blockIdx.y: 4 keys.
template <typename T, int DP>
__global__ void __launch_bounds__(256) tiles_dkv_join_kernel(Args a, const KeyTile* __restrict__ tiles,
                                                             const int64_t* __restrict__ share,
                                                             const int32_t* __restrict__ start, int ctas,
                                                             const float* __restrict__ part,
                                                             const float* __restrict__ largest,
                                                             T* __restrict__ dk, T* __restrict__ dv) {
  pdl_wait();
  const int j = blockIdx.x;
  const int64_t from = share[j], to = share[j + 1];
  if (from >= to) return;
  // the share's last tile: the one in which the next share that is not empty begins
  int next = j + 1;
  while (next < ctas && share[next] >= share[next + 1]) ++next;
  if (next >= ctas) return;
  const KeyTile t = load_tile(tiles + __ldg(start + next));
  if (t.base >= to || t.base < from) return;  // it begins with the next share, or began before
  const int64_t end = t.base + t.steps();
  for (int e = threadIdx.x; e < 2 * 4 * DP / 4; e += 256) {
    const int which = e / (4 * DP / 4), key = blockIdx.y * 4 + e / (DP / 4) % 4, d = e % (DP / 4) * 4;
    if (key >= t.keys || d >= a.D) continue;
    const int k = a.order[static_cast<int64_t>(t.r) * a.N + t.s0 + key];
    if (k < 0 || k >= a.N) continue;
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int q = j; q < ctas && share[q] < end; ++q) {
      if (share[q] >= share[q + 1]) continue;
      const float4 v = *reinterpret_cast<const float4*>(
          part + ((static_cast<int64_t>(q) * 2 + (q == j)) * 2 + which) * (kSub * DP) + key * DP + d);
      s.x += v.x, s.y += v.y, s.z += v.z, s.w += v.w;
    }
    const float pw = Range<T>::kNarrow ? power(largest[t.r]) : 1.f;
    const float scale = which == 0 ? Range<T>::unshift() : a.scale * inverse_power(pw);
    const int b = t.r / a.Hkv, hk = t.r - b * a.Hkv;
    T* out = (which == 0 ? dv : dk) + ((static_cast<int64_t>(b) * a.Hkv + hk) * a.N + k) * a.D + d;
    *reinterpret_cast<uint2*>(out) = make_uint2(mma::pack2<T>(s.x * scale, s.y * scale), mma::pack2<T>(s.z * scale, s.w * scale));
  }
}

struct GradLayout {
  UnitPlan plan;
  size_t part, first, tiles, share, start, dkv_part, total;
};

GradLayout grad_layout(const Args& a, uint8_t* ws) {
  GradLayout l{};
  const int64_t R = static_cast<int64_t>(a.batch) * a.Hkv;
  const int64_t DP = a.D <= 64 ? 64 : 128;
  size_t at = carve_units(a, a.Nq, true, ws, &l.plan);
  auto take = [&](int64_t bytes) {
    const size_t p = at;
    at += align_up(static_cast<size_t>(bytes), 256);
    return p;
  };
  l.part = take(l.plan.units_max * kUnitRows * DP * kPartBytes);
  l.first = take(R * 16);
  l.tiles = take(R * row_tiles_max(a.K, a.N) * static_cast<int64_t>(sizeof(KeyTile)));
  l.share = take((kMaxCtas + 1) * 8);
  l.start = take(kMaxCtas * 4);
  l.dkv_part = take(static_cast<int64_t>(std::min(sm_count(), kMaxCtas)) * 4 * kSub * DP * 4);
  l.total = at;
  return l;
}

template <typename T, int DP>
int grad_typed(const Args& a, int dtype, const float* lse, float* delta, const T* dout, T* dq, T* dk,
               T* dv, uint8_t* ws, cudaStream_t stream) {
  const GradLayout l = grad_layout(a, ws);
  const int64_t R = static_cast<int64_t>(a.batch) * a.Hkv;
  CUtensorMap tm_q, tm_k, tm_v, tm_do;
  RowMap rq, rk, rv, rdo;
  const Strides flat{static_cast<int64_t>(a.Hq) * a.Nq * a.D, static_cast<int64_t>(a.Nq) * a.D, a.D};
  FKC_TRY(encode_rows(a.q, a.qs, a.batch, a.Hq, a.Nq, a.D, dtype, &tm_q, &rq));
  FKC_TRY(encode_rows(a.k, a.ks, a.batch, a.Hkv, a.N, a.D, dtype, &tm_k, &rk));
  FKC_TRY(encode_rows(a.v, a.vs, a.batch, a.Hkv, a.N, a.D, dtype, &tm_v, &rv));
  FKC_TRY(encode_rows(dout, flat, a.batch, a.Hq, a.Nq, a.D, dtype, &tm_do, &rdo));
  const int ctas = static_cast<int>(std::min<int64_t>(std::min(sm_count(), kMaxCtas), l.plan.units_max));
  FKC_TRY(launch_units(a, 0, a.Nq, rq, l.plan, ctas, lse, stream));
  int32_t* odd = l.plan.odd;
  const int32_t *q_row = l.plan.q_row, *do_row = l.plan.do_row, *pos = l.plan.row_pos;
  const float *row_lse = l.plan.row_lse, *row_delta = l.plan.row_delta;
  auto walk = [&](auto kern) -> int {
    const int smem = static_cast<int>(DqSmem<DP>::kBytes);
    FKC_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    return launch_pdl(kern, dim3(ctas), dim3(kGradThreads), smem, stream, tm_q, tm_k, tm_v, tm_do, rk, rv, a,
                       q_row, do_row, pos, row_lse, row_delta, static_cast<const float*>(l.plan.row_power),
                      static_cast<const Unit*>(l.plan.units), static_cast<const int32_t*>(l.plan.start), ws + l.part, l.plan.units_max,
                      device_error_word());
  };
  FKC_TRY(walk(tiles_dq_kernel<T, DP, true>));
  const int64_t rows = R * a.Nq * a.G;
  FKC_TRY(launch_pdl(tiles_delta_join_kernel<T>, dim3(static_cast<unsigned>((rows + 255) / 256)), dim3(256), 0, stream, a,
                     static_cast<const int32_t*>(l.plan.pair_row), reinterpret_cast<const float2*>(ws + l.part),
                     l.plan.units_max, delta, l.plan.row_delta, l.plan.row_power, l.plan.largest, rows));
  if (dq != nullptr) {
    FKC_TRY(walk(tiles_dq_kernel<T, DP, false>));
    const int gp = join_heads(a.G), chunks = (a.G + gp - 1) / gp;
    const int64_t warps = R * a.Nq * chunks;
    FKC_TRY(launch_pdl(tiles_dq_join_kernel<T, DP>, dim3(static_cast<unsigned>((warps + 7) / 8)), dim3(256), 0,
                       stream, a, gp, chunks, static_cast<const int32_t*>(l.plan.pair_row),
                       static_cast<const uint8_t*>(ws + l.part), dq, odd, warps));
  }
  if (dk == nullptr)
    return launch_again(a, dtype, odd, lse, delta, dout, dq, nullptr, nullptr, nullptr, nullptr, stream);
  const size_t bytes = static_cast<size_t>(R) * a.N * a.D * sizeof(T);
  FKC_TRY(launch_zero_fill(dk, bytes, stream));
  FKC_TRY(launch_zero_fill(dv, bytes, stream));
  int64_t* first = reinterpret_cast<int64_t*>(ws + l.first);
  int64_t* share = reinterpret_cast<int64_t*>(ws + l.share);
  KeyTile* tiles = reinterpret_cast<KeyTile*>(ws + l.tiles);
  int32_t* start = reinterpret_cast<int32_t*>(ws + l.start);
  float* part = reinterpret_cast<float*>(ws + l.dkv_part);
  const int shares = std::min(sm_count(), kMaxCtas);
  const int32_t* inv = l.plan.inv_offsets;
  FKC_TRY(launch_pdl(key_count_kernel, dim3(static_cast<unsigned>(R)), dim3(1024), 0, stream, a, inv, first));
  FKC_TRY(launch_pdl(key_tiles_kernel, dim3(static_cast<unsigned>(R)), dim3(1024), 0, stream, a, inv,
                     static_cast<const int32_t*>(l.plan.first_unit), static_cast<const int64_t*>(first), tiles,
                     share, start, shares, static_cast<int>(R)));
  auto kern = tiles_dkv_kernel<T, DP>;
  const int smem = static_cast<int>(DkvSmem<DP>::kBytes);
  FKC_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  FKC_TRY(launch_pdl(kern, dim3(shares), dim3(kGradThreads), smem, stream, tm_q, tm_k, tm_v, tm_do, rk, rv, a,
                     q_row, do_row, pos, row_lse, row_delta, static_cast<const KeyTile*>(tiles),
                     static_cast<const int64_t*>(share), static_cast<const int32_t*>(start),
                     static_cast<const float*>(l.plan.largest), dk, dv, part, odd, device_error_word()));
  FKC_TRY(launch_pdl(tiles_dkv_join_kernel<T, DP>, dim3(shares, kSub / 4), dim3(256), 0, stream, a,
                     static_cast<const KeyTile*>(tiles), static_cast<const int64_t*>(share),
                     static_cast<const int32_t*>(start), shares, static_cast<const float*>(part),
                     static_cast<const float*>(l.plan.largest), dk, dv));
  return launch_again(a, dtype, odd, lse, delta, dout, dq, l.plan.inv_order, inv, dk, dv, stream);
}

template <typename T>
int grad_dtype(const Args& a, int dtype, const float* lse, float* delta, const void* dout, void* dq,
               void* dk, void* dv, uint8_t* ws, cudaStream_t stream) {
  const T* d = static_cast<const T*>(dout);
  T *q = static_cast<T*>(dq), *k = static_cast<T*>(dk), *v = static_cast<T*>(dv);
  return a.D <= 64 ? grad_typed<T, 64>(a, dtype, lse, delta, d, q, k, v, ws, stream)
                   : grad_typed<T, 128>(a, dtype, lse, delta, d, q, k, v, ws, stream);
}

}  // namespace

// In us, as use_tiles, fitted to the gradients of the same calls (the walk within 16% on average, this form
// within 9%): the form that it chooses took 1.8% longer on average than the faster one. The
// walk's chains: a warp's key tiles, twice, and a CTA's columns. Measured (walk, by clusters), the
// gradients alone, D = 128 but for the last two:
// G 1, 171 queries x 2 rows, 16 of 256 clusters of 24 keys: 95, 98; 348 x 2, 16 of 128 of 24: 94, 80. G 4,
// 409 x 4, 8 of 256 of 32: 156, 142. G 32, 190 x 2, 16 of 128 of 16: 177, 195; 3296 x 1, 3 of 16 of 8:
// 1906, 273. D = 64: G 4, 1297 x 8, 2 of 32 of 24: 90, 117; 2356 x 4, 3 of 32 of 24: 153, 134.
bool use_tiles_grad(const Args& a) {
  if (!tiles_fit(a, a.Nq, 1ll << 33)) return false;  // all queries at once
  const FormWork w = form_work(a, a.Nq);
  const double columns = static_cast<double>(a.Nq) * a.top * a.G / a.K;  // of a cluster
  const double walk = 35.7 + 107.6e-6 * w.reads * w.width + 1.27 * a.top * w.keys / 16 + 1.85 * columns / 32 +
                      575e-6 * w.rows * (w.keys / 64 + 0.5) * w.width;
  const double tiles = 63.9 + w.units * (0.0274 + 0.000535 * w.keys * w.width) + w.rows * (165e-6 + 326e-6 * w.width);
  return tiles < walk;
}

size_t tiles_backward_workspace_bytes(const Args& a) { return grad_layout(a, nullptr).total; }

int launch_tiles_backward(const Args& a, int dtype, const float* lse, float* delta, const void* dout,
                          void* dq, void* dk, void* dv, void* ws, cudaStream_t stream) {
  uint8_t* w = static_cast<uint8_t*>(ws);
  return dtype == FKC_DTYPE_F16
             ? grad_dtype<__half>(a, dtype, lse, delta, dout, dq, dk, dv, w, stream)
             : grad_dtype<__nv_bfloat16>(a, dtype, lse, delta, dout, dq, dk, dv, w, stream);
}

}  // namespace attn
}  // namespace fkc
