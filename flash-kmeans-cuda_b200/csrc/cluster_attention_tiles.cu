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
// tiles_fwd_kernel is persistent, one CTA per SM, over units of 256 rows (two MMAs of 128)
// of one cluster: TMA row gathers (four rows an instruction) fetch Q, and the cluster's keys and
// values in steps of 128; one
// thread issues S = Q K^T (tcgen05, both operands in shared memory) and O += P V (P from
// TMEM, V as MN-major operand) into TMEM; two warpgroups turn S into P in place, a thread a
// row, with the running maximum and sum in fp32, and write O out. P is rounded to the 16-bit
// input type for the second product, as its operand type demands.
#include <algorithm>
#include <numeric>

#include "cluster_attention.cuh"
#include "cluster_tiles.cuh"

namespace fkc {
namespace attn {
namespace {

// Appends the units of row r. Which place they get is up to the order of the rows' claims;
// what a unit computes and writes does not depend on it.
__global__ void __launch_bounds__(1024) tile_units_kernel(Args a,
                                                          const int32_t* __restrict__ inv_offsets,
                                                          Unit* __restrict__ units, int32_t* count,
                                                          int units_max) {
  constexpr int rows = kUnitRows;
  __shared__ int warp_total[32];
  __shared__ int first;
  pdl_wait();
  const int r = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int32_t* of = inv_offsets + static_cast<int64_t>(r) * (a.K + 1);
  for (int c0 = 0; c0 < a.K; c0 += 1024) {
    const int c = c0 + threadIdx.x;
    int s0 = 0, s1 = 0, e0 = 0;
    int64_t all = 0;
    if (c < a.K) {
      cluster_span(a, r, c, s0, s1);
      e0 = of[c];
      if (s1 > s0) all = static_cast<int64_t>(of[c + 1] - e0) * a.G;
    }
    const int n = static_cast<int>((all + rows - 1) / rows);
    int inc = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xFFFFFFFFu, inc, o);
      if (lane >= o) inc += u;
    }
    __syncthreads();
    if (lane == 31) warp_total[warp] = inc;
    __syncthreads();
    int at = inc - n, sum = 0;
    for (int w = 0; w < 32; ++w) {
      if (w < warp) at += warp_total[w];
      sum += warp_total[w];
    }
    if (threadIdx.x == 0) first = atomicAdd(count, sum);
    __syncthreads();
    at += first;
    for (int t = 0; t < n; ++t)
      if (at + t < units_max)  // always, with the workspace of carve_units
        units[at + t] = Unit{c, t * rows, s0, s1, e0, static_cast<int>(min(static_cast<int64_t>(rows), all - static_cast<int64_t>(t) * rows)), r, 0};
  }
}

// The rows of the units, one warp a unit: a lane takes rows lane + 32 j.
__global__ void __launch_bounds__(256) tile_rows_kernel(Args a, int i0, int nq, RowMap rq,
                                                        const int32_t* __restrict__ inv_order,
                                                        Unit* __restrict__ units,
                                                        const int32_t* __restrict__ count,
                                                        int32_t* __restrict__ q_row,
                                                        int2* __restrict__ slot_pos) {
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int64_t u = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  if (u >= *count) return;
  const Unit un = units[u];
  const int b = un.r / a.Hkv, hk = un.r - b * a.Hkv;
  const int32_t* list = inv_order + static_cast<int64_t>(un.r) * nq * a.top + un.e0;
  int high = -1;
#pragma unroll
  for (int j = 0; j < kUnitRows / 32; ++j) {
    const int rr = j * 32 + lane;
    int slot = -1, pos = -1, row = rq.rows;
    if (rr < un.nrows) {
      const int at = un.row0 + rr, e = at / a.G, h = at - e * a.G;
      const int p = list[e], i = i0 + p / a.top;
      slot = p * a.G + h;
      pos = max(-1, min(a.q_pos != nullptr ? a.q_pos[static_cast<int64_t>(b) * a.Nq + i] : a.N, a.N));
      if (pos >= 0) row = rq.at(b, hk * a.G + h, i);
    }
    q_row[u * kUnitRows + rr] = row;
    slot_pos[u * kUnitRows + rr] = make_int2(slot, pos);
    high = max(high, pos);
  }
  high = __reduce_max_sync(0xFFFFFFFFu, high);
  if (lane == 0) units[u].high = high;
}

// Shared memory of the forward kernel: operand tiles (1024-byte aligned), then the rest.
template <int DP>
struct FwdSmem {
  static constexpr uint32_t kTile = tc_tile_bytes<DP>();
  static constexpr uint32_t kQ = 0;              // one tile per 128 rows
  static constexpr uint32_t kK = 2 * kTile;      // two stages
  static constexpr uint32_t kV = 4 * kTile;      // two stages
  static constexpr uint32_t kMeta = 6 * kTile;
  struct Meta {
    int32_t key[2][kKeysStep]; // positions of a stage's keys; INT_MAX behind the last
    uint64_t k_full[2], v_full[2], kv_free[2], q_full[2], q_free[2];
    uint64_t s_full[2], p_full[2], o_full[2], o_free[2];
    uint64_t drain;
    uint32_t tmem;
    int abort;
  };
  static constexpr uint32_t kBytes = kMeta + sizeof(Meta) + 1024;
};

enum : int { kErrLoad = 151, kErrMma = 152, kErrSoftmax = 153 };

// Warps 0-3 and 4-7: softmax and output of rows 0-127 and 128-255 of a unit (a thread a
// row); warp 8: the MMAs; warps 9, 10: gathers of keys and of values; 11, 12: of Q.
constexpr int kFwdThreads = 32 * 13;

// The steps of a CTA's units in turn, the next unit always fetched ahead.
struct StepIter {
  const Unit* units;
  int n, total, stride, step;
  Unit un, next;
  __device__ __forceinline__ StepIter(const Unit* u, int first, int count, int str)
      : units(u), n(first), total(count), stride(str), step(0) {
    if (n < total) un = load_unit(units + n);
    if (n + stride < total) next = load_unit(units + n + stride);
  }
  __device__ __forceinline__ bool valid() const { return n < total; }
  __device__ __forceinline__ void advance() {
    if (++step < un.steps()) return;
    next_unit();
  }
  __device__ __forceinline__ void next_unit() {
    step = 0;
    n += stride;
    un = next;
    if (n + stride < total) next = load_unit(units + n + stride);
  }
};

template <typename T, int DP>
__global__ void __launch_bounds__(kFwdThreads, 1) tiles_fwd_kernel(
    const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
    const __grid_constant__ CUtensorMap tm_v, RowMap rq, RowMap rk, RowMap rv, Args a, int i0, int nq,
    const int32_t* __restrict__ q_row, const int2* __restrict__ slot_pos,
    const Unit* __restrict__ units, const int32_t* __restrict__ count, float* __restrict__ part_o,
    float* __restrict__ part_lse, int* err) {
  using namespace ptx;
  using S = FwdSmem<DP>;
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
      mbar_init(smem_u32(&mt.q_full[x]), 1);
      mbar_init(smem_u32(&mt.kv_free[x]), 1);
      mbar_init(smem_u32(&mt.q_free[x]), 1);
      mbar_init(smem_u32(&mt.s_full[x]), 1);
      mbar_init(smem_u32(&mt.p_full[x]), 128);
      mbar_init(smem_u32(&mt.o_full[x]), 1);
      mbar_init(smem_u32(&mt.o_free[x]), 128);
    }
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
  const uint32_t tmem = mt.tmem;  // sub-tile x: S (then P) at 256 x, O at 256 x + 128
  pdl_wait();
  const int total = *count;
  const int stride = gridDim.x;

  if (warp < 8) {
    // ------------------------------------------------------------ softmax, output
    const int sub = warp >> 2, row = (warp & 3) * 32 + lane;
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t t_s = tmem + lanes + sub * 256, t_o = t_s + 128;
    const float sc = a.scale * kLog2e;
    uint32_t item = 0, uses = 0, s_uses = 0;
    bool ok = true;
    StepIter it(units, blockIdx.x, total, stride);
    const int2* meta = slot_pos + sub * kSub + row;
    int2 ahead = it.valid() ? __ldg(meta + static_cast<int64_t>(it.n) * kUnitRows) : make_int2(-1, -1);
    for (; ok && it.valid(); it.next_unit()) {
      const Unit& un = it.un;
      const int steps = un.steps();
      const int slot = ahead.x, pos = ahead.y;
      if (it.n + stride < total) ahead = __ldg(meta + static_cast<int64_t>(it.n + stride) * kUnitRows);
      if (un.nrows <= sub * kSub) {
        item += steps;
        continue;
      }
      const int pos_min = __reduce_min_sync(0xFFFFFFFFu, slot < 0 ? INT_MAX : pos);
      float m = -INFINITY, l = 0.f;
      for (int step = 0; step < steps; ++step, ++item, ++s_uses) {
        const int st = item & 1;
        ok = warp_mbar_wait(&mt.k_full[st], (item >> 1) & 1, abort) &&
             warp_mbar_wait(&mt.s_full[sub], s_uses & 1, abort);
        if (!ok) {
          give_up(abort, err, kErrSoftmax);
          break;
        }
        tc_fence_after();
        const int keys = un.keys(step);
        const int32_t* key = mt.key[st];
        float tops[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
        uint32_t open = 0;  // 32-key chunks that every row of the warp sees whole
#pragma unroll
        for (int c = 0; c < kKeysStep / 32; ++c) {
          if (c * 32 >= keys) break;
          uint32_t s[32];
          tmem_ld_32x32b_x32(t_s + c * 32, s);
          const bool whole = __reduce_max_sync(0xFFFFFFFFu, key[c * 32 + lane]) <= pos_min;
          tmem_wait_ld();
          if (whole) {
            open |= 1u << c;
#pragma unroll
            for (int j = 0; j < 32; ++j) tops[j & 3] = fmaxf(tops[j & 3], __uint_as_float(s[j]));
          } else {
#pragma unroll
            for (int j = 0; j < 32; j += 4) {
              const int4 k4 = *reinterpret_cast<const int4*>(key + c * 32 + j);
              tops[0] = fmaxf(tops[0], k4.x <= pos ? __uint_as_float(s[j]) : -INFINITY);
              tops[1] = fmaxf(tops[1], k4.y <= pos ? __uint_as_float(s[j + 1]) : -INFINITY);
              tops[2] = fmaxf(tops[2], k4.z <= pos ? __uint_as_float(s[j + 2]) : -INFINITY);
              tops[3] = fmaxf(tops[3], k4.w <= pos ? __uint_as_float(s[j + 3]) : -INFINITY);
            }
          }
        }
        const float top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
        const float mn = fmaxf(m, top * sc);  // the scale is positive
        const float from = mn == -INFINITY ? 0.f : mn;
        const float alpha = ex2(m - from);
        m = mn;
        if (step > 0 && __any_sync(0xFFFFFFFFu, alpha != 1.f)) {
          // the product of the step before has ended: its commit came before this S's
#pragma unroll
          for (int c = 0; c < DP / 32; ++c) {
            uint32_t o[32];
            tmem_ld_32x32b_x32(t_o + c * 32, o);
            tmem_wait_ld();
#pragma unroll
            for (int j = 0; j < 32; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * alpha);
            tmem_st_32x32b_x32(t_o + c * 32, o);
          }
        }
        float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < kKeysStep / 32; ++c) {
          if (c * 32 >= keys) break;
          uint32_t s[32], p[16];
          tmem_ld_32x32b_x32(t_s + c * 32, s);
          tmem_wait_ld();
          if (open >> c & 1u) {
#pragma unroll
            for (int j = 0; j < 32; ++j)
              s[j] = __float_as_uint(ex2(fmaf(__uint_as_float(s[j]), sc, -from)));
          } else {
#pragma unroll
            for (int j = 0; j < 32; j += 4) {
              const int4 k4 = *reinterpret_cast<const int4*>(key + c * 32 + j);
              const int k[4] = {k4.x, k4.y, k4.z, k4.w};
#pragma unroll
              for (int e = 0; e < 4; ++e)
                s[j + e] = __float_as_uint(
                    ex2(k[e] <= pos ? fmaf(__uint_as_float(s[j + e]), sc, -from) : -INFINITY));
            }
          }
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            const float p0 = __uint_as_float(s[2 * j]), p1 = __uint_as_float(s[2 * j + 1]);
            sum[(2 * j) & 3] += p0;
            sum[(2 * j + 1) & 3] += p1;
            p[j] = mma::pack2<T>(p0, p1);
          }
          tmem_st_32x32b_x16(t_s + c * 16, p);  // over scores that are read already
        }
        l = l * alpha + ((sum[0] + sum[1]) + (sum[2] + sum[3]));
        tmem_wait_st();
        tc_fence_before();
        mbar_arrive(smem_u32(&mt.p_full[sub]));
      }
      if (!ok) break;
      ok = warp_mbar_wait(&mt.o_full[sub], uses & 1, abort);
      if (!ok) {
        give_up(abort, err, kErrSoftmax);
        break;
      }
      tc_fence_after();
      const float inv = l == 0.f ? 0.f : 1.f / l;
      const int64_t at = static_cast<int64_t>(un.r) * nq * a.top * a.G + slot;
      float* out = part_o + at * a.D;
#pragma unroll
      for (int c = 0; c < DP / 32; ++c) {
        uint32_t o[32];
        tmem_ld_32x32b_x32(t_o + c * 32, o);
        tmem_wait_ld();
#pragma unroll
        for (int j = 0; j < 32; j += 8) {
          float v[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] = __uint_as_float(o[j + e]) * inv;
          if (slot >= 0 && c * 32 + j < a.D) st_global_v8(out + c * 32 + j, v);
        }
        __syncwarp();
      }
      if (slot >= 0) part_lse[at] = l == 0.f ? -INFINITY : m + log2f(l);
      tc_fence_before();
      mbar_arrive(smem_u32(&mt.o_free[sub]));
      ++uses;
    }
  } else if (warp == 8) {
    // ------------------------------------------------------------ MMAs (one thread)
    if (lane == 0) {
      const int dsteps = (a.D + 15) / 16;
      constexpr uint32_t idesc_o = umma_idesc_f16(kBf16, kSub, DP) | kIdescMnB;
      uint32_t item = 0, q_uses[2] = {0, 0}, p_uses[2] = {0, 0};
      struct Pending {
        bool has, first, last;
        int stage, ksteps;
        uint32_t parity;  // of the stage's values
      } pend[2] = {};
      bool ok = true;
      auto product = [&](int sub) {  // O (+)= P V of the pending step
        Pending& p = pend[sub];
        if (!p.has) return;
        p.has = false;
        ok = ok && mbar_wait(smem_u32(&mt.p_full[sub]), p_uses[sub] & 1, abort);
        ++p_uses[sub];
        // the output of the use before: q_uses counts the S of this one already
        if (ok && p.first) ok = mbar_wait(smem_u32(&mt.o_free[sub]), q_uses[sub] & 1, abort);
        ok = ok && mbar_wait(smem_u32(&mt.v_full[p.stage]), p.parity, abort);
        if (!ok) return;
        tc_fence_after();
        mma_tmem_rows(tmem + sub * 256 + 128, tmem + sub * 256, sb + S::kV + p.stage * S::kTile,
                      idesc_o, p.ksteps, p.first);
        if (p.last) umma_commit(smem_u32(&mt.o_full[sub]));
      };
      for (StepIter it(units, blockIdx.x, total, stride); ok && it.valid(); it.next_unit()) {
        const Unit& un = it.un;
        const int steps = un.steps();
        for (int step = 0; ok && step < steps; ++step, ++item) {
          const int st = item & 1;
          const int k16 = (un.keys(step) + 15) / 16;
          const uint32_t idesc_s = umma_idesc_f16(kBf16, kSub, 16 * k16);
          for (int sub = 0; sub < 2; ++sub) {
            product(sub);
            if (!ok || un.nrows <= sub * kSub) continue;
            ok = mbar_wait(smem_u32(&mt.k_full[st]), (item >> 1) & 1, abort);
            if (ok && step == 0) {
              ok = mbar_wait(smem_u32(&mt.q_full[sub]), q_uses[sub] & 1, abort);
              ++q_uses[sub];
            }
            if (!ok) break;
            mma_kmajor<DP>(tmem + sub * 256, sb + S::kQ + sub * S::kTile, sb + S::kK + st * S::kTile,
                           idesc_s, dsteps);
            umma_commit(smem_u32(&mt.s_full[sub]));
            if (step == steps - 1) umma_commit(smem_u32(&mt.q_free[sub]));
            pend[sub] = {true, step == 0, step == steps - 1, st, k16, (item >> 1) & 1};
          }
          if (ok && item > 0) umma_commit(smem_u32(&mt.kv_free[st ^ 1]));
        }
      }
      for (int sub = 0; sub < 2; ++sub)
        if (ok) product(sub);
      if (!ok) give_up(abort, err, kErrMma);
      umma_commit(smem_u32(&mt.drain));  // nothing is in flight when TMEM is freed
      const int never = 0;
      mbar_wait(smem_u32(&mt.drain), 0, &never);
    }
  } else {
    // ------------------------------------------------------------ gathers
    // The next step's (or unit's) row numbers are fetched while this one's copies run.
    bool ok = true;
    if (warp <= 10) {
      const bool values = warp == 10;
      const CUtensorMap* tm = values ? &tm_v : &tm_k;
      const RowMap rm = values ? rv : rk;
      const uint32_t tiles = sb + (values ? S::kV : S::kK);
      StepIter it(units, blockIdx.x, total, stride);
      auto fetch = [&](int (&idx)[4]) {  // positions of keys 4 lane .. of the step
        const int32_t* order = a.order + static_cast<int64_t>(it.un.r) * a.N;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int s = it.un.s0 + it.step * kKeysStep + lane * 4 + j;
          const int row = s < it.un.s1 ? __ldg(order + s) : -1;
          idx[j] = row >= 0 && row < a.N ? row : INT_MAX;
        }
      };
      int idx[4];
      if (it.valid()) fetch(idx);
      for (uint32_t item = 0; it.valid(); ++item) {
        const int st = item & 1;
        const int b = it.un.r / a.Hkv, hk = it.un.r - b * a.Hkv;
        const int quads = (it.un.keys(it.step) + 15) / 16 * 4;
        int rows[4];
#pragma unroll
        for (int j = 0; j < 4; ++j)  // a key that no row sees is not read
          rows[j] = idx[j] <= it.un.high ? rm.at(b, hk, idx[j]) : rm.rows;
        const int4 key = make_int4(idx[0], idx[1], idx[2], idx[3]);
        it.advance();
        if (it.valid()) fetch(idx);
        ok = warp_mbar_wait(&mt.kv_free[st], ((item >> 1) & 1) ^ 1, abort);
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
      const int sub = warp - 11;
      const int4* src = reinterpret_cast<const int4*>(q_row) + sub * (kSub / 4) + lane;
      StepIter it(units, blockIdx.x, total, stride);
      int4 ahead = it.valid() ? __ldg(src + static_cast<int64_t>(it.n) * (kUnitRows / 4)) : make_int4(0, 0, 0, 0);
      uint32_t uses = 0;
      for (; it.valid(); it.next_unit()) {
        const int4 rows = ahead;
        if (it.n + stride < total) ahead = __ldg(src + static_cast<int64_t>(it.n + stride) * (kUnitRows / 4));
        if (it.un.nrows <= sub * kSub) continue;
        ok = warp_mbar_wait(&mt.q_free[sub], (uses & 1) ^ 1, abort);
        if (!ok) break;
        if (lane == 0) mbar_arrive_expect_tx(smem_u32(&mt.q_full[sub]), S::kTile);
        gather_rows4<DP>(sb + S::kQ + sub * S::kTile, &tm_q, &mt.q_full[sub], lane * 4, rows.x, rows.y,
                         rows.z, rows.w);
        __syncwarp();
        ++uses;
      }
    }
    if (!ok) give_up(abort, err, kErrLoad);
    // copies in flight end before the CTA does: the MMA warp waits for all of them, and
    // after a wait that gave up they are waited for here
    if (!ok || *abort) {
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
  uint32_t has = 0;  // bit s of lane l: slot 32 s + l has a part
  for (int s0 = 0; s0 < a.top; s0 += 32) {
    const int s = s0 + lane;
    int from = 0, to = 0;
    if (s < a.top) cluster_span(a, r, sel[s], from, to);
    if (to > from) {
      has |= 1u << (s0 >> 5);
      top = fmaxf(top, pl[static_cast<int64_t>(s) * a.G]);
    }
  }
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
  const float from = top == -INFINITY ? 0.f : top;
  float acc[4] = {0.f, 0.f, 0.f, 0.f}, sum = 0.f;
  const bool on = lane * 4 < a.D;
  constexpr int kAhead = 8;  // parts in flight
  for (int s0 = 0; s0 < a.top; s0 += kAhead) {
    float4 v[kAhead];
    float w[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int s = s0 + u;
      const bool part = s < a.top && (__shfl_sync(0xFFFFFFFFu, has, s & 31) >> (s >> 5) & 1u);
      w[u] = part ? pl[static_cast<int64_t>(s) * a.G] : -INFINITY;
      v[u] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (part && on)
        v[u] = __ldcs(reinterpret_cast<const float4*>(po + static_cast<int64_t>(s) * a.G * a.D + lane * 4));
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      if (w[u] == -INFINITY) continue;  // sees nothing of this cluster
      const float e = exp2f(w[u] - from);
      sum += e;
      acc[0] += e * v[u].x;
      acc[1] += e * v[u].y;
      acc[2] += e * v[u].z;
      acc[3] += e * v[u].w;
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
  UnitPlan plan;
  size_t part_lse, part_o, total;
  int64_t nq;
};

Layout fwd_layout(const Args& a, uint8_t* ws) {
  Layout l{};
  const int64_t R = static_cast<int64_t>(a.batch) * a.Hkv;
  l.nq = queries_per_round(a);
  size_t at = carve_units(a, l.nq, ws, &l.plan);
  auto take = [&](int64_t bytes) {
    const size_t p = at;
    at += align_up(static_cast<size_t>(bytes), 256);
    return p;
  };
  l.part_lse = take(R * l.nq * a.top * a.G * 4);
  l.part_o = take(R * l.nq * a.top * a.G * a.D * 4);
  l.total = at;
  return l;
}

template <typename T, int DP>
int fwd_typed(const Args& a, int dtype, T* out, float* lse, uint8_t* ws, cudaStream_t stream) {
  const Layout l = fwd_layout(a, ws);
  const int64_t R = static_cast<int64_t>(a.batch) * a.Hkv;
  float* part_lse = reinterpret_cast<float*>(ws + l.part_lse);
  float* part_o = reinterpret_cast<float*>(ws + l.part_o);
  CUtensorMap tm_q, tm_k, tm_v;
  RowMap rq, rk, rv;
  FKC_TRY(encode_rows(a.q, a.qs, a.batch, a.Hq, a.Nq, a.D, dtype, &tm_q, &rq));
  FKC_TRY(encode_rows(a.k, a.ks, a.batch, a.Hkv, a.N, a.D, dtype, &tm_k, &rk));
  FKC_TRY(encode_rows(a.v, a.vs, a.batch, a.Hkv, a.N, a.D, dtype, &tm_v, &rv));
  auto kern = tiles_fwd_kernel<T, DP>;
  const int smem = static_cast<int>(FwdSmem<DP>::kBytes);
  FKC_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  for (int64_t i0 = 0; i0 < a.Nq; i0 += l.nq) {
    const int nq = static_cast<int>(std::min<int64_t>(l.nq, a.Nq - i0));
    FKC_TRY(launch_units(a, i0, nq, rq, l.plan, stream));
    const int64_t grid = std::min<int64_t>(sm_count(), l.plan.units_max);
    FKC_TRY(launch_pdl(kern, dim3(static_cast<unsigned>(grid)), dim3(kFwdThreads), smem, stream, tm_q,
                       tm_k, tm_v, rq, rk, rv, a, static_cast<int>(i0), nq, static_cast<const int32_t*>(l.plan.q_row),
                       static_cast<const int2*>(l.plan.slot_pos),
                       static_cast<const Unit*>(l.plan.units),
                       static_cast<const int32_t*>(l.plan.count), part_o, part_lse,
                       device_error_word()));
    const int64_t rows = R * nq * a.G;
    FKC_TRY(launch_pdl(tiles_join_kernel<T>, dim3(static_cast<unsigned>((rows + 7) / 8)), dim3(256), 0,
                       stream, a, static_cast<int>(i0), nq, static_cast<const float*>(part_o),
                       static_cast<const float*>(part_lse), out, lse, rows));
  }
  return FKC_OK;
}

template <typename T>
int fwd_dtype(const Args& a, int dtype, void* out, float* lse, void* ws, cudaStream_t stream) {
  T* o = static_cast<T*>(out);
  uint8_t* w = static_cast<uint8_t*>(ws);
  return a.D <= 64 ? fwd_typed<T, 64>(a, dtype, o, lse, w, stream)
                   : fwd_typed<T, 128>(a, dtype, o, lse, w, stream);
}

}  // namespace

int sm_count() {
  const DeviceInfo* di = nullptr;
  return current_device_info(&di) == FKC_OK ? di->sm_count : 148;
}

bool row_map(const Strides& s, int64_t nb, int64_t nh, int64_t nn, int64_t D, RowMap* map,
             int64_t* unit) {
  const int64_t u0 = std::gcd(std::gcd(s.b, s.h), s.n);
  const int64_t u = u0 == 0 ? D : u0;
  const int64_t last = ((nb - 1) * s.b + (nh - 1) * s.h + (nn - 1) * s.n) / u;
  if (u < D || last >= 2147483647ll - 1) return false;
  if (map != nullptr) *map = {s.b / u, s.h / u, s.n / u, static_cast<int>(last + 1)};
  if (unit != nullptr) *unit = u;
  return true;
}

int encode_rows(const void* base, const Strides& s, int64_t nb, int64_t nh, int64_t nn, int64_t D,
                int dtype, CUtensorMap* tm, RowMap* map) {
  int64_t unit = 0;
  FKC_REQUIRE(row_map(s, nb, nh, nn, D, map, &unit), "attention: strides without a common unit");
  return encode_tmap_rows(
      tm, dtype == FKC_DTYPE_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16,
      base, static_cast<uint64_t>(D), static_cast<uint64_t>(map->rows),
      static_cast<uint64_t>(unit) * 2);
}

size_t carve_units(const Args& a, int64_t nq, uint8_t* ws, UnitPlan* out) {
  const int64_t R = static_cast<int64_t>(a.batch) * a.Hkv;
  const int64_t pairs = nq * a.top;
  UnitPlan p{};
  // every cluster with pairs may end in a unit that is not full
  p.units_max = R * (pairs * a.G / kUnitRows + std::min<int64_t>(a.K, pairs));
  size_t at = 0;
  auto take = [&](int64_t bytes) -> void* {
    void* q = ws != nullptr ? ws + at : nullptr;
    at += align_up(static_cast<size_t>(bytes), 256);
    return q;
  };
  p.inv_order = static_cast<int32_t*>(take(R * pairs * 4));
  p.inv_offsets = static_cast<int32_t*>(take(R * (a.K + 1) * 4));
  p.units = static_cast<Unit*>(take(p.units_max * static_cast<int64_t>(sizeof(Unit))));
  p.count = static_cast<int32_t*>(take(4));
  p.q_row = static_cast<int32_t*>(take(p.units_max * kUnitRows * 4));
  p.slot_pos = static_cast<int2*>(take(p.units_max * kUnitRows * 8));
  p.group_ws = take(static_cast<int64_t>(group_workspace_bytes(R, pairs, a.K)));
  if (out != nullptr) *out = p;
  return at;
}

int launch_units(const Args& a, int64_t i0, int64_t nq, const RowMap& rq, const UnitPlan& p,
                 cudaStream_t stream) {
  const int64_t R = static_cast<int64_t>(a.batch) * a.Hkv;
  FKC_REQUIRE(p.units_max <= 2147483647ll, "attention: too many tiles");
  FKC_TRY(launch_zero_fill(p.count, 4, stream));
  FKC_TRY(launch_group(a.sel + i0 * a.top, false, static_cast<int64_t>(a.Nq) * a.top, p.inv_order,
                       p.inv_offsets, R, nq * a.top, a.K, p.group_ws, stream));
  FKC_TRY(launch_pdl(tile_units_kernel, dim3(static_cast<unsigned>(R)), dim3(1024), 0, stream, a,
                     static_cast<const int32_t*>(p.inv_offsets), p.units, p.count,
                     static_cast<int>(p.units_max)));
  return launch_pdl(tile_rows_kernel, dim3(static_cast<unsigned>((p.units_max + 7) / 8)), dim3(256), 0,
                    stream, a, static_cast<int>(i0), static_cast<int>(nq), rq,
                    static_cast<const int32_t*>(p.inv_order), p.units,
                    static_cast<const int32_t*>(p.count), p.q_row, p.slot_pos);
}

bool use_tiles(const Args& a) {
  const int64_t R = static_cast<int64_t>(a.batch) * a.Hkv;
  const int64_t per_round = queries_per_round(a) * a.top;
  // rows of a cluster fill half a tile, keys of a cluster repay its parts, and there are
  // enough tiles for the GPU
  // the gathers' maps
  if (!row_map(a.qs, a.batch, a.Hq, a.Nq, a.D, nullptr, nullptr) ||
      !row_map(a.ks, a.batch, a.Hkv, a.N, a.D, nullptr, nullptr) ||
      !row_map(a.vs, a.batch, a.Hkv, a.N, a.D, nullptr, nullptr))
    return false;
  // 32-bit numbers of a row's (pair, head)
  if (queries_per_round(a) * a.top * a.G > (1ll << 30)) return false;
  return a.scale > 0.f && per_round * a.G >= 64ll * a.K && a.N / a.K >= 4 * a.G + 8 &&
         R * a.Nq * a.top * a.G >= 148ll * kSub;
}

size_t tiles_forward_workspace_bytes(const Args& a) { return fwd_layout(a, nullptr).total; }

int launch_tiles_forward(const Args& a, int dtype, void* out, float* lse, void* ws,
                         cudaStream_t stream) {
  return dtype == FKC_DTYPE_F16 ? fwd_dtype<__half>(a, dtype, out, lse, ws, stream)
                                : fwd_dtype<__nv_bfloat16>(a, dtype, out, lse, ws, stream);
}

}  // namespace attn
}  // namespace fkc
