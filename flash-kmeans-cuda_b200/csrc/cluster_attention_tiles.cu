// Attention over selected clusters, cluster by cluster: the form for many queries.
//
// The walk of cluster_attention.cu reads every selected key once per query: 4 * D bytes
// a key for 4 * D * G flops, from L2. Here the queries that selected a cluster are brought
// together instead: sel is grouped by cluster (cluster_group.cu: entry e is query
// e / top), the heads of its queries become the rows of units of 256, and a unit reads the
// cluster's keys once for all of them. A unit leaves, for every (query, slot of sel, head),
// the output over that cluster (a part, three bytes a value) and its log-sum-exp, and tiles_join_kernel
// joins a query's top parts. So the traffic is D * (2 + 3 + 3) bytes per (query, slot, head)
// instead of 4 * D per (query, key): at G = 4 and 64 keys a cluster an eighth.
//
// tiles_fwd_kernel is persistent, one CTA per SM, over shares of the units of equal estimated cost.
// TMA row gathers (four rows an instruction) fetch Q, and the cluster's keys and values in steps
// of 128, which stay for the next unit of the same cluster; one thread issues S = Q K^T (tcgen05,
// both operands in shared memory) and O += P V (P from TMEM, V as MN-major operand) into
// TMEM; two warpgroups turn S into P in place, a thread a row, with the running maximum and sum
// in fp32; two others write O out by bulk copies meanwhile. P enters the second product as two terms
// (cluster_attention.cu), which lie side by side in the columns of S that they came from; that took the
// call below from 551 to 615 us, out's error against 64 bits from 0.0023 of its norm to 0.0017.
//
// At 4096 queries x 8 rows of G = 4, 16 of 256 clusters of 64 keys, D = 128 (2.1 M (query, slot,
// head) rows, 69 GFLOP): the units and rows are listed in 55 us, tiles_fwd_kernel takes 383 us, the
// join 143 us (the call 600 us: each from cold caches alone; the larger of the skewed clusters are
// selected more often, 1779 keys a query instead of 1024, which makes it 119 GFLOP). The kernel is bound by its
// SMs' instruction issue (50% of all slots, softmax and output) and by the gathers, which it waits
// for at the start of every unit; its tensor pipe is busy for 29% of the time and DRAM for near a
// half (1.1 GB: the parts do not fit L2, Q rows come from it). The join moves 824 MB at 5.8 TB/s.
// What was measured on the way, the same call: the walk 3860 us; by clusters with warp-level
// matrix instructions 1250; tcgen05 with operands copied 16 bytes a thread 940, by row gathers
// 900; rows listed beforehand instead of by the gathering warps 740; shares by cost, kept keys,
// 16-bit parts and bulk stores 680; joins of four heads side by side 630; warpgroups of
// their own for the output and loops kept rolled (the roles' unrolled code outgrew the
// instruction cache) 490; parts of three bytes, whose columns may lie any factor apart, 550; two terms of P 615; three CTAs an SM for the joins again 600.
#include <algorithm>
#include <atomic>
#include <numeric>

#include "cluster_attention.cuh"
#include "cluster_tiles.cuh"

namespace fkc {
namespace attn {
namespace {

__global__ void __launch_bounds__(256) tile_init_kernel(int64_t* count, int32_t* __restrict__ pair_row,
                                                        int64_t pairs, int32_t* odd, float* largest, int R) {
  pdl_wait();
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i == 0) *count = 0;
  if (i == 0 && odd != nullptr) *odd = 0;
  if (largest != nullptr)
    for (int64_t r = i; r < R; r += static_cast<int64_t>(gridDim.x) * 256) largest[r] = 0.f;
  for (int64_t p = i; p < pairs; p += static_cast<int64_t>(gridDim.x) * 256) pair_row[p] = -1;
}

// Appends the units of row r. Which place they get is up to the order of the rows' claims;
// what a unit computes and writes does not depend on it.
__global__ void __launch_bounds__(1024) tile_units_kernel(Args a,
                                                          const int32_t* __restrict__ inv_offsets,
                                                          Unit* __restrict__ units, int64_t* count,
                                                          int32_t* __restrict__ cum,
                                                          int32_t* __restrict__ first_unit, int i0,
                                                          int nq, int units_max) {
  constexpr int rows = kUnitRows;
  __shared__ int warp_total[32];
  __shared__ unsigned long long warp_sum[32];
  __shared__ unsigned long long first;
  pdl_wait();
  const int r = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int32_t* of = inv_offsets + static_cast<int64_t>(r) * (a.K + 1);
  int high = a.q_pos != nullptr ? -1 : a.N;
  if (a.q_pos != nullptr) {
    const int32_t* pos = a.q_pos + static_cast<int64_t>(r / a.Hkv) * a.Nq + i0;
    for (int i = threadIdx.x; i < nq; i += 1024) high = max(high, min(pos[i], a.N));
    high = __reduce_max_sync(0xFFFFFFFFu, high);
    if (lane == 0) warp_total[warp] = high;
    __syncthreads();
    for (int w = 0; w < 32; ++w) high = max(high, warp_total[w]);
  }
  for (int c0 = 0; c0 < a.K; c0 += 1024) {
    const int c = c0 + threadIdx.x;
    int s0 = 0, s1 = 0, e0 = 0;
    int64_t all = 0;
    if (c < a.K) {
      cluster_span(a, r, c, s0, s1);
      e0 = of[c];
      if (s1 > s0) all = static_cast<int64_t>(of[c + 1] - e0) * a.G;
    }
    // units, and their cost above 2^32
    const int n = static_cast<int>((all + rows - 1) / rows);
    Unit un{c, 0, s0, s1, e0, 0, r, high};
    const unsigned long long own =
        (static_cast<unsigned long long>(n) * un.cost() << 32) | static_cast<unsigned>(n);
    unsigned long long inc = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned long long u = __shfl_up_sync(0xFFFFFFFFu, inc, o);
      if (lane >= o) inc += u;
    }
    __syncthreads();
    if (lane == 31) warp_sum[warp] = inc;
    __syncthreads();
    unsigned long long at = inc - own, sum = 0;
    for (int w = 0; w < 32; ++w) {
      if (w < warp) at += warp_sum[w];
      sum += warp_sum[w];
    }
    if (threadIdx.x == 0) first = atomicAdd(reinterpret_cast<unsigned long long*>(count), sum);
    __syncthreads();
    at += first;
    if (n > 0) first_unit[static_cast<int64_t>(r) * a.K + c] = static_cast<int32_t>(at & 0xFFFFFFFFu);
    for (int t = 0; t < n; ++t) {
      const int64_t u = static_cast<int64_t>(at & 0xFFFFFFFFu) + t;
      un.row0 = t * rows;
      un.nrows = static_cast<int>(min(static_cast<int64_t>(rows), all - static_cast<int64_t>(t) * rows)) |
                 (t + 1 < n ? Unit::kMore : 0);
      if (u < units_max) {  // always, with the workspace of carve_units
        units[u] = un;
        cum[u] = static_cast<int32_t>((at >> 32) + static_cast<unsigned long long>(t) * un.cost());
      }
    }
  }
}

// The rows of the units, one warp a unit: a lane takes rows lane + 32 j.
__global__ void __launch_bounds__(256) tile_rows_kernel(Args a, int i0, int nq, RowMap rq,
                                                        const int32_t* __restrict__ inv_order,
                                                        const Unit* __restrict__ units,
                                                        const int64_t* __restrict__ count,
                                                        const int32_t* __restrict__ cum,
                                                        int32_t* __restrict__ start, int ctas,
                                                        int32_t* __restrict__ q_row,
                                                        int32_t* __restrict__ row_pos,
                                                        int32_t* __restrict__ pair_row,
                                                        const float* __restrict__ lse,
                                                        int32_t* __restrict__ do_row,
                                                        float* __restrict__ row_lse) {
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int64_t u = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  const int64_t total = *count & 0xFFFFFFFFll, cost = *count >> 32;
  if (u == 0 && total == 0)
    for (int j = lane; j <= ctas; j += 32) start[j] = 0;
  if (u >= total) return;
  const Unit un = units[u];
  {
    // CTA j starts at the first unit whose cost begins at j / ctas of the whole or later
    const int64_t to = cum[u], from = u == 0 ? -1 : cum[u - 1];
    const int64_t j0 = u == 0 ? 0 : from * ctas / cost + 1;
    for (int64_t j = j0 + lane; j <= ctas && j * cost <= to * ctas; j += 32) start[j] = static_cast<int32_t>(u);
    if (u == total - 1)
      for (int64_t j = to * ctas / cost + 1 + lane; j <= ctas; j += 32) start[j] = static_cast<int32_t>(total);
  }
  const int b = un.r / a.Hkv, hk = un.r - b * a.Hkv;
  const int64_t pairs0 = static_cast<int64_t>(un.r) * nq * a.top;
  const int32_t* list = inv_order + pairs0 + un.e0;
#pragma unroll
  for (int j = 0; j < kUnitRows / 32; ++j) {
    const int rr = j * 32 + lane;
    int pos = -1, row = rq.rows;
    int64_t flat = -1;  // row of (batch, Hq, Nq)
    if (rr < (un.nrows & (Unit::kMore - 1))) {
      const int at = un.row0 + rr, e = at / a.G, h = at - e * a.G;
      const int p = list[e], i = i0 + p / a.top;
      if (h == 0) pair_row[pairs0 + p] = static_cast<int32_t>(u * kUnitRows + rr);
      pos = max(-1, min(a.q_pos != nullptr ? a.q_pos[static_cast<int64_t>(b) * a.Nq + i] : a.N, a.N));
      if (pos >= 0) {
        row = rq.at(b, hk * a.G + h, i);
        flat = (static_cast<int64_t>(b) * a.Hq + hk * a.G + h) * a.Nq + i;
      }
    }
    if (lse != nullptr) {
      do_row[u * kUnitRows + rr] = static_cast<int32_t>(flat >= 0 ? flat : static_cast<int64_t>(a.batch) * a.Hq * a.Nq);
      row_lse[u * kUnitRows + rr] = flat >= 0 ? lse[flat] * kLog2e : 0.f;
    }
    q_row[u * kUnitRows + rr] = row;
    row_pos[u * kUnitRows + rr] = pos;
  }
}

// Shared memory of the forward kernel: operand tiles (1024-byte aligned), then the rest.
template <int DP>
struct FwdSmem {
  static constexpr uint32_t kTile = tc_tile_bytes<DP>();
  static constexpr uint32_t kQ = 0;              // one tile per 128 rows
  static constexpr uint32_t kK = 2 * kTile;      // two stages
  static constexpr uint32_t kV = 4 * kTile;      // two stages
  static constexpr uint32_t kOut = 6 * kTile;    // 4 KB per output warp
  static constexpr uint32_t kMeta = kOut + 8 * 4096;
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

// Warps 0-3 and 4-7: softmax of rows 0-127 and 128-255 of a unit (a thread a row); 8-11 and
// 12-15: their output, while the softmax goes on to the next unit; warp 16: the MMAs; warps 17,
// 18: gathers of keys and of values; 19-22: of Q, 64 rows each (a gather takes its warp some 70
// cycles to issue, so they are spread over warps); 23 has nothing to do.
constexpr int kFwdThreads = 32 * 24;
// Registers of the three kinds of warpgroups: as many in all as the launch's 80 a thread.
constexpr int kLaunchRegs = 80, kSoftmaxRegs = 112, kOutputRegs = 72, kOtherRegs = 56;
static_assert(256 * (kSoftmaxRegs + kOutputRegs + kOtherRegs) <= kFwdThreads * kLaunchRegs,
              "setmaxnreg would wait for registers that the block does not have");

template <typename T, int DP>
__global__ void __launch_bounds__(kFwdThreads, 1) tiles_fwd_kernel(
    const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
    const __grid_constant__ CUtensorMap tm_v, RowMap rk, RowMap rv, Args a,
    const int32_t* __restrict__ q_row, const int32_t* __restrict__ row_pos,
    const Unit* __restrict__ units, const int32_t* __restrict__ start, uint8_t* __restrict__ part_o,
    float2* __restrict__ part_lse, int* err) {
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
      mbar_init(smem_u32(&mt.q_full[x]), 2);
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
  if (warp == 16) {
    tmem_alloc(smem_u32(&mt.tmem), 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = mt.tmem;  // sub-tile x: S (then P) at 256 x, O at 256 x + 128
  pdl_wait();

  if (warp < 8) {
    // ------------------------------------------------------------ softmax
    more_registers<kSoftmaxRegs>();
    const int sub = warp >> 2, row = (warp & 3) * 32 + lane;
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t t_s = tmem + lanes + sub * 256, t_o = t_s + 128;
    const float sc = a.scale * kLog2e;
    uint32_t s_uses = 0;
    bool ok = true;
    UnitIter it(units, start);
    const int32_t* meta = row_pos + sub * kSub + row;
    int ahead = it.valid() ? __ldg(meta + static_cast<int64_t>(it.n) * kUnitRows) : -1;
    for (; ok && it.valid(); it.advance()) {
      const Unit& un = it.un;
      const int steps = un.steps();
      const int pos = ahead;
      if (it.n + 1 < it.total) ahead = __ldg(meta + static_cast<int64_t>(it.n + 1) * kUnitRows);
      if (un.nrows <= sub * kSub) continue;
      const int pos_min =
          __reduce_min_sync(0xFFFFFFFFu, sub * kSub + row < un.nrows ? pos : INT_MAX);
      float m = -INFINITY, l = 0.f;
      for (int step = 0; step < steps; ++step, ++s_uses) {
        const uint32_t load = it.load + step;
        const int st = load & 1;
        ok = warp_mbar_wait(&mt.k_full[st], (load >> 1) & 1, abort) &&
             warp_mbar_wait(&mt.s_full[sub], s_uses & 1, abort);
        if (!ok) {
          give_up(abort, err, kErrSoftmax);
          break;
        }
        tc_fence_after();
        const int keys = un.keys(step);
        const int32_t* key = mt.key[st];
        // (loops over chunks stay loops: unrolled, the code of the kernel's roles outgrew the
        // instruction cache)
        float tops[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
        uint32_t open = 0;  // 32-key chunks that every row of the warp sees whole
#pragma unroll 1
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
        const float base = mn == -INFINITY ? 0.f : mn, from = base - Range<T>::kShift;
        const float alpha = ex2(m - base);
        m = mn;
        if (step > 0 && __any_sync(0xFFFFFFFFu, alpha != 1.f)) {
          // the product of the step before has ended: its commit came before this S's
#pragma unroll 1
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
#pragma unroll 1
        for (int c = 0; c < kKeysStep / 32; ++c) {
          if (c * 32 >= keys) break;
          float s[32];
          tmem_ld_f32_x32(t_s + c * 32, s);
          tmem_wait_ld();
          if (open >> c & 1u) {
#pragma unroll
            for (int j = 0; j < 32; ++j)
              s[j] = ex2(fmaf(s[j], sc, -from));
          } else {
#pragma unroll
            for (int j = 0; j < 32; j += 4) {
              const int4 k4 = *reinterpret_cast<const int4*>(key + c * 32 + j);
              const int k[4] = {k4.x, k4.y, k4.z, k4.w};
#pragma unroll
              for (int e = 0; e < 4; ++e)
                s[j + e] = ex2(k[e] <= pos ? fmaf(s[j + e], sc, -from) : -INFINITY);
            }
          }
#pragma unroll
          for (int j = 0; j < 32; ++j) sum[j & 3] += s[j];
          split32<T, true>(t_s + c * 32, s);
        }
        l = l * alpha + ((sum[0] + sum[1]) + (sum[2] + sum[3]));
        tmem_wait_st();
        tc_fence_before();
        mbar_arrive(smem_u32(&mt.p_full[sub]));
      }
      if (!ok) break;
      part_lse[static_cast<int64_t>(it.n) * kUnitRows + sub * kSub + row] =
          make_float2(l == 0.f ? -INFINITY : m - Range<T>::kShift + log2f(l), l == 0.f ? 0.f : 1.f / l);
    }
  } else if (warp < 16) {
    // ------------------------------------------------------------ output
    fewer_registers<kOutputRegs>();
    const int sub = (warp >> 2) - 2, row = (warp & 3) * 32 + lane;
    const uint32_t t_o = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16) + sub * 256 + 128;
    uint32_t uses = 0;
    bool ok = true;
    for (UnitIter it(units, start); ok && it.valid(); it.advance()) {
      if (it.un.nrows <= sub * kSub) continue;
      ok = warp_mbar_wait(&mt.o_full[sub], uses & 1, abort);
      if (!ok) {
        give_up(abort, err, kErrSoftmax);
        break;
      }
      tc_fence_after();
      const int64_t urow = static_cast<int64_t>(it.n) * kUnitRows + sub * kSub + row;
      const uint32_t buf = sb + S::kOut + (warp - 8) * 4096;
      uint8_t* dst = part_o + (urow - lane) * (DP * kPartBytes);
#pragma unroll 1
      for (int c = 0; c < DP / 32; ++c) {
        uint32_t o[32];
        tmem_ld_32x32b_x32(t_o + c * 32, o);
        tmem_wait_ld();
        put_segment(buf, o, dst + c * kSegment);
      }
      tc_fence_before();
      mbar_arrive(smem_u32(&mt.o_free[sub]));
      ++uses;
    }
    if (lane == 0) bulk_wait_all();
  } else {
    fewer_registers<kOtherRegs>();
    if (warp == 16 && lane == 0) {
      // ---------------------------------------------------------- MMAs (one thread)
      const int dsteps = (a.D + 15) / 16;
      constexpr uint32_t idesc_o = umma_idesc_f16(kBf16, kSub, DP) | kIdescMnB;
      uint32_t q_uses[2] = {0, 0}, p_uses[2] = {0, 0};
      struct Pending {
        bool has, first, last;
        int stage, ksteps;
        uint32_t parity;  // of the stage's values
      } pend[2] = {};
      int to_free = -1;  // the stage of the step before, if nothing uses it again
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
        mma_tmem_rows<8>(tmem + sub * 256 + 128, tmem + sub * 256, sb + S::kV + p.stage * S::kTile,
                      idesc_o, p.ksteps, p.first);
        if (p.last) umma_commit(smem_u32(&mt.o_full[sub]));
      };
      for (UnitIter it(units, start); ok && it.valid(); it.advance()) {
        const Unit& un = it.un;
        const int steps = un.steps();
        for (int step = 0; ok && step < steps; ++step) {
          const uint32_t load = it.load + step;
          const int st = load & 1;
          const int k16 = (un.keys(step) + 15) / 16;
          const uint32_t idesc_s = umma_idesc_f16(kBf16, kSub, 16 * k16);
          for (int sub = 0; sub < 2; ++sub) {
            product(sub);
            if (!ok || un.nrows <= sub * kSub) continue;
            ok = mbar_wait(smem_u32(&mt.k_full[st]), (load >> 1) & 1, abort);
            if (ok && step == 0) {
              ok = mbar_wait(smem_u32(&mt.q_full[sub]), q_uses[sub] & 1, abort);
              ++q_uses[sub];
            }
            if (!ok) break;
            mma_kmajor<DP>(tmem + sub * 256, sb + S::kQ + sub * S::kTile, sb + S::kK + st * S::kTile,
                           idesc_s, dsteps);
            umma_commit(smem_u32(&mt.s_full[sub]));
            if (step == steps - 1) umma_commit(smem_u32(&mt.q_free[sub]));
            pend[sub] = {true, step == 0, step == steps - 1, st, k16, (load >> 1) & 1};
          }
          if (ok && to_free >= 0) umma_commit(smem_u32(&mt.kv_free[to_free]));
          to_free = it.keep ? -1 : st;
        }
      }
      for (int sub = 0; sub < 2; ++sub)
        if (ok) product(sub);
      if (!ok) give_up(abort, err, kErrMma);
      umma_commit(smem_u32(&mt.drain));  // nothing is in flight when TMEM is freed
      const int never = 0;
      mbar_wait(smem_u32(&mt.drain), 0, &never);
    }
    // ------------------------------------------------------------ gathers
    // The next step's (or unit's) row numbers are fetched while this one's copies run.
    bool ok = true;
    if (warp == 17 || warp == 18) {
      const bool values = warp == 18;
      const CUtensorMap* tm = values ? &tm_v : &tm_k;
      const RowMap rm = values ? rv : rk;
      const uint32_t tiles = sb + (values ? S::kV : S::kK);
      UnitIter it(units, start);
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
    } else if (warp >= 19 && warp < 23) {
      const int x = (warp - 19) >> 1, row0 = ((warp - 19) & 1) * 64 + (lane & 15) * 4;
      const int4* src = reinterpret_cast<const int4*>(q_row) + (x * kSub + row0) / 4;
      UnitIter it(units, start);
      int4 ahead = it.valid() ? __ldg(src + static_cast<int64_t>(it.n) * (kUnitRows / 4)) : make_int4(0, 0, 0, 0);
      uint32_t uses = 0;
      for (; it.valid(); it.advance()) {
        const int4 rows = ahead;
        if (it.n + 1 < it.total) ahead = __ldg(src + static_cast<int64_t>(it.n + 1) * (kUnitRows / 4));
        if (it.un.nrows <= x * kSub) continue;
        ok = warp_mbar_wait(&mt.q_free[x], (uses & 1) ^ 1, abort);
        if (!ok) break;
        if (lane == 0) mbar_arrive_expect_tx(smem_u32(&mt.q_full[x]), S::kTile / 2);
        // a block of 64 elements by each half of the warp
        const int blk = lane >> 4;
        if (blk < DP / 64)
          tma_gather4(sb + S::kQ + x * S::kTile + blk * (128 * kSub) + row0 * 128, &tm_q,
                      smem_u32(&mt.q_full[x]), blk * 64, rows.x, rows.y, rows.z, rows.w);
        __syncwarp();
        ++uses;
      }
    }
    if (!ok) give_up(abort, err, kErrLoad);
    // copies in flight end before the CTA does: the MMA warp waits for all of them, and
    // after a wait that gave up they are waited for here
    if (warp > 16 && (!ok || *abort)) {
      const uint64_t t0 = globaltimer_ns();
      while (globaltimer_ns() - t0 < 1000000ull) {
      }
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == 16) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// One warp per (query, GP heads): joins the parts of its clusters, whose log-sum-exps are to
// base 2. Bound by the parts' loads: three CTAs an SM (80 registers) take 143 us for 824 MB, two 174.
template <typename T, int DP>
__global__ void __launch_bounds__(256, 3) tiles_join_kernel(Args a, int i0, int nq, int gp, int chunks,
                                                         const int32_t* __restrict__ pair_row,
                                                         const uint8_t* __restrict__ part_o,
                                                         const float2* __restrict__ part_lse,
                                                         T* __restrict__ out,
                                                         float* __restrict__ lse,
                                                         int32_t* __restrict__ odd, int64_t warps) {
  constexpr int E = 8, SEGS = DP / 64;
  constexpr int kAhead = 8 / SEGS;  // slots in flight per lane
  pdl_wait();
  const int64_t w0 = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);  // (r, i - i0, heads)
  if (w0 >= warps) return;
  const JoinLane me(gp);
  const int h = static_cast<int>(w0 % chunks) * gp + me.head;
  const int64_t qi = w0 / chunks;
  const int r = static_cast<int>(qi / nq), i = i0 + static_cast<int>(qi % nq);
  const int b = r / a.Hkv, per = 4 / gp;
  const int32_t* pairs = pair_row + qi * a.top;
  float top = -INFINITY, sum = 0.f, acc[SEGS][E];
#pragma unroll
  for (int g = 0; g < SEGS; ++g)
#pragma unroll
    for (int e = 0; e < E; ++e) acc[g][e] = 0.f;
  for (int s0 = 0; s0 < a.top; s0 += kAhead * per) {
    Part8 v[kAhead][SEGS];
    float2 w[kAhead];
    float big = top;
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int s = s0 + u * per + me.slot;
      const int64_t n = s < a.top && h < a.G ? pairs[s] : -1;
      w[u] = n >= 0 ? part_lse[n + h] : make_float2(-INFINITY, 0.f);
#pragma unroll
      for (int g = 0; g < SEGS; ++g) {
        v[u][g] = Part8{};
        if (n >= 0) v[u][g] = load_part<DP>(part_o, n + h, g * 8 + me.piece);
      }
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) big = fmaxf(big, w[u].x);
    const float from = big == -INFINITY ? 0.f : big, alpha = exp2f(top - from);
    top = big;
    sum *= alpha;
#pragma unroll
    for (int g = 0; g < SEGS; ++g)
#pragma unroll
      for (int e = 0; e < E; ++e) acc[g][e] *= alpha;
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      if (w[u].x == -INFINITY) continue;  // no part, or it sees nothing of its cluster
      const float p = exp2f(w[u].x - from);
      sum += p;
#pragma unroll
      for (int g = 0; g < SEGS; ++g) add_part(acc[g], v[u][g], p * w[u].y);
    }
  }
  for (int o = 8 * gp; o < 32; o <<= 1) {  // the slots' lanes
    const float other = __shfl_xor_sync(0xFFFFFFFFu, top, o), big = fmaxf(top, other);
    const float from = big == -INFINITY ? 0.f : big;
    const float mine = exp2f(top - from), its = exp2f(other - from);
    sum = sum * mine + __shfl_xor_sync(0xFFFFFFFFu, sum, o) * its;
#pragma unroll
    for (int g = 0; g < SEGS; ++g)
#pragma unroll
      for (int e = 0; e < E; ++e)
        acc[g][e] = acc[g][e] * mine + __shfl_xor_sync(0xFFFFFFFFu, acc[g][e], o) * its;
    top = big;
  }
  if (me.slot != 0 || h >= a.G) return;
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  const int64_t at = (static_cast<int64_t>(b) * a.Hq + (r - b * a.Hkv) * a.G + h) * a.Nq + i;
#pragma unroll
  for (int g = 0; g < SEGS; ++g) {
    const int d = (g * 8 + me.piece) * E;
    if (d < a.D) store_out<T>(out + at * a.D + d, acc[g], inv);
  }
  float bad = 0.f;
#pragma unroll
  for (int g = 0; g < SEGS; ++g)
#pragma unroll
    for (int e = 0; e < E; ++e) bad = not_finite(acc[g][e], bad);
  if (bad != 0.f) *odd = 1;
  if (me.piece == 0) lse[at] = sum == 0.f ? -INFINITY : (top + log2f(sum)) * kLn2;
}

// Queries that one round takes: rounds of equal size whose rows take some 1.5 GB (a round has its own
// grouping, so short ones cost launches), 64 queries at least.
int64_t queries_per_round(const Args& a) {
  const int64_t R = static_cast<int64_t>(a.batch) * a.Hkv;
  const int64_t per = R * a.top * a.G * unit_row_bytes(a);
  const int64_t most = std::max<int64_t>(64, (3ll << 29) / per);
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
  l.nq = queries_per_round(a);
  size_t at = carve_units(a, l.nq, false, ws, &l.plan);
  auto take = [&](int64_t bytes) {
    const size_t p = at;
    at += align_up(static_cast<size_t>(bytes), 256);
    return p;
  };
  l.part_lse = take(l.plan.units_max * kUnitRows * 8);
  l.part_o = take(l.plan.units_max * kUnitRows * (a.D <= 64 ? 64 : 128) * kPartBytes);
  l.total = at;
  return l;
}

template <typename T, int DP>
int fwd_typed(const Args& a, int dtype, T* out, float* lse, uint8_t* ws, cudaStream_t stream) {
  const Layout l = fwd_layout(a, ws);
  const int64_t R = static_cast<int64_t>(a.batch) * a.Hkv;
  float2* part_lse = reinterpret_cast<float2*>(ws + l.part_lse);
  uint8_t* part_o = ws + l.part_o;
  CUtensorMap tm_q, tm_k, tm_v;
  RowMap rq, rk, rv;
  FKC_TRY(encode_rows(a.q, a.qs, a.batch, a.Hq, a.Nq, a.D, dtype, &tm_q, &rq));
  FKC_TRY(encode_rows(a.k, a.ks, a.batch, a.Hkv, a.N, a.D, dtype, &tm_k, &rk));
  FKC_TRY(encode_rows(a.v, a.vs, a.batch, a.Hkv, a.N, a.D, dtype, &tm_v, &rv));
  auto kern = tiles_fwd_kernel<T, DP>;
  const int smem = static_cast<int>(FwdSmem<DP>::kBytes);
  // the compiler gives the block as many registers as its warpgroups take in all, or they would wait
  static std::atomic<int> regs{0};  // of this kernel, the same on every device
  if (regs.load(std::memory_order_relaxed) == 0) {
    cudaFuncAttributes fa{};
    FKC_CUDA_TRY(cudaFuncGetAttributes(&fa, kern));
    regs.store(fa.numRegs, std::memory_order_relaxed);
  }
  FKC_REQUIRE(regs.load(std::memory_order_relaxed) >= kLaunchRegs, "attention: the kernel was built with %d registers",
              regs.load(std::memory_order_relaxed));
  FKC_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  for (int64_t i0 = 0; i0 < a.Nq; i0 += l.nq) {
    const int nq = static_cast<int>(std::min<int64_t>(l.nq, a.Nq - i0));
    const int ctas = static_cast<int>(std::min<int64_t>(std::min(sm_count(), kMaxCtas), l.plan.units_max));
    FKC_TRY(launch_units(a, i0, nq, rq, l.plan, ctas, nullptr, stream));
    FKC_TRY(launch_pdl(kern, dim3(ctas), dim3(kFwdThreads), smem, stream, tm_q, tm_k, tm_v, rk, rv, a,
                       static_cast<const int32_t*>(l.plan.q_row),
                       static_cast<const int32_t*>(l.plan.row_pos),
                       static_cast<const Unit*>(l.plan.units),
                       static_cast<const int32_t*>(l.plan.start), part_o, part_lse,
                       device_error_word()));
    const int gp = join_heads(a.G), chunks = (a.G + gp - 1) / gp;
    const int64_t warps = R * nq * chunks;
    FKC_TRY(launch_pdl(tiles_join_kernel<T, DP>, dim3(static_cast<unsigned>((warps + 7) / 8)), dim3(256),
                       0, stream, a, static_cast<int>(i0), nq, gp, chunks,
                       static_cast<const int32_t*>(l.plan.pair_row),
                       static_cast<const uint8_t*>(part_o), static_cast<const float2*>(part_lse), out,
                       lse, l.plan.odd, warps));
  }
  return launch_again(a, dtype, l.plan.odd, lse, nullptr, nullptr, out, nullptr, nullptr, nullptr, nullptr, stream);
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

size_t carve_units(const Args& a, int64_t nq, bool grad, uint8_t* ws, UnitPlan* out) {
  const int64_t R = static_cast<int64_t>(a.batch) * a.Hkv;
  const int64_t pairs = nq * a.top;
  UnitPlan p{};
  p.units_max = units_most(a, nq);
  size_t at = 0;
  auto take = [&](int64_t bytes) -> void* {
    void* q = ws != nullptr ? ws + at : nullptr;
    at += align_up(static_cast<size_t>(bytes), 256);
    return q;
  };
  p.inv_order = static_cast<int32_t*>(take(R * pairs * 4));
  p.inv_offsets = static_cast<int32_t*>(take(R * (a.K + 1) * 4));
  p.units = static_cast<Unit*>(take(p.units_max * static_cast<int64_t>(sizeof(Unit))));
  p.count = static_cast<int64_t*>(take(8));
  p.start = static_cast<int32_t*>(take((kMaxCtas + 1) * 4));
  p.cum = static_cast<int32_t*>(take(p.units_max * 4));
  p.q_row = static_cast<int32_t*>(take(p.units_max * kUnitRows * 4));
  p.row_pos = static_cast<int32_t*>(take(p.units_max * kUnitRows * 4));
  p.pair_row = static_cast<int32_t*>(take(R * pairs * 4));
  p.first_unit = static_cast<int32_t*>(take(R * a.K * 4));
  p.odd = static_cast<int32_t*>(take(4));
  if (grad) {
    p.do_row = static_cast<int32_t*>(take(p.units_max * kUnitRows * 4));
    p.row_lse = static_cast<float*>(take(p.units_max * kUnitRows * 4));
    p.row_delta = static_cast<float*>(take(p.units_max * kUnitRows * 4));
    p.row_power = static_cast<float*>(take(p.units_max * kUnitRows * 4));
    p.largest = static_cast<float*>(take(R * 4));
  }
  p.group_ws = take(static_cast<int64_t>(group_workspace_bytes(R, pairs, a.K)));
  if (out != nullptr) *out = p;
  return at;
}

int launch_units(const Args& a, int64_t i0, int64_t nq, const RowMap& rq, const UnitPlan& p, int ctas,
                 const float* lse, cudaStream_t stream) {
  const int64_t R = static_cast<int64_t>(a.batch) * a.Hkv;
  FKC_REQUIRE(p.units_max * kUnitRows <= 2147483647ll, "attention: too many tiles");
  const int64_t blocks = std::min<int64_t>((R * nq * a.top + 255) / 256, sm_count() * 8ll);
  FKC_TRY(launch_pdl(tile_init_kernel, dim3(static_cast<unsigned>(blocks)), dim3(256), 0, stream, p.count,
                     p.pair_row, R * nq * a.top, i0 == 0 ? p.odd : nullptr, p.largest,
                     static_cast<int>(R)));
  FKC_TRY(launch_group(a.sel + i0 * a.top, false, static_cast<int64_t>(a.Nq) * a.top, p.inv_order,
                       p.inv_offsets, R, nq * a.top, a.K, p.group_ws, stream));
  FKC_TRY(launch_pdl(tile_units_kernel, dim3(static_cast<unsigned>(R)), dim3(1024), 0, stream, a,
                     static_cast<const int32_t*>(p.inv_offsets), p.units, p.count, p.cum, p.first_unit,
                     static_cast<int>(i0), static_cast<int>(nq), static_cast<int>(p.units_max)));
  return launch_pdl(tile_rows_kernel, dim3(static_cast<unsigned>((p.units_max + 7) / 8)), dim3(256), 0,
                    stream, a, static_cast<int>(i0), static_cast<int>(nq), rq,
                    static_cast<const int32_t*>(p.inv_order),
                    static_cast<const Unit*>(p.units),
                    static_cast<const int64_t*>(p.count), static_cast<const int32_t*>(p.cum),
                    p.start, ctas, p.q_row, p.row_pos, p.pair_row, lse, p.do_row,
                    p.row_lse);
}

FormWork form_work(const Args& a, int64_t nq) {
  const double R = static_cast<double>(a.batch) * a.Hkv, pairs = static_cast<double>(nq) * a.top;
  FormWork w;
  w.width = a.D <= 64 ? 0.5 : 1.0;
  w.keys = static_cast<double>(a.N) / a.K;
  w.rows = R * a.Nq * a.top * a.G;
  w.reads = R * a.Nq * a.top * w.keys * (a.G <= 8 ? 1.0 : 1.2 * ((a.G + 15) / 16));
  // every cluster with pairs may end in a unit that is not full; fewer units than SMs leave
  // SMs idle
  const double rounds = static_cast<double>((a.Nq + nq - 1) / nq);
  w.units = std::max(rounds * R * std::min<double>(a.K, pairs) + w.rows / kUnitRows, 148.0);
  return w;
}

bool tiles_fit(const Args& a, int64_t nq, int64_t bytes) {
  // 32-bit row numbers; a running maximum of unscaled scores; the gathers' maps
  if (!(a.scale > 0.f) ||
      !row_map(a.qs, a.batch, a.Hq, a.Nq, a.D, nullptr, nullptr) ||
      !row_map(a.ks, a.batch, a.Hkv, a.N, a.D, nullptr, nullptr) ||
      !row_map(a.vs, a.batch, a.Hkv, a.N, a.D, nullptr, nullptr))
    return false;
  const int64_t rows = units_most(a, nq) * kUnitRows;
  return rows <= (1ll << 30) && rows * unit_row_bytes(a) <= bytes;
}

// In us, fitted to 200 calls of 8 to 200 keys a cluster, 32 to 4096 queries, 1 to 32 heads a row and 1 to 32
// clusters a query, both widths and types (the walk within 16% on average, this form within 9%): the
// form that it chooses took 0.5% longer on average than the faster one. The walk's last term is the
// chain of one warp's key tiles. Measured (walk, by clusters), D = 128 but for the last two:
// G 8, 218 queries x 8 rows, 4 of 64 clusters of 64 keys: 45, 45. G 4, 375 x 1, 16 of 512 of 100: 46, 49;
// 142 x 4, 8 of 64 of 100: 37, 35; 2191 x 4, 16 of 256 of 100: 930, 171. G 16, 996 x 4, 3 of 16 of 12:
// 43, 71. G 1, 886 x 8, 2 of 16 of 32: 50, 35. D = 64: G 4, 444 x 4, 3 of 64 of 16: 8, 29. G 1, 2139 x 4,
// 16 of 16 of 100: 480, 58.
bool use_tiles(const Args& a) {
  const int64_t nq = queries_per_round(a);
  if (!tiles_fit(a, nq, 1ll << 32)) return false;
  const FormWork w = form_work(a, nq);
  const double walk = 7.9 + 79.7e-6 * w.reads * w.width + 0.0705 * a.top * w.keys / 16 / split_count(a);
  const double tiles = 27.8 + w.units * (0.0079 + 0.000162 * w.keys * w.width) + w.rows * (38e-6 + 111e-6 * w.width);
  return tiles < walk;
}

size_t tiles_forward_workspace_bytes(const Args& a) { return fwd_layout(a, nullptr).total; }

int launch_tiles_forward(const Args& a, int dtype, void* out, float* lse, void* ws,
                         cudaStream_t stream) {
  return dtype == FKC_DTYPE_F16 ? fwd_dtype<__half>(a, dtype, out, lse, ws, stream)
                                : fwd_dtype<__nv_bfloat16>(a, dtype, out, lse, ws, stream);
}

}  // namespace attn
}  // namespace fkc
