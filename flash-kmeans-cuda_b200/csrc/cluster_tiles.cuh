// Tiles of attention by clusters (cluster_attention_tiles.cu and its backward): the units
// of work, and operand tiles gathered row by row into the layout that tcgen05.mma reads.
//
// A pair is one entry of sel: query i's slot s, number p = (i - i0) * top + s of its row r.
// Grouping sel by cluster (cluster_group.cu) brings the pairs of a cluster together; the
// G heads of its pairs, one after another, are the cluster's rows. A unit is up to 256 of them.
#pragma once

#include <algorithm>

#include "cluster_attention.cuh"
#include "fkc_ptx.cuh"

namespace fkc {
namespace attn {

constexpr int kSub = 128;        // rows of one MMA
constexpr int kKeysStep = 128;   // keys per step

// One unit: cluster c of row r, whose slots are [s0, s1) and whose pairs start at e0; rows
// [row0, row0 + nrows) of the cluster; high: the last position that one of them sees.
struct __align__(16) Unit {
  int c, row0, s0, s1;
  int e0, nrows, r, high;

  __device__ __forceinline__ int steps() const { return (s1 - s0 + kKeysStep - 1) / kKeysStep; }
  __device__ __forceinline__ int keys(int step) const {
    return min(kKeysStep, s1 - s0 - step * kKeysStep);
  }
};

__device__ __forceinline__ Unit load_unit(const Unit* u) {
  Unit x;
  const int4 lo = __ldg(reinterpret_cast<const int4*>(u));
  const int4 hi = __ldg(reinterpret_cast<const int4*>(u) + 1);
  x.c = lo.x, x.row0 = lo.y, x.s0 = lo.z, x.s1 = lo.w;
  x.e0 = hi.x, x.nrows = hi.y, x.r = hi.z, x.high = hi.w;
  return x;
}

// Operand tile of 128 rows x DP 16-bit elements: column blocks of 64 elements (128 rows x
// 128 bytes each, 128-byte swizzle). As K-major operand a row is a row; as MN-major operand a
// row is a k. Elements past D are filled with zeros by the copy.
template <int DP>
constexpr uint32_t tc_tile_bytes() {
  return kSub * DP * 2;
}

// D (+)= A B^T over the first `depth` elements (a multiple of 16) of K-major tiles.
template <int DP>
__device__ __forceinline__ void mma_kmajor(uint32_t d, uint32_t a_tile, uint32_t b_tile,
                                           uint32_t idesc, int ksteps) {
  constexpr uint32_t hi = ptx::umma_desc_hi(1024, ptx::kLayoutSwizzle128B);
  const uint32_t a = ptx::umma_desc_lo(a_tile), b = ptx::umma_desc_lo(b_tile);
#pragma unroll
  for (int k = 0; k < DP / 16; ++k) {
    if (k >= ksteps) break;
    const uint32_t o = ((k >> 2) * (128 * kSub) + (k & 3) * 32) >> 4;
    ptx::umma_f16(d, ptx::umma_desc(a + o, hi), ptx::umma_desc(b + o, hi), idesc, k > 0);
  }
}

// D (+)= A B, A [lanes x 16 * ksteps] in TMEM, B the first 16 * ksteps rows of a tile (MN-major).
__device__ __forceinline__ void mma_tmem_rows(uint32_t d, uint32_t a_tmem, uint32_t b_tile,
                                              uint32_t idesc, int ksteps, bool fresh) {
  for (int k = 0; k < ksteps; ++k)
    ptx::umma_f16_ta(d, a_tmem + k * 8, ptx::umma_desc_mn(b_tile + k * 2048, 128 * kSub), idesc,
                     !(fresh && k == 0));
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Eight floats to a 32-byte aligned address.
__device__ __forceinline__ void st_global_v8(float* p, const float (&v)[8]) {
  asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "f"(v[0]),
               "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7])
               : "memory");
}

__device__ __forceinline__ void named_barrier(int id, int threads) {
  asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}
// The same; true in all of the threads when `any` is in one.
__device__ __forceinline__ bool named_barrier_any(int id, int threads, bool any) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 p, %3, 0;\n\t"
      "bar.red.or.pred q, %1, %2, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"(id), "r"(threads), "r"(any ? 1u : 0u)
      : "memory");
  return r != 0;
}

// Bounded wait of a whole warp; the same answer in every lane.
__device__ __forceinline__ bool warp_mbar_wait(const uint64_t* bar, uint32_t parity,
                                               const volatile int* abort) {
  return __all_sync(0xFFFFFFFFu, ptx::mbar_wait(ptx::smem_u32(bar), parity, abort));
}

// A bounded wait gave up: every role leaves, the host reads the code (fkc_device_status).
__device__ __forceinline__ void give_up(volatile int* abort, int* err, int code) {
  *abort = 1;
  if (err != nullptr) atomicCAS(err, 0, code);
}

// A strided (batch, heads, positions) tensor as rows of a 2-D map: row b * b_ + h * h_ + n * n_,
// `rows` of them; row number `rows` reads as zeros.
struct RowMap {
  int64_t b, h, n;
  int rows;
  __device__ __forceinline__ int at(int ib, int ih, int in) const {
    return static_cast<int>(ib * b + ih * h + in * n);
  }
};
// False where the strides have no common unit of a row's length, or there are 2^31 rows.
bool row_map(const Strides& s, int64_t nb, int64_t nh, int64_t nn, int64_t D, RowMap* map,
             int64_t* unit);
int encode_rows(const void* base, const Strides& s, int64_t nb, int64_t nh, int64_t nn, int64_t D,
                int dtype, CUtensorMap* tm, RowMap* map);

// Four rows of an operand tile, the rows' 16 * CH bytes in blocks of 64 elements.
template <int DP>
__device__ __forceinline__ void gather_rows4(uint32_t tile, const CUtensorMap* tm, const uint64_t* bar,
                                             int row, int r0, int r1, int r2, int r3) {
#pragma unroll
  for (int blk = 0; blk < DP / 64; ++blk)
    ptx::tma_gather4(tile + blk * (128 * kSub) + row * 128, tm, ptx::smem_u32(bar), blk * 64, r0, r1,
                     r2, r3);
}

// The grouping, units and rows of a range of queries, in the caller's workspace. Unit u's row
// j is entry kUnitRows * u + j of the rows' arrays.
constexpr int kUnitRows = 2 * kSub;
struct UnitPlan {
  int32_t* inv_order;    // (R, nq * top) pairs by cluster
  int32_t* inv_offsets;  // (R, K + 1)
  Unit* units;
  int32_t* count;        // of units
  int32_t* q_row;        // row of Q's map; the one past its last for a row that sees nothing
  int2* slot_pos;        // (pair, head) number within r, or -1 past the unit's last row; last
                         // position that the row sees
  void* group_ws;
  int64_t units_max;
};
size_t carve_units(const Args& a, int64_t nq, uint8_t* ws, UnitPlan* out);
// Groups sel of the queries [i0, i0 + nq), lists the units and fills the rows.
int launch_units(const Args& a, int64_t i0, int64_t nq, const RowMap& rq, const UnitPlan& p,
                 cudaStream_t stream);
int sm_count();

}  // namespace attn
}  // namespace fkc
