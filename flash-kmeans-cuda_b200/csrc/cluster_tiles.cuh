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
// [row0, row0 + nrows) of the cluster; high: the last position that a query of the range
// sees. Units of one cluster follow one another.
struct __align__(16) Unit {
  int c, row0, s0, s1;
  int e0, nrows, r, high;

  // in memory, nrows carries a flag: another unit of the cluster follows
  static constexpr int kMore = 1 << 16;

  __device__ __forceinline__ int steps() const { return (s1 - s0 + kKeysStep - 1) / kKeysStep; }
  // in about 580 cycles: each of the one or two steps whose keys stay in shared memory from
  // unit to unit (16), or each step of more, which every unit loads again (18), and what a
  // unit takes besides; capped, so that sums stay below 2^31
  __device__ __forceinline__ int cost() const {
    return min(steps() <= 2 ? 1 + 16 * steps() : 8 + 18 * steps(), 1020);
  }
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

// The issue loops below run in one thread, whose instructions per MMA bound them: descriptors are
// two halves of which a step adds a constant to one, and the usual depth is unrolled.
//
// D = A B^T over 16 * ksteps elements of K-major tiles.
template <int DP>
__device__ __forceinline__ void mma_kmajor(uint32_t d, uint32_t a_tile, uint32_t b_tile,
                                           uint32_t idesc, int ksteps) {
  constexpr uint32_t hi = ptx::umma_desc_hi(1024, ptx::kLayoutSwizzle128B);
  const uint32_t a = ptx::umma_desc_lo(a_tile), b = ptx::umma_desc_lo(b_tile);
  auto step = [&](int k) {
    const uint32_t o = ((k >> 2) * (128 * kSub) + (k & 3) * 32) >> 4;
    ptx::umma_f16(d, ptx::umma_desc(a + o, hi), ptx::umma_desc(b + o, hi), idesc, k > 0);
  };
  if (ksteps == DP / 16) {
#pragma unroll
    for (int k = 0; k < DP / 16; ++k) step(k);
  } else {
    for (int k = 0; k < ksteps; ++k) step(k);
  }
}

// D (+)= A B, A [lanes x 16 * ksteps] in TMEM as split32 leaves it, B the first 16 * ksteps rows of a tile
// (MN-major). MOST: the usual number of steps.
template <int MOST>
__device__ __forceinline__ void mma_tmem_rows(uint32_t d, uint32_t a_tmem, uint32_t b_tile,
                                              uint32_t idesc, int ksteps, bool fresh) {
  constexpr uint32_t hi = ptx::umma_desc_hi(1024, ptx::kLayoutSwizzle128B);
  const uint32_t b = ((b_tile >> 4) & 0x3FFFu) | ((128u * kSub >> 4) << 16);
  auto step = [&](int k, uint32_t accumulate) {
    const uint32_t at = a_tmem + (k >> 1) * 32 + (k & 1) * 8;
    const uint64_t rows = ptx::umma_desc(b + k * 128, hi);
    ptx::umma_f16_ta(d, at, rows, idesc, accumulate);
    ptx::umma_f16_ta(d, at + 16, rows, idesc, 1u);
  };
  step(0, fresh ? 0u : 1u);
  if (ksteps == MOST) {
#pragma unroll
    for (int k = 1; k < MOST; ++k) step(k, 1u);
  } else {
    for (int k = 1; k < ksteps; ++k) step(k, 1u);
  }
}
// 32 fp32 values of a row as two 16-bit terms each: the first ones in 16 columns, what their rounding
// left in the 16 behind them, so that they take the place of the 32 columns that they came from.
// kWeights: values that are not negative.
template <typename T, bool kWeights>
__device__ __forceinline__ void split32(uint32_t taddr, const float (&v)[32]) {
  uint32_t y[32];
#pragma unroll
  for (int j = 0; j < 16; ++j) {
    if constexpr (kWeights)
      mma::split2_weights<T>(v[2 * j], v[2 * j + 1], y[j], y[16 + j]);
    else
      mma::split2<T>(v[2 * j], v[2 * j + 1], y[j], y[16 + j]);
  }
  ptx::tmem_st_32x32b_x32(taddr, y);
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ void st_shared_v4(uint32_t at, const uint4& v) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(v.x), "r"(v.y), "r"(v.z),
               "r"(v.w)
               : "memory");
}

// What the units' rows leave for the join: a row's output over one cluster, in 24 bits a value (the
// upper three bytes of its fp32). Sign and exponent are whole, so that columns of a row may lie any
// factor apart, infinities beside them; what is dropped is at most 2^-16 of the value, against the
// 2^-12 that the last rounding of out may take from it (2^-9 with bf16). In 16 bits (fp16 under a power
// of two of the row's own) a column 2^-39 of the row's largest was lost; 4 bytes a value cost the prompt
// of cluster_attention_tiles.cu 90 us more than 2 did.
//
// 32 rows are stored as the warps write them, in segments of 32 columns (3 KB): the rows' upper halves,
// 64 bytes a row, then their third bytes, 32 a row. The 16-byte pieces of a row are permuted by the
// row's number, so that eight lanes that store a piece each meet different banks.
constexpr int kPartBytes = 3;
constexpr int kSegment = 32 * 32 * kPartBytes;
__device__ __forceinline__ uint32_t part_hi(int r, int j) {  // 16-byte piece j of the upper halves
  return static_cast<uint32_t>(r * 64 + ((j ^ (r >> 1 & 3)) << 4));
}
__device__ __forceinline__ uint32_t part_lo(int r, int j) {  // of the third bytes
  return static_cast<uint32_t>(2048 + r * 32 + ((j ^ (r >> 2 & 1)) << 4));
}
// One segment: the lane's 32 values of its row, to dst through the warp's buffer; the copy goes on while
// the warp does other things (the stores themselves, 16 bytes a lane to rows or to whole lines
// alike, held the warps for some 170 cycles each).
__device__ __forceinline__ void put_segment(uint32_t buf, const uint32_t (&v)[32], uint8_t* dst) {
  const int lane = threadIdx.x & 31;
  if (lane == 0) ptx::bulk_wait_read();  // the buffer's last copy
  __syncwarp();
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    uint32_t y[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] = __byte_perm(v[8 * j + 2 * e], v[8 * j + 2 * e + 1], 0x7632);
    st_shared_v4(buf + part_hi(lane, j), make_uint4(y[0], y[1], y[2], y[3]));
  }
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    uint32_t y[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int c = 16 * j + 4 * e;
      y[e] = __byte_perm(__byte_perm(v[c], v[c + 1], 0x51), __byte_perm(v[c + 2], v[c + 3], 0x51), 0x5410);
    }
    st_shared_v4(buf + part_lo(lane, j), make_uint4(y[0], y[1], y[2], y[3]));
  }
  ptx::fence_proxy_async_smem();
  __syncwarp();
  if (lane == 0) {
    ptx::bulk_store(dst, buf, kSegment);
    ptx::bulk_commit();
  }
}
// Eight columns of a row, from column 8 * j on, as a lane of the joins reads them.
struct Part8 {
  uint4 hi;
  uint2 lo;
};
template <int DP>
__device__ __forceinline__ Part8 load_part(const uint8_t* parts, int64_t n, int j) {
  const int r = static_cast<int>(n & 31);
  const uint8_t* seg = parts + (n >> 5) * (32 * DP * kPartBytes) + (j >> 2) * kSegment;
  Part8 p;
  p.hi = __ldcs(reinterpret_cast<const uint4*>(seg + part_hi(r, j & 3)));
  p.lo = __ldcs(reinterpret_cast<const uint2*>(seg + part_lo(r, (j & 3) >> 1) + (j & 1) * 8));
  return p;
}
// acc += f * the values. The byte that was dropped is filled with the one before it, which keeps
// zeros and infinities what they are and whose mean is that of the byte.
__device__ __forceinline__ void add_part(float (&acc)[8], const Part8& p, float f) {
  const uint32_t hi[4] = {p.hi.x, p.hi.y, p.hi.z, p.hi.w}, lo[2] = {p.lo.x, p.lo.y};
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const uint32_t b = 4 + (e & 3), h = (e & 1) * 2;
    acc[e] = fmaf(f, __uint_as_float(__byte_perm(hi[e >> 1], lo[e >> 2], (h + 1) << 12 | h << 8 | b << 4 | b)), acc[e]);
  }
}

// Registers of the warpgroup's threads from here on.
template <int N>
__device__ __forceinline__ void more_registers() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void fewer_registers() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

// Bounded wait of a whole warp; the same answer in every lane.
__device__ __forceinline__ bool warp_mbar_wait(const uint64_t* bar, uint32_t parity,
                                               const volatile int* abort) {
  return __all_sync(0xFFFFFFFFu, ptx::mbar_wait(ptx::smem_u32(bar), parity, abort));
}

__device__ __forceinline__ void tmem_ld_f32_x32(uint32_t taddr, float (&v)[32]) {
  uint32_t r[32];
  ptx::tmem_ld_32x32b_x32(taddr, r);
#pragma unroll
  for (int j = 0; j < 32; ++j) v[j] = __uint_as_float(r[j]);
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
  int64_t* count;        // units; their cost above 2^32
  int32_t* cum;          // cost of the units before each
  int32_t* start;        // first unit of each CTA, and their number
  int32_t* q_row;        // row of Q's map; the one past its last for a row that sees nothing
  int32_t* row_pos;      // last position that the row sees; -1: none, or no row
  int32_t* pair_row;     // (R, nq * top) unit row of a pair's first head; -1: no key
  int32_t* first_unit;   // (R, K) of clusters that have units
  int32_t* odd;          // a result is not finite (cluster_masked.cu)
  // for the gradients: row of dout's map, as q_row; lse to base 2 of the row; its delta and the power of
  // two of its dS, and per row of clusters the largest A (see Range), which cluster_attention_tiles_grad.cu sets
  int32_t* do_row;
  float *row_lse, *row_delta, *row_power, *largest;
  void* group_ws;
  int64_t units_max;
};
size_t carve_units(const Args& a, int64_t nq, bool grad, uint8_t* ws, UnitPlan* out);
// Groups sel of the queries [i0, i0 + nq), lists the units, fills the rows and shares the
// units among `ctas` CTAs. lse (batch, Hq, Nq) with rows of the gradients only.
int launch_units(const Args& a, int64_t i0, int64_t nq, const RowMap& rq, const UnitPlan& p, int ctas,
                 const float* lse, cudaStream_t stream);
constexpr int kMaxCtas = 1024;

// What the choice between the two forms weighs, with nq queries a round: keys of a cluster on
// average, (query, slot, head) rows, keys that the walk reads (of more than 8 heads, more than
// once), units, and the width of the tiles' columns, of 128.
struct FormWork {
  double keys, rows, reads, units, width;
};
FormWork form_work(const Args& a, int64_t nq);
// Whether the form by clusters can take nq queries at once, the scratch of their units' rows (nearly
// all there is) within `bytes`.
bool tiles_fit(const Args& a, int64_t nq, int64_t bytes);
inline int64_t unit_row_bytes(const Args& a) {  // the part, and up to eight words beside it
  return (a.D <= 64 ? 64 : 128) * kPartBytes + 32;
}
inline int64_t units_most(const Args& a, int64_t nq) {  // every cluster with pairs may end in one that is not full
  const int64_t pairs = nq * a.top;
  return static_cast<int64_t>(a.batch) * a.Hkv * (pairs * a.G / kUnitRows + std::min<int64_t>(a.K, pairs));
}

// A CTA's units [start[blockIdx.x], start[blockIdx.x + 1]) in turn. The next one is fetched while
// one is worked on, and nothing but its turn waits for it. Keys and values are loaded into two
// stages, load number `load` into stage load & 1; a unit of the same cluster as the one
// before it, whose steps both stages hold, uses them again.
struct UnitIter {
  const Unit* units;
  int n, total;
  uint32_t load;        // number of the unit's first step among the loads
  bool again, keep;     // the unit uses the loads of the one before; the next one will use its
  Unit un, next;

  __device__ __forceinline__ UnitIter(const Unit* u, const int32_t* start)
      : units(u), n(__ldg(start + blockIdx.x)), total(__ldg(start + blockIdx.x + 1)), load(0), again(false) {
    if (n < total) next = load_unit(units + n);
    open();
  }
  __device__ __forceinline__ void open() {
    keep = false;
    if (n >= total) return;
    un = next;
    if (n + 1 < total) next = load_unit(units + n + 1);
    const bool more = (un.nrows & Unit::kMore) != 0;
    un.nrows &= Unit::kMore - 1;
    keep = more && n + 1 < total && un.steps() <= 2;
  }
  __device__ __forceinline__ bool valid() const { return n < total; }
  __device__ __forceinline__ void advance() {
    if (!keep) load += un.steps();
    again = keep;
    ++n;
    open();
  }
};

// How a warp of the joins reads the parts of GP neighbouring heads of a query (the largest power
// of two up to 4 and G): eight lanes take 64 columns of a head's row, GP heads side by side, and 4 / GP
// slots of sel at once.
struct JoinLane {
  int piece, head, slot;  // of 8 columns; of the heads; of the slots
  __device__ __forceinline__ JoinLane(int gp) {
    const int lane = threadIdx.x & 31;
    piece = lane & 7;
    head = (lane >> 3) & (gp - 1);
    slot = (lane >> 3) / gp;
  }
};
inline int join_heads(int G) { return G >= 4 ? 4 : G >= 2 ? 2 : 1; }
// Eight values times f, rounded to T.
template <typename T>
__device__ __forceinline__ void store_out(T* out, const float (&v)[8], float f) {
  uint32_t y[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) y[e] = mma::pack2<T>(v[2 * e] * f, v[2 * e + 1] * f);
  *reinterpret_cast<uint4*>(out) = make_uint4(y[0], y[1], y[2], y[3]);
}

}  // namespace attn
}  // namespace fkc
