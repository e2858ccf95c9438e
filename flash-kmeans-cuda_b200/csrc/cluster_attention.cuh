// What the forward and backward kernels of attention over selected clusters share:
// the call's arguments, the walk over the keys of a query's clusters and the
// gathered shared-memory tiles.
#pragma once

#include <cstdint>

#include "fkc_internal.h"
#include "fkc_launch.cuh"
#include "fkc_mma.cuh"

namespace fkc {
namespace attn {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

struct Strides {
  int64_t b, h, n;  // elements between sequences, heads and positions
};

// Rows r = batch index * Hkv + kv head; Hq = Hkv * G.
struct Args {
  const void *q, *k, *v;
  Strides qs, ks, vs;
  const int32_t* sel;      // (R, Nq, top) cluster ids; outside [0, K): none
  const int32_t* order;    // (R, N) positions by cluster
  const int32_t* offsets;  // (R, K + 1)
  const int32_t* q_pos;    // (batch, Nq) or null: every key is visible
  int batch, Hq, Hkv, G, Nq, N, K, top, D;
  float scale;
};

// One cluster's slots, kept inside [0, N) whatever offsets holds.
__device__ __forceinline__ void cluster_span(const Args& a, int r, int c, int& s, int& e) {
  s = e = 0;
  if (c < 0 || c >= a.K) return;
  const int32_t* of = a.offsets + static_cast<int64_t>(r) * (a.K + 1) + c;
  s = min(max(of[0], 0), a.N);
  e = min(max(of[1], s), a.N);
}

// The concatenated keys of the clusters that one query selected, for one warp:
// pre[j] is the first place of the j-th cluster in the concatenation, at[j] its
// first slot in order. Lists live in shared memory, 2 * top + 1 words.
struct KeyList {
  int* pre;
  int* at;
  int total;  // keys in the concatenation

  __device__ __forceinline__ void build(const Args& a, int r, int i, int* buf) {
    const int lane = threadIdx.x & 31;
    pre = buf;
    at = buf + a.top + 1;
    const int32_t* sel = a.sel + (static_cast<int64_t>(r) * a.Nq + i) * a.top;
    int run = 0;
    for (int j0 = 0; j0 < a.top; j0 += 32) {
      const int j = j0 + lane;
      int s = 0, e = 0;
      if (j < a.top) cluster_span(a, r, sel[j], s, e);
      int inc = e - s;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xFFFFFFFFu, inc, o);
        if (lane >= o) inc += u;
      }
      if (j < a.top) {
        pre[j] = run + inc - (e - s);
        at[j] = s;
      }
      run += __shfl_sync(0xFFFFFFFFu, inc, 31);
    }
    if (lane == 0) pre[a.top] = run;
    total = run;
    __syncwarp();
  }

  // What order holds for place p (a lane's places ascend; cur is its cursor); -1 past the end.
  // Nothing here waits for the load: visible() does, at its use.
  __device__ __forceinline__ int key(const Args& a, const int32_t* order, int p, int& cur) const {
    if (p >= total) return -1;
    while (cur + 1 < a.top && p >= pre[cur + 1]) ++cur;
    return order[at[cur] + (p - pre[cur])];
  }
  // The key, or -1 where a query at pos does not see it.
  static __device__ __forceinline__ int visible(const Args& a, int row, int pos) {
    return row >= 0 && row < a.N && row <= pos ? row : -1;
  }
};

// Byte offset of 16-byte chunk c of row r in a tile of rows of DP 16-bit elements:
// the chunk index is xored with the row's low bits, so that the eight rows of an
// ldmatrix fall into eight different bank groups.
template <int DP>
__device__ __forceinline__ uint32_t tile_at(int r, int c) {
  return static_cast<uint32_t>(r * (DP * 2) + ((c ^ (r & 7)) << 4));
}

// A fragment (16 rows x 16 columns at column 16 * kk) of a row-major tile.
template <int DP>
__device__ __forceinline__ void load_a(uint32_t (&f)[4], uint32_t tile, int row0, int kk) {
  const int lane = threadIdx.x & 31;
  mma::ldmatrix_x4(f, tile + tile_at<DP>(row0 + (lane & 15), kk * 2 + (lane >> 4)));
}
// A fragment of the transposed tile: 16 columns (from 16 * md) x 16 rows.
template <int DP>
__device__ __forceinline__ void load_a_trans(uint32_t (&f)[4], uint32_t tile, int row0, int md) {
  const int lane = threadIdx.x & 31, m = lane >> 3;
  mma::ldmatrix_x4_trans(f, tile + tile_at<DP>(row0 + (lane & 7) + (m >> 1) * 8, md * 2 + (m & 1)));
}
// B fragments of two neighbouring 8-row groups (rows are the columns of B) at depth 16 * kk:
// f[0], f[1] of the first group, f[2], f[3] of the second.
template <int DP>
__device__ __forceinline__ void load_b(uint32_t (&f)[4], uint32_t tile, int row0, int kk) {
  const int lane = threadIdx.x & 31, m = lane >> 3;
  mma::ldmatrix_x4(f, tile + tile_at<DP>(row0 + (lane & 7) + (m >> 1) * 8, kk * 2 + (m & 1)));
}
// B fragments of two neighbouring groups of 8 tile columns (from 16 * nd), rows as depth:
// f[0], f[1] of the first group, f[2], f[3] of the second.
template <int DP>
__device__ __forceinline__ void load_b_trans(uint32_t (&f)[4], uint32_t tile, int row0, int nd) {
  const int lane = threadIdx.x & 31, m = lane >> 3;
  mma::ldmatrix_x4_trans(f, tile + tile_at<DP>(row0 + (lane & 7) + (m & 1) * 8, nd * 2 + (m >> 1)));
}

// 0 while all of x are finite (from a so_far of 0).
__device__ __forceinline__ float not_finite(float x, float so_far) { return fmaf(x, 0.f, so_far); }

// The 16-bit operands P and dS of fp16 inputs, whose normal range ends at 2^-14: P (at most 1) is
// held as 2^14 P, and dS under a power of two that the sum A of P |dP| over a row's keys gives, since
// |dS| <= 2 A: power(A) * A lies in [2^13, 2^14), or below where A is less than 2^-47 (a product of
// two fp16 rows, 2^39 at most, times the power stays finite). dQ has a power per row, dK one per row of
// clusters, from the largest A of its queries. (With dout near 1e-4 and 512 keys, dS below 2^-24 made
// dQ off by 0.004 of its norm.) bf16 has fp32's exponents and needs neither.
template <typename T>
struct Range {
  static constexpr bool kNarrow = std::is_same<T, __half>::value;
  static constexpr int kShift = kNarrow ? 14 : 0;  // of P
  static __host__ __device__ constexpr float unshift() { return kNarrow ? 0x1p-14f : 1.f; }
};
__device__ __forceinline__ float power(float A) {  // 1 where A is not finite
  const int e = static_cast<int>(__float_as_uint(A) >> 23);
  return __uint_as_float(static_cast<uint32_t>(e >= 255 ? 127 : min(267 - e, 127 + 60)) << 23);
}
__device__ __forceinline__ float inverse_power(float p) {
  return __uint_as_float((254u << 23) - __float_as_uint(p));
}
// The largest A of a row of clusters; A is not negative, so its bits are ordered as it is.
__device__ __forceinline__ void note_largest(float* word, float A) {
  if (A > *reinterpret_cast<volatile float*>(word)) atomicMax(reinterpret_cast<int*>(word), __float_as_int(A));
}

int sm_count();  // of the current device

// Launchers (cluster_select.cu, cluster_attention.cu, cluster_attention_grad.cu); dtype is
// FKC_DTYPE_F16 or FKC_DTYPE_BF16. out, dout and the gradients are contiguous.
size_t select_workspace_bytes(int64_t R, int64_t Nq, int64_t K);
int launch_select(const Args& a, const void* centroids, const float* bias, double scale, int dtype,
                  int32_t* sel, void* ws, cudaStream_t stream);
int split_count(const Args& a);  // warps that share the keys of a query in the walk
size_t forward_workspace_bytes(const Args& a);
int launch_forward(const Args& a, int dtype, void* out, float* lse, void* ws, cudaStream_t stream);
// The form by clusters (cluster_attention_tiles.cu), taken where use_tiles says so.
bool use_tiles(const Args& a);
size_t tiles_forward_workspace_bytes(const Args& a);
int launch_tiles_forward(const Args& a, int dtype, void* out, float* lse, void* ws,
                         cudaStream_t stream);
bool use_tiles_grad(const Args& a);
size_t tiles_backward_workspace_bytes(const Args& a);
int launch_tiles_backward(const Args& a, int dtype, const float* lse, float* delta, const void* dout,
                          void* dq, void* dk, void* dv, void* ws, cudaStream_t stream);
// After the kernels above, where they set *odd: results that are not finite, from what their rows
// see alone (cluster_masked.cu). Forward: rows is out. Gradients (dout given): rows is dq.
int launch_again(const Args& a, int dtype, const int32_t* odd, const float* lse, const float* delta,
                 const void* dout, void* rows, const int32_t* inv_order, const int32_t* inv_offsets,
                 void* dk, void* dv, cudaStream_t stream);
size_t backward_workspace_bytes(const Args& a);
int launch_backward(const Args& a, int dtype, const float* lse, const void* dout, void* dq,
                    void* dk, void* dv, void* ws, cudaStream_t stream);

}  // namespace attn
}  // namespace fkc
