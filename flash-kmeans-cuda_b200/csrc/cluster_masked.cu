// Attention results that masks cut through.
//
// A tile multiplies what one of its rows does not see by zeros, which is no product where the
// other factor is an infinity or a NaN: another row of the tile may see that key, this one must
// not. So where q_pos is given, the kernels that work in such tiles report a result that is not
// finite (an fma per value that is in a register anyway), and again_kernel, their last launch,
// forms every such result again from what its row alone sees, a warp a row. Without a report
// it ends at once. Such values are rare; if they are the row's
// own, its sum is given up as soon as all of it is NaN, so that a run whose values have all become
// NaN stays usable. (Formed where it is found, in the joins, the code cost the usual
// case 28 of 486 us of a prefill and 75 of 497 us of a training step in registers.)
#include <algorithm>

#include "cluster_attention.cuh"

namespace fkc {
namespace attn {
namespace {

constexpr int kWarps = 16;

template <typename T>
__device__ __forceinline__ bool row_is_odd(const T* row, int D) {
  float odd = 0.f;
  for (int d = threadIdx.x & 31; d < D; d += 32) odd = not_finite(static_cast<float>(row[d]), odd);
  return __any_sync(0xFFFFFFFFu, odd != 0.f);
}
// A warp's sum over the columns of two rows.
template <typename T>
__device__ __forceinline__ float dot(const T* x, const T* y, int D) {
  float s = 0.f;
  for (int d = threadIdx.x & 31; d < D; d += 32) s = fmaf(static_cast<float>(x[d]), static_cast<float>(y[d]), s);
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, o);
  return s;
}
// acc[j] += w * row[lane + 32 j]; true if all that the lanes hold is NaN.
template <typename T>
__device__ __forceinline__ bool add_row(float (&acc)[4], const T* row, float w, int D) {
  bool lost = true;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int d = (threadIdx.x & 31) + 32 * j;
    if (d >= D) continue;
    acc[j] = fmaf(w, static_cast<float>(row[d]), acc[j]);
    lost = lost && isnan(acc[j]);
  }
  return __all_sync(0xFFFFFFFFu, lost);
}
template <typename T>
__device__ __forceinline__ void put_row(T* row, const float (&acc)[4], float scale, int D) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int d = (threadIdx.x & 31) + 32 * j;
    if (d < D) row[d] = static_cast<T>(acc[j] * scale);
  }
}

// Without dout, rows are those of out: sum of P V. With it, those of dq (or null), scale * sum of
// dS K, and dk, dv (or null) follow, for which inv lists the entries of sel by cluster.
template <typename T>
__global__ void __launch_bounds__(32 * kWarps) again_kernel(Args a, const int32_t* __restrict__ odd,
                                                            const float* __restrict__ lse,
                                                            const float* __restrict__ delta,
                                                            const T* __restrict__ dout, T* rows,
                                                            const int32_t* __restrict__ inv_order,
                                                            const int32_t* __restrict__ inv_offsets,
                                                            T* dk, T* dv) {
  pdl_wait();
  if (*odd == 0) return;
  const int64_t first = static_cast<int64_t>(blockIdx.x) * kWarps + (threadIdx.x >> 5);
  const int64_t step = static_cast<int64_t>(gridDim.x) * kWarps;
  const T *q = static_cast<const T*>(a.q), *k = static_cast<const T*>(a.k), *v = static_cast<const T*>(a.v);
  const float sc = a.scale * kLog2e;
  const int64_t nrows = rows != nullptr ? static_cast<int64_t>(a.batch) * a.Hq * a.Nq : 0;
  for (int64_t at = first; at < nrows; at += step) {
    if (!row_is_odd(rows + at * a.D, a.D)) continue;
    const int i = static_cast<int>(at % a.Nq), h = static_cast<int>(at / a.Nq % a.Hq);
    const int b = static_cast<int>(at / a.Nq / a.Hq), hk = h / a.G, r = b * a.Hkv + hk;
    const T* qr = q + b * a.qs.b + h * a.qs.h + i * a.qs.n;
    const T *kr = k + b * a.ks.b + hk * a.ks.h, *vr = v + b * a.vs.b + hk * a.vs.h;
    const int pos = a.q_pos[static_cast<int64_t>(b) * a.Nq + i];
    const int32_t* sel = a.sel + (static_cast<int64_t>(r) * a.Nq + i) * a.top;
    const float ls = lse[at] * kLog2e, dl = dout != nullptr ? delta[at] : 0.f;
    float acc[4] = {0.f, 0.f, 0.f, 0.f};
    bool lost = false;
    for (int j = 0; j < a.top && !lost; ++j) {
      int s, end;
      cluster_span(a, r, sel[j], s, end);
      for (; s < end && !lost; ++s) {
        const int n = a.order[static_cast<int64_t>(r) * a.N + s];
        if (n < 0 || n >= a.N || n > pos) continue;
        const T *kn = kr + n * a.ks.n, *vn = vr + n * a.vs.n;
        const float p = exp2f(fmaf(dot(qr, kn, a.D), sc, -ls));
        lost = dout == nullptr ? add_row(acc, vn, p, a.D)
                               : add_row(acc, kn, p * (dot(dout + at * a.D, vn, a.D) - dl), a.D);
      }
    }
    put_row(rows + at * a.D, acc, dout == nullptr ? 1.f : a.scale, a.D);
  }
  if (dk == nullptr) return;
  const int64_t slots = static_cast<int64_t>(a.batch) * a.Hkv * a.N;
  for (int64_t x = first; x < slots; x += step) {
    const int n = a.order[x], r = static_cast<int>(x / a.N), slot = static_cast<int>(x - static_cast<int64_t>(r) * a.N);
    if (n < 0 || n >= a.N) continue;
    const int64_t at = (static_cast<int64_t>(r) * a.N + n) * a.D;
    const bool odd_k = row_is_odd(dk + at, a.D), odd_v = row_is_odd(dv + at, a.D);
    if (!odd_k && !odd_v) continue;
    const int b = r / a.Hkv, hk = r - b * a.Hkv;
    const T *kn = k + b * a.ks.b + hk * a.ks.h + n * a.ks.n, *vn = v + b * a.vs.b + hk * a.vs.h + n * a.vs.n;
    const int32_t* list = inv_order + static_cast<int64_t>(r) * a.Nq * a.top;
    float gk[4] = {0.f, 0.f, 0.f, 0.f}, gv[4] = {0.f, 0.f, 0.f, 0.f};
    bool lost = false;
    for (int c = 0; c < a.K && !lost; ++c) {
      int s, end;
      cluster_span(a, r, c, s, end);
      if (slot < s || slot >= end) continue;
      const int32_t* of = inv_offsets + static_cast<int64_t>(r) * (a.K + 1) + c;
      for (int e = of[0]; e < of[1] && !lost; ++e) {
        const int i = list[e] / a.top;
        if (n > a.q_pos[static_cast<int64_t>(b) * a.Nq + i]) continue;
        for (int g = 0; g < a.G && !lost; ++g) {
          const int h = hk * a.G + g;
          const int64_t row = (static_cast<int64_t>(b) * a.Hq + h) * a.Nq + i;
          const T *qr = q + b * a.qs.b + h * a.qs.h + i * a.qs.n, *gr = dout + row * a.D;
          const float p = exp2f(fmaf(dot(qr, kn, a.D), sc, -lse[row] * kLog2e));
          const bool lost_k = add_row(gk, qr, p * (dot(gr, vn, a.D) - delta[row]), a.D);
          lost = add_row(gv, gr, p, a.D) && lost_k;
        }
      }
    }
    put_row(dk + at, gk, a.scale, a.D);
    put_row(dv + at, gv, 1.f, a.D);
  }
}

template <typename T>
int again_typed(const Args& a, const int32_t* odd, const float* lse, const float* delta, const void* dout,
                void* rows, const int32_t* inv_order, const int32_t* inv_offsets, void* dk, void* dv,
                cudaStream_t stream) {
  return launch_pdl(again_kernel<T>, dim3(sm_count()), dim3(32 * kWarps), 0, stream, a, odd, lse, delta,
                    static_cast<const T*>(dout), static_cast<T*>(rows), inv_order, inv_offsets,
                    static_cast<T*>(dk), static_cast<T*>(dv));
}

}  // namespace

int launch_again(const Args& a, int dtype, const int32_t* odd, const float* lse, const float* delta,
                 const void* dout, void* rows, const int32_t* inv_order, const int32_t* inv_offsets,
                 void* dk, void* dv, cudaStream_t stream) {
  if (a.q_pos == nullptr) return FKC_OK;  // every row of a tile sees all of its keys
  return dtype == FKC_DTYPE_F16
             ? again_typed<__half>(a, odd, lse, delta, dout, rows, inv_order, inv_offsets, dk, dv, stream)
             : again_typed<__nv_bfloat16>(a, odd, lse, delta, dout, rows, inv_order, inv_offsets, dk, dv, stream);
}

}  // namespace attn
}  // namespace fkc
