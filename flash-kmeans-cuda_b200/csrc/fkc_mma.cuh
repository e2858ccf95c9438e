// Warp-level matrix instructions (m16n8k16, fp32 accumulators), the shared-memory
// loads that feed them and 16-byte asynchronous copies, for kernels whose operand
// rows are gathered one by one: a tile of 8 heads is far below the 64 rows that a
// tcgen05.mma takes at least, and its operands could not come from registers.
//
// Fragment layouts, lane = 4 * g + t: A (16 x 16, row-major) a0 = (g, 2t), a1 =
// (g + 8, 2t), a2 = (g, 2t + 8), a3 = (g + 8, 2t + 8); B (16 x 8) b0 = (2t, g), b1 =
// (2t + 8, g); C (16 x 8) c0, c1 = (g, 2t), (g, 2t + 1), c2, c3 = the same of row g + 8.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>
#include <type_traits>

namespace fkc {
namespace mma {

template <typename T>
__device__ __forceinline__ void m16n8k16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                         uint32_t b1) {
  if constexpr (std::is_same<T, __half>::value)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9},"
        " {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7},"
        " {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Four 8 x 8 matrices; lane l gives the address of row l % 8 of matrix l / 8.
__device__ __forceinline__ void ldmatrix_x4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}

// The transpose of an 8 x 8 matrix held over the warp.
__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

// Two fp32 values rounded to nearest, lo in the low half.
template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if constexpr (std::is_same<T, __half>::value) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}
template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t v) {
  if constexpr (std::is_same<T, __half>::value)
    return __half22float2(*reinterpret_cast<const __half2*>(&v));
  else
    return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&v));
}

// 16 bytes to shared memory; zeros, and no read, when !valid.
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool valid) {
  const uint32_t bytes = valid ? 16u : 0u;
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes)
               : "memory");
}
__device__ __forceinline__ void cp_async_commit() {
  asm volatile("cp.async.commit_group;" ::: "memory");
}
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// The same as two terms: rounded, and what that left, rounded (2^-18 of the value with bf16).
template <typename T>
__device__ __forceinline__ void split2(float lo, float hi, uint32_t& first, uint32_t& second) {
  first = pack2<T>(lo, hi);
  const float2 f = unpack2<T>(first);
  second = pack2<T>(lo - f.x, hi - f.y);
}

// The same for values that are not negative, as terms that are not either: the first is cut off below
// the value (2^-16 of it less, so that a value of 16 bits is too), and the second positive wherever the
// value is, so that a product with an infinity is that infinity and not a sum of two of either sign.
template <typename T>
__device__ __forceinline__ void split2_weights(float lo, float hi, uint32_t& first, uint32_t& second) {
  constexpr float kBelow = 1.f - 0x1p-16f;
  if constexpr (std::is_same<T, __half>::value) {
    asm("cvt.rz.f16x2.f32 %0, %1, %2;" : "=r"(first) : "f"(hi * kBelow), "f"(lo * kBelow));
    const float2 f = unpack2<T>(first);
    second = pack2<T>(lo - f.x, hi - f.y);
  } else {
    const uint32_t x = __float_as_uint(lo * kBelow), y = __float_as_uint(hi * kBelow);
    first = __byte_perm(x, y, 0x7632);
    second = pack2<T>(lo - __uint_as_float(x & 0xFFFF0000u), hi - __uint_as_float(y & 0xFFFF0000u));
  }
}

}  // namespace mma
}  // namespace fkc
