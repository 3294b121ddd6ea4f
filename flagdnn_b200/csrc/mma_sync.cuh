// Warp-wide products and the copies and loads that feed them, shared by the gated delta rule and the products of few rows.
#pragma once
#include <stdint.h>

#include <type_traits>

#include "conv_convert.cuh"

namespace fdnn {

// D += A B, 16 x 8 x 16.  A: rows lane / 4 (+ 8 in a[1], a[3]), pairs of k at 2 (lane % 4) (+ 8 in a[2], a[3]); B: column lane / 4, pairs
// of k likewise; D: rows lane / 4 (+ 8 in d[2], d[3]), columns 2 (lane % 4) and the next.
// fp32: the same of 16 x 8 x 8 in TF32, A at (row, k = lane % 4), (row + 8, k), (row, k + 4), (row + 8, k + 4), B at k = lane % 4, + 4.
template <typename T>
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<T, __half>::value)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else if constexpr (std::is_same<T, __nv_bfloat16>::value)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Four 8 x 8 matrices of 16-bit values, 16-byte rows at each lane's address; TRANS: transposed.
template <bool TRANS>
__device__ __forceinline__ void ldmatrix(uint32_t (&r)[4], uint32_t at) {
  if constexpr (TRANS)
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
  else
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void copy16(uint32_t to, const void* from, int bytes) {   // the rest of the 16 is zeros
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(bytes) : "memory");
}
// fp32 as a TF32 number, rounded to nearest (by the integer unit: the conversion's instruction takes as long as the products), and what it
// leaves, of either sign, whose last bits the tensor core does not read.  The first part is finite: the largest numbers do not become infinite,
// and an infinity or NaN is all in the second.
__device__ __forceinline__ void two_parts(float v, uint32_t& hi, uint32_t& lo) {
  constexpr float kLargest = 3.4011621342146535e38f;   // of TF32: 2^127 (2 - 2^-10)
  float h;
  asm("min.xorsign.abs.f32 %0, %1, %2;" : "=f"(h) : "f"(__uint_as_float((__float_as_uint(v) + 0x1000u) & 0xffffe000u)), "f"(kLargest));
  hi = __float_as_uint(h);
  lo = __float_as_uint(v - h);
}

}  // namespace fdnn
