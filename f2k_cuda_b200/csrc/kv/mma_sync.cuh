// Warp-level matrix pieces of the token kernel: ldmatrix, m16n8k16 products and packing for bf16 and fp16.
#pragma once

#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

namespace f2k {

__device__ __forceinline__ void ldmatrix_x4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}

// An 8 x 8 matrix of 16-bit elements, two to a lane, transposed across the warp.
__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t w) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(w));
    return r;
}

template <class T> struct Half16;      // what differs between the 16-bit types
template <> struct Half16<__nv_bfloat16> {
    static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
        uint32_t r;
        asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
        return r;
    }
    static __device__ __forceinline__ float lo(uint32_t w) { return __uint_as_float(w << 16); }
    static __device__ __forceinline__ float hi(uint32_t w) { return __uint_as_float(w & 0xFFFF0000u); }
    static __device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
};
template <> struct Half16<__half> {
    static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
        uint32_t r;
        asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
        return r;
    }
    static __device__ __forceinline__ float lo(uint32_t w) { return __half2float(__ushort_as_half((unsigned short)(w & 0xFFFFu))); }
    static __device__ __forceinline__ float hi(uint32_t w) { return __half2float(__ushort_as_half((unsigned short)(w >> 16))); }
    static __device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
};

// Two e4m3 values (the low 16 bits of w) as two fp16, exactly.
__device__ __forceinline__ uint32_t f16x2_of_e4m3x2(uint32_t w) {
    uint32_t r;
    asm("{\n\t.reg .b16 x;\n\tcvt.u16.u32 x, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, x;\n\t}" : "=r"(r) : "r"(w));
    return r;
}

// What scores over e4m3 keys are multiplied by, never below the smallest normal number: as 0 it would make NaN of a masked score's
// -inf. Scores of fp16 products are below 2^33, so with a factor this small their weights are all alike.
__device__ __forceinline__ float score_factor(float scale_log2, const float* k_scale, int head) {
    const float c = k_scale ? scale_log2 * k_scale[head] : scale_log2;
    return c < 1.17549435e-38f ? 1.17549435e-38f : c;
}
// bf16 queries over e4m3 keys: the exponent field f of the power of two 2^(f - 127) that brings a row's largest element `top` into
// [2^14, 2^15), for the products in fp16. An infinite one is left as it is, and a row next to nothing is not brought further
// up than its factor c of the scores can go down by the same power and stay normal: what is lost in front of such a factor has
// no weight.
__device__ __forceinline__ unsigned fp16_row_power(float top, float c) {
    const unsigned e = __float_as_uint(top) >> 23, least = __float_as_uint(c) >> 23;
    return e == 255u ? 127u : min(min(253u, 268u - e), least + 126u);
}

}  // namespace f2k
