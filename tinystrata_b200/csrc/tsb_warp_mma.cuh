// tsb_warp_mma.cuh - warp-level matrix instructions and the typed loads and stores of the serving-step operators
// (tsb_cache.cu, tsb_delta.cu).
//
// Those kernels keep their running state (softmax statistics, output rows, the recurrent state) in the registers of one
// warp between matrix products whose result feeds the next product's left operand.  mma.sync's accumulator layout is
// its left operand's layout, so the chain needs no trip through shared or tensor memory; a tcgen05 tile (64 or 128
// rows, read back from tensor memory) would be mostly padding at the 8..64 rows these products have.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cstdint>

namespace tsb {

enum : int { E_F32 = 0, E_F16 = 1, E_BF16 = 30 };   // element types by their ggml ids

__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_f16(float4& c, const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c.x), "+f"(c.y), "+f"(c.z), "+f"(c.w)
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// The same from zero.
__device__ __forceinline__ void mma_f16_zero(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
}
__device__ __forceinline__ void mma_s8_zero(int (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=r"(c[0]), "=r"(c[1]), "=r"(c[2]), "=r"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "r"(0));
}
// 16 x 8 x 32 on int8 (a lane's words: columns 4 (lane % 4) .. + 3 and 16 more on).
__device__ __forceinline__ void mma_s8(int (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// An 8x8 matrix of 16-bit values held two a lane by rows, transposed.
__device__ __forceinline__ uint32_t transpose8(uint32_t a) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(a));
    return r;
}
// Four 8x8 matrices of 16-bit values; lane l gives the address of row l % 8 of matrix l / 8 (16 bytes each).  Volatile:
// ordered against the barrier waits and synchronisations that make the rows visible.
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr));
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr));
}

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ float load_elem(const void* p, int64_t i, int type) {
    if (type == E_F32) return ((const float*) p)[i];
    if (type == E_F16) return __half2float(((const __half*) p)[i]);
    return __bfloat162float(((const __nv_bfloat16*) p)[i]);
}
__device__ __forceinline__ void store_elem(void* p, int64_t i, int type, float v) {
    if (type == E_F32) ((float*) p)[i] = v;
    else if (type == E_F16) ((__half*) p)[i] = __float2half_rn(v);
    else ((__nv_bfloat16*) p)[i] = __float2bfloat16_rn(v);
}
__host__ __device__ constexpr int elem_bytes(int type) { return type == E_F32 ? 4 : 2; }

// 8 values from element i on; `wide`: 16-byte aligned (the caller checked base and strides).
__device__ __forceinline__ void load8(float (&x)[8], const void* p, int64_t i, int type, bool wide) {
    if (!wide) {
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = load_elem(p, i + j, type);
        return;
    }
    if (type == E_F32) {
        const float4 a = *(const float4*) ((const float*) p + i), b = *(const float4*) ((const float*) p + i + 4);
        x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
        return;
    }
    const uint4 w = *(const uint4*) ((const uint16_t*) p + i);
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if (type == E_F16) {
            const float2 f = __half22float2(*(const __half2*) &u[j]);
            x[2 * j] = f.x, x[2 * j + 1] = f.y;
        } else {
            x[2 * j] = __uint_as_float(u[j] << 16), x[2 * j + 1] = __uint_as_float(u[j] & 0xffff0000u);
        }
    }
}

}  // namespace tsb
