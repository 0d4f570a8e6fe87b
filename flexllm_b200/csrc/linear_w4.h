// Products with 4-bit weights: the call, shared by its kernels (linear_w4.cu: few tokens and fp32, linear_w4_tc.cu: tensor cores).
#pragma once
#include "float_common.cuh"

namespace flexllm {

struct W4Call {
    const void* a; long lda;
    const uint8_t* w;
    const void* scale; int scale_f32;
    const uint8_t* zero;
    int group;
    const float* bias;
    int M, N, K;
    void* y; long ldy; int y_f32;
};
int linear_w4_tc(const W4Call& c, cudaStream_t st);      // bf16

__device__ __forceinline__ uint32_t and_or(uint32_t a, uint32_t mask, uint32_t bits) {
    uint32_t r;
    asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(r) : "r"(a), "r"(mask), "r"(bits));
    return r;
}
__device__ __forceinline__ uint32_t sub_bf2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("sub.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
__device__ __forceinline__ uint32_t pick(uint32_t a, uint32_t b, uint32_t sel) {
    uint32_t r;
    asm("prmt.b32 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(sel));
    return r;
}
// Nibbles i and i + 4 of a word as bf16, less the zero point: 0x4300 | q is 128 + q, and z2 holds 128 + z twice.
__device__ __forceinline__ uint32_t weights2(uint32_t word, int i, uint32_t z2) { return sub_bf2(and_or(word >> (4 * i), 0x000f000fu, 0x43004300u), z2); }
__device__ __forceinline__ uint32_t zero2(uint32_t z) { return (z & 15u) * 0x10001u + 0x43004300u; }

}  // namespace flexllm
