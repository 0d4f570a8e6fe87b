// Products with 4-bit weights: the call, shared by its kernels (linear_w4.cu: few tokens, linear_w4_tc.cu: tensor cores).
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
    int* error_flag;
};
// Zero points of more than four bits (`seen`: those of a thread, one on top of the other) are used without the upper ones, and reported.
__device__ __forceinline__ void check_zeros(uint32_t seen, int* flag) { if ((seen & 0xf0f0f0f0u) && flag) atomicOr(flag, 2); }
int linear_w4_tc(const W4Call& c, bool f32, cudaStream_t st);

__device__ __forceinline__ uint32_t pick(uint32_t a, uint32_t b, uint32_t sel) {
    uint32_t r;
    asm("prmt.b32 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(sel));
    return r;
}
// 8 fp32 activations as the pairs (0,4) (1,5) (2,6) (3,7) of their three bf16 parts: the upper 16 bits of a number, of what they leave, and of what that
// leaves, eight significant bits each. (Cut, since the nearest bf16 of a number above 3.39e38 is an infinity.) An infinity leaves nothing, a NaN a NaN.
struct Eight { uint4 part[3]; };
__device__ __forceinline__ Eight eight(float (&f)[8]) {
    Eight r;
#pragma unroll
    for (int k = 0; k < 3; k++) {
        uint32_t w[4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            w[j] = pick(__float_as_uint(f[j]), __float_as_uint(f[j + 4]), 0x7632);
            f[j] = fabsf(f[j]) == INFINITY ? 0.0f : f[j] - bf_lo(w[j]);
            f[j + 4] = fabsf(f[j + 4]) == INFINITY ? 0.0f : f[j + 4] - bf_hi(w[j]);
        }
        r.part[k] = make_uint4(w[0], w[1], w[2], w[3]);
    }
    return r;
}

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
// Nibbles i and i + 4 of a word as bf16, less the zero point: 0x4300 | q is 128 + q, and z2 holds 128 + z twice.
__device__ __forceinline__ uint32_t weights2(uint32_t word, int i, uint32_t z2) { return sub_bf2(and_or(word >> (4 * i), 0x000f000fu, 0x43004300u), z2); }
__device__ __forceinline__ uint32_t zero2(uint32_t z) { return (z & 15u) * 0x10001u + 0x43004300u; }

}  // namespace flexllm
