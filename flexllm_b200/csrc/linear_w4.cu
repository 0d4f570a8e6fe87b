// Products with 4-bit weights, one scale and zero point per group of the inner index:
//   y[m][n] = sum_groups s[n][g] * sum_{k in g} a[m][k] (q[n][k] - z[n][g])
// HBM bound for few tokens: half a byte per weight. Weights stream from memory into the registers of the lanes that multiply them: a warp has
// 16 rows on the 16-row side of bf16 warp MMAs and 8 tokens per MMA on the other. q - z is an integer of five bits, exact in bf16, and sums
// over a group stay in the MMA's fp32 accumulators; the scale multiplies them in fp32, so no weight is ever rounded. fp32 activations are
// cut into three bf16 parts of eight bits each, which hold them to the last bit, at three MMAs instead of one.
//
// Two nibbles j and j + 4 of a word become a pair of bf16 in three instructions (shift, mask and exponent at once: 0x4300 | q is 128 + q, one
// subtraction of 128 + z). The inner index may go through the MMA in any order, the same one in both operands: a lane's words are as they lie
// in memory, and the activations are put into that order on their way into shared memory.
#include "float_common.cuh"

namespace flexllm {

namespace {

struct W4Args {
    const void* a; long lda;
    const uint8_t* w;
    const void* scale; int scale_f32;
    const uint8_t* zero;
    int group;
    const float* bias;
    int M, N, K;
    void* y; long ldy; int y_f32;
    int ks;                                // warps of a CTA along K
    int kc;                                // inner elements staged at a time
};
constexpr int W4_WARPS = 8;

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
template <int VW> struct Words { uint32_t v[VW]; };
template <int VW> __device__ __forceinline__ Words<VW> load_words(const uint8_t* p) {
    Words<VW> r;
    if (VW == 4) asm("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(r.v[0]), "=r"(r.v[1 % VW]), "=r"(r.v[2 % VW]), "=r"(r.v[3 % VW]) : "l"(p));
    else if (VW == 2) asm("ld.global.nc.v2.u32 {%0, %1}, [%2];" : "=r"(r.v[0]), "=r"(r.v[1 % VW]) : "l"(p));
    else asm("ld.global.nc.u32 %0, [%1];" : "=r"(r.v[0]) : "l"(p));
    return r;
}

// 8 activations k .. k + 7 as the bf16 pairs (0,4) (1,5) (2,6) (3,7), PL parts
template <int PL> struct Eight { uint4 part[PL]; };
__device__ __forceinline__ Eight<1> eight(const bf16* p) {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    Eight<1> r;
    r.part[0] = make_uint4(pick(v.x, v.z, 0x5410), pick(v.x, v.z, 0x7632), pick(v.y, v.w, 0x5410), pick(v.y, v.w, 0x7632));
    return r;
}
__device__ __forceinline__ Eight<3> eight(const float* p) {
    float f[8];
    load8(p, f);
    Eight<3> r;
#pragma unroll
    for (int k = 0; k < 3; k++) {
        r.part[k] = make_uint4(bf_pack(f[0], f[4]), bf_pack(f[1], f[5]), bf_pack(f[2], f[6]), bf_pack(f[3], f[7]));
        const uint32_t w[4] = {r.part[k].x, r.part[k].y, r.part[k].z, r.part[k].w};
#pragma unroll
        for (int j = 0; j < 4; j++) {
            // what the part leaves; nothing of an infinity or NaN (the first part carries it)
            f[j] = fabsf(f[j]) <= 3.0e38f ? f[j] - bf_lo(w[j]) : 0.0f;
            f[j + 4] = fabsf(f[j + 4]) <= 3.0e38f ? f[j + 4] - bf_hi(w[j]) : 0.0f;
        }
    }
    return r;
}

// VW words per lane and row: a quad of lanes covers 32 VW elements of one group. MT tiles of 8 tokens.
template <class T, int VW, int MT>
__global__ void __launch_bounds__(W4_WARPS * 32, 2) linear_w4_kernel(const __grid_constant__ W4Args p) {
    constexpr int PL = sizeof(T) == 2 ? 1 : 3;
    constexpr int BK = 32 * VW;                            // elements of a block
    constexpr int U = 4 / VW;                              // blocks per step: four words per lane and row
    extern __shared__ __align__(16) uint8_t x_sm[];        // [PL][tokens][kc] bf16, pitch of 64 bytes more than a multiple of 128
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, lr = lane >> 2, lc = lane & 3;
    const int m0 = blockIdx.y * 64, Mb = min(p.M - m0, 8 * MT);
    const int kw = warp % p.ks, rt = blockIdx.x * (W4_WARPS / p.ks) + warp / p.ks;
    const int n_lo = rt * 16 + lr, n_hi = n_lo + 8;
    const int groups = p.K / p.group;
    const uint8_t* w_lo = p.w + (long)min(n_lo, p.N - 1) * (p.K / 2) + lc * 4 * VW;
    const uint8_t* w_hi = p.w + (long)min(n_hi, p.N - 1) * (p.K / 2) + lc * 4 * VW;
    const long g_lo = (long)min(n_lo, p.N - 1) * groups, g_hi = (long)min(n_hi, p.N - 1) * groups;
    auto scale_at = [&](long i) { return p.scale_f32 ? ((const float*)p.scale)[i] : to_f(((const bf16*)p.scale)[i]); };
    // 128 + z, twice
    auto zero_at = [&](long i) { return (p.zero ? (uint32_t)(p.zero[i] & 15u) : 8u) * 0x10001u + 0x43004300u; };
    float acc[MT][4];
#pragma unroll
    for (int t = 0; t < MT; t++)
#pragma unroll
        for (int i = 0; i < 4; i++) acc[t][i] = 0.0f;
    pdl_sync();
    for (int k0 = 0; k0 < p.K; k0 += p.kc) {
        const int kc = min(p.kc, p.K - k0), pitch = p.kc * 2 + ((p.kc & 63) ? 0 : 64);
        if (k0) __syncthreads();
        for (int e = tid; e < Mb * (kc / 8); e += W4_WARPS * 32) {
            const int m = e / (kc / 8), k = (e - m * (kc / 8)) * 8;
            const Eight<PL> x = eight((const T*)p.a + (long)(m0 + m) * p.lda + k0 + k);
            const int blk = k / BK, c = (k % BK) / (8 * VW), j = k % (8 * VW) / 8;
#pragma unroll
            for (int q = 0; q < PL; q++)
                *reinterpret_cast<uint4*>(x_sm + (long)(q * Mb + m) * pitch + (blk * BK + j * 32 + c * 8) * 2) = x.part[q];
        }
        __syncthreads();
        const int nb = kc / BK, b_beg = nb * kw / p.ks, b_end = nb * (kw + 1) / p.ks;
        for (int b0 = b_beg; b0 < b_end; b0 += U) {
            Words<VW> wl[U], wh[U];
            float sl[U], sh[U];
            uint32_t zl[U], zh[U];
#pragma unroll
            for (int u = 0; u < U; u++) {
                const int b = min(b0 + u, b_end - 1), k = k0 + b * BK;
                wl[u] = load_words<VW>(w_lo + k / 2); wh[u] = load_words<VW>(w_hi + k / 2);
                sl[u] = scale_at(g_lo + k / p.group); sh[u] = scale_at(g_hi + k / p.group);
                zl[u] = zero_at(g_lo + k / p.group); zh[u] = zero_at(g_hi + k / p.group);
            }
#pragma unroll
            for (int u = 0; u < U; u++) {
                if (b0 + u >= b_end) break;
                float part[MT][4];
#pragma unroll
                for (int t = 0; t < MT; t++)
#pragma unroll
                    for (int i = 0; i < 4; i++) part[t][i] = 0.0f;
#pragma unroll
                for (int j = 0; j < VW; j++) {
                    uint32_t al[4], ah[4];
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        al[i] = sub_bf2(and_or(wl[u].v[j] >> (4 * i), 0x000f000fu, 0x43004300u), zl[u]);
                        ah[i] = sub_bf2(and_or(wh[u].v[j] >> (4 * i), 0x000f000fu, 0x43004300u), zh[u]);
                    }
#pragma unroll
                    for (int t = 0; t < MT; t++) {
                        const int m = t * 8 + lr;
#pragma unroll
                        for (int q = 0; q < PL; q++) {
                            uint4 x = make_uint4(0, 0, 0, 0);
                            if (m < Mb) x = *reinterpret_cast<const uint4*>(x_sm + (long)(q * Mb + m) * pitch + ((b0 + u) * BK + j * 32 + lc * 8) * 2);
                            mma_bf16(part[t], al[0], ah[0], al[1], ah[1], x.x, x.y);
                            mma_bf16(part[t], al[2], ah[2], al[3], ah[3], x.z, x.w);
                        }
                    }
                }
#pragma unroll
                for (int t = 0; t < MT; t++) {
                    acc[t][0] = __fmaf_rn(part[t][0], sl[u], acc[t][0]); acc[t][1] = __fmaf_rn(part[t][1], sl[u], acc[t][1]);
                    acc[t][2] = __fmaf_rn(part[t][2], sh[u], acc[t][2]); acc[t][3] = __fmaf_rn(part[t][3], sh[u], acc[t][3]);
                }
            }
        }
    }
    // the warps' parts of K, joined in their order; [ks][tokens][rows of the CTA]
    __syncthreads();
    float* red = reinterpret_cast<float*>(x_sm);
    const int rows = 16 * (W4_WARPS / p.ks), r0 = 16 * (warp / p.ks);
#pragma unroll
    for (int t = 0; t < MT; t++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int m = t * 8 + 2 * lc + (i & 1);
            if (m < Mb) red[((long)kw * Mb + m) * rows + r0 + lr + 8 * (i >> 1)] = acc[t][i];
        }
    __syncthreads();
    for (int e = tid; e < Mb * rows; e += W4_WARPS * 32) {
        const int m = e / rows, n = blockIdx.x * rows + e % rows;
        if (n >= p.N) continue;
        float v = 0.0f;
        for (int k = 0; k < p.ks; k++) v += red[(long)k * Mb * rows + e];
        if (p.bias) v += p.bias[n];
        const long at = (long)(m0 + m) * p.ldy + n;
        if (p.y_f32) ((float*)p.y)[at] = v;
        else ((T*)p.y)[at] = from_f<T>(v);
    }
}

template <class T, int VW, int MT> int launch_w4(W4Args& p, cudaStream_t st) {
    const int PL = sizeof(T) == 2 ? 1 : 3;
    const int tokens = p.M < 8 * MT ? p.M : 8 * MT;
    // warps along K while the CTAs are fewer than two per SM
    p.ks = 1;
    const long tiles = (p.N + 15) / 16;
    while (p.ks < W4_WARPS && tiles * p.ks < 2L * W4_WARPS * gemm_sm_count()) p.ks *= 2;
    const int least = 32 * VW * p.ks;                     // a block for every warp
    const int most = 96 * 1024 / (PL * tokens * 2) / 128 * 128;
    p.kc = p.K <= most ? p.K : most;
    if (p.kc < p.K && p.kc > least) p.kc = p.kc / least * least;
    const size_t pitch = (size_t)p.kc * 2 + ((p.kc & 63) ? 0 : 64);
    size_t smem = pitch * PL * tokens;
    const size_t red = (size_t)W4_WARPS * 16 * tokens * 4;
    if (red > smem) smem = red;
    auto kern = linear_w4_kernel<T, VW, MT>;
    TRY_RC(allow_shared(kern, smem));
    const long ctas = (tiles * p.ks + W4_WARPS - 1) / W4_WARPS;
    launch_k(kern, dim3((unsigned)ctas, (p.M + 63) / 64), dim3(W4_WARPS * 32), smem, st, p);
    return launch_status();
}
template <class T, int VW> int pick_w4(W4Args& p, cudaStream_t st) {
    if (p.M <= 8) return launch_w4<T, VW, 1>(p, st);
    if (p.M <= 16) return launch_w4<T, VW, 2>(p, st);
    if (p.M <= 32) return launch_w4<T, VW, 4>(p, st);
    return launch_w4<T, VW, 8>(p, st);
}
template <class T> int run_w4(W4Args& p, cudaStream_t st) {
    if (p.group % 128 == 0) return pick_w4<T, 4>(p, st);
    if (p.group % 64 == 0) return pick_w4<T, 2>(p, st);
    return pick_w4<T, 1>(p, st);
}

}  // namespace

}  // namespace flexllm

using namespace flexllm;

extern "C" int flexllm_linear_w4(int dtype, const void* a, long lda, const uint8_t* w, const void* scale, int scale_dtype, const uint8_t* zero, int group,
                                 const float* bias, int M, int N, int K, void* y, long ldy, int y_f32, void* stream) {
    FLEXLLM_REQUIRE((dtype == FLEXLLM_F32 || dtype == FLEXLLM_BF16) && (scale_dtype == FLEXLLM_F32 || scale_dtype == FLEXLLM_BF16));
    FLEXLLM_REQUIRE(M >= 0 && N > 0 && K > 0 && group > 0 && group % 32 == 0 && K % group == 0 && lda >= K && lda % 8 == 0 && ldy >= N);
    if ((M + 63) / 64 > 65535) return FLEXLLM_ENOTSUP;
    if (M == 0) return FLEXLLM_OK;
    FLEXLLM_REQUIRE(a && w && scale && y && aligned(a, 16) && aligned(w, 16));
    W4Args p = {a, lda, w, scale, scale_dtype == FLEXLLM_F32, zero, group, bias, M, N, K, y, ldy, y_f32 != 0, 1, 0};
    const SetUpEarly early;
    return dtype == FLEXLLM_BF16 ? run_w4<bf16>(p, (cudaStream_t)stream) : run_w4<float>(p, (cudaStream_t)stream);
}
