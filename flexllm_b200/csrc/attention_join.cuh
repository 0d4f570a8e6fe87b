// The tensor-core forms of paged attention: the end of a tile whose keys were cut.
#pragma once
#include "attention_paged.cuh"
#include "tc_common.cuh"

namespace flexllm {

constexpr float kSlack = 8.0f;             // log2 units by which a score may exceed its row's shift
constexpr float kNoScore = -1e30f;         // where a row's shift starts: weights of scores below it are zero, and a row of such scores is computed key by key

__device__ __forceinline__ void store8f(bf16* p, const float (&f)[8], bool vec) {
    if (vec) *reinterpret_cast<uint4*>(p) = make_uint4(bf_pack(f[0], f[1]), bf_pack(f[2], f[3]), bf_pack(f[4], f[5]), bf_pack(f[6], f[7]));
    else
#pragma unroll
        for (int x = 0; x < 8; x++) p[x] = __float2bfloat16_rn(f[x]);
}
__device__ __forceinline__ void store8f(float* p, const float (&f)[8], bool vec) {
    if (vec) { store4(p, make_float4(f[0], f[1], f[2], f[3])); store4(p + 4, make_float4(f[4], f[5], f[6], f[7])); }
    else
#pragma unroll
        for (int x = 0; x < 8; x++) p[x] = f[x];
}
template <class T> __device__ __forceinline__ bool whole_stores(const PagedAttn& a) { return a.ldo % (16 / (int)sizeof(T)) == 0 && aligned16(a.out); }

constexpr int kJoinRows = 144;             // rows of a tile and 16 CTAs, a multiple of their number: up to 15 more

// scale * log2 e; for a scale of 0 the smallest number, so that masked scores of -infinity stay that: 3.4e38 becomes 4.8e-7, a weight of 1 but for the last bits
inline float score_factor(const PagedAttn& a) {
    const float f = a.scale * kLog2e;
    return f > 1.401298464e-45f ? f : 1.401298464e-45f;
}

// The parts of a tile of 128 rows, STEP of them in each of the n_split CTAs of a cluster, joined by all nt threads of every CTA: maxima (log2 units) and
// sums at m_at and l_at, [STEP][128], outputs at o_at, [STEP][128][dv + 4], at the same addresses in every CTA and fenced. CTA r of the
// cluster has rows r, r + n_split, ..: first the parts' weights (over the sums; parts x rows of a CTA are kJoinRows STEP at most), then the outputs.
template <class T, int STEP>
__device__ __forceinline__ void join_parts(const PagedAttn& a, const SeqRows& s, int i0, int RC, int TQ, int heads, int h0, int n_split, int split, uint32_t o_at,
                                           uint32_t m_at, uint32_t l_at, float* w_sm, unsigned* redo_sm, int nt) {
    using namespace tc;
    constexpr int N = 8 * STEP;                        // parts looked at together: set p % STEP of CTA p / STEP
    const int rows = min(TQ, s.n - i0) * RC, per = a.dv / 8, mine = (rows - split + n_split - 1) / n_split, parts = n_split * STEP;
    for (int e = threadIdx.x; e < mine; e += nt) {
        const int row = split + e * n_split;
        float top = kNoScore, sum = 0.0f;
        for (int p0 = 0; p0 < parts; p0 += N) {
            float mk[N], lk[N];
            const float before = top;
#pragma unroll
            for (int p = 0; p < N; p++)
                if (p0 + p < parts) {
                    mk[p] = ld_cluster_f32(cluster_addr(m_at + ((p % STEP) * 128 + row) * 4, (p0 + p) / STEP));
                    lk[p] = ld_cluster_f32(cluster_addr(l_at + ((p % STEP) * 128 + row) * 4, (p0 + p) / STEP));
                }
#pragma unroll
            for (int p = 0; p < N; p++)
                if (p0 + p < parts) top = fmaxf(top, mk[p]);
            sum *= ex2_fast(before - top);
#pragma unroll
            for (int p = 0; p < N; p++)
                if (p0 + p < parts) { sum = __fmaf_rn(lk[p], ex2_fast(mk[p] - top), sum); w_sm[(p0 + p) * mine + e] = mk[p]; }
        }
        const float r = sum == 0.0f ? 0.0f : 1.0f / sum;
        if (sum == 0.0f && row % RC < heads && sees_any(a, s, i0 + row / RC)) atomicOr(&redo_sm[row >> 5], 1u << (row & 31));
        for (int p = 0; p < parts; p++) w_sm[p * mine + e] = sum == 0.0f ? 0.0f : ex2_fast(w_sm[p * mine + e] - top) * r;
    }
    __syncthreads();
    for (int e = threadIdx.x; e < mine * per; e += nt) {
        const int i = e / per, row = split + i * n_split, d = e % per * 8;
        if (row % RC >= heads) continue;
        float f[8];
#pragma unroll
        for (int x = 0; x < 8; x++) f[x] = 0.0f;
        for (int p0 = 0; p0 < parts; p0 += 4) {        // the loads of four parts are under way together
            float4 x[4], y[4];
#pragma unroll
            for (int p = 0; p < 4; p++)
                if (p0 + p < parts) {
                    const uint32_t at = cluster_addr(o_at + (uint32_t)(((p0 + p) % STEP * 128 + row) * (a.dv + 4) + d) * 4u, (p0 + p) / STEP);
                    x[p] = ld_cluster_f32x4(at); y[p] = ld_cluster_f32x4(at + 16);
                }
#pragma unroll
            for (int p = 0; p < 4; p++)
                if (p0 + p < parts) {
                    const float w = w_sm[(p0 + p) * mine + i];
                    f[0] = __fmaf_rn(x[p].x, w, f[0]); f[1] = __fmaf_rn(x[p].y, w, f[1]); f[2] = __fmaf_rn(x[p].z, w, f[2]); f[3] = __fmaf_rn(x[p].w, w, f[3]);
                    f[4] = __fmaf_rn(y[p].x, w, f[4]); f[5] = __fmaf_rn(y[p].y, w, f[5]); f[6] = __fmaf_rn(y[p].z, w, f[6]); f[7] = __fmaf_rn(y[p].w, w, f[7]);
                }
        }
        bool odd = false;
#pragma unroll
        for (int x = 0; x < 8; x++) odd = odd || not_finite(f[x]);
        if (odd) atomicOr(&redo_sm[row >> 5], 1u << (row & 31));
        store8f((T*)a.out + (long)(s.row0 + i0 + row / RC) * a.ldo + (long)(h0 + row % RC) * a.dv + d, f, whole_stores<T>(a));
    }
}

// Bits of the keys 32 c .. 32 c + 31 of a tile that begins at key key0 that a row sees.
__device__ __forceinline__ uint32_t seen_word(int c, int sure, unsigned long long bits, int ctx, int key0) {
    const int nv = min(max(sure - key0 - 32 * c, 0), 32), sh = 32 * c - (ctx - key0);
    uint32_t see = nv == 32 ? 0xffffffffu : (1u << nv) - 1u;
    if (sh > -32 && sh < 64) see |= sh >= 0 ? (uint32_t)(bits >> sh) : (uint32_t)bits << -sh;
    return see;
}

}  // namespace flexllm
