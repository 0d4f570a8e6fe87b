// Attention of packed rows over their sequences' pages: what its kernels share.
//   p_ij = exp(scale q_i . k_j - m_i) / l_i over the keys j that row i sees,  out_i = sum_j p_ij v_j;  a row that sees nothing: 0
// Causal: row i of a sequence sees the positions up to ctx + i. Trees: it sees the ctx cached ones and, of the new ones, those whose
// bit is set in its mask. The R = H / G query heads of a key/value head are rows of the same tile.
#pragma once
#include "paged.cuh"

namespace flexllm {

struct PagedAttn {
    PackedSeqs seq;
    int H, G, dk, dv;
    float scale;
    const void* q; long ldq;              // T [T][ldq], heads side by side
    const unsigned long long* mask;       // [T], nullptr: causal
    const void *k, *v;                    // pages
    void* out; long ldo;
};

// Number of keys that row i of a sequence sees without asking the mask, and whether it sees a later one.
__device__ __forceinline__ int sure_keys(const PagedAttn& a, const SeqRows& s, int i) { return a.mask ? s.ctx : s.ctx + i + 1; }
// The mask's bits of tokens that the sequence has.
__device__ __forceinline__ unsigned long long mask_bits(const PagedAttn& a, const SeqRows& s, int i) {
    if (!a.mask) return 0ull;
    const unsigned long long bits = a.mask[s.row0 + i];
    return s.n < 64 ? bits & ((1ull << s.n) - 1) : bits;
}
__device__ __forceinline__ bool sees_key(int key, int sure, unsigned long long bits, int ctx) {
    return key < sure || (unsigned)(key - ctx) < 64u && ((bits >> (key - ctx)) & 1u);
}

__device__ __forceinline__ bool sees_any(const PagedAttn& a, const SeqRows& s, int i) { return sure_keys(a, s, i) > 0 || mask_bits(a, s, i) != 0; }
// One row, key by key, by a whole warp. Rows come here whose result was not finite: a product of a weight of zero and an infinity or
// NaN in a value that the row does not see must not reach it (and a result that is truly not finite comes out again). And rows that see a key, but whose
// weights were all zero: scores below where the running maximum starts, or so large that their exponents in one rounding and in two are far apart.
template <class T> __device__ __noinline__ void attn_row_by_key(const PagedAttn& a, int b, const SeqRows& s, int i, int h) {
    const int lane = threadIdx.x & 31, g = h / (a.H / a.G);
    const T* q = (const T*)a.q + (long)(s.row0 + i) * a.ldq + (long)h * a.dk;
    const unsigned long long bits = mask_bits(a, s, i);
    const int sure = sure_keys(a, s, i), end = a.mask ? s.ctx + s.n : sure;
    float m = -INFINITY, l = 0.0f, o[8];
#pragma unroll
    for (int e = 0; e < 8; e++) o[e] = 0.0f;
    for (int key = 0; key < end; key++) {
        if (!sees_key(key, sure, bits, s.ctx)) continue;
        const long page = page_of(a.seq, b, key / kPage);
        const int slot = key & (kPage - 1);
        const T* k = (const T*)a.k + ((page * a.G + g) * kPage + slot) * a.dk;
        const T* v = (const T*)a.v + (page * a.G + g) * (long)a.dv * kPage + slot;
        float d = 0.0f;
        for (int e = lane; e < a.dk; e += 32) d = __fmaf_rn(to_f(q[e]), to_f(k[e]), d);
        const float x = warp_sum(d) * a.scale;
        const float mn = x > m ? x : m, al = m == -INFINITY ? 0.0f : expf(m - mn);
        const float w = x == -INFINITY ? 0.0f : expf(x - mn);
        m = mn;
        l = __fmaf_rn(l, al, w);
#pragma unroll
        for (int e = 0; e < 8; e++)
            if (lane + 32 * e < a.dv) {
                o[e] *= al;
                if (w != 0.0f) o[e] = __fmaf_rn(w, to_f(v[(long)(lane + 32 * e) * kPage]), o[e]);
            }
    }
    T* out = (T*)a.out + (long)(s.row0 + i) * a.ldo + (long)h * a.dv;
#pragma unroll
    for (int e = 0; e < 8; e++)
        if (lane + 32 * e < a.dv) out[lane + 32 * e] = from_f<T>(l == 0.0f ? 0.0f : o[e] / l);
}
__device__ __forceinline__ bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }
__device__ __forceinline__ bool not_finite(float v) { return !(fabsf(v) <= 3.402823466e38f); }

// CTAs of a cluster among which a tile's keys are cut, for `tiles` (tile, head) pairs of up to `pages` key pages each: as many as all run at once
// while each part keeps `least` pages, and 16 in clusters of more than 8.
inline int key_splits(long tiles, bool two, int pages, int least, int most) {
    int best = 1;
    for (int s = 2; s <= most && pages >= s * (s > 8 ? 16 : least); s++)
        if (cluster_slots(s, two) >= tiles) best = s;
    return best;
}

int attn_paged_simt(const PagedAttn& a, cudaStream_t st);      // fp32
int attn_paged_f32(const PagedAttn& a, cudaStream_t st);       // fp32, heads up to 128
int attn_paged_tc(const PagedAttn& a, cudaStream_t st);        // bf16, scale >= 0

}  // namespace flexllm
