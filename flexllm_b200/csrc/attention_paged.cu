// Attention of packed rows over their sequences' pages on the CUDA cores, for the 32-bit mode. A CTA of 256 threads takes RT rows
// (TQ tokens x the query heads of one key/value head) and walks the sequence's pages, one page of 64 keys per step: S = Q K^T and
// O += P V are both dot products of rows in shared memory (Q and K along the head, P and V^T along the keys), RT/16 x 4 and RT/16 x dv/16
// of them per thread, two partial sums each (even and odd elements) in packed fp32 pairs. K of the next page comes in under P V, V of
// this page under Q K^T. Few tiles: a cluster of CTAs cuts the keys, and its partial maxima, sums and outputs meet in shared memory.
#include "attention_paged.cuh"
#include "tc_common.cuh"

namespace flexllm {

using namespace tc;

namespace {

constexpr int PPITCH = kPage + 4;         // pitch of P and V^T rows: 16-byte reads of eight consecutive rows meet no bank twice

struct SimtArgs { PagedAttn a; int RC, HC, TQ; };      // heads per tile, head chunks per group, tokens per tile

__host__ __device__ inline size_t simt_floats(int RT, int dk, int dv16) { return (size_t)(RT + kPage) * (dk + 4) + (size_t)(dv16 + RT) * PPITCH; }

__device__ __forceinline__ void copy16(float* dst, const float* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

template <int RT, int NV>
__global__ void __launch_bounds__(256) attn_paged_simt_kernel(const __grid_constant__ SimtArgs sa, int n_split) {
    constexpr int RR = RT / 16;           // rows per thread
    extern __shared__ __align__(16) float sm[];
    __shared__ float m_sm[RT], l_sm[RT];
    __shared__ Unit unit_sm;
    __shared__ unsigned redo_sm[2];
    const PagedAttn& a = sa.a;
    const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
    const int tile = blockIdx.x / n_split, split = blockIdx.x % n_split;
    const int g = blockIdx.y / sa.HC, h0 = g * (a.H / a.G) + (blockIdx.y % sa.HC) * sa.RC;
    const int heads = min(sa.RC, (g + 1) * (a.H / a.G) - h0);
    pdl_sync();
    if (tid < 32) {
        const int TQ = sa.TQ;
        const Unit u = find_unit(a.seq, tile, [TQ](const SeqRows& s) { return (s.n + TQ - 1) / TQ; });
        if (tid == 0) { unit_sm = u; redo_sm[0] = redo_sm[1] = 0; }
    }
    __syncthreads();
    const int b = unit_sm.b;
    if (b < 0) return;                    // the same for the whole cluster
    const SeqRows s = unit_sm.s;
    const int i0 = unit_sm.i * sa.TQ;     // first row of the tile within the sequence
    const int DP = a.dk + 4;
    float *q_sm = sm, *k_sm = q_sm + RT * DP, *v_sm = k_sm + kPage * DP, *p_sm = v_sm + NV * 16 * PPITCH;
    const int end = a.mask ? s.ctx + s.n : min(s.ctx + i0 + sa.TQ, s.ctx + s.n);
    const int n_pg = (end + kPage - 1) / kPage;
    const int t_beg = (int)((long)n_pg * split / n_split), t_end = (int)((long)n_pg * (split + 1) / n_split);

    // rows of this thread: ty + 16 r; token and head of a row
    int sure[RR];
    unsigned long long bits[RR];
    bool live[RR];
#pragma unroll
    for (int r = 0; r < RR; r++) {
        const int row = ty + 16 * r, i = i0 + row / sa.RC;
        live[r] = row < sa.TQ * sa.RC && i < s.n && row % sa.RC < heads;
        sure[r] = live[r] ? sure_keys(a, s, i) : 0;
        bits[r] = live[r] ? mask_bits(a, s, i) : 0ull;
    }
    for (int e = tid; e < RT * (a.dk / 4); e += 256) {
        const int row = e / (a.dk / 4), c = (e - row * (a.dk / 4)) * 4, i = i0 + row / sa.RC;
        const bool on = row < sa.TQ * sa.RC && i < s.n && row % sa.RC < heads;
        if (on) copy16(q_sm + row * DP + c, (const float*)a.q + (long)(s.row0 + i) * a.ldq + (long)(h0 + row % sa.RC) * a.dk + c);
        else store4(q_sm + row * DP + c, make_float4(0.0f, 0.0f, 0.0f, 0.0f));
    }
    auto load_k = [&](int t) {
        const float* kp = (const float*)a.k + ((long)page_of(a.seq, b, t) * a.G + g) * kPage * a.dk;
        for (int e = tid; e < kPage * (a.dk / 4); e += 256) {
            const int key = e / (a.dk / 4), c = (e - key * (a.dk / 4)) * 4;
            copy16(k_sm + key * DP + c, kp + (long)key * a.dk + c);
        }
        copies_commit();
    };
    // keys from `end` on were never written: zeros in their place, so that a weight of zero stays without effect
    auto load_v = [&](int t) {
        const float* vp = (const float*)a.v + ((long)page_of(a.seq, b, t) * a.G + g) * a.dv * kPage;
        const int left = end - t * kPage;
        for (int e = tid; e < a.dv * (kPage / 4); e += 256) {
            const int d = e / (kPage / 4), c = (e % (kPage / 4)) * 4;
            const float* src = vp + (long)d * kPage + c;
            float* dst = v_sm + d * PPITCH + c;
            if (c + 4 <= left) copy16(dst, src);
            else
                for (int x = 0; x < 4; x++) dst[x] = c + x < left ? src[x] : 0.0f;
        }
        copies_commit();
    };
    f32x2 acc[RR][NV];
    float m[RR], l[RR];
#pragma unroll
    for (int r = 0; r < RR; r++) {
        m[r] = -INFINITY; l[r] = 0.0f;
#pragma unroll
        for (int j = 0; j < NV; j++) acc[r][j] = pack2(0.0f, 0.0f);
    }
    if (t_beg < t_end) { load_k(t_beg); load_v(t_beg); }
    for (int t = t_beg; t < t_end; t++) {
        copies_wait<1>();
        __syncthreads();
        f32x2 sc[RR][4];
#pragma unroll
        for (int r = 0; r < RR; r++)
#pragma unroll
            for (int j = 0; j < 4; j++) sc[r][j] = pack2(0.0f, 0.0f);
#pragma unroll 2
        for (int c = 0; c < a.dk; c += 4) {
            float4 qv[RR], kv[4];
#pragma unroll
            for (int r = 0; r < RR; r++) qv[r] = load4(q_sm + (ty + 16 * r) * DP + c);
#pragma unroll
            for (int j = 0; j < 4; j++) kv[j] = load4(k_sm + (tx + 16 * j) * DP + c);
#pragma unroll
            for (int r = 0; r < RR; r++)
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    sc[r][j] = fma2(pack2(qv[r].x, qv[r].y), pack2(kv[j].x, kv[j].y), sc[r][j]);
                    sc[r][j] = fma2(pack2(qv[r].z, qv[r].w), pack2(kv[j].z, kv[j].w), sc[r][j]);
                }
        }
#pragma unroll
        for (int r = 0; r < RR; r++) {
            float x[4], mx = -INFINITY;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                float u, w;
                unpack2(sc[r][j], u, w);
                x[j] = sees_key(t * kPage + tx + 16 * j, sure[r], bits[r], s.ctx) ? (u + w) * a.scale : -INFINITY;
                mx = fmaxf(mx, x[j]);
            }
#pragma unroll
            for (int o = 8; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
            const float mn = fmaxf(m[r], mx), ref = mn == -INFINITY ? 0.0f : mn;
            const float al = m[r] == -INFINITY ? 0.0f : expf(m[r] - ref);
            m[r] = mn;
            float sum = 0.0f;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                x[j] = expf(x[j] - ref);
                sum += x[j];
                p_sm[(ty + 16 * r) * PPITCH + tx + 16 * j] = x[j];
            }
            l[r] = __fmaf_rn(l[r], al, sum);              // this thread's keys: summed over the lanes at the end
            const f32x2 al2 = pack2(al, al);
#pragma unroll
            for (int j = 0; j < NV; j++) acc[r][j] = mul2(acc[r][j], al2);
        }
        __syncthreads();                                  // P is there, K has been read
        if (t + 1 < t_end) { load_k(t + 1); copies_wait<1>(); } else copies_wait<0>();
        __syncthreads();                                  // V is there
#pragma unroll 2
        for (int c = 0; c < kPage; c += 4) {
            float4 pv[RR];
#pragma unroll
            for (int r = 0; r < RR; r++) pv[r] = load4(p_sm + (ty + 16 * r) * PPITCH + c);
#pragma unroll
            for (int j = 0; j < NV; j++) {
                const float4 vv = load4(v_sm + (tx + 16 * j) * PPITCH + c);
#pragma unroll
                for (int r = 0; r < RR; r++) {
                    acc[r][j] = fma2(pack2(pv[r].x, pv[r].y), pack2(vv.x, vv.y), acc[r][j]);
                    acc[r][j] = fma2(pack2(pv[r].z, pv[r].w), pack2(vv.z, vv.w), acc[r][j]);
                }
            }
        }
        __syncthreads();                                  // V and P have been read
        if (t + 1 < t_end) load_v(t + 1);
    }
    copies_wait<0>();
    __syncthreads();
    // ---- this part's maxima, sums and outputs into shared memory; the parts' rows are joined by the CTAs of the cluster in turn
    float* o_sm = sm;                                     // [RT][dv]
#pragma unroll
    for (int r = 0; r < RR; r++) {
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) l[r] += __shfl_xor_sync(0xffffffffu, l[r], o);
        if (tx == 0) { m_sm[ty + 16 * r] = m[r]; l_sm[ty + 16 * r] = l[r]; }
#pragma unroll
        for (int j = 0; j < NV; j++) {
            float u, w;
            unpack2(acc[r][j], u, w);
            if (tx + 16 * j < a.dv) o_sm[(ty + 16 * r) * a.dv + tx + 16 * j] = u + w;
        }
    }
    if (n_split > 1) cluster_sync(); else __syncthreads();
    const int rows = min(sa.TQ, s.n - i0) * sa.RC;
    for (int e = tid; e < rows * a.dv; e += 256) {
        const int row = e / a.dv, d = e - row * a.dv;
        if (row % n_split != split || row % sa.RC >= heads) continue;
        float mx = -INFINITY, sum = 0.0f, v = 0.0f;
        if (n_split == 1) {
            sum = l_sm[row]; v = o_sm[e];
        } else {
            for (int k = 0; k < n_split; k++) mx = fmaxf(mx, ld_cluster_f32(cluster_addr(smem_u32(m_sm + row), k)));
            for (int k = 0; k < n_split; k++) {
                const float mk = ld_cluster_f32(cluster_addr(smem_u32(m_sm + row), k)), w = mk == -INFINITY ? 0.0f : expf(mk - mx);
                sum = __fmaf_rn(ld_cluster_f32(cluster_addr(smem_u32(l_sm + row), k)), w, sum);
                v = __fmaf_rn(ld_cluster_f32(cluster_addr(smem_u32(o_sm + e), k)), w, v);
            }
        }
        v = sum == 0.0f ? 0.0f : v / sum;
        if (not_finite(v)) atomicOr(&redo_sm[row >> 5], 1u << (row & 31));
        ((float*)a.out)[(long)(s.row0 + i0 + row / sa.RC) * a.ldo + (long)(h0 + row % sa.RC) * a.dv + d] = v;
    }
    if (n_split > 1) cluster_sync(); else __syncthreads();
    if (redo_sm[0] | redo_sm[1])
        for (int row = tid >> 5; row < rows; row += 8)
            if (redo_sm[row >> 5] >> (row & 31) & 1) attn_row_by_key<float>(a, b, s, i0 + row / sa.RC, h0 + row % sa.RC);
}

template <int RT, int NV> int launch_simt(const SimtArgs& sa, int tiles, int splits, cudaStream_t st) {
    const size_t smem = simt_floats(RT, sa.a.dk, NV * 16) * 4;
    auto kern = attn_paged_simt_kernel<RT, NV>;
    TRY_RC(allow_shared(kern, smem));
    launch_cluster(kern, dim3(tiles * splits, sa.a.G * sa.HC), dim3(256), splits, smem, st, sa, splits);
    return launch_status();
}
template <int RT> int run_simt(const PagedAttn& a, cudaStream_t st) {
    SimtArgs sa;
    const int R = a.H / a.G;
    sa.a = a;
    sa.RC = R < RT ? R : RT; sa.HC = (R + sa.RC - 1) / sa.RC; sa.TQ = RT / sa.RC;
    const long tiles = a.seq.T / sa.TQ + (a.seq.B < a.seq.T ? a.seq.B : a.seq.T);
    const int splits = key_splits(tiles * a.G * sa.HC, gemm_sm_count(), (a.seq.max_ctx + kPage) / kPage, 1);
    if (tiles * splits > 0x7fffffffL || a.G * sa.HC > 65535) return FLEXLLM_ENOTSUP;
    if (a.dv <= 64) return launch_simt<RT, 4>(sa, (int)tiles, splits, st);
    if (a.dv <= 128) return launch_simt<RT, 8>(sa, (int)tiles, splits, st);
    return launch_simt<RT, 16>(sa, (int)tiles, splits, st);
}

}  // namespace

int attn_paged_simt(const PagedAttn& a, cudaStream_t st) {
    const long rows = (long)(a.seq.T / a.seq.B) * (a.H / a.G);          // of an average sequence and a key/value head
    return rows <= 16 ? run_simt<16>(a, st) : run_simt<64>(a, st);
}

namespace {
int attn_paged(int dtype, const flexllm_kv_pages* kv, int heads, float scale, const void* q, long ldq, const uint64_t* mask, const int32_t* cu,
               const int32_t* ctx, const int32_t* page_table, int max_pages, int max_ctx, int B, int T, void* out, long ldo, void* stream) {
    FLEXLLM_REQUIRE(dtype == FLEXLLM_F32 || dtype == FLEXLLM_BF16);
    FLEXLLM_REQUIRE(kv && kv->k && kv->v && kv->hkv > 0 && heads > 0 && heads % kv->hkv == 0 && kv->kdim > 0 && kv->vdim > 0);
    PagedAttn a = {};
    a.seq = {cu, ctx, page_table, max_pages, max_ctx, B, T, kv->n_pages, mask ? 64 : 0x7fffffff, nullptr};
    a.H = heads; a.G = kv->hkv; a.dk = kv->kdim; a.dv = kv->vdim;
    a.scale = scale; a.q = q; a.ldq = ldq; a.mask = (const unsigned long long*)mask; a.k = kv->k; a.v = kv->v; a.out = out; a.ldo = ldo;
    const long per16 = dtype == FLEXLLM_BF16 ? 8 : 4;                   // elements of 16 bytes
    FLEXLLM_REQUIRE(packed_ok(a.seq) && ldq >= (long)heads * a.dk && ldo >= (long)heads * a.dv && ldq % per16 == 0 && scale >= 0.0f && scale <= 1e30f);
    if (a.dk % 8 || a.dv % 8 || a.dk > 256 || a.dv > 256) return FLEXLLM_ENOTSUP;
    if (T == 0) return FLEXLLM_OK;
    FLEXLLM_REQUIRE(q && out && aligned(q, 16) && aligned(kv->k, 16) && aligned(kv->v, 16) && aligned(out, dtype == FLEXLLM_BF16 ? 2 : 4));
    a.seq.error_flag = device_error_flag();
    const SetUpEarly early;
    return dtype == FLEXLLM_BF16 ? attn_paged_tc(a, (cudaStream_t)stream) : attn_paged_simt(a, (cudaStream_t)stream);
}
}  // namespace

}  // namespace flexllm

using namespace flexllm;

extern "C" int flexllm_attn_packed(int dtype, const flexllm_kv_pages* kv, int heads, float scale, const void* q, long ldq, const int32_t* cu,
                                   const int32_t* ctx, const int32_t* page_table, int max_pages, int max_ctx, int B, int T, void* out, long ldo,
                                   void* stream) {
    return attn_paged(dtype, kv, heads, scale, q, ldq, nullptr, cu, ctx, page_table, max_pages, max_ctx, B, T, out, ldo, stream);
}
extern "C" int flexllm_attn_tree(int dtype, const flexllm_kv_pages* kv, int heads, float scale, const void* q, long ldq, const uint64_t* mask,
                                 const int32_t* cu, const int32_t* ctx, const int32_t* page_table, int max_pages, int max_ctx, int B, int T, void* out,
                                 long ldo, void* stream) {
    FLEXLLM_REQUIRE((mask || T == 0) && aligned(mask, 8));
    return attn_paged(dtype, kv, heads, scale, q, ldq, T == 0 ? (const uint64_t*)8 : mask, cu, ctx, page_table, max_pages, max_ctx, B, T, out, ldo, stream);
}
