// Attention of packed rows over their sequences' pages on the CUDA cores, for the 32-bit mode with heads of more than 128 (others:
// attention_paged_f32.cu). A CTA of 256 threads takes RT rows
// (TQ tokens x the query heads of one key/value head) and walks the sequence's pages, one page of 64 keys per step: S = Q K^T and
// O += P V are both dot products of rows in shared memory (Q and K along the head, P and V^T along the keys), RT/16 x 4 and RT/16 x dv/16
// of them per thread, two partial sums each (even and odd elements) in packed fp32 pairs. A row's 16 threads are half a warp, so that its weights
// change hands without a barrier; the next page comes in under this one's products where shared memory holds two.
// Few tiles: a cluster of CTAs cuts the keys, and its partial maxima, sums and outputs meet in shared memory.
// Bound by the fp32 units and the reads of shared memory that feed them: 8 / 2 heads of 256, two prompts of 750 behind 500: 422 us, 25 TFLOP/s; four trees
// of 25 over 3000: 153 us.
#include "attention_paged.cuh"
#include "tc_common.cuh"

namespace flexllm {

using namespace tc;

namespace {

constexpr int PPITCH = kPage + 4;         // pitch of P and V^T rows: 16-byte reads of eight consecutive rows meet no bank twice

template <int N> struct Const { static constexpr int value = N; };
struct SimtArgs { PagedAttn a; int RC, HC, TQ, bufs; };      // heads per tile, head chunks per group, tokens per tile, pages in shared memory

__host__ __device__ inline size_t simt_floats(int RT, int dk, int dv16, int bufs) {
    return (size_t)(RT + bufs * kPage) * (dk + 4) + (size_t)(bufs * dv16 + RT) * PPITCH;
}

__device__ __forceinline__ void copy16(float* dst, const float* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

template <int RT, int NV>
__global__ void __launch_bounds__(256, RT * NV <= 256 ? 2 : 1) attn_paged_simt_kernel(const __grid_constant__ SimtArgs sa, int n_split) {
    constexpr int RR = RT / 16;           // rows per thread
    extern __shared__ __align__(16) float sm[];
    __shared__ float m_sm[RT], l_sm[RT], w_sm[RT + 8];
    __shared__ Unit unit_sm;
    __shared__ unsigned redo_sm[2];
    const PagedAttn& a = sa.a;
    const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
    const int tile = blockIdx.x / n_split, split = blockIdx.x % n_split, all = a.G * sa.HC, hg = tile % all;
    const int g = hg / sa.HC, h0 = g * (a.H / a.G) + (hg % sa.HC) * sa.RC;
    const int heads = min(sa.RC, (g + 1) * (a.H / a.G) - h0);
    pdl_sync();
    if (tid < 32) {
        const int TQ = sa.TQ;
        const Unit u = find_unit(a.seq, tile / all, TQ, 1, [TQ](const SeqRows& s) { return (s.n + TQ - 1) / TQ; });
        if (tid == 0) { unit_sm = u; redo_sm[0] = redo_sm[1] = 0; }
    }
    __syncthreads();
    const int b = unit_sm.b;
    if (b < 0) return;                    // the same for the whole cluster
    const SeqRows s = unit_sm.s;
    const int i0 = unit_sm.i * sa.TQ;     // first row of the tile within the sequence
    const int DP = a.dk + 4;
    float *q_sm = sm, *p_sm = q_sm + RT * DP, *kv_sm = p_sm + RT * PPITCH;      // a page: K [64][DP], V^T [16 NV][PPITCH]
    const int kv_floats = kPage * DP + NV * 16 * PPITCH, warp = tid >> 5, lane = tid & 31;
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
    for (int row = warp; row < RT; row += 8) {
        const int i = i0 + row / sa.RC;
        const bool on = row < sa.TQ * sa.RC && i < s.n && row % sa.RC < heads;
        for (int c = lane * 4; c < a.dk; c += 128)
            if (on) copy16(q_sm + row * DP + c, (const float*)a.q + (long)(s.row0 + i) * a.ldq + (long)(h0 + row % sa.RC) * a.dk + c);
            else store4(q_sm + row * DP + c, make_float4(0.0f, 0.0f, 0.0f, 0.0f));
    }
    copies_commit();                      // also where this part has no page: the wait at the end covers what was committed
    // page ids are asked for a page ahead: the copies of a page would wait for its id
    int next_page = t_beg < t_end ? page_of(a.seq, b, t_beg) : 0;
    auto load_page = [&](int t) {
        float *k_sm = kv_sm + (sa.bufs == 2 ? (t - t_beg) & 1 : 0) * kv_floats, *v_sm = k_sm + kPage * DP;
        const long at = ((long)next_page * a.G + g) * kPage;
        const float *kp = (const float*)a.k + at * a.dk, *vp = (const float*)a.v + at * a.dv;
        if (t + 1 < t_end) next_page = page_of(a.seq, b, t + 1);
        for (int key = warp; key < kPage; key += 8)
            for (int c = lane * 4; c < a.dk; c += 128) copy16(k_sm + key * DP + c, kp + (long)key * a.dk + c);
        // keys from `end` on were never written: zeros for their values, so that a weight of zero stays without effect
        const int left = end - t * kPage, c = (tid & 15) * 4;
        for (int d = tid >> 4; d < a.dv; d += 16) {
            const float* src = vp + (long)d * kPage + c;
            float* dst = v_sm + d * PPITCH + c;
            if (c + 4 <= left) copy16(dst, src);
            else
                for (int x = 0; x < 4; x++) dst[x] = c + x < left ? src[x] : 0.0f;
        }
        copies_commit();
    };
    // products of the groups of 16 rows that have any: a sequence's last tile is seldom full
    const int groups = (min(sa.TQ, s.n - i0) * sa.RC + 15) / 16;
    auto by_rows = [&](auto f) {
        if (RR == 1 || groups == 1) f(Const<1>());
        else if (RR == 2 || groups == 2) f(Const<2>());
        else f(Const<RR>());
    };
    f32x2 acc[RR][NV];
    float m[RR], l[RR];
#pragma unroll
    for (int r = 0; r < RR; r++) {
        m[r] = -INFINITY; l[r] = 0.0f;
#pragma unroll
        for (int j = 0; j < NV; j++) acc[r][j] = pack2(0.0f, 0.0f);
    }
    if (t_beg < t_end) load_page(t_beg);
    for (int t = t_beg; t < t_end; t++) {
        const float *k_sm = kv_sm + (sa.bufs == 2 ? (t - t_beg) & 1 : 0) * kv_floats, *v_sm = k_sm + kPage * DP;
        copies_wait<0>();
        __syncthreads();                                  // the page is there, the one before has been read
        if (sa.bufs == 2 && t + 1 < t_end) load_page(t + 1);
        f32x2 sc[RR][4];
#pragma unroll
        for (int r = 0; r < RR; r++)
#pragma unroll
            for (int j = 0; j < 4; j++) sc[r][j] = pack2(0.0f, 0.0f);
        by_rows([&](auto rows) {
            constexpr int L = decltype(rows)::value;
#pragma unroll 4
            for (int c = 0; c < a.dk; c += 4) {
                float4 qv[L], kv[4];
#pragma unroll
                for (int r = 0; r < L; r++) qv[r] = load4(q_sm + (ty + 16 * r) * DP + c);
#pragma unroll
                for (int j = 0; j < 4; j++) kv[j] = load4(k_sm + (tx + 16 * j) * DP + c);
#pragma unroll
                for (int r = 0; r < L; r++)
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        sc[r][j] = fma2(pack2(qv[r].x, qv[r].y), pack2(kv[j].x, kv[j].y), sc[r][j]);
                        sc[r][j] = fma2(pack2(qv[r].z, qv[r].w), pack2(kv[j].z, kv[j].w), sc[r][j]);
                    }
            }
        });
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
        __syncwarp();                                     // a row's weights are read by the half warp that wrote them
        // a page's keys in sums of their own: thousands of terms one after the other in one sum would cost it digits
        by_rows([&](auto rows) {
            constexpr int L = decltype(rows)::value, NJ = NV > 8 ? 8 : NV;
#pragma unroll
            for (int j0 = 0; j0 < NV; j0 += NJ) {
                f32x2 part[L][NJ];
#pragma unroll
                for (int r = 0; r < L; r++)
#pragma unroll
                    for (int j = 0; j < NJ; j++) part[r][j] = pack2(0.0f, 0.0f);
#pragma unroll 4
                for (int c = 0; c < kPage; c += 4) {
                    float4 pv[L];
#pragma unroll
                    for (int r = 0; r < L; r++) pv[r] = load4(p_sm + (ty + 16 * r) * PPITCH + c);
#pragma unroll
                    for (int j = 0; j < NJ; j++) {
                        const float4 vv = load4(v_sm + (tx + 16 * (j0 + j)) * PPITCH + c);
#pragma unroll
                        for (int r = 0; r < L; r++) {
                            part[r][j] = fma2(pack2(pv[r].x, pv[r].y), pack2(vv.x, vv.y), part[r][j]);
                            part[r][j] = fma2(pack2(pv[r].z, pv[r].w), pack2(vv.z, vv.w), part[r][j]);
                        }
                    }
                }
#pragma unroll
                for (int r = 0; r < L; r++)
#pragma unroll
                    for (int j = 0; j < NJ; j++) acc[r][j0 + j] = add2(acc[r][j0 + j], part[r][j]);
            }
        });
        __syncwarp();
        if (sa.bufs == 1 && t + 1 < t_end) {
            __syncthreads();
            load_page(t + 1);
        }
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
    // CTA r of the cluster has rows r, r + n_split, ..: the parts' weights over the sums, then the outputs
    const int rows = min(sa.TQ, s.n - i0) * sa.RC, mine = (rows - split + n_split - 1) / n_split;
    for (int e = tid; e < mine; e += 256) {
        const int row = split + e * n_split;
        float mk[8], lk[8], mx = -INFINITY, sum = 0.0f;
#pragma unroll
        for (int k = 0; k < 8; k++)
            if (k < n_split) {
                mk[k] = ld_cluster_f32(cluster_addr(smem_u32(m_sm + row), k));
                lk[k] = ld_cluster_f32(cluster_addr(smem_u32(l_sm + row), k));
            }
#pragma unroll
        for (int k = 0; k < 8; k++)
            if (k < n_split) mx = fmaxf(mx, mk[k]);
#pragma unroll
        for (int k = 0; k < 8; k++)
            if (k < n_split) {
                mk[k] = mk[k] == -INFINITY ? 0.0f : expf(mk[k] - mx);
                sum = __fmaf_rn(lk[k], mk[k], sum);
            }
#pragma unroll
        for (int k = 0; k < 8; k++)
            if (k < n_split) w_sm[k * mine + e] = sum == 0.0f ? 0.0f : mk[k] / sum;
    }
    __syncthreads();
    for (int e = tid; e < mine * (a.dv / 4); e += 256) {
        const int at = e / (a.dv / 4), row = split + at * n_split, d = (e - at * (a.dv / 4)) * 4;
        if (row % sa.RC >= heads) continue;
        float4 x[8], v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int k = 0; k < 8; k++)
            if (k < n_split) x[k] = ld_cluster_f32x4(cluster_addr(smem_u32(o_sm + row * a.dv + d), k));
#pragma unroll
        for (int k = 0; k < 8; k++)
            if (k < n_split) {
                const float w = w_sm[k * mine + at];
                v = make_float4(__fmaf_rn(x[k].x, w, v.x), __fmaf_rn(x[k].y, w, v.y), __fmaf_rn(x[k].z, w, v.z), __fmaf_rn(x[k].w, w, v.w));
            }
        if (not_finite(v.x) || not_finite(v.y) || not_finite(v.z) || not_finite(v.w)) atomicOr(&redo_sm[row >> 5], 1u << (row & 31));
        float* out = (float*)a.out + (long)(s.row0 + i0 + row / sa.RC) * a.ldo + (long)(h0 + row % sa.RC) * a.dv + d;
        if ((a.ldo & 3) == 0 && aligned16(a.out)) store4(out, v);
        else { out[0] = v.x; out[1] = v.y; out[2] = v.z; out[3] = v.w; }
    }
    if (n_split > 1) cluster_sync(); else __syncthreads();
    if (redo_sm[0] | redo_sm[1])
        for (int row = tid >> 5; row < rows; row += 8)
            if (redo_sm[row >> 5] >> (row & 31) & 1) attn_row_by_key<float>(a, b, s, i0 + row / sa.RC, h0 + row % sa.RC);
}

template <int RT, int NV> int launch_simt(SimtArgs& sa, int tiles, int splits, cudaStream_t st) {
    sa.bufs = simt_floats(RT, sa.a.dk, NV * 16, 2) * 4 <= 220 * 1024 ? 2 : 1;
    const size_t smem = simt_floats(RT, sa.a.dk, NV * 16, sa.bufs) * 4;
    auto kern = attn_paged_simt_kernel<RT, NV>;
    TRY_RC(allow_shared(kern, smem));
    launch_cluster(kern, dim3((unsigned)tiles * splits * sa.a.G * sa.HC), dim3(256), splits, smem, st, sa, splits);
    return launch_status();
}
template <int RT> int run_simt(const PagedAttn& a, cudaStream_t st) {
    SimtArgs sa;
    const int R = a.H / a.G;
    sa.a = a;
    sa.RC = R < RT ? R : RT; sa.HC = (R + sa.RC - 1) / sa.RC; sa.TQ = RT / sa.RC;
    const long seqs = a.seq.B < a.seq.T ? a.seq.B : a.seq.T;
    const long tiles = most_units(a.seq, sa.TQ), real = ((a.seq.T + seqs - 1) / seqs + sa.TQ - 1) / sa.TQ * seqs;      // at most; with sequences of equal length
    const int splits = key_splits(real * a.G * sa.HC, false, (a.seq.max_ctx + kPage) / kPage, 1, 8);
    if (tiles * splits * a.G * sa.HC > 0x7fffffffL) return FLEXLLM_ENOTSUP;
    if (a.dv <= 64) return launch_simt<RT, 4>(sa, (int)tiles, splits, st);
    if (a.dv <= 128) return launch_simt<RT, 8>(sa, (int)tiles, splits, st);
    return launch_simt<RT, 16>(sa, (int)tiles, splits, st);
}

}  // namespace

int attn_paged_simt(const PagedAttn& a, cudaStream_t st) {
    if (a.dk <= 128 && a.dv <= 128) return attn_paged_f32(a, st);
    const long rows = (long)(a.seq.T / a.seq.B) * (a.H / a.G);          // of an average sequence and a key/value head
    return rows <= 16 ? run_simt<16>(a, st) : run_simt<64>(a, st);
}

namespace {
int attn_paged(int dtype, const flexllm_kv_pages* kv, int heads, float scale, const void* q, long ldq, const uint64_t* mask, const int32_t* cu,
               const int32_t* ctx, const int32_t* page_table, int max_pages, int max_ctx, int B, int T, void* out, long ldo, void* stream) {
    FLEXLLM_REQUIRE(dtype == FLEXLLM_F32 || dtype == FLEXLLM_BF16);
    FLEXLLM_REQUIRE(kv && kv->k && kv->v && kv->hkv > 0 && heads > 0 && heads <= 65535 && heads % kv->hkv == 0 && kv->kdim > 0 && kv->vdim > 0);
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
