// Products with 4-bit weights, one scale and zero point per group of the inner index, for up to 8 tokens:
//   y[m][n] = sum_groups s[n][g] * sum_{k in g} a[m][k] (q[n][k] - z[n][g])
// HBM bound for few tokens: half a byte per weight. Weights stream from memory into the registers of the lanes that multiply them: a warp has
// 16 rows on the 16-row side of bf16 warp MMAs and 8 tokens per MMA on the other. q - z is an integer of five bits, exact in bf16, and sums
// over a group stay in the MMA's fp32 accumulators; the scale multiplies them in fp32, so no weight is ever rounded. fp32 activations are
// cut into three bf16 parts of eight bits each, which hold them to the last bit, at three MMAs instead of one.
//
// Two nibbles j and j + 4 of a word become a pair of bf16 in three instructions (shift, mask and exponent at once: 0x4300 | q is 128 + q, one
// subtraction of 128 + z). The inner index may go through the MMA in any order, the same one in both operands: a lane's words are as they lie
// in memory, and the activations follow (16 bytes at a time on their way into shared memory, pairs when they are read).
// Measured: one token, 8192 x 2048, 7.2 us (launch, first words, joining K); 128256 x 2048, 41 us, 3.2 TB/s, where unpacking fills the math pipes; fp32
// activations, 8192 x 2048: one token 8.4 us, eight 9.7 us.
#include "linear_w4.h"

namespace flexllm {

namespace {

struct W4Args : W4Call {
    int ks;                                // warps of a CTA along K
    int per_group; uint32_t magic;         // blocks of a group, and 2^32 / per_group rounded up: the quotient of block numbers below 2^16
    int red_at, rows_log;                  // where the parts meet in shared memory; log2 of a CTA's rows
    int steps, chunks;                     // steps of kStep elements per staged chunk of activations (a multiple of ks), chunks
};
constexpr int kStep = 128;
constexpr int kWarps = 16;                 // of a CTA

template <int VW> struct Words { uint32_t v[VW]; };
template <int VW> __device__ __forceinline__ Words<VW> load_words(const uint8_t* p) {
    Words<VW> r;
    if (VW == 4) asm("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(r.v[0]), "=r"(r.v[1 % VW]), "=r"(r.v[2 % VW]), "=r"(r.v[3 % VW]) : "l"(p));
    else if (VW == 2) asm("ld.global.nc.v2.u32 {%0, %1}, [%2];" : "=r"(r.v[0]), "=r"(r.v[1 % VW]) : "l"(p));
    else asm("ld.global.nc.u32 %0, [%1];" : "=r"(r.v[0]) : "l"(p));
    return r;
}

// 8 bf16 activations k .. k + 7 as the pairs (0,4) (1,5) (2,6) (3,7)
__device__ __forceinline__ uint4 pairs(const uint4& v) {
    return make_uint4(pick(v.x, v.z, 0x5410), pick(v.x, v.z, 0x7632), pick(v.y, v.w, 0x5410), pick(v.y, v.w, 0x7632));
}

__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}

// d [16 x 8] = a [16 x 16] b [16 x 8]
__device__ __forceinline__ void mma_bf16_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
                 : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}

// A step is 128 elements of 32 rows (two MMA tiles, which share the activations' operands): four words per lane and row, U blocks of VW words (a quad of lanes covers the 32 VW elements of a block, which
// are of one group). A CTA's warps are ks along K, the others along the rows; the tokens' activations are staged in chunks, two in shared
// memory, and serve all its rows. Where one chunk holds them all, a CTA goes on with further rows. Weights, scales and zero points are asked
// for D steps ahead, over the end of a chunk and of the rows.
// In shared memory 32 elements, those of one word of a quad's lanes, lie together for all tokens: [chunk][8 tokens][64 bytes], so that eight
// lanes read 128 bytes in a row and every address but the step's is a constant.
// PACKED: K of whole steps, a group per block, bf16 scales: a step's scales and zero points come in one load each.
template <class T, int VW, bool PACKED>
__global__ void __launch_bounds__(kWarps * 32, 1) linear_w4_kernel(const __grid_constant__ W4Args p) {
    constexpr int PL = sizeof(T) == 2 ? 1 : 3, NW = kWarps;
    constexpr int BK = 32 * VW, U = 4 / VW;                // elements of a block, blocks per step
    constexpr int D = 2;
    constexpr int XC = 8 * 64, XS = 4 * XC;           // bytes of 32 elements of all tokens, of a step
    constexpr int SW = PACKED ? (U + 1) / 2 : U, ZW = PACKED ? 1 : U;
    extern __shared__ __align__(16) uint8_t x_sm[];        // [2][PL][steps] XS
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, lr = lane >> 2, lc = lane & 3;
    const int kw = warp & (p.ks - 1), per_cta = NW / p.ks, rows = 32 * per_cta, r0 = 32 * (warp / p.ks);
    const int groups = p.K / p.group, plane = p.steps * XS;
    // a step's words, scales and zero points of this lane's four rows, as they are in memory: a conversion here would wait for the load
    struct Step { Words<VW> w[4][U]; uint32_t s[4][SW], z[4][ZW]; };
    auto scale_of = [&](const uint32_t (&v)[SW], int u) {
        if (PACKED) return __uint_as_float(u & 1 ? v[u >> 1] & 0xffff0000u : v[u >> 1] << 16);
        return __uint_as_float(p.scale_f32 ? v[u % SW] : v[u % SW] << 16);
    };
    auto zero_of = [&](const uint32_t (&v)[ZW], int u) {           // 128 + z, twice
        return zero2(PACKED ? v[0] >> (8 * u) : v[u % ZW]);
    };
    // the next step to ask for: its round (ks steps side by side) and, with 32-bit offsets of this lane's rows from the tile's first row
    const int all = (p.K + kStep - 1) / kStep, rounds = (all + p.ks - 1) / p.ks;
    int f_round = 0, f_tile = blockIdx.x;
    uint32_t w_at[4], g_at[4];
    auto aim = [&] {
        const int last = max(p.N - 1 - f_tile * rows, 0);
        if (f_tile * rows >= p.N) f_tile = 0;             // behind the last rows: something to load, not used
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const uint32_t n = min(r0 + lr + 8 * r, last);
            w_at[r] = n * (p.K / 2) + lc * 4 * VW; g_at[r] = n * groups;
        }
    };
    auto fetch = [&](Step& s) {
        const long row0 = (long)f_tile * rows;
        // in the last round a warp may have no step: something to load, not used
        const int st = f_round * p.ks + kw < all ? kw : 0;
        if (PACKED) {
            const uint8_t* w = p.w + row0 * (p.K / 2) + (f_round * p.ks + st) * (kStep / 2);
            const long g0 = row0 * groups + (f_round * p.ks + st) * U;
            const uint16_t* sc = (const uint16_t*)p.scale + g0;
#pragma unroll
            for (int r = 0; r < 4; r++) {
#pragma unroll
                for (int u = 0; u < U; u++) s.w[r][u] = load_words<VW>(w + w_at[r] + u * (BK / 2));
                if (U == 1) s.s[r][0] = sc[g_at[r]];
                else if (U == 2) s.s[r][0] = *(const uint32_t*)(sc + g_at[r]);
                else {
                    const uint2 x = *(const uint2*)(sc + g_at[r]);
                    s.s[r][0] = x.x; s.s[r][1 % SW] = x.y;
                }
                s.z[r][0] = 0x08080808u;
            }
            if (p.zero) {
                const uint8_t* z = p.zero + g0;
#pragma unroll
                for (int r = 0; r < 4; r++) s.z[r][0] = U == 1 ? z[g_at[r]] : U == 2 ? *(const uint16_t*)(z + g_at[r]) : *(const uint32_t*)(z + g_at[r]);
            }
        } else {
#pragma unroll
            for (int u = 0; u < U; u++) {
                const int k = min((f_round * p.ks + st) * kStep + u * BK, p.K - BK), g = p.per_group == 1 ? k / BK : (int)__umulhi(k / BK, p.magic);
                const uint8_t* w = p.w + row0 * (p.K / 2) + k / 2;
                const long g0 = row0 * groups + g;
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    s.w[r][u] = load_words<VW>(w + w_at[r]);
                    s.s[r][u % SW] = p.scale_f32 ? ((const uint32_t*)p.scale)[g0 + g_at[r]] : (uint32_t)((const uint16_t*)p.scale)[g0 + g_at[r]];
                    s.z[r][u % ZW] = 8;
                    if (p.zero) s.z[r][u % ZW] = p.zero[g0 + g_at[r]];
                }
            }
        }
        if (++f_round == rounds) { f_round = 0; f_tile += gridDim.x; aim(); }
    };
    // Activations of a chunk into its buffer, 16 bytes per lane: 4 VW lanes read the 64 VW bytes of a token's block in a row. Elements k .. k + 7 of
    // lane c's word j are k = BK block + 8 VW c + 8 j.
    const int kc = p.steps * kStep;
    auto pieces = [&](int chunk, auto f) {
        constexpr int LT = 4 * VW, TW = 32 / LT;           // lanes of a token, tokens of a warp
        const int n = min(kc, p.K - chunk * kc) / BK, piece = lane % LT, c = piece / VW, j = piece % VW;
        uint8_t* to = x_sm + (chunk & 1) * PL * plane + j * XC + (lane / LT) * 64 + c * 16;
        const int k = chunk * kc + piece * 8;
        for (int e = warp; e < n * (8 / TW); e += NW) {
            const int b = e / (8 / TW), mt = (e - b * (8 / TW)) * TW, m = mt + lane / LT;
            if (m < p.M) f(to + b * VW * XC + mt * 64, m, k + b * BK);
        }
    };
    auto stage = [&](int chunk) {
        pieces(chunk, [&](uint8_t* to, int m, int k) {
            const T* src = (const T*)p.a + (long)m * p.lda + k;
            if (PL == 1) copy16((uint32_t)__cvta_generic_to_shared(to), src);
            else {
                float f[8];
                load8((const float*)src, f);
                const Eight x = eight(f);
#pragma unroll
                for (int q = 0; q < 3; q++) *reinterpret_cast<uint4*>(to + q * plane) = x.part[q];
            }
        });
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    // the same pieces once they are there: their elements in the order of the weights' pairs
    auto settle = [&](int chunk) {
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        if (PL == 1) pieces(chunk, [&](uint8_t* at, int, int) { *reinterpret_cast<uint4*>(at) = pairs(*reinterpret_cast<const uint4*>(at)); });
    };
    float acc[2][4];
    auto clear = [&] {
#pragma unroll
        for (int h = 0; h < 2; h++)
#pragma unroll
            for (int i = 0; i < 4; i++) acc[h][i] = 0.0f;
    };
    // one step of the warp: elements k0 .. of its rows, activations at xb
    auto multiply = [&](const Step& cur, int k0, const uint8_t* xb) {
#pragma unroll
        for (int u = 0; u < U; u++) {
            if (!PACKED && k0 + u * BK >= p.K) break;
            // an MMA cuts its fp32 sums instead of rounding them: the small parts' products have sums of their own, and do not cut the large ones
            float sc[4], part[PL == 3 ? 2 : 1][2][4];
            uint32_t z[4];
#pragma unroll
            for (int r = 0; r < 4; r++) { z[r] = zero_of(cur.z[r], u); sc[r] = scale_of(cur.s[r], u); }
#pragma unroll
            for (int j = 0; j < VW; j++) {
                uint32_t a[4][4];
#pragma unroll
                for (int r = 0; r < 4; r++)
#pragma unroll
                    for (int i = 0; i < 4; i++) a[r][i] = weights2(cur.w[r][u].v[j], i, z[r]);
#pragma unroll
                for (int q = 0; q < PL; q++) {
                    const uint4 x = *reinterpret_cast<const uint4*>(xb + q * plane + (u * VW + j) * XC);
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        if (j == 0 && q < 2) mma_bf16_first(part[q > 0][h], a[2 * h][0], a[2 * h + 1][0], a[2 * h][1], a[2 * h + 1][1], x.x, x.y);
                        else mma_bf16(part[q > 0][h], a[2 * h][0], a[2 * h + 1][0], a[2 * h][1], a[2 * h + 1][1], x.x, x.y);
                    }
#pragma unroll
                    for (int h = 0; h < 2; h++) mma_bf16(part[q > 0][h], a[2 * h][2], a[2 * h + 1][2], a[2 * h][3], a[2 * h + 1][3], x.z, x.w);
                }
            }
#pragma unroll
            for (int h = 0; h < 2; h++)
#pragma unroll
                for (int i = 0; i < 4; i++) acc[h][i] = __fmaf_rn(PL == 3 ? part[0][h][i] + part[PL == 3][h][i] : part[0][h][i], sc[2 * h + (i >> 1)], acc[h][i]);
        }
    };
    // the warps' parts of K, joined in their order; [ks][tokens][rows of the CTA + 4], behind the activations when these are needed again
    float* red = reinterpret_cast<float*>(x_sm + p.red_at);
    const int red_row = rows + 4;
    auto finish = [&](int tile) {
        __syncthreads();
#pragma unroll
        for (int h = 0; h < 2; h++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int m = 2 * lc + (i & 1);
                if (m < p.M) red[(kw * p.M + m) * red_row + r0 + 16 * h + lr + 8 * (i >> 1)] = acc[h][i];
            }
        __syncthreads();
        for (int e0 = tid; e0 < p.M * rows; e0 += 4 * NW * 32) {
            float v[4];
#pragma unroll
            for (int x = 0; x < 4; x++) {
                const int e = min(e0 + x * NW * 32, p.M * rows - 1), at = (e >> p.rows_log) * red_row + (e & (rows - 1));
                v[x] = 0.0f;
                for (int k = 0; k < p.ks; k++) v[x] += red[k * p.M * red_row + at];
            }
#pragma unroll
            for (int x = 0; x < 4; x++) {
                const int e = e0 + x * NW * 32, m = e >> p.rows_log, n = tile * rows + (e & (rows - 1));
                if (m >= p.M || n >= p.N) continue;
                if (p.bias) v[x] += p.bias[n];
                const long at = (long)m * p.ldy + n;
                if (p.y_f32) ((float*)p.y)[at] = v[x];
                else ((T*)p.y)[at] = from_f<T>(v[x]);
            }
        }
    };
    // the zero points of this CTA's rows, to look at their upper bits while something else is on its way: the first words, or (fp32, whose registers are
    // full then) the first activations. Looked at where they are used: 5 to 15 % slower.
    auto look_at_zeros = [&] {
        if (!p.zero) return;
        uint32_t seen = 0;
        for (int t = blockIdx.x; t * rows < p.N; t += gridDim.x) {
            const uint8_t* z = p.zero + (long)t * rows * groups;
            const int n = min(rows, p.N - t * rows) * groups, whole = ((uintptr_t)z & 15) == 0 ? n & ~15 : 0;
            for (int e = tid * 16; e < whole; e += NW * 32 * 16) {
                const uint4 v = *reinterpret_cast<const uint4*>(z + e);
                seen |= v.x | v.y | v.z | v.w;
            }
            for (int e = whole + tid; e < n; e += NW * 32) seen |= z[e];
        }
        check_zeros(seen, p.error_flag);
    };
    pdl_sync();
    if (PL == 3) look_at_zeros();
    stage(0);
    Step ring[D];
    aim();
#pragma unroll
    for (int d = 0; d < D; d++) fetch(ring[d]);
    if (PL == 1) look_at_zeros();
    clear();
    const int per_chunk = p.chunks > 1 ? p.steps / p.ks : rounds;      // rounds
    int tile = blockIdx.x, round = 0, chunk = 0, left = 0;             // left: rounds of the chunk at hand
    // a ring slot is refilled where it was used, with its index known to the compiler: moved from register to register, a load would be waited for
    while (tile * rows < p.N)
#pragma unroll
        for (int d = 0; d < D; d++) {
            if (tile * rows >= p.N) break;
            if (left == 0) {
                if (tile == blockIdx.x) {
                    settle(chunk);
                    __syncthreads();                       // the chunk is there, the one before has been read
                    if (chunk + 1 < p.chunks) stage(chunk + 1);
                }
                left = per_chunk;
            }
            const int st = round * p.ks + kw;
            if (st < all) multiply(ring[d], st * kStep, x_sm + (chunk & 1) * PL * plane + (st - chunk * p.steps) * XS + lr * 64 + lc * 16);
            fetch(ring[d]);
            if (--left == 0) chunk++;
            if (++round == rounds) {
                finish(tile);
                clear();
                round = chunk = left = 0;
                tile += gridDim.x;
            }
        }
}

template <class T, int VW, bool PACKED> int launch_w4(W4Args& p, cudaStream_t st) {
    constexpr int NW = kWarps, PL = sizeof(T) == 2 ? 1 : 3, per_step = PL * 8 * 2 * kStep;       // bytes of activations
    const int all = (p.K + kStep - 1) / kStep;             // steps of a row
    p.per_group = p.group / (32 * VW);
    p.magic = (uint32_t)(((1ull << 32) + p.per_group - 1) / p.per_group);
    // warps along K while their CTAs find an SM each and every warp keeps a step
    p.ks = 1;
    const long tiles = (p.N + 31) / 32, sms = gemm_sm_count();
    while (p.ks < NW && 2 * p.ks <= all && (tiles * 2 * p.ks + NW - 1) / NW <= sms) p.ks *= 2;
    // all activations at once, or two chunks in turn
    const int red = NW * 36 * p.M * 4, room = 220 * 1024;
    int steps = (room - red) / per_step;
    if (steps < all) steps = room / 2 / per_step;
    while (p.ks > steps) p.ks /= 2;
    p.steps = steps < all ? steps / p.ks * p.ks : all;
    p.chunks = (all + p.steps - 1) / p.steps;
    const int x_bytes = p.steps * per_step;
    p.red_at = p.chunks > 1 ? 0 : x_bytes;
    const size_t smem = p.chunks > 1 ? (2 * x_bytes > red ? 2 * x_bytes : red) : x_bytes + red;
    const int per_cta = NW / p.ks;
    for (p.rows_log = 5; 32 * per_cta > 1 << p.rows_log;) p.rows_log++;
    auto kern = linear_w4_kernel<T, VW, PACKED>;
    TRY_RC(allow_shared(kern, smem));
    long ctas = (tiles + per_cta - 1) / per_cta;
    if (p.chunks == 1 && ctas > sms) ctas = sms;
    launch_k(kern, dim3((unsigned)ctas), dim3(NW * 32), smem, st, p);
    return launch_status();
}
bool packed_groups(const W4Args& p, int block) { return !p.scale_f32 && p.group == block && p.K % kStep == 0 && aligned(p.scale, 8) && aligned(p.zero, 4); }
template <class T, int VW> int run_w4(W4Args& p, cudaStream_t st) { return packed_groups(p, 32 * VW) ? launch_w4<T, VW, true>(p, st) : launch_w4<T, VW, false>(p, st); }
template <class T> int pick_w4(W4Args& p, cudaStream_t st) {
    if (p.group % 128 == 0) return run_w4<T, 4>(p, st);
    if (p.group % 64 == 0) return run_w4<T, 2>(p, st);
    return run_w4<T, 1>(p, st);
}

}  // namespace

}  // namespace flexllm

using namespace flexllm;

extern "C" int flexllm_linear_w4(int dtype, const void* a, long lda, const uint8_t* w, const void* scale, int scale_dtype, const uint8_t* zero, int group,
                                 const float* bias, int M, int N, int K, void* y, long ldy, int y_f32, void* stream) {
    FLEXLLM_REQUIRE((dtype == FLEXLLM_F32 || dtype == FLEXLLM_BF16) && (scale_dtype == FLEXLLM_F32 || scale_dtype == FLEXLLM_BF16));
    FLEXLLM_REQUIRE(M >= 0 && N > 0 && K > 0 && group > 0 && group % 32 == 0 && K % group == 0 && lda >= K && lda % 8 == 0 && ldy >= N);
    // tiles of up to 512 rows are counted a grid beyond the last one, in 31 bits
    if (M > 32 * 65535 || N > 1 << 30 || K > 1 << 20) return FLEXLLM_ENOTSUP;
    if (M == 0) return FLEXLLM_OK;
    FLEXLLM_REQUIRE(a && w && scale && y && aligned(a, 16) && aligned(w, 16) && aligned(scale, scale_dtype == FLEXLLM_F32 ? 4 : 2) && aligned(bias, 4) &&
                    aligned(y, y_f32 || dtype == FLEXLLM_F32 ? 4 : 2));
    const W4Call c = {a, lda, w, scale, scale_dtype == FLEXLLM_F32, zero, group, bias, M, N, K, y, ldy, y_f32 != 0, zero ? device_error_flag() : nullptr};
    const SetUpEarly early;
    // the tensor cores for more than 8 tokens (16 x 8192 x 2048: 9.1 us, fp32 11.8), and for more than 2 (fp32: any) where K is long and one wave has all rows: each CTA
    // there has a part of K (4 x 2048 x 8192: 10.6 us against 13.6, fp32 13.9 against 17.8; 1 x 1024 x 4096 in fp32: 8.2
    // against 17.3; 8 x 8192 x 8192: 21.2 against 26.6, but fp32 31 against 28;
    // 8 x 128256 x 2048: 79 against 49)
    const bool f32 = dtype == FLEXLLM_F32;
    if (M > 8 || ((M > 2 || f32) && K >= 4096 && N <= (f32 ? 32L : 128L) * gemm_sm_count())) return linear_w4_tc(c, f32, (cudaStream_t)stream);
    W4Args p = {};
    static_cast<W4Call&>(p) = c;
    return f32 ? pick_w4<float>(p, (cudaStream_t)stream) : pick_w4<bf16>(p, (cudaStream_t)stream);
}
