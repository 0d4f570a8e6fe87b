// Attention of packed rows over their sequences' pages in fp32, on the tensor cores (heads up to 128). A number is the sum of three bf16 parts of eight bits
// each, which hold it to the last bit; a product is the six of nine products of parts that reach 2^-24 of it, summed in fp32. Six bf16 MMAs
// are a quarter of what the same product takes the fp32 units.
// An MMA cuts its fp32 sums instead of rounding them: half a step on average, for every 16 products. So the sums in TMEM are short, the small products
// first and the large ones of one page last, and the pages' outputs are added up by fp32 units, rounded (all pages in one sum in TMEM:
// 5e-5 low after 10,000 keys, 5e-4 after 80,000).
// A tile is 128 rows (tokens x the query heads of one key/value head), walked page by page with the running softmax of the bf16 kernel:
//   warps 12, 14   bring K and V^T of a page in pieces of up to 4 KB, a lane for each cutting warp (one warp for both would hold the one back for
//                  the other: with two slots, heads of 128, a fifth slower)
//   warps 4 .. 11  cut them into parts, in swizzled shared memory (Q at the start, into TMEM)
//   warp 13        S = Q K^T of the next page, then P V of this one; Q and P come from TMEM
//   warps 0 .. 3   one row per thread: maximum, weights 2^(S scale log2 e - m) in three parts, sums of the weights and of the pages' outputs. The latter
//                  are in TMEM, or in shared memory where the columns are taken (heads of more than 96). (Held in registers by the cutting warps,
//                  whose code is left too few: 10 to 20 % slower)
// Few tiles: a cluster of CTAs cuts the keys.
// Shared memory bounds it: for a page of heads of 128, 512 clocks of copies, 512 of reads and 768 of writes to cut it, 1536 of reads by the MMAs, 1024 for the
// sums of a full tile, and the cutting waits for its turn in between; the tensor cores run a fifth of the time. 66 tokens of four sequences over 1350 to 3000,
// 16 / 4 heads of 128: 46 us; three prompts of 380 behind 280 to 700, 8 / 2 heads of 64: 32 us; one token over 84500, one head of 128: 290 us; 1500 tokens
// behind 1000, 32 / 8 heads of 128: 324 us, 133 TFLOP/s, nearly twice what the fp32 units could. The rounded sums cost 7 to 10 % of these times.
#include "attention_join.cuh"

namespace flexllm {

using namespace tc;

namespace {

constexpr int kF32Threads = 480, kMostSlots = 4;     // slots for pieces per cutting warp: 4 or 2
constexpr uint32_t kPieceBytes = 4096;

struct F32Args {
    PagedAttn a;
    int RC, HC, TQ, heads;                 // heads per tile, head chunks per group, tokens per tile, head chunks
    int kc, kq, vr, n_split;               // 128-byte blocks of a part's K row, 32-element chunks of a Q row, rows of a V^T part
    int v_rows, slots_log, two;            // rows of V^T of a cutting warp; its slots; K's and V's parts have two stages (1) or one (0)
    int x_log, sum_at;                     // log2 of the buffers of a page's outputs in TMEM; column of the sums, 0: in shared memory
    float a2;                              // scale * log2 e
};
struct F32Smem { uint32_t v, raw, sums, bars, total; };      // K's parts, V's, pieces, the outputs' sums
__host__ __device__ inline F32Smem f32_smem(int kc, int vr, int slots_log, int two, bool sums) {
    F32Smem o;
    o.v = (3u << two) * kc * 8192u;
    o.raw = o.v + (3u << two) * vr * 128u;
    o.sums = o.raw + (8u << slots_log) * kPieceBytes;
    o.bars = o.sums + (sums ? (uint32_t)(vr + 31) / 32 * 32 * 512u : 0u);
    o.total = o.bars + 1024u + 1024u;
    return o;
}

// TMEM: S, P, then the outputs of a page (one or two buffers), their sums where there is room, Q at the end
constexpr uint32_t kPCol = 64, kXCol = 160;
__host__ __device__ inline uint32_t q_col(int kq) { return 512u - 48u * (uint32_t)kq; }
__host__ __device__ inline uint32_t x_stride(int vr) { return (uint32_t)(vr + 31) / 32 * 32; }

// Two numbers less what is nearest to them in bf16, which is `w`: exact
__device__ __forceinline__ f32x2 rest2(f32x2 f, uint32_t w) { return fma2(pack2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)), pack2(-1.0f, -1.0f), f); }
__device__ __forceinline__ uint32_t near2(f32x2 f) {
    float x, y;
    unpack2(f, x, y);
    return bf_pack(x, y);
}
// 8 numbers as their three parts: twice what is nearest in eight bits, and the rest. Where an infinity or a NaN is among them, a NaN is in some part.
__device__ __forceinline__ void cut8(const float (&f)[8], uint4 (&part)[3]) {
    f32x2 v[4];
#pragma unroll
    for (int j = 0; j < 4; j++) v[j] = pack2(f[2 * j], f[2 * j + 1]);
#pragma unroll
    for (int p = 0; p < 3; p++) {
        const uint32_t w[4] = {near2(v[0]), near2(v[1]), near2(v[2]), near2(v[3])};
        part[p] = make_uint4(w[0], w[1], w[2], w[3]);
#pragma unroll
        for (int j = 0; j < 4; j++) v[j] = rest2(v[j], w[j]);
    }
}
// 32 bytes per lane, the lanes' side by side. Every other four lanes read their second half first (flip 16), so that eight lanes meet all banks once.
__device__ __forceinline__ void load8_shared(uint32_t at, uint32_t flip, float (&f)[8]) {
    float x[4], y[4];
    asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(x[0]), "=f"(x[1]), "=f"(x[2]), "=f"(x[3]) : "r"(at + flip));
    asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(y[0]), "=f"(y[1]), "=f"(y[2]), "=f"(y[3]) : "r"(at + (flip ^ 16u)));
#pragma unroll
    for (int i = 0; i < 4; i++) { f[i] = flip ? y[i] : x[i]; f[4 + i] = flip ? x[i] : y[i]; }
}
__device__ __forceinline__ void store_shared(uint32_t at, const uint4& v) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
__device__ __forceinline__ void bulk_copy(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}

__global__ void __launch_bounds__(kF32Threads, 1) attn_paged_f32_kernel(const __grid_constant__ F32Args t) {
    extern __shared__ uint8_t smem_raw[];
    __shared__ Unit unit_sm;
    __shared__ unsigned redo_sm[4];
    const uint32_t raw = smem_u32(smem_raw), base = (raw + 1023u) & ~1023u;
    uint8_t* base_ptr = smem_raw + (base - raw);
    const PagedAttn& a = t.a;
    const F32Smem o = f32_smem(t.kc, t.vr, t.slots_log, t.two, t.sum_at == 0);
    uint64_t* bars = reinterpret_cast<uint64_t*>(base_ptr + o.bars);
    const uint32_t bar_rf = smem_u32(bars), bar_re = bar_rf + 64 * kMostSlots, bar_q = bar_re + 64 * kMostSlots, bar_k = bar_q + 8, bar_ke = bar_k + 16, bar_v = bar_ke + 16,
                   bar_ve = bar_v + 16, bar_s = bar_ve + 16, bar_r = bar_s + 8, bar_p = bar_r + 8, bar_o = bar_p + 8, bar_x = bar_o + 8;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 96);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int i = 0; i < 8 * kMostSlots; i++) { mbar_init(bar_rf + 8 * i, 1); mbar_init(bar_re + 8 * i, 1); }
        for (int i = 0; i < 2; i++) { mbar_init(bar_k + 8 * i, 4); mbar_init(bar_ke + 8 * i, 1); mbar_init(bar_v + 8 * i, 4); mbar_init(bar_ve + 8 * i, 1); mbar_init(bar_x + 8 * i, 4); }
        mbar_init(bar_q, 8); mbar_init(bar_s, 1); mbar_init(bar_r, 4); mbar_init(bar_p, 4); mbar_init(bar_o, 1);
        *abort_flag = 0;
        fence_barrier_init();
    }
    if (threadIdx.x < 4) redo_sm[threadIdx.x] = 0;
    if (warp == 13) { tmem_alloc(smem_u32(tmem_slot), 512); tmem_relinquish(); }
    pdl_wait();
    const int tile = blockIdx.x / t.n_split, split = blockIdx.x % t.n_split, hg = tile % t.heads;
    if (warp == 0) {
        const int TQ = t.TQ;
        const Unit u = find_unit(a.seq, tile / t.heads, TQ, 1, [TQ](const SeqRows& s) { return (s.n + TQ - 1) / TQ; });
        if (lane == 0) unit_sm = u;
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    pdl_launch();                                         // behind the allocation: no later kernel may hold the TMEM that this one waits for
    const uint32_t tmem = *tmem_slot, tP = tmem + kPCol, tX = tmem + kXCol, tQ = tmem + q_col(t.kq);      // S at the start
    const int b = unit_sm.b;
    const SeqRows s = unit_sm.s;
    const int R = a.H / a.G, g = hg / t.HC, h0 = g * R + (hg % t.HC) * t.RC, heads = min(t.RC, (g + 1) * R - h0);
    const int i0 = unit_sm.i * t.TQ;                      // first row of the tile within the sequence
    const int end = b < 0 ? 0 : a.mask ? s.ctx + s.n : min(s.ctx + i0 + t.TQ, s.ctx + s.n), n_pg = (end + kPage - 1) / kPage;
    const int t0 = (int)((long)n_pg * split / t.n_split), t1 = (int)((long)n_pg * (split + 1) / t.n_split);
    auto wait = [&](uint32_t bar, uint32_t parity) { return __all_sync(0xffffffffu, mbar_spin(bar, parity, abort_flag)) != 0; };
    if (b >= 0) {
    if (warp == 12 || warp == 14) {
        // lane w brings what the cutting warp w (K) or w + 4 (V) has of a page, in two pieces
        const bool keys = warp == 12;
        const int c = lane & 3, rows = lane >= 4 ? 0 : keys ? 16 : max(min(t.v_rows, a.dv - c * t.v_rows), 0), half = keys ? 8 : t.v_rows / 2;
        const int width = keys ? a.dk : kPage;
        const float* from = keys ? (const float*)a.k + (long)c * 16 * a.dk : (const float*)a.v + (long)c * t.v_rows * kPage;
        const long page_size = (long)a.G * kPage * (keys ? a.dk : a.dv), head = (long)g * kPage * (keys ? a.dk : a.dv);
        bool ok = true;
        int ids = 0, u = 0;
        for (int j = t0; j < t1; j++) {
            const int n = j - t0;
            if ((n & 31) == 0) ids = j + lane < t1 ? page_of(a.seq, b, j + lane) : 0;
            const float* src = from + __shfl_sync(0xffffffffu, ids, n & 31) * page_size + head;
            for (int r = 0; r < rows; r += half, u++) {
                const int slot = ((keys ? lane : lane + 4) << t.slots_log) + (u & ((1 << t.slots_log) - 1));
                ok = ok && mbar_spin(bar_re + 8 * slot, (uint32_t)(u >> t.slots_log & 1) ^ 1u, abort_flag);
                if (!ok) continue;
                const uint32_t bytes = (uint32_t)(min(half, rows - r) * width) * 4u;
                mbar_expect_tx(bar_rf + 8 * slot, bytes);
                bulk_copy(base + o.raw + slot * kPieceBytes, src + r * width, bytes, bar_rf + 8 * slot);
            }
            __syncwarp();
        }
    } else if (warp == 13) {
        const uint32_t leader = elect_leader(), u_tmem = (uint32_t)uniform_max((int)tmem);
        const int u0 = uniform_max(t0), u1 = uniform_max(t1);
        const uint32_t idesc_qk = umma_idesc_bf16(128, kPage), idesc_pv = umma_idesc_bf16(128, t.vr);
        const int ksteps = (a.dk + 15) / 16;
        const uint32_t k_lo = umma_desc_lo(base), v_lo = umma_desc_lo(base + o.v);
        // products of parts, the small ones first
        auto parts = [](int x, uint32_t& pa, uint32_t& pb) {
            pa = x == 1 ? 2u : x == 2 || x == 4 ? 1u : 0u;
            pb = x == 0 ? 2u : x == 2 || x == 3 ? 1u : 0u;
        };
        auto qk = [&](int n) {
            const uint32_t st = n & t.two;
            if (!wait(bar_k + 8 * st, (uint32_t)(n >> t.two & 1))) return false;
            if (n > 0 && !wait(bar_r, (uint32_t)(n - 1 & 1))) return false;      // the scores in front have been read
            tc_fence_after();
#pragma unroll
            for (int x = 0; x < 6; x++) {
                uint32_t pa, pb;
                parts(x, pa, pb);
                const uint32_t qa = u_tmem + q_col(t.kq) + pa * (uint32_t)t.kq * 16u, ka = k_lo + (st * 3u + pb) * (uint32_t)t.kc * 512u;
                for (int k = 0; k < ksteps; k++) umma_bf16_ts_lo(leader, u_tmem, qa + 8 * k, ka + (k >> 2) * 512u + 2 * (k & 3), idesc_qk, x > 0 || k > 0);
            }
            umma_commit_by(leader, bar_s);
            umma_commit_by(leader, bar_ke + 8 * st);
            return true;
        };
        bool ok = u0 < u1 && wait(bar_q, 0) && qk(0);
        for (int j = u0; ok && j < u1; j++) {
            const int n = j - u0;
            const uint32_t st = n & t.two, xb = n & ((1 << t.x_log) - 1), before = n >> t.x_log;
            if (j + 1 < u1 && !qk(n + 1)) break;          // under this page's softmax
            ok = wait(bar_v + 8 * st, (uint32_t)(n >> t.two & 1)) && wait(bar_p, (uint32_t)(n & 1));
            ok = ok && (before == 0 || wait(bar_x + 8 * xb, before - 1 & 1));      // the outputs that were in this buffer have been added up
            if (!ok) break;
            tc_fence_after();
#pragma unroll
            for (int x = 0; x < 6; x++) {
                uint32_t pa, pb;
                parts(x, pa, pb);
#pragma unroll
                for (uint32_t k = 0; k < 4; k++)
                    umma_bf16_ts_lo(leader, u_tmem + kXCol + xb * x_stride(t.vr), u_tmem + kPCol + 32 * pa + 8 * k, v_lo + (st * 3u + pb) * (uint32_t)t.vr * 8u + 2 * k, idesc_pv, x > 0 || k > 0);
            }
            umma_commit_by(leader, bar_o);
            umma_commit_by(leader, bar_ve + 8 * st);
        }
    } else if (warp >= 4 && warp < 12) {
        // ---- numbers into parts: 8 of them per thread and piece
        const int ct = threadIdx.x - 128, per = a.dk / 8;
        uint4 part[3];
        auto put = [&](uint32_t at, uint32_t stride, int row, int c) {         // the 16 bytes c of a row of all parts; `at` the row's block
#pragma unroll
            for (int p = 0; p < 3; p++) store_shared(base + at + p * stride + row * 128 + (((c ^ row) & 7) << 4), part[p]);
        };
        const uint32_t k_part = (uint32_t)t.kc * 8192u, v_part = (uint32_t)t.vr * 128u;
        if (t0 < t1) {
            // Q's parts into TMEM, two elements per column: warps w and w + 4 have the same rows, and 32-element chunks in turn
            const int row = threadIdx.x & 127, i = i0 + row / t.RC;
            const bool live = row < t.TQ * t.RC && i < s.n && row % t.RC < heads;
            const float* src = (const float*)a.q + (long)(s.row0 + i) * a.ldq + (long)(h0 + row % t.RC) * a.dk;
            for (int c = (warp - 4) >> 2; c < t.kq; c += 2) {
                uint32_t pk[3][16];
#pragma unroll
                for (int x = 0; x < 4; x++) {
                    float f[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
                    if (live && 32 * c + 8 * x < a.dk) load8(src + 32 * c + 8 * x, f);
                    cut8(f, part);
#pragma unroll
                    for (int p = 0; p < 3; p++) { pk[p][4 * x] = part[p].x; pk[p][4 * x + 1] = part[p].y; pk[p][4 * x + 2] = part[p].z; pk[p][4 * x + 3] = part[p].w; }
                }
                __syncwarp();
#pragma unroll
                for (int p = 0; p < 3; p++) tmem_st_32x16(tQ + (uint32_t)(p * t.kq + c) * 16u + ((uint32_t)((warp & 3) * 32) << 16), pk[p]);
            }
            if ((per & 1) && ct < kPage) {                // the last 16 elements of a product reach beyond the row: zeros in K
                part[0] = part[1] = part[2] = make_uint4(0, 0, 0, 0);
                for (uint32_t st = 0; st <= (uint32_t)t.two; st++) put((st * 3u * t.kc + (uint32_t)(per >> 3)) * 8192u, k_part, ct, per);
            }
            fence_proxy_async_smem();
            tmem_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar_q);
        }
        // warps 4 .. 7: 16 keys of K each, 8 .. 11: rows of V^T. A warp goes through its pieces without the others; a piece is in registers when the next
        // one is asked for
        const int w = warp - 4, c = w & 3, rows = w < 4 ? 16 : max(min(t.v_rows, a.dv - c * t.v_rows), 0), half = w < 4 ? 8 : t.v_rows / 2, wide = w < 4 ? per : 8;
        const uint32_t inv = 65535u / (uint32_t)wide + 1u, raw_at = base + o.raw, flip = (uint32_t)(lane >> 2 & 1) * 16u;
        const uint32_t full = w < 4 ? bar_k : bar_v, empty = w < 4 ? bar_ke : bar_ve;
        bool ok = true;
        int u = 0;
        for (int j = t0; ok && j < t1; j++) {
            const int n = j - t0, left = end - j * kPage;
            const uint32_t st = n & t.two, before = (uint32_t)(n >> t.two & 1) ^ 1u, to = w < 4 ? st * 3 * k_part : o.v + st * 3 * v_part;
            if (rows == 0) ok = wait(empty + 8 * st, before);
            for (int r = 0; ok && r < rows; r += half, u++) {
                const int count = min(half, rows - r) * wide;      // of 8 numbers, at most 128
                const int slot = (w << t.slots_log) + (u & ((1 << t.slots_log) - 1));
                ok = wait(bar_rf + 8 * slot, (uint32_t)(u >> t.slots_log & 1));
                if (!ok) break;
                float f[4][8];
#pragma unroll
                for (int x = 0; x < 4; x++)
                    if (lane + 32 * x < count) load8_shared(raw_at + slot * kPieceBytes + (lane + 32 * x) * 32, flip, f[x]);
                __syncwarp();
                if (lane == 0) mbar_arrive(bar_re + 8 * slot);
                if (r == 0) ok = wait(empty + 8 * st, before);
                if (!ok) break;
#pragma unroll
                for (int x = 0; x < 4; x++) {
                    const int e = lane + 32 * x;
                    if (e >= count) continue;
                    const int row = (int)(e * inv >> 16), col = e - row * wide;
                    // keys behind the sequence's last one were never written: zeros, so that a weight of zero stays without effect
                    if (w >= 4 && col * 8 + 8 > left)
#pragma unroll
                        for (int y = 0; y < 8; y++)
                            if (col * 8 + y >= left) f[x][y] = 0.0f;
                    cut8(f[x], part);
                    if (w < 4) put(to + (uint32_t)(col >> 3) * 8192u, k_part, c * 16 + r + row, col);
                    else put(to, v_part, c * t.v_rows + r + row, col);
                }
            }
            if (!ok) break;
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(full + 8 * st);
        }
    } else if (warp < 4) {
        // ---- one row per thread
        const int row = threadIdx.x;
        const uint32_t lane_addr = (uint32_t)(warp * 32) << 16;
        const int i = i0 + row / t.RC, hr = row % t.RC;
        const bool live = row < t.TQ * t.RC && i < s.n && hr < heads;
        const int sure = live ? sure_keys(a, s, i) : 0x40000000;
        const unsigned long long bits = live ? mask_bits(a, s, i) : 0ull;
        const bool busy = __any_sync(0xffffffffu, live);                                  // other warps' rows are nowhere read
        float m = kNoScore, l = 0.0f, al = 0.0f;
        // sums in shared memory: rows of whole 128 bytes, their 16-byte pieces turned by the row, so that eight lanes meet all banks once
        float* const sums = reinterpret_cast<float*>(base_ptr + o.sums) + (uint32_t)row * x_stride(t.vr);
        auto piece = [&](int d) { return sums + ((((uint32_t)d >> 2) ^ ((uint32_t)row & 7u)) << 2); };
        const uint32_t tSum = tmem + t.sum_at + lane_addr;
        // sums = sums * f + outputs of page n
        auto add_page = [&](int n, float f) {
            const int xb = n & ((1 << t.x_log) - 1);
            if (busy) {
                for (int d = 0; d < t.vr; d += 16) {
                    uint32_t u[16], v[16];
                    tmem_ld_32x16(tX + xb * x_stride(t.vr) + d + lane_addr, u);
                    if (n > 0) {
                        if (t.sum_at) tmem_ld_32x16(tSum + d, v);
                        else
#pragma unroll
                            for (int x = 0; x < 16; x += 4) *reinterpret_cast<uint4*>(v + x) = *reinterpret_cast<const uint4*>(piece(d + x));
                    }
                    tmem_ld_wait();
                    if (n > 0)
#pragma unroll
                        for (int x = 0; x < 16; x++) u[x] = __float_as_uint(__fmaf_rn(__uint_as_float(v[x]), f, __uint_as_float(u[x])));
                    if (t.sum_at) tmem_st_32x16(tSum + d, u);
                    else
#pragma unroll
                        for (int x = 0; x < 16; x += 4) *reinterpret_cast<uint4*>(piece(d + x)) = *reinterpret_cast<const uint4*>(u + x);
                }
                tmem_st_wait();
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar_x + 8 * xb);
        };
        bool ok = true;
        for (int j = t0; j < t1; j++) {
            const int n = j - t0;
            if (!wait(bar_s, (uint32_t)(n & 1))) { ok = false; break; }
            tc_fence_after();
            uint32_t v[2][32];
            tmem_ld_32x32(tmem + lane_addr, v[0]);
            tmem_ld_32x32(tmem + 32 + lane_addr, v[1]);
            tmem_ld_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar_r);
            if (!__all_sync(0xffffffffu, sure - j * kPage >= kPage))
#pragma unroll
                for (int c = 0; c < 2; c++) {
                    const uint32_t see = seen_word(c, sure, bits, s.ctx, j * kPage);
#pragma unroll
                    for (int x = 0; x < 32; x++)
                        if (!(see >> x & 1u)) v[c][x] = 0xff800000u;
                }
            float mx = fmaxf(__uint_as_float(v[0][0]), __uint_as_float(v[1][0])), my = fmaxf(__uint_as_float(v[0][1]), __uint_as_float(v[1][1]));
#pragma unroll
            for (int x = 2; x < 32; x += 2) {
                mx = max3(mx, __uint_as_float(v[0][x]), __uint_as_float(v[1][x]));
                my = max3(my, __uint_as_float(v[0][x + 1]), __uint_as_float(v[1][x + 1]));
            }
            const float top = fmaxf(mx, my) * t.a2, m_new = top > m + kSlack ? top : m, al_n = ex2_fast(m - m_new);
            m = m_new;
            l *= al_n;
            f32x2 sum = pack2(0.0f, 0.0f);
#pragma unroll
            for (int c = 0; c < 2; c++) {
                uint32_t pk[3][16];
#pragma unroll
                for (int x = 0; x < 32; x += 2) {
                    const float e0 = ex2_fast(__fmaf_rn(__uint_as_float(v[c][x]), t.a2, -m)), e1 = ex2_fast(__fmaf_rn(__uint_as_float(v[c][x + 1]), t.a2, -m));
                    f32x2 e = pack2(e0, e1);
                    sum = add2(sum, e);
#pragma unroll
                    for (int p = 0; p < 3; p++) {
                        pk[p][x >> 1] = near2(e);
                        e = rest2(e, pk[p][x >> 1]);
                    }
                }
                if (c == 0 && n > 0) {                    // the weights in front have been read
                    if (!wait(bar_o, (uint32_t)((n - 1) & 1))) { ok = false; break; }
                    tc_fence_after();
                }
#pragma unroll
                for (int p = 0; p < 3; p++) tmem_st_32x16(tP + 32 * p + 16 * c + lane_addr, pk[p]);
            }
            if (!ok) break;
            float s0, s1;
            unpack2(sum, s0, s1);
            l += s0 + s1;
            tmem_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar_p);
            if (n > 0) add_page(n - 1, al);               // under the products with this page
            al = al_n;
        }
        const bool any = t0 < t1;
        if (ok && any) ok = wait(bar_o, (uint32_t)((t1 - t0 - 1) & 1));
        if (ok) {
            tc_fence_after();
            if (any) add_page(t1 - t0 - 1, al);
            const float rl = t.n_split > 1 ? 1.0f : l == 0.0f ? 0.0f : 1.0f / l;
            bool odd = live && t.n_split == 1 && l == 0.0f && (sure > 0 || bits != 0);
            float* orow = reinterpret_cast<float*>(base_ptr) + (long)row * (a.dv + 4);
            float* out = (float*)a.out + (long)(s.row0 + i) * a.ldo + (long)(h0 + hr) * a.dv;
            const bool vec = whole_stores<float>(a);
            for (int d0 = 0; d0 < t.vr; d0 += 16) {
                uint32_t u[16];
                if (any && t.sum_at) {
                    tmem_ld_32x16(tSum + d0, u);
                    tmem_ld_wait();
                } else if (any) {
#pragma unroll
                    for (int x = 0; x < 16; x += 4) *reinterpret_cast<uint4*>(u + x) = *reinterpret_cast<const uint4*>(piece(d0 + x));
                } else {
#pragma unroll
                    for (int x = 0; x < 16; x++) u[x] = 0;
                }
#pragma unroll
                for (int c = 0; c < 16; c += 8) {
                    if (d0 + c >= a.dv) continue;
                    float f[8];
#pragma unroll
                    for (int x = 0; x < 8; x++) f[x] = t.n_split == 1 && l == 0.0f ? 0.0f : __uint_as_float(u[c + x]) * rl;
                    if (t.n_split > 1) {                  // this part's row into shared memory, over the operands (every product has been waited for)
                        store8f(orow + d0 + c, f, true);
                    } else if (live) {
#pragma unroll
                        for (int x = 0; x < 8; x++) odd = odd || not_finite(f[x]);
                        store8f(out + d0 + c, f, vec);
                    }
                }
            }
            if (t.n_split > 1) {
                float* ml = reinterpret_cast<float*>(base_ptr) + 128 * (a.dv + 4);
                ml[row] = m; ml[128 + row] = l;
            } else {
                const unsigned bad = __ballot_sync(0xffffffffu, odd);
                if (lane == 0) redo_sm[warp] = bad;
            }
        }
    }
    }
    if (b >= 0 && t.n_split > 1) {
        cluster_sync();
        float* ml = reinterpret_cast<float*>(base_ptr) + 128 * (a.dv + 4);
        join_parts<float, 1>(a, s, i0, t.RC, t.TQ, heads, h0, t.n_split, split, base, smem_u32(ml), smem_u32(ml + 128), ml + 256, redo_sm, kF32Threads);
        cluster_sync();
    }
    tc_fence_before();
    __syncthreads();
    if ((redo_sm[0] | redo_sm[1] | redo_sm[2] | redo_sm[3]) && !*abort_flag)
        for (int row = warp; row < 128; row += kF32Threads / 32)
            if (redo_sm[row >> 5] >> (row & 31) & 1) attn_row_by_key<float>(a, b, s, i0 + row / t.RC, h0 + row % t.RC);
    if (*abort_flag) {
        const unsigned long long t_0 = globaltimer_ns();
        while (globaltimer_ns() - t_0 < 200000ull) { __nanosleep(1000); }
        if (threadIdx.x == 0 && a.seq.error_flag) atomicOr(a.seq.error_flag, 1);
        __syncthreads();
    }
    if (warp == 13) { tc_fence_after(); tmem_dealloc(tmem, 512); }
}

}  // namespace

int attn_paged_f32(const PagedAttn& a, cudaStream_t st) {
    F32Args t = {};
    const int R = a.H / a.G;
    t.a = a;
    t.RC = R < 128 ? R : 128; t.HC = (R + t.RC - 1) / t.RC; t.TQ = 128 / t.RC;
    t.kc = (a.dk + 63) / 64; t.kq = (a.dk + 31) / 32; t.vr = (a.dv + 15) / 16 * 16;
    t.v_rows = (a.dv + 31) / 32 * 8;
    t.a2 = score_factor(a);
    const long heads = (long)a.G * t.HC, seqs = a.seq.B < a.seq.T ? a.seq.B : a.seq.T, ones = most_units(a.seq, t.TQ);
    t.heads = (int)heads;
    if (ones * 16 * heads > 0x7fffffffL) return FLEXLLM_ENOTSUP;
    const long tiles = ((a.seq.T + seqs - 1) / seqs + t.TQ - 1) / t.TQ * seqs * heads;
    t.n_split = key_splits(tiles, false, (a.seq.max_ctx + kPage) / kPage, 2, 16);
    // the sums of the outputs in TMEM where a page's outputs leave room, twice, so that the next page's products need not wait for the addition, or once
    const uint32_t xs = x_stride(t.vr), room = q_col(t.kq) - kXCol;
    t.x_log = 2 * xs + t.vr <= room;
    t.sum_at = (1u << t.x_log) * xs + t.vr <= room ? kXCol + (xs << t.x_log) : 0;
    // two stages while two slots fit beside them; four slots where they fit
    auto fits = [&](int slots_log, int two) { return f32_smem(t.kc, t.vr, slots_log, two, t.sum_at == 0).total <= 226u * 1024u; };
    t.two = fits(1, 1);
    t.slots_log = fits(2, t.two) ? 2 : 1;
    const F32Smem o = f32_smem(t.kc, t.vr, t.slots_log, t.two, t.sum_at == 0);
    if (o.total > 226u * 1024u || (128u * (a.dv + 4) + 256u + kJoinRows) * 4u > o.sums) return FLEXLLM_ENOTSUP;
    TRY_RC(allow_shared(attn_paged_f32_kernel, o.total));
    TRY_RC(allow_cluster(attn_paged_f32_kernel, t.n_split));
    launch_cluster(attn_paged_f32_kernel, dim3((unsigned)(ones * t.n_split * heads)), dim3(kF32Threads), t.n_split, o.total, st, t);
    return launch_status();
}

}  // namespace flexllm
