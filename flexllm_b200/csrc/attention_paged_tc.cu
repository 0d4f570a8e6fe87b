// Attention of packed rows over their sequences' pages in bf16, on the tensor cores (tcgen05). A tile is 128 rows: TQ consecutive tokens of a
// sequence x the RC query heads of a key/value head (row = token * RC + head), so that a group's heads share every K and V tile. The kernel
// walks the keys in tiles of 128 (two pages) with a running softmax:
//   S = Q K^T into TMEM; one thread per row reads its 128 scores, P = 2^(S scale log2 e - m) goes back over them as bf16, and
//   O += P V takes P from TMEM and V^T from the pages as they lie (keys along the inner index)
// m is lazy: only a row whose maximum exceeds it by more than kSlack moves it and rescales its O in TMEM.
// P is rounded to bf16 since both operands of an MMA have one type, and a second part would double the products with V: results are off by 1.9e-3 to 2.3e-3
// (root of the mean square, relative), where rounding the result alone leaves 1.6e-3. The weights' sum is of the unrounded ones, in fp32. O is the
// tensor core's fp32 sum, which it cuts instead of rounding: 5e-4 low after 80,000 keys in one part and 2.5e-3 after a million, when half a step of the result is 2e-3 to 3.9e-3.
//   kPair   two tiles per CTA, so that one tile's softmax runs under the other's products: prompts
//   kOne    one tile per CTA, two CTAs per SM: more tiles than SMs; and heads of more than 128
//   kTurns  one tile per CTA with two sets of scores, outputs and softmax warps that take the key tiles in turn: fewer tiles than SMs (trees,
//           decoding), whose keys are also cut among the CTAs of a cluster
// Where a tile's keys are cut, the parts' maxima, sums and outputs meet in shared memory, in a fixed order.
// Warps 0 .. 4 W - 1 softmax (W sets, one row per thread), then one for TMA, one for the MMAs.
// Bound by, and measured: prompts (kPair) by the chain from scores to weights and back, the tensor cores busy 42 % (16384 tokens, 32 / 8 heads of 128: 2.0 ms,
// 1.08 PFLOP/s, 66 % of the measured bf16 rate; 4000 tokens 151 us, 0.87 PFLOP/s); trees (kOne) by that chain and the differences
// between sequences (16 of 25 tokens over 8000: 89 us, 4.2 TB/s); single tokens by the products, which take 128 rows for a few (one over 84500: 81 us,
// 4.3 TB/s, the tensor cores busy 73 % on 80 SMs); short calls by latency (26 tokens over 1000: 14 us, eight prompts of 143: 11.6 us).
// Keys behind a sequence's last one were never written: their scores are replaced, their values zeroed in shared memory. Any other value
// that a row does not see meets a weight of zero; a row whose result is not finite, or whose weights are all zero
// although it sees a key, is computed again, key by key.
#include "attention_join.cuh"

namespace flexllm {

using namespace tc;

namespace {

enum { kOne, kPair, kTurns };
constexpr int KT = 128;                    // keys per tile

struct TcArgs {
    PagedAttn a;
    int RC, HC, TQ, heads;                 // heads per tile, head chunks per group, tokens per tile, head chunks
    uint32_t q_block;                      // bytes of a 128-byte block of the rows of Q. The products take 128 rows, so those of a short tile read on into K
    int kc, vr;                            // 128-byte blocks of a Q or K row, rows of a V^T tile (dv rounded up to 16)
    int ks, vs;                            // stages of K and V
    float a2;                              // scale * log2 e
    int tmem_cols, o_stride, n_split;
};
// Stage of a ring and the parity of its round, counted up: a quotient by a stage count that is only known at run time takes one thread 250 clocks
// (a tile's four of them took as long as its products).
struct Ring {
    int st; uint32_t ph; const int n;
    __device__ __forceinline__ Ring(int n_, int at) : st(at % n_), ph((uint32_t)(at / n_) & 1u), n(n_) {}
    __device__ __forceinline__ void next() { if (++st == n) { st = 0; ph ^= 1u; } }
};
struct TcSmem { uint32_t k, v, bars, total; };
__host__ __device__ inline TcSmem tc_smem(int NQ, uint32_t q_block, int kc, int vr, int ks, int vs) {
    TcSmem o;
    o.k = (uint32_t)(NQ * kc) * q_block;
    o.v = o.k + (uint32_t)(ks * kc) * 16384u;
    o.bars = o.v + (uint32_t)(vs * vr) * 256u;
    o.total = o.bars + 256u + 1024u;
    return o;
}
constexpr int kMaxStages = 4;
constexpr uint32_t kHalfSm = 108 * 1024, kWholeSm = 224 * 1024;       // dynamic shared memory; a few KB are static

template <int MODE>
__global__ void __launch_bounds__(MODE == kOne ? 192 : 320, MODE == kOne ? 2 : 1) attn_paged_tc_kernel(const __grid_constant__ CUtensorMap tmapQ, const __grid_constant__ CUtensorMap tmapK,
                                                                         const __grid_constant__ CUtensorMap tmapV, const __grid_constant__ TcArgs t) {
    constexpr int NQ = MODE == kPair ? 2 : 1;             // tiles
    constexpr int W = MODE == kOne ? 1 : 2;               // sets of scores and outputs
    constexpr int STEP = MODE == kTurns ? 2 : 1;          // set w takes the key tiles w * (STEP - 1), + STEP, ..
    constexpr int WT = W * 4, WM = WT + 1, NT = W * 128 + 64;      // the TMA warp, the MMA warp, threads
    extern __shared__ uint8_t smem_raw[];
    __shared__ Unit unit_sm;
    __shared__ unsigned redo_sm[4 * NQ];
    __shared__ float m_sm[W * 128], l_sm[W * 128], w_sm[NQ == 2 ? 1 : kJoinRows * STEP];
    const uint32_t raw = smem_u32(smem_raw), base = (raw + 1023u) & ~1023u;
    uint8_t* base_ptr = smem_raw + (base - raw);
    const PagedAttn& a = t.a;
    const TcSmem o = tc_smem(NQ, t.q_block, t.kc, t.vr, t.ks, t.vs);
    uint64_t* bars = reinterpret_cast<uint64_t*>(base_ptr + o.bars);
    const uint32_t bar_q = smem_u32(bars), bar_kf = bar_q + 8, bar_ke = bar_kf + 8 * kMaxStages, bar_vf = bar_ke + 8 * kMaxStages,
                   bar_ve = bar_vf + 8 * kMaxStages, bar_s = bar_ve + 8 * kMaxStages, bar_p = bar_s + 16, bar_o = bar_p + 16, bar_f = bar_o + 16, bar_h = bar_f + 16;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 28);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        mbar_init(bar_q, 1);
        for (int i = 0; i < kMaxStages; i++) { mbar_init(bar_kf + 8 * i, 1); mbar_init(bar_ke + 8 * i, 1); mbar_init(bar_vf + 8 * i, 1); mbar_init(bar_ve + 8 * i, 1); }
        for (int i = 0; i < 2; i++) { mbar_init(bar_s + 8 * i, 1); mbar_init(bar_p + 8 * i, 4); mbar_init(bar_o + 8 * i, 1); mbar_init(bar_f + 8 * i, 1); mbar_init(bar_h + 8 * i, 4); }
        *abort_flag = 0;
        fence_barrier_init();
    }
    if (threadIdx.x < 4 * NQ) redo_sm[threadIdx.x] = 0;
    if (warp == WM) { tmem_alloc(smem_u32(tmem_slot), t.tmem_cols); tmem_relinquish(); }
    if (warp == WT && lane == 0) { tma_prefetch_desc(&tmapQ); tma_prefetch_desc(&tmapK); tma_prefetch_desc(&tmapV); }
    pdl_wait();
    // tiles' heads before tiles, so that CTAs without a tile (the host knows the most there can be) start when no other is left
    const int tile = blockIdx.x / t.n_split, split = blockIdx.x % t.n_split, hg = tile % t.heads;
    if (warp == 0) {
        const int per = NQ * t.TQ;
        const Unit u = find_unit(a.seq, tile / t.heads, per, 1, [per](const SeqRows& s) { return (s.n + per - 1) / per; });
        if (lane == 0) unit_sm = u;
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    pdl_launch();                                         // behind the allocation: no later kernel may hold the TMEM that this one waits for
    const uint32_t tmem = *tmem_slot;
    const int b = unit_sm.b;
    const SeqRows s = unit_sm.s;
    const int R = a.H / a.G, g = hg / t.HC, h0 = g * R + (hg % t.HC) * t.RC, heads = min(t.RC, (g + 1) * R - h0);
    const int i0 = unit_sm.i * NQ * t.TQ;                 // first row of the first tile within the sequence
    // key tiles [t0, t1[q]) of the tiles q; `end`: keys that exist for the last row
    int end = 0, t0 = 0, t1[NQ];
#pragma unroll
    for (int q = 0; q < NQ; q++) {
        t1[q] = 0;
        if (b < 0 || i0 + q * t.TQ >= s.n) continue;
        end = a.mask ? s.ctx + s.n : min(s.ctx + i0 + (q + 1) * t.TQ, s.ctx + s.n);
        const int n = (end + KT - 1) / KT;
        t0 = (int)((long)n * split / t.n_split);          // pairs are never cut
        t1[q] = (int)((long)n * (split + 1) / t.n_split);
    }
    const int t_last = t1[0] > t1[NQ - 1] ? t1[0] : t1[NQ - 1];

    if (b >= 0) {
    if (warp == WT) {
        // ---- Q, then K and V page by page; the page ids of 32 pages at a time in the warp's lanes
        if (lane == 0 && t0 < t_last) {
            mbar_expect_tx(bar_q, (uint32_t)(NQ * t.kc * t.TQ * t.RC) * 128u);
            for (int q = 0; q < NQ; q++)
                for (int i = 0; i < t.kc; i++) tma_load_3d(base + (uint32_t)(q * t.kc + i) * t.q_block, &tmapQ, bar_q, i * 128, h0, s.row0 + i0 + q * t.TQ);
        }
        const int n_pg = (end + kPage - 1) / kPage;
        int ids = 0;
        Ring rk(t.ks, 0), rv(t.vs, 0);
        for (int j = t0; j < t_last; j++, rk.next(), rv.next()) {
            const int n = j - t0, sk = rk.st, sv = rv.st;
            if ((n & 15) == 0) ids = 2 * j + lane < n_pg ? page_of(a.seq, b, 2 * j + lane) : 0;
            const int p0 = __shfl_sync(0xffffffffu, ids, 2 * (n & 15)), p1 = __shfl_sync(0xffffffffu, ids, 2 * (n & 15) + 1);
            const int pages = 2 * j + 1 < n_pg ? 2 : 1;
            int ok = 1;
            if (lane == 0) {
                ok = mbar_spin(bar_ke + 8 * sk, rk.ph ^ 1u, abort_flag);
                if (ok) {
                    mbar_expect_tx(bar_kf + 8 * sk, (uint32_t)(t.kc * pages) * 8192u);
                    for (int p = 0; p < pages; p++)
                        for (int i = 0; i < t.kc; i++)
                            tma_load_2d(base + o.k + (uint32_t)(sk * t.kc + i) * 16384u + p * 8192u, &tmapK, bar_kf + 8 * sk, i * 128, ((p ? p1 : p0) * a.G + g) * kPage);
                    ok = mbar_spin(bar_ve + 8 * sv, rv.ph ^ 1u, abort_flag);
                }
                if (ok) {
                    mbar_expect_tx(bar_vf + 8 * sv, (uint32_t)(t.vr * pages) * 128u);
                    for (int p = 0; p < pages; p++)
                        tma_load_2d(base + o.v + (uint32_t)(sv * 2 + p) * t.vr * 128u, &tmapV, bar_vf + 8 * sv, 0, ((p ? p1 : p0) * a.G + g) * a.dv);
                }
            }
            if (!__shfl_sync(0xffffffffu, ok, 0)) break;
        }
    } else if (warp == WM) {
        const uint32_t idesc_qk = umma_idesc_bf16(128, KT), idesc_pv = umma_idesc_bf16(128, t.vr);
        const int ksteps = (a.dk + 15) / 16;
        const uint32_t leader = elect_leader();
        // the same for all lanes, and known to be: the bounds of this warp's loops
        const int u0 = uniform_max(t0), u_last = uniform_max(t_last), u_end = uniform_max(end);
        int u1[NQ];
#pragma unroll
        for (int q = 0; q < NQ; q++) u1[q] = uniform_max(t1[q]);
        auto wait = [&](uint32_t bar, uint32_t parity) { return __all_sync(0xffffffffu, mbar_spin(bar, parity, abort_flag)) != 0; };
        const uint32_t u_tmem = (uint32_t)uniform_max((int)tmem), tP = u_tmem + W * KT, page = (uint32_t)t.vr * 8u;
        const uint32_t q_lo = umma_desc_lo(base), k_lo = umma_desc_lo(base + o.k), v_lo = umma_desc_lo(base + o.v);
        // S of set w = Q K_j^T, over the weights that the product in front has read
        auto qk = [&](int w, int j, const Ring& r) {
            const int q = NQ == 2 ? w : 0;
            if (!wait(bar_kf + 8 * r.st, r.ph)) return false;
            tc_fence_after();
            const uint32_t q_step = t.q_block >> 4, a_at = q_lo + (uint32_t)(q * t.kc) * q_step, b_at = k_lo + (uint32_t)(r.st * t.kc) * 1024u, d_at = u_tmem + w * KT;
            for (int blk = 0; blk < ksteps >> 2; blk++)
#pragma unroll
                for (uint32_t k = 0; k < 4; k++) umma_bf16_lo(leader, d_at, a_at + blk * q_step + 2 * k, b_at + blk * 1024u + 2 * k, idesc_qk, blk + k > 0);
            for (int k = ksteps & ~3; k < ksteps; k++)
                umma_bf16_lo(leader, d_at, a_at + (k >> 2) * q_step + 2 * (k & 3), b_at + (k >> 2) * 1024u + 2 * (k & 3), idesc_qk, k > 0);
            umma_commit_by(leader, bar_s + 8 * w);
            if (q == NQ - 1 || j >= u1[NQ - 1]) umma_commit_by(leader, bar_ke + 8 * r.st);      // the last product with K_j
            return true;
        };
        bool ok = u0 < u_last && wait(bar_q, 0);
        for (int w = 0; w < W; w++) {
            const int j = u0 + w * (STEP - 1);
            if (ok && j < u1[NQ == 2 ? w : 0]) ok = qk(w, j, Ring(t.ks, j - u0));
        }
        Ring rk(t.ks, STEP), rv(t.vs, 0);                  // K of the tile that follows in the same set, V of this one
        for (int j = u0; ok && j < u_last; j++, rk.next(), rv.next()) {
            const int n = j - u0;
            ok = wait(bar_vf + 8 * rv.st, rv.ph);
#pragma unroll
            for (int q = 0; q < NQ; q++) {
                if (!ok || j >= u1[q]) continue;
                const int w = MODE == kTurns ? n & 1 : q;
                const uint32_t b_at = v_lo + (uint32_t)(rv.st * 2) * page, p_at = u_tmem + w * KT, d_at = tP + w * t.o_stride;
                // the weights of the first 64 keys, then the others. A tile that ends early is only right when its values' zeros are there too
#pragma unroll
                for (uint32_t half = 0; half < 2; half++) {
                    ok = ok && wait((half == 0 && u_end - j * KT >= KT ? bar_h : bar_p) + 8 * w, (uint32_t)(n / STEP & 1));
                    if (!ok) break;
                    tc_fence_after();
#pragma unroll
                    for (uint32_t k = 0; k < 4; k++) umma_bf16_ts_lo(leader, d_at, p_at + 32 * half + 8 * k, b_at + half * page + 2 * k, idesc_pv, n >= STEP || half + k > 0 ? 1u : 0u);
                }
                if (!ok) continue;
                umma_commit_by(leader, (j + STEP < u1[q] ? bar_o : bar_f) + 8 * w);        // the last one has a barrier of its own
                if (q == NQ - 1 || j >= u1[NQ - 1]) umma_commit_by(leader, bar_ve + 8 * rv.st);
                if (j + STEP < u1[q]) ok = qk(w, j + STEP, rk);
            }
        }
    } else {
        // ---- one row per thread
        const int w = warp >> 2, q = NQ == 2 ? w : 0, row = threadIdx.x & 127;
        const uint32_t lane_addr = (uint32_t)((warp & 3) * 32) << 16;
        const int i = i0 + q * t.TQ + row / t.RC, hr = row % t.RC;
        const bool live = row < t.TQ * t.RC && i < s.n && hr < heads;
        const bool busy = __any_sync(0xffffffffu, live);                                  // other warps' rows are nowhere read
        const int sure = live ? sure_keys(a, s, i) : 0x40000000;                          // rows of the tile without a token mask nothing
        const unsigned long long bits = live ? mask_bits(a, s, i) : 0ull;
        const uint32_t tO = tmem + W * KT + w * t.o_stride + lane_addr;
        const int my_t0 = t0 + w * (STEP - 1), my_t1 = q == 1 ? t1[NQ - 1] : t1[0];
        auto wait_bar = [&](uint32_t bar, uint32_t parity) { return __all_sync(0xffffffffu, mbar_spin(bar, parity, abort_flag)) != 0; };
        float m = kNoScore;
        f32x2 l2[2] = {pack2(0.0f, 0.0f), pack2(0.0f, 0.0f)};
        const f32x2 a22 = pack2(t.a2, t.a2);
        bool ok = true;
        for (int j = my_t0; j < my_t1; j += STEP) {
            const int n = j - t0, turn = n / STEP, left = end - j * KT;
            if (!wait_bar(bar_s + 8 * w, (uint32_t)(turn & 1))) { ok = false; break; }
            tc_fence_after();
            const uint32_t tS = tmem + w * KT + lane_addr;
            if (!busy) {
                if (lane == 0) mbar_arrive(bar_h + 8 * w);
            } else {
            uint32_t v[4][32];
#pragma unroll
            for (int c = 0; c < 4; c++) tmem_ld_32x32(tS + 32 * c, v[c]);
            tmem_ld_wait();
            const int hi = sure - j * KT;
            const bool masked = !__all_sync(0xffffffffu, hi >= KT);
            if (masked) {
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    const uint32_t see = seen_word(c, sure, bits, s.ctx, j * KT);
#pragma unroll
                    for (int x = 0; x < 32; x++)
                        if (!(see >> x & 1u)) v[c][x] = 0xff800000u;
                }
            }
            float mx[4];
#pragma unroll
            for (int c = 0; c < 4; c++) {
                mx[c] = fmaxf(__uint_as_float(v[c][0]), __uint_as_float(v[c][1]));
#pragma unroll
                for (int x = 2; x < 32; x += 2) mx[c] = max3(mx[c], __uint_as_float(v[c][x]), __uint_as_float(v[c][x + 1]));
            }
            const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * t.a2;
            const bool grow = live && top > m + kSlack;
            if (__any_sync(0xffffffffu, grow)) {
                const float m_new = grow ? top : m, al = ex2_fast(m - m_new);
                m = m_new;
                l2[0] = mul2(l2[0], pack2(al, al)); l2[1] = mul2(l2[1], pack2(al, al));
                if (turn > 0) {
                    if (!wait_bar(bar_o + 8 * w, (uint32_t)((turn - 1) & 1))) { ok = false; break; }      // the products so far
                    tc_fence_after();
                    for (int d = 0; d < t.vr; d += 16) {
                        uint32_t u[16];
                        tmem_ld_32x16(tO + d, u);
                        tmem_ld_wait();
#pragma unroll
                        for (int x = 0; x < 16; x++) u[x] = __float_as_uint(__uint_as_float(u[x]) * al);
                        tmem_st_32x16(tO + d, u);
                    }
                }
            }
            const f32x2 nm = pack2(-m, -m);
#pragma unroll
            for (int c = 0; c < 4; c++) {
                uint32_t pk[16];
#pragma unroll
                for (int x = 0; x < 32; x += 2) {
                    float e0, e1;
                    unpack2(fma2(pack2(__uint_as_float(v[c][x]), __uint_as_float(v[c][x + 1])), a22, nm), e0, e1);
                    e0 = ex2_fast(e0); e1 = ex2_fast(e1);
                    l2[(x >> 1) & 1] = add2(l2[(x >> 1) & 1], pack2(e0, e1));
                    pk[x >> 1] = bf_pack(e0, e1);
                }
                tmem_st_32x16(tS + 16 * c, pk);
                if (c == 1) {                             // half the weights are there: their product may start
                    tmem_st_wait();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(bar_h + 8 * w);
                }
            }
            }
            if (left < KT) {                              // the sequence ends inside the tile: zeros for the values behind its end
                const int sv = n % t.vs, c0 = left >> 3;
                if (!wait_bar(bar_vf + 8 * sv, (uint32_t)(n / t.vs & 1))) { ok = false; break; }
                for (int d = row; d < t.vr; d += 128) {
                    uint8_t* vrow = base_ptr + o.v + (uint32_t)(sv * 2) * t.vr * 128u + d * 128;
                    for (int c = c0; c < 16; c++) {        // keys 8 c .. 8 c + 7
                        uint8_t* at = vrow + (uint32_t)(c >> 3) * t.vr * 128u + (((c ^ d) & 7) << 4);
                        if (c > c0 || !(left & 7)) *reinterpret_cast<uint4*>(at) = make_uint4(0, 0, 0, 0);
                        else
                            for (int x = left & 7; x < 8; x++) reinterpret_cast<uint16_t*>(at)[x] = 0;
                    }
                }
                fence_proxy_async_smem();
            }
            tmem_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar_p + 8 * w);
        }
        float l, l1;
        unpack2(add2(l2[0], l2[1]), l, l1);
        l += l1;
        const bool any = my_t0 < my_t1;
        if (ok && any) ok = wait_bar(bar_f + 8 * w, 0);
        if (MODE == kTurns) named_sync<1, 256>();          // every product of both sets has been waited for
        if (ok) {
            tc_fence_after();
            if (MODE == kPair || (MODE == kOne && t.n_split == 1)) {
                const float rl = l == 0.0f ? 0.0f : 1.0f / l;
                bool odd = live && l == 0.0f && (sure > 0 || bits != 0);
                bf16* out = (bf16*)a.out + (long)(s.row0 + i) * a.ldo + (long)(h0 + hr) * a.dv;
                const bool vec = (a.ldo & 7) == 0 && aligned16(a.out);
                for (int d0 = 0; d0 < t.vr; d0 += 32) {
                    uint32_t u[32];
                    tmem_ld_32x32(tO + d0, u);            // o_stride columns are this tile's
                    tmem_ld_wait();
                    if (!live) continue;
#pragma unroll
                    for (int c = 0; c < 32; c += 8) {
                        if (d0 + c >= a.dv) continue;
                        float f[8];
#pragma unroll
                        for (int x = 0; x < 8; x++) {
                            f[x] = l == 0.0f ? 0.0f : __uint_as_float(u[c + x]) * rl;
                            odd = odd || not_finite(f[x]);
                        }
                        if (vec) *reinterpret_cast<uint4*>(out + d0 + c) = make_uint4(bf_pack(f[0], f[1]), bf_pack(f[2], f[3]), bf_pack(f[4], f[5]), bf_pack(f[6], f[7]));
                        else
#pragma unroll
                            for (int x = 0; x < 8; x++) out[d0 + c + x] = __float2bfloat16_rn(f[x]);
                    }
                }
                const unsigned bad = __ballot_sync(0xffffffffu, odd);
                if (lane == 0) redo_sm[warp] = bad;
            } else {
                // this part's row into shared memory, over the operands
                float* orow = reinterpret_cast<float*>(base_ptr) + (long)(w * 128 + row) * (a.dv + 4);
                for (int d0 = 0; d0 < t.vr; d0 += 32) {
                    uint32_t u[32];
                    if (any) {
                        tmem_ld_32x32(tO + d0, u);
                        tmem_ld_wait();
                    } else {
#pragma unroll
                        for (int x = 0; x < 32; x++) u[x] = 0;
                    }
#pragma unroll
                    for (int x = 0; x < 32; x += 4)
                        if (d0 + x < a.dv) *reinterpret_cast<uint4*>(orow + d0 + x) = make_uint4(u[x], u[x + 1], u[x + 2], u[x + 3]);
                }
                m_sm[w * 128 + row] = m; l_sm[w * 128 + row] = l;
            }
        }
    }
    }
    if (b >= 0 && (MODE == kTurns || (MODE == kOne && t.n_split > 1))) {
        if (t.n_split > 1) cluster_sync(); else __syncthreads();
        join_parts<bf16, STEP>(a, s, i0, t.RC, t.TQ, heads, h0, t.n_split, split, base, smem_u32(m_sm), smem_u32(l_sm), w_sm, redo_sm, NT);
        if (t.n_split > 1) cluster_sync();
    }
    tc_fence_before();
    __syncthreads();
    unsigned redo = 0;
#pragma unroll
    for (int w = 0; w < 4 * NQ; w++) redo |= redo_sm[w];
    if (redo && !*abort_flag)
        for (int row = warp; row < NQ * 128; row += NT / 32)
            if (redo_sm[row >> 5] >> (row & 31) & 1) attn_row_by_key<bf16>(a, b, s, i0 + (row >> 7) * t.TQ + (row & 127) / t.RC, h0 + (row & 127) % t.RC);
    if (*abort_flag) {
        const unsigned long long t_0 = globaltimer_ns();
        while (globaltimer_ns() - t_0 < 200000ull) { __nanosleep(1000); }
        if (threadIdx.x == 0 && a.seq.error_flag) atomicOr(a.seq.error_flag, 1);
        __syncthreads();
    }
    if (warp == WM) { tc_fence_after(); tmem_dealloc(tmem, t.tmem_cols); }
}

template <int MODE> int launch_tc(TcArgs& t, long tiles, cudaStream_t st) {
    const PagedAttn& a = t.a;
    constexpr int NQ = MODE == kPair ? 2 : 1, W = MODE == kOne ? 1 : 2, NT = W * 128 + 64;
    // stages while they fit, of K and V in turn; kOne: two CTAs per SM where that is possible
    const bool two = MODE == kOne && KT + t.o_stride <= 256 && tc_smem(1, t.q_block, t.kc, t.vr, 1, 1).total <= kHalfSm;
    t.tmem_cols = two ? 256 : 512;
    t.ks = t.vs = 1;
    for (int i = 0; i < 2 * (kMaxStages - 1); i++) {
        int& n = i & 1 ? t.vs : t.ks;
        n++;
        if (tc_smem(NQ, t.q_block, t.kc, t.vr, t.ks, t.vs).total > (two ? kHalfSm : kWholeSm)) { n--; break; }
    }
    TcSmem o = tc_smem(NQ, t.q_block, t.kc, t.vr, t.ks, t.vs);
    // the parts of a tile go over the operands, not over the barriers
    const uint32_t parts = MODE == kTurns || t.n_split > 1 ? (uint32_t)(W * 128 * (a.dv + 4) * 4) : 0;
    if (o.total > kWholeSm || parts > o.bars) return FLEXLLM_ENOTSUP;
    CUtensorMap tq, tk, tv;
    TRY_RC(make_tmap_rows3_u8(&tq, a.q, (uint64_t)a.seq.T, (uint64_t)a.H, (uint64_t)a.dk * 2, (uint32_t)t.TQ, (uint32_t)t.RC, (uint64_t)a.ldq * 2));
    TRY_RC(make_tmap_2d_u8(&tk, a.k, (uint64_t)a.seq.n_pages * a.G * kPage, (uint64_t)a.dk * 2, kPage));
    TRY_RC(make_tmap_2d_u8(&tv, a.v, (uint64_t)a.seq.n_pages * a.G * a.dv, kPage * 2, (uint32_t)t.vr));
    auto kern = attn_paged_tc_kernel<MODE>;
    TRY_RC(allow_shared(kern, o.total));
    TRY_RC(allow_cluster(kern, t.n_split));
    launch_cluster(kern, dim3((unsigned)(tiles * t.n_split * t.heads)), dim3(NT), t.n_split, o.total, st, tq, tk, tv, t);
    return launch_status();
}

int most_clusters(int size) {
    auto kern = attn_paged_tc_kernel<kTurns>;
    const size_t smem = kWholeSm - 4096;
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = size; at[0].val.clusterDim.y = 1; at[0].val.clusterDim.z = 1;
    cfg.gridDim = dim3(size); cfg.blockDim = dim3(320); cfg.dynamicSmemBytes = smem; cfg.attrs = at; cfg.numAttrs = 1;
    int n = 0;
    if (allow_shared(kern, smem) || allow_cluster(kern, size) || cudaOccupancyMaxActiveClusters(&n, kern, &cfg) != cudaSuccess) {
        cudaGetLastError();                               // not known: keys are not cut
        return 0;
    }
    return n;
}

}  // namespace

int cluster_slots(int size, bool two) {
    struct Table {
        int n[17];
        Table() { for (int s = 1; s <= 16; s++) n[s] = most_clusters(s); }
    };
    static const Table table;
    return two ? (size == 1 ? 2 * table.n[1] : table.n[(size + 1) / 2]) : table.n[size];
}

int attn_paged_tc(const PagedAttn& a, cudaStream_t st) {
    TcArgs t = {};
    const int R = a.H / a.G;
    t.a = a;
    t.RC = R < 128 ? R : 128; t.HC = (R + t.RC - 1) / t.RC;
    t.kc = (a.dk + 63) / 64; t.vr = (a.dv + 15) / 16 * 16; t.o_stride = (t.vr + 31) / 32 * 32;
    t.a2 = score_factor(a);
    const long heads = (long)a.G * t.HC, seqs = a.seq.B < a.seq.T ? a.seq.B : a.seq.T, each = (a.seq.T + seqs - 1) / seqs;
    // short tiles where two of them would hold what sequences have on average: shared memory for Q becomes stages (one token over 84500, 8 key/value
    // heads: 105 us and 81)
    const int most = each * t.RC <= 16 ? 32 : 128;
    t.TQ = most / t.RC;
    t.q_block = most * 128u;
    const long pairs = most_units(a.seq, 2 * t.TQ), ones = most_units(a.seq, t.TQ);
    t.heads = (int)heads;
    // rows of the pages are counted in 31 bits
    if (ones * 16 * heads > 0x7fffffffL || (long)a.seq.n_pages * a.G * (a.dv > kPage ? a.dv : kPage) > 0x7fffffffL) return FLEXLLM_ENOTSUP;
    const long sms = gemm_sm_count(), tiles = (each + t.TQ - 1) / t.TQ * seqs * heads;      // if all sequences are of equal length
    const int pages = (a.seq.max_ctx + kPage) / kPage;
    t.n_split = 1;
    if (a.dk <= 128 && a.dv <= 128) {
        if (tiles <= sms) {
            // What the call takes in microseconds, cut into s parts, by one CTA of kTurns or two of kOne per SM: a time per key tile, one for the call, and
            // one per part for joining rows (a tree of 26 over 1000, kTurns and kOne: 17.6 and 15.2; 16 of 25 over 8000: 103 and 89; 9 of 10
            // over 4000: 34 and 44; one token over 84500, one head: 62 and 157; where several sequences are named, their lengths are 0.4 to 1 of the figure)
            const float rows = (float)((each < t.TQ ? each : t.TQ) * t.RC) / 128;
            const int n = (pages + 1) / 2;
            float best = 3e38f;
            bool turns = true;
            for (int s = 1; s <= 16 && s <= n; s++) {
                const float part = (float)((n + s - 1) / s);
                const int alone = cluster_slots(s, false);
                const float two_sets = 1.1f * part + 11.0f + 1.6f * s * rows;
                const float one_set = (alone >= tiles ? 1.85f * part + 8.0f : 2.1f * part + 9.0f) + (s > 1 ? 2.5f + 0.8f * s * rows : 0.0f);
                if (two_sets < best && alone >= tiles) { best = two_sets; turns = true; t.n_split = s; }
                if (one_set < best && cluster_slots(s, true) >= tiles) { best = one_set; turns = false; t.n_split = s; }
            }
            return turns ? launch_tc<kTurns>(t, ones, st) : launch_tc<kOne>(t, ones, st);
        }
        // pairs where sequences fill them and every SM has one
        if ((long)a.seq.T >= 2L * t.TQ * seqs && tiles >= 2 * sms) return launch_tc<kPair>(t, pairs, st);
        // long ones are cut although each has its place: sequences differ (20 trees of 20 over 6000: 105 us against 112, 32 of 28 over 8000: 199 against
        // 228, 32 single tokens over 8000: 154 against 152, over 2000: 56 against 48)
        if (tiles <= 4 * sms && pages >= 80) t.n_split = 2;
        return launch_tc<kOne>(t, ones, st);
    }
    t.n_split = key_splits(tiles, false, pages, KT / kPage, 16);
    return launch_tc<kOne>(t, ones, st);
}

}  // namespace flexllm
