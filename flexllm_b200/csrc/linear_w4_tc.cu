// Products with 4-bit weights on the tensor cores (tcgen05), for more than a few tokens:
//   y[m][n] = sum_groups s[n][g] * sum_{k in g} a[m][k] (q[n][k] - z[n][g])
// Weights are on the 128-row side, up to 64 tokens on the other (32 in fp32: three bf16 parts, which hold a number to the last bit, and three products into
// the same sums). A CTA walks K in steps of 128:
//   warp 12        brings words (eight steps ahead, six in fp32) and bf16 activations by TMA
//   warps 4 .. 11  put q - z, exact in bf16, into swizzled shared memory, four of them a step, the others the next (48 tokens, 16384 x 2048: all eight a
//                  step 13.2 us, by fours 11.7; three teams of four leave too few registers for the sums: 12.9). They load nothing from memory
//                  themselves: their fence towards the tensor core would wait for it (words in registers, asked for four steps ahead: 18.8 us)
//   warp 13        issues the MMAs, accumulators of their own for each group of a step, two steps' worth
//   warps 0 .. 3   take a step's sums out of TMEM and add them up in fp32 registers, times the groups' scales: no weight is ever rounded;
//                  they also hand the zero points to the converting warps, six steps ahead, and cut fp32 activations into their parts
// Few rows: the CTAs of a cluster cut K, and their sums meet in shared memory, in a fixed order.
// Bound by the chain of a step: words from shared memory, unpacked and put back (about 600 clocks), their fence, eight MMAs. 48 tokens, 16384 x 2048: 12.1 us;
// 64 tokens, 8192 x 8192: 22.4 us, 383 TFLOP/s, 1.5 TB/s; 64 tokens, 128256 x 2048: 88 us; fp32, 64 tokens, 8192 x 2048: 23 us (warp MMAs, 68).
#include "linear_w4.h"
#include "tc_common.cuh"

namespace flexllm {

using namespace tc;

namespace {

constexpr int kStepK = 128, kStages = 3, kTeams = 2, kTmaWarp = 4 + 4 * kTeams, kMmaWarp = kTmaWarp + 1, kTcThreads = (kMmaWarp + 1) * 32;
constexpr int kZeros = 8, kZerosAhead = 6;      // zero points: slots, steps ahead of the sums

struct W4Tc {
    W4Call c;
    int steps, n_split;
    int* error_flag;
    int per_group; uint32_t magic;         // blocks of a group, and 2^32 / per_group rounded up: the quotient of block numbers below 2^16
};
// shared memory: A [stage][2][128 rows][128 bytes], activations [stage][P][2][NT][128 bytes], words [words][128 rows][64 bytes], zero points [kZeros][4][128]
template <int NT, int P> struct W4Smem {
    static constexpr int words = P == 3 ? 6 : 8;
    static constexpr uint32_t x = kStages * 32768u, x_part = NT * 256u, x_stage = P * x_part, w = x + kStages * x_stage, z = w + words * 8192u, bars = z + kZeros * 512u,
                              total = bars + 512u + 1024u;
};

// U groups (or parts of one) per step; P = 3: fp32 activations
template <int NT, int U, int P>
__global__ void __launch_bounds__(kTcThreads, 1) linear_w4_tc_kernel(const __grid_constant__ CUtensorMap tmapX, const __grid_constant__ CUtensorMap tmapW,
                                                                     const __grid_constant__ W4Tc t) {
    constexpr int BK = kStepK / U;                         // elements of a block
    using S = W4Smem<NT, P>;
    constexpr int kWords = S::words, kTokens = P == 3 ? 32 : 64;
    extern __shared__ uint8_t smem_raw[];
    const W4Call& c = t.c;
    const uint32_t raw = smem_u32(smem_raw), base = (raw + 1023u) & ~1023u;
    uint8_t* base_ptr = smem_raw + (base - raw);
    uint64_t* bars = reinterpret_cast<uint64_t*>(base_ptr + S::bars);
    // operands there (conversion and activations) and read; sums there and read; words there; zero points there
    const uint32_t bar_a = smem_u32(bars), bar_e = bar_a + 8 * kStages, bar_d = bar_e + 8 * kStages, bar_de = bar_d + 16, bar_w = bar_de + 16,
                   bar_z = bar_w + 8 * kWords;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 32);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    constexpr uint32_t need = 2 * U * NT, cols = need <= 32 ? 32 : need <= 64 ? 64 : need <= 128 ? 128 : need <= 256 ? 256 : 512;
    if (threadIdx.x == 0) {
        for (int i = 0; i < kStages; i++) { mbar_init(bar_a + 8 * i, P == 3 ? 8 : 5); mbar_init(bar_e + 8 * i, 1); }
        for (int i = 0; i < 2; i++) { mbar_init(bar_d + 8 * i, 1); mbar_init(bar_de + 8 * i, 4); }
        for (int i = 0; i < kWords; i++) mbar_init(bar_w + 8 * i, 1);
        for (int i = 0; i < kZeros; i++) mbar_init(bar_z + 8 * i, 4);
        *abort_flag = 0;
        fence_barrier_init();
    }
    if (warp == kMmaWarp) { tmem_alloc(smem_u32(tmem_slot), cols); tmem_relinquish(); }
    if (warp == kTmaWarp && lane == 0) { if (P == 1) tma_prefetch_desc(&tmapX); tma_prefetch_desc(&tmapW); }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    pdl_sync();                                           // behind the allocation: no later kernel may hold the TMEM that this one waits for
    const int split = blockIdx.x % t.n_split, n0 = blockIdx.x / t.n_split * 128, m0 = blockIdx.y * kTokens;
    const int s0 = (int)((long)t.steps * split / t.n_split), s1 = (int)((long)t.steps * (split + 1) / t.n_split);
    // all lanes look: one that looks for the others and tells them takes twice as long
    auto wait_warp = [&](uint32_t bar, uint32_t parity) { return __all_sync(0xffffffffu, mbar_spin(bar, parity, abort_flag)) != 0; };
    float acc[NT];
#pragma unroll
    for (int x = 0; x < NT; x++) acc[x] = 0.0f;
    if (warp == kTmaWarp) {
        if (lane == 0) {
            // the words of step n lie where those of step n - kWords were, which the conversion has read when the products of that step are done
            auto words = [&](int n) {
                if (s0 + n >= s1) return;
                mbar_expect_tx(bar_w + 8 * (n % kWords), 8192u);
                tma_load_2d(base + S::w + (uint32_t)(n % kWords) * 8192u, &tmapW, bar_w + 8 * (n % kWords), (s0 + n) * (kStepK / 2), n0);
            };
            for (int n = 0; n < kWords; n++) words(n);
            for (int n = 0; s0 + n < s1; n++) {
                const int st = n % kStages;
                if (!mbar_spin(bar_e + 8 * st, (uint32_t)(n / kStages & 1) ^ 1u, abort_flag)) break;
                if (P == 1) {
                    mbar_expect_tx(bar_a + 8 * st, NT * 256u);
                    for (int b = 0; b < 2; b++)
                        tma_load_2d(base + S::x + (uint32_t)(st * 2 + b) * (NT * 128u), &tmapX, bar_a + 8 * st, ((s0 + n) * kStepK + b * 64) * 2, m0);
                }
                if (n >= kStages) words(n - kStages + kWords);
            }
        }
    } else if (warp == kMmaWarp) {
        const uint32_t leader = elect_leader(), u_tmem = (uint32_t)uniform_max((int)tmem);
        const uint32_t idesc = umma_idesc_bf16(128, NT), a_lo = umma_desc_lo(base), x_lo = umma_desc_lo(base + S::x);
        for (int n = 0; s0 + n < s1; n++) {
            const int st = n % kStages, buf = n & 1;
            if (!wait_warp(bar_de + 8 * buf, (uint32_t)(n >> 1 & 1) ^ 1u)) break;
            if (!wait_warp(bar_a + 8 * st, (uint32_t)(n / kStages & 1))) break;
            tc_fence_after();
#pragma unroll
            for (int p = P - 1; p >= 0; p--)               // the small parts first
#pragma unroll
                for (int k = 0; k < 8; k++)
                    umma_bf16_lo(leader, u_tmem + (buf * U + k / (8 / U)) * NT, a_lo + st * 2048 + (k >> 2) * 1024 + 2 * (k & 3),
                                 x_lo + (st * P + p) * (NT * 16) + (k >> 2) * (NT * 8) + 2 * (k & 3), idesc, p < P - 1 || k % (8 / U) > 0);
            umma_commit_by(leader, bar_d + 8 * buf);
            umma_commit_by(leader, bar_e + 8 * st);
        }
    } else if (warp >= 4) {
        // a row per lane: eight lanes in a row meet eight different 16-byte columns, in the words as in the operand
        const int r = (warp & 3) * 32 + lane;
        for (int n = (warp - 4) >> 2; s0 + n < s1; n += kTeams) {
            const int st = n % kStages, sw = n % kWords;
            uint8_t* to = base_ptr + st * 32768 + r * 128;
            if (!wait_warp(bar_w + 8 * sw, (uint32_t)(n / kWords & 1))) break;
            uint4 v[4];
#pragma unroll
            for (int x = 0; x < 4; x++) v[x] = *reinterpret_cast<const uint4*>(base_ptr + S::w + sw * 8192 + r * 64 + ((x ^ (r >> 1 & 3)) << 4));
            if (!wait_warp(bar_e + 8 * st, (uint32_t)(n / kStages & 1) ^ 1u)) break;
            uint32_t z2[U];
#pragma unroll
            for (int u = 0; u < U; u++) z2[u] = zero2(8u);
            if (c.zero) {
                if (!wait_warp(bar_z + 8 * (n % kZeros), (uint32_t)(n / kZeros & 1))) break;
#pragma unroll
                for (int u = 0; u < U; u++) z2[u] = zero2(base_ptr[S::z + n % kZeros * 512 + u * 128 + r]);
            }
#pragma unroll
            for (int x = 0; x < 4; x++) {
                const uint32_t z = z2[x * U / 4];
                const uint32_t word[4] = {v[x].x, v[x].y, v[x].z, v[x].w};
#pragma unroll
                for (int y = 0; y < 4; y++) {
                    const uint32_t p0 = weights2(word[y], 0, z), p1 = weights2(word[y], 1, z), p2 = weights2(word[y], 2, z), p3 = weights2(word[y], 3, z);
                    *reinterpret_cast<uint4*>(to + (x >> 1) * 16384 + ((((x & 1) * 4 + y) ^ (r & 7)) << 4)) =
                        make_uint4(pick(p0, p1, 0x5410), pick(p2, p3, 0x5410), pick(p0, p1, 0x7632), pick(p2, p3, 0x7632));
                }
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar_a + 8 * st);
        }
    } else {
        const int groups = c.K / c.group, rr = warp * 32 + lane;
        const long g0 = (long)min(n0 + rr, c.N - 1) * groups;
        const uint32_t lane_addr = (uint32_t)(warp * 32) << 16;
        auto group_at = [&](int i, int u) {               // behind K: the last one, for zeros
            const int kb = min(i * U + u, c.K / BK - 1);
            return g0 + (t.per_group == 1 ? kb : (int)__umulhi(kb, t.magic));
        };
        uint32_t next[U];
        auto fetch = [&](int i) {
#pragma unroll
            for (int u = 0; u < U; u++) next[u] = c.scale_f32 ? ((const uint32_t*)c.scale)[group_at(i, u)] : (uint32_t)((const uint16_t*)c.scale)[group_at(i, u)];
        };
        // zero points of step n into a slot that the conversion of step n - kZeros has left: its products are among the sums
        struct Zeros { uint32_t v[U]; } zero;
        auto fetch_zero = [&](int n) {
            Zeros z;
#pragma unroll
            for (int u = 0; u < U; u++) z.v[u] = c.zero[group_at(s0 + n, u)];
            return z;
        };
        auto hand_zero = [&](int n, const Zeros& z) {
            uint32_t seen = 0;
#pragma unroll
            for (int u = 0; u < U; u++) { base_ptr[S::z + n % kZeros * 512 + u * 128 + rr] = (uint8_t)z.v[u]; seen |= z.v[u]; }
            check_zeros(seen, c.error_flag);
            __syncwarp();
            if (lane == 0) mbar_arrive(bar_z + 8 * (n % kZeros));
        };
        // fp32 activations of a step: loaded a step before they are cut, since the fence behind the cut waits for what is on its way
        constexpr int E = P == 3 ? NT / 8 : 1;             // of 8 numbers, per thread
        float xs[E][8];
        auto load_x = [&](int n) {
#pragma unroll
            for (int i = 0; i < E; i++) {
                const int e = threadIdx.x + 128 * i, m = m0 + (e >> 4), k = (s0 + n) * kStepK + (e & 15) * 8;
                if (m < c.M && k < c.K) load8((const float*)c.a + (long)m * c.lda + k, xs[i]);
                else
#pragma unroll
                    for (int y = 0; y < 8; y++) xs[i][y] = 0.0f;
            }
        };
        auto cut_x = [&](int n) {
            const int st = n % kStages;
            if (!wait_warp(bar_e + 8 * st, (uint32_t)(n / kStages & 1) ^ 1u)) return false;
#pragma unroll
            for (int i = 0; i < E; i++) {
                const int e = threadIdx.x + 128 * i, row = e >> 4, col = e & 15;
                float f[8] = {xs[i][0], xs[i][2], xs[i][4], xs[i][6], xs[i][1], xs[i][3], xs[i][5], xs[i][7]};
                const Eight parts = eight(f);
#pragma unroll
                for (int p = 0; p < 3; p++)
                    *reinterpret_cast<uint4*>(base_ptr + S::x + st * S::x_stage + p * S::x_part + (col >> 3) * (NT * 128) + row * 128 + (((col ^ row) & 7) << 4)) = parts.part[p];
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar_a + 8 * st);
            return true;
        };
        bool ok = s0 < s1;
        if (ok) fetch(s0);
        if (P == 3 && ok) {
            load_x(0);
            for (int n = 0; ok && n < 2 && s0 + n < s1; n++) { ok = cut_x(n); load_x(n + 1); }
        }
        if (ok && c.zero) {
            Zeros first[kZerosAhead];
#pragma unroll
            for (int n = 0; n < kZerosAhead; n++) first[n] = fetch_zero(n);
#pragma unroll
            for (int n = 0; n < kZerosAhead; n++) if (s0 + n < s1) hand_zero(n, first[n]);
            zero = fetch_zero(kZerosAhead);
        }
        for (int n = 0; ok && s0 + n < s1; n++) {
            float sc[U];
#pragma unroll
            for (int u = 0; u < U; u++) sc[u] = __uint_as_float(c.scale_f32 ? next[u] : next[u] << 16);
            fetch(s0 + n + 1);
            ok = wait_warp(bar_d + 8 * (n & 1), (uint32_t)(n >> 1 & 1));
            if (!ok) break;
            tc_fence_after();
#pragma unroll
            for (int x0 = 0; x0 < U * NT; x0 += 16) {
                uint32_t v[16];
                tmem_ld_32x16(tmem + (n & 1) * (U * NT) + x0 + lane_addr, v);
                tmem_ld_wait();
#pragma unroll
                for (int x = 0; x < 16; x++) acc[x0 % NT + x] = __fmaf_rn(__uint_as_float(v[x]), sc[x0 / NT], acc[x0 % NT + x]);
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar_de + 8 * (n & 1));
            if (P == 3 && s0 + n + 2 < s1) {
                ok = cut_x(n + 2);
                load_x(n + 3);
            }
            if (c.zero && s0 + n + kZerosAhead < s1) {
                hand_zero(n + kZerosAhead, zero);
                zero = fetch_zero(n + kZerosAhead + 1);
            }
        }
    }
    // the sums into shared memory (every product has been waited for), [token][132]; the CTAs of the cluster join the tokens in turn
    float* red = reinterpret_cast<float*>(base_ptr);
    __syncthreads();
    if (warp < 4)
#pragma unroll
        for (int x = 0; x < NT; x++) red[x * 132 + warp * 32 + lane] = acc[x];
    if (t.n_split > 1) cluster_sync(); else __syncthreads();
    const int Mb = min(c.M - m0, NT), rows = min(128, c.N - n0);
    for (int e = threadIdx.x; e < (Mb - split + t.n_split - 1) / t.n_split * 32; e += kTcThreads) {
        const int m = split + (e >> 5) * t.n_split, r = (e & 31) * 4;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        if (t.n_split == 1) v = *reinterpret_cast<const float4*>(red + m * 132 + r);
        else
            for (int p = 0; p < t.n_split; p++) {
                const float4 x = ld_cluster_f32x4(cluster_addr(base + (uint32_t)(m * 132 + r) * 4u, p));
                v.x += x.x; v.y += x.y; v.z += x.z; v.w += x.w;
            }
        const long at = (long)(m0 + m) * c.ldy + n0 + r;
        const float f[4] = {v.x, v.y, v.z, v.w};
        float o[4];
#pragma unroll
        for (int x = 0; x < 4; x++) o[x] = f[x] + (c.bias && r + x < rows ? c.bias[n0 + r + x] : 0.0f);
        const bool whole = r + 4 <= rows && (c.ldy & 3) == 0;
        if (c.y_f32) {
            float* y = (float*)c.y + at;
            if (whole && ((uintptr_t)c.y & 15) == 0) store4(y, make_float4(o[0], o[1], o[2], o[3]));
            else
                for (int x = 0; x < 4; x++) if (r + x < rows) y[x] = o[x];
        } else {
            bf16* y = (bf16*)c.y + at;
            if (whole && ((uintptr_t)c.y & 7) == 0) store4(y, make_float4(o[0], o[1], o[2], o[3]));
            else
                for (int x = 0; x < 4; x++) if (r + x < rows) y[x] = __float2bfloat16_rn(o[x]);
        }
    }
    if (t.n_split > 1) cluster_sync();
    tc_fence_before();
    __syncthreads();
    if (*abort_flag) {
        const unsigned long long t_0 = globaltimer_ns();
        while (globaltimer_ns() - t_0 < 200000ull) { __nanosleep(1000); }
        if (threadIdx.x == 0 && t.error_flag) atomicOr(t.error_flag, 1);
        __syncthreads();
    }
    if (warp == kMmaWarp) { tc_fence_after(); tmem_dealloc(tmem, cols); }
}

template <int NT, int U, int P> int launch_tc(W4Tc& t, cudaStream_t st) {
    const W4Call& c = t.c;
    t.steps = (c.K + kStepK - 1) / kStepK;
    t.per_group = c.group / (kStepK / U);
    t.magic = (uint32_t)(((1ull << 32) + t.per_group - 1) / t.per_group);
    const long tiles = (c.N + 127) / 128, blocks = (c.M + (P == 3 ? 31 : 63)) / (P == 3 ? 32 : 64);
    t.n_split = 1;
    for (int k = 2; k <= 16 && t.steps >= k * (k > 8 ? 4 : 2); k++)
        if (cluster_slots(k, false) >= tiles * blocks) t.n_split = k;
    CUtensorMap tx = {}, tw;
    if (P == 1) TRY_RC(make_tmap_2d_u8_ld(&tx, c.a, (uint64_t)c.M, (uint64_t)c.K * 2, NT, (uint64_t)c.lda * 2));
    TRY_RC(make_tmap_2d_u8_box(&tw, c.w, (uint64_t)c.N, (uint64_t)c.K / 2, 64, 128, 64));
    auto kern = linear_w4_tc_kernel<NT, U, P>;
    constexpr uint32_t smem = W4Smem<NT, P>::total;
    TRY_RC(allow_shared(kern, smem));
    TRY_RC(allow_cluster(kern, t.n_split));
    launch_cluster(kern, dim3((unsigned)(tiles * t.n_split), (unsigned)blocks), dim3(kTcThreads), t.n_split, smem, st, tx, tw, t);
    return launch_status();
}
template <int NT, int P> int pick_tc(W4Tc& t, cudaStream_t st) {
    if (t.c.group % 128 == 0) return launch_tc<NT, 1, P>(t, st);
    if (t.c.group % 64 == 0) return launch_tc<NT, 2, P>(t, st);
    return launch_tc<NT, 4, P>(t, st);
}

}  // namespace

int linear_w4_tc(const W4Call& c, bool f32, cudaStream_t st) {
    W4Tc t = {};
    t.c = c; t.c.y_f32 = c.y_f32 || f32; t.error_flag = device_error_flag();
    if (f32) return c.M <= 16 ? pick_tc<16, 3>(t, st) : pick_tc<32, 3>(t, st);
    if (c.M <= 16) return pick_tc<16, 1>(t, st);
    if (c.M <= 32) return pick_tc<32, 1>(t, st);
    if (c.M <= 48) return pick_tc<48, 1>(t, st);
    return pick_tc<64, 1>(t, st);
}

}  // namespace flexllm
