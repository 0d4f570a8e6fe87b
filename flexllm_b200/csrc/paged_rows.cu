// Rows of packed sequences on their way into the floating-point paged cache, and within it:
//   qk_norm_rope  norm of every q and k head, rotation, q to a dense tensor, k and v to the pages
//   kv_keep       the entries of an accepted path moved together
#include "paged.cuh"

namespace flexllm {

namespace {

// Norm and rotation.  y = x / sqrt(mean x^2 + eps) * gain;  pair p < rot/2 turns elements p and p + rot/2 by the angle whose cosine and sine
// the tables hold at [pos[axis of p]][p]; elements from rot on stay. All in fp32, rounded once.
// HBM bound: every row is read and written once, the tables' rows come from L2. A group of L lanes holds a head: lane c the pairs
// 4 c .. 4 c + 3 (two vectors of four elements, so that both halves of a pair meet in one thread), the lanes behind them eight of the unrotated
// elements each. A warp stays with one token, whose sequence, positions and table entries it looks up once for eight heads. In bf16 the
// instructions count as much as the bytes: pairs of fp32 throughout. 16384 tokens, 16 / 8 heads of 128, three axes: 67 us, 4.0 TB/s, issue slots 60 % full; 32 tokens,
// 32 / 8 heads: 4.3 us, a launch and four dependent loads.
struct RopeArgs {
    PackedSeqs seq;
    int H, G, dk, dv, rot;
    const void* proj; long ldp;
    const float *q_gain, *k_gain;
    float eps;
    const int32_t* pos; int axes, sec_end[4];      // pairs below sec_end[a] (and not below sec_end[a - 1]) turn by axis a's position
    const float *cos_t, *sin_t; int table_len;
    void *k, *v;
    void* q; long ldq;
    int chunks, qk_ctas;                           // warps of a token, CTAs of such warps
    bool fours;                                    // the pairs of a lane are of one axis, the tables' rows 16-byte aligned
};
constexpr int kRopeHeads = 8;                      // heads of a warp

// four elements as two pairs
struct Four { f32x2 a, b; };
__device__ __forceinline__ Four load_four(const float* p) { const float4 v = load4(p); return {pack2(v.x, v.y), pack2(v.z, v.w)}; }
// four elements as they are in memory
template <class T> struct Raw;
template <> struct Raw<bf16> {
    static constexpr int kRounds = 4;              // of heads under way together
    uint2 v;
    __device__ __forceinline__ void load(const bf16* p) { v = *reinterpret_cast<const uint2*>(p); }
    __device__ __forceinline__ Four four() const { return {pack2(bf_lo(v.x), bf_hi(v.x)), pack2(bf_lo(v.y), bf_hi(v.y))}; }
};
template <> struct Raw<float> {
    static constexpr int kRounds = 2;
    float4 v;
    __device__ __forceinline__ void load(const float* p) { v = load4(p); }
    __device__ __forceinline__ Four four() const { return {pack2(v.x, v.y), pack2(v.z, v.w)}; }
};
template <class T> __device__ __forceinline__ void store_four(T* p, const Four& v) {
    float4 f;
    unpack2(v.a, f.x, f.y); unpack2(v.b, f.z, f.w);
    store4(p, f);
}
__device__ __forceinline__ Four times(const Four& x, const Four& y) { return {mul2(x.a, y.a), mul2(x.b, y.b)}; }
__device__ __forceinline__ Four times_plus(const Four& x, const Four& y, const Four& z) { return {fma2(x.a, y.a, z.a), fma2(x.b, y.b, z.b)}; }
__device__ __forceinline__ Four all_four(float v) { return {pack2(v, v), pack2(v, v)}; }

template <class T, int L> __device__ __forceinline__ void rope_warp(const RopeArgs& a, unsigned w) {
    constexpr int kRounds = Raw<T>::kRounds * (32 / L) <= kRopeHeads ? Raw<T>::kRounds : kRopeHeads * L / 32;
    const int lane = threadIdx.x & 31, c = lane % L, sub = lane / L;
    const int t = w / (unsigned)a.chunks, h0 = (w - t * a.chunks) * kRopeHeads, h1 = min(h0 + kRopeHeads, a.H + a.G);
    if (t >= a.seq.T) return;
    const int half = a.rot >> 1, nrot = half >> 2;
    const bool turns = c < nrot, rest = !turns && a.rot + (c - nrot) * 8 < a.dk, mine = turns || rest;
    const int e0 = turns ? 4 * c : a.rot + (c - nrot) * 8, e1 = turns ? e0 + half : e0 + 4;
    const T* src = (const T*)a.proj + (long)t * a.ldp;
    // a round: 32 / L heads
    Raw<T> x[kRounds], y[kRounds];
    auto load = [&](int h) {
#pragma unroll
        for (int j = 0; j < kRounds; j++) {
            const int hj = h + j * (32 / L) + sub;
            if (hj < h1 && mine) { x[j].load(src + hj * a.dk + e0); y[j].load(src + hj * a.dk + e1); }
        }
    };
    load(h0);
    // the sequence of the row: the last one that starts at or before it
    const int b = count_below(a.seq.B, [&](int i) { return a.seq.cu[i] <= t; }) - 1;
    Four co = all_four(1.0f), si = all_four(0.0f);         // the other elements do not turn
    bool outside = false;                                  // an error only if the row is a sequence's
    if (turns) {
        auto row_of = [&](int pair) {
            int axis = 0;
            while (axis < a.axes - 1 && pair >= a.sec_end[axis]) axis++;
            int row = a.pos[(long)axis * a.seq.T + t];
            if ((unsigned)row >= (unsigned)a.table_len) { outside = true; row = row < 0 ? 0 : a.table_len - 1; }
            return (long)row * half + pair;
        };
        if (a.fours) {
            const long at = row_of(e0);
            co = load_four(a.cos_t + at); si = load_four(a.sin_t + at);
        } else {
            float f[8];
#pragma unroll
            for (int p = 0; p < 4; p++) { const long at = row_of(e0 + p); f[p] = a.cos_t[at]; f[4 + p] = a.sin_t[at]; }
            co = {pack2(f[0], f[1]), pack2(f[2], f[3])}; si = {pack2(f[4], f[5]), pack2(f[6], f[7])};
        }
    }
    const Four minus_si = times(si, all_four(-1.0f));
    if (b < 0) return;
    const SeqRows s = seq_rows(a.seq, b);
    if (t < s.row0 || t >= s.row0 + s.n) return;
    if (outside) data_error(a.seq.error_flag);
    const int at = s.ctx + t - s.row0;
    const long page = h1 <= a.H ? 0 : s.sound ? page_or_none(a.seq, b, at / kPage) : -1;
    const float inv_dk = 1.0f / (float)a.dk;
    for (int h = h0; h < h1; h += kRounds * (32 / L)) {
        if (h > h0) load(h);
#pragma unroll
        for (int j = 0; j < kRounds; j++) {
            const int hj = h + j * (32 / L) + sub;
            const float* gain = hj < a.H ? a.q_gain : a.k_gain;
            Four u = all_four(0.0f), v = u;
            if (hj < h1 && mine) { u = x[j].four(); v = y[j].four(); }
            float s0, s1;
            unpack2(fma2(u.a, u.a, fma2(u.b, u.b, fma2(v.a, v.a, mul2(v.b, v.b)))), s0, s1);
            float ss = s0 + s1;
#pragma unroll
            for (int o = L / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
            if (hj >= h1 || !mine) continue;
            if (gain) {
                const Four r = all_four(rsqrtf(__fmaf_rn(ss, inv_dk, a.eps)));
                u = times(times(u, r), load_four(gain + e0));
                v = times(times(v, r), load_four(gain + e1));
            }
            T* dst = hj < a.H ? (T*)a.q + (long)t * a.ldq + (long)hj * a.dk
                              : (T*)a.k + ((page * a.G + (hj - a.H)) * kPage + (at & (kPage - 1))) * a.dk;
            const Four lo = times_plus(v, minus_si, times(u, co)), hi = times_plus(u, si, times(v, co));
            if (hj >= a.H && page < 0) continue;           // looked at here and no earlier: the page's id is on its way until now
            store_four(dst + e0, lo);
            store_four(dst + e1, hi);
        }
    }
}

// 16 bytes of consecutive slots of a V^T row
template <class T> struct Slots;
template <> struct Slots<bf16> { static constexpr int N = 8; };
template <> struct Slots<float> { static constexpr int N = 4; };

// CTAs below qk_ctas: eight warps of the above. Then one (page of a sequence, key/value head) each: the page's new value rows through shared
// memory into its columns, whole 16-byte pieces where the call fills them.
template <class T, int L> __global__ void __launch_bounds__(256, 4) qk_norm_rope_kernel(const __grid_constant__ RopeArgs a) {
    extern __shared__ __align__(16) uint8_t raw[];
    __shared__ Unit unit_sm;
    pdl_sync();
    if ((int)blockIdx.x < a.qk_ctas) {
        rope_warp<T, L>(a, blockIdx.x * 8u + (threadIdx.x >> 5));
        return;
    }
    const int id = blockIdx.x - a.qk_ctas, g = id % a.G, tid = threadIdx.x;
    if (tid < 32) {
        const Unit u = find_unit(a.seq, id / a.G, kPage, 2, [](const SeqRows& s) { return (s.ctx + s.n - 1) / kPage - s.ctx / kPage + 1; });
        if (tid == 0) unit_sm = u;
    }
    __syncthreads();
    if (unit_sm.b < 0 || !unit_sm.s.sound) return;
    const SeqRows s = unit_sm.s;
    const int pg = s.ctx / kPage + unit_sm.i;
    const int lo = max(s.ctx, pg * kPage) - pg * kPage, hi = min(s.ctx + s.n - pg * kPage, kPage);      // slots [lo, hi)
    constexpr int N = Slots<T>::N;
    const int pitch = a.dv + 4 / (int)sizeof(T);          // elements: consecutive rows one word apart
    T* tile = reinterpret_cast<T*>(raw);                  // [slot][pitch]
    const T* src = (const T*)a.proj + (long)(s.row0 + pg * kPage - s.ctx) * a.ldp + (long)(a.H + a.G) * a.dk + (long)g * a.dv;
    const int vec = a.dv / N;
    for (int e = tid; e < (hi - lo) * vec; e += 256) {
        const int t = lo + e / vec, d = (e % vec) * N;
        const uint4 w = *reinterpret_cast<const uint4*>(src + (long)t * a.ldp + d);
        uint32_t* dst = reinterpret_cast<uint32_t*>(tile + (long)t * pitch + d);
        dst[0] = w.x; dst[1] = w.y; dst[2] = w.z; dst[3] = w.w;
    }
    const long page = page_or_none(a.seq, unit_sm.b, pg);
    __syncthreads();
    if (page < 0) return;
    T* vp = (T*)a.v + (page * a.G + g) * (long)a.dv * kPage;
    constexpr int PIECES = kPage / N;
    for (int e = tid; e < a.dv * PIECES; e += 256) {
        const int d = e / PIECES, t0 = (e % PIECES) * N;
        if (t0 + N <= lo || t0 >= hi) continue;
        __align__(16) T x[N];
#pragma unroll
        for (int i = 0; i < N; i++) x[i] = t0 + i >= lo && t0 + i < hi ? tile[(long)(t0 + i) * pitch + d] : from_f<T>(0.0f);
        T* dst = vp + (long)d * kPage + t0;
        if (t0 >= lo && t0 + N <= hi) *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(x);
        else
#pragma unroll
            for (int i = 0; i < N; i++)
                if (t0 + i >= lo && t0 + i < hi) dst[i] = x[i];
    }
}

template <class T, int L> int launch_rope(RopeArgs& a, cudaStream_t st) {
    a.chunks = (a.H + a.G + kRopeHeads - 1) / kRopeHeads;
    const long qk = ((long)a.seq.T * a.chunks + 7) / 8;
    // a sequence's first row opens a page, the next one another, and so does every 64th
    const long seqs = a.seq.B < a.seq.T ? a.seq.B : a.seq.T, next = a.seq.T - seqs,
               units = a.seq.B > kLookThrough ? a.seq.T / kPage + 2L * a.seq.B : seqs + (next + (kPage - 1) * (next < seqs ? next : seqs)) / kPage;
    if (qk + units * a.G > 0x7fffffffL || qk > 0x1fffffffL) return FLEXLLM_ENOTSUP;      // warps are counted in 32 bits
    a.qk_ctas = (int)qk;
    const size_t smem = (size_t)kPage * (a.dv * sizeof(T) + 4);
    auto kern = qk_norm_rope_kernel<T, L>;
    TRY_RC(allow_shared(kern, smem));
    launch_k(kern, dim3((unsigned)(qk + units * a.G)), dim3(256), smem, st, a);
    return launch_status();
}
template <class T> int run_rope(RopeArgs& a, cudaStream_t st) {
    if (a.dk <= 64) return launch_rope<T, 8>(a, st);
    if (a.dk <= 128) return launch_rope<T, 16>(a, st);
    return launch_rope<T, 32>(a, st);
}

// new[ctx + i] = old[ctx + keep[i]], i < count: one CTA per (sequence, key/value head, several layers of like shape, where there are enough CTAs). All old
// entries are in shared memory before the first new one is written, so the indices may come in any order. Bound by latency (counts, indices, page
// table, entries, one after the other) and by the sectors of V^T: an element of two bytes is read and written with its 32.
struct KeepLayer { void *k, *v; int hkv, dk, dv, n_pages; };
constexpr int kKeepLayers = 64;
struct KeepArgs {
    PackedSeqs seq;                        // cu unused
    const int32_t *keep, *count;
    int most, layers, per;                 // per: layers of a CTA
    KeepLayer layer[kKeepLayers];
};

template <class T> __global__ void __launch_bounds__(256) kv_keep_kernel(const __grid_constant__ KeepArgs a) {
    extern __shared__ __align__(16) uint8_t raw[];
    __shared__ int src_page[64], src_slot[64], dst_page[64], dst_slot[64], n_moves;
    const int l0 = blockIdx.z * a.per, layers = min(a.per, a.layers - l0);
    const KeepLayer& y = a.layer[l0];      // the shape of all of them
    const int b = blockIdx.x, g = blockIdx.y, tid = threadIdx.x;
    pdl_sync();
    if (g >= y.hkv) return;
    if (tid == 0) n_moves = 0;
    __syncthreads();
    int count = a.count[b], ctx = a.seq.ctx[b];
    if (count < 0 || count > a.most) { if (tid == 0) data_error(a.seq.error_flag); count = min(max(count, 0), a.most); }
    if (tid < count) {
        PackedSeqs p = a.seq;
        p.n_pages = y.n_pages;
        const int from = a.keep[(long)b * a.most + tid];
        if (ctx < 0 || from < 0 || from >= 64 || max(from, tid) > a.seq.max_ctx - ctx) data_error(a.seq.error_flag);      // such an entry is not moved
        else if (from != tid) {
            const int s = ctx + from, d = ctx + tid;
            const int sp = page_or_none(p, b, s / kPage), dp = page_or_none(p, b, d / kPage);
            if (sp >= 0 && dp >= 0) {
                const int m = atomicAdd(&n_moves, 1);
                src_page[m] = sp; src_slot[m] = s & (kPage - 1);
                dst_page[m] = dp; dst_slot[m] = d & (kPage - 1);
            }
        }
    }
    __syncthreads();
    const int n = n_moves;
    if (n == 0) return;
    const int vec = y.dk * (int)sizeof(T) / 16, kn = n * vec, vn = n * y.dv;
    T* ks = reinterpret_cast<T*>(raw);                    // [layer][n][dk]
    T* vs = ks + (long)layers * n * y.dk;                 // [layer][dv][n]
    // quotients of numbers below 2^17 by numbers below 2^15 (1 apart), as they are needed for every element
    struct Quotient {
        uint32_t by, magic;
        __device__ Quotient(int d) : by(d), magic(d > 1 ? 0xffffffffu / (uint32_t)d + 1u : 0u) {}
        __device__ __forceinline__ uint32_t operator()(uint32_t x) const { return by > 1 ? __umulhi(x, magic) : x; }
    };
    const Quotient by_kn(kn), by_vec(vec), by_vn(vn), by_n(n);
    auto k_at = [&](uint32_t e, const int* page, const int* slot) {
        const uint32_t l = by_kn(e), r = e - l * kn, i = by_vec(r), c = r - i * vec;
        return reinterpret_cast<uint4*>((T*)a.layer[l0 + l].k + (((long)page[i] * y.hkv + g) * kPage + slot[i]) * y.dk) + c;
    };
    auto v_at = [&](uint32_t e, const int* page, const int* slot) {
        const uint32_t l = by_vn(e), r = e - l * vn, d = by_n(r), i = r - d * n;
        return (T*)a.layer[l0 + l].v + ((long)page[i] * y.hkv + g) * y.dv * kPage + (long)d * kPage + slot[i];
    };
    for (int e = tid; e < layers * kn; e += 256) reinterpret_cast<uint4*>(ks)[e] = *k_at(e, src_page, src_slot);
    for (int e0 = tid; e0 < layers * vn; e0 += 8 * 256) {      // eight loads under way
        T x[8];
#pragma unroll
        for (int j = 0; j < 8; j++) if (e0 + j * 256 < layers * vn) x[j] = *v_at(e0 + j * 256, src_page, src_slot);
#pragma unroll
        for (int j = 0; j < 8; j++) if (e0 + j * 256 < layers * vn) vs[e0 + j * 256] = x[j];
    }
    __syncthreads();
    for (int e = tid; e < layers * kn; e += 256) *k_at(e, dst_page, dst_slot) = reinterpret_cast<const uint4*>(ks)[e];
    for (int e = tid; e < layers * vn; e += 256) *v_at(e, dst_page, dst_slot) = vs[e];
}

template <class T> int run_keep(KeepArgs& a, int heads, int widest, bool alike, cudaStream_t st) {
    // several layers per CTA, up to 4, while every SM has its eight CTAs (48 sequences, 8 heads, 16 layers: 20.1 us with one, 16.2 with 4)
    const long all = (long)a.seq.B * heads * a.layers, room = 8L * gemm_sm_count();
    a.per = 1;
    while (alike && a.per < 4 && all >= 2 * a.per * room && 2 * a.per * a.most * widest * (int)sizeof(T) <= 24 * 1024) a.per *= 2;
    const size_t smem = (size_t)a.per * a.most * widest * sizeof(T);
    auto kern = kv_keep_kernel<T>;
    TRY_RC(allow_shared(kern, smem));
    launch_k(kern, dim3(a.seq.B, heads, (a.layers + a.per - 1) / a.per), dim3(256), smem, st, a);
    return launch_status();
}

bool pages_ok(const flexllm_kv_pages* kv) {
    return kv && kv->k && kv->v && aligned(kv->k, 16) && aligned(kv->v, 16) && kv->n_pages > 0 && kv->hkv > 0 && kv->kdim > 0 && kv->vdim > 0;
}
bool dims_ok(const flexllm_kv_pages* kv) { return kv->kdim % 8 == 0 && kv->vdim % 8 == 0 && kv->kdim <= 256 && kv->vdim <= 256; }

}  // namespace

}  // namespace flexllm

using namespace flexllm;

extern "C" int flexllm_qk_norm_rope(int dtype, const flexllm_kv_pages* kv, int heads, const void* proj, long ldp, const float* q_gain, const float* k_gain,
                                    float eps, const int32_t* pos, int axes, const int* sections_host, const float* cos_t, const float* sin_t, int rot,
                                    int table_len, const int32_t* cu, const int32_t* ctx, const int32_t* page_table, int max_pages, int max_ctx, int B,
                                    int T, void* q, long ldq, void* stream) {
    FLEXLLM_REQUIRE(dtype == FLEXLLM_F32 || dtype == FLEXLLM_BF16);
    FLEXLLM_REQUIRE(pages_ok(kv) && heads > 0 && heads <= 65535 && kv->hkv <= 65535 && eps >= 0.0f);
    RopeArgs a = {};
    a.seq = {cu, ctx, page_table, max_pages, max_ctx, B, T, kv->n_pages, 0x7fffffff, nullptr};
    a.H = heads; a.G = kv->hkv; a.dk = kv->kdim; a.dv = kv->vdim; a.rot = rot;
    const long per16 = dtype == FLEXLLM_BF16 ? 8 : 4;
    FLEXLLM_REQUIRE(packed_ok(a.seq) && ldp >= (long)(a.H + a.G) * a.dk + (long)a.G * a.dv && ldq >= (long)a.H * a.dk && ldp % per16 == 0 && ldq % per16 == 0);
    FLEXLLM_REQUIRE(rot >= 0 && rot <= a.dk && axes >= 1 && axes <= 4 && (axes == 1 || sections_host) && (rot == 0 || (cos_t && sin_t && aligned(cos_t, 4) && aligned(sin_t, 4) && table_len > 0)));
    if (!dims_ok(kv) || rot % 8) return FLEXLLM_ENOTSUP;
    int end = 0;
    for (int i = 0; i < axes; i++) {
        const int n = sections_host ? sections_host[i] : rot / 2;
        FLEXLLM_REQUIRE(n >= 0 && n <= rot / 2 - end);
        end += n;
        a.sec_end[i] = end;
    }
    FLEXLLM_REQUIRE(end == rot / 2);
    if (T == 0) return FLEXLLM_OK;
    FLEXLLM_REQUIRE(proj && q && (rot == 0 || pos) && aligned(pos, 4) && aligned(proj, 16) && aligned(q, 16) && aligned(q_gain, 16) && aligned(k_gain, 16));
    a.fours = aligned(cos_t, 16) && aligned(sin_t, 16);
    for (int i = 0; i < axes; i++) a.fours = a.fours && a.sec_end[i] % 4 == 0;
    a.proj = proj; a.ldp = ldp; a.q_gain = q_gain; a.k_gain = k_gain; a.eps = eps; a.pos = pos; a.axes = axes;
    a.cos_t = cos_t; a.sin_t = sin_t; a.table_len = table_len; a.k = kv->k; a.v = kv->v; a.q = q; a.ldq = ldq;
    a.seq.error_flag = device_error_flag();
    const SetUpEarly early;
    return dtype == FLEXLLM_BF16 ? run_rope<bf16>(a, (cudaStream_t)stream) : run_rope<float>(a, (cudaStream_t)stream);
}

extern "C" int flexllm_kv_keep(int dtype, const flexllm_kv_pages* layers_host, int layers, const int32_t* page_table, int max_pages, const int32_t* ctx,
                               int max_ctx, const int32_t* keep, const int32_t* count, int most, int B, void* stream) {
    FLEXLLM_REQUIRE(dtype == FLEXLLM_F32 || dtype == FLEXLLM_BF16);
    PackedSeqs seq = {nullptr, ctx, page_table, max_pages, max_ctx, B, 0, 0, 0, nullptr};
    FLEXLLM_REQUIRE(layers_host && layers > 0 && most >= 0 && B > 0 && table_ok(seq));
    if (most > 64) return FLEXLLM_ENOTSUP;
    for (int i = 0; i < layers; i++) {
        FLEXLLM_REQUIRE(pages_ok(layers_host + i));
        if (!dims_ok(layers_host + i) || layers_host[i].hkv > 65535) return FLEXLLM_ENOTSUP;
    }
    if (most == 0) return FLEXLLM_OK;
    FLEXLLM_REQUIRE(keep && count && aligned(keep, 4) && aligned(count, 4));
    seq.error_flag = device_error_flag();
    const SetUpEarly early;
    for (int l0 = 0; l0 < layers; l0 += kKeepLayers) {
        const int n = layers - l0 < kKeepLayers ? layers - l0 : kKeepLayers;
        KeepArgs a = {};
        a.seq = seq;
        a.keep = keep; a.count = count; a.most = most; a.layers = n;
        int heads = 0, widest = 0;
        bool alike = true;
        for (int i = 0; i < n; i++) {
            const flexllm_kv_pages& p = layers_host[l0 + i];
            const flexllm_kv_pages& o = layers_host[l0];
            a.layer[i] = {p.k, p.v, p.hkv, p.kdim, p.vdim, p.n_pages};
            alike = alike && p.hkv == o.hkv && p.kdim == o.kdim && p.vdim == o.vdim && p.n_pages == o.n_pages;
            heads = p.hkv > heads ? p.hkv : heads;
            widest = p.kdim + p.vdim > widest ? p.kdim + p.vdim : widest;
        }
        TRY_RC(dtype == FLEXLLM_BF16 ? run_keep<bf16>(a, heads, widest, alike, (cudaStream_t)stream) : run_keep<float>(a, heads, widest, alike, (cudaStream_t)stream));
    }
    return FLEXLLM_OK;
}
