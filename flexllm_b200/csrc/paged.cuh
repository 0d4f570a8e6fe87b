// What the operators over packed sequences and the floating-point paged cache share: sequence b of a call has the packed rows
// cu[b] .. cu[b+1] - 1, at cache positions ctx[b] .., in pages of 64 tokens, K [page][G][64][dk], V transposed [page][G][dv][64].
// cu, ctx and the page table are device memory that the host never sees: values out of range are clamped (a page id: reads take page 0; entries that no
// position needs are not looked at) and reported through the device's error word, so that no access leaves its buffer. What a sequence with such
// values, or a page that the table does not name, would receive is left out.
#pragma once
#include "float_common.cuh"

namespace flexllm {

constexpr int kPage = 64;

struct PackedSeqs {
    const int32_t *cu, *ctx, *page_table;
    int max_pages, max_ctx, B, T, n_pages;
    int max_new;                           // most rows of one sequence
    int* error_flag;
};
struct SeqRows { int row0, n, ctx; bool sound; };      // first packed row, rows, tokens already in the cache; as the call says, not clamped

__device__ __forceinline__ void data_error(int* flag) { if (flag) atomicOr(flag, 2); }

__device__ __forceinline__ SeqRows seq_rows(const PackedSeqs& p, int b) {
    const int c0 = p.cu[b], c1 = p.cu[b + 1], x0 = p.ctx[b];
    SeqRows s;
    s.row0 = min(max(c0, 0), p.T);
    s.n = min(max(c1, s.row0), p.T) - s.row0;
    s.n = min(min(s.n, p.max_new), p.max_ctx + 1);
    s.ctx = min(max(x0, 0), p.max_ctx + 1 - s.n);
    s.sound = s.row0 == c0 && s.n == c1 - c0 && (s.n == 0 || s.ctx == x0);
    if (!s.sound) data_error(p.error_flag);
    return s;
}
// Page i of sequence b, or -1. Nothing is written for a page that the table does not name: page 0 may be another sequence's.
__device__ __forceinline__ int page_or_none(const PackedSeqs& p, int b, int i) {
    const int page = p.page_table[(long)b * p.max_pages + i];
    if ((unsigned)page < (unsigned)p.n_pages) return page;
    data_error(p.error_flag);
    return -1;
}
// The same for reads: page 0 in its place.
__device__ __forceinline__ int page_of(const PackedSeqs& p, int b, int i) { return max(page_or_none(p, b, i), 0); }

// How many of `n` are below a border, where below(i) holds up to it; 32 looks at a time. One whole warp.
template <class Below> __device__ __forceinline__ int count_below(int n, Below below) {
    const int lane = threadIdx.x & 31;
    int lo = 0, hi = n;
    while (lo < hi) {
        const int step = (hi - lo + 31) / 32, at = lo + step * (lane + 1) - 1;
        const int c = __popc(__ballot_sync(0xffffffffu, at < hi && below(at)));
        lo += step * c;
        hi = min(hi, lo + step - 1);
    }
    return lo;
}

// Unit `u` of a call whose sequences have count(rows) units each, at most rows / per + extra, counted from the last unit of the last sequence (in causal
// attention the longest first). One whole warp; b < 0: no such unit. Up to 64 sequences are looked through, units one after the other and those
// that do not exist at the end; more are searched, with units numbered cu / per + extra b + i, so that some numbers between them have no unit
// (1024 single tokens over up to 200: 135 us looked through, 84 searched).
struct Unit { int b, i; SeqRows s; };
constexpr int kLookThrough = 64;
template <class Count> __device__ __forceinline__ Unit find_unit(const PackedSeqs& p, int u, int per, int extra, Count count) {
    const int lane = threadIdx.x & 31;
    Unit r;
    r.b = -1; r.i = 0; r.s.row0 = r.s.n = r.s.ctx = 0; r.s.sound = true;
    if (p.B > kLookThrough) {
        if ((long)u * 32 + lane < p.B) seq_rows(p, u * 32 + lane);        // for what it reports
        const int id = p.T / per + extra * p.B - 1 - u;
        auto first = [&](int b) { return min(max(p.cu[b], 0), p.T) / per + extra * b; };
        const int b = count_below(p.B, [&](int i) { return first(i) <= id; }) - 1;
        if (b < 0) return r;
        const SeqRows s = seq_rows(p, b);
        const int i = id - first(b);
        if (s.n > 0 && i >= 0 && i < count(s)) { r.b = b; r.i = i; r.s = s; }
        return r;
    }
    int base = 0;
    for (int b0 = 0; b0 < p.B; b0 += 32) {
        const int b = p.B - 1 - b0 - lane;
        SeqRows s = {0, 0, 0, true};
        if (b >= 0) s = seq_rows(p, b);
        const int c = s.n > 0 ? count(s) : 0;
        int incl = c;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int t = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += t;
        }
        const unsigned hit = __ballot_sync(0xffffffffu, u < base + incl);
        if (hit) {
            const int src = __ffs(hit) - 1;
            r.b = __shfl_sync(0xffffffffu, b, src);
            r.i = base + __shfl_sync(0xffffffffu, incl, src) - 1 - u;
            r.s.row0 = __shfl_sync(0xffffffffu, s.row0, src);
            r.s.n = __shfl_sync(0xffffffffu, s.n, src);
            r.s.ctx = __shfl_sync(0xffffffffu, s.ctx, src);
            r.s.sound = __shfl_sync(0xffffffffu, (int)s.sound, src);
            return r;
        }
        base += __shfl_sync(0xffffffffu, incl, 31);
    }
    return r;
}

// How many units find_unit has to be asked for: of `per` rows each, the first row of a sequence opening one.
inline long most_units(const PackedSeqs& p, int per) {
    const long seqs = p.B < p.T ? p.B : p.T;
    return p.B > kLookThrough ? p.T / per + (long)p.B : seqs + (p.T - seqs) / per;
}

// The host's checks of those arguments. Positions stay far from the end of 32 bits, so that a sum with a row's index does.
inline bool table_ok(const PackedSeqs& p) {
    return p.ctx && p.page_table && aligned(p.ctx, 4) && aligned(p.page_table, 4) && p.max_pages > 0 && p.max_ctx >= 0 && p.max_ctx < 1 << 30 &&
           (long)p.max_ctx < (long)p.max_pages * kPage;
}
inline bool packed_ok(const PackedSeqs& p) {
    return p.cu && aligned(p.cu, 4) && p.B > 0 && p.T >= 0 && p.n_pages > 0 && table_ok(p);
}

}  // namespace flexllm
