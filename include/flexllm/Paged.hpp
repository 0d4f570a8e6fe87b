// Packed sequences over a floating-point paged cache, and products with 4-bit weights (no counterparts in Modules/)
#pragma once
#include "common.hpp"
namespace flexllm {
// One step's sequences: rows cu[b] .. cu[b+1] - 1 at cache positions ctx[b] .. of the pages page_table[b] (device memory)
struct PackedSequences {
    const int32_t *cu, *ctx, *page_table;
    int max_pages, max_ctx, sequences, rows;
};
// A floating-point cache whose layers are handed out as pages
class FloatKVCache {
  public:
    FloatKVCache() = default;
    FloatKVCache(const FloatKVCache&) = delete;
    FloatKVCache& operator=(const FloatKVCache&) = delete;
    ~FloatKVCache() { flexllm_kv_cache_destroy(h_); }
    int create(int layers, int n_pages, const flexllm_kv_shape* shapes, int dtype) {
        return flexllm_kv_cache_create_float(&h_, layers, n_pages, shapes, 64, dtype == FLEXLLM_BF16 ? 2 : 4);
    }
    int pages(int layer, flexllm_kv_pages* out) { return flexllm_kv_cache_pages(h_, layer, out); }
    flexllm_kv_cache* handle() const { return h_; }
  private:
    flexllm_kv_cache* h_ = nullptr;
};
inline int qk_norm_rope(int dtype, const flexllm_kv_pages& kv, int heads, const void* proj, long ldp, const float* q_gain, const float* k_gain, float eps,
                        const int32_t* pos, int axes, const int* sections_host, const float* cos_t, const float* sin_t, int rot, int table_len,
                        const PackedSequences& s, void* q, long ldq, stream_t st = nullptr) {
    return flexllm_qk_norm_rope(dtype, &kv, heads, proj, ldp, q_gain, k_gain, eps, pos, axes, sections_host, cos_t, sin_t, rot, table_len, s.cu, s.ctx,
                                s.page_table, s.max_pages, s.max_ctx, s.sequences, s.rows, q, ldq, st);
}
inline int attn_packed(int dtype, const flexllm_kv_pages& kv, int heads, float scale, const void* q, long ldq, const PackedSequences& s, void* out, long ldo,
                       stream_t st = nullptr) {
    return flexllm_attn_packed(dtype, &kv, heads, scale, q, ldq, s.cu, s.ctx, s.page_table, s.max_pages, s.max_ctx, s.sequences, s.rows, out, ldo, st);
}
inline int attn_tree(int dtype, const flexllm_kv_pages& kv, int heads, float scale, const void* q, long ldq, const uint64_t* mask, const PackedSequences& s,
                     void* out, long ldo, stream_t st = nullptr) {
    return flexllm_attn_tree(dtype, &kv, heads, scale, q, ldq, mask, s.cu, s.ctx, s.page_table, s.max_pages, s.max_ctx, s.sequences, s.rows, out, ldo, st);
}
inline int kv_keep(int dtype, const flexllm_kv_pages* layers_host, int layers, const PackedSequences& s, const int32_t* keep, const int32_t* count, int most,
                   stream_t st = nullptr) {
    return flexllm_kv_keep(dtype, layers_host, layers, s.page_table, s.max_pages, s.ctx, s.max_ctx, keep, count, most, s.sequences, st);
}
inline int linear_w4(int dtype, const void* a, long lda, const uint8_t* w, const void* scale, int scale_dtype, const uint8_t* zero, int group,
                     const float* bias, int M, int N, int K, void* y, long ldy, bool y_f32 = false, stream_t st = nullptr) {
    return flexllm_linear_w4(dtype, a, lda, w, scale, scale_dtype, zero, group, bias, M, N, K, y, ldy, y_f32 ? 1 : 0, st);
}
}  // namespace flexllm
