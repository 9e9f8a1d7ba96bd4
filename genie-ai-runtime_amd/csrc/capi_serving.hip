// capi_serving.hip -- C ABI of the batched serving kernels: the attention front
// over a paged KV cache, paged decode attention and logits processing.
#include "capi_common.h"
#include "serving.h"

using namespace jllm_hip;

namespace {
inline bool aligned(const void* p, unsigned n) { return ((uintptr_t)p & (n - 1)) == 0; }
inline bool finite_pos(float x) { return x > 0.0f && x <= 3.402823466e+38f; }

int refuse(const char* tag, const char* what) {
    fprintf(stderr, "[%s] %s\n", tag, what);
    return JLLM_ERR_INVALID;
}

constexpr int MAX_BATCH = 65535;                 // grid dimension

bool attn_shape_ok(int B, int n_heads, int n_kv, int hd, int max_seq, int window) {
    return B >= 0 && B <= MAX_BATCH && n_kv > 0 && n_heads > 0 && n_heads % n_kv == 0 && n_heads / n_kv <= 16 &&
           n_heads <= 4096 && hd > 0 && hd % 32 == 0 && hd <= 128 && max_seq >= 0 && window >= 0 &&
           paged_attn_blocks(B, n_kv, max_seq, window) < SERVING_MAX_BLOCKS;
}
}  // namespace

extern "C" {

int jllm_hip_qk_norm_rope_store_kv_paged(uint16_t* q_out, int64_t q_out_stride, const uint16_t* q, int64_t q_stride,
                                         const uint16_t* k, int64_t k_stride, const uint16_t* v, int64_t v_stride,
                                         const void* q_norm, const void* k_norm, int norm_fp32, float eps,
                                         void* k_pages, void* v_pages, float* k_scales, float* v_scales,
                                         int64_t n_slots, const int32_t* positions, const int32_t* slots,
                                         int n_heads, int n_kv_heads, int head_dim, int cache_head_dim, int N,
                                         float theta_base, int neox, int kv_int8, void* stream) {
    static const char tag[] = "qk_norm_rope_store_kv_paged";
    if (N < 0 || n_heads <= 0 || n_kv_heads <= 0 || n_heads > 4096 || n_kv_heads > 4096 || n_slots < 0 ||
        n_slots > INT32_MAX)
        return refuse(tag, "a count out of range");
    if (head_dim <= 0 || head_dim % 8 != 0 || head_dim > 2 * ROPE_MAX_HALF || cache_head_dim < head_dim ||
        ((int64_t)cache_head_dim * (kv_int8 ? 1 : 2)) % 16 != 0)
        return refuse(tag, "need head_dim % 8 == 0, head_dim <= 128, cache_head_dim >= head_dim and cache rows of a "
                           "multiple of 16 bytes");
    if (!finite_pos(theta_base) || !(eps >= 0.0f)) return refuse(tag, "need theta_base > 0 and eps >= 0");
    if (q_out_stride < (int64_t)n_heads * head_dim || q_stride < (int64_t)n_heads * head_dim ||
        k_stride < (int64_t)n_kv_heads * head_dim || v_stride < (int64_t)n_kv_heads * head_dim ||
        q_out_stride % 4 || q_stride % 4 || k_stride % 4 || v_stride % 4)
        return refuse(tag, "row strides must hold a row and be multiples of 4 halves");
    if (N == 0) return JLLM_OK;
    if (!q_out || !q || !k || !v || !k_pages || !v_pages || !positions || !slots) return refuse(tag, "null pointer");
    if ((q_norm == nullptr) != (k_norm == nullptr)) return refuse(tag, "q_norm and k_norm: both or neither");
    if (kv_int8 && (!k_scales || !v_scales)) return refuse(tag, "an INT8 cache needs both scale arrays");
    if (!aligned(q_out, 8) || !aligned(q, 8) || !aligned(k, 8) || !aligned(v, 8) || !aligned16(k_pages) ||
        !aligned16(v_pages) || !aligned(positions, 4) || !aligned(slots, 4) ||
        (kv_int8 && (!aligned(k_scales, 4) || !aligned(v_scales, 4))) ||
        !aligned(q_norm, norm_fp32 ? 4 : 2) || !aligned(k_norm, norm_fp32 ? 4 : 2))
        return refuse(tag, "q, k, v must be 8-byte and the pages 16-byte aligned");
    if (q_out == q && q_out_stride != q_stride) return refuse(tag, "q in place needs q_out_stride == q_stride");
    PagedFrontArgs a;
    a.q_out = q_out; a.q = q; a.k = k; a.v = v;
    a.q_out_stride = q_out_stride; a.q_stride = q_stride; a.k_stride = k_stride; a.v_stride = v_stride;
    a.q_norm = q_norm; a.k_norm = k_norm; a.k_pages = k_pages; a.v_pages = v_pages;
    a.k_scales = k_scales; a.v_scales = v_scales; a.n_slots = n_slots; a.positions = positions; a.slots = slots;
    a.n_heads = n_heads; a.n_kv = n_kv_heads; a.head_dim = head_dim; a.cache_head_dim = cache_head_dim; a.N = N;
    // (the reciprocal root takes a subnormal for 0, which would make a row of zeros NaN; of
    // other rows the mean square is above 2^-56, where neither eps is seen)
    a.eps = eps > 0.0f && eps < 1.17549435e-38f ? 1.17549435e-38f : eps;
    a.norm_fp32 = norm_fp32 != 0; a.neox = neox != 0; a.kv_int8 = kv_int8 != 0;
    if (paged_front_blocks(a) >= SERVING_MAX_BLOCKS) return refuse(tag, "too many tokens for one launch");
    rope_turns(a.rt, head_dim, theta_base);
    return launch_status(paged_front_launch(a, (hipStream_t)stream), tag);
}

int64_t jllm_hip_flash_attention_decode_paged_workspace(int B, int n_heads, int n_kv_heads, int head_dim, int max_seq,
                                                        int window) {
    if (!attn_shape_ok(B, n_heads, n_kv_heads, head_dim, max_seq, window)) return JLLM_ERR_INVALID;
    return paged_attn_workspace(B, n_heads, n_kv_heads, head_dim, max_seq, window);
}

int jllm_hip_flash_attention_decode_paged(uint16_t* out, const uint16_t* q, int64_t q_stride, const void* k_pages,
                                          const void* v_pages, const float* k_scales, const float* v_scales,
                                          int n_pages, int page_size, const int32_t* block_table,
                                          int64_t table_stride, const int32_t* seq_lens, int B, int n_heads,
                                          int n_kv_heads, int head_dim, int cache_head_dim, int max_seq, float scale,
                                          int kv_int8, int window, void* workspace, int64_t workspace_bytes,
                                          void* stream) {
    static const char tag[] = "flash_attention_decode_paged";
    if (!attn_shape_ok(B, n_heads, n_kv_heads, head_dim, max_seq, window))
        return refuse(tag, "need n_heads % n_kv_heads == 0, <= 16 q heads per KV head, head_dim a multiple of 32 up "
                           "to 128, B <= 65535, max_seq >= 0, window >= 0 and fewer than 2^24 workgroups");
    if (cache_head_dim < head_dim || cache_head_dim > 4096 || ((int64_t)cache_head_dim * (kv_int8 ? 1 : 2)) % 16 != 0)
        return refuse(tag, "need head_dim <= cache_head_dim <= 4096 and cache rows of a multiple of 16 bytes");
    if (page_size < 16 || page_size > 4096 || (page_size & (page_size - 1)) || n_pages < 0 ||
        (int64_t)n_pages * page_size > INT32_MAX)
        return refuse(tag, "need page_size a power of two from 16 to 4096 and n_pages * page_size < 2^31");
    if (table_stride < ((int64_t)max_seq + page_size - 1) / page_size)
        return refuse(tag, "block_table rows are shorter than max_seq");
    if (q_stride < (int64_t)n_heads * head_dim || q_stride % 8 != 0)
        return refuse(tag, "q_stride must hold a row and be a multiple of 8 halves");
    if (!(scale - scale == 0.0f)) return refuse(tag, "scale must be finite");
    if (B == 0) return JLLM_OK;
    if (!out || !q || !seq_lens || (max_seq > 0 && !block_table) || (max_seq > 0 && n_pages > 0 && (!k_pages || !v_pages)))
        return refuse(tag, "null pointer");
    if (!aligned16(out) || !aligned16(q) || !aligned16(k_pages) || !aligned16(v_pages) || !aligned(k_scales, 4) ||
        !aligned(v_scales, 4) || !aligned(block_table, 4) || !aligned(seq_lens, 4))
        return refuse(tag, "out, q and the pages must be 16-byte aligned");
    const int64_t need = paged_attn_workspace(B, n_heads, n_kv_heads, head_dim, max_seq, window);
    if (need > 0 && (!workspace || workspace_bytes < need || !aligned16(workspace)))
        return refuse(tag, "workspace: null, not 16-byte aligned or smaller than "
                           "jllm_hip_flash_attention_decode_paged_workspace says");
    PagedAttnArgs a;
    a.out = out; a.q = q; a.q_stride = q_stride; a.k = k_pages; a.v = v_pages;
    a.ks = kv_int8 ? k_scales : nullptr; a.vs = kv_int8 ? v_scales : nullptr;
    a.table = block_table; a.lens = seq_lens; a.part = (float*)workspace; a.table_stride = table_stride;
    a.n_pages = n_pages; a.page_shift = __builtin_ctz((unsigned)page_size); a.B = B; a.n_heads = n_heads;
    a.n_kv = n_kv_heads; a.head_dim = head_dim; a.cache_head_dim = cache_head_dim; a.max_seq = max_seq;
    a.window = window; a.scale = scale;
    return launch_status(paged_attn_launch(a, kv_int8 != 0, (hipStream_t)stream), tag);
}

int64_t jllm_hip_logits_process_workspace(int B, int V) {
    if (B < 0 || B > MAX_BATCH || V <= 0) return JLLM_ERR_INVALID;
    return logits_workspace(B, V);
}

int jllm_hip_logits_process(float* out, int64_t out_stride, const float* logits, int64_t logits_stride, int B, int V,
                            const int32_t* tokens, int64_t token_stride, const int32_t* n_prompt,
                            const int32_t* n_tokens, const float* repetition, const float* frequency,
                            const float* presence, const int32_t* bias_ids, const float* bias, int64_t bias_stride,
                            const int32_t* n_bias, const uint32_t* mask, int64_t mask_stride, int32_t* next_token,
                            void* workspace, int64_t workspace_bytes, void* stream) {
    static const char tag[] = "logits_process";
    if (B < 0 || B > MAX_BATCH || V <= 0 || out_stride < V || logits_stride < V)
        return refuse(tag, "need 0 <= B <= 65535, V > 0 and row strides of at least V");
    if (tokens && (!n_tokens || token_stride < 0 || token_stride > INT32_MAX))
        return refuse(tag, "tokens need n_tokens and a stride below 2^31");
    if (bias_ids && (!bias || !n_bias || bias_stride < 0 || bias_stride > INT32_MAX))
        return refuse(tag, "bias_ids need bias, n_bias and a stride below 2^31");
    if (mask && mask_stride < ((int64_t)V + 31) / 32) return refuse(tag, "mask rows hold less than V bits");
    if (B == 0) return JLLM_OK;
    if (!out || !logits) return refuse(tag, "null pointer");
    if (out == logits && out_stride != logits_stride) return refuse(tag, "in place needs equal strides");
    const void* words[] = {out, logits, tokens, n_prompt, n_tokens, repetition, frequency, presence, bias_ids, bias,
                           n_bias, mask, next_token};
    for (const void* p : words)
        if (!aligned(p, 4)) return refuse(tag, "pointers must be 4-byte aligned");
    if ((int64_t)B * (((int64_t)V + 1023) / 1024) >= SERVING_MAX_BLOCKS) return refuse(tag, "too many logits for one launch");
    const int64_t need = next_token ? logits_workspace(B, V) : 0;
    if (need > 0 && (!workspace || workspace_bytes < need || !aligned(workspace, 8)))
        return refuse(tag, "workspace: null, not 8-byte aligned or smaller than jllm_hip_logits_process_workspace says");
    LogitsArgs a;
    a.out = out; a.x = logits; a.out_stride = out_stride; a.x_stride = logits_stride; a.B = B; a.V = V;
    a.tokens = tokens; a.token_stride = token_stride; a.n_prompt = n_prompt; a.n_tokens = n_tokens;
    a.repetition = repetition; a.frequency = frequency; a.presence = presence;
    a.bias_ids = bias_ids; a.bias = bias; a.bias_stride = bias_stride; a.n_bias = n_bias;
    a.mask = mask; a.mask_stride = mask_stride; a.next_token = next_token; a.cand = (uint64_t*)workspace;
    return launch_status(logits_launch(a, (hipStream_t)stream), tag);
}

}  // extern "C"
