// serving.h -- internal interface of the batched serving kernels: the paged
// attention front (paged_front.hip), paged decode attention
// (paged_attention.hip) and logits processing (logits.hip).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>
#include "layer_ops.h"

namespace jllm_hip {

constexpr int64_t SERVING_MAX_BLOCKS = (int64_t)1 << 24;   // 2^32 threads of 256-thread workgroups

// ---- paged attention front ----

// Rotary frequencies in turns: f[i] = theta^(-2i / head_dim) / 2 pi as a 64-bit
// fraction of a turn, so that position * f[i] modulo 2^64 is the angle's
// fraction of a turn whatever the position.
struct RopeTurns {
    uint64_t f[ROPE_MAX_HALF];
};
void rope_turns(RopeTurns& rt, int head_dim, double theta);

struct PagedFrontArgs {
    uint16_t* q_out;          // [N][q_out_stride]
    const uint16_t* q;        // [N][q_stride]: n_heads * hd values
    const uint16_t* k;        // [N][k_stride]: n_kv * hd values
    const uint16_t* v;        // [N][v_stride]
    int64_t q_out_stride, q_stride, k_stride, v_stride;
    const void* q_norm;       // [hd] or null (neither q nor k is normed)
    const void* k_norm;
    void* k_pages;            // [n_slots][n_kv][cache_head_dim]
    void* v_pages;
    float* k_scales;          // [n_slots][n_kv] (int8 only)
    float* v_scales;
    int64_t n_slots;
    const int32_t* positions; // [N]
    const int32_t* slots;     // [N]
    int n_heads, n_kv, head_dim, cache_head_dim, N;
    float eps;
    int norm_fp32, neox, kv_int8;
    RopeTurns rt;
};
hipError_t paged_front_launch(const PagedFrontArgs& a, hipStream_t st);
int64_t paged_front_blocks(const PagedFrontArgs& a);

// ---- paged decode attention ----

struct PagedAttnArgs {
    uint16_t* out;            // [B][n_heads * hd]
    const uint16_t* q;        // [B][q_stride]
    int64_t q_stride;
    const void* k;            // [n_pages][page_size][n_kv][cache_head_dim]
    const void* v;
    const float* ks;          // [n_pages][page_size][n_kv] (int8 only; null = 1)
    const float* vs;
    const int32_t* table;     // [B][table_stride] page ids
    const int32_t* lens;      // [B]
    float* part;              // partials, see paged_attention.hip
    int64_t table_stride;
    int n_pages, page_shift, B, n_heads, n_kv, head_dim, cache_head_dim, max_seq, window;
    float scale;
};
// workgroups that a call of these sizes launches (below SERVING_MAX_BLOCKS)
int64_t paged_attn_blocks(int B, int n_kv, int max_seq, int window);
// bytes of partials for these sizes (0 when no row is cut)
int64_t paged_attn_workspace(int B, int n_heads, int n_kv, int head_dim, int max_seq, int window);
hipError_t paged_attn_launch(const PagedAttnArgs& a, bool kv_int8, hipStream_t st);

// ---- logits ----

struct LogitsArgs {
    float* out;               // [B][out_stride]
    const float* x;           // [B][x_stride]
    int64_t out_stride, x_stride;
    int B, V;
    const int32_t* tokens;    // [B][token_stride] or null
    int64_t token_stride;
    const int32_t* n_prompt;  // [B] or null (0)
    const int32_t* n_tokens;  // [B]
    const float* repetition;  // [B] or null (1)
    const float* frequency;   // [B] or null (0)
    const float* presence;    // [B] or null (0)
    const int32_t* bias_ids;  // [B][bias_stride] or null
    const float* bias;        // [B][bias_stride]
    int64_t bias_stride;
    const int32_t* n_bias;    // [B]
    const uint32_t* mask;     // [B][mask_stride] or null
    int64_t mask_stride;
    int32_t* next_token;      // [B] or null
    uint64_t* cand;           // [B][chunks] (next_token with more than one chunk)
};
int64_t logits_workspace(int B, int V);
hipError_t logits_launch(const LogitsArgs& a, hipStream_t st);

}  // namespace jllm_hip
