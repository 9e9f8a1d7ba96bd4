// paged_attention.hip -- decode attention of a batch of query rows, each over the
// pages of its own sequence.
//
//   s_t = scale * ks_t * (q . k_t),  out = sum_t e^(s_t - m) vs_t v_t / sum_t e^(s_t - m)
//
// over the keys t of the row: [max(0, len - window), len).  Key t lies in slot
// t % page_size of page table[row][t / page_size].
#include "attn_common.h"
#include "serving.h"

namespace jllm_hip {

__device__ __forceinline__ float page_val(const void* p, int64_t i, bool int8) {
    return int8 ? (float)((const int8_t*)p)[i] : f16_bits_to_f32(((const uint16_t*)p)[i]);
}

// one wave per (row, query head), lane l: d = l and l + 64
template <bool INT8>
__global__ __launch_bounds__(64) void paged_attn_kernel(PagedAttnArgs a) {
    const int b = blockIdx.y, h = blockIdx.x, l = threadIdx.x, hd = a.head_dim;
    const int kvh = h / (a.n_heads / a.n_kv);
    int len = a.lens[b];
    len = len < 0 ? 0 : (len > a.max_seq ? a.max_seq : len);
    const int lo = a.window > 0 && len > a.window ? len - a.window : 0;
    const bool a0 = l < hd, a1 = l + 64 < hd;
    const uint16_t* q = a.q + b * a.q_stride + (int64_t)h * hd;
    const float q0 = a0 ? f16_bits_to_f32(q[l]) : 0.0f, q1 = a1 ? f16_bits_to_f32(q[l + 64]) : 0.0f;
    float m = -INFINITY, L = 0.0f, o0 = 0.0f, o1 = 0.0f;
    for (int t = lo; t < len; t++) {
        const int page = a.table[b * a.table_stride + (t >> a.page_shift)];
        if (page < 0 || page >= a.n_pages) continue;
        const int64_t slot = ((int64_t)page << a.page_shift) + (t & ((1 << a.page_shift) - 1));
        const int64_t row = slot * a.n_kv + kvh, at = row * a.cache_head_dim;
        const float k0 = a0 ? page_val(a.k, at + l, INT8) : 0.0f, k1 = a1 ? page_val(a.k, at + l + 64, INT8) : 0.0f;
        const float s = wave_sum(q0 * k0 + q1 * k1) * (INT8 && a.ks ? a.ks[row] : 1.0f) * a.scale;
        const float mn = fmaxf(m, s), base = mn == -INFINITY ? 0.0f : mn;
        const float c = expf(m - base), p = expf(s - base);
        const float pv = p * (INT8 && a.vs ? a.vs[row] : 1.0f);
        L = L * c + p;
        o0 = o0 * c + (a0 ? pv * page_val(a.v, at + l, INT8) : 0.0f);
        o1 = o1 * c + (a1 ? pv * page_val(a.v, at + l + 64, INT8) : 0.0f);
        m = mn;
    }
    // rows without a key (or with none of finite score) are zero; a NaN stays
    uint16_t* o = a.out + ((int64_t)b * a.n_heads + h) * hd;
    if (a0) o[l] = f32_to_f16_bits(L == 0.0f ? 0.0f : o0 / L);
    if (a1) o[l + 64] = f32_to_f16_bits(L == 0.0f ? 0.0f : o1 / L);
}

int64_t paged_attn_workspace(int, int, int, int, int, int) { return 0; }

hipError_t paged_attn_launch(const PagedAttnArgs& a, bool kv_int8, hipStream_t st) {
    const dim3 grid(a.n_heads, a.B);
    if (kv_int8) hipLaunchKernelGGL((paged_attn_kernel<true>), grid, dim3(64), 0, st, a);
    else         hipLaunchKernelGGL((paged_attn_kernel<false>), grid, dim3(64), 0, st, a);
    return hipGetLastError();
}

}  // namespace jllm_hip
