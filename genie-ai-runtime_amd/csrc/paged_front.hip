// paged_front.hip -- the attention front of a batch of tokens over a paged KV
// cache: q / k RMSNorm per head, RoPE of q and k, and the store of k and v into
// the cache slot of each token, in one launch.
//
//   n = x / sqrt(mean(x^2) + eps) * w
//   (a, b) -> (a cos t - b sin t, a sin t + b cos t),  t = position * theta^(-2i/hd)
//   cache: fp16(v), or code = rint(v * 127 / max|v|) with scale max|v| / 127
//
// All of it in fp32 from the fp16 inputs, rounded once, where q or the cache row
// is stored.  The contiguous front (qk_post_kernel, which replaces
// decode.cu:1441-1478) keeps the reference's fp16 roundings between the steps and
// its fp32 angle, which at position p is off by up to p * 2^-24 radians; here the
// angle is a 64-bit fraction of a turn, exact to 2^-32 turns at every position.
#include "kq_common.h"
#include "serving.h"
#include <math.h>

namespace jllm_hip {

typedef uint32_t u32x2f __attribute__((ext_vector_type(2)));

void rope_turns(RopeTurns& rt, int head_dim, double theta) {
    for (int i = 0; i < ROPE_MAX_HALF; i++) {
        if (i >= head_dim / 2) { rt.f[i] = 0; continue; }
        const double turns = pow(theta, -2.0 * i / head_dim) / 6.283185307179586476925286766559;
        rt.f[i] = (uint64_t)ldexp(turns - floor(turns), 64);
    }
}

// max of the bit patterns of |x|: NaN above infinity above every finite value
template <int CTRL>
__device__ __forceinline__ uint32_t dpp_max_u(uint32_t v) {
    const uint32_t o = (uint32_t)__builtin_amdgcn_mov_dpp((int)v, CTRL, 0xF, 0xF, false);
    return o > v ? o : v;
}
// reductions over aligned groups of GL lanes (4, 8 or 16): DPP steps as in wave_sum
template <int GL>
__device__ __forceinline__ float group_sum_dpp(float v) {
    v += dpp_mov_f<0xB1>(v);
    v += dpp_mov_f<0x4E>(v);
    if (GL > 4) v += dpp_mov_f<0x141>(v);
    if (GL > 8) v += dpp_mov_f<0x140>(v);
    return v;
}
template <int GL>
__device__ __forceinline__ uint32_t group_max_dpp(uint32_t v) {
    v = dpp_max_u<0xB1>(v);
    v = dpp_max_u<0x4E>(v);
    if (GL > 4) v = dpp_max_u<0x141>(v);
    if (GL > 8) v = dpp_max_u<0x140>(v);
    return v;
}

__device__ __forceinline__ u32x2f pack4(const float* x) {
    return u32x2f{(uint32_t)f32_to_f16_bits(x[0]) | ((uint32_t)f32_to_f16_bits(x[1]) << 16),
                  (uint32_t)f32_to_f16_bits(x[2]) | ((uint32_t)f32_to_f16_bits(x[3]) << 16)};
}
__device__ __forceinline__ uint32_t code4(const float* x, float inv) {
    uint32_t w = 0;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        int c = (int)__builtin_rintf(x[j] * inv);
        c = c > 127 ? 127 : (c < -127 ? -127 : c);
        w |= ((uint32_t)c & 0xFFu) << (8 * j);
    }
    return w;
}

// One wave takes 64 / GL rows (heads) of one token, GL lanes a row, 8 values a
// lane: values e0 + [0, 4) and e1 + [0, 4) with, in split pairs (neox), e0 = 4 gl
// and e1 = e0 + hd / 2, in interleaved pairs e0 = 8 gl and e1 = e0 + 4; either way
// the lane's four pairs are its own and have the frequencies 4 gl + [0, 4).
template <int GL, bool INT8>
__global__ __launch_bounds__(256) void paged_front_kernel(PagedFrontArgs a) {
    constexpr int RG = 64 / GL;                        // rows a wave takes at once
    const int hd = a.head_dim, R = a.n_heads + 2 * a.n_kv;
    const int groups = (R + RG - 1) / RG;
    const int64_t gw = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int l = threadIdx.x & 63, sub = l / GL, gl = l % GL;
    const int64_t t = gw / groups;
    const int g = (int)(gw % groups);
    if (t >= a.N) return;
    const int slot = a.slots[t];
    if (slot < 0 || slot >= a.n_slots) return;         // padding: nothing of this token is written
    const int r = g * RG + sub;
    const bool act = 8 * gl < hd && r < R;
    const int kind = r < a.n_heads ? 0 : (r < a.n_heads + a.n_kv ? 1 : 2);   // q, k, v
    const int head = kind == 0 ? r : (kind == 1 ? r - a.n_heads : r - a.n_heads - a.n_kv);
    const int e0 = a.neox ? 4 * gl : 8 * gl, e1 = a.neox ? e0 + hd / 2 : e0 + 4;
    const uint16_t* src = (kind == 0 ? a.q + t * a.q_stride : (kind == 1 ? a.k + t * a.k_stride : a.v + t * a.v_stride)) +
                          (int64_t)head * hd;
    u32x2f ra = {0u, 0u}, rb = {0u, 0u};
    if (act) { ra = *(const u32x2f*)(src + e0); rb = *(const u32x2f*)(src + e1); }
    float x[8];
#pragma unroll
    for (int j = 0; j < 2; j++) {
        x[2 * j] = f16_bits_to_f32(ra[j] & 0xFFFFu); x[2 * j + 1] = f16_bits_to_f32(ra[j] >> 16);
        x[4 + 2 * j] = f16_bits_to_f32(rb[j] & 0xFFFFu); x[5 + 2 * j] = f16_bits_to_f32(rb[j] >> 16);
    }
    if (a.q_norm) {
        float ss = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; j++) ss += x[j] * x[j];
        ss = group_sum_dpp<GL>(ss);
        if (kind < 2 && act) {
            const void* w = kind == 0 ? a.q_norm : a.k_norm;
            const float rrms = 1.0f / sqrtf(ss / (float)hd + a.eps);
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const int e = j < 4 ? e0 + j : e1 + j - 4;
                x[j] *= rrms * (a.norm_fp32 ? ((const float*)w)[e] : f16_bits_to_f32(((const uint16_t*)w)[e]));
            }
        }
    }
    if (kind < 2 && act) {
        const int64_t pos = a.positions[t];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            // signed fraction of a turn in units of 2^-32; sin and cos of pi * (2 frac)
            const int32_t fr = (int32_t)((a.rt.f[4 * gl + j] * (uint64_t)pos) >> 32);
            float s, c;
            sincospif((float)fr * 0x1p-31f, &s, &c);
            float& p = a.neox ? x[j] : x[2 * j];
            float& q = a.neox ? x[4 + j] : x[2 * j + 1];
            const float u = p * c - q * s, w = p * s + q * c;
            p = u;
            q = w;
        }
    }
    if (kind == 0) {
        if (act) {
            uint16_t* o = a.q_out + t * a.q_out_stride + (int64_t)head * hd;
            *(u32x2f*)(o + e0) = pack4(x);
            *(u32x2f*)(o + e1) = pack4(x + 4);
        }
    }
    const int64_t row = (int64_t)slot * a.n_kv + head;
    void* pages = kind == 1 ? a.k_pages : a.v_pages;
    if (INT8) {
        uint32_t mb = 0;
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const uint32_t b = __builtin_bit_cast(uint32_t, x[j]) & 0x7FFFFFFFu;
            mb = b > mb ? b : mb;
        }
        mb = group_max_dpp<GL>(mb);
        if (kind > 0 && act) {
            const float mx = __builtin_bit_cast(float, mb);
            const bool fine = mb < 0x7F800000u;        // a row with a NaN or an infinity reads as NaN
            const float inv = fine && mx > 1e-35f ? 127.0f / mx : 0.0f;
            int8_t* o = (int8_t*)pages + row * a.cache_head_dim;
            *(uint32_t*)(o + e0) = fine ? code4(x, inv) : 0u;
            *(uint32_t*)(o + e1) = fine ? code4(x + 4, inv) : 0u;
            if (gl == 0) (kind == 1 ? a.k_scales : a.v_scales)[row] = fine ? mx / 127.0f : __builtin_nanf("");
        }
    } else if (kind > 0 && act) {
        uint16_t* o = (uint16_t*)pages + row * a.cache_head_dim;
        *(u32x2f*)(o + e0) = pack4(x);
        *(u32x2f*)(o + e1) = pack4(x + 4);
    }
}

namespace {
int lanes_of(int hd) { return hd <= 32 ? 4 : (hd <= 64 ? 8 : 16); }
}  // namespace

int64_t paged_front_blocks(const PagedFrontArgs& a) {
    const int rg = 64 / lanes_of(a.head_dim);
    const int64_t groups = (a.n_heads + 2 * (int64_t)a.n_kv + rg - 1) / rg;
    return ((int64_t)a.N * groups + 3) / 4;
}

hipError_t paged_front_launch(const PagedFrontArgs& a, hipStream_t st) {
    const dim3 grid((unsigned)paged_front_blocks(a));
#define FRONT_CASE(GL)                                                                              \
    if (a.kv_int8) hipLaunchKernelGGL((paged_front_kernel<GL, true>), grid, dim3(256), 0, st, a);   \
    else           hipLaunchKernelGGL((paged_front_kernel<GL, false>), grid, dim3(256), 0, st, a);
    switch (lanes_of(a.head_dim)) {
    case 4:  FRONT_CASE(4) break;
    case 8:  FRONT_CASE(8) break;
    default: FRONT_CASE(16) break;
    }
#undef FRONT_CASE
    return hipGetLastError();
}

}  // namespace jllm_hip
