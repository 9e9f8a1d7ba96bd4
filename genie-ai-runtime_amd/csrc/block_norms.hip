// block_norms.hip -- what stands between two blocks of a layer, gfx950:
//
//   t = x, or x / sqrt(mean x^2 + eps) * w_post             the block's output
//   h = residual_scale * residual + branch_scale * gate * t    the residual stream
//   y = h / sqrt(mean h^2 + eps) * w_pre                       the next block's input
//
// with y as fp16 rows or as int8 codes rint(y * 127 / max |y|) and the scale max |y| / 127
// of each row.  One workgroup a row: the row stays in registers between its two sums, so
// every input is read and every output written once, and the bytes are the bound (8191 rows
// of 4096, gated and normed twice, 335 MB, 68 us: 4.9 TB/s, a copy of 1 GiB 5.1; one row of
// 2560 2.7 us, of which a launch is two).  fp32 from the inputs to the stores; y is formed
// from h before h is rounded, so each output carries one rounding.  For the codes
// 1 / sqrt(..) cancels: y / max |y| is h w / max |h w|, and that maximum is found in the same
// pass through LDS as the sum of squares (8191 rows of 4096, the block's output normed, 235 MB,
// 55 us: 4.3 TB/s); only where h w leaves fp32's range does a row take a second maximum.  Loading the weights and the gate with x instead of
// where they are used: 47.5 -> 45 us without a gate, 68.5 -> 67.6 with one, but 73 -> 102 for
// rows of 16384 (registers) and 2.8 -> 3.0 for one row.
#include "kq_common.h"
#include "serving.h"

namespace jllm_hip {

typedef uint32_t u32x4n __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2n __attribute__((ext_vector_type(2)));
typedef float f32x4n __attribute__((ext_vector_type(4)));

namespace {

__device__ __forceinline__ void load8_h(const uint16_t* p, float (&v)[8]) {
    const u32x4n u = *(const u32x4n*)p;
#pragma unroll
    for (int e = 0; e < 4; e++) {
        const half2_t h = as_h2(u[e]);
        v[2 * e] = (float)h[0];
        v[2 * e + 1] = (float)h[1];
    }
}
__device__ __forceinline__ void load8(const void* p, bool fp32, int64_t at, float (&v)[8]) {
    if (!fp32) return load8_h((const uint16_t*)p + at, v);
    const f32x4n a = *(const f32x4n*)((const float*)p + at), b = *(const f32x4n*)((const float*)p + at + 4);
#pragma unroll
    for (int e = 0; e < 4; e++) { v[e] = a[e]; v[4 + e] = b[e]; }
}
__device__ __forceinline__ u32x4n pack8_h(const float (&v)[8]) {
    u32x4n u;
#pragma unroll
    for (int e = 0; e < 4; e++) u[e] = (uint32_t)f32_to_f16_bits(v[2 * e]) | (uint32_t)f32_to_f16_bits(v[2 * e + 1]) << 16;
    return u;
}
__device__ __forceinline__ uint32_t wave_max_u32(uint32_t v) {
    auto step = [&](int x) { v = max(v, (uint32_t)x); };
    step(__builtin_amdgcn_mov_dpp((int)v, 0xB1, 0xF, 0xF, false));
    step(__builtin_amdgcn_mov_dpp((int)v, 0x4E, 0xF, 0xF, false));
    step(__builtin_amdgcn_mov_dpp((int)v, 0x141, 0xF, 0xF, false));
    step(__builtin_amdgcn_mov_dpp((int)v, 0x140, 0xF, 0xF, false));
    const uint32_t a = max((uint32_t)__builtin_amdgcn_readlane((int)v, 0), (uint32_t)__builtin_amdgcn_readlane((int)v, 16));
    const uint32_t b = max((uint32_t)__builtin_amdgcn_readlane((int)v, 32), (uint32_t)__builtin_amdgcn_readlane((int)v, 48));
    return max(a, b);
}
__device__ __forceinline__ float gate_of(float g, int kind) {
    return kind == 0 ? g : (kind == 1 ? 1.0f / (1.0f + expf(-g)) : tanhf(g));
}

// T threads a row, up to E pieces of 8 values each
template <int T, int E>
__global__ __launch_bounds__(T) void block_norms_kernel(BlockNormsArgs a) {
    constexpr int W = T / 64;
    __shared__ float sSum[2][W];
    __shared__ uint32_t sTop[W];
    const int64_t row = blockIdx.x;
    const int t = (int)threadIdx.x, lane = t & 63, wave = t >> 6;
    const int pieces = a.hidden / 8;
    float v[E][8], r[E][8];
#pragma unroll
    for (int i = 0; i < E; i++) {
        const int p = t + i * T;
#pragma unroll
        for (int e = 0; e < 8; e++) v[i][e] = r[i][e] = 0.0f;
        if (p < pieces) {
            load8_h(a.x + row * a.x_stride + 8 * p, v[i]);
            if (a.residual) load8(a.residual, a.h_fp32, row * a.residual_stride + 8 * p, r[i]);
        }
    }
    const float inv_n = 1.0f / (float)a.hidden;
    if (a.post) {
        float ss = 0.0f;
#pragma unroll
        for (int i = 0; i < E; i++)
#pragma unroll
            for (int e = 0; e < 8; e++) ss = fmaf(v[i][e], v[i][e], ss);
        ss = wave_sum(ss);
        if (W > 1) {
            if (lane == 0) sSum[0][wave] = ss;
            __syncthreads();
            ss = 0.0f;
#pragma unroll
            for (int w = 0; w < W; w++) ss += sSum[0][w];
        }
        const float f = 1.0f / sqrtf(ss * inv_n + a.eps);
#pragma unroll
        for (int i = 0; i < E; i++) {
            const int p = t + i * T;
            if (p >= pieces) continue;
            float w[8];
            load8(a.post, a.norm_fp32, 8 * p, w);
#pragma unroll
            for (int e = 0; e < 8; e++) v[i][e] = v[i][e] * f * w[e];
        }
    }
    float ss = 0.0f;
#pragma unroll
    for (int i = 0; i < E; i++) {
        const int p = t + i * T;
        if (p >= pieces) continue;
        if (a.gate) {
            float g[8];
            load8_h(a.gate + row * a.gate_stride + 8 * p, g);
#pragma unroll
            for (int e = 0; e < 8; e++) v[i][e] *= gate_of(g[e], a.gate_kind);
        }
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const float b = a.branch_scale * v[i][e];
            v[i][e] = a.residual ? fmaf(a.residual_scale, r[i][e], b) : b;
            ss = fmaf(v[i][e], v[i][e], ss);
        }
        if (a.h) {
            if (a.h_fp32) {
                float* o = (float*)a.h + row * a.h_stride + 8 * p;
                *(f32x4n*)o = f32x4n{v[i][0], v[i][1], v[i][2], v[i][3]};
                *(f32x4n*)(o + 4) = f32x4n{v[i][4], v[i][5], v[i][6], v[i][7]};
            } else {
                *(u32x4n*)((uint16_t*)a.h + row * a.h_stride + 8 * p) = pack8_h(v[i]);
            }
        }
    }
    if (!a.y && !a.codes) return;
    // h times the weights in v; maximum of their magnitudes as bits, so that a NaN is the largest
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < E; i++) {
        const int p = t + i * T;
        if (p >= pieces) continue;
        float w[8];
        load8(a.pre, a.norm_fp32, 8 * p, w);
#pragma unroll
        for (int e = 0; e < 8; e++) {
            r[i][e] = w[e];
            if (a.codes) top = max(top, __builtin_bit_cast(uint32_t, v[i][e] * w[e]) & 0x7FFFFFFFu);
        }
    }
    ss = wave_sum(ss);
    if (a.codes) top = wave_max_u32(top);
    if (W > 1) {
        if (lane == 0) { sSum[1][wave] = ss; sTop[wave] = top; }
        __syncthreads();
        ss = 0.0f;
        top = 0;
#pragma unroll
        for (int w = 0; w < W; w++) { ss += sSum[1][w]; top = max(top, sTop[w]); }
    }
    const float f = 1.0f / sqrtf(ss * inv_n + a.eps);
    if (a.y) {
#pragma unroll
        for (int i = 0; i < E; i++) {
            const int p = t + i * T;
            if (p >= pieces) continue;
            float y[8];
#pragma unroll
            for (int e = 0; e < 8; e++) y[e] = v[i][e] * f * r[i][e];
            *(u32x4n*)(a.y + row * a.y_stride + 8 * p) = pack8_h(y);
        }
    }
    if (a.codes) {
        float m = __builtin_bit_cast(float, top), by = 1.0f, scale;
        const bool far = !(m >= 0x1p-100f && m <= 0x1p126f);
        if (far) by = f;
#pragma unroll
        for (int i = 0; i < E; i++)
#pragma unroll
            for (int e = 0; e < 8; e++) r[i][e] *= v[i][e] * by;
        scale = f * m * (1.0f / 127.0f);
        if (far) {
            // h times the weights has left fp32's range, or is about to, where y need not: the
            // codes are y's own then, by a maximum of their own.  (Rows of zeros, infinities and
            // NaN come here too.)
            top = 0;
#pragma unroll
            for (int i = 0; i < E; i++)
#pragma unroll
                for (int e = 0; e < 8; e++)
                    if (t + i * T < pieces) top = max(top, __builtin_bit_cast(uint32_t, r[i][e]) & 0x7FFFFFFFu);
            top = wave_max_u32(top);
            if (W > 1) {
                __syncthreads();                       // (the first maximum has been read)
                if (lane == 0) sTop[wave] = top;
                __syncthreads();
                top = 0;
#pragma unroll
                for (int w = 0; w < W; w++) top = max(top, sTop[w]);
            }
            m = __builtin_bit_cast(float, top);
            scale = m * (1.0f / 127.0f);
        }
        const bool fine = m <= 3.402823466e+38f && scale <= 3.402823466e+38f;   // a row with an infinity or NaN has no scale
        // (magnitudes under 2^-100: 127 / m might be infinite)
        const float lift = m < 0x1p-100f ? 0x1p96f : 1.0f, ml = m * lift;
        const float inv = ml > 0.0f ? 127.0f / ml : 0.0f;
        if (t == 0) a.code_scales[row] = fine ? scale : NAN;
#pragma unroll
        for (int i = 0; i < E; i++) {
            const int p = t + i * T;
            if (p >= pieces) continue;
            u32x2n o = {0u, 0u};
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const float q = fminf(fmaxf(__builtin_rintf(r[i][e] * lift * inv), -127.0f), 127.0f);
                o[e / 4] |= (uint32_t)((int)(fine ? q : 0.0f) & 0xFF) << (8 * (e % 4));
            }
            *(u32x2n*)(a.codes + row * a.code_stride + 8 * p) = o;
        }
    }
}

// As many threads as a row has pieces, up to 512: a row's loads are one round trip and its
// waves' sums are short (8192 rows of 4096 with the first norm, 268 MB, 48.9 us; 52.4 with
// 256 threads and two pieces each; rows of 512 8.4, 12.1 with 256 threads).  Rows of more
// than 512 pieces take 1024 threads while two workgroups a CU hold them all (1 row of 8192
// 3.5 us, 4.0 with 512 threads), and 512 with two pieces each beyond (8192 rows 107 us, 115
// with 1024).
template <int T, int E>
hipError_t norms_go(const BlockNormsArgs& a, hipStream_t st) {
    hipLaunchKernelGGL((block_norms_kernel<T, E>), dim3((unsigned)a.rows), dim3(T), 0, st, a);
    return hipGetLastError();
}
}  // namespace

hipError_t block_norms_launch(const BlockNormsArgs& a, hipStream_t st) {
    const int pieces = a.hidden / 8;
    if (pieces <= 64)   return norms_go<64, 1>(a, st);
    if (pieces <= 128)  return norms_go<128, 1>(a, st);
    if (pieces <= 256)  return norms_go<256, 1>(a, st);
    if (pieces <= 384)  return norms_go<384, 1>(a, st);
    if (pieces <= 512)  return norms_go<512, 1>(a, st);
    if (pieces <= 1024) return a.rows <= 512 ? norms_go<1024, 1>(a, st) : norms_go<512, 2>(a, st);
    if (pieces <= 2048) return norms_go<1024, 2>(a, st);
    return norms_go<1024, 4>(a, st);
}

}  // namespace jllm_hip
