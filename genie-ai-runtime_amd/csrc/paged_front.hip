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
// frequency is a 64-bit fraction of a turn and the angle a 32-bit one, within 2^-31
// turns at every position (theta >= 1): 2^-33.5 from the frequency's rounding times
// a position below 2^31, 2^-32 from the bits that are cut off.
//
// Measured (32 / 8 heads x 128): 2048 tokens into INT8 pages 11.5 us (46 MB, 4.0
// TB/s; half of it instructions), 8000 into fp16 pages 43.6 us (4.5 TB/s); 64 tokens
// 3.8 us, one 3.5 us, where the chain of scalar and vector loads is all there is.
#include "kq_common.h"
#include "serving.h"
#include <math.h>

namespace jllm_hip {

typedef uint32_t u32x2f __attribute__((ext_vector_type(2)));

namespace {
typedef unsigned __int128 u128;
// the upper half of the 256-bit product, short by less than 4
u128 mul_hi(u128 a, u128 b) {
    const uint64_t a1 = (uint64_t)(a >> 64), a0 = (uint64_t)a, b1 = (uint64_t)(b >> 64), b0 = (uint64_t)b;
    return (u128)a1 * b1 + (((u128)a1 * b0) >> 64) + (((u128)a0 * b1) >> 64);
}
}  // namespace

// f[i] = theta^(-2 i / hd) / 2 pi, each from one before it in 128-bit fixed point and
// rounded to 64 bits at the end: off by less than 0.51 of 2^-64 turns for theta from 1 to
// 2^64, 0.7 above (64-bit products added up to 30 of 2^-64).  The host's time for 64 of
// them is 0.2 us.
void rope_turns(RopeTurns& rt, int head_dim, double theta) {
    const int n = head_dim / 2;
    if (theta > 1.0) {
        u128 r;                                              // theta^(-1 / n)
        if (theta < 18446744073709551616.0) {
            // A Newton step on r^n theta = 1 from a double: the error, some 2^-50, is squared
            // (and times n / 2).  theta = m 2^e, m a whole number of 24 bits (it is a float),
            // so r^n m less 2^(128 - e) is 2^(128 - e) times the relative error of r^n,
            // and fits a signed word.
            const double ratio = pow(theta, -1.0 / n);
            r = (u128)(uint64_t)ldexp(ratio, 64) << 64;
            int e;
            const uint32_t m = (uint32_t)ldexp(frexp(theta, &e), 24);
            e -= 24;
            u128 power = ~(u128)0, x = r;
            for (int k = n; k > 0; k >>= 1, x = mul_hi(x, x))
                if (k & 1) power = mul_hi(power, x);
            const u128 one = e > 0 ? (u128)1 << (128 - e) : 0;       // modulo 2^128
            const __int128 above = (__int128)(power * m - one);
            r -= (u128)(__int128)(ldexp((double)above, e) * ratio / n);
        } else {
            // (r^n has too few bits here, but the powers of r fall so fast that 64 of r do)
            r = (u128)(uint64_t)ldexpl(powl((long double)theta, -1.0L / n), 64) << 64;
        }
        // four chains, so that a product need not wait for the one before it (n is a multiple of 4)
        const u128 r2 = mul_hi(r, r), r4 = mul_hi(r2, r2);
        u128 f[4] = {((u128)0x28BE60DB9391054Aull << 64) | 0x7F09D5F47D4D3770ull};     // 2^128 / 2 pi
        f[1] = mul_hi(f[0], r);
        f[2] = mul_hi(f[0], r2);
        f[3] = mul_hi(f[1], r2);
        for (int i = 0; i < n; i += 4)
            for (int j = 0; j < 4; j++) {
                rt.f[i + j] = (uint64_t)((f[j] + ((u128)1 << 63)) >> 64);
                f[j] = mul_hi(f[j], r4);
            }
    } else {
        for (int i = 0; i < n; i++) {
            const long double turns = powl((long double)theta, -2.0L * i / head_dim) / 6.283185307179586476925286766559L;
            rt.f[i] = (uint64_t)ldexpl(turns - floorl(turns), 64);
        }
    }
    for (int i = n; i < ROPE_MAX_HALF; i++) rt.f[i] = 0;
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
    return u32x2f{h2_bits(half2_t{(_Float16)x[0], (_Float16)x[1]}), h2_bits(half2_t{(_Float16)x[2], (_Float16)x[3]})};
}
// the codes rint(x * inv), the product rounded first as the KV quantiser does
// (fp16_to_int8_kernel, convert.cu:26-69): adding 1.5 * 2^23 leaves the code in the
// lowest byte
__device__ __forceinline__ uint32_t code4(const float* x, float inv) {
#pragma clang fp contract(off)
    uint32_t b[4];
#pragma unroll
    for (int j = 0; j < 4; j++) b[j] = __builtin_bit_cast(uint32_t, x[j] * inv + 12582912.0f);
    const uint32_t lo = __builtin_amdgcn_perm(b[1], b[0], 0x0c0c0400u), hi = __builtin_amdgcn_perm(b[3], b[2], 0x0c0c0400u);
    return lo | (hi << 16);
}

// sine and cosine of 2 pi turn 2^-32.  The nearest quarter turn goes into a swap and two
// signs; what is left, |r| <= pi / 4, into the Taylor polynomials up to r^9 and r^8
// (next terms: 2e-9 and 3e-8).  A third of the instructions of sincospif.
__device__ __forceinline__ void sincos_turn(uint32_t turn, float& s, float& c) {
    const uint32_t quarter = (turn + 0x20000000u) >> 30;
    const float r = (float)(int32_t)(turn - (quarter << 30)) * 1.46291807926715968e-9f;     // 2 pi 2^-32
    const float r2 = r * r;
    const float ps = __builtin_fmaf(__builtin_fmaf(__builtin_fmaf(__builtin_fmaf(r2, 1.0f / 362880.0f, -1.0f / 5040.0f), r2,
                                    1.0f / 120.0f), r2, -1.0f / 6.0f), r2 * r, r);
    const float pc = __builtin_fmaf(__builtin_fmaf(__builtin_fmaf(__builtin_fmaf(r2, 1.0f / 40320.0f, -1.0f / 720.0f), r2,
                                    1.0f / 24.0f), r2, -0.5f), r2, 1.0f);
    const bool swap = quarter & 1u;
    s = swap ? pc : ps;
    c = swap ? ps : pc;
    // quarters 2, 3 turn the sine's sign, 1, 2 the cosine's
    s = __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, s) ^ ((quarter & 2u) << 30));
    c = __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, c) ^ (((quarter + 1u) & 2u) << 30));
}

typedef float f32x4w __attribute__((ext_vector_type(4), aligned(4)));
typedef uint16_t u16x4w __attribute__((ext_vector_type(4), aligned(2)));

// the lane's eight norm weights
__device__ __forceinline__ void load_weights(const void* p, bool fp32, int e0, int e1, float (&w)[8]) {
    if (fp32) {
        const f32x4w x = *(const f32x4w*)((const float*)p + e0), y = *(const f32x4w*)((const float*)p + e1);
#pragma unroll
        for (int j = 0; j < 4; j++) { w[j] = x[j]; w[4 + j] = y[j]; }
    } else {
        const u16x4w x = *(const u16x4w*)((const uint16_t*)p + e0), y = *(const u16x4w*)((const uint16_t*)p + e1);
#pragma unroll
        for (int j = 0; j < 4; j++) { w[j] = f16_bits_to_f32(x[j]); w[4 + j] = f16_bits_to_f32(y[j]); }
    }
}

// One wave takes 64 / GL rows (heads) of one token at a time, GL lanes a row, 8 values
// a lane: values e0 + [0, 4) and e1 + [0, 4) with, in split pairs (neox), e0 = 4 gl
// and e1 = e0 + hd / 2, in interleaved pairs e0 = 8 gl and e1 = e0 + 4; either way
// the lane's four pairs are its own and have the frequencies 4 gl + [0, 4).  A wave
// goes through iters groups of rows of its token, with the next group's values on
// the way.  The kernel is bound by its instructions, not by the bytes, so what the
// groups share is computed once: sines, cosines, and their products with the norm
// weights, which a new kind of rows (q, then k) or a group of both renews.
template <int GL, bool INT8, bool NEOX>
__global__ __launch_bounds__(256) void paged_front_kernel(PagedFrontArgs a, int groups, int iters, int per) {
    constexpr int RG = 64 / GL;                        // rows a wave takes at once
    const int hd = a.head_dim, R = a.n_heads + 2 * a.n_kv, QK = a.n_heads + a.n_kv;
    const unsigned tb = blockIdx.x / (unsigned)per;    // the block's four waves: four tokens, the same groups
    const int64_t t = (int64_t)tb * 4 + __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    if (t >= a.N) return;
    const int g0 = (int)(blockIdx.x - tb * per) * iters, g1 = min(g0 + iters, groups);
    const int l = threadIdx.x & 63, sub = l / GL, gl = l % GL;
    const int e0 = NEOX ? 4 * gl : 8 * gl, e1 = NEOX ? e0 + hd / 2 : e0 + 4;
    const bool in_row = 8 * gl < hd;
    const float inv_hd = 1.0f / (float)hd;
    const uint64_t qr = (uint64_t)(a.q + t * a.q_stride), kr0 = (uint64_t)(a.k + t * a.k_stride),
                   vr0 = (uint64_t)(a.v + t * a.v_stride);

    u32x2f ra = {0u, 0u}, rb = {0u, 0u};
    auto load = [&](int g) {
        const int r = g * RG + sub;
        if (!in_row || r >= R) return;
        const int kr = r - a.n_heads, vr = kr - a.n_kv;
        typedef const __attribute__((address_space(1))) u32x2f* global_t;
        uint64_t src = qr + 2 * (uint64_t)(r * hd);
        if (kr >= 0) src = kr0 + 2 * (uint64_t)(kr * hd);
        if (vr >= 0) src = vr0 + 2 * (uint64_t)(vr * hd);
        ra = *(global_t)(src + 2 * e0);
        rb = *(global_t)(src + 2 * e1);
    };
    const int slot = a.slots[t], pos = a.positions[t];
    load(g0);
    float wq[8], wk[8];
#pragma unroll
    for (int j = 0; j < 8; j++) wq[j] = wk[j] = 1.0f;
    if (a.q_norm && in_row) {
        load_weights(a.q_norm, a.norm_fp32 != 0, e0, e1, wq);
        load_weights(a.k_norm, a.norm_fp32 != 0, e0, e1, wk);
    }
    uint64_t fr[4];
#pragma unroll
    for (int j = 0; j < 4; j++) fr[j] = a.rt.f[4 * gl + j];
    __builtin_amdgcn_sched_barrier(0);
    if (slot < 0 || slot >= a.n_slots) return;         // padding: nothing of this token is written

    float sn[4], cs[4];
#pragma unroll
    for (int j = 0; j < 4; j++) {
        // bits 32 to 63 of fr * pos; a negative position counts 2^32 too much above
        const uint32_t f0 = (uint32_t)fr[j], f1 = (uint32_t)(fr[j] >> 32);
        sincos_turn(__umulhi(f0, (uint32_t)pos) + f1 * (uint32_t)pos - (pos < 0 ? f0 : 0u), sn[j], cs[j]);
    }
    // pair (p, q) -> (p c0 - q s0, p s1 + q c1)
    float c0[4] = {}, s0[4] = {}, c1[4] = {}, s1[4] = {};
    int have = -1;                                     // kind of the rows that these are for: 0 q, 1 k, 2 a mixture
    for (int g = g0; g < g1; g++) {
        const int r = g * RG + sub, kr = r - a.n_heads, vr = kr - a.n_kv;
        const bool act = in_row && r < R;
        const int first = g * RG, last = first + RG - 1;
        if (first < QK) {
            const int kind = last < a.n_heads ? 0 : (first >= a.n_heads ? 1 : 2);
            if (kind != have) {
                have = kind;
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const int p = NEOX ? j : 2 * j, q = NEOX ? 4 + j : 2 * j + 1;
                    const float wp = kr < 0 ? wq[p] : wk[p], wz = kr < 0 ? wq[q] : wk[q];
                    c0[j] = cs[j] * wp; s0[j] = sn[j] * wz; s1[j] = sn[j] * wp; c1[j] = cs[j] * wz;
                }
            }
        }
        float x[8];
#pragma unroll
        for (int j = 0; j < 2; j++) {
            x[2 * j] = f16_bits_to_f32(ra[j] & 0xFFFFu); x[2 * j + 1] = f16_bits_to_f32(ra[j] >> 16);
            x[4 + 2 * j] = f16_bits_to_f32(rb[j] & 0xFFFFu); x[5 + 2 * j] = f16_bits_to_f32(rb[j] >> 16);
        }
        if (g + 1 < g1) load(g + 1);
        if (first < QK) {
            float rrms = 1.0f;
            if (a.q_norm) {
                float ss = 0.0f;
#pragma unroll
                for (int j = 0; j < 8; j++) ss += x[j] * x[j];
                rrms = __builtin_amdgcn_rsqf(group_sum_dpp<GL>(ss) * inv_hd + a.eps);     // 1 ulp
            }
            if (vr < 0) {
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    float &p = x[NEOX ? j : 2 * j], &q = x[NEOX ? 4 + j : 2 * j + 1];
                    const float y = p * rrms, z = q * rrms;
                    p = y * c0[j] - z * s0[j];
                    q = y * s1[j] + z * c1[j];
                }
            }
        }
        if (kr < 0 && act) {
            uint16_t* o = a.q_out + t * a.q_out_stride + r * hd;
            *(u32x2f*)(o + e0) = pack4(x);
            *(u32x2f*)(o + e1) = pack4(x + 4);
        }
        if (last < a.n_heads) continue;                // only q heads in this group
        const int64_t row = (int64_t)slot * a.n_kv + (vr < 0 ? kr : vr);
        void* pages = vr < 0 ? a.k_pages : a.v_pages;
        if (INT8) {
            uint32_t mb = 0;
#pragma unroll
            for (int j = 0; j < 8; j++) mb = max(mb, __builtin_bit_cast(uint32_t, x[j]) & 0x7FFFFFFFu);
            mb = group_max_dpp<GL>(mb);
            if (kr >= 0 && act) {
                const float mx = __builtin_bit_cast(float, mb);
                const bool fine = mb < 0x7F800000u;    // a row with a NaN or an infinity reads as NaN
                const bool some = fine && mx > 1e-35f; // below: 127 / mx overflows; the row is zero
                const float inv = 127.0f / mx;
                int8_t* o = (int8_t*)pages + row * a.cache_head_dim;
                *(uint32_t*)(o + e0) = some ? code4(x, inv) : 0u;
                *(uint32_t*)(o + e1) = some ? code4(x + 4, inv) : 0u;
                if (gl == 0) (vr < 0 ? a.k_scales : a.v_scales)[row] = fine ? mx / 127.0f : __builtin_nanf("");
            }
        } else if (kr >= 0 && act) {
            uint16_t* o = (uint16_t*)pages + row * a.cache_head_dim;
            *(u32x2f*)(o + e0) = pack4(x);
            *(u32x2f*)(o + e1) = pack4(x + 4);
        }
    }
}

namespace {
int lanes_of(int hd) { return hd <= 32 ? 4 : (hd <= 64 ? 8 : 16); }
int groups_of(const PagedFrontArgs& a) {
    const int rg = 64 / lanes_of(a.head_dim);
    return (a.n_heads + 2 * a.n_kv + rg - 1) / rg;
}
// Groups of rows per wave: one while the waves do not fill the card, more (up to
// all of a token's) beyond that.
int iters_of(const PagedFrontArgs& a) {
    const int groups = groups_of(a);
    const int64_t it = (int64_t)a.N * groups / 4096;
    return it < 1 ? 1 : (it > groups ? groups : (int)it);
}
}  // namespace

int64_t paged_front_blocks(const PagedFrontArgs& a) {
    const int groups = groups_of(a), iters = iters_of(a);
    return ((int64_t)a.N + 3) / 4 * ((groups + iters - 1) / iters);
}

template <int GL, bool INT8>
static void front_go(const PagedFrontArgs& a, hipStream_t st) {
    const dim3 grid((unsigned)paged_front_blocks(a));
    const int groups = groups_of(a), iters = iters_of(a), per = (groups + iters - 1) / iters;
    if (a.neox) hipLaunchKernelGGL((paged_front_kernel<GL, INT8, true>), grid, dim3(256), 0, st, a, groups, iters, per);
    else        hipLaunchKernelGGL((paged_front_kernel<GL, INT8, false>), grid, dim3(256), 0, st, a, groups, iters, per);
}

hipError_t paged_front_launch(const PagedFrontArgs& a, hipStream_t st) {
    switch (lanes_of(a.head_dim) + (a.kv_int8 ? 1 : 0)) {
    case 4:  front_go<4, false>(a, st); break;
    case 5:  front_go<4, true>(a, st); break;
    case 8:  front_go<8, false>(a, st); break;
    case 9:  front_go<8, true>(a, st); break;
    case 16: front_go<16, false>(a, st); break;
    default: front_go<16, true>(a, st); break;
    }
    return hipGetLastError();
}

}  // namespace jllm_hip
