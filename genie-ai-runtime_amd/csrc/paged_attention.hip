// paged_attention.hip -- decode attention of a batch of query rows, each over the
// pages of its own sequence, gfx950.
//
//   s_t = scale * ks_t * (q . k_t),  out = sum_t e^(s_t - m) vs_t v_t / sum_t e^(s_t - m)
//
// over the keys t of the row: [max(0, len - window), len).  Key t lies in slot
// t % page_size of page table[row][t / page_size].
//
// One pass over K and V, all query heads of a KV head together.  A wave takes
// tiles of 32 keys, two blocks of 16 (a page holds whole blocks, so a block is one
// base address).  With lane (li = l & 15, lg = l >> 4) of v_mfma_f32_16x16x32_f16:
//   S^T = K q^T   rows = keys, columns = heads: the lane gets the scores of head li
//                 and keys 4 lg + [0, 4) of each block;
//   O^T = V^T P^T those eight keys are just what the lane's B operand wants, so P
//                 goes from the softmax into the matrix cores without leaving its
//                 registers, and maximum, sum and rescale factor are the lane's own
//                 head's.  V^T's A operand needs one d of eight keys: the lane loads
//                 hd / 16 neighbouring d of its eight keys and one byte permute per
//                 two values transposes them (and, for int8, converts them: a code + 128
//                 with a zero byte above it is the subnormal half (code + 128) 2^-24;
//                 the 128 leaves through the accumulator's start value for K, and through
//                 the sum of the weights for V).
// Sums, maxima and accumulators are fp32.  The weights are rounded to fp16 for
// the matrix cores (2^-12 of a weight, less than the output's own rounding),
// times 2^14 so that they become subnormal only below 2^-28 of the largest.
// With int8 the V scales go into the exponent, e^(s_t - m) vs_t = 2^(s'_t + log2
// vs_t), with a maximum of their own: no scale can overflow or swamp the others.
#include "attn_common.h"
#include "serving.h"

namespace jllm_hip {

typedef float f32x4p __attribute__((ext_vector_type(4)));

constexpr int PA_TILE = 32;            // keys a wave takes at once
constexpr int PA_BLOCK = 16;           // keys behind one base address
constexpr int PA_MAX_CHUNK = 1024;     // 64 blocks: one lane each
constexpr int PA_WAVES = 4;
constexpr float PA_LIFT = 14.0f;       // log2 of the factor on fp16 weights
constexpr float PA_LOG2E = 1.44269504088896340736f;

bool attn_splitk_enabled();

// maximum / sum over the four 16-lane rows, in every lane
__device__ __forceinline__ float rows_op(float v, bool sum) {
    const unsigned u = __builtin_bit_cast(unsigned, v);
    const auto s = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    const float a = __builtin_bit_cast(float, (unsigned)s[0]), b = __builtin_bit_cast(float, (unsigned)s[1]);
    float lo, hi;
    wave_halves(sum ? a + b : fmaxf(a, b), lo, hi);
    return sum ? lo + hi : fmaxf(lo, hi);
}
// lane N of each 16-lane row, in the whole row
template <int N>
__device__ __forceinline__ float row_bcast(float v) { return dpp_mov_f<0x150 + N>(v); }

// four int8 codes -> (code + 128) 2^-24 as four halves
__device__ __forceinline__ u32x2a codes_to_h4(uint32_t w) {
    const uint32_t u = w ^ 0x80808080u;
    return u32x2a{__builtin_amdgcn_perm(u, u, 0x0c010c00u), __builtin_amdgcn_perm(u, u, 0x0c030c02u)};
}

// the weights' exponent base: a row without a finite score yet has base 0
__device__ __forceinline__ float base_of(float m) { return m == -INFINITY ? 0.0f : m; }

struct PagedSplit { int chunk, splits; };

template <bool INT8, int HD>
__global__ __launch_bounds__(64 * PA_WAVES)
void paged_attn_kernel(PagedAttnArgs a, int chunk, int S) {
    constexpr int EB = INT8 ? 1 : 2;
    constexpr int NST = HD / 32;                       // Q.K^T steps
    constexpr int KC = INT8 ? HD / 64 : HD / 32;       // 16-byte pieces of a K row per lane
    constexpr bool KT = INT8 && HD % 64 != 0;          // and an 8-byte one
    constexpr int NT = HD / 16;                        // 16-wide d tiles of O
    constexpr int V0 = HD == 96 ? 4 : NT;              // neighbouring d per lane, first part ...
    constexpr int V1 = NT - V0;                        // ... and second (from d = 64)
    constexpr int W0 = (V0 * EB + 3) / 4, W1 = (V1 * EB + 3) / 4, VW = W0 + W1;   // in words
    extern __shared__ __attribute__((aligned(16))) float smem[];

    const int kvh = blockIdx.x, split = blockIdx.y, b = blockIdx.z;
    const int wv = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int l = (int)threadIdx.x & 63, li = l & 15, lg = l >> 4;
    const int G = a.n_heads / a.n_kv;
    int len = a.lens[b];
    len = len < 0 ? 0 : (len > a.max_seq ? a.max_seq : len);
    const int lo = a.window > 0 && len > a.window ? len - a.window : 0;
    const int kv0 = (lo & ~(PA_BLOCK - 1)) + split * chunk, kv1 = min(kv0 + chunk, len);
    uint16_t* out = a.out + ((int64_t)b * a.n_heads + kvh * G) * HD;
    if (kv0 >= kv1) {
        // behind the row's end; an empty row is written here unless the join does it
        if (S == 1)
            for (int i = (int)threadIdx.x; i < G * HD; i += 64 * PA_WAVES) out[i] = 0;
        return;
    }
    // lane j: slot of the first key of block j, and which blocks are there
    const int nblk = (kv1 - kv0 + PA_BLOCK - 1) / PA_BLOCK;
    const int bpos = kv0 + PA_BLOCK * min(l, nblk - 1);
    const int page = a.table[b * a.table_stride + (bpos >> a.page_shift)];
    const uint64_t there = __builtin_amdgcn_ballot_w64(l < nblk && (unsigned)page < (unsigned)a.n_pages);
    const int slot0 = (page << a.page_shift) + (bpos & ((1 << a.page_shift) - 1));

    const uint32_t row = (uint32_t)a.n_kv * a.cache_head_dim * EB;      // bytes
    const int64_t hoff = (int64_t)kvh * a.cache_head_dim * EB;

    // this wave's tiles wv, wv + W, ... of which a block is there: bit 2 i
    uint64_t todo = (there | (there >> 1)) & ((~(uint64_t)0 / ((1 << 2 * PA_WAVES) - 1)) << (2 * wv));
    auto next_tile = [&]() {
        const int i = todo ? __builtin_ctzll(todo) / 2 : -1;
        todo &= todo - 1;
        return i;
    };
    auto bases = [&](int i, int& s0, int& s1) {        // slots of a tile's blocks; a missing one takes the other's
        const int x = __builtin_amdgcn_readlane(slot0, 2 * i), y = __builtin_amdgcn_readlane(slot0, 2 * i + 1);
        s0 = (there >> (2 * i)) & 1 ? x : y;
        s1 = (there >> (2 * i + 1)) & 1 ? y : x;
    };

    // (zeroed: where a path leaves such registers undefined, this compiler has
    // given words of a loaded row to other values while they were still needed)
    u32x4a rk[2][KC > 0 ? KC : 1] = {};
    u32x2a rt[2] = {};
    uint32_t rv[8][VW] = {};
    float rs = 1.0f;
    auto load_k = [&](int s0, int s1) {
#pragma unroll
        for (int q = 0; q < 2; q++) {
            const uint8_t* p = (const uint8_t*)a.k + (int64_t)(q ? s1 : s0) * row + hoff;
            const uint32_t o = (uint32_t)li * row;
#pragma unroll
            for (int c = 0; c < KC; c++) rk[q][c] = *(const u32x4a*)(p + (o + 64 * c + 16 * lg));
            if (KT) rt[q] = *(const u32x2a*)(p + (o + 64 * KC + 8 * lg));
        }
        if (INT8) {
            // lane li: K (li < 8) or V scale of key 4 lg + li % 4 of block (li >> 2) & 1
            const float* p = li < 8 ? a.ks : a.vs;
            const int64_t s = (li & 4 ? s1 : s0) + 4 * lg + (li & 3);
            rs = p ? p[s * a.n_kv + kvh] : 1.0f;
        }
    };
    auto load_v = [&](int s0, int s1) {
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const uint8_t* p = (const uint8_t*)a.v + (int64_t)(e < 4 ? s0 : s1) * row + hoff;
            const uint32_t o = (uint32_t)(4 * lg + (e & 3)) * row;
            const uint8_t* x = p + (o + V0 * EB * li);
            if (V0 * EB == 16) { const u32x4a w = *(const u32x4a*)x; rv[e][0] = w.x; rv[e][1 % VW] = w.y; rv[e][2 % VW] = w.z; rv[e][3 % VW] = w.w; }
            else if (V0 * EB == 8) { const u32x2a w = *(const u32x2a*)x; rv[e][0] = w.x; rv[e][1 % VW] = w.y; }
            else if (V0 * EB == 4) rv[e][0] = *(const uint32_t*)x;
            else rv[e][0] = *(const uint16_t*)x;
            if (V1 > 0) {
                const uint8_t* y = p + (o + 64 * EB + V1 * EB * li);
                rv[e][VW - 1] = V1 * EB == 4 ? *(const uint32_t*)y : *(const uint16_t*)y;
            }
        }
    };

    int i = next_tile();
    if (i >= 0) {
        int s0, s1;
        bases(i, s0, s1);
        load_k(s0, s1);
        load_v(s0, s1);
    }
    __builtin_amdgcn_sched_barrier(0);

    // q operand: head li (columns past the last head stay zero), the d that K's pieces bring
    h8 qb[NST];
#pragma unroll
    for (int st = 0; st < NST; st++) {
        const int d = !INT8 ? 32 * st + 8 * lg : (KT && st == NST - 1 ? 64 * KC + 8 * lg : 64 * (st / 2) + 16 * lg + 8 * (st % 2));
        const u32x4a w = *(const u32x4a*)(a.q + b * a.q_stride + (int64_t)(kvh * G + min(li, G - 1)) * HD + d);
        qb[st] = __builtin_bit_cast(h8, li < G ? w : u32x4a{0u, 0u, 0u, 0u});
    }
    // - sum_d 128 2^-24 q_d: takes the codes' offset out of every score
    f32x4p start = {};
    if (INT8) {
        const h8 off = __builtin_bit_cast(h8, u32x4a{0x00800080u, 0x00800080u, 0x00800080u, 0x00800080u});
#pragma unroll
        for (int st = 0; st < NST; st++) start = __builtin_amdgcn_mfma_f32_16x16x32_f16(off, qb[st], start, 0, 0, 0);
        start = -start;
    }
    const float f0 = a.scale * PA_LOG2E, f8 = f0 * 16777216.0f;

    float m = -INFINITY, L = 0.0f, M = -INFINITY;      // maximum, this lane's sum; maximum with the V scales
    f32x4p acc[NT], wsum = {};
#pragma unroll
    for (int j = 0; j < NT; j++) acc[j] = f32x4p{};
    const h8 ones = __builtin_bit_cast(h8, u32x4a{0x3C003C00u, 0x3C003C00u, 0x3C003C00u, 0x3C003C00u});

    while (i >= 0) {
        const int p0 = kv0 + PA_TILE * i;
        const bool v0 = (there >> (2 * i)) & 1, v1 = (there >> (2 * i + 1)) & 1;
        // 1. scores of the tile, in units of log2
        float s[8];
#pragma unroll
        for (int q = 0; q < 2; q++) {
            f32x4p c = start;
#pragma unroll
            for (int st = 0; st < NST; st++) {
                h8 kb;
                if (!INT8) {
                    kb = __builtin_bit_cast(h8, rk[q][st % (KC > 0 ? KC : 1)]);
                } else {
                    const bool tail = KT && st == NST - 1;
                    const u32x4a w = rk[q][tail ? 0 : (st / 2) % (KC > 0 ? KC : 1)];
                    const u32x2a x = codes_to_h4(tail ? rt[q].x : (st % 2 ? w.z : w.x));
                    const u32x2a y = codes_to_h4(tail ? rt[q].y : (st % 2 ? w.w : w.y));
                    kb = __builtin_bit_cast(h8, u32x4a{x.x, x.y, y.x, y.y});
                }
                c = __builtin_amdgcn_mfma_f32_16x16x32_f16(kb, qb[st], c, 0, 0, 0);
            }
#pragma unroll
            for (int r = 0; r < 4; r++) s[4 * q + r] = c[r];
        }
        // lanes li < 8: the K factor, li >= 8: log2 of the V scale
        const float sraw = rs;
        const int in = next_tile();
        int n0 = 0, n1 = 0;
        if (in >= 0) {
            bases(in, n0, n1);
            load_k(n0, n1);
        }
        __builtin_amdgcn_sched_barrier(0);
        float sv = 0.0f;
        if (INT8) {
            sv = li < 8 ? sraw * f8 : __builtin_amdgcn_logf(fabsf(sraw));
            s[0] *= row_bcast<0>(sv); s[1] *= row_bcast<1>(sv); s[2] *= row_bcast<2>(sv); s[3] *= row_bcast<3>(sv);
            s[4] *= row_bcast<4>(sv); s[5] *= row_bcast<5>(sv); s[6] *= row_bcast<6>(sv); s[7] *= row_bcast<7>(sv);
        } else {
#pragma unroll
            for (int e = 0; e < 8; e++) s[e] *= f0;
        }
        const bool full = v0 && v1 && p0 >= lo && p0 + PA_TILE <= kv1;
        uint32_t live = 0xFFu;                         // bit e: the lane's key e counts
        if (!full) {
            live = 0;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const int t = p0 + PA_BLOCK * (e >> 2) + 4 * lg + (e & 3);
                if ((e < 4 ? v0 : v1) && t >= lo && t < kv1) live |= 1u << e;
            }
#pragma unroll
            for (int e = 0; e < 8; e++) s[e] = live >> e & 1 ? s[e] : -INFINITY;
        }
        // 2. softmax
        float mx = s[0];
#pragma unroll
        for (int e = 1; e < 8; e++) mx = fmaxf(mx, s[e]);
        const float mn = fmaxf(m, rows_op(mx, false)), mb = base_of(mn);
        float corr = __builtin_amdgcn_exp2f(m - mb);
        m = mn;
        float p[8], ps = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; e++) {
            p[e] = __builtin_amdgcn_exp2f(s[e] - (INT8 ? mb : mb - PA_LIFT));
            ps += p[e];
        }
        L = L * corr + ps;
        if (INT8) {
            // the weights times the V scales, under a maximum of their own
            float t[8];
            t[0] = s[0] + row_bcast<8>(sv); t[1] = s[1] + row_bcast<9>(sv); t[2] = s[2] + row_bcast<10>(sv); t[3] = s[3] + row_bcast<11>(sv);
            t[4] = s[4] + row_bcast<12>(sv); t[5] = s[5] + row_bcast<13>(sv); t[6] = s[6] + row_bcast<14>(sv); t[7] = s[7] + row_bcast<15>(sv);
            if (!full) {
#pragma unroll
                for (int e = 0; e < 8; e++) t[e] = live >> e & 1 ? t[e] : -INFINITY;
            }
            float tx = t[0];
#pragma unroll
            for (int e = 1; e < 8; e++) tx = fmaxf(tx, t[e]);
            const float Mn = fmaxf(M, rows_op(tx, false)), Mb = base_of(Mn);
            corr = __builtin_amdgcn_exp2f(M - Mb);
            M = Mn;
#pragma unroll
            for (int e = 0; e < 8; e++) p[e] = __builtin_amdgcn_exp2f(t[e] - (Mb - PA_LIFT));
            // a negative V scale: its sign back onto the weight (no quantiser here writes one)
            if (__builtin_amdgcn_ballot_w64(li >= 8 && sraw < 0.0f)) {
                p[0] = __builtin_copysignf(p[0], row_bcast<8>(sraw)); p[1] = __builtin_copysignf(p[1], row_bcast<9>(sraw));
                p[2] = __builtin_copysignf(p[2], row_bcast<10>(sraw)); p[3] = __builtin_copysignf(p[3], row_bcast<11>(sraw));
                p[4] = __builtin_copysignf(p[4], row_bcast<12>(sraw)); p[5] = __builtin_copysignf(p[5], row_bcast<13>(sraw));
                p[6] = __builtin_copysignf(p[6], row_bcast<14>(sraw)); p[7] = __builtin_copysignf(p[7], row_bcast<15>(sraw));
            }
        }
        // no head's maximum moved: every factor is 1
        if (__builtin_amdgcn_ballot_w64(corr != 1.0f)) {
#pragma unroll
            for (int j = 0; j < NT; j++) acc[j] *= corr;
            if (INT8) wsum *= corr;
        }
        h8 pb;
#pragma unroll
        for (int e = 0; e < 8; e++) pb[e] = (_Float16)p[e];
        // 3. O^T += V^T P^T
        if (!INT8 && !full) {                          // what a slot without a key holds may be NaN
#pragma unroll
            for (int e = 0; e < 8; e++)
#pragma unroll
                for (int w = 0; w < VW; w++) rv[e][w] = live >> e & 1 ? rv[e][w] : 0u;
        }
        if (INT8) {
#pragma unroll
            for (int e = 0; e < 8; e++)
#pragma unroll
                for (int w = 0; w < VW; w++) rv[e][w] ^= 0x80808080u;
        }
#pragma unroll
        for (int j = 0; j < NT; j++) {
            const int jj = j < V0 ? j : j - V0;
            const int w = (j < V0 ? 0 : W0) + jj * EB / 4, at = jj % (4 / EB);
            const uint32_t sel = INT8 ? 0x0c040c00u + 0x00010001u * at : (at ? 0x07060302u : 0x05040100u);
            u32x4a va;
#pragma unroll
            for (int e = 0; e < 4; e++) va[e] = __builtin_amdgcn_perm(rv[2 * e + 1][w], rv[2 * e][w], sel);
            acc[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, va), pb, acc[j], 0, 0, 0);
        }
        if (INT8) wsum = __builtin_amdgcn_mfma_f32_16x16x32_f16(ones, pb, wsum, 0, 0, 0);
        __builtin_amdgcn_sched_barrier(0);
        if (in >= 0) load_v(n0, n1);
        i = in;
    }

    // the wave's state: m, l, numerators; acc[j][r] is d = V0 (4 lg + r) + j, or 64 + V1 (4 lg + r) + j - V0
    L = rows_op(L, true);
    if (INT8) {
        const float f = __builtin_amdgcn_exp2f(base_of(M) - base_of(m) - PA_LIFT);
#pragma unroll
        for (int j = 0; j < NT; j++)
#pragma unroll
            for (int r = 0; r < 4; r++) acc[j][r] = (acc[j][r] * 16777216.0f - 128.0f * wsum[0]) * f;
    }
    constexpr int LD = HD + 4;
    float* sO = smem + (size_t)wv * G * LD;
    float* sML = smem + (size_t)PA_WAVES * G * LD;     // m [W][16], l [W][16]
    if (li < G) {
#pragma unroll
        for (int j = 0; j < NT; j++)
#pragma unroll
            for (int r = 0; r < 4; r++)
                sO[li * LD + (j < V0 ? V0 * (4 * lg + r) + j : 64 + V1 * (4 * lg + r) + j - V0)] = acc[j][r];
    }
    if (l < 16) { sML[wv * 16 + l] = m; sML[(PA_WAVES + wv) * 16 + l] = L; }
    __syncthreads();
    // join of the waves in wave order
    for (int e = (int)threadIdx.x; e < G * HD; e += 64 * PA_WAVES) {
        const int h = e / HD, d = e % HD;
        float top = sML[h];
#pragma unroll
        for (int w = 1; w < PA_WAVES; w++) top = fmaxf(top, sML[w * 16 + h]);
        const float tb = base_of(top);
        float num = 0.0f, den = 0.0f;
#pragma unroll
        for (int w = 0; w < PA_WAVES; w++) {
            const float f = __builtin_amdgcn_exp2f(sML[w * 16 + h] - tb);
            num += f * smem[((size_t)w * G + h) * LD + d];
            den += f * sML[(PA_WAVES + w) * 16 + h];
        }
        if (S == 1) {
            // no key of finite score: zero; a NaN stays
            out[e] = f32_to_f16_bits(den == 0.0f ? 0.0f : num / den);
        } else {
            const int64_t at = ((int64_t)b * a.n_heads + kvh * G + h) * S + split;
            const int64_t n = (int64_t)a.B * a.n_heads * S;
            a.part[2 * n + at * HD + d] = num;
            if (d == 0) { a.part[at] = top; a.part[n + at] = den; }
        }
    }
}

// out = sum_s 2^(m_s - M) num_s / sum_s 2^(m_s - M) l_s over the splits that the
// row has, in a fixed order: wave w of the head's workgroup adds splits w, w + NW,
// ..., lane l d = 2 l and 2 l + 1; then the waves' sums in wave order.
template <int NW>
__global__ __launch_bounds__(64 * NW) void paged_join_kernel(PagedAttnArgs a, int chunk, int S) {
    __shared__ float sM[NW];
    __shared__ float sSum[NW][130];
    const int b = blockIdx.y, h = blockIdx.x, hd = a.head_dim;
    const int w = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), l = (int)threadIdx.x & 63;
    int len = a.lens[b];
    len = len < 0 ? 0 : (len > a.max_seq ? a.max_seq : len);
    const int lo = a.window > 0 && len > a.window ? len - a.window : 0;
    const int ns = (len - (lo & ~(PA_BLOCK - 1)) + chunk - 1) / chunk;
    const int64_t n = (int64_t)a.B * a.n_heads * S, at = ((int64_t)b * a.n_heads + h) * S;
    const float* pm = a.part + at;
    const float* pl = a.part + n + at;
    const float* pn = a.part + 2 * n + at * hd;
    float top = -INFINITY;
    for (int s = (int)threadIdx.x; s < ns; s += 64 * NW) top = fmaxf(top, pm[s]);
    top = wave_max(top);
    if (NW > 1) {
        if (l == 0) sM[w] = top;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < NW; i++) top = fmaxf(top, sM[i]);
    }
    const float tb = base_of(top);
    float den = 0.0f;
    float2 num = make_float2(0.0f, 0.0f);
    const int d2 = 2 * l < hd ? 2 * l : 0;
#pragma unroll 8
    for (int s = w; s < ns; s += NW) {
        const float f = __builtin_amdgcn_exp2f(pm[s] - tb);
        const float2 v = *(const float2*)(pn + (int64_t)s * hd + d2);
        den += f * pl[s];
        num.x += f * v.x;
        num.y += f * v.y;
    }
    if (NW > 1) {
        sSum[w][2 * l] = num.x;
        sSum[w][2 * l + 1] = num.y;
        if (l == 0) sSum[w][128] = den;
        __syncthreads();
        if (w > 0) return;
#pragma unroll
        for (int i = 1; i < NW; i++) {
            num.x += sSum[i][2 * l];
            num.y += sSum[i][2 * l + 1];
            den += sSum[i][128];
        }
    }
    if (2 * l < hd) {
        const float x = den == 0.0f ? 0.0f : num.x / den, y = den == 0.0f ? 0.0f : num.y / den;
        *(uint32_t*)(a.out + ((int64_t)b * a.n_heads + h) * hd + 2 * l) =
            (uint32_t)f32_to_f16_bits(x) | ((uint32_t)f32_to_f16_bits(y) << 16);
    }
}

namespace {
// Keys per workgroup: enough splits for 2048 workgroups when every row is as long
// as it can be, at least a tile per wave, at most one block per lane.
PagedSplit split_of(int B, int n_kv, int max_seq, int window) {
    int64_t span = max_seq;
    if (window > 0 && window + (int64_t)PA_BLOCK - 1 < span) span = window + (int64_t)PA_BLOCK - 1;
    PagedSplit p;
    if (span < 1) span = 1;
    const int64_t rows = (int64_t)(B > 0 ? B : 1) * n_kv;
    const int64_t want = (2048 + rows - 1) / rows;
    int64_t chunk = (span + want - 1) / want;
    chunk = (chunk + PA_TILE * PA_WAVES - 1) / (PA_TILE * PA_WAVES) * (PA_TILE * PA_WAVES);
    if (chunk > PA_MAX_CHUNK) chunk = PA_MAX_CHUNK;
    p.chunk = (int)chunk;
    p.splits = (int)((span + chunk - 1) / chunk);
    return p;
}
}  // namespace

int64_t paged_attn_workspace(int B, int n_heads, int n_kv, int head_dim, int max_seq, int window) {
    const PagedSplit p = split_of(B, n_kv, max_seq, window);
    if (p.splits == 1) return 0;
    return ((int64_t)B * n_heads * p.splits * (2 + head_dim) * 4 + 15) & ~(int64_t)15;
}

hipError_t paged_attn_launch(const PagedAttnArgs& a, bool kv_int8, hipStream_t st) {
    const PagedSplit p = split_of(a.B, a.n_kv, a.max_seq, a.window);
    const int G = a.n_heads / a.n_kv;
    const dim3 grid(a.n_kv, p.splits, a.B);
    const size_t lds = ((size_t)PA_WAVES * G * (a.head_dim + 4) + PA_WAVES * 32) * 4;
#define PAGED_CASE(HD)                                                                                                     \
    if (kv_int8) hipLaunchKernelGGL((paged_attn_kernel<true, HD>), grid, dim3(64 * PA_WAVES), lds, st, a, p.chunk, p.splits);  \
    else         hipLaunchKernelGGL((paged_attn_kernel<false, HD>), grid, dim3(64 * PA_WAVES), lds, st, a, p.chunk, p.splits);
    switch (a.head_dim) {
    case 32:  PAGED_CASE(32) break;
    case 64:  PAGED_CASE(64) break;
    case 96:  PAGED_CASE(96) break;
    case 128: PAGED_CASE(128) break;
    default: return hipErrorInvalidValue;
    }
#undef PAGED_CASE
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || p.splits == 1) return e;
    if (p.splits <= 16) hipLaunchKernelGGL((paged_join_kernel<1>), dim3(a.n_heads, a.B), dim3(64), 0, st, a, p.chunk, p.splits);
    else                hipLaunchKernelGGL((paged_join_kernel<8>), dim3(a.n_heads, a.B), dim3(512), 0, st, a, p.chunk, p.splits);
    return hipGetLastError();
}

}  // namespace jllm_hip
