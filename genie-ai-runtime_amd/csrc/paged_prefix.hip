// paged_prefix.hip -- decode attention of a batch over the keys that all its rows share,
// gfx950: the parts of every row's softmax that the shared prefix makes, which the
// attention over the rows' own keys (paged_attention.hip) then joins.
//
//   m = max s_t, l = sum e^(s_t - m), num = sum e^(s_t - m) vs_t v_t,  s_t = scale ks_t q . k_t
//
// over the keys t of a part of the prefix, for every query head of every row.  The prefix
// is read once for all rows: the query heads that share a KV head, of all rows together,
// are the columns of the matrix products, 16 to a group.  The products, the softmax and
// the roundings are those of paged_attention.hip (scores and weights in one lane's
// registers between the two products, weights in two fp16 parts, V scales in the weights'
// exponent); here a wave's keys meet NR column groups.
//
// Two forms.  Few columns (query heads of one KV head, of all rows): keys straight to
// registers, four waves; 8 rows over 16384 INT8 keys of 32 / 8 heads x 128 22 us, both
// launches, of which the prefix's 34 MB need 6.6.  More: keys through LDS, eight waves,
// so that up to 256 columns meet each key that is read; bound by the softmax's VALU
// instructions beside the matrix products (64 rows of 32 / 8 heads over 32768 fp16 keys 68
// us: VALU issue 52 %, matrix cores 39 %, 2.0 TB/s).
// A short prefix is a chain of latencies: 4 rows over 2048 INT8 keys 6.0 us, of which the
// length, the table and the first keys are 2, the instructions' own first reading much of
// the rest.
//
// Four waves are RW row waves (columns of their own) times KW key waves (keys of their
// own, joined in LDS at the end).  With a window a row sees the last of the prefix only:
// a key that one column sees and another does not is weighed 0 there, and where it holds
// an infinity or NaN in fp16 V, which 0 would turn into NaN, that value is taken out of
// the product and added to the columns that see it.
#include <type_traits>
#include "paged_common.h"
#include "prefix_window.h"

namespace jllm_hip {

namespace {

constexpr int PP_MAX_SPLITS = 256;

// columns per wave and wave grid for a batch: cols = B * heads per KV head
struct PrefixPlan { int nr, rw, lds, tiles, splits; };
PrefixPlan prefix_plan(int B, int n_heads, int n_kv, int max_prefix, int window, bool int8) {
    PrefixPlan p;
    const int64_t cols = (int64_t)(B > 0 ? B : 1) * (n_heads / n_kv);
    const int64_t span = window > 0 && window < max_prefix ? window : max_prefix;
    // keys through LDS: over 64 columns, and of fp16 keys over 32 where each of 256 workgroups
    // has 256 keys (12 rows of 32 / 8 heads over 8192 keys 21.7 us, 26.2 without; over 4096 18.5
    // and 17.8; INT8, 16384 keys 33.2 and 31.7: its conversions take longer with few columns)
    p.lds = cols > 64 || (cols > 32 && !int8 && span * n_kv >= 256 * 256);
    // (with a window the code for columns that do not see a key leaves no registers for two
    // groups: 16 rows of 16 / 4 heads x 128 15.3 us.  Of fp16 keys and head_dim 128 it spills
    // even so: 11 registers here, through LDS 4 with four row waves and 37, 52 bytes a lane,
    // with eight.  32 / 8 heads, the last 4096 of 8192 keys and a whole prefix of 4096: 16 rows
    // 27.0 and 22.0 us, 64 rows 41.4 and 37.0.)
    p.nr = p.lds || (cols > 16 && window == 0) ? 2 : 1;
    p.rw = p.lds ? (cols > 128 ? 8 : 4) : (cols > 16 * p.nr ? (cols > 32 * p.nr ? 4 : 2) : 1);
    const int per = 16 * p.nr * p.rw;
    p.tiles = (int)((cols + per - 1) / per);
    // parts: as many workgroups as the CUs hold, of at least a stage (48 rows over 1500 INT8 keys
    // 39.1 us, 40.6 with two stages; 64 over 32768 fp16 keys 90, 121 with half the workgroups),
    // or two tiles a wave
    const int unit = p.lds ? 2 * PA_TILE : 2 * PA_TILE * (PA_WAVES / p.rw), fill = 256;
    const int64_t units = (span + unit - 1) / unit, wgs = (int64_t)p.tiles * n_kv;
    int64_t s = (fill + wgs - 1) / wgs;
    if (s > units) s = units;
    if (s > PP_MAX_SPLITS) s = PP_MAX_SPLITS;
    p.splits = s < 1 ? 1 : (int)s;
    return p;
}

// 1 in each half that is not 0, in one operation
__device__ __forceinline__ uint32_t ones_of(uint32_t h) {
    uint32_t x;
    asm("v_pk_min_u16 %0, %1, 1 op_sel_hi:[1,0]" : "=v"(x) : "v"(h));
    return x;
}

// WINDOW: with the code for rows that see the last keys only
template <bool INT8, int HD, int NR, int RW, bool WINDOW>
__global__ __launch_bounds__(64 * PA_WAVES, 2)
void paged_prefix_kernel(PagedAttnArgs a, PagedPrefixArgs pre) {
    constexpr int EB = INT8 ? 1 : 2;
    constexpr int KW = PA_WAVES / RW;                  // waves that share the columns
    constexpr int UNIT = PA_TILE * KW;
    constexpr int COLS = 16 * NR * RW;                 // columns of the workgroup
    constexpr int NST = HD / 32;                       // Q.K^T steps
    constexpr int KC = INT8 ? HD / 64 : HD / 32;       // 16-byte pieces of a K row per lane
    constexpr bool KT = INT8 && HD % 64 != 0;          // and an 8-byte one
    constexpr int NT = HD / 16;                        // 16-wide d tiles of O
    constexpr int V0 = HD == 96 ? 4 : NT;              // neighbouring d per lane, first part ...
    constexpr int V1 = NT - V0;                        // ... and second (from d = 64)
    constexpr int W0 = (V0 * EB + 3) / 4, W1 = (V1 * EB + 3) / 4, VW = W0 + W1;   // in words
    constexpr int LD = HD + 4;
    extern __shared__ __attribute__((aligned(16))) float smem[];
    __shared__ int sLo[PA_WAVES], sAt[COLS];           // (sAt: a column's place in the parts)

    const int tiles = (a.B * (a.n_heads / a.n_kv) + COLS - 1) / COLS;
    // (the row tiles of one part and head are neighbours: they read the same keys)
    const int tile = (int)(blockIdx.x % (unsigned)tiles), rest = (int)(blockIdx.x / (unsigned)tiles);
    const int kvh = rest % a.n_kv, part = rest / a.n_kv;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), wv = wave % KW, rg = wave / KW;
    const int l = (int)threadIdx.x & 63, li = l & 15, lg = l >> 4;
    const int G = a.n_heads / a.n_kv;
    const int cols = a.B * G;
    const int len = min(max(*pre.len, 0), pre.max_len);

    // the first key that any row sees
    int base = 0;
    if (WINDOW) {
        int lo = len;
        for (int b = (int)threadIdx.x; b < a.B; b += 64 * PA_WAVES) {
            const int n = min(a.lens[b], a.max_seq);
            if (n >= 0) lo = min(lo, first_seen(len, n, a.window));
        }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) lo = min(lo, __shfl_xor(lo, o, 64));
        if (l == 0) sLo[wave] = lo;
        __syncthreads();
        base = min(min(sLo[0], sLo[1]), min(sLo[2], sLo[3])) & ~(PA_BLOCK - 1);
    }
    const int units = (int)(((unsigned)(len - base) + UNIT - 1) / (unsigned)UNIT);
    const int n_parts = min(units, a.prefix_splits);
    if (blockIdx.x == 0 && threadIdx.x == 0) *(int*)a.prefix = n_parts;
    if (part >= n_parts) return;
    const int kv0 = base + part_begin(units, n_parts, part) * UNIT;
    const int kv1 = (int)min((unsigned)base + (unsigned)part_begin(units, n_parts, part + 1) * UNIT, (unsigned)len);

    // the lane's columns: row and head, the first key it sees
    const int c0 = tile * COLS + 16 * NR * rg + li;
    int lo[NR], lo_max = 0;
    bool dead[NR];                                     // sees nothing of the prefix (or no column)
    h8 qb[NR][NST];
#pragma unroll
    for (int j = 0; j < NR; j++) {
        const int c = min(c0 + 16 * j, cols - 1), b = c / G, g = c - b * G;
        const bool is = c0 + 16 * j < cols;
        lo[j] = 0;
        dead[j] = !is;
        if (WINDOW) {
            const int n = min(a.lens[b], a.max_seq);
            const int first = first_seen(len, n, a.window);
            dead[j] = dead[j] || n < 0 || first >= len;
            lo[j] = dead[j] ? 0 : first;
        }
        lo_max = max(lo_max, lo[j]);
#pragma unroll
        for (int st = 0; st < NST; st++) {
            const int d = !INT8 ? 32 * st + 8 * lg : (KT && st == NST - 1 ? 64 * KC + 8 * lg : 64 * (st / 2) + 16 * lg + 8 * (st % 2));
            const u32x4a w = *(const u32x4a*)(a.q + b * a.q_stride + (int64_t)(kvh * G + g) * HD + d);
            qb[j][st] = __builtin_bit_cast(h8, is ? w : u32x4a{0u, 0u, 0u, 0u});
        }
    }
    if (WINDOW) {
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) lo_max = max(lo_max, __shfl_xor(lo_max, o, 64));
        lo_max = __builtin_amdgcn_readfirstlane(lo_max);
    }

    // Passes of 1024 keys: lane j looks up block j, one pass ahead.
    auto look_up = [&](unsigned k0) {
        const unsigned t = k0 + PA_BLOCK * l;
        return t < (unsigned)kv1 ? pre.table[t >> a.page_shift] : -1;
    };
    int pass = kv0, slot0 = 0;
    uint64_t there = 0, todo = 0;                      // blocks of the pass that are there; this wave's tiles of those (bit 2 i)
    int pg = look_up(kv0);
    auto enter = [&](unsigned k0) {
        pass = (int)k0;
        const unsigned t = k0 + PA_BLOCK * l;
        there = __builtin_amdgcn_ballot_w64(t < (unsigned)kv1 && (unsigned)pg < (unsigned)a.n_pages);
        slot0 = (pg << a.page_shift) + (int)(t & ((1u << a.page_shift) - 1));
        todo = (there | (there >> 1)) & ((~(uint64_t)0 / (((uint64_t)1 << 2 * KW) - 1)) << (2 * wv));
        pg = look_up(k0 + PA_PASS);
    };
    enter(kv0);

    const uint32_t row = (uint32_t)a.n_kv * a.cache_head_dim * EB;      // bytes
    const int64_t hoff = (int64_t)kvh * a.cache_head_dim * EB;

    struct Tile { int p0, s0, s1; bool v0, v1; };
    auto next_tile = [&]() {
        Tile x = {-1, 0, 0, false, false};
        while (!todo) {
            if ((unsigned)pass + PA_PASS >= (unsigned)kv1) return x;
            enter((unsigned)pass + PA_PASS);
        }
        const int i = __builtin_ctzll(todo);
        todo &= todo - 1;
        x.p0 = pass + PA_BLOCK * i;
        x.v0 = (there >> i) & 1;
        x.v1 = (there >> (i + 1)) & 1;
        const int p = __builtin_amdgcn_readlane(slot0, i), q = __builtin_amdgcn_readlane(slot0, i + 1);
        x.s0 = __builtin_amdgcn_readfirstlane(x.v0 ? p : q);
        x.s1 = __builtin_amdgcn_readfirstlane(x.v1 ? q : p);
        return x;
    };

    u32x4a rk[2][KC > 0 ? KC : 1] = {};
    u32x2a rt[2] = {};
    uint32_t rv[8][VW] = {};
    float rs = 1.0f;
    auto lane_offset = [](uint32_t x) {
        asm("" : "+v"(x));
        return x;
    };
    auto block_base = [&](const void* pages, int slot) {
        uint64_t x = (uint64_t)pages + (uint64_t)((int64_t)slot * row + hoff);
        asm("" : "+s"(x));
        return x;
    };
    auto load_k = [&](int s0, int s1) {
        const uint32_t o = lane_offset((uint32_t)li * row + 16 * lg), o8 = lane_offset((uint32_t)li * row + 8 * lg);
#pragma unroll
        for (int q = 0; q < 2; q++) {
            const uint64_t p = block_base(a.k, q ? s1 : s0);
#pragma unroll
            for (int c = 0; c < KC; c++) rk[q][c] = *(global_ptr<u32x4a>)(p + o + 64 * c);
            if (KT) rt[q] = *(global_ptr<u32x2a>)(p + o8 + 64 * KC);
        }
        if (INT8) {
            // lane li: K (li < 8) or V scale of key 4 lg + li % 4 of block (li >> 2) & 1
            const float* p = li < 8 ? a.ks : a.vs;
            const int64_t s = (li & 4 ? s1 : s0) + 4 * lg + (li & 3);
            rs = p ? p[s * a.n_kv + kvh] : 1.0f;
        }
    };
    auto load_v = [&](int s0, int s1) {
        uint32_t o[4], o1[4];
#pragma unroll
        for (int r = 0; r < 4; r++) {
            o[r] = lane_offset((uint32_t)(4 * lg + r) * row + V0 * EB * li);
            if (V1 > 0) o1[r] = lane_offset((uint32_t)(4 * lg + r) * row + V1 * EB * li);
        }
#pragma unroll
        for (int q = 0; q < 2; q++) {
            const uint64_t p = block_base(a.v, q ? s1 : s0);
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const uint64_t x = p + o[r];
                uint32_t (&v)[VW] = rv[4 * q + r];
                if (V0 * EB == 16) { const u32x4a w = *(global_ptr<u32x4a>)x; v[0] = w.x; v[1 % VW] = w.y; v[2 % VW] = w.z; v[3 % VW] = w.w; }
                else if (V0 * EB == 8) { const u32x2a w = *(global_ptr<u32x2a>)x; v[0] = w.x; v[1 % VW] = w.y; }
                else if (V0 * EB == 4) v[0] = *(global_ptr<uint32_t>)x;
                else v[0] = *(global_ptr<uint16_t>)x;
                if (V1 > 0) {
                    const uint64_t y = p + o1[r] + 64 * EB;
                    v[VW - 1] = V1 * EB == 4 ? *(global_ptr<uint32_t>)y : *(global_ptr<uint16_t>)y;
                }
            }
        }
    };
    // the eight keys' values of d tile j as the A operand
    auto v_operand = [&](const uint32_t (&v)[8][VW], int j) {
        const int jj = j < V0 ? j : j - V0;
        const int w = (j < V0 ? 0 : W0) + jj * EB / 4, at = jj % (4 / EB);
        const uint32_t sel = INT8 ? 0x0c040c00u + 0x00010001u * at : (at ? 0x07060302u : 0x05040100u);
        u32x4a va;
#pragma unroll
        for (int e = 0; e < 4; e++) va[e] = __builtin_amdgcn_perm(v[2 * e + 1][w], v[2 * e][w], sel);
        return __builtin_bit_cast(h8, va);
    };

    Tile cur = next_tile();
    if (cur.p0 >= 0) {
        load_k(cur.s0, cur.s1);
        load_v(cur.s0, cur.s1);
    }

    // - sum_d 128 2^-24 q_d: takes the codes' offset out of every score
    f32x4p start[NR] = {};
    if (INT8) {
        const h8 off = __builtin_bit_cast(h8, u32x4a{0x00800080u, 0x00800080u, 0x00800080u, 0x00800080u});
#pragma unroll
        for (int j = 0; j < NR; j++) {
#pragma unroll
            for (int st = 0; st < NST; st++) start[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(off, qb[j][st], start[j], 0, 0, 0);
            start[j] = -start[j];
        }
    }
    const float f0 = a.scale * PA_LOG2E;

    float m[NR], L[NR], M[NR];                         // maximum, this lane's sum; maximum with the V scales
    f32x4p acc[NR][NT], wsum[NR];
#pragma unroll
    for (int j = 0; j < NR; j++) {
        m[j] = M[j] = -INFINITY;
        L[j] = 0.0f;
        wsum[j] = f32x4p{};
#pragma unroll
        for (int t = 0; t < NT; t++) acc[j][t] = f32x4p{};
    }
    const h8 ones = __builtin_bit_cast(h8, u32x4a{0x3C003C00u, 0x3C003C00u, 0x3C003C00u, 0x3C003C00u});

    while (cur.p0 >= 0) {
        const int p0 = cur.p0;
        const bool v0 = cur.v0, v1 = cur.v1;
        // 1. scores of the tile, in units of log2
        float s[NR][8];
#pragma unroll
        for (int q = 0; q < 2; q++) {
            f32x4p c[NR];
#pragma unroll
            for (int j = 0; j < NR; j++) c[j] = start[j];
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
#pragma unroll
                for (int j = 0; j < NR; j++) c[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kb, qb[j][st], c[j], 0, 0, 0);
            }
#pragma unroll
            for (int j = 0; j < NR; j++)
#pragma unroll
                for (int r = 0; r < 4; r++) s[j][4 * q + r] = c[j][r];
        }
        const float sraw = rs;
        const Tile next = next_tile();
        if (next.p0 >= 0) load_k(next.s0, next.s1);
        // lanes li < 8: the K factor, li >= 8: log2 of the V scale
        const float sv = INT8 ? (li < 8 ? sraw * f0 * 16777216.0f : __builtin_amdgcn_logf(fabsf(sraw))) : 0.0f;
        float kf[8], vf[8];
        if (INT8) {
            kf[0] = row_bcast<0>(sv); kf[1] = row_bcast<1>(sv); kf[2] = row_bcast<2>(sv); kf[3] = row_bcast<3>(sv);
            kf[4] = row_bcast<4>(sv); kf[5] = row_bcast<5>(sv); kf[6] = row_bcast<6>(sv); kf[7] = row_bcast<7>(sv);
            vf[0] = row_bcast<8>(sv); vf[1] = row_bcast<9>(sv); vf[2] = row_bcast<10>(sv); vf[3] = row_bcast<11>(sv);
            vf[4] = row_bcast<12>(sv); vf[5] = row_bcast<13>(sv); vf[6] = row_bcast<14>(sv); vf[7] = row_bcast<15>(sv);
        }
        const bool whole = v0 && v1 && kv1 - p0 >= PA_TILE;         // every key of the tile is one
        const bool full = whole && (!WINDOW || p0 >= lo_max);                    // and every column sees it
        uint32_t keys = 0xFFu;                         // bit e: the lane's key e is one
        if (!whole) {
            keys = 0;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const int o = PA_BLOCK * (e >> 2) + 4 * lg + (e & 3);      // key p0 + o
                if ((e < 4 ? v0 : v1) && o < kv1 - p0) keys |= 1u << e;
            }
        }
        h8 pb[NR], pl[NR];
        uint32_t seen[NR];
#pragma unroll
        for (int j = 0; j < NR; j++) {
            uint32_t live = keys;
            if (WINDOW && !full) {
#pragma unroll
                for (int e = 0; e < 8; e++)
                    if (PA_BLOCK * (e >> 2) + 4 * lg + (e & 3) < lo[j] - p0) live &= ~(1u << e);
            }
            seen[j] = live;
#pragma unroll
            for (int e = 0; e < 8; e++) s[j][e] *= INT8 ? kf[e] : f0;
            if (!full) {
#pragma unroll
                for (int e = 0; e < 8; e++) s[j][e] = live >> e & 1 ? s[j][e] : -INFINITY;
            }
            // 2. softmax
            float mx = s[j][0];
#pragma unroll
            for (int e = 1; e < 8; e++) mx = fmaxf(mx, s[j][e]);
            const float mn = fmaxf(m[j], rows_op(mx, false)), mb = base_of(mn);
            float corr = __builtin_amdgcn_exp2f(m[j] - mb);
            m[j] = mn;
            float p[8], ps = 0.0f;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                p[e] = __builtin_amdgcn_exp2f(s[j][e] - mb);
                ps += p[e];
            }
            L[j] = L[j] * corr + ps;
            if (INT8) {
                // the weights times the V scales, under a maximum of their own
                float t[8];
#pragma unroll
                for (int e = 0; e < 8; e++) t[e] = s[j][e] + vf[e];
                if (!full) {
#pragma unroll
                    for (int e = 0; e < 8; e++) t[e] = live >> e & 1 ? t[e] : -INFINITY;
                }
                float tx = t[0];
#pragma unroll
                for (int e = 1; e < 8; e++) tx = fmaxf(tx, t[e]);
                const float Mn = fmaxf(M[j], rows_op(tx, false)), Mb = base_of(Mn);
                corr = __builtin_amdgcn_exp2f(M[j] - Mb);
                M[j] = Mn;
#pragma unroll
                for (int e = 0; e < 8; e++) p[e] = __builtin_amdgcn_exp2f(t[e] - Mb);
                // a negative V scale: its sign back onto the weight (no quantiser here writes one)
                if (__builtin_amdgcn_ballot_w64(li >= 8 && sraw < 0.0f)) {
                    p[0] = __builtin_copysignf(p[0], row_bcast<8>(sraw)); p[1] = __builtin_copysignf(p[1], row_bcast<9>(sraw));
                    p[2] = __builtin_copysignf(p[2], row_bcast<10>(sraw)); p[3] = __builtin_copysignf(p[3], row_bcast<11>(sraw));
                    p[4] = __builtin_copysignf(p[4], row_bcast<12>(sraw)); p[5] = __builtin_copysignf(p[5], row_bcast<13>(sraw));
                    p[6] = __builtin_copysignf(p[6], row_bcast<14>(sraw)); p[7] = __builtin_copysignf(p[7], row_bcast<15>(sraw));
                }
            }
            // no column's maximum moved: every factor is 1
            if (__builtin_amdgcn_ballot_w64(corr != 1.0f)) {
#pragma unroll
                for (int t = 0; t < NT; t++) acc[j][t] *= corr;
                if (INT8) wsum[j] *= corr;
            }
            // p * PA_LIFT in two parts, each rounded down; of a weight that is not 0 the low
            // part is not 0 either (fp16 V may be infinite)
            u32x4a hw, lw;
#pragma unroll
            for (int e = 0; e < 8; e += 2) {
                const float x = p[e] * PA_LIFT, y = p[e + 1] * PA_LIFT;
                const auto hi = __builtin_amdgcn_cvt_pkrtz(x, y);
                const auto low = __builtin_amdgcn_cvt_pkrtz(x - (float)hi[0], y - (float)hi[1]);
                const uint32_t h = __builtin_bit_cast(uint32_t, hi);
                hw[e / 2] = h;
                lw[e / 2] = __builtin_bit_cast(uint32_t, low) | (INT8 ? 0u : ones_of(h));
            }
            pb[j] = __builtin_bit_cast(h8, hw);
            pl[j] = __builtin_bit_cast(h8, lw);
        }
        // 3. O^T += V^T P^T
        if (!INT8 && !whole) {                         // what a slot without a key holds may be NaN
#pragma unroll
            for (int e = 0; e < 8; e++)
#pragma unroll
                for (int w = 0; w < VW; w++) rv[e][w] = keys >> e & 1 ? rv[e][w] : 0u;
        }
        if (WINDOW && !INT8 && p0 < lo_max) {
            // keys that some columns do not see: infinities and NaN out of V, and into those that do
            uint32_t any = 0;
#pragma unroll
            for (int e = 0; e < 8; e++)
#pragma unroll
                for (int w = 0; w < VW; w++) any |= ((rv[e][w] & 0x7C007C00u) + 0x04000400u) & 0x80008000u;
            if (__builtin_amdgcn_ballot_w64(any != 0)) {
#pragma unroll 1
                for (int kind = 0; kind < 3; kind++) {   // +inf, -inf, NaN
                    // 1.0 where the value is of this kind
                    const uint32_t nan = kind == 2 ? ~0u : 0u, neg = kind == 1 ? ~0u : 0u;
                    uint32_t at[8][VW];
#pragma unroll
                    for (int e = 0; e < 8; e++)
#pragma unroll
                        for (int w = 0; w < VW; w++) {
                            const uint32_t x = rv[e][w], odd = ((x & 0x7C007C00u) + 0x04000400u) >> 15;
                            const uint32_t mantissa = ((x & 0x03FF03FFu) + 0x03FF03FFu) >> 10;
                            at[e][w] = (odd & ~(mantissa ^ nan) & (~((x >> 15) ^ neg) | nan) & 0x00010001u) * 0x3C00u;
                        }
                    const float bad = kind == 0 ? INFINITY : (kind == 1 ? -INFINITY : NAN);
#pragma unroll
                    for (int j = 0; j < NR; j++) {
                        u32x4a on;
#pragma unroll
                        for (int e = 0; e < 4; e++)
                            on[e] = (seen[j] >> (2 * e) & 1 ? 0x3C00u : 0u) | (seen[j] >> (2 * e + 1) & 1 ? 0x3C000000u : 0u);
#pragma unroll
                        for (int t = 0; t < NT; t++) {
                            const f32x4p c = __builtin_amdgcn_mfma_f32_16x16x32_f16(v_operand(at, t), __builtin_bit_cast(h8, on), f32x4p{}, 0, 0, 0);
#pragma unroll
                            for (int r = 0; r < 4; r++)
                                if (c[r] > 0.0f) acc[j][t][r] += bad;
                        }
                    }
                }
#pragma unroll
                for (int e = 0; e < 8; e++)
#pragma unroll
                    for (int w = 0; w < VW; w++) {
                        const uint32_t x = rv[e][w], f = ((x & 0x7C007C00u) + 0x04000400u) >> 15 & 0x00010001u;
                        rv[e][w] = x & ~(f * 0xFFFFu);
                    }
            }
        }
        if (INT8) {
#pragma unroll
            for (int e = 0; e < 8; e++)
#pragma unroll
                for (int w = 0; w < VW; w++) rv[e][w] ^= 0x80808080u;
        }
#pragma unroll
        for (int t = 0; t < NT; t++) {
            const h8 va = v_operand(rv, t);
#pragma unroll
            for (int j = 0; j < NR; j++) acc[j][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, pb[j], acc[j][t], 0, 0, 0);
#pragma unroll
            for (int j = 0; j < NR; j++) acc[j][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, pl[j], acc[j][t], 0, 0, 0);
        }
        if (INT8) {
#pragma unroll
            for (int j = 0; j < NR; j++) {
                wsum[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ones, pb[j], wsum[j], 0, 0, 0);
                wsum[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ones, pl[j], wsum[j], 0, 0, 0);
            }
        }
        if (next.p0 >= 0) load_v(next.s0, next.s1);
        cur = next;
    }

    // the waves' states: [wave][16 NR][LD] numerators, then m and l [wave][16 NR]
    float* sO = smem + (size_t)wave * 16 * NR * LD;
    float* sML = smem + (size_t)PA_WAVES * 16 * NR * LD;
#pragma unroll
    for (int j = 0; j < NR; j++) {
        const float sum = rows_op(L[j], true);
        float f = 1.0f / PA_LIFT;
        if (INT8) f = M[j] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(M[j] - base_of(m[j])) * (1.0f / PA_LIFT);
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const float x = INT8 ? (acc[j][t][r] * 16777216.0f - 128.0f * wsum[j][0]) * f : acc[j][t][r] * f;
                sO[(16 * j + li) * LD + (t < V0 ? V0 * (4 * lg + r) + t : 64 + V1 * (4 * lg + r) + t - V0)] = dead[j] ? 0.0f : x;
            }
        if (lg == 0) {
            sML[wave * 16 * NR + 16 * j + li] = dead[j] ? -INFINITY : m[j];
            sML[(PA_WAVES + wave) * 16 * NR + 16 * j + li] = dead[j] ? 0.0f : sum;
            const int c = c0 + 16 * j, b = c / G;
            sAt[16 * (NR * rg + j) + li] = b * a.n_heads + kvh * G + (c - b * G);
        }
    }
    __syncthreads();
    // Join of the key waves in wave order: a thread a column, for the factors, then four d a
    // thread (element by element, with the division for every element, the join was 8 of 14
    // us: 16 rows of 32 / 8 heads x 128 over 1153 keys).
    const int64_t step = (int64_t)a.B * a.n_heads;
    float2* oml = (float2*)(a.prefix + 4) + part * step;
    float* onum = a.prefix + prefix_num_at(a.prefix_splits, step) + part * step * HD;
    if ((int)threadIdx.x < COLS && tile * COLS + (int)threadIdx.x < cols) {
        const int cl = (int)threadIdx.x, w0 = cl / (16 * NR) * KW, cc = cl % (16 * NR);
        float top = sML[w0 * 16 * NR + cc], den = 0.0f;
#pragma unroll
        for (int w = 1; w < KW; w++) top = fmaxf(top, sML[(w0 + w) * 16 * NR + cc]);
        const float tb = base_of(top);
#pragma unroll
        for (int w = 0; w < KW; w++) {
            float& x = sML[(w0 + w) * 16 * NR + cc];
            x = __builtin_amdgcn_exp2f(x - tb);
            den += x * sML[(PA_WAVES + w0 + w) * 16 * NR + cc];
        }
        oml[sAt[cl]] = make_float2(top, den);
    }
    __syncthreads();
    constexpr int EACH = (COLS * (HD / 4) + 64 * PA_WAVES - 1) / (64 * PA_WAVES);
#pragma unroll
    for (int i = 0; i < EACH; i++) {
        const int e = (int)threadIdx.x + i * 64 * PA_WAVES, cl = e / (HD / 4), d = 4 * (e % (HD / 4));
        if (cl >= COLS || tile * COLS + cl >= cols) break;
        const int w0 = cl / (16 * NR) * KW, cc = cl % (16 * NR);
        f32x4p num = {};
#pragma unroll
        for (int w = 0; w < KW; w++)
            num += sML[(w0 + w) * 16 * NR + cc] * *(const f32x4p*)(smem + ((size_t)(w0 + w) * 16 * NR + cc) * LD + d);
        *(f32x4p*)(onum + (int64_t)sAt[cl] * HD + d) = num;
    }
}

// ---- many columns: keys through LDS ----

// Eight waves, RW of them with 32 columns of their own each, KW = 8 / RW that share columns and
// take alternate tiles of 32 keys.  Stages of 64 keys lie in LDS as fp16 rows, two of them:
// one is worked on, the next goes there through registers (INT8 codes converted on the way,
// once for all columns), the one behind it is on its way.  16-byte piece c of key r lies at
// place c ^ kswz(r) or c ^ vswz(r): K is read as the A operand lies (16 keys, four pieces), V
// transposed by the read itself (4 keys x 16 d to a 16-lane row).  (Loads straight to LDS
// are waited for before every transposing read, by the compiler: 125 us for 64 rows over
// 32768 fp16 keys.)
constexpr int PT_WAVES = 8;
constexpr int PT_STAGE = 64;
// Factor on the weights' fp16 parts, and how far (in log2) a weight may pass 1: 2^15.9 is
// still an fp16.  The parts' last bit is 2^-36 of the reference.
constexpr float PT_LIFT_LOG = 12.0f, PT_LIFT = 4096.0f, PT_SLACK = 3.9f;
template <int HD> __device__ __forceinline__ int kswz(int r) { return HD == 128 ? r & 15 : (HD == 64 ? (r >> 1) & 7 : (r >> 2) & 3); }
template <int HD> __device__ __forceinline__ int vswz(int r) { return HD == 128 ? 2 * r & 15 : (HD == 64 ? r & 6 : (r >> 1) & 2); }

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
__device__ __forceinline__ u32x2a read_tr(const uint8_t* p) {
    return __builtin_bit_cast(u32x2a, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)p));
}

// x minus the low / high half of h, in one operation
__device__ __forceinline__ float less_low(float x, uint32_t h) {
    float y;
    asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]" : "=v"(y) : "v"(h), "v"(x));
    return y;
}
__device__ __forceinline__ float less_high(float x, uint32_t h) {
    float y;
    asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(y) : "v"(h), "v"(x));
    return y;
}

template <bool INT8, int HD>
constexpr int pt_lds() {
    constexpr int MAIN = 2 * 2 * PT_STAGE * HD * 2 + (INT8 ? 2 * (3 * PT_STAGE + 4) * 4 : 0), OUT = PT_WAVES * 32 * (HD + 4 + 3) * 4;
    return MAIN > OUT ? MAIN : OUT;
}

template <bool INT8, int HD, int RW, bool WINDOW>
__global__ __launch_bounds__(64 * PT_WAVES, 2)
void prefix_tile_kernel(PagedAttnArgs a, PagedPrefixArgs pre) {
    constexpr int EB = INT8 ? 1 : 2, NR = 2;
    constexpr int KW = PT_WAVES / RW, COLS = 32 * RW;
    constexpr int NST = HD / 32, NT = HD / 16, LD = HD + 4;
    constexpr int ROWB = HD * 2, HALF = PT_STAGE * ROWB;          // K rows of a stage, then V rows
    constexpr int PC = HD * EB / 16, PIECES = PT_STAGE * PC;       // 16-byte pieces of a row, of K's rows of a stage
    constexpr int NI = (2 * PIECES + 511) / 512;                  // a thread's
    extern __shared__ __attribute__((aligned(128))) uint8_t ring[];
    float* sScale = (float*)(ring + 2 * 2 * HALF);             // (INT8) [slot]: K factor, log2 |V scale|, V scale of each key, any below 0
    __shared__ int sLo[PT_WAVES], sAt[COLS];           // (sAt: a column's place in the parts)

    const int G = a.n_heads / a.n_kv, cols = a.B * G;
    const int tiles = (cols + COLS - 1) / COLS, groups = a.n_kv * a.prefix_splits;
    // the column tiles of one part and head read the same keys: on one XCD, one after the other
    int tile, rest;
    if (groups % 8 == 0) {
        const int x = (int)(blockIdx.x & 7u), y = (int)(blockIdx.x >> 3);
        tile = y % tiles;
        rest = y / tiles * 8 + x;
    } else {
        tile = (int)(blockIdx.x % (unsigned)tiles);
        rest = (int)(blockIdx.x / (unsigned)tiles);
    }
    const int kvh = rest % a.n_kv, part = rest / a.n_kv;
    const int tid = (int)threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), wv = wave % KW, rg = wave / KW;
    const int l = tid & 63, li = l & 15, lg = l >> 4;
    // (a block that is not there is loaded from page 0 and not counted: so there has to be one)
    const int len = a.n_pages > 0 ? min(max(*pre.len, 0), pre.max_len) : 0;

    // the first key that any row sees
    int base = 0;
    if (WINDOW) {
        int lo = len;
        for (int b = tid; b < a.B; b += 64 * PT_WAVES) {
            const int n = min(a.lens[b], a.max_seq);
            if (n >= 0) lo = min(lo, first_seen(len, n, a.window));
        }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) lo = min(lo, __shfl_xor(lo, o, 64));
        if (l == 0) sLo[wave] = lo;
        __syncthreads();
        base = len;
#pragma unroll
        for (int w = 0; w < PT_WAVES; w++) base = min(base, sLo[w]);
        base &= ~(PA_BLOCK - 1);
    }
    const int units = (int)(((unsigned)(len - base) + PT_STAGE - 1) / (unsigned)PT_STAGE);
    const int n_parts = min(units, a.prefix_splits);
    if (blockIdx.x == 0 && tid == 0) *(int*)a.prefix = n_parts;
    if (part >= n_parts) return;
    const int kv0 = base + part_begin(units, n_parts, part) * PT_STAGE;
    const int kv1 = (int)min((unsigned)base + (unsigned)part_begin(units, n_parts, part + 1) * PT_STAGE, (unsigned)len);
    const int stages = (int)(((unsigned)(kv1 - kv0) + PT_STAGE - 1) / (unsigned)PT_STAGE);

    // Passes of 1024 keys: lane j looks up block j, one pass ahead; the loads run ahead of the
    // products, so each has its own pass.
    auto look_up = [&](unsigned k0) {
        const unsigned t = k0 + PA_BLOCK * l;
        return t < (unsigned)kv1 ? pre.table[t >> a.page_shift] : -1;
    };
    int slot0 = 0, pg = look_up(kv0);                             // slot of the lane's block, 0 where there is none
    uint64_t there_load = 0, there = 0;                           // blocks that are there: of the loads' pass, of the products'
    auto enter = [&](unsigned k0) {
        const unsigned t = k0 + PA_BLOCK * l;
        const bool is = t < (unsigned)kv1 && (unsigned)pg < (unsigned)a.n_pages;
        there_load = __builtin_amdgcn_ballot_w64(is);
        slot0 = is ? (pg << a.page_shift) + (int)(t & ((1u << a.page_shift) - 1)) : 0;
        pg = look_up(k0 + PA_PASS);
    };
    const uint32_t row = (uint32_t)a.n_kv * a.cache_head_dim * EB;      // bytes
    const int64_t hoff = (int64_t)kvh * a.cache_head_dim * EB;

    // what follows from the thread alone is found anew where it is used: kept, it would take
    // registers that the products need
    auto anew = [](int x) {
        asm("" : "+v"(x));
        return x;
    };
    // a thread's ith piece: V's or K's, key, piece of the row
    struct Piece { bool v; int r, c; };
    auto piece = [](int t, int i) {
        Piece x;
        if (PIECES % 512 == 0) {
            x.v = 512 * i >= PIECES;
            x.r = t / PC + 512 * i % PIECES / PC;
            x.c = t % PC;
        } else {
            const int e = min(t + 512 * i, 2 * PIECES - 1);
            x.v = e >= PIECES;
            x.r = (x.v ? e - PIECES : e) / PC;
            x.c = (x.v ? e - PIECES : e) % PC;
        }
        return x;
    };
    u32x4a data[NI];
    float ksr = 0.0f, vsr = 0.0f;
    auto fetch = [&](int s) {                                     // stage s on its way
        if (s % 16 == 0) enter((unsigned)kv0 + (unsigned)s * PT_STAGE);
        auto slot = [&](int r) { return __builtin_amdgcn_ds_bpermute(4 * (4 * (s % 16) + (r >> 4)), slot0) + (r & 15); };
        const int tid_ = anew(tid);
#pragma unroll
        for (int i = 0; i < NI; i++) {
            const Piece x = piece(tid_, i);
            const bool v = x.v;
            const int r = x.r, c = x.c;
            data[i] = *(global_ptr<u32x4a>)((uint64_t)(v ? a.v : a.k) + (uint64_t)((int64_t)slot(r) * row + hoff) + 16 * c);
        }
        if (INT8) {
            const int64_t at = (int64_t)slot(l) * a.n_kv + kvh;
            ksr = a.ks ? a.ks[at] : 1.0f;
            vsr = a.vs ? a.vs[at] : 1.0f;
        }
    };
    // the scale's sign goes into q, so that the largest product is the largest score; with fp16
    // keys a scale of 0 is one that no finite product brings near 1 (masked products are -inf
    // before they meet it; those of INT8 keys, which may have any scale, after)
    const float f0 = fmaxf(fabsf(a.scale) * PA_LOG2E, INT8 ? 0.0f : 1e-30f);
    auto put = [&](int s) {                                       // the fetched stage into LDS
        uint8_t* st = ring + (s & 1) * 2 * HALF;
        const int tid_ = anew(tid);
#pragma unroll
        for (int i = 0; i < NI; i++) {
            if (2 * PIECES % 512 != 0 && tid_ + 512 * i >= 2 * PIECES) break;
            const Piece x = piece(tid_, i);
            const bool v = x.v;
            const int r = x.r, c = x.c;
            const int z = v ? vswz<HD>(r) : kswz<HD>(r);
            uint8_t* to = st + (v ? HALF : 0) + r * ROWB;
            if (INT8) {
                const u32x2a x0 = i8x4_to_h4(data[i].x), x1 = i8x4_to_h4(data[i].y), x2 = i8x4_to_h4(data[i].z), x3 = i8x4_to_h4(data[i].w);
                *(u32x4a*)(to + 16 * (2 * c ^ z)) = u32x4a{x0.x, x0.y, x1.x, x1.y};
                *(u32x4a*)(to + 16 * ((2 * c + 1) ^ z)) = u32x4a{x2.x, x2.y, x3.x, x3.y};
            } else {
                *(u32x4a*)(to + 16 * (c ^ z)) = data[i];
            }
        }
        if (INT8 && tid < PT_STAGE) {
            float* sc = sScale + (s & 1) * (3 * PT_STAGE + 4);
            sc[tid] = ksr * f0;
            sc[PT_STAGE + tid] = __builtin_amdgcn_logf(fabsf(vsr));
            sc[2 * PT_STAGE + tid] = vsr;
            const uint64_t below = __builtin_amdgcn_ballot_w64(vsr < 0.0f);
            if (tid == 0) sc[3 * PT_STAGE] = below ? 1.0f : 0.0f;
        }
    };

    // the lane's columns: row and head, the first key it sees
    const int c0 = tile * COLS + 32 * rg + li;
    int lo[NR], lo_max = 0;
    bool dead[NR];                                     // sees nothing of the prefix (or no column)
    h8 qb[NR][NST];
    const uint32_t flip = a.scale < 0.0f ? 0x80008000u : 0u;
#pragma unroll
    for (int j = 0; j < NR; j++) {
        const int c = min(c0 + 16 * j, cols - 1), b = c / G, g = c - b * G;
        const bool is = c0 + 16 * j < cols;
        lo[j] = 0;
        dead[j] = !is;
        if (WINDOW) {
            const int n = min(a.lens[b], a.max_seq);
            const int first = first_seen(len, n, a.window);
            dead[j] = dead[j] || n < 0 || first >= len;
            lo[j] = dead[j] ? 0 : first;
        }
        lo_max = max(lo_max, lo[j]);
#pragma unroll
        for (int st = 0; st < NST; st++) {
            u32x4a w = *(const u32x4a*)(a.q + b * a.q_stride + (int64_t)(kvh * G + g) * HD + 32 * st + 8 * lg);
            w ^= flip;
            qb[j][st] = __builtin_bit_cast(h8, is ? w : u32x4a{0u, 0u, 0u, 0u});
        }
    }
    if (WINDOW) {
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) lo_max = max(lo_max, __shfl_xor(lo_max, o, 64));
        lo_max = __builtin_amdgcn_readfirstlane(lo_max);
    }

    float m[NR], L[NR], M[NR];                         // maximum, this lane's sum; maximum with the V scales
    f32x4p acc[NR][NT];
#pragma unroll
    for (int j = 0; j < NR; j++) {
        m[j] = M[j] = -INFINITY;
        L[j] = 0.0f;
#pragma unroll
        for (int t = 0; t < NT; t++) acc[j][t] = f32x4p{};
    }

    // A tile's keys that are keys (bit e: the lane's key e), and that column j sees.
    auto keys_of = [&](int p0, bool v0, bool v1, int lg) {
        uint32_t keys = 0;
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const int o = PA_BLOCK * (e >> 2) + 4 * lg + (e & 3);          // key p0 + o
            if ((e < 4 ? v0 : v1) && o < kv1 - p0) keys |= 1u << e;
        }
        return keys;
    };
    auto seen_by = [&](uint32_t keys, int j, int p0, int lg) {
        if (WINDOW) {
#pragma unroll
            for (int e = 0; e < 8; e++)
                if (PA_BLOCK * (e >> 2) + 4 * lg + (e & 3) < lo[j] - p0) keys &= ~(1u << e);
        }
        return keys;
    };
    // Where the lane reads: piece lg of key li in K's rows, the (li / 4)th key of four and eight
    // bytes of a 16-wide d tile in V's.  Step t is 64 or 32 bytes further in the row, under
    // the place's exclusive or (rows of 192 bytes: the places move pieces within four only).
    const int at_k = li * ROWB + 16 * (lg ^ kswz<HD>(li));
    const int rv = 4 * lg + (li >> 2), at_v = HALF + rv * ROWB + 8 * (li & 1) + 16 * (((li & 3) >> 1) ^ vswz<HD>(rv));
    const int turn_v = 16 * vswz<HD>(rv);
    auto k_piece = [&](const uint8_t* tile, int q, int t) {
        return *(const u32x4a*)(HD == 96 ? tile + at_k + 64 * t + 16 * q * ROWB : ring + (((int)(tile - ring) + at_k) ^ 64 * t) + 16 * q * ROWB);
    };
    auto v_piece = [&](const uint8_t* tile, int t) {
        const uint8_t* x = HD == 96 ? tile + (t % 2 ? at_v - 2 * turn_v : at_v) + 32 * t : ring + (((int)(tile - ring) + at_v) ^ 32 * t);
        const u32x2a lo4 = read_tr(x), hi4 = read_tr(x + 16 * ROWB);
        return u32x4a{lo4.x, lo4.y, hi4.x, hi4.y};
    };
    // Tile of 32 keys from p0, at `tile` in LDS, its scales at sc.  m is a column's reference,
    // not its maximum: it moves up only where a score passes it by PT_SLACK, so that most
    // tiles rescale nothing and compare within a lane.
    auto work = [&](auto whole, const uint8_t* tile, const float* sc, int p0, bool v0, bool v1) {
        constexpr bool full = decltype(whole)::value;  // every key of the tile is one and every column sees it
        float s[NR][8];
#pragma unroll
        for (int q = 0; q < 2; q++) {
            f32x4p c[NR] = {};
#pragma unroll
            for (int t = 0; t < NST; t++) {
                const h8 kb = __builtin_bit_cast(h8, k_piece(tile, q, t));
#pragma unroll
                for (int j = 0; j < NR; j++) c[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kb, qb[j][t], c[j], 0, 0, 0);
            }
#pragma unroll
            for (int j = 0; j < NR; j++)
#pragma unroll
                for (int r4 = 0; r4 < 4; r4++) s[j][4 * q + r4] = c[j][r4];
        }
        float kf[8], vf[8];
        if (INT8) {
#pragma unroll
            for (int q = 0; q < 2; q++) {
                const f32x4p x = *(const f32x4p*)(sc + 16 * q + 4 * lg), y = *(const f32x4p*)(sc + PT_STAGE + 16 * q + 4 * lg);
#pragma unroll
                for (int e = 0; e < 4; e++) { kf[4 * q + e] = x[e]; vf[4 * q + e] = y[e]; }
            }
        }
        h8 pb[NR], pl[NR];
#pragma unroll
        for (int j = 0; j < NR; j++) {
            if (INT8) {
#pragma unroll
                for (int e = 0; e < 8; e++) s[j][e] *= kf[e];
            }
            if (!full) {
                const uint32_t live = seen_by(keys_of(p0, v0, v1, lg), j, p0, lg);
#pragma unroll
                for (int e = 0; e < 8; e++) s[j][e] = live >> e & 1 ? s[j][e] : -INFINITY;
            }
            // (f: from the products to units of log2)
            const float f = INT8 ? 1.0f : f0;
            float mx = fmaxf(fmaxf(s[j][0], s[j][1]), s[j][2]);
            mx = fmaxf(fmaxf(mx, s[j][3]), s[j][4]);
            mx = fmaxf(fmaxf(mx, s[j][5]), s[j][6]);
            mx = fmaxf(mx, s[j][7]) * f;
            if (__builtin_amdgcn_ballot_w64(mx > m[j] + PT_SLACK)) {
                const float mn = fmaxf(m[j], rows_op(mx, false)), corr = __builtin_amdgcn_exp2f(m[j] - base_of(mn));
                m[j] = mn;
                L[j] *= corr;
                if (!INT8) {
#pragma unroll
                    for (int t = 0; t < NT; t++) acc[j][t] *= corr;
                }
            }
            // weights times PT_LIFT, their sum too
            const float mb = PT_LIFT_LOG - base_of(m[j]);
            float p[8];
#pragma unroll
            for (int e = 0; e < 8; e++) {
                p[e] = __builtin_amdgcn_exp2f(INT8 ? s[j][e] + mb : fmaf(s[j][e], f, mb));
                L[j] += p[e];
            }
            if (INT8) {
                // the weights times the V scales, under a reference of their own
                float t[8];
#pragma unroll
                for (int e = 0; e < 8; e++) t[e] = s[j][e] + vf[e];
                if (!full) {
                    const uint32_t live = seen_by(keys_of(p0, v0, v1, lg), j, p0, lg);
#pragma unroll
                    for (int e = 0; e < 8; e++) t[e] = live >> e & 1 ? t[e] : -INFINITY;
                }
                float tx = fmaxf(fmaxf(t[0], t[1]), t[2]);
                tx = fmaxf(fmaxf(tx, t[3]), t[4]);
                tx = fmaxf(fmaxf(tx, t[5]), t[6]);
                tx = fmaxf(tx, t[7]);
                if (__builtin_amdgcn_ballot_w64(tx > M[j] + PT_SLACK)) {
                    const float Mn = fmaxf(M[j], rows_op(tx, false)), corr = __builtin_amdgcn_exp2f(M[j] - base_of(Mn));
                    M[j] = Mn;
#pragma unroll
                    for (int t2 = 0; t2 < NT; t2++) acc[j][t2] *= corr;
                }
                const float Mb = PT_LIFT_LOG - base_of(M[j]);
#pragma unroll
                for (int e = 0; e < 8; e++) p[e] = __builtin_amdgcn_exp2f(t[e] + Mb);
                // a negative V scale: its sign back onto the weight (no quantiser here writes one)
                if (__builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, sc[3 * PT_STAGE - (p0 - kv0) % PT_STAGE]))) {
#pragma unroll
                    for (int e = 0; e < 8; e++) p[e] = __builtin_copysignf(p[e], sc[2 * PT_STAGE + 16 * (e >> 2) + 4 * lg + (e & 3)]);
                }
            }
            // Two fp16 parts, the first rounded down, the second to nearest.  fp16 V may be
            // infinite, and 0 * inf is no part of inf: where the first is not 0 the second's last
            // bit is set.
            u32x4a hw, lw;
#pragma unroll
            for (int e = 0; e < 8; e += 2) {
                const auto hi = __builtin_amdgcn_cvt_pkrtz(p[e], p[e + 1]);
                const uint32_t h = __builtin_bit_cast(uint32_t, hi);
                const half2_t low = {(_Float16)less_low(p[e], h), (_Float16)less_high(p[e + 1], h)};
                hw[e / 2] = h;
                lw[e / 2] = h2_bits(low) | (INT8 ? 0u : ones_of(h));
            }
            pb[j] = __builtin_bit_cast(h8, hw);
            pl[j] = __builtin_bit_cast(h8, lw);
        }
        // O^T += V^T P^T: the lane's d (li of tile t) of keys 4 lg + [0, 4) of both blocks
        if (full) {
#pragma unroll
            for (int t = 0; t < NT; t++) {
                const h8 va = __builtin_bit_cast(h8, v_piece(tile, t));
#pragma unroll
                for (int j = 0; j < NR; j++) acc[j][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, pb[j], acc[j][t], 0, 0, 0);
#pragma unroll
                for (int j = 0; j < NR; j++) acc[j][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, pl[j], acc[j][t], 0, 0, 0);
            }
            return;
        }
        // a tile with keys that are none, or that some columns do not see
        const uint32_t keys = keys_of(p0, v0, v1, lg);
        uint32_t mask[4];
#pragma unroll
        for (int e = 0; e < 4; e++) mask[e] = (keys >> (2 * e) & 1 ? 0xFFFFu : 0u) | (keys >> (2 * e + 1) & 1 ? 0xFFFF0000u : 0u);
#pragma unroll
        for (int t = 0; t < NT; t++) {
            u32x4a w = v_piece(tile, t);
#pragma unroll
            for (int e = 0; e < 4; e++) w[e] &= mask[e];           // what a slot without a key holds may be NaN
            if (WINDOW && !INT8) {
                // infinities and NaN out of the product, and into the columns that see them
                u32x4a odd, nan, neg;
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    odd[e] = ((w[e] & 0x7C007C00u) + 0x04000400u) >> 15 & 0x00010001u;
                    nan[e] = ((w[e] & 0x03FF03FFu) + 0x03FF03FFu) >> 10 & 0x00010001u;
                    neg[e] = w[e] >> 15 & 0x00010001u;
                }
                if (__builtin_amdgcn_ballot_w64((odd[0] | odd[1] | odd[2] | odd[3]) != 0)) {
#pragma unroll
                    for (int kind = 0; kind < 3; kind++) {         // +inf, -inf, NaN
                        u32x4a at;
#pragma unroll
                        for (int e = 0; e < 4; e++)
                            at[e] = (odd[e] & (kind == 2 ? nan[e] : ~nan[e] & (kind == 1 ? neg[e] : ~neg[e])) & 0x00010001u) * 0x3C00u;
                        const float bad = kind == 0 ? INFINITY : (kind == 1 ? -INFINITY : NAN);
#pragma unroll
                        for (int j = 0; j < NR; j++) {
                            const uint32_t seen = seen_by(keys, j, p0, lg);
                            u32x4a on;
#pragma unroll
                            for (int e = 0; e < 4; e++)
                                on[e] = (seen >> (2 * e) & 1 ? 0x3C00u : 0u) | (seen >> (2 * e + 1) & 1 ? 0x3C000000u : 0u);
                            const f32x4p c = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, at), __builtin_bit_cast(h8, on), f32x4p{}, 0, 0, 0);
#pragma unroll
                            for (int r = 0; r < 4; r++)
                                if (c[r] > 0.0f) acc[j][t][r] += bad;
                        }
                    }
#pragma unroll
                    for (int e = 0; e < 4; e++) w[e] &= ~(odd[e] * 0xFFFFu);
                }
            }
            const h8 va = __builtin_bit_cast(h8, w);
#pragma unroll
            for (int j = 0; j < NR; j++) {
                acc[j][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, pb[j], acc[j][t], 0, 0, 0);
                acc[j][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, pl[j], acc[j][t], 0, 0, 0);
            }
        }
    };

    fetch(0);
    there = there_load;
    put(0);
    if (stages > 1) fetch(1);
    auto next = [&](int s) {
        if (s + 1 < stages) {
            put(s + 1);
            if (s + 2 < stages) fetch(s + 2);
        }
    };
    // Two waves share a SIMD: waves 4 to 7 see to the next stages first, 0 to 3 last, so that
    // one's matrix products run beside the other's softmax.  Whole stages have a loop of
    // their own, in which the sums stay in place.
    auto begin = [&](int s) {
        __syncthreads();
        if (wave >= PT_WAVES / 2) next(s);
    };
    auto end = [&](int s) {
        if (wave < PT_WAVES / 2) next(s);
    };
    auto blocks = [&](int s) {                                    // bits of the stage's four blocks
        if (s > 0 && s % 16 == 0) there = there_load;
        return (uint32_t)(there >> 4 * (s % 16)) & 15u;
    };
    int s = 0;
    while (s < stages) {
        uint32_t is = blocks(s);
        while (is == 15u && kv1 - (kv0 + s * PT_STAGE) >= PT_STAGE && (!WINDOW || kv0 + s * PT_STAGE >= lo_max)) {
            begin(s);
            const uint8_t* st = ring + (s & 1) * 2 * HALF;
            const float* sc = sScale + (s & 1) * (3 * PT_STAGE + 4);
            const int p0 = kv0 + s * PT_STAGE;
            if (KW == 2) work(std::true_type{}, st + 32 * wv * ROWB, sc + 32 * wv, p0 + 32 * wv, true, true);
            else {
#pragma unroll 1
                for (int u = 0; u < 2; u++) work(std::true_type{}, st + 32 * u * ROWB, sc + 32 * u, p0 + 32 * u, true, true);
            }
            end(s);
            if (++s == stages) break;
            is = blocks(s);
        }
        if (s == stages) break;
        begin(s);
#pragma unroll 1
        for (int u = KW == 2 ? wv : 0; u < (KW == 2 ? wv + 1 : 2); u++) {
            const int p0 = kv0 + s * PT_STAGE + 32 * u;
            const bool v0 = is >> 2 * u & 1, v1 = is >> (2 * u + 1) & 1;
            if (p0 < kv1 && (v0 || v1)) work(std::false_type{}, ring + (s & 1) * 2 * HALF + 32 * u * ROWB, sScale + (s & 1) * (3 * PT_STAGE + 4) + 32 * u, p0, v0, v1);
        }
        end(s);
        s++;
    }
    __syncthreads();

    // the waves' states: [wave][32][LD] numerators, then m, l and the numerators' factor [wave][32]
    float* smem = (float*)ring;
    float* sO = smem + (size_t)wave * 32 * LD;
    float* sML = smem + (size_t)PT_WAVES * 32 * LD;
    float* sF = sML + 2 * PT_WAVES * 32;
#pragma unroll
    for (int j = 0; j < NR; j++) {
        const float sum = rows_op(L[j], true) * (1.0f / PT_LIFT);
        float f = 1.0f / PT_LIFT;
        if (INT8) f = M[j] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(M[j] - base_of(m[j])) * (1.0f / PT_LIFT);
#pragma unroll
        for (int t = 0; t < NT; t++) {
            f32x4p x = acc[j][t];
            if (WINDOW && dead[j]) x = f32x4p{};       // (without a window only columns that are none)
            *(f32x4p*)(sO + (16 * j + li) * LD + 16 * t + 4 * lg) = x;
        }
        if (lg == 0) {
            sML[wave * 32 + 16 * j + li] = dead[j] ? -INFINITY : m[j];
            sML[(PT_WAVES + wave) * 32 + 16 * j + li] = dead[j] ? 0.0f : sum;
            sF[wave * 32 + 16 * j + li] = WINDOW && dead[j] ? 0.0f : f;
            const int c = c0 + 16 * j, b = c / G;
            sAt[32 * rg + 16 * j + li] = b * a.n_heads + kvh * G + (c - b * G);
        }
    }
    __syncthreads();
    // join of the key waves in wave order: a thread a column, for the factors, then four d a thread
    const int64_t step = (int64_t)a.B * a.n_heads;
    float2* oml = (float2*)(a.prefix + 4) + part * step;
    float* onum = a.prefix + prefix_num_at(a.prefix_splits, step) + part * step * HD;
    if (tid < COLS && tile * COLS + tid < cols) {
        const int w0 = tid / 32 * KW, cc = tid % 32;
        float top = sML[w0 * 32 + cc], den = sML[(PT_WAVES + w0) * 32 + cc];
        if (KW == 2) {
            const float m0 = top, m1 = sML[(w0 + 1) * 32 + cc];
            top = fmaxf(m0, m1);
            const float tb = base_of(top), f0_ = __builtin_amdgcn_exp2f(m0 - tb), f1_ = __builtin_amdgcn_exp2f(m1 - tb);
            den = f0_ * den + f1_ * sML[(PT_WAVES + w0 + 1) * 32 + cc];
            sF[w0 * 32 + cc] *= f0_;
            sF[(w0 + 1) * 32 + cc] *= f1_;
        }
        oml[sAt[tid]] = make_float2(top, den);
    }
    if (KW == 2) __syncthreads();
    constexpr int EACH = COLS * (HD / 4) / (64 * PT_WAVES);
#pragma unroll 4
    for (int i = 0; i < EACH; i++) {
        const int e = tid + i * 64 * PT_WAVES, cl = e / (HD / 4), d = 4 * (e % (HD / 4));
        if (tile * COLS + cl >= cols) break;
        const int w0 = cl / 32 * KW, cc = cl % 32;
        f32x4p num = sF[w0 * 32 + cc] * *(const f32x4p*)(smem + ((size_t)w0 * 32 + cc) * LD + d);
        if (KW == 2) num += sF[(w0 + 1) * 32 + cc] * *(const f32x4p*)(smem + ((size_t)(w0 + 1) * 32 + cc) * LD + d);
        *(f32x4p*)(onum + (int64_t)sAt[cl] * HD + d) = num;
    }
}

template <bool INT8, int HD, int RW, bool WINDOW>
hipError_t tile_go(const PagedAttnArgs& a, const PagedPrefixArgs& pre, const PrefixPlan& p, hipStream_t st) {
    constexpr int LDS = pt_lds<INT8, HD>();
    if (const hipError_t e = allow_lds<prefix_tile_kernel<INT8, HD, RW, WINDOW>>(LDS)) return e;
    hipLaunchKernelGGL((prefix_tile_kernel<INT8, HD, RW, WINDOW>), dim3((unsigned)p.tiles * (unsigned)a.n_kv * (unsigned)a.prefix_splits),
                       dim3(64 * PT_WAVES), LDS, st, a, pre);
    return hipGetLastError();
}

template <bool INT8, int HD, int NR, int RW, bool WINDOW>
hipError_t prefix_go(const PagedAttnArgs& a, const PagedPrefixArgs& pre, const PrefixPlan& p, hipStream_t st) {
    constexpr size_t lds = (size_t)PA_WAVES * 16 * NR * (HD + 4 + 2) * 4;
    if (const hipError_t e = allow_lds<paged_prefix_kernel<INT8, HD, NR, RW, WINDOW>>((int)lds)) return e;
    hipLaunchKernelGGL((paged_prefix_kernel<INT8, HD, NR, RW, WINDOW>), dim3((unsigned)p.tiles * (unsigned)a.n_kv * (unsigned)a.prefix_splits),
                       dim3(64 * PA_WAVES), lds, st, a, pre);
    return hipGetLastError();
}

template <bool INT8, int HD>
hipError_t prefix_hd(const PagedAttnArgs& a, const PagedPrefixArgs& pre, const PrefixPlan& p, hipStream_t st) {
    if (a.window > 0) {
        if (p.lds) return p.rw == 8 ? tile_go<INT8, HD, 8, true>(a, pre, p, st) : tile_go<INT8, HD, 4, true>(a, pre, p, st);
        return p.rw == 1 ? prefix_go<INT8, HD, 1, 1, true>(a, pre, p, st) : (p.rw == 2 ? prefix_go<INT8, HD, 1, 2, true>(a, pre, p, st) : prefix_go<INT8, HD, 1, 4, true>(a, pre, p, st));
    }
    if (p.lds) return p.rw == 8 ? tile_go<INT8, HD, 8, false>(a, pre, p, st) : tile_go<INT8, HD, 4, false>(a, pre, p, st);
    if (p.nr == 1) return prefix_go<INT8, HD, 1, 1, false>(a, pre, p, st);
    return p.rw == 1 ? prefix_go<INT8, HD, 2, 1, false>(a, pre, p, st) : prefix_go<INT8, HD, 2, 2, false>(a, pre, p, st);
}
}  // namespace

int paged_prefix_splits(int B, int n_heads, int n_kv, int max_prefix, int window, bool kv_int8) {
    return prefix_plan(B, n_heads, n_kv, max_prefix, window, kv_int8).splits;
}

int64_t paged_prefix_blocks(int B, int n_heads, int n_kv, int max_prefix, int window, bool kv_int8) {
    const PrefixPlan p = prefix_plan(B, n_heads, n_kv, max_prefix, window, kv_int8);
    return (int64_t)p.tiles * n_kv * p.splits;
}

int64_t paged_prefix_workspace(int B, int n_heads, int n_kv, int head_dim, int max_prefix, int window, bool kv_int8) {
    const int64_t splits = paged_prefix_splits(B, n_heads, n_kv, max_prefix, window, kv_int8), step = (int64_t)B * n_heads;
    return (prefix_num_at(splits, step) + splits * step * head_dim) * 4;
}

hipError_t paged_prefix_launch(const PagedAttnArgs& a, const PagedPrefixArgs& pre, bool kv_int8, hipStream_t st) {
    const PrefixPlan p = prefix_plan(a.B, a.n_heads, a.n_kv, pre.max_len, a.window, kv_int8);
    switch (a.head_dim + (kv_int8 ? 1 : 0)) {
    case 32:  return prefix_hd<false, 32>(a, pre, p, st);
    case 33:  return prefix_hd<true, 32>(a, pre, p, st);
    case 64:  return prefix_hd<false, 64>(a, pre, p, st);
    case 65:  return prefix_hd<true, 64>(a, pre, p, st);
    case 96:  return prefix_hd<false, 96>(a, pre, p, st);
    case 97:  return prefix_hd<true, 96>(a, pre, p, st);
    case 128: return prefix_hd<false, 128>(a, pre, p, st);
    case 129: return prefix_hd<true, 128>(a, pre, p, st);
    default: return hipErrorInvalidValue;
    }
}

}  // namespace jllm_hip
