// paged_attention.hip -- decode attention of a batch of query rows, each over the
// pages of its own sequence, gfx950.
//
//   s_t = scale * ks_t * (q . k_t),  out = sum_t e^(s_t - m) vs_t v_t / sum_t e^(s_t - m)
//
// over the keys t of the row: [max(0, len - window), len).  Key t lies in slot
// t % page_size of page table[row][t / page_size].
//
// One pass over K and V, all query heads of a KV head together.  The keys of all
// rows are dealt out to as many workgroups as the card holds, in equal parts whatever
// the rows' lengths are (the host knows only their maximum), and joined.  A wave takes
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
// Sums, maxima and accumulators are fp32.  For the matrix cores a weight is split into
// two fp16 parts, as in the other attention kernels: together within 2^-21
// of the weight, so the output's rounding is the only one to 11 bits (with one part,
// 2^-12 of sum w |v|, values that cancel lost their difference).  The second product
// and the split cost 0.5 % of 24 fp16 rows of up to 16384, 1.5 % of 48 INT8 rows of up
// to 4096 and at most 2.5 % (64 INT8 rows of 4 / 1 heads x 32, 15.2 us).  The parts are
// of the weight times 2^14, so that they become subnormal only below 2^-28 of the largest.
// With int8 the V scales go into the exponent, e^(s_t - m) vs_t = 2^(s'_t + log2
// vs_t), with a maximum of their own: no scale overflows the weights (below 1e34 the
// fp32 sums neither) or swamps the others, and a scale of 0 is a weight of 0.
//
// Measured (32 / 8 heads x 128, both launches): 131072 fp16 keys of one row 92 us and
// 24 rows of up to 16384 103 us (5.8 TB/s: the reads are the bound), 48 INT8 rows of
// up to 4096 39.8 us (3.8 TB/s; start, join and the scales' lines are the rest), one
// INT8 row of 700 9.3 us.
#include "attention.h"
#include "attn_common.h"
#include "serving.h"

namespace jllm_hip {

typedef float f32x4p __attribute__((ext_vector_type(4)));
template <typename T> using global_ptr = const __attribute__((address_space(1))) T*;
template <bool ONCE, typename T>
__device__ __forceinline__ T load_once(global_ptr<T> p) {
    if (ONCE) return __builtin_nontemporal_load(p);
    return *p;
}

constexpr int PA_TILE = 32;            // keys a wave takes at once
constexpr int PA_BLOCK = 16;           // keys behind one base address
constexpr int PA_PASS = 1024;          // keys whose pages a wave looks up at once: a block per lane
constexpr int PA_WAVES = 4;
constexpr int PA_MAX_ROWS = 1024;      // rows that a workgroup counts through (16 per lane)
constexpr float PA_LIFT = 16384.0f;    // factor on the weights' fp16 parts
constexpr float PA_LOG2E = 1.44269504088896340736f;

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

// How the keys are dealt out.  A unit is a tile for each of the waves that share a
// KV head.
//   whole: a workgroup per row (and heads): writes the row's output itself
//   else: the units of all rows, one row behind the other, cut into nw equal parts
//     whatever the rows' lengths are; a part may hold pieces of several rows, a row
//     pieces of several parts.  Piece (part w, row b) has partial w + b.  A row in
//     one piece is written by its workgroup, the others by the join, which a row's
//     first piece tells where they lie.
struct PagedPlan { int whole, nw, heads; };

struct RowKeys { int lo, base, len; };                 // keys [lo, len); base: lo rounded down to a block
__device__ __forceinline__ RowKeys row_keys(const PagedAttnArgs& a, int len) {
    RowKeys r;
    r.len = len < 0 ? 0 : (len > a.max_seq ? a.max_seq : len);
    r.lo = a.window > 0 && r.len > a.window ? r.len - a.window : 0;
    r.base = r.lo & ~(PA_BLOCK - 1);
    return r;
}
__device__ __forceinline__ int row_units(const RowKeys& r, int unit) { return (int)(((unsigned)(r.len - r.base) + unit - 1) / (unsigned)unit); }

template <int CTRL, int ROWS>
__device__ __forceinline__ int dpp_add(int v) { return v + __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xF, false); }
// inclusive prefix sum over the wave
__device__ __forceinline__ int wave_scan(int v) {
    v = dpp_add<0x111, 0xF>(v);     // row_shr 1, 2, 4, 8
    v = dpp_add<0x112, 0xF>(v);
    v = dpp_add<0x114, 0xF>(v);
    v = dpp_add<0x118, 0xF>(v);
    v = dpp_add<0x142, 0xA>(v);     // row_bcast 15 to rows 1 and 3
    v = dpp_add<0x143, 0xC>(v);     // row_bcast 31 to rows 2 and 3
    return v;
}
// units of row r, 0 behind the last row
__device__ __forceinline__ int units_of(const PagedAttnArgs& a, int r, int unit, int& len) {
    len = r < a.B ? a.lens[r] : 0;
    return row_units(row_keys(a, len), unit);
}
// first unit of part w when total units are cut into n parts
__device__ __forceinline__ int part_begin(int total, int n, int w) {
    const int q = total / n, rem = total - q * n;
    return w * q + min(w, rem);
}
// the part that unit u falls into
__device__ __forceinline__ int part_of(int total, int n, int u) {
    const int q = total / n, rem = total - q * n;
    return u < rem * (q + 1) ? u / (q + 1) : rem + (u - rem * (q + 1)) / q;
}
// Parts of total units: a workgroup on every CU as long as each has a unit, more (up
// to nw, three on every CU) only with two units each: 17 rows with a window of 1024
// 9.6 us against 12.7 with two units from the start, one row of 2000 9.0 against 10.0,
// but 8 rows of 1500 16.3 with single units throughout against 15.3.
__device__ __forceinline__ int parts_of(int total, int nw) {
    return max(1, min(nw, max(total / 2, min(total, nw / 3))));
}

// the weights' exponent base: a row without a finite score yet has base 0
__device__ __forceinline__ float base_of(float m) { return m == -INFINITY ? 0.0f : m; }

// WHOLE: a workgroup per row, without the code of the parts (one row of 30 keys 5.4 us
// with both in one kernel)
template <bool INT8, int HD, int HW, bool WHOLE>
__global__ __launch_bounds__(64 * PA_WAVES, 3)
void paged_attn_kernel(PagedAttnArgs a, PagedPlan plan) {
    constexpr int EB = INT8 ? 1 : 2;
    constexpr int W = PA_WAVES / HW;                   // waves that share a KV head's keys
    constexpr int UNIT = PA_TILE * W;
    constexpr int NST = HD / 32;                       // Q.K^T steps
    constexpr int KC = INT8 ? HD / 64 : HD / 32;       // 16-byte pieces of a K row per lane
    constexpr bool KT = INT8 && HD % 64 != 0;          // and an 8-byte one
    constexpr int NT = HD / 16;                        // 16-wide d tiles of O
    constexpr int V0 = HD == 96 ? 4 : NT;              // neighbouring d per lane, first part ...
    constexpr int V1 = NT - V0;                        // ... and second (from d = 64)
    constexpr int W0 = (V0 * EB + 3) / 4, W1 = (V1 * EB + 3) / 4, VW = W0 + W1;   // in words
    // V rows that one load reads in whole lines are not kept in the caches, where they
    // would push out lines of which half is still to be read (K's: a load reads 64
    // bytes of a row): 24 fp16 rows of up to 16384 118 -> 110 us, 48 INT8 rows of up to
    // 4096 44.2 -> 39.2.  Rows read in pieces, and K, lose by it (17 rows of head_dim
    // 96: 9.9 -> 10.4; K 3 %).
    constexpr bool VONCE = V1 == 0 && HD * EB % 128 == 0;
    constexpr int LD = HD + 4;
    extern __shared__ __attribute__((aligned(16))) float smem[];

    const unsigned hg = (unsigned)a.n_kv / HW, part = blockIdx.x / hg;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), hs = wave % HW, wv = wave / HW;
    const int kvh = (int)(blockIdx.x - part * hg) * HW + hs;
    const int lane = (int)threadIdx.x & 63;
    const int G = a.n_heads / a.n_kv;
    float* sH = smem + (size_t)hs * W * (G * LD + 32);  // this KV head's part: numerators [W][G], m [W][16], l [W][16]
    float* sO = sH + (size_t)wv * G * LD;
    float* sML = sH + (size_t)W * G * LD;

    // the part's units [at, end), and the rows that they lie in
    // (two levels: lane j counts rows j span + [0, span); of the group that a unit
    // falls into the rows go to the lanes.  Up to 64 rows are one group.)
    const int span = a.B <= 64 ? 64 : (a.B + 63) / 64;
    int at = 0, end = 0, total = 0, n_parts = 1;
    int group = 0, gincl = 0, lens = 0, incl = 0;       // incl: units up to the lane's row
    auto enter_group = [&](int g, int base) {
        group = g * span;
        incl = base + wave_scan(lane < span ? units_of(a, group + lane, UNIT, lens) : 0);
    };
    if (!WHOLE) {
        if (a.B <= 64) {
            enter_group(0, 0);
            total = __builtin_amdgcn_readlane(incl, 63);
        } else {
            int x, sum = 0;
#pragma unroll 4
            for (int i = 0; i < span; i++) sum += units_of(a, lane * span + i, UNIT, x);
            gincl = wave_scan(sum);
            total = __builtin_amdgcn_readlane(gincl, 63);
        }
        n_parts = parts_of(total, plan.nw);
        if ((int)part >= n_parts) return;
        at = part_begin(total, n_parts, (int)part);
        end = part_begin(total, n_parts, (int)part + 1);
        if (at >= end) return;
    }

  do {
    // what follows from the lane is found anew for each piece: kept across the pieces it
    // would take registers that the tiles need (24 fp16 rows of up to 16384 117 us, not 110)
    int l = lane;
    asm("" : "+v"(l));
    const int li = l & 15, lg = l >> 4;
    int b = (int)part, u0 = 0, u1 = 0, units = 0, len; // row, its units [u0, u1) that are this piece
    if (WHOLE) {
        len = a.lens[b];
    } else {
        uint64_t beyond = __builtin_amdgcn_ballot_w64(incl > at);
        if (!beyond) {                                 // (more than 64 rows only)
            const int g = __builtin_ctzll(__builtin_amdgcn_ballot_w64(gincl > at));
            enter_group(g, g > 0 ? __builtin_amdgcn_readlane(gincl, g - 1) : 0);
            beyond = __builtin_amdgcn_ballot_w64(incl > at);
            if (!beyond) return;                       // (lengths that changed since they were counted)
        }
        const int j = __builtin_ctzll(beyond);
        b = group + j;
        len = __builtin_amdgcn_readlane(lens, j);
        units = row_units(row_keys(a, len), UNIT);
        const int first = __builtin_amdgcn_readlane(incl, j) - units;
        u0 = at - first;
        u1 = min(units, end - first);
        at = first + u1;
        // a row's first piece tells the join how many there are
        if (u0 == 0 && blockIdx.x == part * hg && threadIdx.x == 0) {
            int2* pieces = (int2*)(a.part + (int64_t)(plan.nw + a.B) * a.n_heads * (2 + HD));
            pieces[b] = make_int2((int)part, u1 == units ? 1 : part_of(total, n_parts, first + units - 1) - (int)part + 1);
        }
    }
    const RowKeys keys = row_keys(a, len);
    const int lo = keys.lo;
    if (WHOLE) u1 = units = row_units(keys, UNIT);
    uint16_t* out = a.out + ((int64_t)b * a.n_heads + kvh * G) * HD;
    if (units == 0) {                                  // (whole rows only: pieces have units)
        for (int i = wv * 64 + l; i < G * HD; i += 64 * W) out[i] = 0;
        return;
    }
    // (key numbers up to 2^31: sums that may pass it are unsigned)
    const int kv0 = keys.base + u0 * UNIT, kv1 = (int)min((unsigned)keys.base + (unsigned)u1 * UNIT, (unsigned)keys.len);

    // Passes of 1024 keys: lane j looks up block j, one pass ahead.
    auto look_up = [&](unsigned k0) {
        const unsigned t = k0 + PA_BLOCK * l;
        return t < (unsigned)kv1 ? a.table[b * a.table_stride + (t >> a.page_shift)] : -1;
    };
    int pass = kv0, slot0 = 0;
    uint64_t there = 0, todo = 0;                      // blocks of the pass that are there; this wave's tiles of those (bit 2 i)
    int pg = look_up(kv0);
    auto enter = [&](unsigned k0) {
        pass = (int)k0;
        const unsigned t = k0 + PA_BLOCK * l;
        there = __builtin_amdgcn_ballot_w64(t < (unsigned)kv1 && (unsigned)pg < (unsigned)a.n_pages);
        slot0 = (pg << a.page_shift) + (int)(t & ((1u << a.page_shift) - 1));
        todo = (there | (there >> 1)) & ((~(uint64_t)0 / (((uint64_t)1 << 2 * W) - 1)) << (2 * wv));
        pg = look_up(k0 + PA_PASS);
    };
    enter(kv0);

    const uint32_t row = (uint32_t)a.n_kv * a.cache_head_dim * EB;      // bytes
    const int64_t hoff = (int64_t)kvh * a.cache_head_dim * EB;

    // the wave's next tile: its first key, the slots of its blocks (a missing one
    // takes the other's), which are there; p0 < 0: none
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
        x.s0 = __builtin_amdgcn_readfirstlane(x.v0 ? p : q);     // (scalar base addresses)
        x.s1 = __builtin_amdgcn_readfirstlane(x.v1 ? q : p);
        return x;
    };

    // (zeroed: some dozen instructions a wave, so that no path has them undefined.  The
    // listings show no need: with and without, no word of a loaded row is written
    // before it is read in the loop.)
    u32x4a rk[2][KC > 0 ? KC : 1] = {};
    u32x2a rt[2] = {};
    uint32_t rv[8][VW] = {};
    float rs = 1.0f;
    // A block's base address stays scalar, the lane's offset 32 bits (both opaque, or
    // the compiler keeps a 64-bit address per load, which costs a wave per SIMD).
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
                if (V0 * EB == 16) { const u32x4a w = load_once<VONCE>((global_ptr<u32x4a>)x); v[0] = w.x; v[1 % VW] = w.y; v[2 % VW] = w.z; v[3 % VW] = w.w; }
                else if (V0 * EB == 8) { const u32x2a w = load_once<VONCE>((global_ptr<u32x2a>)x); v[0] = w.x; v[1 % VW] = w.y; }
                else if (V0 * EB == 4) v[0] = *(global_ptr<uint32_t>)x;
                else v[0] = *(global_ptr<uint16_t>)x;
                if (V1 > 0) {
                    const uint64_t y = p + o1[r] + 64 * EB;
                    v[VW - 1] = V1 * EB == 4 ? *(global_ptr<uint32_t>)y : *(global_ptr<uint16_t>)y;
                }
            }
        }
    };

    Tile cur = next_tile();
    if (cur.p0 >= 0) {
        load_k(cur.s0, cur.s1);
        load_v(cur.s0, cur.s1);
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

    while (cur.p0 >= 0) {
        const int p0 = cur.p0;
        const bool v0 = cur.v0, v1 = cur.v1;
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
        const Tile next = next_tile();
        if (next.p0 >= 0) load_k(next.s0, next.s1);
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
        const bool full = v0 && v1 && p0 >= lo && kv1 - p0 >= PA_TILE;
        uint32_t live = 0xFFu;                         // bit e: the lane's key e counts
        if (!full) {
            live = 0;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const int o = PA_BLOCK * (e >> 2) + 4 * lg + (e & 3);      // key p0 + o
                if ((e < 4 ? v0 : v1) && o >= lo - p0 && o < kv1 - p0) live |= 1u << e;
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
            p[e] = __builtin_amdgcn_exp2f(s[e] - mb);
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
            for (int e = 0; e < 8; e++) p[e] = __builtin_amdgcn_exp2f(t[e] - Mb);
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
        // p * PA_LIFT in two parts, each rounded down.  fp16 V may be infinite, and 0 * inf
        // is no part of inf: there the low part of a weight that is not 0 gets its last bit.
        u32x4a hw, lw;
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
            const float x = p[e] * PA_LIFT, y = p[e + 1] * PA_LIFT;
            const auto hi = __builtin_amdgcn_cvt_pkrtz(x, y);
            const auto lo = __builtin_amdgcn_cvt_pkrtz(x - (float)hi[0], y - (float)hi[1]);
            const uint32_t h = __builtin_bit_cast(uint32_t, hi);       // (no sign bits)
            hw[e / 2] = h;
            lw[e / 2] = __builtin_bit_cast(uint32_t, lo) | (INT8 ? 0u : (h + 0x7FFF7FFFu) >> 15 & 0x00010001u);
        }
        const h8 pb = __builtin_bit_cast(h8, hw), pl = __builtin_bit_cast(h8, lw);
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
            acc[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, va), pl, acc[j], 0, 0, 0);
        }
        if (INT8) {
            wsum = __builtin_amdgcn_mfma_f32_16x16x32_f16(ones, pb, wsum, 0, 0, 0);
            wsum = __builtin_amdgcn_mfma_f32_16x16x32_f16(ones, pl, wsum, 0, 0, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
        if (next.p0 >= 0) load_v(next.s0, next.s1);
        cur = next;
    }

    // the wave's state: m, l, numerators; acc[j][r] is d = V0 (4 lg + r) + j, or 64 + V1 (4 lg + r) + j - V0
    L = rows_op(L, true);
    if (INT8) {
        // (no V scale but 0: the numerators are 0, and with the base of an M of -inf the
        // factor would be infinite under scores below -2^7)
        const float f = M == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(M - base_of(m)) * (1.0f / PA_LIFT);
#pragma unroll
        for (int j = 0; j < NT; j++)
#pragma unroll
            for (int r = 0; r < 4; r++) acc[j][r] = (acc[j][r] * 16777216.0f - 128.0f * wsum[0]) * f;
    } else {
#pragma unroll
        for (int j = 0; j < NT; j++) acc[j] *= 1.0f / PA_LIFT;
    }
    if (li < G) {
#pragma unroll
        for (int j = 0; j < NT; j++)
#pragma unroll
            for (int r = 0; r < 4; r++)
                sO[li * LD + (j < V0 ? V0 * (4 * lg + r) + j : 64 + V1 * (4 * lg + r) + j - V0)] = acc[j][r];
    }
    if (l < 16) { sML[wv * 16 + l] = m; sML[(W + wv) * 16 + l] = L; }
    __syncthreads();
    // join of the waves in wave order
    for (int e = wv * 64 + l; e < G * HD; e += 64 * W) {
        const int h = e / HD, d = e % HD;
        float top = sML[h];
#pragma unroll
        for (int w = 1; w < W; w++) top = fmaxf(top, sML[w * 16 + h]);
        const float tb = base_of(top);
        float num = 0.0f, den = 0.0f;
#pragma unroll
        for (int w = 0; w < W; w++) {
            const float f = __builtin_amdgcn_exp2f(sML[w * 16 + h] - tb);
            num += f * sH[((size_t)w * G + h) * LD + d];
            den += f * sML[(W + w) * 16 + h];
        }
        if (u1 - u0 == units) {
            // no key of finite score: zero; a NaN stays
            out[e] = f32_to_f16_bits(den == 0.0f ? 0.0f : num / den);
        } else {
            const int64_t n = (int64_t)(plan.nw + a.B) * a.n_heads, at_ = ((int64_t)part + b) * a.n_heads + kvh * G + h;
            a.part[2 * n + at_ * HD + d] = num;
            if (d == 0) { a.part[at_] = top; a.part[n + at_] = den; }
        }
    }
    if (!WHOLE && at < end) __syncthreads();      // the next piece writes the states again
  } while (!WHOLE && at < end);
}

// out = sum_s 2^(m_s - M) num_s / sum_s 2^(m_s - M) l_s over the pieces of a row that
// has several, in a fixed order: wave w of the head's workgroup adds pieces w, w + NW,
// ..., lane l d = 2 l and 2 l + 1; then the waves' sums in wave order.  Rows without a
// key are written here too.
template <int NW>
__global__ __launch_bounds__(64 * NW) void paged_join_kernel(PagedAttnArgs a, PagedPlan plan) {
    constexpr int AHEAD = 8;                           // pieces a wave has on the way
    __shared__ float sTop[NW], sDen[NW];
    __shared__ float sSum[NW][128];
    const int b = blockIdx.y, h = blockIdx.x, hd = a.head_dim;
    const int w = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), l = (int)threadIdx.x & 63;
    const int64_t slots = (int64_t)(plan.nw + a.B) * a.n_heads;
    const int2 pieces = *(const int2*)(a.part + slots * (2 + hd) + 2 * b);      // first part, count; of rows that have keys
    uint32_t* out = (uint32_t*)(a.out + ((int64_t)b * a.n_heads + h) * hd + 2 * l);
    if (row_keys(a, a.lens[b]).len == 0) {
        if (w == 0 && 2 * l < hd) *out = 0;
        return;
    }
    // (bounded, so that lengths or a workspace that others write meanwhile spoil values only)
    const int w0 = min(max(pieces.x, 0), plan.nw - 1), ns = min(pieces.y, plan.nw - w0);
    if (ns <= 1) return;
    const int64_t n = slots, at = ((int64_t)w0 + b) * a.n_heads + h;
    const int64_t H = a.n_heads;
    const float* pm = a.part + at;
    const float* pl = a.part + n + at;
    const float* pn = a.part + 2 * n + at * hd + (2 * l < hd ? 2 * l : 0);
    // a wave's first pieces set out together with the maxima
    float2 v[AHEAD];
    float pmax[AHEAD], psum[AHEAD];
    auto load = [&](int s0) {
#pragma unroll
        for (int i = 0; i < AHEAD; i++) {
            const int s = s0 + NW * i;
            const bool is = s < ns;
            v[i] = is ? *(const float2*)(pn + s * H * hd) : make_float2(0.0f, 0.0f);
            pmax[i] = is ? pm[s * H] : -INFINITY;
            psum[i] = is ? pl[s * H] : 0.0f;
        }
    };
    load(w);
    float top = -INFINITY;
    for (int s = (int)threadIdx.x; s < ns; s += 64 * NW) top = fmaxf(top, pm[s * H]);
    top = wave_max(top);
    if (NW > 1) {
        if (l == 0) sTop[w] = top;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < NW; i++) top = fmaxf(top, sTop[i]);
    }
    const float tb = base_of(top);
    float den = 0.0f;
    float2 num = make_float2(0.0f, 0.0f);
    for (int s0 = w; s0 < ns; s0 += NW * AHEAD) {
        if (s0 > w) load(s0);
#pragma unroll
        for (int i = 0; i < AHEAD; i++) {
            const float f = __builtin_amdgcn_exp2f(pmax[i] - tb);
            den += f * psum[i];
            num.x += f * v[i].x;
            num.y += f * v[i].y;
        }
    }
    if (NW > 1) {
        sSum[w][2 * l] = num.x;
        sSum[w][2 * l + 1] = num.y;
        if (l == 0) sDen[w] = den;
        __syncthreads();
        if (w > 0) return;
#pragma unroll
        for (int i = 1; i < NW; i++) {
            num.x += sSum[i][2 * l];
            num.y += sSum[i][2 * l + 1];
            den += sDen[i];
        }
    }
    if (2 * l < hd) {
        const float x = den == 0.0f ? 0.0f : num.x / den, y = den == 0.0f ? 0.0f : num.y / den;
        *out = (uint32_t)f32_to_f16_bits(x) | ((uint32_t)f32_to_f16_bits(y) << 16);
    }
}

namespace {
// Whole rows where the longest is short: the join and its launch cost more than the
// cut gains (32 / 8 heads x 128, whole against cut: 1 row of 400 fp16 keys 8.2 us
// against 9.8, of 600 9.7 against 8.8, of 1000 13.2 against 9.0; 16 rows of 700 13.1
// against 15.2; 64 of 1000 54 against 60; 256 of 700 INT8 77 against 100; 8 of 1500 20.5
// against 15.4).
// Also for more rows than PA_MAX_ROWS: that is as far as a workgroup counts through all
// lengths, no gain.  1500 rows up to 2000 of 4 / 1 heads x 32 29 us whole, 38 cut, and 1500
// INT8 rows of 1100 of 16 / 2 heads 161 against 189, but 1100 fp16 rows up to 1200 101
// against 84, and one long row among them is a single workgroup's, 8 us for 1000 keys.
// Parts: as many as the card holds at once, three workgroups on each of 256 CUs.
// Heads per workgroup: KV heads that run side by side read neighbouring pieces of the
// same rows.  Pieces under 128 bytes share their lines (all lengths drawn; one head
// against two: 128 INT8 rows up to 4000 of 8 heads x 64 78.5 us against 62.1, of 2 x 64
// up to 8000 38.1 against 30.5; 128 fp16 rows up to 8000 of 4 x 32 60.3 against 45.4).
// Whole lines gain little, and with few heads lose (24 fp16 rows of 8 x 128 up to 16384
// 109.9 against 107.9, 16 INT8 rows of 8192 69 against 64; 64 INT8 rows up to 16000 of
// 2 x 128 46.9 against 49.5, with 4 heads the same).  Both only while the two waves that
// are left per head have enough of a row: the least number of keys over all heads from
// which it pays is 2^19 up to 128 bytes and 2^20 from there (16 INT8 rows up to 2000 of
// 2 x 64 9.3 against 9.8; 40 fp16 rows up to 1700 of 8 x 128 23.8 against 25.7).
// piece: bytes of a key's row of one head.
PagedPlan plan_of(int B, int n_kv, int max_seq, int window, int piece) {
    int64_t span = max_seq;
    if (window > 0 && window + (int64_t)PA_BLOCK - 1 < span) span = window + (int64_t)PA_BLOCK - 1;
    const int64_t rows = (int64_t)(B > 0 ? B : 1) * n_kv;
    PagedPlan p;
    p.whole = !attn_splitk_enabled() || span <= (rows >= 128 ? 1024 : 512) || B > PA_MAX_ROWS ||
              B * ((span + PA_TILE - 1) / PA_TILE) > (1 << 30);
    if (p.whole) p.heads = rows >= 2048 ? 4 : (rows >= 512 ? 2 : 1);
    else p.heads = rows * span >= (piece <= 128 ? 1 << 19 : 1 << 20) && (piece < 128 || n_kv >= 8) ? 2 : 1;
    while (n_kv % p.heads) p.heads /= 2;
    const int hg = n_kv / p.heads;
    p.nw = p.whole ? 0 : (768 / hg > 1 ? 768 / hg : 1);
    return p;
}

template <bool INT8, int HD>
void paged_go(const PagedAttnArgs& a, const PagedPlan& p, hipStream_t st) {
    const dim3 grid((unsigned)(a.n_kv / p.heads) * (unsigned)(p.whole ? a.B : p.nw));
    const size_t lds = (size_t)PA_WAVES * (a.n_heads / a.n_kv * (HD + 4) + 32) * 4;
    switch (p.heads + (p.whole ? 0 : 4)) {
    case 1:  hipLaunchKernelGGL((paged_attn_kernel<INT8, HD, 1, true>), grid, dim3(64 * PA_WAVES), lds, st, a, p); break;
    case 2:  hipLaunchKernelGGL((paged_attn_kernel<INT8, HD, 2, true>), grid, dim3(64 * PA_WAVES), lds, st, a, p); break;
    case 4:  hipLaunchKernelGGL((paged_attn_kernel<INT8, HD, 4, true>), grid, dim3(64 * PA_WAVES), lds, st, a, p); break;
    case 5:  hipLaunchKernelGGL((paged_attn_kernel<INT8, HD, 1, false>), grid, dim3(64 * PA_WAVES), lds, st, a, p); break;
    default: hipLaunchKernelGGL((paged_attn_kernel<INT8, HD, 2, false>), grid, dim3(64 * PA_WAVES), lds, st, a, p); break;
    }
}
}  // namespace

int64_t paged_attn_blocks(int B, int n_kv, int max_seq, int window) {
    // (of wide rows, whose workgroups take fewer heads)
    const PagedPlan p = plan_of(B, n_kv, max_seq, window, 256);
    return (int64_t)(n_kv / p.heads) * (p.whole ? B : p.nw);
}

int64_t paged_attn_workspace(int B, int n_heads, int n_kv, int head_dim, int max_seq, int window) {
    // of int8, which has at least as many parts
    const PagedPlan p = plan_of(B, n_kv, max_seq, window, head_dim);
    if (p.whole) return 0;
    return ((int64_t)(p.nw + B) * n_heads * (2 + head_dim) * 4 + (int64_t)B * 8 + 15) & ~(int64_t)15;
}

hipError_t paged_attn_launch(const PagedAttnArgs& a, bool kv_int8, hipStream_t st) {
    const PagedPlan p = plan_of(a.B, a.n_kv, a.max_seq, a.window, a.head_dim * (kv_int8 ? 1 : 2));
    switch (a.head_dim + (kv_int8 ? 1 : 0)) {
    case 32:  paged_go<false, 32>(a, p, st); break;
    case 33:  paged_go<true, 32>(a, p, st); break;
    case 64:  paged_go<false, 64>(a, p, st); break;
    case 65:  paged_go<true, 64>(a, p, st); break;
    case 96:  paged_go<false, 96>(a, p, st); break;
    case 97:  paged_go<true, 96>(a, p, st); break;
    case 128: paged_go<false, 128>(a, p, st); break;
    case 129: paged_go<true, 128>(a, p, st); break;
    default: return hipErrorInvalidValue;
    }
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || p.whole) return e;
    if (p.nw <= 16 * a.B) hipLaunchKernelGGL((paged_join_kernel<1>), dim3(a.n_heads, a.B), dim3(64), 0, st, a, p);
    else                  hipLaunchKernelGGL((paged_join_kernel<8>), dim3(a.n_heads, a.B), dim3(512), 0, st, a, p);
    return hipGetLastError();
}

}  // namespace jllm_hip
