// gemm_i8.hip -- product of 8-bit codes with a scale for each token and channel, gfx950:
//
//   y[n][m] = xs[n] ws[m] sum_k x[n][k] w[m][k] (+ bias[m])
//
// The sums are int32 on the matrix cores and exact (K <= 131056), whatever their order;
// the fp32 epilogue multiplies by the token's scale, then the channel's.
// Bounds: up to 16 tokens the bytes of W (151936 x 2560 74 us, 5.3 TB/s), but of few channels
// its 16 a workgroup leave CUs idle (2560 x 9728 9.1 us on 160 of 256).  To about 1000 tokens the
// waves wait, for the next stage or at its barrier (64 tokens x 6144 x 2560 8.8 us, 59 % of their
// time; 251 x 32003 x 2064 34.5 us, 42 %).  Beyond, the matrix cores and the clock that their power leaves: 8192^3 492 us,
// 2.23 POP/s, at 1.9 GHz, of whose cycles they are busy 57 %.  There a wave waits 47 % of its
// time, for a stage's barrier or for its operands (a quarter's reads from LDS stand right before
// its matrix instructions, and are waited for); which of them costs more is not measured.
#include "gemm_i8_plan.h"
#include "kq_common.h"
#include "serving.h"

namespace jllm_hip {

typedef int i32x4g __attribute__((ext_vector_type(4)));
typedef int i32x16g __attribute__((ext_vector_type(16)));
typedef uint32_t u32x2g __attribute__((ext_vector_type(2)));
typedef float f32x4g __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) void lds_void_g;

namespace {

// Every form rounds alike, the product before the bias is added (a fused multiply and add
// where the compiler sees both would give a token other bits among many than among few).
__device__ __forceinline__ float scaled_by(int sum, float xs, float ws, bool biased, float bias) {
#pragma clang fp contract(off)
    const float v = (float)sum * xs * ws;
    return biased ? v + bias : v;
}
__device__ __forceinline__ float scaled(const GemmI8Args& a, int sum, float xs, int m) {
    return scaled_by(sum, xs, a.ws[m], a.bias != nullptr, a.bias ? a.bias[m] : 0.0f);
}
__device__ __forceinline__ void store1(const GemmI8Args& a, int n, int m, float v) {
    const int64_t at = (int64_t)n * a.y_stride + m;
    if (a.y_fp32) ((float*)a.y)[at] = v;
    else ((uint16_t*)a.y)[at] = f32_to_f16_bits(v);
}
// Four neighbouring channels m .. m + 3 of token n.
__device__ __forceinline__ void store4(const GemmI8Args& a, int n, int m, const int (&sum)[4], float xs, bool packed) {
    if (packed && m + 3 < a.M) {
        float v[4];
#pragma unroll
        for (int r = 0; r < 4; r++) v[r] = scaled(a, sum[r], xs, m + r);
        const int64_t at = (int64_t)n * a.y_stride + m;
        if (a.y_fp32) *(f32x4g*)((float*)a.y + at) = f32x4g{v[0], v[1], v[2], v[3]};
        else *(u32x2g*)((uint16_t*)a.y + at) = u32x2g{(uint32_t)f32_to_f16_bits(v[0]) | (uint32_t)f32_to_f16_bits(v[1]) << 16,
                                                      (uint32_t)f32_to_f16_bits(v[2]) | (uint32_t)f32_to_f16_bits(v[3]) << 16};
        return;
    }
#pragma unroll
    for (int r = 0; r < 4; r++)
        if (m + r < a.M) store1(a, n, m + r, scaled(a, sum[r], xs, m + r));
}
// rows whose four channels are one aligned store
__device__ __forceinline__ bool packed_rows(const GemmI8Args& a) {
    return a.y_stride % 4 == 0 && ((uintptr_t)a.y & (a.y_fp32 ? 15 : 7)) == 0;
}

// ---- few tokens: the weights are read once, and are what bounds it ----

// 16 channels x up to 16 tokens a workgroup; its waves take the 64-byte pieces of K in turn
// (an even U: two pieces in turn) and their sums meet in LDS.  Lane (li, lg) of
// v_mfma_i32_16x16x64_i8: 16 codes of channel li / token li.  Codes go straight to registers,
// two batches of U pieces on the way.  Waves x U:
//   one token     151936 x 2560   19456 x 2560   6144 x 2560   2560 x 9728   1024 x 9728
//   4 x 5             76.8            13.9           6.3           9.9           9.4
//   4 x 8             74.2            13.9           6.4          10.9          10.4
//   16 x 5           108              17.1           7.5           9.5           9.1
// (us, calls one behind the other, W from memory.  A workgroup for up to 64 tokens, without tiles: its own
// reading of all tokens took longer than its weights: 28 us for 2560 x 9728 against 14.)
template <int GF_WAVES, int U>
__global__ __launch_bounds__(64 * GF_WAVES) void gemm_i8_few_kernel(GemmI8Args a) {
    constexpr int STEP = 64 * GF_WAVES * U, RUN = U % 2 == 0 ? 2 : 1;
    __shared__ int sums[GF_WAVES][4][64];
    const int lane = (int)threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int li = lane & 15, lg = lane >> 4, m0 = (int)blockIdx.x * 16;
    const int8_t* w = a.w + (int64_t)min(m0 + li, a.M - 1) * a.w_stride;
    const int8_t* x = a.x + (int64_t)min(li, a.N - 1) * a.x_stride;
    i32x4g acc = {};
    i32x4g wv[2][U], xv[2][U];
    auto load = [&](int q, int k0) {
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int k = k0 + 64 * (GF_WAVES * RUN * (u / RUN) + u % RUN) + 16 * lg;
            const bool is = k < a.K;
            wv[q][u] = is ? __builtin_nontemporal_load((const i32x4g*)(w + k)) : i32x4g{};
            xv[q][u] = is ? *(const i32x4g*)(x + k) : i32x4g{};
        }
    };
    auto work = [&](int q) {
#pragma unroll
        for (int u = 0; u < U; u++) acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(wv[q][u], xv[q][u], acc, 0, 0, 0);
    };
    load(0, 64 * RUN * wave);
    for (int k0 = 64 * RUN * wave; k0 < a.K; k0 += 2 * STEP) {
        load(1, k0 + STEP);
        __builtin_amdgcn_sched_barrier(0);
        work(0);
        load(0, k0 + 2 * STEP);
        __builtin_amdgcn_sched_barrier(0);
        work(1);
    }
#pragma unroll
    for (int r = 0; r < 4; r++) sums[wave][r][lane] = acc[r];
    __syncthreads();
    const int e = (int)threadIdx.x, m = e & 15, n = e >> 4;
    if (e >= 256 || n >= a.N || m0 + m >= a.M) return;
    int s = 0;
#pragma unroll
    for (int v = 0; v < GF_WAVES; v++) s += sums[v][m & 3][(m >> 2) * 16 + n];
    store1(a, n, m0 + m, scaled(a, s, a.xs[n], m0 + m));
}

// ---- many tokens: tiles through LDS ----

// Results [ROWS][TM] of ES bytes in LDS, rows `pitch` bytes apart (a multiple of 16, TM * ES + 16 or
// more), to the rows token(r) of out (`row` elements apart) from channel m0; T threads.  Rows
// may begin anywhere: whole pieces between the 16-byte boundaries, which LDS gives at any
// element, then the ends of all rows element by element (1124 tokens x 41131 channels of
// fp16 43 us, 82 with element stores throughout; 41136 channels 36).
template <int TM, int ROWS, int T, int ES, typename Token>
__device__ __forceinline__ void put_rows(const uint8_t* lds, int pitch, uint8_t* out, int64_t row, int m0, int M, int N, Token token) {
    constexpr int PER = 16 / ES;
    const int live = min(TM, M - m0);
    auto put = [&](const uint8_t* from, uint8_t* to, int i) {
        if (ES == 2) ((uint16_t*)to)[i] = ((const uint16_t*)from)[i];
        else         ((uint32_t*)to)[i] = ((const uint32_t*)from)[i];
    };
    if (((uintptr_t)out & 15) == 0 && row * ES % 16 == 0) {
        for (int e = (int)threadIdx.x; e < ROWS * (TM / PER); e += T) {
            const int r = e / (TM / PER), m = (e - r * (TM / PER)) * PER, n = token(r);
            if (n >= N || m >= live) continue;
            const uint8_t* from = lds + r * pitch + m * ES;
            uint8_t* o = out + ((int64_t)n * row + m0 + m) * ES;
            if (m + PER <= live) *(i32x4g*)o = *(const i32x4g*)from;
            else
                for (int i = 0; i < live - m; i++) put(from, o, i);
        }
        return;
    }
    auto row_at = [&](int n) { return out + ((int64_t)n * row + m0) * ES; };
    auto front = [&](const uint8_t* o) { return min((int)(-(uintptr_t)o & 15) / ES, live); };
    for (int e = (int)threadIdx.x; e < ROWS * (TM / PER); e += T) {
        const int r = e / (TM / PER), j = e - r * (TM / PER), n = token(r);
        if (n >= N) continue;
        uint8_t* o = row_at(n);
        const uint8_t* from = lds + r * pitch;
        const int m = front(o) + j * PER;
        if (m + PER > live) continue;
        i32x4g w;
        if (ES == 4) {
#pragma unroll
            for (int i = 0; i < 4; i++) w[i] = ((const int*)from)[m + i];
        } else {
            const uint32_t* p = (const uint32_t*)from + (m >> 1);
            uint32_t x[5];
#pragma unroll
            for (int i = 0; i < 5; i++) x[i] = p[i];   // (the fifth may be the row's padding)
#pragma unroll
            for (int i = 0; i < 4; i++) w[i] = (int)__builtin_amdgcn_alignbit(x[i + 1], x[i], 16u * (m & 1));
        }
        *(i32x4g*)(o + m * ES) = w;
    }
    // the ends, an element a lane: PER in front, PER behind
    for (int e = (int)threadIdx.x; e < ROWS * 2 * PER; e += T) {
        const int r = e / (2 * PER), i = e - r * 2 * PER, n = token(r);
        if (n >= N) continue;
        uint8_t* o = row_at(n);
        const int head = front(o), tail = head + (live - head) / PER * PER;
        const int m = i < PER ? i : tail + i - PER;
        if (i < PER ? m < head : m < live) put(lds + r * pitch, o, m);
    }
}

// A workgroup of WM x WN waves, each 32 FM channels x 32 FN tokens on
// v_mfma_i32_32x32x32_i8.  Stages of 128 codes of every row go straight from memory into
// LDS, the next one on its way while one is worked on.  Piece c (16 bytes) of row r lies
// at place c ^ (r / 2 % 8): two rows fill the 64 banks, and the same piece of any 16 rows that
// a read takes at once falls on each of them once.

// 16 bytes a lane from base + offset straight to LDS, lane after lane
__device__ __forceinline__ void load_lds(__amdgpu_buffer_rsrc_t base, uint8_t* lds, int offset) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(base, (lds_void_g*)lds, 16, offset, 0, 0, 0);
}

template <int FM, int FN, int WM, int WN, int R>
__device__ __forceinline__ void tile_body(const GemmI8Args& a, uint8_t* tiles, int m0, int n0, int part, int splits) {
    constexpr int TM = 32 * FM * WM, TN = 32 * FN * WN, NW = WM * WN;
    constexpr int STAGE = (TM + TN) * GT_K;
    constexpr int LA = TM / 8 / NW, LB = TN / 8 / NW;  // loads of 8 rows per wave and stage
    const int lane = (int)threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int li = lane & 31, g = lane >> 5, wm = wave % WM, wn = wave / WM;

    const int stages = (a.K + GT_K - 1) / GT_K;
    const int s0 = (int)((int64_t)stages * part / splits), s1 = (int)((int64_t)stages * (part + 1) / splits);

    // lane l of load i of a wave: row 8 i + l / 8 of its share (8 LA or 8 LB rows), place l % 8
    auto piece = [&](int row8) { return 16 * ((lane & 7) ^ ((4 * row8 + (lane >> 4)) & 7)); };
    const int8_t* wbase = a.w + (int64_t)m0 * a.w_stride;
    const int8_t* xbase = a.x + (int64_t)n0 * a.x_stride;
    const __amdgpu_buffer_rsrc_t rW = __builtin_amdgcn_make_buffer_rsrc((void*)wbase, (short)0, 0x7FFFFFFF, 0x00020000);
    const __amdgpu_buffer_rsrc_t rX = __builtin_amdgcn_make_buffer_rsrc((void*)xbase, (short)0, 0x7FFFFFFF, 0x00020000);
    int rowW[LA], rowX[LB];                            // (rows past the last re-read it)
#pragma unroll
    for (int i = 0; i < LA; i++) rowW[i] = min(8 * (wave * LA + i) + (lane >> 3), a.M - 1 - m0) * (int)a.w_stride;
#pragma unroll
    for (int i = 0; i < LB; i++) rowX[i] = min(8 * (wave * LB + i) + (lane >> 3), a.N - 1 - n0) * (int)a.x_stride;
    auto slot = [](int s) { return R == 2 ? s & 1 : (R == 4 ? s & 3 : s % R); };
    auto issue = [&](int s) {
        uint8_t* st = tiles + slot(s) * STAGE;
        // (a last stage that K ends in: pieces past the end re-read the last one)
#pragma unroll
        for (int i = 0; i < LA; i++) load_lds(rW, st + (wave * LA + i) * 1024, rowW[i] + min(s * GT_K + piece(wave * LA + i), a.K - 16));
#pragma unroll
        for (int i = 0; i < LB; i++) load_lds(rX, st + TM * GT_K + (wave * LB + i) * 1024, rowX[i] + min(s * GT_K + piece(wave * LB + i), a.K - 16));
    };

    i32x16g acc[FM][FN];
#pragma unroll
    for (int i = 0; i < FM; i++)
#pragma unroll
        for (int j = 0; j < FN; j++) acc[i][j] = i32x16g{};
    const int sw = (li >> 1) & 7;
    const uint8_t* pa = tiles + (32 * FM * wm + li) * GT_K;
    const uint8_t* pb = tiles + TM * GT_K + (32 * FN * wn + li) * GT_K;
    auto work = [&](int s, bool tail) {
        const int off = slot(s) * STAGE;
#pragma unroll
        for (int h = 0; h < 4; h++) {
            const int at = off + 16 * ((2 * h + g) ^ sw);
            i32x4g av[FM], bv[FN];
#pragma unroll
            for (int i = 0; i < FM; i++) av[i] = *(const i32x4g*)(pa + at + 32 * GT_K * i);
#pragma unroll
            for (int j = 0; j < FN; j++) bv[j] = *(const i32x4g*)(pb + at + 32 * GT_K * j);
            if (tail && s * GT_K + 32 * h + 16 * g >= a.K) {
#pragma unroll
                for (int i = 0; i < FM; i++) av[i] = i32x4g{};
            }
#pragma unroll
            for (int i = 0; i < FM; i++)
#pragma unroll
                for (int j = 0; j < FN; j++) acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(av[i], bv[j], acc[i][j], 0, 0, 0);
        }
    };
    // stage s is in LDS, and every wave is done with stage s - 1
    auto arrive = [&](int s) {
        constexpr int AHEAD = (R - 2) * (LA + LB);     // loads of the stages behind it
        if (R > 2 && s + R - 2 < s1) __builtin_amdgcn_s_waitcnt(0x0F70 | (AHEAD & 15) | (AHEAD >> 4) << 14);
        else                         __builtin_amdgcn_s_waitcnt(0x0F70);
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_sched_barrier(0);
    };
#pragma unroll
    for (int i = 0; i < R - 1; i++)
        if (s0 + i < s1) issue(s0 + i);
    const int full = min(s1, a.K / GT_K);
    for (int s = s0; s < full; s++) {
        arrive(s);
        if (s + R - 1 < s1) issue(s + R - 1);
        work(s, false);
    }
    if (s0 < s1 && full < s1) {
        arrive(full);
        work(full, true);
    }

    // The tile goes out through LDS, 32 WN tokens at a time, so that rows are stored in whole
    // lines: [32 WN][TM] results (fp16, or 4 bytes), rows 16 bytes apart from a power of two.
    const bool half = splits == 1 && !a.y_fp32;
    const int es = half ? 2 : 4, pitch = TM * es + 16;
    float* sw_ = (float*)(tiles + 32 * WN * (TM * 4 + 16));          // the channels' scales and biases
    float* sb_ = sw_ + TM;
    __syncthreads();
    if (splits == 1)
        for (int e = (int)threadIdx.x; e < TM; e += 64 * NW) {
            const int m = min(m0 + e, a.M - 1);
            sw_[e] = a.ws[m];
            sb_[e] = a.bias ? a.bias[m] : 0.0f;
        }
    const int64_t row = splits > 1 ? (int64_t)a.M : a.y_stride;
    uint8_t* out = splits > 1 ? (uint8_t*)(a.part + (int64_t)part * a.N * a.M) : (uint8_t*)a.y;
#pragma unroll
    for (int j = 0; j < FN; j++) {
        __syncthreads();
        const float xs = splits > 1 ? 0.0f : a.xs[min(n0 + 32 * (FN * wn + j) + li, a.N - 1)];
        uint8_t* to = tiles + (32 * wn + li) * pitch;
#pragma unroll
        for (int i = 0; i < FM; i++)
#pragma unroll
            for (int v = 0; v < 4; v++) {
                const int m = 32 * (FM * wm + i) + 8 * v + 4 * g;
                i32x4g sum = {acc[i][j][4 * v], acc[i][j][4 * v + 1], acc[i][j][4 * v + 2], acc[i][j][4 * v + 3]};
                if (splits > 1) { *(i32x4g*)(to + 4 * m) = sum; continue; }
                const f32x4g ws = *(const f32x4g*)(sw_ + m), bias = *(const f32x4g*)(sb_ + m);
                f32x4g y;
#pragma unroll
                for (int r = 0; r < 4; r++) y[r] = scaled_by(sum[r], xs, ws[r], a.bias != nullptr, bias[r]);
                if (half) *(u32x2g*)(to + 2 * m) = u32x2g{(uint32_t)f32_to_f16_bits(y[0]) | (uint32_t)f32_to_f16_bits(y[1]) << 16,
                                                          (uint32_t)f32_to_f16_bits(y[2]) | (uint32_t)f32_to_f16_bits(y[3]) << 16};
                else      *(f32x4g*)(to + 4 * m) = y;
            }
        __syncthreads();
        auto token = [&](int r) { return n0 + 32 * (FN * (r / 32) + j) + r % 32; };
        if (half) put_rows<TM, 32 * WN, 64 * NW, 2>(tiles, pitch, out, row, m0, a.M, a.N, token);
        else      put_rows<TM, 32 * WN, 64 * NW, 4>(tiles, pitch, out, row, m0, a.M, a.N, token);
    }
}

// Workgroups go round the eight XCDs: each gets a run of neighbouring tiles, in columns of
// four, so that what its L2 holds serves several.  Tile t of mt x nt.
__device__ __forceinline__ int xcd_run(int b, int total) {
    const int q = total / 8, rem = total % 8, xcd = b % 8;
    return xcd * q + min(xcd, rem) + b / 8;
}
__device__ __forceinline__ void tile_at(int t, int mt, int nt, int& i, int& j) {
    const int col = t / (4 * nt), in = t - col * 4 * nt, wide = min(4, mt - 4 * col);
    i = 4 * col + in % wide;
    j = in / wide;
}

template <int FM, int FN, int WM, int WN, int R>
__global__ __launch_bounds__(64 * WM * WN, 1) void gemm_i8_tile_kernel(GemmI8Args a, int splits) {
    constexpr int TM = 32 * FM * WM, TN = 32 * FN * WN;
    extern __shared__ __attribute__((aligned(128))) uint8_t tiles[];
    const int mt = (a.M + TM - 1) / TM, nt = (a.N + TN - 1) / TN, total = mt * nt;
    const int part = (int)(blockIdx.x / (unsigned)total), b = (int)(blockIdx.x - (unsigned)part * (unsigned)total);
    int i, j;
    tile_at(xcd_run(b, total), mt, nt, i, j);
    tile_body<FM, FN, WM, WN, R>(a, tiles, i * TM, j * TN, part, splits);
}

// `whole` tiles of 256 x 256, as many as fill every CU the same number of times, then the
// rest of the tiles in halves of 256 x 128.
__global__ __launch_bounds__(512, 1) void gemm_i8_rounds_kernel(GemmI8Args a, int whole) {
    extern __shared__ __attribute__((aligned(128))) uint8_t tiles[];
    const int mt = (a.M + 255) / 256, nt = (a.N + 255) / 256, b = (int)blockIdx.x;
    int i, j;
    if (b < whole) {
        tile_at(xcd_run(b, whole), mt, nt, i, j);
        tile_body<4, 2, 2, 4, 2>(a, tiles, 256 * i, 256 * j, 0, 1);
    } else {
        tile_at(whole + (b - whole) / 2, mt, nt, i, j);
        const int n0 = 256 * j + 128 * ((b - whole) & 1);
        if (n0 < a.N) tile_body<4, 1, 2, 4, 3>(a, tiles, 256 * i, n0, 0, 1);
    }
}

// sums of the parts, scaled: a token's channels in fours
__global__ __launch_bounds__(256) void gemm_i8_join_kernel(GemmI8Args a, int splits) {
    const int n = (int)blockIdx.y, m = 4 * ((int)blockIdx.x * 256 + (int)threadIdx.x);
    if (m >= a.M) return;
    const int64_t step = (int64_t)a.N * a.M;
    const int32_t* p = a.part + (int64_t)n * a.M + m;
    int s[4] = {0, 0, 0, 0};
    const float xs = a.xs[n];
    if (a.M % 4 == 0) {
#pragma unroll 8
        for (int i = 0; i < splits; i++) {
            const i32x4g v = *(const i32x4g*)(p + i * step);
#pragma unroll
            for (int r = 0; r < 4; r++) s[r] += v[r];
        }
    } else {
        for (int i = 0; i < splits; i++)
#pragma unroll
            for (int r = 0; r < 4; r++) s[r] += m + r < a.M ? p[i * step + r] : 0;
    }
    store4(a, n, m, s, xs, packed_rows(a));
}

// Rows of codes so far apart that a tile's offsets pass 31 bits: 16 channels x 64 tokens a
// wave, straight from memory.
__global__ __launch_bounds__(256) void gemm_i8_far_kernel(GemmI8Args a) {
    const int lane = (int)threadIdx.x & 63, wave = (int)threadIdx.x >> 6, li = lane & 15, lg = lane >> 4;
    const int mt = (a.M + 63) / 64;
    const int m0 = (int)(blockIdx.x % (unsigned)mt) * 64 + 16 * wave, n0 = (int)(blockIdx.x / (unsigned)mt) * 64;
    const int8_t* w = a.w + (int64_t)min(m0 + li, a.M - 1) * a.w_stride;
    const int8_t* x[4];
#pragma unroll
    for (int j = 0; j < 4; j++) x[j] = a.x + (int64_t)min(n0 + 16 * j + li, a.N - 1) * a.x_stride;
    i32x4g acc[4] = {};
    for (int k0 = 0; k0 < a.K; k0 += 64) {
        const int k = k0 + 16 * lg;
        i32x4g wv = {}, xv[4] = {};
        if (k < a.K) {
            wv = *(const i32x4g*)(w + k);
#pragma unroll
            for (int j = 0; j < 4; j++) xv[j] = *(const i32x4g*)(x[j] + k);
        }
#pragma unroll
        for (int j = 0; j < 4; j++) acc[j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wv, xv[j], acc[j], 0, 0, 0);
    }
    const bool packed = packed_rows(a);
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const int n = n0 + 16 * j + li, m = m0 + 4 * lg;
        const int sum[4] = {acc[j][0], acc[j][1], acc[j][2], acc[j][3]};
        if (n < a.N && m < a.M) store4(a, n, m, sum, a.xs[n], packed);
    }
}

template <int FM, int FN, int WM, int WN, int R>
constexpr int tile_lds() {
    constexpr int TM = 32 * FM * WM, TN = 32 * FN * WN, MAIN = R * (TM + TN) * GT_K, OUT = 32 * WN * (TM * 4 + 16) + 8 * TM;
    return MAIN > OUT ? MAIN : OUT;
}
template <int FM, int FN, int WM, int WN, int R>
hipError_t tile_go(const GemmI8Args& a, int splits, hipStream_t st) {
    constexpr int TM = 32 * FM * WM, TN = 32 * FN * WN, LDS = tile_lds<FM, FN, WM, WN, R>();
    if (const hipError_t e = allow_lds<gemm_i8_tile_kernel<FM, FN, WM, WN, R>>(LDS)) return e;
    const unsigned n = (unsigned)((a.M + TM - 1) / TM) * (unsigned)((a.N + TN - 1) / TN);
    hipLaunchKernelGGL((gemm_i8_tile_kernel<FM, FN, WM, WN, R>), dim3(n * (unsigned)splits), dim3(64 * WM * WN), LDS, st, a, splits);
    return hipGetLastError();
}
hipError_t rounds_go(const GemmI8Args& a, int whole, hipStream_t st) {
    constexpr int LDS = tile_lds<4, 2, 2, 4, 2>() > tile_lds<4, 1, 2, 4, 3>() ? tile_lds<4, 2, 2, 4, 2>() : tile_lds<4, 1, 2, 4, 3>();
    if (const hipError_t e = allow_lds<gemm_i8_rounds_kernel>(LDS)) return e;
    const int n = (a.M + 255) / 256 * ((a.N + 255) / 256);
    hipLaunchKernelGGL(gemm_i8_rounds_kernel, dim3((unsigned)(whole + 2 * (n - whole))), dim3(512), LDS, st, a, whole);
    return hipGetLastError();
}
}  // namespace

int64_t gemm_i8_workspace(int M, int N, int K) {
    const GemmPlan p = gemm_plan(M, N, K);
    return p.splits > 1 ? ((int64_t)p.splits * M * N * 4 + 15) & ~(int64_t)15 : 0;
}

// (an upper bound over the forms)
int64_t gemm_i8_blocks(int M, int N, int) { return (((int64_t)M + 15) / 16) * (((int64_t)N + 63) / 64); }

hipError_t gemm_i8_launch(const GemmI8Args& a, hipStream_t st) {
    const GemmPlan p = gemm_plan(a.M, a.N, a.K);
    if (p.few) {
        const dim3 grid((unsigned)(a.M + 15) / 16);
        if (p.few == FEW_MANY_CHANNELS) hipLaunchKernelGGL((gemm_i8_few_kernel<4, 8>), grid, dim3(256), 0, st, a);
        else if (p.few == FEW_LONG_K) hipLaunchKernelGGL((gemm_i8_few_kernel<16, 5>), grid, dim3(1024), 0, st, a);
        else hipLaunchKernelGGL((gemm_i8_few_kernel<4, 5>), grid, dim3(256), 0, st, a);
        return hipGetLastError();
    }
    if (a.w_stride * 256 >= ((int64_t)1 << 31) || a.x_stride * 256 >= ((int64_t)1 << 31)) {
        hipLaunchKernelGGL(gemm_i8_far_kernel, dim3((unsigned)(((a.M + 63) / 64) * ((a.N + 63) / 64))), dim3(256), 0, st, a);
        return hipGetLastError();
    }
    hipError_t e;
    if (p.whole) return rounds_go(a, p.whole, st);
    switch (p.tile) {
    case 0:  e = tile_go<4, 2, 2, 4, 2>(a, p.splits, st); break;
    case 1:  e = tile_go<2, 2, 2, 4, 3>(a, p.splits, st); break;
    case 2:  e = tile_go<2, 2, 2, 2, 2>(a, p.splits, st); break;
    case 3:  e = tile_go<1, 1, 2, 2, 4>(a, p.splits, st); break;
    default: e = tile_go<1, 1, 1, 2, 4>(a, p.splits, st); break;
    }
    if (e != hipSuccess || p.splits == 1) return e;
    hipLaunchKernelGGL(gemm_i8_join_kernel, dim3((unsigned)(a.M + 1023) / 1024, (unsigned)a.N), dim3(256), 0, st, a, p.splits);
    return hipGetLastError();
}

}  // namespace jllm_hip
