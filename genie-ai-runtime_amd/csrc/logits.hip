// logits.hip -- what a sampler does to a batch's logits before it picks: penalties
// for repeated tokens, biases, grammar masks; and the greedy pick itself.
//
//   y = x > 0 ? x / r : x * r    tokens of the row's prompt or output
//   y = y - f * count            count of the token in the row's output
//   y = y - p                    where count > 0
//   y = y + bias                 listed tokens (listed twice: the last entry counts)
//   y = -inf                     where the token's mask bit is 0
//   token = lowest index of the largest finite y, -1 when there is none
//
// Measured (both launches, replayed): 64 rows x 151936 with up to 4096 listed tokens,
// biases and masks 20.0 us (4.0 TB/s), without any 15.3; 251 rows x 32003 17.0 us; one
// row 5.8 us, of which the kernels run 4.0 and 1.9 (7.9 us where the host launches them).
#include "kq_common.h"
#include "serving.h"

namespace jllm_hip {

constexpr int LG_THREADS = 256;
constexpr uint32_t LG_PROMPT = 0x80000000u;    // "in the prompt" bit of a count

// rows begin at any 4-byte address
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));
typedef int32_t i32x4u __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t u32x4l __attribute__((ext_vector_type(4)));

// entries of a list row that count (below 2^30: a count keeps its topmost bits, and
// the loops' places stay ints)
__device__ __forceinline__ int list_length(int n, int64_t stride) {
    return (int)max((int64_t)0, min(min((int64_t)n, stride), (int64_t)1 << 30));
}

// (value, index) as one word that grows with the value and falls with the index;
// 0: nothing to pick
__device__ __forceinline__ uint64_t pick_key(float y, int i) {
    const uint32_t b = __builtin_bit_cast(uint32_t, y + 0.0f);      // -0 counts as +0
    const uint32_t o = b & 0x80000000u ? ~b : b | 0x80000000u;
    return ((uint64_t)o << 32) | (uint32_t)~i;
}
template <int CTRL>
__device__ __forceinline__ uint32_t dpp_umax(uint32_t v) {
    return max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, CTRL, 0xF, 0xF, false));
}
__device__ __forceinline__ uint32_t wave_umax(uint32_t v) {
    v = dpp_umax<0xB1>(v);
    v = dpp_umax<0x4E>(v);
    v = dpp_umax<0x141>(v);
    v = dpp_umax<0x140>(v);
    const uint32_t a = max((uint32_t)__builtin_amdgcn_readlane((int)v, 0), (uint32_t)__builtin_amdgcn_readlane((int)v, 16));
    const uint32_t b = max((uint32_t)__builtin_amdgcn_readlane((int)v, 32), (uint32_t)__builtin_amdgcn_readlane((int)v, 48));
    return max(a, b);
}
__device__ __forceinline__ uint64_t wave_max_key(uint64_t k) {
    const uint32_t hi = wave_umax((uint32_t)(k >> 32));
    const uint32_t lo = wave_umax((uint32_t)(k >> 32) == hi ? (uint32_t)k : 0u);
    return ((uint64_t)hi << 32) | lo;
}

// A workgroup takes CH = 1024 J tokens of a row, a thread J times four neighbours.
// The logits and mask words are on their way while the lists are searched: every
// workgroup goes through its row's whole lists and counts the tokens that fall
// into its part in LDS (integers: the order of the atomics does not matter).
template <int J>
__global__ __launch_bounds__(LG_THREADS) void logits_kernel(LogitsArgs a) {
#pragma clang fp contract(off)
    constexpr int CH = 1024 * J;
    extern __shared__ __attribute__((aligned(16))) uint32_t sLists[];
    __shared__ uint64_t sKey[LG_THREADS / 64];
    uint32_t* sCount = sLists;                             // [CH] when there are tokens
    uint32_t* sBias = sLists + (a.tokens ? CH : 0);        // [CH] when there are biases: entry + 1
    const int64_t b = blockIdx.y;
    const int t = threadIdx.x, c0 = blockIdx.x * CH, n = min(CH, a.V - c0);
    const float* x = a.x + b * a.x_stride + c0;
    float* out = a.out + b * a.out_stride + c0;

    // The first round of the lists is read before it is known how much of it counts:
    // up to the stride there is the row's or the next row's memory.  Behind the last
    // row there may be none: it is read as far as it counts.  (By limits, not by a way
    // of its own around the loads: 64 rows with lists and masks 20.3 us against 20.7.)
    const bool ahead = b + 1 < a.B;
    const int first = ahead ? LG_THREADS : 0;
    const int32_t* ids = a.tokens + b * a.token_stride;
    const int32_t* bids = a.bias_ids + b * a.bias_stride;
    i32x4u id4 = {-1, -1, -1, -1};
    if (a.tokens && 4 * t + 4 <= (ahead ? a.token_stride : 0)) id4 = *(const i32x4u*)(ids + 4 * t);
    const int bid = a.bias_ids && t < (ahead ? a.bias_stride : 0) ? bids[t] : -1;
    f32x4u y[J];
    uint32_t word[J];
#pragma unroll
    for (int j = 0; j < J; j++) {
        const int i = 1024 * j + 4 * t;
        if (i + 4 <= n) y[j] = *(const f32x4u*)(x + i);
        else
#pragma unroll
            for (int e = 0; e < 4; e++) y[j][e] = i + e < n ? x[i + e] : -INFINITY;
        word[j] = a.mask && i < n ? a.mask[b * a.mask_stride + ((c0 + i) >> 5)] : ~0u;
    }
    __builtin_amdgcn_sched_barrier(0);

    const int lists = (a.tokens ? CH : 0) + (a.bias_ids ? CH : 0);
    if (lists) {
        for (int i = 4 * t; i < lists; i += 4 * LG_THREADS) *(u32x4l*)(sLists + i) = u32x4l{0u, 0u, 0u, 0u};
        __syncthreads();
    }
    if (a.tokens) {
        const int nt = list_length(a.n_tokens[b], a.token_stride);
        const int np = a.n_prompt ? max(0, min(a.n_prompt[b], nt)) : 0;
        auto count = [&](uint32_t at, int i) {             // at: place in this part
            if (at < (uint32_t)n && i < nt) {
                if (i < np) atomicOr(&sCount[at], LG_PROMPT);
                else atomicAdd(&sCount[at], 1u);
            }
        };
        auto count4 = [&](i32x4u id, int i) {              // few of the ids fall into this part: one test for four
            const uint32_t p0 = (uint32_t)id[0] - c0, p1 = (uint32_t)id[1] - c0, p2 = (uint32_t)id[2] - c0, p3 = (uint32_t)id[3] - c0;
            if (min(min(p0, p1), min(p2, p3)) >= (uint32_t)n) return;
            count(p0, i);
            count(p1, i + 1);
            count(p2, i + 2);
            count(p3, i + 3);
        };
        // whole fours of what may be read, then the last entries
        const int fours = (ahead ? (int)a.token_stride : nt) & ~3;
        count4(id4, 4 * t);                            // (the last row begins in the loop)
#pragma unroll 2
        for (int i = 4 * (first + t); i < min(nt, fours); i += 4 * LG_THREADS) count4(*(const i32x4u*)(ids + i), i);
        if (fours + t < nt) count((uint32_t)ids[fours + t] - c0, fours + t);
    }
    if (a.bias_ids) {
        const int nb = list_length(a.n_bias[b], a.bias_stride);
        auto list = [&](int id, int i) {
            const uint32_t at = (uint32_t)id - (uint32_t)c0;
            if (at < (uint32_t)n && i < nb) atomicMax(&sBias[at], (uint32_t)i + 1u);
        };
        list(bid, t);
        for (int i = first + t; i < nb; i += LG_THREADS) list(bids[i], i);
    }
    if (lists) __syncthreads();
    const float rep = a.tokens && a.repetition ? a.repetition[b] : 1.0f;
    const float freq = a.tokens && a.frequency ? a.frequency[b] : 0.0f;
    const float pres = a.tokens && a.presence ? a.presence[b] : 0.0f;
    float best = -INFINITY;
    int at = -1;
#pragma unroll
    for (int j = 0; j < J; j++) {
        const int i = 1024 * j + 4 * t;
        if (a.tokens) {
            const u32x4l c4 = *(const u32x4l*)(sCount + i);
#pragma unroll
            for (int e = 0; e < 4; e++) {
                if (c4[e]) {
                    y[j][e] = y[j][e] > 0.0f ? y[j][e] / rep : y[j][e] * rep;
                    const uint32_t cnt = c4[e] & ~LG_PROMPT;
                    if (cnt) { y[j][e] = y[j][e] - freq * (float)cnt; y[j][e] = y[j][e] - pres; }
                }
            }
        }
        if (a.bias_ids) {
            const u32x4l c4 = *(const u32x4l*)(sBias + i);
#pragma unroll
            for (int e = 0; e < 4; e++)
                if (c4[e]) y[j][e] = y[j][e] + a.bias[b * a.bias_stride + c4[e] - 1];
        }
        const uint32_t bits = word[j] >> (i & 31);
#pragma unroll
        for (int e = 0; e < 4; e++) {
            if (!(bits >> e & 1u)) y[j][e] = -INFINITY;
            // (-inf, which masked tokens and those behind the row's end have, and NaN are
            // not above the start value)
            if (y[j][e] > best && y[j][e] < INFINITY) { best = y[j][e]; at = i + e; }
        }
        // (not kept in the L2, where it would push out logits on their way in: 21.4 us
        // -> 19.8 for 64 rows with lists and masks; loads marked so cost as much)
        if (i + 4 <= n) __builtin_nontemporal_store(y[j], (f32x4u*)(out + i));
        else
#pragma unroll
            for (int e = 0; e < 4; e++) if (i + e < n) out[i + e] = y[j][e];
    }
    if (!a.next_token) return;
    uint64_t key = wave_max_key(at >= 0 ? pick_key(best, c0 + at) : 0);
    if ((t & 63) == 0) sKey[t >> 6] = key;
    __syncthreads();
    if (t == 0) {
#pragma unroll
        for (int w = 1; w < LG_THREADS / 64; w++) key = max(key, sKey[w]);
        if (gridDim.x == 1) a.next_token[b] = key ? (int32_t)~(uint32_t)key : -1;
        else a.cand[b * gridDim.x + blockIdx.x] = key;
    }
}

// one wave per row
__global__ __launch_bounds__(LG_THREADS) void logits_pick_kernel(int32_t* tok, const uint64_t* cand, int chunks, int B) {
    const int64_t b = (int64_t)blockIdx.x * (LG_THREADS / 64) + (threadIdx.x >> 6);
    const int l = threadIdx.x & 63;
    if (b >= B) return;
    uint64_t key = 0;
#pragma unroll 4
    for (int i = l; i < chunks; i += 64) key = max(key, cand[b * chunks + i]);
    key = wave_max_key(key);
    if (l == 0) tok[b] = key ? (int32_t)~(uint32_t)key : -1;
}

namespace {
// Parts of 2048 tokens, which search the lists half as often, once they fill the
// card, else of 1024 (one row of 151936 with 700 tokens listed: 5.8 us against 7.1 with
// parts of 4096; 64 rows with lists, biases and masks, when they took 22.3 us: 24.6 with
// 4096).
int logits_part(int B, int V) { return (int64_t)B * (((int64_t)V + 2047) / 2048) < 1024 ? 1 : 2; }
int logits_chunks(int B, int V) {
    const int ch = 1024 * logits_part(B, V);
    return (int)(((int64_t)V + ch - 1) / ch);
}
}  // namespace

int64_t logits_workspace(int B, int V) {
    const int n = logits_chunks(B, V);
    return n > 1 ? (int64_t)B * n * 8 : 0;
}

hipError_t logits_launch(const LogitsArgs& a, hipStream_t st) {
    const int n = logits_chunks(a.B, a.V), J = logits_part(a.B, a.V);
    const dim3 grid(n, a.B);
    const size_t lds = (size_t)((a.tokens ? 1 : 0) + (a.bias_ids ? 1 : 0)) * J * 4096;
    if (J == 1) hipLaunchKernelGGL((logits_kernel<1>), grid, dim3(LG_THREADS), lds, st, a);
    else        hipLaunchKernelGGL((logits_kernel<2>), grid, dim3(LG_THREADS), lds, st, a);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || !a.next_token || n == 1) return e;
    hipLaunchKernelGGL(logits_pick_kernel, dim3((a.B + 3) / 4), dim3(LG_THREADS), 0, st, a.next_token,
                       (const uint64_t*)a.cand, n, a.B);
    return hipGetLastError();
}

}  // namespace jllm_hip
