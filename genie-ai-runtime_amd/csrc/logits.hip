// logits.hip -- what a sampler does to a batch's logits before it picks: penalties
// for repeated tokens, biases, grammar masks; and the greedy pick itself.
//
//   y = x > 0 ? x / r : x * r    tokens of the row's prompt or output
//   y = y - f * count            count of the token in the row's output
//   y = y - p                    where count > 0
//   y = y + bias                 listed tokens (listed twice: the last entry counts)
//   y = -inf                     where the token's mask bit is 0
//   token = lowest index of the largest finite y, -1 when there is none
#include "kq_common.h"
#include "serving.h"

namespace jllm_hip {

constexpr int LG_THREADS = 256;
constexpr int LG_CHUNK = 4096;                 // tokens a workgroup takes
constexpr uint32_t LG_PROMPT = 0x80000000u;    // "in the prompt" bit of a count

typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t u32x4l __attribute__((ext_vector_type(4)));

// (value, index) as one word that grows with the value and falls with the index;
// 0 for what the pick ignores
__device__ __forceinline__ uint64_t pick_key(float y, int i) {
    if (!isfinite(y)) return 0;
    const uint32_t b = __builtin_bit_cast(uint32_t, y + 0.0f);      // -0 counts as +0
    const uint32_t o = b & 0x80000000u ? ~b : b | 0x80000000u;
    return ((uint64_t)o << 32) | (uint32_t)~i;
}
__device__ __forceinline__ uint64_t wave_max_key(uint64_t k) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        const uint64_t v = __shfl_xor((unsigned long long)k, o, 64);
        k = v > k ? v : k;
    }
    return k;
}

__global__ __launch_bounds__(LG_THREADS) void logits_kernel(LogitsArgs a) {
#pragma clang fp contract(off)
    __shared__ uint32_t sCount[LG_CHUNK];
    __shared__ uint32_t sBias[LG_CHUNK];
    __shared__ uint64_t sKey[LG_THREADS / 64];
    const int64_t b = blockIdx.y;
    const int t = threadIdx.x, c0 = blockIdx.x * LG_CHUNK, n = min(LG_CHUNK, a.V - c0);
    if (a.tokens) for (int i = t; i < LG_CHUNK; i += LG_THREADS) sCount[i] = 0;
    if (a.bias_ids) for (int i = t; i < LG_CHUNK; i += LG_THREADS) sBias[i] = 0;
    __syncthreads();
    if (a.tokens) {
        const int nt = (int)max((int64_t)0, min((int64_t)a.n_tokens[b], a.token_stride));
        const int np = a.n_prompt ? max(0, min(a.n_prompt[b], nt)) : 0;
        const int32_t* ids = a.tokens + b * a.token_stride;
        for (int i = t; i < nt; i += LG_THREADS) {
            const uint32_t at = (uint32_t)ids[i] - (uint32_t)c0;
            if (at < (uint32_t)n) {
                if (i < np) atomicOr(&sCount[at], LG_PROMPT);
                else atomicAdd(&sCount[at], 1u);
            }
        }
    }
    if (a.bias_ids) {
        const int nb = (int)max((int64_t)0, min((int64_t)a.n_bias[b], a.bias_stride));
        const int32_t* ids = a.bias_ids + b * a.bias_stride;
        for (int i = t; i < nb; i += LG_THREADS) {
            const uint32_t at = (uint32_t)ids[i] - (uint32_t)c0;
            if (at < (uint32_t)n) atomicMax(&sBias[at], (uint32_t)i + 1u);
        }
    }
    __syncthreads();
    const float rep = a.repetition ? a.repetition[b] : 1.0f;
    const float freq = a.frequency ? a.frequency[b] : 0.0f, pres = a.presence ? a.presence[b] : 0.0f;
    const float* x = a.x + b * a.x_stride + c0;
    float* out = a.out + b * a.out_stride + c0;
    uint64_t best = 0;
    for (int i = t; i < n; i += LG_THREADS) {
        float y = x[i];
        if (a.tokens) {
            const uint32_t c = sCount[i];
            if (c) {
                y = y > 0.0f ? y / rep : y * rep;
                const uint32_t cnt = c & ~LG_PROMPT;
                if (cnt) { y = y - freq * (float)cnt; y = y - pres; }
            }
        }
        if (a.bias_ids) {
            const uint32_t j = sBias[i];
            if (j) y = y + a.bias[b * a.bias_stride + j - 1];
        }
        if (a.mask && !((a.mask[b * a.mask_stride + ((c0 + i) >> 5)] >> (i & 31)) & 1u)) y = -INFINITY;
        out[i] = y;
        const uint64_t k = pick_key(y, c0 + i);
        best = k > best ? k : best;
    }
    if (!a.next_token) return;
    best = wave_max_key(best);
    if ((t & 63) == 0) sKey[t >> 6] = best;
    __syncthreads();
    if (t == 0) {
        for (int w = 1; w < LG_THREADS / 64; w++) best = sKey[w] > best ? sKey[w] : best;
        if (gridDim.x == 1) a.next_token[b] = best ? (int32_t)~(uint32_t)best : -1;
        else a.cand[b * gridDim.x + blockIdx.x] = best;
    }
}

__global__ __launch_bounds__(64) void logits_pick_kernel(int32_t* tok, const uint64_t* cand, int chunks) {
    const int64_t b = blockIdx.x;
    uint64_t best = 0;
    for (int i = threadIdx.x; i < chunks; i += 64) {
        const uint64_t k = cand[b * chunks + i];
        best = k > best ? k : best;
    }
    best = wave_max_key(best);
    if (threadIdx.x == 0) tok[b] = best ? (int32_t)~(uint32_t)best : -1;
}

namespace {
int logits_chunks(int V) { return (int)(((int64_t)V + LG_CHUNK - 1) / LG_CHUNK); }
}  // namespace

int64_t logits_workspace(int B, int V) {
    const int n = logits_chunks(V);
    return n > 1 ? (int64_t)B * n * 8 : 0;
}

hipError_t logits_launch(const LogitsArgs& a, hipStream_t st) {
    const int n = logits_chunks(a.V);
    hipLaunchKernelGGL(logits_kernel, dim3(n, a.B), dim3(LG_THREADS), 0, st, a);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || !a.next_token || n == 1) return e;
    hipLaunchKernelGGL(logits_pick_kernel, dim3(a.B), dim3(64), 0, st, a.next_token, (const uint64_t*)a.cand, n);
    return hipGetLastError();
}

}  // namespace jllm_hip
