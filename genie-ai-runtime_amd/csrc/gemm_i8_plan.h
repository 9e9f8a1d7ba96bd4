// gemm_i8_plan.h -- which form of the product of 8-bit codes a size takes (host only).
#pragma once
#include <stdint.h>

namespace jllm_hip {

constexpr int GT_K = 128;              // codes of a row in a stage of a tile

// How the product is cut.  What a stage of 128 codes costs a CU with one tile of a kind at
// work and with as many as fit, and what a tile costs beside its stages, alone and full, in
// us (fitted to 64 stages and 16, half a round of tiles to twelve):
//   256 x 256            1.71        10.3
//   128 x 256            0.93         6.3       (251 tokens x 32003 channels in 128 x 128 45 us where this took 39)
//   128 x 128, two       0.86, 0.98   3.5, 7.0
//   64 x 64, two         0.28, 0.49   3.0, 3.3  (256 tokens, 4096 x 4096 14.6; 21 with 128 x 128)
//   32 x 64, up to three 0.24, 0.55   2.5, 3.0  (64 tokens, 6144 x 2560 9.5; 11 with 64 x 64)
// Sums of parts: 4 us and their bytes twice at 6 TB/s (64 tokens, 2560 x 9728 in 6 parts
// 14.1; 26 in one).  The plan is what these say takes least.
// Few tokens: from 16384 channels a wave has 16 pieces on the way; from 8192 codes 16 waves
// share K, where there is no more than a workgroup for each CU (4096 x 28672, one token 25.1 us,
// 27.8 with four; with two a CU it is near: 8192 x 9728 18.3 and 19.2, 8 tokens 21.5 either way).
enum { FEW_NONE, FEW, FEW_MANY_CHANNELS, FEW_LONG_K };
struct GemmPlan { int few, tile, splits, whole; };
struct TileKind { int tm, tn, share; float alone, full, tile, tiles; };
constexpr TileKind GEMM_TILES[] = {{256, 256, 1, 1.71f, 1.71f, 10.3f, 10.3f}, {128, 256, 1, 0.93f, 0.93f, 6.3f, 6.3f}, {128, 128, 2, 0.86f, 0.98f, 3.5f, 7.0f},
                              {64, 64, 2, 0.28f, 0.49f, 3.0f, 3.3f}, {32, 64, 3, 0.24f, 0.55f, 2.5f, 3.0f}};
inline GemmPlan gemm_plan(int M, int N, int K) {
    GemmPlan best = {};
    best.splits = 1;
    if (N <= 16) {
        best.few = M >= 16384 ? FEW_MANY_CHANNELS : (K >= 8192 && M <= 4096 ? FEW_LONG_K : FEW);
        return best;
    }
    float least = 1e30f;
    const int stages = (K + GT_K - 1) / GT_K;
    for (int k = 0; k < 5; k++) {
        const TileKind& t = GEMM_TILES[k];
        const int64_t n = (((int64_t)M + t.tm - 1) / t.tm) * (((int64_t)N + t.tn - 1) / t.tn), room = 256 * t.share;
        for (int s = 1; s <= 16; s++) {
            if (s > 1 && (s * 4 > stages || n * s > room)) break;
            const float st = (float)((stages + s - 1) / s);
            const int64_t wgs = n * s, rest = wgs % room;
            float us = (float)(wgs / room) * (st * t.full + t.tiles);
            int whole = 0;
            if (k == 0 && s == 1 && n > room && rest > 0 && rest <= room / 2) {
                whole = (int)(n - rest);               // the rest as halves
                us += st * 1.05f + 6.5f;
            } else if (rest > 0) {
                const float f = t.share > 1 ? (float)((rest - 1) / 256) / (float)(t.share - 1) : 0.0f;
                us += st * (t.alone + f * (t.full - t.alone)) + t.tile + f * (t.tiles - t.tile);
            }
            if (s > 1) us += 4.0f + (float)s * (float)M * (float)N * (8.0f / 6e6f);
            if (us < least) {
                least = us;
                best.tile = k; best.splits = s; best.whole = whole;
            }
        }
    }
    return best;
}

}  // namespace jllm_hip
