// CPU check of the forms that sizes of the product of 8-bit codes take
// (genie-ai-runtime_amd/csrc/gemm_i8_plan.h): reads "M N K" lines, prints the plan of each.
// Test infrastructure, not part of the library.
#include <cstdio>
#include "gemm_i8_plan.h"

int main() {
    int M, N, K;
    while (std::scanf("%d %d %d", &M, &N, &K) == 3) {
        const jllm_hip::GemmPlan p = jllm_hip::gemm_plan(M, N, K);
        std::printf("%d %d %d %d\n", p.few, p.tile, p.splits, p.whole);
    }
    return 0;
}
