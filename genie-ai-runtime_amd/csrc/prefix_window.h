// prefix_window.h -- which keys of a shared prefix a window leaves a row.
#pragma once
#include <stdint.h>

namespace jllm_hip {

// The first of the prefix's len keys that a row with n tokens of its own sees when it attends
// to the last `window` of both: [0, len], len for none.  (len + n may pass 31 bits.)
constexpr int first_seen(int len, int n, int window) {
    const int64_t first = (int64_t)len + n - window;
    return first < 0 ? 0 : (first < len ? (int)first : len);
}

}  // namespace jllm_hip
