// What the kernels of attention over paged caches share (paged_attention.cu, paged_attention_tc.cu).
#pragma once
#include "paged.cuh"

namespace paged {

constexpr float kLog2e = 1.4426950408889634f;

struct AttendArgs {
    View p;
    const void* q;             // [T, H, D]
    void* out;                 // [T, H * E]
    const float* sink;         // [H], nullable
    float* lse;                // [T, H] in units of log 2; where mass is kept
    int H, window, first;
    float c;                   // scale log2 e
};

}  // namespace paged
