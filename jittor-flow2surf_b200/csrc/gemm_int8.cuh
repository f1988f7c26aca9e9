// The 8-bit product's operands and its two tensor-core forms (linear_int8.cu
// chooses).
#pragma once

#include "common.cuh"

namespace f2s {

struct Int8Args {
    const int8_t* x;  // (rows, K), pitch ldx
    int64_t ldx;
    const float* xs;
    const int8_t* w;  // (cols, K), pitch ldw
    int64_t ldw;
    const float* ws;
    const void* bias;  // of y's type, or null
    void* y;           // (rows, cols), pitch ldy
    int64_t ldy;
    int dtype;
    int rows, cols, K;
};

// x and w 16-byte aligned with pitches of multiples of 16.
int linear_int8_tiles(const Int8Args& g, cudaStream_t st);  // 128 channels x up to 128 tokens, K split
int linear_int8_pairs(const Int8Args& g, cudaStream_t st);  // 256 x 256 tiles by CTA pairs

}  // namespace f2s
