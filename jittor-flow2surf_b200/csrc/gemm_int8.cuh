// The 8-bit product's operands and its tensor-core forms.
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

// On tcgen05: x and w 16-byte aligned with pitches of multiples of 16.
int linear_int8_tensor(const Int8Args& g, cudaStream_t st);

}  // namespace f2s
