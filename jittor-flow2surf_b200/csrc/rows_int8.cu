// Rows of 8-bit integers with one scale each: a row v of m = max |v| becomes
// q = rint(127 v / m) and scale = m / 127, and stands for scale q.
// Bound by memory: 3 bytes per channel of a 16-bit type, 5 of fp32.
#include "kernels.cuh"
#include "row_ops.cuh"

namespace f2s {
namespace {

using namespace rows;

template <typename T, int E, int TPR, Mode kMode>
__global__ void __launch_bounds__(block_threads(TPR), resident(block_threads(TPR), E, held_size(sizeof(T), kMode)))
quantize_rows_kernel(const T* __restrict__ x, int64_t ldx, int64_t nrows, int width, int8_t* __restrict__ q8,
                     int64_t ldq, float* __restrict__ scale) {
    using S = Slice<T, E, TPR, kMode>;
    __shared__ float shared_m[32];
    const int t = TPR <= 32 ? threadIdx.x % TPR : threadIdx.x;
    const int64_t row = TPR <= 32 ? (int64_t)blockIdx.x * (256 / TPR) + threadIdx.x / TPR : (int64_t)blockIdx.x;
    const bool live = row < nrows;
    const int64_t at = live ? row : 0;
    const int C = live ? width : 0;
    const T* from = x + at * ldx;
    Held<T, E, kMode> held;
    load_held<TPR>(from, C, t, held);
    float m = 0.0f, none = 0.0f;
#pragma unroll
    for (int i = 0; i < E; i += 8) {
        float v[8];
        held.get(i, v);
        m = max_abs(v, m);
    }
    row_sum_max<TPR, false, true>(none, m, shared_m, shared_m);
    const Rounding<float> rounding(m);
#pragma unroll
    for (int i = 0; i < E; i += 8) {
        float v[8];
        held.get(i, v);
        store8_chunk<sizeof(T) == 2, S, kMode>(q8 + at * ldq, C, t, i, v, rounding, [&](int j) { return v[j]; });
    }
    if (live && t == 0) scale[row] = m < kInf ? m / 127.0f : __int_as_float(0x7fc00000);
}

// y = scale q, 16 channels (one 16-byte load) per thread.
template <typename T>
__global__ void __launch_bounds__(256)
dequantize_rows_kernel(const int8_t* __restrict__ q8, int64_t ldq, const float* __restrict__ scale, int per_row,
                       int64_t items, T* __restrict__ y, int64_t ldy) {
    const int64_t item = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (item >= items) return;
    const int64_t row = items <= INT32_MAX ? (int64_t)((uint32_t)item / (uint32_t)per_row) : item / per_row;
    const int c = (int)(item - row * per_row) * 16;
    const float s = scale[row];
    const uint4 u = *reinterpret_cast<const uint4*>(q8 + row * ldq + c);
    float v[16];
    widen8(u.x, v);
    widen8(u.y, v + 4);
    widen8(u.z, v + 8);
    widen8(u.w, v + 12);
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] *= s;
    uint4* to = reinterpret_cast<uint4*>(y + row * ldy + c);
#pragma unroll
    for (int i = 0; i < 16 / kVec<T>; ++i) to[i] = pack16<T>(v + i * kVec<T>);
}

// The same for any pitch and width: a warp takes 256 channels of a row, eight
// per lane, 32 apart.
template <typename T>
__global__ void __launch_bounds__(256)
dequantize_any_kernel(const int8_t* __restrict__ q8, int64_t ldq, const float* __restrict__ scale, int width,
                      int per_row, int64_t items, T* __restrict__ y, int64_t ldy) {
    const int64_t item = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    if (item >= items) return;
    const int64_t row = items <= INT32_MAX ? (int64_t)((uint32_t)item / (uint32_t)per_row) : item / per_row;
    const int c = (int)(item - row * per_row) * 256 + (threadIdx.x & 31);
    const int8_t* from = q8 + row * ldq + c;
    T* to = y + row * ldy + c;
    const float s = scale[row];
    int v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = c + 32 * i < width ? from[32 * i] : 0;
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (c + 32 * i < width) to[32 * i] = from_f32<T>((float)v[i] * s);
}

template <typename T>
int quantize_launch(const void* x, int64_t ldx, int64_t nrows, int C, int8_t* q, int64_t ldq, float* scale,
                    cudaStream_t st) {
    const Mode mode = Layout(nrows, C, sizeof(T)).rows(x, ldx).eight(q, ldq).mode();
    const Shape s = pick_shape(kForward, sizeof(T), nrows, C, mode);
    const int64_t blocks = ceil_div64(nrows, block_rows(s.tpr));
    F2S_LIMIT(blocks <= INT32_MAX, "quantize_rows: %lld rows", (long long)nrows);
    TraceScope trace(kTagRows8, st);
    dispatch<kForward, T>(s, mode, [&](auto e, auto tpr, auto m) {
        quantize_rows_kernel<T, e.value, tpr.value, m.value><<<(unsigned)blocks, block_threads(tpr.value), 0, st>>>(
            static_cast<const T*>(x), ldx, nrows, C, q, ldq, scale);
    });
    return check_launch("quantize_rows_kernel");
}

template <typename T>
int dequantize_launch(const int8_t* q, int64_t ldq, const float* scale, int64_t nrows, int C, void* y, int64_t ldy,
                      cudaStream_t st) {
    const bool wide = C % 16 == 0 && aligned16(q) && aligned16(y) &&
                      ((ldq % 16 == 0 && ldy % kVec<T> == 0) || nrows == 1);
    const int per_row = wide ? C / 16 : ceil_div(C, 256);
    const int64_t items = nrows * per_row, blocks = ceil_div64(items, wide ? 256 : 8);
    F2S_LIMIT(blocks <= INT32_MAX, "dequantize_rows: %lld rows of %d", (long long)nrows, C);
    TraceScope trace(kTagRows8, st);
    T* to = static_cast<T*>(y);
    if (wide) dequantize_rows_kernel<T><<<(unsigned)blocks, 256, 0, st>>>(q, ldq, scale, per_row, items, to, ldy);
    else dequantize_any_kernel<T><<<(unsigned)blocks, 256, 0, st>>>(q, ldq, scale, C, per_row, items, to, ldy);
    return check_launch("dequantize_rows_kernel");
}

}  // namespace
}  // namespace f2s

extern "C" int f2s_quantize_rows(const void* x, int64_t ldx, int dtype, int64_t rows, int C, int8_t* q, int64_t ldq,
                                 float* scale, void* stream) {
    F2S_TRY(f2s::rows::check_dtype("quantize_rows", dtype));
    F2S_REQUIRE(rows >= 0 && C >= 1, "quantize_rows: bad shape rows=%lld C=%d", (long long)rows, C);
    F2S_LIMIT(C <= f2s::rows::kMaxRow, "quantize_rows: C=%d, at most %d channels", C, f2s::rows::kMaxRow);
    if (rows == 0) return F2S_OK;
    F2S_REQUIRE(x && q && scale, "quantize_rows: null pointer");
    F2S_REQUIRE(ldx >= C && ldq >= C, "quantize_rows: row pitch below C=%d", C);
    int status = F2S_OK;
    F2S_DTYPE_SWITCH(dtype, status = f2s::quantize_launch<T>(x, ldx, rows, C, q, ldq, scale, f2s::as_stream(stream)));
    return status;
}

extern "C" int f2s_dequantize_rows(const int8_t* q, int64_t ldq, const float* scale, int64_t rows, int C, void* y,
                                   int64_t ldy, int dtype, void* stream) {
    F2S_TRY(f2s::rows::check_dtype("dequantize_rows", dtype));
    F2S_REQUIRE(rows >= 0 && C >= 1, "dequantize_rows: bad shape rows=%lld C=%d", (long long)rows, C);
    F2S_LIMIT(C <= INT32_MAX - 255, "dequantize_rows: C=%d, at most 2^31 - 256 channels", C);
    if (rows == 0) return F2S_OK;
    F2S_REQUIRE(q && scale && y, "dequantize_rows: null pointer");
    F2S_REQUIRE(ldq >= C && ldy >= C, "dequantize_rows: row pitch below C=%d", C);
    int status = F2S_OK;
    F2S_DTYPE_SWITCH(dtype, status = f2s::dequantize_launch<T>(q, ldq, scale, rows, C, y, ldy, f2s::as_stream(stream)));
    return status;
}
