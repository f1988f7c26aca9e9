// Root-mean-square norm of a residual stream, with the residual's addition:
//   s = x + r (rounded to the stream's type, as it is stored)
//   y = s rstd w,  rstd = (mean(s^2) + eps)^-1/2
// and its backward, or y as 8-bit rows with one scale each:
//   q = rint(127 s w / m), m = max |s w|, scale = m rstd / 127.
// rstd cancels in q, so the sum and the maximum come from one reduction and q
// is the exact rounding whatever the order of the sum.
//
// All are bound by memory: the forward reads x, r and writes s, y (8 bytes per
// channel in 16 bits, 7 with 8-bit rows), the backward reads s, dy, ds and
// writes dx (8 bytes). Rows are held in registers (row_ops.cuh), so each is
// read once.
#include <type_traits>

#include "kernels.cuh"
#include "row_ops.cuh"

namespace f2s {
namespace {

using namespace rows;

struct NormArgs {
    const void* x;
    int64_t ldx;
    const void* residual;  // null: none (s = x, `stream` not written)
    int64_t ldr;
    const void* weight;
    int64_t nrows;
    int C;
    float eps;
    void* stream;  // (nrows, C)
    void* y;       // (nrows, C), or
    int8_t* q;     // 8-bit rows of pitch ldq
    int64_t ldq;
    float* scale;
};

// The row, so that what follows from it is computed anew.
__device__ __forceinline__ int64_t opaque(int64_t row) {
    asm volatile("" : "+l"(row));
    return row;
}

// A row that fp32 does not carry, in 64 bits, which hold every square and product of two
// fp32 values: one whose squares leave fp32 (magnitudes above 1e18, or tiny ones with an
// eps that does not hide them: the reciprocal root of a subnormal row is past 3.4e38
// itself), or, for 8-bit rows, one whose largest product s w lies outside of
// [1e-30, 1e30] (beyond 3.4e38 products are infinite in fp32, below 1.2e-38 they lose
// bits). Almost no row is one: it is written again, value by value, after the kernel has
// written it as any other, in a call of its own that is given the row's number alone, so
// that it takes no registers from the others.
template <typename T, int E, int TPR, Mode kMode, bool k8>
__device__ __noinline__ void row_in_64_bits(const NormArgs& g, int64_t row) {
    using S = Slice<T, E, TPR, kMode>;
    __shared__ double shared_a[32];
    __shared__ unsigned long long shared_m[32];
    const int t = TPR <= 32 ? threadIdx.x % TPR : threadIdx.x;
    const bool live = row < g.nrows;
    const int C = live ? g.C : 0;
    if (!live) row = 0;
    // the stream: x, or this thread's own channels of it
    const T* s = g.residual ? static_cast<const T*>(g.stream) + row * (int64_t)g.C
                            : static_cast<const T*>(g.x) + row * g.ldx;
    const T* w = static_cast<const T*>(g.weight);
    double sum = 0.0;
    unsigned long long bits = 0;
#pragma unroll 1
    for (int i = 0; i < S::kEach; ++i) {
        const int c = S::channel(i, t);
        if (c >= C) break;
        const double a = (double)to_f32<T>(s[c]);
        sum = fma(a, a, sum);
        if constexpr (k8) {
            const auto p = (unsigned long long)__double_as_longlong(fabs(a * (double)to_f32<T>(w[c])));
            bits = p > bits ? p : bits;
        }
    }
    row_sum_max<TPR, true, k8>(sum, bits, shared_a, shared_m);
    const double rstd = 1.0 / sqrt(sum / (double)g.C + (double)g.eps);
    const double m = __longlong_as_double((long long)bits);
    const bool finite = m < (double)kInf;
#pragma unroll 1
    for (int i = 0; i < S::kEach; ++i) {
        const int c = S::channel(i, t);
        if (c >= C) break;
        const double a = (double)to_f32<T>(s[c]), b = (double)to_f32<T>(w[c]);
        if constexpr (k8) g.q[row * g.ldq + c] = (int8_t)(finite && m > 0.0 ? nearest_whole(a * b, m) : 0);
        else static_cast<T*>(g.y)[row * (int64_t)g.C + c] = from_f32<T>((float)(a * rstd * b));
    }
    if (k8 && live && t == 0) g.scale[row] = finite ? (float)(m / 127.0 * rstd) : __int_as_float(0x7fc00000);
}

// 8 single bf16 values with 8-bit rows stay at 48 registers for a fifth 256-thread
// block per SM: 65,536 x 191 36 us against 41.
template <typename T, int E, int TPR, Mode kMode, bool k8>
constexpr int norm_resident() {
    constexpr int threads = block_threads(TPR);
    if (k8 && kMode == kSingle && E == 8 && std::is_same<T, __nv_bfloat16>::value && threads <= 256) return 1280 / threads;
    return resident(threads, E, 2 * held_size(sizeof(T), kMode));
}

// k8: 8-bit rows. The products s w of a 16-bit type are exact in fp32 where they stay
// in its range; those of fp32 are taken in 64 bits for the maximum and at rounding
// borders.
template <typename T, int E, int TPR, Mode kMode, bool k8>
__global__ void __launch_bounds__(block_threads(TPR), norm_resident<T, E, TPR, kMode, k8>())
add_rms_norm_kernel(const __grid_constant__ NormArgs g) {
    using S = Slice<T, E, TPR, kMode>;
    constexpr bool kExact64 = k8 && sizeof(T) == 4;
    using M = typename std::conditional<kExact64, unsigned long long, float>::type;
    __shared__ M shared_m[32];
    __shared__ float shared_a[32];
    const int t = TPR <= 32 ? threadIdx.x % TPR : threadIdx.x;
    const int64_t row = TPR <= 32 ? (int64_t)blockIdx.x * (256 / TPR) + threadIdx.x / TPR : (int64_t)blockIdx.x;
    // rows past the end take part in the shuffles and write nothing
    const bool live = row < g.nrows;
    const int C = live ? g.C : 0;
    const int64_t at = live ? row : 0;
    const T* weight = static_cast<const T*>(g.weight);
    const T* from = static_cast<const T*>(g.x) + at * g.ldx;
    Held<T, E, kMode> s, w;
    load_held<TPR>(from, C, t, s);
    if (g.residual) {
        Held<T, E, kMode> r;
        load_held<TPR>(static_cast<const T*>(g.residual) + at * g.ldr, C, t, r);
        load_held<TPR>(weight, C, t, w);
#pragma unroll
        for (int i = 0; i < E; i += 8) {
            float a[8], b[8];
            s.get(i, a);
            r.get(i, b);
#pragma unroll
            for (int j = 0; j < 8; ++j) a[j] += b[j];
            s.set(i, a);
        }
        T* to = static_cast<T*>(g.stream) + at * (int64_t)g.C;
        store_held<TPR>(to, C, t, s);
        from = to;
    } else {
        load_held<TPR>(weight, C, t, w);
    }
    float sum = 0.0f;
    M m = 0;
    uint32_t seen = 0;
    if constexpr (k8 && std::is_same<T, __nv_bfloat16>::value) seen = s.magnitudes();
#pragma unroll
    for (int i = 0; i < E; i += 8) {
        float a[8], b[8];
        s.get(i, a);
        w.get(i, b);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            sum = fmaf(a[j], a[j], sum);
            if constexpr (kExact64) {
                const M p = (M)__double_as_longlong(fabs((double)a[j] * (double)b[j]));
                m = p > m ? p : m;
            } else if constexpr (k8) {
                b[j] *= a[j];
            }
        }
        if constexpr (k8 && !kExact64) m = max_abs(b, m);
    }
    row_sum_max<TPR, true, k8>(sum, m, shared_a, shared_m);
    const float rstd = reciprocal_rms(sum, g.C, g.eps);
    bool odd = live && squares_leave_fp32(sum, g.eps), some = odd;
    if constexpr (k8) {
        using L = typename std::conditional<kExact64, double, float>::type;
        L largest;
        if constexpr (kExact64) largest = __longlong_as_double((long long)m);
        else largest = m;
        const Rounding<L> rounding(largest);
#pragma unroll
        for (int i = 0; i < E; i += 8) {
            float a[8], b[8];
            s.get(i, a);
            w.get(i, b);
#pragma unroll
            for (int j = 0; j < 8; ++j) a[j] *= b[j];
            if constexpr (kExact64) {
                // `from` holds the stream: x, or this thread's own channels of it
                store8_chunk<false, S, kMode>(g.q + at * g.ldq, C, t, i, a, rounding, [&](int j) {
                    const int c = S::channel(i + j, t);
                    return c < C ? (double)from[c] * (double)weight[c] : 0.0;
                });
            } else {
                // products of bf16 have 16 bits, of fp16 22
                store8_chunk<std::is_same<T, __nv_bfloat16>::value, S, kMode>(
                    g.q + at * g.ldq, C, t, i, a, rounding, [&](int j) { return a[j]; });
            }
        }
        if (live && t == 0)
            g.scale[row] = (float)largest < kInf ? (float)((double)largest / 127.0 * (double)rstd)
                                                 : __int_as_float(0x7fc00000);
        const bool outside = live && !((float)largest >= kTiny && (float)largest <= kHuge);
        // a row without products needs no more, one of the rows that pad a batch; where
        // they are 0 in fp32 alone, some of its values are not 0
        some = kExact64 ? largest != (L)0 : largest != (L)0 || seen != 0;
        some = odd || (outside && some);
        odd = odd || outside;
    } else {
#pragma unroll
        for (int i = 0; i < E; i += 8) {
            float a[8], b[8];
            s.get(i, a);
            w.get(i, b);
#pragma unroll
            for (int j = 0; j < 8; ++j) a[j] = a[j] * rstd * b[j];
            s.set(i, a);
        }
        store_held<TPR>(static_cast<T*>(g.y) + at * (int64_t)g.C, C, t, s);
    }
    // fp16 has neither such squares nor such products
    if constexpr (!std::is_same<T, __half>::value) {
        // all threads of a row of several warps agree on `odd`, not on `some`
        bool again = TPR > 32 ? odd : __any_sync(0xffffffffu, odd);
        if (k8 && again) again = TPR > 32 ? __syncthreads_or(some) : __any_sync(0xffffffffu, some);
        if (again) row_in_64_bits<T, E, TPR, kMode, k8>(g, opaque(row));
    }
}

template <bool k8>
int norm_launch(const NormArgs& g, int dtype, cudaStream_t st) {
    const int size = dtype_size(dtype);
    Layout layout(g.nrows, g.C, size);
    layout.rows(g.x, g.ldx).rows(g.residual, g.ldr).rows(g.stream, g.C).rows(g.y, g.C).vector(g.weight);
    if (k8) layout.eight(g.q, g.ldq);
    const Mode mode = layout.mode();
    const Shape s = pick_shape(kForward, size, g.nrows, g.C, mode);
    const int64_t blocks = ceil_div64(g.nrows, block_rows(s.tpr));
    F2S_LIMIT(blocks <= INT32_MAX, "add_rms_norm: %lld rows", (long long)g.nrows);
    TraceScope trace(kTagRmsNorm, st);
    F2S_DTYPE_SWITCH(dtype, dispatch<kForward, T>(s, mode, [&](auto e, auto tpr, auto m) {
        add_rms_norm_kernel<T, e.value, tpr.value, m.value, k8>
            <<<(unsigned)blocks, block_threads(tpr.value), 0, st>>>(g);
    }));
    return check_launch("add_rms_norm_kernel");
}

}  // namespace
}  // namespace f2s

extern "C" int f2s_add_rms_norm(const void* x, int64_t ldx, const void* residual, int64_t ldr, const void* weight,
                                int dtype, int64_t rows, int C, float eps, void* stream_out, void* y, void* stream) {
    F2S_TRY(f2s::check_norm("add_rms_norm", dtype, rows, C, eps));
    if (rows == 0) return F2S_OK;
    F2S_REQUIRE(x && weight && y && (!residual || stream_out), "add_rms_norm: null pointer");
    F2S_REQUIRE(ldx >= C && (!residual || ldr >= C), "add_rms_norm: row pitch below C=%d", C);
    f2s::NormArgs g{x, ldx, residual, ldr, weight, rows, C, eps, stream_out, y, nullptr, 0, nullptr};
    return f2s::norm_launch<false>(g, dtype, f2s::as_stream(stream));
}

extern "C" int f2s_add_rms_norm_int8(const void* x, int64_t ldx, const void* residual, int64_t ldr,
                                     const void* weight, int dtype, int64_t rows, int C, float eps, void* stream_out,
                                     int8_t* q, int64_t ldq, float* scale, void* stream) {
    F2S_TRY(f2s::check_norm("add_rms_norm_int8", dtype, rows, C, eps));
    if (rows == 0) return F2S_OK;
    F2S_REQUIRE(x && weight && q && scale && (!residual || stream_out), "add_rms_norm_int8: null pointer");
    F2S_REQUIRE(ldx >= C && ldq >= C && (!residual || ldr >= C), "add_rms_norm_int8: row pitch below C=%d", C);
    f2s::NormArgs g{x, ldx, residual, ldr, weight, rows, C, eps, stream_out, nullptr, q, ldq, scale};
    return f2s::norm_launch<true>(g, dtype, f2s::as_stream(stream));
}
