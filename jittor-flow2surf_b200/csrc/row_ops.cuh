// Row operators on 16- and 32-bit activations: how a row is spread over
// threads and held in registers, its reductions, and the rounding to 8 bits.
//
// A row of up to kMaxRow channels is read once, held in E fp32 registers of
// each of TPR threads (TPR 8 or 32: several rows per block, reduced with
// shuffles; 128 and up: one row per block), and everything that needs it is
// computed from there.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace f2s {
namespace rows {

constexpr int kMaxRow = 32768;

template <typename T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }

template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }

__device__ __forceinline__ float2 unpack2(uint32_t u, __nv_bfloat16) {
    return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
}
__device__ __forceinline__ float2 unpack2(uint32_t u, __half) {
    return __half22float2(*reinterpret_cast<const __half2*>(&u));
}
__device__ __forceinline__ uint32_t pack2(float a, float b, __nv_bfloat16) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack2(float a, float b, __half) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// One 16-byte access: 8 values of a 16-bit type, 4 of fp32.
template <typename T>
constexpr int kVec = 16 / (int)sizeof(T);

template <typename T>
__device__ __forceinline__ void unpack16(uint4 u, float* v) {
    if constexpr (sizeof(T) == 4) {
        v[0] = __uint_as_float(u.x);
        v[1] = __uint_as_float(u.y);
        v[2] = __uint_as_float(u.z);
        v[3] = __uint_as_float(u.w);
    } else {
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = unpack2(w[i], T());
            v[2 * i] = f.x;
            v[2 * i + 1] = f.y;
        }
    }
}

template <typename T>
__device__ __forceinline__ uint4 pack16(const float* v) {
    if constexpr (sizeof(T) == 4) {
        return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]),
                          __float_as_uint(v[3]));
    } else {
        return make_uint4(pack2(v[0], v[1], T()), pack2(v[2], v[3], T()), pack2(v[4], v[5], T()),
                          pack2(v[6], v[7], T()));
    }
}

// The E channels of a row that thread `t` of TPR holds. kWide: 16-byte
// vectors (the row's start 16-byte aligned, C a multiple of the vector),
// vector i of the thread at (i TPR + t); otherwise single values, value i at
// i TPR + t. Channels past C read as 0 and are not written.
template <typename T, int E, int TPR, bool kWide>
struct Slice {
    static constexpr int V = kWide ? kVec<T> : 1;
    static_assert(E % V == 0, "whole vectors");

    __device__ static __forceinline__ int channel(int i, int t) {
        return ((i / V) * TPR + t) * V + i % V;
    }

    __device__ static __forceinline__ void load(const T* row, int C, int t, float (&v)[E]) {
#pragma unroll
        for (int i = 0; i < E; i += V) {
            const int c = channel(i, t);
            if constexpr (kWide) {
                const uint4 u = c < C ? *reinterpret_cast<const uint4*>(row + c) : make_uint4(0, 0, 0, 0);
                unpack16<T>(u, &v[i]);
            } else {
                v[i] = c < C ? to_f32<T>(row[c]) : 0.0f;
            }
        }
    }

    __device__ static __forceinline__ void store(T* row, int C, int t, const float (&v)[E]) {
#pragma unroll
        for (int i = 0; i < E; i += V) {
            const int c = channel(i, t);
            if (c >= C) continue;
            if constexpr (kWide) *reinterpret_cast<uint4*>(row + c) = pack16<T>(&v[i]);
            else row[c] = from_f32<T>(v[i]);
        }
    }

    // low bytes of q[i]; `row` 8-byte aligned where kWide (a multiple of 16 in fact)
    __device__ static __forceinline__ void store8(int8_t* row, int C, int t, const uint32_t (&q)[E]) {
#pragma unroll
        for (int i = 0; i < E; i += V) {
            const int c = channel(i, t);
            if (c >= C) continue;
            if constexpr (kWide) {
                uint32_t w[V / 4];
#pragma unroll
                for (int j = 0; j < V / 4; ++j)
                    w[j] = __byte_perm(__byte_perm(q[i + 4 * j], q[i + 4 * j + 1], 0x0040),
                                       __byte_perm(q[i + 4 * j + 2], q[i + 4 * j + 3], 0x0040), 0x5410);
                if constexpr (V == 8) *reinterpret_cast<uint2*>(row + c) = make_uint2(w[0], w[1]);
                else *reinterpret_cast<uint32_t*>(row + c) = w[0];
            } else {
                row[c] = (int8_t)(q[i] & 0xffu);
            }
        }
    }
};

// v rounded to T and back: what a row stored in T holds.
template <typename T>
__device__ __forceinline__ float rounded(float v) {
    return to_f32<T>(from_f32<T>(v));
}

__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }
constexpr uint32_t kInfBits = 0x7f800000u;
constexpr unsigned long long kInfBits64 = 0x7ff0000000000000ull;

// Sum of `a` (fp32) and maximum of `m` over the TPR threads of a row; every
// thread gets both. Magnitudes are compared as bit patterns, so that infinity
// and NaN, whose patterns lie above every finite value's, are not lost as in
// a floating-point maximum. `shared` holds 2 * TPR / 32 entries for TPR > 32;
// two uses need a barrier between them.
template <int TPR, typename M>
__device__ __forceinline__ void row_sum_max(float& a, M& m, M* shared_m, float* shared_a) {
    constexpr int kWidth = TPR < 32 ? TPR : 32;
#pragma unroll
    for (int o = kWidth / 2; o > 0; o >>= 1) {
        a += __shfl_xor_sync(0xffffffffu, a, o);
        const M other = __shfl_xor_sync(0xffffffffu, m, o);
        m = other > m ? other : m;
    }
    if constexpr (TPR > 32) {
        constexpr int kWarps = TPR / 32;
        const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
        if (lane == 0) {
            shared_a[warp] = a;
            shared_m[warp] = m;
        }
        __syncthreads();
        a = lane < kWarps ? shared_a[lane] : 0.0f;
        m = lane < kWarps ? shared_m[lane] : M(0);
#pragma unroll
        for (int o = kWarps / 2; o > 0; o >>= 1) {
            a += __shfl_xor_sync(0xffffffffu, a, o);
            const M other = __shfl_xor_sync(0xffffffffu, m, o);
            m = other > m ? other : m;
        }
        a = __shfl_sync(0xffffffffu, a, 0);
        m = __shfl_sync(0xffffffffu, m, 0);
    }
}

// ---- rounding to 8 bits ----------------------------------------------------
// q = the whole number nearest to 127 v / m (m the row's largest magnitude),
// the even one at a tie, of the exact quotient. In fp32, t = v inv with
// inv = 127 / m is off by at most 127 (2^-24 of inv, 2^-24 of a rounded v) =
// 1.6e-5, so the nearest whole number of t is the answer unless t lies within
// kBorder of a half; there (about one value in 15,000) the halves are compared
// in 64 bits, where 254 v and (2 k + 1) m are exact (v of 48 bits: to 2^-53).
constexpr float kMagic = 12582912.0f;  // 1.5 * 2^23: adding it rounds to a whole number
constexpr float kBorder = 0.49997f;
// below this m the fp32 quotient may overflow or lose bits: all in 64 bits
constexpr float kTiny = 1e-30f;

static __device__ __noinline__ uint32_t round8_exact(double v, double m) {
    double k = floor(127.0 * v / m);
    const double twice = 254.0 * v - (2.0 * k + 1.0) * m;
    // k is the floor up to its own rounding next to a whole number, where
    // both neighbours' halves are far
    if (twice > 0.0 || (twice == 0.0 && ((int)k & 1))) k += 1.0;
    k = k > 127.0 ? 127.0 : k < -127.0 ? -127.0 : k;
    return (uint32_t)(int)k;
}

// t's nearest whole number in the low bits; `off` grows to the largest
// distance of a t from it.
__device__ __forceinline__ uint32_t round8(float v, float inv, float& off) {
    const float shifted = __fmaf_rn(v, inv, kMagic);
    const float whole = __fsub_rn(shifted, kMagic);
    off = fmaxf(off, fabsf(__fmaf_rn(v, inv, -whole)));
    return __float_as_uint(shifted);
}

// E values of one thread to 8 bits, v the fp32 values and at(i) the exact
// ones. `fast`: m is finite and at least kTiny; otherwise m is zero or not
// finite (all zero bits), or tiny (all exact).
template <int E, typename F>
__device__ __forceinline__ void round8_row(const float (&v)[E], float inv, double m, bool fast,
                                           uint32_t (&q)[E], F at) {
    if (fast) {
        float off = 0.0f;
#pragma unroll
        for (int i = 0; i < E; ++i) q[i] = round8(v[i], inv, off);
        if (off > kBorder) {
#pragma unroll
            for (int i = 0; i < E; ++i) {
                float o = 0.0f;
                round8(v[i], inv, o);
                if (o > kBorder) q[i] = round8_exact(at(i), m);
            }
        }
    } else {
        const bool tiny = m > 0.0 && m < 1.0;
#pragma unroll
        for (int i = 0; i < E; ++i) q[i] = tiny ? round8_exact(at(i), m) : 0u;
    }
}

// Four 8-bit values of a word as fp32, exactly: the byte with its sign bit
// flipped becomes the low mantissa byte of 2^23.
__device__ __forceinline__ void widen8(uint32_t w, float* v) {
    w ^= 0x80808080u;
    v[0] = __uint_as_float(__byte_perm(w, 0x4b000000u, 0x7440)) - 8388736.0f;
    v[1] = __uint_as_float(__byte_perm(w, 0x4b000000u, 0x7441)) - 8388736.0f;
    v[2] = __uint_as_float(__byte_perm(w, 0x4b000000u, 0x7442)) - 8388736.0f;
    v[3] = __uint_as_float(__byte_perm(w, 0x4b000000u, 0x7443)) - 8388736.0f;
}

// ---- dispatch --------------------------------------------------------------
// (TPR, E) for a row of C channels: the fewest threads whose 32 registers
// each hold it, and then the fewest registers. With few rows (fewer threads
// in all than the SMs hold at one 512-thread block each) more threads per row
// with 8 registers each shorten the one row's latency instead.
struct Shape {
    int tpr, e;
};

inline Shape pick_shape(int64_t nrows, int C, bool wide) {
    static const int kThreads[] = {8, 32, 128, 512, 1024};
    int i = 0;
    while (i < 4 && kThreads[i] * 32 < C) ++i;
    while (i < 3 && C > kThreads[i] * 8 && nrows * kThreads[i] < (int64_t)sm_count() * 512) ++i;
    const int e = ceil_div(ceil_div(C, kThreads[i]), 8) * 8;
    // single values: 8, 16 or 32; 1,024 threads: 32
    return {kThreads[i], i == 4 || (!wide && e > 16) ? 32 : e};
}

// Rows per block and threads per block of a shape.
inline int block_threads(int tpr) { return tpr <= 32 ? 256 : tpr; }
inline int block_rows(int tpr) { return tpr <= 32 ? 256 / tpr : 1; }

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// F2S_ROW_DISPATCH(shape, wide, T, LAUNCH): LAUNCH(T, E, TPR, kWide) for the
// shape's constants.
#define F2S_ROW_E_WIDE(s, T, TPR, LAUNCH)          \
    switch ((s).e) {                               \
        case 8: LAUNCH(T, 8, TPR, true); break;    \
        case 16: LAUNCH(T, 16, TPR, true); break;  \
        case 24: LAUNCH(T, 24, TPR, true); break;  \
        default: LAUNCH(T, 32, TPR, true); break;  \
    }
#define F2S_ROW_E_SINGLE(s, T, TPR, LAUNCH)         \
    switch ((s).e) {                                \
        case 8: LAUNCH(T, 8, TPR, false); break;    \
        case 16: LAUNCH(T, 16, TPR, false); break;  \
        default: LAUNCH(T, 32, TPR, false); break;  \
    }
#define F2S_ROW_DISPATCH(s, wide, T, LAUNCH)                            \
    if (wide) {                                                         \
        switch ((s).tpr) {                                              \
            case 8: F2S_ROW_E_WIDE(s, T, 8, LAUNCH); break;             \
            case 32: F2S_ROW_E_WIDE(s, T, 32, LAUNCH); break;           \
            case 128: F2S_ROW_E_WIDE(s, T, 128, LAUNCH); break;         \
            case 512: F2S_ROW_E_WIDE(s, T, 512, LAUNCH); break;         \
            default: LAUNCH(T, 32, 1024, true); break;                  \
        }                                                               \
    } else {                                                            \
        switch ((s).tpr) {                                              \
            case 8: F2S_ROW_E_SINGLE(s, T, 8, LAUNCH); break;           \
            case 32: F2S_ROW_E_SINGLE(s, T, 32, LAUNCH); break;         \
            case 128: F2S_ROW_E_SINGLE(s, T, 128, LAUNCH); break;       \
            case 512: F2S_ROW_E_SINGLE(s, T, 512, LAUNCH); break;       \
            default: LAUNCH(T, 32, 1024, false); break;                 \
        }                                                               \
    }

// The three element types of these operators (f2s_dtype).
#define F2S_DTYPE_SWITCH(dtype, ...)                                     \
    switch (dtype) {                                                     \
        case F2S_DTYPE_F32: { using T = float; __VA_ARGS__; break; }          \
        case F2S_DTYPE_BF16: { using T = __nv_bfloat16; __VA_ARGS__; break; } \
        default: { using T = __half; __VA_ARGS__; break; }                    \
    }

inline int check_dtype(const char* what, int dtype) {
    F2S_REQUIRE(dtype == F2S_DTYPE_F32 || dtype == F2S_DTYPE_BF16 || dtype == F2S_DTYPE_F16, "%s: unknown dtype %d",
                what, dtype);
    return F2S_OK;
}

inline int dtype_size(int dtype) { return dtype == F2S_DTYPE_F32 ? 4 : 2; }

}  // namespace rows
}  // namespace f2s
