// Row operators on 16- and 32-bit activations: how a row is spread over
// threads and held in registers, its reductions, and the rounding to 8 bits.
//
// A row of up to kMaxRow channels is read once, E channels of it held in the
// registers of each of TPR threads (TPR 8 or 32: several rows per block, reduced
// with shuffles; 128 and up: one row per block), and everything that needs it is
// computed from there in fp32.
//
// Tried and not kept, on a B200: rows of any start by aligned vectors or pairs from
// the boundary before them (8,192 x 4,097 fp16 110 -> 74 and 65 us, but 65,536 x 191
// 29 -> 36 and 33, with 8-bit rows 36 -> 53 and 48: the values at a row's ends and
// the weights, which start elsewhere, cost narrow rows more than they gain).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

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

// How the threads of a row access it: single values, pairs of a 16-bit type (rows
// that start on 4 bytes, C even), or 16-byte vectors (rows that start on 16 bytes, C
// a multiple of the vector).
enum Mode { kSingle, kPair, kWide };

// The E channels of a row that thread `t` of TPR holds: access i of the thread at
// (i TPR + t), so that a warp's are adjacent.
template <typename T, int E, int TPR, Mode kMode>
struct Slice {
    static constexpr int kEach = E;
    static constexpr int V = kMode == kWide ? kVec<T> : kMode == kPair ? 2 : 1;
    static_assert(E % 8 == 0 && (kMode != kPair || sizeof(T) == 2), "whole chunks; pairs of a 16-bit type");

    __device__ static __forceinline__ int channel(int i, int t) { return ((i / V) * TPR + t) * V + i % V; }
};

// A thread's E channels as they are stored: packed pairs of a 16-bit type that is
// not read value by value (half the registers of fp32 values), fp32 otherwise. Used
// in chunks of 8. Channels past C are 0 and not written.
template <typename T, int E, Mode kMode>
struct Held {
    static constexpr bool kPacked = kMode != kSingle && sizeof(T) == 2;
    uint32_t w[kPacked ? E / 2 : 1];
    float f[kPacked ? 1 : E];

    __device__ __forceinline__ void get(int i, float (&v)[8]) const {
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
            if constexpr (kPacked) {
                const float2 two = unpack2(w[(i + j) / 2], T());
                v[j] = two.x;
                v[j + 1] = two.y;
            } else {
                v[j] = f[i + j];
                v[j + 1] = f[i + j + 1];
            }
        }
    }
    // 0 where all values are 0.
    __device__ __forceinline__ uint32_t magnitudes() const {
        uint32_t u = 0;
#pragma unroll
        for (int i = 0; i < (kPacked ? E / 2 : E); ++i) {
            if constexpr (kPacked) u |= w[i];
            else u |= __float_as_uint(f[i]);
        }
        return u & (kPacked ? 0x7fff7fffu : 0x7fffffffu);
    }
    // Values rounded to T.
    __device__ __forceinline__ void set(int i, const float (&v)[8]) {
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
            if constexpr (kPacked) {
                w[(i + j) / 2] = pack2(v[j], v[j + 1], T());
            } else {
                f[i + j] = to_f32<T>(from_f32<T>(v[j]));
                f[i + j + 1] = to_f32<T>(from_f32<T>(v[j + 1]));
            }
        }
    }
};

template <int TPR, typename T, int E, Mode kMode>
__device__ __forceinline__ void load_held(const T* row, int C, int t, Held<T, E, kMode>& h) {
    using S = Slice<T, E, TPR, kMode>;
#pragma unroll
    for (int i = 0; i < E; i += S::V) {
        const int c = S::channel(i, t);
        if constexpr (kMode == kSingle) {
            h.f[i] = c < C ? to_f32<T>(row[c]) : 0.0f;
        } else if constexpr (kMode == kPair) {
            h.w[i / 2] = c < C ? *reinterpret_cast<const uint32_t*>(row + c) : 0u;
        } else {
            const uint4 u = c < C ? *reinterpret_cast<const uint4*>(row + c) : make_uint4(0, 0, 0, 0);
            if constexpr (sizeof(T) == 2) {
                h.w[i / 2] = u.x;
                h.w[i / 2 + 1] = u.y;
                h.w[i / 2 + 2] = u.z;
                h.w[i / 2 + 3] = u.w;
            } else {
                unpack16<T>(u, &h.f[i]);
            }
        }
    }
}

template <int TPR, typename T, int E, Mode kMode>
__device__ __forceinline__ void store_held(T* row, int C, int t, const Held<T, E, kMode>& h) {
    using S = Slice<T, E, TPR, kMode>;
#pragma unroll
    for (int i = 0; i < E; i += S::V) {
        const int c = S::channel(i, t);
        if (c >= C) continue;
        if constexpr (kMode == kSingle) row[c] = from_f32<T>(h.f[i]);
        else if constexpr (kMode == kPair) *reinterpret_cast<uint32_t*>(row + c) = h.w[i / 2];
        else if constexpr (sizeof(T) == 2)
            *reinterpret_cast<uint4*>(row + c) = make_uint4(h.w[i / 2], h.w[i / 2 + 1], h.w[i / 2 + 2], h.w[i / 2 + 3]);
        else *reinterpret_cast<uint4*>(row + c) = pack16<T>(&h.f[i]);
    }
}

constexpr float kInf = __builtin_huge_valf();

// Largest of a and the magnitudes of b and c, keeping a NaN (fmaxf drops it), so
// that a row's largest magnitude tells whether all of the row is finite.
__device__ __forceinline__ float max_abs(float a, float b, float c) {
    float r;
    asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
__device__ __forceinline__ float max_abs(const float (&v)[8], float m) {
#pragma unroll
    for (int j = 0; j < 8; j += 2) m = max_abs(m, v[j], v[j + 1]);
    return m;
}

template <int TPR>
__device__ __forceinline__ float lanes_max(float m) {
    if constexpr (TPR >= 32) {
        float r;  // volatile: all 32 lanes execute it, wherever its result is used
        asm volatile("redux.sync.max.NaN.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(m));
        return r;
    } else {
#pragma unroll
        for (int o = TPR / 2; o > 0; o >>= 1) m = max_abs(m, m, __shfl_xor_sync(0xffffffffu, m, o));
        return m;
    }
}
// In 64 bits, on the bit patterns of magnitudes: infinity's and NaN's lie above
// every finite value's.
template <int TPR>
__device__ __forceinline__ unsigned long long lanes_max(unsigned long long m) {
#pragma unroll
    for (int o = (TPR < 32 ? TPR : 32) / 2; o > 0; o >>= 1) {
        const unsigned long long other = __shfl_xor_sync(0xffffffffu, m, o);
        m = other > m ? other : m;
    }
    return m;
}
template <int TPR, typename A>
__device__ __forceinline__ A lanes_sum(A a) {
#pragma unroll
    for (int o = (TPR < 32 ? TPR : 32) / 2; o > 0; o >>= 1) a += __shfl_xor_sync(0xffffffffu, a, o);
    return a;
}

// Sum of `a` (kSum) and maximum of `m` (kMax) over the TPR threads of a row;
// every thread gets both. The shared arrays hold TPR / 32 entries for TPR > 32;
// two uses need a barrier between them.
template <int TPR, bool kSum, bool kMax, typename A, typename M>
__device__ __forceinline__ void row_sum_max(A& a, M& m, A* shared_a, M* shared_m) {
    if constexpr (kSum) a = lanes_sum<TPR>(a);
    if constexpr (kMax) m = lanes_max<TPR>(m);
    if constexpr (TPR > 32) {
        constexpr int kWarps = TPR / 32;
        const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
        if (lane == 0) {
            if constexpr (kSum) shared_a[warp] = a;
            if constexpr (kMax) shared_m[warp] = m;
        }
        __syncthreads();
        // each lane one of the warps' values, some twice
        if constexpr (kSum) a = lanes_sum<kWarps>(shared_a[lane % kWarps]);
        if constexpr (kMax) m = lanes_max<kWarps>(shared_m[lane % kWarps]);
    }
}

// ---- rounding to 8 bits ----------------------------------------------------
// q = the whole number nearest to 127 v / m (m the row's largest magnitude),
// the even one at a tie, of the exact quotient. In fp32, t = v inv with
// inv = 127 / m is off by at most 127 (2^-23 + 2^-24 of inv, 2^-24 of a rounded
// v, 2^-24 of a rounded m) = 3.8e-5, so the nearest whole number of t is the
// answer unless t lies next to a half, past kBorder. There the sign of
// 254 v - c m with c / 2 that half decides, taken without rounding (one value in
// 10,000).
// Where v and m have at most 16 bits (kShort) there is no such case to look at,
// although exact halves are common then (about one quotient of bf16 values in
// 1,000, which cost SwiGLU's forward a quarter of its instructions): one step
// with the exact remainder makes t the rounded quotient itself, exact where that
// is a half, and no other quotient rounds to a half. For v = a u and m = b w, with
// a and b whole numbers below 2^16 and u and w powers of two, 254 v - c m is a
// multiple of the smaller of u and w, and the quotient's distance from c / 2 is
// that over 2 m: where w is the smaller, at least 1 / (2 b) > 2^-17 against a
// rounding of 2^-18 at most (quotients end at 127); where u is, at least
// t / (254 a) > 2^-23.99 t against a rounding of 2^-24 t.
constexpr float kMagic = 12582912.0f;  // 1.5 * 2^23: adding it rounds to a whole number
constexpr float kBorder = 0.49995f;
// Below 1e-30, 127 / m may overflow and products lose bits, and above 1e30
// 254 v may overflow: such a row is scaled by 2^80 or 2^-80 first, which changes
// no quotient (what falls below the smallest number is far below a half).
constexpr float kTiny = 1e-30f, kHuge = 1e30f;
constexpr float kScaleTiny = 0x1p80f, kScaleHuge = 0x1p-80f;

// 254 v - c m of fp32 values, c odd and below 256 in magnitude: each product is
// the sum of its rounding and an error of at most 8 bits; the two are within
// 2^-10 of each other, so their differences are exact and the sign is right.
__device__ __forceinline__ float half_side(float v, float m, float c) {
    const float p = __fmul_rn(254.0f, v), q = __fmul_rn(c, m);
    return __fadd_rn(__fsub_rn(p, q), __fsub_rn(__fmaf_rn(254.0f, v, -p), __fmaf_rn(c, m, -q)));
}
// The same in 64 bits, of products v and m of two fp32 values (48 bits each).
__device__ __forceinline__ double half_side(double v, double m, float c) {
    const double p = __dmul_rn(254.0, v), q = __dmul_rn((double)c, m);
    return __dadd_rn(__dsub_rn(p, q), __dsub_rn(__fma_rn(254.0, v, -p), __fma_rn((double)c, m, -q)));
}

// 127 v / m of such products to the nearest whole number, m finite and above 0.
__device__ __forceinline__ int nearest_whole(double v, double m) {
    const float below = (float)floor(127.0 * v / m);  // or, next to a whole number, the one beside it
    const double side = half_side(v, m, 2.0f * below + 1.0f);
    const int k = (int)below;
    return side > 0 || (side == 0 && (k & 1)) ? k + 1 : k;
}

__device__ __forceinline__ uint32_t pack_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}

// How a row of largest magnitude m is rounded.
template <typename M>
struct Rounding {
    M m;          // scaled
    float inv;    // 127 / m
    float reciprocal;  // 1 / m
    float scale;  // of the row's values, 1 unless `odd`
    bool odd;     // a tiny, huge, zero or not finite row
    bool zero;    // a row of zeros, or one that is not finite
    __device__ __forceinline__ explicit Rounding(M largest) : m(largest), scale(1.0f) {
        const float mf = (float)largest;
        odd = !(mf >= kTiny && mf <= kHuge);
        zero = !(mf > 0.0f && mf < kInf);
        if (odd) {
            scale = mf < kTiny ? kScaleTiny : kScaleHuge;
            m *= (M)scale;
        }
        reciprocal = zero ? 0.0f : f2s_rcp_approx((float)m);
        inv = 127.0f * reciprocal;
    }
};

// Two fp32 values in a register pair, and their fused multiply-add.
__device__ __forceinline__ uint64_t pair(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void unpair(uint64_t p, float& a, float& b) {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(p));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}

__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

// 8 values of a thread to 8 bits, in the low bytes of q; at(j): value j in m's
// type.
template <bool kShort, typename M, typename F>
__device__ __forceinline__ void round8(float (&v)[8], const Rounding<M>& r, uint32_t (&q)[8], F at) {
    if (r.odd) {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] *= r.scale;
    }
    if constexpr (kShort) {
        const uint64_t top = pair(127.0f, 127.0f), by = pair(r.reciprocal, r.reciprocal),
                       minus_m = pair(-(float)r.m, -(float)r.m), magic = pair(kMagic, kMagic);
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
            const uint64_t a = mul2(pair(v[j], v[j + 1]), top), t = mul2(a, by);
            float s0, s1;
            unpair(add2(fma2(fma2(t, minus_m, a), by, t), magic), s0, s1);
            q[j] = __float_as_uint(s0);
            q[j + 1] = __float_as_uint(s1);
        }
        if (r.zero) {
#pragma unroll
            for (int j = 0; j < 8; ++j) q[j] = 0u;
        }
        return;
    }
    float off = 0.0f;
    const uint64_t inv = pair(r.inv, r.inv), magic = pair(kMagic, kMagic), minus = pair(-1.0f, -1.0f);
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
        const uint64_t two = pair(v[j], v[j + 1]);
        const uint64_t shifted = fma2(two, inv, magic);
        float s0, s1, d0, d1;
        unpair(shifted, s0, s1);
        unpair(fma2(two, inv, fma2(shifted, minus, magic)), d0, d1);  // t minus its whole number
        asm("max.abs.f32 %0, %1, %2, %3;" : "=f"(off) : "f"(off), "f"(d0), "f"(d1));
        q[j] = __float_as_uint(s0);
        q[j + 1] = __float_as_uint(s1);
    }
    if (off > kBorder) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float whole = __fsub_rn(__uint_as_float(q[j]), kMagic);
            const float d = __fmaf_rn(v[j], r.inv, -whole);
            if (fabsf(d) > kBorder) {
                // the half between `below` and the next whole number
                const float below = d > 0.0f ? whole : whole - 1.0f;
                const auto side = half_side(at(j), r.m, 2.0f * below + 1.0f);
                const int k = (int)below;
                q[j] = (uint32_t)(side > 0 || (side == 0 && (k & 1)) ? k + 1 : k);
            }
        }
    }
    if (r.zero) {
#pragma unroll
        for (int j = 0; j < 8; ++j) q[j] = 0u;
    }
}

// Chunk i of a thread's channels, v, to 8 bits in `row` (of a start and pitch that
// keep pairs and vectors aligned). at(j): value j of the chunk in m's type, scaled.
template <bool kShort, typename S, Mode kMode, typename M, typename F>
__device__ __forceinline__ void store8_chunk(int8_t* row, int C, int t, int i, float (&v)[8], const Rounding<M>& r,
                                             F at) {
    uint32_t q[8];
    round8<kShort>(v, r, q, at);
    const int c = S::channel(i, t);
    if constexpr (kMode == kWide && S::V == 8) {
        if (c < C)
            *reinterpret_cast<uint2*>(row + c) =
                make_uint2(pack_bytes(q[0], q[1], q[2], q[3]), pack_bytes(q[4], q[5], q[6], q[7]));
    } else if constexpr (kMode == kWide) {
        const int c4 = S::channel(i + 4, t);
        if (c < C) *reinterpret_cast<uint32_t*>(row + c) = pack_bytes(q[0], q[1], q[2], q[3]);
        if (c4 < C) *reinterpret_cast<uint32_t*>(row + c4) = pack_bytes(q[4], q[5], q[6], q[7]);
    } else if constexpr (kMode == kPair) {
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
            const int c2 = S::channel(i + j, t);
            if (c2 < C) *reinterpret_cast<uint16_t*>(row + c2) = (uint16_t)__byte_perm(q[j], q[j + 1], 0x0040);
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (S::channel(i + j, t) < C) row[S::channel(i + j, t)] = (int8_t)(q[j] & 0xffu);
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

// Whether a row's sum of squares is outside of what fp32 holds well: rows of
// magnitudes above 1e18, or below 1e-14 with an eps that does not hide them. fp16 has no
// values of the first kind and its squares are never below 2^-48.
__device__ __forceinline__ bool squares_leave_fp32(float sum, float eps) {
    return sum > 0x1p120f || (sum < 0x1p-90f && eps < 0x1p-90f);
}

// Reciprocal root of a row's mean square from its sum.
__device__ __forceinline__ float reciprocal_rms(float sum, int C, float eps) {
    return __frsqrt_rn(sum / (float)C + eps);
}

// ---- dispatch --------------------------------------------------------------
// What a kernel's registers hold per channel decides how many channels (of
// `size` bytes) a thread of a TPR-thread row takes at most.
enum Kind {
    kForward,  // one or two packed rows
    kGrad      // s, dy, ds, w and dw; with TPR > 32 the next row's too
};
constexpr int most_channels(Kind kind, int size, int tpr) {
    return kind == kForward ? (size == 2 ? 32 : 16)
                            : tpr <= 32 ? (size == 2 ? 24 : 16) : (size == 2 ? 16 : 8);
}
constexpr int kThreads[] = {8, 32, 128, 256, 512, 1024};

// Single values of a 16-bit type are held in fp32.
constexpr int held_size(int size, Mode mode) { return mode == kSingle ? 4 : size; }

// (TPR, E) for a row of C channels: the fewest threads that hold it, since each
// thread's share of the reduction and of the row's constants costs as much as
// ten channels, and then the fewest registers. Rows past 512 x most_channels
// take up to 32 channels of 512 or 1,024 threads, and spill a little. With few
// rows (fewer threads in all than the SMs hold at one 512-thread block each)
// more threads per row with 8 channels each shorten the one row's latency.
struct Shape {
    int tpr, e;
};

inline Shape pick_shape(Kind kind, int size, int64_t nrows, int C, Mode mode) {
    size = held_size(size, mode);
    const bool single = mode == kSingle;
    int i = 0;
    while (i < 4 && kThreads[i] * most_channels(kind, size, kThreads[i]) < C) ++i;
    while (i < 4 && C > kThreads[i] * 8 && nrows * kThreads[i] < (int64_t)sm_count() * 512) ++i;
    // single values: 8, 16 or 32; the backward's on 1,024 threads before they spill
    // (8,192 x 4,097: 210 us against 466; the forward 157 against 110)
    if (kThreads[i] * 32 < C || (single && kind == kGrad && i == 4 && C > 512 * 8)) i = 5;
    const int e = ceil_div(ceil_div(C, kThreads[i]), 8) * 8;
    const bool all = i == 5 && (!single || kind == kForward);
    return {kThreads[i], all || (single && e > 16) ? 32 : e};
}

// Blocks of `threads` per SM that E channels held in `size` bytes each leave
// registers for: the second launch bound.
constexpr int resident(int threads, int E, int size) {
    return ((E * size <= 32 ? 1536 : 1024) / threads) > 0 ? (E * size <= 32 ? 1536 : 1024) / threads : 1;
}

// Rows per block and threads per block of a shape.
constexpr int block_threads(int tpr) { return tpr <= 32 ? 256 : tpr; }
constexpr int block_rows(int tpr) { return tpr <= 32 ? 256 / tpr : 1; }

template <int kValue>
using Const = std::integral_constant<int, kValue>;

template <Mode kValue>
using ConstMode = std::integral_constant<Mode, kValue>;

template <Kind kKind, int kSize, Mode kMode, int kTpr, typename F>
void dispatch_channels(const Shape& s, F f) {
    constexpr bool single = kMode == kSingle;
    // 512 and 1,024 threads take what is left, but for the backward's single values
    constexpr int most = kTpr == 1024 || (kTpr == 512 && !(single && kKind == kGrad))
                             ? 32
                             : most_channels(kKind, held_size(kSize, kMode), kTpr);
    if constexpr (kTpr < 1024 || (single && kKind == kGrad)) {
        if (s.e == 8) f(Const<8>(), Const<kTpr>(), ConstMode<kMode>());
        if constexpr (most >= 16)
            if (s.e == 16) f(Const<16>(), Const<kTpr>(), ConstMode<kMode>());
        if constexpr (most >= 24 && !single)
            if (s.e == 24) f(Const<24>(), Const<kTpr>(), ConstMode<kMode>());
    }
    if constexpr (most >= 32)
        if (s.e == 32) f(Const<32>(), Const<kTpr>(), ConstMode<kMode>());
}

template <Kind kKind, int kSize, Mode kMode, typename F>
void dispatch_threads(const Shape& s, F f) {
    switch (s.tpr) {
        case 8: dispatch_channels<kKind, kSize, kMode, 8>(s, f); break;
        case 32: dispatch_channels<kKind, kSize, kMode, 32>(s, f); break;
        case 128: dispatch_channels<kKind, kSize, kMode, 128>(s, f); break;
        case 256: dispatch_channels<kKind, kSize, kMode, 256>(s, f); break;
        case 512: dispatch_channels<kKind, kSize, kMode, 512>(s, f); break;
        default: dispatch_channels<kKind, kSize, kMode, 1024>(s, f); break;
    }
}

// f(E, TPR, mode) for the shape, as integral constants: T's type decides whether
// there are pairs, `kSize` (its own, or what a kernel holds) the registers.
template <Kind kKind, typename T, int kSize = sizeof(T), typename F>
void dispatch(const Shape& s, Mode mode, F f) {
    if (mode == kWide) dispatch_threads<kKind, kSize, kWide>(s, f);
    else if (mode == kSingle) dispatch_threads<kKind, kSize, kSingle>(s, f);
    if constexpr (sizeof(T) == 2)
        if (mode == kPair) dispatch_threads<kKind, kSize, kPair>(s, f);
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// The widest mode that all of a kernel's rows allow.
struct Layout {
    int64_t nrows;
    int vec;
    bool wide, pairs;
    Layout(int64_t n, int C, int size)
        : nrows(n), vec(16 / size), wide(C % (16 / size) == 0), pairs(size == 2 && C % 2 == 0) {}
    Layout& vector(const void* p) {
        wide = wide && aligned16(p);
        pairs = pairs && (reinterpret_cast<uintptr_t>(p) & 3) == 0;
        return *this;
    }
    Layout& rows(const void* p, int64_t pitch) {  // null: none
        if (!p) return *this;
        wide = wide && (pitch % vec == 0 || nrows == 1);
        pairs = pairs && (pitch % 2 == 0 || nrows == 1);
        return vector(p);
    }
    Layout& eight(const void* p, int64_t pitch) {
        wide = wide && aligned16(p) && (pitch % vec == 0 || nrows == 1);
        pairs = pairs && (reinterpret_cast<uintptr_t>(p) & 1) == 0 && (pitch % 2 == 0 || nrows == 1);
        return *this;
    }
    Mode mode() const { return wide ? kWide : pairs ? kPair : kSingle; }
};

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

inline int check_norm(const char* what, int dtype, int64_t nrows, int C, float eps) {
    F2S_TRY(check_dtype(what, dtype));
    F2S_REQUIRE(nrows >= 0 && C >= 1 && eps >= 0.0f, "%s: bad shape rows=%lld C=%d eps=%g", what,
                (long long)nrows, C, (double)eps);
    F2S_LIMIT(C <= kMaxRow, "%s: C=%d, at most %d channels", what, C, kMaxRow);
    return F2S_OK;
}

inline int dtype_size(int dtype) { return dtype == F2S_DTYPE_F32 ? 4 : 2; }

}  // namespace rows
}  // namespace f2s
