// The gated activation of a feed-forward layer, h = v g sigma(g) of rows
// [g | v] of 2 H channels:
//   training  the forward can keep g and v as 8-bit checkpoints (groups of
//             128 channels of g, and of v, share a scale), 52% of the bytes
//             of a 16-bit type, and the backward reads those:
//             dv = dy g sigma(g), dg = dy v sigma(g) (1 + g (1 - sigma(g)));
//   serving   h as 8-bit rows with one scale each, for the 8-bit product.
//
// Bound by memory. The forward with checkpoints reads 4 bytes per h channel of
// a 16-bit type and writes 4.06, the backward reads 4.06 and writes 4; the
// special-function unit (an exponential and a reciprocal per channel) stays at
// a third of its rate.
#include "kernels.cuh"
#include "row_ops.cuh"

namespace f2s {
namespace {

using namespace rows;

constexpr int kGroup = F2S_SWIGLU_GROUP;
constexpr int kLanes = 16;                // threads of one group
constexpr int kEach = kGroup / kLanes;    // channels per thread: 8
static_assert(kEach == 8, "one 8-byte store of checkpoints per thread");

// Approximate reciprocal and exponential, 2^-22 relative each: below the
// rounding of 16-bit results, and 4e-7 relative of fp32 ones.
__device__ __forceinline__ float sigmoid(float g) {
    return f2s_rcp_approx(1.0f + f2s_ex2_approx(-1.44269504088896341f * g));
}

// How a thread's 8 channels of a group lie: consecutive where H is a multiple
// of 8 (with 16-byte accesses where the pointers allow it), else 16 apart, so
// that a warp's single accesses are adjacent. H alone decides the order, which
// is also the order of the checkpoint's bytes, in the forward and the backward.
enum Form { kWideRun, kRun, kApart };

// Channels of a group that begins at `row`; those past `left` (a multiple of 8
// unless kApart) are outside the row.
template <typename T, Form kForm>
__device__ __forceinline__ void load_group(const T* row, int lane, int left, float (&v)[kEach]) {
    if constexpr (kForm == kWideRun) {
        const bool in = lane * kEach < left;
#pragma unroll
        for (int j = 0; j < kEach; j += kVec<T>) {
            const uint4 u = in ? *reinterpret_cast<const uint4*>(row + lane * kEach + j) : make_uint4(0, 0, 0, 0);
            unpack16<T>(u, &v[j]);
        }
    } else {
#pragma unroll
        for (int j = 0; j < kEach; ++j) {
            const int c = kForm == kRun ? lane * kEach + j : j * kLanes + lane;
            v[j] = c < left ? to_f32<T>(row[c]) : 0.0f;
        }
    }
}

template <typename T, Form kForm>
__device__ __forceinline__ void store_group(T* row, int lane, int left, const float (&v)[kEach]) {
    if constexpr (kForm == kWideRun) {
        if (lane * kEach >= left) return;
#pragma unroll
        for (int j = 0; j < kEach; j += kVec<T>)
            *reinterpret_cast<uint4*>(row + lane * kEach + j) = pack16<T>(&v[j]);
    } else {
#pragma unroll
        for (int j = 0; j < kEach; ++j) {
            const int c = kForm == kRun ? lane * kEach + j : j * kLanes + lane;
            if (c < left) row[c] = from_f32<T>(v[j]);
        }
    }
}

// One group's checkpoint: thread `lane` keeps its 8 channels, in its own
// order, as 8 consecutive bytes.
__device__ __forceinline__ void keep_group(const float (&v)[kEach], int lane, int8_t* q8, float* scale) {
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < kEach; ++j) m = max(m, abs_bits(v[j]));
#pragma unroll
    for (int o = kLanes / 2; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
    const float largest = __uint_as_float(m);
    const bool finite = m < kInfBits;
    uint32_t q[kEach];
    round8_row(v, 127.0f / largest, finite ? (double)largest : 0.0, finite && largest >= kTiny, q,
               [&](int i) { return (double)v[i]; });
    uint32_t w[2];
#pragma unroll
    for (int j = 0; j < 2; ++j)
        w[j] = __byte_perm(__byte_perm(q[4 * j], q[4 * j + 1], 0x0040),
                           __byte_perm(q[4 * j + 2], q[4 * j + 3], 0x0040), 0x5410);
    if (q8) {
        *reinterpret_cast<uint2*>(q8 + lane * kEach) = make_uint2(w[0], w[1]);
        if (lane == 0) *scale = finite ? largest / 127.0f : __int_as_float(0x7fc00000);
    }
}

// Units of 16 threads, one per (row, group of 128 channels). `kept` of unit u
// is at byte 256 u (gate, then value), its scales at 2 u.
template <typename T, Form kForm, bool kKeep>
__global__ void __launch_bounds__(256)
swiglu_kernel(const T* __restrict__ projected, int64_t ld, int H, int groups, int64_t units, T* __restrict__ y,
              int8_t* __restrict__ kept, float* __restrict__ scales) {
    const int lane = threadIdx.x % kLanes;
    const int64_t unit = (int64_t)blockIdx.x * (256 / kLanes) + threadIdx.x / kLanes;
    const bool live = unit < units;
    const int64_t u = live ? unit : 0;
    const int64_t row = units <= INT32_MAX ? (int64_t)((uint32_t)u / (uint32_t)groups) : u / groups;
    const int first = (int)(u - row * groups) * kGroup;
    const int left = live ? H - first : 0;
    const T* from = projected + row * ld + first;
    float g[kEach], v[kEach], h[kEach];
    load_group<T, kForm>(from, lane, left, g);
    load_group<T, kForm>(from + H, lane, left, v);
#pragma unroll
    for (int j = 0; j < kEach; ++j) h[j] = g[j] * sigmoid(g[j]) * v[j];
    store_group<T, kForm>(y + row * (int64_t)H + first, lane, left, h);
    if constexpr (kKeep) {
        // the shuffles need every lane of the warp, live or not
        keep_group(g, lane, live ? kept + u * (2 * kGroup) : nullptr, scales + 2 * u);
        keep_group(v, lane, live ? kept + u * (2 * kGroup) + kGroup : nullptr, scales + 2 * u + 1);
    }
}

// From the checkpoints (`kept` not null) or the projection itself.
template <typename T, Form kForm, bool kKept>
__global__ void __launch_bounds__(256)
swiglu_grad_kernel(const T* __restrict__ projected, int64_t ld, const int8_t* __restrict__ kept,
                   const float* __restrict__ scales, const T* __restrict__ dy, int64_t lddy, int H, int groups,
                   int64_t units, T* __restrict__ dprojected) {
    const int lane = threadIdx.x % kLanes;
    const int64_t u = (int64_t)blockIdx.x * (256 / kLanes) + threadIdx.x / kLanes;
    if (u >= units) return;
    const int64_t row = units <= INT32_MAX ? (int64_t)((uint32_t)u / (uint32_t)groups) : u / groups;
    const int first = (int)(u - row * groups) * kGroup;
    const int left = H - first;
    float g[kEach], v[kEach], d[kEach];
    load_group<T, kForm>(dy + row * lddy + first, lane, left, d);
    if constexpr (kKept) {
        const int8_t* from = kept + u * (2 * kGroup) + lane * kEach;
        const uint2 qg = *reinterpret_cast<const uint2*>(from);
        const uint2 qv = *reinterpret_cast<const uint2*>(from + kGroup);
        const float2 s = *reinterpret_cast<const float2*>(scales + 2 * u);
        widen8(qg.x, g);
        widen8(qg.y, g + 4);
        widen8(qv.x, v);
        widen8(qv.y, v + 4);
#pragma unroll
        for (int j = 0; j < kEach; ++j) {
            g[j] *= s.x;
            v[j] *= s.y;
        }
    } else {
        const T* from = projected + row * ld + first;
        load_group<T, kForm>(from, lane, left, g);
        load_group<T, kForm>(from + H, lane, left, v);
    }
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
        const float sg = sigmoid(g[j]);
        const float ds = d[j] * sg;
        d[j] = ds * v[j] * fmaf(g[j], 1.0f - sg, 1.0f);  // dg
        v[j] = ds * g[j];                                // dv
    }
    T* to = dprojected + row * (2 * (int64_t)H) + first;
    store_group<T, kForm>(to, lane, left, d);
    store_group<T, kForm>(to + H, lane, left, v);
}

// h as 8-bit rows.
template <typename T, int E, int TPR, bool kWide>
__global__ void __launch_bounds__(TPR <= 32 ? 256 : TPR)
swiglu_int8_kernel(const T* __restrict__ projected, int64_t ld, int64_t nrows, int H, int8_t* __restrict__ q8,
                   int64_t ldq, float* __restrict__ scale) {
    using S = Slice<T, E, TPR, kWide>;
    __shared__ uint32_t shared_m[32];
    __shared__ float shared_a[32];
    const int t = TPR <= 32 ? threadIdx.x % TPR : threadIdx.x;
    const int64_t row = TPR <= 32 ? (int64_t)blockIdx.x * (256 / TPR) + threadIdx.x / TPR : (int64_t)blockIdx.x;
    const bool live = row < nrows;
    const int64_t at = live ? row : 0;
    const int C = live ? H : 0;
    float h[E], v[E];
    S::load(projected + at * ld, C, t, h);
    S::load(projected + at * ld + H, C, t, v);
    uint32_t m = 0;
    float unused = 0.0f;
#pragma unroll
    for (int i = 0; i < E; ++i) {
        h[i] = h[i] * sigmoid(h[i]) * v[i];
        m = max(m, abs_bits(h[i]));
    }
    row_sum_max<TPR>(unused, m, shared_m, shared_a);
    const float largest = __uint_as_float(m);
    const bool finite = m < kInfBits;
    uint32_t q[E];
    round8_row(h, 127.0f / largest, finite ? (double)largest : 0.0, finite && largest >= kTiny, q,
               [&](int i) { return (double)h[i]; });
    S::store8(q8 + at * ldq, C, t, q);
    if (live && t == 0) scale[row] = finite ? largest / 127.0f : __int_as_float(0x7fc00000);
}

int check_swiglu(const char* what, int dtype, int64_t nrows, int H) {
    F2S_TRY(check_dtype(what, dtype));
    F2S_REQUIRE(nrows >= 0 && H >= 1, "%s: bad shape rows=%lld H=%d", what, (long long)nrows, H);
    F2S_LIMIT(H <= (1 << 29), "%s: H=%d", what, H);
    return F2S_OK;
}

struct Units {
    int groups;
    int64_t units;
    unsigned blocks;
};

int units_of(const char* what, int64_t nrows, int H, Units& u) {
    u.groups = ceil_div(H, kGroup);
    u.units = nrows * u.groups;
    const int64_t blocks = ceil_div64(u.units, 256 / kLanes);
    F2S_LIMIT(blocks <= INT32_MAX, "%s: %lld rows of %d", what, (long long)nrows, H);
    u.blocks = (unsigned)blocks;
    return F2S_OK;
}

template <typename T>
int swiglu_launch(const void* projected, int64_t ld, int64_t nrows, int H, void* y, int8_t* kept, float* scales,
                  cudaStream_t st) {
    Units u;
    F2S_TRY(units_of("swiglu", nrows, H, u));
    const bool wide = H % kEach == 0 && aligned16(projected) && aligned16(y) && (ld % kVec<T> == 0 || nrows == 1);
    TraceScope trace(kTagSwiGlu, st);
    auto go = [&](auto kernel) {
        kernel<<<u.blocks, 256, 0, st>>>(static_cast<const T*>(projected), ld, H, u.groups, u.units,
                                         static_cast<T*>(y), kept, scales);
    };
    if (wide) kept ? go(swiglu_kernel<T, kWideRun, true>) : go(swiglu_kernel<T, kWideRun, false>);
    else if (H % kEach == 0) kept ? go(swiglu_kernel<T, kRun, true>) : go(swiglu_kernel<T, kRun, false>);
    else kept ? go(swiglu_kernel<T, kApart, true>) : go(swiglu_kernel<T, kApart, false>);
    return check_launch("swiglu_kernel");
}

template <typename T>
int swiglu_grad_launch(const void* projected, int64_t ld, const int8_t* kept, const float* scales, const void* dy,
                       int64_t lddy, int64_t nrows, int H, void* dprojected, cudaStream_t st) {
    Units u;
    F2S_TRY(units_of("swiglu_backward", nrows, H, u));
    const bool wide = H % kEach == 0 && aligned16(dy) && aligned16(dprojected) && (lddy % kVec<T> == 0 || nrows == 1) &&
                      (kept || (aligned16(projected) && (ld % kVec<T> == 0 || nrows == 1)));
    TraceScope trace(kTagSwiGlu, st);
    auto go = [&](auto kernel) {
        kernel<<<u.blocks, 256, 0, st>>>(static_cast<const T*>(projected), ld, kept, scales, static_cast<const T*>(dy),
                                         lddy, H, u.groups, u.units, static_cast<T*>(dprojected));
    };
    if (wide) kept ? go(swiglu_grad_kernel<T, kWideRun, true>) : go(swiglu_grad_kernel<T, kWideRun, false>);
    else if (H % kEach == 0) kept ? go(swiglu_grad_kernel<T, kRun, true>) : go(swiglu_grad_kernel<T, kRun, false>);
    else kept ? go(swiglu_grad_kernel<T, kApart, true>) : go(swiglu_grad_kernel<T, kApart, false>);
    return check_launch("swiglu_grad_kernel");
}

template <typename T>
int swiglu_int8_launch(const void* projected, int64_t ld, int64_t nrows, int H, int8_t* q, int64_t ldq, float* scale,
                       cudaStream_t st) {
    constexpr int vec = kVec<T>;
    const bool wide = H % vec == 0 && aligned16(projected) && aligned16(q) &&
                      ((ld % vec == 0 && ldq % vec == 0) || nrows == 1);
    const Shape s = pick_shape(nrows, H, wide);
    const int64_t blocks = ceil_div64(nrows, block_rows(s.tpr));
    F2S_LIMIT(blocks <= INT32_MAX, "swiglu_int8: %lld rows", (long long)nrows);
    TraceScope trace(kTagSwiGlu, st);
    const T* from = static_cast<const T*>(projected);
#define F2S_LAUNCH(T, E, TPR, W) \
    swiglu_int8_kernel<T, E, TPR, W><<<(unsigned)blocks, block_threads(TPR), 0, st>>>(from, ld, nrows, H, q, ldq, scale)
    F2S_ROW_DISPATCH(s, wide, T, F2S_LAUNCH);
#undef F2S_LAUNCH
    return check_launch("swiglu_int8_kernel");
}

}  // namespace
}  // namespace f2s

extern "C" int f2s_swiglu(const void* projected, int64_t ld, int dtype, int64_t rows, int H, void* y,
                          int8_t* checkpoint, float* checkpoint_scale, void* stream) {
    F2S_TRY(f2s::check_swiglu("swiglu", dtype, rows, H));
    if (rows == 0) return F2S_OK;
    F2S_REQUIRE(projected && y && (!checkpoint) == (!checkpoint_scale), "swiglu: null pointer");
    F2S_REQUIRE(ld >= 2 * (int64_t)H, "swiglu: row pitch below 2 H = %lld", 2 * (long long)H);
    F2S_REQUIRE((reinterpret_cast<uintptr_t>(checkpoint) & 7) == 0 && (reinterpret_cast<uintptr_t>(checkpoint_scale) & 7) == 0,
                "swiglu: checkpoints start on 8 bytes");
    int status = F2S_OK;
    F2S_DTYPE_SWITCH(dtype, status = f2s::swiglu_launch<T>(projected, ld, rows, H, y, checkpoint, checkpoint_scale,
                                                           f2s::as_stream(stream)));
    return status;
}

extern "C" int f2s_swiglu_backward(const void* projected, int64_t ld, const int8_t* checkpoint,
                                   const float* checkpoint_scale, const void* dy, int64_t lddy, int dtype,
                                   int64_t rows, int H, void* dprojected, void* stream) {
    F2S_TRY(f2s::check_swiglu("swiglu_backward", dtype, rows, H));
    if (rows == 0) return F2S_OK;
    F2S_REQUIRE(dy && dprojected && (projected || checkpoint) && (!checkpoint) == (!checkpoint_scale),
                "swiglu_backward: null pointer");
    F2S_REQUIRE(lddy >= H && (checkpoint || ld >= 2 * (int64_t)H), "swiglu_backward: row pitch below the row");
    F2S_REQUIRE((reinterpret_cast<uintptr_t>(checkpoint) & 7) == 0 && (reinterpret_cast<uintptr_t>(checkpoint_scale) & 7) == 0,
                "swiglu_backward: checkpoints start on 8 bytes");
    int status = F2S_OK;
    F2S_DTYPE_SWITCH(dtype, status = f2s::swiglu_grad_launch<T>(projected, ld, checkpoint, checkpoint_scale, dy, lddy,
                                                                rows, H, dprojected, f2s::as_stream(stream)));
    return status;
}

extern "C" int f2s_swiglu_int8(const void* projected, int64_t ld, int dtype, int64_t rows, int H, int8_t* q,
                               int64_t ldq, float* scale, void* stream) {
    F2S_TRY(f2s::check_swiglu("swiglu_int8", dtype, rows, H));
    F2S_LIMIT(H <= f2s::rows::kMaxRow, "swiglu_int8: H=%d, at most %d channels", H, f2s::rows::kMaxRow);
    if (rows == 0) return F2S_OK;
    F2S_REQUIRE(projected && q && scale, "swiglu_int8: null pointer");
    F2S_REQUIRE(ld >= 2 * (int64_t)H && ldq >= H, "swiglu_int8: row pitch below the row");
    int status = F2S_OK;
    F2S_DTYPE_SWITCH(dtype, status = f2s::swiglu_int8_launch<T>(projected, ld, rows, H, q, ldq, scale,
                                                                f2s::as_stream(stream)));
    return status;
}
