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
constexpr int kLanes = 8;               // threads of one group
constexpr int kEach = kGroup / kLanes;  // channels per thread: 16
static_assert(kEach == 16, "one 16-byte store of checkpoints per thread");

// Approximate reciprocal and exponential, 2^-22 relative each, and the argument
// -1.4427 g rounded before the exponential, whose error grows with |g| where sigma is
// small: below the rounding of 16-bit results. Of fp32 ones 6e-7 relative for gates
// above -3, 2e-6 at -30 and 4e-6 below -50. Below gates of -87.3 sigma, under 2^-126,
// is 0.
__device__ __forceinline__ float sigmoid(float g) {
    return f2s_rcp_approx(1.0f + f2s_ex2_approx(-1.44269504088896341f * g));
}

// v g sigma(g), in one order of products wherever it is computed.
__device__ __forceinline__ float gated(float g, float v) { return __fmul_rn(__fmul_rn(g, sigmoid(g)), v); }

// How a thread's 16 channels of a group lie: two runs of 8, 64 apart, where H is
// a multiple of 8 (with 16-byte accesses where the pointers allow it), else
// single ones, 8 apart, so that a warp's accesses are adjacent. H alone decides
// the order, which is also the order of the checkpoint's bytes, in the forward
// and the backward.
enum Form { kWideRun, kRun, kApart };

template <Form kForm>
__device__ __forceinline__ int channel_of(int j, int lane) {
    return kForm == kApart ? j * kLanes + lane : (j / 8) * 64 + lane * 8 + j % 8;
}

// Channels of a group that begins at `row`; those past `left` (a multiple of 8
// unless kApart) are outside the row.
template <typename T, Form kForm>
__device__ __forceinline__ void load_group(const T* row, int lane, int left, float (&v)[kEach]) {
    if constexpr (kForm == kWideRun) {
#pragma unroll
        for (int j = 0; j < kEach; j += kVec<T>) {
            const int c = channel_of<kForm>(j, lane);
            const uint4 u = c < left ? *reinterpret_cast<const uint4*>(row + c) : make_uint4(0, 0, 0, 0);
            unpack16<T>(u, &v[j]);
        }
    } else {
#pragma unroll
        for (int j = 0; j < kEach; ++j) {
            const int c = channel_of<kForm>(j, lane);
            v[j] = c < left ? to_f32<T>(row[c]) : 0.0f;
        }
    }
}

template <typename T, Form kForm>
__device__ __forceinline__ void store_group(T* row, int lane, int left, const float (&v)[kEach]) {
    if constexpr (kForm == kWideRun) {
#pragma unroll
        for (int j = 0; j < kEach; j += kVec<T>) {
            const int c = channel_of<kForm>(j, lane);
            if (c < left) *reinterpret_cast<uint4*>(row + c) = pack16<T>(&v[j]);
        }
    } else {
#pragma unroll
        for (int j = 0; j < kEach; ++j) {
            const int c = channel_of<kForm>(j, lane);
            if (c < left) row[c] = from_f32<T>(v[j]);
        }
    }
}

// One group's checkpoint: thread `lane` keeps its 16 channels, in its own
// order, as 16 consecutive bytes.
template <bool kShort>
__device__ __forceinline__ void keep_group(const float (&v)[kEach], int lane, int8_t* q8, float* scale) {
    float m = 0.0f;
#pragma unroll
    for (int j = 0; j < kEach; j += 2) m = max_abs(m, v[j], v[j + 1]);
    m = lanes_max<kLanes>(m);
    const Rounding<float> rounding(m);
    uint32_t w[kEach / 4];
#pragma unroll
    for (int i = 0; i < kEach; i += 8) {
        float held[8];
        uint32_t q[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) held[j] = v[i + j];
        round8<kShort>(held, rounding, q, [&](int j) { return held[j]; });
        w[i / 4] = pack_bytes(q[0], q[1], q[2], q[3]);
        w[i / 4 + 1] = pack_bytes(q[4], q[5], q[6], q[7]);
    }
    if (q8) {
        *reinterpret_cast<uint4*>(q8 + lane * kEach) = make_uint4(w[0], w[1], w[2], w[3]);
        if (lane == 0) *scale = m < kInf ? m / 127.0f : __int_as_float(0x7fc00000);
    }
}

// Units of 8 threads, one per (row, group of 128 channels). `kept` of unit u
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
    for (int j = 0; j < kEach; ++j) h[j] = gated(g[j], v[j]);
    store_group<T, kForm>(y + row * (int64_t)H + first, lane, left, h);
    if constexpr (kKeep) {
        // the shuffles need every lane of the warp, live or not
        keep_group<sizeof(T) == 2>(g, lane, live ? kept + u * (2 * kGroup) : nullptr, scales + 2 * u);
        keep_group<sizeof(T) == 2>(v, lane, live ? kept + u * (2 * kGroup) + kGroup : nullptr, scales + 2 * u + 1);
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
        const uint4 qg = *reinterpret_cast<const uint4*>(from);
        const uint4 qv = *reinterpret_cast<const uint4*>(from + kGroup);
        const float2 s = *reinterpret_cast<const float2*>(scales + 2 * u);
        widen8(qg.x, g);
        widen8(qg.y, g + 4);
        widen8(qg.z, g + 8);
        widen8(qg.w, g + 12);
        widen8(qv.x, v);
        widen8(qv.y, v + 4);
        widen8(qv.z, v + 8);
        widen8(qv.w, v + 12);
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
template <typename T, int E, int TPR, Mode kMode>
__global__ void __launch_bounds__(block_threads(TPR), resident(block_threads(TPR), E, 2 * sizeof(T)))
swiglu_int8_kernel(const T* __restrict__ projected, int64_t ld, int64_t nrows, int H, int8_t* __restrict__ q8,
                   int64_t ldq, float* __restrict__ scale) {
    using S = Slice<T, E, TPR, kMode>;
    __shared__ float shared_m[32];
    const int t = TPR <= 32 ? threadIdx.x % TPR : threadIdx.x;
    const int64_t row = TPR <= 32 ? (int64_t)blockIdx.x * (256 / TPR) + threadIdx.x / TPR : (int64_t)blockIdx.x;
    const bool live = row < nrows;
    const int64_t at = live ? row : 0;
    const int C = live ? H : 0;
    const T* from = projected + at * ld;
    Held<T, E, kMode> gate, value;
    load_held<TPR>(from, C, t, gate);
    load_held<TPR>(from + H, C, t, value);
    float h[E];
    float m = 0.0f, none = 0.0f;
#pragma unroll
    for (int i = 0; i < E; i += 8) {
        float g[8], v[8];
        gate.get(i, g);
        value.get(i, v);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            h[i + j] = gated(g[j], v[j]);
            v[j] = h[i + j];
        }
        m = max_abs(v, m);
    }
    row_sum_max<TPR, false, true>(none, m, shared_m, shared_m);
    const Rounding<float> rounding(m);
#pragma unroll
    for (int i = 0; i < E; i += 8) {
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = h[i + j];
        store8_chunk<false, S, kMode>(q8 + at * ldq, C, t, i, v, rounding, [&](int j) { return v[j]; });
    }
    if (live && t == 0) scale[row] = m < kInf ? m / 127.0f : __int_as_float(0x7fc00000);
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
    const bool wide = H % 8 == 0 && aligned16(projected) && aligned16(y) && (ld % kVec<T> == 0 || nrows == 1);
    TraceScope trace(kTagSwiGlu, st);
    auto go = [&](auto kernel) {
        kernel<<<u.blocks, 256, 0, st>>>(static_cast<const T*>(projected), ld, H, u.groups, u.units,
                                         static_cast<T*>(y), kept, scales);
    };
    if (wide) kept ? go(swiglu_kernel<T, kWideRun, true>) : go(swiglu_kernel<T, kWideRun, false>);
    else if (H % 8 == 0) kept ? go(swiglu_kernel<T, kRun, true>) : go(swiglu_kernel<T, kRun, false>);
    else kept ? go(swiglu_kernel<T, kApart, true>) : go(swiglu_kernel<T, kApart, false>);
    return check_launch("swiglu_kernel");
}

template <typename T>
int swiglu_grad_launch(const void* projected, int64_t ld, const int8_t* kept, const float* scales, const void* dy,
                       int64_t lddy, int64_t nrows, int H, void* dprojected, cudaStream_t st) {
    Units u;
    F2S_TRY(units_of("swiglu_backward", nrows, H, u));
    const bool wide = H % 8 == 0 && aligned16(dy) && aligned16(dprojected) && (lddy % kVec<T> == 0 || nrows == 1) &&
                      (kept || (aligned16(projected) && (ld % kVec<T> == 0 || nrows == 1)));
    TraceScope trace(kTagSwiGlu, st);
    auto go = [&](auto kernel) {
        kernel<<<u.blocks, 256, 0, st>>>(static_cast<const T*>(projected), ld, kept, scales, static_cast<const T*>(dy),
                                         lddy, H, u.groups, u.units, static_cast<T*>(dprojected));
    };
    if (wide) kept ? go(swiglu_grad_kernel<T, kWideRun, true>) : go(swiglu_grad_kernel<T, kWideRun, false>);
    else if (H % 8 == 0) kept ? go(swiglu_grad_kernel<T, kRun, true>) : go(swiglu_grad_kernel<T, kRun, false>);
    else kept ? go(swiglu_grad_kernel<T, kApart, true>) : go(swiglu_grad_kernel<T, kApart, false>);
    return check_launch("swiglu_grad_kernel");
}

template <typename T>
int swiglu_int8_launch(const void* projected, int64_t ld, int64_t nrows, int H, int8_t* q, int64_t ldq, float* scale,
                       cudaStream_t st) {
    const Mode mode = Layout(nrows, H, sizeof(T)).rows(projected, ld).eight(q, ldq).mode();
    const Shape s = pick_shape(kForward, 4, nrows, H, mode);  // h is held in fp32
    const int64_t blocks = ceil_div64(nrows, block_rows(s.tpr));
    F2S_LIMIT(blocks <= INT32_MAX, "swiglu_int8: %lld rows", (long long)nrows);
    TraceScope trace(kTagSwiGlu, st);
    dispatch<kForward, T, 4>(s, mode, [&](auto e, auto tpr, auto m) {
        swiglu_int8_kernel<T, e.value, tpr.value, m.value><<<(unsigned)blocks, block_threads(tpr.value), 0, st>>>(
            static_cast<const T*>(projected), ld, nrows, H, q, ldq, scale);
    });
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
    F2S_REQUIRE((reinterpret_cast<uintptr_t>(checkpoint) & 15) == 0 && (reinterpret_cast<uintptr_t>(checkpoint_scale) & 7) == 0,
                "swiglu: checkpoints start on 16 bytes");
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
    F2S_REQUIRE((reinterpret_cast<uintptr_t>(checkpoint) & 15) == 0 && (reinterpret_cast<uintptr_t>(checkpoint_scale) & 7) == 0,
                "swiglu_backward: checkpoints start on 16 bytes");
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
