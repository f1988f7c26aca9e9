// Backward of the root-mean-square norm of a residual stream (rms_norm.cu).
// With u = dy w and n = s rstd:
//   dx = ds + rstd (u - n mean(u n)),   dw = sum over rows of dy n.
// Blocks walk the rows by the grid and keep their part of dw in registers
// (32-bit sums in a fixed order: per thread over its rows, over the block's
// row groups, then over the blocks by weight_grad_kernel), so it costs one
// (blocks x C) array instead of another pass over dy and s.
//
// Bound by memory: it reads s, dy, ds and writes dx, 8 bytes per channel in 16 bits.
#include "kernels.cuh"
#include "row_ops.cuh"

namespace f2s {
namespace {

using namespace rows;

struct NormGradArgs {
    const void* s;
    int64_t lds;
    const void* weight;
    const void* dy;
    int64_t lddy;
    const void* ds;  // gradient of the stream output, or null
    int64_t ldds;
    int64_t nrows;
    int C;
    float eps;
    void* dx;        // (nrows, C)
    float* partial;  // (blocks, C), or null: no weight gradient
};

// Blocks per SM: 1,024 threads with 8 16-bit or 8 single channels each (64
// registers), 512 with more (128).
constexpr int grad_resident(int tpr, int E, int size, Mode mode) {
    const int threads = E * size <= 16 || (mode == kSingle && E == 8) ? 1024 : 512;
    return threads / block_threads(tpr) > 0 ? threads / block_threads(tpr) : 1;
}

// The block's rows once more, for a block that met a row whose squares leave fp32:
// by the whole block, value by value, each row's values multiplied by a power of two
// where they are squared. Apart from the rows' own loop, whose registers it would
// cost (from within, 170 us became 173 to 245 for 32,768 x 4,096).
template <typename T>
__device__ void rows_again(const NormGradArgs& g, int rows_at_once, float* shared_a, float* shared_b) {
    const int threads = blockDim.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const T* w = static_cast<const T*>(g.weight);
    float* mine = g.partial ? g.partial + (int64_t)blockIdx.x * g.C : nullptr;
    auto join = [&](float v, float* shared, bool largest) {
        v = largest ? lanes_max<32>(v) : lanes_sum<32>(v);
        __syncthreads();
        if (lane == 0) shared[warp] = v;
        __syncthreads();
        v = lane < threads / 32 ? shared[lane] : 0.0f;
        return largest ? lanes_max<32>(v) : lanes_sum<32>(v);
    };
    if (mine)
        for (int c = threadIdx.x; c < g.C; c += threads) mine[c] = 0.0f;
    const int64_t stride = (int64_t)gridDim.x * rows_at_once;
    for (int64_t first = (int64_t)blockIdx.x * rows_at_once; first < g.nrows; first += stride) {
        const int64_t last = first + rows_at_once < g.nrows ? first + rows_at_once : g.nrows;
        for (int64_t row = first; row < last; ++row) {
            const T* s = static_cast<const T*>(g.s) + row * g.lds;
            const T* dy = static_cast<const T*>(g.dy) + row * g.lddy;
            const T* ds = g.ds ? static_cast<const T*>(g.ds) + row * g.ldds : nullptr;
            T* dx = static_cast<T*>(g.dx) + row * (int64_t)g.C;
            float m = 0.0f, sum = 0.0f, along = 0.0f;
            for (int c = threadIdx.x; c < g.C; c += threads) m = max_abs(m, m, to_f32<T>(s[c]));
            m = join(m, shared_a, true);
            const float most = m * m * (float)g.C;  // bounds the sum
            const float by = !squares_leave_fp32(most, g.eps) ? 1.0f : most > 1.0f ? 0x1p-80f : 0x1p100f;
            for (int c = threadIdx.x; c < g.C; c += threads) {
                const float a = to_f32<T>(s[c]) * by;
                sum = fmaf(a, a, sum);
                along = fmaf(to_f32<T>(dy[c]) * to_f32<T>(w[c]), a, along);
            }
            sum = join(sum, shared_a, false);
            along = join(along, shared_b, false);
            // the reciprocal root is norm by, which may leave fp32 where the row is tiny
            const float norm = reciprocal_rms(sum, g.C, g.eps * by * by);
            const float mean = along * norm / (float)g.C;
            for (int c = threadIdx.x; c < g.C; c += threads) {
                const float d = to_f32<T>(dy[c]), n = to_f32<T>(s[c]) * by * norm;
                float grad = norm * (d * to_f32<T>(w[c]) - n * mean) * by;
                if (ds) grad += to_f32<T>(ds[c]);
                dx[c] = from_f32<T>(grad);
                if (mine) mine[c] = fmaf(d, n, mine[c]);
            }
        }
    }
}

template <typename T, int E, int TPR, Mode kMode>
__global__ void __launch_bounds__(block_threads(TPR), grad_resident(TPR, E, held_size(sizeof(T), kMode), kMode))
add_rms_norm_grad_kernel(const NormGradArgs g) {
    using S = Slice<T, E, TPR, kMode>;
    constexpr int kRows = TPR <= 32 ? 256 / TPR : 1;
    __shared__ float shared_a[2][32], shared_b[2][32];
    const int t = TPR <= 32 ? threadIdx.x % TPR : threadIdx.x;
    const int group = TPR <= 32 ? threadIdx.x / TPR : 0;
    float dw[E];
#pragma unroll
    for (int i = 0; i < E; ++i) dw[i] = 0.0f;
    // Rows of one warp or less: the other warps' loads hide a row's latency.
    // Rows of a block: its warps wait for one another, so the next row is on
    // its way meanwhile (single values have no registers for that).
    constexpr bool kAhead = TPR > 32 && kMode != kSingle;
    Held<T, E, kMode> w, s, dy, ds, s_next, dy_next, ds_next;
    load_held<TPR>(static_cast<const T*>(g.weight), g.C, t, w);
    auto fetch = [&](int64_t row) {
        const bool in = row < g.nrows;
        const int64_t at = in ? row : 0;
        const int C = in ? g.C : 0;
        load_held<TPR>(static_cast<const T*>(g.s) + at * g.lds, C, t, s_next);
        load_held<TPR>(static_cast<const T*>(g.dy) + at * g.lddy, C, t, dy_next);
        if (g.ds) load_held<TPR>(static_cast<const T*>(g.ds) + at * g.ldds, C, t, ds_next);
    };
    const int64_t stride = (int64_t)gridDim.x * kRows;
    if constexpr (kAhead) fetch(blockIdx.x);
    int parity = 0;
    bool again = false;
    for (int64_t first = (int64_t)blockIdx.x * kRows; first < g.nrows; first += stride) {
        const int64_t row = first + group;
        const bool live = row < g.nrows;
        const int64_t at = live ? row : 0;
        const int C = live ? g.C : 0;
        if constexpr (!kAhead) fetch(row);
        s = s_next;
        dy = dy_next;
        ds = ds_next;
        if constexpr (kAhead) fetch(row + stride);
        float sum = 0.0f, along = 0.0f;  // s^2, dy w s
#pragma unroll
        for (int i = 0; i < E; i += 8) {
            float a[8], b[8], c[8];
            s.get(i, a);
            dy.get(i, b);
            w.get(i, c);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                sum = fmaf(a[j], a[j], sum);
                along = fmaf(b[j] * c[j], a[j], along);
            }
        }
        sum = lanes_sum<TPR>(sum);
        along = lanes_sum<TPR>(along);
        if constexpr (TPR > 32) {
            // two buffers by turns: a row's partial sums are read before the
            // barrier of the next row, and overwritten only after it
            constexpr int kWarps = TPR / 32;
            const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
            if (lane == 0) {
                shared_a[parity][warp] = sum;
                shared_b[parity][warp] = along;
            }
            __syncthreads();
            sum = lanes_sum<kWarps>(shared_a[parity][lane % kWarps]);
            along = lanes_sum<kWarps>(shared_b[parity][lane % kWarps]);
            parity ^= 1;
        }
        again = again || (live && squares_leave_fp32(sum, g.eps));
        // 0 past the last row: with eps = 0 its reciprocal would put NaN into dw
        const float rstd = live ? reciprocal_rms(sum, g.C, g.eps) : 0.0f;
        const float mean = along * rstd / (float)g.C;  // mean(u n)
#pragma unroll
        for (int i = 0; i < E; i += 8) {
            float a[8], b[8], c[8], d[8];
            s.get(i, a);
            dy.get(i, b);
            w.get(i, c);
            if (g.ds) ds.get(i, d);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float n = a[j] * rstd;
                dw[i + j] = fmaf(b[j], n, dw[i + j]);
                a[j] = rstd * (b[j] * c[j] - n * mean);
                if (g.ds) a[j] += d[j];
            }
            s.set(i, a);
        }
        store_held<TPR>(static_cast<T*>(g.dx) + at * (int64_t)g.C, C, t, s);
    }
    // fp16 has no such rows
    if constexpr (!std::is_same<T, __half>::value) {
        if (__syncthreads_or(again)) {
            rows_again<T>(g, kRows, shared_a[0], shared_b[0]);
            return;
        }
    }
    if (!g.partial) return;
    float* mine = g.partial + (int64_t)blockIdx.x * g.C;
    if constexpr (TPR <= 32) {
        // the block's row groups, in order: the groups of a warp by shuffles,
        // then the warps through shared memory
#pragma unroll
        for (int o = TPR; o < 32; o <<= 1) {
#pragma unroll
            for (int i = 0; i < E; ++i) dw[i] += __shfl_xor_sync(0xffffffffu, dw[i], o);
        }
        __shared__ float sums[8][TPR * E];
        const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
        if (lane < TPR) {
#pragma unroll
            for (int i = 0; i < E; ++i) sums[warp][S::channel(i, t)] = dw[i];
        }
        __syncthreads();
        for (int c = threadIdx.x; c < g.C; c += 256) {
            float a = sums[0][c];
#pragma unroll
            for (int k = 1; k < 8; ++k) a += sums[k][c];
            mine[c] = a;
        }
    } else {
#pragma unroll
        for (int i = 0; i < E; ++i) {
            const int c = S::channel(i, t);
            if (c < g.C) mine[c] = dw[i];
        }
    }
}

// dw[c] = sum over blocks of partial[block][c]: kCols channels x 1,024 / kCols
// slices of the blocks per CTA. 8 channels keep a slice's few loads in flight at
// once and fill more SMs; from 2,048 channels on 32 do that too, with fewer CTAs
// (8,192 x 1,000: 21.7 us for the backward against 24.2; 300 x 8,192 18.4 against
// 15.2).
template <typename T, int kCols>
__global__ void __launch_bounds__(1024) weight_grad_kernel(const float* __restrict__ partial, int blocks, int C,
                                                           T* __restrict__ dw) {
    constexpr int kSlices = 1024 / kCols;
    __shared__ float sums[kCols][kSlices + 1];
    const int slice = threadIdx.x / kCols, col = threadIdx.x % kCols, c = blockIdx.x * kCols + col;
    float a = 0.0f;
    if (c < C) {
#pragma unroll 8
        for (int b = slice; b < blocks; b += kSlices) a += partial[(int64_t)b * C + c];
    }
    sums[col][slice] = a;
    __syncthreads();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (warp >= kCols) return;
    // warp w sums the slices of channel w
    a = sums[warp][lane];
#pragma unroll
    for (int k = 32; k < kSlices; k += 32) a += sums[warp][lane + k];
    a = f2s_warp_sum(a);
    const int at = blockIdx.x * kCols + warp;
    if (lane == 0 && at < C) dw[at] = from_f32<T>(a);
}

template <typename T>
void weight_grad_launch(const float* partial, int blocks, int C, void* dw, cudaStream_t st) {
    if (C < 2048) weight_grad_kernel<T, 8><<<ceil_div(C, 8), 1024, 0, st>>>(partial, blocks, C, static_cast<T*>(dw));
    else weight_grad_kernel<T, 32><<<ceil_div(C, 32), 1024, 0, st>>>(partial, blocks, C, static_cast<T*>(dw));
}

// Blocks of the backward: those that are resident at one time, each with
// several rows to share its dw over.
int grad_blocks(int64_t nrows, const Shape& s, int size, Mode mode) {
    const int64_t all = ceil_div64(nrows, block_rows(s.tpr));
    const int64_t most = (int64_t)sm_count() * grad_resident(s.tpr, s.e, held_size(size, mode), mode);
    return (int)(all < most ? all : most);
}

// Enough for any type and layout of (nrows, C): the most blocks of its shapes.
size_t grad_workspace(int64_t nrows, int C) {
    int blocks = 0;
    for (int size : {4, 2})
        for (Mode mode : {kSingle, kPair, kWide}) {
            const int b = grad_blocks(nrows, pick_shape(kGrad, size, nrows, C, mode), size, mode);
            blocks = b > blocks ? b : blocks;
        }
    return (size_t)blocks * C * sizeof(float);
}

}  // namespace
}  // namespace f2s

extern "C" int f2s_add_rms_norm_backward_workspace_bytes(int64_t rows, int C, size_t* bytes) {
    F2S_TRY(f2s::check_norm("add_rms_norm_backward", F2S_DTYPE_F32, rows, C, 0.0f));
    F2S_REQUIRE(bytes, "add_rms_norm_backward: null pointer");
    *bytes = f2s::grad_workspace(rows, C);
    return F2S_OK;
}

extern "C" int f2s_add_rms_norm_backward(const void* s, int64_t lds, const void* weight, int dtype, int64_t rows,
                                         int C, float eps, const void* dy, int64_t lddy, const void* ds, int64_t ldds,
                                         void* dx, void* dweight, void* workspace, size_t workspace_bytes,
                                         void* stream) {
    using namespace f2s;
    using namespace f2s::rows;
    F2S_TRY(check_norm("add_rms_norm_backward", dtype, rows, C, eps));
    cudaStream_t st = as_stream(stream);
    if (rows == 0) {
        if (dweight) F2S_CUDA_TRY(cudaMemsetAsync(dweight, 0, (size_t)C * dtype_size(dtype), st));
        return F2S_OK;
    }
    F2S_REQUIRE(s && weight && dy && dx, "add_rms_norm_backward: null pointer");
    F2S_REQUIRE(lds >= C && lddy >= C && (!ds || ldds >= C), "add_rms_norm_backward: row pitch below C=%d", C);
    const size_t needed = grad_workspace(rows, C);
    if (dweight && (!workspace || workspace_bytes < needed))
        return fail(F2S_ERR_WORKSPACE, "add_rms_norm_backward: workspace of %zu bytes, %zu needed", workspace_bytes,
                    needed);
    const int size = dtype_size(dtype);
    const Mode mode =
        Layout(rows, C, size).rows(s, lds).rows(dy, lddy).rows(ds, ldds).rows(dx, C).vector(weight).mode();
    NormGradArgs g{s, lds, weight, dy, lddy, ds, ldds, rows, C, eps, dx, dweight ? static_cast<float*>(workspace) : nullptr};
    const Shape shape = pick_shape(kGrad, size, rows, C, mode);
    const int blocks = grad_blocks(rows, shape, size, mode);
    TraceScope trace(kTagRmsNorm, st);
    F2S_DTYPE_SWITCH(dtype, dispatch<kGrad, T>(shape, mode, [&](auto e, auto tpr, auto m) {
        add_rms_norm_grad_kernel<T, e.value, tpr.value, m.value><<<blocks, block_threads(tpr.value), 0, st>>>(g);
    }));
    F2S_TRY(check_launch("add_rms_norm_grad_kernel"));
    if (!dweight) return F2S_OK;
    F2S_DTYPE_SWITCH(dtype, weight_grad_launch<T>(static_cast<const float*>(workspace), blocks, C, dweight, st));
    return check_launch("weight_grad_kernel");
}
