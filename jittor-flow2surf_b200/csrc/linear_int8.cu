// Product of 8-bit integer rows with scales for each token and channel:
//   y[t, n] = xs[t] ws[n] sum_k x[t, k] w[n, k] + b[n],
// the sum exact in 32 bits (K <= 131,071 keeps 2^14 K below 2^31).
#include "gemm_int8.cuh"
#include "row_ops.cuh"

namespace f2s {
namespace {

using namespace rows;

constexpr int kMaxK = 131071;

// A few tokens: bound by the weights' bytes and by latency. A warp takes two
// channels (and 1 / kSplit of their K, joined in shared memory), 16 bytes of
// each per lane and step, four products and sums per dp4a; its loads of several
// steps are in flight at once.
//
// Against the tensor cores, which take 4.5 us at least and little more for more
// tokens (both in us):   1 x 4096 -> 4096 6.2, 7.5;   4 x 192 -> 1536 3.1, 4.2;
// 4 x 8192 -> 1024 4.4, 7.2;   4 x 4096 -> 4096 9.7, 8.0;   1 x 8192 -> 8192 18.6,
// 17.8: past 2^25 products of 8-bit values this form's arithmetic costs more.
constexpr int kFew = 4;  // tokens at most
constexpr int64_t kFewProducts = 1 << 25;
constexpr int kFewWarps = 8;  // per block

template <typename T, int R>
__global__ void __launch_bounds__(32 * kFewWarps) linear_int8_few_kernel(const Int8Args g, int split) {
    __shared__ int sums[kFewWarps][2 * R];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int group = warp / split, part = warp - group * split;
    const int n0 = ((int)blockIdx.x * (kFewWarps / split) + group) * 2;
    const int chunks = g.K / 16;  // whole 16-byte chunks
    const int c0 = (int)((int64_t)part * chunks / split), c1 = (int)((int64_t)(part + 1) * chunks / split);
    int acc[2][R] = {};
    // a channel past the last one reads the last one and is not written
    const int8_t* w0 = g.w + (int64_t)(n0 < g.cols ? n0 : g.cols - 1) * g.ldw;
    const int8_t* w1 = g.w + (int64_t)(n0 + 1 < g.cols ? n0 + 1 : g.cols - 1) * g.ldw;
#pragma unroll 4
    for (int c = c0 + lane; c < c1; c += 32) {
        const int4 a = __ldg(reinterpret_cast<const int4*>(w0) + c), b = __ldg(reinterpret_cast<const int4*>(w1) + c);
#pragma unroll
        for (int r = 0; r < R; ++r) {
            if (r >= g.rows) break;
            const int4 x = __ldg(reinterpret_cast<const int4*>(g.x + r * g.ldx) + c);
            acc[0][r] = __dp4a(a.w, x.w, __dp4a(a.z, x.z, __dp4a(a.y, x.y, __dp4a(a.x, x.x, acc[0][r]))));
            acc[1][r] = __dp4a(b.w, x.w, __dp4a(b.z, x.z, __dp4a(b.y, x.y, __dp4a(b.x, x.x, acc[1][r]))));
        }
    }
    // the bytes past the last whole chunk, one per lane of the first part
    const int k = chunks * 16 + lane;
    if (part == 0 && k < g.K) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
            if (r >= g.rows) break;
            const int x = g.x[r * g.ldx + k];
            acc[0][r] += w0[k] * x;
            acc[1][r] += w1[k] * x;
        }
    }
#pragma unroll
    for (int i = 0; i < 2 * R; ++i) {
        const int sum = __reduce_add_sync(0xffffffffu, acc[i & 1][i >> 1]);
        if (lane == 0) sums[warp][i] = sum;
    }
    if (split > 1) __syncthreads();
    else __syncwarp();
    if (part == 0 && lane < 2 * R) {
        const int n = n0 + (lane & 1), r = lane >> 1;
        if (n < g.cols && r < g.rows) {
            int sum = 0;
            for (int p = 0; p < split; ++p) sum += sums[warp + p][lane];
            const float b = g.bias ? to_f32<T>(static_cast<const T*>(g.bias)[n]) : 0.0f;
            static_cast<T*>(g.y)[r * g.ldy + n] = from_f32<T>(fmaf((float)sum * g.xs[r], g.ws[n], b));
        }
    }
}

template <typename T>
int few_launch(const Int8Args& g, cudaStream_t st) {
    // K split until every SM has 16 warps, at least two steps each
    int split = 1;
    while (split < kFewWarps && (int64_t)ceil_div(g.cols, 2) * split < 16 * sm_count() && g.K >= 2 * 512 * 2 * split)
        split *= 2;
    const int blocks = ceil_div(g.cols, 2 * (kFewWarps / split));
    auto go = [&](auto kernel) { kernel<<<blocks, 32 * kFewWarps, 0, st>>>(g, split); };
    if (g.rows == 1) go(linear_int8_few_kernel<T, 1>);
    else if (g.rows == 2) go(linear_int8_few_kernel<T, 2>);
    else go(linear_int8_few_kernel<T, 4>);
    return check_launch("linear_int8_few_kernel");
}

// Any pitch and alignment: 64 x 64 outputs per block of 256 threads, 4 x 4
// each, K in steps of 64 staged in shared memory as words of four, four
// products and sums per dp4a.
template <typename T>
__global__ void __launch_bounds__(256) linear_int8_any_kernel(const Int8Args g) {
    __shared__ int8_t xa[64][68], wa[64][68];
    const int m0 = blockIdx.x * 64, n0 = blockIdx.y * 64;
    const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
    int acc[4][4] = {};
    for (int k0 = 0; k0 < g.K; k0 += 64) {
        for (int i = threadIdx.x; i < 64 * 64; i += 256) {
            const int r = i / 64, k = i % 64;
            const bool in = k0 + k < g.K;
            xa[r][k] = in && m0 + r < g.rows ? g.x[(m0 + r) * g.ldx + k0 + k] : (int8_t)0;
            wa[r][k] = in && n0 + r < g.cols ? g.w[(n0 + r) * g.ldw + k0 + k] : (int8_t)0;
        }
        __syncthreads();
#pragma unroll 4
        for (int k = 0; k < 64; k += 4) {
            int a[4], b[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                a[i] = *reinterpret_cast<const int*>(&xa[ty + 16 * i][k]);
                b[i] = *reinterpret_cast<const int*>(&wa[tx + 16 * i][k]);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] = __dp4a(a[i], b[j], acc[i][j]);
        }
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int m = m0 + ty + 16 * i;
        if (m >= g.rows) continue;
        const float xs = g.xs[m];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int n = n0 + tx + 16 * j;
            if (n >= g.cols) continue;
            const float b = g.bias ? to_f32<T>(static_cast<const T*>(g.bias)[n]) : 0.0f;
            static_cast<T*>(g.y)[m * g.ldy + n] = from_f32<T>(fmaf((float)acc[i][j] * xs, g.ws[n], b));
        }
    }
}

template <typename T>
int any_launch(const Int8Args& g, cudaStream_t st) {
    F2S_LIMIT(ceil_div(g.cols, 64) <= 65535, "linear_int8: %d columns of an unaligned pitch", g.cols);
    linear_int8_any_kernel<T><<<dim3(ceil_div(g.rows, 64), ceil_div(g.cols, 64)), 256, 0, st>>>(g);
    return check_launch("linear_int8_any_kernel");
}

}  // namespace
}  // namespace f2s

extern "C" int f2s_linear_int8(const int8_t* x, int64_t ldx, const float* x_scale, const int8_t* w, int64_t ldw,
                               const float* w_scale, const void* bias, void* y, int64_t ldy, int dtype, int rows,
                               int cols, int K, void* stream) {
    F2S_TRY(f2s::rows::check_dtype("linear_int8", dtype));
    F2S_REQUIRE(rows >= 0 && cols >= 1 && K >= 1, "linear_int8: bad shape rows=%d cols=%d K=%d", rows, cols, K);
    F2S_LIMIT(K <= f2s::kMaxK, "linear_int8: K=%d, at most %d for an exact 32-bit sum", K, f2s::kMaxK);
    // a tile's last row and column are 32-bit numbers
    F2S_LIMIT(rows <= INT32_MAX - 255 && cols <= INT32_MAX - 255, "linear_int8: %d x %d outputs, at most 2^31 - 256 a side",
              rows, cols);
    if (rows == 0) return F2S_OK;
    F2S_REQUIRE(x && x_scale && w && w_scale && y, "linear_int8: null pointer");
    F2S_REQUIRE(ldx >= K && ldw >= K && ldy >= cols, "linear_int8: row pitch below the row");
    f2s::Int8Args g{x, ldx, x_scale, w, ldw, w_scale, bias, y, ldy, dtype, rows, cols, K};
    cudaStream_t st = f2s::as_stream(stream);
    f2s::TraceScope trace(f2s::kTagGemmInt8, st);
    using f2s::rows::aligned16;
    const bool aligned = aligned16(x) && aligned16(w) && (ldx % 16 == 0 || rows == 1) && (ldw % 16 == 0 || cols == 1);
    if (aligned && !(rows <= f2s::kFew && (int64_t)rows * cols * K <= f2s::kFewProducts))
        return f2s::linear_int8_tensor(g, st);
    int status = F2S_OK;
    if (aligned) F2S_DTYPE_SWITCH(dtype, status = f2s::few_launch<T>(g, st))
    else F2S_DTYPE_SWITCH(dtype, status = f2s::any_launch<T>(g, st));
    return status;
}
