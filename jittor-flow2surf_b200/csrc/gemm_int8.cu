// Tensor-core forms of the 8-bit product (tcgen05 kind::i8, exact 32-bit
// sums): y[t, n] = xs[t] ws[n] sum_k x[t, k] w[n, k] + b[n].
//
// tiles  few tokens, or few tiles: one CTA per 128 channels x BN tokens, the
//        weights as the M = 128 operand (their bytes are what bounds the call),
//        K split over the CTAs of a cluster, which add their integer sums
//        through shared memory: the result does not depend on the split.
// pairs  many tokens: persistent CTA pairs (cta_group::2) on 256 x bn tiles.
//        Each CTA stages its 128 token rows and half of the channels, so a
//        pair moves 32 KB per 128-byte K block and SM where single CTAs of
//        128 x 256 would move 48 KB, more than L2 delivers at the int8 rate.
//
// Operands come by TMA in 128-byte rows (K blocks of 128) with the 128-byte
// swizzle; columns past K and rows past the matrix read as zeros.
#include "gemm_int8.cuh"
#include "row_ops.cuh"
#include "tc_common.cuh"

namespace f2s {
namespace {

using rows::from_f32;
using rows::to_f32;

constexpr size_t kSmemLimit = 227 * 1024;
constexpr int kBlockK = 128;

// Instruction descriptor of kind::i8: 32-bit integer sums, both operands
// signed and K-major.
constexpr uint32_t idesc_i8(int M, int N) {
    return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}

__device__ __forceinline__ void umma_i8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}

// Bounded wait on polls, as tc::mbar_wait_poll, that gives up early only for a wait
// that ran out elsewhere: the error word may hold another kernel's report (a value
// out of the fp16 range), which is no reason to stop this one.
__device__ __forceinline__ bool wait_poll(uint64_t* bar, uint32_t parity, int* err) {
    for (uint32_t i = 0; i < tc::kSpinLimit; ++i) {
        if (tc::mbar_try_wait_now(bar, parity)) return true;
        if ((i & 63u) == 63u && *reinterpret_cast<volatile int*>(err) == tc::kTcWaitTimeout) return false;
    }
    atomicExch(err, tc::kTcWaitTimeout);
    return false;
}

// ---- clusters ----
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
// Address of this CTA's shared address `a` in the CTA of cluster rank `r`.
__device__ __forceinline__ uint32_t map_rank(uint32_t a, uint32_t r) {
    uint32_t d;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(r));
    return d;
}
__device__ __forceinline__ void store_cluster(uint32_t a, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
    asm volatile("st.shared::cluster.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(a), "r"(x), "r"(y), "r"(z), "r"(w)
                 : "memory");
}

__device__ __forceinline__ void store_cluster(uint32_t a, uint32_t x) {
    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(a), "r"(x) : "memory");
}

template <typename T>
__device__ __forceinline__ float bias_at(const void* bias, int n) {
    return bias ? to_f32<T>(static_cast<const T*>(bias)[n]) : 0.0f;
}

// ---- tiles -------------------------------------------------------------------

struct TileArgs {
    const float* xs;
    const float* ws;
    const void* bias;
    void* y;
    int64_t ldy;
    int rows, cols;
    int k_blocks, stages, split, partial_bytes;
    int* err;
};

constexpr int kTileThreads = 192;  // TMA warp, MMA warp, 4 epilogue warps

template <typename T, int BN>
__global__ void __launch_bounds__(kTileThreads)
linear_int8_tiles_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x,
                         const TileArgs g) {
    constexpr uint32_t kA = 128 * 128, kB = BN * 128, kStage = kA + kB;
    constexpr uint32_t kCols = BN < 32 ? 32 : BN;
    extern __shared__ unsigned char raw[];
    unsigned char* smem =
        reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
    const int S = g.stages;
    int4* partial = reinterpret_cast<int4*>(smem + (size_t)S * kStage);  // [own][split][128] of 4 tokens
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + (size_t)S * kStage + g.partial_bytes);
    uint64_t* empty = full + S;
    uint64_t* done = empty + S;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + 1);
    int* issued = reinterpret_cast<int*>(tmem_slot + 1);  // K blocks loaded,
    int* used = issued + 1;                               // and multiplied

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int split = g.split;
    const int rank = (int)blockIdx.x % split;
    const int n0 = (int)blockIdx.x / split * 128, m0 = (int)blockIdx.y * BN;
    const int kb0 = (int)((int64_t)rank * g.k_blocks / split);
    const int kb1 = (int)((int64_t)(rank + 1) * g.k_blocks / split);

    auto load = [&](int i) {
        const int s = i % S;
        unsigned char* st = smem + (size_t)s * kStage;
        tc::mbar_arrive_expect_tx(&full[s], kStage);
        tc::tma_load_2d(st, &map_w, &full[s], (kb0 + i) * kBlockK, n0);
        tc::tma_load_2d(st + kA, &map_x, &full[s], (kb0 + i) * kBlockK, m0);
    };
    const int blocks = kb1 - kb0, ahead = min(min(blocks, S), 2);
    if (threadIdx.x == 0) {
        for (int s = 0; s < S; ++s) {
            tc::mbar_init(&full[s], 1);
            tc::mbar_init(&empty[s], 1);
        }
        tc::mbar_init(done, 1);
        tc::fence_barrier_init();
        // the first blocks are on their way while the CTA sets up (an issue takes
        // 0.1 us and more: all of a ring's would hold the other warps up)
        for (int i = 0; i < ahead; ++i) load(i);
    }
    if (warp == 1) tc::tmem_alloc(tmem_slot, kCols);
    tc::tc_fence_before();
    __syncthreads();
    tc::tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    // the other CTAs write into this one's `partial` only once it has started
    if (split > 1) cluster_arrive();

    if (warp == 0) {
        if (lane == 0) {
            int i = ahead;
            for (; i < blocks; ++i) {
                if (i >= S && !wait_poll(&empty[i % S], ((uint32_t)(i / S) & 1u) ^ 1u, g.err)) break;
                load(i);
            }
            *issued = i;
        }
        __syncwarp();
    } else if (warp == 1) {
        if (lane == 0) {
            int i = 0;
            for (; i < blocks; ++i) {
                const int s = i % S;
                if (!wait_poll(&full[s], (uint32_t)(i / S) & 1u, g.err)) break;
                tc::tc_fence_after();
                const uint32_t st = tc::smem_u32(smem + (size_t)s * kStage);
                const uint64_t a = tc::sw128_desc(st), b = tc::sw128_desc(st + kA);
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    umma_i8(tmem, a + 2 * k, b + 2 * k, idesc_i8(128, BN), (i | k) ? 1u : 0u);
                tc::umma_commit(&empty[s]);
            }
            *used = i;
            // every MMA issued has completed (TMEM is freed below)
            tc::umma_commit(done);
            tc::mbar_drain(done, 0);
        }
        __syncwarp();
    }
    // The accumulators come into registers and tensor memory is freed before this
    // CTA waits for the others of its cluster: one that held it meanwhile, while
    // another one could not get its own beside a kernel that waits for this
    // CTA's, would wait forever.
    const int channel = (warp & 3) * 32 + lane;  // a warp reads its TMEM lane quarter
    const int n = n0 + channel;
    bool ok = true;
    uint32_t v[BN];
    float ws = 0.0f, b = 0.0f;
    if (warp >= 2) {
        if (n < g.cols) {
            ws = __ldg(g.ws + n);
            b = bias_at<T>(g.bias, n);
        }
        ok = __all_sync(0xffffffffu, wait_poll(done, 0, g.err));
        tc::tc_fence_after();
        const uint32_t from = tmem + ((uint32_t)((warp & 3) * 32) << 16);
        if constexpr (BN == 16) {
            tc::tmem_ld16_issue(from, v);
            tc::tmem_ld16_wait(v);
        } else {
#pragma unroll
            for (int j = 0; j < BN; j += 32) {
                uint32_t (&part)[32] = *reinterpret_cast<uint32_t(*)[32]>(&v[j]);
                tc::tmem_ld32_issue(from + j, part);
                tc::tmem_ld32_wait(part);
            }
        }
        tc::tc_fence_before();
    }
    __syncthreads();
    tc::tc_fence_after();
    if (warp == 1) tc::tmem_dealloc(tmem, kCols);
    // where a wait ran out, the copies still under way land before the CTA exits
    auto land = [&]() {
        if (threadIdx.x == 0)
            for (int i = *used; i < *issued; ++i) tc::mbar_drain(&full[i % S], (uint32_t)(i / S) & 1u);
    };

    auto store = [&](int m, int acc) {
        static_cast<T*>(g.y)[m * g.ldy + n] = from_f32<T>(fmaf((float)acc * __ldg(g.xs + m), ws, b));
    };
    if (split == 1) {
        if (warp >= 2 && ok && n < g.cols) {
#pragma unroll
            for (int j = 0; j < BN; ++j)
                if (m0 + j < g.rows) store(m0 + j, (int)v[j]);
        }
        land();
        return;
    }
    cluster_wait();
    if (warp >= 2 && ok) {
        // four tokens at a time go to the CTAs of the cluster in turn, which
        // finish them (split is a power of two)
        const uint32_t mine = tc::smem_u32(partial + rank * 128 + channel);
#pragma unroll
        for (int j = 0; j < BN; j += 4) {
            const uint32_t four = (uint32_t)j / 4, to = four & (split - 1);
            store_cluster(map_rank(mine + (four & ~(uint32_t)(split - 1)) * 2048u, to), v[j], v[j + 1], v[j + 2],
                          v[j + 3]);
        }
    }
    cluster_arrive();
    cluster_wait();
    land();
    if (warp < 2 || !ok || n >= g.cols) return;
    for (int four = rank; four < BN / 4; four += split) {
        const int m = m0 + four * 4;
        if (m >= g.rows) break;
        const int4* from = partial + (four - rank) * 128 + channel;
        int4 acc = from[0];
        for (int r = 1; r < split; ++r) {
            const int4 more = from[r * 128];
            acc.x += more.x;
            acc.y += more.y;
            acc.z += more.z;
            acc.w += more.w;
        }
        store(m, acc.x);
        if (m + 1 < g.rows) store(m + 1, acc.y);
        if (m + 2 < g.rows) store(m + 2, acc.z);
        if (m + 3 < g.rows) store(m + 3, acc.w);
    }
}

int operand_map(CUtensorMap* map, const int8_t* p, int64_t ld, int nrows, int K, int box_rows) {
    // one row has no pitch of its own
    return make_tensor_map_2d_typed(map, p, kTmaU8, 128, nrows, K, nrows == 1 ? ceil_div64(K, 16) * 16 : ld, box_rows,
                                    kBlockK);
}

template <typename T, int BN>
int tiles_launch(const Int8Args& a, int split, cudaStream_t st) {
    CUtensorMap mw, mx;
    F2S_TRY(operand_map(&mw, a.w, a.ldw, a.cols, a.K, 128));
    F2S_TRY(operand_map(&mx, a.x, a.ldx, a.rows, a.K, BN));
    // fours of tokens per CTA, from every CTA of the cluster
    const int partial = split > 1 ? ceil_div(BN / 4, split) * split * 128 * 16 : 0;
    TileArgs g{a.xs, a.ws, a.bias, a.y, a.ldy, a.rows, a.cols, ceil_div(a.K, kBlockK), 0, split, partial, tc_error_word()};
    if (!g.err) return fail(F2S_ERR_CUDA, "linear_int8: device error word unavailable");
    const size_t stage = 128 * 128 + BN * 128;
    const size_t fixed = 1024 + 512 + partial;
    // two CTAs per SM where there are that many
    const int per_cta = ceil_div(g.k_blocks, split);
    const int64_t ctas = (int64_t)ceil_div(a.cols, 128) * split * ceil_div(a.rows, BN);
    const size_t budget = ctas > sm_count() ? kSmemLimit / 2 - 1024 : kSmemLimit;
    int stages = (int)((budget - fixed) / stage);
    stages = stages < 12 ? stages : 12;
    stages = stages < per_cta ? stages : per_cta;
    g.stages = stages;
    const size_t smem = fixed + stages * stage;
    auto kernel = linear_int8_tiles_kernel<T, BN>;
    F2S_TRY(allow_shared(kernel, smem));
    const int token_tiles = ceil_div(a.rows, BN);
    F2S_LIMIT(token_tiles <= 65535, "linear_int8: %d rows", a.rows);
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(ceil_div(a.cols, 128) * split), (unsigned)token_tiles);
    cfg.blockDim = dim3(kTileThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)split;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    F2S_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, mw, mx, g));
    return check_launch("linear_int8_tiles_kernel");
}

// ---- pairs -------------------------------------------------------------------

struct PairArgs;

// A pair's output tiles: t, t + pairs, ... of an order in bands of 8 token
// tiles, channels outer, so that the operands of the tiles that run at one
// time stay in L2. Advanced by additions: a division costs a warp as much as
// the arithmetic of ten output columns.
struct Walk {
    int t, band, in_band;
    __device__ __forceinline__ void start(const PairArgs& g, int first);
    __device__ __forceinline__ void next(const PairArgs& g, int pairs);
    __device__ __forceinline__ void at(const PairArgs& g, int& m0, int& n0) const;
};

struct PairArgs {
    const float* xs;
    const float* ws;
    const void* bias;
    void* y;
    int64_t ldy;
    int rows, cols;
    int bn;          // channels of a tile: 64, 128, 192 or 256
    int k_blocks, stages;
    int m_tiles, n_tiles;
    int step_bands, step_rest;  // the number of pairs, in bands and tiles
    int boxes;       // y written by TMA
    uint32_t idesc;
    int* err;
};

__device__ __forceinline__ void Walk::start(const PairArgs& g, int first) {
    t = first;
    band = first / (8 * g.n_tiles);
    in_band = first - band * 8 * g.n_tiles;
}
__device__ __forceinline__ void Walk::next(const PairArgs& g, int pairs) {
    t += pairs;
    band += g.step_bands;
    in_band += g.step_rest;
    if (in_band >= 8 * g.n_tiles) {
        in_band -= 8 * g.n_tiles;
        ++band;
    }
}
__device__ __forceinline__ void Walk::at(const PairArgs& g, int& m0, int& n0) const {
    const int high = g.m_tiles - band * 8;  // of the last band, if below 8
    const int n = high >= 8 ? in_band >> 3 : in_band / high;
    m0 = (band * 8 + in_band - n * (high >= 8 ? 8 : high)) * 256;
    n0 = n * g.bn;
}

constexpr int kPairThreads = 64 + 32 * 8;
constexpr int kBox = 32 * 128;      // 32 rows of 128 bytes of y

// TMA load by either CTA of a pair, signalling a barrier of the pair's leader.
__device__ __forceinline__ void tma_load_pair(void* dst, const CUtensorMap* map, uint32_t bar, int c0, int c1) {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%3, %4}], [%2];" ::"r"(tc::smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1)
        : "memory");
}

__device__ __forceinline__ void umma_i8_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}

// Arrive on `bar` in both CTAs of the pair once the MMAs issued so far complete.
__device__ __forceinline__ void commit_pair(uint64_t* bar) {
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
            tc::smem_u32(bar)),
        "h"((uint16_t)3)
        : "memory");
}

// Arrive on a barrier of either CTA of the pair. Only tensor memory is handed
// over, ordered by the tcgen05 fences around it: a release of cluster scope would
// wait for this thread's stores of y first, 1 us a tile.
__device__ __forceinline__ void arrive_pair(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}

// K blocks `used` to `loaded` or `other` are loaded by the leader or the other CTA, at
// most one of each stage, and not waited for: until they land. A barrier counts both
// CTAs' bytes; a part that one of them no longer loaded is taken off, or not expected.
__device__ __forceinline__ void drain_pair(uint64_t* full, int S, uint32_t stage_bytes, int used, int loaded, int other) {
    for (int i = used; i < loaded || i < other; ++i) {
        uint64_t* bar = &full[i % S];
        if (i >= other)
            asm volatile("mbarrier.complete_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(tc::smem_u32(bar)),
                         "r"(stage_bytes)
                         : "memory");
        if (i >= loaded) tc::mbar_arrive_expect_tx(bar, stage_bytes);
        tc::mbar_drain(bar, (uint32_t)(i / S) & 1u);
    }
}

// 16 lanes x 64 columns of TMEM: register 4 j + 2 i + k holds lane t / 4 + 8 i of
// column 8 j + 2 (t % 4) + k, for thread t.
__device__ __forceinline__ void tmem_ld16_issue(uint32_t taddr, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.16x256b.x8.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr));
}

// Four 8 x 8 matrices of 16-bit values, a thread holding row t / 4, columns 2 (t % 4)
// and the next of each; lane 8 i + k points at row k of matrix i.
__device__ __forceinline__ void store_matrices(unsigned char* to, const uint32_t (&r)[4]) {
    asm volatile("stmatrix.sync.aligned.m8n8.x4.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(tc::smem_u32(to)), "r"(r[0]),
                 "r"(r[1]), "r"(r[2]), "r"(r[3])
                 : "memory");
}

// The warp's last store has read its box.
__device__ __forceinline__ void box_free(int lane) {
    if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
    __syncwarp();
}

// Eight epilogue warps, two per TMEM lane quarter with every other box of 128
// bytes of y. Where K is small their shared memory traffic bounds the kernel: a
// 16-bit y with a whole row in a lane, which takes every scale and bias to every
// lane, takes 53 us for 65,536 x 192 -> 1,536 against 49 for the split of rows
// below. A 32-bit y is bound by its writes (75 us, 5.4 TB/s). With a row in a lane
// sixteen warps, on two accumulators by turns, took 54 (16-bit) and 84 us (32-bit),
// and two boxes of a warp by turns 52 and 82.
template <typename T>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kPairThreads, 1)
linear_int8_pairs_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w,
                         const __grid_constant__ CUtensorMap map_y, const PairArgs g) {
    constexpr int kBoxCols = 128 / (int)sizeof(T);
    constexpr int kWarps = 8;
    constexpr int kCols = 128;  // columns of a warp
    extern __shared__ unsigned char raw[];
    unsigned char* smem =
        reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
    const int S = g.stages;
    const uint32_t a_bytes = 128 * 128, b_bytes = (uint32_t)g.bn * 64, stage_bytes = a_bytes + b_bytes;
    unsigned char* boxes = smem + (size_t)S * stage_bytes;  // kWarps x kBox
    float* vectors = reinterpret_cast<float*>(boxes + kWarps * kBox);  // a warp's [ws kCols | bias kCols]
    uint64_t* full = reinterpret_cast<uint64_t*>(vectors + kWarps * 2 * kCols);  // leader's: both CTAs' bytes
    uint64_t* empty = full + S;
    uint64_t* tfull = empty + S;   // [2]
    uint64_t* tempty = tfull + 2;  // [2] leader's: eight epilogue warps of both CTAs
    uint64_t* done = tempty + 2;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + 1);
    int* issued = reinterpret_cast<int*>(tmem_slot + 1);  // [2] leader's: K blocks that each CTA loaded
    int* used = issued + 2;                               // leader's: and multiplied

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_rank();
    const int tiles = g.m_tiles * g.n_tiles, pairs = (int)gridDim.x / 2, pair = (int)blockIdx.x / 2;
    Walk walk;
    walk.start(g, pair);

    if (threadIdx.x == 0) {
        for (int s = 0; s < S; ++s) {
            tc::mbar_init(&full[s], 1);
            tc::mbar_init(&empty[s], 1);
        }
        for (int b = 0; b < 2; ++b) {
            tc::mbar_init(&tfull[b], 1);
            tc::mbar_init(&tempty[b], 16);
        }
        tc::mbar_init(done, 1);
        tc::fence_barrier_init();
        tc::prefetch_tensormap(&map_x);
        tc::prefetch_tensormap(&map_w);
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tc::smem_u32(tmem_slot)),
                     "r"(512u)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    tc::tc_fence_before();
    __syncthreads();
    cluster_arrive();
    cluster_wait();
    tc::tc_fence_after();
    const uint32_t tmem = *tmem_slot;

    if (warp == 0) {
        if (lane == 0) {
            int stage = 0, count = 0;
            uint32_t phase = 0;
            bool ok = true;
            for (; ok && walk.t < tiles; walk.next(g, pairs)) {
                int m0, n0;
                walk.at(g, m0, n0);
                for (int kb = 0; kb < g.k_blocks; ++kb) {
                    if (!wait_poll(&empty[stage], phase ^ 1u, g.err)) {
                        ok = false;
                        break;
                    }
                    unsigned char* st = smem + (size_t)stage * stage_bytes;
                    const uint32_t bar = map_rank(tc::smem_u32(&full[stage]), 0);
                    if (rank == 0) tc::mbar_arrive_expect_tx(&full[stage], 2 * stage_bytes);
                    tma_load_pair(st, &map_x, bar, kb * kBlockK, m0 + (int)rank * 128);
                    tma_load_pair(st + a_bytes, &map_w, bar, kb * kBlockK, n0 + (int)rank * (g.bn / 2));
                    ++count;
                    if (++stage == S) {
                        stage = 0;
                        phase ^= 1u;
                    }
                }
            }
            store_cluster(map_rank(tc::smem_u32(issued + rank), 0), (uint32_t)count);
        }
        __syncwarp();
    } else if (warp == 1) {
        if (lane == 0 && rank == 0) {
            int stage = 0, iter = 0, count = 0;
            uint32_t phase = 0;
            bool ok = true;
            for (int t = pair; ok && t < tiles; t += pairs, ++iter) {
                const int buf = iter & 1;
                if (!wait_poll(&tempty[buf], ((uint32_t)(iter >> 1) & 1u) ^ 1u, g.err)) break;
                tc::tc_fence_after();
                const uint32_t d = tmem + (uint32_t)(buf * 256);
                for (int kb = 0; kb < g.k_blocks; ++kb) {
                    if (!wait_poll(&full[stage], phase, g.err)) {
                        ok = false;
                        break;
                    }
                    ++count;
                    tc::tc_fence_after();
                    const uint32_t st = tc::smem_u32(smem + (size_t)stage * stage_bytes);
                    const uint64_t a = tc::sw128_desc(st), b = tc::sw128_desc(st + a_bytes);
#pragma unroll
                    for (int k = 0; k < 4; ++k) umma_i8_pair(d, a + 2 * k, b + 2 * k, g.idesc, (kb | k) ? 1u : 0u);
                    commit_pair(&empty[stage]);
                    if (++stage == S) {
                        stage = 0;
                        phase ^= 1u;
                    }
                }
                if (ok) commit_pair(&tfull[buf]);
            }
            *used = count;
            commit_pair(done);
            tc::mbar_drain(done, 0);
        }
        __syncwarp();
    } else {
        const int e = warp - 2;
        const int quarter = warp & 3;      // TMEM lanes of this warp
        const int half = e >> 2;           // boxes half, half + 2, ...
        unsigned char* box = boxes + e * kBox;
        float* ws = vectors + e * 2 * kCols;
        float* bs = ws + kCols;
        const uint32_t to_leader[2] = {map_rank(tc::smem_u32(&tempty[0]), 0), map_rank(tc::smem_u32(&tempty[1]), 0)};
        // a tile's token scale and the scales and biases of this warp's columns
        // (box by box), on their way while the tile before is written; for this
        // warp alone, so there is no barrier that another warp could miss. Past
        // the last row or column: the last one's, not written.
        int m0 = 0, n0 = 0;
        float xs_next = 0.0f, ws_next[kCols / 32], bs_next[kCols / 32];
        auto fetch = [&]() {
            if (walk.t >= tiles) return;
            walk.at(g, m0, n0);
            xs_next = __ldg(g.xs + min(m0 + (int)rank * 128 + quarter * 32 + lane, g.rows - 1));
#pragma unroll
            for (int i = 0; i < kCols / 32; ++i) {
                const int l = lane + 32 * i;
                const int n = min(n0 + (half + 2 * (l / kBoxCols)) * kBoxCols + l % kBoxCols, g.cols - 1);
                ws_next[i] = __ldg(g.ws + n);
                bs_next[i] = bias_at<T>(g.bias, n);
            }
        };
        fetch();
        for (int t = pair, iter = 0; t < tiles; t += pairs, ++iter) {
            const int buf = iter & 1;
            const int row0 = m0 + (int)rank * 128 + quarter * 32, col0 = n0;
            const float xs = xs_next;
            float xs4[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) xs4[i] = __shfl_sync(0xffffffffu, xs, (lane >> 2) + 8 * i);
#pragma unroll
            for (int i = 0; i < kCols / 32; ++i) {
                ws[lane + 32 * i] = ws_next[i];
                bs[lane + 32 * i] = bs_next[i];
            }
            __syncwarp();
            walk.next(g, pairs);
            fetch();
            const bool ok = wait_poll(&tfull[buf], (uint32_t)(iter >> 1) & 1u, g.err);
            // a warp that gave up stops with its lanes together
            if (!__all_sync(0xffffffffu, ok)) break;
            tc::tc_fence_after();
            const uint32_t acc = tmem + (uint32_t)(buf * 256) + ((uint32_t)(quarter * 32) << 16);
            int held_at = 0;  // this box's columns in ws, bs
            for (int c = half * kBoxCols; c < g.bn; c += 2 * kBoxCols, held_at += kBoxCols) {
                // through registers into the box, 128 bytes of y per row, its 16-byte chunks
                // swizzled
                if constexpr (sizeof(T) == 4) {
                    // a lane's row
                    uint32_t v[32];
                    tc::tmem_ld32_issue(acc + c, v);
                    tc::tmem_ld32_wait(v);
                    box_free(lane);
#pragma unroll
                    for (int j = 0; j < 32; j += 4) {
                        const float4 w4 = *reinterpret_cast<const float4*>(ws + held_at + j);
                        const float4 b4 = *reinterpret_cast<const float4*>(bs + held_at + j);
                        *reinterpret_cast<float4*>(box + lane * 128 + (((j / 4) ^ (lane & 7)) << 4)) =
                            make_float4(fmaf((float)(int)v[j] * xs, w4.x, b4.x), fmaf((float)(int)v[j + 1] * xs, w4.y, b4.y),
                                        fmaf((float)(int)v[j + 2] * xs, w4.z, b4.z), fmaf((float)(int)v[j + 3] * xs, w4.w, b4.w));
                    }
                } else {
                    // columns 8 j + 2 (lane % 4) and the next one of the rows lane / 4 + 8 i: with
                    // these, a lane reads 32 scales and biases of the box, not 128
                    float2 w2[8], b2[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        w2[j] = *reinterpret_cast<const float2*>(ws + held_at + 8 * j + 2 * (lane & 3));
                        b2[j] = *reinterpret_cast<const float2*>(bs + held_at + 8 * j + 2 * (lane & 3));
                    }
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        uint32_t v[32];
                        tmem_ld16_issue(acc + c + ((uint32_t)(16 * h) << 16), v);
                        tc::tmem_ld32_wait(v);
                        if (h == 0) box_free(lane);
#pragma unroll
                        for (int j = 0; j < 8; j += 2) {
                            uint32_t y8[4];  // rows 0-7 and 8-15 of columns 8 j .., then of 8 j + 8 ..
#pragma unroll
                            for (int k = 0; k < 4; ++k) {
                                const int n = j + k / 2, at = 4 * n + 2 * (k & 1);
                                const float scale = xs4[2 * h + (k & 1)];
                                y8[k] = rows::pack2(fmaf((float)(int)v[at] * scale, w2[n].x, b2[n].x),
                                                    fmaf((float)(int)v[at + 1] * scale, w2[n].y, b2[n].y), T());
                            }
                            const int r = 16 * h + (lane & 15);  // the row that this lane points at
                            store_matrices(box + r * 128 + (((j + (lane >> 4)) ^ (r & 7)) << 4), y8);
                        }
                    }
                }
                if (c + 2 * kBoxCols >= g.bn) {
                    // this warp's last read of the accumulator
                    tc::tc_fence_before();
                    __syncwarp();
                    if (lane == 0) arrive_pair(to_leader[buf]);
                }
                if (col0 + c >= g.cols) continue;  // past the last column
                if (g.boxes) {
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    __syncwarp();
                    if (lane == 0) {
                        asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];" ::"l"(
                                         reinterpret_cast<uint64_t>(&map_y)),
                                     "r"(tc::smem_u32(box)), "r"(col0 + c), "r"(row0)
                                     : "memory");
                        asm volatile("cp.async.bulk.commit_group;" ::: "memory");
                    }
                } else {
                    // any pitch: the box's rows one by one, lanes along the row
                    __syncwarp();
                    const T* held = reinterpret_cast<const T*>(box);
                    T* to = static_cast<T*>(g.y) + (int64_t)row0 * g.ldy + col0 + c;
#pragma unroll 8
                    for (int r = 0; r < 32; ++r, to += g.ldy) {
#pragma unroll
                        for (int k = lane; k < kBoxCols; k += 32) {
                            const int chunk = k * (int)sizeof(T) / 16, in = k % (16 / (int)sizeof(T));
                            if (row0 + r < g.rows && col0 + c + k < g.cols)
                                to[k] = held[(r * 128 + ((chunk ^ (r & 7)) << 4)) / (int)sizeof(T) + in];
                        }
                    }
                }
            }
            // a warp without a box in this tile frees its share too
            if (half * kBoxCols >= g.bn) {
                tc::tc_fence_before();
                __syncwarp();
                if (lane == 0) arrive_pair(to_leader[buf]);
            }
        }
        if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
        __syncwarp();
    }
    // neither CTA leaves, or frees its TMEM, while the other still uses it
    tc::tc_fence_before();
    __syncthreads();
    cluster_arrive();
    cluster_wait();
    tc::tc_fence_after();
    // what is still under way to this CTA lands before either leaves: the arrivals of the
    // leader's commits at the other CTA and, where a wait ran out, copies
    if (threadIdx.x == 0) {
        if (rank == 0) drain_pair(full, S, stage_bytes, *used, issued[0], issued[1]);
        else tc::mbar_drain(done, 0);
    }
    if (warp == 1)
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
    __syncthreads();
    cluster_arrive();
    cluster_wait();
}

template <typename T>
int pairs_launch(const Int8Args& a, int bn, cudaStream_t st) {
    CUtensorMap mx, mw, my;
    F2S_TRY(operand_map(&mx, a.x, a.ldx, a.rows, a.K, 128));
    F2S_TRY(operand_map(&mw, a.w, a.ldw, a.cols, a.K, bn / 2));
    PairArgs g{};
    g.xs = a.xs;
    g.ws = a.ws;
    g.bias = a.bias;
    g.y = a.y;
    g.ldy = a.ldy;
    g.rows = a.rows;
    g.cols = a.cols;
    g.bn = bn;
    g.k_blocks = ceil_div(a.K, kBlockK);
    g.m_tiles = ceil_div(a.rows, 256);
    g.n_tiles = ceil_div(a.cols, bn);
    g.idesc = idesc_i8(256, bn);
    g.err = tc_error_word();
    if (!g.err) return fail(F2S_ERR_CUDA, "linear_int8: device error word unavailable");
    F2S_LIMIT((int64_t)g.m_tiles * g.n_tiles <= INT32_MAX / 2, "linear_int8: %d x %d outputs", a.rows, a.cols);
    g.boxes = rows::aligned16(a.y) && a.ldy * (int64_t)sizeof(T) % 16 == 0;
    if (g.boxes)
        F2S_TRY(make_tensor_map_2d_typed(&my, a.y, sizeof(T) == 4 ? kTmaF32 : kTmaBF16, 128, a.rows, a.cols, a.ldy, 32,
                                         128 / (int)sizeof(T)));
    else my = mx;
    const size_t stage = 128 * 128 + (size_t)bn * 64;
    const size_t fixed = 1024 + 8 * (kBox + 2 * 128 * sizeof(float)) + 512;
    int stages = (int)((kSmemLimit - fixed) / stage);
    g.stages = stages > 8 ? 8 : stages;
    const size_t smem = fixed + g.stages * stage;
    auto kernel = linear_int8_pairs_kernel<T>;
    F2S_TRY(allow_shared(kernel, smem));
    const int tiles = g.m_tiles * g.n_tiles, most = sm_count() / 2, pairs = tiles < most ? tiles : most;
    g.step_bands = pairs / (8 * g.n_tiles);
    g.step_rest = pairs % (8 * g.n_tiles);
    kernel<<<2 * pairs, kPairThreads, smem, st>>>(mx, mw, my, g);
    return check_launch("linear_int8_pairs_kernel");
}

// The forms' times on a B200, in us, fitted to 60 shapes of 1 to 2,048 tokens: a
// CTA of `tiles` takes 3 and 0.45 per K block and the kernel 2 around that; joining
// K parts takes up to 0.6 with the tokens, and clusters of 4 and 8 leave some SMs
// without a CTA (a GPU processing cluster holds whole ones). `pairs` takes 5.5 and
// 0.38 per K block of each 256 x bn tile.
float tiles_time(const Int8Args& a, int bn, int split) {
    const int64_t ctas = (int64_t)ceil_div(a.cols, 128) * ceil_div(a.rows, bn) * split;
    const int sms = sm_count(), usable = split == 8 ? sms * 7 / 10 : split == 4 ? sms * 9 / 10 : sms;
    return 2.0f + (split > 1 ? 0.6f * (float)bn / 64.0f : 0.0f) +
           (float)ceil_div64(ctas, usable) * (3.0f + 0.45f * (float)ceil_div(ceil_div(a.K, kBlockK), split));
}

int tile_tokens(const Int8Args& a) { return a.rows <= 16 ? 16 : a.rows <= 32 ? 32 : 64; }

int tile_split(const Int8Args& a, int bn) {
    int split = 1;
    for (int s = 2; s <= 8 && s <= ceil_div(a.K, kBlockK); s *= 2)
        if (tiles_time(a, bn, s) < tiles_time(a, bn, split)) split = s;
    return split;
}

// The channel tile with the fewest columns computed (one of 64 takes as long as
// one of 128), the larger on ties.
int pair_channels(const Int8Args& a) {
    int bn = 256;
    for (int c : {192, 128, 64})
        if (ceil_div(a.cols, c) * (c < 128 ? 128 : c) < ceil_div(a.cols, bn) * bn) bn = c;
    return bn;
}

float pairs_time(const Int8Args& a, int bn) {
    const int64_t tiles = (int64_t)ceil_div(a.rows, 256) * ceil_div(a.cols, bn);
    return 5.5f + 0.38f * (float)ceil_div64(tiles, sm_count() / 2) * (float)ceil_div(a.K, kBlockK);
}

}  // namespace

int linear_int8_tensor(const Int8Args& a, cudaStream_t st) {
    const int bn = tile_tokens(a), split = tile_split(a, bn), channels = pair_channels(a);
    int status = F2S_OK;
    if (pairs_time(a, channels) < tiles_time(a, bn, split)) {
        F2S_DTYPE_SWITCH(a.dtype, status = pairs_launch<T>(a, channels, st));
        return status;
    }
    F2S_DTYPE_SWITCH(a.dtype, switch (bn) {
        case 16: status = tiles_launch<T, 16>(a, split, st); break;
        case 32: status = tiles_launch<T, 32>(a, split, st); break;
        default: status = tiles_launch<T, 64>(a, split, st); break;
    });
    return status;
}

}  // namespace f2s
