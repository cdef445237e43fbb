// Tensor-core kernels of the adapters for few rows: x.A of a tile of rows
// (any batch; k_ad_shrink) and the product with W and B for decode-sized
// batches (k_ad_skinny).
//
// Both put the long matrix on the M side of the MMA (128 of its columns, or
// of the stacked adapters' rank columns, fill the 128 TMEM lanes) and up to
// 128 rows of x on the N side, so that a batch of one row costs a 16-column
// MMA and the kernel is a stream of W (bytes bound).  K is split over a
// cluster of up to 8 blocks so that a narrow W still reaches most SMs; the
// partial tiles are added up in rank order through distributed shared memory,
// so results do not depend on timing.
//
// k_ad_skinny is launched as a programmatic dependent of k_ad_shrink: it
// streams W while x.A is still being made and waits for it (griddepcontrol)
// only before the extension blocks.
#include <cooperative_groups.h>
#include <cuda.h>

#include <mutex>

#include "adapter_mma.cuh"

namespace latent {

namespace {

namespace cg = cooperative_groups;
using namespace adapter;

constexpr int kThreads = 256;  // warp 0: TMA, 1: MMA, 2: TMEM, 4..7: rows (segments, x.A parts, epilogue)
constexpr int kMaxStages = 10;

struct Shared {
    uint64_t full[kMaxStages], empty[kMaxStages];
    uint64_t acc, t_full[2], t_empty[2];
    uint32_t tmem;
    volatile int abort;
    uint8_t wide[kRows];   // fp16: rows finished in fp32
    Segments seg;
};

struct Plan {
    int rows;       // N of the MMA: rows of x per tile, a multiple of 16
    int stages;
    int cluster;
    int parts;
    int chunk;      // blocks per accumulator
    uint32_t cols;  // TMEM columns
    size_t smem;
};

__device__ __forceinline__ uint8_t *align1024(uint8_t *p) {
    return reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(p) + 1023) & ~uintptr_t(1023));
}

__device__ __forceinline__ void give_up(Shared &sh, uint32_t *err) {
    atomicOr(err, kErrTimeout);
    sh.abort = 1;
}

// The loads of the last stages issued must land before the block exits.
__device__ __forceinline__ void drain(Shared &sh, int issued, int stages) {
    for (int j = 0; j < stages && j < issued; ++j) {
        const int i = issued - 1 - j;
        mbar_wait(sh.full + i % stages, (uint32_t)(i / stages) & 1u);
    }
}

__device__ __forceinline__ void setup(Shared &sh, int stages, uint32_t cols, int builders) {
    if (threadIdx.x == 0) {
        for (int s = 0; s < stages; ++s) {
            mbar_init(sh.full + s, 1);
            mbar_init(sh.empty + s, 1);
        }
        mbar_init(&sh.acc, 1);
        for (int b = 0; b < 2; ++b) {
            mbar_init(sh.t_full + b, builders);
            mbar_init(sh.t_empty + b, 1);
        }
        sh.abort = 0;
        fence_barrier_init();
    }
    if (threadIdx.x / 32 == 2) {
        tmem_alloc(&sh.tmem, cols);
        tmem_relinquish();
    }
}

// This block's accumulator (lane = M row, column = row of x) as part[row][128].
__device__ __forceinline__ void store_partial(float *part, uint32_t tmem, int rows, int groups, int tid) {
    for (int c = 0; c < rows; c += 32) {  // columns behind `rows` inside the last 32 are allocated and dropped
        float s[32];
        for (int g = 0; g < groups; ++g) {
            uint32_t v[32];
            tmem_ld32(tmem + ((uint32_t)(tid & ~31) << 16) + (uint32_t)(g * rows + c), v);
            tmem_ld_wait();
#pragma unroll
            for (int j = 0; j < 32; ++j) s[j] = g ? s[j] + __uint_as_float(v[j]) : __uint_as_float(v[j]);
        }
#pragma unroll
        for (int j = 0; j < 32; ++j)
            if (c + j < rows) part[(c + j) * 128 + tid] = s[j];
    }
}

// x.A.  Block (cluster rank, slot, row tile); the stacked rank columns of the
// tile's adapters in tiles of 128, slot, slot + gridDim.y, ...
template <bool BF>
__global__ void __launch_bounds__(kThreads, 1) k_ad_shrink(const __grid_constant__ CUtensorMap mA,
                                                           const __grid_constant__ CUtensorMap mX, AdapterArgs g,
                                                           Plan p) {
    extern __shared__ uint8_t raw[];
    uint8_t *ring = align1024(raw);
    const uint32_t stage = 16384u + (uint32_t)p.rows * 128u;
    float *part = reinterpret_cast<float *>(ring + p.stages * stage);
    __shared__ Shared sh;
    cg::cluster_group cluster = cg::this_cluster();
    const int q = blockIdx.x, CS = gridDim.x;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const latent_adapter_desc &d = g.d;
    const int t0 = blockIdx.z * g.tile_rows, nt = min(g.tile_rows, d.n_tokens - t0);
    const int rank = d.rank;
    launch_dependents();
    setup(sh, p.stages, p.cols, 1);
    if (warp >= 4) build_segments(sh.seg, d, t0, nt, threadIdx.x - 128, 1, q == 0 && blockIdx.y == 0);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sh.tmem;
    const int nk = (d.n_in + kBK - 1) / kBK;
    const int k0 = (int)((int64_t)nk * q / CS), k1 = (int)((int64_t)nk * (q + 1) / CS);
    const int total = sh.seg.n * rank;  // stacked rank columns
    int it = 0;                         // stages issued or used by this role
    uint32_t tile = 0;
    for (int m = blockIdx.y * 128; m < total; m += gridDim.y * 128, ++tile) {
        if (warp == 0 && lane == 0 && !sh.abort) {
            const int boxes = min(8, (total - m) / 16);
            bool ok = true;
            for (int k = k0; k < k1; ++k, ++it) {
                const int s = it % p.stages;
                if (it >= p.stages && !mbar_wait(sh.empty + s, (uint32_t)(it / p.stages - 1) & 1u)) { ok = false; break; }
                if (sh.abort) { ok = false; break; }
                uint8_t *st = ring + s * stage;
                mbar_arrive_expect_tx(sh.full + s, (uint32_t)boxes * 2048u + (uint32_t)p.rows * 128u);
                for (int i = 0; i < boxes; ++i) {
                    const int r = m + 16 * i;
                    tma_load_2d(st + i * 2048, &mA, k * kBK, sh.seg.id[r / rank] * rank + r % rank, sh.full + s);
                }
                tma_load_2d(st + 16384, &mX, k * kBK, t0, sh.full + s);
            }
            if (!ok) {
                give_up(sh, d.err);
                drain(sh, it, p.stages);
            }
        } else if (warp == 1 && lane == 0 && !sh.abort) {
            const uint32_t id = idesc(BF, p.rows, false, false);
            bool ok = true;
            for (int k = k0; k < k1; ++k, ++it) {
                const int s = it % p.stages;
                if (!mbar_wait(sh.full + s, (uint32_t)(it / p.stages) & 1u) || sh.abort) { ok = false; break; }
                tc_fence_after();
                const uint32_t a = smem_addr(ring + s * stage), x = a + 16384u;
#pragma unroll
                for (int kk = 0; kk < 4; ++kk)
                    mma_f16(tmem, desc_kmajor_sw128(a + kk * 32), desc_kmajor_sw128(x + kk * 32), id, (k > k0) | kk);
                mma_commit(sh.empty + s);
            }
            if (!ok) give_up(sh, d.err);
            mma_commit(&sh.acc);
        } else if (warp >= 4 && !sh.abort) {
            if (!mbar_wait(&sh.acc, tile & 1u)) give_up(sh, d.err);
            tc_fence_after();
            store_partial(part, tmem, p.rows, 1, threadIdx.x - 128);
            tc_fence_before();
        }
        __syncwarp();
        cluster.sync();
        // this block's share of the rows: t[row][j] = scale * sum over the cluster, in rank order
        const int per = (nt + CS - 1) / CS;
        const int r0 = q * per, r1 = min(nt, r0 + per);
        for (int i = threadIdx.x; i < (r1 - r0) * rank; i += kThreads) {
            const int r = r0 + i / rank, j = i % rank;
            const int s = sh.seg.row[r];
            const int at = s * rank + j - m;
            if (s < 0 || at < 0 || at >= 128) continue;
            float v = 0.f;
            for (int c = 0; c < CS; ++c) v += cluster.map_shared_rank(part, c)[r * 128 + at];
            g.t[(int64_t)(t0 + r) * rank + j] = v * __ldg(d.scale + sh.seg.id[s]);
        }
        __syncwarp();
        cluster.sync();
        tc_fence_after();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 2) tmem_dealloc(tmem, p.cols);
}

// The product.  Block (cluster rank, 128 output columns, row tile).
template <bool BF, bool KN, int PARTS, typename Y>
__global__ void __launch_bounds__(kThreads, 1) k_ad_skinny(const __grid_constant__ CUtensorMap mW,
                                                           const __grid_constant__ CUtensorMap mB,
                                                           const __grid_constant__ CUtensorMap mX, AdapterArgs g,
                                                           Plan p) {
    extern __shared__ uint8_t raw[];
    uint8_t *ring = align1024(raw);
    const uint32_t xbytes = (uint32_t)p.rows * 128u, stage = 16384u + xbytes;
    uint8_t *tbuf = ring + p.stages * stage;              // 2 x PARTS x [rows][128 bytes]
    float *part = reinterpret_cast<float *>(ring);        // after the last MMA
    __shared__ Shared sh;
    cg::cluster_group cluster = cg::this_cluster();
    const int q = blockIdx.x, CS = gridDim.x;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const latent_adapter_desc &d = g.d;
    const int n0 = blockIdx.y * 128, t0 = blockIdx.z * g.tile_rows, nt = min(g.tile_rows, d.n_tokens - t0);
    const int rank = d.rank;
    setup(sh, p.stages, p.cols, 128);
    if (warp >= 4) build_segments(sh.seg, d, t0, nt, threadIdx.x - 128, 1, false);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sh.tmem;
    const int nk = (d.n_in + kBK - 1) / kBK;
    const int k0 = (int)((int64_t)nk * q / CS), k1 = (int)((int64_t)nk * (q + 1) / CS);
    const int ext = sh.seg.n * rank, ne = (ext + kBK - 1) / kBK;
    const int e0 = (int)((int64_t)ne * q / CS), e1 = (int)((int64_t)ne * (q + 1) / CS);
    const int groups = (k1 - k0 + p.chunk - 1) / p.chunk;  // accumulators; the extension goes to the last
    if (warp == 0 && lane == 0) {
        int it = 0;
        bool ok = true;
        for (int k = k0; k < k1 + (e1 - e0); ++k, ++it) {
            const int s = it % p.stages;
            if (it >= p.stages && !mbar_wait(sh.empty + s, (uint32_t)(it / p.stages - 1) & 1u)) { ok = false; break; }
            if (sh.abort) { ok = false; break; }
            uint8_t *st = ring + s * stage;
            if (k < k1) {
                mbar_arrive_expect_tx(sh.full + s, stage);
                if (KN) {
                    tma_load_2d(st, &mW, n0, k * kBK, sh.full + s);
                    tma_load_2d(st + 8192, &mW, n0 + 64, k * kBK, sh.full + s);
                } else {
                    tma_load_2d(st, &mW, k * kBK, n0, sh.full + s);
                }
                tma_load_2d(st + 16384, &mX, k * kBK, t0, sh.full + s);
            } else {
                const int r0 = (e0 + k - k1) * kBK, boxes = min(4, (ext - r0) / 16);
                mbar_arrive_expect_tx(sh.full + s, (uint32_t)boxes * 4096u);
                for (int i = 0; i < boxes; ++i) {
                    const int r = r0 + 16 * i, row = sh.seg.id[r / rank] * rank + r % rank;
                    tma_load_2d(st + i * 2048, &mB, n0, row, sh.full + s);
                    tma_load_2d(st + 8192 + i * 2048, &mB, n0 + 64, row, sh.full + s);
                }
            }
        }
        if (!ok) {
            give_up(sh, d.err);
            drain(sh, it, p.stages);
        }
    } else if (warp == 1 && lane == 0) {
        const uint32_t id = idesc(BF, p.rows, KN, false), idx = idesc(BF, p.rows, true, false);
        int it = 0;
        bool ok = true;
        for (int k = k0; k < k1; ++k, ++it) {
            const int s = it % p.stages;
            if (!mbar_wait(sh.full + s, (uint32_t)(it / p.stages) & 1u) || sh.abort) { ok = false; break; }
            tc_fence_after();
            const uint32_t a = smem_addr(ring + s * stage), x = a + 16384u;
            const int grp = (k - k0) / p.chunk, first = grp * p.chunk + k0;
#pragma unroll
            for (int kk = 0; kk < 4; ++kk)
                mma_f16(tmem + (uint32_t)(grp * p.rows), KN ? desc_mnmajor_sw128(a + kk * 2048) : desc_kmajor_sw128(a + kk * 32),
                        desc_kmajor_sw128(x + kk * 32), id, (k > first) | kk);
            mma_commit(sh.empty + s);
        }
        for (int e = e0; ok && e < e1; ++e, ++it) {
            const int s = it % p.stages, b = (e - e0) & 1;
            if (!mbar_wait(sh.full + s, (uint32_t)(it / p.stages) & 1u) ||
                !mbar_wait(sh.t_full + b, (uint32_t)((e - e0) >> 1) & 1u) || sh.abort) { ok = false; break; }
            tc_fence_after();
            const uint32_t a = smem_addr(ring + s * stage), t = smem_addr(tbuf) + (uint32_t)(b * PARTS) * xbytes;
            const int steps = min(4, (ext - e * kBK) / 16);
            for (int kk = 0; kk < steps; ++kk)
#pragma unroll
                for (int w = 0; w < PARTS; ++w)
                    mma_f16(tmem + (uint32_t)((groups - 1) * p.rows), desc_mnmajor_sw128(a + kk * 2048),
                            desc_kmajor_sw128(t + w * xbytes + kk * 32), idx, 1);
            mma_commit(sh.empty + s);
            mma_commit(sh.t_empty + b);
        }
        if (!ok) give_up(sh, d.err);
        mma_commit(&sh.acc);
    } else if (warp >= 4) {
        const int r = threadIdx.x - 128;
        const int seg = sh.seg.row[r];
        const float *t = g.t + (int64_t)(t0 + r) * rank;
        dependency_wait();
        const bool wide = !BF && seg >= 0 && beyond_f16(t, rank);
        sh.wide[r] = wide;
        bool ok = true;
        for (int e = e0; e < e1; ++e) {
            const int b = (e - e0) & 1;
            if (e - e0 >= 2 && !mbar_wait(sh.t_empty + b, (uint32_t)((e - e0) / 2 - 1) & 1u)) { ok = false; break; }
            if (sh.abort) { ok = false; break; }
            if (r < p.rows) build_t_row<BF, PARTS, 8>(tbuf + (uint32_t)(b * PARTS) * xbytes, xbytes, r, wide ? -1 : seg, rank, t, e * kBK);
            fence_async_shared();
            mbar_arrive(sh.t_full + b);
        }
        if (!ok || !mbar_wait(&sh.acc, 0u)) give_up(sh, d.err);
        tc_fence_after();
        store_partial(part, tmem, p.rows, groups, r);
        tc_fence_before();
    }
    __syncwarp();
    cluster.sync();
    // this block's share of the rows, two columns per thread: the cluster's partial tiles in rank order
    const int per = (nt + CS - 1) / CS;
    const int r0 = q * per, r1 = min(nt, r0 + per);
    const int n = n0 + 2 * (threadIdx.x & 63);
    for (int r = r0 + (threadIdx.x >> 6); r < r1; r += kThreads / 64) {
        float2 v = make_float2(0.f, 0.f);
        for (int c = 0; c < CS; ++c) {
            const float2 u = *reinterpret_cast<const float2 *>(cluster.map_shared_rank(part, c) + r * 128 + 2 * (threadIdx.x & 63));
            v.x += u.x;
            v.y += u.y;
        }
        if (n >= d.n_out) continue;
        if (!BF && sh.wide[r]) {
            const float *t = g.t + (int64_t)(t0 + r) * rank;
            const int a = sh.seg.id[sh.seg.row[r]];
            v.x += adapter_dot<BF>(d, t, a, n);
            v.y += adapter_dot<BF>(d, t, a, n + 1);
        }
        if constexpr (sizeof(Y) == 4)
            *reinterpret_cast<float2 *>(static_cast<float *>(d.y) + (int64_t)(t0 + r) * d.ldy + n) = v;
        else
            *reinterpret_cast<uint32_t *>(static_cast<Y *>(d.y) + (int64_t)(t0 + r) * d.ldy + n) = pack2<BF>(v.x, v.y);
    }
    __syncwarp();
    cluster.sync();  // the others' partial tiles stay until every block has read them
    tc_fence_after();
    if (warp == 2) tmem_dealloc(tmem, p.cols);
}

typedef CUresult (*EncodeTiledFn)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *,
                                  const cuuint64_t *, const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn encode_fn() {
    static EncodeTiledFn fn = nullptr;
    static std::once_flag once;
    std::call_once(once, [] {
        void *p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
            q == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<EncodeTiledFn>(p);
    });
    return fn;
}

uint32_t tmem_cols(int n) {
    uint32_t c = 32;
    while ((int)c < n) c *= 2;
    return c;
}

constexpr size_t kSmemLimit = 220 * 1024;  // dynamic; the static part holds Shared

cudaError_t launch_cluster(const void *fn, dim3 grid, size_t smem, int cluster, bool dependent, void **args,
                           cudaStream_t s) {
    cudaError_t err = ensure_smem(fn, smem);
    if (err != cudaSuccess) return err;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = (unsigned)cluster;
    at[0].val.clusterDim.y = 1;
    at[0].val.clusterDim.z = 1;
    at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = dependent ? 2 : 1;
    return cudaLaunchKernelExC(&cfg, fn, args);
}

// Blocks of a cluster: as many of 8, 4, 2, 1 as the contraction has blocks for
// and the SMs have room for beside the other clusters.
int pick_cluster(int64_t others, int blocks, int sms) {
    int c = 8;
    while (c > 1 && (c > blocks || others * c > sms)) c /= 2;
    return c;
}

template <typename Y>
const void *skinny_fn(bool bf, bool kn, int parts) {
    if (bf) {
        if (parts == 3) return kn ? (const void *)k_ad_skinny<true, true, 3, Y> : (const void *)k_ad_skinny<true, false, 3, Y>;
        return kn ? (const void *)k_ad_skinny<true, true, 2, Y> : (const void *)k_ad_skinny<true, false, 2, Y>;
    }
    return kn ? (const void *)k_ad_skinny<false, true, 2, Y> : (const void *)k_ad_skinny<false, false, 2, Y>;
}

}  // namespace

bool adapter_map(void *map, bool bf16, const void *base, uint64_t rows, uint64_t cols, uint64_t ld, uint32_t box_rows) {
    EncodeTiledFn fn = encode_fn();
    if (!fn) return false;
    cuuint64_t dims[2] = {cols, rows};
    cuuint64_t strides[1] = {ld * 2};
    cuuint32_t box[2] = {(cuuint32_t)adapter::kBK, box_rows};
    cuuint32_t es[2] = {1, 1};
    return fn(static_cast<CUtensorMap *>(map), bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
              2, const_cast<void *>(base), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) ==
           CUDA_SUCCESS;
}

cudaError_t launch_adapter_shrink(const AdapterArgs &g, int sms, cudaStream_t s) {
    const latent_adapter_desc &d = g.d;
    const bool bf = d.type == LATENT_TYPE_BF16;
    const int tiles = (d.n_tokens + g.tile_rows - 1) / g.tile_rows;
    const int most = ((d.n_adapter < g.tile_rows ? d.n_adapter : g.tile_rows) * d.rank + 127) / 128;
    const int nk = (d.n_in + kBK - 1) / kBK;
    Plan p{};
    p.rows = (g.tile_rows + 15) / 16 * 16;
    const size_t part = (size_t)p.rows * 512, stage = 16384 + (size_t)p.rows * 128;
    p.cluster = pick_cluster(tiles, nk, sms);
    int slots = sms / (tiles * p.cluster);  // tiles of stacked rank columns side by side
    slots = slots < 1 ? 1 : slots > most ? most : slots;
    const int per = (nk + p.cluster - 1) / p.cluster;
    p.stages = (int)((kSmemLimit - 1024 - part) / stage);
    if (p.stages > kMaxStages) p.stages = kMaxStages;
    if (p.stages > per) p.stages = per;
    p.cols = tmem_cols(p.rows);
    p.smem = 1024 + p.stages * stage + part;
    CUtensorMap mA, mX;
    if (!adapter_map(&mA, bf, d.a, (uint64_t)d.n_adapter * d.rank, d.n_in, d.lda, 16) ||
        !adapter_map(&mX, bf, d.x, d.n_tokens, d.n_in, d.ldx, p.rows))
        return cudaErrorInvalidValue;
    AdapterArgs a = g;
    void *args[] = {&mA, &mX, &a, &p};
    return launch_cluster(bf ? (const void *)k_ad_shrink<true> : (const void *)k_ad_shrink<false>,
                          dim3(p.cluster, slots, tiles), p.smem, p.cluster, false, args, s);
}

cudaError_t launch_adapter_skinny(const AdapterArgs &g, int sms, cudaStream_t s) {
    const latent_adapter_desc &d = g.d;
    const bool bf = d.type == LATENT_TYPE_BF16, kn = !(d.flags & LATENT_ADAPTER_W_TRANSPOSED);
    const bool f32 = d.y_type == LATENT_TYPE_F32;
    const int tiles = (d.n_tokens + g.tile_rows - 1) / g.tile_rows, ntn = (d.n_out + 127) / 128;
    const int nk = (d.n_in + kBK - 1) / kBK;
    Plan p{};
    p.rows = (g.tile_rows + 15) / 16 * 16;
    p.parts = bf && f32 ? 3 : 2;
    p.cluster = pick_cluster((int64_t)tiles * ntn, nk, sms);
    // The tensor cores cut a sum off instead of rounding it: a chain over K
    // = 7168 is off by 8e-6 of the result, one over 512 by 5e-7 (measured).
    // fp32 results therefore use an accumulator per 512 of K, added up in
    // fp32, as far as the 512 TMEM columns go, and clusters long enough.
    const int read = (p.rows + 31) / 32 * 32;  // columns the epilogue reads of an accumulator
    const int groups = (512 - read) / p.rows + 1;
    if (f32)
        while (p.cluster < 8 && p.cluster < nk && (nk + p.cluster - 1) / p.cluster > 8 * groups) p.cluster *= 2;
    const int per = (nk + p.cluster - 1) / p.cluster;
    p.chunk = per;
    if (f32) p.chunk = per <= 8 * groups ? 8 : (per + groups - 1) / groups;
    const int used = (per + p.chunk - 1) / p.chunk;
    p.cols = tmem_cols((used - 1) * p.rows + read);
    const size_t stage = 16384 + (size_t)p.rows * 128, tb = 2 * (size_t)p.parts * p.rows * 128;
    p.stages = (int)((kSmemLimit - 1024 - tb) / stage);
    if (p.stages > kMaxStages) p.stages = kMaxStages;
    const int least = (int)(((size_t)p.rows * 512 + stage - 1) / stage);  // the partial tile lies in the ring
    if (p.stages > per + 4) p.stages = per + 4;
    if (p.stages < least) p.stages = least;
    p.smem = 1024 + p.stages * stage + tb;
    CUtensorMap mW, mB, mX;
    if (!(kn ? adapter_map(&mW, bf, d.w, d.n_in, d.n_out, d.ldw, kBK) : adapter_map(&mW, bf, d.w, d.n_out, d.n_in, d.ldw, 128)) ||
        !adapter_map(&mB, bf, d.b, (uint64_t)d.n_adapter * d.rank, d.n_out, d.ldb, 16) ||
        !adapter_map(&mX, bf, d.x, d.n_tokens, d.n_in, d.ldx, p.rows))
        return cudaErrorInvalidValue;
    const void *fn = f32 ? skinny_fn<float>(bf, kn, p.parts)
                         : bf ? skinny_fn<__nv_bfloat16>(bf, kn, p.parts) : skinny_fn<__half>(bf, kn, p.parts);
    AdapterArgs a = g;
    void *args[] = {&mW, &mB, &mX, &a, &p};
    return launch_cluster(fn, dim3(p.cluster, ntn, tiles), p.smem, p.cluster, true, args, s);
}

}  // namespace latent
