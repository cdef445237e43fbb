// Tensor-core kernels of the adapters for few rows: x.A of a tile of rows
// (any batch; k_ad_shrink) and the product with W and B for decode-sized
// batches (k_ad_skinny).
//
// Both put the long matrix on the M side of the MMA (128 of its columns, or
// of the stacked adapters' rank columns, fill the 128 TMEM lanes) and up to
// 128 rows of x on the N side, so that a batch of one row costs a 16-column
// MMA and the kernel is a stream of W (bytes bound).  K is split over a
// cluster of up to 16 blocks so that a narrow W still reaches most SMs; the
// partial tiles are added up in rank order through distributed shared memory,
// so results do not depend on timing.
//
// k_ad_skinny is launched as a programmatic dependent of k_ad_shrink (unless it
// makes x.A itself): on the SMs that the shrink leaves it streams W while x.A is
// still being made, and it waits for x.A (griddepcontrol) only before the
// extension blocks.
#include <cuda.h>

#include <mutex>
#include <set>
#include <utility>

#include "adapter_mma.cuh"

namespace latent {

namespace {

using namespace adapter;

constexpr int kThreads = 256;  // warp 0: TMA, 1: MMA, 2: TMEM, 4..7: rows (segments, x.A parts, epilogue)
constexpr int kMaxStages = 12;
constexpr int kMaxTBufs = 4;

struct Shared {
    uint64_t full[kMaxStages], empty[kMaxStages];
    uint64_t acc_full[2], acc_empty[2], t_full[kMaxTBufs], t_empty[kMaxTBufs], seg;
    uint32_t tmem;
    volatile int abort;
    Segments segs;
    alignas(16) float down[kRows];     // fp16: RowScale's, of the rows' t
    alignas(16) uint32_t dest[kRows];  // where a row's sums go: its owner's shared memory, kNoRow behind the last row
};
constexpr uint32_t kNoRow = 0xffffffffu;

struct Plan {
    int rows;       // N of the MMA: rows of x per tile, a multiple of 16
    int stages;
    int chunk;      // blocks per accumulator (k_ad_skinny)
    int tbufs;      // tiles of x.A parts
    int next_col;   // the accumulator behind the product's: x.A's (SELF), else in fp16 the adapters' part's
    uint32_t cols;  // TMEM columns
};

__device__ __forceinline__ uint8_t *align1024(uint8_t *p) {
    return reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(p) + 1023) & ~uintptr_t(1023));
}

__device__ __forceinline__ void give_up(Shared &sh, uint32_t *err) {
    atomicOr(err, kErrTimeout);
    sh.abort = 1;
}

// After a failure: the loads in flight land well within 20 ms.
__device__ __forceinline__ void drain() {
    const unsigned long long t0 = global_ns();
    while (global_ns() - t0 < 20000000ull) __nanosleep(1000);
}

// Barriers by warp 0, which goes on at once (its first loads wait for nobody),
// TMEM by warp 2, which then lets a dependent kernel start.
template <bool DEPENDENTS>
__device__ __forceinline__ void setup(Shared &sh, const Plan &p, int warp, int lane) {
    if (warp == 0) {
        if (lane == 0) {
            for (int s = 0; s < p.stages; ++s) {
                mbar_init(sh.full + s, 1);
                mbar_init(sh.empty + s, 1);
            }
            for (int b = 0; b < 2; ++b) {
                mbar_init(sh.acc_full + b, 1);
                mbar_init(sh.acc_empty + b, 128);
            }
            for (int b = 0; b < kMaxTBufs; ++b) {
                mbar_init(sh.t_full + b, 4);  // the builders' warps
                mbar_init(sh.t_empty + b, 1);
            }
            mbar_init(&sh.seg, 128);
            sh.abort = 0;
            fence_barrier_init();
        }
        __syncwarp();
        asm volatile("bar.arrive 3, 256;" ::: "memory");
        return;
    }
    if (warp == 2) {
        tmem_alloc(&sh.tmem, p.cols);
        tmem_relinquish();
        if (DEPENDENTS) launch_dependents();
    }
    tc_fence_before();
    bar_sync(3, kThreads);
    tc_fence_after();
}

__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire;" ::: "memory"); }
__device__ __forceinline__ uint32_t map_rank(uint32_t addr, int rank) {
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
__device__ __forceinline__ void st_cluster(uint32_t addr, float v) {
    asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(addr), "f"(v) : "memory");
}

template <int N>
__device__ __forceinline__ void load_words(const void *p, uint32_t (&v)[N]) {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
        const uint4 u = reinterpret_cast<const uint4 *>(p)[i / 4];
        v[i] = u.x;
        v[i + 1] = u.y;
        v[i + 2] = u.z;
        v[i + 3] = u.w;
    }
}

// By the thread of row r: rows are dealt to the cluster in runs of `per`; rank
// q's sums of a row (row_bytes) lie at place q * per + r % per of its owner.
__device__ __forceinline__ void set_dest(Shared &sh, const float *recv, int r, int nt, int per, int q, uint32_t row_bytes) {
    sh.dest[r] = r < nt ? map_rank(smem_addr(recv) + (uint32_t)(q * per + r % per) * row_bytes, r / per) : kNoRow;
}

// By the load warp: the K blocks [k0, k1) of stacked rank columns m .. m + 127 (rows of A) and of x.
__device__ __forceinline__ bool load_stacked(Shared &sh, const Plan &p, Ring &at, uint8_t *ring, uint32_t stage,
                                             const CUtensorMap *mA, const CUtensorMap *mX, int m, int total, int k0,
                                             int k1, int t0, int rank, int log2r) {
    const int cols = min(128, total - m), boxes = cols >> log2r, lane = threadIdx.x & 31;
    const int row = lane < boxes ? sh.segs.id[(m >> log2r) + lane] << log2r : 0;  // of the lane-th adapter
    int rows[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) rows[i] = __shfl_sync(kAll, row, i);
    for (int k = k0; k < k1; ++k, at.next(p.stages)) {
        if (at.wrapped && !wait_warp(sh.empty + at.s, at.phase ^ 1u, &sh.abort)) return false;
        if (elect()) {
            uint8_t *st = ring + at.s * stage;
            mbar_arrive_expect_tx(sh.full + at.s, (uint32_t)(cols + p.rows) * 128u);
            tma_load_2d(st + 16384, mX, k * kBK, t0, sh.full + at.s);
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (i < boxes) tma_load_2d(st + ((uint32_t)i << log2r) * 128u, mA, k * kBK, rows[i], sh.full + at.s);
        }
    }
    return true;
}

// By the MMA warp: their product into acc.
__device__ __forceinline__ bool multiply_stacked(Shared &sh, const Plan &p, Ring &at, uint8_t *ring, uint32_t stage,
                                                 uint32_t acc, uint32_t id, int k0, int k1) {
    for (int k = k0; k < k1; ++k, at.next(p.stages)) {
        if (!wait_warp(sh.full + at.s, at.phase, &sh.abort)) return false;
        tc_fence_after();
        if (elect()) {
            const uint32_t w = smem_addr(ring + at.s * stage), x = w + 16384u;
#pragma unroll
            for (int kk = 0; kk < 4; ++kk)
                mma_f16(acc, desc_kmajor_sw128(w + kk * 32), desc_kmajor_sw128(x + kk * 32), id, (k > k0) | kk);
            mma_commit(sh.empty + at.s);
        }
    }
    return true;
}

// By the epilogue warps: x.A of the tile at stacked column m (acc: lane = stacked column, column = row of x) to the
// rows' owners, `off` bytes into a row's place.
__device__ __forceinline__ void send_stacked(const Shared &sh, const Plan &p, uint32_t acc, int m, int rank, int log2r,
                                             int tid, uint32_t off) {
    const int seg = (m + tid) >> log2r;
    off += ((uint32_t)(m + tid) & (uint32_t)(rank - 1)) * 4u;
    for (int c = 0; c < p.rows; c += 32) {
        uint32_t v[32], to[32], of[32];
        __syncwarp();
        tmem_ld32(acc + ((uint32_t)(tid & ~31) << 16) + (uint32_t)c, v);
        load_words(sh.dest + c, to);
        load_words(sh.segs.row + c, of);
        tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 32; ++i)
            if ((int)of[i] == seg) st_cluster(to[i] + off, __uint_as_float(v[i]));
    }
}

// The same of several accumulators: each into the sums, then these to the owners.
__device__ __forceinline__ void add_stacked(const Plan &p, uint32_t acc, int tid, float (&sums)[kRows]) {
#pragma unroll
    for (int c = 0; c < kRows; c += 16) {
        if (c >= p.rows) break;
        uint32_t v[16];
        __syncwarp();
        tmem_ld16(acc + ((uint32_t)(tid & ~31) << 16) + (uint32_t)c, v);
        tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 16; ++i) sums[c + i] += __uint_as_float(v[i]);
    }
}
__device__ __forceinline__ void send_sums(const Shared &sh, const Plan &p, const float (&sums)[kRows], int m, int rank,
                                          int log2r, int tid) {
    const int seg = (m + tid) >> log2r;
    const uint32_t off = ((uint32_t)(m + tid) & (uint32_t)(rank - 1)) * 4u;
#pragma unroll
    for (int c = 0; c < kRows; c += 16) {
        if (c >= p.rows) break;
        uint32_t to[16], of[16];
        load_words(sh.dest + c, to);
        load_words(sh.segs.row + c, of);
#pragma unroll
        for (int i = 0; i < 16; ++i)
            if ((int)of[i] == seg) st_cluster(to[i] + off, sums[c + i]);
    }
}

// x.A.  Block (cluster rank, slot, row tile); the stacked rank columns of the
// tile's adapters in tiles of 128: slot, slot + gridDim.y, ...  Rank q of the
// cluster sums K blocks of its share; every block sends the t of a row to the
// row's owner (rows are dealt to the cluster in runs), which adds them up in
// rank order.
// Measured: 64 rows of K = 7168 with 24 adapters of rank 64 10.4 us (22 MB of A,
// 2.2 TB/s); 2047 rows of K = 4096 with one adapter of rank 64 11.5 us, without
// any 4.8 (start, adapter list, the cluster's barriers): in between the blocks
// fetch 27 MB of x and A, 4 TB/s.
// For fp32 results a block with more than 512 of K has its two accumulators take
// turns every 512, as the products do, and the epilogue keeps their sums in
// registers: over K = 7168 x.A is then off by 4.8e-7 (fp16 6.5e-7) instead of
// 7.9e-6, at 131.1 us instead of 130.5 for 18900 rows with N = 256, 45.6 for
// 44.0 for 8192 rows of 4096 x 256, nothing for decode batches.  16-bit results
// keep one chain: x.A enters them in two parts, to 2^-16.
template <bool BF, bool F32>
__global__ void __launch_bounds__(kThreads, 1) k_ad_shrink(const __grid_constant__ CUtensorMap mA,
                                                           const __grid_constant__ CUtensorMap mX, AdapterArgs g,
                                                           Plan p) {
    extern __shared__ uint8_t raw[];
    uint8_t *ring = align1024(raw);
    const uint32_t stage = 16384u + (uint32_t)p.rows * 128u;
    float *recv = reinterpret_cast<float *>(ring + p.stages * stage);  // [cluster][rows of a rank][rank]
    __shared__ Shared sh;
    const int q = blockIdx.x, CS = gridDim.x;
    const int warp = warp_index(), lane = threadIdx.x & 31;
    const latent_adapter_desc &d = g.d;
    const int t0 = blockIdx.z * g.tile_rows, nt = min(g.tile_rows, d.n_tokens - t0);
    const int rank = d.rank, log2r = g.log2r;
    cluster_arrive();  // the others may send once every block has started
    int a = -1;
    if (warp == 0 && lane == 0) {
        prefetch_tensormap(&mA);
        prefetch_tensormap(&mX);
    } else if (warp >= 4) {
        const int r = threadIdx.x - 128;
        a = row_adapter(d, t0 + r, r < nt, q == 0 && blockIdx.y == 0);
    }
    setup<true>(sh, p, warp, lane);
    const uint32_t tmem = warp ? (uint32_t)uniform((int)sh.tmem) : 0u, read = (uint32_t)(p.rows + 31) & ~31u;
    const int nk = (d.n_in + kBK - 1) / kBK;
    const int k0 = (int)((int64_t)nk * q / CS), k1 = (int)((int64_t)nk * (q + 1) / CS);
    const int per = (nt + CS - 1) / CS;  // rows of an owner
    const int chunk = F32 ? 8 : max(1, k1 - k0);  // K blocks per accumulator
    bool ok = true;
    if (warp >= 4) {
        build_segments(sh.segs, a, nt, threadIdx.x - 128, 1);
        set_dest(sh, recv, threadIdx.x - 128, nt, per, q, (uint32_t)rank * 4u);
        mbar_arrive(&sh.seg);
    }
    ok = wait_warp(&sh.seg, 0u, &sh.abort);
    const int total = ok ? uniform(sh.segs.n) * rank : 0;  // stacked rank columns
    if (warp == 0) {
        Ring at;
        for (int m = blockIdx.y * 128; m < total && ok; m += gridDim.y * 128)
            ok = load_stacked(sh, p, at, ring, stage, &mA, &mX, m, total, k0, k1, t0, rank, log2r);
        if (ok) ok = ring_drained(at, sh.empty, p.stages, &sh.abort);
    } else if (warp == 1) {
        const uint32_t id = idesc(BF, p.rows, false, false);
        Ring at;
        uint32_t n = 0;
        for (int m = blockIdx.y * 128; m < total && ok; m += gridDim.y * 128)
            for (int k = k0; k < k1 && ok; k += chunk, ++n) {
                const uint32_t b = n & 1u;
                if (n >= 2 && !wait_warp(sh.acc_empty + b, ((n >> 1) - 1u) & 1u, &sh.abort)) { ok = false; break; }
                tc_fence_after();
                ok = multiply_stacked(sh, p, at, ring, stage, tmem + b * read, id, k, min(k1, k + chunk));
                if (ok && elect()) mma_commit(sh.acc_full + b);
            }
        if (!ok && elect()) {
            mma_commit(sh.acc_full);
            mma_commit(sh.acc_full + 1);
        }
    } else if (warp >= 4) {
        const int tid = threadIdx.x - 128;
        cluster_wait();
        uint32_t n = 0;
        for (int m = blockIdx.y * 128; m < total && ok; m += gridDim.y * 128) {
            float sums[F32 ? kRows : 1] = {};
            for (int k = k0; k < k1; k += chunk, ++n) {
                const uint32_t b = n & 1u;
                if (!wait(sh.acc_full + b, (n >> 1) & 1u) || sh.abort) ok = false;
                if (__any_sync(0xffffffffu, !ok)) { ok = false; break; }
                tc_fence_after();
                const bool all = k1 - k0 <= chunk;
                if (all) send_stacked(sh, p, tmem + b * read, m, rank, log2r, tid, 0u);
                if constexpr (F32) {
                    if (!all) add_stacked(p, tmem + b * read, tid, sums);
                    if (!all && k + chunk >= k1) send_sums(sh, p, sums, m, rank, log2r, tid);
                }
                tc_fence_before();
                mbar_arrive(sh.acc_empty + b);
            }
        }
    }
    if (!ok) {
        give_up(sh, d.err);
        drain();
    }
    __syncwarp();
    if (warp < 4) cluster_wait();
    cluster_arrive();
    cluster_wait();
    // this block's rows: t[row][j] = sum over the cluster, in rank order
    const int r0 = q * per, r1 = min(nt, r0 + per);
    for (int i = threadIdx.x; i < (r1 - r0) << log2r; i += kThreads) {
        const int r = i >> log2r, s = sh.segs.row[r0 + r];
        // rows without an adapter, and rows of another slot's tiles
        if (s < 0 || ((uint32_t)(s << log2r) / 128u) % gridDim.y != blockIdx.y) continue;
        float v = 0.f;
        for (int c = 0; c < CS; ++c) v += recv[((c * per) << log2r) + i];
        g.t[((int64_t)(t0 + r0) << log2r) + i] = v;
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 2) tmem_dealloc(tmem, p.cols);
}

template <typename Y> __device__ __forceinline__ Y to_y(float v);
template <> __device__ __forceinline__ float to_y<float>(float v) { return v; }
template <> __device__ __forceinline__ __half to_y<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 to_y<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// The product.  Block (cluster rank, 128 output columns, row tile).
//
// SELF (one launch, one tile of rows): every cluster makes all of x.A itself,
// behind its W loads, and the owner of a row adds x.A.B for its 128 columns on
// the CUDA cores: no trip of x.A through global memory, at the price of every
// cluster loading the adapters' A.
//
// Measured: one row of 2048 x 2048, rank 16, SELF: 8.3 us against 1.3 for its 8.5
// MB: start, one trip to DRAM, two cluster barriers and the end of the grid are
// what is left.  64 rows of 7168 x 2048, 24 adapters of rank 64: 15.1 us for 36
// MB of W and B (2.4 TB/s; the extension blocks wait for x.A).
//
// fp16: the adapters' part has the accumulator behind x.W's (next_col), its rows
// scaled (RowScale).
template <bool BF, bool KN, int PARTS, typename Y, bool SELF>
__global__ void __launch_bounds__(kThreads, 1) k_ad_skinny(const __grid_constant__ CUtensorMap mW,
                                                           const __grid_constant__ CUtensorMap mB,
                                                           const __grid_constant__ CUtensorMap mX,
                                                           const __grid_constant__ CUtensorMap mA, AdapterArgs g,
                                                           Plan p) {
    constexpr uint32_t kTiles = (PARTS + 1) / 2;
    extern __shared__ uint8_t raw[];
    uint8_t *ring = align1024(raw);
    const uint32_t xbytes = (uint32_t)p.rows * 128u, stage = 16384u + xbytes;
    uint8_t *tbuf = ring + p.stages * stage;                                      // tbufs x kTiles x [rows][128 bytes]
    // [cluster][rows of a rank][128 sums, SELF: and those of x.A]
    float *recv = reinterpret_cast<float *>(tbuf + p.tbufs * kTiles * xbytes);
    __shared__ Shared sh;
    const int q = blockIdx.x, CS = gridDim.x;
    const int warp = warp_index(), lane = threadIdx.x & 31;
    const latent_adapter_desc &d = g.d;
    const int n0 = blockIdx.y * 128, t0 = blockIdx.z * g.tile_rows, nt = min(g.tile_rows, d.n_tokens - t0);
    const int rank = d.rank, log2r = g.log2r;
    const int pitch = SELF ? 128 + rank : 128;
    cluster_arrive();
    int a = -1;
    if (warp == 0 && lane == 0) {
        prefetch_tensormap(&mW);
        prefetch_tensormap(&mX);
        prefetch_tensormap(&mB);
        if (SELF) prefetch_tensormap(&mA);
    } else if (warp >= 4) {
        const int r = threadIdx.x - 128;
        a = row_adapter(d, t0 + r, r < nt, SELF && q == 0 && blockIdx.y == 0);
    }
    setup<false>(sh, p, warp, lane);
    const uint32_t tmem = warp ? (uint32_t)uniform((int)sh.tmem) : 0u;
    const int nk = (d.n_in + kBK - 1) / kBK;
    const int k0 = (int)((int64_t)nk * q / CS), k1 = (int)((int64_t)nk * (q + 1) / CS);
    const int per = (nt + CS - 1) / CS;  // rows of an owner
    bool ok = true;
    if (warp == 0) {
        Ring at;
        for (int k = k0; ok && k < k1; ++k, at.next(p.stages)) {
            if (at.wrapped && !wait_warp(sh.empty + at.s, at.phase ^ 1u, &sh.abort)) { ok = false; break; }
            if (elect()) {
                uint8_t *st = ring + at.s * stage;
                mbar_arrive_expect_tx(sh.full + at.s, stage);
                if (KN) {
                    tma_load_2d(st, &mW, n0, k * kBK, sh.full + at.s);
                    tma_load_2d(st + 8192, &mW, n0 + 64, k * kBK, sh.full + at.s);
                } else {
                    tma_load_2d(st, &mW, k * kBK, n0, sh.full + at.s);
                }
                tma_load_2d(st + 16384, &mX, k * kBK, t0, sh.full + at.s);
            }
        }
        if (ok) ok = wait_warp(&sh.seg, 0u, &sh.abort);
        if (SELF && ok) {
            const int total = uniform(sh.segs.n) * rank;  // 128 at most
            if (total) ok = load_stacked(sh, p, at, ring, stage, &mA, &mX, 0, total, k0, k1, t0, rank, log2r);
        }
        if (!SELF && ok) {
            const int ext = uniform(sh.segs.n) * rank, ne = (ext + kExt - 1) / kExt;
            const int e1 = (int)((int64_t)ne * (q + 1) / CS), box = min(rank, kExt);
            for (int e = (int)((int64_t)ne * q / CS); e < e1; ++e, at.next(p.stages)) {
                if (at.wrapped && !wait_warp(sh.empty + at.s, at.phase ^ 1u, &sh.abort)) { ok = false; break; }
                const int rows = min(kExt, ext - e * kExt), r = e * kExt + lane * box;  // one box of 32 rows or two of 16
                const int src = lane * box < rows ? (sh.segs.id[r >> log2r] << log2r) + (r & (rank - 1)) : 0;
                const int src0 = __shfl_sync(kAll, src, 0), src1 = __shfl_sync(kAll, src, 1);
                if (elect()) {
                    uint8_t *st = ring + at.s * stage;
                    mbar_arrive_expect_tx(sh.full + at.s, (uint32_t)rows * 256u);
                    tma_load_2d(st, &mB, n0, src0, sh.full + at.s);
                    tma_load_2d(st + 8192, &mB, n0 + 64, src0, sh.full + at.s);
                    if (box < rows) {
                        tma_load_2d(st + 2048, &mB, n0, src1, sh.full + at.s);
                        tma_load_2d(st + 8192 + 2048, &mB, n0 + 64, src1, sh.full + at.s);
                    }
                }
            }
        }
        if (ok) ok = ring_drained(at, sh.empty, p.stages, &sh.abort);
    } else if (warp == 1) {
        const uint32_t id = idesc(BF, p.rows, KN, false), idx = idesc(BF, p.rows, true, false);
        Ring at;
        int in_chunk = 0;
        uint32_t acc = tmem;
        for (int k = k0; ok && k < k1; ++k, at.next(p.stages)) {
            if (!wait_warp(sh.full + at.s, at.phase, &sh.abort)) { ok = false; break; }
            tc_fence_after();
            if (in_chunk == p.chunk) {
                in_chunk = 0;
                acc += (uint32_t)p.rows;
            }
            if (elect()) {
                const uint32_t w = smem_addr(ring + at.s * stage), x = w + 16384u;
#pragma unroll
                for (int kk = 0; kk < 4; ++kk)
                    mma_f16(acc, KN ? desc_mnmajor_sw128(w + kk * 2048) : desc_kmajor_sw128(w + kk * 32),
                            desc_kmajor_sw128(x + kk * 32), id, in_chunk | kk);
                mma_commit(sh.empty + at.s);
            }
            ++in_chunk;
        }
        if (SELF && ok && elect()) mma_commit(sh.acc_full);
        if (ok) ok = wait_warp(&sh.seg, 0u, &sh.abort);
        if (SELF && ok && uniform(sh.segs.n)) {
            ok = multiply_stacked(sh, p, at, ring, stage, tmem + (uint32_t)p.next_col, idesc(BF, p.rows, false, false), k0, k1);
            if (ok && elect()) mma_commit(sh.acc_full + 1);
        }
        if (!SELF && ok) {
            const int ext = uniform(sh.segs.n) * rank, ne = (ext + kExt - 1) / kExt;
            const int e0 = (int)((int64_t)ne * q / CS), e1 = (int)((int64_t)ne * (q + 1) / CS);
            Ring tb;
            for (int e = e0; e < e1; ++e, at.next(p.stages), tb.next(p.tbufs)) {
                if (!wait_warp(sh.full + at.s, at.phase, &sh.abort) || !wait_warp(sh.t_full + tb.s, tb.phase, &sh.abort)) {
                    ok = false;
                    break;
                }
                tc_fence_after();
                if (elect()) {
                    const uint32_t w = smem_addr(ring + at.s * stage), t = smem_addr(tbuf) + (uint32_t)tb.s * kTiles * xbytes;
                    const int steps = min(kExt / 16, (ext - e * kExt) / 16);
                    const uint32_t to = BF ? acc : tmem + (uint32_t)p.next_col, more = BF || e > e0;
                    for (int kk = 0; kk < steps; ++kk)
#pragma unroll
                        for (int w2 = 0; w2 < PARTS; ++w2)
                            mma_f16(to, desc_mnmajor_sw128(w + kk * 2048), desc_kmajor_sw128(t + t_offset(w2, kk, xbytes)),
                                    idx, more | kk | w2);
                    mma_commit(sh.empty + at.s);
                    mma_commit(sh.t_empty + tb.s);
                }
            }
        }
        if (elect()) {
            if (!ok && SELF) mma_commit(sh.acc_full + 1);
            if (!SELF || !ok) mma_commit(sh.acc_full);
        }
    } else if (warp >= 4) {
        const int r = threadIdx.x - 128;
        build_segments(sh.segs, a, nt, r, 1);
        set_dest(sh, recv, r, nt, per, q, (uint32_t)pitch * 4u);
        mbar_arrive(&sh.seg);
        ok = wait(&sh.seg, 0u);
        const int ext = ok ? sh.segs.n * rank : 0;
        // column c of the accumulator = row c of x, to its owner; `part`: with the adapters' part from its own
        auto send_product = [&](bool part) {
            const int groups = (k1 - k0 + p.chunk - 1) / p.chunk;  // accumulators in use; bf16: the extension went to the last
            for (int c = 0; c < p.rows; c += 32) {  // columns behind `rows` in the last 32 are allocated and dropped
                float s[32];
                uint32_t to[32];
                load_words(sh.dest + c, to);
                for (int gr = 0; gr < groups; ++gr) {
                    uint32_t v[32];
                    __syncwarp();
                    tmem_ld32(tmem + ((uint32_t)(r & ~31) << 16) + (uint32_t)(gr * p.rows + c), v);
                    tmem_ld_wait();
#pragma unroll
                    for (int j = 0; j < 32; ++j) s[j] = gr ? s[j] + __uint_as_float(v[j]) : __uint_as_float(v[j]);
                }
                if (!BF && part) {
                    uint32_t v[32], down[32];
                    __syncwarp();
                    tmem_ld32(tmem + ((uint32_t)(r & ~31) << 16) + (uint32_t)(p.next_col + c), v);
                    load_words(sh.down + c, down);
                    tmem_ld_wait();
#pragma unroll
                    for (int j = 0; j < 32; ++j) s[j] = fmaf(__uint_as_float(v[j]), __uint_as_float(down[j]), s[j]);
                }
#pragma unroll
                for (int j = 0; j < 32; ++j)
                    if (to[j] != kNoRow) st_cluster(to[j] + (uint32_t)r * 4u, s[j]);
            }
            tc_fence_before();
        };
        if constexpr (SELF) {
            ok = __all_sync(0xffffffffu, wait(sh.acc_full, 0u) && !sh.abort);
            tc_fence_after();
            cluster_wait();
            if (ok) send_product(false);
            if (ext && ok) {
                ok = __all_sync(0xffffffffu, wait(sh.acc_full + 1, 0u) && !sh.abort);
                tc_fence_after();
                if (ok) send_stacked(sh, p, tmem + (uint32_t)p.next_col, 0, rank, log2r, r, 512u);
                tc_fence_before();
            }
        }
        if constexpr (!SELF) {
            const int seg = ok ? sh.segs.row[r] : -1;
            const int ne = (ext + kExt - 1) / kExt;
            const int e0 = (int)((int64_t)ne * q / CS), e1 = (int)((int64_t)ne * (q + 1) / CS);
            const float *t = g.t + ((int64_t)(t0 + r) << log2r);
            const float scale = seg >= 0 ? __ldg(d.scale + a) : 0.f;
            dependency_wait();
            RowScale rs;
            if constexpr (!BF) {
                if (seg >= 0 && e0 < e1) rs.set(t, scale, rank);
                sh.down[r] = rs.down;
                bar_sync(1, kRows);  // for all of these warps' send_product
            }
            float4 v[8];
            if (e0 < e1) load_t_row(v, seg, rank, log2r, t, e0 * kExt);
            Ring tb;
            for (int e = e0; e < e1; ++e, tb.next(p.tbufs)) {
                if (tb.wrapped && !wait_warp(sh.t_empty + tb.s, tb.phase ^ 1u, &sh.abort)) { ok = false; break; }
                if (r < p.rows) store_t_row<BF, PARTS>(v, tbuf + (uint32_t)tb.s * kTiles * xbytes, xbytes, r, scale, rs.up);
                fence_async_shared();
                __syncwarp();
                if (lane == 0) mbar_arrive(sh.t_full + tb.s);
                if (e + 1 < e1) load_t_row(v, seg, rank, log2r, t, (e + 1) * kExt);
            }
            if (warp == 4 && __all_sync(kAll, ok)) ok = ring_drained(tb, sh.t_empty, p.tbufs, &sh.abort);
            if (!ok) give_up(sh, d.err);  // before the wait below, so that it ends
            __syncwarp();
            if (!wait(sh.acc_full, 0u)) ok = false;
            __syncwarp();
            tc_fence_after();
            cluster_wait();
            send_product(e0 < e1);
        }
    }
    if (!ok) {
        give_up(sh, d.err);
        drain();
    }
    __syncwarp();
    if (warp < 4) cluster_wait();
    cluster_arrive();
    cluster_wait();
    // this block's rows, two columns per thread: the cluster's parts in rank order
    const int r0 = q * per, r1 = min(nt, r0 + per);
    float *own_t = reinterpret_cast<float *>(ring);  // SELF: [row][rank] scale * x.A (the ring's loads have all been used)
    if constexpr (SELF) {
        for (int i = threadIdx.x; i < max(0, r1 - r0) << log2r; i += kThreads) {
            const int row = i >> log2r, s = sh.segs.row[r0 + row];
            float v = 0.f;
            if (s >= 0) {
                for (int c = 0; c < CS; ++c) v += recv[(c * per + row) * pitch + 128 + (i & (rank - 1))];
                v *= __ldg(d.scale + sh.segs.id[s]);
            }
            own_t[i] = v;
        }
        __syncthreads();
    }
    const int n = n0 + 2 * (threadIdx.x & 63);
    for (int r = r0 + (threadIdx.x >> 6); r < r1 && n < d.n_out; r += kThreads / 64) {
        float2 v = make_float2(0.f, 0.f);
        for (int c = 0; c < CS; ++c) {
            const float2 u = *reinterpret_cast<const float2 *>(recv + (c * per + r - r0) * pitch + 2 * (threadIdx.x & 63));
            v.x += u.x;
            v.y += u.y;
        }
        if constexpr (SELF) {
            const int s = sh.segs.row[r];
            if (s >= 0) {
                const uint16_t *b = static_cast<const uint16_t *>(d.b) + (((int64_t)sh.segs.id[s] << log2r) * d.ldb + n);
                const float *t = own_t + ((r - r0) << log2r);
#pragma unroll 16
                for (int j = 0; j < rank; ++j) {
                    const float2 u = unpack2<BF>(__ldg(reinterpret_cast<const uint32_t *>(b + j * d.ldb)));
                    v.x = fmaf(t[j], u.x, v.x);
                    v.y = fmaf(t[j], u.y, v.y);
                }
            }
        }
        Y *y = static_cast<Y *>(d.y) + (int64_t)(t0 + r) * d.ldy + n;
        if (n + 1 < d.n_out && (uintptr_t)y % (2 * sizeof(Y)) == 0) {
            if constexpr (sizeof(Y) == 4) *reinterpret_cast<float2 *>(y) = v;
            else *reinterpret_cast<uint32_t *>(y) = pack2<BF>(v.x, v.y);
        } else {  // rows of y that are not aligned, the last column of an odd width
            y[0] = to_y<Y>(v.x);
            if (n + 1 < d.n_out) y[1] = to_y<Y>(v.y);
        }
    }
    tc_fence_before();
    __syncthreads();
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

// Dynamic shared memory of a block beside the static: all of an SM's, whatever
// the ring needs, so that no block of another kernel that wants TMEM starts
// beside it: clusters whose blocks wait for columns that the other's hold would
// wait for each other.
constexpr size_t kSmem = 227 * 1024 - sizeof(Shared);

// Clusters of more than 8 blocks, once per kernel and device.
cudaError_t allow_clusters(const void *fn) {
    static std::mutex mu;
    static std::set<std::pair<const void *, int>> done;
    int dev = 0;
    cudaError_t err = cudaGetDevice(&dev);
    if (err != cudaSuccess) return err;
    std::lock_guard<std::mutex> lock(mu);
    if (done.count({fn, dev})) return cudaSuccess;
    err = cudaFuncSetAttribute(fn, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (err == cudaSuccess) done.insert({fn, dev});
    return err;
}

cudaError_t launch_cluster(const void *fn, dim3 grid, bool dependent, void **args, cudaStream_t s) {
    cudaError_t err = ensure_smem(fn, kSmem);
    if (err != cudaSuccess || (grid.x > 8 && (err = allow_clusters(fn)) != cudaSuccess)) return err;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = kSmem;
    cfg.stream = s;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = grid.x;
    at[0].val.clusterDim.y = 1;
    at[0].val.clusterDim.z = 1;
    at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = dependent ? 2 : 1;
    return cudaLaunchKernelExC(&cfg, fn, args);
}

// Clusters of 1..16 blocks that the device holds at once, one block per SM (a
// cluster stays within a GPC: 7 of 16, 15 of 9, 22 of 6, 33 of 4 on 148 SMs).
// More than 8 are not portable to every device; the kernels ask for them.
const int *cluster_room() {
    struct Table {
        bool set = false;
        int n[kMaxCluster + 1];
    };
    static std::mutex mu;
    static Table tables[64];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return nullptr;
    std::lock_guard<std::mutex> lock(mu);
    Table &t = tables[dev];
    if (!t.set) {
        const void *fn = (const void *)k_ad_shrink<true, false>;
        if (ensure_smem(fn, kSmem) != cudaSuccess || allow_clusters(fn) != cudaSuccess) return nullptr;
        for (int c = 1; c <= kMaxCluster; ++c) {
            cudaLaunchConfig_t cfg{};
            cfg.gridDim = dim3(c, 256);
            cfg.blockDim = dim3(kThreads);
            cfg.dynamicSmemBytes = kSmem;
            cudaLaunchAttribute at[1];
            at[0].id = cudaLaunchAttributeClusterDimension;
            at[0].val.clusterDim.x = (unsigned)c;
            at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
            cfg.attrs = at;
            cfg.numAttrs = 1;
            if (cudaOccupancyMaxActiveClusters(&t.n[c], fn, &cfg) != cudaSuccess) return nullptr;
        }
        t.set = true;
    }
    return t.n;
}

// Blocks of a cluster for `others` clusters: as many as the contraction has
// blocks for and as run at once.
int pick_cluster(int64_t others, int blocks, const int *room) {
    int c = blocks < kMaxCluster ? blocks : kMaxCluster;
    while (c > 1 && others > room[c]) --c;
    return c;
}

// What the cluster sends to one block: a row of `row` bytes per rank and owned row.
size_t recv_bytes(int tile_rows, int cluster, int row) {
    return (size_t)cluster * ((tile_rows + cluster - 1) / cluster) * row;
}

// Stages beside `other` bytes of shared memory, no more than there are loads.
int pick_stages(size_t stage, size_t other, int loads) {
    int n = (int)((kSmem - 1024 - other) / stage);
    if (n > kMaxStages) n = kMaxStages;
    return n < loads ? n : loads;
}

template <typename Y, bool SELF>
const void *skinny_fn(bool bf, bool kn) {
    constexpr int P = sizeof(Y) == 4 ? 3 : 2;
    if (bf) return kn ? (const void *)k_ad_skinny<true, true, P, Y, SELF> : (const void *)k_ad_skinny<true, false, P, Y, SELF>;
    return kn ? (const void *)k_ad_skinny<false, true, 2, Y, SELF> : (const void *)k_ad_skinny<false, false, 2, Y, SELF>;
}
template <bool SELF>
const void *skinny_fn(bool bf, bool kn, bool f32) {
    if (f32) return skinny_fn<float, SELF>(bf, kn);
    return bf ? skinny_fn<__nv_bfloat16, SELF>(bf, kn) : skinny_fn<__half, SELF>(bf, kn);
}

}  // namespace

namespace {
bool encode(void *map, CUtensorMapDataType type, int size, const void *base, uint64_t rows, uint64_t cols, uint64_t ld,
            uint32_t box_rows) {
    EncodeTiledFn fn = encode_fn();
    if (!fn) return false;
    cuuint64_t dims[2] = {cols, rows};
    cuuint64_t strides[1] = {ld * size};
    cuuint32_t box[2] = {128u / size, box_rows};
    cuuint32_t es[2] = {1, 1};
    return fn(static_cast<CUtensorMap *>(map), type, 2, const_cast<void *>(base), dims, strides, box, es,
              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
}  // namespace

bool adapter_map(void *map, bool bf16, const void *base, uint64_t rows, uint64_t cols, uint64_t ld, uint32_t box_rows) {
    return encode(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, base, rows, cols, ld,
                  box_rows);
}

bool adapter_out_map(void *map, int y_type, void *base, uint64_t rows, uint64_t cols, uint64_t ld, uint32_t box_rows) {
    if (y_type == LATENT_TYPE_F32) return encode(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 4, base, rows, cols, ld, box_rows);
    return adapter_map(map, y_type == LATENT_TYPE_BF16, base, rows, cols, ld, box_rows);
}

namespace {

struct ShrinkPlan {
    Plan p;
    int cluster, slots, tiles;
};
ShrinkPlan plan_shrink(const AdapterArgs &g, const int *room) {
    const latent_adapter_desc &d = g.d;
    ShrinkPlan r{};
    Plan &p = r.p;
    r.tiles = (d.n_tokens + g.tile_rows - 1) / g.tile_rows;
    const int most = ((d.n_adapter < g.tile_rows ? d.n_adapter : g.tile_rows) * d.rank + 127) / 128;
    const int nk = (d.n_in + kBK - 1) / kBK;
    p.rows = (g.tile_rows + 15) / 16 * 16;
    const size_t stage = 16384 + (size_t)p.rows * 128;
    // Clusters, and tiles of stacked rank columns side by side: the fewest K blocks one after the other.  A batch of
    // one row tile may use every adapter; longer ones are packed prompts with few to a tile.
    const int expect = r.tiles == 1 ? most : 1;
    int64_t best = INT64_MAX;
    for (int c = 1; c <= kMaxCluster && c <= nk; ++c) {
        if (room[c] < 1) continue;
        int slots = room[c] / r.tiles;
        slots = slots < 1 ? 1 : slots > most ? most : slots;
        const int64_t turns = ((int64_t)r.tiles * slots + room[c] - 1) / room[c];
        const int64_t cost = turns * ((expect + slots - 1) / slots) * ((nk + c - 1) / c);
        if (cost < best) {
            best = cost;
            r.cluster = c;
            r.slots = slots;
        }
    }
    const size_t recv = recv_bytes(g.tile_rows, r.cluster, d.rank * 4);
    p.stages = pick_stages(stage, recv, (nk + r.cluster - 1) / r.cluster * ((most + r.slots - 1) / r.slots));
    p.cols = tmem_cols(2 * ((p.rows + 31) / 32 * 32));
    return r;
}

// Accumulators of `rows` columns in k_ad_skinny's TMEM.  The tensor cores cut a
// sum off instead of rounding it (figures at k_ad_wide): fp32 results use an
// accumulator per 512 of K, added up in fp32, as far as the TMEM columns go,
// and clusters long enough.
// `next`: with one more accumulator behind them.
int accumulators(int rows, bool next) {
    const int read = (rows + 31) / 32 * 32;  // columns the epilogue reads of an accumulator
    return (512 - (next ? 2 : 1) * read) / rows + 1;
}

// Blocks of a cluster of k_ad_skinny.  Where both kernels are small, its
// clusters start beside the shrink's blocks and stream W meanwhile, so those
// SMs are not counted on as long as two blocks per cluster are left (8 rows of
// 4096 x 4096 with 8 of 64 adapters of rank 16: 13.0 us, 14.7 with all SMs; of
// 4096 x 8192, where one block of two would be left: 24.7 us, 17.8 with all).
int plan_skinny(const AdapterArgs &g, const int *room, int beside, int sms) {
    const latent_adapter_desc &d = g.d;
    const int64_t others = ((int64_t)d.n_tokens + g.tile_rows - 1) / g.tile_rows * ((d.n_out + 127) / 128);
    const int nk = (d.n_in + kBK - 1) / kBK;
    int c = pick_cluster(others, nk, room);
    while (beside && c > 2 && others * c > sms - beside) --c;
    if (d.y_type == LATENT_TYPE_F32) {
        const int groups = accumulators((g.tile_rows + 15) / 16 * 16, d.type == LATENT_TYPE_F16);
        while (c < kMaxCluster && c < nk && room[c + 1] > 0 && (nk + c - 1) / c > 8 * groups) ++c;
    }
    return c;
}

}  // namespace

cudaError_t launch_adapter_shrink(const AdapterArgs &g, const void *x_map, cudaStream_t s) {
    const latent_adapter_desc &d = g.d;
    const bool bf = d.type == LATENT_TYPE_BF16;
    const int *room = cluster_room();
    if (!room) return cudaErrorInvalidConfiguration;
    ShrinkPlan r = plan_shrink(g, room);
    if (r.p.stages < 1) return cudaErrorInvalidConfiguration;
    CUtensorMap mA;
    if (!adapter_map(&mA, bf, d.a, (uint64_t)d.n_adapter * d.rank, d.n_in, d.lda, d.rank)) return cudaErrorInvalidValue;
    AdapterArgs a = g;
    void *args[] = {&mA, const_cast<void *>(x_map), &a, &r.p};
    const void *fn = d.y_type == LATENT_TYPE_F32 ? bf ? (const void *)k_ad_shrink<true, true> : (const void *)k_ad_shrink<false, true>
                                                 : bf ? (const void *)k_ad_shrink<true, false> : (const void *)k_ad_shrink<false, false>;
    return launch_cluster(fn, dim3(r.cluster, r.slots, r.tiles), false, args, s);
}

cudaError_t launch_adapter_skinny(const AdapterArgs &g, const void *x_map, int sms, bool self, cudaStream_t s) {
    const latent_adapter_desc &d = g.d;
    const bool bf = d.type == LATENT_TYPE_BF16, kn = !(d.flags & LATENT_ADAPTER_W_TRANSPOSED);
    const bool f32 = d.y_type == LATENT_TYPE_F32;
    const int tiles = (d.n_tokens + g.tile_rows - 1) / g.tile_rows, ntn = (d.n_out + 127) / 128;
    const int nk = (d.n_in + kBK - 1) / kBK;
    const int *room = cluster_room();
    if (!room) return cudaErrorInvalidConfiguration;
    Plan p{};
    p.rows = (g.tile_rows + 15) / 16 * 16;
    const int parts = bf && f32 ? 3 : 2;
    // as far as the ring still holds the loads of a trip to DRAM
    p.tbufs = self ? 0 : p.rows <= 64 ? kMaxTBufs : 2;
    const size_t stage = 16384 + (size_t)p.rows * 128, tb = (size_t)p.tbufs * ((parts + 1) / 2) * p.rows * 128;
    const int cluster = self ? adapter_self_cluster(g) : adapter_skinny_cluster(g, sms);
    const int read = (p.rows + 31) / 32 * 32, groups = accumulators(p.rows, self || !bf);
    const int per = (nk + cluster - 1) / cluster;
    p.chunk = per;
    if (f32) p.chunk = per <= 8 * groups ? 8 : (per + groups - 1) / groups;
    p.next_col = ((per + p.chunk - 1) / p.chunk - 1) * p.rows + read;
    p.cols = tmem_cols(p.next_col + (self || !bf ? read : 0));
    const size_t recv = recv_bytes(g.tile_rows, cluster, self ? 512 + d.rank * 4 : 512);
    p.stages = pick_stages(stage, tb + recv, per * (self ? 2 : 1) + 4);
    if (p.stages < 1) return cudaErrorInvalidConfiguration;
    CUtensorMap mW, mB, mA{};
    if (!(kn ? adapter_map(&mW, bf, d.w, d.n_in, d.n_out, d.ldw, kBK) : adapter_map(&mW, bf, d.w, d.n_out, d.n_in, d.ldw, 128)) ||
        !adapter_map(&mB, bf, d.b, (uint64_t)d.n_adapter * d.rank, d.n_out, d.ldb, d.rank < kExt ? d.rank : kExt) ||
        (self && !adapter_map(&mA, bf, d.a, (uint64_t)d.n_adapter * d.rank, d.n_in, d.lda, d.rank)))
        return cudaErrorInvalidValue;
    const void *fn = self ? skinny_fn<true>(bf, kn, f32) : skinny_fn<false>(bf, kn, f32);
    AdapterArgs a = g;
    void *args[] = {&mW, &mB, const_cast<void *>(x_map), &mA, &a, &p};
    return launch_cluster(fn, dim3(cluster, ntn, tiles), !self, args, s);
}

int adapter_skinny_cluster(const AdapterArgs &g, int sms) {
    const int *room = cluster_room();
    if (!room) return 1;
    const ShrinkPlan r = plan_shrink(g, room);
    const int shrink = r.cluster * r.slots * r.tiles;
    return plan_skinny(g, room, shrink <= sms / 3 ? shrink : 0, sms);
}

int adapter_waves(int64_t clusters, int cluster) {
    const int *room = cluster_room();
    return room && room[cluster] > 0 ? (int)((clusters + room[cluster] - 1) / room[cluster]) : 1;
}

int adapter_self_cluster(const AdapterArgs &g) {
    const int *room = cluster_room();
    const latent_adapter_desc &d = g.d;
    return room ? pick_cluster((d.n_out + 127) / 128, (d.n_in + kBK - 1) / kBK, room) : 1;
}

}  // namespace latent
