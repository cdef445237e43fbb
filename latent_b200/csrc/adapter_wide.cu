// The adapters' product for prompt-sized batches: y = x.W + the adapters'
// part, tiles of 256 rows x 256 columns (fp32 results: 128) on pairs of SMs
// (tcgen05 cta_group::2).
//
// Persistent, one cluster of two blocks per tile at a time.  Each block holds
// 128 rows of x and half the tile's columns of W per stage (a ring of 5) and
// its 128 rows of the accumulator in TMEM, twice, so that the epilogue of one
// tile runs under the MMAs of the next.  Per block: warp 0 loads (TMA, plain
// per-block loads that complete on the leader's barrier), warp 1 of the leader
// issues the pair's MMAs, warps 4..7 drain accumulators (through shared memory
// to TMA stores, which also clip the ragged edges), warps 8..11 list the
// adapters of the tile's 256 rows and build the x.A parts of the extension
// blocks (32 stacked B rows each).
//
// A pair tile of 256 columns costs 512 cycles of MMA per 64 of K against 64 KB
// of loads: half the L2 traffic per operation of one block working alone.
// Measured: 8192 rows of 4096 x 14336, bf16: 602 us, 1.60 PFLOP/s, tensor pipe
// 93% active (power bound in a long run: 650 us).  2047 rows of 4096 x 4096: 51
// us without adapters (128 tiles on 74 pairs: two turns, the second of 54), 56
// with five packed prompts of rank 64, 65 with six adapters mixed over all rows.
//
// fp32 results: the tensor cores cut a sum off instead of rounding it, so the
// two accumulators take turns every 512 of K and the epilogue adds them up in
// fp32 registers, 128 a thread, hence the narrower tile.  Measured at K = 7168,
// root mean squares: one chain 7.9e-6 of the result (fp16 8.4e-6; terms of one
// sign 2.2e-5, fp16 4.4e-5), chains of 512 4.8e-7 (6.5e-7; 2.4e-7, 2.4e-6), a
// plain fp32 product 8.8e-7 (1.5e-6; 1.2e-6, 1.2e-6).  16-bit results keep the
// one chain: their rounding is 1.66e-3 (fp16 2.07e-4) with it as without, with
// terms of one sign 1.29e-3 (fp16 1.67e-4 for 1.61e-4).
//
// fp16 to fp32: the adapters' part takes one more turn of the accumulators, its
// rows scaled (RowScale).
#include <cooperative_groups.h>
#include <cuda.h>

#include "adapter_mma.cuh"

namespace latent {

namespace {

namespace cg = cooperative_groups;
using namespace adapter;

constexpr int kThreads = 384;
constexpr int kPairRows = 256;
constexpr int kGroupM = 8;       // row tiles that share a sweep over the columns (L2 reuse)
constexpr uint32_t kXBytes = 16384;
constexpr uint32_t kOut = 4096;  // a warp's staging: 32 rows of 128 bytes
// All of an SM's shared memory, more than the kernel needs, so that no block of
// another kernel that wants TMEM starts beside it: clusters whose blocks wait
// for columns that the other's hold would wait for each other.
constexpr size_t kStatic = 6144;
constexpr size_t kSmem = 227 * 1024 - kStatic;

template <bool BF, bool F32>
struct Cfg {
    static constexpr int kCols = F32 ? 128 : 256;                    // of a pair's tile
    static constexpr int kStages = 5;
    static constexpr uint32_t kStage = kXBytes + kCols / 2 * 128;    // x, W
    static constexpr int kParts = BF && F32 ? 3 : 2;
    static constexpr bool kScaled = !BF && F32;                      // the adapters' part has an accumulator of its own
    static constexpr bool kWide = !BF && !F32;                       // rows that fp16 parts cannot hold
    static constexpr uint32_t kTTile = 16384u * ((kParts + 1) / 2);  // 128 rows x (2 parts x 32) of x.A, and the third part
    static constexpr int kChunk = F32 ? 8 : 1 << 30;                 // K blocks per accumulator
    static constexpr int kTBufs = 2;
    static_assert(1024 + kStages * kStage + kTBufs * kTTile + 4 * kOut <= kSmem, "shared memory");
};

struct PairSegments {
    int n;
    int id[kPairRows];
    int16_t row[128];     // of this block's rows
    uint8_t wide[128];    // fp16 results: finished in fp32 by the epilogue
    float down[128];      // fp16 to fp32: RowScale's, of the rows' t
};

struct Shared {
    uint64_t full[5], empty[5];
    uint64_t acc_full[2], acc_empty[2], t_full[2], t_empty[2], seg_full[2], seg_empty[2];
    uint32_t tmem;
    volatile int abort;
    alignas(16) int ids[kPairRows];
    int first[kPairRows];
    int warp_n[8];
    PairSegments seg[2];
};

static_assert(sizeof(Shared) <= kStatic, "static shared memory");

__device__ __forceinline__ uint32_t peer_addr(const void *p, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_addr(p)), "r"(rank));
    return r;
}
// Releases what this thread did and has observed in shared memory to the pair:
// all that the other block's threads take over from an arrival (the x.A parts;
// TMEM reads are over before it).  A release of global memory too has an
// extension block wait for its loads: 1.3 us instead of 0.5 (made by a warp
// of its own: 0.9).
__device__ __forceinline__ void arrive_cluster(uint32_t bar) {
    asm volatile(
        "fence.release.sync_restrict::shared::cta.cluster;\n\t"
        "mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar)
        : "memory");
}
__device__ __forceinline__ void load_pair(void *dst, const CUtensorMap *map, int c0, int c1, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], "
        "[%4];" ::"r"(smem_addr(dst)),
        "l"(map), "r"(c0), "r"(c1), "r"(bar)
        : "memory");
}
__device__ __forceinline__ void mma_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t id, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(id), "r"(accumulate)
        : "memory");
}
// Arrives on the barrier at this offset in both blocks once the MMAs issued so far are complete.
__device__ __forceinline__ void commit_pair(uint64_t *bar) {
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
            smem_addr(bar)),
        "h"((uint16_t)3)
        : "memory");
}

__device__ __forceinline__ void store_box(const CUtensorMap *map, int c0, int c1, const void *src) {
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%1, %2}], [%3];" ::"l"(map), "r"(c0), "r"(c1),
                 "r"(smem_addr(src))
                 : "memory");
}
__device__ __forceinline__ void store_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void store_wait_read() {
    asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void store_wait() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }

struct Tile {
    int t0, n0;
};
// Tiles in sweeps of kGroupM row tiles: all columns of one sweep before the next.
template <int COLS>
__device__ __forceinline__ Tile tile_at(int i, int tm, int tn) {
    const int per = kGroupM * tn, g = i / per, first = g * kGroupM;
    const int rows = min(kGroupM, tm - first), j = i - g * per;
    return {(first + j % rows) * kPairRows, (j / rows) * COLS};
}

// M = 256 over the pair.
__host__ __device__ constexpr uint32_t idesc_pair(bool bf16, int cols, bool b_mn) {
    return (1u << 4) | ((bf16 ? 1u : 0u) << 7) | ((bf16 ? 1u : 0u) << 10) | ((b_mn ? 1u : 0u) << 16) |
           ((uint32_t)(cols >> 3) << 17) | ((uint32_t)(kPairRows >> 4) << 24);
}

template <bool BF, bool KN, bool F32>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
k_ad_wide(const __grid_constant__ CUtensorMap mX, const __grid_constant__ CUtensorMap mW,
          const __grid_constant__ CUtensorMap mB, const __grid_constant__ CUtensorMap mY, AdapterArgs g) {
    using C = Cfg<BF, F32>;
    constexpr int kStages = C::kStages, kPairCols = C::kCols, kHalf = kPairCols / 2;
    constexpr uint32_t kStage = C::kStage;
    extern __shared__ uint8_t raw[];
    uint8_t *ring = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
    uint8_t *tbuf = ring + kStages * kStage;
    uint8_t *obuf = tbuf + C::kTBufs * C::kTTile;
    __shared__ Shared sh;
    cg::cluster_group cluster = cg::this_cluster();
    const int cta = blockIdx.x & 1;  // its rank in the cluster
    const int warp = warp_index(), lane = threadIdx.x & 31;
    const latent_adapter_desc &d = g.d;
    const int rank = d.rank;
    const int tm = (d.n_tokens + kPairRows - 1) / kPairRows, tn = (d.n_out + kPairCols - 1) / kPairCols;
    const int tiles = tm * tn, pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
    const int nk = (d.n_in + kBK - 1) / kBK, chunks = (nk - 1) / C::kChunk + 1;  // of K per tile

    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s) {
            mbar_init(sh.full + s, 1);
            mbar_init(sh.empty + s, 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(sh.acc_full + b, 1);
            mbar_init(sh.acc_empty + b, 8);    // the epilogue warps of both blocks
            mbar_init(sh.t_full + b, 8);       // the builders' warps of both
            mbar_init(sh.t_empty + b, 1);
            mbar_init(sh.seg_full + b, 128);
            mbar_init(sh.seg_empty + b, 6);    // loader, MMA warp and epilogue warps of this block
        }
        sh.abort = 0;
        fence_barrier_init();
    }
    if (warp == 2) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&sh.tmem)),
                     "r"(512)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    cluster.sync();  // both blocks' barriers exist before either arrives on the other's
    tc_fence_after();
    const uint32_t tmem = (uint32_t)uniform((int)sh.tmem);
    bool ok = true;
    Ring tb_last;  // the builders' x.A tiles

    if (warp == 0) {
        // ---------------- loads ----------------
        Ring at;
        int tl = 0;
        const uint32_t full0 = peer_addr(sh.full, 0);
        for (int i = pair; i < tiles && ok; i += pairs, ++tl) {
            const Tile tile = tile_at<kPairCols>(i, tm, tn);
            const int row = tile.t0 + cta * 128, col = tile.n0 + cta * kHalf;
            for (int k = 0; k < nk; ++k, at.next(kStages)) {
                if (at.wrapped && !wait_warp(sh.empty + at.s, at.phase ^ 1u, &sh.abort)) { ok = false; break; }
                if (elect()) {
                    uint8_t *st = ring + at.s * kStage;
                    const uint32_t bar = full0 + at.s * 8;
                    if (cta == 0) mbar_arrive_expect_tx(sh.full + at.s, 2 * kStage);
                    load_pair(st, &mX, k * kBK, row, bar);
                    if (KN) {
                        load_pair(st + kXBytes, &mW, col, k * kBK, bar);
                        if (kHalf > 64) load_pair(st + kXBytes + 8192, &mW, col + 64, k * kBK, bar);
                    } else {
                        load_pair(st + kXBytes, &mW, k * kBK, col, bar);
                    }
                }
            }
            if (!ok || !wait_warp(sh.seg_full + (tl & 1), (uint32_t)(tl >> 1) & 1u, &sh.abort)) { ok = false; break; }
            const PairSegments &seg = sh.seg[tl & 1];
            const int ext = uniform(seg.n) * rank, box = min(rank, kExt);
            for (int r0 = 0; r0 < ext; r0 += kExt, at.next(kStages)) {
                if (at.wrapped && !wait_warp(sh.empty + at.s, at.phase ^ 1u, &sh.abort)) { ok = false; break; }
                const int rows = min(kExt, ext - r0), r = r0 + lane * box;  // one box of 32 rows or two of 16
                const int src = lane * box < rows ? (seg.id[r >> g.log2r] << g.log2r) + (r & (rank - 1)) : 0;
                const int src0 = __shfl_sync(kAll, src, 0), src1 = __shfl_sync(kAll, src, 1);
                if (elect()) {
                    uint8_t *st = ring + at.s * kStage + kXBytes;
                    const uint32_t bar = full0 + at.s * 8;
                    if (cta == 0) mbar_arrive_expect_tx(sh.full + at.s, (uint32_t)(rows * kPairCols * 2));
                    load_pair(st, &mB, col, src0, bar);
                    if (kHalf > 64) load_pair(st + 8192, &mB, col + 64, src0, bar);
                    if (box < rows) {
                        load_pair(st + 2048, &mB, col, src1, bar);
                        if (kHalf > 64) load_pair(st + 8192 + 2048, &mB, col + 64, src1, bar);
                    }
                }
            }
            if (ok && lane == 0) mbar_arrive(sh.seg_empty + (tl & 1));
        }
        if (ok) ok = ring_drained(at, sh.empty, kStages, &sh.abort);
    } else if (warp == 1) {
        // ---------------- MMAs (the leader's warp, for both blocks) ----------------
        Ring at, tb;
        int tl = 0, cc = 0;  // tiles, accumulators
        constexpr uint32_t id = idesc_pair(BF, kPairCols, KN), idx = idesc_pair(BF, kPairCols, true);
        for (int i = pair; i < tiles && ok; i += pairs, ++tl) {
            uint32_t acc = 0;
            if (cta == 0) {
                int left = 0;  // blocks until the next accumulator
                for (int k = 0; k < nk; ++k, at.next(kStages)) {
                    if (left == 0) {
                        if (k && elect()) commit_pair(sh.acc_full + ((cc - 1) & 1));
                        if (cc >= 2 && !wait_warp<true>(sh.acc_empty + (cc & 1), (uint32_t)((cc >> 1) - 1) & 1u, &sh.abort)) {
                            ok = false;
                            break;
                        }
                        tc_fence_after();
                        acc = tmem + (uint32_t)(cc & 1) * (uint32_t)kPairCols;
                        left = min(C::kChunk, nk - k);
                        ++cc;
                    }
                    if (!wait_warp(sh.full + at.s, at.phase, &sh.abort)) { ok = false; break; }
                    tc_fence_after();
                    if (elect()) {
                        const uint32_t x = smem_addr(ring + at.s * kStage), w = x + kXBytes;
                        const uint32_t more = left != min(C::kChunk, nk - k / C::kChunk * C::kChunk);  // not the first of its accumulator
#pragma unroll
                        for (int kk = 0; kk < 4; ++kk)
                            mma_pair(acc, desc_kmajor_sw128(x + kk * 32),
                                     KN ? desc_mnmajor_sw128(w + kk * 2048) : desc_kmajor_sw128(w + kk * 32), id, more | kk);
                        commit_pair(sh.empty + at.s);
                    }
                    --left;
                }
                if (!ok) break;
            }
            if (!wait_warp(sh.seg_full + (tl & 1), (uint32_t)(tl >> 1) & 1u, &sh.abort)) { ok = false; break; }
            const int ext = uniform(sh.seg[tl & 1].n) * rank;
            if (cta == 0) {  // the adapters' part goes to the last accumulator, or to the next
                uint32_t more = 1;
                if (C::kScaled && ext) {
                    if (elect()) commit_pair(sh.acc_full + ((cc - 1) & 1));
                    if (cc >= 2 && !wait_warp<true>(sh.acc_empty + (cc & 1), (uint32_t)((cc >> 1) - 1) & 1u, &sh.abort)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    acc = tmem + (uint32_t)(cc & 1) * (uint32_t)kPairCols;
                    more = 0;
                    ++cc;
                }
                for (int r0 = 0; r0 < ext; r0 += kExt, at.next(kStages), tb.next(C::kTBufs)) {
                    if (!wait_warp(sh.full + at.s, at.phase, &sh.abort) ||
                        !wait_warp<true>(sh.t_full + tb.s, tb.phase, &sh.abort)) { ok = false; break; }
                    tc_fence_after();
                    if (elect()) {
                        const uint32_t w = smem_addr(ring + at.s * kStage) + kXBytes, t = smem_addr(tbuf + tb.s * C::kTTile);
                        const int steps = min(kExt / 16, (ext - r0) / 16);
                        for (int kk = 0; kk < steps; ++kk)
#pragma unroll
                            for (int q = 0; q < C::kParts; ++q)
                                mma_pair(acc, desc_kmajor_sw128(t + t_offset(q, kk, 16384u)), desc_mnmajor_sw128(w + kk * 2048), idx,
                                         more | kk | q);
                        commit_pair(sh.empty + at.s);
                        commit_pair(sh.t_empty + tb.s);
                    }
                    more = 1;
                }
                if (!ok) break;
                if (elect()) commit_pair(sh.acc_full + ((cc - 1) & 1));
            }
            if (lane == 0) mbar_arrive(sh.seg_empty + (tl & 1));
        }
        if (!ok && cta == 0 && elect()) {
            commit_pair(sh.acc_full);  // lets the waiting epilogues go on to the abort flag
            commit_pair(sh.acc_full + 1);
        }
    } else if (warp >= 4 && warp < 8) {
        // ---------------- epilogue: lane = row ----------------
        const int r = threadIdx.x - 128, w = warp - 4;
        uint8_t *out = obuf + w * kOut;
        const uint32_t lanes = tmem + ((uint32_t)(w * 32) << 16);
        int tl = 0, cc = 0;
        for (int i = pair; i < tiles; i += pairs, ++tl) {
            const Tile tile = tile_at<kPairCols>(i, tm, tn);
            if (!wait_warp(sh.seg_full + (tl & 1), (uint32_t)(tl >> 1) & 1u, &sh.abort)) { ok = false; break; }
            const PairSegments &seg = sh.seg[tl & 1];
            const int t = tile.t0 + cta * 128 + r, row0 = tile.t0 + cta * 128 + w * 32;
            const bool wide = C::kWide && t < d.n_tokens && seg.wide[r];
            const int a = wide ? seg.id[seg.row[r]] : 0;
            const uint32_t wide_rows = C::kWide ? __ballot_sync(kAll, wide) : 0u;
            float v[F32 ? kPairCols : 64];
            if constexpr (F32) {
                const int sums = chunks + (C::kScaled && uniform(seg.n) ? 1 : 0);
                for (int c = 0; c < sums; ++c, ++cc) {
                    const float down = C::kScaled && c == chunks ? seg.down[r] : 1.f;
                    if (!wait_warp(sh.acc_full + (cc & 1), (uint32_t)(cc >> 1) & 1u, &sh.abort)) { ok = false; break; }
                    tc_fence_after();
#pragma unroll
                    for (int n = 0; n < kPairCols; n += 16) {
                        uint32_t u[16];
                        tmem_ld16(lanes + (uint32_t)((cc & 1) * kPairCols + n), u);
                        tmem_ld_wait();
#pragma unroll
                        for (int j = 0; j < 16; ++j) {
                            const float p = C::kScaled ? __uint_as_float(u[j]) * down : __uint_as_float(u[j]);
                            v[n + j] = c ? v[n + j] + p : p;
                        }
                    }
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) arrive_cluster(peer_addr(sh.acc_empty + (cc & 1), 0));
                }
                if (!ok) break;
            } else {
                if (!wait_warp(sh.acc_full + (cc & 1), (uint32_t)(cc >> 1) & 1u, &sh.abort)) { ok = false; break; }
                tc_fence_after();
            }
            // 128 bytes of a row at a time: registers, swizzled shared memory, one TMA store per warp
            constexpr int kRun = F32 ? 32 : 64;
#pragma unroll
            for (int c = 0; c < kPairCols; c += kRun) {
                if constexpr (!F32) {
#pragma unroll
                    for (int h = 0; h < 64; h += 32) {
                        uint32_t u[32];
                        tmem_ld32(lanes + (uint32_t)((cc & 1) * kPairCols + c + h), u);
                        tmem_ld_wait();
#pragma unroll
                        for (int j = 0; j < 32; ++j) v[h + j] = __uint_as_float(u[j]);
                    }
                }
                float *x = v + (F32 ? c : 0);
                if constexpr (C::kWide) {  // rows whose x.A fp16 parts cannot hold: the warp makes a row's part, its lane takes it
                    for (uint32_t rest = wide_rows; rest; rest &= rest - 1) {
                        const int b = __ffs(rest) - 1, ad = __shfl_sync(kAll, a, b);
                        const float *tb = g.t + (int64_t)(row0 + b) * rank;
                        const int n = tile.n0 + c + lane * (kRun / 32);
                        float p0 = 0.f, p1 = 0.f;
                        if (n < d.n_out) p0 = adapter_dot<BF>(d, tb, ad, n);
                        if (kRun > 32 && n + 1 < d.n_out) p1 = adapter_dot<BF>(d, tb, ad, n + 1);
#pragma unroll
                        for (int j = 0; j < kRun; ++j) {
                            const float p = kRun > 32 ? __shfl_sync(kAll, j & 1 ? p1 : p0, j >> 1) : __shfl_sync(kAll, p0, j);
                            if (lane == b) x[j] += p;
                        }
                    }
                }
                __syncwarp();
                if (elect()) store_wait_read<0>();  // the store before has left the buffer
                __syncwarp();
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    uint4 o;
                    if constexpr (F32) {
                        o = make_uint4(__float_as_uint(x[4 * j]), __float_as_uint(x[4 * j + 1]), __float_as_uint(x[4 * j + 2]),
                                       __float_as_uint(x[4 * j + 3]));
                    } else {
                        o = make_uint4(pack2<BF>(x[8 * j], x[8 * j + 1]), pack2<BF>(x[8 * j + 2], x[8 * j + 3]),
                                       pack2<BF>(x[8 * j + 4], x[8 * j + 5]), pack2<BF>(x[8 * j + 6], x[8 * j + 7]));
                    }
                    *reinterpret_cast<uint4 *>(out + lane * 128 + ((j ^ (lane & 7)) * 16)) = o;
                }
                fence_async_shared();
                __syncwarp();
                if (row0 < d.n_tokens && tile.n0 + c < d.n_out && elect()) {
                    store_box(&mY, tile.n0 + c, row0, out);
                    store_commit();
                }
            }
            if constexpr (!F32) {
                tc_fence_before();
                __syncwarp();
                if (lane == 0) arrive_cluster(peer_addr(sh.acc_empty + (cc & 1), 0));
                ++cc;
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(sh.seg_empty + (tl & 1));
        }
        __syncwarp();
        if (elect()) store_wait();
    } else if (warp >= 8) {
        // ---------------- adapters of the tile, x.A parts ----------------
        const int tid = threadIdx.x - 256;
        int tl = 0;
        Ring &tb = tb_last;
        dependency_wait();
        for (int i = pair; i < tiles; i += pairs, ++tl) {
            const Tile tile = tile_at<kPairCols>(i, tm, tn);
            if (tl >= 2 && ok) ok = wait(sh.seg_empty + (tl & 1), (uint32_t)((tl >> 1) - 1) & 1u);
            // all 128 go on or none: the named barriers below have no limit of their own
            if (!bar_all(2, 128, ok && !sh.abort)) { ok = false; break; }
            PairSegments &seg = sh.seg[tl & 1];
            // two rows per thread, numbered by the first row of the pair's 256 that has the same adapter
            int a[2], lead[2], at[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int t = tile.t0 + h * 128 + tid;
                a[h] = t < d.n_tokens ? __ldg(d.ids + t) : -1;
                if (a[h] >= d.n_adapter) a[h] = -1;
                sh.ids[h * 128 + tid] = a[h];
                lead[h] = h * 128 + tid;
            }
            bar_sync(1, 128);
#pragma unroll 4
            for (int j = kPairRows - 4; j >= 0; j -= 4) {
                const int4 v = *reinterpret_cast<const int4 *>(sh.ids + j);
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    if (v.w == a[h]) lead[h] = j + 3;
                    if (v.z == a[h]) lead[h] = j + 2;
                    if (v.y == a[h]) lead[h] = j + 1;
                    if (v.x == a[h]) lead[h] = j;
                }
            }
            unsigned m[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                m[h] = __ballot_sync(0xffffffffu, a[h] >= 0 && lead[h] == h * 128 + tid);
                if (lane == 0) sh.warp_n[h * 4 + (tid >> 5)] = __popc(m[h]);
            }
            bar_sync(1, 128);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                int base = 0;
                for (int w = 0; w < h * 4 + (tid >> 5); ++w) base += sh.warp_n[w];
                at[h] = base + __popc(m[h] & ((1u << lane) - 1u));
                if (m[h] >> lane & 1u) {
                    seg.id[at[h]] = a[h];
                    sh.first[h * 128 + tid] = at[h];
                }
            }
            if (tid == 0) {
                int n = 0;
                for (int w = 0; w < 8; ++w) n += sh.warp_n[w];
                seg.n = n;
            }
            bar_sync(1, 128);
            const int mine = cta;
            const int my = a[mine] >= 0 ? sh.first[lead[mine]] : -1;
            const int t = tile.t0 + mine * 128 + tid;
            const float *tp = g.t + (int64_t)t * rank;
            const float scale = my >= 0 ? __ldg(d.scale + a[mine]) : 0.f;
            const bool wide = C::kWide && my >= 0 && beyond_f16(tp, scale, rank);
            RowScale rs;
            if (C::kScaled && my >= 0) rs.set(tp, scale, rank);
            seg.row[tid] = (int16_t)my;
            seg.wide[tid] = wide;
            seg.down[tid] = rs.down;
            const int ext = seg.n * rank;
            mbar_arrive(sh.seg_full + (tl & 1));
            const int live = wide ? -1 : my;
            float4 v[8];
            if (ext) load_t_row(v, live, rank, g.log2r, tp, 0);
            for (int r0 = 0; r0 < ext; r0 += kExt, tb.next(C::kTBufs)) {  // a thread that gives up here is heard at the next tile
                if (tb.wrapped && !wait_warp(sh.t_empty + tb.s, tb.phase ^ 1u, &sh.abort)) { ok = false; break; }
                store_t_row<BF, C::kParts>(v, tbuf + tb.s * C::kTTile, 16384u, tid, scale, rs.up);
                if (r0 + kExt < ext) load_t_row(v, live, rank, g.log2r, tp, r0 + kExt);
                fence_async_shared();
                __syncwarp();
                if (lane == 0) arrive_cluster(peer_addr(sh.t_full + tb.s, 0));
            }
        }
    }
    if (warp == 8 && __all_sync(kAll, ok)) ok = ring_drained(tb_last, sh.t_empty, C::kTBufs, &sh.abort);
    if (!ok) {
        atomicOr(d.err, kErrTimeout);
        sh.abort = 1;
        const unsigned long long t0 = global_ns();  // loads in flight land well within this
        while (global_ns() - t0 < 20000000ull) __nanosleep(1000);
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    cluster.sync();
    tc_fence_after();
    if (warp == 2)
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
}

}  // namespace

cudaError_t launch_adapter_wide(const AdapterArgs &g, const void *x_map, int sms, cudaStream_t s) {
    const latent_adapter_desc &d = g.d;
    const bool bf = d.type == LATENT_TYPE_BF16, kn = !(d.flags & LATENT_ADAPTER_W_TRANSPOSED);
    const bool f32 = d.y_type == LATENT_TYPE_F32;
    const int cols = f32 ? Cfg<true, true>::kCols : Cfg<true, false>::kCols;
    CUtensorMap mW, mB, mY;
    if (!(kn ? adapter_map(&mW, bf, d.w, d.n_in, d.n_out, d.ldw, kBK)
             : adapter_map(&mW, bf, d.w, d.n_out, d.n_in, d.ldw, cols / 2)) ||
        !adapter_map(&mB, bf, d.b, (uint64_t)d.n_adapter * d.rank, d.n_out, d.ldb, d.rank < kExt ? d.rank : kExt) ||
        !adapter_out_map(&mY, d.y_type, d.y, d.n_tokens, d.n_out, d.ldy, 32))
        return cudaErrorInvalidValue;
    const void *fn = f32 ? bf ? kn ? (const void *)k_ad_wide<true, true, true> : (const void *)k_ad_wide<true, false, true>
                              : kn ? (const void *)k_ad_wide<false, true, true> : (const void *)k_ad_wide<false, false, true>
                     : bf ? kn ? (const void *)k_ad_wide<true, true, false> : (const void *)k_ad_wide<true, false, false>
                          : kn ? (const void *)k_ad_wide<false, true, false> : (const void *)k_ad_wide<false, false, false>;
    cudaError_t err = ensure_smem(fn, kSmem);
    if (err != cudaSuccess) return err;
    const int64_t tiles = ((int64_t)d.n_tokens + kPairRows - 1) / kPairRows * ((d.n_out + cols - 1) / cols);
    const int pairs = tiles < sms / 2 ? (int)tiles : sms / 2;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(2 * pairs);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = kSmem;
    cfg.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    AdapterArgs a = g;
    void *args[] = {const_cast<void *>(x_map), &mW, &mB, &mY, &a};
    return cudaLaunchKernelExC(&cfg, fn, args);
}

}  // namespace latent
