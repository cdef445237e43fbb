// The adapters' product for prompt-sized batches: y = x.W + the adapters'
// part, tiles of 256 rows x 256 columns on pairs of SMs (tcgen05 cta_group::2).
//
// Persistent, one cluster of two blocks per tile at a time.  Each block holds
// 128 rows of x and 128 columns of W per stage (32 KB, a ring of 5) and the
// 128 x 256 half of the accumulator in TMEM, twice, so that the epilogue of
// one tile runs under the MMAs of the next.  Per block: warp 0 loads (TMA,
// plain per-block loads that complete on the leader's barrier), warp 1 of the
// leader issues the pair's MMAs, warps 4..7 drain accumulators, warps 8..11
// list the adapters of the tile's 256 rows and build the x.A parts of the
// extension blocks (32 stacked B rows each: both parts side by side in one
// 128-byte row).
//
// A pair tile costs 512 cycles of MMA per 64 of K against 64 KB of loads: half
// the L2 traffic per operation of one block working alone.
#include <cooperative_groups.h>
#include <cuda.h>

#include "adapter_mma.cuh"

namespace latent {

namespace {

namespace cg = cooperative_groups;
using namespace adapter;

constexpr int kThreads = 384;
constexpr int kStages = 5;
constexpr int kPairRows = 256, kPairCols = 256;
constexpr uint32_t kStage = 32768;             // 16 KB of x, 16 KB of W
constexpr uint32_t kTTile = 16384;             // 128 rows x (2 parts x 32) of x.A
constexpr int kParts = 2;
constexpr int kGroupM = 8;                     // row tiles that share a sweep over the columns (L2 reuse)
// All of an SM's shared memory, more than the ring needs: the block takes all
// TMEM columns, and no other block that wants some may start beside it.
constexpr size_t kStatic = 6144;
constexpr size_t kSmem = 227 * 1024 - kStatic;
static_assert(1024 + kStages * kStage + 2 * kTTile <= kSmem, "ring and x.A tiles");

struct PairSegments {
    int n;
    int id[kPairRows];
    int16_t row[128];     // of this block's rows
    uint8_t wide[128];    // fp16: finished in fp32 by the epilogue
};

struct Shared {
    uint64_t full[kStages], empty[kStages];
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
__device__ __forceinline__ void arrive_cluster(uint32_t bar) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
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

struct Tile {
    int t0, n0;
};
// Tiles in sweeps of kGroupM row tiles: all columns of one sweep before the next.
__device__ __forceinline__ Tile tile_at(int i, int tm, int tn) {
    const int per = kGroupM * tn, g = i / per, first = g * kGroupM;
    const int rows = min(kGroupM, tm - first), j = i - g * per;
    return {(first + j % rows) * kPairRows, (j / rows) * kPairCols};
}

// M = 256 over the pair.
__host__ __device__ constexpr uint32_t idesc_pair(bool bf16, bool b_mn) {
    return (1u << 4) | ((bf16 ? 1u : 0u) << 7) | ((bf16 ? 1u : 0u) << 10) | ((b_mn ? 1u : 0u) << 16) |
           ((uint32_t)(kPairCols >> 3) << 17) | ((uint32_t)(kPairRows >> 4) << 24);
}

template <bool BF, bool KN>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
k_ad_wide(const __grid_constant__ CUtensorMap mX, const __grid_constant__ CUtensorMap mW,
          const __grid_constant__ CUtensorMap mB, AdapterArgs g) {
    extern __shared__ uint8_t raw[];
    uint8_t *ring = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
    uint8_t *tbuf = ring + kStages * kStage;
    __shared__ Shared sh;
    cg::cluster_group cluster = cg::this_cluster();
    const int cta = blockIdx.x & 1;  // its rank in the cluster
    const int warp = warp_index(), lane = threadIdx.x & 31;
    const latent_adapter_desc &d = g.d;
    const int rank = d.rank;
    const int tm = (d.n_tokens + kPairRows - 1) / kPairRows, tn = (d.n_out + kPairCols - 1) / kPairCols;
    const int tiles = tm * tn, pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
    const int nk = (d.n_in + kBK - 1) / kBK;

    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s) {
            mbar_init(sh.full + s, 1);
            mbar_init(sh.empty + s, 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(sh.acc_full + b, 1);
            mbar_init(sh.acc_empty + b, 256);  // the epilogue threads of both blocks
            mbar_init(sh.t_full + b, 256);     // the builders of both
            mbar_init(sh.t_empty + b, 1);
            mbar_init(sh.seg_full + b, 128);
            mbar_init(sh.seg_empty + b, 130);  // loader, MMA warp and epilogue threads of this block
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
    const uint32_t tmem = sh.tmem;
    bool ok = true;

    if (warp == 0) {
        // ---------------- loads ----------------
        Ring at;
        int tl = 0;
        const uint32_t full0 = peer_addr(sh.full, 0);
        for (int i = pair; i < tiles && ok; i += pairs, ++tl) {
            const Tile tile = tile_at(i, tm, tn);
            const int row = tile.t0 + cta * 128, col = tile.n0 + cta * 128;
            for (int k = 0; k < nk; ++k, at.next(kStages)) {
                if (at.wrapped && !wait_warp(sh.empty + at.s, at.phase ^ 1u, &sh.abort)) { ok = false; break; }
                if (elect()) {
                    uint8_t *st = ring + at.s * kStage;
                    const uint32_t bar = full0 + at.s * 8;
                    if (cta == 0) mbar_arrive_expect_tx(sh.full + at.s, 2 * kStage);
                    load_pair(st, &mX, k * kBK, row, bar);
                    if (KN) {
                        load_pair(st + 16384, &mW, col, k * kBK, bar);
                        load_pair(st + 16384 + 8192, &mW, col + 64, k * kBK, bar);
                    } else {
                        load_pair(st + 16384, &mW, k * kBK, col, bar);
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
                    uint8_t *st = ring + at.s * kStage + 16384;
                    const uint32_t bar = full0 + at.s * 8;
                    if (cta == 0) mbar_arrive_expect_tx(sh.full + at.s, (uint32_t)rows * 512u);
                    load_pair(st, &mB, col, src0, bar);
                    load_pair(st + 8192, &mB, col + 64, src0, bar);
                    if (box < rows) {
                        load_pair(st + 2048, &mB, col, src1, bar);
                        load_pair(st + 8192 + 2048, &mB, col + 64, src1, bar);
                    }
                }
            }
            if (ok && lane == 0) mbar_arrive(sh.seg_empty + (tl & 1));
        }
    } else if (warp == 1) {
        // ---------------- MMAs (the leader's warp, for both blocks) ----------------
        Ring at, tb;
        int tl = 0;
        constexpr uint32_t id = idesc_pair(BF, KN), idx = idesc_pair(BF, true);
        for (int i = pair; i < tiles && ok; i += pairs, ++tl) {
            const int b = tl & 1;
            const uint32_t acc = tmem + (uint32_t)b * 256u;
            if (cta == 0) {
                if (tl >= 2 && !wait_warp<true>(sh.acc_empty + b, (uint32_t)((tl >> 1) - 1) & 1u, &sh.abort)) { ok = false; break; }
                tc_fence_after();
                for (int k = 0; k < nk; ++k, at.next(kStages)) {
                    if (!wait_warp(sh.full + at.s, at.phase, &sh.abort)) { ok = false; break; }
                    tc_fence_after();
                    if (elect()) {
                        const uint32_t x = smem_addr(ring + at.s * kStage), w = x + 16384u;
#pragma unroll
                        for (int kk = 0; kk < 4; ++kk)
                            mma_pair(acc, desc_kmajor_sw128(x + kk * 32),
                                     KN ? desc_mnmajor_sw128(w + kk * 2048) : desc_kmajor_sw128(w + kk * 32), id, k | kk);
                        commit_pair(sh.empty + at.s);
                    }
                }
                if (!ok) break;
            }
            if (!wait_warp(sh.seg_full + b, (uint32_t)(tl >> 1) & 1u, &sh.abort)) { ok = false; break; }
            const int ext = uniform(sh.seg[b].n) * rank;
            if (cta == 0) {
                for (int r0 = 0; r0 < ext; r0 += kExt, at.next(kStages), tb.next(2)) {
                    if (!wait_warp(sh.full + at.s, at.phase, &sh.abort) ||
                        !wait_warp<true>(sh.t_full + tb.s, tb.phase, &sh.abort)) { ok = false; break; }
                    tc_fence_after();
                    if (elect()) {
                        const uint32_t w = smem_addr(ring + at.s * kStage) + 16384u, t = smem_addr(tbuf + tb.s * kTTile);
                        const int steps = min(kExt / 16, (ext - r0) / 16);
                        for (int kk = 0; kk < steps; ++kk)
#pragma unroll
                            for (int q = 0; q < kParts; ++q)
                                mma_pair(acc, desc_kmajor_sw128(t + t_offset(q, kk, 0u)), desc_mnmajor_sw128(w + kk * 2048), idx, 1);
                        commit_pair(sh.empty + at.s);
                        commit_pair(sh.t_empty + tb.s);
                    }
                }
                if (!ok) break;
                if (elect()) commit_pair(sh.acc_full + b);
            }
            if (lane == 0) mbar_arrive(sh.seg_empty + b);
        }
        if (!ok && cta == 0 && elect()) {
            commit_pair(sh.acc_full);  // lets the waiting epilogues go on to the abort flag
            commit_pair(sh.acc_full + 1);
        }
    } else if (warp >= 4 && warp < 8) {
        // ---------------- epilogue: lane = row ----------------
        const int r = threadIdx.x - 128;
        int tl = 0;
        for (int i = pair; i < tiles; i += pairs, ++tl) {
            const int b = tl & 1;
            const Tile tile = tile_at(i, tm, tn);
            if (!wait(sh.seg_full + b, (uint32_t)(tl >> 1) & 1u) ||
                !wait(sh.acc_full + b, (uint32_t)(tl >> 1) & 1u) || sh.abort) { ok = false; break; }
            tc_fence_after();
            const int t = tile.t0 + cta * 128 + r;
            const bool live = t < d.n_tokens;
            const bool wide = !BF && sh.seg[b].wide[r];
            const int a = wide ? sh.seg[b].id[sh.seg[b].row[r]] : 0;
            const uint32_t acc = tmem + (uint32_t)b * 256u + ((uint32_t)(r & ~31) << 16);
            uint16_t *y = static_cast<uint16_t *>(d.y) + (int64_t)t * d.ldy + tile.n0;
#pragma unroll 1
            for (int c = 0; c < kPairCols; c += 32) {
                uint32_t v[32];
                __syncwarp();
                tmem_ld32(acc + (uint32_t)c, v);
                tmem_ld_wait();
                if (live) {
                    if (!BF && wide) {
#pragma unroll
                        for (int j = 0; j < 32; ++j)
                            if (tile.n0 + c + j < d.n_out)
                                v[j] = __float_as_uint(__uint_as_float(v[j]) +
                                                       adapter_dot<BF>(d, g.t + (int64_t)t * rank, a, tile.n0 + c + j));
                    }
#pragma unroll
                    for (int j = 0; j < 32; j += 8) {
                        uint4 o;
                        o.x = pack2<BF>(__uint_as_float(v[j]), __uint_as_float(v[j + 1]));
                        o.y = pack2<BF>(__uint_as_float(v[j + 2]), __uint_as_float(v[j + 3]));
                        o.z = pack2<BF>(__uint_as_float(v[j + 4]), __uint_as_float(v[j + 5]));
                        o.w = pack2<BF>(__uint_as_float(v[j + 6]), __uint_as_float(v[j + 7]));
                        if (tile.n0 + c + j < d.n_out) *reinterpret_cast<uint4 *>(y + c + j) = o;
                    }
                }
            }
            tc_fence_before();
            arrive_cluster(peer_addr(sh.acc_empty + b, 0));
            mbar_arrive(sh.seg_empty + b);
        }
    } else if (warp >= 8) {
        // ---------------- adapters of the tile, x.A parts ----------------
        const int tid = threadIdx.x - 256;
        int tl = 0, eb = 0;
        dependency_wait();
        for (int i = pair; i < tiles; i += pairs, ++tl) {
            const Tile tile = tile_at(i, tm, tn);
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
            const bool wide = !BF && my >= 0 && beyond_f16(tp, scale, rank);
            seg.row[tid] = (int16_t)my;
            seg.wide[tid] = wide;
            const int ext = seg.n * rank;
            mbar_arrive(sh.seg_full + (tl & 1));
            const int live = wide ? -1 : my;
            float4 v[8];
            if (ext) load_t_row(v, live, rank, g.log2r, tp, 0);
            for (int r0 = 0; r0 < ext; r0 += kExt, ++eb) {  // a thread that gives up here is heard at the next tile
                if (eb >= 2 && !wait(sh.t_empty + (eb & 1), (uint32_t)((eb >> 1) - 1) & 1u)) { ok = false; break; }
                if (sh.abort) { ok = false; break; }
                store_t_row<BF, kParts>(v, tbuf + (eb & 1) * kTTile, 0u, tid, scale);
                if (r0 + kExt < ext) load_t_row(v, live, rank, g.log2r, tp, r0 + kExt);
                fence_async_shared();
                arrive_cluster(peer_addr(sh.t_full + (eb & 1), 0));
            }
        }
    }
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
    CUtensorMap mW, mB;
    if (!(kn ? adapter_map(&mW, bf, d.w, d.n_in, d.n_out, d.ldw, kBK) : adapter_map(&mW, bf, d.w, d.n_out, d.n_in, d.ldw, 128)) ||
        !adapter_map(&mB, bf, d.b, (uint64_t)d.n_adapter * d.rank, d.n_out, d.ldb,
                     d.rank < kExt ? d.rank : kExt))
        return cudaErrorInvalidValue;
    const void *fn = bf ? kn ? (const void *)k_ad_wide<true, true> : (const void *)k_ad_wide<true, false>
                        : kn ? (const void *)k_ad_wide<false, true> : (const void *)k_ad_wide<false, false>;
    cudaError_t err = ensure_smem(fn, kSmem);
    if (err != cudaSuccess) return err;
    const int64_t tiles = ((int64_t)d.n_tokens + kPairRows - 1) / kPairRows * ((d.n_out + kPairCols - 1) / kPairCols);
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
    void *args[] = {const_cast<void *>(x_map), &mW, &mB, &a};
    return cudaLaunchKernelExC(&cfg, fn, args);
}

}  // namespace latent
