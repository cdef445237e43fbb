// Shared by the tensor-core kernels of the adapters (csrc/adapter_*.cu):
// operand descriptors, the list of adapters a tile of rows uses, and the
// tile of x.A parts that the extension of the contraction multiplies by B.
//
// The adapters enter a product tile as more contraction length.  For a tile
// of up to 128 rows with the distinct adapters a_0 .. a_{S-1},
//   y = [x | t^0 | .. | t^{S-1}] . [W ; B_{a_0} ; .. ; B_{a_{S-1}}]
// where t^s holds t of the rows that use a_s and zero in the others: the same
// accumulator, no second pass over y.  t (fp32) enters as 2 or 3 parts of the
// 16-bit operand type that add up to it (each part rounds what the ones
// before left: 2 parts of bf16 leave 2^-16 of t, 3 of bf16 2^-24, 2 of fp16
// 2^-22 or half a step of its subnormals, 2^-25, whichever is more), multiplied
// by the same B rows.  fp16's range is too short for that as it stands: where
// TMEM has room for another accumulator, the adapters' part goes there, each
// row's t scaled by a power of two that the epilogue takes back (RowScale);
// elsewhere the rows that do not fit are made in fp32 (beyond_f16).
#pragma once

#include "internal.h"
#include "sm100.cuh"

namespace latent {

struct AdapterArgs {
    latent_adapter_desc d;
    float *t;        // [T][rank] x.A (fp32)
    int tile_rows;   // rows per tile: 128, fewer rounded up to 16
    int log2r;       // rank = 1 << log2r
};

constexpr int kMaxCluster = 16;

// x_map: the CUtensorMap of x with a box of tile_rows rows.
cudaError_t launch_adapter_shrink(const AdapterArgs &a, const void *x_map, cudaStream_t s);
// self: with x.A in the same launch (one tile of rows).
cudaError_t launch_adapter_skinny(const AdapterArgs &a, const void *x_map, int sms, bool self, cudaStream_t s);
cudaError_t launch_adapter_wide(const AdapterArgs &a, const void *x_map, int sms, cudaStream_t s);
// What the choice between them goes by: blocks that split K (with x.A in a launch of its own, and in the same), and
// how often that many clusters have to take turns.
int adapter_skinny_cluster(const AdapterArgs &a, int sms);
int adapter_self_cluster(const AdapterArgs &a);
int adapter_waves(int64_t clusters, int cluster);

namespace adapter {

using namespace sm100;

constexpr int kBK = 64;          // contraction per stage: 128 bytes, one swizzle atom
constexpr int kRows = 128;       // rows of a tile at most (TMEM lanes or columns)

// kind::f16 with fp32 accumulation, M = 128; mn: the operand's other dimension
// (not the contraction) is the contiguous one.
__host__ __device__ constexpr uint32_t idesc(bool bf16, int n, bool a_mn, bool b_mn) {
    return (1u << 4) | ((bf16 ? 1u : 0u) << 7) | ((bf16 ? 1u : 0u) << 10) | ((a_mn ? 1u : 0u) << 15) |
           ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
}

// Operand tile stored as boxes of [64 contraction rows][64 columns] of 128
// bytes a row, 128B swizzle: 8-row atoms 1024 bytes apart (stride offset),
// the next 64 columns 8192 bytes further (leading offset).
__device__ __forceinline__ uint64_t desc_mnmajor_sw128(uint32_t saddr) {
    uint64_t d = 0;
    d |= (uint64_t)((saddr & 0x3FFFFu) >> 4);
    d |= (uint64_t)(8192 >> 4) << 16;
    d |= (uint64_t)(1024 >> 4) << 32;
    d |= (uint64_t)1 << 46;
    d |= (uint64_t)2 << 61;
    return d;
}

// Bounded wait for the phase with parity `parity`; CLUSTER: acquires what
// threads of the other blocks wrote before they arrived.  Each try suspends for
// a while; the clock is read after every 32.
template <bool CLUSTER = false>
__device__ __forceinline__ bool wait(uint64_t *bar, uint32_t parity) {
    const uint32_t a = smem_addr(bar);
    unsigned long long t0 = 0;
    for (unsigned i = 1;; ++i) {
        uint32_t done;
        if constexpr (CLUSTER)
            asm volatile(
                "{\n\t.reg .pred p;\n\t"
                "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
                "selp.u32 %0, 1, 0, p;\n\t}"
                : "=r"(done) : "r"(a), "r"(parity) : "memory");
        else
            asm volatile(
                "{\n\t.reg .pred p;\n\t"
                "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
                "selp.u32 %0, 1, 0, p;\n\t}"
                : "=r"(done) : "r"(a), "r"(parity) : "memory");
        if (done) return true;
        if ((i & 31u) == 0) {
            const unsigned long long now = global_ns();
            if (i == 32) t0 = now;
            else if (now - t0 > kWaitNs) return false;
        }
    }
}

// The loads and MMAs take their addresses and coordinates from uniform
// registers.  Issued under `lane == 0`, or with operands that the compiler
// cannot prove equal over the warp, each of them is wrapped in a loop over the
// lanes' values: about 100 cycles an instruction more (measured: a one-warp
// load loop at 315 cycles a turn against 194).  So their loops are run by whole
// warps, on values and conditions that are uniform by construction (block
// indexes, votes, shuffles from a constant lane), and only the instructions
// themselves by one elected lane, always the same.
constexpr uint32_t kAll = 0xffffffffu;
__device__ __forceinline__ bool elect() {
    uint32_t p;
    asm volatile(
        "{\n\t.reg .pred q;\n\t"
        "elect.sync _|q, 0xffffffff;\n\t"
        "selp.u32 %0, 1, 0, q;\n\t}"
        : "=r"(p));
    return p != 0;
}
__device__ __forceinline__ int uniform(int v) { return __shfl_sync(kAll, v, 0); }
__device__ __forceinline__ int warp_index() { return uniform((int)threadIdx.x >> 5); }

// By a whole warp, with one result for all lanes; false as well once *abort is set.
template <bool CLUSTER = false>
__device__ __forceinline__ bool wait_warp(uint64_t *bar, uint32_t parity, volatile int *abort) {
    const bool done = wait<CLUSTER>(bar, parity) && !*abort;
    return __all_sync(kAll, done);
}

// Position in a ring: slot and the parity of its current phase.
struct Ring {
    int s = 0;
    uint32_t phase = 0;
    bool wrapped = false;
    __device__ __forceinline__ void next(int slots) {
        if (++s == slots) {
            s = 0;
            phase ^= 1u;
            wrapped = true;
        }
    }
};

// By a whole warp, behind its last use of a ring: until the MMAs have handed
// the last slot back (commits arrive in their order).  These arrivals are made
// by the tensor core on its own; none may reach a block that has gone.
__device__ __forceinline__ bool ring_drained(const Ring &at, uint64_t *empty, int slots, volatile int *abort) {
    if (!at.wrapped && at.s == 0) return true;
    return at.s ? wait_warp(empty + at.s - 1, at.phase, abort) : wait_warp(empty + slots - 1, at.phase ^ 1u, abort);
}

__device__ __forceinline__ void fence_async_shared() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void launch_dependents() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void dependency_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void bar_sync(int id, int threads) {
    asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}

__device__ __forceinline__ bool bar_all(int id, int threads, bool v) {
    uint32_t r;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.u32 p, %3, 0;\n\t"
        "barrier.red.and.pred q, %1, %2, p;\n\t"
        "selp.u32 %0, 1, 0, q;\n\t}"
        : "=r"(r)
        : "r"(id), "r"(threads), "r"((uint32_t)v)
        : "memory");
    return r != 0;
}

// 32 lanes x 16 columns of 32-bit TMEM words into 16 registers per thread.
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&v)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
          "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
        : "r"(taddr)
        : "memory");
}

// Distinct adapters of a tile's rows, in order of first use.
struct Segments {
    alignas(16) int ids[kRows];  // scratch, read four at a time
    int id[kRows];               // the distinct adapters' ids
    int row[kRows];              // a row's index into id; -1: no adapter
    int first[kRows];
    int warp_n[4];
    int n;                       // distinct adapters
};

// A row's adapter, -1 for none (ids that no adapter has are reported and count as none).
__device__ __forceinline__ int row_adapter(const latent_adapter_desc &d, int t, bool live, bool report) {
    const int a = live ? __ldg(d.ids + t) : -1;
    if (a < d.n_adapter) return a;
    if (report) atomicOr(d.err, kErrExpertId);
    return -1;
}

// By 128 threads (tid 0..127, named barrier `bar`), a: the adapter of row tid
// (-1 behind row nt): thread i finds the first row with row i's adapter; the
// rows that are their own first are numbered.  The other warps see the result
// behind a barrier of the caller's.
__device__ __forceinline__ void build_segments(Segments &s, int a, int nt, int tid, int bar) {
    s.ids[tid] = a;
    bar_sync(bar, kRows);
    int lead = tid;
#pragma unroll 4
    for (int j = (nt - 1) & ~3; j >= 0; j -= 4) {
        const int4 v = *reinterpret_cast<const int4 *>(s.ids + j);
        if (v.w == a) lead = j + 3;
        if (v.z == a) lead = j + 2;
        if (v.y == a) lead = j + 1;
        if (v.x == a) lead = j;
    }
    const bool mine = a >= 0 && lead == tid;
    const unsigned m = __ballot_sync(0xffffffffu, mine);
    if ((tid & 31) == 0) s.warp_n[tid >> 5] = __popc(m);
    bar_sync(bar, kRows);
    int base = 0;
    for (int w = 0; w < (tid >> 5); ++w) base += s.warp_n[w];
    if (mine) {
        const int i = base + __popc(m & ((1u << (tid & 31)) - 1u));
        s.id[i] = a;
        s.first[tid] = i;
    }
    if (tid == 0) s.n = s.warp_n[0] + s.warp_n[1] + s.warp_n[2] + s.warp_n[3];
    bar_sync(bar, kRows);
    s.row[tid] = a >= 0 ? s.first[lead] : -1;
}

template <bool BF> __device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    if constexpr (BF) {
        const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
        return *reinterpret_cast<const uint32_t *>(&v);
    } else {
        const __half2 v = __floats2half2_rn(lo, hi);
        return *reinterpret_cast<const uint32_t *>(&v);
    }
}
template <bool BF> __device__ __forceinline__ float2 unpack2(uint32_t v) {
    if constexpr (BF) return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162 *>(&v));
    else return __half22float2(*reinterpret_cast<const __half2 *>(&v));
}
template <bool BF> __device__ __forceinline__ float load16(const void *p, int64_t i) {
    if constexpr (BF) return __bfloat162float(__ldg(static_cast<const __nv_bfloat16 *>(p) + i));
    else return __half2float(__ldg(static_cast<const __half *>(p) + i));
}

// The contraction of an extension block: 32 stacked B rows.
constexpr int kExt = 32;

// One row of an extension block (stacked rows r0 .. r0 + 31) in K-major
// 128B-swizzled tiles: t where the row's own segment lies, zeros elsewhere.  A
// 128-byte row holds two parts of the 32 values (a third goes to a second
// tile, tile_bytes further); what a part that is not finite leaves is zero.
// `t`: the row's x.A, taken times scale (and up, a power of two).  load_t_row fetches (one trip to L2,
// which the caller lets run under the block before), store_t_row writes.
__device__ __forceinline__ void load_t_row(float4 (&v)[8], int seg, int rank, int log2r, const float *t, int r0) {
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        const int r = r0 + 8 * c;
        const bool mine = seg >= 0 && (r >> log2r) == seg;
        const float4 *p = reinterpret_cast<const float4 *>(t + (r & (rank - 1)));
        v[2 * c] = mine ? __ldcg(p) : make_float4(0.f, 0.f, 0.f, 0.f);
        v[2 * c + 1] = mine ? __ldcg(p + 1) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
}

template <bool BF, int PARTS>
__device__ __forceinline__ void store_t_row(float4 (&v)[8], uint8_t *tile, uint32_t tile_bytes, int row, float scale,
                                            float up = 1.f) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        v[i].x = v[i].x * scale * up;
        v[i].y = v[i].y * scale * up;
        v[i].z = v[i].z * scale * up;
        v[i].w = v[i].w * scale * up;
    }
#pragma unroll
    for (int p = 0; p < PARTS; ++p)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            uint32_t q[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float &x = i & 1 ? v[2 * c + i / 2].z : v[2 * c + i / 2].x;
                float &y = i & 1 ? v[2 * c + i / 2].w : v[2 * c + i / 2].y;
                q[i] = pack2<BF>(x, y);
                if (p + 1 < PARTS) {
                    const float2 back = unpack2<BF>(q[i]);
                    x = isfinite(back.x) ? x - back.x : 0.f;
                    y = isfinite(back.y) ? y - back.y : 0.f;
                }
            }
            const int run = 4 * (p & 1) + c;
            *reinterpret_cast<uint4 *>(tile + (p >> 1) * tile_bytes + row * 128 + ((run ^ (row & 7)) * 16)) =
                make_uint4(q[0], q[1], q[2], q[3]);
        }
}
// Byte offset of part p, contraction step kk (16 values) in those tiles.
__device__ __forceinline__ uint32_t t_offset(int p, int kk, uint32_t tile_bytes) {
    return (uint32_t)(p >> 1) * tile_bytes + (uint32_t)(p & 1) * 64u + (uint32_t)kk * 32u;
}

// The largest magnitude of a row's t, and whether one is infinite or not a number.
__device__ __forceinline__ float largest(const float *t, float scale, int rank, bool &finite) {
    float most = 0.f;
    finite = true;
    for (int r = 0; r < rank; r += 4) {
        const float4 u = __ldcg(reinterpret_cast<const float4 *>(t + r));
        const float x = fabsf(u.x * scale), y = fabsf(u.y * scale), z = fabsf(u.z * scale), w = fabsf(u.w * scale);
        finite = finite && isfinite(x) && isfinite(y) && isfinite(z) && isfinite(w);
        most = fmaxf(fmaxf(most, fmaxf(x, y)), fmaxf(z, w));
    }
    return most;
}

// The power of two that takes a row's largest t to 2^14 .. 2^15, and its
// inverse: what two fp16 parts leave of a t is then 2^-22 of it or 2^-39 of the
// row's largest.  Rows of zeros, and with values that are not finite: 1.
struct RowScale {
    float up = 1.f, down = 1.f;
    __device__ __forceinline__ void set(const float *t, float scale, int rank) {
        bool finite;
        const float most = largest(t, scale, rank, finite);
        if (!finite || most == 0.f) return;
        const int e = min(141 - (int)(__float_as_uint(most) >> 23), 126);  // 14 less the exponent
        up = __uint_as_float((uint32_t)(127 + e) << 23);
        down = __uint_as_float((uint32_t)(127 - e) << 23);
    }
};

// 16-bit results of the pair kernel, whose accumulators fill TMEM: a row whose
// largest t is beyond fp16's 65504, not finite, or so small that 2^-25 is more
// than 2^-16 of it (what two bf16 parts leave) enters the tile as zeros and is
// finished in fp32 by the epilogue (2047 rows of 4096 x 4096, rank 16: 379 us
// if all rows are, 60 if none is).
__device__ __forceinline__ bool beyond_f16(const float *t, float scale, int rank) {
    bool finite;
    const float most = largest(t, scale, rank, finite);
    return !finite || most > 65504.f || (most > 0.f && most < 0x1p-9f);
}

// The adapter's part of y in column n, in fp32.
template <bool BF>
__device__ __forceinline__ float adapter_dot(const latent_adapter_desc &d, const float *t, int a, int n) {
    float s = 0.f;
    const float scale = __ldg(d.scale + a);
    const int64_t row = (int64_t)a * d.rank;
    for (int r = 0; r < d.rank; ++r) s = fmaf(__ldcg(t + r) * scale, load16<BF>(d.b, (row + r) * d.ldb + n), s);
    return s;
}

}  // namespace adapter

// The output matrix as a 2-D TMA map, a box of 128-byte rows, 128B swizzle.
bool adapter_out_map(void *map, int y_type, void *base, uint64_t rows, uint64_t cols, uint64_t ld, uint32_t box_rows);
// A row-major 16-bit matrix, likewise: a {64, box_rows} box.
bool adapter_map(void *map, bool bf16, const void *base, uint64_t rows, uint64_t cols, uint64_t ld, uint32_t box_rows);

}  // namespace latent
