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
// before left: 2 parts of bf16 leave 2^-16 of t, of fp16 2^-22, 3 of bf16
// 2^-24), multiplied by the same B rows.
#pragma once

#include "internal.h"
#include "sm100.cuh"

namespace latent {

struct AdapterArgs {
    latent_adapter_desc d;
    float *t;        // [T][rank] scale * x.A (fp32)
    int tile_rows;   // rows per tile: 128, fewer rounded up to 16
};

cudaError_t launch_adapter_shrink(const AdapterArgs &a, int sms, cudaStream_t s);
cudaError_t launch_adapter_skinny(const AdapterArgs &a, int sms, cudaStream_t s);
cudaError_t launch_adapter_wide(const AdapterArgs &a, int sms, cudaStream_t s);

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

// Distinct adapters of a tile's rows, in order of first use.
struct Segments {
    alignas(16) int ids[kRows];  // scratch, read four at a time
    int id[kRows];               // the distinct adapters' ids
    int row[kRows];              // a row's index into id; -1: no adapter
    int first[kRows];
    int warp_n[4];
    int n;                       // distinct adapters
};

// By 128 threads (tid 0..127, named barrier `bar`): thread i finds the first
// row with row i's adapter; the rows that are their own first are numbered.
__device__ __forceinline__ void build_segments(Segments &s, const latent_adapter_desc &d, int t0, int nt, int tid,
                                               int bar, bool report) {
    int a = tid < nt ? __ldg(d.ids + t0 + tid) : -1;
    if (a >= d.n_adapter) {
        if (report) atomicOr(d.err, kErrExpertId);
        a = -1;
    }
    s.ids[tid] = a;
    bar_sync(bar, kRows);
    int lead = tid;
#pragma unroll 4
    for (int j = kRows - 4; j >= 0; j -= 4) {
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
    bar_sync(bar, kRows);
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

// Eight values of t as PARTS 16-byte runs of the operand type that add up to
// them; what a part that is not finite leaves is zero.
template <bool BF, int PARTS>
__device__ __forceinline__ void split_t(const float *t, uint4 (&out)[PARTS]) {
    const float4 u = __ldcg(reinterpret_cast<const float4 *>(t)), w = __ldcg(reinterpret_cast<const float4 *>(t) + 1);
    float2 v[4] = {{u.x, u.y}, {u.z, u.w}, {w.x, w.y}, {w.z, w.w}};
#pragma unroll
    for (int p = 0; p < PARTS; ++p) {
        uint32_t q[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            q[i] = pack2<BF>(v[i].x, v[i].y);
            const float2 back = unpack2<BF>(q[i]);
            v[i].x = isfinite(back.x) ? v[i].x - back.x : 0.f;
            v[i].y = isfinite(back.y) ? v[i].y - back.y : 0.f;
        }
        out[p] = make_uint4(q[0], q[1], q[2], q[3]);
    }
}

// One row of an extension block (stacked B rows r0 .. r0 + 8 CHUNKS - 1) in a
// K-major 128B-swizzled tile: t where the row's own segment lies, zeros
// elsewhere.  Part p of chunk c goes to 16-byte run c of tile p (CHUNKS 8), or
// to run 4 p + c of one tile (CHUNKS 4).
template <bool BF, int PARTS, int CHUNKS>
__device__ __forceinline__ void build_t_row(uint8_t *tile, uint32_t part_bytes, int row, int seg, int rank,
                                            const float *t, int r0) {
#pragma unroll 2
    for (int c = 0; c < CHUNKS; ++c) {
        const int r = r0 + 8 * c;
        uint4 out[PARTS];
#pragma unroll
        for (int p = 0; p < PARTS; ++p) out[p] = make_uint4(0u, 0u, 0u, 0u);
        if (seg >= 0 && r / rank == seg) split_t<BF, PARTS>(t + r % rank, out);
#pragma unroll
        for (int p = 0; p < PARTS; ++p) {
            const int run = CHUNKS == 8 ? c : CHUNKS * p + c;
            *reinterpret_cast<uint4 *>(tile + (CHUNKS == 8 ? p * part_bytes : 0u) + row * 128 + ((run ^ (row & 7)) * 16)) = out[p];
        }
    }
}

// fp16 parts reach 65504.  A row whose t goes further (or is not a number)
// enters the tile as zeros and is finished in fp32 by the epilogue.
__device__ __forceinline__ bool beyond_f16(const float *t, int rank) {
    bool in = true;
    for (int r = 0; r < rank; r += 4) {
        const float4 u = __ldcg(reinterpret_cast<const float4 *>(t + r));
        in = in && fabsf(u.x) <= 65504.f && fabsf(u.y) <= 65504.f && fabsf(u.z) <= 65504.f && fabsf(u.w) <= 65504.f;
    }
    return !in;
}

template <bool BF>
__device__ __forceinline__ float adapter_dot(const latent_adapter_desc &d, const float *t, int a, int n) {
    float s = 0.f;
    const int64_t row = (int64_t)a * d.rank;
    for (int r = 0; r < d.rank; ++r) s = fmaf(__ldcg(t + r), load16<BF>(d.b, (row + r) * d.ldb + n), s);
    return s;
}

}  // namespace adapter

// A row-major 16-bit matrix as a 2-D TMA map with a {64, box_rows} box, 128B swizzle.
bool adapter_map(void *map, bool bf16, const void *base, uint64_t rows, uint64_t cols, uint64_t ld, uint32_t box_rows);

}  // namespace latent
