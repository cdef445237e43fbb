// Training side of the router (csrc/router.cu): the load-balance and z losses
// with the per-expert counts and their gradient (latent_balance_loss), and the
// gradient of the routing weights (latent_router_grad).  The reference has no
// training code; the routing rule differentiated here is
// loader/adaptive_topk.py:29-90 with its kept set held fixed.
//
// Balance loss over packed sequences s (rows [cu[s], cu[s+1]), counted rows
// n_s, kept slots c_se, f_se = c_se / max(1, sum_e c_se), S' sequences with a
// counted row, n = sum n_s):
//   L_bal = (1/S') sum_s E sum_e f_se P_se,  P_se = (1/n_s) sum_t p_te
//   L_z   = (1/n) sum_t lse_t^2,             loss = b L_bal + z L_z
// With C_se = E f_se / (S' n_s), numbers per sequence and expert that the ids
// alone give, L_bal = sum_t D_t with D_t = sum_e C_se p_te, and
//   dloss/dl_ti = p_ti (b (C_si - D_t) + 2 z lse_t / n):
// value and gradient need the counts first and then ONE pass over the logits,
// and no per-expert probability sums.
//
// k_balance_count: one cluster of 1 to 8 blocks per sequence; each block counts its
// rows' ids in a shared-memory histogram, the blocks add theirs up through
// distributed shared memory: integers, no global atomics, nothing to zero.  It
// leaves f as well, in fp32: an integer to float conversion per column and row
// runs at a quarter of the rate.
// k_balance_main, its programmatic dependent, takes the softmax of its first
// rows before it waits for the counts: 4 to 32 lanes per row, the row in
// registers; every block leaves its two partial sums (64 bits) and the last one
// adds them up in block order, so that a call's results do not depend on the
// order of execution.
//
// Measured, 16384 rows of 256 fp32 experts, top-8, 8 sequences: both kernels in a
// graph 13.6 us with even loads, 14.4 with skewed ones; under a profiler, caches
// cold, the count 8.5 and main 15.9 (34 MB read and written; about half of its
// blocks' time is waiting on loads and shuffles).  64 rows: 6.7 to 7.5 for both.
#include <cooperative_groups.h>

#include "internal.h"

namespace latent {

namespace {

namespace cg = cooperative_groups;

constexpr int kMaxTrainExperts = 1024;  // 32 logits per lane in registers
constexpr int kMaxTrainTopK = 32;       // one lane per slot
constexpr int kCountThreads = 1024;  // at most
constexpr int kRowWarps = 8;
constexpr unsigned kFull = 0xffffffffu;

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

template <int BYTES> struct Raw;
template <> struct Raw<2> { using type = uint16_t; };
template <> struct Raw<4> { using type = uint32_t; };
template <> struct Raw<8> { using type = uint2; };
template <> struct Raw<16> { using type = uint4; };

// A row of E values held by LPR lanes, PL values each: lane l has, of each run
// of LPR * VEC columns, the VEC adjacent ones from l * VEC (one load or store of
// VEC * sizeof(T) bytes).  E is a multiple of VEC and rows are aligned to it.
template <typename T, int PL, int VEC, int LPR = 32>
struct Row {
    static constexpr int NV = PL / VEC;
    using R = typename Raw<VEC * sizeof(T)>::type;
    static __device__ __forceinline__ int col(int lane, int v) { return (v * LPR + lane) * VEC; }
    static __device__ __forceinline__ void load(const T *row, int E, int lane, float pad, float (&x)[PL]) {
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int c = col(lane, v);
            if (c < E) {
                const R raw = __ldg(reinterpret_cast<const R *>(row + c));
                const T *e = reinterpret_cast<const T *>(&raw);
#pragma unroll
                for (int i = 0; i < VEC; ++i) x[v * VEC + i] = to_f32(e[i]);
            } else {
#pragma unroll
                for (int i = 0; i < VEC; ++i) x[v * VEC + i] = pad;
            }
        }
    }
    // A row that this kernel also writes.
    static __device__ __forceinline__ void load_rw(const T *row, int E, int lane, float (&x)[PL]) {
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int c = col(lane, v);
            R raw = R();
            if (c < E) raw = *reinterpret_cast<const R *>(row + c);
            const T *e = reinterpret_cast<const T *>(&raw);
#pragma unroll
            for (int i = 0; i < VEC; ++i) x[v * VEC + i] = to_f32(e[i]);
        }
    }
    // f(j, value) for fp32 values laid out like the row (0 behind column E).
    template <typename F>
    static __device__ __forceinline__ void floats(const float *row, int E, int lane, F f) {
        constexpr int W = VEC < 4 ? VEC : 4;
        using R4 = typename Raw<W * 4>::type;
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int c = col(lane, v);
#pragma unroll
            for (int i = 0; i < VEC; i += W) {
                R4 raw = R4();
                if (c < E) raw = __ldca(reinterpret_cast<const R4 *>(row + c + i));
                const float *e = reinterpret_cast<const float *>(&raw);
#pragma unroll
                for (int u = 0; u < W; ++u) f(v * VEC + i + u, e[u]);
            }
        }
    }
    static __device__ __forceinline__ void store(T *row, int E, int lane, const float (&x)[PL]) {
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int c = col(lane, v);
            if (c < E) {
                R raw;
                T *e = reinterpret_cast<T *>(&raw);
#pragma unroll
                for (int i = 0; i < VEC; ++i) e[i] = from_f32<T>(x[v * VEC + i]);
                *reinterpret_cast<R *>(row + c) = raw;
            }
        }
    }
};

// exp(x) for x <= 0: 2^(x log2 e), the product rounded once more than expf's
// (|x| 2^-24 of the result) and two steps of the approximation, at a third of
// its instructions.
__device__ __forceinline__ float exp_neg(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x * 1.4426950408889634f));
    return r;
}

__device__ __forceinline__ void launch_dependents() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void dependency_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// Over the LANES lanes that share a row.
template <int LANES = 32>
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(kFull, v, o));
    return v;
}
template <int LANES = 32>
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) v += __shfl_xor_sync(kFull, v, o);
    return v;
}

// Rows [lo, hi) of sequence s; cu == NULL: one sequence of all T rows.  The
// borders are device data: whatever they hold, no row outside [0, T) is touched.
__device__ __forceinline__ void sequence_rows(const int32_t *cu, int s, int T, int &lo, int &hi) {
    if (!cu) {
        lo = 0;
        hi = T;
        return;
    }
    lo = min(max(__ldg(cu + s), 0), T);
    hi = min(max(__ldg(cu + s + 1), lo), T);
}

// Sequence of row t, -1 for a row before the first or behind the last.
__device__ __forceinline__ int sequence_of(const int32_t *cu, int S, int t) {
    if (!cu) return 0;
    if (t < __ldg(cu) || t >= __ldg(cu + S)) return -1;
    int lo = 0, hi = S;  // the last s with cu[s] <= t: empty sequences before it are passed over
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (__ldg(cu + mid) <= t) lo = mid; else hi = mid;
    }
    return lo;
}

struct BalanceArgs {
    const void *logits;
    const int32_t *ids;
    const uint8_t *valid;
    const int32_t *cu;
    int T, E, k, S;
    float b, z;
    const float *d_loss;  // gradient with respect to losses[0]; NULL: 1
    bool d_losses;        // and behind it those with respect to losses[1] and [2]
    float *losses;
    int32_t *counts;    // [S][E]
    void *grad;
    int32_t *seq;       // [S] counted rows
    float *share;       // [S][row pitch] each expert's share of the sequence's kept slots
    int share_ld;
    double *partial;    // [blocks][2]
    uint32_t *ticket;
};

template <int CS>
__global__ void __cluster_dims__(CS, 1, 1) __launch_bounds__(kCountThreads)
k_balance_count(BalanceArgs a) {
    __shared__ int hist[kMaxTrainExperts];
    __shared__ int tot[2];  // counted rows, kept slots of this block
    cg::cluster_group cluster = cg::this_cluster();
    const int rank = (int)cluster.block_rank();
    const int s = blockIdx.x / CS;
    launch_dependents();
    for (int e = threadIdx.x; e < a.E; e += blockDim.x) hist[e] = 0;
    if (threadIdx.x < 2) tot[threadIdx.x] = 0;
    if (blockIdx.x == 0 && threadIdx.x == 0) *a.ticket = 0u;
    __syncthreads();
    int lo, hi;
    sequence_rows(a.cu, s, a.T, lo, hi);
    const int per = (hi - lo + CS - 1) / CS;
    const int r0 = min(hi, lo + rank * per), r1 = min(hi, r0 + per);
    int rows = 0, slots = 0;
    const int end = r1 * a.k;
    for (int i = r0 * a.k + threadIdx.x; i < end; i += 4 * blockDim.x) {
        int e[4];  // four loads on the way at once
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int at = i + u * blockDim.x;
            e[u] = at < end && (!a.valid || __ldg(a.valid + at / a.k)) ? __ldg(a.ids + at) : -1;
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            if (e[u] >= 0 && e[u] < a.E) {
                atomicAdd(&hist[e[u]], 1);
                ++slots;
            }
        }
    }
    if (a.valid) {
        for (int t = r0 + threadIdx.x; t < r1; t += blockDim.x) rows += __ldg(a.valid + t) != 0;
    } else if (threadIdx.x == 0) {
        rows = r1 - r0;
    }
    rows = __reduce_add_sync(kFull, rows);
    slots = __reduce_add_sync(kFull, slots);
    if ((threadIdx.x & 31) == 0) {
        if (rows) atomicAdd(&tot[0], rows);
        if (slots) atomicAdd(&tot[1], slots);
    }
    cluster.sync();
    // lanes 2q and 2q + 1 have block q's rows and slots: sums over even and over odd lanes
    int all = (threadIdx.x & 31) < 2 * CS ? cluster.map_shared_rank(tot, (threadIdx.x & 31) >> 1)[threadIdx.x & 1] : 0;
#pragma unroll
    for (int o = 16; o > 1; o >>= 1) all += __shfl_xor_sync(kFull, all, o);
    const int counted = __shfl_sync(kFull, all, 0), kept = __shfl_sync(kFull, all, 1);
    const float inv = 1.f / (float)max(1, kept);
    const int step = (a.E + CS - 1) / CS;
    const int e0 = rank * step, e1 = min(a.E, e0 + step);
    for (int e = e0 + threadIdx.x; e < e1; e += blockDim.x) {
        int c = 0;
#pragma unroll
        for (int q = 0; q < CS; ++q) c += *cluster.map_shared_rank(&hist[e], q);
        a.counts[(int64_t)s * a.E + e] = c;
        a.share[(int64_t)s * a.share_ld + e] = (float)c * inv;
    }
    if (rank == 0 && threadIdx.x == 0) a.seq[s] = counted;
    cluster.sync();  // the others' shared memory stays until every block has read it
}

constexpr int kBalanceWarps = 4;
// One turn of resident blocks that loop over the rows: none starts behind the
// counts' wait and the launch of the others (65536 rows of 64 experts 15.9 us,
// 20.6 with 16 blocks per SM, 20.0 with 4).
constexpr int kBalanceBlocksPerSm = 7;

// LPR lanes per row: the sums over a row, its logarithm, its divisions and its
// place among the sequences cost instructions per group of lanes, so few lanes
// with up to 32 values each take fewer of them per row than a whole warp.
template <typename T, int PL, int VEC, int LPR>
__global__ void __launch_bounds__(kBalanceWarps * 32, kBalanceBlocksPerSm) k_balance_main(BalanceArgs a) {
    using RW = Row<T, PL, VEC, LPR>;
    constexpr int kRows = 32 / LPR;  // rows of a warp
    __shared__ double part[kBalanceWarps][2];
    __shared__ bool last;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, sub = lane % LPR;
    const T *logits = static_cast<const T *>(a.logits);
    T *grad = static_cast<T *>(a.grad);
    bool first = true;
    int used = 0;    // sequences that have a counted row
    int64_t n = 0;   // counted rows
    float gb = 0.f, gz = 0.f;
    double sb = 0.0, sz = 0.0;
    for (int t0 = (blockIdx.x * kBalanceWarps + warp) * kRows; first || t0 < a.T; t0 += gridDim.x * kBalanceWarps * kRows) {
        const int t = t0 + lane / LPR;
        float x[PL];
        RW::load(logits + (int64_t)t * a.E, t < a.T ? a.E : 0, sub, -INFINITY, x);
        const int seq = t >= a.T || (a.valid && !__ldg(a.valid + t)) ? -1 : sequence_of(a.cu, a.S, t);
        float m = -INFINITY;
#pragma unroll
        for (int j = 0; j < PL; ++j) m = fmaxf(m, x[j]);
        m = warp_max<LPR>(m);
        bool nan = false;
        if (m == -INFINITY) {
#pragma unroll
            for (int j = 0; j < PL; ++j) nan |= x[j] != x[j];
        }
        nan = warp_max<LPR>(nan ? 1.f : 0.f) != 0.f;
        // a padded row, whatever it holds, gives nothing and gets a zero gradient; so does one with every expert masked
        const bool none = seq < 0 || (m == -INFINITY && !nan);
        if (none) {
            m = 0.f;
#pragma unroll
            for (int j = 0; j < PL; ++j) x[j] = -INFINITY;
        }
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < PL; ++j) {
            x[j] = exp_neg(x[j] - m);
            sum += x[j];
        }
        sum = warp_sum<LPR>(sum);
        const float inv = none ? 0.f : 1.f / sum;
        const float lse = none ? 0.f : m + logf(sum);
        if (first) {  // the counts are needed only now
            first = false;
            dependency_wait();
            for (int s = lane; s < a.S; s += 32) {
                const int c = __ldcg(a.seq + s);
                n += c;
                used += c > 0;
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) n += __shfl_xor_sync(kFull, n, o);
            used = __reduce_add_sync(kFull, used);
            const float up = a.d_loss ? __ldg(a.d_loss) : 1.f;
            gb = up * a.b;
            gz = n > 0 ? up * (2.f * a.z / (float)n) : 0.f;
            if (a.d_losses) {
                gb += __ldg(a.d_loss + 1);
                if (n > 0) gz += __ldg(a.d_loss + 2) * (2.f / (float)n);
            }
        }
        const int rows = __ldcg(a.seq + max(seq, 0));
        const float scale = seq >= 0 ? (float)a.E / ((float)used * (float)rows) : 0.f;  // C = scale * share
        const float *share = a.share + (int64_t)max(seq, 0) * a.share_ld;
        const int cols = seq >= 0 ? a.E : 0;
        float d = 0.f;
        RW::floats(share, cols, sub, [&](int j, float c) { d = fmaf(c, x[j], d); });
        d = warp_sum<LPR>(d) * (inv * scale);
        if (sub == 0) {
            sb += d;
            sz += (double)lse * lse;
        }
        if (grad && t < a.T) {  // the shares once more, from L1: kept, they would cost a register per column
            const float ca = gb * scale * inv, cb = inv * (gz * lse - gb * d);
            RW::floats(share, cols, sub, [&](int j, float c) { x[j] *= fmaf(ca, c, cb); });
            RW::store(grad + (int64_t)t * a.E, a.E, sub, x);
        }
    }
#pragma unroll
    for (int o = 16; o >= LPR; o >>= 1) {
        sb += __shfl_xor_sync(kFull, sb, o);
        sz += __shfl_xor_sync(kFull, sz, o);
    }
    if (lane == 0) {
        part[warp][0] = sb;
        part[warp][1] = sz;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        double b = 0.0, z = 0.0;
        for (int w = 0; w < kBalanceWarps; ++w) {
            b += part[w][0];
            z += part[w][1];
        }
        reinterpret_cast<double2 *>(a.partial)[blockIdx.x] = make_double2(b, z);
        uint32_t done;  // releases the partial sums, acquires the others'
        asm volatile("atom.acq_rel.gpu.global.add.u32 %0, [%1], 1;" : "=r"(done) : "l"(a.ticket) : "memory");
        last = done == gridDim.x - 1;
    }
    __syncthreads();
    if (!last) return;
    // thread i adds blocks i, i + 128, ... in order, then lanes and warps by a fixed tree
    double b = 0.0, z = 0.0;
#pragma unroll 8
    for (int i = threadIdx.x; i < (int)gridDim.x; i += kBalanceWarps * 32) {
        const double2 v = __ldcg(reinterpret_cast<const double2 *>(a.partial) + i);
        b += v.x;
        z += v.y;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        b += __shfl_xor_sync(kFull, b, o);
        z += __shfl_xor_sync(kFull, z, o);
    }
    if (lane == 0) {
        part[warp][0] = b;
        part[warp][1] = z;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        b = z = 0.0;
        for (int w = 0; w < kBalanceWarps; ++w) {
            b += part[w][0];
            z += part[w][1];
        }
        z = n > 0 ? z / (double)n : 0.0;
        a.losses[0] = (float)(a.b * b + a.z * z);
        a.losses[1] = (float)b;
        a.losses[2] = (float)z;
    }
}

// Gradient of the routing weights.  Slot j of row t (id i_j, kept when
// 0 <= i_j < E) has the weight w_j = s_j, or s_j / sum_kept s with RENORM; the
// scores s are given (SOFTMAX: as logits).  With c = sum_kept dw_j w_j:
//   scores: ds_j = (dw_j - c) / sum_kept s with RENORM, else dw_j;
//   logits, RENORM: the softmax's own sum cancels, w is the softmax over the
//     kept logits alone and dl_j = w_j (dw_j - c), zero elsewhere;
//   logits, raw: dl_i = p_i (dw_i - c) over the whole row.
// An id held by several slots of a row gets the sum of their parts.  ACCUM adds
// to what dscores holds.
__device__ __forceinline__ float same_id_sum(int key, float g, unsigned &same) {
    same = __match_any_sync(kFull, key);
    if (!__any_sync(kFull, (same & (same - 1)) != 0u)) return g;
    float total = 0.f;  // in slot order
    for (unsigned rest = same; __any_sync(kFull, rest != 0u);) {
        const int src = rest ? __ffs(rest) - 1 : 0;
        const float add = __shfl_sync(kFull, g, src);
        if (rest) total += add;
        rest &= rest - 1;
    }
    return total;
}

// All forms but the raw logits: the kept scores alone decide, the rest of a row
// is zero (ACCUM: left alone).  A warp has 32 / kw rows side by side, kw = the
// power of two that holds top_k: lane = slot.  The rows' zeros are stored first
// (they wait for nothing), the kept columns after a __syncwarp.
// Measured: 16384 rows of 256 fp32 experts, top-8: 5.9 us, 18.4 MB, 3.1 TB/s
// (write bound); 64 rows 2.6.
template <typename T, bool WIDE, bool SOFTMAX, bool RENORM, bool ACCUM>
__global__ void __launch_bounds__(kRowWarps * 32) k_router_grad_kept(const T *__restrict__ scores,
                                                                     const int32_t *__restrict__ ids,
                                                                     const float *__restrict__ dw, int T_, int E,
                                                                     int k, int log2kw, T *__restrict__ out) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int kw = 1 << log2kw, rows = 32 >> log2kw;
    const int64_t t0 = ((int64_t)blockIdx.x * kRowWarps + warp) * rows;
    if (t0 >= T_) return;
    const int group = lane >> log2kw, slot = lane & (kw - 1);
    const int64_t t = t0 + group;
    const bool have = t < T_ && slot < k;
    int id = have ? __ldg(ids + t * k + slot) : -1;
    const bool kept = id >= 0 && id < E;
    const float d = kept ? __ldg(dw + t * k + slot) : 0.f;
    if (!ACCUM) {
        T *o = out + t0 * E;
        const int64_t n = (T_ - t0 < rows ? T_ - t0 : rows) * E;
        if (WIDE) {
            constexpr int W = 16 / (int)sizeof(T);
            for (int64_t i = (int64_t)lane * W; i < n; i += 32 * W)
                *reinterpret_cast<uint4 *>(o + i) = make_uint4(0u, 0u, 0u, 0u);
        } else {
            for (int64_t i = lane; i < n; i += 32) o[i] = from_f32<T>(0.f);
        }
    }
    const float v = kept && (SOFTMAX || RENORM) ? to_f32(__ldg(scores + t * E + id)) : 0.f;
    const float old = ACCUM && kept ? to_f32(out[t * E + id]) : 0.f;
    auto sum = [&](float x) {
        for (int o = kw >> 1; o > 0; o >>= 1) x += __shfl_xor_sync(kFull, x, o);
        return x;
    };
    float g = d;
    if (SOFTMAX) {  // w: the softmax over the kept logits
        float m = kept ? v : -INFINITY;
        for (int o = kw >> 1; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(kFull, m, o));
        const float e = kept ? expf(v - m) : 0.f;
        const float total = sum(e);
        const float w = kept ? e / total : 0.f;
        g = w * (d - sum(w * d));
    } else if (RENORM) {
        const float total = sum(v);
        const float c = sum(kept ? v / total * d : 0.f);
        g = kept ? (d - c) / total : 0.f;
    }
    unsigned same;
    g = same_id_sum(kept ? group * kMaxTrainExperts + id : -1 - lane, g, same);  // (also orders the zeros before the rest)
    __syncwarp();
    if (kept && lane == __ffs(same) - 1) out[t * E + id] = from_f32<T>(old + g);
}

// Raw weights of logits: dl_i = p_i (dw_i - c) over the whole row.  LPR lanes
// per row, as in k_balance_main, and no fewer than top_k: lane = slot; the row
// is written as -c p_i, then the kept columns.
// Measured: 9001 rows of 160 bf16 experts 3.7 us, 5.4 with a warp per row; 65536
// rows of 64 fp32 experts 8.7 (34 MB, 3.9 TB/s) and 23.4; of 256 24.8, 5.4 TB/s.
template <typename T, int PL, int VEC, int LPR, bool ACCUM>
__global__ void __launch_bounds__(kRowWarps * 32) k_router_grad_raw(const T *__restrict__ scores,
                                                                    const int32_t *__restrict__ ids,
                                                                    const float *__restrict__ dw, int T_, int E, int k,
                                                                    T *__restrict__ out) {
    using RW = Row<T, PL, VEC, LPR>;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, group = lane / LPR, sub = lane % LPR;
    const int64_t t0 = ((int64_t)blockIdx.x * kRowWarps + warp) * (32 / LPR), t = t0 + group;
    if (t0 >= T_) return;
    const int cols = t < T_ ? E : 0;
    const T *row = scores + t * E;
    T *o = out + t * E;
    const int id = sub < k && t < T_ ? __ldg(ids + t * k + sub) : -1;
    const bool kept = id >= 0 && id < E;
    const float d = kept ? __ldg(dw + t * k + sub) : 0.f;
    const unsigned of_row = LPR == 32 ? kFull : ((1u << (LPR & 31)) - 1u) << (group * LPR);
    const bool any = __ballot_sync(kFull, kept) & of_row;
    const float v = kept ? to_f32(__ldg(row + id)) : 0.f, old = ACCUM && kept ? to_f32(o[id]) : 0.f;
    float x[PL];
    RW::load(row, cols, sub, -INFINITY, x);
    float m = -INFINITY;
#pragma unroll
    for (int j = 0; j < PL; ++j) m = fmaxf(m, x[j]);
    m = warp_max<LPR>(m);
    float sum = 0.f;
#pragma unroll
    for (int j = 0; j < PL; ++j) {
        x[j] = expf(x[j] - m);
        sum += x[j];
    }
    sum = warp_sum<LPR>(sum);
    const float p = kept ? expf(v - m) / sum : 0.f;
    const float c = warp_sum<LPR>(d * p);
    const float cn = -c / sum;
    float y[PL];
    if (ACCUM) RW::load_rw(o, cols, sub, y);
#pragma unroll
    for (int j = 0; j < PL; ++j) x[j] = (any ? x[j] * cn : 0.f) + (ACCUM ? y[j] : 0.f);
    unsigned same;
    const float g = same_id_sum(kept ? group * kMaxTrainExperts + id : -1 - lane, p * d, same);
    __syncwarp();
    RW::store(o, cols, sub, x);
    __syncwarp();
    if (kept && lane == __ffs(same) - 1) o[id] = from_f32<T>(old + (g - c * p));  // p (sum of its slots' dw - c)
}

bool is_aligned(const void *p, size_t a) { return ((uintptr_t)p % a) == 0; }
size_t round256(size_t x) { return (x + 255) / 256 * 256; }

int sm_count(int *sms) {
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess ||
        cudaDeviceGetAttribute(sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
        return LATENT_ERR_CUDA;
    return LATENT_OK;
}

constexpr int kMaxBalanceBlocks = 4096;  // partial sums in the workspace

struct BalanceLayout {
    size_t seq, share, partial, ticket, total;
    int share_ld;
};
BalanceLayout balance_layout(int S, int E) {
    BalanceLayout L;
    L.share_ld = (E + 3) / 4 * 4;  // rows of 16 bytes' multiples
    L.seq = 0;
    L.share = round256((size_t)S * 4);
    L.partial = L.share + round256((size_t)S * L.share_ld * 4);
    L.ticket = L.partial + (size_t)kMaxBalanceBlocks * 16;
    L.total = L.ticket + 256;
    return L;
}

template <typename T, int PL, int LPR>
cudaError_t launch_balance_rows(const BalanceArgs &a, bool vec, int sms, cudaStream_t s) {
    constexpr int V = 16 / (int)sizeof(T);
    constexpr int rows = kBalanceWarps * (32 / LPR);
    int blocks = (a.T + rows - 1) / rows;
    const int most = sms * kBalanceBlocksPerSm < kMaxBalanceBlocks ? sms * kBalanceBlocksPerSm : kMaxBalanceBlocks;
    blocks = blocks < 1 ? 1 : blocks > most ? most : blocks;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(blocks);
    cfg.blockDim = dim3(kBalanceWarps * 32);
    cfg.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    return vec && a.E % V == 0 ? cudaLaunchKernelEx(&cfg, k_balance_main<T, PL, V, LPR>, a)
                               : cudaLaunchKernelEx(&cfg, k_balance_main<T, PL, 1, LPR>, a);
}

template <typename T>
int launch_balance(const BalanceArgs &a, int sms, cudaStream_t s) {
    const bool vec = is_aligned(a.logits, 16) && is_aligned(a.grad, 16);
    cudaError_t err;
    if (a.E <= 32) err = launch_balance_rows<T, 8, 4>(a, vec, sms, s);
    else if (a.E <= 64) err = launch_balance_rows<T, 8, 8>(a, vec, sms, s);
    else if (a.E <= 128) err = launch_balance_rows<T, 16, 8>(a, vec, sms, s);
    else if (a.E <= 192) err = launch_balance_rows<T, 24, 8>(a, vec, sms, s);
    else if (a.E <= 256) err = launch_balance_rows<T, 32, 8>(a, vec, sms, s);
    else if (a.E <= 512) err = launch_balance_rows<T, 32, 16>(a, vec, sms, s);
    else err = launch_balance_rows<T, 32, 32>(a, vec, sms, s);
    if (err == cudaSuccess) return LATENT_OK;
    cudaGetLastError();  // not left for the caller's next check
    return LATENT_ERR_CUDA;
}

template <typename T, bool SOFTMAX, bool RENORM>
int launch_kept(const T *scores, const int32_t *ids, const float *dw, int n, int E, int k, bool accum, T *out,
                cudaStream_t s) {
    int log2kw = 0;
    while ((1 << log2kw) < k) ++log2kw;
    const int rows = kRowWarps * (32 >> log2kw);
    const unsigned g = (unsigned)((n + rows - 1) / rows);
    const bool wide = E * sizeof(T) % 16 == 0 && is_aligned(out, 16);
    if (accum)
        k_router_grad_kept<T, false, SOFTMAX, RENORM, true><<<g, kRowWarps * 32, 0, s>>>(scores, ids, dw, n, E, k, log2kw, out);
    else if (wide)
        k_router_grad_kept<T, true, SOFTMAX, RENORM, false><<<g, kRowWarps * 32, 0, s>>>(scores, ids, dw, n, E, k, log2kw, out);
    else
        k_router_grad_kept<T, false, SOFTMAX, RENORM, false><<<g, kRowWarps * 32, 0, s>>>(scores, ids, dw, n, E, k, log2kw, out);
    return cudaGetLastError() == cudaSuccess ? LATENT_OK : LATENT_ERR_CUDA;
}

template <typename T, int PL, int LPR>
int launch_raw(const latent_router_grad_desc &d, bool vec, cudaStream_t s) {
    constexpr int V = 16 / (int)sizeof(T), rows = kRowWarps * (32 / LPR);
    const T *sc = static_cast<const T *>(d.scores);
    T *o = static_cast<T *>(d.d_scores);
    const int n = d.n_tokens, E = d.n_expert, k = d.top_k;
    const unsigned g = (unsigned)((n + rows - 1) / rows);
    const bool accum = d.flags & LATENT_ROUTER_ACCUMULATE;
    vec = vec && E % V == 0;
    if (vec && accum) k_router_grad_raw<T, PL, V, LPR, true><<<g, kRowWarps * 32, 0, s>>>(sc, d.ids, d.d_weights, n, E, k, o);
    else if (vec) k_router_grad_raw<T, PL, V, LPR, false><<<g, kRowWarps * 32, 0, s>>>(sc, d.ids, d.d_weights, n, E, k, o);
    else if (accum) k_router_grad_raw<T, PL, 1, LPR, true><<<g, kRowWarps * 32, 0, s>>>(sc, d.ids, d.d_weights, n, E, k, o);
    else k_router_grad_raw<T, PL, 1, LPR, false><<<g, kRowWarps * 32, 0, s>>>(sc, d.ids, d.d_weights, n, E, k, o);
    return cudaGetLastError() == cudaSuccess ? LATENT_OK : LATENT_ERR_CUDA;
}

template <typename T>
int launch_router_grad(const latent_router_grad_desc &d, cudaStream_t s) {
    const T *sc = static_cast<const T *>(d.scores);
    T *o = static_cast<T *>(d.d_scores);
    const int32_t *ids = d.ids;
    const float *dw = d.d_weights;
    const int n = d.n_tokens, E = d.n_expert, k = d.top_k;
    const uint32_t flags = d.flags;
    const bool softmax = flags & LATENT_ROUTER_SOFTMAX, renorm = flags & LATENT_ROUTER_RENORMALIZE;
    const bool accum = flags & LATENT_ROUTER_ACCUMULATE;
    if (softmax && renorm) return launch_kept<T, true, true>(sc, ids, dw, n, E, k, accum, o, s);
    if (renorm) return launch_kept<T, false, true>(sc, ids, dw, n, E, k, accum, o, s);
    if (!softmax) return launch_kept<T, false, false>(sc, ids, dw, n, E, k, accum, o, s);
    const bool vec = is_aligned(sc, 16) && is_aligned(o, 16);
    if (k <= 8) {
        if (E <= 32 && k <= 4) return launch_raw<T, 8, 4>(d, vec, s);
        if (E <= 64) return launch_raw<T, 8, 8>(d, vec, s);
        if (E <= 128) return launch_raw<T, 16, 8>(d, vec, s);
        if (E <= 256) return launch_raw<T, 32, 8>(d, vec, s);
    }
    if (E <= 256) return launch_raw<T, 8, 32>(d, vec, s);
    if (E <= 512 && k <= 16) return launch_raw<T, 32, 16>(d, vec, s);
    return launch_raw<T, 32, 32>(d, vec, s);
}

bool float_type(int t) { return t == LATENT_TYPE_F32 || t == LATENT_TYPE_F16 || t == LATENT_TYPE_BF16; }
size_t type_size(int t) { return t == LATENT_TYPE_F32 ? 4 : 2; }

int train_shape(int32_t T, int32_t E, int32_t k) {
    if (T < 0 || E < 1 || k < 1) return LATENT_ERR_SHAPE;
    if ((int64_t)T * k > (int64_t)1 << 30) return LATENT_ERR_SHAPE;
    if (E > kMaxTrainExperts) return LATENT_ERR_UNSUPPORTED;
    return LATENT_OK;
}

}  // namespace

}  // namespace latent

extern "C" LATENT_API int latent_balance_workspace_size(const latent_balance_desc *d, size_t *bytes) {
    if (!d || !bytes) return LATENT_ERR_INVALID;
    if (d->n_sequences < 1 || d->n_expert < 1) return LATENT_ERR_SHAPE;
    *bytes = latent::balance_layout(d->n_sequences, d->n_expert).total;
    return LATENT_OK;
}

extern "C" LATENT_API int latent_balance_loss(const latent_balance_desc *d, CUstream_st *stream) {
    using namespace latent;
    if (!d) return LATENT_ERR_INVALID;
    int st = train_shape(d->n_tokens, d->n_expert, d->top_k);
    if (st) return st;
    if (d->n_sequences < 1 || (d->n_sequences > 1 && !d->cu_seqlens)) return LATENT_ERR_SHAPE;
    if (!float_type(d->type)) return LATENT_ERR_DTYPE;
    const bool d_losses = d->flags & LATENT_BALANCE_D_LOSSES;
    if ((d->flags & ~(uint32_t)LATENT_BALANCE_D_LOSSES) || (d_losses && !d->d_loss) || !d->losses || !d->counts || !d->workspace || (d->n_tokens > 0 && (!d->logits || !d->ids)))
        return LATENT_ERR_INVALID;
    const size_t es = type_size(d->type);
    if (!is_aligned(d->logits, es) || !is_aligned(d->grad, es) || !is_aligned(d->ids, 4) ||
        !is_aligned(d->cu_seqlens, 4) || !is_aligned(d->d_loss, 4) || !is_aligned(d->losses, 4) ||
        !is_aligned(d->counts, 4) || !is_aligned(d->workspace, 256))
        return LATENT_ERR_ALIGN;
    const BalanceLayout L = balance_layout(d->n_sequences, d->n_expert);
    if (d->workspace_bytes < L.total) return LATENT_ERR_WORKSPACE;
    int sms = 0;
    if ((st = sm_count(&sms))) return st;
    char *ws = static_cast<char *>(d->workspace);
    const BalanceArgs a{d->logits, d->ids, d->valid, d->cu_seqlens, d->n_tokens, d->n_expert, d->top_k, d->n_sequences,
                        d->balance_coef, d->z_coef, d->d_loss, d_losses, d->losses, d->counts, d->grad,
                        reinterpret_cast<int32_t *>(ws + L.seq), reinterpret_cast<float *>(ws + L.share), L.share_ld,
                        reinterpret_cast<double *>(ws + L.partial), reinterpret_cast<uint32_t *>(ws + L.ticket)};
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    // as many blocks for a sequence as run at once (both kernels in a graph: 16384 rows of 256 experts in 8 sequences
    // 13.5 us with 8 blocks each, 15.1 with one; 16384 of 64 in 1024 sequences 67.8 and 16.7), of 1024 threads where each
    // has many ids (65536 rows of 128 experts in one sequence 27.2 us, 35.1 with 512; 9001 of 160 in 37 12.0 and 10.8)
    const unsigned S = (unsigned)d->n_sequences;
    const int share = sms / d->n_sequences;
    const int cluster = share >= 8 ? 8 : share >= 4 ? 4 : share >= 2 ? 2 : 1;
    const int threads = (int64_t)d->n_tokens * d->top_k / S / cluster >= 8 * kCountThreads ? kCountThreads : kCountThreads / 2;
    if (cluster == 8) k_balance_count<8><<<8 * S, threads, 0, s>>>(a);
    else if (cluster == 4) k_balance_count<4><<<4 * S, threads, 0, s>>>(a);
    else if (cluster == 2) k_balance_count<2><<<2 * S, threads, 0, s>>>(a);
    else k_balance_count<1><<<S, threads, 0, s>>>(a);
    if (cudaGetLastError() != cudaSuccess) return LATENT_ERR_CUDA;
    switch (d->type) {
        case LATENT_TYPE_F32: return launch_balance<float>(a, sms, s);
        case LATENT_TYPE_F16: return launch_balance<__half>(a, sms, s);
        default: return launch_balance<__nv_bfloat16>(a, sms, s);
    }
}

extern "C" LATENT_API int latent_router_grad(const latent_router_grad_desc *d, CUstream_st *stream) {
    using namespace latent;
    if (!d) return LATENT_ERR_INVALID;
    const int st = train_shape(d->n_tokens, d->n_expert, d->top_k);
    if (st) return st;
    if (d->reserved ||
        (d->flags & ~(uint32_t)(LATENT_ROUTER_RENORMALIZE | LATENT_ROUTER_SOFTMAX | LATENT_ROUTER_ACCUMULATE)))
        return LATENT_ERR_INVALID;
    if (!float_type(d->type)) return LATENT_ERR_DTYPE;
    if (d->top_k > kMaxTrainTopK) return LATENT_ERR_UNSUPPORTED;
    if (d->n_tokens == 0) return LATENT_OK;
    if (!d->scores || !d->ids || !d->d_weights || !d->d_scores) return LATENT_ERR_INVALID;
    const size_t es = type_size(d->type);
    if (!is_aligned(d->scores, es) || !is_aligned(d->d_scores, es) || !is_aligned(d->ids, 4) ||
        !is_aligned(d->d_weights, 4))
        return LATENT_ERR_ALIGN;
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    switch (d->type) {
        case LATENT_TYPE_F32: return launch_router_grad<float>(*d, s);
        case LATENT_TYPE_F16: return launch_router_grad<__half>(*d, s);
        default: return launch_router_grad<__nv_bfloat16>(*d, s);
    }
}
