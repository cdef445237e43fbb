// Low-rank adapters of many requests beside one shared projection
// (latent_adapter_project): y[t] = x[t].W + s_a (x[t].A_a).B_a, a = ids[t].
//
// Two steps: t = x[t].A_a (fp32, [T][rank] in the workspace), then a product
// kernel that adds s_a t.B_a to x.W.  This file has the entry points and
// both steps on the CUDA cores (k_ad_shrink_any, k_ad_any), for what the
// tensor-core kernels cannot read: strides of x or W that are not multiples of
// 8, unaligned rows, and the adapters' part alone (no dense W).
#include "adapter_mma.cuh"

namespace latent {

namespace {

template <typename T> __device__ __forceinline__ float ad_f32(T v);
template <> __device__ __forceinline__ float ad_f32<__half>(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float ad_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }

__device__ __forceinline__ void ad_store(void *y, int y_type, int64_t i, float v) {
    if (y_type == LATENT_TYPE_F32) static_cast<float *>(y)[i] = v;
    else if (y_type == LATENT_TYPE_F16) static_cast<__half *>(y)[i] = __float2half_rn(v);
    else static_cast<__nv_bfloat16 *>(y)[i] = __float2bfloat16_rn(v);
}
__device__ __forceinline__ float ad_load(const void *y, int y_type, int64_t i) {
    if (y_type == LATENT_TYPE_F32) return static_cast<const float *>(y)[i];
    if (y_type == LATENT_TYPE_F16) return __half2float(static_cast<const __half *>(y)[i]);
    return __bfloat162float(static_cast<const __nv_bfloat16 *>(y)[i]);
}

constexpr int kShrinkWarps = 8;

// One warp per (row, rank column): block (t, j0 / 8).
template <typename T>
__global__ void __launch_bounds__(kShrinkWarps * 32) k_ad_shrink_any(latent_adapter_desc d, float *tt) {
    const int t = blockIdx.x;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int j = blockIdx.y * kShrinkWarps + warp;
    const int a = __ldg(d.ids + t);
    if (a >= d.n_adapter && blockIdx.y == 0 && threadIdx.x == 0) atomicOr(d.err, kErrExpertId);
    if (a < 0 || a >= d.n_adapter) return;
    const T *x = static_cast<const T *>(d.x) + (int64_t)t * d.ldx;
    const T *w = static_cast<const T *>(d.a) + ((int64_t)a * d.rank + j) * d.lda;
    float s = 0.f;
    for (int k = lane; k < d.n_in; k += 32) s = fmaf(ad_f32(x[k]), ad_f32(w[k]), s);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (lane == 0) tt[(int64_t)t * d.rank + j] = s * __ldg(d.scale + a);
}

// 64 x 64 outputs per block, 4 x 4 per thread, K in steps of 16 through shared memory.
constexpr int kSB = 64, kSK = 16;

template <typename T>
__global__ void __launch_bounds__(256) k_ad_any(latent_adapter_desc d, const float *tt) {
    __shared__ float xs[kSK][kSB + 4], ws[kSK][kSB + 4];
    const int row0 = blockIdx.y * kSB, col0 = blockIdx.x * kSB;
    const int tr = threadIdx.x / 16, tc = threadIdx.x % 16;
    const T *x = static_cast<const T *>(d.x), *w = static_cast<const T *>(d.w), *b = static_cast<const T *>(d.b);
    const bool tn = d.flags & LATENT_ADAPTER_W_TRANSPOSED;
    const int64_t sk = tn ? 1 : d.ldw, sn = tn ? d.ldw : 1;
    float acc[4][4] = {};
    for (int k0 = 0; w && k0 < d.n_in; k0 += kSK) {
        for (int i = threadIdx.x; i < kSB * kSK; i += 256) {
            const int r = i / kSK, k = i % kSK;
            xs[k][r] = row0 + r < d.n_tokens && k0 + k < d.n_in ? ad_f32(x[(int64_t)(row0 + r) * d.ldx + k0 + k]) : 0.f;
            const int wk = tn ? i % kSK : i / kSB, wn = tn ? i / kSK : i % kSB;
            ws[wk][wn] = col0 + wn < d.n_out && k0 + wk < d.n_in ? ad_f32(w[(k0 + wk) * sk + (col0 + wn) * sn]) : 0.f;
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < kSK; ++k) {
            float xv[4], wv[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                xv[i] = xs[k][tr * 4 + i];
                wv[i] = ws[k][tc + 16 * i];
            }
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(xv[i], wv[j], acc[i][j]);
        }
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int t = row0 + tr * 4 + i;
        if (t >= d.n_tokens) continue;
        const int a = __ldg(d.ids + t);
        if (a >= 0 && a < d.n_adapter) {
            const float *tv = tt + (int64_t)t * d.rank;
            const T *bv = b + (int64_t)a * d.rank * d.ldb;
            for (int r = 0; r < d.rank; ++r) {
                const float s = tv[r];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int n = col0 + tc + 16 * j;
                    if (n < d.n_out) acc[i][j] = fmaf(s, ad_f32(bv[(int64_t)r * d.ldb + n]), acc[i][j]);
                }
            }
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int n = col0 + tc + 16 * j;
            if (n >= d.n_out) continue;
            const int64_t at = (int64_t)t * d.ldy + n;
            ad_store(d.y, d.y_type, at, w ? acc[i][j] : ad_load(d.y, d.y_type, at) + acc[i][j]);
        }
    }
}

// Clears the error that is being reported and no other: calls on other streams
// may record theirs between the read and this.
__global__ void k_ad_clear(uint32_t *err, uint32_t bit) { atomicAnd(err, ~bit); }

bool ad_aligned(const void *p, size_t a) { return ((uintptr_t)p % a) == 0; }

int ad_validate(const latent_adapter_desc *d) {
    if (!d) return LATENT_ERR_INVALID;
    if (d->n_adapter < 0 || d->n_in < 1 || d->n_out < 1 || d->n_tokens < 0) return LATENT_ERR_SHAPE;
    if (d->n_in > 1 << 30 || d->n_out > 1 << 30) return LATENT_ERR_SHAPE;  // tiles reach past the end in 32 bits
    if (d->rank != 16 && d->rank != 32 && d->rank != 64 && d->rank != 128) return LATENT_ERR_UNSUPPORTED;
    if (d->type != LATENT_TYPE_F16 && d->type != LATENT_TYPE_BF16) return LATENT_ERR_DTYPE;
    if (d->y_type != d->type && d->y_type != LATENT_TYPE_F32) return LATENT_ERR_DTYPE;
    if (d->flags & ~(uint32_t)LATENT_ADAPTER_W_TRANSPOSED) return LATENT_ERR_INVALID;
    return LATENT_OK;
}

// What TMA loads need: rows from 16-byte boundaries (of any width: a map ends where the matrix does), coordinates of
// 32 bits, and a grid over the columns.
bool ad_tensor_cores(const latent_adapter_desc *d) {
    return d->w && d->n_adapter > 0 && (int64_t)d->n_adapter * d->rank <= INT32_MAX && d->n_out <= 65535 * 128 &&
           (d->ldx | d->ldw | d->lda | d->ldb) % 8 == 0 && ad_aligned(d->x, 16) && ad_aligned(d->w, 16) &&
           ad_aligned(d->a, 16) && ad_aligned(d->b, 16);
}

enum AdapterPath { kPathSelf, kPathSkinny, kPathWide };

int tile_rows(int n, AdapterPath path) { return path == kPathWide || n >= adapter::kRows ? adapter::kRows : (n + 15) / 16 * 16; }

// Which kernels serve a call, by what they cost in measured steps (B200,
// bf16): k_ad_skinny takes 2 us per wave and 0.45 us (fp32 results 0.5) per 64
// of a block's share of K at 128 rows (as many bytes less at fewer), k_ad_wide
// 3 us and 0.23 us (fp32 results 0.26) per 64 of K.  An extension block of 32
// stacked rank columns, of which a batch of single tokens may need one per
// adapter and 32 ranks, costs 0.5 us (fp32 results 0.6) of one of a cluster's
// blocks, or of the pair.  E.g. skinny and wide, rank 16: 320 rows of
// 2048 x 2048 16.1 and 18.9 us, 1024 rows 26.9 and 18.3, 1024 rows of
// 7168 x 512 25.1 and 39.6; 24 adapters of rank 64 in 200 rows of
// 1024 x 14336, fp32 results: 105.0 and 87.9.  Over 187 shapes of 100 to 2048
// rows the slower of the two is taken by more than 5% on nine (bf16; 1.19 times
// at worst) and on three (fp32 results; 1.13).
// Up to 64 rows whose adapters fit one tile of 128 stacked rank columns, with
// at most 8 steps of K per block, k_ad_skinny makes x.A itself (one row of
// 1024 x 4096: 8.5 us against 10.3 in two launches, of 7168 x 2048: 15.7
// against 11.5).
AdapterPath pick_path(const AdapterArgs &g, int sms) {
    const latent_adapter_desc &d = g.d;
    AdapterArgs a = g;
    a.tile_rows = tile_rows(d.n_tokens, kPathSkinny);
    const int64_t nk = (d.n_in + 63) / 64;
    const int64_t stacked = (int64_t)(d.n_adapter < d.n_tokens ? d.n_adapter : d.n_tokens) * d.rank;
    if (d.n_tokens <= 64 && stacked <= 128) {
        const int c = adapter_self_cluster(a);
        if ((nk + c - 1) / c <= 8) return kPathSelf;
    }
    // k_ad_wide stores through TMA, which ends a row at a multiple of 16 bytes, with zeros behind the last column
    if (d.n_tokens <= 96 || (d.ldy | d.n_out) % 8 || !ad_aligned(d.y, 16)) return kPathSkinny;
    const int64_t ext = d.n_tokens <= 256 ? (stacked + 31) / 32 : 0;  // longer batches: packed prompts, few adapters a tile
    const int c = adapter_skinny_cluster(a, sms);
    const int64_t clusters = ((int64_t)d.n_tokens + 127) / 128 * ((d.n_out + 127) / 128);
    const bool f32 = d.y_type == LATENT_TYPE_F32;
    const int step = f32 ? 60 : 50;  // of an extension block; all in 10 ns
    const int64_t skinny = adapter_waves(clusters, c) * ((nk + c - 1) / c * (f32 ? 50 : 45) + (ext + c - 1) / c * step + 200);
    const int cols = f32 ? 128 : 256;
    const int64_t tiles = ((int64_t)d.n_tokens + 255) / 256 * ((d.n_out + cols - 1) / cols);
    const int64_t wide = (tiles + sms / 2 - 1) / (sms / 2) * (nk * (f32 ? 26 : 23) + ext * step) + 300;
    return wide < skinny ? kPathWide : kPathSkinny;
}

}  // namespace

}  // namespace latent

extern "C" LATENT_API int latent_adapter_workspace_size(const latent_adapter_desc *d, size_t *bytes) {
    const int st = latent::ad_validate(d);
    if (st) return st;
    if (!bytes) return LATENT_ERR_INVALID;
    *bytes = ((size_t)d->n_tokens * d->rank * 4 + 511) / 256 * 256;
    return LATENT_OK;
}

extern "C" LATENT_API int latent_adapter_project(const latent_adapter_desc *d, CUstream_st *stream) try {
    using namespace latent;
    const int st = ad_validate(d);
    if (st) return st;
    if (d->n_tokens == 0) return LATENT_OK;
    const bool tn = d->flags & LATENT_ADAPTER_W_TRANSPOSED;
    if (!d->x || !d->ids || !d->y || !d->err || !d->workspace || (d->n_adapter > 0 && (!d->a || !d->b || !d->scale)))
        return LATENT_ERR_INVALID;
    if (d->ldx < d->n_in || d->ldy < d->n_out || (d->w && d->ldw < (tn ? d->n_in : d->n_out)) ||
        (d->n_adapter > 0 && (d->lda < d->n_in || d->ldb < d->n_out)))
        return LATENT_ERR_SHAPE;
    if (!ad_aligned(d->x, 2) || !ad_aligned(d->w, 2) || !ad_aligned(d->a, 2) || !ad_aligned(d->b, 2) ||
        !ad_aligned(d->scale, 4) || !ad_aligned(d->ids, 4) || !ad_aligned(d->y, d->y_type == LATENT_TYPE_F32 ? 4 : 2) ||
        !ad_aligned(d->err, 4) || !ad_aligned(d->workspace, 256))
        return LATENT_ERR_ALIGN;
    size_t need = 0;
    latent_adapter_workspace_size(d, &need);
    if (d->workspace_bytes < need) return LATENT_ERR_WORKSPACE;
    if (d->n_tokens > 65535 * kSB) return LATENT_ERR_SHAPE;  // row tiles of the CUDA-core grid
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    float *tt = static_cast<float *>(d->workspace);
    if (ad_tensor_cores(d)) {
        int dev = 0, sms = 0;
        if (cudaGetDevice(&dev) != cudaSuccess ||
            cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
            return LATENT_ERR_CUDA;
        AdapterArgs a{};
        a.d = *d;
        a.t = tt;
        a.log2r = d->rank == 16 ? 4 : d->rank == 32 ? 5 : d->rank == 64 ? 6 : 7;
        const AdapterPath path = pick_path(a, sms);
        a.tile_rows = tile_rows(d->n_tokens, path);
        CUtensorMap x;
        if (!adapter_map(&x, d->type == LATENT_TYPE_BF16, d->x, d->n_tokens, d->n_in, d->ldx, a.tile_rows))
            return LATENT_ERR_CUDA;
        cudaError_t err = cudaSuccess;
        if (path != kPathSelf) err = launch_adapter_shrink(a, &x, s);
        if (err == cudaSuccess)
            err = path == kPathWide ? launch_adapter_wide(a, &x, sms, s) : launch_adapter_skinny(a, &x, sms, path == kPathSelf, s);
        if (err != cudaSuccess) {
            cudaGetLastError();  // not left for the caller's next check
            return LATENT_ERR_CUDA;
        }
        return LATENT_OK;
    }
    const dim3 gs((unsigned)d->n_tokens, (unsigned)d->rank / kShrinkWarps);
    const dim3 gp((unsigned)((d->n_out + kSB - 1) / kSB), (unsigned)((d->n_tokens + kSB - 1) / kSB));
    if (d->type == LATENT_TYPE_F16) {
        k_ad_shrink_any<__half><<<gs, kShrinkWarps * 32, 0, s>>>(*d, tt);
        k_ad_any<__half><<<gp, 256, 0, s>>>(*d, tt);
    } else {
        k_ad_shrink_any<__nv_bfloat16><<<gs, kShrinkWarps * 32, 0, s>>>(*d, tt);
        k_ad_any<__nv_bfloat16><<<gp, 256, 0, s>>>(*d, tt);
    }
    return cudaGetLastError() == cudaSuccess ? LATENT_OK : LATENT_ERR_CUDA;
} catch (...) {  // the tables of kernel attributes allocate on the host
    return LATENT_ERR_CUDA;
}

extern "C" LATENT_API int latent_adapter_check(uint32_t *err, CUstream_st *stream) {
    using namespace latent;
    if (!err) return LATENT_ERR_INVALID;
    uint32_t bits = 0;
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    if (cudaMemcpyAsync(&bits, err, 4, cudaMemcpyDeviceToHost, s) != cudaSuccess || cudaStreamSynchronize(s) != cudaSuccess)
        return LATENT_ERR_CUDA;
    const uint32_t bit = bits & kErrTimeout ? kErrTimeout : bits & kErrExpertId;
    if (!bit) return LATENT_OK;
    k_ad_clear<<<1, 1, 0, s>>>(err, bit);
    if (cudaGetLastError() != cudaSuccess || cudaStreamSynchronize(s) != cudaSuccess) return LATENT_ERR_CUDA;
    return bit == kErrTimeout ? LATENT_ERR_TIMEOUT : LATENT_ERR_EXPERT_ID;
}
