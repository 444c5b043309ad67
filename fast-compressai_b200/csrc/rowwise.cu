// rowwise.cu -- layer norm, activations and 8-bit checkpoints of the pointwise
// layers (include/fcai_layers.h).  All of them are bound by memory: the work
// is to touch every byte once, in 16-byte accesses.
//
// Two ways through a [rows][channels] matrix:
//   * strips: a CTA takes 128 channels (one 8-bit block, 16 lanes of 8) and
//     walks down its share of the rows, 16 rows at a time; sums over rows stay
//     in registers, meet in shared memory, and leave as one partial row per
//     CTA, which colsum_kernel adds in a fixed order (the same bits every run);
//   * rows: a CTA takes whole rows, for sums over channels.
#include <cuda_runtime.h>

#include <algorithm>

#include "layers_common.cuh"

namespace rw {

using namespace ly;

constexpr int kThreads = 256;
constexpr int kBlock = FCAI_KEEP_BLOCK;
constexpr int kRowsIter = kThreads / 16;  // rows a strip CTA handles at a time

// Eight channels from col on (zeros past the row's end).
template <typename T>
__device__ __forceinline__ void load8(const T *row, int col, int n, bool vec, float (&v)[8]) {
    if (vec) {
        if (col < n) Vec8<T>::load(row + col, v);
        else
            for (int i = 0; i < 8; ++i) v[i] = 0.f;
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = col + i < n ? to_f32(row[col + i]) : 0.f;
    }
}
template <typename T>
__device__ __forceinline__ void store8(T *row, int col, int n, bool vec, const float (&v)[8]) {
    if (vec) {
        if (col < n) Vec8<T>::store(row + col, v);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (col + i < n) row[col + i] = from_f32<T>(v[i]);
    }
}
__device__ __forceinline__ void load_codes(const uint8_t *row, int col, int n, bool vec, uint32_t &lo, uint32_t &hi) {
    lo = hi = 0;
    if (vec) {
        if (col < n) {
            const uint2 q = __ldg(reinterpret_cast<const uint2 *>(row + col));
            lo = q.x, hi = q.y;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (col + i < n) (i < 4 ? lo : hi) |= (uint32_t)row[col + i] << (8 * (i & 3));
    }
}
__device__ __forceinline__ void store_codes(uint8_t *row, int col, int n, bool vec, uint32_t lo, uint32_t hi) {
    if (vec) {
        if (col < n) *reinterpret_cast<uint2 *>(row + col) = make_uint2(lo, hi);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (col + i < n) row[col + i] = (uint8_t)((i < 4 ? lo : hi) >> (8 * (i & 3)));
    }
}

// What a backward pass reads x from.
struct Kept {
    const void *x;
    int64_t ldx;
    const uint8_t *codes;
    const float *scales;
    int keep;
};
template <typename T>
__device__ __forceinline__ void load_kept(const Kept &k, int64_t row, int col, int n, int nblk, bool vec, float (&v)[8]) {
    if (k.keep == FCAI_KEEP_FULL) {
        load8(static_cast<const T *>(k.x) + row * k.ldx, col, n, vec, v);
    } else {
        uint32_t lo, hi;
        load_codes(k.codes + row * n, col, n, vec, lo, hi);
        const float s = col < n ? __ldg(k.scales + row * nblk + col / kBlock) : 0.f;
        if (k.keep == FCAI_KEEP_E4M3) {
            decode4<true>(lo, s, v);
            decode4<true>(hi, s, v + 4);
        } else {
            decode4<false>(lo, s, v);
            decode4<false>(hi, s, v + 4);
        }
    }
}

// A block's codes and scale, from the 16 lanes that hold its channels (8 each).
template <bool kE4m3>
__device__ __forceinline__ void keep_block(const float (&v)[8], uint8_t *codes_row, float *scale, int col, int n, bool vec) {
    float amax = fabsf(v[0]);
#pragma unroll
    for (int i = 1; i < 8; ++i) amax = max_nan(amax, fabsf(v[i]));
#pragma unroll
    for (int d = 8; d >= 1; d >>= 1) amax = max_nan(amax, __shfl_xor_sync(0xffffffffu, amax, d));
    const float s = block_scale<kE4m3>(amax);
    const float inv = __frcp_rn(s);
    store_codes(codes_row, col, n, vec, encode4<kE4m3>(v, inv), encode4<kE4m3>(v + 4, inv));
    if ((threadIdx.x & 15) == 0 && col < n) *scale = s;
}

__device__ __forceinline__ void act8(int kind, const float (&x)[8], float (&y)[8]) {
    switch (kind) {
        case FCAI_ACT_RELU:
#pragma unroll
            for (int i = 0; i < 8; ++i) y[i] = act<FCAI_ACT_RELU>(x[i]);
            break;
        case FCAI_ACT_GELU:
#pragma unroll
            for (int i = 0; i < 8; ++i) y[i] = act<FCAI_ACT_GELU>(x[i]);
            break;
        case FCAI_ACT_SILU:
#pragma unroll
            for (int i = 0; i < 8; ++i) y[i] = act<FCAI_ACT_SILU>(x[i]);
            break;
        default:
#pragma unroll
            for (int i = 0; i < 8; ++i) y[i] = x[i];
    }
}
__device__ __forceinline__ void act_grad8(int kind, const float (&x)[8], float (&g)[8]) {
    switch (kind) {
        case FCAI_ACT_RELU:
#pragma unroll
            for (int i = 0; i < 8; ++i) g[i] *= act_grad<FCAI_ACT_RELU>(x[i]);
            break;
        case FCAI_ACT_GELU:
#pragma unroll
            for (int i = 0; i < 8; ++i) g[i] *= act_grad<FCAI_ACT_GELU>(x[i]);
            break;
        case FCAI_ACT_SILU:
#pragma unroll
            for (int i = 0; i < 8; ++i) g[i] *= act_grad<FCAI_ACT_SILU>(x[i]);
            break;
        default: break;
    }
}

// ---- activation forward, checkpoint load -------------------------------------
// One (row, block) per 16 lanes and step.
template <typename T>
__global__ void __launch_bounds__(kThreads)
    act_forward_kernel(const T *__restrict__ x, int64_t ldx, T *__restrict__ y, int64_t ldy, uint8_t *__restrict__ codes,
                       float *__restrict__ scales, int64_t rows, int n, int nblk, int act, int keep, int vec) {
    const int64_t items = rows * nblk;
    const int64_t step = (int64_t)gridDim.x * kRowsIter;
    // both halves of a warp run the same number of steps: the shuffles of a block need the whole warp
    for (int64_t base = (int64_t)blockIdx.x * kRowsIter + (threadIdx.x >> 5) * 2; base < items; base += step) {
        const int64_t it = base + ((threadIdx.x >> 4) & 1);
        const bool in = it < items;
        const int64_t row = in ? it / nblk : 0;
        const int blk = (int)(it - row * nblk);
        const int col = in ? blk * kBlock + (threadIdx.x & 15) * 8 : n;
        float v[8];
        load8(x + row * ldx, col, n, vec, v);
        if (keep == FCAI_KEEP_INT8) keep_block<false>(v, codes + row * n, scales + it, col, n, vec);
        else if (keep == FCAI_KEEP_E4M3) keep_block<true>(v, codes + row * n, scales + it, col, n, vec);
        if (y) {
            float o[8];
            act8(act, v, o);
            store8(y + row * ldy, col, n, vec, o);
        }
    }
}

template <typename T>
__global__ void __launch_bounds__(kThreads)
    checkpoint_load_kernel(Kept k, T *__restrict__ out, int64_t ldo, int64_t rows, int n, int nblk, int vec) {
    const int64_t items = rows * nblk;
    for (int64_t it = (int64_t)blockIdx.x * kRowsIter + (threadIdx.x >> 4); it < items; it += (int64_t)gridDim.x * kRowsIter) {
        const int64_t row = it / nblk;
        const int col = (int)(it - row * nblk) * kBlock + (threadIdx.x & 15) * 8;
        float v[8];
        load_kept<T>(k, row, col, n, nblk, vec, v);
        store8(out + row * ldo, col, n, vec, v);
    }
}

// ---- strips --------------------------------------------------------------------
// Adds the 16 row groups' sums of a strip CTA and writes its partial row.
__device__ __forceinline__ void strip_sums(const float (&acc)[8], float *partial_row, int col, int n, float (*sh)[kBlock]) {
    const int g = threadIdx.x >> 4, l = threadIdx.x & 15;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; ++i) sh[g][l * 8 + i] = acc[i];
    __syncthreads();
    if (threadIdx.x < kBlock) {
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < kRowsIter; ++i) s += sh[i][threadIdx.x];
        const int c = col - l * 8 + threadIdx.x;
        if (c < n) partial_row[c] = s;
    }
}

// dx = dy act'(x); grid (strips, row shares)
template <typename T>
__global__ void __launch_bounds__(kThreads)
    act_backward_kernel(const T *__restrict__ dy, int64_t lddy, Kept k, T *__restrict__ dx, int64_t lddx,
                        float *__restrict__ partial, int64_t rows, int n, int nblk, int act, int vec) {
    __shared__ float sh[kRowsIter][kBlock];
    const int col = blockIdx.x * kBlock + (threadIdx.x & 15) * 8;
    float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    for (int64_t row = (int64_t)blockIdx.y * kRowsIter + (threadIdx.x >> 4); row < rows; row += (int64_t)gridDim.y * kRowsIter) {
        float g[8], x[8];
        load8(dy + row * lddy, col, n, vec, g);
        if (act != FCAI_ACT_NONE) {
            load_kept<T>(k, row, col, n, nblk, vec, x);
            act_grad8(act, x, g);
        }
        if (dx) store8(dx + row * lddx, col, n, vec, g);
#pragma unroll
        for (int i = 0; i < 8; ++i) acc[i] += g[i];
    }
    if (partial) strip_sums(acc, partial + (int64_t)blockIdx.y * n, col, n, sh);
}

// out[c] = sum over the partial rows, in order.
template <typename T>
__global__ void colsum_kernel(const float *__restrict__ partial, int rows, int64_t stride, T *__restrict__ out, int n) {
    const int c = blockIdx.x * blockDim.x + threadIdx.x;
    if (c >= n) return;
    float s = 0.f;
    for (int r = 0; r < rows; ++r) s += partial[r * stride + c];
    out[c] = from_f32<T>(s);
}

// ---- layer norm ----------------------------------------------------------------
// Sums over the CTA; every thread gets them.
__device__ __forceinline__ float2 block_sum2(float a, float b, float2 *sh) {
#pragma unroll
    for (int d = 16; d >= 1; d >>= 1) {
        a += __shfl_xor_sync(0xffffffffu, a, d);
        b += __shfl_xor_sync(0xffffffffu, b, d);
    }
    __syncthreads();  // the previous sums have been read
    if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = make_float2(a, b);
    __syncthreads();
    float2 s = make_float2(0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) s.x += sh[w].x, s.y += sh[w].y;
    return s;
}
struct Affine {
    const void *w, *b;
    int f32, vec;
};
template <typename T>
__device__ __forceinline__ void load_affine(const Affine &a, const void *p, int col, int n, float dflt, float (&v)[8]) {
    if (!p) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = dflt;
    } else if (a.f32) {
        load8(static_cast<const float *>(p), col, n, a.vec, v);
    } else {
        load8(static_cast<const T *>(p), col, n, a.vec, v);
    }
}

// A CTA per row; the row is read three times (from cache after the first).
template <typename T>
__global__ void __launch_bounds__(kThreads)
    norm_forward_kernel(const T *__restrict__ x, int64_t ldx, Affine af, T *__restrict__ y, int64_t ldy,
                        float *__restrict__ mean_out, float *__restrict__ rstd_out, uint8_t *__restrict__ codes,
                        float *__restrict__ scales, int64_t rows, int n, int nblk, float eps, int keep, int vec) {
    __shared__ float2 sh[kThreads / 32];
    for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
        const T *xr = x + row * ldx;
        float s = 0.f, v[8];
        for (int col = threadIdx.x * 8; col < n; col += kThreads * 8) {
            load8(xr, col, n, vec, v);
#pragma unroll
            for (int i = 0; i < 8; ++i) s += v[i];
        }
        const float mean = block_sum2(s, 0.f, sh).x / n;
        s = 0.f;
        for (int col = threadIdx.x * 8; col < n; col += kThreads * 8) {
            load8(xr, col, n, vec, v);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float d = col + i < n ? v[i] - mean : 0.f;
                s = fmaf(d, d, s);
            }
        }
        const float rstd = 1.f / sqrtf(block_sum2(s, 0.f, sh).x / n + eps);
        if (threadIdx.x == 0 && mean_out) {
            mean_out[row] = mean;
            rstd_out[row] = rstd;
        }
        // whole warps stay in the loop: a block's shuffles need them
        for (int c0 = (threadIdx.x & ~31) * 8; c0 < n; c0 += kThreads * 8) {
            const int col = c0 + (threadIdx.x & 31) * 8;
            load8(xr, col, n, vec, v);
            float *sc = scales + row * nblk + col / kBlock;
            if (keep == FCAI_KEEP_INT8) keep_block<false>(v, codes + row * n, sc, col, n, vec);
            else if (keep == FCAI_KEEP_E4M3) keep_block<true>(v, codes + row * n, sc, col, n, vec);
            float w[8], b[8];
            load_affine<T>(af, af.w, col, n, 1.f, w);
            load_affine<T>(af, af.b, col, n, 0.f, b);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = fmaf((v[i] - mean) * rstd, w[i], b[i]);
            store8(y + row * ldy, col, n, vec, v);
        }
    }
}

// Per row: mean(t), mean(t xhat) into stats.
template <typename T>
__global__ void __launch_bounds__(kThreads)
    norm_backward_stats_kernel(const T *__restrict__ dy, int64_t lddy, Kept k, const float *__restrict__ mean,
                               const float *__restrict__ rstd, Affine af, float2 *__restrict__ stats, int64_t rows, int n,
                               int nblk, int vec) {
    __shared__ float2 sh[kThreads / 32];
    for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
        const float mu = mean[row], rs = rstd[row];
        float s1 = 0.f, s2 = 0.f;
        for (int col = threadIdx.x * 8; col < n; col += kThreads * 8) {
            float g[8], x[8], w[8];
            load8(dy + row * lddy, col, n, vec, g);
            load_kept<T>(k, row, col, n, nblk, vec, x);
            load_affine<T>(af, af.w, col, n, 1.f, w);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float t = g[i] * w[i];  // zero past the row's end: g is
                s1 += t;
                s2 = fmaf(t, (x[i] - mu) * rs, s2);
            }
        }
        const float2 s = block_sum2(s1, s2, sh);
        if (threadIdx.x == 0) stats[row] = make_float2(s.x / n, s.y / n);
    }
}

template <typename T>
__global__ void __launch_bounds__(kThreads)
    norm_backward_strip_kernel(const T *__restrict__ dy, int64_t lddy, Kept k, const float *__restrict__ mean,
                               const float *__restrict__ rstd, Affine af, const float2 *__restrict__ stats,
                               T *__restrict__ dx, int64_t lddx, float *__restrict__ partial, int64_t rows, int n, int nblk,
                               int vec) {
    __shared__ float sh[kRowsIter][kBlock];
    const int col = blockIdx.x * kBlock + (threadIdx.x & 15) * 8;
    float w[8], aw[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}, ab[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    load_affine<T>(af, af.w, col, n, 1.f, w);
    for (int64_t row = (int64_t)blockIdx.y * kRowsIter + (threadIdx.x >> 4); row < rows; row += (int64_t)gridDim.y * kRowsIter) {
        const float mu = mean[row], rs = rstd[row];
        const float2 m = stats[row];
        float g[8], x[8], o[8];
        load8(dy + row * lddy, col, n, vec, g);
        load_kept<T>(k, row, col, n, nblk, vec, x);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float xh = (x[i] - mu) * rs;
            o[i] = rs * (g[i] * w[i] - m.x - xh * m.y);
            aw[i] = fmaf(g[i], xh, aw[i]);
            ab[i] += g[i];
        }
        if (dx) store8(dx + row * lddx, col, n, vec, o);
    }
    if (partial) {
        float *pr = partial + (int64_t)blockIdx.y * 2 * n;
        strip_sums(aw, pr, col, n, sh);
        strip_sums(ab, pr + n, col, n, sh);
    }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------

static int64_t round256(int64_t v) { return (v + 255) / 256 * 256; }
static int blocks_of(int n) { return (n + kBlock - 1) / kBlock; }
static bool codes_vec(const void *codes, int n) { return !codes || ((reinterpret_cast<uintptr_t>(codes) & 7) == 0 && n % 8 == 0); }

// CTAs down the rows for `strips` strips: about 4 per SM in all, none without rows.
static int row_shares(int64_t rows, int strips) {
    const int64_t want = std::max<int64_t>(1, ((int64_t)fcai::sm_count() * 4 + strips - 1) / strips);
    return (int)std::max<int64_t>(1, std::min<int64_t>({want, (rows + kRowsIter - 1) / kRowsIter, 65535}));
}
static int64_t act_workspace(int64_t rows, int n) { return round256((int64_t)row_shares(rows, blocks_of(n)) * n * 4); }
static int64_t norm_workspace(int64_t rows, int n) {
    return round256(rows * 8) + round256((int64_t)row_shares(rows, blocks_of(n)) * 2 * n * 4);
}

static int check_sizes(const char *op, int64_t rows, int n, int dtype) {
    if (dtype < FCAI_DTYPE_BF16 || dtype > FCAI_DTYPE_F32) return fcai::fail(FCAI_ERR_INVALID, "%s: unknown dtype %d", op, dtype);
    if (rows < 0 || rows > 0x7FFFFFFF || n < 1 || n > (1 << 24))
        return fcai::fail(FCAI_ERR_INVALID, "%s: sizes out of range (rows %lld, channels %d)", op, (long long)rows, n);
    return FCAI_OK;
}
static bool bad_matrix(const void *p, int64_t ld, int n, int dtype) {
    return ld < n || ld > (1ll << 36) || (reinterpret_cast<uintptr_t>(p) & (dtype_size(dtype) - 1));
}
// x as the backward calls take it
static int check_kept(const char *op, const Kept &k, int64_t rows, int n, int dtype) {
    if (k.keep == FCAI_KEEP_FULL) {
        if (bad_matrix(k.x, k.ldx, n, dtype) || (rows && !k.x)) return fcai::fail(FCAI_ERR_INVALID, "%s: bad x", op);
    } else if (k.keep == FCAI_KEEP_INT8 || k.keep == FCAI_KEEP_E4M3) {
        if ((rows && (!k.codes || !k.scales)) || (reinterpret_cast<uintptr_t>(k.scales) & 3))
            return fcai::fail(FCAI_ERR_INVALID, "%s: bad codes or scales", op);
    } else {
        return fcai::fail(FCAI_ERR_INVALID, "%s: unknown keep %d", op, k.keep);
    }
    return FCAI_OK;
}
static int check_ws(const char *op, int64_t need, const void *ws, int64_t bytes) {
    if (need > 0 && (!ws || bytes < need || (reinterpret_cast<uintptr_t>(ws) & 255)))
        return fcai::fail(FCAI_ERR_WORKSPACE, "%s: needs a 256-byte aligned workspace of %lld bytes", op, (long long)need);
    return FCAI_OK;
}
static int item_grid(int64_t rows, int nblk) {
    return (int)std::max<int64_t>(1, std::min<int64_t>((rows * nblk + kRowsIter - 1) / kRowsIter, (int64_t)fcai::sm_count() * 8));
}
static int colsum(const float *partial, int rows, int64_t stride, void *out, int n, int dtype, cudaStream_t st) {
    const int grid = (n + 127) / 128;
    if (dtype == FCAI_DTYPE_BF16) colsum_kernel<<<grid, 128, 0, st>>>(partial, rows, stride, static_cast<__nv_bfloat16 *>(out), n);
    else if (dtype == FCAI_DTYPE_F16) colsum_kernel<<<grid, 128, 0, st>>>(partial, rows, stride, static_cast<__half *>(out), n);
    else colsum_kernel<<<grid, 128, 0, st>>>(partial, rows, stride, static_cast<float *>(out), n);
    FCAI_CUDA_TRY(cudaGetLastError());
    return FCAI_OK;
}
static bool affine_vec(const void *p, int wdtype) { return !p || aligned16(p, 0, wdtype); }

template <typename T>
static int act_forward(const void *x, int64_t ldx, void *y, int64_t ldy, void *codes, float *scales, int64_t rows, int n,
                       int dtype, int act, int keep, cudaStream_t st) {
    const bool q = keep == FCAI_KEEP_INT8 || keep == FCAI_KEEP_E4M3;
    const int vec = n % 8 == 0 && aligned16(x, ldx, dtype) && (!y || aligned16(y, ldy, dtype)) && (!q || codes_vec(codes, n));
    act_forward_kernel<T><<<item_grid(rows, blocks_of(n)), kThreads, 0, st>>>(
        static_cast<const T *>(x), ldx, static_cast<T *>(y), ldy, static_cast<uint8_t *>(codes), scales, rows, n, blocks_of(n), act,
        keep, vec);
    FCAI_CUDA_TRY(cudaGetLastError());
    return FCAI_OK;
}
template <typename T>
static int act_backward(const void *dy, int64_t lddy, const Kept &k, void *dx, int64_t lddx, void *bias_grad, int64_t rows, int n,
                        int dtype, int act, float *ws, cudaStream_t st) {
    const int strips = blocks_of(n), shares = row_shares(rows, strips);
    const bool full = k.keep == FCAI_KEEP_FULL;
    const int vec = n % 8 == 0 && aligned16(dy, lddy, dtype) && (!dx || aligned16(dx, lddx, dtype)) &&
                    (act == FCAI_ACT_NONE || (full ? aligned16(k.x, k.ldx, dtype) : codes_vec(k.codes, n)));
    act_backward_kernel<T><<<dim3(strips, shares), kThreads, 0, st>>>(static_cast<const T *>(dy), lddy, k, static_cast<T *>(dx), lddx,
                                                                    bias_grad ? ws : nullptr, rows, n, strips, act, vec);
    FCAI_CUDA_TRY(cudaGetLastError());
    return bias_grad ? colsum(ws, shares, n, bias_grad, n, dtype, st) : FCAI_OK;
}
template <typename T>
static int load_checkpoint(const Kept &k, void *out, int64_t ldo, int64_t rows, int n, int dtype, cudaStream_t st) {
    const int vec = n % 8 == 0 && aligned16(out, ldo, dtype) && codes_vec(k.codes, n);
    checkpoint_load_kernel<T><<<item_grid(rows, blocks_of(n)), kThreads, 0, st>>>(k, static_cast<T *>(out), ldo, rows, n, blocks_of(n),
                                                                                vec);
    FCAI_CUDA_TRY(cudaGetLastError());
    return FCAI_OK;
}
template <typename T>
static int norm_forward(const void *x, int64_t ldx, Affine af, int wdtype, void *y, int64_t ldy, float *mean, float *rstd,
                        void *codes, float *scales, int64_t rows, int n, float eps, int dtype, int keep, cudaStream_t st) {
    const bool q = keep == FCAI_KEEP_INT8 || keep == FCAI_KEEP_E4M3;
    const int vec = n % 8 == 0 && aligned16(x, ldx, dtype) && aligned16(y, ldy, dtype) && (!q || codes_vec(codes, n));
    af.vec = n % 8 == 0 && affine_vec(af.w, wdtype) && affine_vec(af.b, wdtype);
    const int grid = (int)std::min<int64_t>(rows, (int64_t)fcai::sm_count() * 8);
    norm_forward_kernel<T><<<grid, kThreads, 0, st>>>(static_cast<const T *>(x), ldx, af, static_cast<T *>(y), ldy, mean, rstd,
                                                    static_cast<uint8_t *>(codes), scales, rows, n, blocks_of(n), eps, keep, vec);
    FCAI_CUDA_TRY(cudaGetLastError());
    return FCAI_OK;
}
template <typename T>
static int norm_backward(const void *dy, int64_t lddy, const Kept &k, const float *mean, const float *rstd, Affine af, int wdtype,
                         void *dx, int64_t lddx, void *dweight, void *dbias, int64_t rows, int n, int dtype, unsigned char *ws,
                         cudaStream_t st) {
    const int strips = blocks_of(n), shares = row_shares(rows, strips);
    const int vec = n % 8 == 0 && aligned16(dy, lddy, dtype) && (!dx || aligned16(dx, lddx, dtype)) &&
                    (k.keep == FCAI_KEEP_FULL ? aligned16(k.x, k.ldx, dtype) : codes_vec(k.codes, n));
    af.vec = n % 8 == 0 && affine_vec(af.w, wdtype);
    float2 *stats = reinterpret_cast<float2 *>(ws);
    float *partial = reinterpret_cast<float *>(ws + round256(rows * 8));
    norm_backward_stats_kernel<T><<<(int)std::min<int64_t>(rows, (int64_t)fcai::sm_count() * 8), kThreads, 0, st>>>(
        static_cast<const T *>(dy), lddy, k, mean, rstd, af, stats, rows, n, strips, vec);
    FCAI_CUDA_TRY(cudaGetLastError());
    norm_backward_strip_kernel<T><<<dim3(strips, shares), kThreads, 0, st>>>(static_cast<const T *>(dy), lddy, k, mean, rstd, af, stats,
                                                                           static_cast<T *>(dx), lddx,
                                                                           dweight || dbias ? partial : nullptr, rows, n, strips, vec);
    FCAI_CUDA_TRY(cudaGetLastError());
    int rc = FCAI_OK;
    if (dweight) rc = colsum(partial, shares, 2 * (int64_t)n, dweight, n, wdtype, st);
    if (!rc && dbias) rc = colsum(partial + n, shares, 2 * (int64_t)n, dbias, n, wdtype, st);
    return rc;
}

// Sums over no rows.
static int zero_sums(void *out, int n, int dtype, cudaStream_t st) {
    if (out) FCAI_CUDA_TRY(cudaMemsetAsync(out, 0, (size_t)n * dtype_size(dtype), st));
    return FCAI_OK;
}

#define RW_BY_DTYPE(call)                                          \
    (dtype == FCAI_DTYPE_BF16  ? call(__nv_bfloat16)               \
     : dtype == FCAI_DTYPE_F16 ? call(__half)                      \
                               : call(float))

}  // namespace rw

extern "C" {

int fcai_activation_forward(const void *x, int64_t ldx, void *y, int64_t ldy, void *codes, float *scales, int64_t rows,
                            int32_t channels, int32_t dtype, int32_t act, int32_t keep, fcai_stream_t stream) {
    using namespace rw;
    fcai::clear_error();
    int rc = check_sizes("activation", rows, channels, dtype);
    if (rc) return rc;
    if (act < FCAI_ACT_NONE || act > FCAI_ACT_SILU) return fcai::fail(FCAI_ERR_INVALID, "activation: unknown activation %d", act);
    if (keep < FCAI_KEEP_NONE || keep > FCAI_KEEP_E4M3) return fcai::fail(FCAI_ERR_INVALID, "activation: unknown keep %d", keep);
    if (bad_matrix(x, ldx, channels, dtype) || (y && bad_matrix(y, ldy, channels, dtype)))
        return fcai::fail(FCAI_ERR_INVALID, "activation: a row stride is smaller than its row, or a misaligned pointer");
    const bool q = keep >= FCAI_KEEP_INT8;
    if (rows && (!x || (q && (!codes || !scales)) || (!q && !y)) || (reinterpret_cast<uintptr_t>(scales) & 3))
        return fcai::fail(FCAI_ERR_INVALID, "activation: null or misaligned pointer");
    if (rows == 0) return FCAI_OK;
    auto st = static_cast<cudaStream_t>(stream);
#define CALL(T) act_forward<T>(x, ldx, y, ldy, codes, scales, rows, channels, dtype, act, keep, st)
    return RW_BY_DTYPE(CALL);
#undef CALL
}

int64_t fcai_activation_workspace(int64_t rows, int32_t channels) {
    if (rows < 0 || rows > 0x7FFFFFFF || channels < 1 || channels > (1 << 24)) return -1;
    return rw::act_workspace(rows, channels);
}

int fcai_activation_backward(const void *dy, int64_t lddy, const void *x, int64_t ldx, const void *codes, const float *scales,
                             void *dx, int64_t lddx, void *bias_grad, int64_t rows, int32_t channels, int32_t dtype, int32_t act,
                             int32_t keep, void *workspace, int64_t workspace_bytes, fcai_stream_t stream) {
    using namespace rw;
    fcai::clear_error();
    int rc = check_sizes("activation", rows, channels, dtype);
    if (rc) return rc;
    if (act < FCAI_ACT_NONE || act > FCAI_ACT_SILU) return fcai::fail(FCAI_ERR_INVALID, "activation: unknown activation %d", act);
    const Kept k{x, ldx, static_cast<const uint8_t *>(codes), scales, keep};
    if (act != FCAI_ACT_NONE && (rc = check_kept("activation", k, rows, channels, dtype))) return rc;
    if (bad_matrix(dy, lddy, channels, dtype) || (dx && bad_matrix(dx, lddx, channels, dtype)) || (rows && !dy))
        return fcai::fail(FCAI_ERR_INVALID, "activation: null or misaligned pointer, or a row stride smaller than its row");
    if (rows && !dx && !bias_grad) return fcai::fail(FCAI_ERR_INVALID, "activation: nothing to write");
    auto st = static_cast<cudaStream_t>(stream);
    if (rows == 0) return zero_sums(bias_grad, channels, dtype, st);
    if (bias_grad && (rc = check_ws("activation", act_workspace(rows, channels), workspace, workspace_bytes))) return rc;
#define CALL(T) act_backward<T>(dy, lddy, k, dx, lddx, bias_grad, rows, channels, dtype, act, static_cast<float *>(workspace), st)
    return RW_BY_DTYPE(CALL);
#undef CALL
}

int fcai_checkpoint_load(const void *codes, const float *scales, void *out, int64_t ldo, int64_t rows, int32_t channels,
                         int32_t dtype, int32_t keep, fcai_stream_t stream) {
    using namespace rw;
    fcai::clear_error();
    int rc = check_sizes("checkpoint", rows, channels, dtype);
    if (rc) return rc;
    const Kept k{nullptr, 0, static_cast<const uint8_t *>(codes), scales, keep};
    if (keep == FCAI_KEEP_FULL) return fcai::fail(FCAI_ERR_INVALID, "checkpoint: keep must be int8 or e4m3");
    if ((rc = check_kept("checkpoint", k, rows, channels, dtype))) return rc;
    if (bad_matrix(out, ldo, channels, dtype) || (rows && !out))
        return fcai::fail(FCAI_ERR_INVALID, "checkpoint: null or misaligned pointer, or a row stride smaller than its row");
    if (rows == 0) return FCAI_OK;
    auto st = static_cast<cudaStream_t>(stream);
#define CALL(T) load_checkpoint<T>(k, out, ldo, rows, channels, dtype, st)
    return RW_BY_DTYPE(CALL);
#undef CALL
}

int fcai_layer_norm_forward(const void *x, int64_t ldx, const void *weight, const void *bias, int32_t wdtype, void *y, int64_t ldy,
                            float *mean, float *rstd, void *codes, float *scales, int64_t rows, int32_t channels, float eps,
                            int32_t dtype, int32_t keep, fcai_stream_t stream) {
    using namespace rw;
    fcai::clear_error();
    int rc = check_sizes("layer_norm", rows, channels, dtype);
    if (rc) return rc;
    if (wdtype != dtype && wdtype != FCAI_DTYPE_F32) return fcai::fail(FCAI_ERR_INVALID, "layer_norm: weights are of x's type or f32");
    if (keep < FCAI_KEEP_NONE || keep > FCAI_KEEP_E4M3) return fcai::fail(FCAI_ERR_INVALID, "layer_norm: unknown keep %d", keep);
    if (!(eps >= 0.f) || eps > FLT_MAX) return fcai::fail(FCAI_ERR_INVALID, "layer_norm: eps must be finite and not negative");
    if (bad_matrix(x, ldx, channels, dtype) || bad_matrix(y, ldy, channels, dtype) ||
        ((reinterpret_cast<uintptr_t>(weight) | reinterpret_cast<uintptr_t>(bias)) & (dtype_size(wdtype) - 1)))
        return fcai::fail(FCAI_ERR_INVALID, "layer_norm: a row stride is smaller than its row, or a misaligned pointer");
    if ((mean == nullptr) != (rstd == nullptr)) return fcai::fail(FCAI_ERR_INVALID, "layer_norm: mean and rstd go together");
    if (((reinterpret_cast<uintptr_t>(mean) | reinterpret_cast<uintptr_t>(rstd) | reinterpret_cast<uintptr_t>(scales)) & 3) ||
        (rows && (!x || !y || (keep >= FCAI_KEEP_INT8 && (!codes || !scales)))))
        return fcai::fail(FCAI_ERR_INVALID, "layer_norm: null or misaligned pointer");
    if (rows == 0) return FCAI_OK;
    const Affine af{weight, bias, wdtype == FCAI_DTYPE_F32, 0};
    auto st = static_cast<cudaStream_t>(stream);
#define CALL(T) norm_forward<T>(x, ldx, af, wdtype, y, ldy, mean, rstd, codes, scales, rows, channels, eps, dtype, keep, st)
    return RW_BY_DTYPE(CALL);
#undef CALL
}

int64_t fcai_layer_norm_workspace(int64_t rows, int32_t channels) {
    if (rows < 0 || rows > 0x7FFFFFFF || channels < 1 || channels > (1 << 24)) return -1;
    return rw::norm_workspace(rows, channels);
}

int fcai_layer_norm_backward(const void *dy, int64_t lddy, const void *x, int64_t ldx, const void *codes, const float *scales,
                             const float *mean, const float *rstd, const void *weight, int32_t wdtype, void *dx, int64_t lddx,
                             void *dweight, void *dbias, int64_t rows, int32_t channels, int32_t dtype, int32_t keep,
                             void *workspace, int64_t workspace_bytes, fcai_stream_t stream) {
    using namespace rw;
    fcai::clear_error();
    int rc = check_sizes("layer_norm", rows, channels, dtype);
    if (rc) return rc;
    if (wdtype != dtype && wdtype != FCAI_DTYPE_F32) return fcai::fail(FCAI_ERR_INVALID, "layer_norm: weights are of x's type or f32");
    const Kept k{x, ldx, static_cast<const uint8_t *>(codes), scales, keep};
    if ((rc = check_kept("layer_norm", k, rows, channels, dtype))) return rc;
    if (bad_matrix(dy, lddy, channels, dtype) || (dx && bad_matrix(dx, lddx, channels, dtype)) ||
        ((reinterpret_cast<uintptr_t>(weight) | reinterpret_cast<uintptr_t>(dweight) | reinterpret_cast<uintptr_t>(dbias)) &
         (dtype_size(wdtype) - 1)) ||
        ((reinterpret_cast<uintptr_t>(mean) | reinterpret_cast<uintptr_t>(rstd)) & 3) || (rows && (!dy || !mean || !rstd)))
        return fcai::fail(FCAI_ERR_INVALID, "layer_norm: null or misaligned pointer, or a row stride smaller than its row");
    if (rows && !dx && !dweight && !dbias) return fcai::fail(FCAI_ERR_INVALID, "layer_norm: nothing to write");
    auto st = static_cast<cudaStream_t>(stream);
    if (rows == 0) {
        rc = zero_sums(dweight, channels, wdtype, st);
        return rc ? rc : zero_sums(dbias, channels, wdtype, st);
    }
    if ((rc = check_ws("layer_norm", norm_workspace(rows, channels), workspace, workspace_bytes))) return rc;
    const Affine af{weight, nullptr, wdtype == FCAI_DTYPE_F32, 0};
#define CALL(T)                                                                                                                \
    norm_backward<T>(dy, lddy, k, mean, rstd, af, wdtype, dx, lddx, dweight, dbias, rows, channels, dtype,                      \
                     static_cast<unsigned char *>(workspace), st)
    return RW_BY_DTYPE(CALL);
#undef CALL
}

}  // extern "C"
