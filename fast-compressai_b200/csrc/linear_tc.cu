// linear_tc.cu -- the pointwise layer's matrix products on the sm_100a tensor
// cores (tcgen05) and their C ABI (include/fcai_layers.h).
//
// One kernel computes D[M][N] = sum_k A(m, k) B(n, k) for the three products
// of a layer with x[rows][cin], w[cout][cin], dp[rows][cout]:
//   forward          y  = x w^T     A = x  (K contiguous)  B = w  (K contiguous)
//   backward input   dx = dp w      A = dp (K contiguous)  B = w  (N contiguous)
//   backward weight  dw = dp^T x    A = dp (M contiguous)  B = x  (N contiguous)
// Operands stay where they are: an operand whose rows run along K is loaded as
// K-major tiles (TMA boxes of 64 k x rows), one whose rows run along M or N as
// MN-major tiles (boxes of 64 mn x 64 k), and the instruction descriptor's
// major bits say which; no transposed copy exists.  A matrix whose address or
// row stride is not 16-byte aligned, which TMA cannot read, is copied once
// into the workspace with a padded stride (repack_kernel).
//
// CTA organisation (persistent, one CTA per SM, 10 warps):
//   warps 0-7  epilogue: TMEM -> registers -> a per-warp 32 x 32 fp32 staging
//              tile (XOR-swizzled, so both directions are free of bank
//              conflicts) -> bias, activation, residual and rounding in a
//              layout where 4 lanes cover 32 columns of a row, 16 bytes each
//   warp 8     TMA producer
//   warp 9     MMA issuer; owns the TMEM allocation
// Two TMEM accumulators let the epilogue of a tile overlap the next mainloop.
//
// Work units are (tile, split): when a product has fewer tiles than SMs (few
// rows, or a weight gradient whose long axis is the contraction), K is split
// and each unit writes an fp32 partial tile to the workspace; reduce_kernel
// sums the splits in order (bitwise the same on every run) and applies the
// epilogue.
#include <cuda_runtime.h>
#include <cudaTypedefs.h>

#include <algorithm>
#include <mutex>

#include "layers_common.cuh"
#include "tc_ptx.h"

namespace tcx {
template <> struct T16<__nv_bfloat16> { static constexpr bool kBf16 = true; };
template <> struct T16<__half> { static constexpr bool kBf16 = false; };
}  // namespace tcx

namespace ln {

using namespace tcx;
using namespace ly;

constexpr int kBM = 128;            // tile rows of one CTA
constexpr int kBK = 64;             // K per ring stage: one 128-byte swizzled row
constexpr int kEpiWarps = 8;
constexpr int kThreads = (kEpiWarps + 2) * 32;
constexpr int kStagingWarp = 32 * 32 * 4;
constexpr uint64_t kWaitNs = 1000000000ull;

struct Params {
    int M, N;
    int tiles_m, tiles_n, group_m;
    int splits, ksteps, ksteps_split;  // K steps in all and per split
    int units;
    int ldp;                           // partial tiles: row stride (N rounded up to 8)
    int vec;                           // y, residual, pre and bias take 16-byte accesses
    int act;
    const void *bias, *residual;
    void *y, *pre;
    int64_t ldy, ldr, ldpre;
    float *partial;                    // [splits][M][ldp], or NULL
};

// A tile is kPair ? 256 : 128 rows by kBN columns.
template <int kBN, bool kPair>
struct Layout {
    static constexpr int kNB = kPair ? kBN / 2 : kBN;  // rows of B this CTA stages
    static constexpr int kTileM = kPair ? 2 * kBM : kBM;
    static constexpr int kA = kBM * kBK * 2;
    static constexpr int kB = kNB * kBK * 2;
    static constexpr int kStage = kA + kB;
    static constexpr int kStages = kNB == 64 ? 8 : 6;
    static constexpr int offStaging = kStages * kStage;
    static constexpr int offBar = offStaging + kEpiWarps * kStagingWarp;
    static constexpr int kBars = 2 * kStages + 2 * 2 + 1;
    static constexpr int offSlot = offBar + kBars * 8;
    static constexpr int kBytes = offSlot + 16;
    static constexpr int kAlloc = kBytes + 1024;  // the base is rounded up to 1024
    static_assert(kAlloc <= 227 * 1024, "shared memory");
};

// Unit -> (row tile, column tile, split).  Tiles run through groups of group_m
// row tiles, column by column, so that the CTAs of a wave share operand tiles
// in L2; the splits of a tile are neighbours.
__device__ __forceinline__ void unit_coords(const Params &p, int unit, int &tm, int &tn, int &sp) {
    const int t = unit / p.splits;
    sp = unit - t * p.splits;
    const int per = p.group_m * p.tiles_n;
    const int g = t / per;
    const int rest = t - g * per;
    const int gm = min(p.group_m, p.tiles_m - g * p.group_m);
    tn = rest / gm;
    tm = g * p.group_m + rest - tn * gm;
}

// Epilogue of kR rows' 8 neighbouring columns from `col` on; rows at
// `row + i * row_step`, those from M on left out.  All rows go through each
// step together, so that their loads and arithmetic overlap.
template <typename T, int kR>
__device__ __forceinline__ void finish(const Params &p, int64_t row, int row_step, int col, float (&v)[kR * 8]) {
    if (p.bias) {
        float bias[8];
        Vec8<T>::load(static_cast<const T *>(p.bias) + col, bias);
#pragma unroll
        for (int i = 0; i < kR * 8; ++i) v[i] += bias[i & 7];
    }
    if (p.pre) {
#pragma unroll
        for (int i = 0; i < kR; ++i)
            if (row + i * row_step < p.M) {
                float o[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) o[e] = v[i * 8 + e];
                Vec8<T>::store(static_cast<T *>(p.pre) + (row + i * row_step) * p.ldpre + col, o);
            }
    }
    uint4 res[kR];
    if (p.residual) {
#pragma unroll
        for (int i = 0; i < kR; ++i)
            if (row + i * row_step < p.M)
                res[i] = __ldg(reinterpret_cast<const uint4 *>(static_cast<const T *>(p.residual) + (row + i * row_step) * p.ldr + col));
    }
    if (p.act != FCAI_ACT_NONE) {
        F2 w[kR * 4];
#pragma unroll
        for (int i = 0; i < kR * 4; ++i) w[i] = f2(v[2 * i], v[2 * i + 1]);
        act_n(p.act, w);
#pragma unroll
        for (int i = 0; i < kR * 4; ++i) {
            const float2 o = split(w[i]);
            v[2 * i] = o.x, v[2 * i + 1] = o.y;
        }
    }
#pragma unroll
    for (int i = 0; i < kR; ++i) {
        if (row + i * row_step >= p.M) continue;
        float o[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] = v[i * 8 + e];
        if (p.residual) {
            float r[8];
            Vec8<T>::unpack(res[i], r);
#pragma unroll
            for (int e = 0; e < 8; ++e) o[e] += r[e];
        }
        Vec8<T>::store(static_cast<T *>(p.y) + (row + i * row_step) * p.ldy + col, o);
    }
}
template <typename T>
__device__ __forceinline__ void finish1(const Params &p, int64_t row, int col, float v, float bias) {
    v += bias;
    if (p.pre) static_cast<T *>(p.pre)[row * p.ldpre + col] = from_f32<T>(v);
    v = act_1(p.act, v);
    if (p.residual) v += to_f32(static_cast<const T *>(p.residual)[row * p.ldr + col]);
    static_cast<T *>(p.y)[row * p.ldy + col] = from_f32<T>(v);
}

// One 32 x 32 chunk of a warp: rows [row0, row0 + 32) from the staging tile.
template <typename T>
__device__ __forceinline__ void write_chunk(const Params &p, const unsigned char *stg, int row0, int col0, int sp,
                                            int lane) {
    if (col0 >= p.N) return;
    if (p.partial || p.vec) {
        const int col = col0 + (lane & 3) * 8, r0 = lane >> 2;
        if (col >= (p.partial ? p.ldp : p.N)) return;  // both multiples of 8
        float v[32];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int r = i * 8 + r0;
            const float4 a = *reinterpret_cast<const float4 *>(stg + r * 128 + (((2 * (lane & 3)) ^ (r & 7)) << 4));
            const float4 b = *reinterpret_cast<const float4 *>(stg + r * 128 + (((2 * (lane & 3) + 1) ^ (r & 7)) << 4));
            v[8 * i] = a.x, v[8 * i + 1] = a.y, v[8 * i + 2] = a.z, v[8 * i + 3] = a.w;
            v[8 * i + 4] = b.x, v[8 * i + 5] = b.y, v[8 * i + 6] = b.z, v[8 * i + 7] = b.w;
        }
        if (p.partial) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int row = row0 + i * 8 + r0;
                if (row >= p.M) break;
                float4 *dst = reinterpret_cast<float4 *>(p.partial + ((int64_t)sp * p.M + row) * p.ldp + col);
                dst[0] = make_float4(v[8 * i], v[8 * i + 1], v[8 * i + 2], v[8 * i + 3]);
                dst[1] = make_float4(v[8 * i + 4], v[8 * i + 5], v[8 * i + 6], v[8 * i + 7]);
            }
        } else {
            finish<T, 4>(p, row0 + r0, 8, col, v);
        }
    } else {
        const int col = col0 + lane;
        if (col >= p.N) return;
        const float bias = p.bias ? to_f32(static_cast<const T *>(p.bias)[col]) : 0.f;
#pragma unroll 4
        for (int r = 0; r < 32; ++r) {
            if (row0 + r >= p.M) break;
            const float v = *reinterpret_cast<const float *>(stg + r * 128 + (((lane >> 2) ^ (r & 7)) << 4) + (lane & 3) * 4);
            finish1<T>(p, row0 + r, col, v, bias);
        }
    }
}

// kTA / kTB: the operand's rows run along K (its M / N axis is contiguous).
// kPair: clusters of two CTAs share each MMA (cta_group::2, M = 256): each CTA
// stages its 128 rows of A and half the columns' rows of B and owns 128 rows
// of the accumulator; the rank-0 CTA issues for both.
template <typename T, int kBN, bool kPair, bool kTA, bool kTB>
__global__ void __launch_bounds__(kThreads, 1)
    linear_tc_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB, const Params p) {
    using Lay = Layout<kBN, kPair>;
    constexpr int kStages = Lay::kStages;
    extern __shared__ unsigned char smem_raw[];
    unsigned char *smem =
        reinterpret_cast<unsigned char *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t *full = reinterpret_cast<uint64_t *>(smem + Lay::offBar);  // pairs: rank 0's counts both CTAs' loads
    uint64_t *empty = full + kStages;
    uint64_t *accf = empty + kStages;  // accumulator filled (by the MMA warp; pairs: in both CTAs)
    uint64_t *acce = accf + 2;         // accumulator read: one arrival per epilogue warp (pairs: of both CTAs, at rank 0)
    uint64_t *dbar = acce + 2;         // abort path: this CTA's MMAs drained
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(smem + Lay::offSlot);
    volatile int *abort = reinterpret_cast<volatile int *>(smem + Lay::offSlot + 4);

    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    const uint32_t rank = kPair ? cluster_ctarank() : 0u;
    const bool leader = rank == 0;
    const int unit0 = kPair ? (int)(blockIdx.x >> 1) : (int)blockIdx.x;
    const int unit_step = kPair ? (int)(gridDim.x >> 1) : (int)gridDim.x;
    constexpr uint32_t kTmemCols = 2 * kBN;

    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(&accf[b], 1);
            mbar_init(&acce[b], kPair ? 2 * kEpiWarps : kEpiWarps);
        }
        mbar_init(dbar, 1);
        *abort = 0;
        fence_barrier_init();
    }
    if (warp == kEpiWarps + 1) {
        if (kPair) {
            tmem_alloc_pair(tmem_slot, kTmemCols);
            tmem_relinquish_pair();
        } else {
            tmem_alloc(tmem_slot, kTmemCols);
            tmem_relinquish();
        }
    }
    tc_fence_before();
    __syncthreads();
    // pairs: both CTAs' barriers exist before any remote arrive or load names them
    if (kPair) cluster_sync_all();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;

    if (warp == kEpiWarps) {
        // ------------------------------------------------------------ producer
        if (lane == 0) {
            tma_prefetch_desc(&tmA);
            tma_prefetch_desc(&tmB);
        }
        __syncwarp();
        uint32_t it = 0;
        bool stop = false;
        for (int unit = unit0; unit < p.units && !stop; unit += unit_step) {
            int tm, tn, sp;
            unit_coords(p, unit, tm, tn, sp);
            const int m0 = tm * Lay::kTileM + (int)rank * kBM, n0 = tn * kBN + (int)rank * Lay::kNB;
            const int k1 = min((sp + 1) * p.ksteps_split, p.ksteps);
            for (int ks = sp * p.ksteps_split; ks < k1; ++ks, ++it) {
                const int s = it % kStages;
                const uint32_t r = it / kStages;
                if (!mbar_wait_warp(&empty[s], (r & 1) ^ 1, abort, kWaitNs)) {
                    *abort = 1;
                    stop = true;
                    break;
                }
                unsigned char *st = smem + s * Lay::kStage;
                const int k0 = ks * kBK;
                if constexpr (kPair) {
                    const uint32_t fb = mapa_shared(smem_u32(&full[s]), 0);
                    if (leader) mbar_arrive_expect_tx_w(&full[s], 2 * Lay::kStage);
                    if (kTA) {
                        tma_load_2d_pair_w(st, &tmA, fb, m0, k0);
                        tma_load_2d_pair_w(st + 8192, &tmA, fb, m0 + 64, k0);
                    } else {
                        tma_load_2d_pair_w(st, &tmA, fb, k0, m0);
                    }
                    if (kTB) {
#pragma unroll
                        for (int n = 0; n < Lay::kNB; n += 64)
                            tma_load_2d_pair_w(st + Lay::kA + n * 128, &tmB, fb, n0 + n, k0);
                    } else {
                        tma_load_2d_pair_w(st + Lay::kA, &tmB, fb, k0, n0);
                    }
                } else {
                    mbar_arrive_expect_tx_w(&full[s], Lay::kStage);
                    if (kTA) {
                        tma_load_2d_w(st, &tmA, &full[s], m0, k0);
                        tma_load_2d_w(st + 8192, &tmA, &full[s], m0 + 64, k0);
                    } else {
                        tma_load_2d_w(st, &tmA, &full[s], k0, m0);
                    }
                    if (kTB) {
#pragma unroll
                        for (int n = 0; n < Lay::kNB; n += 64)
                            tma_load_2d_w(st + Lay::kA + n * 128, &tmB, &full[s], n0 + n, k0);
                    } else {
                        tma_load_2d_w(st + Lay::kA, &tmB, &full[s], k0, n0);
                    }
                }
            }
        }
        if (*abort && leader) {
            // the loads in flight land before the CTA exits (pairs: rank 0's
            // barriers also count the peer's loads): the last rounds issued
            for (int s = 0; s < kStages; ++s)
                if (it > (uint32_t)s) mbar_wait(&full[s], ((it - 1 - s) / kStages) & 1, nullptr, kWaitNs / 10);
        }
        __syncwarp();
    } else if (warp == kEpiWarps + 1) {
        // ---------------------------------------------------------- MMA issuer
        if (leader) {
            constexpr uint32_t idesc = idesc_f16kind<T>(Lay::kTileM, kBN, kTA, kTB);
            uint32_t it = 0;
            int j = 0;
            bool ok = true;
            for (int unit = unit0; unit < p.units && ok; unit += unit_step, ++j) {
                int tm, tn, sp;
                unit_coords(p, unit, tm, tn, sp);
                const int buf = j & 1;
                if (!mbar_wait_warp(&acce[buf], ((j >> 1) & 1) ^ 1, abort, kWaitNs, kPair)) {
                    *abort = 1;
                    break;
                }
                tc_fence_after();
                const uint32_t d = tmem_base + buf * kBN;
                const int k0 = sp * p.ksteps_split, k1 = min(k0 + p.ksteps_split, p.ksteps);
                for (int ks = k0; ks < k1; ++ks, ++it) {
                    const int s = it % kStages;
                    if (!mbar_wait_warp(&full[s], (it / kStages) & 1, abort, kWaitNs)) {
                        *abort = 1;
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    const uint32_t a0 = smem_u32(smem + s * Lay::kStage), b0 = a0 + Lay::kA;
#pragma unroll
                    for (int kk = 0; kk < kBK / 16; ++kk) {
                        // K-major tiles: 16 k are 32 bytes of the 128-byte row, row
                        // groups of 8 are 1024 bytes apart.  MN-major tiles: 16 k
                        // are two groups of 8 rows, 1024 bytes apart, and blocks
                        // of 64 along M / N are 8192 bytes apart.
                        const uint64_t ad = kTA ? smem_desc(a0 + kk * 2048, 8192, 1024, 2) : smem_desc(a0 + kk * 32, 16, 1024, 2);
                        const uint64_t bd = kTB ? smem_desc(b0 + kk * 2048, 8192, 1024, 2) : smem_desc(b0 + kk * 32, 16, 1024, 2);
                        const uint32_t acc = (ks > k0 || kk > 0) ? 1u : 0u;
                        if (kPair) mma_bf16_pair_w(d, ad, bd, idesc, acc);
                        else mma_bf16_w(d, ad, bd, idesc, acc);
                    }
                    if (kPair) mma_commit_pair_both_w(&empty[s], 3);
                    else mma_commit_w(&empty[s]);
                }
                if (!ok) break;
                if (kPair) mma_commit_pair_both_w(&accf[buf], 3);
                else mma_commit_w(&accf[buf]);
            }
        }
        __syncwarp();
    } else {
        // ------------------------------------------------------------ epilogue
        const int q = warp & 3, half = warp >> 2;
        unsigned char *stg = smem + Lay::offStaging + warp * kStagingWarp;
        int j = 0;
        for (int unit = unit0; unit < p.units; unit += unit_step, ++j) {
            int tm, tn, sp;
            unit_coords(p, unit, tm, tn, sp);
            const int buf = j & 1;
            if (!mbar_wait_warp(&accf[buf], (j >> 1) & 1, abort, kWaitNs)) {
                *abort = 1;
                break;
            }
            tc_fence_after();
            const int row0 = tm * Lay::kTileM + (int)rank * kBM + q * 32;
            const uint32_t taddr = tmem_base + buf * kBN + ((uint32_t)(q * 32) << 16);
#pragma unroll 1
            for (int c = half * (kBN / 2); c < (half + 1) * (kBN / 2); c += 32) {
                uint32_t v[32];
                tmem_ld32(taddr + c, v);
                tmem_wait_ld();
                if (c + 32 == (half + 1) * (kBN / 2)) {  // this warp has read its part of the accumulator
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) {
                        if (kPair) mbar_arrive_cluster(mapa_shared(smem_u32(&acce[buf]), 0));
                        else mbar_arrive(&acce[buf]);
                    }
                }
                if (row0 < p.M) {
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        *reinterpret_cast<uint4 *>(stg + lane * 128 + ((e ^ (lane & 7)) << 4)) =
                            make_uint4(v[4 * e], v[4 * e + 1], v[4 * e + 2], v[4 * e + 3]);
                    __syncwarp();
                    write_chunk<T>(p, stg, row0, tn * kBN + c, sp, lane);
                    __syncwarp();
                }
            }
        }
    }

    // ---------------------------------------------------------------- teardown
    __syncthreads();
    if (*abort && leader) {
        // TMEM is freed only once every MMA issued has completed
        if (warp == kEpiWarps + 1) {
            if (lane == 0) {
                if (kPair) mma_commit_pair(dbar);
                else mma_commit(dbar);
                mbar_wait(dbar, 0, nullptr, kWaitNs / 10);
            }
            __syncwarp();
        }
        __syncthreads();
    }
    // pairs: no remote arrive, load or MMA reaches a CTA that has left
    if (kPair) cluster_sync_all();
    if (warp == kEpiWarps + 1) {
        __syncwarp();
        tc_fence_after();
        if (kPair) tmem_dealloc_pair(tmem_base, kTmemCols);
        else tmem_dealloc(tmem_base, kTmemCols);
    }
}

// Sums the splits of 8 neighbouring columns in order and applies the epilogue.
template <typename T>
__global__ void reduce_kernel(const Params p) {
    const int per_row = p.ldp / 8;
    const int64_t n = (int64_t)p.M * per_row;
    const int64_t step = (int64_t)p.M * p.ldp;
    for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < n; i += (int64_t)gridDim.x * blockDim.x) {
        const int64_t row = i / per_row;
        const int col = (int)(i - row * per_row) * 8;
        float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        const float *src = p.partial + row * p.ldp + col;
        for (int s = 0; s < p.splits; ++s, src += step) {
            float u[8];
            Vec8<float>::load(src, u);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] += u[e];
        }
        if (p.vec) {
            finish<T, 1>(p, row, 0, col, v);
        } else {
            for (int e = 0; e < 8 && col + e < p.N; ++e)
                finish1<T>(p, row, col + e, v[e], p.bias ? to_f32(static_cast<const T *>(p.bias)[col + e]) : 0.f);
        }
    }
}

// src[rows][cols] (row stride ld) -> dst[rows][ldd], for matrices TMA cannot read.
__global__ void repack_kernel(const uint16_t *__restrict__ src, int64_t ld, uint16_t *__restrict__ dst, int64_t rows,
                              int cols, int ldd) {
    const int64_t n = rows * ldd;
    for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < n; i += (int64_t)gridDim.x * blockDim.x) {
        const int64_t row = i / ldd;
        const int col = (int)(i - row * ldd);
        dst[i] = col < cols ? __ldg(src + row * ld + col) : (uint16_t)0;
    }
}

// y = act(bias) + residual, for an empty contraction (a weight gradient over no rows).
template <typename T>
__global__ void empty_product_kernel(const Params p) {
    const int64_t n = (int64_t)p.M * p.N;
    for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < n; i += (int64_t)gridDim.x * blockDim.x)
        static_cast<T *>(p.y)[i / p.N * p.ldy + i % p.N] = from_f32<T>(0.f);
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------

static PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
    static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
    static std::once_flag once;
    std::call_once(once, [] {
        void *ptr = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) == cudaSuccess &&
            q == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(ptr);
    });
    return fn;
}

// A row-major matrix [outer][inner] as 128-byte swizzled boxes of 64 elements x box_rows.
static int make_map(CUtensorMap *map, const void *base, int64_t inner, int64_t outer, int64_t ld, int box_rows, int dtype) {
    auto fn = encode_fn();
    if (!fn) return fcai::fail(FCAI_ERR_CUDA, "cuTensorMapEncodeTiled is unavailable");
    const cuuint64_t dims[2] = {(cuuint64_t)inner, (cuuint64_t)outer};
    const cuuint64_t strides[1] = {(cuuint64_t)ld * 2};
    const cuuint32_t box[2] = {64, (cuuint32_t)box_rows};
    const cuuint32_t es[2] = {1, 1};
    const CUresult r = fn(map, dtype == FCAI_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
                          2, const_cast<void *>(base), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
                          CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fcai::fail(FCAI_ERR_INVALID, "cuTensorMapEncodeTiled failed (%d)", (int)r);
    return FCAI_OK;
}

static int64_t round256(int64_t v) { return (v + 255) / 256 * 256; }
static int round8(int v) { return (v + 7) / 8 * 8; }

// How a product of M x N x K runs.  Three tile shapes; the estimate below (in
// SM clocks) picks the one that ends first.
//   pair 256 x 256: 64 KB of operands a K step for both CTAs, 512 clocks of MMA;
//   128 x 128: 32 KB for 256 clocks of MMA, held to about 560 by the operand
//     feed from L2 (measured: 1.01 PFLOP/s over 16384 x 8192 x 8192);
//   128 x 64: 24 KB, about 400.
struct Plan {
    int bn, pair, splits, ksteps, ksteps_split, tiles_m, tiles_n;
    int64_t partial_bytes;
};
static Plan make_plan(int64_t M, int64_t N, int64_t K) {
    struct Shape {
        int bn, pair;
        double kstep, epilogue;  // clocks a K step; clocks of a tile's epilogue
    };
    static const Shape shapes[3] = {{256, 1, 540., 5000.}, {128, 0, 560., 2500.}, {64, 0, 400., 1300.}};
    const int sms = fcai::sm_count();
    Plan best{};
    double best_time = 0.;
    for (const Shape &sh : shapes) {
        if (sh.bn > 64 && N <= sh.bn / 2) continue;
        Plan pl{};
        pl.bn = sh.bn;
        pl.pair = sh.pair;
        const int tile_m = sh.pair ? 256 : 128;
        pl.tiles_m = (int)((M + tile_m - 1) / tile_m);
        pl.tiles_n = (int)((N + pl.bn - 1) / pl.bn);
        pl.ksteps = (int)((K + kBK - 1) / kBK);
        const int64_t tiles = (int64_t)pl.tiles_m * pl.tiles_n;
        const int64_t slots = sh.pair ? sms / 2 : sms;
        int splits = tiles >= slots ? 1 : (int)(slots / tiles);
        splits = std::max(1, std::min(splits, pl.ksteps / 4));
        pl.ksteps_split = (pl.ksteps + splits - 1) / splits;
        pl.splits = (pl.ksteps + pl.ksteps_split - 1) / pl.ksteps_split;  // none is empty
        pl.partial_bytes = pl.splits > 1 ? round256((int64_t)pl.splits * M * round8((int)N) * 4) : 0;
        const int64_t waves = (tiles * pl.splits + slots - 1) / slots;
        // a tile's epilogue runs under the next tile's K steps
        double time = waves * std::max(pl.ksteps_split * sh.kstep, sh.epilogue) + sh.epilogue;
        if (pl.splits > 1) time += 5000. + 2. * pl.partial_bytes / 4000.;  // the second launch and the partial tiles
        if (best.bn == 0 || time < best_time) {
            best = pl;
            best_time = time;
        }
    }
    return best;
}

struct Operand {
    const void *ptr;
    int64_t ld, rows;  // stored [rows][cols]
    int cols;
};

static int64_t repack_bytes(int64_t rows, int cols) { return round256(rows * round8(cols) * 2); }

static int elementwise_grid(int64_t n, int threads) {
    return (int)std::max<int64_t>(1, std::min<int64_t>((n + threads - 1) / threads, (int64_t)fcai::sm_count() * 8));
}

// Makes `o` readable by TMA, from the workspace if it has to be copied.
static int prepare_operand(Operand &o, int dtype, unsigned char *&ws, cudaStream_t stream) {
    if (aligned16(o.ptr, o.ld, dtype)) return FCAI_OK;
    const int ldd = round8(o.cols);
    repack_kernel<<<elementwise_grid(o.rows * ldd, 256), 256, 0, stream>>>(static_cast<const uint16_t *>(o.ptr), o.ld,
                                                                         reinterpret_cast<uint16_t *>(ws), o.rows,
                                                                         o.cols, ldd);
    FCAI_CUDA_TRY(cudaGetLastError());
    o.ptr = ws;
    o.ld = ldd;
    ws += repack_bytes(o.rows, o.cols);
    return FCAI_OK;
}

template <typename T, int kBN, bool kPair, bool kTA, bool kTB>
static int launch(const CUtensorMap &a, const CUtensorMap &b, const Params &p, cudaStream_t stream) {
    using Lay = Layout<kBN, kPair>;
    auto kernel = linear_tc_kernel<T, kBN, kPair, kTA, kTB>;
    static int slots[64] = {0};  // CTAs (pairs) resident at once
    int dev = 0;
    FCAI_CUDA_TRY(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 64) return fcai::fail(FCAI_ERR_CUDA, "device ordinal %d unsupported", dev);
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = 2;
    attr.val.clusterDim.y = 1;
    attr.val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg{};
    cfg.blockDim = dim3(kThreads, 1, 1);
    cfg.dynamicSmemBytes = Lay::kAlloc;
    cfg.stream = stream;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    if (!slots[dev]) {
        FCAI_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Lay::kAlloc));
        int n = fcai::sm_count();
        if (kPair) {
            cfg.gridDim = dim3(2, 1, 1);
            FCAI_CUDA_TRY(cudaOccupancyMaxActiveClusters(&n, kernel, &cfg));
            if (n < 1) return fcai::fail(FCAI_ERR_CUDA, "no CTA pair of this product fits on the device");
        }
        slots[dev] = n;
    }
    const int n = std::min(p.units, slots[dev]);
    if (kPair) {
        cfg.gridDim = dim3(2 * n, 1, 1);
        FCAI_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, a, b, p));
    } else {
        kernel<<<n, kThreads, Lay::kAlloc, stream>>>(a, b, p);
    }
    FCAI_CUDA_TRY(cudaGetLastError());
    return FCAI_OK;
}

template <typename T, bool kTA, bool kTB>
static int run(Operand A, Operand B, int64_t M, int N, int64_t K, int dtype, Params p, unsigned char *ws,
               cudaStream_t stream) {
    const Plan pl = make_plan(M, N, K);
    p.M = (int)M;
    p.N = N;
    p.tiles_m = pl.tiles_m;
    p.tiles_n = pl.tiles_n;
    p.group_m = 8;
    p.splits = pl.splits;
    p.ksteps = pl.ksteps;
    p.ksteps_split = pl.ksteps_split;
    p.units = pl.tiles_m * pl.tiles_n * pl.splits;
    p.ldp = round8(N);
    p.vec = N % 8 == 0 && aligned16(p.y, p.ldy, dtype) && (!p.pre || aligned16(p.pre, p.ldpre, dtype)) &&
            (!p.residual || aligned16(p.residual, p.ldr, dtype)) && (!p.bias || aligned16(p.bias, 0, dtype));
    p.partial = nullptr;
    if (pl.splits > 1) {
        p.partial = reinterpret_cast<float *>(ws);
        ws += pl.partial_bytes;
    }
    int rc;
    if ((rc = prepare_operand(A, dtype, ws, stream))) return rc;
    if ((rc = prepare_operand(B, dtype, ws, stream))) return rc;
    CUtensorMap ma, mb;
    if ((rc = make_map(&ma, A.ptr, A.cols, A.rows, A.ld, kTA ? kBK : kBM, dtype))) return rc;
    if ((rc = make_map(&mb, B.ptr, B.cols, B.rows, B.ld, kTB ? kBK : pl.pair ? pl.bn / 2 : pl.bn, dtype)))
        return rc;
    rc = pl.pair        ? launch<T, 256, true, kTA, kTB>(ma, mb, p, stream)
         : pl.bn == 128 ? launch<T, 128, false, kTA, kTB>(ma, mb, p, stream)
                        : launch<T, 64, false, kTA, kTB>(ma, mb, p, stream);
    if (rc) return rc;
    if (pl.splits > 1) {
        reduce_kernel<T><<<elementwise_grid(M * (p.ldp / 8), 256), 256, 0, stream>>>(p);
        FCAI_CUDA_TRY(cudaGetLastError());
    }
    return FCAI_OK;
}

// Checks shared by the three products.
static int check_common(int64_t rows, int cin, int cout, int dtype, const void *a, int64_t lda, int acols, const void *b,
                        int64_t ldb, int bcols, const void *out, int64_t ldo, int ocols) {
    if (dtype != FCAI_DTYPE_BF16 && dtype != FCAI_DTYPE_F16)
        return fcai::fail(FCAI_ERR_INVALID, "linear: dtype must be bf16 or f16");
    if (rows < 0 || rows > 0x7FFFFFFF - 256 || cin < 1 || cout < 1 || cin > (1 << 24) || cout > (1 << 24))
        return fcai::fail(FCAI_ERR_INVALID, "linear: sizes out of range (rows %lld, cin %d, cout %d)", (long long)rows, cin,
                          cout);
    if (lda < acols || ldb < bcols || ldo < ocols || std::max({lda, ldb, ldo}) > (1ll << 36))
        return fcai::fail(FCAI_ERR_INVALID, "linear: a row stride is smaller than its row or too large");
    if (((reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b) | reinterpret_cast<uintptr_t>(out)) & 1) != 0)
        return fcai::fail(FCAI_ERR_INVALID, "linear: misaligned pointer");
    return FCAI_OK;
}

static int64_t workspace_bytes(int op, int64_t rows, int cin, int cout, int repack) {
    if (rows < 0 || rows > 0x7FFFFFFF - 256 || cin < 1 || cout < 1 || cin > (1 << 24) || cout > (1 << 24)) return -1;
    if (rows == 0) return 0;
    int64_t n;
    switch (op) {
        case FCAI_LINEAR_FORWARD:
            n = make_plan(rows, cout, cin).partial_bytes;
            if (repack & 1) n += repack_bytes(rows, cin);
            if (repack & 2) n += repack_bytes(cout, cin);
            return n;
        case FCAI_LINEAR_BACKWARD_INPUT:
            n = make_plan(rows, cin, cout).partial_bytes;
            if (repack & 1) n += repack_bytes(rows, cout);
            if (repack & 2) n += repack_bytes(cout, cin);
            return n;
        case FCAI_LINEAR_BACKWARD_WEIGHT:
            n = make_plan(cout, cin, rows).partial_bytes;
            if (repack & 1) n += repack_bytes(rows, cout);
            if (repack & 2) n += repack_bytes(rows, cin);
            return n;
        default:
            return -1;
    }
}
static int check_workspace(int op, int64_t rows, int cin, int cout, const void *a, int64_t lda, const void *b, int64_t ldb,
                           int dtype, const void *ws, int64_t bytes) {
    const int repack = (aligned16(a, lda, dtype) ? 0 : 1) | (aligned16(b, ldb, dtype) ? 0 : 2);
    const int64_t need = workspace_bytes(op, rows, cin, cout, repack);
    if (need > 0 && (!ws || bytes < need || (reinterpret_cast<uintptr_t>(ws) & 255)))
        return fcai::fail(FCAI_ERR_WORKSPACE, "linear: needs a 256-byte aligned workspace of %lld bytes", (long long)need);
    return FCAI_OK;
}

}  // namespace ln

extern "C" {

int64_t fcai_linear_workspace(int32_t op, int64_t rows, int32_t cin, int32_t cout, int32_t repack) {
    return ln::workspace_bytes(op, rows, cin, cout, repack);
}

int fcai_linear_forward(const void *x, int64_t ldx, const void *w, int64_t ldw, const void *bias,
                        const void *residual, int64_t ldr, void *y, int64_t ldy, void *pre, int64_t ldpre,
                        int64_t rows, int32_t cin, int32_t cout, int32_t dtype, int32_t act, void *workspace,
                        int64_t workspace_bytes, fcai_stream_t stream) {
    using namespace ln;
    fcai::clear_error();
    int rc = check_common(rows, cin, cout, dtype, x, ldx, cin, w, ldw, cin, y, ldy, cout);
    if (rc) return rc;
    if (act < FCAI_ACT_NONE || act > FCAI_ACT_SILU) return fcai::fail(FCAI_ERR_INVALID, "linear: unknown activation %d", act);
    if ((residual && ldr < cout) || (pre && ldpre < cout))
        return fcai::fail(FCAI_ERR_INVALID, "linear: a row stride is smaller than its row");
    if (rows == 0) return FCAI_OK;
    if (!x || !w || !y) return fcai::fail(FCAI_ERR_INVALID, "linear: null pointer");
    if ((rc = check_workspace(FCAI_LINEAR_FORWARD, rows, cin, cout, x, ldx, w, ldw, dtype, workspace, workspace_bytes)))
        return rc;
    Params p{};
    p.act = act;
    p.bias = bias;
    p.residual = residual;
    p.ldr = ldr;
    p.y = y;
    p.ldy = ldy;
    p.pre = pre;
    p.ldpre = ldpre;
    const Operand A{x, ldx, rows, cin}, B{w, ldw, cout, cin};
    auto *ws = static_cast<unsigned char *>(workspace);
    auto st = static_cast<cudaStream_t>(stream);
    return dtype == FCAI_DTYPE_BF16 ? run<__nv_bfloat16, false, false>(A, B, rows, cout, cin, dtype, p, ws, st)
                                    : run<__half, false, false>(A, B, rows, cout, cin, dtype, p, ws, st);
}

int fcai_linear_backward_input(const void *dp, int64_t lddp, const void *w, int64_t ldw, void *dx, int64_t lddx,
                               int64_t rows, int32_t cin, int32_t cout, int32_t dtype, void *workspace,
                               int64_t workspace_bytes, fcai_stream_t stream) {
    using namespace ln;
    fcai::clear_error();
    int rc = check_common(rows, cin, cout, dtype, dp, lddp, cout, w, ldw, cin, dx, lddx, cin);
    if (rc) return rc;
    if (rows == 0) return FCAI_OK;
    if (!dp || !w || !dx) return fcai::fail(FCAI_ERR_INVALID, "linear: null pointer");
    if ((rc = check_workspace(FCAI_LINEAR_BACKWARD_INPUT, rows, cin, cout, dp, lddp, w, ldw, dtype, workspace,
                              workspace_bytes)))
        return rc;
    Params p{};
    p.y = dx;
    p.ldy = lddx;
    const Operand A{dp, lddp, rows, cout}, B{w, ldw, cout, cin};
    auto *ws = static_cast<unsigned char *>(workspace);
    auto st = static_cast<cudaStream_t>(stream);
    return dtype == FCAI_DTYPE_BF16 ? run<__nv_bfloat16, false, true>(A, B, rows, cin, cout, dtype, p, ws, st)
                                    : run<__half, false, true>(A, B, rows, cin, cout, dtype, p, ws, st);
}

int fcai_linear_backward_weight(const void *dp, int64_t lddp, const void *x, int64_t ldx, void *dw, int64_t lddw,
                                int64_t rows, int32_t cin, int32_t cout, int32_t dtype, void *workspace,
                                int64_t workspace_bytes, fcai_stream_t stream) {
    using namespace ln;
    fcai::clear_error();
    int rc = check_common(rows, cin, cout, dtype, dp, lddp, cout, x, ldx, cin, dw, lddw, cin);
    if (rc) return rc;
    if (!dw || (rows && (!dp || !x))) return fcai::fail(FCAI_ERR_INVALID, "linear: null pointer");
    Params p{};
    p.y = dw;
    p.ldy = lddw;
    auto st = static_cast<cudaStream_t>(stream);
    if (rows == 0) {
        p.M = cout;
        p.N = cin;
        // zero is the same bits in both types
        empty_product_kernel<__half><<<elementwise_grid((int64_t)cout * cin, 256), 256, 0, st>>>(p);
        FCAI_CUDA_TRY(cudaGetLastError());
        return FCAI_OK;
    }
    if ((rc = check_workspace(FCAI_LINEAR_BACKWARD_WEIGHT, rows, cin, cout, dp, lddp, x, ldx, dtype, workspace,
                              workspace_bytes)))
        return rc;
    const Operand A{dp, lddp, rows, cout}, B{x, ldx, rows, cin};
    auto *ws = static_cast<unsigned char *>(workspace);
    return dtype == FCAI_DTYPE_BF16 ? run<__nv_bfloat16, true, true>(A, B, cout, cin, rows, dtype, p, ws, st)
                                    : run<__half, true, true>(A, B, cout, cin, rows, dtype, p, ws, st);
}

}  // extern "C"
