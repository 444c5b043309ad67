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
// CTA organisation (persistent, one CTA per SM, 18 warps):
//   16 warps      epilogue: a row of the tile a lane, 32 columns at a time, from
//                 TMEM to bias, activation, residual and rounding; the 32 x 32
//                 results go to a swizzled tile in shared memory and from there
//                 by TMA (which also brought the residual's into the same
//                 tile).  The first form moved fp32 values through shared memory
//                 to store them from registers, and shared memory's bandwidth,
//                 which the MMA's operands need too, was what bounded layers
//                 with short contractions.
//   one warp      TMA producer
//   one warp      MMA issuer; owns the TMEM allocation
// Two or four TMEM accumulators let the epilogue of a tile overlap the next
// mainloops.  Layers with short contractions are bound by the epilogue, so its
// warps form as many groups as there are accumulators, each with every n-th
// tile of its own: the groups are in different steps at any time, which hides
// the latencies of one group behind the arithmetic of another.  A CTA with one
// or two tiles in all lets every warp work on each tile instead.
//
// A forward product that keeps the activation's input in 8 bits makes the
// codes here: a warp has whole 128-column blocks of its rows, takes their
// largest magnitudes in a first pass over the accumulator, and the codes leave
// beside y, so the activation's input does not go through memory in more than 8
// bits.  (It does, as fp32 in the workspace, where reduce_kernel makes the codes: up
// to 32 rows, where K is split, and for small results whose columns are no multiple
// of 16, which the codes' tensor map asks for.)
//
// Work units are (tile, split): when a product has fewer tiles than SMs (few
// rows, or a weight gradient whose long axis is the contraction), K is split
// and each unit writes an fp32 partial tile to the workspace; reduce_kernel
// sums the splits in order (bitwise the same on every run) and applies the
// epilogue.
//
// Every wait is bounded (1 s).  One that runs out, which no product should see,
// makes its CTA stop, drain what it has in flight and set its device's word in host
// memory, from which the device's next call returns FCAI_ERR_CUDA.
//
// Up to 32 rows the forward product is a matter of reading w once:
// few_rows_kernel does it with warp-level MMAs, w as their 16-row operand.
#include <cuda_runtime.h>
#include <cudaTypedefs.h>

#include <algorithm>
#include <atomic>
#include <initializer_list>
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
constexpr int kTileBytes = 32 * 32 * 2;       // a 32 x 32 tile of results
constexpr int kStagingWarp = 2 * kTileBytes;  // two of them, or one of fp32 values
constexpr uint64_t kWaitNs = 1000000000ull;

// Division of n < 2^31 by a divisor known on the host (Granlund and Montgomery,
// Division by Invariant Integers using Multiplication, 1994).
struct FastDiv {
    uint32_t d, mul, shift;
};
static FastDiv fast_div(uint32_t d) {
    uint32_t l = 0;
    while (l < 32 && (1ull << l) < d) ++l;
    return {d, (uint32_t)((((1ull << l) - d) << 32) / d + 1), l};
}
__device__ __forceinline__ int divide(int n, const FastDiv &f) { return (int)((__umulhi((uint32_t)n, f.mul) + (uint32_t)n) >> f.shift); }

struct Params {
    int M, N;
    int tiles_m, group_m;
    FastDiv splits, group, gm, gm_last;  // group: tiles of a group; gm: row tiles of a full / the last group
    int ksteps, ksteps_split;            // K steps in all and per split
    int units;
    int ldp;                             // partial tiles: row stride (N rounded up to 8)
    int coop;                            // all epilogue warps on each tile
    int vec;                             // N % 8 == 0, and y, residual, pre, bias and codes take wide accesses
    int tma;                             // y, residual, pre and codes are tiles of tensor maps; bias takes wide accesses, to a multiple of 8
    int act;
    const void *bias, *residual;
    void *y, *pre;
    int64_t ldy, ldr, ldpre;
    float *partial;                      // [splits][M][ldp], or NULL
    uint8_t *codes;                      // [M][N] (through a tensor map: rows of N up to a multiple of 16), or NULL
    float *scales;                       // [M][nblk]
    int nblk, keep;
    int32_t *error;                      // host memory: set if a wait ran out
};

// A tile is kPair ? 256 : 128 rows by kBN columns.  kKeep: what a backward pass
// needs leaves too, through a third tile of each epilogue warp.
template <int kBN, bool kPair, bool kKeep>
struct Layout {
    static constexpr int kNB = kPair ? kBN / 2 : kBN;  // rows of B this CTA stages
    static constexpr int kTileM = kPair ? 2 * kBM : kBM;
    static constexpr int kEpiWarps = 16;
    static constexpr int kBufs = kBN == 256 ? 2 : 4;     // accumulators, and groups of epilogue warps
    static constexpr int kGroupWarps = kEpiWarps / kBufs;
    static constexpr int kSpan = kBN < 128 ? kBN : 128;  // columns of a warp in a group
    static constexpr int kThreads = (kEpiWarps + 2) * 32;
    static constexpr int kA = kBM * kBK * 2;
    static constexpr int kB = kNB * kBK * 2;
    static constexpr int kStage = kA + kB;
    static constexpr int kStages = kNB == 64 ? (kKeep ? 5 : 6) : (kKeep ? 4 : 5);
    static constexpr int offStaging = kStages * kStage;
    static constexpr int kWarpTile = kStagingWarp + (kKeep ? kTileBytes : 0);
    static constexpr int offBar = offStaging + kEpiWarps * kWarpTile;
    static constexpr int kBars = 2 * kStages + 3 * kBufs + 1 + 2 * kEpiWarps;
    static constexpr int offSlot = offBar + kBars * 8;
    static constexpr int kBytes = offSlot + 16;
    static constexpr int kAlloc = kBytes + 1024;  // the base is rounded up to 1024
    static_assert(kAlloc <= 227 * 1024, "shared memory");
};

// Unit -> (row tile, column tile, split).  Tiles run through groups of group_m
// row tiles, column by column, so that the CTAs of a wave share operand tiles
// in L2; the splits of a tile are neighbours.
__device__ __forceinline__ void unit_coords(const Params &p, int unit, int &tm, int &tn, int &sp) {
    const int t = divide(unit, p.splits);
    sp = unit - t * (int)p.splits.d;
    const int g = divide(t, p.group);
    const int rest = t - g * (int)p.group.d;
    const int m0 = g * p.group_m;
    const bool last = p.tiles_m - m0 < p.group_m;
    tn = last ? divide(rest, p.gm_last) : divide(rest, p.gm);
    tm = m0 + rest - tn * (int)(last ? p.gm_last.d : p.gm.d);
}

// A block's scale, and the codes of eight of its values.
__device__ __forceinline__ float keep_scale(int keep, float amax) {
    return keep == FCAI_KEEP_E4M3 ? block_scale<true>(amax) : block_scale<false>(amax);
}
__device__ __forceinline__ uint2 keep_codes(int keep, const V8 &v, float scale) {
    const float inv = __frcp_rn(scale);
    return keep == FCAI_KEEP_E4M3 ? encode8<true>(v, inv) : encode8<false>(v, inv);
}
__device__ __forceinline__ float amax8(const F2 *v) {
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = split(v[i]);
        m = max_nan(m, max_nan(fabsf(f.x), fabsf(f.y)));
    }
    return m;
}

template <typename T>
__device__ __forceinline__ uint4 pack8(const F2 *v) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = split(v[i]);
        w[i] = pack2(f.x, f.y, T());
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}
template <typename T>
__device__ __forceinline__ void unpack8(const uint4 &q, F2 *v) {
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = unpack2(w[i], T());
        v[i] = f2(f.x, f.y);
    }
}

template <typename T>
__device__ __forceinline__ void finish1(const Params &p, int64_t row, int col, float v) {
    if (p.pre) static_cast<T *>(p.pre)[row * p.ldpre + col] = from_f32<T>(v);
    v = act_1(p.act, v);
    if (p.residual) v += to_f32(static_cast<const T *>(p.residual)[row * p.ldr + col]);
    static_cast<T *>(p.y)[row * p.ldy + col] = from_f32<T>(v);
}
template <typename T>
__device__ __forceinline__ void add_bias8(const Params &p, int col, F2 (&v)[4]) {
    if (!p.bias) return;
    F2 b[4];
    unpack8<T>(__ldg(reinterpret_cast<const uint4 *>(static_cast<const T *>(p.bias) + col)), b);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = add2(v[i], b[i]);
}

// Shared memory by its 32-bit address: through a pointer computed from a
// rounded base the compiler would use generic accesses.
__device__ __forceinline__ void sts128(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ float4 lds128(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ uint4 lds128u(uint32_t addr) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ float lds32(uint32_t addr) {
    float v;
    asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
    return v;
}

// The bias of 32 columns that every lane has alike, 8 at a time (a ragged or
// unaligned bias was copied: narrow loads here, even where no call takes them,
// cost every product registers; 36864 x 192 -> 768 took 34.3 us in a graph instead
// of 32.1).
template <typename T>
__device__ __forceinline__ void add_bias32(const Params &p, int col0, F2 (&v)[16]) {
    if (!p.bias) return;
#pragma unroll
    for (int g = 0; g < 4; ++g) {
        if (col0 + 8 * g >= p.N) break;
        F2 b[4];
        unpack8<T>(__ldg(reinterpret_cast<const uint4 *>(static_cast<const T *>(p.bias) + col0 + 8 * g)), b);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[4 * g + e] = add2(v[4 * g + e], b[e]);
    }
}
// A lane's 32 values as its row of a 32 x 32 tile: 64 bytes, in the 64-byte
// swizzle of the tensor maps (free of bank conflicts).
template <typename T>
__device__ __forceinline__ void put_row(uint32_t tile, int lane, const F2 (&v)[16]) {
#pragma unroll
    for (int g = 0; g < 4; ++g) {
        const uint4 q = pack8<T>(v + 4 * g);
        sts128(tile + lane * 64 + ((g ^ ((lane >> 1) & 3)) << 4), q.x, q.y, q.z, q.w);
    }
}

// The two ways around TMA: fp32 partial tiles, and outputs whose rows do not
// take 16-byte accesses.  `stg`: the warp's 32 x 32 fp32 tile, row-swizzled.
template <typename T>
__device__ __forceinline__ void write_plain(const Params &p, uint32_t stg, int row0, int col0, int sp, int lane) {
    if (p.partial) {
        const int col = col0 + (lane & 3) * 8, r0 = lane >> 2, row = row0 + r0;
        if (col >= p.ldp) return;  // a multiple of 8
        const uint32_t src = stg + r0 * 128;
        const uint32_t c0 = ((2 * (lane & 3)) ^ r0) << 4;  // r0 < 8: the rows' swizzle
        float *dst = p.partial + ((int64_t)sp * p.M + row) * p.ldp + col;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (row + i * 8 >= p.M) break;
            reinterpret_cast<float4 *>(dst + (int64_t)i * 8 * p.ldp)[0] = lds128(src + i * 1024 + c0);
            reinterpret_cast<float4 *>(dst + (int64_t)i * 8 * p.ldp)[1] = lds128(src + i * 1024 + (c0 ^ 16));
        }
        return;
    }
    const int col = col0 + lane;
    if (col >= p.N) return;
    const float bias = p.bias ? to_f32(static_cast<const T *>(p.bias)[col]) : 0.f;
    // eight rows' residuals at a time are on their way before the first is used
#pragma unroll 1
    for (int r = 0; r < 32 && row0 + r < p.M; r += 8) {
        const int left = p.M - row0 - r;
        float res[8], v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e)
            res[e] = p.residual && e < left ? to_f32(static_cast<const T *>(p.residual)[(row0 + r + e) * p.ldr + col]) : 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = lds32(stg + (r + e) * 128 + (((lane >> 2) ^ e) << 4) + (lane & 3) * 4) + bias;
        if (p.pre) {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (e < left) static_cast<T *>(p.pre)[(row0 + r + e) * p.ldpre + col] = from_f32<T>(v[e]);
        }
        F2 w[4] = {f2(v[0], v[1]), f2(v[2], v[3]), f2(v[4], v[5]), f2(v[6], v[7])};
        act_n<4, true>(p.act, w);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float2 f = split(w[e / 2]);
            if (e < left) static_cast<T *>(p.y)[(row0 + r + e) * p.ldy + col] = from_f32<T>((e & 1 ? f.y : f.x) + res[e]);
        }
    }
}

struct Maps {
    CUtensorMap a, b;           // operands
    CUtensorMap y, res, extra;  // 32 x 32 tiles of y, the residual, and pre or the codes (where they are used)
};

// kTA / kTB: the operand's rows run along K (its M / N axis is contiguous).
// kPair: clusters of two CTAs share each MMA (cta_group::2, M = 256): each CTA
// stages its 128 rows of A and half the columns' rows of B and owns 128 rows
// of the accumulator; the rank-0 CTA issues for both.
template <typename T, int kBN, bool kPair, bool kTA, bool kTB, bool kKeep>
__global__ void __launch_bounds__(Layout<kBN, kPair, kKeep>::kThreads, 1)
    linear_tc_kernel(const __grid_constant__ Maps maps, const Params p) {
    using Lay = Layout<kBN, kPair, kKeep>;
    const CUtensorMap &tmA = maps.a, &tmB = maps.b;
    constexpr int kStages = Lay::kStages, kEpiWarps = Lay::kEpiWarps, kBufs = Lay::kBufs;
    extern __shared__ unsigned char smem_raw[];
    unsigned char *smem =
        reinterpret_cast<unsigned char *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t *full = reinterpret_cast<uint64_t *>(smem + Lay::offBar);  // pairs: rank 0's counts both CTAs' loads
    uint64_t *empty = full + kStages;
    uint64_t *accf = empty + kStages;  // accumulator filled (by the MMA warp; pairs: in both CTAs)
    uint64_t *acce = accf + kBufs;     // accumulator read: one arrival per epilogue warp of this CTA that reads it
    uint64_t *pacce = acce + kBufs;    // pairs, rank 0: the peer's accumulator read
    uint64_t *resbar = pacce + kBufs;  // residual tiles loaded: two per epilogue warp
    uint64_t *dbar = resbar + 2 * kEpiWarps;        // abort path: this CTA's MMAs drained
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(smem + Lay::offSlot);
    volatile int *abort = reinterpret_cast<volatile int *>(smem + Lay::offSlot + 4);

    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    const uint32_t rank = kPair ? cluster_ctarank() : 0u;
    const bool leader = rank == 0;
    const int unit0 = kPair ? (int)(blockIdx.x >> 1) : (int)blockIdx.x;
    const int unit_step = kPair ? (int)(gridDim.x >> 1) : (int)gridDim.x;
    constexpr uint32_t kTmemCols = kBufs * kBN;

    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        for (int b = 0; b < kBufs; ++b) {
            mbar_init(&accf[b], 1);
            mbar_init(&acce[b], p.coop ? (kBN < 128 ? kBN / 32 * 4 : kEpiWarps) : Lay::kGroupWarps);
            mbar_init(&pacce[b], 1);
        }
        for (int b = 0; b < 2 * kEpiWarps; ++b) mbar_init(&resbar[b], 1);
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
                if (!mbar_wait_warp_idle(&empty[s], (r & 1) ^ 1, abort, kWaitNs)) {
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
                const int buf = j % kBufs;
                const uint32_t parity = ((j / kBufs) & 1) ^ 1;
                if (!mbar_wait_warp(&acce[buf], parity, abort, kWaitNs) ||
                    (kPair && !mbar_wait_warp(&pacce[buf], parity, abort, kWaitNs, true))) {
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
        } else {
            // The peer's accumulators are free: passed on by this warp, since an
            // arrival in another CTA waits until the arriving thread's earlier
            // stores have been seen, and the epilogue's lanes always have some.
            int j = 0;
            for (int unit = unit0; unit < p.units; unit += unit_step, ++j) {
                if (!mbar_wait_warp_idle(&acce[j % kBufs], (j / kBufs) & 1, abort, kWaitNs)) {
                    *abort = 1;
                    break;
                }
                if (lane == 0) mbar_arrive_cluster(mapa_shared(smem_u32(&pacce[j % kBufs]), 0));
            }
        }
        __syncwarp();
    } else {
        // ------------------------------------------------------------ epilogue
        const int q = warp & 3;
        // the warp's tiles (every jstep-th from j0 on) and its columns of each
        const int j0 = p.coop ? 0 : warp / Lay::kGroupWarps, jstep = p.coop ? 1 : kBufs;
        const int cbegin = p.coop ? (warp >> 2) * 32 : (warp % Lay::kGroupWarps) / 4 * 128;
        const int cstep = p.coop ? 128 : 32, cend = p.coop ? kBN : cbegin + Lay::kSpan;
        const uint32_t staging = smem_u32(smem + Lay::offStaging) + warp * Lay::kWarpTile;
        const uint32_t extra = staging + kStagingWarp;
        const uint32_t stg = staging + lane * 128 + ((lane & 7) << 4);  // this row of an fp32 tile, chunk 0
        const uint32_t rbar = smem_u32(&resbar[2 * warp]);
        const bool tma = p.tma, residual = tma && p.residual;
        uint32_t n = 0;  // chunks through the two tiles so far
        // Lane 0: the residual's rows and columns of chunk `i` into tile i % 2,
        // whose last store (chunk i - 2) has been read.
        auto fetch_residual = [&](uint32_t i, int col, int row) {
            const uint32_t bar = rbar + (i & 1) * 8;
            asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(kTileBytes) : "memory");
            tma_load_2d(staging + (i & 1) * kTileBytes, &maps.res, bar, col, row);
        };
        if (cbegin < kBN)
            for (int j = j0, unit = unit0 + j0 * unit_step; unit < p.units; j += jstep, unit += jstep * unit_step) {
                int tm, tn, sp;
                unit_coords(p, unit, tm, tn, sp);
                const int buf = j % kBufs;
                const int row0 = tm * Lay::kTileM + (int)rank * kBM + q * 32;
                const int ctile = tn * kBN;
                const int cmax = row0 < p.M ? min(cend, p.N - ctile) : cbegin;  // columns that are there: chunks below it
                if (residual && cbegin < cmax && lane == 0) {  // on its way while the accumulator fills
                    bulk_wait_read_but_one();
                    fetch_residual(n, ctile + cbegin, row0);
                }
                if (!mbar_wait_warp_idle(&accf[buf], (j / kBufs) & 1, abort, kWaitNs)) {
                    *abort = 1;
                    if (residual && cbegin < cmax) mbar_wait(&resbar[2 * warp + (n & 1)], (n >> 1) & 1, nullptr, kWaitNs / 10);
                    break;
                }
                tc_fence_after();
                const uint32_t taddr = tmem_base + buf * kBN + ((uint32_t)(q * 32) << 16);
                float inv = 1.f;  // codes: 1 / scale of this lane's row
                if (kKeep && p.codes && !p.partial && cbegin < cmax) {
                    // first pass: the largest magnitude of the row's block
                    float m = 0.f;
#pragma unroll 1
                    for (int c = cbegin; c < cmax; c += 32) {
                        uint32_t w[32];
                        tmem_ld32(taddr + c, w);
                        tmem_wait_ld();
                        F2 v[16];
#pragma unroll
                        for (int e = 0; e < 16; ++e) v[e] = f2(__uint_as_float(w[2 * e]), __uint_as_float(w[2 * e + 1]));
                        add_bias32<T>(p, ctile + c, v);
#pragma unroll
                        for (int e = 0; e < 16; e += 4) m = max_nan(m, amax8(v + e));
                    }
                    const float s = keep_scale(p.keep, m);
                    if (row0 + lane < p.M) p.scales[(int64_t)(row0 + lane) * p.nblk + (ctile + cbegin) / FCAI_KEEP_BLOCK] = s;
                    inv = __frcp_rn(s);
                }
                bool ok = true;
#pragma unroll 1
                for (int c = cbegin; c < cend; c += cstep) {
                    uint32_t w[32];
                    tmem_ld32(taddr + c, w);
                    tmem_wait_ld();
                    if (c + cstep >= cend) {  // this warp has read its part of the accumulator
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&acce[buf]);
                    }
                    if (c >= cmax) continue;
                    const int col0 = ctile + c;
                    if (!tma) {
#pragma unroll
                        for (int e = 0; e < 8; ++e) sts128(stg ^ (e << 4), w[4 * e], w[4 * e + 1], w[4 * e + 2], w[4 * e + 3]);
                        __syncwarp();
                        write_plain<T>(p, staging, row0, col0, sp, lane);
                        __syncwarp();
                        continue;
                    }
                    F2 v[16];
#pragma unroll
                    for (int e = 0; e < 16; ++e) v[e] = f2(__uint_as_float(w[2 * e]), __uint_as_float(w[2 * e + 1]));
                    add_bias32<T>(p, col0, v);
                    const uint32_t tile = staging + (n & 1) * kTileBytes;
                    if (lane == 0) bulk_wait_read_but_one();  // this chunk's tile, and the extra one, may be written
                    __syncwarp();
                    if (kKeep && p.codes) {
                        // the row's 32 codes, in the 32-byte swizzle of their map
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const V8 x = {v[8 * h], v[8 * h + 1], v[8 * h + 2], v[8 * h + 3]}, y = {v[8 * h + 4], v[8 * h + 5], v[8 * h + 6], v[8 * h + 7]};
                            const uint2 a = p.keep == FCAI_KEEP_E4M3 ? encode8<true>(x, inv) : encode8<false>(x, inv);
                            const uint2 b = p.keep == FCAI_KEEP_E4M3 ? encode8<true>(y, inv) : encode8<false>(y, inv);
                            sts128(extra + lane * 32 + ((h ^ ((lane >> 2) & 1)) << 4), a.x, a.y, b.x, b.y);
                        }
                    } else if (kKeep && p.pre) {
                        put_row<T>(extra, lane, v);
                    }
                    if (kKeep && (p.codes || p.pre)) {
                        fence_proxy_async_smem();
                        __syncwarp();
                        if (lane == 0) {
                            tma_store_2d(&maps.extra, extra, col0, row0);
                            bulk_commit_group();
                        }
                    }
                    act_n(p.act, v);
                    if (residual) {
                        if (lane == 0 && c + cstep < cmax) {
                            // the other tile's store (the previous chunk's) has been read; the extra one's may be pending
                            if (kKeep && (p.codes || p.pre)) bulk_wait_read_but_one();
                            else bulk_wait_read_all();
                            fetch_residual(n + 1, col0 + cstep, row0);
                        }
                        __syncwarp();
                        ok = mbar_wait_warp_idle(&resbar[2 * warp + (n & 1)], (n >> 1) & 1, abort, kWaitNs);
                        if (!ok) {
                            *abort = 1;
                            if (c + cstep < cmax) mbar_wait(&resbar[2 * warp + ((n + 1) & 1)], ((n + 1) >> 1) & 1, nullptr, kWaitNs / 10);
                            break;
                        }
#pragma unroll
                        for (int g = 0; g < 4; ++g) {
                            F2 r[4];
                            unpack8<T>(lds128u(tile + lane * 64 + ((g ^ ((lane >> 1) & 3)) << 4)), r);
#pragma unroll
                            for (int e = 0; e < 4; ++e) v[4 * g + e] = add2(v[4 * g + e], r[e]);
                        }
                    }
                    put_row<T>(tile, lane, v);
                    fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) {
                        tma_store_2d(&maps.y, tile, col0, row0);
                        bulk_commit_group();
                    }
                    ++n;
                }
                if (!ok) break;
            }
        if (lane == 0) bulk_wait_all();  // stores complete before the CTA exits
        __syncwarp();
    }

    // ---------------------------------------------------------------- teardown
    __syncthreads();
    if (*abort) {
        if (threadIdx.x == 0) *static_cast<volatile int32_t *>(p.error) = 1;
        // TMEM is freed only once every MMA issued has completed
        if (leader && warp == kEpiWarps + 1) {
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

// Sums the splits in a fixed order and applies the epilogue: 16 lanes a row's 128
// columns, 8 each, so that an 8-bit block is theirs.  Few rows: kParts groups of
// 16 lanes share a row's splits (every kParts-th each) and the first one adds
// their sums, since one group's loads alone would leave most SMs idle.  Also the
// second half of a product that keeps codes but whose rows do not take wide
// accesses.
template <typename T, int kParts>
__global__ void __launch_bounds__(256) reduce_kernel(const Params p) {
    __shared__ __align__(16) float sums[16][128];  // the parts' sums; rows on their way to narrow stores
    constexpr int kRows = 16 / kParts;  // rows a CTA and step
    const int group = threadIdx.x >> 4, split0 = group / kRows;
    const int col = blockIdx.x * FCAI_KEEP_BLOCK + (threadIdx.x & 15) * 8;
    const int64_t step = (int64_t)p.M * p.ldp;
    // every thread runs the same steps: barriers, and a block's shuffles need whole warps
    for (int64_t r0 = (int64_t)blockIdx.y * kRows; r0 < p.M; r0 += (int64_t)gridDim.y * kRows) {
        const int64_t row = r0 + group % kRows;
        bool in = row < p.M && col < p.N;
        F2 v[4] = {f2(0.f), f2(0.f), f2(0.f), f2(0.f)};
        if (in) {
            const float *src = p.partial + row * p.ldp + col + split0 * step;
#pragma unroll 4
            for (int s = split0; s < (int)p.splits.d; s += kParts, src += kParts * step) {
                const float4 a = __ldg(reinterpret_cast<const float4 *>(src)), b = __ldg(reinterpret_cast<const float4 *>(src) + 1);
                v[0] = add2(v[0], f2(a.x, a.y)), v[1] = add2(v[1], f2(a.z, a.w));
                v[2] = add2(v[2], f2(b.x, b.y)), v[3] = add2(v[3], f2(b.z, b.w));
            }
        }
        if constexpr (kParts > 1) {
            float *mine = &sums[group][(threadIdx.x & 15) * 8];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float2 f = split(v[e]);
                mine[2 * e] = f.x, mine[2 * e + 1] = f.y;
            }
            __syncthreads();
            in = in && split0 == 0;
            if (in) {
#pragma unroll
                for (int q = 1; q < kParts; ++q) {
                    const float *o = &sums[group + q * kRows][(threadIdx.x & 15) * 8];
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] = add2(v[e], f2(o[2 * e], o[2 * e + 1]));
                }
            }
            __syncthreads();
        }
        if (in) {
            if (p.vec) {
                add_bias8<T>(p, col, v);
            } else if (p.bias) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    auto at = [&](int c) { return c < p.N ? to_f32(static_cast<const T *>(p.bias)[c]) : 0.f; };
                    v[e] = add2(v[e], f2(at(col + 2 * e), at(col + 2 * e + 1)));
                }
            }
        }
        uint2 codes = make_uint2(0u, 0u);
        if (p.codes) {
            // columns from N on are zeros: their weights were, and no bias was added
            float m = in ? amax8(v) : 0.f;
#pragma unroll
            for (int d = 8; d >= 1; d >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, d));
            if (in) {
                const float s = keep_scale(p.keep, m);
                const uint2 q = keep_codes(p.keep, V8{v[0], v[1], v[2], v[3]}, s);
                if (p.vec) *reinterpret_cast<uint2 *>(p.codes + row * p.N + col) = q;
                codes = q;
                if ((threadIdx.x & 15) == 0) p.scales[row * p.nblk + blockIdx.x] = s;
            }
        }
        if (p.vec) {
            if (!in) continue;
            if (p.pre) *reinterpret_cast<uint4 *>(static_cast<T *>(p.pre) + row * p.ldpre + col) = pack8<T>(v);
            act_n(p.act, v);
            if (p.residual) {
                F2 r[4];
                unpack8<T>(__ldg(reinterpret_cast<const uint4 *>(static_cast<const T *>(p.residual) + row * p.ldr + col)), r);
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = add2(v[e], r[e]);
            }
            *reinterpret_cast<uint4 *>(static_cast<T *>(p.y) + row * p.ldy + col) = pack8<T>(v);
        } else {
            // narrow accesses: the row through shared memory, so that neighbouring lanes have neighbouring columns
            float *mine = sums[group];
            const int l = threadIdx.x & 15;
            auto put = [&]() {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float2 f = split(v[e]);
                    mine[l * 8 + 2 * e] = f.x, mine[l * 8 + 2 * e + 1] = f.y;
                }
            };
            const bool here = row < p.M && (kParts == 1 || split0 == 0);
            __syncwarp();
            if (p.codes) {
                reinterpret_cast<uint2 *>(mine)[l] = codes;
                __syncwarp();
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const int c = blockIdx.x * FCAI_KEEP_BLOCK + l + 16 * e;
                    if (here && c < p.N) p.codes[row * p.N + c] = reinterpret_cast<const uint8_t *>(mine)[l + 16 * e];
                }
                __syncwarp();
            }
            if (p.pre) {
                put();
                __syncwarp();
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const int c = blockIdx.x * FCAI_KEEP_BLOCK + l + 16 * e;
                    if (here && c < p.N) static_cast<T *>(p.pre)[row * p.ldpre + c] = from_f32<T>(mine[l + 16 * e]);
                }
                __syncwarp();
            }
            act_n(p.act, v);
            put();
            __syncwarp();
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int c = blockIdx.x * FCAI_KEEP_BLOCK + l + 16 * e;
                if (!here || c >= p.N) continue;
                const float r = p.residual ? to_f32(static_cast<const T *>(p.residual)[row * p.ldr + c]) : 0.f;
                static_cast<T *>(p.y)[row * p.ldy + c] = from_f32<T>(mine[l + 16 * e] + r);
            }
            if constexpr (kParts > 1) __syncthreads();  // the rows' sums come to the same memory
            else __syncwarp();
        }
    }
}

// Up to four matrices that TMA cannot read, [rows][cols] with row stride ld,
// into dst[rows][ldd], 16 bytes a thread and step.  Rows start at any element,
// so a thread's eight come as 4-byte words: four of them, or, from an odd
// element on, three between two single elements, shifted together; nothing
// outside the row is read.
struct Repack {
    const uint16_t *src;
    uint16_t *dst;
    int64_t ld, rows;
    int cols, ldd;
    FastDiv chunks;  // of 8 elements a row
    int step;        // rows of a CTA and step
};
struct Repacks {
    Repack r[4];
};
__global__ void __launch_bounds__(256) repack_kernel(const Repacks all) {
    const Repack &o = all.r[blockIdx.y];
    const int chunks = (int)o.chunks.d;
    for (int64_t row0 = (int64_t)blockIdx.x * o.step; row0 < o.rows; row0 += (int64_t)gridDim.x * o.step) {
        const int n = (int)min((int64_t)o.step, o.rows - row0) * chunks;
#pragma unroll 2
        for (int i = threadIdx.x; i < n; i += 256) {
            const int r = divide(i, o.chunks), col = (i - r * chunks) * 8;
            const uint16_t *src = o.src + (row0 + r) * o.ld + col;
            uint32_t w[4];
            if (col + 8 > o.cols) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    w[e] = col + 2 * e < o.cols ? (uint32_t)__ldg(src + 2 * e) : 0u;
                    if (col + 2 * e + 1 < o.cols) w[e] |= (uint32_t)__ldg(src + 2 * e + 1) << 16;
                }
            } else if (reinterpret_cast<uintptr_t>(src) & 2) {
                const uint32_t first = __ldg(src), end = __ldg(src + 7);
                const uint32_t *q = reinterpret_cast<const uint32_t *>(src + 1);
                const uint32_t q0 = __ldg(q), q1 = __ldg(q + 1), q2 = __ldg(q + 2);
                w[0] = first | q0 << 16;
                w[1] = __funnelshift_r(q0, q1, 16);
                w[2] = __funnelshift_r(q1, q2, 16);
                w[3] = q2 >> 16 | end << 16;
            } else {
                const uint32_t *q = reinterpret_cast<const uint32_t *>(src);
#pragma unroll
                for (int e = 0; e < 4; ++e) w[e] = __ldg(q + e);
            }
            *reinterpret_cast<uint4 *>(o.dst + (row0 + r) * o.ldd + col) = make_uint4(w[0], w[1], w[2], w[3]);
        }
    }
}

// The way back: padded rows src[rows][lds] to dst[rows][cols] with row stride ldd,
// whose rows start at any element.  A thread's 16 bytes are aligned in dst, so
// that all but a row's first and last sectors are written whole; the direct narrow
// stores left most sectors partial, and the backward pass of 28106 x 1730 -> 24 took
// 197 us instead of 167.  The padding, to 16 bytes at least, takes the words that
// reach past the row's end.
struct Unpad {
    const void *src;
    void *dst;
    int64_t lds, ldd, rows;
    int cols;
    FastDiv chunks;  // aligned 16-byte pieces of a row: one more than its length asks for
    int step;        // rows of a CTA and step
};
template <typename E>
__global__ void __launch_bounds__(256) unpad_kernel(const Unpad o) {
    constexpr int kChunk = 16 / sizeof(E);
    const int chunks = (int)o.chunks.d;
    for (int64_t row0 = (int64_t)blockIdx.x * o.step; row0 < o.rows; row0 += (int64_t)gridDim.x * o.step) {
        const int n = (int)min((int64_t)o.step, o.rows - row0) * chunks;
#pragma unroll 2
        for (int i = threadIdx.x; i < n; i += 256) {
            const int r = divide(i, o.chunks);
            E *dst = static_cast<E *>(o.dst) + (row0 + r) * o.ldd;
            const int col = (i - r * chunks) * kChunk - (int)((reinterpret_cast<uintptr_t>(dst) & 15) / sizeof(E));
            const E *src = static_cast<const E *>(o.src) + (row0 + r) * o.lds + col;
            if (col >= 0 && col + kChunk <= o.cols) {
                const uint32_t shift = (uint32_t)(reinterpret_cast<uintptr_t>(src) & 3) * 8;
                const uint32_t *q = reinterpret_cast<const uint32_t *>(reinterpret_cast<uintptr_t>(src) & ~uintptr_t(3));
                const uint32_t q0 = __ldg(q), q1 = __ldg(q + 1), q2 = __ldg(q + 2), q3 = __ldg(q + 3), q4 = shift ? __ldg(q + 4) : 0u;
                *reinterpret_cast<uint4 *>(dst + col) = make_uint4(__funnelshift_r(q0, q1, shift), __funnelshift_r(q1, q2, shift),
                                                                   __funnelshift_r(q2, q3, shift), __funnelshift_r(q3, q4, shift));
            } else {
#pragma unroll
                for (int e = 0; e < kChunk; ++e)
                    if (col + e >= 0 && col + e < o.cols) dst[col + e] = __ldg(src + e);
            }
        }
    }
}

// ---- few rows -----------------------------------------------------------------
// y for up to 8 * kNB rows of x: every weight is read once, 16 bytes a lane, and
// the sums run on warp-level MMAs (m16n8k16: 16 rows of w by 8 rows of x).
// Lane (g, t) = (lane / 4, lane % 4) holds 8 consecutive k of w's rows g and g + 8
// and of x's row g; an MMA takes k in any order as long as both operands agree,
// so these 8 serve two MMAs as they were loaded.  A CTA owns 16 columns of y;
// its warps take K in turns of 32, and their sums meet in shared memory in a
// fixed order.  Bound by reading w, and by the launch: a warp has 8 loads of 512
// bytes of w in flight (4 above 16 rows), 16 warps a CTA for long rows (1 x 4096 ->
// 4096 in a graph: 4.8 us with w in L2, 9.1 with w from memory).  Rows that do not
// take 16-byte accesses are read by single elements.
template <typename T> __device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma16816<__nv_bfloat16>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma16816<__half>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
struct FewRows {
    const void *x, *w;
    int64_t ldx, ldw;
    int K;
};
// k .. k + 7 of a row (zeros past K, and everything for a row that is not there)
template <bool kV>
__device__ __forceinline__ uint4 load_k8(const uint16_t *row, int k, int K, bool in) {
    uint4 q = make_uint4(0u, 0u, 0u, 0u);
    if (kV) {
        if (in && k < K) q = __ldg(reinterpret_cast<const uint4 *>(row + k));
    } else {
        uint32_t w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (in && k + i < K) w[i / 2] |= (uint32_t)__ldg(row + k + i) << (16 * (i & 1));
        q = make_uint4(w[0], w[1], w[2], w[3]);
    }
    return q;
}
template <typename T, int kNB, int kWarps, bool kV>
__global__ void __launch_bounds__(kWarps * 32) few_rows_kernel(const FewRows f, const Params p) {
    __shared__ float sums[kWarps][kNB * 128];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int n0 = blockIdx.x * 16;
    const uint16_t *w0 = static_cast<const uint16_t *>(f.w) + (int64_t)(n0 + g) * f.ldw;
    const uint16_t *w1 = w0 + 8 * f.ldw;
    const bool in0 = n0 + g < p.N, in1 = n0 + g + 8 < p.N;
    float d[kNB][4];
#pragma unroll
    for (int b = 0; b < kNB; ++b) d[b][0] = d[b][1] = d[b][2] = d[b][3] = 0.f;
    constexpr int kUnroll = kNB == 4 ? 2 : 4;
    for (int k0 = warp * 32; k0 < f.K; k0 += kWarps * 32 * kUnroll) {
        uint4 a0[kUnroll], a1[kUnroll], x[kUnroll][kNB];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            const int k = k0 + u * kWarps * 32 + t * 8;
            a0[u] = load_k8<kV>(w0, k, f.K, in0);
            a1[u] = load_k8<kV>(w1, k, f.K, in1);
#pragma unroll
            for (int b = 0; b < kNB; ++b)
                x[u][b] = load_k8<kV>(static_cast<const uint16_t *>(f.x) + (int64_t)(b * 8 + g) * f.ldx, k, f.K, b * 8 + g < p.M);
        }
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            const uint32_t lo[4] = {a0[u].x, a1[u].x, a0[u].y, a1[u].y}, hi[4] = {a0[u].z, a1[u].z, a0[u].w, a1[u].w};
#pragma unroll
            for (int b = 0; b < kNB; ++b) {
                mma16816<T>(d[b], lo, x[u][b].x, x[u][b].y);
                mma16816<T>(d[b], hi, x[u][b].z, x[u][b].w);
            }
        }
    }
    // d: rows g, g + 8 of w by rows 2 t, 2 t + 1 of x -> sums[warp][x row][w row]
#pragma unroll
    for (int b = 0; b < kNB; ++b) {
        float *s = sums[warp] + (b * 8 + 2 * t) * 16 + g;
        s[0] = d[b][0], s[16] = d[b][1], s[8] = d[b][2], s[24] = d[b][3];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < kNB * 128; i += kWarps * 32) {
        const int row = i >> 4, col = n0 + (i & 15);
        if (row >= p.M || col >= (p.partial ? p.ldp : p.N)) continue;  // columns from N to ldp: zeros
        float v = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) v += sums[w][i];
        if (p.partial) {  // the epilogue follows in reduce_kernel, which sees whole 8-bit blocks
            p.partial[(int64_t)row * p.ldp + col] = v;
            continue;
        }
        if (p.bias) v += to_f32(static_cast<const T *>(p.bias)[col]);
        finish1<T>(p, row, col, v);
    }
}

// y = 0, a weight gradient over no rows; zero is the same bits in both types.
__global__ void empty_product_kernel(const Params p) {
    const int64_t n = (int64_t)p.M * p.N;
    for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < n; i += (int64_t)gridDim.x * blockDim.x)
        static_cast<uint16_t *>(p.y)[i / p.N * p.ldy + i % p.N] = 0;
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

// One word for each device, of pinned memory that the device can write; NULL
// without a device.  It is made outside any capture that a first call is part of.
static volatile int32_t *error_word() {
    static std::atomic<int32_t *> words[64];
    static std::mutex making;
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return nullptr;
    int32_t *word = words[dev].load(std::memory_order_acquire);
    if (word) return word;
    const std::lock_guard<std::mutex> lock(making);
    word = words[dev].load(std::memory_order_acquire);
    if (word) return word;
    cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
    if (cudaThreadExchangeStreamCaptureMode(&mode) != cudaSuccess) return nullptr;
    void *p = nullptr;
    if (cudaHostAlloc(&p, sizeof(int32_t), cudaHostAllocPortable | cudaHostAllocMapped) == cudaSuccess) {
        word = static_cast<int32_t *>(p);
        *word = 0;
        words[dev].store(word, std::memory_order_release);
    }
    cudaThreadExchangeStreamCaptureMode(&mode);
    return word;
}
static int check_errors() {
    volatile int32_t *word = error_word();
    if (!word) return fcai::fail(FCAI_ERR_CUDA, "linear: no device, or no pinned memory for its error word");
    if (!*word) return FCAI_OK;
    *word = 0;
    return fcai::fail(FCAI_ERR_CUDA, "linear: a pipeline wait of an earlier product on this device ran out; its results are wrong");
}

constexpr int kCodeType = 100;  // a map of codes: bytes
// A row-major matrix [outer][inner] as boxes of box_cols x box_rows elements,
// swizzled over the box's row: 64 16-bit columns 128 bytes (operands), 32 64
// bytes, 32 codes 32 bytes (results).
static int make_map(CUtensorMap *map, const void *base, int64_t inner, int64_t outer, int64_t ld, int box_rows, int dtype,
                    int box_cols = 64) {
    auto fn = encode_fn();
    if (!fn) return fcai::fail(FCAI_ERR_CUDA, "cuTensorMapEncodeTiled is unavailable");
    const int size = dtype == kCodeType ? 1 : 2;
    const cuuint64_t dims[2] = {(cuuint64_t)inner, (cuuint64_t)outer};
    const cuuint64_t strides[1] = {(cuuint64_t)ld * size};
    const cuuint32_t box[2] = {(cuuint32_t)box_cols, (cuuint32_t)box_rows};
    const cuuint32_t es[2] = {1, 1};
    const CUtensorMapSwizzle sw = box_cols * size == 128 ? CU_TENSOR_MAP_SWIZZLE_128B
                                  : box_cols * size == 64 ? CU_TENSOR_MAP_SWIZZLE_64B
                                                          : CU_TENSOR_MAP_SWIZZLE_32B;
    const CUtensorMapDataType type = dtype == kCodeType         ? CU_TENSOR_MAP_DATA_TYPE_UINT8
                                     : dtype == FCAI_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                                : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    const CUresult r = fn(map, type, 2, const_cast<void *>(base), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE, sw,
                          CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
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
// reduce: the epilogue runs in reduce_kernel even without splits; codes: tiles hold whole 8-bit blocks.
static Plan make_plan(int64_t M, int64_t N, int64_t K, bool reduce = false, bool codes = false) {
    struct Shape {
        int bn, pair;
        double kstep, epilogue;  // clocks a K step; clocks of a tile's epilogue
    };
    static const Shape shapes[3] = {{256, 1, 540., 3000.}, {128, 0, 560., 1500.}, {64, 0, 400., 1300.}};
    const int sms = fcai::sm_count();
    Plan best{};
    double best_time = 0.;
    for (const Shape &sh : shapes) {
        if (sh.bn > 64 && N <= sh.bn / 2) continue;
        if (codes && sh.bn < FCAI_KEEP_BLOCK && N > sh.bn) continue;
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
        pl.partial_bytes = pl.splits > 1 || reduce ? round256((int64_t)pl.splits * M * round8((int)N) * 4) : 0;
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

// Rows a CTA copies at a time: 2048 chunks' worth, or fewer where that would leave
// SMs idle (777 x 321 and 577 x 321: 5.1 us with 16 CTAs each).
static int rows_a_step(int64_t rows, int chunks) {
    const int64_t share = rows * chunks / (2 * fcai::sm_count());
    return (int)std::max<int64_t>(1, std::min<int64_t>(64, std::max<int64_t>(256, std::min<int64_t>(2048, share)) / chunks));
}
// Makes matrices readable by TMA, from the workspace if they have to be copied.
static int prepare_operands(std::initializer_list<Operand *> all, int dtype, unsigned char *&ws, cudaStream_t stream) {
    Repacks r{};
    int n = 0;
    int64_t steps = 0;
    for (Operand *o : all) {
        if (!o->ptr || aligned16(o->ptr, o->ld, dtype)) continue;
        const int ldd = round8(o->cols), step = rows_a_step(o->rows, ldd / 8);
        r.r[n++] = {static_cast<const uint16_t *>(o->ptr), reinterpret_cast<uint16_t *>(ws), o->ld, o->rows, o->cols, ldd,
                    fast_div(ldd / 8), step};
        steps = std::max(steps, (o->rows + step - 1) / step);
        o->ptr = ws;
        o->ld = ldd;
        ws += repack_bytes(o->rows, o->cols);
    }
    if (!n) return FCAI_OK;
    const int grid = (int)std::min<int64_t>(steps, (int64_t)fcai::sm_count() * 16);
    repack_kernel<<<dim3(grid, n), 256, 0, stream>>>(r);
    FCAI_CUDA_TRY(cudaGetLastError());
    return FCAI_OK;
}
// Outputs of at least this many elements go through padded rows when their own
// are not 16-byte aligned; below, the second launch and pass cost more than the
// narrow stores (4000 x 1027 from 2023: 52 against 48 us; 20000 x 333 from 501: 44
// against 50).
constexpr int64_t kPadFrom = 6 << 20;

template <typename T, int kBN, bool kPair, bool kTA, bool kTB, bool kKeep>
static int launch(const Maps &maps, const Params &p, cudaStream_t stream) {
    using Lay = Layout<kBN, kPair, kKeep>;
    auto kernel = linear_tc_kernel<T, kBN, kPair, kTA, kTB, kKeep>;
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
    cfg.blockDim = dim3(Lay::kThreads, 1, 1);
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
        FCAI_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, maps, p));
    } else {
        kernel<<<n, Lay::kThreads, Lay::kAlloc, stream>>>(maps, p);
    }
    FCAI_CUDA_TRY(cudaGetLastError());
    return FCAI_OK;
}

template <typename T>
static int launch_reduce(const Params &p, cudaStream_t stream) {
    const int64_t sms = fcai::sm_count(), ctas = ((int64_t)p.M + 15) / 16 * p.nblk;  // with one part
    const int parts = p.splits.d < 8 || ctas >= 2 * sms ? 1 : ctas * 4 >= 2 * sms ? 4 : 16;
    const int rows = 16 / parts;
    const int shares = (int)std::min<int64_t>({((int64_t)p.M + rows - 1) / rows, std::max<int64_t>(1, sms * 8 / p.nblk), 65535});
    const dim3 grid(p.nblk, shares);
    if (parts == 1) reduce_kernel<T, 1><<<grid, 256, 0, stream>>>(p);
    else if (parts == 4) reduce_kernel<T, 4><<<grid, 256, 0, stream>>>(p);
    else reduce_kernel<T, 16><<<grid, 256, 0, stream>>>(p);
    FCAI_CUDA_TRY(cudaGetLastError());
    return FCAI_OK;
}

// Whether the epilogue can use wide accesses; the codes are [M][N] bytes.
static bool wide_outputs(const Params &p, int N, int dtype) {
    return N % 8 == 0 && aligned16(p.y, p.ldy, dtype) && (!p.pre || aligned16(p.pre, p.ldpre, dtype)) &&
           (!p.residual || aligned16(p.residual, p.ldr, dtype)) && (!p.bias || aligned16(p.bias, 0, dtype)) &&
           (reinterpret_cast<uintptr_t>(p.codes) & (N % 16 ? 7 : 15)) == 0;
}
// Codes whose rows the tensor map cannot take: small results make them in
// reduce_kernel, from at most 4 * kPadFrom bytes of fp32 values (the workspace is
// asked for by sizes); larger ones send them through rows padded to 16 bytes, as
// they do y.  Other widths' outputs take tiles of codes, which the entry point has
// checked.
static bool codes_padded(int64_t M, int N) { return N % 16 != 0 && M * N >= kPadFrom; }
static bool codes_by_reduce(int64_t M, int N) { return N % 16 != 0 && M * N < kPadFrom; }
static int64_t code_row(int N) { return (N + 15) / 16 * 16; }
static int unpad_grid(const Unpad &o) {
    return (int)std::min<int64_t>((o.rows + o.step - 1) / o.step, (int64_t)fcai::sm_count() * 16);
}
template <typename T, bool kTA, bool kTB>
static int run(Operand A, Operand B, int64_t M, int N, int64_t K, int dtype, Params p, unsigned char *ws,
               cudaStream_t stream) {
    p.error = const_cast<int32_t *>(error_word());
    p.vec = wide_outputs(p, N, dtype);
    const Plan pl = make_plan(M, N, K, p.codes && codes_by_reduce(M, N), p.codes != nullptr);
    p.M = (int)M;
    p.N = N;
    p.tiles_m = pl.tiles_m;
    p.group_m = pl.pair ? 8 : 16;
    p.splits = fast_div(pl.splits);
    p.group = fast_div((uint32_t)p.group_m * pl.tiles_n);
    p.gm = fast_div(p.group_m);
    p.gm_last = fast_div(pl.tiles_m % p.group_m ? pl.tiles_m % p.group_m : p.group_m);
    p.ksteps = pl.ksteps;
    p.ksteps_split = pl.ksteps_split;
    p.units = pl.tiles_m * pl.tiles_n * pl.splits;
    p.ldp = round8(N);
    p.nblk = (N + FCAI_KEEP_BLOCK - 1) / FCAI_KEEP_BLOCK;
    p.coop = !p.codes && p.units <= 2 * (pl.pair ? fcai::sm_count() / 2 : fcai::sm_count());
    p.partial = nullptr;
    if (pl.partial_bytes) {
        p.partial = reinterpret_cast<float *>(ws);
        ws += pl.partial_bytes;
    }
    // unaligned results and residual: through copies with padded rows, or (few elements, or a split product) narrow accesses
    const bool y_aligned = aligned16(p.y, p.ldy, dtype), r_aligned = !p.residual || aligned16(p.residual, p.ldr, dtype);
    const bool pad = !p.partial && M * N >= kPadFrom && (!y_aligned || !r_aligned);
    p.tma = !p.partial && (pad || (y_aligned && r_aligned)) && (!p.pre || aligned16(p.pre, p.ldpre, dtype));
    Operand R{p.tma ? p.residual : nullptr, p.ldr, M, N}, bias{p.tma ? p.bias : nullptr, N, 1, N};
    int rc;
    if ((rc = prepare_operands({&A, &B, &R, &bias}, dtype, ws, stream))) return rc;
    Unpad back{}, codes_back{};
    if (p.tma) {
        p.residual = R.ptr;
        p.ldr = R.ld;
        p.bias = bias.ptr;
        if (!y_aligned) {
            const int chunks = (N + 7) / 8 + 1;
            back = {ws, p.y, round8(N), p.ldy, M, N, fast_div(chunks), rows_a_step(M, chunks)};
            p.y = ws;
            p.ldy = round8(N);
            ws += repack_bytes(M, N);
        }
        if (p.codes && N % 16) {
            const int chunks = (N + 15) / 16 + 1;
            codes_back = {ws, p.codes, code_row(N), N, M, N, fast_div(chunks), rows_a_step(M, chunks)};
            p.codes = ws;
        }
    }
    Maps maps;
    if ((rc = make_map(&maps.a, A.ptr, A.cols, A.rows, A.ld, kTA ? kBK : kBM, dtype))) return rc;
    if ((rc = make_map(&maps.b, B.ptr, B.cols, B.rows, B.ld, kTB ? kBK : pl.pair ? pl.bn / 2 : pl.bn, dtype))) return rc;
    const bool keep = !kTA && !kTB && p.tma && (p.pre || p.codes);
    if (p.tma) {
        if ((rc = make_map(&maps.y, p.y, N, M, p.ldy, 32, dtype, 32))) return rc;
        if (p.residual && (rc = make_map(&maps.res, p.residual, N, M, p.ldr, 32, dtype, 32))) return rc;
        if (p.codes && (rc = make_map(&maps.extra, p.codes, N, M, code_row(N), 32, kCodeType, 32))) return rc;
        if (p.pre && (rc = make_map(&maps.extra, p.pre, N, M, p.ldpre, 32, dtype, 32))) return rc;
    }
#define LN_LAUNCH(keep_)                                                              \
    (pl.pair        ? launch<T, 256, true, kTA, kTB, keep_>(maps, p, stream)          \
     : pl.bn == 128 ? launch<T, 128, false, kTA, kTB, keep_>(maps, p, stream)         \
                    : launch<T, 64, false, kTA, kTB, keep_>(maps, p, stream))
    if constexpr (!kTA && !kTB) rc = keep ? LN_LAUNCH(true) : LN_LAUNCH(false);
    else rc = LN_LAUNCH(false);
#undef LN_LAUNCH
    if (rc) return rc;
    if (back.src) {
        unpad_kernel<uint16_t><<<unpad_grid(back), 256, 0, stream>>>(back);
        FCAI_CUDA_TRY(cudaGetLastError());
    }
    if (codes_back.src) {
        unpad_kernel<uint8_t><<<unpad_grid(codes_back), 256, 0, stream>>>(codes_back);
        FCAI_CUDA_TRY(cudaGetLastError());
    }
    return p.partial ? launch_reduce<T>(p, stream) : FCAI_OK;
}

// Up to this many rows the forward product runs without tiles.
constexpr int kFewRows = 32;
template <typename T, int kNB, bool kV>
static int launch_few(const FewRows &f, const Params &p, cudaStream_t stream) {
    // long rows: more warps share a group's K, so that about all of w is in flight at once
    const int grid = (p.N + 15) / 16;
    if (f.K < 2048) few_rows_kernel<T, kNB, 8, kV><<<grid, 256, 0, stream>>>(f, p);
    else few_rows_kernel<T, kNB, 16, kV><<<grid, 512, 0, stream>>>(f, p);
    FCAI_CUDA_TRY(cudaGetLastError());
    return FCAI_OK;
}
template <typename T, int kNB>
static int launch_few(const FewRows &f, const Params &p, bool vec, cudaStream_t stream) {
    return vec ? launch_few<T, kNB, true>(f, p, stream) : launch_few<T, kNB, false>(f, p, stream);
}
template <typename T>
static int run_few(const FewRows &f, int rows, int N, int dtype, Params p, void *ws, cudaStream_t stream) {
    p.M = rows;
    p.N = N;
    p.ldp = round8(N);
    p.nblk = (N + FCAI_KEEP_BLOCK - 1) / FCAI_KEEP_BLOCK;
    p.splits = fast_div(1);
    p.vec = wide_outputs(p, N, dtype);
    p.partial = p.codes ? static_cast<float *>(ws) : nullptr;
    const bool vec = f.K % 8 == 0 && aligned16(f.x, f.ldx, dtype) && aligned16(f.w, f.ldw, dtype);
    const int rc = rows <= 8    ? launch_few<T, 1>(f, p, vec, stream)
                   : rows <= 16 ? launch_few<T, 2>(f, p, vec, stream)
                                : launch_few<T, 4>(f, p, vec, stream);
    return rc || !p.partial ? rc : launch_reduce<T>(p, stream);
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

static int64_t workspace_bytes(int op, int64_t rows, int cin, int cout, int repack, int keep) {
    if (rows < 0 || rows > 0x7FFFFFFF - 256 || cin < 1 || cout < 1 || cin > (1 << 24) || cout > (1 << 24)) return -1;
    if (op < FCAI_LINEAR_FORWARD || op > FCAI_LINEAR_BACKWARD_WEIGHT) return -1;
    if (rows == 0) return 0;
    const bool forward = op == FCAI_LINEAR_FORWARD, weight = op == FCAI_LINEAR_BACKWARD_WEIGHT;
    const bool k8 = forward && keep >= FCAI_KEEP_INT8;
    if (forward && rows <= kFewRows) return k8 ? round256(rows * round8(cout) * 4) : 0;
    // the product's sizes, and its operands'
    const int64_t M = weight ? cout : rows, K = weight ? rows : forward ? cin : cout, a_rows = rows, b_rows = weight ? rows : cout;
    const int N = forward ? cout : cin, a_cols = forward ? cin : cout, b_cols = cin;
    const int64_t partial = make_plan(M, N, K, k8 && codes_by_reduce(M, N), k8).partial_bytes;
    int64_t n = partial;
    if (repack & 1) n += repack_bytes(a_rows, a_cols);
    if (repack & 2) n += repack_bytes(b_rows, b_cols);
    if (!partial && (repack & 16)) n += repack_bytes(1, N);
    if (!partial && M * N >= kPadFrom) {
        if (repack & 4) n += repack_bytes(M, N);
        if (repack & 8) n += repack_bytes(M, N);
    }
    if (!partial && k8 && codes_padded(M, N)) n += round256(M * code_row(N));
    return n;
}
// The last check before a launch.
static int check_workspace(int op, int64_t rows, int cin, int cout, const void *a, int64_t lda, const void *b, int64_t ldb,
                           const void *y, int64_t ldy, const void *residual, int64_t ldr, const void *bias, int dtype, int keep,
                           const void *ws, int64_t bytes) {
    const int repack = (aligned16(a, lda, dtype) ? 0 : 1) | (aligned16(b, ldb, dtype) ? 0 : 2) | (aligned16(y, ldy, dtype) ? 0 : 4) |
                       (!residual || aligned16(residual, ldr, dtype) ? 0 : 8) | (!bias || aligned16(bias, cout, dtype) ? 0 : 16);
    const int64_t need = workspace_bytes(op, rows, cin, cout, repack, keep);
    if (need > 0 && (!ws || bytes < need || (reinterpret_cast<uintptr_t>(ws) & 255)))
        return fcai::fail(FCAI_ERR_WORKSPACE, "linear: needs a 256-byte aligned workspace of %lld bytes", (long long)need);
    return check_errors();
}

}  // namespace ln

extern "C" {

int32_t *fcai_linear_error_word(void) { return const_cast<int32_t *>(ln::error_word()); }

int64_t fcai_linear_workspace(int32_t op, int64_t rows, int32_t cin, int32_t cout, int32_t repack, int32_t keep) {
    return ln::workspace_bytes(op, rows, cin, cout, repack, keep);
}

int fcai_linear_forward(const void *x, int64_t ldx, const void *w, int64_t ldw, const void *bias,
                        const void *residual, int64_t ldr, void *y, int64_t ldy, void *pre, int64_t ldpre,
                        void *codes, float *scales, int64_t rows, int32_t cin, int32_t cout, int32_t dtype, int32_t act,
                        int32_t keep, void *workspace, int64_t workspace_bytes, fcai_stream_t stream) {
    using namespace ln;
    fcai::clear_error();
    int rc = check_common(rows, cin, cout, dtype, x, ldx, cin, w, ldw, cin, y, ldy, cout);
    if (rc) return rc;
    if (act < FCAI_ACT_NONE || act > FCAI_ACT_SILU) return fcai::fail(FCAI_ERR_INVALID, "linear: unknown activation %d", act);
    if (keep < FCAI_KEEP_NONE || keep > FCAI_KEEP_E4M3) return fcai::fail(FCAI_ERR_INVALID, "linear: unknown keep %d", keep);
    const bool k8 = keep >= FCAI_KEEP_INT8;
    if ((rows && k8 && (!codes || !scales)) || (keep == FCAI_KEEP_FULL && rows && !pre) || (reinterpret_cast<uintptr_t>(scales) & 3))
        return fcai::fail(FCAI_ERR_INVALID, "linear: the keep needs its output");
    if ((residual && (ldr < cout || ldr > (1ll << 36))) || (keep == FCAI_KEEP_FULL && (ldpre < cout || ldpre > (1ll << 36))))
        return fcai::fail(FCAI_ERR_INVALID, "linear: a row stride is smaller than its row or too large");
    if (((reinterpret_cast<uintptr_t>(bias) | reinterpret_cast<uintptr_t>(residual) | reinterpret_cast<uintptr_t>(pre)) & 1) != 0)
        return fcai::fail(FCAI_ERR_INVALID, "linear: misaligned pointer");
    if (rows == 0) return FCAI_OK;
    if (!x || !w || !y) return fcai::fail(FCAI_ERR_INVALID, "linear: null pointer");
    Params p{};
    p.act = act;
    p.bias = bias;
    p.residual = residual;
    p.ldr = ldr;
    p.y = y;
    p.ldy = ldy;
    p.pre = keep == FCAI_KEEP_FULL ? pre : nullptr;
    p.ldpre = ldpre;
    p.codes = k8 ? static_cast<uint8_t *>(codes) : nullptr;
    p.scales = scales;
    p.keep = keep;
    if (k8 && rows > kFewRows && cout % 8 == 0 && !wide_outputs(p, cout, dtype))
        return fcai::fail(FCAI_ERR_INVALID, "linear: codes need 16-byte aligned y, bias and residual rows, and 16-byte aligned codes");
    if ((rc = check_workspace(FCAI_LINEAR_FORWARD, rows, cin, cout, x, ldx, w, ldw, y, ldy, residual, ldr, bias, dtype, keep,
                              workspace, workspace_bytes)))
        return rc;
    const Operand A{x, ldx, rows, cin}, B{w, ldw, cout, cin};
    auto *ws = static_cast<unsigned char *>(workspace);
    auto st = static_cast<cudaStream_t>(stream);
    if (rows <= kFewRows) {
        const FewRows f{x, w, ldx, ldw, cin};
        return dtype == FCAI_DTYPE_BF16 ? run_few<__nv_bfloat16>(f, (int)rows, cout, dtype, p, ws, st)
                                        : run_few<__half>(f, (int)rows, cout, dtype, p, ws, st);
    }
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
    if ((rc = check_workspace(FCAI_LINEAR_BACKWARD_INPUT, rows, cin, cout, dp, lddp, w, ldw, dx, lddx, nullptr, 0, nullptr, dtype, 0,
                              workspace, workspace_bytes)))
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
        empty_product_kernel<<<elementwise_grid((int64_t)cout * cin, 256), 256, 0, st>>>(p);
        FCAI_CUDA_TRY(cudaGetLastError());
        return FCAI_OK;
    }
    if ((rc = check_workspace(FCAI_LINEAR_BACKWARD_WEIGHT, rows, cin, cout, dp, lddp, x, ldx, dw, lddw, nullptr, 0, nullptr, dtype, 0,
                              workspace, workspace_bytes)))
        return rc;
    const Operand A{dp, lddp, rows, cout}, B{x, ldx, rows, cin};
    auto *ws = static_cast<unsigned char *>(workspace);
    return dtype == FCAI_DTYPE_BF16 ? run<__nv_bfloat16, true, true>(A, B, cout, cin, rows, dtype, p, ws, st)
                                    : run<__half, true, true>(A, B, cout, cin, rows, dtype, p, ws, st);
}

}  // extern "C"
