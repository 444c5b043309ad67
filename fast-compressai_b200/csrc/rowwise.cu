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
//
// The strips read through a ring of shared memory that cp.async fills, every thread
// its own 16 bytes a row, several rows ahead of the one it works on: what is in
// flight costs no registers, needs no barrier, and never drains while a row is
// worked on (with the next rows in registers instead, too few bytes were in
// flight: 3.3 to 4.7 TB/s).  Rows that do not take 16-byte accesses go by single
// elements, with the next row in registers or with more warps.  The layer norm
// keeps its next rows in registers (a ring for it was slower, 89 us against 62 at
// 16384 x 4096).
#include <cuda_runtime.h>

#include <algorithm>
#include <type_traits>

#include "layers_common.cuh"

namespace rw {

using namespace ly;

constexpr int kThreads = 256;
constexpr int kBlock = FCAI_KEEP_BLOCK;
// Lanes a row of a strip: 16 cover a block of 128 channels; rows of up to 32
// channels take 4, or most lanes would idle.
constexpr int strip_lanes(int n) { return n <= 32 ? 4 : 16; }
constexpr int kRowsIter = kThreads / 16;  // rows a strip CTA handles at a time (with 16 lanes)

// The eight channels a thread holds of its group's 8 * g: consecutive ones where
// rows take 16-byte accesses (kV), else every g-th, so that neighbouring lanes
// still touch neighbouring elements.
template <bool kV>
struct Cols {
    int first, step;
    __device__ __forceinline__ Cols(int base, int l, int g) : first(kV ? base + l * 8 : base + l), step(kV ? 1 : g) {}
    __device__ __forceinline__ int operator[](int i) const { return first + i * step; }
};
template <typename T, bool kV>
__device__ __forceinline__ void load8(const T *row, const Cols<kV> &c, int n, bool in, float (&v)[8]) {
    if (kV) {
        if (in && c.first < n) Vec8<T>::load(row + c.first, v);
        else
            for (int i = 0; i < 8; ++i) v[i] = 0.f;
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = in && c[i] < n ? to_f32(row[c[i]]) : 0.f;
    }
}
template <typename T, bool kV>
__device__ __forceinline__ void store8(T *row, const Cols<kV> &c, int n, bool in, const float (&v)[8]) {
    if (kV) {
        if (in && c.first < n) Vec8<T>::store(row + c.first, v);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (in && c[i] < n) row[c[i]] = from_f32<T>(v[i]);
    }
}
template <typename T, bool kV>
__device__ __forceinline__ void store8(T *row, const Cols<kV> &c, int n, bool in, const V8 &v) {
    float f[8];
    v.get(f);
    store8(row, c, n, in, f);
}
template <bool kV>
__device__ __forceinline__ uint2 load_codes(const uint8_t *row, const Cols<kV> &c, int n, bool in) {
    uint2 q = make_uint2(0u, 0u);
    if (kV) {
        if (in && c.first < n) q = __ldg(reinterpret_cast<const uint2 *>(row + c.first));
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (in && c[i] < n) (i < 4 ? q.x : q.y) |= (uint32_t)__ldg(row + c[i]) << (8 * (i & 3));
    }
    return q;
}
template <bool kV>
__device__ __forceinline__ void store_codes(uint8_t *row, const Cols<kV> &c, int n, bool in, uint2 q) {
    if (kV) {
        if (in && c.first < n) *reinterpret_cast<uint2 *>(row + c.first) = q;
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (in && c[i] < n) row[c[i]] = (uint8_t)((i < 4 ? q.x : q.y) >> (8 * (i & 3)));
    }
}

template <typename T> struct Pair;
template <> struct Pair<__half> { using type = __half2; };
template <> struct Pair<__nv_bfloat16> { using type = __nv_bfloat162; };
// Eight elements as they lie in memory, 4 or 8 registers: what is in flight or waits for a sum.
template <typename T, bool kV>
struct Raw8 {
    uint32_t w[sizeof(T) * 2];
    __device__ __forceinline__ void load(const T *row, const Cols<kV> &c, int n, bool in) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) * 2; ++i) w[i] = 0u;
        if constexpr (kV) {
            if (in && c.first < n) {
#pragma unroll
                for (int i = 0; i < (int)sizeof(T) / 2; ++i) {
                    const uint4 q = __ldg(reinterpret_cast<const uint4 *>(row + c.first) + i);
                    w[4 * i] = q.x, w[4 * i + 1] = q.y, w[4 * i + 2] = q.z, w[4 * i + 3] = q.w;
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                if (!in || c[i] >= n) continue;
                if constexpr (sizeof(T) == 4) w[i] = __float_as_uint(__ldg(row + c[i]));
                else w[i / 2] |= (uint32_t)__ldg(reinterpret_cast<const unsigned short *>(row) + c[i]) << (16 * (i & 1));
            }
        }
    }
    __device__ __forceinline__ V8 get() const {
        V8 v;
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < 4; ++i) v.p[i] = f2(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]));
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float2 f = unpack2(w[i], T());
                v.p[i] = f2(f.x, f.y);
            }
        }
        return v;
    }
    // largest magnitude; NaN if there is one
    __device__ __forceinline__ float amax() const {
        if constexpr (sizeof(T) == 4) {
            float m = fabsf(__uint_as_float(w[0]));
#pragma unroll
            for (int i = 1; i < 8; ++i) m = max_nan(m, fabsf(__uint_as_float(w[i])));
            return m;
        } else {
            using T2 = typename Pair<T>::type;
            T2 m = __habs2(*reinterpret_cast<const T2 *>(&w[0]));
#pragma unroll
            for (int i = 1; i < 4; ++i) m = __hmax2_nan(m, __habs2(*reinterpret_cast<const T2 *>(&w[i])));
            const float2 f = unpack2(*reinterpret_cast<uint32_t *>(&m), T());
            return max_nan(f.x, f.y);
        }
    }
};

// What a backward pass reads x from.
struct Kept {
    const void *x;
    int64_t ldx;
    const uint8_t *codes;
    const float *scales;
    int keep;
};
__device__ __forceinline__ V8 decode8(int keep, uint2 q, float s) {
    V8 v;
    if (keep == FCAI_KEEP_E4M3) {
        decode4<true>(q.x, s, v.p[0], v.p[1]);
        decode4<true>(q.y, s, v.p[2], v.p[3]);
    } else {
        decode4<false>(q.x, s, v.p[0], v.p[1]);
        decode4<false>(q.y, s, v.p[2], v.p[3]);
    }
    return v;
}
// A kept value's bits as they are loaded, before they are decoded: loads of several rows go out together.
template <typename T, bool kV, bool k8>
struct KeptRaw {
    Raw8<T, kV> x;
    uint2 q;
    float s;
    __device__ __forceinline__ void load(const Kept &k, int64_t row, const Cols<kV> &c, int n, int nblk, bool in) {
        if constexpr (k8) {
            q = load_codes(k.codes + row * n, c, n, in);
            s = in && c.first < n ? __ldg(k.scales + row * nblk + c.first / kBlock) : 0.f;
        } else {
            x.load(static_cast<const T *>(k.x) + row * k.ldx, c, n, in);
        }
    }
    __device__ __forceinline__ V8 get(const Kept &k) const {
        if constexpr (k8) return decode8(k.keep, q, s);
        else return x.get();
    }
};

// ---- rows in flight ----------------------------------------------------------
template <int kBytes>
__device__ __forceinline__ void cp_async(uint32_t dst, const void *src, bool in) {
    const uint64_t g = __cvta_generic_to_global(src);
    if constexpr (kBytes == 16)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(g), "r"(in ? 16 : 0) : "memory");
    else
        asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(g), "n"(kBytes), "r"(in ? kBytes : 0) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int kPending>
__device__ __forceinline__ void cp_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(kPending) : "memory");
}
constexpr int kRingBytes = 32768;  // a CTA's ring at most

// kCta threads, kPer chunks of 8 values a thread and step; kAsync: through the
// ring at `base`, else the next step waits in registers.
template <typename T, bool kV, bool kAsync, int kCta, int kPer>
struct RowFeed {
    static constexpr int kPieces = sizeof(T) / 2;
    static constexpr int kStep = kPer * kPieces * kCta * 16;  // ring bytes a step
    Raw8<T, kV> reg[kAsync ? 1 : kPer];
    __device__ __forceinline__ void issue(uint32_t base, int i, const T *m, int64_t offset, const Cols<kV> &c, int n, bool in) {
        if constexpr (kAsync) {
            const bool ok = in && c.first < n;
            const T *src = ok ? m + offset + c.first : m;
#pragma unroll
            for (int q = 0; q < kPieces; ++q)
                cp_async<16>(base + ((i * kPieces + q) * kCta + threadIdx.x) * 16, src + (ok ? q * (16 / (int)sizeof(T)) : 0), ok);
        } else {
            reg[i].load(m + offset, c, n, in);
        }
    }
    __device__ __forceinline__ Raw8<T, kV> get(uint32_t base, int i) const {
        if constexpr (kAsync) {
            Raw8<T, kV> r;
#pragma unroll
            for (int q = 0; q < kPieces; ++q)
                asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                             : "=r"(r.w[4 * q]), "=r"(r.w[4 * q + 1]), "=r"(r.w[4 * q + 2]), "=r"(r.w[4 * q + 3])
                             : "r"(base + ((i * kPieces + q) * kCta + threadIdx.x) * 16)
                             : "memory");
            return r;
        } else {
            return reg[i];
        }
    }
};
template <typename T, bool kV, bool k8, bool kAsync, int kCta, int kPer>
struct KeptFeed {
    using Values = RowFeed<T, kV, kAsync, kCta, kPer>;
    static constexpr int kStep = k8 ? kPer * kCta * 12 : Values::kStep;
    Values x;
    KeptRaw<T, kV, true> reg[kAsync || !k8 ? 1 : kPer];
    __device__ __forceinline__ void issue(uint32_t base, int i, const Kept &k, int64_t row, const Cols<kV> &c, int n, int nblk, bool in) {
        if constexpr (!k8) {
            x.issue(base, i, static_cast<const T *>(k.x), row * k.ldx, c, n, in);
        } else if constexpr (kAsync) {
            const bool ok = in && c.first < n;
            cp_async<8>(base + (i * kCta + threadIdx.x) * 8, ok ? k.codes + row * n + c.first : k.codes, ok);
            cp_async<4>(base + kPer * kCta * 8 + (i * kCta + threadIdx.x) * 4, ok ? k.scales + row * nblk + c.first / kBlock : k.scales, ok);
        } else {
            reg[i].load(k, row, c, n, nblk, in);
        }
    }
    __device__ __forceinline__ KeptRaw<T, kV, k8> get(uint32_t base, int i) const {
        KeptRaw<T, kV, k8> r;
        if constexpr (!k8) {
            r.x = x.get(base, i);
        } else if constexpr (kAsync) {
            asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(r.q.x), "=r"(r.q.y) : "r"(base + (i * kCta + threadIdx.x) * 8) : "memory");
            asm volatile("ld.shared.f32 %0, [%1];" : "=f"(r.s) : "r"(base + kPer * kCta * 8 + (i * kCta + threadIdx.x) * 4) : "memory");
        } else {
            r = reg[i];
        }
        return r;
    }
};
// Steps in flight: as many as the ring holds, at most four.
constexpr int ring_depth(int step_bytes) { return step_bytes * 4 <= kRingBytes ? 4 : step_bytes * 2 <= kRingBytes ? kRingBytes / step_bytes : 1; }

// A block's codes and scale, from the kLanes (at most 16) lanes that hold its
// channels, 8 each (amax: the lane's own); the whole warp calls it.
template <int kLanes, bool kV>
__device__ __forceinline__ void keep_block(int keep, float amax, const V8 &v, uint8_t *codes_row, float *scale, const Cols<kV> &c,
                                           int n, bool in) {
#pragma unroll
    for (int d = (kLanes < 16 ? kLanes : 16) / 2; d >= 1; d >>= 1) amax = max_nan(amax, __shfl_xor_sync(0xffffffffu, amax, d));
    uint2 q;
    float s;
    if (keep == FCAI_KEEP_E4M3) {
        s = block_scale<true>(amax);
        q = encode8<true>(v, __frcp_rn(s));
    } else {
        s = block_scale<false>(amax);
        q = encode8<false>(v, __frcp_rn(s));
    }
    store_codes(codes_row, c, n, in, q);
    if (in && c.first % kBlock == 0 && c.first < n) *scale = s;
}

// ---- strips: activations, checkpoint load ------------------------------------
// grid (strips, row shares): the CTAs that run at the same time cover whole rows, which DRAM pages like.
template <typename T, bool kV, int kLanes>
__global__ void __launch_bounds__(kThreads, kV ? 5 : 4)
    act_forward_kernel(const T *__restrict__ x, int64_t ldx, T *__restrict__ y, int64_t ldy, uint8_t *__restrict__ codes,
                       float *__restrict__ scales, int64_t rows, int n, int nblk, int act, int keep) {
    using Feed = RowFeed<T, kV, kV, kThreads, 1>;
    constexpr int kD = kV ? ring_depth(Feed::kStep) : 1;
    __shared__ __align__(16) unsigned char ring[kV ? kD * Feed::kStep : 16];
    const uint32_t base = (uint32_t)__cvta_generic_to_shared(ring);
    const int strip = blockIdx.x;
    const Cols<kV> c(strip * kBlock, threadIdx.x % kLanes, kLanes);
    const int64_t step = (int64_t)gridDim.y * (kThreads / kLanes);
    const int sub = (threadIdx.x & 31) / kLanes;
    // the loop runs on the warp's first row: a block's shuffles need the whole warp
    int64_t r0 = (int64_t)blockIdx.y * (kThreads / kLanes) + (threadIdx.x >> 5) * (32 / kLanes);
    Feed feed;
#pragma unroll
    for (int d = 0; d < kD; ++d) {
        feed.issue(base + d * Feed::kStep, 0, x, (r0 + d * step + sub) * ldx, c, n, r0 + d * step + sub < rows);
        cp_commit();
    }
    for (int slot = 0; r0 < rows; r0 += step, slot = slot + 1 == kD ? 0 : slot + 1) {
        cp_wait<kD - 1>();
        const Raw8<T, kV> raw = feed.get(base + slot * Feed::kStep, 0);
        V8 v = raw.get();
        const int64_t row = r0 + sub;
        const bool in = row < rows;
        if (keep != FCAI_KEEP_NONE) keep_block<kLanes>(keep, raw.amax(), v, codes + row * n, scales + row * nblk + strip, c, n, in);
        feed.issue(base + slot * Feed::kStep, 0, x, (row + kD * step) * ldx, c, n, row + kD * step < rows);
        cp_commit();
        if (y) {
            act_n(act, v.p);
            store8(y + row * ldy, c, n, in, v);
        }
    }
    cp_wait<0>();
}

// Rows a thread has in flight: 8 + 4 bytes a row are too little for the ring to
// pay.  By single elements one row and more warps (31 us -> 27 at 30000 x 1021).
template <typename T, bool kV, int kLanes>
__global__ void __launch_bounds__(kThreads, 6)
    checkpoint_load_kernel(Kept k, T *__restrict__ out, int64_t ldo, int64_t rows, int n, int nblk) {
    constexpr int kLoadRows = kV ? 2 : 1;
    const Cols<kV> c(blockIdx.x * kBlock, threadIdx.x % kLanes, kLanes);
    const int64_t step = (int64_t)gridDim.y * (kThreads / kLanes);
    for (int64_t r0 = (int64_t)blockIdx.y * (kThreads / kLanes) + threadIdx.x / kLanes; r0 < rows; r0 += step * kLoadRows) {
        KeptRaw<T, kV, true> raw[kLoadRows];
#pragma unroll
        for (int u = 0; u < kLoadRows; ++u) raw[u].load(k, r0 + u * step, c, n, nblk, r0 + u * step < rows);
#pragma unroll
        for (int u = 0; u < kLoadRows; ++u) {
            if (r0 + u * step >= rows) break;
            store8(out + (r0 + u * step) * ldo, c, n, true, raw[u].get(k));
        }
    }
}

// Adds the sums of a CTA's groups of kLanes threads (8 * kLanes channels from
// base on) and writes them to a partial row.
template <int kLanes, int kCta, bool kV>
__device__ __forceinline__ void group_sums(const V8 &sums, float *partial_row, int base, int n, float *sh) {
    constexpr int kSpan = kLanes * 8;
    const int g = threadIdx.x / kLanes, l = threadIdx.x % kLanes;
    const Cols<kV> c(0, l % 16 + (kV ? l / 16 * 16 : 0), kLanes < 16 ? kLanes : 16);
    const int blk = kV ? 0 : l / 16 * kBlock;
    float acc[8];
    sums.get(acc);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; ++i) sh[g * kSpan + blk + c[i]] = acc[i];
    __syncthreads();
    for (int j = threadIdx.x; j < kSpan; j += kCta) {
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < kCta / kLanes; ++i) s += sh[i * kSpan + j];
        if (base + j < n) partial_row[base + j] = s;
    }
}

// Rows that take single elements only: with the next row in registers, packing it
// waits for its loads in the middle of this one's work, and 24 warps an SM do not
// hide that (30000 x 1021 bf16 from int8: 127 us); 48 warps without a row ahead do
// (59).  f32 from f32, with nothing to pack, stays ahead (64 us, 77 without).
template <typename T, bool k8>
constexpr bool act_ahead() {
    return sizeof(T) == 4 && !k8;
}
// dx = dy act'(x) and partial sums of it over the CTA's rows; kAct: x is read
template <typename T, bool kV, bool k8, bool kAct, int kLanes>
__global__ void __launch_bounds__(kThreads, !kV ? (act_ahead<T, k8>() ? 3 : 6) : sizeof(T) == 4 ? 3 : 4)
    act_backward_kernel(const T *__restrict__ dy, int64_t lddy, Kept k, T *__restrict__ dx, int64_t lddx,
                        float *__restrict__ partial, int64_t rows, int n, int nblk, int act) {
    using FeedG = RowFeed<T, kV, kV, kThreads, 1>;
    using FeedX = KeptFeed<T, kV, k8, kV, kThreads, 1>;
    constexpr int kStep = FeedG::kStep + (kAct ? FeedX::kStep : 0);
    constexpr int kD = kV ? ring_depth(kStep) : 1;
    constexpr int kSums = kThreads * 8 * 4;
    // the sums meet in the ring's memory when the rows are through
    __shared__ __align__(16) unsigned char ring[kV && kD * kStep > kSums ? kD * kStep : kSums];
    const uint32_t base = (uint32_t)__cvta_generic_to_shared(ring);
    const Cols<kV> c(blockIdx.x * kBlock, threadIdx.x % kLanes, kLanes);
    const int64_t step = (int64_t)gridDim.y * (kThreads / kLanes);
    V8 acc = {f2(0.f), f2(0.f), f2(0.f), f2(0.f)};
    int64_t row = (int64_t)blockIdx.y * (kThreads / kLanes) + threadIdx.x / kLanes;
    FeedG feed_g;
    FeedX feed_x;
    auto issue = [&](int slot, int64_t r) {
        feed_g.issue(base + slot * kStep, 0, dy, r * lddy, c, n, r < rows);
        if (kAct) feed_x.issue(base + slot * kStep + FeedG::kStep, 0, k, r, c, n, nblk, r < rows);
        cp_commit();
    };
    auto finish = [&](V8 g, V8 x) {
        if (kAct) act_grad_n(act, x.p, g.p);
        if (dx) store8(dx + row * lddx, c, n, true, g);
#pragma unroll
        for (int i = 0; i < 4; ++i) acc.p[i] = add2(acc.p[i], g.p[i]);
    };
    if constexpr (kV || act_ahead<T, k8>()) {
#pragma unroll
        for (int d = 0; d < kD; ++d) issue(d, row + d * step);
        for (int slot = 0; row < rows; row += step, slot = slot + 1 == kD ? 0 : slot + 1) {
            cp_wait<kD - 1>();
            V8 g = feed_g.get(base + slot * kStep, 0).get(), x;
            if (kAct) x = feed_x.get(base + slot * kStep + FeedG::kStep, 0).get(k);
            issue(slot, row + kD * step);
            finish(g, x);
        }
        cp_wait<0>();
    } else {
        for (; row < rows; row += step) {
            Raw8<T, kV> raw_g;
            KeptRaw<T, kV, k8> raw_x;
            raw_g.load(dy + row * lddy, c, n, true);
            V8 x;
            if (kAct) {
                raw_x.load(k, row, c, n, nblk, true);
                x = raw_x.get(k);
            }
            finish(raw_g.get(), x);
        }
    }
    if (partial) {
        group_sums<kLanes, kThreads, kV>(acc, partial + (int64_t)blockIdx.y * n, blockIdx.x * kBlock, n, reinterpret_cast<float *>(ring));
    }
}

// Column sums of partial[rows][stride], in a fixed order: columns [0, n0) to
// out0, [n0, n0 + n1) to out1.  32 columns a CTA, 32 threads down the rows.
template <typename T>
__global__ void __launch_bounds__(1024)
    colsum_kernel(const float *__restrict__ partial, int rows, int64_t stride, T *__restrict__ out0, int n0, T *__restrict__ out1,
                  int n1) {
    __shared__ float sh[32][33];
    const int col = blockIdx.x * 32 + threadIdx.x;
    float s = 0.f;
    if (col < n0 + n1) {
#pragma unroll 8
        for (int r = threadIdx.y; r < rows; r += 32) s += partial[r * stride + col];
    }
    sh[threadIdx.y][threadIdx.x] = s;
    __syncthreads();
    if (threadIdx.y == 0 && col < n0 + n1) {
        s = 0.f;
#pragma unroll
        for (int i = 0; i < 32; ++i) s += sh[i][threadIdx.x];
        if (col < n0) {
            if (out0) out0[col] = from_f32<T>(s);
        } else if (out1) {
            out1[col - n0] = from_f32<T>(s);
        }
    }
}

// ---- layer norm ----------------------------------------------------------------
// A group of kLanes threads holds a row in registers, kChunks x 8 channels a
// thread, and reads it from memory once.  Up to 32 lanes the group is part of a
// warp and sums with shuffles; above, it is the whole CTA and one exchange
// through shared memory follows (two buffers in turn, so that a sum needs one
// barrier).
template <int kLanes>
struct Group {
    static constexpr int kCta = kLanes <= 32 ? kThreads : kLanes;
    static constexpr int kGroups = kCta / kLanes;
    static constexpr int kWarpsRow = kLanes <= 32 ? 1 : kLanes / 32;
};
// CTAs an SM is to hold of the norm kernels, which also sets their grids: whole
// CTAs a row with two chunks a thread get 128 registers (the forward kernel of
// 16-bit rows makes do with 84).
constexpr int norm_ctas(int lanes, int chunks, bool f32, int warp_groups, bool lean = false) {
    if (lanes <= 32) return f32 && chunks == 2 ? 1 : f32 ? 2 : warp_groups;
    const int threads = f32 ? 512 : chunks == 1 ? 1024 : lean ? 768 : 512;
    return threads > lanes ? threads / lanes : 1;
}
// Sums of kN values over the group, exchanged together.
template <int kLanes, int kN>
__device__ __forceinline__ void group_sum(float (&v)[kN], float (*sh)[16][kN], int &turn) {
#pragma unroll
    for (int d = (kLanes < 32 ? kLanes : 32) / 2; d >= 1; d >>= 1)
#pragma unroll
        for (int i = 0; i < kN; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], d);
    if constexpr (kLanes > 32) {
        if ((threadIdx.x & 31) == 0) {
#pragma unroll
            for (int i = 0; i < kN; ++i) sh[turn][threadIdx.x >> 5][i] = v[i];
        }
        __syncthreads();
        // every warp adds the warps' sums, a lane each
#pragma unroll
        for (int i = 0; i < kN; ++i) v[i] = sh[turn][threadIdx.x & (kLanes / 32 - 1)][i];
#pragma unroll
        for (int d = kLanes / 64; d >= 1; d >>= 1)
#pragma unroll
            for (int i = 0; i < kN; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], d);
        turn ^= 1;
    }
}
template <int kLanes, bool kV>
__device__ __forceinline__ Cols<kV> chunk_cols(int chunk) {
    const int l = threadIdx.x % kLanes;
    if (kLanes <= 16) return Cols<kV>(0, l, kLanes);
    return Cols<kV>(chunk * kLanes * 8 + l / 16 * kBlock, l % 16, 16);
}

struct Affine {
    const void *w, *b;
    int f32, vec;
};
template <typename T, bool kV>
__device__ __forceinline__ V8 load_affine(const Affine &a, const void *p, const Cols<kV> &c, int n, float dflt) {
    float v[8];
    if (!p) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = dflt;
    } else if (kV && a.vec) {
        if (a.f32) load8(static_cast<const float *>(p), c, n, true, v);
        else load8(static_cast<const T *>(p), c, n, true, v);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            v[i] = c[i] >= n ? 0.f : a.f32 ? static_cast<const float *>(p)[c[i]] : to_f32(static_cast<const T *>(p)[c[i]]);
    }
    V8 o;
    o.set(v);
    return o;
}

// kRows rows a group and step, their sums exchanged together; the next step's
// rows are fetched before this one's are summed.  16 channels a thread of a
// whole-CTA group: with 8, a row's sums (shuffles, which share the data path of
// shared memory, and the exchange) took half of all instructions.
template <typename T, bool kV, bool k8, int kLanes, int kChunks, int kRows>
__global__ void __launch_bounds__(Group<kLanes>::kCta, norm_ctas(kLanes, kChunks, sizeof(T) == 4, k8 || kChunks == 2 ? 2 : 3, !k8 && kV))
    norm_forward_kernel(const T *__restrict__ x, int64_t ldx, Affine af, T *__restrict__ y, int64_t ldy,
                        float *__restrict__ mean_out, float *__restrict__ rstd_out, uint8_t *__restrict__ codes,
                        float *__restrict__ scales, int64_t rows, int n, int nblk, float eps, int keep) {
    using G = Group<kLanes>;
    __shared__ float sh[2][16][kRows];
    int turn = 0;
    const float inv_n = 1.f / n;
    const int64_t step = (int64_t)gridDim.x * G::kGroups * kRows;
    const int sub = threadIdx.x / kLanes;
    // the loop runs on the CTA's first row: shuffles and barriers need everyone
    int64_t r0 = (int64_t)blockIdx.x * G::kGroups * kRows;
    Raw8<T, kV> next[kRows][kChunks];
    auto fetch = [&](int64_t first) {
#pragma unroll
        for (int u = 0; u < kRows; ++u) {
            const int64_t row = first + u * G::kGroups + sub;
#pragma unroll
            for (int j = 0; j < kChunks; ++j) next[u][j].load(x + row * ldx, chunk_cols<kLanes, kV>(j), n, row < rows);
        }
    };
    fetch(r0);
    V8 w[kChunks], b[kChunks];
#pragma unroll
    for (int j = 0; j < kChunks; ++j) {
        w[j] = load_affine<T>(af, af.w, chunk_cols<kLanes, kV>(j), n, 1.f);
        b[j] = load_affine<T>(af, af.b, chunk_cols<kLanes, kV>(j), n, 0.f);
    }
    for (; r0 < rows; r0 += step) {
        Raw8<T, kV> raw[kRows][kChunks];
#pragma unroll
        for (int u = 0; u < kRows; ++u)
#pragma unroll
            for (int j = 0; j < kChunks; ++j) raw[u][j] = next[u][j];
        if (r0 + step < rows) fetch(r0 + step);
        float mean[kRows], rstd[kRows];
#pragma unroll
        for (int u = 0; u < kRows; ++u) {
            F2 s = f2(0.f);
#pragma unroll
            for (int j = 0; j < kChunks; ++j) {
                const V8 v = raw[u][j].get();
                s = add2(s, add2(add2(v.p[0], v.p[1]), add2(v.p[2], v.p[3])));
            }
            mean[u] = hsum(s);
        }
        group_sum<kLanes>(mean, sh, turn);
#pragma unroll
        for (int u = 0; u < kRows; ++u) {
            // sum / n as the product with 1 / n and one step of iterative refinement (the remainder sum - m n is exact):
            // equal 16-bit values, whose sum is exact, have themselves as mean, and their row comes out as the bias
            // (448 x 29952 gave 0.53 instead of 0 without it; a division takes 10.2 us at 36864 x 192, this 9.2)
            const float m = mean[u] * inv_n;
            mean[u] = fmaf(fmaf(-m, (float)n, mean[u]), inv_n, m);
            F2 s = f2(0.f);
#pragma unroll
            for (int j = 0; j < kChunks; ++j) {
                const Cols<kV> c = chunk_cols<kLanes, kV>(j);
                const V8 v = raw[u][j].get();
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    F2 d = add2(v.p[i], f2(-mean[u]));
                    if (kV) {
                        if (c.first >= n) d = f2(0.f);
                    } else {
                        const float2 e = split(d);
                        d = f2(c[2 * i] < n ? e.x : 0.f, c[2 * i + 1] < n ? e.y : 0.f);
                    }
                    s = fma2(d, d, s);
                }
            }
            rstd[u] = hsum(s);
        }
        group_sum<kLanes>(rstd, sh, turn);
#pragma unroll
        for (int u = 0; u < kRows; ++u) {
            const int64_t row = r0 + u * G::kGroups + sub;
            const bool in = row < rows;
            const float rs = rsqrtf(fmaf(rstd[u], inv_n, eps));
            if (mean_out && in && threadIdx.x % kLanes == 0) {
                mean_out[row] = mean[u];
                rstd_out[row] = rs;
            }
#pragma unroll
            for (int j = 0; j < kChunks; ++j) {
                const Cols<kV> c = chunk_cols<kLanes, kV>(j);
                V8 v = raw[u][j].get();
                if (k8)
                    keep_block<kLanes>(keep, raw[u][j].amax(), v, codes + row * n, scales + row * nblk + c.first / kBlock, c, n, in);
#pragma unroll
                for (int i = 0; i < 4; ++i) v.p[i] = fma2(mul2(add2(v.p[i], f2(-mean[u])), f2(rs)), w[j].p[i], b[j].p[i]);
                store8(y + row * ldy, c, n, in, v);
            }
        }
    }
}

// dx, and the CTA's sums of dy xhat and dy over its rows in partial[CTA][2][n].
// Each thread keeps its channels' sums in registers from row to row.  Rows wait
// for their sums as they came from memory (4 registers per 8 16-bit values) and
// are converted again after it: registers, which set how many rows are in
// flight, are dearer here than instructions.
template <typename T, bool kV, bool k8, int kLanes, int kChunks, int kRows>
__global__ void __launch_bounds__(Group<kLanes>::kCta, norm_ctas(kLanes, kChunks, sizeof(T) == 4, 2))
    norm_backward_kernel(const T *__restrict__ dy, int64_t lddy, Kept k, const float *__restrict__ mean,
                         const float *__restrict__ rstd, Affine af, T *__restrict__ dx, int64_t lddx,
                         float *__restrict__ partial, int64_t rows, int n, int nblk) {
    using G = Group<kLanes>;
    __shared__ float sh[2][16][2 * kRows];
    __shared__ float sums[G::kGroups > 1 ? kThreads * 8 : 1];
    int turn = 0;
    const float inv_n = 1.f / n;
    V8 aw[kChunks], ab[kChunks], w[kChunks];
#pragma unroll
    for (int j = 0; j < kChunks; ++j) {
        w[j] = load_affine<T>(af, af.w, chunk_cols<kLanes, kV>(j), n, 1.f);
        aw[j] = ab[j] = V8{f2(0.f), f2(0.f), f2(0.f), f2(0.f)};
    }
    const int64_t step = (int64_t)gridDim.x * G::kGroups * kRows;
    const int sub = threadIdx.x / kLanes;
    int64_t r0 = (int64_t)blockIdx.x * G::kGroups * kRows;
    Raw8<T, kV> next_g[kRows][kChunks];
    KeptRaw<T, kV, k8> next_x[kRows][kChunks];
    float next_mu[kRows], next_rs[kRows];
    auto fetch = [&](int64_t first) {
#pragma unroll
        for (int u = 0; u < kRows; ++u) {
            const int64_t row = first + u * G::kGroups + sub;
            const bool in = row < rows;
            next_mu[u] = in ? __ldg(mean + row) : 0.f;
            next_rs[u] = in ? __ldg(rstd + row) : 0.f;
#pragma unroll
            for (int j = 0; j < kChunks; ++j) {
                const Cols<kV> c = chunk_cols<kLanes, kV>(j);
                next_g[u][j].load(dy + row * lddy, c, n, in);
                next_x[u][j].load(k, row, c, n, nblk, in);
            }
        }
    };
    fetch(r0);
    for (; r0 < rows; r0 += step) {
        Raw8<T, kV> raw_g[kRows][kChunks];
        KeptRaw<T, kV, k8> raw_x[kRows][kChunks];
        float mu[kRows], rs[kRows], s[2 * kRows];
#pragma unroll
        for (int u = 0; u < kRows; ++u) {
            mu[u] = next_mu[u], rs[u] = next_rs[u];
#pragma unroll
            for (int j = 0; j < kChunks; ++j) raw_g[u][j] = next_g[u][j], raw_x[u][j] = next_x[u][j];
        }
        if (r0 + step < rows) fetch(r0 + step);
#pragma unroll
        for (int u = 0; u < kRows; ++u) {
            F2 s1 = f2(0.f), s2 = f2(0.f);
#pragma unroll
            for (int j = 0; j < kChunks; ++j) {
                const V8 g = raw_g[u][j].get(), x = raw_x[u][j].get(k);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    // past the row's end dy is zero, which keeps xhat there out of every sum
                    const F2 xh = mul2(add2(x.p[i], f2(-mu[u])), f2(rs[u]));
                    const F2 t = mul2(g.p[i], w[j].p[i]);
                    s1 = add2(s1, t);
                    s2 = fma2(t, xh, s2);
                    aw[j].p[i] = fma2(g.p[i], xh, aw[j].p[i]);
                    ab[j].p[i] = add2(ab[j].p[i], g.p[i]);
                }
            }
            s[2 * u] = hsum(s1);
            s[2 * u + 1] = hsum(s2);
        }
        group_sum<kLanes>(s, sh, turn);
        if (!dx) continue;
#pragma unroll
        for (int u = 0; u < kRows; ++u) {
            const int64_t row = r0 + u * G::kGroups + sub;
            const float m1 = s[2 * u] * inv_n, m2 = s[2 * u + 1] * inv_n;
#pragma unroll
            for (int j = 0; j < kChunks; ++j) {
                V8 g = raw_g[u][j].get();
                const V8 x = raw_x[u][j].get(k);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const F2 xh = mul2(add2(x.p[i], f2(-mu[u])), f2(rs[u]));
                    g.p[i] = mul2(f2(rs[u]), fma2(xh, f2(-m2), fma2(g.p[i], w[j].p[i], f2(-m1))));
                }
                store8(dx + row * lddx, chunk_cols<kLanes, kV>(j), n, row < rows, g);
            }
        }
    }
    if (!partial) return;
    float *pr = partial + (int64_t)blockIdx.x * 2 * n;
#pragma unroll
    for (int j = 0; j < kChunks; ++j) {
        const Cols<kV> c = chunk_cols<kLanes, kV>(j);
        if constexpr (G::kGroups > 1) {
            group_sums<kLanes, kThreads, kV>(aw[j], pr, j * kLanes * 8, n, sums);
            group_sums<kLanes, kThreads, kV>(ab[j], pr + n, j * kLanes * 8, n, sums);
        } else {
            float vw[8], vb[8];
            aw[j].get(vw);
            ab[j].get(vb);
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (c[i] < n) {
                    pr[c[i]] = vw[i];
                    pr[n + c[i]] = vb[i];
                }
        }
    }
}

// Rows of more than kMaxHeld channels: a CTA per row that reads it again (from
// cache) for each step.
constexpr int kMaxHeld = 8192;
template <bool kV>
__device__ __forceinline__ Cols<kV> wide_cols(int c0) {  // c0: a multiple of the CTA's 2048 channels
    return Cols<kV>(c0 + (threadIdx.x / 16) * kBlock, threadIdx.x & 15, 16);
}
template <typename T, bool kV>
__global__ void __launch_bounds__(kThreads)
    norm_forward_wide_kernel(const T *__restrict__ x, int64_t ldx, Affine af, T *__restrict__ y, int64_t ldy,
                             float *__restrict__ mean_out, float *__restrict__ rstd_out, uint8_t *__restrict__ codes,
                             float *__restrict__ scales, int64_t rows, int n, int nblk, float eps, int keep) {
    __shared__ float sh[2][16][1];
    int turn = 0;
    for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
        const T *xr = x + row * ldx;
        float s[1] = {0.f}, v[8];
        for (int c0 = 0; c0 < n; c0 += kThreads * 8) {
            load8(xr, wide_cols<kV>(c0), n, true, v);
#pragma unroll
            for (int i = 0; i < 8; ++i) s[0] += v[i];
        }
        group_sum<kThreads>(s, sh, turn);
        const float mean = s[0] / n;
        s[0] = 0.f;
        for (int c0 = 0; c0 < n; c0 += kThreads * 8) {
            const Cols<kV> c = wide_cols<kV>(c0);
            load8(xr, c, n, true, v);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float d = c[i] < n ? v[i] - mean : 0.f;
                s[0] = fmaf(d, d, s[0]);
            }
        }
        group_sum<kThreads>(s, sh, turn);
        const float rstd = 1.f / sqrtf(s[0] / n + eps);
        if (threadIdx.x == 0 && mean_out) {
            mean_out[row] = mean;
            rstd_out[row] = rstd;
        }
        for (int c0 = 0; c0 < n; c0 += kThreads * 8) {
            const Cols<kV> c = wide_cols<kV>(c0);
            Raw8<T, kV> raw;
            raw.load(xr, c, n, true);
            V8 o = raw.get();
            if (keep >= FCAI_KEEP_INT8)
                keep_block<16>(keep, raw.amax(), o, codes + row * n, scales + row * nblk + c.first / kBlock, c, n, true);
            const V8 w = load_affine<T>(af, af.w, c, n, 1.f), b = load_affine<T>(af, af.b, c, n, 0.f);
#pragma unroll
            for (int i = 0; i < 4; ++i) o.p[i] = fma2(mul2(add2(o.p[i], f2(-mean)), f2(rstd)), w.p[i], b.p[i]);
            store8(y + row * ldy, c, n, true, o);
        }
    }
}

// Per row: mean(t), mean(t xhat) into stats.
template <typename T, bool kV, bool k8>
__global__ void __launch_bounds__(kThreads)
    norm_backward_stats_kernel(const T *__restrict__ dy, int64_t lddy, Kept k, const float *__restrict__ mean,
                               const float *__restrict__ rstd, Affine af, float2 *__restrict__ stats, int64_t rows, int n,
                               int nblk) {
    __shared__ float sh[2][16][2];
    int turn = 0;
    for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
        const float mu = mean[row], rs = rstd[row];
        float s[2] = {0.f, 0.f};
        for (int c0 = 0; c0 < n; c0 += kThreads * 8) {
            const Cols<kV> c = wide_cols<kV>(c0);
            Raw8<T, kV> raw_g;
            KeptRaw<T, kV, k8> raw_x;
            raw_g.load(dy + row * lddy, c, n, true);
            raw_x.load(k, row, c, n, nblk, true);
            const V8 g = raw_g.get(), x = raw_x.get(k), w = load_affine<T>(af, af.w, c, n, 1.f);
            F2 s1 = f2(0.f), s2 = f2(0.f);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const F2 t = mul2(g.p[i], w.p[i]);  // zero past the row's end: g is
                s1 = add2(s1, t);
                s2 = fma2(t, mul2(add2(x.p[i], f2(-mu)), f2(rs)), s2);
            }
            s[0] += hsum(s1);
            s[1] += hsum(s2);
        }
        group_sum<kThreads>(s, sh, turn);
        if (threadIdx.x == 0) stats[row] = make_float2(s[0] / n, s[1] / n);
    }
}

template <typename T, bool kV, bool k8>
__global__ void __launch_bounds__(kThreads)
    norm_backward_strip_kernel(const T *__restrict__ dy, int64_t lddy, Kept k, const float *__restrict__ mean,
                               const float *__restrict__ rstd, Affine af, const float2 *__restrict__ stats,
                               T *__restrict__ dx, int64_t lddx, float *__restrict__ partial, int64_t rows, int n, int nblk) {
    __shared__ float sh[kThreads * 8];
    const int base = blockIdx.x * kBlock;
    const Cols<kV> c(base, threadIdx.x & 15, 16);
    V8 aw = {f2(0.f), f2(0.f), f2(0.f), f2(0.f)}, ab = aw;
    const V8 w = load_affine<T>(af, af.w, c, n, 1.f);
    for (int64_t row = (int64_t)blockIdx.y * kRowsIter + (threadIdx.x >> 4); row < rows; row += (int64_t)gridDim.y * kRowsIter) {
        const float mu = mean[row], rs = rstd[row];
        const float2 m = stats[row];
        Raw8<T, kV> raw_g;
        KeptRaw<T, kV, k8> raw_x;
        raw_g.load(dy + row * lddy, c, n, true);
        raw_x.load(k, row, c, n, nblk, true);
        const V8 g = raw_g.get();
        V8 x = raw_x.get(k);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const F2 xh = mul2(add2(x.p[i], f2(-mu)), f2(rs));
            aw.p[i] = fma2(g.p[i], xh, aw.p[i]);
            ab.p[i] = add2(ab.p[i], g.p[i]);
            x.p[i] = mul2(f2(rs), fma2(xh, f2(-m.y), fma2(g.p[i], w.p[i], f2(-m.x))));
        }
        if (dx) store8(dx + row * lddx, c, n, true, x);
    }
    if (partial) {
        float *pr = partial + (int64_t)blockIdx.y * 2 * n;
        group_sums<16, kThreads, kV>(aw, pr, base, n, sh);
        group_sums<16, kThreads, kV>(ab, pr + n, base, n, sh);
    }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------

static int64_t round256(int64_t v) { return (v + 255) / 256 * 256; }
static int blocks_of(int n) { return (n + kBlock - 1) / kBlock; }
static bool codes_vec(const void *codes, int n) { return !codes || ((reinterpret_cast<uintptr_t>(codes) & 7) == 0 && n % 8 == 0); }

// Row shares of the strip kernels: enough CTAs to fill the device, and from
// there on CTAs of 16 steps of 16 rows, long enough for the ring to run full and
// for partial sums to be few, short enough to end evenly.
static int row_shares(int64_t rows, int strips, int lanes = 16) {
    const int64_t steps = (rows + kThreads / lanes - 1) / (kThreads / lanes);
    const int64_t fill = std::max<int64_t>(1, ((int64_t)fcai::sm_count() * 4 + strips - 1) / strips);
    return (int)std::min<int64_t>(steps <= fill ? steps : std::max(fill, (steps + 15) / 16), 65535);
}
// How the layer norm runs rows of n channels: threads a row, 8-channel chunks a thread.
struct Held {
    int lanes, chunks;
};
static Held held(int n) {
    if (n <= 32) return {4, 1};
    if (n <= 128) return {16, 1};
    if (n <= 256) return {32, 1};
    if (n <= 512) return {32, 2};
    if (n <= 1024) return {128, 1};
    if (n <= 2048) return {128, 2};
    if (n <= 4096) return {256, 2};
    return {512, 2};
}
// Rows a group has in flight in the backward kernel.
constexpr int backward_rows(int lanes, int chunks) { return lanes <= 32 ? 2 / chunks : 1; }
// CTAs of the backward kernel: each leaves a partial row of 2 n sums, so it is to
// have 6 steps of rows, once there are two CTAs an SM; rows by single elements 3,
// whose loads more warps hide (fp16 from int8, inputs in memory: 1000 x 1024 10.8 us,
// with as many CTAs as fit 17.3; 5003 x 1024 20.5 and 23.0; 20000 x 200 12.0 and 14.2;
// 2000 x 1021 13.7 with 3 steps, 16.1 with 6).  The workspace is asked for by sizes,
// so rows that are unaligned by address or stride alone have the 6 steps too.
static int norm_backward_grid(int64_t rows, int n) {
    const Held h = held(n);
    const int groups = (h.lanes <= 32 ? kThreads / h.lanes : 1) * backward_rows(h.lanes, h.chunks);
    const int per_sm = h.lanes <= 32 ? 3 : norm_ctas(h.lanes, h.chunks, false, 0);
    const int64_t sms = fcai::sm_count(), steps = (rows + groups - 1) / groups;
    const int64_t want = std::max<int64_t>(std::min<int64_t>(steps, sms * 2), steps / (n % 8 ? 3 : 6));
    return (int)std::max<int64_t>(1, std::min<int64_t>(want, sms * per_sm));
}
static int64_t act_workspace(int64_t rows, int n) {
    return rows ? round256((int64_t)row_shares(rows, blocks_of(n), strip_lanes(n)) * n * 4) : 0;
}
static int64_t norm_workspace(int64_t rows, int n) {
    if (rows == 0) return 0;
    if (n <= kMaxHeld) return round256((int64_t)norm_backward_grid(rows, n) * 2 * n * 4);
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
static int colsum(const float *partial, int rows, int64_t stride, void *out0, int n0, void *out1, int n1, int dtype,
                  cudaStream_t st) {
    const dim3 block(32, 32);
    const int grid = (n0 + n1 + 31) / 32;
    if (dtype == FCAI_DTYPE_BF16)
        colsum_kernel<<<grid, block, 0, st>>>(partial, rows, stride, static_cast<__nv_bfloat16 *>(out0), n0, static_cast<__nv_bfloat16 *>(out1), n1);
    else if (dtype == FCAI_DTYPE_F16)
        colsum_kernel<<<grid, block, 0, st>>>(partial, rows, stride, static_cast<__half *>(out0), n0, static_cast<__half *>(out1), n1);
    else
        colsum_kernel<<<grid, block, 0, st>>>(partial, rows, stride, static_cast<float *>(out0), n0, static_cast<float *>(out1), n1);
    FCAI_CUDA_TRY(cudaGetLastError());
    return FCAI_OK;
}
static bool affine_vec(const void *p, int wdtype) { return !p || aligned16(p, 0, wdtype); }

template <typename T>
static int act_forward(const void *x, int64_t ldx, void *y, int64_t ldy, void *codes, float *scales, int64_t rows, int n,
                       int dtype, int act, int keep, cudaStream_t st) {
    const bool q = keep == FCAI_KEEP_INT8 || keep == FCAI_KEEP_E4M3;
    // f32 goes by single elements: a lane's 32 bytes as two 16-byte accesses leave
    // every store half a sector (30000 x 1024: 60 us, 65 with codes, against 44 and 55;
    // only 64 channels with codes lose by it, 200000 x 64: 32 against 39)
    constexpr bool kWide = sizeof(T) == 2;
    const bool vec = kWide && n % 8 == 0 && aligned16(x, ldx, dtype) && (!y || aligned16(y, ldy, dtype)) && (!q || codes_vec(codes, n));
    const int strips = blocks_of(n);
    const dim3 grid(strips, row_shares(rows, strips, strip_lanes(n)));
    auto kernel = strip_lanes(n) == 4 ? (vec ? act_forward_kernel<T, kWide, 4> : act_forward_kernel<T, false, 4>)
                                      : (vec ? act_forward_kernel<T, kWide, 16> : act_forward_kernel<T, false, 16>);
    kernel<<<grid, kThreads, 0, st>>>(static_cast<const T *>(x), ldx, static_cast<T *>(y), ldy, static_cast<uint8_t *>(codes), scales,
                                      rows, n, strips, act, q ? keep : FCAI_KEEP_NONE);
    FCAI_CUDA_TRY(cudaGetLastError());
    return FCAI_OK;
}
template <typename T>
static int act_backward(const void *dy, int64_t lddy, const Kept &k, void *dx, int64_t lddx, void *bias_grad, int64_t rows, int n,
                        int dtype, int act, float *ws, cudaStream_t st) {
    const int strips = blocks_of(n), shares = row_shares(rows, strips, strip_lanes(n));
    const bool k8 = act != FCAI_ACT_NONE && k.keep != FCAI_KEEP_FULL;
    const bool vec = n % 8 == 0 && aligned16(dy, lddy, dtype) && (!dx || aligned16(dx, lddx, dtype)) &&
                     (act == FCAI_ACT_NONE || (k8 ? codes_vec(k.codes, n) : aligned16(k.x, k.ldx, dtype)));
    auto pick = [&](auto lanes) {
        constexpr int kL = decltype(lanes)::value;
        return act == FCAI_ACT_NONE ? (vec ? act_backward_kernel<T, true, false, false, kL> : act_backward_kernel<T, false, false, false, kL>)
               : k8 ? (vec ? act_backward_kernel<T, true, true, true, kL> : act_backward_kernel<T, false, true, true, kL>)
                    : (vec ? act_backward_kernel<T, true, false, true, kL> : act_backward_kernel<T, false, false, true, kL>);
    };
    auto kernel = strip_lanes(n) == 4 ? pick(std::integral_constant<int, 4>()) : pick(std::integral_constant<int, 16>());
    kernel<<<dim3(strips, shares), kThreads, 0, st>>>(static_cast<const T *>(dy), lddy, k, static_cast<T *>(dx), lddx,
                                                      bias_grad ? ws : nullptr, rows, n, strips, act);
    FCAI_CUDA_TRY(cudaGetLastError());
    return bias_grad ? colsum(ws, shares, n, bias_grad, n, nullptr, 0, dtype, st) : FCAI_OK;
}
template <typename T>
static int load_checkpoint(const Kept &k, void *out, int64_t ldo, int64_t rows, int n, int dtype, cudaStream_t st) {
    const bool vec = n % 8 == 0 && aligned16(out, ldo, dtype) && codes_vec(k.codes, n);
    const int strips = blocks_of(n);
    auto kernel = strip_lanes(n) == 4 ? (vec ? checkpoint_load_kernel<T, true, 4> : checkpoint_load_kernel<T, false, 4>)
                                      : (vec ? checkpoint_load_kernel<T, true, 16> : checkpoint_load_kernel<T, false, 16>);
    kernel<<<dim3(strips, row_shares(rows, strips, strip_lanes(n))), kThreads, 0, st>>>(k, static_cast<T *>(out), ldo, rows, n, strips);
    FCAI_CUDA_TRY(cudaGetLastError());
    return FCAI_OK;
}

struct NormForward {
    const void *x, *w, *b;
    int64_t ldx, ldy, rows;
    void *y, *codes;
    float *mean, *rstd, *scales, eps;
    int n, keep;
    Affine af;
    cudaStream_t st;
};
template <typename T, bool kV, bool k8, int kLanes, int kChunks>
static int launch_norm_forward(const NormForward &a) {
    constexpr int kRows = kLanes <= 32 && kChunks == 1 ? 2 : 1;
    constexpr int64_t kPerCta = (int64_t)Group<kLanes>::kGroups * kRows;
    const int64_t want = (a.rows + kPerCta - 1) / kPerCta;
    const int grid = (int)std::min<int64_t>(want, (int64_t)fcai::sm_count() * (kLanes > 32 ? norm_ctas(kLanes, kChunks, sizeof(T) == 4, 0, !k8 && kV) : 6));
    norm_forward_kernel<T, kV, k8, kLanes, kChunks, kRows><<<grid, Group<kLanes>::kCta, 0, a.st>>>(
        static_cast<const T *>(a.x), a.ldx, a.af, static_cast<T *>(a.y), a.ldy, a.mean, a.rstd, static_cast<uint8_t *>(a.codes),
        a.scales, a.rows, a.n, blocks_of(a.n), a.eps, a.keep);
    FCAI_CUDA_TRY(cudaGetLastError());
    return FCAI_OK;
}
struct NormBackward {
    const void *dy;
    int64_t lddy, lddx, rows;
    Kept k;
    const float *mean, *rstd;
    Affine af;
    void *dx;
    float *partial;
    int n;
    cudaStream_t st;
};
template <typename T, bool kV, bool k8, int kLanes, int kChunks>
static int launch_norm_backward(const NormBackward &a) {
    norm_backward_kernel<T, kV, k8, kLanes, kChunks, backward_rows(kLanes, kChunks)><<<norm_backward_grid(a.rows, a.n), Group<kLanes>::kCta, 0, a.st>>>(
        static_cast<const T *>(a.dy), a.lddy, a.k, a.mean, a.rstd, a.af, static_cast<T *>(a.dx), a.lddx, a.partial, a.rows, a.n,
        blocks_of(a.n));
    FCAI_CUDA_TRY(cudaGetLastError());
    return FCAI_OK;
}
#define RW_BY_HELD(call)                                             \
    switch (h.lanes * 8 + h.chunks) {                                \
        case 4 * 8 + 1: return call(4, 1);                           \
        case 16 * 8 + 1: return call(16, 1);                         \
        case 32 * 8 + 1: return call(32, 1);                         \
        case 32 * 8 + 2: return call(32, 2);                         \
        case 128 * 8 + 1: return call(128, 1);                       \
        case 128 * 8 + 2: return call(128, 2);                       \
        case 256 * 8 + 2: return call(256, 2);                       \
        default: return call(512, 2);                                \
    }
template <typename T, bool kV, bool k8>
static int norm_forward_held(const NormForward &a) {
    const Held h = held(a.n);
#define CALL(lanes, chunks) launch_norm_forward<T, kV, k8, lanes, chunks>(a)
    RW_BY_HELD(CALL)
#undef CALL
}
template <typename T, bool kV, bool k8>
static int norm_backward_held(const NormBackward &a) {
    const Held h = held(a.n);
#define CALL(lanes, chunks) launch_norm_backward<T, kV, k8, lanes, chunks>(a)
    RW_BY_HELD(CALL)
#undef CALL
}

template <typename T>
static int norm_forward(const void *x, int64_t ldx, Affine af, int wdtype, void *y, int64_t ldy, float *mean, float *rstd,
                        void *codes, float *scales, int64_t rows, int n, float eps, int dtype, int keep, cudaStream_t st) {
    const bool q = keep == FCAI_KEEP_INT8 || keep == FCAI_KEEP_E4M3;
    const bool vec = n % 8 == 0 && aligned16(x, ldx, dtype) && aligned16(y, ldy, dtype) && (!q || codes_vec(codes, n));
    af.vec = n % 8 == 0 && affine_vec(af.w, wdtype) && affine_vec(af.b, wdtype);
    if (n <= kMaxHeld) {
        const NormForward a{x, af.w, af.b, ldx, ldy, rows, y, codes, mean, rstd, scales, eps, n, keep, af, st};
        if (q) return vec ? norm_forward_held<T, true, true>(a) : norm_forward_held<T, false, true>(a);
        return vec ? norm_forward_held<T, true, false>(a) : norm_forward_held<T, false, false>(a);
    }
    auto kernel = vec ? norm_forward_wide_kernel<T, true> : norm_forward_wide_kernel<T, false>;
    kernel<<<(int)std::min<int64_t>(rows, (int64_t)fcai::sm_count() * 8), kThreads, 0, st>>>(
        static_cast<const T *>(x), ldx, af, static_cast<T *>(y), ldy, mean, rstd, static_cast<uint8_t *>(codes), scales, rows, n,
        blocks_of(n), eps, keep);
    FCAI_CUDA_TRY(cudaGetLastError());
    return FCAI_OK;
}
template <typename T, bool kV, bool k8>
static int norm_backward_any(const NormBackward &a, float2 *stats, int shares) {
    if (a.n <= kMaxHeld) return norm_backward_held<T, kV, k8>(a);
    const int strips = blocks_of(a.n);
    norm_backward_stats_kernel<T, kV, k8><<<(int)std::min<int64_t>(a.rows, (int64_t)fcai::sm_count() * 8), kThreads, 0, a.st>>>(
        static_cast<const T *>(a.dy), a.lddy, a.k, a.mean, a.rstd, a.af, stats, a.rows, a.n, strips);
    FCAI_CUDA_TRY(cudaGetLastError());
    norm_backward_strip_kernel<T, kV, k8><<<dim3(strips, shares), kThreads, 0, a.st>>>(
        static_cast<const T *>(a.dy), a.lddy, a.k, a.mean, a.rstd, a.af, stats, static_cast<T *>(a.dx), a.lddx, a.partial, a.rows,
        a.n, strips);
    FCAI_CUDA_TRY(cudaGetLastError());
    return FCAI_OK;
}
template <typename T>
static int norm_backward(const void *dy, int64_t lddy, const Kept &k, const float *mean, const float *rstd, Affine af, int wdtype,
                         void *dx, int64_t lddx, void *dweight, void *dbias, int64_t rows, int n, int dtype, unsigned char *ws,
                         cudaStream_t st) {
    const bool k8 = k.keep != FCAI_KEEP_FULL;
    const bool vec = n % 8 == 0 && aligned16(dy, lddy, dtype) && (!dx || aligned16(dx, lddx, dtype)) &&
                     (k8 ? codes_vec(k.codes, n) : aligned16(k.x, k.ldx, dtype));
    af.vec = n % 8 == 0 && affine_vec(af.w, wdtype);
    float2 *stats = nullptr;
    int parts = norm_backward_grid(rows, n);
    if (n > kMaxHeld) {
        stats = reinterpret_cast<float2 *>(ws);
        ws += round256(rows * 8);
        parts = row_shares(rows, blocks_of(n));
    }
    float *partial = dweight || dbias ? reinterpret_cast<float *>(ws) : nullptr;
    const NormBackward a{dy, lddy, lddx, rows, k, mean, rstd, af, dx, partial, n, st};
    const int rc = k8 ? (vec ? norm_backward_any<T, true, true>(a, stats, parts) : norm_backward_any<T, false, true>(a, stats, parts))
                      : (vec ? norm_backward_any<T, true, false>(a, stats, parts) : norm_backward_any<T, false, false>(a, stats, parts));
    if (rc || !partial) return rc;
    return colsum(partial, parts, 2 * (int64_t)n, dweight, n, dbias, n, wdtype, st);
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
