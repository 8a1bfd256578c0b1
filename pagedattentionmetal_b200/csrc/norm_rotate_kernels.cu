// Norm of queries and keys for each head and the rotation by position in one pass, with the
// append of the keys and values to the pages, and the gradient of it.
//
//   n = x * rsqrt(mean(x^2) + eps) * w,   y_a = n_a cos - n_b sin,   y_b = n_b cos + n_a sin
//
// for the pairs (a, b) of the first rotaryDim elements: (i, i + rotaryDim / 2), or
// (2 i, 2 i + 1) when interleaved; angle = position * invFreq[i].  Gradient, with dn the
// rotated gradient turned back, xhat = x * r and g = dn * w:
//
//   dx = r * (g - xhat * mean(g * xhat)),   dw = sum over rows and heads of dn * xhat
//
// The passes are bound by HBM: every element is read and written once.  A thread holds two
// 16-byte pieces of a head's row that contain both members of every pair it turns, so that the
// rotation needs no exchange between threads; the sum of squares is reduced over the few
// consecutive lanes that share a head.  Everything between the load and the one rounding of
// the result is float32, the angle is a float64 product reduced to one turn before it is
// rounded (a float32 product is off by 2^-24 of the position: 0.06 rad at a million tokens).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <type_traits>

#include "kernels.h"
#include "tc_common.cuh"

namespace pam {
namespace {

// Two float32 in one register pair: the passes are close to the issue rate, and a packed product or
// sum is one instruction.
using F2 = unsigned long long;
using tc::add2;
using tc::fma2;
using tc::mul2;
using tc::pack2;
using tc::unpack2;
__device__ __forceinline__ float sumOf(F2 v) {
    float lo, hi;
    unpack2(v, lo, hi);
    return lo + hi;
}

__device__ __forceinline__ float toFloat(float v) { return v; }
__device__ __forceinline__ float toFloat(__half v) { return __half2float(v); }
__device__ __forceinline__ float toFloat(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T fromFloat(float v);
template <> __device__ __forceinline__ float fromFloat<float>(float v) { return v; }
template <> __device__ __forceinline__ __half fromFloat<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 fromFloat<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// cos and sin of position * freq: the angle in half turns, reduced to one turn in float64.
__device__ __forceinline__ float2 turnOf(int position, float freq) {
    constexpr double kInvPi = 0.318309886183790671537768;
    const double t = static_cast<double>(position) * static_cast<double>(freq) * kInvPi;
    float2 cs;
    sincospif(static_cast<float>(t - 2.0 * rint(0.5 * t)), &cs.y, &cs.x);
    return cs;
}

// 16 bytes of a row: E elements.
template <typename T>
struct Piece {
    static constexpr int E = 16 / sizeof(T);
    union {
        uint4 raw;
        uint32_t word[4];
    };
    __device__ __forceinline__ Piece() {
#pragma unroll
        for (int i = 0; i < 4; ++i) word[i] = 0u;
    }
    __device__ __forceinline__ void load(const T* p) { raw = *reinterpret_cast<const uint4*>(p); }
    __device__ __forceinline__ void store(T* p) const { *reinterpret_cast<uint4*>(p) = raw; }
    // The compiler may not keep what was unpacked before: unpacking again costs less than the registers
    // that hold it (more rows in flight).
    __device__ __forceinline__ void forget() {
#pragma unroll
        for (int i = 0; i < 4; ++i) asm volatile("" : "+r"(word[i]));
    }
    __device__ __forceinline__ void unpack(F2 (&f)[E / 2]) const {
#pragma unroll
        for (int e = 0; e < E / 2; ++e) {
            if constexpr (sizeof(T) == 4) f[e] = pack2(__uint_as_float(word[2 * e]), __uint_as_float(word[2 * e + 1]));
            else if constexpr (std::is_same_v<T, __half>) {
                const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&word[e]));
                f[e] = pack2(v.x, v.y);
            } else f[e] = pack2(__uint_as_float(word[e] << 16), __uint_as_float(word[e] & 0xFFFF0000u));
        }
    }
    __device__ __forceinline__ void pack(const F2 (&f)[E / 2]) {
#pragma unroll
        for (int e = 0; e < E / 2; ++e) {
            float lo, hi;
            unpack2(f[e], lo, hi);
            if constexpr (sizeof(T) == 4) { word[2 * e] = __float_as_uint(lo); word[2 * e + 1] = __float_as_uint(hi); }
            else if constexpr (std::is_same_v<T, __half>) {
                const __half2 v = __floats2half2_rn(lo, hi);
                word[e] = *reinterpret_cast<const uint32_t*>(&v);
            } else {
                const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
                word[e] = *reinterpret_cast<const uint32_t*>(&v);
            }
        }
    }
};

// How the pieces of a row are dealt to lanes.  Lane t of a head takes pieces (a, b):
//  rotated, halves:       (t, t + rotaryDim / (2 E));  interleaved: (2 t, 2 t + 1)
//  the tail behind rotaryDim: neighbouring pieces, b may not exist.
struct Layout {
    int lanes;         // lanes that share a head: a power of two
    int pairs;         // lanes with rotated pieces
    int pieces;        // pieces of a row
    int half;          // halves: distance of a pair's pieces; interleaved: 0
    __host__ __device__ void lane(int t, int& a, int& b) const {
        if (half && t < pairs) { a = t; b = t + half; }
        else { a = 2 * t; b = 2 * t + 1; }           // (tail: 2 pairs pieces come before it)
    }
};

template <int E>
Layout layoutOf(int headDim, int rotaryDim, int interleaved) {
    Layout l{};
    l.pieces = headDim / E;
    l.pairs = interleaved ? (rotaryDim / E + 1) / 2 : rotaryDim / (2 * E);
    l.half = interleaved ? 0 : l.pairs;
    const int need = (l.pieces + 1) / 2;
    for (l.lanes = 1; l.lanes < need; l.lanes *= 2) {}
    return l;
}

// The turn of the pieces' pairs by the angles that `cs` (cosines, and sines `half` behind them) holds
// from the piece's first one on: sign * angle.
template <int E>
__device__ __forceinline__ void rotateHalves(F2 (&x)[E / 2], F2 (&y)[E / 2], const float* cs, int half, float sign) {
    const F2 s2 = pack2(sign, sign), minus = pack2(-sign, -sign);
#pragma unroll
    for (int q = 0; q < E / 4; ++q) {
        const float4 c = *reinterpret_cast<const float4*>(cs + 4 * q), s = *reinterpret_cast<const float4*>(cs + half + 4 * q);
        const F2 cc[2] = {pack2(c.x, c.y), pack2(c.z, c.w)}, ss[2] = {pack2(s.x, s.y), pack2(s.z, s.w)};
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const F2 a = x[2 * q + e], b = y[2 * q + e];
            x[2 * q + e] = fma2(mul2(b, ss[e]), minus, mul2(a, cc[e]));
            y[2 * q + e] = fma2(mul2(a, ss[e]), s2, mul2(b, cc[e]));
        }
    }
}
template <int E>
__device__ __forceinline__ void rotatePairs(F2 (&x)[E / 2], const float* cs, int half, float sign) {
#pragma unroll
    for (int e = 0; e < E / 2; ++e) {
        const float c = cs[e], s = sign * cs[half + e];
        float a, b;
        unpack2(x[e], a, b);
        x[e] = pack2(a * c - b * s, b * c + a * s);
    }
}

// Where a slot's row starts in a pool [block][kvHeads][blockSize][dim], head 0: element offset, or -1
// outside the pool.  (One division per row of the launch, not per head.)
__device__ __forceinline__ int64_t poolBase(int64_t slot, int64_t numSlots, int kvHeads, int blockSize, int dim) {
    if (slot < 0 || slot >= numSlots) return -1;
    int64_t blk;
    int off;
    if ((blockSize & (blockSize - 1)) == 0) {
        blk = slot >> (__ffs(blockSize) - 1);
        off = static_cast<int>(slot & (blockSize - 1));
    } else {
        blk = slot / blockSize;
        off = static_cast<int>(slot - blk * blockSize);
    }
    return (blk * kvHeads * blockSize + off) * dim;
}

// What a block looks up of its rows before it works on them.
struct RowInfo {
    int64_t pool;      // poolBase of the row's slot
    int position;      // negative: skipped
};

// Positions, slots and turns of rows [row0, row0 + n) into shared memory.  rowPools: the pools are rows back to
// back, row r at place r.
__device__ __forceinline__ void lookRowsUp(RowInfo* info, float* turns, int64_t row0, int n, const int32_t* positions, const int64_t* slots,
                                           int64_t numSlots, const float* invFreq, int half, int kvHeads, int blockSize, int dim, bool rowPools) {
    for (int i = threadIdx.x; i < n; i += blockDim.x) {
        info[i].position = positions[row0 + i];
        info[i].pool = rowPools ? (row0 + i) * kvHeads * dim : slots ? poolBase(slots[row0 + i], numSlots, kvHeads, blockSize, dim) : -1;
    }
    for (int i = threadIdx.x; i < n * half; i += blockDim.x) {
        const int r = i / half, pos = positions[row0 + r];
        if (pos >= 0) {
            const float2 cs = turnOf(pos, invFreq[i - r * half]);
            turns[r * half + i] = cs.x;              // a row's cosines, then its sines
            turns[r * half + i + half] = cs.y;
        }
    }
    __syncthreads();
}

template <int E>
__device__ __forceinline__ void turnPieces(F2 (&fa)[E / 2], F2 (&fb)[E / 2], const Layout& l, int lane, int pa, int pb, int rotaryDim,
                                           const float* cs, float sign) {
    const int half = rotaryDim / 2;
    if (l.half) {
        if (lane < l.pairs) rotateHalves<E>(fa, fb, cs + pa * E, half, sign);
    } else {
        if (pa * E < rotaryDim) rotatePairs<E>(fa, cs + pa * E / 2, half, sign);
        if (pb * E < rotaryDim) rotatePairs<E>(fb, cs + pb * E / 2, half, sign);
    }
}

// ---- forward ----------------------------------------------------------------

// 16 bytes to shared memory, or zeros.
__device__ __forceinline__ void copyAhead(void* to, const void* from, bool there) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(static_cast<uint32_t>(__cvta_generic_to_shared(to))), "l"(from), "r"(there ? 16 : 0) : "memory");
}
constexpr int kForwardStages = 4;        // rows in shared memory or on their way there

// A block takes `rowsPer` rows.  A group of l.lanes lanes keeps one head of them (of the queries,
// keys and values of a row, one after the other), so that its weights stay in registers and nothing
// is divided inside the loop; rows come to shared memory by asynchronous copies, three ahead, each
// thread its own pieces.  Measured at 32768 rows of 32 + 8 + 8 heads of 128, float16 (806 MB), call after call on
// the same buffers: 138 us = 5.8 TB/s, 0.89 of the copy rate (156 us, 0.79, where every call has buffers of its
// own); two rows ahead 142 us, 96 registers (one block less on an SM) 195 us, 56 154 us; one row ahead in
// registers 155 us; one row a block with a division per head 277 us; 8-byte pieces 242 us (twice the
// instructions per byte).  float32 (1.6 GB) 255 us, 0.96 of the copy rate.
template <typename T>
__global__ void __maxnreg__(80)
normRotateKernel(const __grid_constant__ NormRotateParams p, const Layout l, int rowsPer) {
    using P = Piece<T>;
    constexpr int E = P::E;
    extern __shared__ __align__(16) unsigned char rowSmem[];
    unsigned char* ring = rowSmem;                                        // [kForwardStages][2][threads][16]
    RowInfo* info = reinterpret_cast<RowInfo*>(ring + kForwardStages * 2 * 16 * blockDim.x);              // [rowsPer]
    float* turns = reinterpret_cast<float*>(info + rowsPer);              // [rowsPer][rotaryDim]
    const int tid = threadIdx.x, half = p.rotaryDim / 2;
    const int64_t row0 = static_cast<int64_t>(blockIdx.x) * rowsPer;
    const int n = static_cast<int>(min(static_cast<int64_t>(rowsPer), p.numRows - row0));
    lookRowsUp(info, turns, row0, n, p.positions, p.slots, p.numSlots, p.invFreq, half, p.kvHeads, p.blockSize, p.headDim, p.slotsOut != nullptr);
    if (p.slotsOut && blockIdx.y == 0)
        for (int i = tid; i < n; i += blockDim.x) p.slotsOut[row0 + i] = info[i].position >= 0 ? p.slots[row0 + i] : -1;
    const int lane = tid & (l.lanes - 1), group = tid / l.lanes, groups = blockDim.x / l.lanes;
    const int perRow = p.heads + 2 * p.kvHeads;       // queries, keys, values
    int pa, pb;
    l.lane(lane, pa, pb);
    const bool hasA = pa < l.pieces, hasB = pb < l.pieces;
    const float invDim = 1.f / static_cast<float>(p.headDim);
    // (whole warps stay in the loops for the shuffles)
    const int h = static_cast<int>(blockIdx.y) * groups + group;
    const bool isQ = h < p.heads, isV = h >= p.heads + p.kvHeads;
    const int kvh = isQ ? 0 : isV ? h - p.heads - p.kvHeads : h - p.heads;
    const bool wanted = h < perRow && !(isV && !p.vPool);
    const T* src = isQ ? static_cast<const T*>(p.q) + static_cast<int64_t>(h) * p.headDim
                 : isV ? static_cast<const T*>(p.v) + static_cast<int64_t>(kvh) * p.headDim
                       : static_cast<const T*>(p.k) + static_cast<int64_t>(kvh) * p.headDim;
    const int64_t stride = isQ ? p.qStride : isV ? p.vStride : p.kStride;
    T* rows = static_cast<T*>(isQ ? p.qOut : isV ? nullptr : p.kOut);
    const int64_t rowsStride = isQ ? p.qOutStride : p.kOutStride;
    if (rows) rows += static_cast<int64_t>(isQ ? h : kvh) * p.headDim;
    T* pool = isQ ? nullptr : static_cast<T*>(isV ? p.vPool : p.kPool);
    if (pool) pool += static_cast<int64_t>(kvh) * (p.slotsOut ? 1 : p.blockSize) * p.headDim;
    P wa, wb;
    if (wanted && !isV && hasA) {
        const T* weight = static_cast<const T*>(isQ ? p.qWeight : p.kWeight);
        wa.load(weight + pa * E);
        if (hasB) wb.load(weight + pb * E);
    }
    auto place = [&](int r, int which) { return ring + static_cast<size_t>(((r % kForwardStages) * 2 + which) * blockDim.x + tid) * 16; };
    auto fetch = [&](int r) {
        if (wanted && hasA && r < n && info[r].position >= 0) {
            const T* at = src + (row0 + r) * stride;
            copyAhead(place(r, 0), at + pa * E, true);
            copyAhead(place(r, 1), at + (hasB ? pb : pa) * E, hasB);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll
    for (int r = 0; r < kForwardStages - 1; ++r) fetch(r);
#pragma unroll 1
    for (int r = 0; r < n; ++r) {
        asm volatile("cp.async.wait_group %0;" ::"n"(kForwardStages - 2) : "memory");
        P a, b;
        if (hasA) {                               // (lanes without a piece add zeros)
            a.raw = *reinterpret_cast<const uint4*>(place(r, 0));
            b.raw = *reinterpret_cast<const uint4*>(place(r, 1));
        }
        fetch(r + kForwardStages - 1);            // (where the row before this one was)
        F2 sq = 0ull;
        {
            F2 fa[E / 2], fb[E / 2];
            a.unpack(fa);
            b.unpack(fb);
#pragma unroll
            for (int e = 0; e < E / 2; ++e) sq = fma2(fb[e], fb[e], fma2(fa[e], fa[e], sq));
        }
        float sum = sumOf(sq);
        for (int o = l.lanes >> 1; o > 0; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
        a.forget(); b.forget(); wa.forget(); wb.forget();
        if (wanted && hasA && info[r].position >= 0) {
            if (!isV) {
                F2 fa[E / 2], fb[E / 2], ga[E / 2], gb[E / 2];
                a.unpack(fa);
                b.unpack(fb);
                wa.unpack(ga);
                wb.unpack(gb);
                const float root = rsqrtf(sum * invDim + p.eps);
                const F2 scale = pack2(root, root);
#pragma unroll
                for (int e = 0; e < E / 2; ++e) {
                    fa[e] = mul2(mul2(fa[e], scale), ga[e]);
                    fb[e] = mul2(mul2(fb[e], scale), gb[e]);
                }
                turnPieces<E>(fa, fb, l, lane, pa, pb, p.rotaryDim, turns + r * 2 * half, 1.f);
                a.pack(fa);
                b.pack(fb);
            }
            const int64_t row = row0 + r, at = info[r].pool;
            if (rows) {
                a.store(rows + row * rowsStride + pa * E);
                if (hasB) b.store(rows + row * rowsStride + pb * E);
            }
            if (pool && at >= 0) {
                a.store(pool + at + pa * E);
                if (hasB) b.store(pool + at + pb * E);
            }
        }
    }
}

// Address of a slot's row in a pool [block][kvHeads][blockSize][dim], element offset.
__device__ __forceinline__ int64_t poolOffset(int64_t slot, int kvh, int kvHeads, int blockSize, int dim) {
    const int64_t blk = slot / blockSize, off = slot - blk * blockSize;
    return ((blk * kvHeads + kvh) * blockSize + off) * static_cast<int64_t>(dim);
}

constexpr int kForwardRows = 16;
constexpr int kMaxDim = 256;

// Any head_dim, rotaryDim and alignment: one warp per (row, head), element by element, the row
// in shared memory so that outputs may lie over the inputs.  Cosine and sine are taken anew for every element of
// every head: 8192 rows of 32 + 8 + 8 heads of 96, float16, with 24 rotated elements 195 us, where the pieces
// (all 96 rotated) take 45 us.
template <typename T>
__global__ void __launch_bounds__(128)
normRotateAnyKernel(const __grid_constant__ NormRotateParams p) {
    __shared__ float xs[4][kMaxDim];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, half = p.rotaryDim / 2;
    const int perRow = p.heads + 2 * p.kvHeads;
    const int64_t total = static_cast<int64_t>(p.numRows) * perRow;
    float* x = xs[warp];
    for (int64_t w = blockIdx.x * static_cast<int64_t>(4) + warp; w < total; w += gridDim.x * static_cast<int64_t>(4)) {
        const int64_t row = w / perRow;
        const int h = static_cast<int>(w % perRow), pos = p.positions[row];
        if (p.slotsOut && h == 0 && lane == 0) p.slotsOut[row] = pos >= 0 ? p.slots[row] : -1;
        if (pos < 0) continue;
        const bool isQ = h < p.heads, isV = h >= p.heads + p.kvHeads;
        if (isV && !p.vPool) continue;
        const int kvh = isQ ? 0 : isV ? h - p.heads - p.kvHeads : h - p.heads;
        const T* src = isQ ? static_cast<const T*>(p.q) + row * p.qStride + static_cast<int64_t>(h) * p.headDim
                     : isV ? static_cast<const T*>(p.v) + row * p.vStride + static_cast<int64_t>(kvh) * p.headDim
                           : static_cast<const T*>(p.k) + row * p.kStride + static_cast<int64_t>(kvh) * p.headDim;
        float sum = 0.f;
        for (int d = lane; d < p.headDim; d += 32) {
            x[d] = toFloat(src[d]);
            sum += x[d] * x[d];
        }
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
        __syncwarp();
        const float r = rsqrtf(sum / static_cast<float>(p.headDim) + p.eps);
        const T* weight = static_cast<const T*>(isQ ? p.qWeight : p.kWeight);
        T* dst[2] = {nullptr, nullptr};
        if (isQ) dst[0] = static_cast<T*>(p.qOut) + row * p.qOutStride + static_cast<int64_t>(h) * p.headDim;
        else {
            void* pool = isV ? p.vPool : p.kPool;
            if (!isV && p.kOut) dst[0] = static_cast<T*>(p.kOut) + row * p.kOutStride + static_cast<int64_t>(kvh) * p.headDim;
            if (pool) {
                const int64_t slot = p.slots[row];
                if (p.slotsOut) dst[1] = static_cast<T*>(pool) + (row * p.kvHeads + kvh) * p.headDim;
                else if (slot >= 0 && slot < p.numSlots)
                    dst[1] = static_cast<T*>(pool) + poolOffset(slot, kvh, p.kvHeads, p.blockSize, p.headDim);
            }
        }
        for (int d = lane; d < p.headDim; d += 32) {
            float y = x[d];
            if (!isV) {
                y *= r * toFloat(weight[d]);
                if (d < p.rotaryDim) {
                    const int i = p.interleaved ? d >> 1 : d % half;
                    const bool first = p.interleaved ? !(d & 1) : d < half;
                    const int other = p.interleaved ? d ^ 1 : first ? d + half : d - half;
                    const float2 cs = turnOf(pos, p.invFreq[i]);
                    const float z = x[other] * r * toFloat(weight[other]);
                    y = first ? y * cs.x - z * cs.y : y * cs.x + z * cs.y;
                }
            }
            if (dst[0]) dst[0][d] = fromFloat<T>(y);
            if (dst[1]) dst[1][d] = fromFloat<T>(y);
        }
        __syncwarp();
    }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// The 16-byte pieces need every address and stride on 16 bytes, no pair cut by a piece's end,
// and a head within a warp.
template <int E>
bool piecesApply(int headDim, int rotaryDim, int interleaved) {
    if (headDim % E || headDim / E > 64) return false;
    return interleaved ? rotaryDim % E == 0 : rotaryDim % (2 * E) == 0;
}

// Heads of a row that one block takes, and its threads: chunks of equal size, about kThreadsWanted
// threads each.
constexpr int kThreadsWanted = 512;
inline void headChunks(int perRow, int lanes, int* chunks, int* threads) {
    *chunks = std::max(1, (perRow * lanes + kThreadsWanted - 1) / kThreadsWanted);
    const int heads = (perRow + *chunks - 1) / *chunks;
    *threads = (heads * lanes + 31) / 32 * 32;
    *chunks = (perRow * lanes + *threads - 1) / *threads;
}

template <typename T>
cudaError_t normRotateOf(const NormRotateParams& p, int smCount, cudaStream_t stream, int* launches) {
    constexpr int E = Piece<T>::E;
    const void* ptrs[] = {p.q, p.k, p.v, p.qWeight, p.kWeight, p.qOut, p.kOut, p.kPool, p.vPool};
    bool pieces = piecesApply<E>(p.headDim, p.rotaryDim, p.interleaved);
    for (const void* ptr : ptrs) pieces = pieces && aligned16(ptr);
    for (int64_t s : {p.qStride, p.kStride, p.vStride, p.qOutStride, p.kOutStride}) pieces = pieces && s % E == 0;
    const int perRow = p.heads + 2 * p.kvHeads;
    if (!pieces) {
        const int64_t warps = static_cast<int64_t>(p.numRows) * perRow;
        normRotateAnyKernel<T><<<static_cast<unsigned>(std::min<int64_t>((warps + 3) / 4, smCount * 16)), 128, 0, stream>>>(p);
    } else {
        const Layout l = layoutOf<E>(p.headDim, p.rotaryDim, p.interleaved);
        int chunks, threads;
        headChunks(perRow, l.lanes, &chunks, &threads);
        // enough blocks for every SM first, then rows to share the look-ups and the weights
        const int rowsPer = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(kForwardRows, p.numRows / (smCount * 4))));
        const size_t smem = static_cast<size_t>(threads) * kForwardStages * 2 * 16 + static_cast<size_t>(rowsPer) * (sizeof(RowInfo) + (p.rotaryDim / 2) * sizeof(float2));
        // (at most 544 threads, 68 KB of rows, and 16 KB of turns)
        static std::atomic<unsigned long long> done{0};
        const cudaError_t allowed = allowSmem(normRotateKernel<T>, 100 * 1024, done);
        if (allowed != cudaSuccess) return allowed;
        const dim3 grid(static_cast<unsigned>((static_cast<int64_t>(p.numRows) + rowsPer - 1) / rowsPer), chunks);
        normRotateKernel<T><<<grid, threads, smem, stream>>>(p, l, rowsPer);
    }
    *launches += 1;
    return cudaGetLastError();
}

// ---- backward ---------------------------------------------------------------

constexpr int kBackwardRows = 32;        // rows that a block looks up at a time
constexpr int kBackwardShare = 4;        // rows that a block has at least
constexpr int kBackwardStages = 3;       // rows in shared memory or on their way there


// As the forward kernel, every block with an equal share of the rows.  A group of lanes keeps one head
// of a row and each lane its pieces of it, so that its share of the weight gradients stays in
// registers over all its rows; then the groups of the queries and those of the keys are summed through
// shared memory in a fixed order and the block writes its [2][dim] partial sums: no atomics, the same
// bits for the same grid.  Rows come to shared memory by asynchronous copies, two ahead, each thread its
// own pieces, so that no registers wait for them and no barrier stands in the loop.  Measured at 8192
// rows of 32 + 8 heads of 128, bfloat16 (252 MB): 55.4 us = 4.5 TB/s, 0.69 of the copy rate, bound by
// instructions: 455 a warp for each 16 elements of its lanes, 67% of the issue slots taken with 4.4 warps a
// scheduler; one row ahead in registers, with look-ups for 8 rows at a time, 76 us; three rows ahead 55.5 us;
// 80 registers, with spills, 61 us; four blocks on an SM 59 us.
template <typename T>
__global__ void __maxnreg__(96)
normRotateBackwardKernel(const __grid_constant__ NormRotateBackwardParams p, const Layout l, int share) {
    using P = Piece<T>;
    constexpr int E = P::E;
    extern __shared__ __align__(16) unsigned char rowSmem[];
    const int tid = threadIdx.x, half = p.rotaryDim / 2, threads = blockDim.x;
    unsigned char* ring = rowSmem;                                        // [kBackwardStages][4][threads][16]
    float* sums = reinterpret_cast<float*>(rowSmem);                      // [threads][2 E], behind the loop
    static_assert(2 * E * sizeof(float) <= kBackwardStages * 4 * 16, "the sums take the place of the rows");
    RowInfo* info = reinterpret_cast<RowInfo*>(ring + kBackwardStages * 4 * 16 * threads);                // [kBackwardRows]
    float* turns = reinterpret_cast<float*>(info + kBackwardRows);        // [kBackwardRows][rotaryDim]
    const int lane = tid & (l.lanes - 1), group = tid / l.lanes, groups = threads / l.lanes;
    const int perRow = p.heads + p.kvHeads + (p.dV ? p.kvHeads : 0);
    const int64_t begin = static_cast<int64_t>(blockIdx.x) * share, end = min(begin + share, static_cast<int64_t>(p.numRows));
    int pa, pb;
    l.lane(lane, pa, pb);
    const bool hasA = pa < l.pieces, hasB = pb < l.pieces;
    const float invDim = 1.f / static_cast<float>(p.headDim);
    const int h0 = static_cast<int>(blockIdx.y) * groups, h = h0 + group;
    const bool isQ = h < p.heads, isV = h >= p.heads + p.kvHeads, wanted = h < perRow;
    const int kvh = isQ ? 0 : isV ? h - p.heads - p.kvHeads : h - p.heads;
    const T* src = isQ ? static_cast<const T*>(p.q) + static_cast<int64_t>(h) * p.headDim : static_cast<const T*>(p.k) + static_cast<int64_t>(kvh) * p.headDim;
    const int64_t srcStride = isQ ? p.qStride : p.kStride;
    // the gradient with respect to the rotated row: rows, or (keys and values) pages
    const T* up = isQ ? static_cast<const T*>(p.dQOut) + static_cast<int64_t>(h) * p.headDim
                : !isV && p.dKOut ? static_cast<const T*>(p.dKOut) + static_cast<int64_t>(kvh) * p.headDim
                : static_cast<const T*>(isV ? p.dVPool : p.dKPool) + static_cast<int64_t>(kvh) * p.blockSize * p.headDim;
    const int64_t upStride = static_cast<int64_t>(isQ ? p.heads : p.kvHeads) * p.headDim;
    const bool fromPool = !isQ && (isV || !p.dKOut);
    T* dst = static_cast<T*>(isQ ? p.dQ : isV ? p.dV : p.dK) + static_cast<int64_t>(isQ ? h : kvh) * p.headDim;
    const int64_t dstStride = isQ ? p.dQStride : isV ? p.dVStride : p.dKStride;
    P wa, wb;
    if (wanted && !isV && hasA) {
        const T* weight = static_cast<const T*>(isQ ? p.qWeight : p.kWeight);
        wa.load(weight + pa * E);
        if (hasB) wb.load(weight + pb * E);
    }
    F2 accA[E / 2], accB[E / 2];
#pragma unroll
    for (int e = 0; e < E / 2; ++e) accA[e] = accB[e] = 0ull;
    for (int64_t row0 = begin; row0 < end; row0 += kBackwardRows) {
        const int n = static_cast<int>(min(static_cast<int64_t>(kBackwardRows), end - row0));
        __syncthreads();
        lookRowsUp(info, turns, row0, n, p.positions, p.slots, p.numSlots, p.invFreq, half, p.kvHeads, p.blockSize, p.headDim, false);
        // A thread copies what it will read itself, two rows ahead; nobody waits for anybody.
        auto place = [&](int r, int which) { return ring + static_cast<size_t>(((r % kBackwardStages) * 4 + which) * threads + tid) * 16; };
        auto fetch = [&](int r) {
            if (wanted && hasA && r < n && info[r].position >= 0) {
                if (!isV) {
                    const T* at = src + (row0 + r) * srcStride;
                    copyAhead(place(r, 0), at + pa * E, true);
                    copyAhead(place(r, 1), at + (hasB ? pb : pa) * E, hasB);
                }
                const int64_t slot = info[r].pool;
                const T* from = fromPool ? up + (slot >= 0 ? slot : 0) : up + (row0 + r) * upStride;
                const bool there = !fromPool || slot >= 0;
                copyAhead(place(r, 2), from + pa * E, there);
                copyAhead(place(r, 3), from + (hasB ? pb : pa) * E, there && hasB);
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
#pragma unroll
        for (int r = 0; r < kBackwardStages - 1; ++r) fetch(r);
#pragma unroll 1
        for (int r = 0; r < n; ++r) {
            asm volatile("cp.async.wait_group %0;" ::"n"(kBackwardStages - 2) : "memory");
            struct { P xa, xb, ya, yb; } w;
            if (hasA) {                           // (lanes without a piece add zeros)
                w.xa.raw = *reinterpret_cast<const uint4*>(place(r, 0));
                w.xb.raw = *reinterpret_cast<const uint4*>(place(r, 1));
                w.ya.raw = *reinterpret_cast<const uint4*>(place(r, 2));
                w.yb.raw = *reinterpret_cast<const uint4*>(place(r, 3));
            }
            fetch(r + kBackwardStages - 1);       // (where the row before this one was)
            const bool live = wanted && hasA && info[r].position >= 0;
            T* to = dst + (row0 + r) * dstStride;
            if (live && isV) {
                w.ya.store(to + pa * E);
                if (hasB) w.yb.store(to + pb * E);
            }
            F2 ga[E / 2], gb[E / 2], sq = 0ull, xg = 0ull;                // sums of x^2, and of x * g
            w.ya.unpack(ga); w.yb.unpack(gb);
            turnPieces<E>(ga, gb, l, lane, pa, pb, p.rotaryDim, turns + r * 2 * half, -1.f);
            {
                F2 fa[E / 2], fb[E / 2], va[E / 2], vb[E / 2];
                w.xa.unpack(fa); w.xb.unpack(fb);
                wa.unpack(va); wb.unpack(vb);
#pragma unroll
                for (int e = 0; e < E / 2; ++e) {
                    sq = fma2(fb[e], fb[e], fma2(fa[e], fa[e], sq));
                    xg = fma2(fb[e], mul2(gb[e], vb[e]), fma2(fa[e], mul2(ga[e], va[e]), xg));
                }
            }
            w.xa.forget(); w.xb.forget(); wa.forget(); wb.forget();
            float sum = sumOf(sq), dot = sumOf(xg);
            for (int o = l.lanes >> 1; o > 0; o >>= 1) {
                sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
                dot += __shfl_xor_sync(0xFFFFFFFFu, dot, o);
            }
            if (live && !isV) {
                const float root = rsqrtf(sum * invDim + p.eps);
                const float mean = dot * root * invDim;               // of xhat * g
                const F2 scale = pack2(root, root), minusMean = pack2(-mean, -mean);
                F2 fa[E / 2], fb[E / 2], va[E / 2], vb[E / 2], ha[E / 2], hb[E / 2];
                w.xa.unpack(fa); w.xb.unpack(fb);
                wa.unpack(va); wb.unpack(vb);
#pragma unroll
                for (int e = 0; e < E / 2; ++e) {
                    const F2 ua = mul2(fa[e], scale), ub = mul2(fb[e], scale);        // xhat
                    ha[e] = mul2(scale, fma2(ua, minusMean, mul2(ga[e], va[e])));
                    hb[e] = mul2(scale, fma2(ub, minusMean, mul2(gb[e], vb[e])));
                    accA[e] = fma2(ga[e], ua, accA[e]);
                    accB[e] = fma2(gb[e], ub, accB[e]);
                }
                P out;
                out.pack(ha);
                out.store(to + pa * E);
                if (hasB) {
                    out.pack(hb);
                    out.store(to + pb * E);
                }
            }
        }
    }
    if (!p.partials) return;
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();
#pragma unroll
    for (int e = 0; e < E / 2; ++e) {
        *reinterpret_cast<F2*>(sums + tid * 2 * E + 2 * e) = accA[e];
        *reinterpret_cast<F2*>(sums + tid * 2 * E + E + 2 * e) = accB[e];
    }
    __syncthreads();
    // element i of a head: the lane and place that hold it, its groups in order, queries and keys apart
    for (int i = tid; i < l.lanes * 2 * E; i += threads) {
        int a, b;
        l.lane(i / (2 * E), a, b);
        const int e = i % (2 * E), piece = e < E ? a : b;
        if (piece >= l.pieces) continue;
        const int d = piece * E + e % E, queries = min(max(p.heads - h0, 0), groups);
        const int both = min(max(p.heads + p.kvHeads - h0, 0), groups);
        float q = 0.f, k = 0.f;
        for (int g = 0; g < queries; ++g) q += sums[g * l.lanes * 2 * E + i];
        for (int g = queries; g < both; ++g) k += sums[g * l.lanes * 2 * E + i];
        float* out = p.partials + (static_cast<int64_t>(blockIdx.y) * gridDim.x + blockIdx.x) * 2 * p.headDim;
        out[d] = q;
        out[p.headDim + d] = k;
    }
}

// Any shape and alignment, one warp per (row, head) at a time: the warp's share of the weight
// gradients is added up in shared memory, each element by the lane that owns it.  As the forward one, and with the
// few blocks that the partial sums are counted for: 8192 rows of 32 + 8 heads of 96, float16, with 24 rotated
// elements 754 us, where the pieces (all 96 rotated) take 58 us.
template <typename T>
__global__ void __launch_bounds__(128)
normRotateBackwardAnyKernel(const __grid_constant__ NormRotateBackwardParams p) {
    extern __shared__ float smemAny[];                // per warp: x, g (dn), accQ, accK, [dim] each
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, half = p.rotaryDim / 2, D = p.headDim;
    float *x = smemAny + static_cast<size_t>(warp) * 4 * D, *g = x + D, *accQ = g + D, *accK = accQ + D;
    for (int d = lane; d < D; d += 32) accQ[d] = accK[d] = 0.f;
    const int perRow = p.heads + p.kvHeads + (p.dV ? p.kvHeads : 0);
    const int64_t total = static_cast<int64_t>(p.numRows) * perRow;
    for (int64_t w = blockIdx.x * static_cast<int64_t>(4) + warp; w < total; w += gridDim.x * static_cast<int64_t>(4)) {
        const int64_t row = w / perRow;
        const int h = static_cast<int>(w % perRow), pos = p.positions[row];
        if (pos < 0) continue;
        const bool isQ = h < p.heads, isV = h >= p.heads + p.kvHeads;
        const int kvh = isQ ? 0 : isV ? h - p.heads - p.kvHeads : h - p.heads;
        const int64_t slot = p.slots ? p.slots[row] : -1;
        const bool inPool = slot >= 0 && slot < p.numSlots;
        const int64_t off = inPool && !isQ ? poolOffset(slot, kvh, p.kvHeads, p.blockSize, D) : 0;
        if (isV) {
            T* dst = static_cast<T*>(p.dV) + row * p.dVStride + static_cast<int64_t>(kvh) * D;
            for (int d = lane; d < D; d += 32) dst[d] = inPool ? static_cast<const T*>(p.dVPool)[off + d] : fromFloat<T>(0.f);
            continue;
        }
        const T* src = isQ ? static_cast<const T*>(p.q) + row * p.qStride + static_cast<int64_t>(h) * D
                           : static_cast<const T*>(p.k) + row * p.kStride + static_cast<int64_t>(kvh) * D;
        const T* dy = isQ ? static_cast<const T*>(p.dQOut) + (row * p.heads + h) * static_cast<int64_t>(D)
                    : p.dKOut ? static_cast<const T*>(p.dKOut) + (row * p.kvHeads + kvh) * static_cast<int64_t>(D)
                    : inPool ? static_cast<const T*>(p.dKPool) + off : nullptr;
        const T* weight = static_cast<const T*>(isQ ? p.qWeight : p.kWeight);
        float sum = 0.f, dot = 0.f;
        for (int d = lane; d < D; d += 32) {
            x[d] = toFloat(src[d]);
            sum += x[d] * x[d];
            float dn = dy ? toFloat(dy[d]) : 0.f;
            if (dy && d < p.rotaryDim) {
                const int i = p.interleaved ? d >> 1 : d % half;
                const bool first = p.interleaved ? !(d & 1) : d < half;
                const float z = toFloat(dy[p.interleaved ? d ^ 1 : first ? d + half : d - half]);
                const float2 cs = turnOf(pos, p.invFreq[i]);
                dn = first ? dn * cs.x + z * cs.y : dn * cs.x - z * cs.y;
            }
            g[d] = dn;
            dot += x[d] * dn * toFloat(weight[d]);
        }
        for (int o = 16; o > 0; o >>= 1) {
            sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
            dot += __shfl_xor_sync(0xFFFFFFFFu, dot, o);
        }
        const float r = rsqrtf(sum / static_cast<float>(D) + p.eps), mean = dot * r / static_cast<float>(D);
        T* dst = isQ ? static_cast<T*>(p.dQ) + row * p.dQStride + static_cast<int64_t>(h) * D
                     : static_cast<T*>(p.dK) + row * p.dKStride + static_cast<int64_t>(kvh) * D;
        float* acc = isQ ? accQ : accK;
        __syncwarp();                                 // dst may lie over src or dy: every lane has read its elements
        for (int d = lane; d < D; d += 32) {
            const float xhat = x[d] * r;
            dst[d] = fromFloat<T>(r * (g[d] * toFloat(weight[d]) - xhat * mean));
            acc[d] += g[d] * xhat;
        }
        __syncwarp();
    }
    if (!p.partials) return;
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * D; i += 128) {
        const int which = i / D, d = i % D;
        float t = 0.f;
        for (int w = 0; w < 4; ++w) t += smemAny[static_cast<size_t>(w) * 4 * D + (2 + which) * D + d];
        p.partials[(static_cast<int64_t>(blockIdx.x) * 2 + which) * D + d] = t;
    }
}

// dw = the blocks' partial sums added up in block order (float64: the sum of up to a few
// thousand terms costs nothing here and adds no error of its own).
__global__ void __launch_bounds__(1024)
weightGradientKernel(const float* __restrict__ partials, int blocks, int dim, float* dQWeight, float* dKWeight) {
    __shared__ double part[32][32];
    cudaGridDependencySynchronize();                  // launched early; the partial sums are there from here on
    const int lane = threadIdx.x & 31, slice = threadIdx.x >> 5;
    const int d = blockIdx.x * 32 + lane, which = blockIdx.y;
    double sum = 0.0;
    if (d < dim)
#pragma unroll 4
        for (int b = slice; b < blocks; b += 32) sum += partials[(static_cast<int64_t>(b) * 2 + which) * dim + d];
    part[slice][lane] = sum;
    __syncthreads();
    if (slice == 0 && d < dim) {
        for (int s = 1; s < 32; ++s) sum += part[s][lane];
        float* out = which ? dKWeight : dQWeight;
        if (out) out[d] = static_cast<float>(sum);
    }
}

// Blocks that share the rows: two for every SM, each with a few rows at least.
int backwardBlocks(const NormRotateBackwardParams& p, int smCount) {
    return static_cast<int>(std::min<int64_t>((static_cast<int64_t>(p.numRows) + kBackwardShare - 1) / kBackwardShare, static_cast<int64_t>(smCount) * 2));
}
// Lanes and threads of the launch that the pieces allow (chunks 1, threads 0: the other kernel runs).
template <typename T>
int backwardChunks(const NormRotateBackwardParams& p, Layout* l, int* threads) {
    constexpr int E = Piece<T>::E;
    *threads = 0;
    if (!piecesApply<E>(p.headDim, p.rotaryDim, p.interleaved)) return 1;
    *l = layoutOf<E>(p.headDim, p.rotaryDim, p.interleaved);
    int chunks;
    headChunks(p.heads + (p.dV ? 2 : 1) * p.kvHeads, l->lanes, &chunks, threads);
    return chunks;
}

template <typename T>
cudaError_t normRotateBackwardOf(const NormRotateBackwardParams& p, int smCount, cudaStream_t stream, int* launches) {
    constexpr int E = Piece<T>::E;
    const void* ptrs[] = {p.q, p.k, p.qWeight, p.kWeight, p.dQOut, p.dKOut, p.dKPool, p.dVPool, p.dQ, p.dK, p.dV};
    Layout l{};
    int threads, chunks = backwardChunks<T>(p, &l, &threads);
    bool pieces = threads > 0;
    for (const void* ptr : ptrs) pieces = pieces && aligned16(ptr);
    for (int64_t s : {p.qStride, p.kStride, p.dQStride, p.dKStride, p.dVStride}) pieces = pieces && s % E == 0;
    const int blocks = backwardBlocks(p, smCount);
    if (pieces) {
        const int share = static_cast<int>((static_cast<int64_t>(p.numRows) + blocks - 1) / blocks);
        const size_t smem = static_cast<size_t>(threads) * kBackwardStages * 4 * 16 +
                            kBackwardRows * (sizeof(RowInfo) + (p.rotaryDim / 2) * sizeof(float2));
        // (at most 544 threads, 102 KB of rows, and 33 KB of turns)
        static std::atomic<unsigned long long> done{0};
        const cudaError_t allowed = allowSmem(normRotateBackwardKernel<T>, 160 * 1024, done);
        if (allowed != cudaSuccess) return allowed;
        normRotateBackwardKernel<T><<<dim3(blocks, chunks), threads, smem, stream>>>(p, l, share);
    } else {
        chunks = 1;
        normRotateBackwardAnyKernel<T><<<blocks, 128, static_cast<size_t>(16) * p.headDim * sizeof(float), stream>>>(p);
    }
    *launches += 1;
    cudaError_t e = cudaGetLastError();
    if (e == cudaSuccess && p.partials) {
        cudaLaunchAttribute attr{};
        attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr.val.programmaticStreamSerializationAllowed = 1;
        cudaLaunchConfig_t cfg{};
        cfg.gridDim = dim3((p.headDim + 31) / 32, 2);
        cfg.blockDim = dim3(1024);
        cfg.stream = stream;
        cfg.attrs = &attr;
        cfg.numAttrs = 1;
        e = cudaLaunchKernelEx(&cfg, weightGradientKernel, static_cast<const float*>(p.partials), blocks * chunks, p.headDim, p.dQWeight, p.dKWeight);
        *launches += 1;
    }
    return e;
}

}  // namespace

cudaError_t launchNormRotate(const NormRotateParams& p, int smCount, cudaStream_t stream, int* launches) {
    switch (p.ioType) {
        case kF32: return normRotateOf<float>(p, smCount, stream, launches);
        case kBF16: return normRotateOf<__nv_bfloat16>(p, smCount, stream, launches);
        default: return normRotateOf<__half>(p, smCount, stream, launches);
    }
}

size_t normRotateBackwardWorkspaceBytes(const NormRotateBackwardParams& p, int smCount) {
    if (!p.dQWeight && !p.dKWeight) return 0;
    Layout l{};
    int threads;
    const int chunks = p.ioType == kF32 ? backwardChunks<float>(p, &l, &threads) : backwardChunks<__half>(p, &l, &threads);
    return static_cast<size_t>(backwardBlocks(p, smCount)) * chunks * 2 * p.headDim * sizeof(float);
}

cudaError_t launchNormRotateBackward(const NormRotateBackwardParams& p, int smCount, cudaStream_t stream, int* launches) {
    switch (p.ioType) {
        case kF32: return normRotateBackwardOf<float>(p, smCount, stream, launches);
        case kBF16: return normRotateBackwardOf<__nv_bfloat16>(p, smCount, stream, launches);
        default: return normRotateBackwardOf<__half>(p, smCount, stream, launches);
    }
}

}  // namespace pam
