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

#include "kernels.h"

namespace pam {
namespace {

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

// E elements of 16 bytes: 8 of a 16-bit type, 4 of float32.
template <typename T>
struct Piece {
    static constexpr int E = 16 / sizeof(T);
    uint4 raw;
    __device__ __forceinline__ void load(const T* p) { raw = *reinterpret_cast<const uint4*>(p); }
    __device__ __forceinline__ void store(T* p) const { *reinterpret_cast<uint4*>(p) = raw; }
    __device__ __forceinline__ void unpack(float (&f)[E]) const {
        const T* t = reinterpret_cast<const T*>(&raw);
#pragma unroll
        for (int e = 0; e < E; ++e) f[e] = toFloat(t[e]);
    }
    __device__ __forceinline__ void pack(const float (&f)[E]) {
        T* t = reinterpret_cast<T*>(&raw);
#pragma unroll
        for (int e = 0; e < E; ++e) t[e] = fromFloat<T>(f[e]);
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

template <typename T>
Layout layoutOf(int headDim, int rotaryDim, int interleaved) {
    constexpr int E = Piece<T>::E;
    Layout l{};
    l.pieces = headDim / E;
    l.pairs = interleaved ? (rotaryDim / E + 1) / 2 : rotaryDim / (2 * E);
    l.half = interleaved ? 0 : l.pairs;
    const int need = (l.pieces + 1) / 2;
    for (l.lanes = 1; l.lanes < need; l.lanes *= 2) {}
    return l;
}

// Elements [first, first + E) of a piece and their index in the head: the turn of element d.
// `cs` holds (cos, sin) of the row's rotaryDim / 2 angles.
template <int E>
__device__ __forceinline__ void rotateHalves(float (&x)[E], float (&y)[E], const float2* cs, float sign) {
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const float2 t = cs[e];
        const float s = sign * t.y, a = x[e], b = y[e];
        x[e] = a * t.x - b * s;
        y[e] = b * t.x + a * s;
    }
}
template <int E>
__device__ __forceinline__ void rotatePairs(float (&x)[E], const float2* cs, float sign) {
#pragma unroll
    for (int e = 0; e < E; e += 2) {
        const float2 t = cs[e / 2];
        const float s = sign * t.y, a = x[e], b = x[e + 1];
        x[e] = a * t.x - b * s;
        x[e + 1] = b * t.x + a * s;
    }
}

// Address of a slot's row in a pool [block][kvHeads][blockSize][dim], element offset.
__device__ __forceinline__ int64_t poolOffset(int64_t slot, int kvh, int kvHeads, int blockSize, int dim) {
    const int64_t blk = slot / blockSize, off = slot - blk * blockSize;
    return ((blk * kvHeads + kvh) * blockSize + off) * static_cast<int64_t>(dim);
}

// ---- forward ----------------------------------------------------------------

// A block takes `rowsPer` rows: first the turns of the rows' angles into shared memory, then
// every group of l.lanes lanes takes one (row, head) of queries, keys and values after the other.
template <typename T>
__global__ void __launch_bounds__(512)
normRotateKernel(const NormRotateParams p, const Layout l, int rowsPer) {
    constexpr int E = Piece<T>::E;
    extern __shared__ float2 turns[];                 // [rowsPer][rotaryDim / 2]
    const int tid = threadIdx.x, half = p.rotaryDim / 2;
    const int64_t row0 = static_cast<int64_t>(blockIdx.x) * rowsPer;
    for (int i = tid; i < rowsPer * half; i += blockDim.x) {
        const int64_t row = row0 + i / half;
        const int pos = row < p.numRows ? p.positions[row] : -1;
        if (pos >= 0) turns[i] = turnOf(pos, p.invFreq[i % half]);
    }
    if (p.slotsOut && tid < rowsPer && row0 + tid < p.numRows)
        p.slotsOut[row0 + tid] = p.positions[row0 + tid] >= 0 ? p.slots[row0 + tid] : -1;
    __syncthreads();
    const int lane = tid % l.lanes, group = tid / l.lanes, groups = blockDim.x / l.lanes;
    const int perRow = p.heads + 2 * p.kvHeads;       // queries, keys, values
    int pa, pb;
    l.lane(lane, pa, pb);
    const bool hasA = pa < l.pieces, hasB = pb < l.pieces;
    // whole warps stay in the loop for the shuffles
    const int total = rowsPer * perRow, rounds = (total + groups - 1) / groups;
    for (int it = 0; it < rounds; ++it) {
        const int w = it * groups + group;
        const int64_t row = row0 + w / perRow;
        const int h = w % perRow;
        const bool live = w < total && row < p.numRows && p.positions[row] >= 0;
        const bool isQ = h < p.heads, isV = h >= p.heads + p.kvHeads;
        const int kvh = isQ ? 0 : isV ? h - p.heads - p.kvHeads : h - p.heads;
        const T* src = nullptr;
        if (live) {
            if (isQ) src = static_cast<const T*>(p.q) + row * p.qStride + static_cast<int64_t>(h) * p.headDim;
            else if (!isV) src = static_cast<const T*>(p.k) + row * p.kStride + static_cast<int64_t>(kvh) * p.headDim;
            else if (p.vPool || p.vOut) src = static_cast<const T*>(p.v) + row * p.vStride + static_cast<int64_t>(kvh) * p.headDim;
        }
        Piece<T> a{}, b{};
        if (src && hasA) a.load(src + pa * E);
        if (src && hasB) b.load(src + pb * E);
        float fa[E], fb[E];
        a.unpack(fa);
        b.unpack(fb);
        float sum = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) sum += fa[e] * fa[e] + fb[e] * fb[e];
        for (int o = l.lanes >> 1; o > 0; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
        if (!src || !hasA) continue;                  // (no shuffle below)
        if (!isV) {
            const float r = rsqrtf(sum / static_cast<float>(p.headDim) + p.eps);
            const T* weight = static_cast<const T*>(isQ ? p.qWeight : p.kWeight);
            Piece<T> wa{}, wb{};
            wa.load(weight + pa * E);
            if (hasB) wb.load(weight + pb * E);
            float ga[E], gb[E];
            wa.unpack(ga);
            wb.unpack(gb);
#pragma unroll
            for (int e = 0; e < E; ++e) { fa[e] *= r * ga[e]; fb[e] *= r * gb[e]; }
            const float2* cs = turns + (w / perRow) * half;
            if (l.half) {
                if (lane < l.pairs) rotateHalves<E>(fa, fb, cs + pa * E, 1.f);
            } else {
                if (pa * E < p.rotaryDim) rotatePairs<E>(fa, cs + pa * E / 2, 1.f);
                if (pb * E < p.rotaryDim) rotatePairs<E>(fb, cs + pb * E / 2, 1.f);
            }
            a.pack(fa);
            b.pack(fb);
        }
        T* dst[2] = {nullptr, nullptr};
        if (isQ) dst[0] = static_cast<T*>(p.qOut) + row * p.qOutStride + static_cast<int64_t>(h) * p.headDim;
        else {
            void* rows = isV ? p.vOut : p.kOut;
            void* pool = isV ? p.vPool : p.kPool;
            if (rows) dst[0] = static_cast<T*>(rows) + row * (isV ? p.vOutStride : p.kOutStride) + static_cast<int64_t>(kvh) * p.headDim;
            if (pool) {
                const int64_t slot = p.slots[row];
                if (slot >= 0 && slot < p.numSlots)
                    dst[1] = static_cast<T*>(pool) + poolOffset(slot, kvh, p.kvHeads, p.blockSize, p.headDim);
            }
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            if (!dst[i]) continue;
            a.store(dst[i] + pa * E);
            if (hasB) b.store(dst[i] + pb * E);
        }
    }
}

constexpr int kMaxDim = 256;

// Any head_dim, rotaryDim and alignment: one warp per (row, head), element by element, the row
// in shared memory so that outputs may lie over the inputs.
template <typename T>
__global__ void __launch_bounds__(128)
normRotateAnyKernel(const NormRotateParams p) {
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
        if (isV && !p.vPool && !p.vOut) continue;
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
            void* rows = isV ? p.vOut : p.kOut;
            void* pool = isV ? p.vPool : p.kPool;
            if (rows) dst[0] = static_cast<T*>(rows) + row * (isV ? p.vOutStride : p.kOutStride) + static_cast<int64_t>(kvh) * p.headDim;
            if (pool) {
                const int64_t slot = p.slots[row];
                if (slot >= 0 && slot < p.numSlots)
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
template <typename T>
bool piecesApply(int headDim, int rotaryDim, int interleaved) {
    constexpr int E = Piece<T>::E;
    if (headDim % E || headDim / E > 64) return false;
    return interleaved ? rotaryDim % E == 0 : rotaryDim % (2 * E) == 0;
}

template <typename T>
cudaError_t normRotateOf(const NormRotateParams& p, cudaStream_t stream, int* launches) {
    constexpr int E = Piece<T>::E;
    const void* ptrs[] = {p.q, p.k, p.v, p.qWeight, p.kWeight, p.qOut, p.kOut, p.vOut, p.kPool, p.vPool};
    bool pieces = piecesApply<T>(p.headDim, p.rotaryDim, p.interleaved);
    for (const void* ptr : ptrs) pieces = pieces && aligned16(ptr);
    for (int64_t s : {p.qStride, p.kStride, p.vStride, p.qOutStride, p.kOutStride, p.vOutStride}) pieces = pieces && s % E == 0;
    const int perRow = p.heads + 2 * p.kvHeads;
    if (!pieces) {
        const int64_t warps = static_cast<int64_t>(p.numRows) * perRow;
        normRotateAnyKernel<T><<<static_cast<unsigned>(std::min<int64_t>((warps + 3) / 4, 148 * 16)), 128, 0, stream>>>(p);
    } else {
        const Layout l = layoutOf<T>(p.headDim, p.rotaryDim, p.interleaved);
        const int rowLanes = perRow * l.lanes;
        const int threads = std::min(512, (rowLanes + 31) / 32 * 32);
        // short rows share a block, as far as their angles fit
        const int rowsPer = std::max(1, std::min(256 / std::max(rowLanes, 1), 64));
        const int block = rowsPer > 1 ? 256 : threads;
        const size_t smem = static_cast<size_t>(rowsPer) * (p.rotaryDim / 2) * sizeof(float2);
        const int64_t grid = (static_cast<int64_t>(p.numRows) + rowsPer - 1) / rowsPer;
        normRotateKernel<T><<<static_cast<unsigned>(grid), block, smem, stream>>>(p, l, rowsPer);
    }
    *launches += 1;
    return cudaGetLastError();
}

// ---- backward ---------------------------------------------------------------

constexpr int kBackwardThreads = 256;

// The rows are dealt to the blocks round robin.  A thread always holds the same pieces of a head,
// so that its share of the weight gradients stays in registers over all its rows; at the end the
// block's groups are summed through shared memory in a fixed order and the block writes its
// [2][dim] partial sums: no atomics, the same bits for the same grid.
template <typename T>
__global__ void __launch_bounds__(kBackwardThreads)
normRotateBackwardKernel(const NormRotateBackwardParams p, const Layout l) {
    constexpr int E = Piece<T>::E;
    extern __shared__ float2 turns[];                 // [rotaryDim / 2], then floats [groups][2 E lanes]
    const int tid = threadIdx.x, half = p.rotaryDim / 2;
    const int lane = tid % l.lanes, group = tid / l.lanes, groups = kBackwardThreads / l.lanes;
    const int perRow = p.heads + p.kvHeads + (p.dV ? p.kvHeads : 0);
    const int rounds = (perRow + groups - 1) / groups;
    int pa, pb;
    l.lane(lane, pa, pb);
    const bool hasA = pa < l.pieces, hasB = pb < l.pieces;
    float accQ[2 * E], accK[2 * E];
#pragma unroll
    for (int e = 0; e < 2 * E; ++e) accQ[e] = accK[e] = 0.f;
    const float invDim = 1.f / static_cast<float>(p.headDim);
    for (int64_t row = blockIdx.x; row < p.numRows; row += gridDim.x) {
        const int pos = p.positions[row];
        if (pos < 0) continue;                        // the same for the whole block
        __syncthreads();
        for (int i = tid; i < half; i += kBackwardThreads) turns[i] = turnOf(pos, p.invFreq[i]);
        __syncthreads();
        const int64_t slot = p.slots ? p.slots[row] : -1;
        const bool inPool = slot >= 0 && slot < p.numSlots;
        for (int it = 0; it < rounds; ++it) {
            const int h = it * groups + group;
            const bool isQ = h < p.heads, isV = h >= p.heads + p.kvHeads, live = h < perRow;
            const int kvh = isQ ? 0 : isV ? h - p.heads - p.kvHeads : h - p.heads;
            const T *x = nullptr, *dy = nullptr;
            T* dst = nullptr;
            if (live && isQ) {
                x = static_cast<const T*>(p.q) + row * p.qStride + static_cast<int64_t>(h) * p.headDim;
                dy = static_cast<const T*>(p.dQOut) + (row * p.heads + h) * static_cast<int64_t>(p.headDim);
                dst = static_cast<T*>(p.dQ) + row * p.dQStride + static_cast<int64_t>(h) * p.headDim;
            } else if (live && !isV) {
                x = static_cast<const T*>(p.k) + row * p.kStride + static_cast<int64_t>(kvh) * p.headDim;
                if (p.dKOut) dy = static_cast<const T*>(p.dKOut) + (row * p.kvHeads + kvh) * static_cast<int64_t>(p.headDim);
                else if (inPool) dy = static_cast<const T*>(p.dKPool) + poolOffset(slot, kvh, p.kvHeads, p.blockSize, p.headDim);
                dst = static_cast<T*>(p.dK) + row * p.dKStride + static_cast<int64_t>(kvh) * p.headDim;
            } else if (live) {
                if (inPool) dy = static_cast<const T*>(p.dVPool) + poolOffset(slot, kvh, p.kvHeads, p.blockSize, p.headDim);
                dst = static_cast<T*>(p.dV) + row * p.dVStride + static_cast<int64_t>(kvh) * p.headDim;
            }
            Piece<T> xa{}, xb{}, ya{}, yb{};
            if (x && hasA) xa.load(x + pa * E);
            if (x && hasB) xb.load(x + pb * E);
            if (dy && hasA) ya.load(dy + pa * E);
            if (dy && hasB) yb.load(dy + pb * E);
            if (isV) {                                // (a group's lanes agree; the shuffles below name them alone)
                if (dst && hasA) ya.store(dst + pa * E);
                if (dst && hasB) yb.store(dst + pb * E);
            }
            float fa[E], fb[E], ga[E], gb[E];
            xa.unpack(fa); xb.unpack(fb);
            ya.unpack(ga); yb.unpack(gb);
            if (l.half) {
                if (lane < l.pairs) rotateHalves<E>(ga, gb, turns + pa * E, -1.f);
            } else {
                if (pa * E < p.rotaryDim) rotatePairs<E>(ga, turns + pa * E / 2, -1.f);
                if (pb * E < p.rotaryDim) rotatePairs<E>(gb, turns + pb * E / 2, -1.f);
            }
            const T* weight = static_cast<const T*>(isQ ? p.qWeight : p.kWeight);
            Piece<T> wa{}, wb{};
            if (hasA) wa.load(weight + pa * E);
            if (hasB) wb.load(weight + pb * E);
            float va[E], vb[E];
            wa.unpack(va); wb.unpack(vb);
            float sum = 0.f, dot = 0.f;               // of x^2, and of x * g
#pragma unroll
            for (int e = 0; e < E; ++e) {
                sum += fa[e] * fa[e] + fb[e] * fb[e];
                dot += fa[e] * ga[e] * va[e] + fb[e] * gb[e] * vb[e];
            }
            for (int o = l.lanes >> 1; o > 0; o >>= 1) {
                sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
                dot += __shfl_xor_sync(0xFFFFFFFFu, dot, o);
            }
            if (!live || isV || !hasA) continue;      // (no shuffle below)
            const float r = rsqrtf(sum * invDim + p.eps);
            const float mean = dot * r * invDim;      // of xhat * g
            float ha[E], hb[E];
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const float xa_ = fa[e] * r, xb_ = fb[e] * r;
                ha[e] = r * (ga[e] * va[e] - xa_ * mean);
                hb[e] = r * (gb[e] * vb[e] - xb_ * mean);
                if (isQ) {
                    accQ[e] += ga[e] * xa_;
                    accQ[E + e] += gb[e] * xb_;
                } else {
                    accK[e] += ga[e] * xa_;
                    accK[E + e] += gb[e] * xb_;
                }
            }
            xa.pack(ha);
            xb.pack(hb);
            xa.store(dst + pa * E);
            if (hasB) xb.store(dst + pb * E);
        }
    }
    if (!p.partials) return;
    float* sums = reinterpret_cast<float*>(turns + half + (half & 1));
    const int width = 2 * E * l.lanes;                // floats of a group
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        __syncthreads();
#pragma unroll
        for (int e = 0; e < 2 * E; ++e) sums[group * width + lane * 2 * E + e] = which ? accK[e] : accQ[e];
        __syncthreads();
        for (int i = tid; i < width; i += kBackwardThreads) {
            int a, b;
            l.lane(i / (2 * E), a, b);
            const int e = i % (2 * E), piece = e < E ? a : b;
            if (piece >= l.pieces) continue;
            float total = 0.f;
            for (int g = 0; g < groups; ++g) total += sums[g * width + i];
            p.partials[(static_cast<int64_t>(blockIdx.x) * 2 + which) * p.headDim + piece * E + e % E] = total;
        }
    }
}

// Any shape and alignment, one warp per (row, head) at a time: the warp's share of the weight
// gradients is added up in shared memory, each element by the lane that owns it.
template <typename T>
__global__ void __launch_bounds__(128)
normRotateBackwardAnyKernel(const NormRotateBackwardParams p) {
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
__global__ void __launch_bounds__(256)
weightGradientKernel(const float* __restrict__ partials, int blocks, int dim, float* dQWeight, float* dKWeight) {
    __shared__ double part[8][32];
    const int lane = threadIdx.x & 31, slice = threadIdx.x >> 5;
    const int d = blockIdx.x * 32 + lane, which = blockIdx.y;
    double sum = 0.0;
    if (d < dim)
        for (int b = slice; b < blocks; b += 8) sum += partials[(static_cast<int64_t>(b) * 2 + which) * dim + d];
    part[slice][lane] = sum;
    __syncthreads();
    if (slice == 0 && d < dim) {
        for (int s = 1; s < 8; ++s) sum += part[s][lane];
        float* out = which ? dKWeight : dQWeight;
        if (out) out[d] = static_cast<float>(sum);
    }
}

int backwardBlocks(const NormRotateBackwardParams& p, int smCount) {
    return static_cast<int>(std::min<int64_t>(p.numRows, static_cast<int64_t>(smCount) * 4));
}

template <typename T>
cudaError_t normRotateBackwardOf(const NormRotateBackwardParams& p, int smCount, cudaStream_t stream, int* launches) {
    constexpr int E = Piece<T>::E;
    const void* ptrs[] = {p.q, p.k, p.qWeight, p.kWeight, p.dQOut, p.dKOut, p.dKPool, p.dVPool, p.dQ, p.dK, p.dV};
    bool pieces = piecesApply<T>(p.headDim, p.rotaryDim, p.interleaved);
    for (const void* ptr : ptrs) pieces = pieces && aligned16(ptr);
    for (int64_t s : {p.qStride, p.kStride, p.dQStride, p.dKStride, p.dVStride}) pieces = pieces && s % E == 0;
    const int blocks = backwardBlocks(p, smCount);
    if (pieces) {
        const Layout l = layoutOf<T>(p.headDim, p.rotaryDim, p.interleaved);
        const int half = p.rotaryDim / 2;
        const size_t smem = (half + (half & 1)) * sizeof(float2) + (p.partials ? kBackwardThreads * 2 * E * sizeof(float) : 0);
        normRotateBackwardKernel<T><<<blocks, kBackwardThreads, smem, stream>>>(p, l);
    } else {
        normRotateBackwardAnyKernel<T><<<blocks, 128, static_cast<size_t>(16) * p.headDim * sizeof(float), stream>>>(p);
    }
    *launches += 1;
    cudaError_t e = cudaGetLastError();
    if (e == cudaSuccess && p.partials) {
        weightGradientKernel<<<dim3((p.headDim + 31) / 32, 2), 256, 0, stream>>>(p.partials, blocks, p.headDim, p.dQWeight, p.dKWeight);
        *launches += 1;
        e = cudaGetLastError();
    }
    return e;
}

}  // namespace

cudaError_t launchNormRotate(const NormRotateParams& p, cudaStream_t stream, int* launches) {
    switch (p.ioType) {
        case kF32: return normRotateOf<float>(p, stream, launches);
        case kBF16: return normRotateOf<__nv_bfloat16>(p, stream, launches);
        default: return normRotateOf<__half>(p, stream, launches);
    }
}

size_t normRotateBackwardWorkspaceBytes(const NormRotateBackwardParams& p, int smCount) {
    if (!p.dQWeight && !p.dKWeight) return 0;
    return static_cast<size_t>(backwardBlocks(p, smCount)) * 2 * p.headDim * sizeof(float);
}

cudaError_t launchNormRotateBackward(const NormRotateBackwardParams& p, int smCount, cudaStream_t stream, int* launches) {
    switch (p.ioType) {
        case kF32: return normRotateBackwardOf<float>(p, smCount, stream, launches);
        case kBF16: return normRotateBackwardOf<__nv_bfloat16>(p, smCount, stream, launches);
        default: return normRotateBackwardOf<__half>(p, smCount, stream, launches);
    }
}

}  // namespace pam
