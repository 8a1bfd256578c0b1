// What the kernels of the tree attention share: how a launch's work is laid out in one list of
// tiles, where partial results go, and which keys a row sees.
//
// A request's rows under one KV head, (node, query head of the group) with the head running
// fastest, are cut into row tiles of MR rows; the keys they can see, the visible tail of the
// cache and then the tree's own rows, into key tiles of KT keys.  A pair (request, KV head, row
// tile) has nT key tiles.  All pairs' tiles are laid end to end and every block takes an equal
// contiguous piece of that list, whatever the lengths: a pair that lies inside one piece is
// finished by its block, a pair that several pieces share gets one record (O, m, l per row,
// float32) per piece, joined in piece order by a second kernel.  A block shares at most two
// pairs (one it continues, one it starts), so that the places of the records are fixed by the
// block's number and nothing is counted or cleared: equal inputs give equal bits, and a captured
// launch can be replayed.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "kernels.h"

namespace pam {
namespace tree {

struct SeqInfo {
    int start, n;            // rows [start, start + n) of the request
    uint32_t len, held, lo;  // tokens in the cache; reachable through the table; first that any row sees
    __device__ __forceinline__ SeqInfo() {}
    __device__ __forceinline__ SeqInfo(const TreeParams& p, int b) {
        start = min(max(p.rowStarts[b], 0), p.numRows);
        const int end = min(max(p.rowStarts[b + 1], start), p.numRows);
        n = min(end - start, p.maxNew);
        len = p.lens[b];
        const unsigned long long reach = static_cast<unsigned long long>(p.maxNumBlocks) * p.blockSize;
        held = static_cast<uint32_t>(min(static_cast<unsigned long long>(len), reach));
        // a row's position is at least len, its window starts at position + 1 - window
        const uint32_t w = static_cast<uint32_t>(p.window);
        lo = w > 0 && len + 1u > w ? min(len + 1u - w, held) : 0u;
    }
    // key tiles of the cache part: tile j holds tokens [(lo / KT + j) * KT, + KT)
    template <int KT> __device__ __forceinline__ int cacheTiles() const {
        return held > lo ? static_cast<int>((held - 1) / KT - lo / KT) + 1 : 0;
    }
    template <int KT> __device__ __forceinline__ int tiles() const { return cacheTiles<KT>() + (n + KT - 1) / KT; }
    __device__ __forceinline__ int rowTiles(int group, int mr) const { return (n * group + mr - 1) / mr; }
};

// bfloat16 keeps 8 bits of a weight, which shows when few keys carry the result: requests that see fewer keys than
// this, and all if the caller wants it so, carry the weights into the second product as two operands (16 bits).
constexpr uint32_t kShortKeys = 256;
__device__ __forceinline__ bool twoOperands(const TreeParams& p, const SeqInfo& s) {
    return p.exactWeights == 2 || (p.exactWeights == 1 && s.held - s.lo + static_cast<uint32_t>(s.n) < kShortKeys);
}

// Position of a row (node i of its tree); one below the cache length counts as the cache length.
__device__ __forceinline__ long long positionOf(const TreeParams& p, const SeqInfo& s, int i) {
    if (!p.positions) return static_cast<long long>(s.len) + i;
    return max(static_cast<long long>(p.positions[s.start + i]), static_cast<long long>(s.len));
}
// First cache token that node i sees.
__device__ __forceinline__ uint32_t firstOf(const TreeParams& p, const SeqInfo& s, int i) {
    if (p.window <= 0) return 0u;
    const long long f = positionOf(p, s, i) + 1 - p.window;
    return f <= 0 ? 0u : f >= s.held ? s.held : static_cast<uint32_t>(f);
}
// Nodes 32 w .. 32 w + 31 that node i sees, as bits (n bounds them; without masks: up to itself).
__device__ __forceinline__ uint32_t treeBits(const TreeParams& p, const SeqInfo& s, int i, int w) {
    uint32_t bits;
    if (p.masks) bits = w < p.maskWords ? p.masks[static_cast<int64_t>(s.start + i) * p.maskWords + w] : 0u;
    else bits = i >= 32 * w + 31 ? 0xFFFFFFFFu : i < 32 * w ? 0u : (2u << (i - 32 * w)) - 1u;
    const int left = s.n - 32 * w;
    if (left <= 0) return 0u;
    if (left < 32) bits &= (1u << left) - 1u;
    if (p.window > 0) {
        const long long me = positionOf(p, s, i);
        for (uint32_t rest = bits; rest; rest &= rest - 1) {
            const int j = 32 * w + __ffs(rest) - 1;
            if (positionOf(p, s, j) <= me - p.window) bits &= ~(1u << (j - 32 * w));
        }
    }
    return bits;
}

// ---- the list of tiles --------------------------------------------------------

// prefix[b] = tiles before request b, for b = 0 .. batch; every block builds it by itself.
// THREADS is a multiple of 32, at most 1024.  `scratch` holds THREADS / 32 ints.
template <int MR, int KT, int THREADS>
__device__ __forceinline__ void buildPrefix(const TreeParams& p, int* prefix, int* scratch) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, group = p.heads / p.kvHeads;
    const int per = (p.batch + THREADS - 1) / THREADS, b0 = tid * per, b1 = min(p.batch, b0 + per);
    int sum = 0;
    for (int b = b0; b < b1; ++b) {
        const SeqInfo s(p, b);
        const int t = p.kvHeads * s.rowTiles(group, MR) * s.tiles<KT>();
        prefix[b + 1] = t;
        sum += t;
    }
    int inc = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xFFFFFFFFu, inc, o);
        if (lane >= o) inc += v;
    }
    if (lane == 31) scratch[warp] = inc;
    __syncthreads();
    int before = inc - sum;
    for (int w = 0; w < warp; ++w) before += scratch[w];
    if (tid == 0) prefix[0] = 0;
    for (int b = b0; b < b1; ++b) {
        before += prefix[b + 1];
        prefix[b + 1] = before;
    }
    __syncthreads();
}

// Part of a pair that lies in one block's piece: key tiles [first, last) of nT.
struct Segment {
    int b, kvh, rt, first, last, nT;
    SeqInfo s;
    __device__ __forceinline__ bool whole() const { return first == 0 && last == nT; }
};
// The segment that starts at tile t of the list, t < end <= prefix[batch].
template <int MR, int KT>
__device__ __forceinline__ Segment segmentAt(const TreeParams& p, const int* prefix, int t, int end) {
    int a = 0, z = p.batch - 1;                        // the last request whose tiles start at or before t
    while (a < z) {
        const int mid = (a + z + 1) >> 1;
        if (prefix[mid] <= t) a = mid; else z = mid - 1;
    }
    Segment g;
    g.b = a;
    g.s = SeqInfo(p, a);
    g.nT = g.s.tiles<KT>();
    const int rel = t - prefix[a], pair = rel / g.nT, rowTiles = g.s.rowTiles(p.heads / p.kvHeads, MR);
    g.first = rel - pair * g.nT;
    g.kvh = pair / rowTiles;
    g.rt = pair - g.kvh * rowTiles;
    g.last = min(g.nT, g.first + (end - t));
    return g;
}

// ---- records --------------------------------------------------------------------

// Written by every block of the attention kernel: the pair whose first record is its own (the
// pair it starts and does not finish), the last block that shares it, and for both of its records
// whether a value that is not a finite number was left out (see leftOut).
struct Header {
    int b, kvh, rt, lastBlock;      // lastBlock < 0: the block starts no shared pair
    int odd[2];                     // record 0: the pair the block continues, 1: the pair it starts
    int pad[2];
};
__host__ __device__ __forceinline__ size_t headerBytes(int blocks) { return (static_cast<size_t>(blocks) * sizeof(Header) + 255) / 256 * 256; }
// A record: O [MR][dimPad], then m [MR], l [MR].
__host__ __device__ __forceinline__ size_t recordFloats(int mr, int dimPad) { return static_cast<size_t>(mr) * (dimPad + 2); }
__device__ __forceinline__ Header* headerOf(const TreeParams& p, int block) { return reinterpret_cast<Header*>(p.workspace) + block; }
__device__ __forceinline__ float* recordOf(const TreeParams& p, int blocks, int block, int which, int mr, int dimPad) {
    return reinterpret_cast<float*>(reinterpret_cast<unsigned char*>(p.workspace) + headerBytes(blocks)) +
           (static_cast<size_t>(block) * 2 + which) * recordFloats(mr, dimPad);
}

// ---- values that are not finite ---------------------------------------------------

// A weight of zero times a value that is infinite or NaN would put NaN into rows that do not
// see the value.  Of the keys that some row of a row tile may not see (the tree's, and the cache
// tokens before the last first token, see lastFirst) the kernels therefore take such values as
// zero and note it; a row that does see one gets the sum of
// the values left out added at the end (its result is infinite or NaN: the weight, which is
// positive, does not matter).
__device__ __forceinline__ bool isOdd(float v) { return !(fabsf(v) <= 3.402823466e38f); }

__device__ __forceinline__ float valueOf(const float* p) { return *p; }
__device__ __forceinline__ float valueOf(const __half* p) { return __half2float(*p); }
__device__ __forceinline__ float valueOf(const __nv_bfloat16* p) { return __bfloat162float(*p); }

__device__ __forceinline__ int64_t poolRow(const TreeParams& p, int b, uint32_t token, int kvh, int64_t* block) {
    const uint32_t page = token / static_cast<uint32_t>(p.blockSize);
    const int64_t blk = min(max(p.tables[static_cast<int64_t>(b) * p.maxNumBlocks + page], 0), p.poolBlocks - 1);
    if (block) *block = blk;
    return ((blk * p.kvHeads + kvh) * p.blockSize + (token - page * p.blockSize)) * static_cast<int64_t>(p.headDim);
}

// The key scale of a page.  One that is not a finite number makes the scores of the rows that see the page NaN
// (infinity times a code may be NaN or an infinity of either sign, by the code: kernels that scale the score
// instead of the codes could not tell).
__device__ __forceinline__ float keyScaleOf(__half scale) {
    const float s = __half2float(scale);
    return isOdd(s) ? __int_as_float(0x7FFFFFFF) : s;
}

// A pool's element; FP8: code times scale, in float32.
template <typename KT_>
__device__ __forceinline__ float poolValue(const TreeParams& p, const void* pool, const void* scale, int64_t at, int64_t blk, int kvh) {
    if constexpr (sizeof(KT_) == 1)
        return __half2float(__half(__nv_cvt_fp8_to_halfraw(static_cast<const uint8_t*>(pool)[at], __NV_E4M3))) *
               __half2float(static_cast<const __half*>(scale)[blk * p.kvHeads + kvh]);
    else
        return valueOf(static_cast<const KT_*>(pool) + at);
}

// First token that every row of a row tile sees (the largest of the rows' first tokens).
__device__ __forceinline__ uint32_t lastFirst(const TreeParams& p, const SeqInfo& s, int rt, int mr) {
    if (p.window <= 0) return 0u;
    const int group = p.heads / p.kvHeads, rows = s.n * group;
    uint32_t hi = 0u;
    for (int i = rt * mr / group; i < s.n && i * group < min(rows, (rt + 1) * mr); ++i) hi = max(hi, firstOf(p, s, i));
    return hi;
}

// The same by a whole warp.
__device__ __forceinline__ uint32_t lastFirstOfWarp(const TreeParams& p, const SeqInfo& s, int rt, int mr) {
    if (p.window <= 0) return 0u;
    const int group = p.heads / p.kvHeads, rows = s.n * group;
    uint32_t hi = 0u;
    for (int i = rt * mr / group + static_cast<int>(threadIdx.x & 31); i < s.n && i * group < min(rows, (rt + 1) * mr); i += 32) hi = max(hi, firstOf(p, s, i));
    return __reduce_max_sync(0xFFFFFFFFu, hi);
}

template <typename T> __device__ __forceinline__ T narrow(float v);
template <> __device__ __forceinline__ float narrow<float>(float v) { return v; }
template <> __device__ __forceinline__ __half narrow<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 narrow<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Adds the values that were taken as zero although node i sees them to columns [d0, d1) of its row
// of the result, which this thread (or its warp, before a __syncwarp) has stored.  hi: the first token
// that every row of the row tile sees.  Behind it only FP8 pages are left out, those whose value scale is not a
// finite number.  A key scale that is not (see keyScaleOf) makes the row NaN here, whatever the kernel took it for.
template <typename QT, typename KT_>
__device__ __noinline__ void addLeftOut(const TreeParams& p, SeqInfo s, int b, int kvh, int i, uint32_t hi, QT* row, int d0, int d1) {
    auto addToken = [&](uint32_t t) {
        int64_t blk;
        const int64_t at = poolRow(p, b, t, kvh, &blk);
        for (int d = d0; d < d1; ++d) {
            const float v = poolValue<KT_>(p, p.vPool, p.vScale, at + d, blk, kvh);
            if (isOdd(v)) row[d] = narrow<QT>(valueOf(row + d) + v);
        }
    };
    const uint32_t from = firstOf(p, s, i);
    if constexpr (sizeof(KT_) == 1) {
        for (uint32_t t = from; t < s.held;) {
            const unsigned long long pageEnd = (static_cast<unsigned long long>(t / p.blockSize) + 1) * p.blockSize;
            const uint32_t end = static_cast<uint32_t>(min(pageEnd, static_cast<unsigned long long>(s.held)));
            int64_t blk;
            poolRow(p, b, t, kvh, &blk);
            const int64_t pair = blk * p.kvHeads + kvh;
            const bool odd = isOdd(__half2float(static_cast<const __half*>(p.vScale)[pair]));
            if (isOdd(__half2float(static_cast<const __half*>(p.kScale)[pair])))
                for (int d = d0; d < d1; ++d) row[d] = narrow<QT>(__int_as_float(0x7FFFFFFF));
            for (; t < (odd ? end : min(end, hi)); ++t) addToken(t);
            t = end;
        }
    } else {
        for (uint32_t t = from; t < hi; ++t) addToken(t);
    }
    for (int w = 0; w * 32 < s.n; ++w)
        for (uint32_t bits = treeBits(p, s, i, w); bits; bits &= bits - 1) {
            const QT* v = static_cast<const QT*>(p.vNew) + static_cast<int64_t>(s.start + 32 * w + __ffs(bits) - 1) * p.vStride + static_cast<int64_t>(kvh) * p.headDim;
            for (int d = d0; d < d1; ++d)
                if (isOdd(valueOf(v + d))) row[d] = narrow<QT>(valueOf(row + d) + valueOf(v + d));
        }
}

}  // namespace tree

// A launch whose blocks may be set up while the kernel before it on the stream still runs: the kernel
// calls cudaGridDependencySynchronize() before it reads or writes anything.
template <typename... Params, typename... Args>
cudaError_t launchEarly(void (*kernel)(Params...), dim3 grid, int threads, size_t smem, cudaStream_t stream, Args... args) {
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

// How a request is launched: the kernel, its tiles, the columns of a record, the blocks.
struct TreePlan {
    int variant;       // 0: treeGeneralKernel, 1: treeMmaKernel, 2: treeTcKernel
    int rows, keys, dimPad, blocks;
};
// Each of the two: whether it takes such sizes and types at all (its workspace is counted then), and
// whether it takes the request, buffers and strides included.
// tree_mma_kernel.cu: 16-bit and FP8 pools, head_dim up to 128, everything on 16 bytes.
bool treeMmaSizes(const TreeParams& p);
bool treeMmaApplies(const TreeParams& p);
TreePlan treeMmaPlan(const TreeParams& p, int smCount);
cudaError_t launchTreeMma(const TreeParams& p, const TreePlan& plan, cudaStream_t stream);
// tree_tc_kernel.cu: 16-bit and FP8 pools, head_dim 64, 80, ... 128, block sizes that are multiples of 8 (FP8: 16).
bool treeTcSizes(const TreeParams& p);
bool treeTcApplies(const TreeParams& p);
TreePlan treeTcPlan(const TreeParams& p, int smCount);
cudaError_t launchTreeTc(const TreeParams& p, const TreePlan& plan, cudaStream_t stream);

}  // namespace pam
