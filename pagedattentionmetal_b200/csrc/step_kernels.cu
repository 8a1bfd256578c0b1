// The integer work around a speculative step: what a scheduler hands to the kernels of the
// step (row starts, positions, slots, block tables, ancestor masks), and what the tokens of
// the target model make of the drafted trees (accepted path, slots, next token).
//
// Both kernels move a few hundred KB at most and are bound by latency: one launch each, every
// block derives what it needs of the other requests by itself, no intermediate goes through
// memory, nothing is synchronised between blocks.  Measured call after call: the plan of 256 requests
// with one new token 5.0 us, of 64 trees of up to 64 nodes, masks included, 6.5 to 7.5 us; acceptance of 8 trees
// of up to 16 nodes 5.0 to 5.6 us, of 256 of up to 64 nodes 6.1 us.  A launch and the checks before it
// take about 5 us of a processor; what a step of kernels in a graph pays is less.
#include <algorithm>

#include "kernels.h"

namespace pam {
namespace {

constexpr int kPlanThreads = 256;
constexpr int kPlanChunk = 2048;      // rows and table columns of a request that one block takes

__device__ __forceinline__ long long warpSum(long long v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
    return v;
}

__device__ __forceinline__ int newOf(const StepPlanParams& p, int b) { return min(max(p.newTokens[b], 0), p.maxNew); }

// A parent has to come before its child; anything else counts as "no parent".
__device__ __forceinline__ int parentOf(int parent, int i) { return parent >= 0 && parent < i ? parent : -1; }

// Block (b, chunk): request b's entries [chunk * kPlanChunk, + kPlanChunk) of its table and of
// its rows, and a share of the rows behind the last request.  The row start of a request is the
// sum of the new tokens before it: every block adds the (at most a few thousand) counts up
// itself, which costs one pass over an L2-resident array and saves a second launch.
__global__ void __launch_bounds__(kPlanThreads)
planStepKernel(const StepPlanParams p) {
    __shared__ long long part[2][kPlanThreads / 32];
    __shared__ int par[kMaxTreeNodes];
    const int b = blockIdx.x, chunk = blockIdx.y, tid = threadIdx.x;
    long long before = 0, all = 0;
    for (int i = tid; i < p.batch; i += kPlanThreads) {
        const int n = newOf(p, i);
        all += n;
        if (i < b) before += n;
    }
    before = warpSum(before);
    all = warpSum(all);
    if ((tid & 31) == 0) { part[0][tid >> 5] = before; part[1][tid >> 5] = all; }
    __syncthreads();
    before = all = 0;
#pragma unroll
    for (int i = 0; i < kPlanThreads / 32; ++i) { before += part[0][i]; all += part[1][i]; }
    const int start = static_cast<int>(min(before, static_cast<long long>(p.numRows)));
    const int end = static_cast<int>(min(before + newOf(p, b), static_cast<long long>(p.numRows)));
    const int rowsUsed = static_cast<int>(min(all, static_cast<long long>(p.numRows)));
    const int n = end - start, len = max(p.lengths[b], 0);
    const long long total = static_cast<long long>(len) + n;
    const int idx = p.listIndex ? p.listIndex[b] : b;
    // a list index outside the array is an empty list
    const int stride = idx >= 0 && idx < p.numLists ? p.listStride : 0;
    const int32_t* list = p.lists + static_cast<int64_t>(stride ? idx : 0) * p.listStride;
    if (chunk == 0 && tid == 0) {
        if (p.rowStarts) {
            p.rowStarts[b] = start;
            if (b == p.batch - 1) p.rowStarts[p.batch] = end;
        }
        if (p.totalLengths) p.totalLengths[b] = static_cast<uint32_t>(total);
    }
    if (p.tables) {
        const long long used = min((total + p.blockSize - 1) / p.blockSize, static_cast<long long>(stride));
        const int hi = min(p.maxNumBlocks, (chunk + 1) * kPlanChunk);
        int32_t* row = p.tables + static_cast<int64_t>(b) * p.maxNumBlocks;
        for (int j = chunk * kPlanChunk + tid; j < hi; j += kPlanThreads) row[j] = j < used ? list[j] : 0;
    }
    const int lo = chunk * kPlanChunk, hi = min(n, lo + kPlanChunk);
    if (p.parents && lo < hi) {                       // a tree has at most kMaxTreeNodes rows: chunk 0 has them all
        for (int i = tid; i < n; i += kPlanThreads) par[i] = parentOf(p.parents[start + i], i);
        __syncthreads();
    }
    for (int i = lo + tid; i < hi; i += kPlanThreads) {
        int depth = i;
        if (p.parents) {
            depth = 0;
            uint32_t* mask = p.masks ? p.masks + static_cast<int64_t>(start + i) * p.maskWords : nullptr;
            // up the tree; ancestors come in falling order, so that a word is complete when the
            // walk leaves it
            int word = p.maskWords - 1;
            uint32_t bits = 0;
            for (int j = i; j >= 0; j = par[j]) {
                if (mask) {
                    while (word > j >> 5) { mask[word--] = bits; bits = 0; }
                    bits |= 1u << (j & 31);
                }
                depth += j != i;
            }
            if (mask)
                while (word >= 0) { mask[word--] = bits; bits = 0; }
        } else if (p.masks) {
            uint32_t* mask = p.masks + static_cast<int64_t>(start + i) * p.maskWords;
            for (int w = 0; w < p.maskWords; ++w)
                mask[w] = i >= 32 * w + 31 ? 0xFFFFFFFFu : i < 32 * w ? 0u : (2u << (i - 32 * w)) - 1u;
        }
        const long long pos = static_cast<long long>(len) + depth;
        if (p.positions) p.positions[start + i] = static_cast<int32_t>(pos);
        if (p.slots) {
            const long long page = pos / p.blockSize;
            const int block = page < stride ? list[page] : -1;
            p.slots[start + i] = block >= 0 ? static_cast<int64_t>(block) * p.blockSize + pos % p.blockSize : -1;
        }
    }
    // rows behind the last request: position and slot -1, nothing visible
    const int blocks = gridDim.x * gridDim.y, me = chunk * gridDim.x + b;
    for (int64_t r = rowsUsed + static_cast<int64_t>(me) * kPlanThreads + tid; r < p.numRows; r += static_cast<int64_t>(blocks) * kPlanThreads) {
        if (p.positions) p.positions[r] = -1;
        if (p.slots) p.slots[r] = -1;
        if (p.masks)
            for (int w = 0; w < p.maskWords; ++w) p.masks[r * p.maskWords + w] = 0;
    }
}

// One block per request.  A node is accepted when it has no parent, or its parent is accepted
// and the target model's token at the parent is the drafted one.  Every thread walks from its
// node to the root (the depth of the tree in steps, out of shared memory); the deepest accepted
// node, the lowest index among equals, is the largest key (depth, -index).
__global__ void __launch_bounds__(256)
acceptTreeKernel(const AcceptParams p) {
    __shared__ int par[kMaxTreeNodes];            // parent; bit 30 set: the node's token disagrees with its parent's target
    __shared__ int rank[kMaxTreeNodes];           // place on the accepted path, or -1
    __shared__ unsigned best;
    const int b = blockIdx.x, tid = threadIdx.x, threads = blockDim.x;
    const int start = min(max(p.rowStarts[b], 0), p.numRows);
    const int end = min(max(p.rowStarts[b + 1], start), p.numRows);
    const int n = min(end - start, p.maxTree);
    const int len = max(p.lengths[b], 0);         // (read by all before the barriers: newLengths may lie over lengths)
    constexpr int kDisagrees = 1 << 30;
    if (tid == 0) best = 0;
    for (int i = tid; i < n; i += threads) {
        const int up = parentOf(p.parents[start + i], i);
        const bool agrees = up < 0 || p.draft[start + i] == p.target[start + up];
        par[i] = up < 0 ? -1 : up | (agrees ? 0 : kDisagrees);
        rank[i] = -1;
    }
    __syncthreads();
    unsigned mine = 0;
    for (int i = tid; i < n; i += threads) {
        int depth = 0, j = par[i];
        bool ok = true;
        while (j >= 0) {
            ok = ok && !(j & kDisagrees);
            j = par[j & ~kDisagrees];
            ++depth;
        }
        if (ok) mine = max(mine, (static_cast<unsigned>(depth + 1) << 11) | static_cast<unsigned>(kMaxTreeNodes - 1 - i));
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mine = max(mine, __shfl_xor_sync(0xFFFFFFFFu, mine, o));
    if ((tid & 31) == 0 && mine) atomicMax(&best, mine);          // (integers: the order does not matter)
    __syncthreads();
    const int count = static_cast<int>(best >> 11);
    const int node = count ? kMaxTreeNodes - 1 - static_cast<int>(best & 2047u) : 0;
    if (tid == 0) {
        int j = node;
        for (int d = count - 1; d >= 0; --d) {
            rank[j] = d;
            j = par[j];
        }
        if (p.counts) p.counts[b] = count;
        if (p.next) p.next[b] = count ? p.target[start + node] : -1;
        if (p.newLengths) p.newLengths[b] = static_cast<uint32_t>(len + count);
    }
    __syncthreads();
    if (p.path) {
        int32_t* path = p.path + static_cast<int64_t>(b) * p.maxPath;
        for (int d = count + tid; d < p.maxPath; d += threads) path[d] = -1;
        for (int i = tid; i < n; i += threads)
            if (rank[i] >= 0 && rank[i] < p.maxPath) path[rank[i]] = start + i;
    }
    if (p.slots) {
        const int32_t* table = p.tables + static_cast<int64_t>(b) * p.maxNumBlocks;
        for (int i = tid; i < end - start; i += threads) {
            int64_t slot = -1;
            if (i < n && rank[i] >= 0) {
                const long long pos = static_cast<long long>(len) + rank[i], page = pos / p.blockSize;
                const int block = page < p.maxNumBlocks ? table[page] : -1;
                if (block >= 0) slot = static_cast<int64_t>(block) * p.blockSize + pos % p.blockSize;
            }
            p.slots[start + i] = slot;
        }
        // rows outside every tree
        const int first = min(max(p.rowStarts[0], 0), p.numRows), last = min(max(p.rowStarts[p.batch], 0), p.numRows);
        const int64_t stride = static_cast<int64_t>(gridDim.x) * threads, me = static_cast<int64_t>(b) * threads + tid;
        for (int64_t r = me; r < first; r += stride) p.slots[r] = -1;
        for (int64_t r = last + me; r < p.numRows; r += stride) p.slots[r] = -1;
    }
}

}  // namespace

cudaError_t launchPlanStep(const StepPlanParams& p, cudaStream_t stream, int* launches) {
    const int widest = std::max(p.tables ? p.maxNumBlocks : 1, p.maxNew);
    const dim3 grid(static_cast<unsigned>(p.batch), static_cast<unsigned>((static_cast<int64_t>(widest) + kPlanChunk - 1) / kPlanChunk));
    planStepKernel<<<grid, kPlanThreads, 0, stream>>>(p);
    *launches += 1;
    return cudaGetLastError();
}

cudaError_t launchAcceptTree(const AcceptParams& p, cudaStream_t stream, int* launches) {
    const int threads = std::min(256, (p.maxTree + 31) / 32 * 32);
    acceptTreeKernel<<<static_cast<unsigned>(p.batch), threads, 0, stream>>>(p);
    *launches += 1;
    return cudaGetLastError();
}

}  // namespace pam
