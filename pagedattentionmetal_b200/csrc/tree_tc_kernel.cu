// Tree attention on the 5th-generation tensor cores: float16, bfloat16 and FP8 pools, head_dim 64, 80,
// ... 128, block sizes that are multiples of 8 (FP8: 16).  S = Q K^T and O += P V as tcgen05.mma
// 128 x 128 x 16 with S, P and O in tensor memory, one softmax thread per row, keys and values by TMA
// straight from the pages.  The work is few rows (node, query head) against a long cache, so that the
// keys are what is cut up: every block takes an equal piece of the launch's list of key tiles
// (tree_common.cuh) and leaves the parts of pairs that it shares as records.
//
// A pair is a request's up to 256 rows under one KV head.  With more than 128 rows both softmax groups
// work on every key tile, each on 128 rows, and the tile is fetched once for both (a tile counts as
// two in the list).  With at most 128 rows the groups take the key tiles in turn, each with its own
// running maximum, sum and accumulator, and the output warps join the two: the tensor pipe and the
// loads then work for one group while the other is in its softmax, as with two row tiles.
//
//   warps 0-3, 4-7   softmax groups: thread t owns row t of the group's rows.  In tiles with keys
//                    that are not there or that only some rows see it also clears row t of V.
//   warps 8, 9       TMA producers of K (tiles) and V (half tiles: a stage is free again after half
//                    a P V product): pages in pieces of 16 or 8 rows, or boxes of the step's own keys and
//                    values for a tile of the tree.  FP8: warp 8 alone, codes by bulk copies.
//   warp 11          walks the list and leaves the block's spans (its parts of pairs) in a ring in
//                    shared memory, a few ahead of the warps that work on them: a step of that walk is
//                    some loads and divisions in a row, a microsecond that nobody else waits for.
//   warp 10          issues the products, S products up to two steps ahead of the P V product that waits
//                    for its weights.
//   warps 12-15      outputs and records: thread t owns row t, out of tensor memory.  Before that they
//                    bring the queries of the next span into shared memory, once the span's last S product
//                    is complete: boxes where the group divides 128, else row by row.
//   warps 16-19      FP8 only: codes to float16, which holds every e4m3 value, in the swizzled layout of
//                    the operands.  The key scale multiplies the scores; the value scale the weights, with
//                    the running maximum over score plus logarithm of the value scale, so that the weights
//                    that go into the second product as float16 stay near 1 however small the scales are.
//
// Two forms: when no request of the launch can have more than 128 rows under a KV head there is one
// query tile and room for three K stages and five half stages of V; else two query tiles, two and four.
//
// What bounds it, measured with 32 requests of 4096 tokens, 8 KV heads of 128, pages of 16: 4 rows,
// bfloat16, 100 us = 0.82 of the copy rate, 64 rows 109 us = 0.77: HBM.  256 rows (dual) 178 us, 0.95 us a tile
// and group: the chain S -> softmax -> P V of each group (some 3000 cycles), whose instructions come from
// caches that six kinds of warps share; half of the tensor pipe's rate.  FP8 64 rows 116 us, the same
// chain with scales in it, where the codes would take 38 us.  One request of 1024 tokens 16 us: 9 us of
// a block's way from start to end, 5 us of the join, launches.
//
// Every wait is bounded as in the prefill kernel; a block that gives up waits for the copies and products
// that it has under way before it ends.
#include <algorithm>
#include <type_traits>

#include "tc_common.cuh"
#include "tree_common.cuh"

namespace pam {
namespace {

using namespace tc;
using namespace tree;

constexpr int kRows = 128, kKeys = 128, kHd = 128;
constexpr int kTileBytes = kKeys * kHd * 2, kHalfBytes = kTileBytes / 2;      // a 64-dim block of a tile
constexpr int kVHalfBytes = kTileBytes / 2, kVBlockBytes = kVHalfBytes / 2;   // 64 keys of V, a 64-dim block of them
constexpr float kRescaleThreshold = 8.0f;
// Weights are kept times 2^7, as far up as the threshold leaves float16 room (2^15): those down to 2^-21 of a row's
// reference then keep all their bits, not those down to 2^-14 alone.  (bfloat16 has float32's range.)
template <bool BF16> constexpr float kWeightLift = BF16 ? 0.f : 7.f;
constexpr long long kWaitCycles = 400000000LL;
constexpr long long kDrainCycles = 4000000LL;          // for the copies in flight when a wait ran out
constexpr int kKProducerWarp = 8, kVProducerWarp = 9, kMmaWarp = 10, kPlanWarp = 11, kOutputWarp0 = 12;
constexpr int kConvertWarp0 = 16;                      // FP8: four more warps
template <bool FP8> constexpr int kThreads = FP8 ? 640 : 512;

// The part of a pair that lies in the block's piece: key tiles [first, last) of nT.
struct Span {
    SeqInfo s;
    int b, kvh, rp, first, last, nT, cacheTiles, rows;   // rows: of the request under the KV head
    int lastBlock;                                       // that shares the pair
    uint32_t hi;                                         // see lastFirst
    int tile;                                            // the block's tiles before this span
    int dual;                                            // both groups on every tile
    int valid;                                           // 0: the list ends here
    __device__ __forceinline__ int step() const { return dual ? 1 : 2; }
    // tiles of group x
    __device__ __forceinline__ int tilesOf(int x) const { return dual ? last - first : (last - first + 1 - x) >> 1; }
    __device__ __forceinline__ bool whole() const { return first == 0 && last == nT; }
};

// Of the ring.  A warp keeps a span only while it works on it, and looks two ahead of that at most (the issuer): it may
// not keep one while it looks for the next with work for it, since there may be any number of spans in between.
constexpr int kSpans = 8;

// FP8, of a key tile: per 16 keys (a page holds a multiple of them) the key scale times log2(e) /
// sqrt(dim), the logarithm of the value scale, and one over it.  Pages with other than positive finite scales
// are rare and prepared apart (preparePages): where the value scale is zero or not a finite number the bit in
// `zeros` is set, the values are converted to zeros and the scale counts as one; a key scale that is not a
// finite number counts as one.  Smem::spanOdd notes the latter two for addLeftOut.
struct alignas(16) PageScales {
    float key[8], valueLog[8], valueInv[8];
    uint32_t zeros;
};

// WIDE: pairs of up to 256 rows (two query tiles), else of 128.
template <bool WIDE, bool FP8>
struct Smem {
    static constexpr int kPairRows = WIDE ? 256 : 128;
    static constexpr int kQTiles = WIDE ? 2 : 1, kKStages = WIDE || FP8 ? 2 : 3, kVStages = WIDE || FP8 ? 4 : 5;
    static constexpr int kRawStages = FP8 ? 3 : 1, kScaleStages = FP8 ? 8 : 1;
    unsigned char q[kQTiles][kTileBytes];
    unsigned char k[kKStages][kTileBytes];
    unsigned char v[kVStages][kVHalfBytes];
    unsigned char raw[kRawStages][FP8 ? kKeys * kHd : 16];                // FP8: codes of a tile's keys or values as they arrive
    unsigned long long rawFull[kRawStages], rawEmpty[kRawStages];
    PageScales scales[kScaleStages];         // [tile of the block % stages]
    unsigned long long kFull[kKStages], kEmpty[kKStages], vFull[kVStages], vEmpty[kVStages];
    unsigned long long qFull, qEmpty, sFull[2], pFull[2], oFull[2], oEmpty[2];
    unsigned long long spanFull[kSpans], spanEmpty[kSpans];
    // [span of the group & 1][group][row]: sum and reference of the row, and whether the thread left a
    // value out.  Written before the weights of the span's last tile are released, read behind the
    // commit of its last P V product.  Two of each: a group may be in its next span by then, but not
    // in the one after it, whose first S product comes behind a P V product that waits for the read.
    float rowL[2][2][kRows], rowM[2][2][kRows];
    int rowOdd[2][2][kRows];
    // what a softmax thread keeps here to have registers for a row of scores: its node, its first cache
    // token, and in a tree's tile the bits of the nodes that it sees
    int rowNode[2][kRows];
    uint32_t rowFrom[2][kRows], rowBits[2][4][kRows];
    Span span[kSpans];
    int spanOdd[kSpans];                               // FP8: a page of the span has a scale that is not finite
    int scratch[32];
    uint32_t tmemBase;
    int dead;
    int issuedK, issuedV, issuedRaw, issuedQ;          // key tiles, value half tiles, tiles of codes, query tiles asked for
    unsigned long long drained;
    int prefix[1];                                     // [batch + 1]
};
constexpr size_t kSmemLimit = 227 * 1024;
template <bool WIDE, bool FP8> constexpr size_t smemBytes(int batch) { return sizeof(Smem<WIDE, FP8>) + static_cast<size_t>(batch) * sizeof(int); }
static_assert(smemBytes<true, false>(kTreeMaxBatch) <= kSmemLimit, "the block's shared memory must fit the 227 KB a block may opt into");
// warps that read the spans: producers, issuer, output, softmax; FP8: one producer, and the converters
template <bool FP8> constexpr int kSpanReaders = FP8 ? 1 + 1 + 4 + 8 + 4 : 2 + 1 + 4 + 8;

// The block's next span at or after position `pos` of the list (a pair's start, or the block's
// begin); moves pos behind that pair.  False at the end of the piece.
template <bool WIDE>
__device__ __forceinline__ bool nextSpan(const TreeParams& p, const int* prefix, int begin, int end, int quota, int& pos, Span& g) {
    const int group = p.heads / p.kvHeads;
    while (pos < end) {
        int a = 0, z = p.batch - 1;
        while (a < z) {
            const int mid = (a + z + 1) >> 1;
            if (prefix[mid] <= pos) a = mid; else z = mid - 1;
        }
        g.b = a;
        g.s = SeqInfo(p, a);
        g.cacheTiles = g.s.cacheTiles<kKeys>();
        g.nT = g.s.tiles<kKeys>();
        g.rows = g.s.n * group;
        const int rowTiles = (g.rows + kRows - 1) / kRows, perHead = rowTiles * g.nT;
        const int rel = pos - prefix[a];
        g.kvh = rel / perHead;
        const int inHead = rel - g.kvh * perHead;
        constexpr int kTiles = WIDE ? 2 : 1;            // row tiles of a pair
        g.rp = inHead / (kTiles * g.nT);
        g.dual = WIDE && rowTiles - 2 * g.rp >= 2;
        const int start = prefix[a] + g.kvh * perHead + g.rp * kTiles * g.nT, w = g.dual ? 2 : 1;
        // the tiles whose place in the list lies in [begin, end)
        g.first = begin > start ? (begin - start + w - 1) / w : 0;
        g.last = min(g.nT, (end - start + w - 1) / w);
        g.lastBlock = (start + (g.nT - 1) * w) / quota;
        pos = start + g.nT * w;
        if (g.first < g.last) return true;
    }
    return false;
}

// A step of the block's stream: group x on tile j of the span number k, g tiles into the piece.
struct Step {
    int k, first, last, j, g, x;
    bool valid, dual, lo;
    __device__ __forceinline__ bool begins() const { return j == first + (dual ? 0 : x); }        // the group's first of the span
    __device__ __forceinline__ bool ends() const { return j + (dual ? 1 : 2) >= last; }           // ... last
    __device__ __forceinline__ bool endsTile() const { return !dual || x == 1; }
    __device__ __forceinline__ bool opensSpan() const { return j == first && x == 0; }
    __device__ __forceinline__ bool closesSpan() const { return j + 1 == last && endsTile(); }
};

// Scores of keys that are not visible (bit i clear) become -inf.
__device__ __forceinline__ void maskBits(uint32_t (&r)[32], uint32_t bits) {
#pragma unroll
    for (int i = 0; i < 32; ++i)
        if (!(bits >> i & 1u)) r[i] = 0xFF800000u;
}
__device__ __forceinline__ void tmemLd16NoWait(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
}
// FP8: the largest of 16 raw scores, and the weights of 16 keys with their page's scales (the sum
// without the value scale is returned).
template <int BEGIN>
__device__ __forceinline__ float rowMax16(const uint32_t (&r)[32]) {
    float m0 = -INFINITY, m1 = -INFINITY;
#pragma unroll
    for (int i = 0; i < 16; i += 4) {
        m0 = max3(m0, __uint_as_float(r[BEGIN + i]), __uint_as_float(r[BEGIN + i + 1]));
        m1 = max3(m1, __uint_as_float(r[BEGIN + i + 2]), __uint_as_float(r[BEGIN + i + 3]));
    }
    return fmaxf(m0, m1);
}
template <int BEGIN>
__device__ __forceinline__ float pageWeights(const uint32_t (&r)[32], uint32_t (&w)[32], float key, float valueLog, float inv, float negM) {
    return inv * weightsRange<false, false, BEGIN, BEGIN + 16>(r, w, key, negM + valueLog);
}
// Two codes to two float16 values.
__device__ __forceinline__ uint32_t widen(uint32_t codes) {
    uint32_t r;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(static_cast<unsigned short>(codes)));
    return r;
}
// The entries of a tile with pages whose scales are not positive finite numbers; lane i has page i (mod 8).  A
// page of which the request holds nothing counts as one of zeros.
__device__ __forceinline__ void preparePages(PageScales& sc, int* odd, float ks, float vs, bool held, float scaleLog2) {
    const int lane = threadIdx.x & 31;
    const bool zero = !held || isOdd(vs) || !(vs > 0.f);
    if (lane < kKeys / 16) {
        sc.key[lane] = !held || isOdd(ks) ? scaleLog2 : fmaxf(ks * scaleLog2, 1e-30f);
        sc.valueLog[lane] = zero ? 0.f : log2f(vs);
        sc.valueInv[lane] = zero ? 1.f : 1.f / vs;
    }
    const uint32_t zeros = __ballot_sync(0xFFFFFFFFu, zero);
    if (lane == 0) sc.zeros = zeros & 0xFFu;
    if (held && (isOdd(ks) || isOdd(vs))) *odd = 1;
}
__device__ __forceinline__ void bulkLoad(void* dst, const void* src, uint32_t bytes, unsigned long long* bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(smemAddr(dst)), "l"(src), "r"(bytes), "r"(smemAddr(bar)) : "memory");
}
// Whether `v` is set in any of the 128 threads of the output warps (all of them get here).
__device__ __forceinline__ bool anyOfOutput(bool v) {
    uint32_t r = v ? 1u : 0u;
    asm volatile("{\n\t.reg .pred a, b;\n\tsetp.ne.u32 a, %0, 0;\n\tbarrier.cta.red.or.pred b, 1, 128, a;\n\tselp.u32 %0, 1, 0, b;\n\t}" : "+r"(r)::"memory");
    return r != 0;
}

// WHOLE: head_dim 128 (known when the code is compiled: 10% of the time over FP8 pages).
template <bool BF16, bool WIDE, bool FP8, bool WHOLE>
__global__ void __launch_bounds__(kThreads<FP8>, 1)
treeTcKernel(const __grid_constant__ CUtensorMap mapQ, const __grid_constant__ CUtensorMap mapK, const __grid_constant__ CUtensorMap mapV,
             const __grid_constant__ CUtensorMap mapKNew, const __grid_constant__ CUtensorMap mapVNew,
             const __grid_constant__ TreeParams p, float scaleLog2, int* errFlag, long long waitLimit) {
    using T = typename std::conditional<BF16, __nv_bfloat16, __half>::type;
    extern __shared__ __align__(1024) unsigned char rawSmem[];
    using S = Smem<WIDE, FP8>;
    using PoolT = typename std::conditional<FP8, uint8_t, T>::type;
    constexpr int kPairRows = S::kPairRows;
    S* s = reinterpret_cast<S*>(rawSmem);
    if ((smemAddr(rawSmem) & 1023u) != 0) {
        if (threadIdx.x == 0) atomicCAS(errFlag, 0, 40);
        return;
    }
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, group = p.heads / p.kvHeads;
    const int D = WHOLE ? kHd : p.headDim, dimBlocks = WHOLE || D > 64 ? 2 : 1;     // blocks of 64 dims; the second one's end is filled with zeros
    if (threadIdx.x == 0) {
        mbarInit(&s->qFull, kRows % group == 0 ? 1 : kRows);
        mbarInit(&s->qEmpty, 1);
        mbarInit(&s->drained, 1);
        s->issuedK = s->issuedV = s->issuedRaw = s->issuedQ = 0;
        for (int i = 0; i < 2; ++i) {
            mbarInit(&s->sFull[i], 1);
            mbarInit(&s->pFull[i], kRows);
            mbarInit(&s->oFull[i], 1);
            mbarInit(&s->oEmpty[i], 1);
        }
        for (int i = 0; i < S::kKStages; ++i) { mbarInit(&s->kFull[i], FP8 ? kRows : 1); mbarInit(&s->kEmpty[i], 1); }
        for (int i = 0; i < S::kVStages; ++i) { mbarInit(&s->vFull[i], FP8 ? kRows / 2 : 1); mbarInit(&s->vEmpty[i], 1); }
        for (int i = 0; i < S::kRawStages; ++i) { mbarInit(&s->rawFull[i], 1); mbarInit(&s->rawEmpty[i], kRows); }
        for (int i = 0; i < kSpans; ++i) { mbarInit(&s->spanFull[i], 1); mbarInit(&s->spanEmpty[i], kSpanReaders<FP8>); }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        for (const CUtensorMap* m : {&mapQ, &mapK, &mapV, &mapKNew, &mapVNew}) asm volatile("prefetch.tensormap [%0];" ::"l"(m) : "memory");
    }
    if (warp == kMmaWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smemAddr(&s->tmemBase)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    // What came before the launch on its stream is done from here on.
    cudaGridDependencySynchronize();
    if (threadIdx.x == 0) {
        s->dead = *reinterpret_cast<volatile int*>(errFlag) != 0 ? 1 : 0;
        Header h{};
        h.lastBlock = -1;
        *headerOf(p, blockIdx.x) = h;
    }
    buildPrefix<kRows, kKeys, kThreads<FP8>>(p, s->prefix, s->scratch);
    tcFenceBefore();
    __syncthreads();
    tcFenceAfter();
    const uint32_t tmem = s->tmemBase;
    auto tmemS = [&](int x) { return tmem + 128u * static_cast<uint32_t>(x); };
    auto tmemO = [&](int x) { return tmem + 256u + 128u * static_cast<uint32_t>(x); };
    const bool live = *reinterpret_cast<volatile int*>(&s->dead) == 0;
    // The block's span number k.  Null when the wait for it ran out.
    auto spanAt = [&](int k) -> const Span* {
        bool ok = mbarWait(&s->spanFull[k % kSpans], (k / kSpans) & 1, &s->dead, errFlag, waitLimit, 54);
        ok = __all_sync(0xFFFFFFFFu, ok);
        return ok ? &s->span[k % kSpans] : nullptr;
    };
    auto spanDone = [&](int k) {
        __syncwarp();
        if (lane == 0) mbarArrive(&s->spanEmpty[k % kSpans]);
    };

    // 512 x 128 registers at launch: 96 for the service warps, 96 for the output warps, 160 for softmax;
    // FP8 640 x 96: 80, 80, 120, and 80 for the converting warps
    if (warp == kKProducerWarp || warp == kVProducerWarp) {
        if constexpr (FP8) asm volatile("setmaxnreg.dec.sync.aligned.u32 80;"); else asm volatile("setmaxnreg.dec.sync.aligned.u32 96;");
        if (!live) goto done;
        const bool isV = warp == kVProducerWarp;
        const CUtensorMap* pool = isV ? &mapV : &mapK;
        const CUtensorMap* fresh = isV ? &mapVNew : &mapKNew;
        const int tilesPerPage = p.blockSize / 16;
        // 16-bit pages come in pieces of 16 rows, or of 8 (an atom of the swizzle) where 16 does not divide them
        const int pieceRows = p.blockSize % 16 == 0 ? 16 : 8, pieces = kKeys / pieceRows, piecesPerPage = p.blockSize / pieceRows, pieceBytes = pieceRows * 128;
        int gt = 0;                          // tiles of the block's piece so far
        bool ok = true;
        if constexpr (FP8) {
            // One warp for keys and values: pages of 16 rows, 2 KB of codes each (head_dim 128), keys before values in
            // one ring, and the tile's scales, which the ring of eight keeps until the softmax is through:
            // behind the ring of codes this warp is at most five tiles ahead of it.  (The rows of a tree are
            // fetched by the converting warps; their tiles take part in the ring, empty.)  Lane i has page
            // piece i; its entry of the block table is looked up two tiles ahead, its scales one.
            auto entry = [&](const Span& g, const int32_t* table, int j) {
                const int t16 = (static_cast<int>(g.s.lo / kKeys) + j) * (kKeys / 16) + (lane & 7);
                return table[min(t16 / tilesPerPage, p.maxNumBlocks - 1)];
            };
            auto pairOf = [&](const Span& g, int blk) {
                return static_cast<int64_t>(min(max(blk, 0), p.poolBlocks - 1)) * p.kvHeads + g.kvh;
            };
            const __half* kScale = static_cast<const __half*>(p.kScale);
            const __half* vScale = static_cast<const __half*>(p.vScale);
            int raw = 0;
            for (int k = 0; ok && !isV; ++k) {
                const Span* at = spanAt(k);
                if (!at || !at->valid) break;
                const Span& g = *at;
                const int32_t* table = p.tables + static_cast<int64_t>(g.b) * p.maxNumBlocks;
                const int end = min(g.last, g.cacheTiles);           // of the tiles of the cache
                if (lane == 0) s->spanOdd[k % kSpans] = 0;
                __syncwarp();
                int nextBlk = 0;
                int64_t pair = 0;
                __half ksNext = __float2half(0.f), vsNext = ksNext;
                if (g.first < end) {
                    pair = pairOf(g, entry(g, table, g.first));
                    ksNext = kScale[pair];
                    vsNext = vScale[pair];
                    if (g.first + 1 < end) nextBlk = entry(g, table, g.first + 1);
                }
                for (int j = g.first; j < g.last && ok; ++j, ++gt) {
                    const bool inTree = j >= g.cacheTiles;
                    const int t16 = (static_cast<int>(g.s.lo / kKeys) + j) * (kKeys / 16) + (lane & 7);
                    const int64_t from = (pair * p.blockSize + (t16 % tilesPerPage) * 16) * D;
                    const float ks = __half2float(ksNext), vs = __half2float(vsNext);
                    if (j + 1 < end) {
                        pair = pairOf(g, nextBlk);
                        ksNext = kScale[pair];
                        vsNext = vScale[pair];
                        if (j + 2 < end) nextBlk = entry(g, table, j + 2);
                    }
#pragma unroll
                    for (int h = 0; h < 2; ++h, ++raw) {
                        const int st = raw % S::kRawStages;
                        if (raw >= S::kRawStages) ok = mbarWait(&s->rawEmpty[st], ((raw / S::kRawStages) - 1) & 1, &s->dead, errFlag, waitLimit, 56);
                        ok = __all_sync(0xFFFFFFFFu, ok);
                        if (!ok) break;
                        if (h == 0) {
                            PageScales& sc = s->scales[gt % S::kScaleStages];
                            if (__all_sync(0xFFFFFFFFu, inTree || (vs > 0.f && !isOdd(vs) && !isOdd(ks)))) {
                                if (lane < kKeys / 16) {
                                    sc.key[lane] = inTree ? scaleLog2 : fmaxf(ks * scaleLog2, 1e-30f);      // (zero times a masked score would be NaN)
                                    sc.valueLog[lane] = inTree ? 0.f : log2f(vs);
                                    sc.valueInv[lane] = inTree ? 1.f : 1.f / vs;
                                }
                                if (lane == 0) sc.zeros = 0u;
                            } else {
                                const uint32_t piece = static_cast<uint32_t>(t16);
                                preparePages(sc, &s->spanOdd[k % kSpans], ks, vs, piece >= g.s.lo / 16u && piece <= (g.s.held - 1u) / 16u, scaleLog2);
                            }
                        }
                        __syncwarp();
                        if (lane == 0) {
                            if (inTree) mbarArrive(&s->rawFull[st]);
                            else mbarExpectTx(&s->rawFull[st], kKeys * D);
                        }
                        __syncwarp();
                        if (!inTree && lane < kKeys / 16)
                            bulkLoad(s->raw[st] + lane * 16 * D, static_cast<const unsigned char*>(h ? p.vPool : p.kPool) + from, 16 * D, &s->rawFull[st]);
                    }
                }
                spanDone(k);
            }
            if (!isV && lane == 0) s->issuedRaw = raw;
        }
        int issued = 0;
        for (int k = 0; ok && !FP8; ++k) {
            const Span* at = spanAt(k);
            if (!at || !at->valid) break;
            const Span& g = *at;
            const int32_t* table = p.tables + static_cast<int64_t>(g.b) * p.maxNumBlocks;
            for (int j = g.first; j < g.last && ok; ++j, ++gt) {
                const bool inTree = j >= g.cacheTiles;
                const int freshRow = g.s.start + (j - g.cacheTiles) * kKeys;
                int row = 0;
                if (!inTree && lane < pieces) {
                    const int at = (static_cast<int>(g.s.lo / kKeys) + j) * pieces + lane;
                    const int page = min(at / piecesPerPage, p.maxNumBlocks - 1);
                    const int blk = min(max(table[page], 0), p.poolBlocks - 1);
                    row = (blk * p.kvHeads + g.kvh) * p.blockSize + (at % piecesPerPage) * pieceRows;
                }
                if (!isV) {
                    const int st = gt % S::kKStages;
                    if (gt >= S::kKStages) ok = mbarWait(&s->kEmpty[st], ((gt / S::kKStages) - 1) & 1, &s->dead, errFlag, waitLimit, 41);
                    ok = __all_sync(0xFFFFFFFFu, ok);
                    if (!ok) break;
                    if (lane == 0) mbarExpectTx(&s->kFull[st], dimBlocks * kHalfBytes);
                    __syncwarp();
                    ++issued;
                    unsigned char* to = s->k[st];
                    if (inTree) {
                        if (lane < dimBlocks)
                            for (int h = 0; h < 2; ++h)        // (a box is 64 rows)
                                tmaLoad3d(to + lane * kHalfBytes + h * kVBlockBytes, fresh, &s->kFull[st], 64 * lane, g.kvh, freshRow + 64 * h);
                    } else if (lane < pieces) {
                        tmaLoad2d(to + lane * pieceBytes, pool, &s->kFull[st], 0, row);
                        if (dimBlocks == 2) tmaLoad2d(to + kHalfBytes + lane * pieceBytes, pool, &s->kFull[st], 64, row);
                    }
                } else {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const int n = 2 * gt + h, st = n % S::kVStages;
                        if (n >= S::kVStages) ok = mbarWait(&s->vEmpty[st], ((n / S::kVStages) - 1) & 1, &s->dead, errFlag, waitLimit, 42);
                        ok = __all_sync(0xFFFFFFFFu, ok);
                        if (!ok) break;
                        if (lane == 0) mbarExpectTx(&s->vFull[st], dimBlocks * kVBlockBytes);
                        __syncwarp();
                        ++issued;
                        unsigned char* to = s->v[st];
                        if (inTree) {
                            if (lane < dimBlocks) tmaLoad3d(to + lane * kVBlockBytes, fresh, &s->vFull[st], 64 * lane, g.kvh, freshRow + 64 * h);
                        } else if (lane < pieces && (lane >= pieces / 2) == (h == 1)) {
                            const int in = (lane - h * (pieces / 2)) * pieceBytes;
                            tmaLoad2d(to + in, pool, &s->vFull[st], 0, row);
                            if (dimBlocks == 2) tmaLoad2d(to + kVBlockBytes + in, pool, &s->vFull[st], 64, row);
                        }
                    }
                }
            }
            spanDone(k);
        }
        if (!FP8 && lane == 0) (isV ? s->issuedV : s->issuedK) = issued;
    } else if (warp == kMmaWarp) {
        if constexpr (FP8) asm volatile("setmaxnreg.dec.sync.aligned.u32 80;"); else asm volatile("setmaxnreg.dec.sync.aligned.u32 96;");
        if (!live) goto done;
        const bool leader = electOne();
        const uint32_t fmt = BF16 ? 1u : 0u;
        const uint32_t idescS = (1u << 4) | (fmt << 7) | (fmt << 10) | ((128u >> 3) << 17) | ((128u >> 4) << 24);
        // (of one block of dims: N = 64)
        const uint32_t idescO = ((1u << 4) | (fmt << 7) | (fmt << 10) | (static_cast<uint32_t>(dimBlocks * 64 / 8) << 17) | ((128u >> 4) << 24)) | (1u << 16);
        const uint32_t hiK = descHi(1024);
        bool ok = true;
        // The steps of the stream, in order: a tile of a dual span is one step of each group, else tiles
        // alternate between the groups.  Products of a group come in the order S, P V, S, ..., and of
        // two steps in a row (nearly always of two groups) the second one's S must not wait for the
        // first one's weights: c is the next step to have its P V product issued, n the next one to have
        // its S product issued, up to two steps ahead, where the group's step before is through.
        Step c, n;
        auto take = [&](Step& at, int k) {
            const Span* sp = spanAt(k);
            at.k = k;
            at.x = 0;
            at.valid = sp && sp->valid;
            if (!sp) ok = false;
            if (at.valid) { at.first = at.j = sp->first; at.last = sp->last; at.dual = sp->dual != 0; at.lo = twoOperands(p, sp->s); }
        };
        auto advance = [&](Step& at) {
            const bool sameTile = at.dual && at.x == 0;
            at.x ^= 1;
            if (sameTile) return;
            ++at.g;
            if (++at.j == at.last) take(at, at.k + 1);
        };
        c.g = 0;
        take(c, 0);
        n = c;
        int cs = 0, ns = 0;                  // numbers of the two steps
        int nPrev = -1;                      // group of the step before n
        uint32_t pParity = 0, oParity = 0, begun = 0;      // bit x: phase of pFull, of oEmpty; group x has begun a span
        while (c.valid && ok) {
            // ---- S products; while one is held up by its keys or queries, the weights of step c may come
            // first (test_wait: try_wait would sleep through the other condition)
            bool got = false;                // the weights of step c are there
            long long since = 0;
            while (ok && !got) {
                // (the group's step before is n - 1 at the earliest; it is through if that is another group's)
                if (!n.valid || ns > cs + 1 || (ns > cs && n.x == nPrev)) break;
                const int st = n.g % S::kKStages;
                const uint32_t kPar = (n.g / S::kKStages) & 1, qPar = n.k & 1;
                bool there = mbarTest(&s->kFull[st], kPar) && (!n.opensSpan() || mbarTest(&s->qFull, qPar));
                there = __all_sync(0xFFFFFFFFu, there);
                if (!there) {
                    if (ns > cs) got = __all_sync(0xFFFFFFFFu, mbarTest(&s->pFull[c.x], pParity >> c.x & 1));
                    if (since == 0) since = clock64();
                    else if (clock64() - since > waitLimit) {
                        *reinterpret_cast<volatile int*>(&s->dead) = 1;
                        atomicCAS(errFlag, 0, 44);
                    }
                    if (*reinterpret_cast<volatile int*>(&s->dead)) ok = false;
                    ok = __all_sync(0xFFFFFFFFu, ok);
                    continue;
                }
                since = 0;
                tcFenceAfter();
                const uint32_t qLo = descLo(smemAddr(s->q[0]) + (WIDE && n.dual ? n.x * kTileBytes : 0), 16);
                const uint32_t kLo = descLo(smemAddr(s->k[0]) + st * kTileBytes, 16), dS = tmemS(n.x);
                uint64_t dq[kHd / 16], dk[kHd / 16];
#pragma unroll
                for (int ks = 0; ks < kHd / 16; ++ks) {
                    const uint32_t off = ((ks >> 2) * kHalfBytes + (ks & 3) * 32) >> 4;
                    dq[ks] = desc64(qLo + off, hiK);
                    dk[ks] = desc64(kLo + off, hiK);
                }
                if (leader) {
#pragma unroll
                    for (int ks = 0; ks < kHd / 16; ++ks)
                        if (ks < 4 || dimBlocks == 2) umma(dS, dq[ks], dk[ks], idescS, ks > 0);
                    ummaCommit(&s->sFull[n.x]);
                    if (n.endsTile()) ummaCommit(&s->kEmpty[st]);
                    if (n.closesSpan()) ummaCommit(&s->qEmpty);
                }
                __syncwarp();
                nPrev = n.x;
                ++ns;
                advance(n);
            }
            if (ok && !got) ok = mbarWait(&s->pFull[c.x], pParity >> c.x & 1, &s->dead, errFlag, waitLimit, 45);
            ok = __all_sync(0xFFFFFFFFu, ok);
            if (!ok) break;
            // ---- the P V product of step c
            const int x = c.x;
            pParity ^= 1u << x;
            const bool begins = c.begins();
            if (begins) {
                // the accumulator is free once the output of the group's span before was read from it
                if (ok && (begun >> x & 1)) {
                    ok = mbarWait(&s->oEmpty[x], oParity >> x & 1, &s->dead, errFlag, waitLimit, 47);
                    oParity ^= 1u << x;
                }
                begun |= 1u << x;
            }
            const uint32_t sCol = tmemS(x), dO = tmemO(x);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int v = 2 * c.g + h, st = v % S::kVStages;
                if (ok) ok = mbarWait(&s->vFull[st], (v / S::kVStages) & 1, &s->dead, errFlag, waitLimit, 46);
                ok = __all_sync(0xFFFFFFFFu, ok);
                if (!ok) break;
                tcFenceAfter();
                const uint32_t vLo = descLo(smemAddr(s->v[0]) + st * kVHalfBytes, kVBlockBytes);
                uint64_t dv[4];
#pragma unroll
                for (int ks = 0; ks < 4; ++ks) dv[ks] = desc64(vLo + ks * 128, hiK);
                if (leader) {
                    // P of keys 32 i .. 32 i + 31 sits in columns 32 i .. 32 i + 15 of the S buffer (and, with
                    // two operands, its remainder in columns 32 i + 16 .. 32 i + 31)
#pragma unroll
                    for (int ks = 0; ks < 4; ++ks)
                        ummaTs(dO, sCol + 64u * h + 32u * (ks >> 1) + 8u * (ks & 1), dv[ks], idescO, h + ks > 0 || !begins ? 1u : 0u);
                    if (BF16 && c.lo) {
#pragma unroll
                        for (int ks = 0; ks < 4; ++ks)
                            ummaTs(dO, sCol + 64u * h + 32u * (ks >> 1) + 8u * (ks & 1) + 16u, dv[ks], idescO, 1u);
                    }
                    if (h == 1 && c.ends()) ummaCommit(&s->oFull[x]);
                    if (c.endsTile()) ummaCommit(&s->vEmpty[st]);
                }
                __syncwarp();
            }
            if (!ok) break;
            const int k = c.k;
            ++cs;
            advance(c);
            if (c.k != k) spanDone(k);       // (n is in a later span by now)
        }
    } else if (warp == kPlanWarp) {
        if constexpr (FP8) asm volatile("setmaxnreg.dec.sync.aligned.u32 80;"); else asm volatile("setmaxnreg.dec.sync.aligned.u32 96;");
        if (!live) goto done;
        const int total = s->prefix[p.batch];
        // (a piece of at least two, so that every block between a pair's first and last has a tile of it)
        const int quota = max(2, (total + static_cast<int>(gridDim.x) - 1) / static_cast<int>(gridDim.x));
        const int begin = static_cast<int>(min(static_cast<long long>(blockIdx.x) * quota, static_cast<long long>(total)));
        const int end = min(total, begin + quota);
        int pos = begin, tile = 0;
        bool ok = true;
        for (int k = 0; ok; ++k) {
            Span g;
            const bool got = nextSpan<WIDE>(p, s->prefix, begin, end, quota, pos, g);
            g.valid = got;
            g.tile = tile;
            if (got) {
                g.hi = lastFirstOfWarp(p, g.s, g.rp, kPairRows);
                tile += g.last - g.first;
            }
            if (k >= kSpans) ok = mbarWait(&s->spanEmpty[k % kSpans], ((k / kSpans) - 1) & 1, &s->dead, errFlag, waitLimit, 55);
            ok = __all_sync(0xFFFFFFFFu, ok);
            if (!ok) break;
            if (lane == 0) {
                s->span[k % kSpans] = g;
                mbarArrive(&s->spanFull[k % kSpans]);
            }
            __syncwarp();
            if (!got) break;
        }
    } else if (FP8 && warp >= kConvertWarp0) {
        // ------------------------------------------------------------ converting warps
        // They turn the rows of every tile from codes into float16 (exactly) in the swizzled layout of
        // the products' operands.  A tile of the tree comes as float16 already, by TMA.
        if constexpr (FP8) asm volatile("setmaxnreg.dec.sync.aligned.u32 80;");
        if (!live) goto done;
        const int t = (warp & 3) * 32 + lane, half = t >> 6;
        int gt = 0, raw = 0;
        bool ok = true;
        // The warp's 32 rows of codes into the 64-dim blocks of a tile, `block` bytes apart: a lane takes 16
        // codes of a row at a time.  Eight lanes read eight pieces, of row r left of the middle and of row
        // r ^ 1 right of it: their writes then fall on eight different bank groups too.
        const int piece = lane & 7, rowIn = (lane >> 3) ^ (piece >> 2);
        const unsigned rawAt = static_cast<unsigned>(((warp & 3) * 32 + rowIn) * D + piece * 16);
        const unsigned outAt = static_cast<unsigned>(rowIn * 128 + ((((2 * piece) & 7) ^ rowIn) << 4));
        auto convert = [&](const unsigned char* from, unsigned char* to, int block, uint32_t zeros) {
            if (piece >= 4 * dimBlocks) return;
            const bool there = piece * 16 < D;
            from += rawAt;
            to += (piece >> 2) * block;
#pragma unroll
            for (int i0 = 0; i0 < 8; i0 += 4) {
                uint4 w[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) w[i] = there && !(zeros >> (i0 >> 2) & 1u) ? *reinterpret_cast<const uint4*>(from + (i0 + i) * 4 * D) : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    unsigned char* row = to + (i0 + i) * 512;
                    const unsigned at = outAt ^ (i & 1 ? 64u : 0u);
                    *reinterpret_cast<uint4*>(row + at) = make_uint4(widen(w[i].x), widen(w[i].x >> 16), widen(w[i].y), widen(w[i].y >> 16));
                    *reinterpret_cast<uint4*>(row + (at ^ 16u)) = make_uint4(widen(w[i].z), widen(w[i].z >> 16), widen(w[i].w), widen(w[i].w >> 16));
                }
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        };
        for (int k = 0; ok; ++k) {
            const Span* sp = spanAt(k);
            if (!sp || !sp->valid) break;
            const Span& g = *sp;
            for (int j = g.first; j < g.last && ok; ++j, ++gt) {
                const bool inTree = j >= g.cacheTiles;
                const int freshRow = g.s.start + (j - g.cacheTiles) * kKeys;
                const int ks = gt % S::kKStages, n = 2 * gt + half, vs = n % S::kVStages;
                int st = raw % S::kRawStages;
                ok = mbarWait(&s->rawFull[st], (raw / S::kRawStages) & 1, &s->dead, errFlag, waitLimit, 58);
                if (ok && gt >= S::kKStages) ok = mbarWait(&s->kEmpty[ks], ((gt / S::kKStages) - 1) & 1, &s->dead, errFlag, waitLimit, 57);
                if (!ok) break;
                if (!inTree) convert(s->raw[st], s->k[ks] + (warp & 3) * 4096, kHalfBytes, 0u);
                mbarArrive(&s->rawEmpty[st]);
                if (inTree && t == 0) {
                    mbarExpectTx(&s->kFull[ks], dimBlocks * kHalfBytes);
                    for (int i = 0; i < 2 * dimBlocks; ++i)      // (a box is 64 rows of 64 dims)
                        tmaLoad3d(s->k[ks] + (i >> 1) * kHalfBytes + (i & 1) * kVBlockBytes, &mapKNew, &s->kFull[ks], 64 * (i >> 1), g.kvh, freshRow + 64 * (i & 1));
                } else {
                    mbarArrive(&s->kFull[ks]);
                }
                st = ++raw % S::kRawStages;
                ok = mbarWait(&s->rawFull[st], (raw / S::kRawStages) & 1, &s->dead, errFlag, waitLimit, 60);
                if (ok && n >= S::kVStages) ok = mbarWait(&s->vEmpty[vs], ((n / S::kVStages) - 1) & 1, &s->dead, errFlag, waitLimit, 59);
                if (!ok) break;
                if (!inTree) convert(s->raw[st], s->v[vs] + (warp & 1) * 4096, kVBlockBytes, s->scales[gt % S::kScaleStages].zeros >> (2 * (warp & 3)));
                mbarArrive(&s->rawEmpty[st]);
                if (inTree && (t & 63) == 0) {
                    mbarExpectTx(&s->vFull[vs], dimBlocks * kVBlockBytes);
                    for (int i = 0; i < dimBlocks; ++i)
                        tmaLoad3d(s->v[vs] + i * kVBlockBytes, &mapVNew, &s->vFull[vs], 64 * i, g.kvh, freshRow + 64 * half);
                } else {
                    mbarArrive(&s->vFull[vs]);
                }
                ++raw;
            }
            ok = __all_sync(0xFFFFFFFFu, ok);
            spanDone(k);
        }
        if (t == 0) {
            // (only tiles of a tree are copies, and the thread that asks for half of V may be a tile ahead: what
            // counts too much costs the error exit a wait)
            s->issuedK = gt + 1;
            s->issuedV = 2 * gt + 4;
        }
    } else if (warp >= kOutputWarp0) {
        if constexpr (FP8) asm volatile("setmaxnreg.dec.sync.aligned.u32 80;"); else asm volatile("setmaxnreg.dec.sync.aligned.u32 96;");
        if (!live) goto done;
        const int t = (warp & 3) * 32 + lane;
        const uint32_t laneBase = static_cast<uint32_t>((warp & 3) * 32) << 16;
        const bool first = threadIdx.x == kOutputWarp0 * 32;
        int cnt0 = 0, cnt1 = 0;              // spans of a group written: phase of oFull
        int asked = 0;
        // a span's queries into the query tile (a dual span's: tiles), zeros where the request has no
        // such row
        auto fetchQ = [&](const Span& g) {
            ++asked;
            if (kRows % group == 0) {
                // a tile of whole nodes: one box of (64 dims, the KV head's query heads, 128 / group nodes)
                // for each half (rows behind the request's belong to others and are not used)
                if (first) {
                    const int node = g.rp * (kPairRows / group), tiles = WIDE && g.dual ? 2 : 1;
                    mbarExpectTx(&s->qFull, tiles * dimBlocks * kHalfBytes);
                    for (int i = 0; i < 2 * tiles; ++i)
                        if (dimBlocks == 2 || !(i & 1)) tmaLoad3d(s->q[i >> 1] + (i & 1) * kHalfBytes, &mapQ, &s->qFull, 64 * (i & 1), g.kvh * group,
                                  g.s.start + node + (i >> 1) * (kRows / group));
                }
                return;
            }
#pragma unroll 1
            for (int i = 0; i < S::kQTiles; ++i) {
                if (i > 0 && !g.dual) break;
                // every lane looks its row up; half a warp then copies a row, 16 bytes a lane
                const int rr = g.rp * kPairRows + i * kRows + t;
                const int64_t off = rr < g.rows ? static_cast<int64_t>(g.s.start + rr / group) * p.qStride + static_cast<int64_t>(g.kvh * group + rr % group) * D : -1;
                const int c = lane & 15;
#pragma unroll 4
                for (int r = 0; r < 16; ++r) {
                    const int in = 2 * r + (lane >> 4), row = (warp & 3) * 32 + in;
                    int64_t at = __shfl_sync(0xFFFFFFFFu, off, in);
                    if (c * 8 >= D) at = -1;
                    const uint32_t dst = smemAddr(s->q[i]) + row * 128 + (c >> 3) * kHalfBytes + (((c & 7) ^ (row & 7)) << 4);
                    const int n = at >= 0 ? 16 : 0;
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(static_cast<const T*>(p.q) + (at >= 0 ? at + c * 8 : 0)), "r"(n) : "memory");
                }
            }
            asm volatile("cp.async.wait_all;" ::: "memory");
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            mbarArrive(&s->qFull);
        };
        bool ok = true;
        {
            const Span* at = spanAt(0);
            if (at && at->valid) fetchQ(*at);
        }
        for (int k = 0; ok; ++k) {
            const Span* at = spanAt(k);
            ok = !anyOfOutput(at == nullptr);          // (all four warps decide together, so that none waits for one that gave up)
            if (!ok || !at->valid) break;
            const Span& g = *at;
            const Span* next = spanAt(k + 1);
            if (next && next->valid) {
                // the last S product of this span is complete: its queries are no longer read
                ok = mbarWait(&s->qEmpty, k & 1, &s->dead, errFlag, waitLimit, 48);
                ok = __all_sync(0xFFFFFFFFu, ok);
                if (ok) fetchQ(*next);
            }
            const bool has1 = g.tilesOf(1) > 0;
            if (ok) ok = mbarWait(&s->oFull[0], cnt0 & 1, &s->dead, errFlag, waitLimit, 49);
            if (ok && has1) ok = mbarWait(&s->oFull[1], cnt1 & 1, &s->dead, errFlag, waitLimit, 51);
            ok = !anyOfOutput(!ok);
            if (!ok) break;
            tcFenceAfter();
            const int p0 = cnt0 & 1, p1 = cnt1 & 1;
            // values left out anywhere in the span
            const bool odd = anyOfOutput(s->rowOdd[p0][0][t] != 0 || (has1 && s->rowOdd[p1][1][t] != 0) || (FP8 && s->spanOdd[k % kSpans] != 0));
            const bool whole = g.whole();
            const int which = g.first == 0 ? 1 : 0;
            if (!whole && first) {
                Header* h = headerOf(p, blockIdx.x);
                h->odd[which] = odd ? 1 : 0;
                if (which == 1) {
                    h->b = g.b; h->kvh = g.kvh; h->rt = g.rp;
                    h->lastBlock = g.lastBlock;
                }
            }
            float* rec = whole ? nullptr : recordOf(p, gridDim.x, blockIdx.x, which, kPairRows, kHd);
#pragma unroll 1
            for (int x = 0; x < (g.dual ? 2 : 1); ++x) {
                const int rl = (g.dual ? x * kRows : 0) + t, rr = g.rp * kPairRows + rl;
                const bool mine = rr < g.rows;
                float m = s->rowM[x ? p1 : p0][x][t], l = s->rowL[x ? p1 : p0][x][t], a0 = 1.f, a1 = 0.f;
                if (!g.dual && has1) {
                    const float m1 = s->rowM[p1][1][t], top = fmaxf(m, m1), base = top == -INFINITY ? 0.f : top;
                    a0 = ex2Approx(m - base);
                    a1 = ex2Approx(m1 - base);
                    l = l * a0 + s->rowL[p1][1][t] * a1;
                    m = top;
                }
                const float inv = whole ? (l == 0.f ? 0.f : 1.f / l) : 1.f;
                a0 *= inv;
                a1 *= inv;
                T* out = static_cast<T*>(p.out) + (mine ? (static_cast<int64_t>(g.s.start + rr / group) * p.heads + g.kvh * group + rr % group) * D : 0);
                float4* recO = reinterpret_cast<float4*>(rec) + rl;
                const bool both = !g.dual && has1;
                const unsigned long long scale0 = pack2(a0, a0), scale1 = pack2(a1, a1);
                // 16 columns at a time.  (What counts here are instructions: one warp on each scheduler,
                // whose fetches compete with the softmax warps' long loop.  Trading pieces among lanes for
                // wider segments of a row made the loop longer and 1.5 times slower.)
#pragma unroll 1
                for (int c = 0; c < D / 16; ++c) {
                    uint32_t o[16], u[16];
                    tmemLd16NoWait(tmemO(x) + laneBase + 16u * c, o);
                    if (both) tmemLd16NoWait(tmemO(1) + laneBase + 16u * c, u);
                    tmemLdWait();
                    unsigned long long f[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) f[i] = mul2(pack2(__uint_as_float(o[2 * i]), __uint_as_float(o[2 * i + 1])), scale0);
                    if (both)
#pragma unroll
                        for (int i = 0; i < 8; ++i) f[i] = fma2(pack2(__uint_as_float(u[2 * i]), __uint_as_float(u[2 * i + 1])), scale1, f[i]);
                    if (mine) {
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            float lo, hi;
                            unpack2(f[i], lo, hi);
                            o[2 * i] = __float_as_uint(lo);
                            o[2 * i + 1] = __float_as_uint(hi);
                        }
                        if (whole) {
#pragma unroll
                            for (int i = 0; i < 8; ++i) o[i] = pack16<BF16>(__uint_as_float(o[2 * i]), __uint_as_float(o[2 * i + 1]));
                            *reinterpret_cast<uint4*>(out + 16 * c) = make_uint4(o[0], o[1], o[2], o[3]);
                            *reinterpret_cast<uint4*>(out + 16 * c + 8) = make_uint4(o[4], o[5], o[6], o[7]);
                        } else {
                            // records are [32 pieces of 4 columns][256 rows]: consecutive lanes, consecutive 16 bytes
#pragma unroll
                            for (int q = 0; q < 4; ++q)
                                recO[(4 * c + q) * kPairRows] = make_float4(__uint_as_float(o[4 * q]), __uint_as_float(o[4 * q + 1]), __uint_as_float(o[4 * q + 2]), __uint_as_float(o[4 * q + 3]));
                        }
                    }
                    __syncwarp();
                }
                if (whole && odd && mine)
                    addLeftOut<T, PoolT>(p, g.s, g.b, g.kvh, rr / group, g.hi, out, 0, D);
                __syncwarp();
                if (!whole && mine) {
                    rec[kPairRows * kHd + rl] = m;
                    rec[kPairRows * kHd + kPairRows + rl] = l;
                }
            }
            tcFenceBefore();
            anyOfOutput(false);
            if (first) {
                mbarArrive(&s->oEmpty[0]);              // the accumulators and the rows' sums may be overwritten
                if (has1) mbarArrive(&s->oEmpty[1]);
            }
            ++cnt0;
            if (has1) ++cnt1;
            spanDone(k);
        }
        if (first) s->issuedQ = asked;
    } else {
        // ------------------------------------------------------------ softmax groups
        if constexpr (FP8) asm volatile("setmaxnreg.inc.sync.aligned.u32 120;"); else asm volatile("setmaxnreg.inc.sync.aligned.u32 160;");
        if (!live) goto done;
        const int x = warp >> 2, t = (warp & 3) * 32 + lane;
        const uint32_t laneBase = static_cast<uint32_t>((warp & 3) * 32) << 16;
        const uint32_t sAddr = tmemS(x) + laneBase, oAddr = tmemO(x) + laneBase;
        bool ok = true;
        int steps = 0, spans = 0;            // tiles this group has done (phase of sFull), spans
        // the number of the next span at or after k with tiles of this group, or -1; spans without are
        // given back
        auto seek = [&](int k) {
            for (;; ++k) {
                const Span* at = spanAt(k);
                if (!at) ok = false;
                if (!at || !at->valid) return -1;
                if (at->tilesOf(x) > 0) return k;
                spanDone(k);
            }
        };
        int k = seek(0);
        while (k >= 0 && ok) {
            const Span& g = s->span[k % kSpans];
            {
                const int rr = g.rp * kPairRows + (g.dual ? x * kRows : 0) + t, node = rr < g.rows ? rr / group : 0;
                s->rowNode[x][t] = node;
                s->rowFrom[x][t] = max(firstOf(p, g.s, node), g.s.lo);
            }
            const bool useLo = BF16 && twoOperands(p, g.s);
            float mUsed = -INFINITY, l = 0.f;
            int odd = 0;
            const int j0 = g.first + (g.dual ? 0 : x);
            for (int j = j0; j < g.last && ok; j += g.step(), ++steps) {
                const bool inTree = j >= g.cacheTiles;
                const uint32_t k0 = inTree ? static_cast<uint32_t>(j - g.cacheTiles) * kKeys : (g.s.lo / kKeys + j) * kKeys;
                const uint32_t keyEnd = inTree ? static_cast<uint32_t>(g.s.n) : g.s.held;
                const bool edge = inTree || k0 < g.hi || k0 < g.s.lo || k0 + kKeys > keyEnd;
                const bool lastTile = j + g.step() >= g.last;
                if (edge) {
                    // the keys of the tile that the row sees, as bits (loads that the wait below hides)
                    const uint32_t first = s->rowFrom[x][t];
                    const int from = first > k0 ? static_cast<int>(min(first - k0, 128u)) : 0, to = static_cast<int>(min(keyEnd - k0, 128u));
#pragma unroll 1
                    for (int i = 0; i < 4; ++i) {
                        uint32_t bits;
                        if (inTree) bits = treeBits(p, g.s, s->rowNode[x][t], static_cast<int>(k0 / 32) + i);
                        else {
                            const int a = min(max(from - 32 * i, 0), 32), b = min(max(to - 32 * i, 0), 32);
                            bits = (b < 32 ? (1u << b) - 1u : 0xFFFFFFFFu) & (a < 32 ? 0xFFFFFFFFu << a : 0u);
                        }
                        s->rowBits[x][i][t] = bits;
                    }
                }
                ok = mbarWait(&s->sFull[x], steps & 1, &s->dead, errFlag, waitLimit, 52);
                ok = __all_sync(0xFFFFFFFFu, ok);
                if (!ok) break;
                tcFenceAfter();
                // Two passes over the row, half of it at a time: the maximum, then the weights.  (All 128
                // scores in registers, read once, make a loop whose code does not stay in the instruction
                // caches next to the other roles': 129 against 119 us at 64 requests of 2048 tokens.)
                // FP8: per 16 keys, score times key scale plus the logarithm of the value scale, so that the weights
                // come out times the value scale, near 1 whatever the scales are; the sum takes it out again.
                const PageScales& sc = s->scales[(g.tile + j - g.first) % S::kScaleStages];
                float tmax = -INFINITY;
#pragma unroll 1
                for (int c = 0; c < 4; c += 2) {
                    uint32_t r0[32], r1[32];
                    float4 key, add;
                    if constexpr (FP8) { key = reinterpret_cast<const float4*>(sc.key)[c >> 1]; add = reinterpret_cast<const float4*>(sc.valueLog)[c >> 1]; }
                    tmemLd32NoWait(sAddr + 32u * c, r0);
                    tmemLd32NoWait(sAddr + 32u * c + 32u, r1);
                    tmemLdWait();
                    if (edge) {
                        maskBits(r0, s->rowBits[x][c][t]);
                        maskBits(r1, s->rowBits[x][c + 1][t]);
                    }
                    if constexpr (FP8) {
                        tmax = fmaxf(max3(tmax, fmaf(rowMax16<0>(r0), key.x, add.x), fmaf(rowMax16<16>(r0), key.y, add.y)),
                                     fmaxf(fmaf(rowMax16<0>(r1), key.z, add.z), fmaf(rowMax16<16>(r1), key.w, add.w)));
                    } else {
                        tmax = fmaxf(tmax, fmaxf(quarterRowMax(r0), quarterRowMax(r1)));
                    }
                }
                if (!FP8) tmax *= scaleLog2;
                bool raise = false;
                float corr = 1.f;
                if (j == j0) mUsed = tmax;
                else if (tmax > mUsed + kRescaleThreshold) {
                    raise = true;
                    corr = ex2Approx(mUsed - tmax);
                    mUsed = tmax;
                }
                if (j > j0 && __any_sync(0xFFFFFFFFu, raise)) {
                    // (complete up to the group's tile before: this S product was issued behind that P V product)
#pragma unroll 1
                    for (int c = 0; c < 4; ++c) {
                        uint32_t o[32];
                        tmemLd32(oAddr + 32u * c, o);
#pragma unroll
                        for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * corr);
                        tmemSt32(oAddr + 32u * c, o);
                    }
                    tmemStWait();
                    l *= corr;
                }
                const float negM = mUsed == -INFINITY ? 0.f : kWeightLift<BF16> - mUsed;
                if constexpr (FP8) {
                    // (a quarter at a time: there are fewer registers)
#pragma unroll 1
                    for (int c = 0; c < 4; ++c) {
                        uint32_t r[32], wgt[32];
                        const float2 key = reinterpret_cast<const float2*>(sc.key)[c], add = reinterpret_cast<const float2*>(sc.valueLog)[c];
                        const float2 inv = reinterpret_cast<const float2*>(sc.valueInv)[c];
                        tmemLd32NoWait(sAddr + 32u * c, r);
                        tmemLdWait();
                        if (edge) maskBits(r, s->rowBits[x][c][t]);
                        l += pageWeights<0>(r, wgt, key.x, add.x, inv.x, negM);
                        l += pageWeights<16>(r, wgt, key.y, add.y, inv.y, negM);
                        tmemSt16(sAddr + 32u * c, wgt);
                    }
                } else
#pragma unroll 1
                for (int c = 0; c < 4; c += 2) {
                    uint32_t r0[32], r1[32], wgt[32];
                    tmemLd32NoWait(sAddr + 32u * c, r0);
                    tmemLd32NoWait(sAddr + 32u * c + 32u, r1);
                    tmemLdWait();
                    if (edge) {
                        maskBits(r0, s->rowBits[x][c][t]);
                        maskBits(r1, s->rowBits[x][c + 1][t]);
                    }
                    if (useLo) {
                        l += weightsRange<BF16, true, 0, 32>(r0, wgt, scaleLog2, negM);
                        tmemSt32(sAddr + 32u * c, wgt);
                        l += weightsRange<BF16, true, 0, 32>(r1, wgt, scaleLog2, negM);
                        tmemSt32(sAddr + 32u * c + 32u, wgt);
                    } else {
                        l += weightsRange<BF16, false, 0, 32>(r0, wgt, scaleLog2, negM);
                        tmemSt16(sAddr + 32u * c, wgt);
                        l += weightsRange<BF16, false, 0, 32>(r1, wgt, scaleLog2, negM);
                        tmemSt16(sAddr + 32u * c + 32u, wgt);
                    }
                }
                tmemStWait();
                if (edge) {
                    // Row t of V: finite values where there is no such key, or some row may not see it.
                    // (Both groups of a dual span may write the same.  The phase asked for is not two
                    // ahead: this S product was issued after the wait for V of the tile two before.)
                    const int half = 2 * (g.tile + j - g.first) + (t >> 6), st = half % S::kVStages;
                    ok = mbarWait(&s->vFull[st], (half / S::kVStages) & 1, &s->dead, errFlag, waitLimit, 53);
                    ok = __all_sync(0xFFFFFFFFu, ok);
                    if (!ok) break;
                    const uint32_t key = k0 + static_cast<uint32_t>(t);
                    const bool there = key < keyEnd && (inTree || key >= g.s.lo);
                    if (!there || inTree || key < g.hi) {
                        // A weight of zero removes what a row does not see, unless it is infinite or NaN: an
                        // exponent of ones, which carries out of its field when one is added at its end.
                        constexpr uint32_t kExp = BF16 ? 0x7F807F80u : 0x7C007C00u, kOne = BF16 ? 0x00800080u : 0x04000400u;
                        uint32_t carry = 0;
#pragma unroll 4
                        for (int c = 0; c < 8 * dimBlocks; ++c) {
                            // (lane by lane another piece of the row first: no two on one bank)
                            const uint4 w = *reinterpret_cast<const uint4*>(s->v[st] + (c >> 3) * kVBlockBytes + (t & 63) * 128 + (((c ^ t) & 7) << 4));
                            carry |= ((w.x & kExp) + kOne) | ((w.y & kExp) + kOne) | ((w.z & kExp) + kOne) | ((w.w & kExp) + kOne);
                        }
                        if (carry & 0x80008000u) {
#pragma unroll 1
                            for (int c = 0; c < 64 * dimBlocks; ++c) {
                                unsigned short* at = reinterpret_cast<unsigned short*>(s->v[st] + (c >> 6) * kVBlockBytes + (t & 63) * 128 + (c & 63) * 2);
                                if ((*at & kExp & 0xFFFFu) == (kExp & 0xFFFFu)) *at = 0;
                            }
                            if (there) odd = 1;
                        }
                    }
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                }
                if (lastTile) {
                    s->rowL[spans & 1][x][t] = l;
                    s->rowM[spans & 1][x][t] = mUsed;
                    s->rowOdd[spans & 1][x][t] = odd;
                }
                tcFenceBefore();
                mbarArrive(&s->pFull[x]);
            }
            if (!ok) break;
            ++spans;
            // (given back first: a ring full of spans without tiles of this group would wait for it)
            spanDone(k);
            k = seek(k + 1);
        }
    }

done:
    tcFenceBefore();
    __syncthreads();
    if (*reinterpret_cast<volatile int*>(&s->dead)) {
        // A wait ran out: neither the copies nor the products that are under way may outlive the block.
        auto drain = [&](unsigned long long* bar, uint32_t parity) {
            const long long t0 = clock64();
            while (!mbarTest(bar, parity) && clock64() - t0 < kDrainCycles) {}
        };
        if (threadIdx.x == 0) {
            constexpr int kRounds = FP8 ? 2 : 1;
            for (int i = max(0, s->issuedK - kRounds * S::kKStages); i < s->issuedK; ++i) drain(&s->kFull[i % S::kKStages], (i / S::kKStages) & 1);
            for (int i = max(0, s->issuedV - kRounds * S::kVStages); i < s->issuedV; ++i) drain(&s->vFull[i % S::kVStages], (i / S::kVStages) & 1);
            for (int i = max(0, s->issuedRaw - S::kRawStages); i < s->issuedRaw; ++i) drain(&s->rawFull[i % S::kRawStages], (i / S::kRawStages) & 1);
            if (s->issuedQ > 0) drain(&s->qFull, (s->issuedQ - 1) & 1);
        }
        if (warp == kMmaWarp && live) {
            if (electOne()) {
                ummaCommit(&s->drained);
                drain(&s->drained, 0);
            }
            __syncwarp();
        }
        __syncthreads();
    }
    if (warp == kMmaWarp) {
        tcFenceAfter();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
    }
}

}  // namespace

bool treeTcSizes(const TreeParams& p) {
    return p.dtype != kF32 && p.headDim >= 64 && p.headDim <= kHd && p.headDim % 16 == 0 && p.blockSize % (p.dtype == kFP8 ? 16 : 8) == 0;
}

bool treeTcApplies(const TreeParams& p) {
    if (!treeTcSizes(p)) return false;
    if (p.dtype == kFP8 && smemBytes<false, true>(p.batch) > kSmemLimit) return false;
    // (rows of the pool are counted in 32 bits; a pool of unknown length is not taken, since the tensor maps need one)
    if (p.poolBlocks <= 0 || p.poolBlocks >= (1 << 30) / (p.kvHeads * p.blockSize)) return false;
    for (int64_t s : {p.qStride, p.kStride, p.vStride})
        if (s % 8) return false;
    for (const void* ptr : {p.q, p.kNew, p.vNew, p.kPool, p.vPool, static_cast<const void*>(p.out)})
        if (reinterpret_cast<uintptr_t>(ptr) & 15) return false;
    return true;
}

// Two query tiles: when a request can have more than 128 rows under a KV head, or the batch's list does
// not fit beside the longer rings.  Over FP8 pages row tiles are taken one after the other: the ring of
// codes leaves room for two query tiles and one tile of V, which then waits for the products of the
// tile before (both measured before pages of odd scales were told apart: 32 requests of 4096 tokens, 256 rows: 201 us,
// against 207, now 219; one of 8192 tokens 37 against 31).
static bool takesWide(const TreeParams& p) {
    return p.dtype != kFP8 && (static_cast<int64_t>(p.maxNew) * (p.heads / p.kvHeads) > kRows || smemBytes<false, false>(p.batch) > kSmemLimit);
}

TreePlan treeTcPlan(const TreeParams& p, int smCount) {
    TreePlan t{};
    t.variant = 2;
    t.rows = takesWide(p) ? 256 : 128;
    t.keys = kKeys;
    t.dimPad = kHd;
    t.blocks = smCount;
    return t;
}

cudaError_t launchTreeTc(const TreeParams& p, const TreePlan& plan, cudaStream_t stream) {
    EncodeFn encode = encodeFn();
    if (!encode) return cudaErrorNotSupported;
    const CUtensorMapDataType dt = p.dtype == kBF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    const cuuint64_t D = p.headDim;
    CUtensorMap queries, pool[2], fresh[2];
    {
        // queries: [row][head][128]; a box is 64 dims x the heads of a KV head x 128 rows' worth of nodes
        // (used when the group divides 128; else any valid box)
        const int group = p.heads / p.kvHeads, nodes = kRows % group == 0 ? kRows / group : 1, heads = kRows % group == 0 ? group : 1;
        const cuuint64_t dims[3] = {D, static_cast<cuuint64_t>(p.heads), static_cast<cuuint64_t>(p.numRows)};
        const cuuint64_t strides[2] = {D * 2, static_cast<cuuint64_t>(p.qStride) * 2};
        const cuuint32_t box[3] = {64, static_cast<cuuint32_t>(heads), static_cast<cuuint32_t>(nodes)}, one[3] = {1, 1, 1};
        if (encode(&queries, dt, 3, const_cast<void*>(p.q), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                   CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
            return cudaErrorInvalidValue;
    }
    for (int which = 0; which < 2; ++which) {
        if (p.dtype != kFP8) {
        // pools: [block * kv_head * slot][128]; a box is 64 dims x 16 or 8 rows
        const cuuint64_t dims[2] = {D, static_cast<cuuint64_t>(p.poolBlocks) * p.kvHeads * p.blockSize};
        const cuuint64_t strides[1] = {D * 2};
        const cuuint32_t box[2] = {64, p.blockSize % 16 == 0 ? 16u : 8u}, one[2] = {1, 1};
        if (encode(&pool[which], dt, 2, const_cast<void*>(which ? p.vPool : p.kPool), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                   CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
            return cudaErrorInvalidValue;
        }
        // the step's rows: [row][kv_head][128]; a box is 64 dims x 1 head x 64 rows (rows behind the last: zeros)
        const cuuint64_t fdims[3] = {D, static_cast<cuuint64_t>(p.kvHeads), static_cast<cuuint64_t>(p.numRows)};
        const cuuint64_t fstrides[2] = {D * 2, static_cast<cuuint64_t>(which ? p.vStride : p.kStride) * 2};
        const cuuint32_t fbox[3] = {64, 1, 64}, fone[3] = {1, 1, 1};
        if (encode(&fresh[which], dt, 3, const_cast<void*>(which ? p.vNew : p.kNew), fdims, fstrides, fbox, fone, CU_TENSOR_MAP_INTERLEAVE_NONE,
                   CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
            return cudaErrorInvalidValue;
    }
    const float scaleLog2 = 1.4426950408889634f / sqrtf(static_cast<float>(p.headDim));
    auto run = [&](auto kernel, int threads, size_t smem) -> cudaError_t {
        cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kSmemLimit));
        if (e != cudaSuccess) return e;
        return launchEarly(kernel, dim3(plan.blocks), threads, smem, stream, queries, pool[0], pool[1], fresh[0], fresh[1], p, scaleLog2,
                           p.errFlag, p.waitCycles > 0 ? p.waitCycles : kWaitCycles);
    };
    auto whole = [&](auto known) -> cudaError_t {
        constexpr bool W = decltype(known)::value;
        if (p.dtype == kFP8) {
            pool[0] = pool[1] = queries;               // (not read)
            return run(treeTcKernel<false, false, true, W>, kThreads<true>, smemBytes<false, true>(p.batch));
        }
        if (takesWide(p)) {
            const size_t smem = smemBytes<true, false>(p.batch);
            return p.dtype == kBF16 ? run(treeTcKernel<true, true, false, W>, kThreads<false>, smem) : run(treeTcKernel<false, true, false, W>, kThreads<false>, smem);
        }
        const size_t smem = smemBytes<false, false>(p.batch);
        return p.dtype == kBF16 ? run(treeTcKernel<true, false, false, W>, kThreads<false>, smem) : run(treeTcKernel<false, false, false, W>, kThreads<false>, smem);
    };
    return p.headDim == kHd ? whole(std::true_type{}) : whole(std::false_type{});
}

}  // namespace pam
