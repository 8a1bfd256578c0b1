// Tree attention for 16-bit and FP8 pools where the tcgen05 kernel does not apply (head_dim below 64 or
// not a multiple of 16, FP8 pages that are not multiples of 16 tokens, very large batches of FP8, pools of unknown
// length) and for calls too short for it, on mma.sync.m16n8k16.  A key costs 4 head_dim bytes and 4 head_dim flops per
// row, so that 16 rows ask for 16 flops a byte, where the legacy tensor pipe gives several times that;
// at 64 rows the two come close.  Measured with 32 requests of 4096 tokens, 8 KV heads of 128, bfloat16:
// 4 rows 121 us = 0.68 of the copy rate, 64 rows 231 us, 256 rows 821 us (a row tile of 64 after the
// other, each of which reads the keys again); one request of 1024 tokens, 4 rows, 12.6 us.
//
// A block has four warps and walks its piece of the tile list (tree_common.cuh) in key tiles of 64.
// MR = 16, 32 or 64 rows: the warps split into MR / 16 row groups and, where there are fewer than
// four of those, the keys of every tile among 4 / (MR / 16) key groups, each with its own running
// maximum, sum and accumulator; they are joined in shared memory at the end of a pair's part.  Keys
// and values come through a ring of cp.async stages, 16 bytes at a time, each row from the address
// that a lane looked up one tile earlier (page of a block table, or row of the tree): pages may
// be of any size, rows that no query of the request sees are filled with zeros.  The loads run ahead over
// the ends of pairs.  One block-wide wait per tile.
//
// FP8: the ring holds codes; a pass over the arrived tile turns them into float16, exactly (every
// e4m3 value is a float16 value).  The key scale multiplies the scores; the value scale the weights,
// with the running maximum kept over (score + exponent of the value scale): the weights that go
// into the second product as float16 then stay near 1 however small the scales are.
//
// The weights go into the second product in the type of the values: half a step of it per weight,
// at random, against the half step of the result itself.  For bfloat16 that is 2^-8 (see twoOperands).
#include <algorithm>
#include <atomic>
#include <cmath>
#include <type_traits>

#include "tree_common.cuh"

namespace pam {
namespace {

using namespace tree;

constexpr int kThreads = 128, kKeys = 64;
constexpr float kRaise = 6.f;             // the running maximum moves when it is passed by 2^6
// Weights are kept times 2^9, as far up as that leaves float16 room (2^15): those down to 2^-23 of a row's reference
// then keep all their bits, not those down to 2^-14 alone.  (bfloat16 has float32's range.)
template <typename T> constexpr float kWeightLift = std::is_same<T, __half>::value ? 9.f : 0.f;

__device__ __forceinline__ uint32_t smemAddr(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }
__device__ __forceinline__ void ldmatrixX4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];\n"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ void ldmatrixX4Trans(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];\n"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
template <typename T> __device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <> __device__ __forceinline__ void mma16816<__half>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <> __device__ __forceinline__ void mma16816<__nv_bfloat16>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <typename T> __device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <> __device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
    __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&h);
}
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
    __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&h);
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// 16 bytes to shared memory; zeros when there is no source.
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool there) {
    const int n = there ? 16 : 0;
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void commitGroup() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void waitGroups() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// Where the rows of one tile come from (0: nowhere), and for FP8 their scales.  Values whose scale is not a finite
// number come from nowhere, and `odd` says so for either half of the rows (see addLeftOut).
struct RowSource {
    unsigned long long k[kKeys], v[kKeys];
    float kScale[kKeys], vScale[kKeys], vExp[kKeys];
    int odd[2];
};

template <int HD, int MR, bool FP8>
struct Shape {
    static constexpr int kStages = FP8 ? 4 : 3;
    static constexpr int kRowGroups = MR / 16, kKeyGroups = 4 / kRowGroups, kWarpKeys = kKeys / kKeyGroups;
    static constexpr int kRowBytes = HD * 2, kTileBytes = kKeys * kRowBytes;           // a 16-bit tile
    static constexpr int kRawRow = FP8 ? HD : HD * 2, kRawTile = kKeys * kRawRow;      // as it arrives
    static constexpr int kMergeFloats = (HD / 2 + 4) * 32;                             // one warp's state
    static constexpr size_t bytes(int batch) {
        return static_cast<size_t>(kStages) * 2 * kRawTile + (FP8 ? 2 * kTileBytes : 0) + (kStages + 1) * sizeof(RowSource) +
               kMergeFloats * sizeof(float) + (8 + static_cast<size_t>(batch) + 1) * sizeof(int);
    }
};

// Two codes to two float16 values.
__device__ __forceinline__ uint32_t widen(uint32_t codes) {
    uint32_t r;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(static_cast<unsigned short>(codes)));
    return r;
}

template <typename T, int HD, int MR, bool FP8>
__global__ void __launch_bounds__(kThreads, 2)
treeMmaKernel(const __grid_constant__ TreeParams p, float scaleLog2) {
    using S = Shape<HD, MR, FP8>;
    constexpr int NB = S::kWarpKeys / 8;                  // key blocks of 8 of a warp
    extern __shared__ __align__(128) unsigned char raw[];
    unsigned char* ring = raw;                            // [stage][K, V][64 rows]
    unsigned char* wide = ring + static_cast<size_t>(S::kStages) * 2 * S::kRawTile;     // FP8: the tile as float16
    RowSource* sources = reinterpret_cast<RowSource*>(wide + (FP8 ? 2 * S::kTileBytes : 0));
    float* merge = reinterpret_cast<float*>(sources + S::kStages + 1);
    int* scratch = reinterpret_cast<int*>(merge + S::kMergeFloats);
    int* prefix = scratch + 8;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int rowGroup = warp % S::kRowGroups, keyGroup = warp / S::kRowGroups;
    const int gr = lane >> 2, gc = lane & 3;
    cudaGridDependencySynchronize();                      // launched early, as treeTcKernel
    buildPrefix<MR, kKeys, kThreads>(p, prefix, scratch);
    const int blocks = gridDim.x, me = blockIdx.x, total = prefix[p.batch];
    const int quota = (total + blocks - 1) / blocks;
    const int begin = static_cast<int>(min(static_cast<long long>(me) * quota, static_cast<long long>(total))), end = min(total, begin + quota);
    const int group = p.heads / p.kvHeads, D = p.headDim;
    if (tid == 0) {
        Header h{};
        h.lastBlock = -1;
        *headerOf(p, me) = h;
    }
    if (begin >= end) return;

    // ---- the loads' place in the list, ahead of the arithmetic
    Segment ahead = segmentAt<MR, kKeys>(p, prefix, begin, end);
    int aheadT = begin, aheadJ = ahead.first;
    // addresses of the next tile's rows: threads 0 .. 63 the keys', 64 .. 127 the values'
    auto findRows = [&]() {
        if (aheadT >= end) return;
        RowSource& r = sources[(aheadT - begin) % (S::kStages + 1)];
        const int cacheTiles = ahead.s.cacheTiles<kKeys>(), i = tid & 63;
        const bool isV = tid >= 64, inTree = aheadJ >= cacheTiles;
        unsigned long long at = 0;
        bool leftOut = false;
        if (inTree) {
            const int node = (aheadJ - cacheTiles) * kKeys + i;
            if (node < ahead.s.n)
                at = reinterpret_cast<unsigned long long>(static_cast<const T*>(isV ? p.vNew : p.kNew) +
                                                          static_cast<int64_t>(ahead.s.start + node) * (isV ? p.vStride : p.kStride) +
                                                          static_cast<int64_t>(ahead.kvh) * D);
            if (FP8) {
                if (isV) { r.vScale[i] = 1.f; r.vExp[i] = 0.f; }
                else r.kScale[i] = 1.f;
            }
        } else {
            const uint32_t token = (ahead.s.lo / kKeys + aheadJ) * kKeys + i;
            int64_t blk = 0;
            if (token >= ahead.s.lo && token < ahead.s.held) {
                const int64_t row = poolRow(p, ahead.b, token, ahead.kvh, &blk);
                at = reinterpret_cast<unsigned long long>(static_cast<const unsigned char*>(isV ? p.vPool : p.kPool) + row * (FP8 ? 1 : 2));
            }
            if (FP8) {
                const __half scale = at ? static_cast<const __half*>(isV ? p.vScale : p.kScale)[blk * p.kvHeads + ahead.kvh] : __float2half_rn(1.f);
                if (isV) {
                    float s = __half2float(scale);
                    if (isOdd(s)) { s = 1.f; at = 0; leftOut = true; }
                    r.vScale[i] = s;
                    r.vExp[i] = s > 0.f ? static_cast<float>(ilogbf(s) + 1) : -25.f;
                } else {
                    r.kScale[i] = keyScaleOf(scale);
                }
            }
        }
        if (FP8 && isV) {
            leftOut = __any_sync(0xFFFFFFFFu, leftOut);
            if (lane == 0) r.odd[warp & 1] = leftOut ? 1 : 0;
        }
        (isV ? r.v : r.k)[i] = at;
        ++aheadT;
        if (++aheadJ == ahead.last && aheadT < end) {
            ahead = segmentAt<MR, kKeys>(p, prefix, aheadT, end);
            aheadJ = ahead.first;
        }
    };
    // the rows of tile t (counted from the piece's begin) into its stage
    auto issue = [&](int t) {
        if (begin + t < end) {
            const RowSource& r = sources[t % (S::kStages + 1)];
            const uint32_t base = smemAddr(ring + static_cast<size_t>(t % S::kStages) * 2 * S::kRawTile);
            constexpr int CPR = S::kRawRow / 16;
            const int chunks = D * (FP8 ? 1 : 2) / 16;
#pragma unroll
            for (int i = 0; i < 2 * kKeys * CPR / kThreads; ++i) {
                const int idx = tid + kThreads * i, row = idx / CPR, c = idx % CPR;     // rows 0 .. 63: K, 64 .. 127: V
                const unsigned long long at = row < kKeys ? r.k[row] : r.v[row - kKeys];
                const bool there = at != 0 && c < chunks;
                const uint32_t dst = base + row * S::kRawRow + (FP8 ? c * 16 : ((c ^ (row & 7)) << 4));
                copy16(dst, reinterpret_cast<const void*>(there ? at + c * 16 : reinterpret_cast<unsigned long long>(p.kPool)), there);
            }
        }
        commitGroup();
    };
    // (a tree's rows are 16 bits wide, not codes: the ring skips them and the arithmetic fetches them)
    auto skipsRing = [&](const Segment& g, int j) { return FP8 && j >= g.s.cacheTiles<kKeys>(); };

    int skipBits = 0;                                         // bit t % 8: tile t skips the ring
    for (int i = 0; i <= S::kStages; ++i) {
        if (aheadT < end && skipsRing(ahead, aheadJ)) skipBits |= 1 << i;
        findRows();
    }
    __syncthreads();
    auto issueOrSkip = [&](int t) {
        if (FP8 && (skipBits >> (t & 7) & 1)) commitGroup();
        else issue(t);
    };
    for (int i = 0; i < S::kStages - 1; ++i) issueOrSkip(i);

    Segment g;
    uint32_t qf[HD / 16][4];
    float o[HD / 8][4];
    float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;
    int node0 = 0, node1 = 0, rows = 0, j = 0, segT = begin;
    uint32_t first0 = 0, first1 = 0, hi = 0;
    bool odd = false, two = false;
    int segEnd = begin;                                       // list index behind the current segment
    for (int t = 0; begin + t < end; ++t) {
        if (begin + t == segEnd) {
            // ---- a new pair: its rows' queries, windows and masks
            segT = segEnd;
            g = segmentAt<MR, kKeys>(p, prefix, segT, end);
            segEnd = segT + g.last - g.first;
            j = g.first;
            rows = g.s.n * group;
            hi = lastFirst(p, g.s, g.rt, MR);
            const int r0 = g.rt * MR + 16 * rowGroup + gr, r1 = r0 + 8;
            node0 = min(r0 / group, g.s.n - 1);
            node1 = min(r1 / group, g.s.n - 1);
            first0 = firstOf(p, g.s, node0);
            first1 = firstOf(p, g.s, node1);
            const T* q0 = static_cast<const T*>(p.q) + static_cast<int64_t>(g.s.start + node0) * p.qStride + static_cast<int64_t>(g.kvh * group + r0 % group) * D;
            const T* q1 = static_cast<const T*>(p.q) + static_cast<int64_t>(g.s.start + node1) * p.qStride + static_cast<int64_t>(g.kvh * group + r1 % group) * D;
#pragma unroll
            for (int ks = 0; ks < HD / 16; ++ks)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int d = 16 * ks + 8 * h + 2 * gc;
                    qf[ks][2 * h] = r0 < rows && d < D ? *reinterpret_cast<const uint32_t*>(q0 + d) : 0u;
                    qf[ks][2 * h + 1] = r1 < rows && d < D ? *reinterpret_cast<const uint32_t*>(q1 + d) : 0u;
                }
#pragma unroll
            for (int n = 0; n < HD / 8; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[n][e] = 0.f;
            m0 = m1 = -INFINITY;
            l0 = l1 = 0.f;
            odd = false;
            two = std::is_same<T, __nv_bfloat16>::value && twoOperands(p, g.s);
        }
        const int cacheTiles = g.s.cacheTiles<kKeys>();
        const bool inTree = j >= cacheTiles;
        const uint32_t k0 = inTree ? static_cast<uint32_t>(j - cacheTiles) * kKeys : (g.s.lo / kKeys + j) * kKeys;
        waitGroups<S::kStages - 2>();
        __syncthreads();
        issueOrSkip(t + S::kStages - 1);
        // the addresses of the tile behind those under way (the slot that tile t - 1 used: `sources`
        // has one more than the ring)
        if (t > 0 && aheadT < end) {
            const int bit = (t + S::kStages) & 7;
            skipBits = (skipBits & ~(1 << bit)) | (skipsRing(ahead, aheadJ) ? 1 << bit : 0);
            findRows();
        }
        unsigned char* kTile = ring + static_cast<size_t>(t % S::kStages) * 2 * S::kRawTile;
        unsigned char* vTile = kTile + S::kRawTile;
        const RowSource& src = sources[t % (S::kStages + 1)];
        if (FP8) {
            if (inTree) {
                constexpr int CPR = S::kRowBytes / 16;
                for (int i = tid; i < 2 * kKeys * CPR; i += kThreads) {
                    const int row = i / CPR, c = i % CPR;
                    const unsigned long long at = row < kKeys ? src.k[row] : src.v[row - kKeys];
                    uint4 w = make_uint4(0u, 0u, 0u, 0u);
                    if (at && c * 8 < D) w = *reinterpret_cast<const uint4*>(at + c * 16);
                    *reinterpret_cast<uint4*>(wide + row * S::kRowBytes + ((c ^ (row & 7)) << 4)) = w;
                }
            } else {
                constexpr int CPR = S::kRawRow / 16;                 // 16 codes become two chunks
#pragma unroll 4
                for (int i = tid; i < 2 * kKeys * CPR; i += kThreads) {
                    const int row = i / CPR, c = i % CPR;
                    const uint4 w = *reinterpret_cast<const uint4*>(kTile + row * S::kRawRow + c * 16);
                    const uint4 a = make_uint4(widen(w.x), widen(w.x >> 16), widen(w.y), widen(w.y >> 16));
                    const uint4 b = make_uint4(widen(w.z), widen(w.z >> 16), widen(w.w), widen(w.w >> 16));
                    unsigned char* dst = wide + row * S::kRowBytes;
                    *reinterpret_cast<uint4*>(dst + (((2 * c) ^ (row & 7)) << 4)) = a;
                    *reinterpret_cast<uint4*>(dst + (((2 * c + 1) ^ (row & 7)) << 4)) = b;
                }
            }
            kTile = wide;
            vTile = wide + S::kTileBytes;
            __syncthreads();
        }
        if (inTree || k0 < hi) {
            // values that are not finite, of keys that some row may not see (tree_common.cuh)
            constexpr int CPR = S::kRowBytes / 16;
            constexpr uint32_t kExp = std::is_same<T, __half>::value ? 0x7C00u : 0x7F80u;
            bool found = false;
            for (int i = tid; i < kKeys * CPR; i += kThreads) {
                const int row = i / CPR;
                if (!inTree && k0 + row >= hi) continue;
                uint32_t* w = reinterpret_cast<uint32_t*>(vTile + row * S::kRowBytes + (i % CPR) * 16);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    uint32_t x = w[e];
                    if ((x & kExp) == kExp) x &= 0xFFFF0000u;
                    if ((x >> 16 & kExp) == kExp) x &= 0x0000FFFFu;
                    if (x != w[e]) { w[e] = x; found = true; }
                }
            }
            odd = __syncthreads_or(found) || odd;
        }
        if (FP8) odd = odd || src.odd[0] != 0 || src.odd[1] != 0;
        // ---- scores of this warp's rows and keys
        float s[NB][4];
#pragma unroll
        for (int n = 0; n < NB; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[n][e] = 0.f;
        const uint32_t kBase = smemAddr(kTile), vBase = smemAddr(vTile);
        const int keyBase = keyGroup * S::kWarpKeys;
#pragma unroll
        for (int ks = 0; ks < HD / 16; ++ks)
#pragma unroll
            for (int n = 0; n < NB; n += 2) {
                const int key = keyBase + 8 * n + 8 * (lane >> 4) + (lane & 7), c = 2 * ks + ((lane >> 3) & 1);
                uint32_t b[4];
                ldmatrixX4(b, kBase + key * S::kRowBytes + ((c ^ (key & 7)) << 4));
                mma16816<T>(s[n], qf[ks], b[0], b[1]);
                mma16816<T>(s[n + 1], qf[ks], b[2], b[3]);
            }
        const bool edge = inTree || k0 < hi || k0 < g.s.lo || k0 + kKeys > g.s.held;
        float top0 = -INFINITY, top1 = -INFINITY;
        unsigned long long bits0 = ~0ull, bits1 = ~0ull;       // keys of the tile that the two rows see
        if (edge) {
            if (inTree) {
                const int w = static_cast<int>(k0 / 32);
                bits0 = treeBits(p, g.s, node0, w) | static_cast<unsigned long long>(treeBits(p, g.s, node0, w + 1)) << 32;
                bits1 = treeBits(p, g.s, node1, w) | static_cast<unsigned long long>(treeBits(p, g.s, node1, w + 1)) << 32;
            } else {
                auto range = [&](uint32_t from) {
                    const int a = from > k0 ? static_cast<int>(min(from - k0, 64u)) : 0, b = static_cast<int>(min(g.s.held - k0, 64u));
                    const unsigned long long below = b >= 64 ? ~0ull : (1ull << b) - 1ull;
                    return a >= 64 ? 0ull : below & (~0ull << a);
                };
                bits0 = range(max(first0, g.s.lo));
                bits1 = range(max(first1, g.s.lo));
            }
        }
        bits0 >>= keyBase;
        bits1 >>= keyBase;
#pragma unroll
        for (int n = 0; n < NB; ++n) {
            float f0 = scaleLog2, f1 = scaleLog2, e0 = 0.f, e1 = 0.f;
            if (FP8) {
                const int c = keyBase + 8 * n + 2 * gc;
                f0 *= src.kScale[c];
                f1 *= src.kScale[c + 1];
                e0 = src.vExp[c];
                e1 = src.vExp[c + 1];
            }
            s[n][0] *= f0; s[n][1] *= f1; s[n][2] *= f0; s[n][3] *= f1;
            if (edge) {
                const int c = 8 * n + 2 * gc;
                if (!(bits0 >> c & 1)) s[n][0] = -INFINITY;
                if (!(bits0 >> (c + 1) & 1)) s[n][1] = -INFINITY;
                if (!(bits1 >> c & 1)) s[n][2] = -INFINITY;
                if (!(bits1 >> (c + 1) & 1)) s[n][3] = -INFINITY;
            }
            top0 = fmaxf(top0, fmaxf(s[n][0] + e0, s[n][1] + e1));
            top1 = fmaxf(top1, fmaxf(s[n][2] + e0, s[n][3] + e1));
        }
#pragma unroll
        for (int x = 1; x < 4; x <<= 1) {
            top0 = fmaxf(top0, __shfl_xor_sync(0xFFFFFFFFu, top0, x));
            top1 = fmaxf(top1, __shfl_xor_sync(0xFFFFFFFFu, top1, x));
        }
        const bool up0 = top0 > m0 + kRaise, up1 = top1 > m1 + kRaise;      // (from -inf: always)
        if (__any_sync(0xFFFFFFFFu, up0 || up1)) {
            const float c0 = up0 ? ex2(m0 - top0) : 1.f, c1 = up1 ? ex2(m1 - top1) : 1.f;
            if (up0) m0 = top0;
            if (up1) m1 = top1;
            l0 *= c0;
            l1 *= c1;
#pragma unroll
            for (int n = 0; n < HD / 8; ++n) { o[n][0] *= c0; o[n][1] *= c0; o[n][2] *= c1; o[n][3] *= c1; }
        }
        const float b0 = m0 == -INFINITY ? 0.f : m0 - kWeightLift<T>, b1 = m1 == -INFINITY ? 0.f : m1 - kWeightLift<T>;
#pragma unroll
        for (int n = 0; n < NB; ++n) {
            s[n][0] = ex2(s[n][0] - b0); s[n][1] = ex2(s[n][1] - b0);
            s[n][2] = ex2(s[n][2] - b1); s[n][3] = ex2(s[n][3] - b1);
            l0 += s[n][0] + s[n][1];
            l1 += s[n][2] + s[n][3];
            if (FP8) {
                const int c = keyBase + 8 * n + 2 * gc;
                const float v0 = src.vScale[c], v1 = src.vScale[c + 1];
                s[n][0] *= v0; s[n][1] *= v1; s[n][2] *= v0; s[n][3] *= v1;
            }
        }
        // ---- weights times values
#pragma unroll
        for (int kk = 0; kk < NB / 2; ++kk) {
            uint32_t a[4], lo[4];
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const float x = s[2 * kk + h][2 * e], y = s[2 * kk + h][2 * e + 1];
                    a[2 * h + e] = pack2<T>(x, y);
                    if (std::is_same<T, __nv_bfloat16>::value && two)
                        lo[2 * h + e] = pack2<T>(x - __uint_as_float(a[2 * h + e] << 16), y - __uint_as_float(a[2 * h + e] & 0xFFFF0000u));
                }
#pragma unroll
            for (int n = 0; n < HD / 8; n += 2) {
                const int key = keyBase + 16 * kk + (lane & 15), c = n + (lane >> 4);
                uint32_t b[4];
                ldmatrixX4Trans(b, vBase + key * S::kRowBytes + ((c ^ (key & 7)) << 4));
                mma16816<T>(o[n], a, b[0], b[1]);
                mma16816<T>(o[n + 1], a, b[2], b[3]);
                if (std::is_same<T, __nv_bfloat16>::value && two) {
                    mma16816<T>(o[n], lo, b[0], b[1]);
                    mma16816<T>(o[n + 1], lo, b[2], b[3]);
                }
            }
        }
        ++j;
        if (begin + t + 1 != segEnd) continue;

        // ---- the end of this block's part of the pair
#pragma unroll
        for (int x = 1; x < 4; x <<= 1) {
            l0 += __shfl_xor_sync(0xFFFFFFFFu, l0, x);
            l1 += __shfl_xor_sync(0xFFFFFFFFu, l1, x);
        }
        if (S::kKeyGroups > 1) {
            // key groups 1, 2, .. of every row group into its first, one after the other
#pragma unroll 1
            for (int step = 0; step < S::kRowGroups * (S::kKeyGroups - 1); ++step) {
                const int rg = step % S::kRowGroups, kg = 1 + step / S::kRowGroups;
                __syncthreads();
                if (rowGroup == rg && keyGroup == kg) {
#pragma unroll
                    for (int n = 0; n < HD / 8; ++n)
#pragma unroll
                        for (int e = 0; e < 4; ++e) merge[(4 * n + e) * 32 + lane] = o[n][e];
                    merge[(HD / 2) * 32 + lane] = m0;
                    merge[(HD / 2 + 1) * 32 + lane] = m1;
                    merge[(HD / 2 + 2) * 32 + lane] = l0;
                    merge[(HD / 2 + 3) * 32 + lane] = l1;
                }
                __syncthreads();
                if (rowGroup == rg && keyGroup == 0) {
                    const float n0 = merge[(HD / 2) * 32 + lane], n1 = merge[(HD / 2 + 1) * 32 + lane];
                    const float t0 = fmaxf(m0, n0), t1 = fmaxf(m1, n1);
                    const float z0 = t0 == -INFINITY ? 0.f : t0, z1 = t1 == -INFINITY ? 0.f : t1;
                    const float a0 = ex2(m0 - z0), a1 = ex2(m1 - z1), c0 = ex2(n0 - z0), c1 = ex2(n1 - z1);
                    m0 = t0;
                    m1 = t1;
                    l0 = l0 * a0 + merge[(HD / 2 + 2) * 32 + lane] * c0;
                    l1 = l1 * a1 + merge[(HD / 2 + 3) * 32 + lane] * c1;
#pragma unroll
                    for (int n = 0; n < HD / 8; ++n) {
                        o[n][0] = o[n][0] * a0 + merge[(4 * n) * 32 + lane] * c0;
                        o[n][1] = o[n][1] * a0 + merge[(4 * n + 1) * 32 + lane] * c0;
                        o[n][2] = o[n][2] * a1 + merge[(4 * n + 2) * 32 + lane] * c1;
                        o[n][3] = o[n][3] * a1 + merge[(4 * n + 3) * 32 + lane] * c1;
                    }
                }
            }
        }
        const bool whole = g.whole();
        const int which = g.first == 0 ? 1 : 0;
        if (!whole && tid == 0) {
            Header* h = headerOf(p, me);
            h->odd[which] = odd ? 1 : 0;
            if (which == 1) {
                h->b = g.b; h->kvh = g.kvh; h->rt = g.rt;
                h->lastBlock = (segT + g.nT - 1) / quota;
            }
        }
        if (keyGroup != 0) continue;
        float* rec = whole ? nullptr : recordOf(p, blocks, me, which, MR, HD);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int rl = 16 * rowGroup + gr + 8 * h, rr = g.rt * MR + rl;
            if (rr >= rows) continue;
            const float l = h ? l1 : l0;
            if (whole) {
                const float inv = l == 0.f ? 0.f : 1.f / l;
                T* out = static_cast<T*>(p.out) + (static_cast<int64_t>(g.s.start + rr / group) * p.heads + g.kvh * group + rr % group) * D;
#pragma unroll
                for (int n = 0; n < HD / 8; ++n) {
                    const int d = 8 * n + 2 * gc;
                    if (d >= D) continue;
                    *reinterpret_cast<uint32_t*>(out + d) = pack2<T>(o[n][2 * h] * inv, o[n][2 * h + 1] * inv);
                }
            } else {
#pragma unroll
                for (int n = 0; n < HD / 8; ++n)
                    *reinterpret_cast<float2*>(rec + rl * HD + 8 * n + 2 * gc) = make_float2(o[n][2 * h], o[n][2 * h + 1]);
                if (gc == 0) {
                    rec[MR * HD + rl] = h ? m1 : m0;
                    rec[MR * HD + MR + rl] = l;
                }
            }
        }
        if (whole && odd) {
            __syncwarp();
            for (int h = 0; h < 2; ++h) {
                const int rr = g.rt * MR + 16 * rowGroup + gr + 8 * h;
                if (gc == 0 && rr < rows)
                    addLeftOut<T, std::conditional_t<FP8, uint8_t, T>>(p, g.s, g.b, g.kvh, rr / group, hi,
                        static_cast<T*>(p.out) + (static_cast<int64_t>(g.s.start + rr / group) * p.heads + g.kvh * group + rr % group) * D, 0, D);
            }
            __syncwarp();
        }
    }
    waitGroups<0>();
}

template <typename T, int HD, int MR, bool FP8>
cudaError_t launchOne(const TreeParams& p, int blocks, float scaleLog2, cudaStream_t stream) {
    static std::atomic<unsigned long long> done{0};
    using S = Shape<HD, MR, FP8>;
    const cudaError_t e = allowSmem(treeMmaKernel<T, HD, MR, FP8>, S::bytes(kTreeMaxBatch), done);
    if (e != cudaSuccess) return e;
    return launchEarly(treeMmaKernel<T, HD, MR, FP8>, dim3(blocks), kThreads, S::bytes(p.batch), stream, p, scaleLog2);
}

template <typename T, bool FP8>
cudaError_t launchShape(const TreeParams& p, const TreePlan& plan, float scaleLog2, cudaStream_t stream) {
    if (plan.dimPad == 64) {
        if (plan.rows == 16) return launchOne<T, 64, 16, FP8>(p, plan.blocks, scaleLog2, stream);
        if (plan.rows == 32) return launchOne<T, 64, 32, FP8>(p, plan.blocks, scaleLog2, stream);
        return launchOne<T, 64, 64, FP8>(p, plan.blocks, scaleLog2, stream);
    }
    if (plan.rows == 16) return launchOne<T, 128, 16, FP8>(p, plan.blocks, scaleLog2, stream);
    if (plan.rows == 32) return launchOne<T, 128, 32, FP8>(p, plan.blocks, scaleLog2, stream);
    return launchOne<T, 128, 64, FP8>(p, plan.blocks, scaleLog2, stream);
}

}  // namespace

bool treeMmaSizes(const TreeParams& p) {
    // 16-byte pieces: of codes 16 dims, of 16-bit values 8
    return p.dtype != kF32 && p.headDim <= 128 && p.headDim % (p.dtype == kFP8 ? 16 : 8) == 0;
}

bool treeMmaApplies(const TreeParams& p) {
    if (!treeMmaSizes(p)) return false;
    for (int64_t s : {p.qStride, p.kStride, p.vStride})
        if (s % 8) return false;
    for (const void* ptr : {p.q, p.kNew, p.vNew, p.kPool, p.vPool, static_cast<const void*>(p.out)})
        if (reinterpret_cast<uintptr_t>(ptr) & 15) return false;
    return true;
}

TreePlan treeMmaPlan(const TreeParams& p, int smCount) {
    TreePlan t{};
    const int64_t rows = static_cast<int64_t>(p.maxNew) * (p.heads / p.kvHeads);
    t.variant = 1;
    t.rows = rows <= 16 ? 16 : rows <= 32 ? 32 : 64;
    t.keys = kKeys;
    t.dimPad = p.headDim <= 64 ? 64 : 128;
    t.blocks = 2 * smCount;
    return t;
}

cudaError_t launchTreeMma(const TreeParams& p, const TreePlan& plan, cudaStream_t stream) {
    const float scaleLog2 = 1.4426950408889634f / sqrtf(static_cast<float>(p.headDim));
    if (p.dtype == kF16) return launchShape<__half, false>(p, plan, scaleLog2, stream);
    if (p.dtype == kBF16) return launchShape<__nv_bfloat16, false>(p, plan, scaleLog2, stream);
    return launchShape<__half, true>(p, plan, scaleLog2, stream);
}

}  // namespace pam
