// Attention of draft trees over the paged cache: the choice of kernel, the general kernel and
// the kernel that joins the records of shared pairs.  The layout of the work is explained in
// tree_common.cuh.
//
//   out_i = sum_j p_ij v_j / sum_j p_ij,   p_ij = exp(q_i . k_j / sqrt(dim)),
//
// over the cache tokens of node i's window and the nodes of its mask; a row that sees nothing is
// zero.  Scores are kept times log2(e), so that the weights are powers of two.
#include <algorithm>
#include <atomic>
#include <cmath>

#include "tree_common.cuh"

namespace pam {
namespace {

using namespace tree;

// ---- general kernel -----------------------------------------------------------

// Any type, any head_dim up to 256, any strides: float32 products on the CUDA cores out of
// shared memory.  4 RW rows (node, head) against 32 keys at a time, 128 threads; warp w owns rows
// RW w .. RW w + RW - 1 from the scores to the result, so that the only block-wide waits are around
// the tile loads.  Lane (c, z) = (lane / 4, lane % 4) sums the RW x 4 scores of its warp's rows and
// keys 4 c .. 4 c + 3 over every fourth 4-element piece of the dimension and, after a sum over z, keeps
// those of rows z and z + 4.  RW 8 takes 12 loads of 16 bytes for 128 products where RW 4 takes 8 for
// 64, and half the fetches of keys and values: chosen when a request can have more than 16 rows (32
// float32 requests of 4096 tokens, 64 rows: 1.40 against 1.66 ms; half of the instructions are products).
// HALVES: blocks of 128 dims.  Above head_dim 128 the 16-bit types run here too, and every tile of 16 rows fetches
// the keys again: bfloat16 with head_dim 256, 32 requests of 4096 tokens, 16 rows 1.75 ms, 64 rows 6.8 ms, where the
// bytes take 165 us.
constexpr int kGenKeys = 32, kGenThreads = 128;

struct GeneralSmem {
    static __host__ __device__ int pad(int dim) { return (dim + 15) / 16 * 16; }
    static __host__ __device__ size_t bytes(int dim, int batch, int rows) {
        const size_t dp = pad(dim);
        return (rows * dp + kGenKeys * (dp + 4) + kGenKeys * dp + kGenKeys * rows) * sizeof(float) +
               2 * kGenKeys * sizeof(long long) * 2 + (kGenThreads / 32 + 4) * sizeof(int) + (static_cast<size_t>(batch) + 1) * sizeof(int);
    }
};

// Four elements in a row, as float32.
__device__ __forceinline__ float4 fourOf(const float* p) { return *reinterpret_cast<const float4*>(p); }
template <typename T>
__device__ __forceinline__ float4 fourOf(const T* p) {
    if constexpr (sizeof(T) == 2) {
        alignas(8) T e[4];
        *reinterpret_cast<uint2*>(e) = *reinterpret_cast<const uint2*>(p);
        return make_float4(valueOf(e), valueOf(e + 1), valueOf(e + 2), valueOf(e + 3));
    } else {
        const uint32_t w = *reinterpret_cast<const uint32_t*>(p);
        auto one = [&](int i) { return __half2float(__half(__nv_cvt_fp8_to_halfraw(static_cast<__nv_fp8_storage_t>(w >> (8 * i)), __NV_E4M3))); };
        return make_float4(one(0), one(1), one(2), one(3));
    }
}

// wide: rows are multiples of four elements, on boundaries of four elements.
template <typename QT, typename KT_, int RW, int HALVES>
__global__ void __launch_bounds__(kGenThreads, 4)
treeGeneralKernel(const __grid_constant__ TreeParams p, float scaleLog2, bool wide) {
    constexpr int kGenRows = 4 * RW, kOwn = RW / 4;        // rows of a tile; rows whose softmax a lane keeps
    extern __shared__ __align__(16) unsigned char raw[];
    const int D = p.headDim, dp = GeneralSmem::pad(D), tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    float* sq = reinterpret_cast<float*>(raw);             // [rows][dp]
    float* sk = sq + kGenRows * dp;                        // [32][dp + 4]
    float* sv = sk + kGenKeys * (dp + 4);                  // [32][dp]
    float* sp = sv + kGenKeys * dp;                        // [32][rows]
    long long* kAt = reinterpret_cast<long long*>(sp + kGenKeys * kGenRows);   // [32] element offsets, -1: no key
    long long* vAt = kAt + kGenKeys;
    long long* blkAt = vAt + kGenKeys;                     // FP8: the block, for its scales
    int* scratch = reinterpret_cast<int*>(blkAt + 2 * kGenKeys);
    int* prefix = scratch + kGenThreads / 32 + 4;
    cudaGridDependencySynchronize();                   // launched early, as treeTcKernel
    buildPrefix<kGenRows, kGenKeys, kGenThreads>(p, prefix, scratch);
    const int blocks = gridDim.x, me = blockIdx.x, total = prefix[p.batch];
    const int quota = (total + blocks - 1) / blocks;
    const int begin = static_cast<int>(min(static_cast<long long>(me) * quota, static_cast<long long>(total))), end = min(total, begin + quota);
    const int group = p.heads / p.kvHeads, c = lane >> 2, z = lane & 3;
    if (tid == 0) {
        Header h{};
        h.lastBlock = -1;
        *headerOf(p, me) = h;
    }
    for (int t = begin; t < end;) {
        const Segment g = segmentAt<kGenRows, kGenKeys>(p, prefix, t, end);
        const SeqInfo& s = g.s;
        const int cacheTiles = s.cacheTiles<kGenKeys>(), rows = s.n * group;
        const uint32_t hi = lastFirst(p, s, g.rt, kGenRows);
        __syncthreads();
        const int pieces = dp / 4;
        if (wide) {
#pragma unroll 4
            for (int i = tid; i < kGenRows * pieces; i += kGenThreads) {
                const int r = i / pieces, d = 4 * (i - r * pieces), rr = g.rt * kGenRows + r;
                float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
                if (rr < rows && d < D)
                    v = fourOf(static_cast<const QT*>(p.q) + static_cast<int64_t>(s.start + rr / group) * p.qStride +
                               static_cast<int64_t>(g.kvh * group + rr % group) * D + d);
                *reinterpret_cast<float4*>(sq + r * dp + d) = make_float4(v.x * scaleLog2, v.y * scaleLog2, v.z * scaleLog2, v.w * scaleLog2);
            }
        } else
        for (int i = tid; i < kGenRows * dp; i += kGenThreads) {
            const int r = i / dp, d = i - r * dp, rr = g.rt * kGenRows + r;
            float v = 0.f;
            if (rr < rows && d < D)
                v = valueOf(static_cast<const QT*>(p.q) + static_cast<int64_t>(s.start + rr / group) * p.qStride +
                            static_cast<int64_t>(g.kvh * group + rr % group) * D + d) * scaleLog2;
            sq[i] = v;
        }
        // the rows whose softmax this lane keeps
        int node[kOwn];
        uint32_t first[kOwn];
        float m[kOwn], l[kOwn];
        bool there[kOwn];
#pragma unroll
        for (int i = 0; i < kOwn; ++i) {
            const int row = g.rt * kGenRows + RW * warp + z + 4 * i;
            there[i] = row < rows;
            node[i] = min(row / group, s.n - 1);
            first[i] = firstOf(p, s, node[i]);
            m[i] = -INFINITY;
            l[i] = 0.f;
        }
        float acc[HALVES][RW][4];                          // [dims lane * 4 (+ 128)][row][dim]
#pragma unroll
        for (int h = 0; h < HALVES; ++h)
#pragma unroll
            for (int r = 0; r < RW; ++r)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[h][r][e] = 0.f;
        bool odd = false;
        for (int j = g.first; j < g.last; ++j) {
            const bool inTree = j >= cacheTiles;
            const uint32_t k0 = inTree ? static_cast<uint32_t>(j - cacheTiles) * kGenKeys : (s.lo / kGenKeys + j) * kGenKeys;
            __syncthreads();
            if (tid < kGenKeys) {
                const uint32_t key = k0 + tid;
                kAt[tid] = vAt[tid] = -1;
                blkAt[tid] = 0;
                if (inTree) {
                    if (key < static_cast<uint32_t>(s.n)) {
                        kAt[tid] = static_cast<int64_t>(s.start + key) * p.kStride + static_cast<int64_t>(g.kvh) * D;
                        vAt[tid] = static_cast<int64_t>(s.start + key) * p.vStride + static_cast<int64_t>(g.kvh) * D;
                    }
                } else if (key >= s.lo && key < s.held) {
                    int64_t blk;
                    kAt[tid] = vAt[tid] = poolRow(p, g.b, key, g.kvh, &blk);
                    blkAt[tid] = blk;
                }
            }
            __syncthreads();
            if (wide) {
                // Four pieces of keys and values each are on their way together: an element at a time, as
                // below, a call of seven short requests spent most of its time on one load after another
                // (dim 80, float32: 38.5 us, now 22).
                constexpr int kAhead = 4;
                for (int i0 = tid; i0 < kGenKeys * pieces; i0 += kAhead * kGenThreads) {
                    float4 kv[kAhead], vv[kAhead];
#pragma unroll
                    for (int u = 0; u < kAhead; ++u) {
                        const int i = i0 + u * kGenThreads, r = min(i / pieces, kGenKeys - 1), d = 4 * (i - r * pieces);
                        kv[u] = vv[u] = make_float4(0.f, 0.f, 0.f, 0.f);
                        if (i < kGenKeys * pieces && kAt[r] >= 0 && d < D) {
                            if (inTree) {
                                kv[u] = fourOf(static_cast<const QT*>(p.kNew) + kAt[r] + d);
                                vv[u] = fourOf(static_cast<const QT*>(p.vNew) + vAt[r] + d);
                            } else {
                                kv[u] = fourOf(static_cast<const KT_*>(p.kPool) + kAt[r] + d);
                                vv[u] = fourOf(static_cast<const KT_*>(p.vPool) + vAt[r] + d);
                            }
                        }
                    }
#pragma unroll
                    for (int u = 0; u < kAhead; ++u) {
                        const int i = i0 + u * kGenThreads, r = i / pieces, d = 4 * (i - r * pieces);
                        if (i >= kGenKeys * pieces) break;
                        float ks = 1.f, vs = 1.f;
                        if (sizeof(KT_) == 1 && !inTree && kAt[r] >= 0) {
                            ks = keyScaleOf(static_cast<const __half*>(p.kScale)[blkAt[r] * p.kvHeads + g.kvh]);
                            vs = __half2float(static_cast<const __half*>(p.vScale)[blkAt[r] * p.kvHeads + g.kvh]);
                        }
                        float e[4] = {vv[u].x * vs, vv[u].y * vs, vv[u].z * vs, vv[u].w * vs};
                        if (inTree || k0 + r < hi) {               // (some row may not see the key)
#pragma unroll
                            for (int c = 0; c < 4; ++c)
                                if (isOdd(e[c])) { e[c] = 0.f; odd = true; }
                        }
                        *reinterpret_cast<float4*>(sk + r * (dp + 4) + d) = make_float4(kv[u].x * ks, kv[u].y * ks, kv[u].z * ks, kv[u].w * ks);
                        *reinterpret_cast<float4*>(sv + r * dp + d) = make_float4(e[0], e[1], e[2], e[3]);
                    }
                }
            } else
            for (int i = tid; i < kGenKeys * dp; i += kGenThreads) {
                const int r = i / dp, d = i - r * dp;
                float kv = 0.f, vv = 0.f;
                if (kAt[r] >= 0 && d < D) {
                    if (inTree) {
                        kv = valueOf(static_cast<const QT*>(p.kNew) + kAt[r] + d);
                        vv = valueOf(static_cast<const QT*>(p.vNew) + vAt[r] + d);
                    } else {
                        kv = poolValue<KT_>(p, p.kPool, p.kScale, kAt[r] + d, blkAt[r], g.kvh);
                        if (sizeof(KT_) == 1 && isOdd(kv)) kv = __int_as_float(0x7FFFFFFF);            // (see keyScaleOf; a code may be NaN itself)
                        vv = poolValue<KT_>(p, p.vPool, p.vScale, vAt[r] + d, blkAt[r], g.kvh);
                    }
                    if ((inTree || k0 + r < hi) && isOdd(vv)) { vv = 0.f; odd = true; }   // (some row may not see the key)
                }
                sk[r * (dp + 4) + d] = kv;
                sv[i] = vv;
            }
            __syncthreads();
            float dot[RW][4];
#pragma unroll
            for (int r = 0; r < RW; ++r)
#pragma unroll
                for (int k = 0; k < 4; ++k) dot[r][k] = 0.f;
            for (int d = 4 * z; d < dp; d += 16) {
                float4 b[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) b[k] = *reinterpret_cast<const float4*>(sk + (4 * c + k) * (dp + 4) + d);
#pragma unroll
                for (int r = 0; r < RW; ++r) {
                    const float4 a = *reinterpret_cast<const float4*>(sq + (RW * warp + r) * dp + d);
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        dot[r][k] += a.x * b[k].x + a.y * b[k].y + a.z * b[k].z + a.w * b[k].w;
                }
            }
            float x[kOwn][4];                              // the lane's rows: scores of keys 4 c .. 4 c + 3
#pragma unroll
            for (int r = 0; r < RW; ++r)
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    float v = dot[r][k];
                    v += __shfl_xor_sync(0xFFFFFFFFu, v, 1);
                    v += __shfl_xor_sync(0xFFFFFFFFu, v, 2);
                    if ((r & 3) == z) x[r >> 2][k] = v;
                }
            float corr[kOwn];
#pragma unroll
            for (int i = 0; i < kOwn; ++i) {
                uint32_t bits = 0u;
                if (there[i]) {
                    if (inTree) bits = treeBits(p, s, node[i], static_cast<int>(k0 / 32));
                    else
                        for (int k = 0; k < 4; ++k) {
                            const uint32_t key = k0 + 4 * c + k;
                            if (key >= first[i] && key < s.held) bits |= 1u << (4 * c + k);
                        }
                }
                float top = -INFINITY;
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    if (!(bits >> (4 * c + k) & 1u)) x[i][k] = -INFINITY;
                    top = fmaxf(top, x[i][k]);
                }
#pragma unroll
                for (int o = 4; o < 32; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
                const float mNew = fmaxf(m[i], top), base = mNew == -INFINITY ? 0.f : mNew;
                corr[i] = exp2f(m[i] - base);
                float sum = 0.f;
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    x[i][k] = exp2f(x[i][k] - base);
                    sum += x[i][k];
                    sp[(4 * c + k) * kGenRows + RW * warp + z + 4 * i] = x[i][k];
                }
#pragma unroll
                for (int o = 4; o < 32; o <<= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
                l[i] = l[i] * corr[i] + sum;
                m[i] = mNew;
            }
            __syncwarp();
            float f[RW];
#pragma unroll
            for (int r = 0; r < RW; ++r) f[r] = __shfl_sync(0xFFFFFFFFu, corr[r >> 2], r & 3);
#pragma unroll
            for (int h = 0; h < HALVES; ++h) {
                const int d = 4 * lane + 128 * h;
                if (d >= dp) break;
#pragma unroll
                for (int r = 0; r < RW; ++r)
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[h][r][e] *= f[r];
#pragma unroll 8
                for (int k = 0; k < kGenKeys; ++k) {
                    const float4 v = *reinterpret_cast<const float4*>(sv + k * dp + d);
                    const float vv[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                    for (int q = 0; q < kOwn; ++q) {
                        const float4 w = *reinterpret_cast<const float4*>(sp + k * kGenRows + RW * warp + 4 * q);
                        const float ww[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                        for (int r = 0; r < 4; ++r)
#pragma unroll
                            for (int e = 0; e < 4; ++e) acc[h][4 * q + r][e] += ww[r] * vv[e];
                    }
                }
            }
            __syncwarp();
        }
        odd = __syncthreads_or(odd);
        const bool whole = g.whole();
        float* rec = nullptr;
        if (!whole) {
            const int which = g.first == 0 ? 1 : 0;
            rec = recordOf(p, blocks, me, which, kGenRows, dp);
            if (tid == 0) {
                Header* h = headerOf(p, me);
                h->odd[which] = odd ? 1 : 0;
                if (which == 1) {
                    h->b = g.b; h->kvh = g.kvh; h->rt = g.rt;
                    h->lastBlock = (t + g.nT - 1) / quota;
                }
            }
        }
#pragma unroll
        for (int r = 0; r < RW; ++r) {
            const float lr = __shfl_sync(0xFFFFFFFFu, l[r >> 2], r & 3), mr = __shfl_sync(0xFFFFFFFFu, m[r >> 2], r & 3);
            const int rl = RW * warp + r, rr = g.rt * kGenRows + rl;
            if (rr >= rows) continue;
#pragma unroll
            for (int h = 0; h < HALVES; ++h) {
                const int d = 4 * lane + 128 * h;
                if (d >= dp) break;
                if (whole) {
                    const float inv = lr == 0.f ? 0.f : 1.f / lr;
                    QT* out = static_cast<QT*>(p.out) + (static_cast<int64_t>(s.start + rr / group) * p.heads + g.kvh * group + rr % group) * D;
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (d + e < D) out[d + e] = narrow<QT>(acc[h][r][e] * inv);
                } else {
                    *reinterpret_cast<float4*>(rec + rl * dp + d) = make_float4(acc[h][r][0], acc[h][r][1], acc[h][r][2], acc[h][r][3]);
                }
            }
            if (whole && odd) {
                __syncwarp();
                if (lane == 0)
                    addLeftOut<QT, KT_>(p, s, g.b, g.kvh, rr / group, hi,
                                        static_cast<QT*>(p.out) + (static_cast<int64_t>(s.start + rr / group) * p.heads + g.kvh * group + rr % group) * D, 0, D);
                __syncwarp();
            }
            if (!whole && lane == 0) {
                rec[kGenRows * dp + rl] = mr;
                rec[kGenRows * dp + kGenRows + rl] = lr;
            }
        }
        t += g.last - g.first;
    }
}

// ---- the records of shared pairs --------------------------------------------------

// Block (i, y): the pair that block i of the attention kernel starts and does not finish, rows
// 8 y .. 8 y + 7 of its row tile, one warp each.  Its records lie in block i (the second) and in
// blocks i + 1 .. lastBlock (the first); their sum in that order is the same in every launch.
template <typename QT, typename KT_>
__global__ void __launch_bounds__(256)
treeJoinKernel(const __grid_constant__ TreeParams p, int blocks, int mr, int dimPad) {
    cudaGridDependencySynchronize();                   // launched early; the records are there from here on
    const Header h = *headerOf(p, blockIdx.x);
    if (h.lastBlock < 0) return;
    const int lane = threadIdx.x & 31, rl = blockIdx.y * 8 + (threadIdx.x >> 5);
    const SeqInfo s(p, h.b);
    const int group = p.heads / p.kvHeads, rr = h.rt * mr + rl;
    if (rl >= mr || rr >= s.n * group) return;
    const int first = blockIdx.x, count = h.lastBlock - first + 1;
    auto record = [&](int i) -> const float* { return recordOf(p, blocks, first + i, i == 0 ? 1 : 0, mr, dimPad); };
    bool odd = false;
    for (int i = lane; i < count; i += 32) odd = odd || headerOf(p, first + i)->odd[i == 0 ? 1 : 0] != 0;
    odd = __any_sync(0xFFFFFFFFu, odd);
    const uint32_t hi = odd ? lastFirst(p, s, h.rt, mr) : 0u;
    QT* out = static_cast<QT*>(p.out) + (static_cast<int64_t>(s.start + rr / group) * p.heads + h.kvh * group + rr % group) * p.headDim;
    for (int d = 4 * lane; d < p.headDim; d += 128) {
        // eight records at a time, maxima, sums and O together: a read is a long wait, and few warps share it
        constexpr int CHUNK = 8;
        float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
        float top = -INFINITY, l = 0.f;
        for (int i0 = 0; i0 < count; i0 += CHUNK) {
            float m[CHUNK], part[CHUNK];
            float4 o[CHUNK];
#pragma unroll
            for (int e = 0; e < CHUNK; ++e) {
                m[e] = -INFINITY;
                part[e] = 0.f;
                o[e] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (i0 + e < count) {
                    const float* r = record(i0 + e);
                    m[e] = r[mr * dimPad + rl];
                    part[e] = r[mr * dimPad + mr + rl];
                    o[e] = *reinterpret_cast<const float4*>(r + rl * dimPad + d);
                }
            }
            const float before = top;
#pragma unroll
            for (int e = 0; e < CHUNK; ++e) top = fmaxf(top, m[e]);
            const float base = top == -INFINITY ? 0.f : top, keep = exp2f(before - base);
            l *= keep;
            sum.x *= keep; sum.y *= keep; sum.z *= keep; sum.w *= keep;
#pragma unroll
            for (int e = 0; e < CHUNK; ++e) {
                const float f = exp2f(m[e] - base);
                l += f * part[e];
                sum.x += f * o[e].x; sum.y += f * o[e].y; sum.z += f * o[e].z; sum.w += f * o[e].w;
            }
        }
        const float inv = l == 0.f ? 0.f : 1.f / l, v[4] = {sum.x, sum.y, sum.z, sum.w};
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (d + e < p.headDim) out[d + e] = narrow<QT>(v[e] * inv);
    }
    if (odd) {
        __syncwarp();
        if (lane == 0) addLeftOut<QT, KT_>(p, s, h.b, h.kvh, rr / group, hi, out, 0, p.headDim);
    }
}

// The same for the records of treeTcKernel, whose O is [piece of 4 columns][MR rows]: block (i, y, z)
// takes rows 32 y .. + 31 and columns 64 z .. + 63, a lane a row and a warp two pieces, so that the
// reads of a record are whole lines.  One request of 8192 tokens leaves 18 records of each pair and
// eight blocks with work: what counts is how many reads in a row a block waits for, so that the records
// are read several at a time, maxima, sums and O together, under a running maximum.
template <typename QT, typename KT_, int MR>
__global__ void __launch_bounds__(256)
treeJoinColumnsKernel(const __grid_constant__ TreeParams p, int blocks) {
    // (pairs of up to 256 rows fill the GPU with work by themselves: there fewer registers and more blocks
    // win, 61.6 against 65.2 us with 8 requests of 4096 tokens and 256 rows; one request of 8192 tokens
    // and 4 rows: 22.7 against 26.5 us)
    constexpr int HD = 128, CHUNK = MR == 256 ? 4 : 8;
    cudaGridDependencySynchronize();
    const Header h = *headerOf(p, blockIdx.x);
    if (h.lastBlock < 0) return;
    const int lane = threadIdx.x & 31, d0 = blockIdx.z * 64 + (threadIdx.x >> 5) * 8, rl = blockIdx.y * 32 + lane;
    const SeqInfo s(p, h.b);
    const int group = p.heads / p.kvHeads, rr = h.rt * MR + rl;
    if (h.rt * MR + static_cast<int>(blockIdx.y) * 32 >= s.n * group) return;
    if (d0 >= p.headDim) return;
    const bool mine = rr < s.n * group;
    const int first = blockIdx.x, count = h.lastBlock - first + 1;
    bool odd = false;
    for (int i = lane; i < count; i += 32) odd = odd || headerOf(p, first + i)->odd[i == 0 ? 1 : 0] != 0;
    float top = -INFINITY, l = 0.f;
    float sum[8] = {};
    if (mine)
        for (int i0 = 0; i0 < count; i0 += CHUNK) {
            float m[CHUNK], part[CHUNK];
            float4 o[CHUNK][2];
#pragma unroll
            for (int e = 0; e < CHUNK; ++e) {
                m[e] = -INFINITY;
                part[e] = 0.f;
                o[e][0] = o[e][1] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (i0 + e < count) {
                    const float* r = recordOf(p, blocks, first + i0 + e, i0 + e == 0 ? 1 : 0, MR, HD);
                    m[e] = r[MR * HD + rl];
                    part[e] = r[MR * HD + MR + rl];
                    for (int q = 0; q < 2; ++q) o[e][q] = reinterpret_cast<const float4*>(r)[(d0 / 4 + q) * MR + rl];
                }
            }
            const float before = top;
#pragma unroll
            for (int e = 0; e < CHUNK; ++e) top = fmaxf(top, m[e]);
            const float base = top == -INFINITY ? 0.f : top, keep = exp2f(before - base);
            l *= keep;
#pragma unroll
            for (int c = 0; c < 8; ++c) sum[c] *= keep;
#pragma unroll
            for (int e = 0; e < CHUNK; ++e) {
                const float f = exp2f(m[e] - base);
                l += f * part[e];
#pragma unroll
                for (int q = 0; q < 2; ++q) {
                    sum[4 * q] += f * o[e][q].x;
                    sum[4 * q + 1] += f * o[e][q].y;
                    sum[4 * q + 2] += f * o[e][q].z;
                    sum[4 * q + 3] += f * o[e][q].w;
                }
            }
        }
    odd = __any_sync(0xFFFFFFFFu, odd);
    if (!mine) return;
    const float inv = l == 0.f ? 0.f : 1.f / l;
    alignas(16) QT out[8];
#pragma unroll
    for (int c = 0; c < 8; ++c) out[c] = narrow<QT>(sum[c] * inv);
    QT* to = static_cast<QT*>(p.out) + (static_cast<int64_t>(s.start + rr / group) * p.heads + h.kvh * group + rr % group) * p.headDim;
    *reinterpret_cast<uint4*>(to + d0) = *reinterpret_cast<const uint4*>(out);
    if (odd) addLeftOut<QT, KT_>(p, s, h.b, h.kvh, rr / group, lastFirst(p, s, h.rt, MR), to, d0, d0 + 8);
}

template <typename QT, typename KT_>
cudaError_t launchJoin(const TreeParams& p, const TreePlan& plan, cudaStream_t stream, int* launches) {
    if (plan.blocks < 2) return cudaSuccess;
    *launches += 1;
    const unsigned blocks = static_cast<unsigned>(plan.blocks - 1);
    if constexpr (sizeof(QT) == 2)
        if (plan.variant == 2) {
            // (slices of rows that some request can have)
            const int64_t rows = std::min<int64_t>(plan.rows, static_cast<int64_t>(p.maxNew) * (p.heads / p.kvHeads));
            const dim3 grid(blocks, static_cast<unsigned>((rows + 31) / 32), 2);
            return plan.rows == 256 ? launchEarly(treeJoinColumnsKernel<QT, KT_, 256>, grid, 256, 0, stream, p, plan.blocks)
                                    : launchEarly(treeJoinColumnsKernel<QT, KT_, 128>, grid, 256, 0, stream, p, plan.blocks);
        }
    return launchEarly(treeJoinKernel<QT, KT_>, dim3(blocks, (plan.rows + 7) / 8), 256, 0, stream, p, plan.blocks, plan.rows, plan.dimPad);
}

TreePlan generalPlan(const TreeParams& p, int smCount) {
    TreePlan t{};
    t.rows = p.headDim <= 128 && static_cast<int64_t>(p.maxNew) * (p.heads / p.kvHeads) > 16 ? 32 : 16;
    t.keys = kGenKeys;
    t.dimPad = GeneralSmem::pad(p.headDim);
    // as many blocks as an SM's shared memory holds, four at most
    const size_t smem = GeneralSmem::bytes(p.headDim, p.batch, t.rows);
    const int perSm = static_cast<int>(std::min<size_t>(4, std::max<size_t>(1, (227u * 1024) / (smem + 1024))));
    t.blocks = smCount * perSm;
    return t;
}

// The tcgen05 kernel wherever it applies: at 32 requests of 4096 tokens (head_dim 128, bfloat16) and 4, 64 and 256
// rows under a KV head 100, 109 and 178 us against 121, 231 and 821 us of the mma kernel, on short lists too, with
// one request of 8192 tokens and 4, 24 and 96 rows, 23, 23 and 24 against 23, 27 and 43.  But a call that cannot have
// work for every block, and few rows, is over sooner in the kernel with the shorter way from start to end (1024
// tokens, 4 rows: 12.6 against 16.4 us).
bool shortCall(const TreeParams& p, int smCount) {
    const int64_t tiles = static_cast<int64_t>(p.batch) * p.kvHeads * ((static_cast<int64_t>(p.maxNumBlocks) * p.blockSize + 127) / 128 + 1);
    return static_cast<int64_t>(p.maxNew) * (p.heads / p.kvHeads) <= 16 && tiles <= smCount;
}

TreePlan treePlan(const TreeParams& p, int smCount) {
    if (treeTcApplies(p) && !(shortCall(p, smCount) && treeMmaApplies(p))) return treeTcPlan(p, smCount);
    if (treeMmaApplies(p)) return treeMmaPlan(p, smCount);
    return generalPlan(p, smCount);
}

size_t planBytes(const TreePlan& t) {
    return headerBytes(t.blocks) + static_cast<size_t>(t.blocks) * 2 * recordFloats(t.rows, t.dimPad) * sizeof(float);
}

template <typename QT, typename KT_, int RW, int HALVES>
cudaError_t launchGeneralShape(const TreeParams& p, const TreePlan& plan, cudaStream_t stream) {
    static std::atomic<unsigned long long> done{0};
    cudaError_t e = allowSmem(treeGeneralKernel<QT, KT_, RW, HALVES>, 227 * 1024, done);
    if (e != cudaSuccess) return e;
    const float scaleLog2 = 1.4426950408889634f / sqrtf(static_cast<float>(p.headDim));
    bool wide = p.headDim % 4 == 0 && p.qStride % 4 == 0 && p.kStride % 4 == 0 && p.vStride % 4 == 0;
    for (const void* rows : {p.q, p.kNew, p.vNew}) wide = wide && reinterpret_cast<uintptr_t>(rows) % (4 * sizeof(QT)) == 0;
    for (const void* pool : {p.kPool, p.vPool}) wide = wide && reinterpret_cast<uintptr_t>(pool) % (4 * sizeof(KT_)) == 0;
    return launchEarly(treeGeneralKernel<QT, KT_, RW, HALVES>, dim3(plan.blocks), kGenThreads, GeneralSmem::bytes(p.headDim, p.batch, plan.rows),
                       stream, p, scaleLog2, wide);
}

template <typename QT, typename KT_>
cudaError_t launchGeneral(const TreeParams& p, const TreePlan& plan, cudaStream_t stream) {
    if (p.headDim > 128) return launchGeneralShape<QT, KT_, 4, 2>(p, plan, stream);
    return plan.rows == 32 ? launchGeneralShape<QT, KT_, 8, 1>(p, plan, stream) : launchGeneralShape<QT, KT_, 4, 1>(p, plan, stream);
}

template <typename QT, typename KT_>
cudaError_t launchOf(const TreeParams& p, const TreePlan& plan, cudaStream_t stream, int* launches) {
    const cudaError_t e = plan.variant == 2 ? launchTreeTc(p, plan, stream) : plan.variant == 1 ? launchTreeMma(p, plan, stream)
                                                                            : launchGeneral<QT, KT_>(p, plan, stream);
    *launches += 1;
    return e == cudaSuccess ? launchJoin<QT, KT_>(p, plan, stream, launches) : e;
}

}  // namespace

int64_t treeTileBound(const TreeParams& p) {
    constexpr int kFewestRows = 16;                    // of a tile of any kernel
    const int64_t rowTiles = (static_cast<int64_t>(p.maxNew) * (p.heads / p.kvHeads) + kFewestRows - 1) / kFewestRows;
    const int64_t keyTiles = static_cast<int64_t>(p.maxNumBlocks) * p.blockSize / kGenKeys + 2 + p.maxNew / kGenKeys + 1;
    return static_cast<int64_t>(p.batch) * p.kvHeads * rowTiles * keyTiles;
}

size_t treeWorkspaceBytes(const TreeParams& p, int smCount) {
    // by sizes and types alone: alignment may change between the query and the call (staged copies)
    size_t n = planBytes(generalPlan(p, smCount));
    if (treeMmaSizes(p)) n = std::max(n, planBytes(treeMmaPlan(p, smCount)));
    if (treeTcSizes(p)) n = std::max(n, planBytes(treeTcPlan(p, smCount)));
    return n;
}

cudaError_t launchTreeAttention(const TreeParams& p, int smCount, cudaStream_t stream, int* launches, bool* bounded) {
    const TreePlan plan = treePlan(p, smCount);
    *bounded = plan.variant == 2;
    switch (p.dtype) {
        case kF32: return launchOf<float, float>(p, plan, stream, launches);
        case kF16: return launchOf<__half, __half>(p, plan, stream, launches);
        case kBF16: return launchOf<__nv_bfloat16, __nv_bfloat16>(p, plan, stream, launches);
        default: return launchOf<__half, uint8_t>(p, plan, stream, launches);
    }
}

}  // namespace pam
