// Attention of one new token per sequence over a paged cache.  For head h of sequence b with `len` tokens:
//
//   z_j = scale q.k_j      z_j = cap tanh(z_j / cap)      z_j += slope_h (j - (len - 1))      max(0, len - window) <= j < len
//   out = sum_j exp(z_j - m) v_j / sum_j exp(z_j - m)     lse = m + log(sum)                  m = max_j z_j
//
// The keys and values of the sequences are read once; memory bounds it.  The work is all tiles of kTile tokens of all units (a
// sequence, a key-value head, a block of its query heads) behind one another; every block takes an equal run of them, so that
// one long sequence and many of different lengths both fill the GPU.  A unit that lies in one block's run is finished there; of
// the others each block leaves (m, sum, sum of exp v) and a second kernel joins them.  A block's run has at most one unit that
// began before it and one that ends behind it: two places a block.
#include "paged.cuh"

namespace rwkvb200 {
namespace {

__device__ int g_error = 0;
constexpr int kThreads = 128, kWarps = kThreads / 32;
constexpr int kTile = 64;
constexpr int kMinTiles = 4;      // a block's run: fewer would cost more to join than they save

struct AttentionArgs {
    int B, Hq, Hkv, N, pages, width, window, group, blocks;   // blocks of query heads per key-value head
    float scale, cap, to_log2;   // to_log2: what makes the partial maxima exponents of 2
    Divisor page;
    const void *q, *k_pages, *v_pages;
    const int *table, *lengths;
    const float* slopes;
    void* out;
    float *lse, *work;
};

struct Range {
    int lo, hi, tiles;   // tokens of a sequence that count, and their tiles: one at least, so that empty sequences get their zeros
    __device__ __forceinline__ Range(const AttentionArgs& p, int b) {
        hi = min(p.lengths[b], p.width * (int)p.page.d);
        lo = p.window > 0 ? max(0, hi - p.window) : 0;
        tiles = hi < 0 ? 0 : max(1, (hi - lo + kTile - 1) / kTile);   // a negative length is a row that only pads the batch
    }
};

// All threads: the number of tiles of all units, and of those of the sequences before b_of.
__device__ __forceinline__ i64 sum_block(i64 v, i64* shared) {
#pragma unroll
    for (int d = 16; d >= 1; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) shared[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) v += shared[w];
    return v;
}
__device__ __forceinline__ i64 tiles_before(const AttentionArgs& p, int end, i64* shared) {
    i64 n = 0;
    for (int b = threadIdx.x; b < end; b += kThreads) n += Range(p, b).tiles;
    return sum_block(n, shared) * (p.Hkv * p.blocks);
}
__device__ __forceinline__ i64 run_length(i64 all, i64 blocks) { return max((i64)kMinTiles, (all + blocks - 1) / blocks); }

// The sequence that tile `begin` of all lies in, and the tiles of those before it.
__device__ __forceinline__ void find_start(const AttentionArgs& p, i64 begin, int units, i64* shared, i64* start) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    i64 base = 0;
    for (int b0 = 0; b0 < p.B; b0 += kThreads) {
        const int b = b0 + threadIdx.x;
        i64 n = b < p.B ? (i64)Range(p, b).tiles * units : 0, x = n;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const i64 o = __shfl_up_sync(0xffffffffu, x, d);
            if (lane >= d) x += o;
        }
        __syncthreads();
        if (lane == 31) shared[warp] = x;
        __syncthreads();
        i64 before = base;
        for (int w = 0; w < kWarps; ++w) {
            if (w < warp) before += shared[w];
            base += shared[w];
        }
        x += before;
        if (begin >= x - n && begin < x) start[0] = b, start[1] = x - n;
        if (base > begin) break;   // (the same for all threads)
    }
    __syncthreads();
}

// One sequence's cache as a lane sees it
template <typename E>
struct Cache {
    const AttentionArgs& p;
    const int* row;
    int head;
    // where token j lies (elements from the pool's start), -1: its page is none of the pool's
    __device__ __forceinline__ i64 at(int j) const {
        const uint32_t col = p.page.quotient((uint32_t)j);
        const int id = row[col];
        if ((unsigned)id >= (unsigned)p.pages) {
            atomicMax(&g_error, kBadPage);
            return -1;
        }
        return (((i64)id * p.Hkv + head) * p.page.d + ((uint32_t)j - col * p.page.d)) * p.N;
    }
};

__device__ __forceinline__ float capped(float z, float cap) { return cap > 0.f ? cap * tanhf(z / cap) : z; }

// Any type, head size and alignment, fp32 arithmetic.  Eight lanes share a token (piece i of W elements of lane l is at
// (i * 8 + l) * W), so a warp has four tokens in hand; every such group keeps a running maximum and sum of its own for HB
// query heads, and they are joined at a run's end.
template <typename E, int W, int HB>
__global__ void __launch_bounds__(kThreads) attention_kernel(const AttentionArgs p) {
    constexpr int kPieces = RWKVB200_MAX_HEAD_SIZE / (8 * W);
    __shared__ i64 shared[kWarps];
    __shared__ float sO[kWarps][HB][RWKVB200_MAX_HEAD_SIZE], sM[kWarps][HB], sL[kWarps][HB];
    __shared__ i64 sStart[2];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, l8 = lane & 7, token = warp * 4 + (lane >> 3);
    const unsigned mask = 0xffu << (lane & 24);   // the lanes that share a token
    const int units = p.Hkv * p.blocks;
    const i64 all = tiles_before(p, p.B, shared), run = run_length(all, gridDim.x);
    const i64 begin = run * blockIdx.x, end = min(begin + run, all);
    if (begin >= end) return;
    find_start(p, begin, units, shared, sStart);
    int b = (int)sStart[0];
    i64 base = sStart[1];
    for (i64 at = begin; at < end;) {
        const Range r(p, b);
        if (at >= base + (i64)r.tiles * units) {   // (a row without tiles is passed over as well)
            base += (i64)r.tiles * units;
            ++b;
            continue;
        }
        const int unit = (int)((at - base) / r.tiles), t0 = (int)((at - base) % r.tiles), t1 = (int)min((i64)r.tiles, t0 + (end - at));
        at += t1 - t0;
        const int head = unit / p.blocks, h0 = head * p.group + unit % p.blocks * HB, heads = min(HB, (head + 1) * p.group - h0);
        const Cache<E> cache{p, p.table + (i64)b * p.width, head};
        if (threadIdx.x == 0 && p.lengths[b] > r.hi) atomicMax(&g_error, kBadLength);
        float q[HB][kPieces * W], o[HB][kPieces * W], m[HB], l[HB];
#pragma unroll
        for (int h = 0; h < HB; ++h) {
            m[h] = -INFINITY;
            l[h] = 0.f;
            const E* from = static_cast<const E*>(p.q) + ((i64)b * p.Hq + h0 + h) * p.N;
#pragma unroll
            for (int i = 0; i < kPieces; ++i)
#pragma unroll
                for (int e = 0; e < W; ++e) {
                    const int n = (i * 8 + l8) * W + e;
                    q[h][i * W + e] = h < heads && n < p.N ? to_f(from[n]) * p.scale : 0.f;
                    o[h][i * W + e] = 0.f;
                }
        }
        struct alignas(sizeof(E) * W) Piece {
            E e[W];
        };
        const int last = min(r.lo + t1 * kTile, r.hi);
        for (int j = r.lo + t0 * kTile + token; j < last; j += kWarps * 4) {
            const i64 place = cache.at(j);
            const bool found = place >= 0;
            const E *k = static_cast<const E*>(p.k_pages) + (found ? place : 0), *v = static_cast<const E*>(p.v_pages) + (found ? place : 0);
            Piece pk[kPieces], pv[kPieces];
#pragma unroll
            for (int i = 0; i < kPieces; ++i) {
                const int n = (i * 8 + l8) * W;
                if (found && n < p.N) {
                    pk[i] = *reinterpret_cast<const Piece*>(k + n);
                    pv[i] = *reinterpret_cast<const Piece*>(v + n);
                } else {
#pragma unroll
                    for (int e = 0; e < W; ++e) pk[i].e[e] = pv[i].e[e] = from_f<E>(0.f);
                }
            }
#pragma unroll
            for (int h = 0; h < HB; ++h) {
                float z = 0.f;
#pragma unroll
                for (int i = 0; i < kPieces; ++i)
#pragma unroll
                    for (int e = 0; e < W; ++e) z = fmaf(q[h][i * W + e], to_f(pk[i].e[e]), z);
#pragma unroll
                for (int d = 4; d >= 1; d >>= 1) z += __shfl_xor_sync(mask, z, d);
                z = capped(z, p.cap);
                if (p.slopes != nullptr && h < heads) z += p.slopes[h0 + h] * (float)(j - (r.hi - 1));
                if (!found) z = -INFINITY;
                // weights of scores of -infinity are 0, also while there is nothing else
                const float top = fmaxf(m[h], z), keep = m[h] == -INFINITY ? 0.f : expf(m[h] - top);
                const float w = z == -INFINITY ? 0.f : expf(z - top);
                m[h] = top;
                l[h] = fmaf(l[h], keep, w);
                if (z != -INFINITY) {   // (else the maximum is what it was, and the value may hold anything)
#pragma unroll
                    for (int i = 0; i < kPieces; ++i)
#pragma unroll
                        for (int e = 0; e < W; ++e) o[h][i * W + e] = fmaf(o[h][i * W + e], keep, w * to_f(pv[i].e[e]));
                }
            }
        }
        __syncwarp();
        // the four groups of a warp, then the warps
        __syncthreads();
#pragma unroll
        for (int h = 0; h < HB; ++h) {
            float top = m[h];
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
            const float keep = m[h] == -INFINITY ? 0.f : expf(m[h] - top);
            float sum = l[h] * keep;
            sum += __shfl_xor_sync(0xffffffffu, sum, 8);
            sum += __shfl_xor_sync(0xffffffffu, sum, 16);
            if (lane == 0) sM[warp][h] = top, sL[warp][h] = sum;
#pragma unroll
            for (int i = 0; i < kPieces; ++i)
#pragma unroll
                for (int e = 0; e < W; ++e) {
                    float x = m[h] == -INFINITY ? 0.f : o[h][i * W + e] * keep;
                    x += __shfl_xor_sync(0xffffffffu, x, 8);
                    x += __shfl_xor_sync(0xffffffffu, x, 16);
                    if (lane < 8) sO[warp][h][(i * 8 + l8) * W + e] = x;
                }
        }
        __syncthreads();
        const bool whole = t0 == 0 && t1 == r.tiles;
        float* part = p.work + ((i64)blockIdx.x * 2 + (t0 == 0)) * HB * (p.N + 2);
        for (int i = threadIdx.x; i < heads * p.N; i += kThreads) {
            const int h = i / p.N, n = i % p.N;
            float top = -INFINITY, x = 0.f, sum = 0.f;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) top = fmaxf(top, sM[w][h]);
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                const float keep = sM[w][h] == -INFINITY ? 0.f : expf(sM[w][h] - top);
                sum += sL[w][h] * keep;
                if (sM[w][h] != -INFINITY) x += sO[w][h][n] * keep;
            }
            if (whole) {
                static_cast<E*>(p.out)[((i64)b * p.Hq + h0 + h) * p.N + n] = from_f<E>(sum == 0.f ? 0.f : x / sum);
                if (n == 0 && p.lse != nullptr) p.lse[(i64)b * p.Hq + h0 + h] = sum == 0.f ? -INFINITY : top + logf(sum);
            } else {
                part[h * (p.N + 2) + n] = x;
                if (n == 0) part[h * (p.N + 2) + p.N] = top, part[h * (p.N + 2) + p.N + 1] = sum;
            }
        }
    }
}

// bf16, heads of whole 16-byte pieces: products on mma.sync m16n8k16 with the tokens in the rows, S^T = K q^T and O^T = V^T P^T, for up
// to 8 HT query heads that share the keys: HT = 1 wastes nothing on groups of 8, and memory bounds both anyway.  Each warp takes
// 16 of a tile's tokens and keeps its own maxima and sums.  The order of the elements of a head (and of the tokens in the second product) is
// free as long as both operands agree, so a lane reads its fragments as 16-byte pieces of rows:
//   keys    lane (g, q): rows g and g + 8, pieces 4 i + q            values  rows 2q, 2q+1, 2q+8, 2q+9, pieces 8 i + g
// They come through shared memory by cp.async (kStages - 1 steps ahead), every lane to a place of its own: no barrier, no bank
// conflict, and rows that do not count are filled with zeros.  Weights are taken into the second product as the sum of two
// bf16 numbers (2^-16 relative; one would double the output's rounding), both above 0, so that an infinite value stays one.
constexpr int kStages = 2;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

__device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transposed(uint32_t v) {   // an 8 x 8 matrix of bf16 over the warp
    uint32_t d;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(v));
    return d;
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float rcp(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// by its series up to 0.25 (five terms leave 0.009 x^10 = 8e-9), else 1 - 2 / (1 + exp(2 x)), which would lose the digits of a small one
__device__ __forceinline__ float hyperbolic_tangent(float x) {
    const float t = x * x;
    float s = fmaf(t, 62.f / 2835.f, -17.f / 315.f);
    s = fmaf(s, t, 2.f / 15.f);
    s = fmaf(s, t, -1.f / 3.f);
    s = fmaf(s * t, x, x);
    return t < 0.0625f ? s : 1.f - 2.f * rcp(1.f + ex2(2.f * kLog2e * x));
}
__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
    const __nv_bfloat162 t = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&t);
}
__device__ __forceinline__ void copy_or_zero(void* to, const bf16* from, bool there) {
    const uint32_t shared = (uint32_t)__cvta_generic_to_shared(to);
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(shared), "l"(from), "r"(there ? 16 : 0) : "memory");
}

template <int NP, int HT>
__global__ void __launch_bounds__(kThreads, 3) attention_mma_kernel(const AttentionArgs p) {
    constexpr int kK = NP / 32, kV = NP / 64;            // pieces of a key's, of a value's row per lane
    constexpr int kPieces = 2 * kK + 4 * kV, kHeads = 8 * HT;
    extern __shared__ __align__(16) uint4 staged[];      // [warp][stage][piece][lane]
    __shared__ i64 shared[kWarps], sStart[2];
    __shared__ float sM[kWarps][kHeads], sL[kWarps][kHeads];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, q = lane & 3;
    const int units = p.Hkv * p.blocks;
    const i64 all = tiles_before(p, p.B, shared), run = run_length(all, gridDim.x);
    const i64 begin = run * blockIdx.x, end = min(begin + run, all);
    if (begin >= end) return;
    find_start(p, begin, units, shared, sStart);
    uint4* mine = staged + warp * kStages * kPieces * 32 + lane;
    float* sO = reinterpret_cast<float*>(staged + warp * kStages * kPieces * 32);   // [head][NP], between the tokens of two units
    const bf16 *keys = static_cast<const bf16*>(p.k_pages), *values = static_cast<const bf16*>(p.v_pages);
    const float scale = p.cap > 0.f ? p.scale / p.cap : p.scale * kLog2e, cap = p.cap * kLog2e;
    int b = (int)sStart[0];
    i64 base = sStart[1];
    for (i64 at = begin; at < end;) {
        const Range r(p, b);
        if (at >= base + (i64)r.tiles * units) {   // (a row without tiles is passed over as well)
            base += (i64)r.tiles * units;
            ++b;
            continue;
        }
        const int unit = (int)((at - base) / r.tiles), t0 = (int)((at - base) % r.tiles), t1 = (int)min((i64)r.tiles, t0 + (end - at));
        at += t1 - t0;
        const int head = unit / p.blocks, h0 = head * p.group + unit % p.blocks * kHeads, heads = min(kHeads, (head + 1) * p.group - h0);
        if (threadIdx.x == 0 && p.lengths[b] > r.hi) atomicMax(&g_error, kBadLength);
        const int* row = p.table + (i64)b * p.width;
        const int from = r.lo + t0 * kTile + warp * 16, last = min(r.lo + t1 * kTile, r.hi), steps = t1 - t0;
        // the row of the pools that token (lane & 15) of a step lies in; -1: the token does not count
        auto rows_of = [&](int step) {
            const int j = from + step * kTile + (lane & 15);
            int n = -1;
            if (step < steps && j < last) {
                const uint32_t col = p.page.quotient((uint32_t)j);
                const int id = row[col];
                if ((unsigned)id < (unsigned)p.pages) n = (id * p.Hkv + head) * (int)p.page.d + (j - (int)(col * p.page.d));
                else atomicMax(&g_error, kBadPage);
            }
            return n;
        };
        auto ask = [&](int n, int stage) {   // copies the step whose rows are n
            uint4* to = mine + stage * kPieces * 32;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int k = __shfl_sync(0xffffffffu, n, g + 8 * i);
                const bf16* at = keys + (i64)max(k, 0) * p.N + q * 8;
#pragma unroll
                for (int j = 0; j < kK; ++j) copy_or_zero(to + (i * kK + j) * 32, at + j * 32, k >= 0 && j * 32 + q * 8 < p.N);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int v = __shfl_sync(0xffffffffu, n, 2 * q + (i & 1) + 8 * (i >> 1));
                const bf16* at = values + (i64)max(v, 0) * p.N + g * 8;
#pragma unroll
                for (int j = 0; j < kV; ++j) copy_or_zero(to + (2 * kK + i * kV + j) * 32, at + j * 64, v >= 0 && j * 64 + g * 8 < p.N);
            }
        };
        // q as the second operand of the scores: head g (and g + 8), the elements that the lane has of the keys
        uint32_t qf[HT][kK][4];
#pragma unroll
        for (int h = 0; h < HT; ++h)
#pragma unroll
            for (int j = 0; j < kK; ++j) {
                const bf16* from = static_cast<const bf16*>(p.q) + ((i64)b * p.Hq + h0 + h * 8 + g) * p.N + j * 32 + q * 8;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    __nv_bfloat162 v = __floats2bfloat162_rn(0.f, 0.f);
                    if (h * 8 + g < heads && j * 32 + q * 8 < p.N) v.x = from[2 * e], v.y = from[2 * e + 1];
                    qf[h][j][e] = *reinterpret_cast<const uint32_t*>(&v);
                }
            }
        float slope[HT][2], m[HT][2], l[HT][2], o[HT][NP / 16][4];   // heads 8 h + 2q, + 1
#pragma unroll
        for (int h = 0; h < HT; ++h) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                slope[h][e] = p.slopes != nullptr && h * 8 + 2 * q + e < heads ? p.slopes[h0 + h * 8 + 2 * q + e] * kLog2e : 0.f;
                m[h][e] = -INFINITY;
                l[h][e] = 0.f;
            }
#pragma unroll
            for (int i = 0; i < NP / 16; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[h][i][e] = 0.f;
        }
        int next = rows_of(0), ahead = rows_of(1);   // rows of the next step, and of the one behind it
        ask(next, 0);
        asm volatile("cp.async.commit_group;" ::: "memory");
        for (int step = 0; step < steps; ++step) {
            const int n = next;
            uint4* in = mine + (step & 1) * kPieces * 32;
            ask(ahead, (step + 1) & 1);
            asm volatile("cp.async.commit_group;" ::: "memory");
            next = ahead;
            ahead = rows_of(step + 2);
            asm volatile("cp.async.wait_group 1;" ::: "memory");
            float z[HT][4];
#pragma unroll
            for (int h = 0; h < HT; ++h)
#pragma unroll
                for (int e = 0; e < 4; ++e) z[h][e] = 0.f;
#pragma unroll
            for (int j = 0; j < kK; ++j) {
                const uint4 x = in[j * 32], y = in[(kK + j) * 32];
#pragma unroll
                for (int h = 0; h < HT; ++h) {
                    mma(z[h], x.x, y.x, x.y, y.y, qf[h][j][0], qf[h][j][1]);
                    mma(z[h], x.z, y.z, x.w, y.w, qf[h][j][2], qf[h][j][3]);
                }
            }
            // scores as exponents of 2: tokens g (elements 0, 1) and g + 8 (2, 3)
            const bool there[2] = {__shfl_sync(0xffffffffu, n, g) >= 0, __shfl_sync(0xffffffffu, n, g + 8) >= 0};
            const float distance = (float)(from + step * kTile + g - (r.hi - 1));
            bool more = false, none = false;   // a new maximum; a score of -infinity
#pragma unroll
            for (int h = 0; h < HT; ++h)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float v = z[h][e] * scale;
                    if (p.cap > 0.f) v = cap * hyperbolic_tangent(v);
                    v = fmaf(slope[h][e & 1], distance + (e >> 1) * 8.f, v);
                    v = there[e >> 1] ? v : -INFINITY;
                    z[h][e] = v;
                    more |= v > m[h][e & 1];
                    none |= v == -INFINITY;
                }
            if (__any_sync(0xffffffffu, more)) {
#pragma unroll
                for (int h = 0; h < HT; ++h) {
                    float keep[2];
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float top = fmaxf(m[h][e], fmaxf(z[h][e], z[h][e + 2]));
#pragma unroll
                        for (int d = 4; d <= 16; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
                        keep[e] = m[h][e] == -INFINITY ? 1.f : ex2(m[h][e] - top);   // (nothing, or NaN, has been summed before)
                        m[h][e] = top;
                        l[h][e] *= keep[e];
                    }
#pragma unroll
                    for (int i = 0; i < NP / 16; ++i)
#pragma unroll
                        for (int e = 0; e < 4; ++e) o[h][i][e] *= keep[e & 1];
                }
            }
            if (__any_sync(0xffffffffu, none)) {
                // a token without weight in any head counts for nothing, whatever its value holds
                bool dead[2] = {true, true};
#pragma unroll
                for (int h = 0; h < HT; ++h)
#pragma unroll
                    for (int e = 0; e < 4; ++e) dead[e >> 1] &= h * 8 + 2 * q + (e & 1) >= heads || z[h][e] == -INFINITY;
                uint32_t gone[2];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    uint32_t x = __ballot_sync(0xffffffffu, dead[i]);
                    x &= x >> 1;
                    gone[i] = x & x >> 2;   // bit 4 g: token g (+ 8)
                }
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (gone[i >> 1] >> (4 * (2 * q + (i & 1))) & 1)
#pragma unroll
                        for (int j = 0; j < kV; ++j) in[(2 * kK + i * kV + j) * 32] = make_uint4(0, 0, 0, 0);
            }
            // weights, and as the second operand of the second product
            uint32_t high[HT][2], low[HT][2];
#pragma unroll
            for (int h = 0; h < HT; ++h) {
                float x[4], y[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float top = m[h][e & 1], w = ex2(z[h][e] - (top == -INFINITY ? 0.f : top));
                    l[h][e & 1] += w;
                    x[e] = __uint_as_float(__float_as_uint(w * (1.f - 1.f / 4096.f)) & 0xffff0000u);
                    y[e] = w - x[e];
                }
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    high[h][i] = transposed(pack_bf16(x[2 * i], x[2 * i + 1]));
                    low[h][i] = transposed(pack_bf16(y[2 * i], y[2 * i + 1]));
                }
            }
            // rows of O^T: g is element i of the lane's first piece, g + 8 of its second (NP = 64: element i + 4 of the only one)
#pragma unroll
            for (int half = 0; half < (NP == 64 ? 1 : 2); ++half) {
                uint32_t v[4][4];   // [token][word]: NP = 128: words 2 half, + 1 of both pieces; 64: all words
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if (NP == 64) {
                        const uint4 x = in[(2 * kK + i) * 32];
                        v[i][0] = x.x, v[i][1] = x.y, v[i][2] = x.z, v[i][3] = x.w;
                    } else {
                        const uint2 x = reinterpret_cast<const uint2*>(&in[(2 * kK + i * kV) * 32])[half], y = reinterpret_cast<const uint2*>(&in[(2 * kK + i * kV + kV - 1) * 32])[half];
                        v[i][0] = x.x, v[i][1] = x.y, v[i][2] = y.x, v[i][3] = y.y;
                    }
                }
#pragma unroll
                for (int w = 0; w < 2; ++w)
#pragma unroll
                    for (int odd = 0; odd < 2; ++odd) {
                        const uint32_t pick = odd ? 0x7632 : 0x5410;
                        const uint32_t a0 = __byte_perm(v[0][w], v[1][w], pick), a1 = __byte_perm(v[0][w + 2], v[1][w + 2], pick);
                        const uint32_t a2 = __byte_perm(v[2][w], v[3][w], pick), a3 = __byte_perm(v[2][w + 2], v[3][w + 2], pick);
#pragma unroll
                        for (int h = 0; h < HT; ++h) {
                            mma(o[h][half * 4 + w * 2 + odd], a0, a1, a2, a3, high[h][0], high[h][1]);
                            mma(o[h][half * 4 + w * 2 + odd], a0, a1, a2, a3, low[h][0], low[h][1]);
                        }
                    }
            }
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        __syncwarp();
        // the warp's shares: O^T back to heads in rows
#pragma unroll
        for (int h = 0; h < HT; ++h) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
#pragma unroll
                for (int d = 4; d <= 16; d <<= 1) l[h][e] += __shfl_xor_sync(0xffffffffu, l[h][e], d);
                if (g == 0) sM[warp][h * 8 + 2 * q + e] = m[h][e], sL[warp][h * 8 + 2 * q + e] = l[h][e];
            }
#pragma unroll
            for (int i = 0; i < NP / 16; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int n = g * 8 + (NP == 64 ? i + (e >> 1) * 4 : i + (e >> 1) * 64);
                    sO[(h * 8 + 2 * q + (e & 1)) * NP + n] = o[h][i][e];
                }
        }
        __syncthreads();
        const bool whole = t0 == 0 && t1 == r.tiles;
        float* part = p.work + ((i64)blockIdx.x * 2 + (t0 == 0)) * kHeads * (p.N + 2);
        const float* all_o = reinterpret_cast<const float*>(staged);
        for (int i = threadIdx.x; i < heads * p.N; i += kThreads) {
            const int h = i / p.N, n = i % p.N;
            float top = -INFINITY, x = 0.f, sum = 0.f;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) top = fmaxf(top, sM[w][h]);
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                const float keep = sM[w][h] == -INFINITY ? 0.f : ex2(sM[w][h] - top);
                sum += sL[w][h] * keep;
                // (a warp whose maximum is -infinity has sums of zeros, or NaN from a NaN score)
                if (sM[w][h] != -INFINITY) x += all_o[w * kStages * kPieces * 128 + h * NP + n] * keep;
            }
            if (whole) {
                static_cast<bf16*>(p.out)[((i64)b * p.Hq + h0 + h) * p.N + n] = __float2bfloat16_rn(sum == 0.f ? 0.f : x / sum);
                if (n == 0 && p.lse != nullptr) p.lse[(i64)b * p.Hq + h0 + h] = sum == 0.f ? -INFINITY : top * kLn2 + logf(sum);
            } else {
                part[h * (p.N + 2) + n] = x;
                if (n == 0) part[h * (p.N + 2) + p.N] = top, part[h * (p.N + 2) + p.N + 1] = sum;
            }
        }
        __syncthreads();
    }
}

// A block per unit: joins what the blocks `parts` of the kernel above have left of it.
template <typename E>
__global__ void __launch_bounds__(kThreads) join_kernel(const AttentionArgs p, int parts, int HB) {
    __shared__ i64 shared[kWarps];
    const int units = p.Hkv * p.blocks, b = blockIdx.x / units, unit = blockIdx.x % units;
    const i64 all = tiles_before(p, p.B, shared), run = run_length(all, parts);
    const Range r(p, b);
    if (r.tiles == 0) return;
    const i64 begin = tiles_before(p, b, shared) + (i64)unit * r.tiles;
    const i64 c0 = begin / run, c1 = (begin + r.tiles - 1) / run;
    if (c0 == c1) return;
    const int head = unit / p.blocks, h0 = head * p.group + unit % p.blocks * HB, heads = min(HB, (head + 1) * p.group - h0);
    const int stride = p.N + 2;
    for (int i = threadIdx.x; i < heads * p.N; i += kThreads) {
        const int h = i / p.N, n = i % p.N;
        float top = -INFINITY, x = 0.f, sum = 0.f;
        for (i64 c = c0; c <= c1; ++c) top = fmaxf(top, p.work[((c * 2 + (c == c0)) * HB + h) * stride + p.N]);
        for (i64 c = c0; c <= c1; ++c) {
            const float* part = p.work + ((c * 2 + (c == c0)) * HB + h) * stride;
            const float m = part[p.N], keep = m == -INFINITY ? 0.f : exp2f((m - top) * p.to_log2);
            sum += part[p.N + 1] * keep;
            if (m != -INFINITY) x += part[n] * keep;
        }
        static_cast<E*>(p.out)[((i64)b * p.Hq + h0 + h) * p.N + n] = from_f<E>(sum == 0.f ? 0.f : x / sum);
        if (n == 0 && p.lse != nullptr) p.lse[(i64)b * p.Hq + h0 + h] = sum == 0.f ? -INFINITY : (top * p.to_log2 + log2f(sum)) * kLn2;
    }
}

constexpr int kBlocksPerSm = 3;
int run_blocks() { return max(1, sm_count()) * kBlocksPerSm; }
int heads_of(int group) { return group >= 4 ? 4 : group >= 2 ? 2 : 1; }
int mma_heads_of(int group) { return group > 8 ? 16 : 8; }

template <typename E, int W, int HB>
int launch(AttentionArgs& p, cudaStream_t st) {
    p.blocks = (p.group + HB - 1) / HB;
    const int parts = run_blocks();
    attention_kernel<E, W, HB><<<parts, kThreads, 0, st>>>(p);
    if (int e = check_launch("paged_attention")) return e;
    join_kernel<E><<<(unsigned)((i64)p.B * p.Hkv * p.blocks), kThreads, 0, st>>>(p, parts, HB);
    return check_launch("paged_attention");
}
template <int NP, int HT>
int launch_mma(AttentionArgs& p, cudaStream_t st) {
    constexpr int smem = kWarps * kStages * (2 * (NP / 32) + 4 * (NP / 64)) * 32 * 16;
    static_assert(kStages * (2 * (NP / 32) + 4 * (NP / 64)) * 32 * 16 >= 8 * HT * NP * 4, "a warp's sums fit its stages");
    if (allow_smem<attention_mma_kernel<NP, HT>>(smem) != cudaSuccess) return check_launch("paged_attention");
    p.blocks = (p.group + 8 * HT - 1) / (8 * HT);
    p.to_log2 = 1.f;
    const int parts = run_blocks();
    attention_mma_kernel<NP, HT><<<parts, kThreads, smem, st>>>(p);
    if (int e = check_launch("paged_attention")) return e;
    join_kernel<bf16><<<(unsigned)((i64)p.B * p.Hkv * p.blocks), kThreads, 0, st>>>(p, parts, 8 * HT);
    return check_launch("paged_attention");
}
// Heads of whole 16-byte pieces that start on such boundaries, and rows of the pools that an int can number.
bool takes_mma(const AttentionArgs& p) {
    const uintptr_t all = reinterpret_cast<uintptr_t>(p.k_pages) | reinterpret_cast<uintptr_t>(p.v_pages);
    return p.N % 8 == 0 && all % 16 == 0 && (i64)p.pages * p.Hkv * p.page.d <= 0x7fffffff;
}
template <typename E>
int dispatch(AttentionArgs& p, cudaStream_t st) {
    if (sizeof(E) == 2 && takes_mma(p)) {
        if (p.group > 8) return p.N <= 64 ? launch_mma<64, 2>(p, st) : launch_mma<128, 2>(p, st);
        return p.N <= 64 ? launch_mma<64, 1>(p, st) : launch_mma<128, 1>(p, st);
    }
    p.to_log2 = kLog2e;
    const uintptr_t all = reinterpret_cast<uintptr_t>(p.k_pages) | reinterpret_cast<uintptr_t>(p.v_pages);
    const bool wide = p.N % 4 == 0 && all % (4 * sizeof(E)) == 0;   // a piece of four elements is one load
    switch (heads_of(p.group) * 2 + wide) {
        case 9: return launch<E, 4, 4>(p, st);
        case 8: return launch<E, 1, 4>(p, st);
        case 5: return launch<E, 4, 2>(p, st);
        case 4: return launch<E, 1, 2>(p, st);
        case 3: return launch<E, 4, 1>(p, st);
        default: return launch<E, 1, 1>(p, st);
    }
}

}  // namespace

int paged_attention_error(int clear) {
    int v = 0;
    if (clear) return cudaMemcpyToSymbol(g_error, &v, sizeof(v)) == cudaSuccess ? 0 : -1;
    return cudaMemcpyFromSymbol(&v, g_error, sizeof(v)) == cudaSuccess ? v : -1;
}

}  // namespace rwkvb200

using namespace rwkvb200;

extern "C" size_t rwkvb200_paged_attention_work_bytes(int dtype, int Hq, int Hkv, int N) {
    if (Hq <= 0 || Hkv <= 0 || N <= 0) return 0;
    const int heads = dtype == RWKVB200_BF16 ? mma_heads_of(Hq / Hkv) : heads_of(Hq / Hkv);
    return (size_t)run_blocks() * 2 * heads * (N + 2) * sizeof(float);
}

extern "C" int rwkvb200_paged_attention(int dtype, int B, int Hq, int Hkv, int N, int pages, int page, int width, const void* q, const void* k_pages,
                                        const void* v_pages, const int* table, const int* lengths, float scale, float cap, int window,
                                        const float* slopes, void* out, float* lse, void* work, void* stream) {
    const char* what = "paged_attention";
    RWKV_REQUIRE(dtype == RWKVB200_F32 || dtype == RWKVB200_BF16, RWKVB200_EINVAL, "%s: unknown dtype %d", what, dtype);
    RWKV_REQUIRE(B > 0 && Hq > 0 && Hkv > 0 && N > 0 && pages > 0 && page > 0 && width > 0, RWKVB200_EINVAL,
                 "%s: B=%d Hq=%d Hkv=%d N=%d pages=%d page=%d width=%d must be positive", what, B, Hq, Hkv, N, pages, page, width);
    RWKV_REQUIRE(Hq % Hkv == 0, RWKVB200_EINVAL, "%s: Hq=%d is not a multiple of Hkv=%d", what, Hq, Hkv);
    RWKV_REQUIRE(N <= RWKVB200_MAX_HEAD_SIZE, RWKVB200_EUNSUPPORTED, "%s: head size %d > %d", what, N, RWKVB200_MAX_HEAD_SIZE);
    RWKV_REQUIRE((i64)width * page <= 0x7fffffff - 1024, RWKVB200_EINVAL, "%s: %d pages of %d tokens are more than 2^31 - 1024", what, width, page);
    RWKV_REQUIRE((i64)B * Hq <= 0x7fffffff, RWKVB200_EINVAL, "%s: B=%d Hq=%d are too many", what, B, Hq);
    RWKV_REQUIRE(window >= 0, RWKVB200_EINVAL, "%s: window=%d is negative", what, window);
    RWKV_REQUIRE(cap >= 0.f, RWKVB200_EINVAL, "%s: cap=%g is negative", what, cap);
    RWKV_NOTNULL(q); RWKV_NOTNULL(k_pages); RWKV_NOTNULL(v_pages); RWKV_NOTNULL(table); RWKV_NOTNULL(lengths); RWKV_NOTNULL(out); RWKV_NOTNULL(work);
    AttentionArgs p{B, Hq, Hkv, N, pages, width, window, Hq / Hkv, 1, scale, cap, 1.f, Divisor((uint32_t)page), q, k_pages, v_pages, table, lengths, slopes, out, lse, static_cast<float*>(work)};
    return dtype == RWKVB200_BF16 ? dispatch<bf16>(p, as_stream(stream)) : dispatch<float>(p, as_stream(stream));
}
