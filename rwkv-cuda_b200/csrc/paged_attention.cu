// Attention of one new token per sequence over a paged cache.  For head h of sequence b with `len` tokens:
//
//   z_j = scale q.k_j      z_j = cap tanh(z_j / cap)      z_j += slope_h (j - (len - 1))      max(0, len - window) <= j < len
//   out = sum_j exp(z_j - m) v_j / sum_j exp(z_j - m)     lse = m + log(sum)                  m = max_j z_j
//
// The keys and values of the sequences are read once for each block of up to 16 (bf16) or 8 (fp32) query heads that share them, with few
// sequences out of L2 from the second time on; memory bounds it up to there, the products beyond (128 sequences of up to 4096
// tokens, 8 key-value heads of 128, bf16: 4 to 8 query heads on each 199 to 252 us, 16 360, 32 685; fp32: 8 468, 16 910, 32 1810).  The work is all tiles (of 64 or 32 tokens) of all units (a
// sequence, a key-value head, a block of its query heads) behind one another; every block takes an equal run of them, so that
// one long sequence and many of different lengths both fill the GPU.  A unit that lies in one block's run is finished there; of
// the others each block leaves (m, sum, sum of exp v) and a second kernel joins them.  A block's run has at most one unit that
// began before it and one that ends behind it: two places a block.
#include "packed.cuh"
#include "paged.cuh"
#include "wkv7_umma.cuh"
#include <cooperative_groups.h>
#include <cuda.h>
#include <type_traits>

namespace rwkvb200 {
namespace {

__device__ int g_error = 0;
constexpr int kThreads = 128, kWarps = kThreads / 32;
constexpr int kMinTokens = 64;    // of a block's run (1000 tokens of 12 heads, fp32: 18.9 us with 256, 14.6 with 128, 12.9, 13.5 with 32)

struct AttentionArgs {
    int B, Hq, Hkv, N, pages, width, window, group, blocks;   // blocks of query heads per key-value head
    int tile_bits;                                            // a tile has 1 << tile_bits tokens, 16 or 8 for each warp
    float scale, cap;
    Divisor page;
    const void *q, *k_pages, *v_pages;
    const int *table, *lengths;
    const float* slopes;
    void* out;
    float *lse, *work;
};

struct Range {
    int lo, hi, start, tiles;   // tokens of a sequence that count; its tiles, from a multiple of 16 on: one at least, so that empty
                                // sequences get their zeros, and none for a row that only pads the batch
    __device__ __forceinline__ Range(const AttentionArgs& p, int b) {
        hi = min(p.lengths[b], p.width * (int)p.page.d);
        lo = p.window > 0 ? max(0, hi - p.window) : 0;
        start = lo & ~15;
        tiles = hi < 0 ? 0 : max(1, (hi - start + (1 << p.tile_bits) - 1) >> p.tile_bits);
    }
};

__device__ __forceinline__ i64 run_length(const AttentionArgs& p, i64 all, int blocks) { return max((i64)(kMinTokens >> p.tile_bits), (all + blocks - 1) / blocks); }

// Where a run begins among the tiles of all units.
struct Start {
    i64 all, run, tile;   // tiles of all units; of a run; the run's first
    i64 base;             // tiles of the sequences before `b`, which `tile` lies in
    int b;
};
// All threads of a block: run number `index` of `runs`; tile >= all: there is none.
template <int THREADS>
__device__ __forceinline__ Start find_start(const AttentionArgs& p, int index, int runs, int units) {
    __shared__ i64 sums[THREADS / 32], found[2];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    // up to a sequence per thread in one pass; more are gone through twice, as their sum has to be known first
    const bool once = p.B <= THREADS;
    Start s;
    s.all = 0;
    if (!once) {
        i64 n = 0;
        for (int b = threadIdx.x; b < p.B; b += THREADS) n += Range(p, b).tiles;
#pragma unroll
        for (int d = 16; d >= 1; d >>= 1) n += __shfl_xor_sync(0xffffffffu, n, d);
        if (lane == 0) sums[warp] = n;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < THREADS / 32; ++w) s.all += sums[w];
        s.all *= units;
        s.run = run_length(p, s.all, runs);
        s.tile = s.run * index;
        __syncthreads();
    }
    i64 base = 0;
    for (int b0 = 0; b0 < p.B; b0 += THREADS) {
        const int b = b0 + threadIdx.x;
        const i64 n = b < p.B ? (i64)Range(p, b).tiles * units : 0;
        i64 x = n;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const i64 o = __shfl_up_sync(0xffffffffu, x, d);
            if (lane >= d) x += o;
        }
        if (lane == 31) sums[warp] = x;
        __syncthreads();
        i64 before = base;
#pragma unroll
        for (int w = 0; w < THREADS / 32; ++w) {
            if (w < warp) before += sums[w];
            base += sums[w];
        }
        x += before;
        if (once) {
            s.all = base;
            s.run = run_length(p, s.all, runs);
            s.tile = s.run * index;
        }
        if (s.tile >= x - n && s.tile < x) found[0] = b, found[1] = x - n;
        __syncthreads();
        if (base > s.tile) break;   // (the same for all threads)
    }
    s.b = (int)found[0];
    s.base = found[1];
    return s;
}

// A step of a warp is 16 (bf16) or 8 (fp32) tokens.  Their keys and values lie in shared memory as boxes of [tokens][128 bytes] in the
// 128-byte swizzle (piece c of 16 bytes of row t is at c ^ (t & 7)), one behind the other for longer rows; heads are filled up
// with zeros to NP = 64 or 128 elements.  A warp has slots for the keys of two steps and the values of two.  They get there
//   kTma:      by one bulk copy each (pages of a multiple of 16 tokens, heads of 64 or 128): a warp's lane 0 asks, keys two steps
//              ahead and values one, and counts the bytes on a barrier of the slot.  A step lies in one page: one lookup;
//   kPieces:   by cp.async in pieces of 16 bytes, rows that do not count filled with zeros (heads of whole pieces);
//   kElements: element by element, by cp.async (fp32) or through registers (bf16).
// (128 sequences of up to 4096 tokens, heads of 128: 205 us by TMA; 273 us by pieces, 267 of them without any product.)
enum { kTma, kPieces, kElements };
// LONE: a cluster of blocks has a unit of its own and nothing is left for a second kernel (launch_steps has the rule).
constexpr int kMaxCluster = 8;
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
// the upper digits of v > 0 as a bf16 number, short of all of it: the rest is 2^-12 to 2^-6.9 of v and exact
__device__ __forceinline__ float upper_half(float v) { return __uint_as_float(__float_as_uint(v * (1.f - 1.f / 4096.f)) & 0xffff0000u); }
// ... of a small weight it would come to 0, and 0 times an infinite value to NaN.  Two weights: their lower parts are the smallest number
// there is (2^-133) at least, but 0 where the upper part, and with it the weight, is 0.
__device__ __forceinline__ uint32_t least_part(uint32_t upper) {
    uint32_t d;
    asm("min.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(upper), "r"(0x00010001u));
    return d;
}
__device__ __forceinline__ uint32_t at_least(uint32_t v, uint32_t least) {
    uint32_t d;
    asm("max.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(v), "r"(least));
    return d;
}
__device__ __forceinline__ void commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int BYTES>
__device__ __forceinline__ void copy_or_zero(uint32_t shared, const void* from, bool there) {
    if (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(shared), "l"(from), "r"(there ? 16 : 0) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(shared), "l"(from), "r"(there ? 4 : 0) : "memory");
}

__device__ __forceinline__ void ldmatrix(uint32_t (&d)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void ldmatrix_transposed(uint32_t (&d)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3]) : "r"(at) : "memory");
}
// a step's rows of a pool, from number `row` on, counted on `bar`
__device__ __forceinline__ void copy_rows(uint32_t to, const CUtensorMap* map, int row, uint64_t* bar, int bytes) {
    const uint32_t b = (uint32_t)__cvta_generic_to_shared(bar);
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(b), "r"(bytes) : "memory");
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(to),
                 "l"(reinterpret_cast<uint64_t>(map)), "r"(0), "r"(row), "r"(0), "r"(b)
                 : "memory");
}
struct Maps {
    CUtensorMap keys, values;
};

// A warp's part of a unit: tokens, pages and slots.
template <typename E, int NP, int MODE>
struct Steps {
    static constexpr bool TMA = MODE == kTma;
    using Place = std::conditional_t<TMA, int, i64>;   // (the coordinate of a bulk copy is an int)
    static constexpr int kTokens = sizeof(E) == 2 ? 16 : 8, kBoxes = NP * (int)sizeof(E) / 128, kBox = kTokens * 128, kRows = kBox * kBoxes;
    static constexpr int kWarpBytes = 4 * kRows;   // the slots: keys, keys, values, values
    const AttentionArgs& p;
    const Maps& maps;
    uint64_t* bars;          // TMA: one per slot
    uint32_t slots;          // address in shared memory
    int lane;
    uint32_t phases = 0;     // of the four barriers
    bool lost = false;       // a wait ran out: nothing more is asked for, and the results are NaN
    // the unit
    const int* row;
    int head, lo, from, last, steps;

    __device__ __forceinline__ Steps(const AttentionArgs& p, const Maps& maps, uint64_t* bars, void* slots, int lane)
        : p(p), maps(maps), bars(bars), slots((uint32_t)__cvta_generic_to_shared(slots)), lane(lane) {
        if (TMA && lane < 4) asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"((uint32_t)__cvta_generic_to_shared(&bars[lane])));
        if (TMA) v7u::proxy_fence();
        __syncwarp();   // (lane 0 uses what the others have made)
    }
    __device__ __forceinline__ void unit(int b, const Range& r, int t0, int t1, int head_, int warp) {
        row = p.table + (i64)b * p.width;
        head = head_;
        lo = r.lo;
        from = r.start + (t0 << p.tile_bits) + warp * kTokens;
        last = min(r.start + (t1 << p.tile_bits), r.hi);
        steps = lost ? 0 : t1 - t0;
    }
    __device__ __forceinline__ int first(int step) const { return from + (step << p.tile_bits); }
    __device__ __forceinline__ bool counts(int j) const { return j >= lo && j < last; }
    // Of a step's tokens a lane answers for one (TMA: all for the first).  Its page is asked for a step before it is looked at.
    __device__ __forceinline__ int token(int step) const { return first(step) + (TMA ? 0 : lane & (kTokens - 1)); }
    __device__ __forceinline__ bool in_use(int step, int j) const { return step < steps && (TMA ? j < last : counts(j)); }
    __device__ __forceinline__ int page(int step) const {
        const int j = token(step);
        return in_use(step, j) ? row[p.page.quotient((uint32_t)j)] : 0;
    }
    // the row of the pools that the token lies in; -1: it does not count
    __device__ __forceinline__ Place place(int step, int id) const {
        const int j = token(step);
        if (!in_use(step, j)) return -1;
        if ((unsigned)id >= (unsigned)p.pages) {
            atomicMax(&g_error, kBadPage);
            return -1;
        }
        return ((Place)id * p.Hkv + head) * (int)p.page.d + (j - (int)(p.page.quotient((uint32_t)j) * p.page.d));
    }
    // whether token t of a step counts, from its place n
    __device__ __forceinline__ bool there(int step, Place n, int t) const {
        return TMA ? n >= 0 && counts(first(step) + t) : __shfl_sync(0xffffffffu, n, t) >= 0;
    }
    __device__ __forceinline__ uint32_t keys(int step) const { return slots + (step & 1) * kRows; }
    __device__ __forceinline__ uint32_t values(int step) const { return slots + (2 + (step & 1)) * kRows; }
    template <bool VALUES>
    __device__ __forceinline__ void ask(int step, Place n) const {
        const uint32_t to = VALUES ? values(step) : keys(step);
        if (TMA) {
            if (lane == 0 && n >= 0) copy_rows(to, VALUES ? &maps.values : &maps.keys, n, &bars[VALUES * 2 + (step & 1)], kRows);
            return;
        }
        const E* pool = static_cast<const E*>(VALUES ? p.v_pages : p.k_pages);
        constexpr int kPer = 16 / sizeof(E);
        if (MODE == kPieces) {
#pragma unroll
            for (int i = 0; i < kRows / 512; ++i) {
                const int piece = i * 32 + lane, t = piece / (8 * kBoxes), c = piece % (8 * kBoxes);
                const Place k = __shfl_sync(0xffffffffu, n, t);
                copy_or_zero<16>(to + (c >> 3) * kBox + t * 128 + (((c ^ t) & 7) << 4), pool + max(k, (Place)0) * p.N + min(c * kPer, p.N - kPer), k >= 0 && c * kPer < p.N);
            }
        } else {
#pragma unroll
            for (int t = 0; t < kTokens; ++t) {
                const Place k = __shfl_sync(0xffffffffu, n, t);
#pragma unroll
                for (int i = 0; i < NP / 32; ++i) {
                    const int e = i * 32 + lane, c = e / kPer;
                    const bool there = k >= 0 && e < p.N;
                    const uint32_t at = to + (c >> 3) * kBox + t * 128 + (((c ^ t) & 7) << 4) + e % kPer * (int)sizeof(E);
                    const E* from = pool + (there ? k * p.N + e : 0);
                    if constexpr (sizeof(E) == 4) {
                        copy_or_zero<4>(at, from, there);
                    } else {
                        const unsigned short v = there ? *reinterpret_cast<const unsigned short*>(from) : (unsigned short)0;
                        asm volatile("st.shared.b16 [%0], %1;" ::"r"(at), "h"(v) : "memory");
                    }
                }
            }
        }
    }
    // waits for the copies of all but the last group (TMA: for those that have been asked for)
    template <bool VALUES>
    __device__ __forceinline__ void arrived(int step, Place n) {
        if (!TMA) {
            asm volatile("cp.async.wait_group 1;" ::: "memory");
        } else if (n >= 0) {
            const int which = VALUES * 2 + (step & 1);
            if (__any_sync(0xffffffffu, !v7u::mbar_wait(&bars[which], phases >> which & 1))) lost = true;
            phases ^= 1u << which;
        }
    }
    __device__ __forceinline__ void finish() {   // nothing is in flight behind it
        if (!TMA) asm volatile("cp.async.wait_group 0;" ::: "memory");
        if (lost) {
            for (int i = 0; i < 4; ++i) v7u::mbar_wait(&bars[i], phases >> i & 1, 1 << 10);
            if (lane == 0) atomicMax(&g_error, kTimeout);
        }
        __syncwarp();
    }
};

// The sums of a unit's warps, sO [head][NP] behind one another every `stride` floats, with their maxima (as exponents of 2) and
// weights: joined, and written as results or as this block's share.
template <typename E, int NP, int HEADS>
__device__ __forceinline__ void write_unit(const AttentionArgs& p, const float* sO, int stride, const float (*sM)[HEADS], const float (*sL)[HEADS], int b, int h0,
                                           int heads, bool whole, bool begins) {
    float* part = p.work + ((i64)blockIdx.x * 2 + begins) * HEADS * (p.N + 2);
    for (int i = threadIdx.x; i < heads * NP; i += kThreads) {
        const int h = i / NP, n = i % NP;
        if (n >= p.N) continue;
        float top = -INFINITY, x = 0.f, sum = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) top = fmaxf(top, sM[w][h]);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            const float keep = sM[w][h] == -INFINITY ? 0.f : ex2(sM[w][h] - top);
            sum += sL[w][h] * keep;
            // (a warp whose maximum is -infinity has sums of zeros, or NaN from a NaN score)
            if (sM[w][h] != -INFINITY) x += sO[w * stride + h * NP + n] * keep;
        }
        if (whole) {
            static_cast<E*>(p.out)[((i64)b * p.Hq + h0 + h) * p.N + n] = from_f<E>(sum == 0.f ? 0.f : x / sum);
            if (n == 0 && p.lse != nullptr) p.lse[(i64)b * p.Hq + h0 + h] = sum == 0.f ? -INFINITY : top * kLn2 + logf(sum);
        } else {
            part[h * (p.N + 2) + n] = x;
            if (n == 0) part[h * (p.N + 2) + p.N] = top, part[h * (p.N + 2) + p.N + 1] = sum;
        }
    }
}

// The same where a cluster of K blocks has a unit to itself: the warps' sums are joined in the block's shared memory (in place of the first
// warp's), then every block joins a K-th of the elements of all blocks and writes the results.
template <typename E, int NP, int HEADS>
__device__ __forceinline__ void write_from_cluster(const AttentionArgs& p, float* sO, int stride, const float (*sM)[HEADS], const float (*sL)[HEADS], float* sTop,
                                                   float* sSum, int b, int h0, int heads) {
    namespace cg = cooperative_groups;
    cg::cluster_group cluster = cg::this_cluster();
    const int K = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    for (int i = threadIdx.x; i < heads * NP; i += kThreads) {
        const int h = i / NP;
        float top = -INFINITY, x = 0.f, sum = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) top = fmaxf(top, sM[w][h]);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            const float keep = sM[w][h] == -INFINITY ? 0.f : ex2(sM[w][h] - top);
            sum += sL[w][h] * keep;
            if (sM[w][h] != -INFINITY) x += sO[w * stride + i] * keep;
        }
        sO[i] = x;
        if (i % NP == 0) sTop[h] = top, sSum[h] = sum;
    }
    cluster.sync();
    const int each = (heads * NP + K - 1) / K, end = min((rank + 1) * each, heads * NP);
    for (int i = rank * each + threadIdx.x; i < end; i += kThreads) {
        const int h = i / NP, n = i % NP;
        if (n >= p.N) continue;
        float m[kMaxCluster], l[kMaxCluster], x[kMaxCluster], top = -INFINITY, all = 0.f, sum = 0.f;
#pragma unroll
        for (int k = 0; k < kMaxCluster; ++k) {
            const bool there = k < K;
            m[k] = there ? *cluster.map_shared_rank(sTop + h, k) : -INFINITY;
            l[k] = there ? *cluster.map_shared_rank(sSum + h, k) : 0.f;
            x[k] = there ? *cluster.map_shared_rank(sO + i, k) : 0.f;
            top = fmaxf(top, m[k]);
        }
#pragma unroll
        for (int k = 0; k < kMaxCluster; ++k) {
            const float keep = m[k] == -INFINITY ? 0.f : ex2(m[k] - top);
            sum += l[k] * keep;
            if (m[k] != -INFINITY) all += x[k] * keep;
        }
        static_cast<E*>(p.out)[((i64)b * p.Hq + h0 + h) * p.N + n] = from_f<E>(sum == 0.f ? 0.f : all / sum);
        if (n == 0 && p.lse != nullptr) p.lse[(i64)b * p.Hq + h0 + h] = sum == 0.f ? -INFINITY : top * kLn2 + logf(sum);
    }
    cluster.sync();   // (a block's shared memory is read until all are done)
}

// bf16: products on mma.sync m16n8k16 with the tokens in the rows, S^T = K q^T and O^T = V^T P^T, for up to 8 HT query heads that share
// the keys.  Eight heads make 52 TFLOP/s at the full rate of memory, which mma.sync does with a seventh of its time: the tiles
// are too narrow for tensor memory to give anything.  Each warp keeps its own maxima and sums.  Both first operands come out of
// shared memory by ldmatrix (the values transposed).  Weights are taken into the second product as the sum of three bf16
// numbers (2^-22 relative, as good as fp32; two leave 2^-16, which shows where values cancel), all above 0, so that an
// infinite value stays one.
// 128 sequences of up to 4096 tokens, 32 heads on 8 of 128: 199 to 203 us with the join, 5.4 TB/s (82 % of the copy rate); one of 131001
// tokens 101 us, 5.3 TB/s.  Short sequences spend their time at the ends of units: 64 of up to 2048 tokens 3.9 TB/s, heads of 64 3.4.
template <int NP, int HT, int MODE, bool LONE>
__global__ void __launch_bounds__(kThreads, 3) attention_mma_kernel(const AttentionArgs p, const __grid_constant__ Maps maps) {
    using Way = Steps<bf16, NP, MODE>;
    using Place = typename Way::Place;
    constexpr bool TMA = MODE == kTma;
    constexpr int kHeads = 8 * HT;
    extern __shared__ __align__(1024) unsigned char staged[];
    __shared__ float sM[kWarps][kHeads], sL[kWarps][kHeads], sTop[kHeads], sSum[kHeads];
    __shared__ uint64_t bars[kWarps][4];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, q = lane & 3;
    const int units = p.Hkv * p.blocks, N = TMA ? NP : p.N;
    unsigned char* mine = staged + warp * Way::kWarpBytes;
    if (TMA && threadIdx.x == 0) {
        asm volatile("prefetch.tensormap [%0];" ::"l"(&maps.keys) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&maps.values) : "memory");
    }
    Way way(p, maps, bars[warp], mine, lane);
    Start start{0, 1, 0, 0, 0};
    if (!LONE) {
        start = find_start<kThreads>(p, blockIdx.x, gridDim.x, units);
        if (start.tile >= start.all) return;
        asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    }
    const i64 end = LONE ? 1 : min(start.tile + start.run, start.all);
    // where a lane's rows for ldmatrix lie: keys: rows lane & 15, piece lane / 16; values: rows by 8 from lane / 16, piece by lane / 8
    const uint32_t key_row = (lane & 15) * 128, key_piece = lane >> 4, value_row = ((lane & 7) + (lane >> 4) * 8) * 128, value_piece = lane >> 3 & 1, swizzle = lane & 7;
    const float scale = p.cap > 0.f ? p.scale / p.cap : p.scale * kLog2e, cap = p.cap * kLog2e;
    int b = start.b;
    i64 base = start.base;
    for (i64 at = start.tile; at < end;) {
        int unit, t0, t1;
        if (LONE) {
            const cooperative_groups::cluster_group cluster = cooperative_groups::this_cluster();
            const int K = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
            unit = blockIdx.x / K;
            b = unit / units;
            unit -= b * units;
            const int tiles = Range(p, b).tiles;
            if (tiles == 0) return;   // (the same for the whole cluster)
            t0 = tiles * rank / K;
            t1 = tiles * (rank + 1) / K;
            at = 1;
        } else {
            const int tiles = Range(p, b).tiles;
            if (at >= base + (i64)tiles * units) {   // (a row without tiles is passed over as well)
                base += (i64)tiles * units;
                ++b;
                continue;
            }
            unit = (int)((at - base) / tiles);
            t0 = (int)((at - base) % tiles);
            t1 = (int)min((i64)tiles, t0 + (end - at));
            at += t1 - t0;
        }
        const Range r(p, b);
        const int head = unit / p.blocks, h0 = head * p.group + unit % p.blocks * kHeads, heads = min(kHeads, (head + 1) * p.group - h0);
        if (threadIdx.x == 0 && p.lengths[b] > r.hi) atomicMax(&g_error, kBadLength);
        way.unit(b, r, t0, t1, head, warp);
        const int id0 = way.page(0), id1 = way.page(1);
        int id2 = way.page(2);
        Place n0 = way.place(0, id0), n1 = way.place(1, id1);
        way.template ask<false>(0, n0);
        commit();
        way.template ask<false>(1, n1);
        way.template ask<true>(0, n0);
        commit();
        // q as the second operand of the scores: head g (and g + 8)
        uint32_t qf[HT][NP / 16][2];
#pragma unroll
        for (int h = 0; h < HT; ++h)
#pragma unroll
            for (int j = 0; j < NP / 8; ++j) {
                const bf16* from = static_cast<const bf16*>(p.q) + ((i64)b * p.Hq + h0 + h * 8 + g) * N + j * 8 + q * 2;
                __nv_bfloat162 v = __floats2bfloat162_rn(0.f, 0.f);
                if (h * 8 + g < heads) {
                    if (j * 8 + q * 2 < N) v.x = from[0];
                    if (j * 8 + q * 2 + 1 < N) v.y = from[1];
                }
                qf[h][j / 2][j % 2] = *reinterpret_cast<const uint32_t*>(&v);
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
        // The scores of a step are made while the step before it is summed.
        float next[HT][4];
        auto scores = [&](int step) {
            const uint32_t in = way.keys(step) + key_row;
#pragma unroll
            for (int h = 0; h < HT; ++h)
#pragma unroll
                for (int e = 0; e < 4; ++e) next[h][e] = 0.f;
#pragma unroll
            for (int j = 0; j < NP / 16; ++j) {
                uint32_t a[4];
                ldmatrix(a, in + j / 4 * Way::kBox + (((j % 4 * 2 + key_piece) ^ swizzle) << 4));
#pragma unroll
                for (int h = 0; h < HT; ++h) mma(next[h], a[0], a[1], a[2], a[3], qf[h][j][0], qf[h][j][1]);
            }
        };
        way.template arrived<false>(0, n0);
        __syncwarp();
        scores(0);
        for (int step = 0; step < way.steps && !way.lost; ++step) {
            float z[HT][4];
#pragma unroll
            for (int h = 0; h < HT; ++h)
#pragma unroll
                for (int e = 0; e < 4; ++e) z[h][e] = next[h][e];
            const Place n2 = way.place(step + 2, id2);
            id2 = way.page(step + 3);
            __syncwarp();                 // (all lanes have read the slots that are asked for)
            way.template ask<false>(step + 2, n2);
            way.template ask<true>(step + 1, n1);
            commit();
            way.template arrived<false>(step + 1, n1);
            way.template arrived<true>(step, n0);
            __syncwarp();
            scores(step + 1);
            const Place n = n0;
            n0 = n1;
            n1 = n2;
            if (!__any_sync(0xffffffffu, n >= 0)) continue;   // no token counts
            // scores as exponents of 2: tokens g (elements 0, 1) and g + 8 (2, 3)
            const bool there[2] = {way.there(step, n, g), way.there(step, n, g + 8)};
            const float distance = (float)(way.first(step) + g - (r.hi - 1));
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
                // a token without weight in any head counts for nothing, whatever its value (or the memory behind the last token) holds
                bool dead[2] = {true, true};
#pragma unroll
                for (int h = 0; h < HT; ++h)
#pragma unroll
                    for (int e = 0; e < 4; ++e) dead[e >> 1] &= h * 8 + 2 * q + (e & 1) >= heads || z[h][e] == -INFINITY;
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    uint32_t gone = __ballot_sync(0xffffffffu, dead[i]);
                    gone &= gone >> 1;
                    gone = gone & gone >> 2 & 0x11111111u;   // bit 4 t: token t (+ 8)
                    for (; gone != 0; gone &= gone - 1) {
                        const int token = i * 8 + (__ffs(gone) - 1) / 4;
                        if (lane < 8 * Way::kBoxes) {
                            unsigned char* to = mine + (2 + (step & 1)) * Way::kRows + lane / 8 * Way::kBox + token * 128 + lane % 8 * 16;
                            *reinterpret_cast<uint4*>(to) = make_uint4(0, 0, 0, 0);
                        }
                    }
                }
                if (TMA) v7u::proxy_fence();
                __syncwarp();
            }
            // weights, and as the second operand of the second product
            uint32_t high[HT][2], middle[HT][2], low[HT][2];
#pragma unroll
            for (int h = 0; h < HT; ++h) {
                float x[4], y[4], r[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float top = m[h][e & 1], w = ex2(z[h][e] - (top == -INFINITY ? 0.f : top));
                    l[h][e & 1] += w;
                    x[e] = upper_half(w);
                    r[e] = w - x[e];
                    y[e] = upper_half(r[e]);
                    r[e] -= y[e];
                }
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const uint32_t upper = pack_bf16(x[2 * i], x[2 * i + 1]), least = least_part(upper);
                    high[h][i] = transposed(upper);
                    middle[h][i] = transposed(at_least(pack_bf16(y[2 * i], y[2 * i + 1]), least));
                    low[h][i] = transposed(at_least(pack_bf16(r[2 * i], r[2 * i + 1]), least));
                }
            }
            const uint32_t in = way.values(step) + value_row;
#pragma unroll
            for (int i = 0; i < NP / 16; ++i) {
                uint32_t a[4];
                ldmatrix_transposed(a, in + i / 4 * Way::kBox + (((i % 4 * 2 + value_piece) ^ swizzle) << 4));
#pragma unroll
                for (int h = 0; h < HT; ++h) {
                    mma(o[h][i], a[0], a[1], a[2], a[3], high[h][0], high[h][1]);
                    mma(o[h][i], a[0], a[1], a[2], a[3], middle[h][0], middle[h][1]);
                    mma(o[h][i], a[0], a[1], a[2], a[3], low[h][0], low[h][1]);
                }
            }
        }
        way.finish();
        // the warp's shares, in its slots: O^T back to heads in rows
        float* sO = reinterpret_cast<float*>(mine);
#pragma unroll
        for (int h = 0; h < HT; ++h) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                if (way.lost) m[h][e] = 0.f, l[h][e] = __int_as_float(0x7fffffff);   // results that cannot pass as such
#pragma unroll
                for (int d = 4; d <= 16; d <<= 1) l[h][e] += __shfl_xor_sync(0xffffffffu, l[h][e], d);
                if (g == 0) sM[warp][h * 8 + 2 * q + e] = m[h][e], sL[warp][h * 8 + 2 * q + e] = l[h][e];
            }
#pragma unroll
            for (int i = 0; i < NP / 16; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) sO[(h * 8 + 2 * q + (e & 1)) * NP + i * 16 + g + (e >> 1) * 8] = o[h][i][e];
        }
        __syncthreads();
        if (LONE) {
            write_from_cluster<bf16, NP, kHeads>(p, reinterpret_cast<float*>(staged), Way::kWarpBytes / 4, sM, sL, sTop, sSum, b, h0, heads);
            return;
        }
        write_unit<bf16, NP, kHeads>(p, reinterpret_cast<const float*>(staged), Way::kWarpBytes / 4, sM, sL, b, h0, heads, t0 == 0 && t1 == r.tiles, t0 == 0);
        if (TMA) v7u::proxy_fence();
        __syncthreads();
    }
}

// fp32: packed multiply-adds, for up to HB query heads that share the keys.  Scores: lane (part, t) takes a quarter of key t
// times all queries (which lie in shared memory, scaled), and the quarters are added so that lane (part, t) ends with the scores of
// HB / 4 heads (q times the scale is rounded once more than q: half a unit of the score).  Sums: a lane has NP / 32 elements of every head, the weights of a token come out of shared memory.  One sequence of
// 100000 tokens, 64 heads on 8 of 128: 5.7 TB/s; 32 of up to 2048 tokens, 32 heads on 8: 4.0.
template <int NP, int HB, int MODE, bool LONE>
__global__ void __launch_bounds__(kThreads, 3) attention_fp32_kernel(const AttentionArgs p, const __grid_constant__ Maps maps) {
    using Way = Steps<float, NP, MODE>;
    using Place = typename Way::Place;
    constexpr bool TMA = MODE == kTma;
    constexpr int kMine = HB / 4, kQuarter = NP / 4, kPad = kQuarter + 4;   // (padded: the four quarters are read at once)
    extern __shared__ __align__(1024) unsigned char staged[];
    __shared__ float sM[kWarps][HB], sL[kWarps][HB], sTop[HB], sSum[HB];
    __shared__ __align__(16) float sQ[HB][4][kPad], sW[kWarps][8][HB];
    __shared__ uint64_t bars[kWarps][4];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, t = lane & 7, part = lane >> 3;
    const int units = p.Hkv * p.blocks;
    unsigned char* mine = staged + warp * Way::kWarpBytes;
    if (TMA && threadIdx.x == 0) {
        asm volatile("prefetch.tensormap [%0];" ::"l"(&maps.keys) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&maps.values) : "memory");
    }
    Way way(p, maps, bars[warp], mine, lane);
    Start start{0, 1, 0, 0, 0};
    if (!LONE) {
        start = find_start<kThreads>(p, blockIdx.x, gridDim.x, units);
        if (start.tile >= start.all) return;
        asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    }
    const i64 end = LONE ? 1 : min(start.tile + start.run, start.all);
    const float scale = p.cap > 0.f ? p.scale / p.cap : p.scale * kLog2e, cap = p.cap * kLog2e;
    int b = start.b;
    i64 base = start.base;
    for (i64 at = start.tile; at < end;) {
        int unit, t0, t1;
        if (LONE) {
            const cooperative_groups::cluster_group cluster = cooperative_groups::this_cluster();
            const int K = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
            unit = blockIdx.x / K;
            b = unit / units;
            unit -= b * units;
            const int tiles = Range(p, b).tiles;
            if (tiles == 0) return;   // (the same for the whole cluster)
            t0 = tiles * rank / K;
            t1 = tiles * (rank + 1) / K;
            at = 1;
        } else {
            const int tiles = Range(p, b).tiles;
            if (at >= base + (i64)tiles * units) {   // (a row without tiles is passed over as well)
                base += (i64)tiles * units;
                ++b;
                continue;
            }
            unit = (int)((at - base) / tiles);
            t0 = (int)((at - base) % tiles);
            t1 = (int)min((i64)tiles, t0 + (end - at));
            at += t1 - t0;
        }
        const Range r(p, b);
        const int head = unit / p.blocks, h0 = head * p.group + unit % p.blocks * HB, heads = min(HB, (head + 1) * p.group - h0);
        if (threadIdx.x == 0 && p.lengths[b] > r.hi) atomicMax(&g_error, kBadLength);
        way.unit(b, r, t0, t1, head, warp);
        const int id0 = way.page(0), id1 = way.page(1);
        int id2 = way.page(2);
        Place n0 = way.place(0, id0), n1 = way.place(1, id1);
        way.template ask<false>(0, n0);
        commit();
        way.template ask<false>(1, n1);
        way.template ask<true>(0, n0);
        commit();
        for (int i = threadIdx.x; i < HB * NP; i += kThreads) {
            const int h = i / NP, n = i % NP;
            sQ[h][n / kQuarter][n % kQuarter] = h < heads && n < p.N ? static_cast<const float*>(p.q)[((i64)b * p.Hq + h0 + h) * p.N + n] * scale : 0.f;
        }
        __syncthreads();
        float slope[kMine], m[kMine], l[kMine];   // heads part * kMine + i
        f2 o[HB][NP / 64];
#pragma unroll
        for (int i = 0; i < kMine; ++i) {
            slope[i] = p.slopes != nullptr && part * kMine + i < heads ? p.slopes[h0 + part * kMine + i] * kLog2e : 0.f;
            m[i] = -INFINITY;
            l[i] = 0.f;
        }
#pragma unroll
        for (int h = 0; h < HB; ++h)
#pragma unroll
            for (int e = 0; e < NP / 64; ++e) o[h][e] = 0;
        float next[kMine];
        auto scores = [&](int step) {
            const unsigned char* in = mine + (step & 1) * Way::kRows + t * 128;
            f2 sum[HB];
#pragma unroll
            for (int h = 0; h < HB; ++h) sum[h] = 0;
#pragma unroll
            for (int c = 0; c < kQuarter / 4; ++c) {
                const int piece = part * (kQuarter / 4) + c;
                const ulonglong2 k = *reinterpret_cast<const ulonglong2*>(in + piece / 8 * Way::kBox + (((piece & 7) ^ t) << 4));
#pragma unroll
                for (int h = 0; h < HB; ++h) {
                    const ulonglong2 v = *reinterpret_cast<const ulonglong2*>(&sQ[h][part][c * 4]);
                    sum[h] = fma2(k.x, v.x, sum[h]);
                    sum[h] = fma2(k.y, v.y, sum[h]);
                }
            }
            // a half of the heads stays, the other goes to the lane across, twice
            float x[HB];
#pragma unroll
            for (int h = 0; h < HB; ++h) x[h] = sum2(sum[h]);
#pragma unroll
            for (int i = 0; i < HB / 2; ++i) {
                const float keep = part & 2 ? x[HB / 2 + i] : x[i], give = part & 2 ? x[i] : x[HB / 2 + i];
                x[i] = keep + __shfl_xor_sync(0xffffffffu, give, 16);
            }
#pragma unroll
            for (int i = 0; i < kMine; ++i) {
                const float keep = part & 1 ? x[kMine + i] : x[i], give = part & 1 ? x[i] : x[kMine + i];
                next[i] = keep + __shfl_xor_sync(0xffffffffu, give, 8);
            }
        };
        way.template arrived<false>(0, n0);
        __syncwarp();
        scores(0);
        for (int step = 0; step < way.steps && !way.lost; ++step) {
            float z[kMine];
#pragma unroll
            for (int i = 0; i < kMine; ++i) z[i] = next[i];
            const Place n2 = way.place(step + 2, id2);
            id2 = way.page(step + 3);
            __syncwarp();                 // (all lanes have read the slots that are asked for, and the weights)
            way.template ask<false>(step + 2, n2);
            way.template ask<true>(step + 1, n1);
            commit();
            way.template arrived<false>(step + 1, n1);
            way.template arrived<true>(step, n0);
            __syncwarp();
            scores(step + 1);
            const Place n = n0;
            n0 = n1;
            n1 = n2;
            if (!__any_sync(0xffffffffu, n >= 0)) continue;   // no token counts
            const bool there = way.there(step, n, t);
            const float distance = (float)(way.first(step) + t - (r.hi - 1));
            bool more = false, dead = true;
#pragma unroll
            for (int i = 0; i < kMine; ++i) {
                float v = z[i];
                if (p.cap > 0.f) v = cap * hyperbolic_tangent(v);
                v = fmaf(slope[i], distance, v);
                v = there ? v : -INFINITY;
                z[i] = v;
                more |= v > m[i];
                dead &= part * kMine + i >= heads || v == -INFINITY;
            }
            // a token without weight in any head counts for nothing, whatever its value (or the memory behind the last token) holds
            uint32_t gone = __ballot_sync(0xffffffffu, dead);
            gone &= gone >> 16;
            gone &= gone >> 8;
            if (__any_sync(0xffffffffu, more)) {
                float keep[kMine];
#pragma unroll
                for (int i = 0; i < kMine; ++i) {
                    float top = fmaxf(m[i], z[i]);
#pragma unroll
                    for (int d = 1; d <= 4; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
                    keep[i] = m[i] == -INFINITY ? 1.f : ex2(m[i] - top);   // (nothing, or NaN, has been summed before)
                    m[i] = top;
                    l[i] *= keep[i];
                }
#pragma unroll
                for (int h = 0; h < HB; ++h) {
                    const float k = __shfl_sync(0xffffffffu, keep[h % kMine], h / kMine * 8);
#pragma unroll
                    for (int e = 0; e < NP / 64; ++e) o[h][e] = mul2(o[h][e], pack2(k, k));
                }
            }
#pragma unroll
            for (int i = 0; i < kMine; ++i) {
                const float w = ex2(z[i] - (m[i] == -INFINITY ? 0.f : m[i]));
                l[i] += w;
                sW[warp][t][part * kMine + i] = w;
            }
            __syncwarp();
            const unsigned char* in = mine + (2 + (step & 1)) * Way::kRows;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                if (gone >> k & 1) continue;
                f2 v[NP / 64];
                if (NP == 128) {
                    const ulonglong2 x = *reinterpret_cast<const ulonglong2*>(in + lane / 8 * Way::kBox + k * 128 + (((lane & 7) ^ k) << 4));
                    v[0] = x.x, v[NP / 64 - 1] = x.y;
                } else {
                    v[0] = *reinterpret_cast<const f2*>(in + lane / 16 * Way::kBox + k * 128 + (((lane / 2 & 7) ^ k) << 4) + (lane & 1) * 8);
                }
#pragma unroll
                for (int h = 0; h < HB; h += 4) {
                    const float4 w = *reinterpret_cast<const float4*>(&sW[warp][k][h]);
#pragma unroll
                    for (int e = 0; e < NP / 64; ++e) {
                        o[h][e] = fma2(pack2(w.x, w.x), v[e], o[h][e]);
                        o[h + 1][e] = fma2(pack2(w.y, w.y), v[e], o[h + 1][e]);
                        o[h + 2][e] = fma2(pack2(w.z, w.z), v[e], o[h + 2][e]);
                        o[h + 3][e] = fma2(pack2(w.w, w.w), v[e], o[h + 3][e]);
                    }
                }
            }
        }
        way.finish();
        float* sO = reinterpret_cast<float*>(mine);
#pragma unroll
        for (int i = 0; i < kMine; ++i) {
            if (way.lost) m[i] = 0.f, l[i] = __int_as_float(0x7fffffff);   // results that cannot pass as such
#pragma unroll
            for (int d = 1; d <= 4; d <<= 1) l[i] += __shfl_xor_sync(0xffffffffu, l[i], d);
            if (t == 0) sM[warp][part * kMine + i] = m[i], sL[warp][part * kMine + i] = l[i];
        }
#pragma unroll
        for (int h = 0; h < HB; ++h)
#pragma unroll
            for (int e = 0; e < NP / 64; ++e) *reinterpret_cast<f2*>(sO + h * NP + lane * (NP / 32) + e * 2) = o[h][e];
        __syncthreads();
        if (LONE) {
            write_from_cluster<float, NP, HB>(p, reinterpret_cast<float*>(staged), Way::kWarpBytes / 4, sM, sL, sTop, sSum, b, h0, heads);
            return;
        }
        write_unit<float, NP, HB>(p, reinterpret_cast<const float*>(staged), Way::kWarpBytes / 4, sM, sL, b, h0, heads, t0 == 0 && t1 == r.tiles, t0 == 0);
        if (TMA) v7u::proxy_fence();
        __syncthreads();
    }
}

// Joins what the `parts` blocks of a kernel above have left.  Block i looks at the border between runs i and i + 1: the blocks of all
// borders that a unit goes over have an equal share of its elements each.  Weights of the runs first, then a thread per element
// and several threads for the runs of one where there are few.  It is launched while the kernel above still runs, and waits for its end before it reads what that left.
constexpr int kJoinThreads = 256;
template <typename E>
__global__ void __launch_bounds__(kJoinThreads) join_kernel(const AttentionArgs p, int parts, int HB) {
    extern __shared__ float weights[];   // [head][run], then [head]: the sums
    __shared__ float sums[kJoinThreads];
    const int units = p.Hkv * p.blocks;
    const Start start = find_start<kJoinThreads>(p, blockIdx.x + 1, parts, units);
    const i64 border = start.tile, run = start.run;
    asm volatile("griddepcontrol.wait;" ::: "memory");   // (all blocks: this kernel must not end before the other)
    if (border >= start.all) return;
    const int b = start.b, tiles = Range(p, b).tiles;
    const int unit = (int)((border - start.base) / tiles);
    const i64 begin = start.base + (i64)unit * tiles;
    if (begin == border) return;   // nothing goes over it
    const int c0 = (int)(begin / run), count = (int)((begin + tiles - 1) / run) - c0 + 1, mine = blockIdx.x - c0;
    const int head = unit / p.blocks, h0 = head * p.group + unit % p.blocks * HB, heads = min(HB, (head + 1) * p.group - h0);
    const int elements = heads * p.N, e0 = (int)((i64)elements * mine / (count - 1)), e1 = (int)((i64)elements * (mine + 1) / (count - 1));
    if (e0 == e1) return;   // (more blocks than elements)
    const int first = e0 / p.N, last = (e1 - 1) / p.N;   // heads
    const int stride = p.N + 2;
    // what run c left of the unit: in the second place of the block where the unit begins, in the first of the others
    auto share = [&](int c, int h) { return p.work + (((i64)(c0 + c) * 2 + (c == 0)) * HB + h) * stride; };
    const int lane = threadIdx.x & 31;
    for (int h = first + (threadIdx.x >> 5); h <= last; h += kJoinThreads / 32) {
        float top = -INFINITY, sum = 0.f;
        for (int c = lane; c < count; c += 32) {
            const float m = share(c, h)[p.N];
            weights[h * count + c] = m;
            top = fmaxf(top, m);
        }
#pragma unroll
        for (int d = 16; d >= 1; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
        for (int c = lane; c < count; c += 32) {
            const float m = weights[h * count + c], w = m == -INFINITY ? 0.f : ex2(m - top);
            weights[h * count + c] = w;
            sum = fmaf(share(c, h)[p.N + 1], w, sum);
        }
#pragma unroll
        for (int d = 16; d >= 1; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
        if (lane == 0) {
            weights[HB * count + h] = sum;
            if (p.lse != nullptr && h * p.N >= e0) p.lse[(i64)b * p.Hq + h0 + h] = sum == 0.f ? -INFINITY : top * kLn2 + logf(sum);
        }
    }
    __syncthreads();
    const int width = min(e1 - e0, kJoinThreads), split = kJoinThreads / width, slice = threadIdx.x / width;
    for (int i0 = e0; i0 < e1; i0 += width) {   // (the same steps for all threads)
        const int i = i0 + threadIdx.x % width, h = i / p.N, n = i % p.N;
        float x = 0.f;
        if (i < e1 && slice < split) {
#pragma unroll 4
            for (int c = slice; c < count; c += split) {
                const float w = weights[h * count + c], v = share(c, h)[n];
                if (w != 0.f) x = fmaf(v, w, x);   // (a run without weight may hold NaN)
            }
        }
        if (split > 1) {
            sums[threadIdx.x] = x;
            __syncthreads();
            if (slice == 0)
                for (int q = 1; q < split; ++q) x += sums[q * width + threadIdx.x];
            __syncthreads();
        }
        if (slice == 0 && i < e1) {
            const float sum = weights[HB * count + h];
            static_cast<E*>(p.out)[((i64)b * p.Hq + h0 + h) * p.N + n] = from_f<E>(sum == 0.f ? 0.f : x / sum);
        }
    }
}

constexpr int kBlocksPerSm = 3, kLoneTokens = 512;
int run_blocks() { return max(1, sm_count()) * kBlocksPerSm; }
template <typename E>
int launch_join(const AttentionArgs& p, int parts, int HB, cudaStream_t st) {
    const int smem = HB * (parts + 1) * (int)sizeof(float);   // (at most 16 heads and three shares per SM: under 48 KB up to 250 SMs)
    cudaLaunchConfig_t config{};
    config.gridDim = dim3(parts - 1);
    config.blockDim = dim3(kJoinThreads);
    config.dynamicSmemBytes = smem;
    config.stream = st;
    cudaLaunchAttribute early;
    early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    early.val.programmaticStreamSerializationAllowed = 1;
    config.attrs = &early;
    config.numAttrs = 1;
    cudaLaunchKernelEx(&config, join_kernel<E>, p, parts, HB);
    return check_launch("paged_attention");
}
int bf16_heads_of(int group) { return group > 8 ? 16 : 8; }
int fp32_heads_of(int group) { return group > 4 ? 8 : 4; }

// A pool as rows of N elements, in boxes of a step's tokens and 128 bytes, one behind the other.
typedef CUresult (*EncodeTiled)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
bool make_row_map(CUtensorMap* map, const void* pool, i64 rows, int N, int element) {
    static const EncodeTiled encode = [] {
        void* fn = nullptr;
        cudaDriverEntryPointQueryResult found;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &found) != cudaSuccess || found != cudaDriverEntryPointSuccess) fn = nullptr;
        return reinterpret_cast<EncodeTiled>(fn);
    }();
    if (encode == nullptr || tensor_maps_disabled()) return false;
    const cuuint32_t size = element == 2 ? 2 : 4, columns = 128 / size, boxes = (cuuint32_t)N / columns;
    const cuuint64_t dims[3] = {columns, (cuuint64_t)rows, boxes}, strides[2] = {(cuuint64_t)N * size, 128};
    const cuuint32_t box[3] = {columns, 32 / size, boxes}, step[3] = {1, 1, 1};
    auto make = [&] {
        return encode(map, size == 2 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 3, const_cast<void*>(pool), dims, strides, box, step,
                      CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
    };
    return make() || (cudaFree(nullptr) == cudaSuccess && make());   // (a thread without a context yet)
}

template <typename E, int NP, int HEADS, int MODE, bool LONE>
constexpr auto steps_kernel() {
    if constexpr (sizeof(E) == 2) return attention_mma_kernel<NP, HEADS / 8, MODE, LONE>;
    else return attention_fp32_kernel<NP, HEADS, MODE, LONE>;
}
template <typename E, int NP, int HEADS, int MODE>
int launch_steps(AttentionArgs& p, const Maps& maps, cudaStream_t st) {
    using Way = Steps<E, NP, MODE>;
    constexpr bool TMA = MODE == kTma;
    constexpr int smem = kWarps * Way::kWarpBytes;
    static_assert(Way::kWarpBytes >= HEADS * NP * 4, "a warp's sums fit its slots");
    p.blocks = (p.group + HEADS - 1) / HEADS;
    p.tile_bits = sizeof(E) == 2 ? 6 : 5;
    // Units of which no block of a cluster gets more than kLoneTokens go to clusters of their own, of up to four blocks or, as long as
    // all clusters are there at once, eight: one launch instead of two, and no share of the work has to be found out (32 heads on 8 of
    // 128: 8 sequences of up to 1024 tokens 12.8 us instead of 16.7, 64 of up to 2048 70.7 and 77.1; 128 of up to 2048 127 and 120).
    // Longer ones are better shared equally (128 sequences of up to 4096 tokens: 261 and 198 us).
    const i64 units = (i64)p.B * p.Hkv * p.blocks, capacity = (i64)p.width * p.page.d, most = p.window > 0 && p.window < capacity ? p.window : capacity;
    int K = 1;
    while (K < kMaxCluster && (most > (i64)K * kLoneTokens || (units * K * 2 <= 2 * sm_count() && most > K * 64))) K *= 2;
    if (TMA && most <= (i64)K * kLoneTokens && (K <= 4 || units * K <= run_blocks()) && units * K <= 0x7fffffff) {
        constexpr auto kernel = steps_kernel<E, NP, HEADS, MODE, TMA>();
        if (allow_smem<kernel>(smem) != cudaSuccess) return check_launch("paged_attention");
        cudaLaunchConfig_t config{};
        config.gridDim = dim3((unsigned)(units * K));
        config.blockDim = dim3(kThreads);
        config.dynamicSmemBytes = smem;
        config.stream = st;
        cudaLaunchAttribute cluster;
        cluster.id = cudaLaunchAttributeClusterDimension;
        cluster.val.clusterDim.x = K;
        cluster.val.clusterDim.y = cluster.val.clusterDim.z = 1;
        config.attrs = &cluster;
        config.numAttrs = 1;
        cudaLaunchKernelEx(&config, kernel, p, maps);
        return check_launch("paged_attention");
    }
    constexpr auto kernel = steps_kernel<E, NP, HEADS, MODE, false>();
    if (allow_smem<kernel>(smem) != cudaSuccess) return check_launch("paged_attention");
    const int parts = run_blocks();
    kernel<<<parts, kThreads, smem, st>>>(p, maps);
    if (int e = check_launch("paged_attention")) return e;
    return launch_join<E>(p, parts, HEADS, st);
}
template <typename E, int NP, int HEADS>
int dispatch_mode(AttentionArgs& p, cudaStream_t st) {
    Maps maps;
    const i64 rows = (i64)p.pages * p.Hkv * p.page.d;
    const uintptr_t all = reinterpret_cast<uintptr_t>(p.k_pages) | reinterpret_cast<uintptr_t>(p.v_pages);
    if (p.N * sizeof(E) % 16 != 0 || all % 16 != 0) return launch_steps<E, NP, HEADS, kElements>(p, maps, st);
    if (p.page.d % 16 == 0 && p.N == NP && rows <= 0x7fffffff && make_row_map(&maps.keys, p.k_pages, rows, p.N, sizeof(E)) &&
        make_row_map(&maps.values, p.v_pages, rows, p.N, sizeof(E)))
        return launch_steps<E, NP, HEADS, kTma>(p, maps, st);
    return launch_steps<E, NP, HEADS, kPieces>(p, maps, st);
}
template <typename E, int FEW, int MANY>
int dispatch(AttentionArgs& p, bool many, cudaStream_t st) {
    if (p.N <= 64) return many ? dispatch_mode<E, 64, MANY>(p, st) : dispatch_mode<E, 64, FEW>(p, st);
    return many ? dispatch_mode<E, 128, MANY>(p, st) : dispatch_mode<E, 128, FEW>(p, st);
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
    const int heads = dtype == RWKVB200_BF16 ? bf16_heads_of(Hq / Hkv) : fp32_heads_of(Hq / Hkv);
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
    if (!(cap < INFINITY)) cap = 0.f;   // (no cap)
    AttentionArgs p{B, Hq, Hkv, N, pages, width, window, Hq / Hkv, 1, 0, scale, cap, Divisor((uint32_t)page), q, k_pages, v_pages, table, lengths, slopes, out, lse, static_cast<float*>(work)};
    return dtype == RWKVB200_BF16 ? dispatch<bf16, 8, 16>(p, bf16_heads_of(p.group) > 8, as_stream(stream)) : dispatch<float, 4, 8>(p, fp32_heads_of(p.group) > 4, as_stream(stream));
}
