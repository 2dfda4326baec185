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
#include "wkv7_umma.cuh"
#include <cuda.h>

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
    int lo, hi, start, tiles;   // tokens of a sequence that count; its tiles, from a multiple of 16 on: one at least, so that empty
                                // sequences get their zeros, and none for a row that only pads the batch
    __device__ __forceinline__ Range(const AttentionArgs& p, int b) {
        hi = min(p.lengths[b], p.width * (int)p.page.d);
        lo = p.window > 0 ? max(0, hi - p.window) : 0;
        start = lo & ~15;
        tiles = hi < 0 ? 0 : max(1, (hi - start + kTile - 1) / kTile);
    }
};

__device__ __forceinline__ i64 run_length(i64 all, i64 blocks) { return max((i64)kMinTiles, (all + blocks - 1) / blocks); }

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
        s.run = run_length(s.all, runs);
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
            s.run = run_length(s.all, runs);
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
    __shared__ float sO[kWarps][HB][RWKVB200_MAX_HEAD_SIZE], sM[kWarps][HB], sL[kWarps][HB];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, l8 = lane & 7, token = warp * 4 + (lane >> 3);
    const unsigned mask = 0xffu << (lane & 24);   // the lanes that share a token
    const int units = p.Hkv * p.blocks;
    const Start start = find_start<kThreads>(p, blockIdx.x, gridDim.x, units);
    const i64 end = min(start.tile + start.run, start.all);
    if (start.tile >= end) return;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    int b = start.b;
    i64 base = start.base;
    for (i64 at = start.tile; at < end;) {
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
        const int last = min(r.start + t1 * kTile, r.hi);
        for (int j = r.start + t0 * kTile + token; j < last; j += kWarps * 4) {
            if (j < r.lo) continue;
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
// 16 of a tile's tokens and keeps its own maxima and sums.  Both operands come out of shared memory by ldmatrix (the values transposed), from
// tiles of [16 tokens][64 elements] in the 128-byte swizzle.  They get there
//   TMA:  by one bulk copy of 16 rows each for keys and values (pages of a multiple of 16 tokens, heads of 64 or 128): a warp's
//         lane 0 asks, keys two steps ahead and values one, and counts the bytes on a barrier of the slot;
//   else: by cp.async in pieces of 16 bytes, rows that do not count filled with zeros.  (Taken for every page size, with a lane's
//         pieces in places of its own, this read 4.0 TB/s at 128 sequences of up to 4096 tokens; without any product 4.1.)
// Weights are taken into the second product as the sum of two bf16 numbers (2^-16 relative; one would double the output's
// rounding), both above 0, so that an infinite value stays one.
constexpr int kTimeout = 3;       // a wait for a copy ran out
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
__device__ __forceinline__ void commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
__device__ __forceinline__ void copy_or_zero(uint32_t shared, const bf16* from, bool there) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(shared), "l"(from), "r"(there ? 16 : 0) : "memory");
}

__device__ __forceinline__ void ldmatrix(uint32_t (&d)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void ldmatrix_transposed(uint32_t (&d)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3]) : "r"(at) : "memory");
}
// 16 rows of a pool, from number `row` on, counted on `bar`
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

template <int NP, int HT, bool TMA>
__global__ void __launch_bounds__(kThreads, 3) attention_mma_kernel(const AttentionArgs p, const __grid_constant__ Maps maps) {
    constexpr int kHalves = NP / 64, kRows = 2048 * kHalves;   // bytes of 16 rows
    constexpr int kHeads = 8 * HT, kWarpBytes = 4 * kRows;     // a warp's slots: keys of two steps, values of two
    extern __shared__ __align__(1024) unsigned char staged[];
    __shared__ float sM[kWarps][kHeads], sL[kWarps][kHeads];
    __shared__ uint64_t bars[kWarps][4];                       // TMA: one per slot
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, q = lane & 3;
    const int units = p.Hkv * p.blocks, N = TMA ? NP : p.N;
    if (TMA && lane < 4) asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"((uint32_t)__cvta_generic_to_shared(&bars[warp][lane])));
    if (TMA) v7u::proxy_fence();
    const Start start = find_start<kThreads>(p, blockIdx.x, gridDim.x, units);
    const i64 end = min(start.tile + start.run, start.all);
    if (start.tile >= end) return;
    unsigned char* mine = staged + warp * kWarpBytes;
    const uint32_t base_keys = (uint32_t)__cvta_generic_to_shared(mine), base_values = base_keys + 2 * kRows;
    float* sO = reinterpret_cast<float*>(mine);                // [head][NP], between the tokens of two units
    // where a lane's rows for ldmatrix lie: keys: rows lane & 15, piece lane / 16; values: rows by 8 from lane / 16, piece by lane / 8
    const uint32_t key_row = (lane & 15) * 128, key_piece = lane >> 4, value_row = ((lane & 7) + (lane >> 4) * 8) * 128, value_piece = lane >> 3 & 1, swizzle = lane & 7;
    const float scale = p.cap > 0.f ? p.scale / p.cap : p.scale * kLog2e, cap = p.cap * kLog2e;
    uint32_t phases = 0;     // of the four barriers
    bool lost = false;       // a wait ran out: nothing more is asked for, and the results are NaN
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    int b = start.b;
    i64 base = start.base;
    for (i64 at = start.tile; at < end;) {
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
        const int from = r.start + t0 * kTile + warp * 16, last = min(r.start + t1 * kTile, r.hi), steps = lost ? 0 : t1 - t0;
        // Of a step's tokens the lane answers for number lane & 15 (TMA: all for the first: they share a page).  Its page is asked for a
        // step before it is looked at.
        auto counts = [&](int j) { return j >= r.lo && j < last; };
        auto token_of = [&](int step) { return from + step * kTile + (TMA ? 0 : lane & 15); };
        auto in_use = [&](int step, int j) { return step < steps && (TMA ? j < last : counts(j)); };
        auto page_of = [&](int step) {
            const int j = token_of(step);
            return in_use(step, j) ? row[p.page.quotient((uint32_t)j)] : 0;
        };
        // the row of the pools that the token lies in; -1: it does not count
        auto row_of = [&](int step, int id) {
            const int j = token_of(step);
            if (!in_use(step, j)) return -1;
            if ((unsigned)id >= (unsigned)p.pages) {
                atomicMax(&g_error, kBadPage);
                return -1;
            }
            return (id * p.Hkv + head) * (int)p.page.d + (j - (int)(p.page.quotient((uint32_t)j) * p.page.d));
        };
        auto ask = [&](bool values, int step, int n) {
            const int slot = step & 1;
            const uint32_t to = (values ? base_values : base_keys) + slot * kRows;
            if (TMA) {
                if (lane == 0 && n >= 0) copy_rows(to, values ? &maps.values : &maps.keys, n, &bars[warp][values * 2 + slot], kRows);
            } else {
                const bf16* pool = static_cast<const bf16*>(values ? p.v_pages : p.k_pages);
#pragma unroll
                for (int i = 0; i < kRows / 512; ++i) {
                    const int piece = i * 32 + lane, token = piece / (8 * kHalves), c = piece % (8 * kHalves);
                    const int k = __shfl_sync(0xffffffffu, n, token);
                    copy_or_zero(to + (c >> 3) * 2048 + token * 128 + (((c ^ token) & 7) << 4), pool + (i64)max(k, 0) * N + min(c * 8, N - 8), k >= 0 && c * 8 < N);
                }
            }
        };
        auto arrived = [&](bool values, int step, int n) {   // TMA: waits for what has been asked for
            const int which = values * 2 + (step & 1);
            if (!TMA || n < 0) return;
            if (__any_sync(0xffffffffu, !v7u::mbar_wait(&bars[warp][which], phases >> which & 1))) lost = true;
            phases ^= 1u << which;
        };
        const int id0 = page_of(0), id1 = page_of(1);
        int id2 = page_of(2);
        int n0 = row_of(0, id0), n1 = row_of(1, id1);
        ask(false, 0, n0);
        commit();
        ask(false, 1, n1);
        ask(true, 0, n0);
        commit();
        // q as the second operand of the scores: head g (and g + 8)
        uint32_t qf[HT][NP / 16][2];
#pragma unroll
        for (int h = 0; h < HT; ++h)
#pragma unroll
            for (int j = 0; j < NP / 8; ++j) {
                const bf16* from = static_cast<const bf16*>(p.q) + ((i64)b * p.Hq + h0 + h * 8 + g) * N + j * 8 + q * 2;
                __nv_bfloat162 v = __floats2bfloat162_rn(0.f, 0.f);
                if (h * 8 + g < heads && j * 8 < N) v.x = from[0], v.y = from[1];
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
            const uint32_t in = base_keys + (step & 1) * kRows + key_row;
#pragma unroll
            for (int h = 0; h < HT; ++h)
#pragma unroll
                for (int e = 0; e < 4; ++e) next[h][e] = 0.f;
#pragma unroll
            for (int j = 0; j < NP / 16; ++j) {
                uint32_t a[4];
                ldmatrix(a, in + j / 4 * 2048 + (((j % 4 * 2 + key_piece) ^ swizzle) << 4));
#pragma unroll
                for (int h = 0; h < HT; ++h) mma(next[h], a[0], a[1], a[2], a[3], qf[h][j][0], qf[h][j][1]);
            }
        };
        if (!TMA) asm volatile("cp.async.wait_group 1;" ::: "memory");
        arrived(false, 0, n0);
        __syncwarp();
        scores(0);
        for (int step = 0; step < steps && !lost; ++step) {
            float z[HT][4];
#pragma unroll
            for (int h = 0; h < HT; ++h)
#pragma unroll
                for (int e = 0; e < 4; ++e) z[h][e] = next[h][e];
            const int n2 = row_of(step + 2, id2);
            id2 = page_of(step + 3);
            __syncwarp();                 // (all lanes have read the slots that are asked for)
            ask(false, step + 2, n2);
            ask(true, step + 1, n1);
            commit();
            if (!TMA) asm volatile("cp.async.wait_group 1;" ::: "memory");
            arrived(false, step + 1, n1);
            arrived(true, step, n0);
            __syncwarp();
            scores(step + 1);
            const int n = n0;
            n0 = n1;
            n1 = n2;
            if (!__any_sync(0xffffffffu, n >= 0)) continue;   // no token counts
            // scores as exponents of 2: tokens g (elements 0, 1) and g + 8 (2, 3)
            const int j = from + step * kTile + g;
            const bool there[2] = {TMA ? counts(j) : __shfl_sync(0xffffffffu, n, g) >= 0, TMA ? counts(j + 8) : __shfl_sync(0xffffffffu, n, g + 8) >= 0};
            const float distance = (float)(j - (r.hi - 1));
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
            const uint32_t in = base_values + (step & 1) * kRows;
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
                        if (lane < 8 * kHalves) {
                            unsigned char* to = mine + 2 * kRows + (step & 1) * kRows + lane / 8 * 2048 + token * 128 + lane % 8 * 16;
                            *reinterpret_cast<uint4*>(to) = make_uint4(0, 0, 0, 0);
                        }
                    }
                }
                if (TMA) v7u::proxy_fence();
                __syncwarp();
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
#pragma unroll
            for (int i = 0; i < NP / 16; ++i) {
                uint32_t a[4];
                ldmatrix_transposed(a, in + value_row + i / 4 * 2048 + (((i % 4 * 2 + value_piece) ^ swizzle) << 4));
#pragma unroll
                for (int h = 0; h < HT; ++h) {
                    mma(o[h][i], a[0], a[1], a[2], a[3], high[h][0], high[h][1]);
                    mma(o[h][i], a[0], a[1], a[2], a[3], low[h][0], low[h][1]);
                }
            }
        }
        if (!TMA) asm volatile("cp.async.wait_group 0;" ::: "memory");
        if (lost) {   // what may still be in flight, and results that cannot pass as such
            for (int i = 0; i < 4; ++i) v7u::mbar_wait(&bars[warp][i], phases >> i & 1, 1 << 10);
            if (lane == 0) atomicMax(&g_error, kTimeout);
#pragma unroll
            for (int h = 0; h < HT; ++h) m[h][0] = m[h][1] = 0.f, l[h][0] = l[h][1] = __int_as_float(0x7fffffff);
        }
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
                for (int e = 0; e < 4; ++e) sO[(h * 8 + 2 * q + (e & 1)) * NP + i * 16 + g + (e >> 1) * 8] = o[h][i][e];
        }
        __syncthreads();
        const bool whole = t0 == 0 && t1 == r.tiles;
        float* part = p.work + ((i64)blockIdx.x * 2 + (t0 == 0)) * kHeads * (N + 2);
        for (int i = threadIdx.x; i < heads * NP; i += kThreads) {
            const int h = i / NP, n = i % NP;
            if (n >= N) continue;
            float top = -INFINITY, x = 0.f, sum = 0.f;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) top = fmaxf(top, sM[w][h]);
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                const float keep = sM[w][h] == -INFINITY ? 0.f : ex2(sM[w][h] - top);
                sum += sL[w][h] * keep;
                // (a warp whose maximum is -infinity has sums of zeros, or NaN from a NaN score)
                if (sM[w][h] != -INFINITY) x += reinterpret_cast<const float*>(staged + w * kWarpBytes)[h * NP + n] * keep;
            }
            if (whole) {
                static_cast<bf16*>(p.out)[((i64)b * p.Hq + h0 + h) * N + n] = __float2bfloat16_rn(sum == 0.f ? 0.f : x / sum);
                if (n == 0 && p.lse != nullptr) p.lse[(i64)b * p.Hq + h0 + h] = sum == 0.f ? -INFINITY : top * kLn2 + logf(sum);
            } else {
                part[h * (N + 2) + n] = x;
                if (n == 0) part[h * (N + 2) + N] = top, part[h * (N + 2) + N + 1] = sum;
            }
        }
        if (TMA) v7u::proxy_fence();
        __syncthreads();
    }
}

// Joins what the `parts` blocks of a kernel above have left.  Block i looks at the border between runs i and i + 1: the blocks of all
// borders that a unit goes over have an equal share of its elements each.  Weights of the runs first, then a thread per element
// and every kSplit-th run.  It is launched while the kernel above still runs, and waits for its end before it reads what that left.
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
            const float m = weights[h * count + c], w = m == -INFINITY ? 0.f : exp2f((m - top) * p.to_log2);
            weights[h * count + c] = w;
            sum = fmaf(share(c, h)[p.N + 1], w, sum);
        }
#pragma unroll
        for (int d = 16; d >= 1; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
        if (lane == 0) {
            weights[HB * count + h] = sum;
            if (p.lse != nullptr && h * p.N >= e0) p.lse[(i64)b * p.Hq + h0 + h] = sum == 0.f ? -INFINITY : (top * p.to_log2 + log2f(sum)) * kLn2;
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

constexpr int kBlocksPerSm = 3;
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
int heads_of(int group) { return group >= 4 ? 4 : group >= 2 ? 2 : 1; }
int mma_heads_of(int group) { return group > 8 ? 16 : 8; }

template <typename E, int W, int HB>
int launch(AttentionArgs& p, cudaStream_t st) {
    p.blocks = (p.group + HB - 1) / HB;
    const int parts = run_blocks();
    attention_kernel<E, W, HB><<<parts, kThreads, 0, st>>>(p);
    if (int e = check_launch("paged_attention")) return e;
    return launch_join<E>(p, parts, HB, st);
}
// A pool as rows of 64 or 128 elements, in boxes of [16 rows][64 elements], one behind the other for rows of 128.
typedef CUresult (*EncodeTiled)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
bool make_row_map(CUtensorMap* map, const void* pool, i64 rows, int N) {
    static const EncodeTiled encode = [] {
        void* fn = nullptr;
        cudaDriverEntryPointQueryResult found;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &found) != cudaSuccess || found != cudaDriverEntryPointSuccess) fn = nullptr;
        return reinterpret_cast<EncodeTiled>(fn);
    }();
    if (encode == nullptr || tensor_maps_disabled()) return false;
    const cuuint64_t dims[3] = {64, (cuuint64_t)rows, (cuuint64_t)N / 64}, strides[2] = {(cuuint64_t)N * 2, 128};
    const cuuint32_t box[3] = {64, 16, (cuuint32_t)N / 64}, step[3] = {1, 1, 1};
    auto make = [&] {
        return encode(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(pool), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                      CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
    };
    return make() || (cudaFree(nullptr) == cudaSuccess && make());   // (a thread without a context yet)
}

template <int NP, int HT, bool TMA>
int launch_mma(AttentionArgs& p, const Maps& maps, cudaStream_t st) {
    constexpr int smem = kWarps * 4 * 2048 * (NP / 64);
    static_assert(4 * 2048 * (NP / 64) >= 8 * HT * NP * 4, "a warp's sums fit its slots");
    if (allow_smem<attention_mma_kernel<NP, HT, TMA>>(smem) != cudaSuccess) return check_launch("paged_attention");
    p.blocks = (p.group + 8 * HT - 1) / (8 * HT);
    p.to_log2 = 1.f;
    const int parts = run_blocks();
    attention_mma_kernel<NP, HT, TMA><<<parts, kThreads, smem, st>>>(p, maps);
    if (int e = check_launch("paged_attention")) return e;
    return launch_join<bf16>(p, parts, 8 * HT, st);
}
// Heads of whole 16-byte pieces that start on such boundaries, and rows of the pools that an int can number.
bool takes_mma(const AttentionArgs& p) {
    const uintptr_t all = reinterpret_cast<uintptr_t>(p.k_pages) | reinterpret_cast<uintptr_t>(p.v_pages);
    return p.N % 8 == 0 && all % 16 == 0 && (i64)p.pages * p.Hkv * p.page.d <= 0x7fffffff;
}
template <typename E>
int dispatch(AttentionArgs& p, cudaStream_t st) {
    if (sizeof(E) == 2 && takes_mma(p)) {
        Maps maps;
        const i64 rows = (i64)p.pages * p.Hkv * p.page.d;
        const bool tma = p.page.d % 16 == 0 && (p.N == 64 || p.N == 128) && make_row_map(&maps.keys, p.k_pages, rows, p.N) &&
                         make_row_map(&maps.values, p.v_pages, rows, p.N);
        switch ((p.N > 64) * 4 + (p.group > 8) * 2 + tma) {
            case 0: return launch_mma<64, 1, false>(p, maps, st);
            case 1: return launch_mma<64, 1, true>(p, maps, st);
            case 2: return launch_mma<64, 2, false>(p, maps, st);
            case 3: return launch_mma<64, 2, true>(p, maps, st);
            case 4: return launch_mma<128, 1, false>(p, maps, st);
            case 5: return launch_mma<128, 1, true>(p, maps, st);
            case 6: return launch_mma<128, 2, false>(p, maps, st);
            default: return launch_mma<128, 2, true>(p, maps, st);
        }
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
