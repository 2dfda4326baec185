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
    float scale, cap;
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
    // the sequence that `begin` lies in: its number, and the tiles before it
    {
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
            if (begin >= x - n && begin < x) sStart[0] = b, sStart[1] = x - n;
            if (base > begin) break;   // (the same for all threads)
        }
        __syncthreads();
    }
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
            const float m = part[p.N], keep = m == -INFINITY ? 0.f : expf(m - top);
            sum += part[p.N + 1] * keep;
            if (m != -INFINITY) x += part[n] * keep;
        }
        static_cast<E*>(p.out)[((i64)b * p.Hq + h0 + h) * p.N + n] = from_f<E>(sum == 0.f ? 0.f : x / sum);
        if (n == 0 && p.lse != nullptr) p.lse[(i64)b * p.Hq + h0 + h] = sum == 0.f ? -INFINITY : top + logf(sum);
    }
}

constexpr int kBlocksPerSm = 3;
int run_blocks() { return max(1, sm_count()) * kBlocksPerSm; }
int heads_of(int group) { return group >= 4 ? 4 : group >= 2 ? 2 : 1; }

template <typename E, int W, int HB>
int launch(AttentionArgs& p, cudaStream_t st) {
    p.blocks = (p.group + HB - 1) / HB;
    const int parts = run_blocks();
    attention_kernel<E, W, HB><<<parts, kThreads, 0, st>>>(p);
    if (int e = check_launch("paged_attention")) return e;
    join_kernel<E><<<(unsigned)((i64)p.B * p.Hkv * p.blocks), kThreads, 0, st>>>(p, parts, HB);
    return check_launch("paged_attention");
}
template <typename E>
int dispatch(AttentionArgs& p, cudaStream_t st) {
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
    return (size_t)run_blocks() * 2 * heads_of(Hq / Hkv) * (N + 2) * sizeof(float);
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
    AttentionArgs p{B, Hq, Hkv, N, pages, width, window, Hq / Hkv, 1, scale, cap, Divisor((uint32_t)page), q, k_pages, v_pages, table, lengths, slopes, out, lse, static_cast<float*>(work)};
    return dtype == RWKVB200_BF16 ? dispatch<bf16>(p, as_stream(stream)) : dispatch<float>(p, as_stream(stream));
}
