// Gated linear recurrence, per channel c:
//
//   L_t = s_c sigmoid(ga_t)      a_t = exp(-L_t)      beta_t = sqrt(1 - a_t^2)      u_t = sigmoid(gx_t) x_t
//   h_t = a_t h_{t-1} + beta_t u_t                    y_t = h_t
//
// At the first token of a document a_t = 0 and beta_t = 1.  Gradients, with e_t = a_{t+1} G_{t+1} and e_{T-1} = dhT:
//
//   G_t = dy_t + e_t       dx = G beta sigmoid(gx)      dgx = G beta u (1 - sigmoid(gx))
//   dL = G a (u a / beta - h_{t-1})                     dga = dL L (1 - sigmoid(ga))     ds = sum dL sigmoid(ga)     dh0 = e_{-1}
//
// (dL = 0 at a document's first token; where L = 0 the term through beta is taken as 0.)
//
// A block owns 32 lanes x 2 channels of one sequence and goes through it in rounds of kWarps x kTokens tokens, a warp owns
// kTokens of them: it makes the gates of its tokens in registers, reduces them to (P, H) (the product of the decays and the end
// state from a zero start), all warps fold those of the warps before theirs onto the block's state, and each walks its tokens
// once more from its own start state.  Every input is read once, y is written once.  Where there are few (sequence, channel)
// blocks, a cluster of blocks shares the rounds: block k of K takes rounds k, k + K, ..., and the (P, H) of their rounds go
// through distributed shared memory, one cluster barrier for K rounds.
//
// Every warp copies its own tokens to shared memory (cp.async), one or two rounds ahead: that keeps enough bytes in flight and
// needs no barrier.  What bounds the kernels is in front of each.
#include "packed.cuh"
#include <cooperative_groups.h>
#include <type_traits>

namespace rwkvb200 {
namespace {

namespace cg = cooperative_groups;

constexpr int kWarps = 8;
constexpr int kTokens = 8;                   // per warp and round
constexpr int kRound = kWarps * kTokens;     // the forward saves the state before every round for the backward
constexpr int kTile = 64;                    // channels of a block
constexpr int kMaxCluster = 8;

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
__device__ __forceinline__ float rsqrt_fast(float x) {
    float y;
    asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// The functions behind the gates: for bf16 tensors the hardware approximations (2e-7 relative: 2^-14 of a step of bf16), for fp32
// CUDA's exponential and one step of Newton's method behind the others.
template <typename E> struct Fn;
template <> struct Fn<bf16> {
    static __device__ __forceinline__ float exp_minus(float x) { return ex2(-1.4426950408889634f * x); }
    static __device__ __forceinline__ float inverse(float x) { return rcp(x); }
    static __device__ __forceinline__ float inverse_root(float v) { return rsqrt_fast(v); }
};
template <> struct Fn<float> {
    static __device__ __forceinline__ float exp_minus(float x) { return expf(-x); }
    static __device__ __forceinline__ float inverse(float x) {   // (of 1 to 4)
        const float r = rcp(x);
        return fmaf(r, fmaf(-x, r, 1.f), r);
    }
    static __device__ __forceinline__ float inverse_root(float v) {
        const float r = rsqrt_fast(v);
        return fmaf(0.5f * r, fmaf(-v * r, r, 1.f), r);
    }
};

__device__ __forceinline__ f2 both(float x) { return pack2(x, x); }
__device__ __forceinline__ float lo(f2 v) {
    float a, b;
    unpack2(v, a, b);
    return a;
}
__device__ __forceinline__ float hi(f2 v) {
    float a, b;
    unpack2(v, a, b);
    return b;
}
template <typename F> __device__ __forceinline__ f2 each(f2 a, F f) { return pack2(f(lo(a)), f(hi(a))); }
template <typename F> __device__ __forceinline__ f2 each(f2 a, f2 b, F f) { return pack2(f(lo(a), lo(b)), f(hi(a), hi(b))); }

// 1 - exp(-L) of two channels, with all its digits where L is small: by its series for L / 8 (five terms leave (1/8)^5/720 = 4e-8),
// doubled three times, 1 - a^2 = (1 - a) (2 - (1 - a)).  That serves L < 1 and takes no special function; beyond it the exponential.
template <typename E>
__device__ __forceinline__ f2 fall(f2 L, bool small) {
    const f2 r = mul2(L, both(0.125f)), two = both(2.f), minus = both(-1.f);
    f2 q = fma2(r, both(1.f / 120.f), both(-1.f / 24.f));
    q = fma2(q, r, both(1.f / 6.f));
    q = fma2(q, r, both(-0.5f));
    q = fma2(q, r, both(1.f));
    q = mul2(q, r);
#pragma unroll
    for (int i = 0; i < 3; ++i) q = mul2(q, fma2(q, minus, two));
    if (small) return q;   // (s <= 1 in all channels of the warp)
    return each(L, q, [](float l, float p) { return l < 1.f ? p : 1.f - Fn<E>::exp_minus(l); });
}
__device__ __forceinline__ f2 square(f2 q) { return mul2(q, fma2(q, both(-1.f), both(2.f))); }
__device__ __forceinline__ f2 decay(f2 q) { return fma2(q, both(-1.f), both(1.f)); }
// 1 / sqrt(1 - a^2); 0 below the normal numbers, where beta counts as 0 (and NaN below 0, which only a negative s makes)
template <typename E>
__device__ __forceinline__ f2 inverse_root(f2 v) {
    return each(v, [](float x) { return fabsf(x) < 1.2e-38f ? 0.f : Fn<E>::inverse_root(x); });
}

// sigmoid(x) and 1 - sigmoid(x) without loss of either: m is the smaller of the two, with the sign of x in front of it
__device__ __forceinline__ float of_pair(float m) { return __float_as_int(m) < 0 ? 1.f + m : m; }
__device__ __forceinline__ float rest_of_pair(float m) { return __float_as_int(m) < 0 ? -m : 1.f - m; }
// Both gates of two channels from one division: exp(-|x|) <= 1, so that no product overflows.
template <typename E>
__device__ __forceinline__ void gates(f2 ga, f2 gx, f2& ea, f2& ex, f2& ra, f2& rx) {
    const f2 one = both(1.f);
    ea = each(ga, [](float v) { return Fn<E>::exp_minus(fabsf(v)); });
    ex = each(gx, [](float v) { return Fn<E>::exp_minus(fabsf(v)); });
    const f2 da = add2(ea, one), dx = add2(ex, one);
    const f2 r = each(mul2(da, dx), [](float v) { return Fn<E>::inverse(v); });
    ra = mul2(r, dx);   // 1 / (1 + exp(-|ga|))
    rx = mul2(r, da);
}
__device__ __forceinline__ f2 sigmoid(f2 x, f2 e, f2 r) {
    const f2 m = mul2(e, r);
    return pack2(lo(x) > 0.f ? lo(r) : lo(m), hi(x) > 0.f ? hi(r) : hi(m));
}
__device__ __forceinline__ f2 sigmoid_pair(f2 x, f2 e, f2 r) {
    const f2 m = mul2(e, r);
    return pack2(lo(x) > 0.f ? -lo(m) : lo(m), hi(x) > 0.f ? -hi(m) : hi(m));
}

// two neighbouring channels in shared memory, and back
__device__ __forceinline__ f2 get2(const bf16* p) {
    const uint32_t w = *reinterpret_cast<const uint32_t*>(p);
    return pack2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
__device__ __forceinline__ f2 get2(const float* p) {
    const float2 w = *reinterpret_cast<const float2*>(p);
    return pack2(w.x, w.y);
}
// ... to global memory: as one word, or one after the other where C is odd or a tensor starts between two words
template <bool PAIRS>
__device__ __forceinline__ void put2(bf16* p, f2 v, bool second) {
    const __nv_bfloat162 t = __floats2bfloat162_rn(lo(v), hi(v));
    if (PAIRS) {
        *reinterpret_cast<__nv_bfloat162*>(p) = t;
    } else {
        p[0] = t.x;
        if (second) p[1] = t.y;
    }
}
template <bool PAIRS>
__device__ __forceinline__ void put2(float* p, f2 v, bool second) {
    if (PAIRS) {
        *reinterpret_cast<float2*>(p) = make_float2(lo(v), hi(v));
    } else {
        p[0] = lo(v);
        if (second) p[1] = hi(v);
    }
}

struct Args {
    int T, C, tiles, rounds;   // channel tiles, rounds of kRound tokens
    const float* h0;
    const void *x, *gx, *ga;
    const float* s;
    const uint8_t* first;
    void* y;
    float* hT;
    float* saved;
    // backward
    const void* dy;
    const float* dhT;
    float* dh0;
    void *dx, *dgx, *dga;
    float* ds;
};

// which of a warp's tokens from t on begin a document, a bit each
__device__ __forceinline__ uint32_t firsts(const uint8_t* first, int t, int T, int lane) {
    if (first == nullptr) return 0;
    const bool f = lane < kTokens && t + lane < T && first[t + lane] != 0;
    return __ballot_sync(0xffffffffu, f);
}

// The [kTokens][kTile] tile of a tensor from token t on: to shared memory, without waiting.  WIDE: every row of C starts on a 16-byte
// boundary, and a piece of 16 bytes is asked for at a time; else element by element, at once.  What lies outside is left alone.
template <typename E, bool WIDE>
__device__ __forceinline__ void fetch(E* tile, const E* from, int t, int T, int C, int c_tile, int lane) {
    if (WIDE) {
        constexpr int n = 16 / sizeof(E), row = kTile / n;   // pieces of a row
#pragma unroll
        for (int i = 0; i < kTokens * row / 32; ++i) {
            const int piece = i * 32 + lane, j = piece / row, c = piece % row * n;
            if (t + j < T && c_tile + c < C) {
                const uint32_t to = (uint32_t)__cvta_generic_to_shared(tile + j * kTile + c);
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from + (i64)(t + j) * C + c) : "memory");
            }
        }
    } else {
#pragma unroll
        for (int j = 0; j < kTokens; ++j) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int c = i * 32 + lane;
                if (t + j < T && c_tile + c < C) tile[j * kTile + c] = from[(i64)(t + j) * C + c];
            }
        }
    }
}
__device__ __forceinline__ void commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void wait_group() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// Shares of a round reduced to one step each: h -> P h + H, or H alone where a document begins in it (P = 0; whatever h is: one document's
// infinities and NaN do not reach the next).  A product of decays that underflows is kept above 0: it must not make an infinite
// state NaN, and 0 means a document.
constexpr float kTiny = 1e-45f;
__device__ __forceinline__ f2 clamp(f2 P) {
    return each(P, [](float v) { return v < kTiny ? kTiny : v; });   // (a NaN stays one)
}
__device__ __forceinline__ f2 step(f2 P, f2 H, f2 h) {
    const f2 n = fma2(P, h, H);
    return pack2(lo(P) == 0.f ? lo(H) : lo(n), hi(P) == 0.f ? hi(H) : hi(n));
}
__device__ __forceinline__ f2 behind(f2 P, f2 before) {   // the product of two shares: 0 if one of them is a document's
    const f2 n = clamp(mul2(P, before));
    return pack2(lo(P) == 0.f || lo(before) == 0.f ? 0.f : lo(n), hi(P) == 0.f || hi(before) == 0.f ? 0.f : hi(n));
}
struct Share {
    f2 P, H;
};
// All shares of the block in the order of time (backward: `reversed`): those before warp `warp` in `mine`, all of them in `all`.
template <bool REVERSED>
__device__ __forceinline__ void fold(const ulonglong2 (*shares)[32], int warp, int lane, bool cuts, Share& mine, Share& all) {
    Share a{both(1.f), both(0.f)};
    if (!cuts) {
#pragma unroll
        for (int i = 0; i < kWarps; ++i) {
            const int q = REVERSED ? kWarps - 1 - i : i;
            if (q == warp) mine = a;
            const ulonglong2 v = shares[q][lane];
            a.H = fma2(v.x, a.H, v.y);
            a.P = mul2(a.P, v.x);
        }
        mine.P = clamp(mine.P);
        a.P = clamp(a.P);
    } else {
#pragma unroll
        for (int i = 0; i < kWarps; ++i) {
            const int q = REVERSED ? kWarps - 1 - i : i;
            if (q == warp) mine = a;
            const ulonglong2 v = shares[q][lane];
            a.H = step(v.x, v.y, a.H);
            a.P = behind(v.x, a.P);
        }
    }
    all = a;
}
// The state before this block's round and the one behind the rounds of all blocks of the cluster, from the state before them.
template <bool REVERSED>
__device__ __forceinline__ f2 through_cluster(cg::cluster_group& cluster, int K, int rank, ulonglong2 (*peers)[32], const Share& all, int warp, int lane, f2& carry) {
    if (K == 1) {
        const f2 start = carry;
        carry = step(all.P, all.H, carry);
        return start;
    }
    if (warp < K) *cluster.map_shared_rank(&peers[rank][lane], warp) = make_ulonglong2(all.P, all.H);
    cluster.sync();
    f2 start = carry;
    for (int i = 0; i < K; ++i) {
        const int q = REVERSED ? K - 1 - i : i;
        if (q == rank) start = carry;
        const ulonglong2 v = peers[q][lane];
        carry = step(v.x, v.y, carry);
    }
    return start;
}

template <typename E> constexpr int kFwdStages = sizeof(E) == 2 ? 3 : 2;
constexpr int kBwdStages = 2;
template <typename E> constexpr int fwd_smem() { return kFwdStages<E> * kWarps * 3 * kTokens * kTile * (int)sizeof(E); }
template <typename E> constexpr int bwd_smem() { return kBwdStages * kWarps * 4 * kTokens * kTile * (int)sizeof(E); }

template <typename E, bool WIDE, bool PAIRS>
__global__ void __launch_bounds__(32 * kWarps, 2) scan_forward_kernel(const Args p) {
    extern __shared__ __align__(16) unsigned char raw[];
    __shared__ ulonglong2 shares[2][kWarps][32], peers[2][kMaxCluster][32];
    constexpr int S = kFwdStages<E>, kPart = kTokens * kTile;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    cg::cluster_group cluster = cg::this_cluster();
    const int K = (int)cluster.num_blocks(), rank = (int)cluster.block_rank(), unit = blockIdx.x / K;
    const int b = unit / p.tiles, c_tile = unit % p.tiles * kTile, c0 = c_tile + lane * 2;
    const bool live = c0 < p.C, second = c0 + 1 < p.C;
    const i64 base = (i64)b * p.T * p.C + c_tile;
    const E *x = static_cast<const E*>(p.x) + base, *gx = static_cast<const E*>(p.gx) + base, *ga = static_cast<const E*>(p.ga) + base;
    E* y = static_cast<E*>(p.y) + base + lane * 2;
    E* mine = reinterpret_cast<E*>(raw) + warp * 3 * kPart;
    const uint8_t* first = p.first ? p.first + (i64)b * p.T : nullptr;
    const f2 s = pack2(live ? p.s[c0] : 0.f, second ? p.s[c0 + 1] : 0.f);
    const i64 row = (i64)b * p.C + c0;
    f2 carry = pack2(live && p.h0 ? p.h0[row] : 0.f, second && p.h0 ? p.h0[row + 1] : 0.f);
    const bool small = __all_sync(0xffffffffu, lo(s) <= 1.f && hi(s) <= 1.f);

    auto ask = [&](int round, int stage) {
        const int t = round * kRound + warp * kTokens;
        E* to = mine + stage * kWarps * 3 * kPart;
        if (t < p.T) {
            fetch<E, WIDE>(to, x, t, p.T, p.C, c_tile, lane);
            fetch<E, WIDE>(to + kPart, gx, t, p.T, p.C, c_tile, lane);
            fetch<E, WIDE>(to + 2 * kPart, ga, t, p.T, p.C, c_tile, lane);
        }
        commit();
    };
#pragma unroll
    for (int i = 0; i < S - 1; ++i) ask(rank + i * K, i);
    if (K > 1) cluster.sync();   // (a block's shared memory is written by others once it has begun)
    int stage = 0, buf = 0;
    for (int r0 = 0; r0 < p.rounds; r0 += K, buf ^= 1) {   // (all blocks of a cluster go through the same barriers)
        const int round = r0 + rank, t = round * kRound + warp * kTokens;
        ask(round + (S - 1) * K, stage == 0 ? S - 1 : stage - 1);
        wait_group<S - 1>();
        __syncwarp();
        const E* in = mine + stage * kWarps * 3 * kPart + lane * 2;
        const uint32_t docs = firsts(first, t, p.T, lane);
        f2 a[kTokens], w[kTokens];
        Share mine_share{both(1.f), both(0.f)};
        auto make = [&](auto plain) {   // plain: all tokens are there, and none begins a document
            constexpr bool kPlain = decltype(plain)::value;
#pragma unroll
            for (int j = 0; j < kTokens; ++j) {
                const f2 vx = get2(in + j * kTile), vgx = get2(in + kPart + j * kTile), vga = get2(in + 2 * kPart + j * kTile);
                f2 ea, ex, ra, rx;
                gates<E>(vga, vgx, ea, ex, ra, rx);
                const f2 q = fall<E>(mul2(s, sigmoid(vga, ea, ra)), small), v = square(q), u = mul2(sigmoid(vgx, ex, rx), vx);
                f2 aj = decay(q), wj = mul2(mul2(v, inverse_root<E>(v)), u);
                if (!kPlain) {
                    if (docs >> j & 1) aj = both(0.f), wj = u;
                    if (t + j >= p.T) aj = both(1.f), wj = both(0.f);
                }
                a[j] = aj;
                w[j] = wj;
                if (kPlain) {
                    mine_share.H = fma2(aj, mine_share.H, wj);
                    mine_share.P = mul2(mine_share.P, aj);
                } else {
                    mine_share.H = docs >> j & 1 ? wj : fma2(aj, mine_share.H, wj);
                    mine_share.P = mul2(mine_share.P, aj);
                }
            }
            mine_share.P = !kPlain && docs ? both(0.f) : clamp(mine_share.P);
        };
        if (docs == 0 && t + kTokens <= p.T) make(std::true_type{}); else make(std::false_type{});
        shares[buf][warp][lane] = make_ulonglong2(mine_share.P, mine_share.H);
        const bool cuts = __syncthreads_or(docs != 0);   // (a buffer is written again two rounds on, behind the next barrier)
        Share before, all;
        fold<false>(shares[buf], warp, lane, cuts, before, all);
        f2 h = through_cluster<false>(cluster, K, rank, peers[buf], all, warp, lane, carry);
        h = step(before.P, before.H, h);
        if (live && t < p.T) {
            if (p.saved != nullptr && warp == 0) {
                float* to = p.saved + ((i64)b * p.rounds + round) * p.C + c0;
                to[0] = lo(h);
                if (second) to[1] = hi(h);
            }
#pragma unroll
            for (int j = 0; j < kTokens; ++j) {
                if (t + j >= p.T) break;
                h = docs >> j & 1 ? w[j] : fma2(a[j], h, w[j]);
                put2<PAIRS>(y + (i64)(t + j) * p.C, h, second);
            }
        }
        stage = stage == S - 1 ? 0 : stage + 1;
        __syncwarp();
    }
    if (p.hT != nullptr && rank == 0 && warp == 0 && live) {
        p.hT[row] = lo(carry);
        if (second) p.hT[row + 1] = hi(carry);
    }
}

// Rounds from the last to the first; e (the gradient that comes into a token from the later ones) goes the same way as h does in
// the forward, with the same products of decays.  h before each token is made again from the saved states.
template <typename E, bool WIDE, bool PAIRS>
__global__ void __launch_bounds__(32 * kWarps, sizeof(E) == 2 ? 2 : 1) scan_backward_kernel(const Args p) {
    extern __shared__ __align__(16) unsigned char raw[];
    __shared__ ulonglong2 shares[2][kWarps][32], forward[2][kWarps][32], peers[2][kMaxCluster][32];
    constexpr int S = kBwdStages, kPart = kTokens * kTile;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    cg::cluster_group cluster = cg::this_cluster();
    const int K = (int)cluster.num_blocks(), rank = (int)cluster.block_rank(), unit = blockIdx.x / K;
    const int b = unit / p.tiles, c_tile = unit % p.tiles * kTile, c0 = c_tile + lane * 2;
    const bool live = c0 < p.C, second = c0 + 1 < p.C;
    const i64 base = (i64)b * p.T * p.C + c_tile;
    const E *x = static_cast<const E*>(p.x) + base, *gx = static_cast<const E*>(p.gx) + base, *ga = static_cast<const E*>(p.ga) + base,
            *dy = static_cast<const E*>(p.dy) + base;
    E *dx = static_cast<E*>(p.dx) + base + lane * 2, *dgx = static_cast<E*>(p.dgx) + base + lane * 2, *dga = static_cast<E*>(p.dga) + base + lane * 2;
    E* mine = reinterpret_cast<E*>(raw) + warp * 4 * kPart;
    const uint8_t* first = p.first ? p.first + (i64)b * p.T : nullptr;
    const f2 s = pack2(live ? p.s[c0] : 0.f, second ? p.s[c0 + 1] : 0.f);
    const i64 row = (i64)b * p.C + c0;
    f2 carry = pack2(live && p.dhT ? p.dhT[row] : 0.f, second && p.dhT ? p.dhT[row + 1] : 0.f), ds = both(0.f);
    const bool small = __all_sync(0xffffffffu, lo(s) <= 1.f && hi(s) <= 1.f);

    auto ask = [&](int round, int stage) {
        const int t = round * kRound + warp * kTokens;
        E* to = mine + stage * kWarps * 4 * kPart;
        if (round >= 0 && t < p.T) {
            fetch<E, WIDE>(to, x, t, p.T, p.C, c_tile, lane);
            fetch<E, WIDE>(to + kPart, gx, t, p.T, p.C, c_tile, lane);
            fetch<E, WIDE>(to + 2 * kPart, ga, t, p.T, p.C, c_tile, lane);
            fetch<E, WIDE>(to + 3 * kPart, dy, t, p.T, p.C, c_tile, lane);
        }
        commit();
    };
    const int turns = (p.rounds + K - 1) / K;
#pragma unroll
    for (int i = 0; i < S - 1; ++i) ask((turns - 1 - i) * K + rank, i);
    if (K > 1) cluster.sync();
    int stage = 0, buf = 0;
    for (int turn = turns - 1; turn >= 0; --turn, buf ^= 1) {
        const int round = turn * K + rank, t = round * kRound + warp * kTokens;
        ask(round - (S - 1) * K, stage == 0 ? S - 1 : stage - 1);
        f2 h = both(0.f);
        if (live && round < p.rounds) {
            const float* from = p.saved + ((i64)b * p.rounds + round) * p.C + c0;
            h = pack2(from[0], second ? from[1] : 0.f);
        }
        wait_group<S - 1>();
        __syncwarp();
        const E* in = mine + stage * kWarps * 4 * kPart + lane * 2;
        const uint32_t docs = firsts(first, t, p.T, lane);
        // per token: 1 - a, the gates as pairs, 1 / beta, and w = beta u, which makes room for h before the token
        f2 q[kTokens], r[kTokens], g[kTokens], inv[kTokens], w[kTokens], P = both(1.f), H = both(0.f), Q = both(0.f);
        auto make = [&](auto plain) {
            constexpr bool kPlain = decltype(plain)::value;
#pragma unroll
            for (int j = 0; j < kTokens; ++j) {
                const f2 vx = get2(in + j * kTile), vgx = get2(in + kPart + j * kTile), vga = get2(in + 2 * kPart + j * kTile);
                f2 ea, ex, ra, rx;
                gates<E>(vga, vgx, ea, ex, ra, rx);
                r[j] = sigmoid_pair(vga, ea, ra);
                g[j] = sigmoid_pair(vgx, ex, rx);
                q[j] = fall<E>(mul2(s, sigmoid(vga, ea, ra)), small);
                const f2 v = square(q[j]), u = mul2(sigmoid(vgx, ex, rx), vx);
                inv[j] = inverse_root<E>(v);
                w[j] = mul2(mul2(v, inv[j]), u);
                if (!kPlain) {
                    if (docs >> j & 1) q[j] = both(1.f), inv[j] = both(0.f), w[j] = u;
                    if (t + j >= p.T) q[j] = both(0.f), w[j] = both(0.f);
                }
                const f2 a = decay(q[j]);
                H = !kPlain && docs >> j & 1 ? w[j] : fma2(a, H, w[j]);
                P = mul2(P, a);
            }
#pragma unroll
            for (int j = kTokens - 1; j >= 0; --j) {
                if (kPlain) {
                    Q = mul2(decay(q[j]), add2(get2(in + 3 * kPart + j * kTile), Q));
                } else if (t + j < p.T) {
                    Q = docs >> j & 1 ? both(0.f) : mul2(decay(q[j]), add2(get2(in + 3 * kPart + j * kTile), Q));
                }
            }
            P = !kPlain && docs ? both(0.f) : clamp(P);
        };
        if (docs == 0 && t + kTokens <= p.T) make(std::true_type{}); else make(std::false_type{});
        shares[buf][warp][lane] = make_ulonglong2(P, Q);
        forward[buf][warp][lane] = make_ulonglong2(P, H);
        const bool cuts = __syncthreads_or(docs != 0);
        Share after, all;
        fold<true>(shares[buf], warp, lane, cuts, after, all);
        f2 e = through_cluster<true>(cluster, K, rank, peers[buf], all, warp, lane, carry);
        e = step(after.P, after.H, e);
        for (int i = 0; i < warp; ++i) {
            const ulonglong2 v = forward[buf][i][lane];
            h = step(v.x, v.y, h);
        }
        if (live && t < p.T) {
#pragma unroll
            for (int j = 0; j < kTokens; ++j) {
                const f2 before = h;
                h = docs >> j & 1 ? w[j] : fma2(decay(q[j]), h, w[j]);
                w[j] = before;
            }
#pragma unroll
            for (int j = kTokens - 1; j >= 0; --j) {
                if (t + j >= p.T) continue;
                const bool doc = docs >> j & 1;
                const f2 vx = get2(in + j * kTile), a = decay(q[j]), G = add2(get2(in + 3 * kPart + j * kTile), e);
                const f2 sr = each(r[j], of_pair), sg = each(g[j], of_pair), beta = doc ? both(1.f) : mul2(square(q[j]), inv[j]);
                const f2 ox = mul2(mul2(G, beta), sg), og = mul2(mul2(ox, vx), each(g[j], rest_of_pair));
                const f2 slope = fma2(w[j], both(-1.f), mul2(mul2(mul2(sg, vx), a), inv[j]));
                const f2 dL = doc ? both(0.f) : mul2(mul2(G, a), slope);
                const f2 oa = mul2(mul2(dL, mul2(s, sr)), each(r[j], rest_of_pair));
                ds = fma2(dL, sr, ds);
                e = doc ? both(0.f) : mul2(a, G);
                const i64 at = (i64)(t + j) * p.C;
                put2<PAIRS>(dx + at, ox, second);
                put2<PAIRS>(dgx + at, og, second);
                put2<PAIRS>(dga + at, oa, second);
            }
        }
        stage = stage == S - 1 ? 0 : stage + 1;
        __syncwarp();
    }
    if (p.dh0 != nullptr && rank == 0 && warp == 0 && live) {
        p.dh0[row] = lo(carry);
        if (second) p.dh0[row + 1] = hi(carry);
    }
    // the warps' shares of ds, in their order
    __syncthreads();
    shares[0][warp][lane] = make_ulonglong2(ds, 0);
    __syncthreads();
    if (warp == 0 && live) {
        f2 sum = both(0.f);
#pragma unroll
        for (int q = 0; q < kWarps; ++q) sum = add2(sum, shares[0][q][lane].x);
        float* to = p.ds + ((i64)b * K + rank) * p.C + c0;
        to[0] = lo(sum);
        if (second) to[1] = hi(sum);
    }
}

// One token: a thread per channel of a row.  Rows that share a slot are tokens of one sequence, in the order of the rows: the
// first of them takes the others along.  A negative slot is a row that only pads the batch; one behind the pool is refused: y
// of that row becomes NaN and the status word says so.
__device__ int g_update_error = 0;
constexpr int kBadSlot = 1;

template <typename E>
__global__ void __launch_bounds__(128) scan_update_kernel(int B, int C, int pool, const int* __restrict__ slots, float* state, const E* __restrict__ x,
                                                          const E* __restrict__ gx, const E* __restrict__ ga, const float* __restrict__ s, E* y) {
    const int b = blockIdx.y, c = blockIdx.x * 128 + threadIdx.x;
    int slot = b;
    bool later = false;
    if (slots != nullptr) {
        slot = slots[b];
        if (slot < 0) return;
        bool before = false;
        for (int q = threadIdx.x; q < B; q += 128) {
            const bool same = slots[q] == slot;
            before |= same && q < b;
            later |= same && q > b;
        }
        before = __syncthreads_or(before);
        later = __syncthreads_or(later);
        if (slot >= pool) {
            if (c < C) y[(i64)b * C + c] = from_f<E>(__int_as_float(0x7fffffff));
            if (threadIdx.x == 0) atomicMax(&g_update_error, kBadSlot);
            return;
        }
        if (before) return;
    }
    if (c >= C) return;
    float* at = state + (i64)slot * C + c;
    const float sc = s[c];
    float h = *at;
    for (int q = b; q < B; ++q) {
        if (q == b || slots[q] == slot) {
            const i64 i = (i64)q * C + c;
            const f2 vga = both(to_f(ga[i])), vgx = both(to_f(gx[i]));
            f2 ea, ex, ra, rx;
            gates<E>(vga, vgx, ea, ex, ra, rx);
            const f2 fallen = fall<E>(mul2(both(sc), sigmoid(vga, ea, ra)), false), v = square(fallen);
            h = fmaf(lo(decay(fallen)), h, lo(mul2(v, inverse_root<E>(v))) * (lo(sigmoid(vgx, ex, rx)) * to_f(x[i])));
            y[i] = from_f<E>(h);
        }
        if (!later) break;
    }
    *at = h;
}

bool aligned(const void* p, uintptr_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

int check(const char* what, int dtype, int B, int T, int C) {
    RWKV_REQUIRE(dtype == RWKVB200_F32 || dtype == RWKVB200_BF16, RWKVB200_EINVAL, "%s: unknown dtype %d", what, dtype);
    RWKV_REQUIRE(B > 0 && T > 0 && C > 0, RWKVB200_EINVAL, "%s: B=%d T=%d C=%d must be positive", what, B, T, C);
    RWKV_REQUIRE((i64)B * ((C + kTile - 1) / kTile) <= 0x7fffffff / kMaxCluster, RWKVB200_EINVAL, "%s: B=%d C=%d: too many blocks", what, B, C);
    RWKV_REQUIRE(T <= 0x7fffffff - 65536, RWKVB200_EINVAL, "%s: T=%d is too long", what, T);
    return RWKVB200_OK;
}

// How many blocks share a (sequence, channel tile): the K for which the rounds that an SM's places go through one after the other are
// fewest, a barrier of a cluster counting as a quarter of a round.
int cluster_size(int units, int rounds, int places) {
    int best = 1;
    double least = 0;
    for (int K = 1; K <= kMaxCluster; K *= 2) {
        if (K > 1 && K > rounds) break;
        const double cost = (double)(((i64)units * K + places - 1) / places) * ((rounds + K - 1) / K) * (K > 1 ? 1.25 : 1.0);
        if (K == 1 || cost < least) best = K, least = cost;
    }
    return best;
}

template <auto Kernel>
int launch(const char* what, const Args& p, int B, int K, int smem, cudaStream_t st) {
    if (allow_smem<Kernel>(smem) != cudaSuccess) return check_launch(what);
    cudaLaunchConfig_t config{};
    config.gridDim = dim3((unsigned)(B * p.tiles * K));
    config.blockDim = dim3(32 * kWarps);
    config.dynamicSmemBytes = smem;
    config.stream = st;
    cudaLaunchAttribute cluster;
    cluster.id = cudaLaunchAttributeClusterDimension;
    cluster.val.clusterDim.x = K;
    cluster.val.clusterDim.y = cluster.val.clusterDim.z = 1;
    config.attrs = &cluster;
    config.numAttrs = 1;
    cudaLaunchKernelEx(&config, Kernel, p);
    return check_launch(what);
}
template <typename E>
int run_forward(const Args& p, int B, int K, cudaStream_t st) {
    const char* what = "gated_scan_forward";
    const bool wide = p.C % (16 / sizeof(E)) == 0 && aligned(p.x, 16) && aligned(p.gx, 16) && aligned(p.ga, 16);
    const bool pairs = p.C % 2 == 0 && aligned(p.y, 2 * sizeof(E));
    constexpr int smem = fwd_smem<E>();
    if (wide && pairs) return launch<scan_forward_kernel<E, true, true>>(what, p, B, K, smem, st);
    return launch<scan_forward_kernel<E, false, false>>(what, p, B, K, smem, st);
}
template <typename E>
int run_backward(const Args& p, int B, int K, cudaStream_t st) {
    const char* what = "gated_scan_backward";
    const bool wide = p.C % (16 / sizeof(E)) == 0 && aligned(p.x, 16) && aligned(p.gx, 16) && aligned(p.ga, 16) && aligned(p.dy, 16);
    const bool pairs = p.C % 2 == 0 && aligned(p.dx, 2 * sizeof(E)) && aligned(p.dgx, 2 * sizeof(E)) && aligned(p.dga, 2 * sizeof(E));
    constexpr int smem = bwd_smem<E>();
    if (wide && pairs) return launch<scan_backward_kernel<E, true, true>>(what, p, B, K, smem, st);
    return launch<scan_backward_kernel<E, false, false>>(what, p, B, K, smem, st);
}

}  // namespace

int gated_scan_error(int clear) {
    int v = 0;
    if (clear) return cudaMemcpyToSymbol(g_update_error, &v, sizeof(v)) == cudaSuccess ? 0 : -1;
    return cudaMemcpyFromSymbol(&v, g_update_error, sizeof(v)) == cudaSuccess ? v : -1;
}

}  // namespace rwkvb200

using namespace rwkvb200;

extern "C" size_t rwkvb200_gated_scan_saved_bytes(int B, int T, int C) {
    if (B <= 0 || T <= 0 || C <= 0) return 0;
    return (size_t)B * ((T + kRound - 1) / kRound) * C * sizeof(float);
}
extern "C" size_t rwkvb200_gated_scan_work_bytes(int B, int T, int C) {
    if (B <= 0 || T <= 0 || C <= 0) return 0;
    return (size_t)B * kMaxCluster * C * sizeof(float);
}

extern "C" int rwkvb200_gated_scan_forward(int dtype, int B, int T, int C, const float* h0, const void* x, const void* gx, const void* ga,
                                           const float* s, const unsigned char* first, void* y, float* hT, void* saved, void* stream) {
    if (int e = check("gated_scan_forward", dtype, B, T, C)) return e;
    RWKV_NOTNULL(x); RWKV_NOTNULL(gx); RWKV_NOTNULL(ga); RWKV_NOTNULL(s); RWKV_NOTNULL(y);
    Args p{};
    p.T = T; p.C = C; p.tiles = (C + kTile - 1) / kTile; p.rounds = (T + kRound - 1) / kRound;
    p.h0 = h0; p.x = x; p.gx = gx; p.ga = ga; p.s = s; p.first = first; p.y = y; p.hT = hT; p.saved = static_cast<float*>(saved);
    const cudaStream_t st = as_stream(stream);
    const int K = cluster_size(B * p.tiles, p.rounds, 2 * sm_count());
    return dtype == RWKVB200_BF16 ? run_forward<bf16>(p, B, K, st) : run_forward<float>(p, B, K, st);
}

extern "C" int rwkvb200_gated_scan_backward(int dtype, int B, int T, int C, const void* x, const void* gx, const void* ga, const float* s,
                                            const unsigned char* first, const void* saved, const void* dy, const float* dhT, float* dh0, void* dx,
                                            void* dgx, void* dga, float* ds, void* work, void* stream) {
    if (int e = check("gated_scan_backward", dtype, B, T, C)) return e;
    RWKV_NOTNULL(x); RWKV_NOTNULL(gx); RWKV_NOTNULL(ga); RWKV_NOTNULL(s); RWKV_NOTNULL(saved); RWKV_NOTNULL(dy);
    RWKV_NOTNULL(dx); RWKV_NOTNULL(dgx); RWKV_NOTNULL(dga); RWKV_NOTNULL(ds); RWKV_NOTNULL(work);
    Args p{};
    p.T = T; p.C = C; p.tiles = (C + kTile - 1) / kTile; p.rounds = (T + kRound - 1) / kRound;
    p.x = x; p.gx = gx; p.ga = ga; p.s = s; p.first = first; p.saved = static_cast<float*>(const_cast<void*>(saved));
    p.dy = dy; p.dhT = dhT; p.dh0 = dh0; p.dx = dx; p.dgx = dgx; p.dga = dga; p.ds = static_cast<float*>(work);
    const cudaStream_t st = as_stream(stream);
    const int K = cluster_size(B * p.tiles, p.rounds, (dtype == RWKVB200_BF16 ? 2 : 1) * sm_count());
    const int rc = dtype == RWKVB200_BF16 ? run_backward<bf16>(p, B, K, st) : run_backward<float>(p, B, K, st);
    return rc != RWKVB200_OK ? rc : sum_rows(RWKVB200_F32, (i64)B * K, C, p.ds, ds, st);
}

extern "C" int rwkvb200_gated_scan_update(int dtype, int B, int C, int pool, float* state, const int* slots, const void* x, const void* gx,
                                          const void* ga, const float* s, void* y, void* stream) {
    if (int e = check("gated_scan_update", dtype, B, 1, C)) return e;
    RWKV_REQUIRE(pool > 0 && (slots != nullptr || pool >= B), RWKVB200_EINVAL, "gated_scan_update: %d states for %d rows", pool, B);
    RWKV_REQUIRE(B <= 65535, RWKVB200_EINVAL, "gated_scan_update: B=%d exceeds 65535", B);
    RWKV_NOTNULL(state); RWKV_NOTNULL(x); RWKV_NOTNULL(gx); RWKV_NOTNULL(ga); RWKV_NOTNULL(s); RWKV_NOTNULL(y);
    const dim3 grid((C + 127) / 128, B);
    const cudaStream_t st = as_stream(stream);
    if (dtype == RWKVB200_BF16)
        scan_update_kernel<bf16><<<grid, 128, 0, st>>>(B, C, pool, slots, state, (const bf16*)x, (const bf16*)gx, (const bf16*)ga, s, (bf16*)y);
    else
        scan_update_kernel<float><<<grid, 128, 0, st>>>(B, C, pool, slots, state, (const float*)x, (const float*)gx, (const float*)ga, s, (float*)y);
    return check_launch("gated_scan_update");
}
