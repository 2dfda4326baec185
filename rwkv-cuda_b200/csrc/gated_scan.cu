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
// A block owns 32 lanes x 2 channels of one sequence and goes through it in rounds of kWarps x 16 (backward and fp32: 8) tokens, a
// warp owns 16 (8) of them: it makes the gates of its tokens in registers, reduces them to (P, H) (the product of the decays and the end
// state from a zero start), all warps fold those of the warps before theirs onto the block's state, and each walks its tokens
// once more from its own start state.  Every input is read once, y is written once.  Where there are few (sequence, channel)
// blocks, a cluster of blocks shares the rounds: block k of K takes rounds k, k + K, ..., and the (P, H) of their rounds go
// through distributed shared memory, one cluster barrier for K rounds.
//
// Every warp copies its own tokens to shared memory (cp.async), a round ahead: that keeps enough bytes in flight and needs no
// barrier.  What bounds the kernels is in front of each.
#include "packed.cuh"
#include <cooperative_groups.h>
#include <atomic>
#include <initializer_list>
#include <type_traits>

namespace rwkvb200 {
namespace {

namespace cg = cooperative_groups;

constexpr int kWarps = 8;
template <typename E> constexpr int kFwdTokens = sizeof(E) == 2 ? 16 : 8;   // per warp and round: what fits two blocks per SM
constexpr int kBwdTokens = 8;                // (three values per token and channel to keep instead of two)
constexpr int kSaved = kWarps * kBwdTokens;  // the forward saves the state before every round of the backward
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

// The functions behind the gates: for bf16 tensors the hardware approximations (2e-7 relative, and for the exponential as many units of
// 2^-24 as its argument is large, from the product with log2 e: 5e-7 at 10, 1.9e-6 at 41; a step of bf16 is 4e-3), for fp32 CUDA's
// exponential and one step of Newton's method behind the others.
constexpr float kLog2e = 1.4426950408889634f;
template <typename E> struct Fn;
template <> struct Fn<bf16> {
    static __device__ __forceinline__ float exp_minus(float x) { return ex2(-kLog2e * x); }
    static __device__ __forceinline__ f2 exp_minus(f2 x) {
        float a, b;
        unpack2(mul2(x, pack2(-kLog2e, -kLog2e)), a, b);
        return pack2(ex2(a), ex2(b));
    }
    static __device__ __forceinline__ float inverse(float x) { return rcp(x); }
    static __device__ __forceinline__ float inverse_any(float x) { return rcp(x); }
    static __device__ __forceinline__ float inverse_root(float v) { return rsqrt_fast(v); }
};
template <> struct Fn<float> {
    static __device__ __forceinline__ float exp_minus(float x) { return expf(-x); }
    static __device__ __forceinline__ f2 exp_minus(f2 x) {
        float a, b;
        unpack2(x, a, b);
        return pack2(expf(-a), expf(-b));
    }
    static __device__ __forceinline__ float inverse(float x) {   // (of finite values from 1 on)
        const float r = rcp(x);
        return fmaf(r, fmaf(-x, r, 1.f), r);
    }
    static __device__ __forceinline__ float inverse_any(float x) { return 1.f / x; }
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

// 1 - exp(-L) of two channels, with all its digits where L is small: for L <= 1 as L times a polynomial (interpolation of
// (1 - exp(-L)) / L at the Chebyshev points of [0, 1]: off by 2.4e-8 with its coefficients in fp32, and by 1.4e-7 as it is evaluated),
// which takes no special function; beyond it -exp(-L), which has the digits of a instead (decay and fallen tell the two apart by the sign).
// SMALL: s <= 1 in all channels of the warp.
template <typename E, bool SMALL>
__device__ __forceinline__ f2 fall(f2 L) {
    f2 q = fma2(L, both(0.0001290763f), both(-0.001300775f));
    q = fma2(q, L, both(0.008275505f));
    q = fma2(q, L, both(-0.04164685f));
    q = fma2(q, L, both(0.16666341f));
    q = fma2(q, L, both(-0.4999998f));
    q = fma2(q, L, both(1.f));
    q = mul2(q, L);
    if (SMALL) return q;
    return each(L, q, [](float l, float p) { return l <= 1.f ? p : -Fn<E>::exp_minus(l); });
}
// s as it is read: -0 becomes 0, as -0 times a gate would come out of the polynomial with the sign of the other form
__device__ __forceinline__ float rate(float s) { return s + 0.f; }
// a and 1 - a^2 = (1 - a) (2 - (1 - a)) of what fall has made
template <bool SMALL>
__device__ __forceinline__ f2 decay(f2 q) {
    if (SMALL) return fma2(q, both(-1.f), both(1.f));
    return each(q, [](float v) { return __float_as_int(v) < 0 ? -v : 1.f - v; });
}
template <bool SMALL>
__device__ __forceinline__ f2 square(f2 q) {
    if (!SMALL) q = each(q, [](float v) { return __float_as_int(v) < 0 ? 1.f + v : v; });
    return mul2(q, fma2(q, both(-1.f), both(2.f)));
}
// 1 / sqrt(1 - a^2); 0 below the normal numbers, where beta counts as 0 (and NaN below 0, which only a negative s makes)
template <typename E>
__device__ __forceinline__ f2 inverse_root(f2 v) {
    return each(v, [](float x) { return fabsf(x) < 1.2e-38f ? 0.f : Fn<E>::inverse_root(x); });
}

// sigmoid(ga), sigmoid(gx) and what they lack of 1, without loss of either.  Two forms: as long as no gate is below kLeast, so that
// exp(-ga) exp(-gx) does not overflow, both come from one division; tiles with a gate that is, or with a NaN, which must not go from
// one gate into the other (EXTREME), take one each.
constexpr float kLeast = -41.f;
template <typename E, bool EXTREME>
struct Gates {
    f2 a, x, ea, ex;
    f2 ga, gx;
    __device__ __forceinline__ Gates(f2 ga, f2 gx) : ga(ga), gx(gx) {
        const f2 one = both(1.f);
        ea = Fn<E>::exp_minus(ga);
        ex = Fn<E>::exp_minus(gx);
        const f2 da = add2(ea, one), dx = add2(ex, one);
        if (EXTREME) {
            a = each(da, [](float v) { return Fn<E>::inverse_any(v); });
            x = each(dx, [](float v) { return Fn<E>::inverse_any(v); });
        } else {
            const f2 r = each(mul2(da, dx), [](float v) { return Fn<E>::inverse(v); });
            a = mul2(r, dx);
            x = mul2(r, da);
        }
    }
    static __device__ __forceinline__ f2 other(f2 g) {
        return each(g, [](float v) { return Fn<E>::inverse_any(1.f + Fn<E>::exp_minus(-v)); });
    }
    __device__ __forceinline__ f2 rest_a() const { return EXTREME ? other(ga) : mul2(ea, a); }
    __device__ __forceinline__ f2 rest_x() const { return EXTREME ? other(gx) : mul2(ex, x); }
};

// two neighbouring channels as they lie in memory
template <typename E> struct Pair;
template <> struct Pair<bf16> {
    __nv_bfloat162 v;
    __device__ __forceinline__ explicit Pair(const bf16* p) : v(*reinterpret_cast<const __nv_bfloat162*>(p)) {}
    __device__ __forceinline__ explicit Pair(float x) : v(__floats2bfloat162_rn(x, x)) {}
    static __device__ __forceinline__ Pair of(uint32_t w) {
        Pair p(0.f);
        p.v = *reinterpret_cast<const __nv_bfloat162*>(&w);
        return p;
    }
    __device__ __forceinline__ f2 get() const {
        const uint32_t w = *reinterpret_cast<const uint32_t*>(&v);
        return pack2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
    }
    __device__ __forceinline__ void least(const Pair& o) { v = __hmin2_nan(v, o.v); }
    __device__ __forceinline__ bool all_from(float x) const { return __low2float(v) >= x && __high2float(v) >= x; }
};
template <> struct Pair<float> {
    float2 v;
    __device__ __forceinline__ explicit Pair(const float* p) : v(*reinterpret_cast<const float2*>(p)) {}
    __device__ __forceinline__ explicit Pair(float x) : v(make_float2(x, x)) {}
    __device__ __forceinline__ f2 get() const { return pack2(v.x, v.y); }
    static __device__ __forceinline__ float min_nan(float a, float b) {
        float m;
        asm("min.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(a), "f"(b));
        return m;
    }
    __device__ __forceinline__ void least(const Pair& o) { v.x = min_nan(v.x, o.v.x), v.y = min_nan(v.y, o.v.y); }
    __device__ __forceinline__ bool all_from(float x) const { return v.x >= x && v.y >= x; }
};
// ... to global memory: as one word, or one after the other where C is odd or a tensor starts between two words
template <bool WORD>
__device__ __forceinline__ void put2(bf16* p, f2 v, bool second) {
    const __nv_bfloat162 t = __floats2bfloat162_rn(lo(v), hi(v));
    if (WORD) {
        *reinterpret_cast<__nv_bfloat162*>(p) = t;
    } else {
        p[0] = t.x;
        if (second) p[1] = t.y;
    }
}
template <bool WORD>
__device__ __forceinline__ void put2(float* p, f2 v, bool second) {
    if (WORD) {
        *reinterpret_cast<float2*>(p) = make_float2(lo(v), hi(v));
    } else {
        p[0] = lo(v);
        if (second) p[1] = hi(v);
    }
}

// j rows of C elements behind p (one wide multiply-add)
template <typename E>
__device__ __forceinline__ E* rows_on(E* p, uint32_t row_bytes, int j) { return reinterpret_cast<E*>(reinterpret_cast<char*>(p) + (uint64_t)row_bytes * (uint32_t)j); }

struct Args {
    int B, T, C, tiles, rounds, saves;   // channel tiles, rounds of the kernel, of the backward
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
template <int L>
__device__ __forceinline__ uint32_t firsts(const uint8_t* first, int t, int T, int lane) {
    if (first == nullptr) return 0;
    const bool f = lane < L && t + lane < T && first[t + lane] != 0;
    return __ballot_sync(0xffffffffu, f);
}

// How rows of C elements lie in memory: each starts on a 16-byte boundary; on one of a pair of channels (C is even); anywhere.
enum { kWideRows, kPairRows, kAnyRows };
// In shared memory a row is kTile elements, or, bf16 anywhere, the 33 words that hold them.
template <typename E, int ROWS> constexpr int kPitch = sizeof(E) == 2 && ROWS == kAnyRows ? kTile + 2 : kTile;

// Tiles of N tensors, L rows each, from token t on: to shared memory, without waiting.  A lane asks for pieces of 16 bytes, for its pair
// of each row, or, anywhere, for single words: there is no asynchronous copy of two bytes, so that bf16 rows come with what shares a
// word with their ends, and are shifted when they are read.  bf16, B8 T4096: C4096 238 and 485 us,
// C4094 435 and 675, C4095 545 and 817.  (Element by element, without running ahead, a step of B4 T1761 C2474 took 1310 us instead of 262.)
// What lies outside is left alone.
template <typename E, int ROWS, int L, int N>
struct Fetch {
    static constexpr int n = 16 / sizeof(E), kRow = kTile / n, kRows = 32 / kRow;   // elements of a piece, pieces of a row, rows at a time
    static constexpr int kPart = L * kPitch<E, ROWS>, kPitchBytes = kPitch<E, ROWS> * (int)sizeof(E), kWords = kTile / 2 + 1;
    static constexpr bool kShifted = sizeof(E) == 2 && ROWS == kAnyRows;
    const E* from[N];
    uint32_t off = 0, off_odd;   // bits by which even and odd rows are off, in five bits for each tensor (kShifted; tiles begin at even tokens)
    int T, C, row, lane, channels;
    i64 at, base, total;   // at: of this lane's first piece
    bool inside, edge;     // its channels; the first or the last sequence
    __device__ __forceinline__ Fetch(int T, int C, int c_tile, int lane, i64 base, i64 total, bool edge)
        : T(T), C(C), row(lane / kRow), lane(lane), channels(min(kTile, C - c_tile)), base(base), total(total), edge(edge) {
        const int c = ROWS == kWideRows ? lane % kRow * n : lane * 2;
        at = (ROWS == kWideRows ? (i64)row * C : 0) + c;
        inside = c_tile + c < C;
    }
    __device__ __forceinline__ void tensor(int k, const void* p) {
        from[k] = static_cast<const E*>(p) + base;
        off |= (uint32_t)(reinterpret_cast<uintptr_t>(from[k]) & 2) * 8 << 5 * k;
        off_odd = off ^ (C & 1 ? 0x84210u : 0u);
    }
    __device__ __forceinline__ uint32_t shift(int k, int j) const { return (j & 1 ? off_odd : off) >> 5 * k; }   // (its low five bits)
    __device__ __forceinline__ void operator()(E* to, int t) const {
        const uint32_t shared = (uint32_t)__cvta_generic_to_shared(to);
        const bool whole = t + L <= T;
        if (ROWS == kWideRows) {
            const i64 first = (i64)t * C + at, step = (i64)kRows * C;
            if (whole) {
                if (inside) {
#pragma unroll
                    for (int k = 0; k < N; ++k) {
                        const E* p = from[k] + first;
#pragma unroll
                        for (int i = 0; i < L / kRows; ++i, p += step) copy<16>(shared + lane * 16 + (k * L + i * kRows) * kPitchBytes, p);
                    }
                }
            } else {
#pragma unroll
                for (int k = 0; k < N; ++k)
#pragma unroll
                    for (int i = 0; i < L / kRows; ++i)
                        if (inside && t + i * kRows + row < T) copy<16>(shared + lane * 16 + (k * L + i * kRows) * kPitchBytes, from[k] + first + i * step);
            }
        } else if (ROWS == kPairRows) {
            if (!inside) return;
            const uint32_t mine = shared + lane * 2 * (int)sizeof(E);
            const uint32_t row_bytes = C * (uint32_t)sizeof(E);
            const int rows = whole ? L : T - t;
#pragma unroll
            for (int k = 0; k < N; ++k) {
                const E* p = from[k] + (i64)t * C + at;
                if (whole) {
#pragma unroll
                    for (int j = 0; j < L; ++j) copy<2 * sizeof(E)>(mine + (k * L + j) * kPitchBytes, rows_on(const_cast<E*>(p), row_bytes, j));
                } else {
#pragma unroll 1
                    for (int j = 0; j < rows; ++j) copy<2 * sizeof(E)>(mine + (k * L + j) * kPitchBytes, rows_on(const_cast<E*>(p), row_bytes, j));
                }
            }
        } else if (!kShifted) {
#pragma unroll
            for (int k = 0; k < N; ++k) {
                const E* p = from[k] + (i64)t * C + lane;
#pragma unroll
                for (int j = 0; j < L; ++j, p += C)
                    if (whole || t + j < T) {
                        if (lane < channels) copy<4>(shared + lane * 4 + (k * L + j) * kPitchBytes, p);
                        if (lane + 32 < channels) copy<4>(shared + lane * 4 + 128 + (k * L + j) * kPitchBytes, p + 32);
                    }
            }
        } else {
            // word i of a row holds its elements 2 i - 1, 2 i or 2 i, 2 i + 1; one at an end of the tensor may be half outside
            if (whole && !(edge && (t == 0 || t + L == T))) {
                const uint32_t row_bytes = C * (uint32_t)sizeof(E);
#pragma unroll
                for (int k = 0; k < N; ++k) {
                    const E* p = from[k] + (i64)t * C + lane * 2;
                    if (lane * 2 < channels) {   // (with one before it or not)
#pragma unroll 4
                        for (int j = 0; j < L; ++j) copy<4>(shared + lane * 4 + (k * L + j) * kPitchBytes, rows_on(const_cast<E*>(p), row_bytes, j) - (shift(k, j) >> 4 & 1));
                    } else if (lane * 2 == channels) {   // (an even row's last channel is in the word before, an odd one's may be here)
#pragma unroll 1
                        for (int j = 0; j < L; ++j)
                            if ((shift(k, j) & 16) != 0) copy<4>(shared + lane * 4 + (k * L + j) * kPitchBytes, rows_on(const_cast<E*>(p), row_bytes, j) - 1);
                    }
                    // (the 33rd word of row `lane`)
                    if (lane < L && (shift(k, lane) & 16) != 0 && channels == kTile)
                        copy<4>(shared + 2 * kTile + (k * L + lane) * kPitchBytes, from[k] + (i64)(t + lane) * C + kTile - 1);
                }
            } else {
#pragma unroll 1
                for (int k = 0; k < N; ++k) {
                    const E* tensor = from[0];
#pragma unroll
                    for (int q = 1; q < N; ++q) tensor = k == q ? from[q] : tensor;
#pragma unroll 1
                    for (int w = lane; w < L * kWords; w += 32) {
                        const int j = w / kWords, i = w % kWords * 2 - (int)(shift(k, j) >> 4 & 1);
                        if (t + j >= T || i >= channels) continue;
                        const uint32_t word = shared + (k * L + j) * kPitchBytes + w % kWords * 4;
                        const i64 nth = (i64)(t + j) * C + i;
                        if (base + nth >= 0 && base + nth + 1 < total) {
                            copy<4>(word, tensor + nth);
                        } else {
                            const int half = base + nth < 0;
                            const uint16_t v = *reinterpret_cast<const uint16_t*>(tensor + nth + half);
                            asm volatile("st.shared.u16 [%0], %1;" ::"r"(word + half * 2), "h"(v) : "memory");
                        }
                    }
                }
            }
        }
    }
    template <int BYTES> static __device__ __forceinline__ void copy(uint32_t to, const E* p) {
        if (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(p) : "memory");
        else asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(to), "l"(p), "n"(BYTES) : "memory");
    }
    // two channels of row j of tensor k, from those of the tile's first row on; `kept` has the bits of those that are there (kShifted)
    __device__ __forceinline__ Pair<E> read(const E* in, int k, int j, uint32_t kept) const {
        const E* p = in + k * kPart + j * kPitch<E, ROWS>;
        if constexpr (kShifted) {
            const uint32_t* w = reinterpret_cast<const uint32_t*>(p);
            return Pair<E>::of(__funnelshift_r(w[0], w[1], shift(k, j)) & kept);
        } else {
            return Pair<E>(p);
        }
    }
};
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
// What leaves the shares before warp `warp` (backward: those behind it, from the last one on) with the state `h`.
template <bool REVERSED>
__device__ __forceinline__ f2 through_block(const ulonglong2 (*shares)[32], int warp, int lane, bool cuts, f2 h) {
    auto walk = [&](auto plain) {
#pragma unroll
        for (int i = 0; i < kWarps - 1; ++i) {
            const int q = REVERSED ? kWarps - 1 - i : i;
            if (REVERSED ? q <= warp : q >= warp) break;
            const ulonglong2 v = shares[q][lane];
            h = decltype(plain)::value ? fma2(v.x, h, v.y) : step(v.x, v.y, h);
        }
    };
    if (cuts) walk(std::false_type{}); else walk(std::true_type{});
    return h;
}
// The state before this block's round, from the state before the rounds of all blocks of the cluster, which becomes the one behind them.
// The shares of the blocks go through distributed shared memory: warp q brings this block's to block q.
template <bool REVERSED>
__device__ __forceinline__ f2 through_cluster(cg::cluster_group& cluster, int K, int rank, const ulonglong2 (*shares)[32], ulonglong2 (*peers)[32], int warp,
                                              int lane, bool cuts, f2& carry) {
    if (warp < K) {
        Share all{both(1.f), both(0.f)};
        if (cuts) {
#pragma unroll
            for (int i = 0; i < kWarps; ++i) {
                const ulonglong2 v = shares[REVERSED ? kWarps - 1 - i : i][lane];
                all.H = step(v.x, v.y, all.H);
                all.P = behind(v.x, all.P);
            }
        } else {
#pragma unroll
            for (int i = 0; i < kWarps; ++i) {
                const ulonglong2 v = shares[REVERSED ? kWarps - 1 - i : i][lane];
                all.H = fma2(v.x, all.H, v.y);
                all.P = mul2(v.x, all.P);
            }
            all.P = clamp(all.P);
        }
        *cluster.map_shared_rank(&peers[rank][lane], warp) = make_ulonglong2(all.P, all.H);
    }
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

constexpr int kFwdStages = 2;
constexpr int kBwdStages = 2;
template <typename E, int ROWS> constexpr int fwd_smem() { return kFwdStages * kWarps * 3 * kFwdTokens<E> * kPitch<E, ROWS> * (int)sizeof(E); }
template <typename E, int ROWS> constexpr int bwd_smem() { return kBwdStages * kWarps * 4 * kBwdTokens * kPitch<E, ROWS> * (int)sizeof(E); }

// A warp's tile: all tokens and channels are there, no document begins and s <= 1; only s <= 1; not even that; or some gate is out of
// range (found on the way)
enum { kSimpleTile, kDocumentTile, kLargeTile, kExtremeTile };
template <int M> using Mode = std::integral_constant<int, M>;

// B8 T4096 C4096 bf16: 238 us, 4.5 TB/s; 176 us without the arithmetic of the gates, 216 without the exchange between the warps.
// Special functions 52 %, issue slots 54 %, four warps per scheduler: three blocks per SM with 8 tokens per warp are no faster.  Of
// the 128 registers a few are short: 112 to 156 bytes of spills a thread (rows anywhere 644 to 704).  With s up to 8 in each tile 320 us, with a gate
// below -41 in each 463.
// One sequence of 32768 tokens, 2048 channels (clusters of 8): 162 us, 111 without the exchange.
template <typename E, int ROWS, bool CLUSTER>
__global__ void __launch_bounds__(32 * kWarps, 2) scan_forward_kernel(const Args p) {
    extern __shared__ __align__(16) unsigned char raw[];
    __shared__ ulonglong2 shares[2][kWarps][32], peers[2][CLUSTER ? kMaxCluster : 1][32];
    __shared__ f2 ends[2][32];   // the state behind a round (a lone block's)
    constexpr int S = kFwdStages, kTokens = kFwdTokens<E>, kRound = kWarps * kTokens, kPart = kTokens * kPitch<E, ROWS>;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    cg::cluster_group cluster = cg::this_cluster();
    const int K = CLUSTER ? (int)cluster.num_blocks() : 1, rank = CLUSTER ? (int)cluster.block_rank() : 0, unit = blockIdx.x / K;
    const int b = unit / p.tiles, c_tile = unit % p.tiles * kTile, c0 = c_tile + lane * 2;
    const bool live = c0 < p.C, second = c0 + 1 < p.C;
    const i64 base = (i64)b * p.T * p.C + c_tile;
    Fetch<E, ROWS, kTokens, 3> fetch(p.T, p.C, c_tile, lane, base, (i64)p.B * p.T * p.C, b == 0 || b == p.B - 1);
    fetch.tensor(0, p.x);
    fetch.tensor(1, p.gx);
    fetch.tensor(2, p.ga);
    E* y = static_cast<E*>(p.y) + base + lane * 2;
    E* mine = reinterpret_cast<E*>(raw) + warp * 3 * kPart;
    const uint32_t kept = second ? 0xffffffffu : 0xffffu;
    if (ROWS == kAnyRows && sizeof(E) == 4) {   // (a last channel's neighbour stays 0)
        for (int i = lane; i < S * kWarps * 3 * kPart; i += 32)
            if (i / (3 * kPart) % kWarps == 0) mine[i] = from_f<E>(0.f);
        __syncwarp();
    }
    const uint32_t row_bytes = p.C * (uint32_t)sizeof(E);
    const uint8_t* first = p.first ? p.first + (i64)b * p.T : nullptr;
    const f2 s = pack2(live ? rate(p.s[c0]) : 0.f, second ? rate(p.s[c0 + 1]) : 0.f);
    const i64 row = (i64)b * p.C + c0;
    f2 carry = pack2(live && p.h0 ? p.h0[row] : 0.f, second && p.h0 ? p.h0[row + 1] : 0.f);
    const bool small = __all_sync(0xffffffffu, lo(s) <= 1.f && hi(s) <= 1.f);

    auto ask = [&](int round, int stage) {
        const int t = round * kRound + warp * kTokens;
        if (t < p.T) fetch(mine + stage * kWarps * 3 * kPart, t);
        commit();
    };
#pragma unroll
    for (int i = 0; i < S - 1; ++i) ask(rank + i * K, i);
    if (CLUSTER) cluster.sync();   // (a block's shared memory is written by others once it has begun)
    else if (warp == kWarps - 1) ends[1][lane] = carry;
    int stage = 0, buf = 0;
    for (int r0 = 0; r0 < p.rounds; r0 += K, buf ^= 1) {   // (all blocks of a cluster go through the same barriers)
        const int round = r0 + rank, t = round * kRound + warp * kTokens;
        ask(round + (S - 1) * K, stage == 0 ? S - 1 : stage - 1);
        wait_group<S - 1>();
        __syncwarp();
        const E* in = mine + stage * kWarps * 3 * kPart + lane * 2;
        const uint32_t docs = firsts<kTokens>(first, t, p.T, lane);
        f2 a[kTokens], w[kTokens];
        Share share;
        Pair<E> least(0.f);
        auto make = [&](auto mode) {
            constexpr bool kSimple = decltype(mode)::value == kSimpleTile, kExtreme = decltype(mode)::value == kExtremeTile, kSmall = decltype(mode)::value <= kDocumentTile;
            share.P = both(1.f);
            share.H = both(0.f);
#pragma unroll
            for (int j = 0; j < kTokens; ++j) {
                const Pair<E> vgx = fetch.read(in, 1, j, kept), vga = fetch.read(in, 2, j, kept);
                const Gates<E, kExtreme> g(vga.get(), vgx.get());
                if (!kExtreme && (kSimple || t + j < p.T)) least.least(vga), least.least(vgx);   // (other rows hold anything)
                const f2 q = fall<E, kSmall>(mul2(s, g.a)), v = square<kSmall>(q), u = mul2(g.x, fetch.read(in, 0, j, kept).get());
                a[j] = decay<kSmall>(q);
                // (v of 0 or below the normal numbers: beta is 0)
                w[j] = kSimple ? mul2(mul2(v, each(v, [](float z) { return Fn<E>::inverse_root(fmaxf(z, 1.2e-38f)); })), u)
                               : mul2(mul2(v, inverse_root<E>(v)), u);
                if (!kSimple) {
                    if (docs >> j & 1) a[j] = both(0.f), w[j] = u;
                    if (t + j >= p.T) a[j] = both(1.f), w[j] = both(0.f);
                }
                share.H = !kSimple && docs >> j & 1 ? w[j] : fma2(a[j], share.H, w[j]);
                share.P = mul2(share.P, a[j]);
            }
            share.P = !kSimple && docs ? both(0.f) : clamp(share.P);
        };
        int mode = !small ? kLargeTile : docs == 0 && t + kTokens <= p.T && c_tile + kTile <= p.C ? kSimpleTile : kDocumentTile;
        if (mode == kSimpleTile) make(Mode<kSimpleTile>{});
        else if (mode == kDocumentTile) make(Mode<kDocumentTile>{});
        else make(Mode<kLargeTile>{});
        if (__any_sync(0xffffffffu, live && !least.all_from(kLeast))) {
            mode = kExtremeTile;
            make(Mode<kExtremeTile>{});
        }
        shares[buf][warp][lane] = make_ulonglong2(share.P, share.H);
        const bool cuts = __syncthreads_or(docs != 0);   // (a buffer is written again two rounds on, behind the next barrier)
        f2 h = CLUSTER ? through_cluster<false>(cluster, K, rank, shares[buf], peers[buf], warp, lane, cuts, carry) : ends[buf ^ 1][lane];
        h = through_block<false>(shares[buf], warp, lane, cuts, h);
        if (p.saved != nullptr && t % kSaved == 0 && live && t < p.T) {
            float* to = p.saved + ((i64)b * p.saves + t / kSaved) * p.C + c0;
            to[0] = lo(h);
            if (second) to[1] = hi(h);
        }
        E* to = y + (i64)t * p.C;
        if (mode == kSimpleTile) {
#pragma unroll
            for (int j = 0; j < kTokens; ++j) {
                h = fma2(a[j], h, w[j]);
                put2<ROWS != kAnyRows>(rows_on(to, row_bytes, j), h, second);
            }
        } else {
#pragma unroll
            for (int j = 0; j < kTokens; ++j) {
                h = docs >> j & 1 ? w[j] : fma2(a[j], h, w[j]);
                if (live && t + j < p.T) put2<ROWS != kAnyRows>(rows_on(to, row_bytes, j), h, second);
            }
        }
        if (!CLUSTER && warp == kWarps - 1) ends[buf][lane] = h;
        stage = stage == S - 1 ? 0 : stage + 1;
        __syncwarp();
    }
    if (!CLUSTER) {
        __syncthreads();
        carry = ends[buf ^ 1][lane];
    }
    if (p.hT != nullptr && rank == 0 && warp == 0 && live) {
        p.hT[row] = lo(carry);
        if (second) p.hT[row + 1] = hi(carry);
    }
}

// Rounds from the last to the first; e (the gradient that comes into a token from the later ones) goes the same way as h does in
// the forward, with the same products of decays.  h before each token is made again from the saved states, and so are the gates
// in the last walk: keeping them would take more registers than two blocks per SM have.  B8 T4096 C4096 bf16: 487 us, 3.9 TB/s; 419
// without the exchange, 358 without the arithmetic of the last walk, 325 without that and the gates'.  T32768 C2048: 330, and 220.
// fp32 takes 198 to 209 registers and 128 KB: one block of eight warps per SM, B8 T512 C1024 46 us for 18 of bytes.
template <typename E, int ROWS, bool CLUSTER>
__global__ void __launch_bounds__(32 * kWarps, sizeof(E) == 2 ? 2 : 1) scan_backward_kernel(const Args p) {
    extern __shared__ __align__(16) unsigned char raw[];
    __shared__ ulonglong2 shares[2][kWarps][32], peers[2][CLUSTER ? kMaxCluster : 1][32];
    __shared__ f2 forward[2][kWarps][32], ends[2][32];
    constexpr int S = kBwdStages, kTokens = kBwdTokens, kRound = kWarps * kTokens, kPart = kTokens * kPitch<E, ROWS>;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    cg::cluster_group cluster = cg::this_cluster();
    const int K = CLUSTER ? (int)cluster.num_blocks() : 1, rank = CLUSTER ? (int)cluster.block_rank() : 0, unit = blockIdx.x / K;
    const int b = unit / p.tiles, c_tile = unit % p.tiles * kTile, c0 = c_tile + lane * 2;
    const bool live = c0 < p.C, second = c0 + 1 < p.C;
    const i64 base = (i64)b * p.T * p.C + c_tile;
    Fetch<E, ROWS, kTokens, 4> fetch(p.T, p.C, c_tile, lane, base, (i64)p.B * p.T * p.C, b == 0 || b == p.B - 1);
    fetch.tensor(0, p.x);
    fetch.tensor(1, p.gx);
    fetch.tensor(2, p.ga);
    fetch.tensor(3, p.dy);
    E *dx = static_cast<E*>(p.dx) + base + lane * 2, *dgx = static_cast<E*>(p.dgx) + base + lane * 2, *dga = static_cast<E*>(p.dga) + base + lane * 2;
    E* mine = reinterpret_cast<E*>(raw) + warp * 4 * kPart;
    const uint32_t kept = second ? 0xffffffffu : 0xffffu;
    if (ROWS == kAnyRows && sizeof(E) == 4) {   // (a last channel's neighbour stays 0)
        for (int i = lane; i < S * kWarps * 4 * kPart; i += 32)
            if (i / (4 * kPart) % kWarps == 0) mine[i] = from_f<E>(0.f);
        __syncwarp();
    }
    const uint32_t row_bytes = p.C * (uint32_t)sizeof(E);
    const uint8_t* first = p.first ? p.first + (i64)b * p.T : nullptr;
    const f2 s = pack2(live ? rate(p.s[c0]) : 0.f, second ? rate(p.s[c0 + 1]) : 0.f);
    const i64 row = (i64)b * p.C + c0;
    f2 carry = pack2(live && p.dhT ? p.dhT[row] : 0.f, second && p.dhT ? p.dhT[row + 1] : 0.f), ds = both(0.f);
    const bool small = __all_sync(0xffffffffu, lo(s) <= 1.f && hi(s) <= 1.f);

    auto ask = [&](int round, int stage) {
        const int t = round * kRound + warp * kTokens;
        if (round >= 0 && t < p.T) fetch(mine + stage * kWarps * 4 * kPart, t);
        commit();
    };
    const int turns = (p.rounds + K - 1) / K;
#pragma unroll
    for (int i = 0; i < S - 1; ++i) ask((turns - 1 - i) * K + rank, i);
    if (CLUSTER) cluster.sync();
    else if (warp == 0) ends[1][lane] = carry;
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
        const uint32_t docs = firsts<kTokens>(first, t, p.T, lane);
        // per token: 1 - a, 1 / beta, and w = beta u, which makes room for h before the token
        f2 q[kTokens], inv[kTokens], w[kTokens], P, H, Q;
        Pair<E> least(0.f);
        auto make = [&](auto mode) {
            constexpr bool kSimple = decltype(mode)::value == kSimpleTile, kExtreme = decltype(mode)::value == kExtremeTile, kSmall = decltype(mode)::value <= kDocumentTile;
            P = both(1.f);
            H = Q = both(0.f);
#pragma unroll
            for (int j = 0; j < kTokens; ++j) {
                const Pair<E> vgx = fetch.read(in, 1, j, kept), vga = fetch.read(in, 2, j, kept);
                const Gates<E, kExtreme> g(vga.get(), vgx.get());
                if (!kExtreme && (kSimple || t + j < p.T)) least.least(vga), least.least(vgx);   // (other rows hold anything)
                q[j] = fall<E, kSmall>(mul2(s, g.a));
                const f2 v = square<kSmall>(q[j]), u = mul2(g.x, fetch.read(in, 0, j, kept).get());
                inv[j] = inverse_root<E>(v);
                w[j] = mul2(mul2(v, inv[j]), u);
                if (!kSimple) {
                    if (docs >> j & 1) q[j] = both(1.f), inv[j] = both(0.f), w[j] = u;
                    if (t + j >= p.T) q[j] = both(0.f), w[j] = both(0.f);
                }
                const f2 a = decay<kSmall>(q[j]);
                H = !kSimple && docs >> j & 1 ? w[j] : fma2(a, H, w[j]);
                P = mul2(P, a);
            }
#pragma unroll
            for (int j = kTokens - 1; j >= 0; --j) {
                if (kSimple) {
                    Q = mul2(decay<kSmall>(q[j]), add2(fetch.read(in, 3, j, kept).get(), Q));
                } else if (t + j < p.T) {
                    Q = docs >> j & 1 ? both(0.f) : mul2(decay<kSmall>(q[j]), add2(fetch.read(in, 3, j, kept).get(), Q));
                }
            }
            P = !kSimple && docs ? both(0.f) : clamp(P);
        };
        int mode = !small ? kLargeTile : docs == 0 && t + kTokens <= p.T && c_tile + kTile <= p.C ? kSimpleTile : kDocumentTile;
        if (mode == kSimpleTile) make(Mode<kSimpleTile>{});
        else if (mode == kDocumentTile) make(Mode<kDocumentTile>{});
        else make(Mode<kLargeTile>{});
        if (__any_sync(0xffffffffu, live && !least.all_from(kLeast))) {
            mode = kExtremeTile;
            make(Mode<kExtremeTile>{});
        }
        shares[buf][warp][lane] = make_ulonglong2(P, Q);
        forward[buf][warp][lane] = H;
        const bool cuts = __syncthreads_or(docs != 0);
        f2 e = CLUSTER ? through_cluster<true>(cluster, K, rank, shares[buf], peers[buf], warp, lane, cuts, carry) : ends[buf ^ 1][lane];
        e = through_block<true>(shares[buf], warp, lane, cuts, e);
        if (cuts) {
            for (int i = 0; i < warp; ++i) h = step(shares[buf][i][lane].x, forward[buf][i][lane], h);
        } else {
#pragma unroll
            for (int i = 0; i < kWarps - 1; ++i) {
                if (i >= warp) break;
                h = fma2(shares[buf][i][lane].x, h, forward[buf][i][lane]);
            }
        }
        auto walk = [&](auto mode) {
            constexpr bool kSimple = decltype(mode)::value == kSimpleTile, kExtreme = decltype(mode)::value == kExtremeTile, kSmall = decltype(mode)::value <= kDocumentTile;
#pragma unroll
            for (int j = 0; j < kTokens; ++j) {
                const f2 before = h;
                h = !kSimple && docs >> j & 1 ? w[j] : fma2(decay<kSmall>(q[j]), h, w[j]);
                w[j] = before;
            }
            const i64 at = (i64)t * p.C;
            E *px = dx + at, *pgx = dgx + at, *pga = dga + at;
#pragma unroll
            for (int j = kTokens - 1; j >= 0; --j) {
                if (!kSimple && t + j >= p.T) continue;
                const bool doc = !kSimple && docs >> j & 1;
                const Gates<E, kExtreme> g(fetch.read(in, 2, j, kept).get(), fetch.read(in, 1, j, kept).get());
                const f2 vx = fetch.read(in, 0, j, kept).get(), a = decay<kSmall>(q[j]), G = add2(fetch.read(in, 3, j, kept).get(), e);
                const f2 beta = doc ? both(1.f) : mul2(square<kSmall>(q[j]), inv[j]);
                const f2 ox = mul2(mul2(G, beta), g.x), og = mul2(mul2(ox, vx), g.rest_x());
                e = mul2(a, G);
                const f2 slope = fma2(w[j], both(-1.f), mul2(mul2(mul2(g.x, vx), a), inv[j]));
                f2 dL = mul2(e, slope);
                if (doc) e = dL = both(0.f);
                const f2 oa = mul2(mul2(dL, mul2(s, g.a)), g.rest_a());
                ds = fma2(dL, g.a, ds);
                if (kSimple || live) {
                    put2<ROWS != kAnyRows>(rows_on(px, row_bytes, j), ox, second);
                    put2<ROWS != kAnyRows>(rows_on(pgx, row_bytes, j), og, second);
                    put2<ROWS != kAnyRows>(rows_on(pga, row_bytes, j), oa, second);
                }
            }
        };
        if (mode == kSimpleTile) walk(Mode<kSimpleTile>{});
        else if (mode == kDocumentTile) walk(Mode<kDocumentTile>{});
        else if (mode == kLargeTile) walk(Mode<kLargeTile>{});
        else walk(Mode<kExtremeTile>{});
        if (!CLUSTER && warp == 0) ends[buf][lane] = e;
        stage = stage == S - 1 ? 0 : stage + 1;
        __syncwarp();
    }
    // the warps' shares of ds, in their order
    __syncthreads();
    if (!CLUSTER) carry = ends[buf ^ 1][lane];
    if (p.dh0 != nullptr && rank == 0 && warp == 0 && live) {
        p.dh0[row] = lo(carry);
        if (second) p.dh0[row + 1] = hi(carry);
    }
    forward[0][warp][lane] = ds;
    __syncthreads();
    if (warp == 0 && live) {
        f2 sum = both(0.f);
#pragma unroll
        for (int q = 0; q < kWarps; ++q) sum = add2(sum, forward[0][q][lane]);
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

constexpr int kUpdateThreads = 128;
template <typename E, int V> struct alignas(sizeof(E) * V) Few { E e[V]; };

// V channels a thread (256 rows of 4096 channels: 6.5 us with four, 9.4 with one).  A chain of loads bounds it: the row's slot, then the
// slots of all rows beside the state.
template <typename E, int V>
__global__ void __launch_bounds__(kUpdateThreads) scan_update_kernel(int B, int C, int pool, const int* __restrict__ slots, float* state, const E* __restrict__ x,
                                                                     const E* __restrict__ gx, const E* __restrict__ ga, const float* __restrict__ s, E* y) {
    const int b = blockIdx.y, c = (blockIdx.x * kUpdateThreads + threadIdx.x) * V;
    const bool live = c < C;
    const int slot = slots != nullptr ? slots[b] : b;
    if (slot < 0) return;
    const bool found = slot < pool;
    // everything is asked for before it is known whether the row is the first of its slot
    using Row = Few<E, V>;
    using Wide = Few<float, V>;
    const i64 at = (i64)b * C + c;
    float* const home = state + (i64)slot * C + c;
    Row rx, rgx, rga;
    Wide h, sc;
    if (live && found) {
        rx = *reinterpret_cast<const Row*>(x + at);
        rgx = *reinterpret_cast<const Row*>(gx + at);
        rga = *reinterpret_cast<const Row*>(ga + at);
        sc = *reinterpret_cast<const Wide*>(s + c);
        h = *reinterpret_cast<const Wide*>(home);
    }
    bool before = false, later = false;
    if (slots != nullptr) {
        for (int q = threadIdx.x; q < B; q += kUpdateThreads) {
            const bool same = slots[q] == slot;
            before |= same && q < b;
            later |= same && q > b;
        }
        before = __syncthreads_or(before);
        later = __syncthreads_or(later);
    }
    if (!found) {
        if (live)
#pragma unroll
            for (int i = 0; i < V; ++i) y[at + i] = from_f<E>(__int_as_float(0x7fffffff));
        if (threadIdx.x == 0) atomicMax(&g_update_error, kBadSlot);
        return;
    }
    if (before || !live) return;
    for (int q = b;;) {
        Row out;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const Gates<E, true> g(both(to_f(rga.e[i])), both(to_f(rgx.e[i])));
            const f2 fallen = fall<E, false>(mul2(both(rate(sc.e[i])), g.a)), v = square<false>(fallen);
            h.e[i] = fmaf(lo(decay<false>(fallen)), h.e[i], lo(mul2(v, inverse_root<E>(v))) * (lo(g.x) * to_f(rx.e[i])));
            out.e[i] = from_f<E>(h.e[i]);
        }
        *reinterpret_cast<Row*>(y + (i64)q * C + c) = out;
        if (!later) break;
        do ++q;
        while (q < B && slots[q] != slot);
        if (q >= B) break;
        const i64 next = (i64)q * C + c;
        rx = *reinterpret_cast<const Row*>(x + next);
        rgx = *reinterpret_cast<const Row*>(gx + next);
        rga = *reinterpret_cast<const Row*>(ga + next);
    }
    *reinterpret_cast<Wide*>(home) = h;
}

bool aligned(std::initializer_list<const void*> ps, size_t bytes) {
    uintptr_t all = 0;
    for (const void* p : ps) all |= reinterpret_cast<uintptr_t>(p);
    return all % bytes == 0;
}

int check(const char* what, int dtype, int B, int T, int C) {
    RWKV_REQUIRE(dtype == RWKVB200_F32 || dtype == RWKVB200_BF16, RWKVB200_EINVAL, "%s: unknown dtype %d", what, dtype);
    RWKV_REQUIRE(B > 0 && T > 0 && C > 0, RWKVB200_EINVAL, "%s: B=%d T=%d C=%d must be positive", what, B, T, C);
    RWKV_REQUIRE(C <= 0x7fffffff - 65536, RWKVB200_EINVAL, "%s: C=%d is too wide", what, C);
    // (the scan counts the bytes of a row in 32 bits)
    RWKV_REQUIRE(T == 1 || (i64)C * (dtype == RWKVB200_BF16 ? 2 : 4) <= 0xffffffffll, RWKVB200_EINVAL, "%s: C=%d: rows of 4 GiB", what, C);
    RWKV_REQUIRE((i64)B * ((C + kTile - 1) / kTile) <= 0x7fffffff / kMaxCluster, RWKVB200_EINVAL, "%s: B=%d C=%d: too many blocks", what, B, C);
    RWKV_REQUIRE(T <= 0x7fffffff - 65536, RWKVB200_EINVAL, "%s: T=%d is too long", what, T);
    return RWKVB200_OK;
}

cudaLaunchAttribute cluster_of(int K) {
    cudaLaunchAttribute a;
    a.id = cudaLaunchAttributeClusterDimension;
    a.val.clusterDim.x = K;
    a.val.clusterDim.y = a.val.clusterDim.z = 1;
    return a;
}
// How many clusters of K blocks of a kernel the current device holds at once (a cluster does not go over the border of a group of SMs, and
// the groups differ in size).  Asked for once per device.
template <auto Kernel>
int clusters_at_once(int K, int smem) {
    static std::atomic<int> known[64][kMaxCluster + 1];   // + 1
    int dev = 0, n = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || allow_smem<Kernel>(smem) != cudaSuccess) return 0;
    if (dev < 64 && (n = known[dev][K].load(std::memory_order_relaxed)) > 0) return n - 1;
    cudaLaunchConfig_t config{};
    config.gridDim = dim3(K);
    config.blockDim = dim3(32 * kWarps);
    config.dynamicSmemBytes = smem;
    cudaLaunchAttribute cluster = cluster_of(K);
    config.attrs = &cluster;
    config.numAttrs = 1;
    if (cudaOccupancyMaxActiveClusters(&n, Kernel, &config) != cudaSuccess) {
        cudaGetLastError();
        return 0;
    }
    if (dev < 64) known[dev][K].store(n + 1, std::memory_order_relaxed);
    return n;
}
// How many blocks share a (sequence, channel tile): as many as are all there at once, one on every SM (the fp32 backward has that many) or two
// (where the kernel has two: it is asked for itself, as rows on any boundary take more shared memory): two side by side take
// 1.38 times the time of one.  B1 T8192 bf16, training step, K = 1 to 8: 20 tiles 454 / 316 / 222 / 166 / 141 / 123 / 151 / 130 us
// (6 are there one by one), 40 tiles 455 / 315 / 224 / 232 / 198 / 177 / 241 / 232 (of 7 not all at once), 60 tiles 452 / 318 / 311 /
// 244 / 310.
template <auto Kernel>
int cluster_size(int units, int rounds, int smem) {
    auto most = [&](auto at_once) {
        int K = kMaxCluster;
        while (K > 1 && (units > 2 * sm_count() / K || at_once(K) < units)) --K;
        return K;
    };
    int K = most([](int K) { return clusters_at_once<scan_backward_kernel<float, kWideRows, true>>(K, bwd_smem<float, kWideRows>()); });
    const int other = most([=](int K) { return clusters_at_once<Kernel>(K, smem); });
    if (other * 100 > K * 138) K = other;
    const int turns = (rounds + K - 1) / K;
    return (rounds + turns - 1) / turns;   // (no block without a round)
}

template <auto Kernel>
int launch(const char* what, const Args& p, int K, int smem, cudaStream_t st) {
    if (allow_smem<Kernel>(smem) != cudaSuccess) return check_launch(what);
    cudaLaunchConfig_t config{};
    config.gridDim = dim3((unsigned)(p.B * p.tiles * K));
    config.blockDim = dim3(32 * kWarps);
    config.dynamicSmemBytes = smem;
    config.stream = st;
    cudaLaunchAttribute cluster = cluster_of(K);
    config.attrs = &cluster;
    config.numAttrs = 1;
    cudaLaunchKernelEx(&config, Kernel, p);
    return check_launch(what);
}
template <typename E>
int rows_of(int C, std::initializer_list<const void*> ps) {
    if (C % (16 / sizeof(E)) == 0 && aligned(ps, 16)) return kWideRows;
    return C % 2 == 0 && aligned(ps, 2 * sizeof(E)) ? kPairRows : kAnyRows;
}
template <typename E, int ROWS>
int forward_cluster(int units, int rounds) { return cluster_size<scan_forward_kernel<E, ROWS, true>>(units, rounds, fwd_smem<E, ROWS>()); }
template <typename E, int ROWS>
int backward_cluster(int units, int rounds) { return cluster_size<scan_backward_kernel<E, ROWS, true>>(units, rounds, bwd_smem<E, ROWS>()); }
template <typename E, int ROWS>
int run_forward(const Args& p, cudaStream_t st) {
    const char* what = "gated_scan_forward";
    constexpr int smem = fwd_smem<E, ROWS>();
    const int K = forward_cluster<E, ROWS>(p.B * p.tiles, p.rounds);
    return K > 1 ? launch<scan_forward_kernel<E, ROWS, true>>(what, p, K, smem, st) : launch<scan_forward_kernel<E, ROWS, false>>(what, p, 1, smem, st);
}
template <typename E>
int run_forward(const Args& p, cudaStream_t st) {
    const int rows = rows_of<E>(p.C, {p.x, p.gx, p.ga, p.y});
    return rows == kWideRows ? run_forward<E, kWideRows>(p, st) : rows == kPairRows ? run_forward<E, kPairRows>(p, st) : run_forward<E, kAnyRows>(p, st);
}
// (leaves B K rows of ds in p.ds)
template <typename E, int ROWS>
int run_backward(const Args& p, int& K, cudaStream_t st) {
    const char* what = "gated_scan_backward";
    constexpr int smem = bwd_smem<E, ROWS>();
    K = backward_cluster<E, ROWS>(p.B * p.tiles, p.rounds);
    return K > 1 ? launch<scan_backward_kernel<E, ROWS, true>>(what, p, K, smem, st) : launch<scan_backward_kernel<E, ROWS, false>>(what, p, 1, smem, st);
}
template <typename E>
int run_backward(const Args& p, int& K, cudaStream_t st) {
    const int rows = rows_of<E>(p.C, {p.x, p.gx, p.ga, p.dy, p.dx, p.dgx, p.dga});
    return rows == kWideRows ? run_backward<E, kWideRows>(p, K, st) : rows == kPairRows ? run_backward<E, kPairRows>(p, K, st) : run_backward<E, kAnyRows>(p, K, st);
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
    return (size_t)B * (((size_t)T + kSaved - 1) / kSaved) * C * sizeof(float);
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
    p.B = B; p.T = T; p.C = C; p.tiles = (C + kTile - 1) / kTile; p.saves = (T + kSaved - 1) / kSaved; const int round = kWarps * (dtype == RWKVB200_BF16 ? kFwdTokens<bf16> : kFwdTokens<float>);
    p.rounds = (T + round - 1) / round;
    p.h0 = h0; p.x = x; p.gx = gx; p.ga = ga; p.s = s; p.first = first; p.y = y; p.hT = hT; p.saved = static_cast<float*>(saved);
    const cudaStream_t st = as_stream(stream);
    return dtype == RWKVB200_BF16 ? run_forward<bf16>(p, st) : run_forward<float>(p, st);
}

extern "C" int rwkvb200_gated_scan_backward(int dtype, int B, int T, int C, const void* x, const void* gx, const void* ga, const float* s,
                                            const unsigned char* first, const void* saved, const void* dy, const float* dhT, float* dh0, void* dx,
                                            void* dgx, void* dga, float* ds, void* work, void* stream) {
    if (int e = check("gated_scan_backward", dtype, B, T, C)) return e;
    RWKV_NOTNULL(x); RWKV_NOTNULL(gx); RWKV_NOTNULL(ga); RWKV_NOTNULL(s); RWKV_NOTNULL(saved); RWKV_NOTNULL(dy);
    RWKV_NOTNULL(dx); RWKV_NOTNULL(dgx); RWKV_NOTNULL(dga); RWKV_NOTNULL(ds); RWKV_NOTNULL(work);
    Args p{};
    p.B = B; p.T = T; p.C = C; p.tiles = (C + kTile - 1) / kTile; p.rounds = p.saves = (T + kSaved - 1) / kSaved;
    p.x = x; p.gx = gx; p.ga = ga; p.s = s; p.first = first; p.saved = static_cast<float*>(const_cast<void*>(saved));
    p.dy = dy; p.dhT = dhT; p.dh0 = dh0; p.dx = dx; p.dgx = dgx; p.dga = dga; p.ds = static_cast<float*>(work);
    const cudaStream_t st = as_stream(stream);
    int K = 1;
    const int rc = dtype == RWKVB200_BF16 ? run_backward<bf16>(p, K, st) : run_backward<float>(p, K, st);
    return rc != RWKVB200_OK ? rc : sum_rows(RWKVB200_F32, (i64)B * K, C, p.ds, ds, st);
}

extern "C" int rwkvb200_gated_scan_update(int dtype, int B, int C, int pool, float* state, const int* slots, const void* x, const void* gx,
                                          const void* ga, const float* s, void* y, void* stream) {
    if (int e = check("gated_scan_update", dtype, B, 1, C)) return e;
    RWKV_REQUIRE(pool > 0 && (slots != nullptr || pool >= B), RWKVB200_EINVAL, "gated_scan_update: %d states for %d rows", pool, B);
    RWKV_REQUIRE(B <= 65535, RWKVB200_EINVAL, "gated_scan_update: B=%d exceeds 65535", B);
    RWKV_NOTNULL(state); RWKV_NOTNULL(x); RWKV_NOTNULL(gx); RWKV_NOTNULL(ga); RWKV_NOTNULL(s); RWKV_NOTNULL(y);
    // four channels a thread where that leaves every SM a block and all rows start on their boundaries
    const bool wide = C % 4 == 0 && (i64)B * C >= 4ll * kUpdateThreads * sm_count() && aligned({state, x, gx, ga, s, y}, 16);
    const int per = wide ? 4 : 1;
    const dim3 grid((C + kUpdateThreads * per - 1) / (kUpdateThreads * per), B);
    const cudaStream_t st = as_stream(stream);
    auto run = [&](auto kernel, auto element) {
        using E = decltype(element);
        kernel<<<grid, kUpdateThreads, 0, st>>>(B, C, pool, slots, state, (const E*)x, (const E*)gx, (const E*)ga, s, (E*)y);
    };
    if (dtype == RWKVB200_BF16) {
        if (wide) run(scan_update_kernel<bf16, 4>, bf16()); else run(scan_update_kernel<bf16, 1>, bf16());
    } else {
        if (wide) run(scan_update_kernel<float, 4>, float()); else run(scan_update_kernel<float, 1>, float());
    }
    return check_launch("gated_scan_update");
}

extern "C" int rwkvb200_test_gated_scan_cluster(int dtype, int B, int T, int C, int rows, int backward, int* at_once) {
    const char* what = "test_gated_scan_cluster";
    if (int e = check(what, dtype, B, T, C)) return e;
    RWKV_REQUIRE(rows >= kWideRows && rows <= kAnyRows, RWKVB200_EINVAL, "%s: rows=%d", what, rows);
    RWKV_NOTNULL(at_once);
    const int units = B * ((C + kTile - 1) / kTile);
    auto ask = [&](auto element, auto mode) {
        using E = decltype(element);
        constexpr int ROWS = decltype(mode)::value, round = kWarps * kFwdTokens<E>;
        const int K = backward ? backward_cluster<E, ROWS>(units, (T + kSaved - 1) / kSaved) : forward_cluster<E, ROWS>(units, (T + round - 1) / round);
        *at_once = backward ? clusters_at_once<scan_backward_kernel<E, ROWS, true>>(K, bwd_smem<E, ROWS>())
                            : clusters_at_once<scan_forward_kernel<E, ROWS, true>>(K, fwd_smem<E, ROWS>());
        return K;
    };
    auto of = [&](auto element) { return rows == kWideRows ? ask(element, Mode<kWideRows>{}) : rows == kPairRows ? ask(element, Mode<kPairRows>{}) : ask(element, Mode<kAnyRows>{}); };
    return dtype == RWKVB200_BF16 ? of(bf16()) : of(0.f);
}
