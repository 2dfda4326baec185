// Gated linear recurrence, per channel c:
//
//   L_t = s_c sigmoid(ga_t)      a_t = exp(-L_t)      beta_t = sqrt(1 - a_t^2)      u_t = sigmoid(gx_t) x_t
//   h_t = a_t h_{t-1} + beta_t u_t                    y_t = h_t
//
// At the first token of a document a_t = 0 and beta_t = 1.  Gradients, with e_t = a_{t+1} G_{t+1} and e_{T-1} = dhT:
//
//   G_t = dy_t + e_t       dx = G beta sigmoid(gx)      dgx = G beta u (1 - sigmoid(gx))
//   dL = G (u a^2 / beta - a h_{t-1})                   dga = dL L (1 - sigmoid(ga))     ds = sum dL sigmoid(ga)     dh0 = e_{-1}
//
// (dL = 0 at a document's first token; where L = 0 the term through beta is taken as 0.)
//
// A block owns 32 lanes x VEC channels of one sequence and goes through it in rounds of kWarps x L tokens, a warp owns L of
// them: it makes the gates of its tokens in registers, reduces them to (P, H) (the product of the decays and the end state from
// a zero start), all warps fold those of the warps before theirs onto the block's state, and each walks its tokens once more
// from its own start state.  Every input is read once, y is written once.
#include "common.cuh"

namespace rwkvb200 {
namespace {

constexpr int kWarps = 8;
constexpr int kFwdTokens = 16;                    // per warp and round
constexpr int kBwdTokens = 8;
constexpr int kSaved = kWarps * kBwdTokens;       // the forward saves the state before every 64th token: a round of the backward

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

// Gates of one channel at one token.  For bf16 tensors by the hardware approximations (2e-7 relative: 2^-14 of a step of bf16),
// for fp32 by CUDA's functions.  1 - a^2 by its series where L is small: the difference would lose its digits there.  A square
// below the normal numbers counts as 0, and its root and inverse root are 0 (below 0, which only a negative s makes, NaN).
template <typename E> struct Gates;
template <> struct Gates<bf16> {
    static __device__ __forceinline__ float exp_minus(float x) { return ex2(-1.4426950408889634f * x); }
    static __device__ __forceinline__ float inverse(float x) { return rcp(x); }
    // 1 - exp(-2L): five terms leave z^5/720 = 7e-6 at z = 0.35
    static __device__ __forceinline__ float square(float L, float a) {
        const float z = 2.f * L;
        const float p = z * fmaf(-z, fmaf(-z, fmaf(-z, fmaf(-z, 1.f / 120.f, 1.f / 24.f), 1.f / 6.f), 0.5f), 1.f);
        return z < 0.35f ? p : fmaf(-a, a, 1.f);
    }
    static __device__ __forceinline__ float inverse_root(float v) { return fabsf(v) < 1.2e-38f ? 0.f : rsqrt_fast(v); }
    static __device__ __forceinline__ float root(float v) { return v * inverse_root(v); }
};
template <> struct Gates<float> {
    static __device__ __forceinline__ float exp_minus(float x) { return expf(-x); }
    static __device__ __forceinline__ float inverse(float x) { return 1.f / x; }
    static __device__ __forceinline__ float square(float L, float a) {   // eight terms: z^8/9! = 6e-10
        const float z = 2.f * L;
        float p = 1.f / 40320.f;
        p = fmaf(-z, p, 1.f / 5040.f);
        p = fmaf(-z, p, 1.f / 720.f);
        p = fmaf(-z, p, 1.f / 120.f);
        p = fmaf(-z, p, 1.f / 24.f);
        p = fmaf(-z, p, 1.f / 6.f);
        p = fmaf(-z, p, 0.5f);
        p = z * fmaf(-z, p, 1.f);
        return z < 0.35f ? p : fmaf(-a, a, 1.f);
    }
    static __device__ __forceinline__ float inverse_root(float v) { return fabsf(v) < 1.2e-38f ? 0.f : 1.f / sqrtf(v); }
    static __device__ __forceinline__ float root(float v) { return fabsf(v) < 1.2e-38f ? 0.f : sqrtf(v); }
};
template <typename E> __device__ __forceinline__ float sigmoid(float x) { return Gates<E>::inverse(1.f + Gates<E>::exp_minus(x)); }
// A sigmoid that keeps the digits of 1 - sigmoid(x) too: the smaller of the two, negative where that is 1 - sigmoid(x).
template <typename E> __device__ __forceinline__ float sigmoid_pair(float x) {
    const float q = Gates<E>::exp_minus(fabsf(x)), m = q * Gates<E>::inverse(1.f + q);
    return x > 0.f ? -m : m;
}
__device__ __forceinline__ float of_pair(float v) { return __float_as_int(v) < 0 ? 1.f + v : v; }
__device__ __forceinline__ float rest_of_pair(float v) { return __float_as_int(v) < 0 ? -v : 1.f - v; }

// VEC neighbouring channels of one token as they lie in memory
template <typename E, int VEC> struct Pack;
template <> struct Pack<bf16, 2> {
    uint32_t w;
    __device__ __forceinline__ float get(int i) const { return __uint_as_float(i ? w & 0xffff0000u : w << 16); }
    __device__ __forceinline__ void set(const float* v) {
        const __nv_bfloat162 t = __floats2bfloat162_rn(v[0], v[1]);
        w = *reinterpret_cast<const uint32_t*>(&t);
    }
};
template <> struct Pack<bf16, 1> {
    bf16 w;
    __device__ __forceinline__ float get(int) const { return __bfloat162float(w); }
    __device__ __forceinline__ void set(const float* v) { w = __float2bfloat16_rn(v[0]); }
};
template <> struct alignas(8) Pack<float, 2> {
    float2 w;
    __device__ __forceinline__ float get(int i) const { return i ? w.y : w.x; }
    __device__ __forceinline__ void set(const float* v) { w = make_float2(v[0], v[1]); }
};
template <> struct Pack<float, 1> {
    float w;
    __device__ __forceinline__ float get(int) const { return w; }
    __device__ __forceinline__ void set(const float* v) { w = v[0]; }
};
template <typename E, int VEC>
__device__ __forceinline__ Pack<E, VEC> load(const E* p) { return *reinterpret_cast<const Pack<E, VEC>*>(p); }
template <typename E, int VEC>
__device__ __forceinline__ Pack<E, VEC> zero() {
    Pack<E, VEC> z;
    const float v[2] = {0.f, 0.f};
    z.set(v);
    return z;
}

struct Args {
    int T, C, tiles, rounds_saved;
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

// A warp's share of a round reduced to one step: h -> P h + H, or H alone where a document begins in it (whatever h is: one
// document's infinities do not reach the next).  A product that underflows must not make an infinite state NaN.
__device__ __forceinline__ float fold(bool cut, float P, float H, float h) { return cut ? H : fmaf(fmaxf(P, 1e-45f), h, H); }

template <typename E, int VEC>
__global__ void __launch_bounds__(32 * kWarps) scan_forward_kernel(const Args p) {
    constexpr int L = kFwdTokens;
    __shared__ float sP[2][kWarps][32 * VEC], sH[2][kWarps][32 * VEC];
    __shared__ int sCut[2][kWarps];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int b = blockIdx.x / p.tiles, c0 = (blockIdx.x % p.tiles) * 32 * VEC + lane * VEC;
    const bool live = c0 < p.C;
    const i64 base = (i64)b * p.T * p.C + c0;
    const E *x = static_cast<const E*>(p.x) + base, *gx = static_cast<const E*>(p.gx) + base, *ga = static_cast<const E*>(p.ga) + base;
    E* y = static_cast<E*>(p.y) + base;
    const uint8_t* first = p.first ? p.first + (i64)b * p.T : nullptr;
    float s[VEC], carry[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
        s[i] = live ? p.s[c0 + i] : 0.f;
        carry[i] = live && p.h0 ? p.h0[(i64)b * p.C + c0 + i] : 0.f;
    }
    for (int t0 = 0, buf = 0; t0 < p.T; t0 += kWarps * L, buf ^= 1) {
        const int t = t0 + warp * L;
        const uint32_t docs = firsts<L>(first, t, p.T, lane);
        Pack<E, VEC> px[L], pgx[L], pga[L];
#pragma unroll
        for (int j = 0; j < L; ++j) {
            const bool in = live && t + j < p.T;
            const i64 at = (i64)(t + j) * p.C;
            px[j] = in ? load<E, VEC>(x + at) : zero<E, VEC>();
            pgx[j] = in ? load<E, VEC>(gx + at) : zero<E, VEC>();
            pga[j] = in ? load<E, VEC>(ga + at) : zero<E, VEC>();
        }
        float a[L][VEC], w[L][VEC], P[VEC], H[VEC];
#pragma unroll
        for (int i = 0; i < VEC; ++i) P[i] = 1.f, H[i] = 0.f;
#pragma unroll
        for (int j = 0; j < L; ++j) {
            const bool doc = docs >> j & 1, past = t + j >= p.T;
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                const float len = s[i] * sigmoid<E>(pga[j].get(i));
                const float d = Gates<E>::exp_minus(len), beta = doc ? 1.f : Gates<E>::root(Gates<E>::square(len, d));
                a[j][i] = past ? 1.f : d;
                w[j][i] = past ? 0.f : beta * (sigmoid<E>(pgx[j].get(i)) * px[j].get(i));
                H[i] = doc ? w[j][i] : fmaf(a[j][i], H[i], w[j][i]);
                P[i] *= a[j][i];
            }
        }
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            sP[buf][warp][lane * VEC + i] = P[i];
            sH[buf][warp][lane * VEC + i] = H[i];
        }
        if (lane == 0) sCut[buf][warp] = docs != 0;
        __syncthreads();   // (a buffer is written again two rounds on, behind the next round's barrier)
        float h[VEC];
#pragma unroll
        for (int q = 0; q < kWarps; ++q) {
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                if (q == warp) h[i] = carry[i];
                carry[i] = fold(sCut[buf][q], sP[buf][q][lane * VEC + i], sH[buf][q][lane * VEC + i], carry[i]);
            }
        }
        if (!live) continue;
        if (p.saved != nullptr && t % kSaved == 0 && t < p.T) {
#pragma unroll
            for (int i = 0; i < VEC; ++i) p.saved[((i64)b * p.rounds_saved + t / kSaved) * p.C + c0 + i] = h[i];
        }
#pragma unroll
        for (int j = 0; j < L; ++j) {
            if (t + j >= p.T) break;
#pragma unroll
            for (int i = 0; i < VEC; ++i) h[i] = docs >> j & 1 ? w[j][i] : fmaf(a[j][i], h[i], w[j][i]);
            Pack<E, VEC> o;
            o.set(h);
            *reinterpret_cast<Pack<E, VEC>*>(y + (i64)(t + j) * p.C) = o;
        }
    }
    if (p.hT != nullptr && warp == 0 && live) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) p.hT[(i64)b * p.C + c0 + i] = carry[i];
    }
}

// Rounds from the last to the first; e (the gradient that comes into a token from the later ones) goes the same way as h does in
// the forward, with the same products of decays.  h before each token is made again from the saved states.
template <typename E, int VEC>
__global__ void __launch_bounds__(32 * kWarps) scan_backward_kernel(const Args p) {
    constexpr int L = kBwdTokens;
    __shared__ float sP[2][kWarps][32 * VEC], sH[2][kWarps][32 * VEC], sQ[2][kWarps][32 * VEC];
    __shared__ int sCut[2][kWarps];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int b = blockIdx.x / p.tiles, c0 = (blockIdx.x % p.tiles) * 32 * VEC + lane * VEC;
    const bool live = c0 < p.C;
    const i64 base = (i64)b * p.T * p.C + c0;
    const E *x = static_cast<const E*>(p.x) + base, *gx = static_cast<const E*>(p.gx) + base, *ga = static_cast<const E*>(p.ga) + base,
            *dy = static_cast<const E*>(p.dy) + base;
    E *dx = static_cast<E*>(p.dx) + base, *dgx = static_cast<E*>(p.dgx) + base, *dga = static_cast<E*>(p.dga) + base;
    const uint8_t* first = p.first ? p.first + (i64)b * p.T : nullptr;
    float s[VEC], carry[VEC], ds[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
        s[i] = live ? p.s[c0 + i] : 0.f;
        carry[i] = live && p.dhT ? p.dhT[(i64)b * p.C + c0 + i] : 0.f;
        ds[i] = 0.f;
    }
    int buf = 0;
    for (int round = p.rounds_saved - 1; round >= 0; --round, buf ^= 1) {
        const int t = round * kSaved + warp * L;
        const uint32_t docs = firsts<L>(first, t, p.T, lane);
        Pack<E, VEC> px[L], pdy[L];
        float r[L][VEC], g[L][VEC], a[L][VEC], P[VEC], H[VEC], Q[VEC], hs[VEC], e[VEC];
        {
            Pack<E, VEC> pgx[L], pga[L];
#pragma unroll
            for (int j = 0; j < L; ++j) {
                const bool in = live && t + j < p.T;
                const i64 at = (i64)(t + j) * p.C;
                px[j] = in ? load<E, VEC>(x + at) : zero<E, VEC>();
                pgx[j] = in ? load<E, VEC>(gx + at) : zero<E, VEC>();
                pga[j] = in ? load<E, VEC>(ga + at) : zero<E, VEC>();
                pdy[j] = in ? load<E, VEC>(dy + at) : zero<E, VEC>();
            }
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                P[i] = 1.f, H[i] = 0.f, Q[i] = 0.f;
                hs[i] = live ? p.saved[((i64)b * p.rounds_saved + round) * p.C + c0 + i] : 0.f;
            }
#pragma unroll
            for (int j = 0; j < L; ++j) {
                const bool doc = docs >> j & 1, past = t + j >= p.T;
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    r[j][i] = sigmoid_pair<E>(pga[j].get(i));
                    g[j][i] = sigmoid_pair<E>(pgx[j].get(i));
                    const float len = s[i] * of_pair(r[j][i]), d = Gates<E>::exp_minus(len);
                    const float w = (doc ? 1.f : Gates<E>::root(Gates<E>::square(len, d))) * (of_pair(g[j][i]) * px[j].get(i));
                    a[j][i] = past ? 1.f : d;
                    H[i] = doc ? w : fmaf(a[j][i], H[i], past ? 0.f : w);
                    P[i] *= a[j][i];
                }
            }
        }
#pragma unroll
        for (int j = L - 1; j >= 0; --j)
#pragma unroll
            for (int i = 0; i < VEC; ++i) Q[i] = docs >> j & 1 ? 0.f : a[j][i] * (pdy[j].get(i) + Q[i]);
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            sP[buf][warp][lane * VEC + i] = P[i];
            sH[buf][warp][lane * VEC + i] = H[i];
            sQ[buf][warp][lane * VEC + i] = Q[i];
        }
        if (lane == 0) sCut[buf][warp] = docs != 0;
        __syncthreads();
#pragma unroll
        for (int q = 0; q < kWarps; ++q) {
            if (q < warp) {
#pragma unroll
                for (int i = 0; i < VEC; ++i) hs[i] = fold(sCut[buf][q], sP[buf][q][lane * VEC + i], sH[buf][q][lane * VEC + i], hs[i]);
            }
        }
#pragma unroll
        for (int q = kWarps - 1; q >= 0; --q) {
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                if (q == warp) e[i] = carry[i];
                carry[i] = fold(sCut[buf][q], sP[buf][q][lane * VEC + i], sQ[buf][q][lane * VEC + i], carry[i]);
            }
        }
        if (!live) continue;
        float before[L][VEC];
#pragma unroll
        for (int j = 0; j < L; ++j) {
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                before[j][i] = hs[i];
                const bool doc = docs >> j & 1;
                const float w = (doc ? 1.f : Gates<E>::root(Gates<E>::square(s[i] * of_pair(r[j][i]), a[j][i]))) * (of_pair(g[j][i]) * px[j].get(i));
                hs[i] = doc ? w : fmaf(a[j][i], hs[i], w);
            }
        }
#pragma unroll
        for (int j = L - 1; j >= 0; --j) {
            if (t + j >= p.T) continue;
            const bool doc = docs >> j & 1;
            float ox[VEC], og[VEC], oa[VEC];
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                const float sr = of_pair(r[j][i]), sg = of_pair(g[j][i]), len = s[i] * sr, v = Gates<E>::square(len, a[j][i]);
                const float G = pdy[j].get(i) + e[i], u = sg * px[j].get(i), beta = doc ? 1.f : Gates<E>::root(v);
                ox[i] = G * beta * sg;
                og[i] = G * beta * u * rest_of_pair(g[j][i]);
                const float dlen = doc ? 0.f : G * (u * (a[j][i] * a[j][i]) * Gates<E>::inverse_root(v) - a[j][i] * before[j][i]);
                oa[i] = dlen * len * rest_of_pair(r[j][i]);
                ds[i] += dlen * sr;
                e[i] = doc ? 0.f : a[j][i] * G;
            }
            Pack<E, VEC> o;
            const i64 at = (i64)(t + j) * p.C;
            o.set(ox);
            *reinterpret_cast<Pack<E, VEC>*>(dx + at) = o;
            o.set(og);
            *reinterpret_cast<Pack<E, VEC>*>(dgx + at) = o;
            o.set(oa);
            *reinterpret_cast<Pack<E, VEC>*>(dga + at) = o;
        }
    }
    if (p.dh0 != nullptr && warp == 0 && live) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) p.dh0[(i64)b * p.C + c0 + i] = carry[i];
    }
    // the warps' shares of ds, in their order
    __syncthreads();
#pragma unroll
    for (int i = 0; i < VEC; ++i) sP[0][warp][lane * VEC + i] = ds[i];
    __syncthreads();
    if (warp == 0 && live) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            float sum = 0.f;
#pragma unroll
            for (int q = 0; q < kWarps; ++q) sum += sP[0][q][lane * VEC + i];
            p.ds[(i64)b * p.C + c0 + i] = sum;
        }
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
            const float len = sc * sigmoid<E>(to_f(ga[i])), a = Gates<E>::exp_minus(len);
            h = fmaf(a, h, Gates<E>::root(Gates<E>::square(len, a)) * (sigmoid<E>(to_f(gx[i])) * to_f(x[i])));
            y[i] = from_f<E>(h);
        }
        if (!later) break;
    }
    *at = h;
}

bool aligned(const void* p, int n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

// Two channels a thread where a pair can be read as one word: C even and pointers aligned to it.
bool pairs(const Args& p, int element) {
    const int n = 2 * element;
    return p.C % 2 == 0 && aligned(p.x, n) && aligned(p.gx, n) && aligned(p.ga, n) && aligned(p.y, n) && aligned(p.dy, n) && aligned(p.dx, n) &&
           aligned(p.dgx, n) && aligned(p.dga, n);
}

int check(const char* what, int dtype, int B, int T, int C) {
    RWKV_REQUIRE(dtype == RWKVB200_F32 || dtype == RWKVB200_BF16, RWKVB200_EINVAL, "%s: unknown dtype %d", what, dtype);
    RWKV_REQUIRE(B > 0 && T > 0 && C > 0, RWKVB200_EINVAL, "%s: B=%d T=%d C=%d must be positive", what, B, T, C);
    RWKV_REQUIRE((i64)B * ((C + 31) / 32) <= 0x7fffffff, RWKVB200_EINVAL, "%s: B=%d C=%d: too many blocks", what, B, C);
    RWKV_REQUIRE(T <= 0x7fffffff - 1024, RWKVB200_EINVAL, "%s: T=%d is too long", what, T);
    return RWKVB200_OK;
}

template <typename E, int VEC>
int run_forward(Args& p, int B, cudaStream_t st) {
    p.tiles = (p.C + 32 * VEC - 1) / (32 * VEC);
    scan_forward_kernel<E, VEC><<<(unsigned)(B * p.tiles), 32 * kWarps, 0, st>>>(p);
    return check_launch("gated_scan_forward");
}
template <typename E, int VEC>
int run_backward(Args& p, int B, cudaStream_t st) {
    p.tiles = (p.C + 32 * VEC - 1) / (32 * VEC);
    scan_backward_kernel<E, VEC><<<(unsigned)(B * p.tiles), 32 * kWarps, 0, st>>>(p);
    return check_launch("gated_scan_backward");
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
    return (size_t)B * ((T + kSaved - 1) / kSaved) * C * sizeof(float);
}
extern "C" size_t rwkvb200_gated_scan_work_bytes(int B, int T, int C) {
    if (B <= 0 || T <= 0 || C <= 0) return 0;
    return (size_t)B * C * sizeof(float);
}

extern "C" int rwkvb200_gated_scan_forward(int dtype, int B, int T, int C, const float* h0, const void* x, const void* gx, const void* ga,
                                           const float* s, const unsigned char* first, void* y, float* hT, void* saved, void* stream) {
    if (int e = check("gated_scan_forward", dtype, B, T, C)) return e;
    RWKV_NOTNULL(x); RWKV_NOTNULL(gx); RWKV_NOTNULL(ga); RWKV_NOTNULL(s); RWKV_NOTNULL(y);
    Args p{};
    p.T = T; p.C = C; p.rounds_saved = (T + kSaved - 1) / kSaved;
    p.h0 = h0; p.x = x; p.gx = gx; p.ga = ga; p.s = s; p.first = first; p.y = y; p.hT = hT; p.saved = static_cast<float*>(saved);
    const cudaStream_t st = as_stream(stream);
    if (dtype == RWKVB200_BF16) return pairs(p, 2) ? run_forward<bf16, 2>(p, B, st) : run_forward<bf16, 1>(p, B, st);
    return pairs(p, 4) ? run_forward<float, 2>(p, B, st) : run_forward<float, 1>(p, B, st);
}

extern "C" int rwkvb200_gated_scan_backward(int dtype, int B, int T, int C, const void* x, const void* gx, const void* ga, const float* s,
                                            const unsigned char* first, const void* saved, const void* dy, const float* dhT, float* dh0, void* dx,
                                            void* dgx, void* dga, float* ds, void* work, void* stream) {
    if (int e = check("gated_scan_backward", dtype, B, T, C)) return e;
    RWKV_NOTNULL(x); RWKV_NOTNULL(gx); RWKV_NOTNULL(ga); RWKV_NOTNULL(s); RWKV_NOTNULL(saved); RWKV_NOTNULL(dy);
    RWKV_NOTNULL(dx); RWKV_NOTNULL(dgx); RWKV_NOTNULL(dga); RWKV_NOTNULL(ds); RWKV_NOTNULL(work);
    Args p{};
    p.T = T; p.C = C; p.rounds_saved = (T + kSaved - 1) / kSaved;
    p.x = x; p.gx = gx; p.ga = ga; p.s = s; p.first = first; p.saved = static_cast<float*>(const_cast<void*>(saved));
    p.dy = dy; p.dhT = dhT; p.dh0 = dh0; p.dx = dx; p.dgx = dgx; p.dga = dga; p.ds = static_cast<float*>(work);
    const cudaStream_t st = as_stream(stream);
    int rc;
    if (dtype == RWKVB200_BF16) rc = pairs(p, 2) ? run_backward<bf16, 2>(p, B, st) : run_backward<bf16, 1>(p, B, st);
    else rc = pairs(p, 4) ? run_backward<float, 2>(p, B, st) : run_backward<float, 1>(p, B, st);
    if (rc != RWKVB200_OK) return rc;
    return sum_rows(RWKVB200_F32, B, C, p.ds, ds, st);
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
