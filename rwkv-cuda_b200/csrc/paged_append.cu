// New tokens go into a paged cache: k and q are rotated by the token's position, k and v are written into its page.
//
//   angle_j = position * inv_freq_j      (a, b) -> (a cos - b sin, a sin + b cos)      j < R/2
//
// with (a, b) the elements (j, j + R/2) of a head or, interleaved, (2j, 2j + 1); cos and sin are multiplied by `factor` and
// elements from R on are left alone.  The angle is taken in fp64 and reduced to one turn before it is rounded: position 10^6 in
// fp32 would leave it 0.06 off.
//
// A token's R/2 cosines and sines are made once for all heads, by the team of threads that does the token: a block where there are few
// tokens, so that the loads run beside the chain behind a place (the sequence, its length, the page), else a warp, so that
// many such chains run side by side.  A thread has the same part of every head it does (an item): it takes its cosines and
// sines into registers once.  Memory bounds it for many tokens, the chain for few.  (Tried: items found by divisions, 185
// instructions a vector; a block for four tokens one after the other.  9216 tokens of 96 heads took 97 and 70 us.)
#include "paged.cuh"

namespace rwkvb200 {
namespace {

__device__ int g_error = 0;
constexpr int kThreads = 256;

struct AppendArgs {
    int M, B, Hq, Hkv, N, R, pages, width, interleaved;
    float factor;
    Divisor page;
    const void *q, *k, *v;
    void *q_out, *k_pages, *v_pages;
    const int *table, *lengths, *cu;
    const float* inv_freq;
};

// VEC elements as they lie in memory
template <typename E, int VEC> struct alignas(sizeof(E) * VEC) Vec {
    E w[VEC];
    __device__ __forceinline__ void get(float (&f)[VEC]) const {
#pragma unroll
        for (int i = 0; i < VEC; ++i) f[i] = to_f(w[i]);
    }
    __device__ __forceinline__ void set(const float (&f)[VEC]) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) w[i] = from_f<E>(f[i]);
    }
};
template <> struct Vec<bf16, 8> {
    uint4 w;
    __device__ __forceinline__ void get(float (&f)[8]) const {
        const uint32_t v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) f[2 * i] = __uint_as_float(v[i] << 16), f[2 * i + 1] = __uint_as_float(v[i] & 0xffff0000u);
    }
    __device__ __forceinline__ void set(const float (&f)[8]) {
        uint32_t v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const __nv_bfloat162 t = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
            v[i] = *reinterpret_cast<const uint32_t*>(&t);
        }
        w = make_uint4(v[0], v[1], v[2], v[3]);
    }
};
template <> struct Vec<float, 4> {
    float4 w;
    __device__ __forceinline__ void get(float (&f)[4]) const { f[0] = w.x, f[1] = w.y, f[2] = w.z, f[3] = w.w; }
    __device__ __forceinline__ void set(const float (&f)[4]) { w = make_float4(f[0], f[1], f[2], f[3]); }
};

// Items of a head of q or k: first the rotated ones: a vector x of the first half and z of the second (half layout), a vector of pairs
// (interleaved), or (interleaved, VEC = 1) a pair's two elements; then the vectors behind R.
template <typename E, int VEC, int TEAM>
__global__ void __launch_bounds__(kThreads) append_kernel(const AppendArgs p) {
    using V = Vec<E, VEC>;
    constexpr bool kBlock = TEAM == kThreads;
    constexpr int kAtOnce = kBlock && VEC > 1 ? 1 : 4;   // heads that a thread has in hand
    __shared__ float cosine[kThreads / TEAM][RWKVB200_MAX_HEAD_SIZE / 2], sine[kThreads / TEAM][RWKVB200_MAX_HEAD_SIZE / 2];
    const int team = threadIdx.x / TEAM, thread = threadIdx.x % TEAM, m = blockIdx.x * (kThreads / TEAM) + team, half = p.R / 2;
    if (m >= p.M) return;   // (a warp of its own: a block's token always is)
    const bool pairs = VEC > 1 && p.interleaved;   // in one vector
    const int rotated = pairs ? p.R / VEC : half / VEC, items = rotated + (p.N - p.R) / VEC, pieces = p.N / VEC;
    const int groups = TEAM / items, group = thread / items, item = thread % items;   // heads at a time
    const int v_groups = TEAM / pieces, v_group = thread / pieces, v_at = thread % pieces * VEC;
    const bool turns = item < rotated, working = group < groups, v_working = v_group < v_groups;
    const int x_at = !turns ? p.R + (item - rotated) * VEC : p.interleaved && !pairs ? 2 * item : item * VEC;
    const int z_at = p.interleaved ? x_at + 1 : half + x_at;
    const bool two = turns && !pairs;
    const int Hq = p.q != nullptr ? p.Hq : 0;
    struct Two {
        V x, z;
    };
    auto load = [&](const void* tensor, int H, int h, Two& i) {
        const E* from = static_cast<const E*>(tensor) + ((i64)m * H + h) * p.N;
        i.x = *reinterpret_cast<const V*>(from + x_at);
        if (two) i.z = *reinterpret_cast<const V*>(from + z_at);
    };
    auto load_v = [&](int h, V& v) { v = *reinterpret_cast<const V*>(static_cast<const E*>(p.v) + ((i64)m * p.Hkv + h) * p.N + v_at); };
    Two q, k;
    V v;
    if (kBlock) {
        if (working && group < Hq) load(p.q, Hq, group, q);
        if (working && group < p.Hkv) load(p.k, p.Hkv, group, k);
        if (v_working && v_group < p.Hkv) load_v(v_group, v);
    }
    int b = m;
    i64 nth = 0;
    if (p.cu != nullptr) {
        int lo = 0, hi = p.B;   // the last b with cu[b] <= m
        while (hi - lo > 1) {
            const int mid = (lo + hi) / 2;
            if (p.cu[mid] <= m) lo = mid; else hi = mid;
        }
        b = lo;
        nth = (i64)m - p.cu[b];
        if (nth < 0 || m >= p.cu[p.B]) return;   // a row that belongs to no sequence
    }
    const int before = p.lengths[b];
    if (before < 0) return;                      // a row that only pads the batch
    const i64 position = before + nth;
    const bool in_table = position < (i64)p.width * p.page.d;
    const uint32_t col = in_table ? p.page.quotient((uint32_t)position) : 0;
    const int id = in_table ? p.table[(i64)b * p.width + col] : -1;
    for (int j = thread; j < half; j += TEAM) {
        const double whole = (double)position * (double)p.inv_freq[j] * 0.15915494309189533577;   // angle / 2 pi
        float s, c;
        sincospif(2.f * (float)(whole - rint(whole)), &s, &c);
        cosine[team][j] = c * p.factor;
        sine[team][j] = s * p.factor;
    }
    // the rows of the first head that the token goes to; -1: nowhere
    i64 place = -1;
    if (id >= 0 && id < p.pages) place = (i64)id * p.Hkv * p.page.d + ((uint32_t)position - col * p.page.d);
    else if (thread == 0) atomicMax(&g_error, in_table ? kBadPage : kBadLength);
    if (kBlock) __syncthreads(); else __syncwarp();
    // the pair that element e belongs to: item * VEC + e, or number e / 2 of the vector's
    float c[VEC], s[VEC];
    if (turns) {
        const int first = pairs ? item * VEC / 2 : item * VEC;
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            const int j = first + (pairs ? e / 2 : e);
            c[e] = cosine[team][j], s[e] = sine[team][j];
        }
    }
    auto turn = [&](Two& i) {
        float a[VEC], b[VEC];
        i.x.get(a);
        if (pairs) {
#pragma unroll
            for (int e = 0; e < VEC; e += 2) {
                const float x = a[e], y = a[(e + 1) % VEC];
                a[e] = x * c[e] - y * s[e];
                a[(e + 1) % VEC] = x * s[e] + y * c[e];
            }
        } else {
            i.z.get(b);
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const float x = a[e], y = b[e];
                a[e] = x * c[e] - y * s[e];
                b[e] = x * s[e] + y * c[e];
            }
            i.z.set(b);
        }
        i.x.set(a);
    };
    // heads from `from` (a head of it every `stride` elements) to `to`; the first of them may be in hand
    auto heads = [&](const void* from, int H, E* to, i64 stride, Two& first) {
        for (int h0 = group; h0 < H; h0 += groups * kAtOnce) {
            Two i[kAtOnce];
#pragma unroll
            for (int u = 0; u < kAtOnce; ++u) {
                const int h = h0 + u * groups;
                if (kBlock && u == 0 && h0 == group) i[u] = first;
                else if (h < H) load(from, H, h, i[u]);
            }
#pragma unroll
            for (int u = 0; u < kAtOnce; ++u) {
                const int h = h0 + u * groups;
                if (h >= H) break;
                if (turns) turn(i[u]);
                *reinterpret_cast<V*>(to + h * stride + x_at) = i[u].x;
                if (two) *reinterpret_cast<V*>(to + h * stride + z_at) = i[u].z;
            }
        }
    };
    if (working) heads(p.q, Hq, static_cast<E*>(p.q_out) + (i64)m * Hq * p.N, p.N, q);
    if (place < 0) return;
    const i64 stride = (i64)p.page.d * p.N;
    if (working) heads(p.k, p.Hkv, static_cast<E*>(p.k_pages) + place * p.N, stride, k);
    if (v_working) {
        E* to = static_cast<E*>(p.v_pages) + place * p.N + v_at;
        for (int h0 = v_group; h0 < p.Hkv; h0 += v_groups * kAtOnce) {
            V i[kAtOnce];
#pragma unroll
            for (int u = 0; u < kAtOnce; ++u) {
                const int h = h0 + u * v_groups;
                if (kBlock && u == 0 && h0 == v_group) i[u] = v;
                else if (h < p.Hkv) load_v(h, i[u]);
            }
#pragma unroll
            for (int u = 0; u < kAtOnce; ++u) {
                const int h = h0 + u * v_groups;
                if (h < p.Hkv) *reinterpret_cast<V*>(to + h * stride) = i[u];
            }
        }
    }
}

template <typename E, int VEC>
void launch(const AppendArgs& p, cudaStream_t st) {
    // a warp a token where that gives every SM sixteen of them, and a head's items are no more than its lanes
    if (p.M >= 16 * sm_count() && p.N / VEC <= 32) {
        constexpr int kPerBlock = kThreads / 32;
        append_kernel<E, VEC, 32><<<((unsigned)p.M + kPerBlock - 1) / kPerBlock, kThreads, 0, st>>>(p);
    } else {
        append_kernel<E, VEC, kThreads><<<p.M, kThreads, 0, st>>>(p);
    }
}
template <typename E>
int launch(const AppendArgs& p, cudaStream_t st) {
    // The widest vectors, up to 16 bytes, of which heads and the rotated part (a half of it in the half layout) are whole numbers and on whose
    // boundaries all tensors begin.  (5000 tokens of 48 heads of 80 with 40 rotated elements, by elements and by four: 65 and 40 us.)
    uintptr_t bytes = 0;
    for (const void* x : {p.q, p.k, p.v, (const void*)p.q_out, (const void*)p.k_pages, (const void*)p.v_pages}) bytes |= reinterpret_cast<uintptr_t>(x);
    const int elements = p.N | (p.interleaved ? p.R : p.R / 2);
    auto fits = [&](int vec) { return elements % vec == 0 && bytes % (vec * sizeof(E)) == 0; };
    if (sizeof(E) == 2 && fits(8)) launch<E, 16 / sizeof(E)>(p, st);
    else if (fits(4)) launch<E, 4>(p, st);
    else if (fits(2)) launch<E, 2>(p, st);
    else launch<E, 1>(p, st);
    return check_launch("paged_append");
}

}  // namespace

int paged_append_error(int clear) {
    int v = 0;
    if (clear) return cudaMemcpyToSymbol(g_error, &v, sizeof(v)) == cudaSuccess ? 0 : -1;
    return cudaMemcpyFromSymbol(&v, g_error, sizeof(v)) == cudaSuccess ? v : -1;
}

}  // namespace rwkvb200

using namespace rwkvb200;

extern "C" int rwkvb200_paged_append(int dtype, int M, int B, int Hq, int Hkv, int N, int R, int pages, int page, int width, const void* q,
                                     const void* k, const void* v, void* q_out, void* k_pages, void* v_pages, const int* table, const int* lengths,
                                     const int* cu_seqlens, const float* inv_freq, int interleaved, float factor, void* stream) {
    const char* what = "paged_append";
    RWKV_REQUIRE(dtype == RWKVB200_F32 || dtype == RWKVB200_BF16, RWKVB200_EINVAL, "%s: unknown dtype %d", what, dtype);
    RWKV_REQUIRE(M > 0 && B > 0 && Hkv > 0 && N > 0 && pages > 0 && page > 0 && width > 0, RWKVB200_EINVAL,
                 "%s: M=%d B=%d Hkv=%d N=%d pages=%d page=%d width=%d must be positive", what, M, B, Hkv, N, pages, page, width);
    RWKV_REQUIRE(N <= RWKVB200_MAX_HEAD_SIZE, RWKVB200_EUNSUPPORTED, "%s: head size %d > %d", what, N, RWKVB200_MAX_HEAD_SIZE);
    RWKV_REQUIRE((i64)width * page <= 0x7fffffff, RWKVB200_EINVAL, "%s: %d pages of %d tokens are more than 2^31 - 1", what, width, page);
    RWKV_REQUIRE(R >= 0 && R % 2 == 0 && R <= N, RWKVB200_EINVAL, "%s: %d rotated elements of %d", what, R, N);
    RWKV_REQUIRE(q == nullptr || Hq > 0, RWKVB200_EINVAL, "%s: Hq=%d must be positive", what, Hq);
    RWKV_REQUIRE((i64)(Hq > 0 ? Hq : 0) * N + 2ll * Hkv * N <= 0xfffffff, RWKVB200_EINVAL, "%s: Hq=%d Hkv=%d are too many heads", what, Hq, Hkv);
    RWKV_REQUIRE(cu_seqlens != nullptr || M == B, RWKVB200_EINVAL, "%s: %d tokens for %d sequences need cu_seqlens", what, M, B);
    RWKV_NOTNULL(k); RWKV_NOTNULL(v); RWKV_NOTNULL(k_pages); RWKV_NOTNULL(v_pages); RWKV_NOTNULL(table); RWKV_NOTNULL(lengths);
    RWKV_REQUIRE((q == nullptr) == (q_out == nullptr), RWKVB200_EINVAL, "%s: q and q_out come together", what);
    if (R > 0) RWKV_NOTNULL(inv_freq);
    const AppendArgs p{M, B, Hq, Hkv, N, R, pages, width, interleaved, factor, Divisor((uint32_t)page), q, k, v, q_out, k_pages, v_pages, table, lengths, cu_seqlens, inv_freq};
    return dtype == RWKVB200_BF16 ? launch<bf16>(p, as_stream(stream)) : launch<float>(p, as_stream(stream));
}
