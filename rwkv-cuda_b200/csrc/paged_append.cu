// New tokens go into a paged cache: k and q are rotated by the token's position, k and v are written into its page.
//
//   angle_j = position * inv_freq_j      (a, b) -> (a cos - b sin, a sin + b cos)      j < R/2
//
// with (a, b) the elements (j, j + R/2) of a head or, interleaved, (2j, 2j + 1); cos and sin are multiplied by `factor` and
// elements from R on are left alone.  The angle is taken in fp64 and reduced to one turn before it is rounded: position 10^6 in
// fp32 would leave it 0.06 off.
//
// A block does one token: its R/2 cosines and sines are made once for all heads.  Memory bounds it.
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

template <typename E, int VEC>
struct alignas(sizeof(E) * VEC) Vec {
    E e[VEC];
};

template <typename E, int VEC>
__global__ void __launch_bounds__(kThreads) append_kernel(const AppendArgs p) {
    __shared__ float cosine[RWKVB200_MAX_HEAD_SIZE / 2], sine[RWKVB200_MAX_HEAD_SIZE / 2];
    using V = Vec<E, VEC>;
    const int m = blockIdx.x;
    int b = m, nth = 0;
    if (p.cu != nullptr) {
        int lo = 0, hi = p.B;   // the last b with cu[b] <= m
        while (hi - lo > 1) {
            const int mid = (lo + hi) / 2;
            if (p.cu[mid] <= m) lo = mid; else hi = mid;
        }
        b = lo;
        nth = m - p.cu[b];
        if (nth < 0 || m >= p.cu[p.B]) return;   // rows that belong to no sequence
    }
    const int before = p.lengths[b];
    if (before < 0) return;                       // a row that only pads the batch
    const i64 position = (i64)before + nth;
    int id = -1;
    uint32_t col = 0, place = 0;
    if (position < (i64)p.width * p.page.d) {
        col = p.page.quotient((uint32_t)position);
        place = (uint32_t)position - col * p.page.d;
        id = p.table[(i64)b * p.width + col];
        if (id < 0 || id >= p.pages) {
            id = -1;
            if (threadIdx.x == 0) atomicMax(&g_error, kBadPage);
        }
    } else if (threadIdx.x == 0) {
        atomicMax(&g_error, kBadLength);
    }
    const int half = p.R / 2;
    for (int j = threadIdx.x; j < half; j += kThreads) {
        const double turns = (double)position * (double)p.inv_freq[j] * 0.15915494309189533577;   // angle / 2 pi
        float s, c;
        sincospif(2.f * (float)(turns - rint(turns)), &s, &c);
        cosine[j] = c * p.factor;
        sine[j] = s * p.factor;
    }
    __syncthreads();
    // items of a rotated head: pairs of vectors (half layout) or vectors of pairs, then the vectors behind R
    const int pieces = p.N / VEC, rotated = p.interleaved ? p.R / VEC : half / VEC, items = rotated + (p.N - p.R) / VEC;
    const int of_q = p.q != nullptr ? p.Hq * items : 0, of_k = p.Hkv * items, all = of_q + of_k + p.Hkv * pieces;
    for (int n = threadIdx.x; n < all; n += kThreads) {
        if (n >= of_q && id < 0) break;
        if (n >= of_q + of_k) {   // v: as it is
            const int i = n - of_q - of_k, head = i / pieces, at = i % pieces * VEC;
            const V x = *reinterpret_cast<const V*>(static_cast<const E*>(p.v) + ((i64)m * p.Hkv + head) * p.N + at);
            *reinterpret_cast<V*>(static_cast<E*>(p.v_pages) + (((i64)id * p.Hkv + head) * p.page.d + place) * p.N + at) = x;
            continue;
        }
        const bool is_q = n < of_q;
        const int i = is_q ? n : n - of_q, head = i / items, item = i % items;
        const E* from = static_cast<const E*>(is_q ? p.q : p.k) + ((i64)m * (is_q ? p.Hq : p.Hkv) + head) * p.N;
        E* to = is_q ? static_cast<E*>(p.q_out) + ((i64)m * p.Hq + head) * p.N
                     : static_cast<E*>(p.k_pages) + (((i64)id * p.Hkv + head) * p.page.d + place) * p.N;
        if (item >= rotated) {
            const int at = p.R + (item - rotated) * VEC;
            *reinterpret_cast<V*>(to + at) = *reinterpret_cast<const V*>(from + at);
        } else if (p.interleaved) {
            if constexpr (VEC > 1) {
                V x = *reinterpret_cast<const V*>(from + item * VEC);
#pragma unroll
                for (int e = 0; e < VEC; e += 2) {
                    const int j = (item * VEC + e) / 2;
                    const float a = to_f(x.e[e]), c = to_f(x.e[e + 1]);
                    x.e[e] = from_f<E>(a * cosine[j] - c * sine[j]);
                    x.e[e + 1] = from_f<E>(a * sine[j] + c * cosine[j]);
                }
                *reinterpret_cast<V*>(to + item * VEC) = x;
            } else if (item % 2 == 0) {   // one thread does both elements of a pair
                const int j = item / 2;
                const float a = to_f(from[item]), c = to_f(from[item + 1]);
                to[item] = from_f<E>(a * cosine[j] - c * sine[j]);
                to[item + 1] = from_f<E>(a * sine[j] + c * cosine[j]);
            }
        } else {
            V x = *reinterpret_cast<const V*>(from + item * VEC), z = *reinterpret_cast<const V*>(from + half + item * VEC);
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const int j = item * VEC + e;
                const float a = to_f(x.e[e]), c = to_f(z.e[e]);
                x.e[e] = from_f<E>(a * cosine[j] - c * sine[j]);
                z.e[e] = from_f<E>(a * sine[j] + c * cosine[j]);
            }
            *reinterpret_cast<V*>(to + item * VEC) = x;
            *reinterpret_cast<V*>(to + half + item * VEC) = z;
        }
    }
}

template <typename E>
int launch(const AppendArgs& p, cudaStream_t st) {
    constexpr int VEC = 16 / sizeof(E);
    uintptr_t all = 0;
    for (const void* x : {p.q, p.k, p.v, (const void*)p.q_out, (const void*)p.k_pages, (const void*)p.v_pages}) all |= reinterpret_cast<uintptr_t>(x);
    // 16 bytes a thread where heads, the rotated part and its halves are whole numbers of them
    const int part = p.interleaved ? p.R : p.R / 2;
    const bool wide = all % 16 == 0 && p.N % VEC == 0 && part % VEC == 0;
    if (wide) append_kernel<E, VEC><<<p.M, kThreads, 0, st>>>(p);
    else append_kernel<E, 1><<<p.M, kThreads, 0, st>>>(p);
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
    RWKV_REQUIRE((i64)(Hq > 0 ? Hq : 0) * N + 2ll * Hkv * N <= 0x3fffffff, RWKVB200_EINVAL, "%s: Hq=%d Hkv=%d are too many heads", what, Hq, Hkv);
    RWKV_REQUIRE(cu_seqlens != nullptr || M == B, RWKVB200_EINVAL, "%s: %d tokens for %d sequences need cu_seqlens", what, M, B);
    RWKV_NOTNULL(k); RWKV_NOTNULL(v); RWKV_NOTNULL(k_pages); RWKV_NOTNULL(v_pages); RWKV_NOTNULL(table); RWKV_NOTNULL(lengths);
    RWKV_REQUIRE((q == nullptr) == (q_out == nullptr), RWKVB200_EINVAL, "%s: q and q_out come together", what);
    if (R > 0) RWKV_NOTNULL(inv_freq);
    const AppendArgs p{M, B, Hq, Hkv, N, R, pages, width, interleaved, factor, Divisor((uint32_t)page), q, k, v, q_out, k_pages, v_pages, table, lengths, cu_seqlens, inv_freq};
    return dtype == RWKVB200_BF16 ? launch<bf16>(p, as_stream(stream)) : launch<float>(p, as_stream(stream));
}
