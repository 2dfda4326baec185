// What the cache's write (paged_append.cu) and the attention that reads it (paged_attention.cu) share.
//
// A cache is two pools of pages (pages, Hkv, page, N): the tokens of one head lie behind one another in a page, so that a head's
// keys are read in runs of page x N elements.  Row b of `table` (B, width) names the pages of sequence b; the token at position j
// lies in page table[b][j / page], at place j % page.
#pragma once
#include "common.cuh"

namespace rwkvb200 {

// n / d for 0 <= n < 2^31 by a multiplication (d >= 1): the high half of n times a 33-bit reciprocal rounded up, whose top bit is the
// addition of n (Granlund and Montgomery, division by invariant integers)
struct Divisor {
    uint32_t d, mul, shift;
    explicit Divisor(uint32_t value) : d(value), mul(0), shift(0) {
        while ((1ull << shift) < d) ++shift;
        mul = (uint32_t)((((1ull << shift) - d) << 32) / d + 1);
    }
    __device__ __forceinline__ uint32_t quotient(uint32_t n) const { return (__umulhi(n, mul) + n) >> shift; }
};

// what the kernels write into the status word of their device
constexpr int kBadPage = 1;      // a page number outside of the pool
constexpr int kBadLength = 2;    // a length beyond what a row of the table holds
constexpr int kTimeout = 3;      // a wait for a copy ran out

int paged_append_error(int clear);      // the last code of the current device, or -1; clear: sets it to 0
int paged_attention_error(int clear);
int gated_scan_error(int clear);

}  // namespace rwkvb200
