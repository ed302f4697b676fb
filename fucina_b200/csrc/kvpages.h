// Checks and device-side addressing shared by the kernels over a paged key-value cache.
#pragma once
#include "common.cuh"

namespace fq {

constexpr int kKvMaxD = 256;

// What a kernel needs of fq_kv_pages, strides resolved.
struct KvView {
    uint8_t* k;
    uint8_t* v;
    __half* k_scale;
    __half* v_scale;
    int n_pages, page_tokens, kv_heads, d;
    size_t page_stride;   // elements of k and v from page to page
    size_t scale_stride;  // elements of the scale planes from page to page
};

// kvcache.cu: FQ_OK and the resolved view, or a decline
int check_kv_pages(const fq_kv_pages* pages, KvView* view);

// Division of numbers below 2^31 by a fixed one (Granlund and Montgomery 1994): n / d = (n * mul) >> (31 + shift) with
// shift = ceil(log2 d) and mul = ceil(2^(31 + shift) / d), below 2^32.
struct FastDiv {
    unsigned d, mul, shift;
    __host__ FastDiv() : d(1), mul(1u << 31), shift(0) {}
    __host__ explicit FastDiv(unsigned d_) : d(d_), shift(0) {
        while ((1ull << shift) < d) ++shift;
        mul = (unsigned)(((1ull << (31 + shift)) + d - 1) / d);
    }
    __host__ __device__ __forceinline__ unsigned div(unsigned n) const {
        return (unsigned)(((unsigned long long)n * mul) >> 31 >> shift);
    }
};

// The row a (sequence, position) pair names, counted in tokens of one head inside its page.
struct KvSlot {
    int page;  // -1: names nothing
    int slot;
};
__device__ __forceinline__ KvSlot kv_slot(const int* __restrict__ table, int n_seqs, int max_pages, const FastDiv& page_tokens, int n_pages,
                                          int seq, int pos) {
    if (seq >= n_seqs || pos < 0) return {-1, 0};
    const int p = (int)page_tokens.div((unsigned)pos);
    if (p >= max_pages) return {-1, 0};
    const int page = table[(size_t)seq * max_pages + p];
    if (page < 0 || page >= n_pages) return {-1, 0};
    return {page, pos - p * (int)page_tokens.d};
}

}  // namespace fq
