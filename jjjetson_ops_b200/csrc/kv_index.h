// Where a token of a paged cache lies, as the kernels and the tests on the CPU compute it.  Plain C++.
#pragma once

#include <cstdint>

#ifdef __CUDACC__
#define JQ_HOST_DEVICE __host__ __device__ __forceinline__
#else
#define JQ_HOST_DEVICE inline
#endif

namespace jq {

// The indices of one cache (see jq_kv_cache); all sizes have been checked to fit.
struct KvIndex {
    const int32_t *table;
    int64_t table_stride;
    int64_t stride_page, stride_slot, stride_head;  // in elements
    int32_t num_seqs, max_pages, num_pages, page_size;
    // token / page_size = token * page_magic / 2^(31 + page_shift): a division costs some 20 instructions, and the page comes first
    uint32_t page_magic;
    int32_t page_shift;
};

// With 2^(s - 1) < d <= 2^s and m = floor(2^(31 + s) / d) + 1, m * d is above 2^(31 + s) by at most 2^s, so that t * m / 2^(31 + s) is
// above t / d by less than 1 / d for t < 2^31: the whole part is the quotient's.  m < 2^32 but for d = 1, where it is 2^31 + 1.
JQ_HOST_DEVICE void kv_set_page_size(KvIndex &ix, int32_t page_size) {
    ix.page_size = page_size;
    ix.page_shift = 0;
    while (((int64_t)1 << ix.page_shift) < page_size) ++ix.page_shift;
    ix.page_magic = (uint32_t)(((uint64_t)1 << (31 + ix.page_shift)) / (uint32_t)page_size + 1);
}
JQ_HOST_DEVICE uint32_t kv_page_of(const KvIndex &ix, uint32_t token) {
    return (uint32_t)(((uint64_t)token * ix.page_magic) >> 31 >> ix.page_shift);
}

// Element offset of token `token`, head 0, in page `page` (what the table says), or -1 when that page does not exist.
JQ_HOST_DEVICE int64_t kv_offset(const KvIndex &ix, uint32_t token, int32_t page) {
    if ((uint32_t)page >= (uint32_t)ix.num_pages) return -1;
    const uint32_t slot = token - kv_page_of(ix, token) * (uint32_t)ix.page_size;
    return (int64_t)page * ix.stride_page + (int64_t)slot * ix.stride_slot;
}

// Tokens of a sequence that has `len` of them by the caller's count: what fits in its row of the table.
JQ_HOST_DEVICE int32_t kv_length(const KvIndex &ix, int32_t len) {
    const int64_t most = (int64_t)ix.max_pages * ix.page_size;
    return len < 0 ? 0 : len > most ? (int32_t)most : len;
}

// A turn is 2^64 steps.  `steps` per position times the position, modulo a turn, is exact.  The nearest quarter turn is taken off it as
// an integer; what is left, in half turns, [-1/4, 1/4], is off by 2^-33 from the cut and by half a bit of its own, 2^-27 at most, from the
// conversion (of a whole half turn it would be 2^-25).
JQ_HOST_DEVICE float rope_half_turns(uint64_t steps, int32_t position, uint32_t *quarters) {
    const uint64_t angle = steps * (uint64_t)(int64_t)position;
    *quarters = (uint32_t)((angle + ((uint64_t)1 << 61)) >> 62);
    return (float)(int32_t)((int64_t)(angle - ((uint64_t)*quarters << 62)) >> 30) * 1.1641532182693481e-10f;  // 2^-33
}
// The cosine and sine of an angle from those of what is left without its quarter turns.
JQ_HOST_DEVICE void rope_add_quarters(uint32_t quarters, float *c, float *s) {
    const float x = quarters & 1 ? -*s : *c, y = quarters & 1 ? *c : *s;
    *c = quarters & 2 ? -x : x;
    *s = quarters & 2 ? -y : y;
}

}  // namespace jq
