// The paged key-value cache as the attention kernels see it, and the checks that its entry points share.
//
// A cache row is one token's key (or value) in one head: D elements, BF16, or 8- or 4-bit codes along D in groups of G, element = code * scale +
// min, the group's scale and min neighbours in one 32-bit word (scale low).  Token p of a sequence lies in page table[p / page] at row p % page:
// row number = page id * page_stride + head * head_stride + (p % page) * row_stride, and a row's words of scales stand at the same number.
#pragma once

#include "common.cuh"

namespace sxb {

struct KvView {
    uint8_t *k, *v;
    uint32_t *k_sm, *v_sm;  // [rows][D / G]; null for BF16
    int64_t page_stride, head_stride, row_stride;
    int n_pages, page_shift, n_kv;
};

// Refuses what the kernels cannot address; on success fills the view.
int kv_view(const char *fn, const SxbKvCache *c, KvView *out);

inline bool is_pow2(int64_t v) { return v > 0 && (v & (v - 1)) == 0; }


__device__ inline int64_t kv_row(const KvView &c, int page, int head, int at) {
    return page * c.page_stride + head * c.head_stride + at * c.row_stride;
}

}  // namespace sxb
