// sxq_paged.h -- the paged key/value cache's index arithmetic (host and device; plain C++, so
// that it is enumerated on the CPU as the kernels use it) and, under hipcc, its launchers.
//
// A cache of one layer is a pool of pages: `page` positions (a power of two) of every KV
// head.  Request r's position p lies in page table[r][p >> shift], at offset p & (page - 1);
// a slot is page * page_size + offset.  Every index that comes from device memory (page
// ids, slots, lengths, rows) is checked against its range before it is used as an address:
// a page id outside the pool counts as absent.
#pragma once
#include <stdint.h>

#if defined(__HIPCC__)
#define SXQ_PG_HD __host__ __device__ __forceinline__
#else
#define SXQ_PG_HD inline
#endif

namespace sxq {

// Types that pages alone have, beside DType's (here, for sxq_common.h is part of the GEMV kernels'
// sources, whose counter summaries go by its text).
enum PageType : int {
    kI8 = 24,
    kE4M3 = 0x101,
};

// One layer's pages.  Strides in elements.
struct KvPool {
    void *k, *v;
    int64_t page_stride, head_stride, pos_stride;
    int32_t dtype, nkv, hd, page, shift, n_pages;
    // 8-bit pages: a scale for every kScaleBlock positions of a page and head.  Strides in floats.
    float *k_scale, *v_scale;
    int64_t scale_page_stride, scale_head_stride;
};
constexpr int kScaleShift = 4, kScaleBlock = 1 << kScaleShift;

SXQ_PG_HD int kv_blocks(int len, int shift) { return (int)(((int64_t)len + (1 << shift) - 1) >> shift); }
// A stored length as the kernels take it: 0 .. the positions its table row can hold.
SXQ_PG_HD int kv_clamp_len(int len, int max_blocks, int shift) {
    const int64_t top = (int64_t)max_blocks << shift;
    return len < 0 ? 0 : len > top ? (int)top : len;
}
SXQ_PG_HD bool kv_page_ok(int id, int n_pages) { return (uint32_t)id < (uint32_t)n_pages; }
SXQ_PG_HD int kv_slot(int id, int pos, int shift, int n_pages) {
    return kv_page_ok(id, n_pages) ? (id << shift) + (pos & ((1 << shift) - 1)) : -1;
}
SXQ_PG_HD int64_t kv_page_base(const KvPool& p, int id, int head) {
    return (int64_t)id * p.page_stride + (int64_t)head * p.head_stride;
}
// Element offset of head `head` at a slot (which lies in the pool).
SXQ_PG_HD int64_t kv_slot_base(const KvPool& p, int slot, int head) {
    return kv_page_base(p, slot >> p.shift, head) + (int64_t)(slot & (p.page - 1)) * p.pos_stride;
}

// Offset of the scale of head `head` at a slot (which lies in the pool).
SXQ_PG_HD int64_t kv_scale_at(const KvPool& p, int slot, int head) {
    return (int64_t)(slot >> p.shift) * p.scale_page_stride + (int64_t)head * p.scale_head_stride +
           ((slot & (p.page - 1)) >> kScaleShift);
}

// Into how many pieces a prefix attention cuts a tile of so many tiles of keys, a place's share of the
// card being `piece` of them: a quarter more stays whole.  Kernel and join, us, by half more / a quarter
// more / none: three f32 prompts of 1412 tokens 55.4 / 53.0 / 63.2, 16 drafts of 5 20.8 / 19.9 / 20.0, a
// chunk of 2048 after 30720 1370 / 1365 / 1495 (none: more pieces than places).
SXQ_PG_HD int kv_pieces(int keys, int piece) { return keys - piece > piece / 4 ? (keys - 1) / piece + 1 : 1; }

}  // namespace sxq
