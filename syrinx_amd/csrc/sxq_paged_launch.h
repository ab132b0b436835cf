// sxq_paged_launch.h -- launchers of the paged cache's kernels (sxq_paged.hip,
// sxq_paged_attn.hip); the arguments are checked by their callers.
#pragma once
#include "sxq_abi.h"
#include "sxq_paged.h"

namespace sxq {

struct KvReserve {
    int shift, n_pages, n_rows, max_blocks;
    int capacity;  // entries of the map
    int limit;     // tokens that may be handed out (the capacity, or more: the rest is not mapped)
    int64_t table_stride;
    const int32_t* add;
    int32_t *lens, *table, *free_list, *free_count, *cu, *slots, *pos, *rows, *status;
};
// moved (or null): set once the launch that moves lengths (and, up to 64 rows, pages) is made,
// which a later one of the call that fails does not take back.
hipError_t launch_kv_reserve(const KvReserve& a, hipStream_t s, bool* moved = nullptr);

struct KvAppend {
    const void* qkv;
    int64_t row_stride;
    int dtype, n_tokens, nh;
    const float *q_norm, *k_norm;
    float eps;
    const float *cos, *sin;
    int max_pos, interleaved;
    const int32_t *pos, *slots;
    void* q_out;
};
hipError_t launch_kv_append(const KvAppend& a, const KvPool& p, hipStream_t s);

struct KvAttend {
    const void* q;
    int64_t q_stride;
    int q_dtype, n_q, nh;
    const int32_t *rows, *lens, *table;
    int n_rows, max_blocks;
    int64_t table_stride;
    float scale;
    void* out;
    int64_t out_stride;
    void* ws;
};
size_t kv_attend_workspace(const KvPool& p, int n_q, int nh);
hipError_t launch_kv_attend(const KvAttend& a, const KvPool& p, hipStream_t s);

// The same over 8-bit pages (sxq_paged8*.hip); with pos (a position a query, or null) query i sees
// the positions 0 .. pos[i] only.
hipError_t launch_kv8_append(const KvAppend& a, const KvPool& p, hipStream_t s);
size_t kv8_attend_workspace(const KvPool& p, int n_q, int nh);
hipError_t launch_kv8_attend(const KvAttend& a, const KvPool& p, hipStream_t s);
size_t kv8_prefix_workspace(const KvPool& p, int n_q, int nh);
hipError_t launch_kv8_prefix(const KvAttend& a, const int32_t* pos, const KvPool& p, hipStream_t s);

// sxq_kv_read, of pages of any type.
struct KvRead {
    const int32_t *cu, *rows, *start, *lens, *table;
    int n_ranges, total, n_rows, max_blocks;
    int64_t table_stride;
    int out_dtype;
    void *k, *v;
    int64_t out_stride;
};
hipError_t launch_kv_read(const KvRead& a, const KvPool& p, hipStream_t s);

inline bool kv_is8(int dtype) { return dtype == kI8 || dtype == kE4M3; }
inline int kv_elem_size(int dtype) { return kv_is8(dtype) ? 1 : type_size(dtype); }

// Up to 16 rows' positions one after another: row i's are start[i] .. start[i + 1] - 1 of start[n].
struct KvSpans {
    int n, start[17];
};
// One layer's KV heads h0 .. h0 + heads - 1 of rows r0 .. r0 + n - 1, each row's positions from p0
// on, as f32 [head][start[n]][hd] (either output may be null).  An absent page reads as zeros.
hipError_t launch_kv_gather(const KvPool& p, const int32_t* table, int64_t table_stride, int max_blocks, const KvSpans& spans,
                            int r0, int h0, int heads, int p0, float* k, float* v, hipStream_t s);
// A free stack of pages 0 .. n - 1, page 0 on top.
hipError_t launch_kv_stack(int32_t* free_list, int n, hipStream_t s);
// The growths of an engine's streams, written to its device array.
struct KvGrowths {
    int n, add[16];
};
hipError_t launch_kv_growths(const KvGrowths& g, int32_t* add, hipStream_t s);
// Row r's slot and position (-1 and 0 without a token) from a map of at most one token a row.
hipError_t launch_kv_by_row(const int32_t* cu, const int32_t* map_slots, const int32_t* map_pos, int rows, int32_t* slots,
                            int32_t* pos, hipStream_t s);
// bf16 (round to nearest even) of n f32 values.
hipError_t launch_f32_to_bf16(const float* x, int64_t n, uint16_t* y, hipStream_t s);
// e4m3 codes of n f32 values times inv (n a multiple of 4).
hipError_t launch_f32_to_e4m3(const float* x, int64_t n, float inv, uint8_t* y, hipStream_t s);
hipError_t launch_fill_f32(float* y, int64_t n, float v, hipStream_t s);

namespace abi {
// The checks every entry point makes of its pages, and their kernel form.
sxq_status kv_pool(const char* who, const sxq_kv_pages* g, bool pointers, KvPool* out);
}  // namespace abi

// f32 <-> the activation and page types (one round-to-nearest-even).
SXQ_DEV float to_f32(float v) { return v; }
SXQ_DEV float to_f32(_Float16 v) { return (float)v; }
SXQ_DEV float to_f32(__bf16 v) { return (float)v; }
template <typename T>
SXQ_DEV T from_f32(float v) {
    return (T)v;
}

}  // namespace sxq
