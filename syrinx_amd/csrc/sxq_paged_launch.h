// sxq_paged_launch.h -- launchers of the paged cache's kernels (sxq_paged.hip,
// sxq_paged_attn.hip); the arguments are checked by their callers.
#pragma once
#include "sxq_abi.h"
#include "sxq_paged.h"

namespace sxq {

struct KvReserve {
    int shift, n_pages, n_rows, max_blocks, capacity;
    int64_t table_stride;
    const int32_t* add;
    int32_t *lens, *table, *free_list, *free_count, *cu, *slots, *pos, *rows, *status;
};
hipError_t launch_kv_reserve(const KvReserve& a, hipStream_t s);

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
