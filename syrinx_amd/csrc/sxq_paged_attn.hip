// sxq_paged_attn.hip -- attention of one new token per request over a paged cache
// (sxq_kv_attention; include/sxq.h states it).
#include <hip/hip_runtime.h>

#include "../../include/sxq.h"
#include "sxq_abi.h"
#include "sxq_paged.h"
#include "sxq_paged_launch.h"

using namespace sxq;
using namespace sxq::abi;

namespace {

// One workgroup per (query, head): 256 positions at a time, a thread per position for the
// scores, then per element of the value for the weighted sum; running maximum and sum.
template <typename TQ, typename TC>
__global__ __launch_bounds__(256) void k_kv_attend(const KvAttend A, const KvPool P) {
    __shared__ float sq[256], sp[256], red[8];
    __shared__ int sid[256];
    const int b = blockIdx.x, h = blockIdx.y, tid = threadIdx.x, hd = P.hd;
    const int r = A.rows ? A.rows[b] : b;
    if (r < 0 || r >= A.n_rows) return;
    const int len = kv_clamp_len(A.lens[r], A.max_blocks, P.shift), kh = h / (A.nh / P.nkv);
    if (tid < hd) sq[tid] = to_f32(((const TQ*)A.q)[b * A.q_stride + (int64_t)h * hd + tid]);
    const TC *kp = (const TC*)P.k, *vp = (const TC*)P.v;
    float m = -INFINITY, l = 0.0f, acc = 0.0f;
    __syncthreads();
    for (int p0 = 0; p0 < len; p0 += 256) {
        const int p = p0 + tid;
        const int id = p < len ? A.table[r * A.table_stride + (p >> P.shift)] : -1;
        const bool ok = kv_page_ok(id, P.n_pages);
        float s = -INFINITY;
        if (ok) {
            const TC* k = kp + kv_page_base(P, id, kh) + (int64_t)(p & (P.page - 1)) * P.pos_stride;
            s = 0.0f;
            for (int d = 0; d < hd; ++d) s += sq[d] * to_f32(k[d]);
            s *= A.scale;
        }
        float mx = s;
        for (int o = 32; o >= 1; o >>= 1) mx = fmaxf(mx, __shfl_xor(mx, o, 64));
        if ((tid & 63) == 0) red[tid >> 6] = mx;
        __syncthreads();
        const float mn = fmaxf(m, fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])));
        const float base = mn > -INFINITY ? mn : 0.0f;  // every score -inf or NaN so far
        const float e = ok ? expf(s - base) : 0.0f;
        float sum = e;
        for (int o = 32; o >= 1; o >>= 1) sum += __shfl_xor(sum, o, 64);
        sp[tid] = e;
        sid[tid] = ok ? id : -1;
        if ((tid & 63) == 0) red[4 + (tid >> 6)] = sum;
        __syncthreads();
        const float al = m > -INFINITY ? expf(m - base) : 1.0f;
        l = l * al + (red[4] + red[5] + red[6] + red[7]);
        acc *= al;
        m = mn;
        if (tid < hd)
            for (int j = 0; j < 256; ++j)
                if (sid[j] >= 0)
                    acc += sp[j] * to_f32(vp[kv_page_base(P, sid[j], kh) + (int64_t)((p0 + j) & (P.page - 1)) * P.pos_stride + tid]);
        __syncthreads();
    }
    if (tid < hd) ((TQ*)A.out)[b * A.out_stride + (int64_t)h * hd + tid] = from_f32<TQ>(l == 0.0f ? 0.0f : acc / l);
}

}  // namespace

namespace sxq {

size_t kv_attend_workspace(const KvPool& p, int n_q, int nh) { return 256; }

hipError_t launch_kv_attend(const KvAttend& a, const KvPool& p, hipStream_t s) {
    const dim3 grid(a.n_q, a.nh);
    if (p.dtype == kF32) hipLaunchKernelGGL((k_kv_attend<float, float>), grid, dim3(256), 0, s, a, p);
    else if (p.dtype == kF16) hipLaunchKernelGGL((k_kv_attend<_Float16, _Float16>), grid, dim3(256), 0, s, a, p);
    else if (a.q_dtype == kF32) hipLaunchKernelGGL((k_kv_attend<float, __bf16>), grid, dim3(256), 0, s, a, p);
    else hipLaunchKernelGGL((k_kv_attend<__bf16, __bf16>), grid, dim3(256), 0, s, a, p);
    return hipGetLastError();
}

}  // namespace sxq

extern "C" {

sxq_status sxq_kv_attention_workspace(const sxq_kv_pages* pages, int n_q, int n_heads, size_t* bytes) {
    if (!bytes) return fail(SXQ_ERR_INVALID, "kv_attention_workspace: null output");
    KvPool p;
    if (sxq_status st = kv_pool("kv_attention_workspace", pages, false, &p)) return st;
    if (n_q < 0 || n_q > 1 << 20 || n_heads < 1 || n_heads > 16384 || n_heads % p.nkv)
        return fail(SXQ_ERR_SHAPE, "kv_attention_workspace: %d queries of %d heads over %d KV heads", n_q, n_heads, p.nkv);
    *bytes = kv_attend_workspace(p, n_q, n_heads);
    return SXQ_OK;
}

sxq_status sxq_kv_attention(int device, const sxq_kv_pages* pages, int q_dtype, const void* q, int64_t q_stride,
                            int n_q, int n_heads, const int32_t* rows, const int32_t* lens, int n_rows,
                            const int32_t* table, int64_t table_stride, int max_blocks, float scale, void* out,
                            int64_t out_stride, void* workspace, size_t workspace_bytes, void* stream) {
    KvPool p;
    if (sxq_status st = kv_pool("kv_attention", pages, n_q > 0, &p)) return st;
    if (q_dtype != p.dtype && !(q_dtype == kF32 && p.dtype == kBF16))
        return fail(SXQ_ERR_DTYPE, "kv_attention: queries of dtype %d over pages of dtype %d", q_dtype, p.dtype);
    if (n_q < 0 || n_q > 1 << 20 || n_heads < 1 || n_heads > 16384 || n_heads % p.nkv)
        return fail(SXQ_ERR_SHAPE, "kv_attention: %d queries of %d heads over %d KV heads", n_q, n_heads, p.nkv);
    const int64_t width = (int64_t)n_heads * p.hd, unit = 16 / type_size(q_dtype);
    if (q_stride < width || out_stride < width || q_stride % unit || out_stride % unit)
        return fail(SXQ_ERR_SHAPE, "kv_attention: q_stride %lld, out_stride %lld (multiples of %lld elements, rows of %lld)",
                    (long long)q_stride, (long long)out_stride, (long long)unit, (long long)width);
    if (n_rows < 1 || max_blocks < 1 || table_stride < max_blocks || (int64_t)max_blocks * p.page > 0x7FFFFFFF)
        return fail(SXQ_ERR_INVALID, "kv_attention: a table of %d rows of %d blocks, stride %lld", n_rows, max_blocks, (long long)table_stride);
    if (!rows && n_q > n_rows) return fail(SXQ_ERR_SHAPE, "kv_attention: %d queries over %d table rows", n_q, n_rows);
    if (!(scale - scale == 0.0f)) return fail(SXQ_ERR_INVALID, "kv_attention: scale is not finite");
    if (n_q == 0) return SXQ_OK;
    if (!q || !lens || !table || !out || !workspace) return fail(SXQ_ERR_INVALID, "kv_attention: null pointer");
    if (((uintptr_t)q | (uintptr_t)out) & 15) return fail(SXQ_ERR_INVALID, "kv_attention: q and out must be 16-byte aligned");
    if ((uintptr_t)workspace & 255) return fail(SXQ_ERR_INVALID, "kv_attention: the workspace must be 256-byte aligned");
    const size_t need = kv_attend_workspace(p, n_q, n_heads);
    if (workspace_bytes < need)
        return fail(SXQ_ERR_INVALID, "kv_attention: a workspace of %zu bytes, %zu needed", workspace_bytes, need);
    DeviceGuard g(device);
    HIP_TRY(g.err, "hipSetDevice");
    KvAttend a;
    a.q = q;
    a.q_stride = q_stride;
    a.q_dtype = q_dtype;
    a.n_q = n_q;
    a.nh = n_heads;
    a.rows = rows;
    a.lens = lens;
    a.table = table;
    a.n_rows = n_rows;
    a.max_blocks = max_blocks;
    a.table_stride = table_stride;
    a.scale = scale;
    a.out = out;
    a.out_stride = out_stride;
    a.ws = workspace;
    HIP_TRY(launch_kv_attend(a, p, (hipStream_t)stream), "kv_attention");
    return SXQ_OK;
}

}  // extern "C"
