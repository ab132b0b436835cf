// sxq_paged8_attn.hip -- attention over the 8-bit paged cache: one new token per request
// (sxq_kv_attention), and several, each over its own prefix (sxq_kv_prefix_attention).
// include/sxq.h states both.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "../../include/sxq.h"
#include "sxq_abi.h"
#include "sxq_paged.h"
#include "sxq_paged_dev.h"

using namespace sxq;
using namespace sxq::abi;

namespace {

// A wave a query and head, 64 positions at a time: a lane's dot product with its key, a running
// maximum and sum, then the weighted values, a lane a column (and every 64th after it).
template <typename TQ, typename C>
__global__ __launch_bounds__(256) void k_kv8_attend_plain(const KvAttend A, const int32_t* pos, const KvPool P) {
    __shared__ float s_q[4][256], s_p[4][64];
    __shared__ int s_slot[4][64];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, hd = P.hd;
    const int b = blockIdx.x, h = blockIdx.y * 4 + wave, kh = min(h, A.nh - 1) / (A.nh / P.nkv);
    const int row = A.rows ? A.rows[b] : b;
    if ((uint32_t)row >= (uint32_t)A.n_rows) return;
    int len = kv_clamp_len(A.lens[row], A.max_blocks, P.shift);
    if (pos) len = min(len, max(pos[b], -1) + 1);
    const bool live = h < A.nh;
    for (int d = lane; d < hd; d += 64) s_q[wave][d] = live ? to_f32(((const TQ*)A.q)[(int64_t)b * A.q_stride + (int64_t)h * hd + d]) : 0.0f;
    float m = -INFINITY, l = 0.0f, acc[4] = {0.f, 0.f, 0.f, 0.f};
    for (int p0 = 0; p0 < len; p0 += 64) {
        const int p = p0 + lane;
        const int slot = p < len ? kv_slot(A.table[(int64_t)row * A.table_stride + (p >> P.shift)], p, P.shift, P.n_pages) : -1;
        __syncthreads();
        float x = -INFINITY;
        if (slot >= 0) {
            const uint32_t* w = (const uint32_t*)((const uint8_t*)P.k + kv_slot_base(P, slot, kh));
            float dot = 0.0f;
            for (int d = 0; d < hd; d += 4) {
                float f[4];
                C::unpack(w[d / 4], f);
#pragma unroll
                for (int e = 0; e < 4; ++e) dot += f[e] * s_q[wave][d + e];
            }
            x = dot * P.k_scale[kv_scale_at(P, slot, kh)] * A.scale;
        }
        float top = x == x ? x : INFINITY;
        for (int o = 32; o >= 1; o >>= 1) top = fmaxf(top, __shfl_xor(top, o, 64));
        const float mn = fmaxf(m, top), up = m > -INFINITY ? expf(m - mn) : 1.0f;
        float e = mn > -INFINITY ? expf(x - mn) : 0.0f, sum = e;
        for (int o = 32; o >= 1; o >>= 1) sum += __shfl_xor(sum, o, 64);
        l = l * up + sum;
        m = mn;
        s_p[wave][lane] = slot >= 0 ? e * P.v_scale[kv_scale_at(P, slot, kh)] : 0.0f;
        s_slot[wave][lane] = slot;
        __syncthreads();
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int d = lane + 64 * q;
            if (d >= hd) break;
            float a = acc[q] * up;
            for (int k = 0; k < 64; ++k) {
                if (s_slot[wave][k] < 0) continue;
                float f[4];
                C::unpack(((const uint8_t*)P.v)[kv_slot_base(P, s_slot[wave][k], kh) + d], f);
                a += s_p[wave][k] * f[0];
            }
            acc[q] = a;
        }
    }
    if (!live) return;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const int d = lane + 64 * q;
        if (d < hd) ((TQ*)A.out)[(int64_t)b * A.out_stride + (int64_t)h * hd + d] = from_f32<TQ>(l == 0.0f ? 0.0f : acc[q] / l);
    }
}

template <typename TQ>
void attend_plain(const KvAttend& a, const int32_t* pos, const KvPool& p, hipStream_t s) {
    const dim3 grid(a.n_q, (a.nh + 3) / 4);
    if (p.dtype == kI8) hipLaunchKernelGGL((k_kv8_attend_plain<TQ, I8>), grid, dim3(256), 0, s, a, pos, p);
    else hipLaunchKernelGGL((k_kv8_attend_plain<TQ, E4M3>), grid, dim3(256), 0, s, a, pos, p);
}

}  // namespace

namespace sxq {

size_t kv8_attend_workspace(const KvPool& p, int n_q, int nh) { return SXQ_KV_COUNTER_BYTES; }
size_t kv8_prefix_workspace(const KvPool& p, int n_q, int nh) { return 256; }

hipError_t launch_kv8_attend(const KvAttend& a, const KvPool& p, hipStream_t s) { return launch_kv8_prefix(a, nullptr, p, s); }
hipError_t launch_kv8_prefix(const KvAttend& a, const int32_t* pos, const KvPool& p, hipStream_t s) {
    if (a.q_dtype == kF32) attend_plain<float>(a, pos, p, s);
    else if (a.q_dtype == kF16) attend_plain<_Float16>(a, pos, p, s);
    else attend_plain<__bf16>(a, pos, p, s);
    return hipGetLastError();
}

}  // namespace sxq
