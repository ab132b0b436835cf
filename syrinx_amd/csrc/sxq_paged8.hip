// sxq_paged8.hip -- the paged cache in 8 bits: new tokens quantized into the pages
// (sxq_kv_append over SXQ_I8 and SXQ_E4M3), and pages of any type read back (sxq_kv_read).
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

// ---------------------------------------------------------------------------- append
// One head's row of a token: eight elements a lane, as two vectors of four at o1 and o2 that hold
// four RoPE pairs (interleaved: 8 j and 8 j + 4; in halves: 4 j and hd / 2 + 4 j), lane j of lh.
// The norm's sum stays among the lh lanes and no element changes lanes.  live: the lane has
// elements; the others give zeros.
template <typename TI>
SXQ_DEV void head_row(const KvAppend& A, int t, int hid, int hd, int j, int lh, bool live, const float* w, bool rot, float* x) {
    const int half = hd / 2, o1 = A.interleaved ? 8 * j : 4 * j, o2 = A.interleaved ? 8 * j + 4 : half + 4 * j;
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = 0.0f;
    float c[4], s[4], g[8];
    if (live) {
        const TI* src = (const TI*)A.qkv + (int64_t)t * A.row_stride + (int64_t)hid * hd;
        load4(src + o1, x);
        load4(src + o2, x + 4);
        if (w) {
            load4(w + o1, g);
            load4(w + o2, g + 4);
        }
        if (rot) {
            const int p = min(max(A.pos[t], 0), A.max_pos - 1);
            load4(A.cos + (int64_t)p * half + 4 * j, c);
            load4(A.sin + (int64_t)p * half + 4 * j, s);
        }
    }
    if (w) {
        float ss = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) ss = fmaf(x[e], x[e], ss);
        for (int o = lh >> 1; o >= 1; o >>= 1) ss += __shfl_xor(ss, o, 64);
        const float inv = 1.0f / sqrtf(ss / (float)hd + A.eps);
        if (live)
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = x[e] * inv * g[e];
    }
    if (rot && live)
#pragma unroll
        for (int e = 0; e < 4; ++e) {  // pair e of the lane
            float &a = A.interleaved ? x[2 * e] : x[e], &b = A.interleaved ? x[2 * e + 1] : x[4 + e];
            const float u = fmaf(a, c[e], -(b * s[e]));
            b = fmaf(b, c[e], a * s[e]);
            a = u;
        }
}

SXQ_DEV float wave_max(float v) {
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, 64));
    return v;
}

// The tokens of a call fall into runs: consecutive tokens at consecutive slots of one block of 16.
// A wave owns a run for one KV head's keys or values: the rows in registers (NP passes of 64 / lh
// tokens, eight elements a lane), the largest of them by a reduction, the scale, the codes; if the
// block's scale has grown, its earlier codes after that.  A wave looks for the runs that begin
// among its `chunk` tokens.  The queries' heads are other workgroups of the launch (from
// kv_groups on), a token and 256 / lh heads each.
template <typename TI, typename C, int NP>
__global__ __launch_bounds__(256) void k_kv8_append(const KvAppend A, const KvPool P, int lh, int chunk, int kv_groups, int q_groups) {
    const int lane = threadIdx.x & 63, hd = P.hd, half = hd / 2;
    const int j = threadIdx.x & (lh - 1);
    const bool live = 8 * j < hd;
    const int o1 = A.interleaved ? 8 * j : 4 * j, o2 = A.interleaved ? 8 * j + 4 : half + 4 * j;
    const uint32_t slots = (uint32_t)P.n_pages << P.shift;
    if ((int)blockIdx.x >= kv_groups) {
        const int b = blockIdx.x - kv_groups, t = b / q_groups, hid = (b - t * q_groups) * (256 / lh) + (int)threadIdx.x / lh;
        if ((uint32_t)A.slots[t] >= slots) return;
        const bool mine = live && hid < A.nh;
        float x[8];
        head_row<TI>(A, t, hid, hd, j, lh, mine, A.q_norm, A.cos != nullptr, x);
        if (!mine) return;
        TI* dst = (TI*)A.q_out + ((int64_t)t * A.nh + hid) * hd;
        store4(dst + o1, x);
        store4(dst + o2, x + 4);
        return;
    }
    const int pairs = 2 * P.nkv, u = (int)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int t0 = u / pairs * chunk, pair = u % pairs;
    if (t0 >= A.n_tokens) return;
    const bool is_k = pair < P.nkv;
    const int head = is_k ? pair : pair - P.nkv;
    uint8_t* pool = (uint8_t*)(is_k ? P.k : P.v);
    float* scales = is_k ? P.k_scale : P.v_scale;
    const float* w = is_k ? A.k_norm : nullptr;

    // lane i: token t0 - 1 + i
    const int ti = t0 - 1 + lane;
    const int slot = ti >= 0 && ti < A.n_tokens ? A.slots[ti] : -1;
    const int before = __shfl_up(slot, 1, 64);
    const bool in = (uint32_t)slot < slots;
    const bool goes_on = in && lane > 0 && slot == before + 1 && (slot & (kScaleBlock - 1)) != 0 && before >= 0;
    const uint64_t on = __ballot(goes_on);
    uint64_t firsts = __ballot(in && !goes_on && lane >= 1 && lane <= chunk);
    const int sub = lane / lh, per = 64 / lh;  // this lane's token of a pass, tokens a pass
    while (firsts) {
        const int i = __builtin_ctzll(firsts);
        firsts &= firsts - 1;
        const int t = t0 - 1 + i, first = __builtin_amdgcn_readlane(slot, i), o = first & (kScaleBlock - 1);
        // (bits i + 1 on of a run: at most 15, ended by the next block)
        const int len = 1 + __builtin_ctzll(~((on >> i) >> 1));
        float x[NP][8], amax = 0.0f;
#pragma unroll
        for (int p = 0; p < NP; ++p)
            if (p * per < len) {
                const int k = p * per + sub;
                head_row<TI>(A, t + min(k, len - 1), A.nh + pair, hd, j, lh, live && k < len, w, is_k && A.cos, x[p]);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float a = fabsf(x[p][e]);
                    amax = a < INFINITY ? fmaxf(amax, a) : amax;
                }
            }
        float* at = scales + kv_scale_at(P, first, head);
        const float had = o ? *at : 0.0f, need = block_scale<C>(wave_max(amax));
        const bool grown = !(had >= need);
        const float s = grown ? need : had, inv = 1.0f / s;
        const int64_t base = kv_slot_base(P, first, head);
#pragma unroll
        for (int p = 0; p < NP; ++p) {
            const int k = p * per + sub;
            if (p * per < len && live && k < len) {
#pragma unroll
                for (int e = 0; e < 8; ++e) x[p][e] *= inv;
                uint8_t* dst = pool + base + (int64_t)k * P.pos_stride;
                *(uint32_t*)(dst + o1) = C::pack(x[p]);
                *(uint32_t*)(dst + o2) = C::pack(x[p] + 4);
            }
        }
        if (grown) {
            if (lane == 0) *at = s;
            const float ratio = had * inv;
            for (int p = 0; p * per < o; ++p) {
                const int k = p * per + sub;
                if (!live || k >= o) continue;
                uint32_t* b = (uint32_t*)(pool + base + (int64_t)(k - o) * P.pos_stride + 8 * j);
                float f[8];
                C::unpack(b[0], f);
                C::unpack(b[1], f + 4);
#pragma unroll
                for (int e = 0; e < 8; ++e) f[e] *= ratio;
                b[0] = C::pack(f);
                b[1] = C::pack(f + 4);
            }
        }
    }
}

template <typename TI, typename C>
hipError_t append_by_width(const KvAppend& a, const KvPool& p, hipStream_t s) {
    int lh = 2;
    while (8 * lh < p.hd) lh *= 2;
    const int chunk = 1, pairs = 2 * p.nkv, q_groups = a.q_out ? (a.nh + 256 / lh - 1) / (256 / lh) : 0;
    const int kv_groups = (int)(((int64_t)(a.n_tokens + chunk - 1) / chunk * pairs + 3) / 4);
    const dim3 grid((unsigned)(kv_groups + (int64_t)a.n_tokens * q_groups));
#define SXQ_AP(NP) hipLaunchKernelGGL((k_kv8_append<TI, C, NP>), grid, dim3(256), 0, s, a, p, lh, chunk, kv_groups, q_groups)
    if (lh <= 4) SXQ_AP(1);
    else if (lh == 8) SXQ_AP(2);
    else if (lh == 16) SXQ_AP(4);
    else SXQ_AP(8);
#undef SXQ_AP
    return hipGetLastError();
}
template <typename TI>
hipError_t append_by_code(const KvAppend& a, const KvPool& p, hipStream_t s) {
    return p.dtype == kI8 ? append_by_width<TI, I8>(a, p, s) : append_by_width<TI, E4M3>(a, p, s);
}

// ---------------------------------------------------------------------------- read
template <typename T>
constexpr bool kCodes = false;
template <>
constexpr bool kCodes<I8> = true;
template <>
constexpr bool kCodes<E4M3> = true;
template <typename T>
constexpr int kElem = sizeof(T);
template <>
constexpr int kElem<I8> = 1;
template <>
constexpr int kElem<E4M3> = 1;

// A workgroup's kReadTokens entries: their slots once (range by search, page by table) through
// LDS, then eight elements of K and V a thread at a time.
constexpr int kReadTokens = 16;
template <typename T, typename TO>
__global__ __launch_bounds__(256) void k_kv_read(const KvRead A, const KvPool P) {
    __shared__ int s_slot[kReadTokens];
    const int t0 = blockIdx.x * kReadTokens, end = min(A.total, A.cu[A.n_ranges]);
    if (t0 >= end) return;
    if (threadIdx.x < kReadTokens) {
        const int t = t0 + threadIdx.x;
        int slot = -1;
        if (t < end) {
            const int i = owner(A.cu, A.n_ranges, t), row = A.rows ? A.rows[i] : i;
            const int64_t pos = (int64_t)(A.start ? A.start[i] : 0) + t - A.cu[i];
            if ((uint32_t)row < (uint32_t)A.n_rows && pos >= 0 && pos < kv_clamp_len(A.lens[row], A.max_blocks, P.shift))
                slot = kv_slot(A.table[(int64_t)row * A.table_stride + (pos >> P.shift)], (int)pos, P.shift, P.n_pages);
        }
        s_slot[threadIdx.x] = slot;
    }
    __syncthreads();
    const int per = P.hd / 8, row = per * P.nkv, n = min(kReadTokens, end - t0) * row;
    for (int i = threadIdx.x; i < n; i += 256) {
        const int t = i / row, h = (i - t * row) / per, d = 8 * (i - t * row - h * per);
        const int slot = s_slot[t];
        float f[2][8] = {};
        if (slot >= 0) {
            const int64_t at = kv_slot_base(P, slot, h) * kElem<T>;
            if constexpr (kCodes<T>) {
                const int64_t sa = kv_scale_at(P, slot, h);
#pragma unroll
                for (int q = 0; q < 2; ++q) {
                    const uint32_t* w = (const uint32_t*)((const uint8_t*)(q ? P.v : P.k) + at + d);
                    const float s = (q ? P.v_scale : P.k_scale)[sa];
                    T::unpack(w[0], f[q]);
                    T::unpack(w[1], f[q] + 4);
#pragma unroll
                    for (int e = 0; e < 8; ++e) f[q][e] *= s;
                }
            } else {
#pragma unroll
                for (int q = 0; q < 2; ++q) {
                    const T* w = (const T*)((const uint8_t*)(q ? P.v : P.k) + at) + d;
                    load4(w, f[q]);
                    load4(w + 4, f[q] + 4);
                }
            }
        }
        const int64_t to = (int64_t)(t0 + t) * A.out_stride + h * P.hd + d;
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            TO* dst = (TO*)(q ? A.v : A.k) + to;
            store4(dst, f[q]);
            store4(dst + 4, f[q] + 4);
        }
    }
}

template <typename T>
void read_by_out(const KvRead& a, const KvPool& p, hipStream_t s) {
    const dim3 grid((unsigned)(((int64_t)a.total + kReadTokens - 1) / kReadTokens));
    if (a.out_dtype == kF32) hipLaunchKernelGGL((k_kv_read<T, float>), grid, dim3(256), 0, s, a, p);
    else if (a.out_dtype == kF16) hipLaunchKernelGGL((k_kv_read<T, _Float16>), grid, dim3(256), 0, s, a, p);
    else hipLaunchKernelGGL((k_kv_read<T, __bf16>), grid, dim3(256), 0, s, a, p);
}

}  // namespace

namespace sxq {

hipError_t launch_kv8_append(const KvAppend& all, const KvPool& p, hipStream_t s) {
    // tokens a launch: the grid (a workgroup for two KV pairs and for 8 or more query heads of a
    // token) may not pass 2^32 threads; a multiple of 16 only helps (a run cut in two at the border
    // is two launches, in order)
    const int64_t groups = (2 * p.nkv + 3) / 4 + (all.nh + 7) / 8;
    const int most = (int)std::max<int64_t>(16, std::min<int64_t>((int64_t)1 << 23, ((int64_t)1 << 23) / groups) & ~(int64_t)15);
    const size_t e = type_size(all.dtype);
    for (int64_t t0 = 0; t0 < all.n_tokens; t0 += most) {
        KvAppend a = all;
        a.n_tokens = (int)std::min<int64_t>(most, all.n_tokens - t0);
        a.qkv = (const char*)all.qkv + t0 * all.row_stride * e;
        if (all.pos) a.pos = all.pos + t0;
        a.slots = all.slots + t0;
        if (all.q_out) a.q_out = (char*)all.q_out + t0 * all.nh * p.hd * e;
        const hipError_t err = a.dtype == kF32   ? append_by_code<float>(a, p, s)
                               : a.dtype == kF16 ? append_by_code<_Float16>(a, p, s)
                                                 : append_by_code<__bf16>(a, p, s);
        if (err != hipSuccess) return err;
    }
    return hipSuccess;
}

hipError_t launch_kv_read(const KvRead& a, const KvPool& p, hipStream_t s) {
    if (p.dtype == kF32) read_by_out<float>(a, p, s);
    else if (p.dtype == kF16) read_by_out<_Float16>(a, p, s);
    else if (p.dtype == kBF16) read_by_out<__bf16>(a, p, s);
    else if (p.dtype == kI8) read_by_out<I8>(a, p, s);
    else read_by_out<E4M3>(a, p, s);
    return hipGetLastError();
}

}  // namespace sxq

extern "C" {

sxq_status sxq_kv_read(int device, const sxq_kv_pages* pages, const int32_t* cu, const int32_t* rows, const int32_t* start,
                       int n_ranges, int total, const int32_t* lens, int n_rows, const int32_t* table, int64_t table_stride,
                       int max_blocks, int out_dtype, void* k, void* v, int64_t out_stride, void* stream) {
    KvPool p;
    if (sxq_status st = kv_pool("kv_read", pages, total > 0, &p)) return st;
    if (out_dtype != kF32 && out_dtype != kF16 && out_dtype != kBF16)
        return fail(SXQ_ERR_DTYPE, "kv_read: out dtype %d (f32, f16 or bf16)", out_dtype);
    if (n_ranges < 0 || total < 0 || total > 1 << 27) return fail(SXQ_ERR_INVALID, "kv_read: %d ranges, %d entries (0..2^27)", n_ranges, total);
    const int64_t width = (int64_t)p.nkv * p.hd, unit = 16 / type_size(out_dtype);
    if (out_stride < width || out_stride % unit || out_stride > (int64_t)1 << 32)
        return fail(SXQ_ERR_SHAPE, "kv_read: out_stride %lld (a multiple of %lld elements, rows of %lld)", (long long)out_stride,
                    (long long)unit, (long long)width);
    if (n_rows < 1 || max_blocks < 1 || table_stride < max_blocks || (int64_t)max_blocks * p.page > 1 << 30)
        return fail(SXQ_ERR_INVALID, "kv_read: a table of %d rows of %d blocks, stride %lld", n_rows, max_blocks, (long long)table_stride);
    if (!rows && n_ranges > n_rows) return fail(SXQ_ERR_SHAPE, "kv_read: %d ranges over %d table rows", n_ranges, n_rows);
    if (total == 0 || n_ranges == 0) return SXQ_OK;
    if (!cu || !lens || !table || !k || !v) return fail(SXQ_ERR_INVALID, "kv_read: null pointer");
    if (((uintptr_t)k | (uintptr_t)v) & 15) return fail(SXQ_ERR_INVALID, "kv_read: k and v must be 16-byte aligned");
    DeviceGuard g(device);
    HIP_TRY(g.err, "hipSetDevice");
    KvRead a;
    a.cu = cu;
    a.rows = rows;
    a.start = start;
    a.lens = lens;
    a.table = table;
    a.n_ranges = n_ranges;
    a.total = total;
    a.n_rows = n_rows;
    a.max_blocks = max_blocks;
    a.table_stride = table_stride;
    a.out_dtype = out_dtype;
    a.k = k;
    a.v = v;
    a.out_stride = out_stride;
    HIP_TRY(launch_kv_read(a, p, (hipStream_t)stream), "kv_read");
    return SXQ_OK;
}

}  // extern "C"
