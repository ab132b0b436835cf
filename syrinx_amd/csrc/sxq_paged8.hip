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
// The norm's sum stays among the lh lanes and no element changes lanes.  A row is loaded as it is and
// by every lane (those past the head's width read its first elements), so that several rows' loads are
// under way together.
template <typename TI>
struct RawRow {
    typedef TI v4t __attribute__((ext_vector_type(4), aligned(sizeof(TI))));
    typedef float v4s __attribute__((ext_vector_type(4), aligned(4)));
    v4t a, b;
    v4s c, s;
};
struct Lane {
    int o1, o2, o3;  // of the row's two vectors and the angles' one
    SXQ_DEV Lane(bool interleaved, int j, int half) {
        o1 = interleaved ? 8 * j : 4 * j;
        o2 = interleaved ? 8 * j + 4 : half + 4 * j;
        o3 = 4 * j;
    }
};
template <typename TI>
SXQ_DEV void load_row(const KvAppend& A, int t, int pos, int hid, int hd, const Lane& at, bool rot, RawRow<TI>& r) {
    typedef RawRow<TI> R;
    const TI* src = (const TI*)A.qkv + (int64_t)t * A.row_stride + (int64_t)hid * hd;
    r.a = *(const typename R::v4t*)(src + at.o1);
    r.b = *(const typename R::v4t*)(src + at.o2);
    if (rot) {
        const int64_t p = (int64_t)min(max(pos, 0), A.max_pos - 1) * (hd / 2) + at.o3;
        r.c = *(const typename R::v4s*)(A.cos + p);
        r.s = *(const typename R::v4s*)(A.sin + p);
    }
}
// The row's eight elements normalised (g: the weights) and rotated; zeros unless live.
template <typename TI>
SXQ_DEV void norm_rope(const KvAppend& A, int hd, int lh, bool live, bool norm, const float* g, bool rot, const RawRow<TI>& r, float* x) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        x[e] = live ? to_f32(r.a[e]) : 0.0f;
        x[4 + e] = live ? to_f32(r.b[e]) : 0.0f;
    }
    if (norm) {
        float ss = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) ss = fmaf(x[e], x[e], ss);
        for (int o = lh >> 1; o >= 1; o >>= 1) ss += __shfl_xor(ss, o, 64);
        // x / rms: a product with the rounded inverse rounds twice, and codes at a border move; its remainder,
        // which a fused product gives exactly, corrects it (Markstein's last step of a division; 8192 bf16
        // tokens of 32 + 16 heads of 128 take 49 us without it, 50 so and 54 by divisions).  Means outside
        // that step's range, zeros and infinities among them, are divided by.
        const float rms = sqrtf(ss / (float)hd + A.eps), inv = 1.0f / rms;
        if (__all(rms > 0x1p-100f && rms < 0x1p100f)) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float q = x[e] * inv;
                x[e] = fmaf(fmaf(-q, rms, x[e]), inv, q) * g[e];
            }
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = x[e] / rms * g[e];
        }
    }
    if (!rot) return;
    auto turn = [&](float& a, float& b, int e) {
        const float u = fmaf(a, r.c[e], -(b * r.s[e]));
        b = fmaf(b, r.c[e], a * r.s[e]);
        a = u;
    };
    if (A.interleaved)
#pragma unroll
        for (int e = 0; e < 4; ++e) turn(x[2 * e], x[2 * e + 1], e);
    else
#pragma unroll
        for (int e = 0; e < 4; ++e) turn(x[e], x[4 + e], e);
}

SXQ_HD int waves_a_unit(int lh) { return lh >= 16 ? 4 : lh == 8 ? 2 : 1; }

SXQ_DEV float wave_max(float v) {
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, 64));
    return v;
}

// The tokens of a call fall into runs: consecutive tokens at consecutive slots of one block of 16.
// A run's keys and values of one head are a unit: their rows in the registers of lh / 4 waves (one to
// four; NP passes of 64 / lh tokens each, eight elements a lane), the largest of each by a reduction
// and through LDS, the scales, the codes; where the block's scale has grown, its earlier codes after
// that.  A workgroup, of 4 waves / waves a unit heads, looks for the runs that begin among its `chunk`
// tokens.  The queries' heads are other workgroups of the launch (from kv_groups on), QT tokens and
// 256 / lh heads each.
// A code needs its block's largest element, so that a block's rows have to meet before any is stored: in
// registers, and each element is read and written once.  What bounds it: 8192 bf16 tokens of 32 + 16
// heads of 128 take 50 us, 185 MB at 3.7 TB/s (a large copy: 5.2), 1412 f32 ones 15.8, 61 MB at 3.9: memory,
// and the start of workgroups; a step's few tokens 4.7, where an empty launch takes 2: the loads of slots,
// rows and angles, which wait for each other.  (The queries by a launch of their own: 70 against 66 us
// for the 8192, before the keys' and values' part was as it is.)
template <typename TI, typename C, int NP, int QT>
__global__ __launch_bounds__(256) void k_kv8_append(const KvAppend A, const KvPool P, int lh, int chunk, int kv_groups, int q_groups) {
    __shared__ float2 s_amax[2][4];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), hd = P.hd;
    const int j = threadIdx.x & (lh - 1);
    const bool live = 8 * j < hd, rot = A.cos != nullptr;
    const Lane el(A.interleaved, live ? j : 0, hd / 2);
    const uint32_t slots = (uint32_t)P.n_pages << P.shift;
    RawRow<TI> raw[2][NP > QT / 2 ? NP : (QT + 1) / 2];
    float g[8];
    if ((int)blockIdx.x >= kv_groups) {
        const int b = blockIdx.x - kv_groups, t0 = b / q_groups * QT, hid = b % q_groups * (256 / lh) + (int)threadIdx.x / lh;
        const bool mine = live && hid < A.nh, norm = A.q_norm != nullptr;
        bool has[QT];
#pragma unroll
        for (int q = 0; q < QT; ++q) {
            const int t = min(t0 + q, A.n_tokens - 1);
            has[q] = (uint32_t)A.slots[t] < slots && t0 + q < A.n_tokens;
            load_row<TI>(A, t, rot ? A.pos[t] : 0, min(hid, A.nh - 1), hd, el, rot, raw[q & 1][q >> 1]);
        }
        if (norm) {
            load4(A.q_norm + el.o1, g);
            load4(A.q_norm + el.o2, g + 4);
        }
#pragma unroll
        for (int q = 0; q < QT; ++q) {
            float x[8];
            norm_rope(A, hd, lh, mine, norm, g, rot, raw[q & 1][q >> 1], x);
            if (!mine || !has[q]) continue;
            TI* dst = (TI*)A.q_out + ((int64_t)(t0 + q) * A.nh + hid) * hd;
            store4(dst + el.o1, x);
            store4(dst + el.o2, x + 4);
        }
        return;
    }
    const int upw = waves_a_unit(lh), units = 4 / upw, groups = (P.nkv + units - 1) / units;  // a chunk's workgroups
    const int t0 = (int)blockIdx.x / groups * chunk, mine = (int)blockIdx.x % groups * units + wave / upw;
    const bool unit = mine < P.nkv;
    const int head = min(mine, P.nkv - 1), part = wave % upw;
    const bool norm = A.k_norm != nullptr;
    if (norm) {
        load4(A.k_norm + el.o1, g);
        load4(A.k_norm + el.o2, g + 4);
    }

    // lane i: token t0 - 1 + i
    const int ti = t0 - 1 + lane;
    const bool there = ti >= 0 && ti < A.n_tokens;
    const int slot = there ? A.slots[ti] : -1, at_pos = there && rot ? A.pos[ti] : 0;
    const int before = __shfl_up(slot, 1, 64);
    const bool in = (uint32_t)slot < slots;
    const bool goes_on = in && lane > 0 && slot == before + 1 && (slot & (kScaleBlock - 1)) != 0 && before >= 0;
    const uint64_t on = __ballot(goes_on);
    uint64_t firsts = __ballot(in && !goes_on && lane >= 1 && lane <= chunk);  // (of the whole workgroup alike)
    const int per = 64 / lh, sub = part * per + lane / lh, all = upw * per;  // this lane's token of a pass, tokens a pass
    for (int turn = 0; firsts; ++turn) {
        const int i = __builtin_ctzll(firsts);
        firsts &= firsts - 1;
        const int t = t0 - 1 + i, first = __builtin_amdgcn_readlane(slot, i), o = first & (kScaleBlock - 1);
        // (bits i + 1 on of a run: at most 15, ended by the next block)
        const int len = 1 + __builtin_ctzll(~((on >> i) >> 1));
        const int64_t at = kv_scale_at(P, first, head), base = kv_slot_base(P, first, head);
        const float had[2] = {o ? P.k_scale[at] : 0.0f, o ? P.v_scale[at] : 0.0f};
        float x[2][NP][8], amax[2] = {0.0f, 0.0f};
#pragma unroll
        for (int p = 0; p < NP; ++p)
            if (p * all + part * per < len) {
                const int k = min(p * all + sub, len - 1);
                load_row<TI>(A, t + k, __shfl(at_pos, i + k, 64), A.nh + head, hd, el, rot, raw[0][p]);
                load_row<TI>(A, t + k, 0, A.nh + P.nkv + head, hd, el, false, raw[1][p]);
            }
#pragma unroll
        for (int p = 0; p < NP; ++p)
            if (p * all + part * per < len)
#pragma unroll
                for (int v = 0; v < 2; ++v) {
                    norm_rope(A, hd, lh, live && p * all + sub < len, norm && !v, g, rot && !v, raw[v][p], x[v][p]);
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const float a = fabsf(x[v][p][e]);
                        amax[v] = a < INFINITY ? fmaxf(amax[v], a) : amax[v];
                    }
                }
#pragma unroll
        for (int v = 0; v < 2; ++v) amax[v] = wave_max(amax[v]);
        if (upw > 1) {
            if (lane == 0) s_amax[turn & 1][wave] = make_float2(amax[0], amax[1]);
            __syncthreads();
            for (int w = 0; w < upw; ++w) {
                const float2 u = s_amax[turn & 1][wave - part + w];
                amax[0] = fmaxf(amax[0], u.x);
                amax[1] = fmaxf(amax[1], u.y);
            }
        }
        if (!unit) continue;
#pragma unroll
        for (int v = 0; v < 2; ++v) {
            uint8_t* const pool = (uint8_t*)(v ? P.v : P.k) + base;
            const float need = block_scale<C>(amax[v]);
            const bool grown = !(had[v] >= need);
            const float s = grown ? need : had[v], inv = 1.0f / s;
#pragma unroll
            for (int p = 0; p < NP; ++p) {
                const int k = p * all + sub;
                if (live && k < len) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) x[v][p][e] *= inv;
                    uint8_t* dst = pool + (int64_t)k * P.pos_stride;
                    *(uint32_t*)(dst + el.o1) = C::pack(x[v][p]);
                    *(uint32_t*)(dst + el.o2) = C::pack(x[v][p] + 4);
                }
            }
            if (!grown) continue;
            if (part == 0 && lane == 0) (v ? P.v_scale : P.k_scale)[at] = s;
            const float ratio = had[v] * inv;
            for (int k = sub; live && k < o; k += all) {
                uint32_t* b = (uint32_t*)(pool + (int64_t)(k - o) * P.pos_stride + 8 * j);
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
    // Few tokens: a workgroup for each (and head), whose latency is the call's.  Many: starting
    // workgroups costs 2 to 3 ns each, so they take more (8192 bf16 tokens of 32 + 16 heads of 128 by 1
    // / 16 / 32 tokens a KV workgroup and 1 / 4 / 4 a query one 139 / 51 / 49 us, 1412 f32 ones by 1 / 4 /
    // 16 / 32 29 / 21 / 15 / 16, 333 by 1 / 4 / 16 6.0 / 5.3 / 7.1); runs of one token, as in a step's map, are
    // taken one after another (16 of them by 1 / 4 / 16: 4.8 / 10 / 31).
    const int chunk = a.n_tokens <= 512 ? 1 : a.n_tokens <= 1024 ? 4 : a.n_tokens <= 4096 ? 16 : 32;
    const int qt = a.n_tokens <= 1024 ? 1 : 4;
    const int units = 4 / waves_a_unit(lh), q_groups = a.q_out ? (a.nh + 256 / lh - 1) / (256 / lh) : 0;
    const int64_t kv_groups = (int64_t)((a.n_tokens + chunk - 1) / chunk) * ((p.nkv + units - 1) / units);
    const dim3 grid((unsigned)(kv_groups + (int64_t)((a.n_tokens + qt - 1) / qt) * q_groups));
#define SXQ_AP(NP, QT) hipLaunchKernelGGL((k_kv8_append<TI, C, NP, QT>), grid, dim3(256), 0, s, a, p, lh, chunk, (int)kv_groups, q_groups)
    if (lh <= 16 && qt == 1) SXQ_AP(1, 1);
    else if (lh <= 16) SXQ_AP(1, 4);
    else if (qt == 1) SXQ_AP(2, 1);
    else SXQ_AP(2, 4);
#undef SXQ_AP
    return hipGetLastError();
}
template <typename TI>
hipError_t append_by_code(const KvAppend& a, const KvPool& p, hipStream_t s) {
    return p.dtype == kI8 ? append_by_width<TI, I8>(a, p, s) : append_by_width<TI, E4M3>(a, p, s);
}

// ---------------------------------------------------------------------------- read
// Eight elements of a page's row as they are loaded, and as f32 (zeros if there is no such position).
template <typename T>
struct Eight {
    typedef T v4t __attribute__((ext_vector_type(4)));
    v4t a, b;
    bool in;
    SXQ_DEV void load(const void* pool, int64_t at, const float*, int64_t, bool there) {
        const v4t* p = (const v4t*)((const T*)pool + at);
        in = there;
        a = p[0];
        b = p[1];
    }
    SXQ_DEV void widen(float* f) const {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            f[e] = in ? to_f32(a[e]) : 0.0f;
            f[4 + e] = in ? to_f32(b[e]) : 0.0f;
        }
    }
};
template <typename C>
struct EightCodes {
    uint32_t a, b;
    float scale;
    SXQ_DEV void load(const void* pool, int64_t at, const float* scales, int64_t sa, bool there) {
        typedef uint32_t v2 __attribute__((ext_vector_type(2)));
        const v2 w = *(const v2*)((const uint8_t*)pool + at);
        a = there ? w.x : 0;
        b = there ? w.y : 0;
        scale = scales[sa];
        if (!there) scale = 0.0f;
    }
    SXQ_DEV void widen(float* f) const {
        C::unpack(a, f);
        C::unpack(b, f + 4);
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] *= scale;
    }
};
template <>
struct Eight<I8> : EightCodes<I8> {};
template <>
struct Eight<E4M3> : EightCodes<E4M3> {};

// A workgroup's `tokens` entries (up to kReadTokens): their slots once (range by search, page by table) through
// LDS, then eight elements of K and V a thread at a time.  Up to kReadRanges ranges are read whole by
// every workgroup, so that a small call is four loads in turn, not a search's too.  What bounds it:
// 64 requests of 1000 to 16384 positions, 8 heads of 128, from int8 into bf16 in 416 us, the codes in and
// the values out at a copy's rate; 500 positions in 4.2.
constexpr int kReadTokens = 16, kReadRanges = 255, kReadAhead = 4;
template <typename T, typename TO>
__global__ __launch_bounds__(256) void k_kv_read(const KvRead A, const KvPool P, int tokens) {
    __shared__ int s_slot[kReadTokens], s_cu[kReadRanges + 1], s_row[kReadRanges], s_start[kReadRanges], s_len[kReadRanges];
    const int t0 = blockIdx.x * tokens, tid = threadIdx.x;
    const bool few = A.n_ranges <= kReadRanges;
    auto len_of = [&](int row) { return (uint32_t)row < (uint32_t)A.n_rows ? kv_clamp_len(A.lens[row], A.max_blocks, P.shift) : 0; };
    int end;
    if (few) {
        if (tid <= A.n_ranges) s_cu[tid] = A.cu[tid];
        if (tid < A.n_ranges) {
            const int row = A.rows ? A.rows[tid] : tid;
            s_row[tid] = row;
            s_start[tid] = A.start ? A.start[tid] : 0;
            s_len[tid] = len_of(row);
        }
        __syncthreads();
        end = min(A.total, s_cu[A.n_ranges]);
    } else {
        end = min(A.total, A.cu[A.n_ranges]);
    }
    if (t0 >= end) return;
    if (tid < tokens) {
        const int t = t0 + tid;
        int slot = -1;
        if (t < end) {
            const int i = few ? owner(s_cu, A.n_ranges, t) : owner(A.cu, A.n_ranges, t);
            const int row = few ? s_row[i] : A.rows ? A.rows[i] : i, len = few ? s_len[i] : len_of(row);
            const int64_t pos = (int64_t)(few ? s_start[i] : A.start ? A.start[i] : 0) + t - (few ? s_cu[i] : A.cu[i]);
            if (pos >= 0 && pos < len)
                slot = kv_slot(A.table[(int64_t)row * A.table_stride + (pos >> P.shift)], (int)pos, P.shift, P.n_pages);
        }
        s_slot[tid] = slot;
    }
    __syncthreads();
    const int per = P.hd / 8, row = per * P.nkv, n = min(tokens, end - t0) * row;
    // (loads of kReadAhead rounds before the first store, which may not pass them)
    for (int i0 = tid; i0 < n; i0 += 256 * kReadAhead) {
        Eight<T> x[kReadAhead][2];
        int64_t to[kReadAhead];
#pragma unroll
        for (int u = 0; u < kReadAhead; ++u) {
            const int i = min(i0 + 256 * u, n - 1);
            const int t = i / row, h = (i - t * row) / per, d = 8 * (i - t * row - h * per), slot = s_slot[t];
            to[u] = (int64_t)(t0 + t) * A.out_stride + h * P.hd + d;
            const int64_t at = slot >= 0 ? kv_slot_base(P, slot, h) + d : 0, sa = slot >= 0 ? kv_scale_at(P, slot, h) : 0;
#pragma unroll
            for (int q = 0; q < 2; ++q) x[u][q].load(q ? P.v : P.k, at, q ? P.v_scale : P.k_scale, sa, slot >= 0);
        }
#pragma unroll
        for (int u = 0; u < kReadAhead; ++u) {
            if (i0 + 256 * u >= n) break;
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                float f[8];
                x[u][q].widen(f);
                TO* dst = (TO*)(q ? A.v : A.k) + to[u];
                store4(dst, f);
                store4(dst + 4, f + 4);
            }
        }
    }
}

template <typename T>
void read_by_out(const KvRead& a, const KvPool& p, hipStream_t s) {
    // (few entries: a thousand pieces of eight a workgroup, one round of loads)
    const int64_t row = (int64_t)p.nkv * (p.hd / 8);
    const int tokens = a.total * row >= 1 << 20 ? kReadTokens : (int)std::max<int64_t>(1, std::min<int64_t>(kReadTokens, 256 * kReadAhead / row));
    const dim3 grid((unsigned)(((int64_t)a.total + tokens - 1) / tokens));
    if (a.out_dtype == kF32) hipLaunchKernelGGL((k_kv_read<T, float>), grid, dim3(256), 0, s, a, p, tokens);
    else if (a.out_dtype == kF16) hipLaunchKernelGGL((k_kv_read<T, _Float16>), grid, dim3(256), 0, s, a, p, tokens);
    else hipLaunchKernelGGL((k_kv_read<T, __bf16>), grid, dim3(256), 0, s, a, p, tokens);
}

}  // namespace

namespace sxq {

hipError_t launch_kv8_append(const KvAppend& all, const KvPool& p, hipStream_t s) {
    // tokens a launch: the grid (a workgroup or less for a KV head and for 8 query heads of a token) may not pass 2^32 threads; a multiple of 16 only helps (a run cut in two at the border
    // is two launches, in order)
    const int64_t groups = p.nkv + (all.nh + 7) / 8;
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
