// sxq_paged_attn.hip -- attention of one new token per request over a paged cache
// (sxq_kv_attention; include/sxq.h states it).
#include <hip/hip_runtime.h>

#include <algorithm>

#include "../../include/sxq.h"
#include "sxq_abi.h"
#include "sxq_paged.h"
#include "sxq_paged_launch.h"
#include "sxq_paged_split.h"

using namespace sxq;
using namespace sxq::abi;

namespace {

constexpr int kTile = 32;
// Workgroups that the card holds at once: four a CU at head widths up to 64, two up to 128, one
// above, by their registers.
inline int attend_places(int hd) { return hd <= 64 ? 1024 : hd <= 128 ? 512 : 256; }

// ---- the matrix operands of each page type -----------------------------------------------
// Scores: A = 16 keys x k head elements, B = the queries' k elements x 16 heads; the sum over
// k may take the elements in any order, so lane (r = lane % 16, g = lane / 16) simply loads 16
// bytes of key r.  A lane of the result holds head r of positions 4 g + i.  Weighted values:
// A = 16 value columns x positions, B = the weights, positions x 16 heads, where again any
// order of the positions does: the weights are used in the registers the scores came in, and
// lane (r, g) loads VW columns of the rows 4 g + i.  16-bit values then want two positions in
// a register where the load gave two columns: one byte permute per result register.
// Result: head r, columns of r' = 4 g + i.
template <typename T>
struct PageOps;

template <>
struct PageOps<float> {
    static constexpr int kHalves = 1;  // 16-position halves of a wave's tile
    static constexpr int kWeightShift = 0;
};
template <>
struct PageOps<__bf16> {
    static constexpr int kHalves = 2;
    static constexpr int kWeightShift = 0;
    typedef v8bf V8;
    static SXQ_DEV v4f mfma(V8 a, V8 b, v4f c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
};
template <>
struct PageOps<_Float16> {
    static constexpr int kHalves = 2;
    // The weights times 2^13, numerator and denominator alike: the second f16 part of a weight
    // is then exact down to 2^-38 of the largest (f16's smallest step, 2^-24, would lose the
    // small weights of a long flat row).
    static constexpr int kWeightShift = 13;
    typedef v8h V8;
    static SXQ_DEV v4f mfma(V8 a, V8 b, v4f c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
};

template <typename T, int HDP>
struct Shape {
    static constexpr int kVW = sizeof(T) == 4 ? 4 : HDP / 16 < 8 ? HDP / 16 : 8;  // value columns a load
    static constexpr int kBlk = HDP / (16 * kVW);
    static constexpr int kD = HDP / 16;       // result registers (x 4) of a lane
    static constexpr int kKS = sizeof(T) == 4 ? HDP / 16 : HDP / 32;  // 16-byte key loads a lane and half
    static constexpr int kH = PageOps<T>::kHalves;
};

// One item of 16 query heads (or fewer) of one KV head: one pass over its keys and values, four
// waves each with its own running maximum m, sum l and weighted values in registers, a tile of
// 32 positions (16 of f32) at a time: scores and weighted values on the matrix cores, the next
// tile's keys in flight once the scores are out, its values once they are used; nothing of a
// tile goes through LDS.  The products cost 16 rows whatever the group size (6 % of the matrix
// cores' time at 5.4 TB/s), so the bound is HBM, or latency for little work.  Measured
// (32 / 8 heads of 128, bf16, us): 64 requests of 1000..16384 positions (1.44 GB) 268, 5.4 TB/s
// where a plain read of 3 GB reaches 6.2; one of 131071 (537 MB) 104; 16 of 256..2040 with f32
// queries (74 MB) 18.2; HBM traffic 1.012, 1.005 and 1.05 of the bytes asked for.  Of the 18
// about 3 are the launch and the loads of lengths and table in turn, 4 the end: partials out, an
// atomic, the join's loads.  Two tiles ahead rather than one (registers for two workgroups a CU
// either way) changed nothing.
// {m, l} and the sum: m is the maximum of scale * log2(e) * score (or
// 0 where none is above -inf), l and the sum carry the weights 2^(x - m + kWeightShift).
template <typename TQ, typename T, int HDP, bool FULL>
__global__ __launch_bounds__(256, HDP <= 64 ? 4 : HDP <= 128 ? 2 : 1) void k_kv_attend(const KvAttend A, const KvPool P,
                                                                                        int target) {
    typedef Shape<T, HDP> S;
    typedef PageOps<T> O;
    constexpr int H = S::kH, KS = S::kKS, VW = S::kVW, BLK = S::kBlk, D = S::kD;
    constexpr bool F32 = sizeof(T) == 4;
    constexpr int QP = F32 || sizeof(TQ) == 2 ? 1 : 3;  // 16-bit parts of a query element, exact together
    constexpr int WP = F32 ? 1 : sizeof(TQ) == 2 ? 2 : 3;  // of a weight (rounded at 2^-18, or 2^-22, of itself)
    __shared__ EndShared<HDP> end;

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r = lane & 15, g = lane >> 4;
    const int hd = FULL ? HDP : P.hd, G = A.nh / P.nkv;
    const int ht = attend_head_tiles(A.nh, P.nkv);
    const int kh = blockIdx.y / ht, h0 = kh * G + (blockIdx.y - kh * ht) * 16;
    const int heads = min(16, (kh + 1) * G - h0);
    const float scale2 = A.scale * 1.44269504088896340736f;
    // where this lane reads within a half tile's 16 positions (bytes): 16 of key r at kcol + 64 s,
    // and its columns of the values 4 g + i
    const uint32_t ps = (uint32_t)P.pos_stride * (uint32_t)sizeof(T), row_bytes = (uint32_t)hd * sizeof(T);
    const uint32_t kcol = 16 * g, koff = r * ps, vcol = VW * r * (uint32_t)sizeof(T);
    uint32_t voff[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) voff[i] = (4 * g + i) * ps;
    const char* kpool = (const char*)P.k + (int64_t)kh * P.head_stride * (int64_t)sizeof(T);
    const char* vpool = (const char*)P.v + (int64_t)kh * P.head_stride * (int64_t)sizeof(T);
    const int64_t page_bytes = P.page_stride * (int64_t)sizeof(T);

    Item it;
    if (!(A.n_q > kScanMax ? planned_item<kTile>(A, P, blockIdx.x, it) : find_item<kTile>(A, P, target, blockIdx.x, it))) return;

    // the queries: B operands, in the element order of the key loads
    const TQ* qrow = (const TQ*)A.q + (int64_t)it.b * A.q_stride + (int64_t)(h0 + min(r, heads - 1)) * hd;
    uint32_t qreg[QP][KS][4];
#pragma unroll
    for (int s = 0; s < KS; ++s) {
        const int col = (F32 ? 16 : 32) * s + (F32 ? 4 : 8) * g;
        const bool in = FULL || col < hd;
        const TQ* src = qrow + (in ? col : 0);
        if constexpr (QP == 1) {
            const v4u v = *(const v4u*)src;
#pragma unroll
            for (int e = 0; e < 4; ++e) qreg[0][s][e] = in ? v[e] : 0;
        } else {
            float f[8];
            *(v4f*)f = *(const v4f*)src;
            *(v4f*)(f + 4) = *(const v4f*)(src + 4);
#pragma unroll
            for (int q = 0; q < QP; ++q) {
                v8bf part;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    part[e] = (__bf16)(in ? f[e] : 0.0f);
                    f[e] -= (float)part[e];
                }
                const v4u u = __builtin_bit_cast(v4u, part);
#pragma unroll
                for (int e = 0; e < 4; ++e) qreg[q][s][e] = u[e];
            }
        }
    }

    const int32_t* table = A.table + (int64_t)it.row * A.table_stride;
    const int t_last = (it.len + 15) / 16 - 1;  // the last half tile (16 positions) with a position
    const int t_end = min((it.first + it.tiles) * (kTile / 16), t_last + 1);
    // Wave w takes the tiles w, w + 4, ... of the segment.  Lane j holds the page of the wave's
    // half tile j of a batch of 64 (-1: absent), so that a tile's addresses wait for no load;
    // the next batch is loaded when one begins.
    const int t0 = it.first * (kTile / 16) + wave * H, log_p = P.shift - 4;
    auto page_batch = [&](int batch) {
        const int t = t0 + (batch * 64 + lane) / H * (kWaves * H) + (lane & (H - 1));
        int id = -1;
        if (t < t_end) id = table[t >> log_p];
        return kv_page_ok(id, P.n_pages) ? id : -1;
    };
    int pages = page_batch(0), pages_next = -1;

    v4f acc[D];
#pragma unroll
    for (int d = 0; d < D; ++d) acc[d] = (v4f){0.f, 0.f, 0.f, 0.f};
    float m = -INFINITY, l = 0.0f;

    uint32_t kreg[H][KS][4], vreg[H][4][BLK][VW * sizeof(T) / 4];
    int id[H];
    // (scalar bases and 32-bit lane offsets: the loads take both as they are)
    int64_t at[H];
    auto place = [&](int t) {
#pragma unroll
        for (int h = 0; h < H; ++h)
            at[h] = max(id[h], 0) * page_bytes + (int64_t)((uint32_t)(((t + h) * 16) & (P.page - 1)) * (uint64_t)ps);
    };
    auto load_k = [&]() {
#pragma unroll
        for (int h = 0; h < H; ++h)
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                v4u v;
                if constexpr (FULL) v = *(const v4u*)(kpool + at[h] + 64 * s + (koff + kcol));
                else v = *(const v4u*)(kpool + at[h] + (koff + (64 * s + kcol < row_bytes ? 64 * s + kcol : 0)));
#pragma unroll
                for (int e = 0; e < 4; ++e) kreg[h][s][e] = v[e];
            }
    };
    auto load_v = [&]() {
#pragma unroll
        for (int h = 0; h < H; ++h)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int b = 0; b < BLK; ++b) {
                    constexpr uint32_t kBlkBytes = 16 * VW * sizeof(T);
                    const char* src;
                    if constexpr (FULL) src = vpool + at[h] + b * kBlkBytes + (voff[i] + vcol);
                    else src = vpool + at[h] + (voff[i] + (b * kBlkBytes + vcol < row_bytes ? b * kBlkBytes + vcol : 0));
                    if constexpr (VW * sizeof(T) == 16) {
                        const v4u v = *(const v4u*)src;
#pragma unroll
                        for (int e = 0; e < 4; ++e) vreg[h][i][b][e] = v[e];
                    } else {
                        const v2u v = *(const v2u*)src;
                        vreg[h][i][b][0] = v[0];
                        vreg[h][i][b][1] = v[1];
                    }
                }
    };

    int t = t0, k = 0;  // the tile's first half, its number in the batch
    auto ids = [&]() {
#pragma unroll
        for (int h = 0; h < H; ++h) id[h] = __builtin_amdgcn_readlane(pages, k * H + h);
    };
    if (t < t_end) {
        // the first tile's pages by scalar loads, which do not queue behind the card's other
        // vector loads
        typedef const __attribute__((address_space(4))) int32_t* scalar_ptr;
        const scalar_ptr st = (scalar_ptr)(uintptr_t)table;
#pragma unroll
        for (int h = 0; h < H; ++h) {
            const int page = st[min(t + h, t_last) >> log_p];
            id[h] = t + h <= t_last && kv_page_ok(page, P.n_pages) ? page : -1;
        }
        place(t);
        load_k();
        load_v();
        if (t + 64 / H * (kWaves * H) < t_end) pages_next = page_batch(1);
    }
    int batch = 1;
    while (t < t_end) {
        const int next = t + kWaves * H;
        const bool more = next < t_end;
        // scores
        float x[H][4];
        int okh[H];
#pragma unroll
        for (int h = 0; h < H; ++h) {
            okh[h] = id[h] >= 0;
            v4f c = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                if constexpr (!FULL) {
                    const bool in = 64 * s + kcol < row_bytes;
#pragma unroll
                    for (int e = 0; e < 4; ++e) kreg[h][s][e] = in ? kreg[h][s][e] : 0;
                }
                if constexpr (F32) {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(kreg[h][s][e]),
                                                                 __uint_as_float(qreg[0][s][e]), c, 0, 0, 0);
                } else {
                    const v4u kk = {kreg[h][s][0], kreg[h][s][1], kreg[h][s][2], kreg[h][s][3]};
#pragma unroll
                    for (int q = QP - 1; q >= 0; --q) {  // the small parts first
                        const v4u qq = {qreg[q][s][0], qreg[q][s][1], qreg[q][s][2], qreg[q][s][3]};
                        c = O::mfma(__builtin_bit_cast(typename O::V8, kk), __builtin_bit_cast(typename O::V8, qq), c);
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) x[h][i] = c[i] * scale2;
        }
        if constexpr (QP > 1) {
            // A query's lower part that is zero, or of the other sign, makes NaN of an infinite
            // key where the whole query gives an infinite score: the first part's product has it
            // (and is NaN where the score is).
            float sum = 0.0f;
#pragma unroll
            for (int h = 0; h < H; ++h)
#pragma unroll
                for (int i = 0; i < 4; ++i) sum += x[h][i];
            if (__any(sum != sum)) {
#pragma unroll
                for (int h = 0; h < H; ++h) {
                    v4f c = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int s = 0; s < KS; ++s) {
                        const v4u kk = {kreg[h][s][0], kreg[h][s][1], kreg[h][s][2], kreg[h][s][3]};
                        const v4u qq = {qreg[0][s][0], qreg[0][s][1], qreg[0][s][2], qreg[0][s][3]};
                        c = O::mfma(__builtin_bit_cast(typename O::V8, kk), __builtin_bit_cast(typename O::V8, qq), c);
                    }
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (x[h][i] != x[h][i]) x[h][i] = c[i] * scale2;
                }
            }
        }
        const bool cut = (t + H) * 16 > it.len;  // some position lies past the end
        bool absent = false;
#pragma unroll
        for (int h = 0; h < H; ++h) absent |= !okh[h];
        const bool partial = cut || absent;
        if (partial)
#pragma unroll
            for (int h = 0; h < H; ++h)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (!okh[h] || (t + h) * 16 + 4 * g + i >= it.len) x[h][i] = -INFINITY;
        if (more) {
            if (++k == 64 / H) {
                k = 0;
                pages = pages_next;
                pages_next = page_batch(++batch);
            }
            ids();
            place(next);
            load_k();
        }
        // the running maximum moves only where a score passes it
        float mx = x[0][0];
#pragma unroll
        for (int h = 0; h < H; ++h)
#pragma unroll
            for (int i = 0; i < 4; ++i) mx = fmaxf(mx, x[h][i]);
        if (__any(mx > m)) {
            const float mn = fmaxf(m, head_max(mx));
            const float al = m > -INFINITY ? exp2_fast(m - mn) : 1.0f;  // nothing but zeros before
            l *= al;
#pragma unroll
            for (int d = 0; d < D; ++d) acc[d] *= al;
            m = mn;
        }
        const float base = (m > -INFINITY ? m : 0.0f) - (float)O::kWeightShift;
        float w[H][4];
#pragma unroll
        for (int h = 0; h < H; ++h)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                w[h][i] = exp2_fast(x[h][i] - base);
                l += w[h][i];
            }
        // values that no weight belongs to may hold anything: zeros in their place
        if (partial)
#pragma unroll
            for (int h = 0; h < H; ++h)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const bool in = okh[h] && (t + h) * 16 + 4 * g + i < it.len;
#pragma unroll
                    for (int b = 0; b < BLK; ++b)
#pragma unroll
                        for (int e = 0; e < (int)(VW * sizeof(T) / 4); ++e) vreg[h][i][b][e] = in ? vreg[h][i][b][e] : 0;
                }
        if constexpr (F32) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int b = 0; b < BLK; ++b)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        acc[4 * b + e] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(vreg[0][i][b][e]), w[0][i],
                                                                              acc[4 * b + e], 0, 0, 0);
        } else {
            typename O::V8 part[WP];
#pragma unroll
            for (int p = 0; p < WP; ++p)
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    part[p][j] = (T)w[j >> 2][j & 3];
                    w[j >> 2][j & 3] -= (float)part[p][j];
                }
            typename O::V8 cols[D];
#pragma unroll
            for (int b = 0; b < BLK; ++b)
#pragma unroll
                for (int e = 0; e < VW; ++e) {
                    v4u a;
#pragma unroll
                    for (int j = 0; j < 4; ++j)  // positions 2 j and 2 j + 1 of the lane's eight
                        a[j] = __builtin_amdgcn_perm(vreg[j >> 1][2 * (j & 1) + 1][b][e / 2], vreg[j >> 1][2 * (j & 1)][b][e / 2],
                                                     e & 1 ? 0x07060302 : 0x05040100);
                    cols[b * VW + e] = __builtin_bit_cast(typename O::V8, a);
                }
#pragma unroll
            for (int p = WP - 1; p >= 0; --p)  // the small parts first; D products between two of one register
#pragma unroll
                for (int d = 0; d < D; ++d) acc[d] = O::mfma(cols[d], part[p], acc[d]);
        }
        if (more) load_v();
        t = next;
    }
    finish_item<TQ, HDP, VW, BLK>(A, it, hd, h0, heads, acc, m, l, end);
}

template <typename TQ, typename T>
void attend_by_width(const KvAttend& a, const KvPool& p, dim3 grid, int target, hipStream_t s) {
#define SXQ_AT(HDP, FULL) hipLaunchKernelGGL((k_kv_attend<TQ, T, HDP, FULL>), grid, dim3(256), 0, s, a, p, target)
    if (p.hd == 64) SXQ_AT(64, true);
    else if (p.hd == 128) SXQ_AT(128, true);
    else if (p.hd == 256) SXQ_AT(256, true);
    else if (p.hd < 64) SXQ_AT(64, false);
    else if (p.hd < 128) SXQ_AT(128, false);
    else SXQ_AT(256, false);
#undef SXQ_AT
}

}  // namespace

namespace sxq {

size_t kv_attend_workspace(const KvPool& p, int n_q, int nh) {
    return kCountBytes + attend_plan_bytes(n_q) + 2 * (size_t)attend_target_max(nh, p.nkv, attend_places(p.hd)) * nh * attend_part_floats(p.hd) * sizeof(float);
}

hipError_t launch_kv_attend(const KvAttend& a, const KvPool& p, hipStream_t s) {
    const int target = attend_target(a.n_q, a.nh, p.nkv, attend_places(p.hd));
    // (no more items than the table's width allows: workgroups that find none cost 1.4 us at
    // one query of 500 positions)
    const int64_t widest = (int64_t)a.n_q * (((int64_t)a.max_blocks * p.page + kTile * kMinTiles - 1) / (kTile * kMinTiles));
    const dim3 grid((unsigned)std::min<int64_t>(target + a.n_q, widest), p.nkv * attend_head_tiles(a.nh, p.nkv));
    if (a.n_q > kScanMax) hipLaunchKernelGGL(k_kv_attend_plan<kTile>, dim3(1), dim3(1024), 0, s, a, p, target);
    if (p.dtype == kF32) attend_by_width<float, float>(a, p, grid, target, s);
    else if (p.dtype == kF16) attend_by_width<_Float16, _Float16>(a, p, grid, target, s);
    else if (a.q_dtype == kF32) attend_by_width<float, __bf16>(a, p, grid, target, s);
    else attend_by_width<__bf16, __bf16>(a, p, grid, target, s);
    return hipGetLastError();
}

}  // namespace sxq

namespace {

// What sxq_kv_attention and sxq_kv_prefix_attention take alike, checked.
sxq_status check_attend(const char* who, const KvPool& p, const KvAttend& a, size_t need, size_t workspace_bytes) {
    const bool known = a.q_dtype == kF32 || a.q_dtype == kF16 || a.q_dtype == kBF16;
    if (kv_is8(p.dtype) ? !known : a.q_dtype != p.dtype && !(a.q_dtype == kF32 && p.dtype == kBF16))
        return fail(SXQ_ERR_DTYPE, "%s: queries of dtype %d over pages of dtype %d", who, a.q_dtype, p.dtype);
    if (a.n_q < 0 || a.n_q > 1 << 20 || a.nh < 1 || a.nh > 16384 || a.nh % p.nkv)
        return fail(SXQ_ERR_SHAPE, "%s: %d queries of %d heads over %d KV heads", who, a.n_q, a.nh, p.nkv);
    const int64_t width = (int64_t)a.nh * p.hd, unit = 16 / type_size(a.q_dtype);
    if (a.q_stride < width || a.out_stride < width || a.q_stride % unit || a.out_stride % unit)
        return fail(SXQ_ERR_SHAPE, "%s: q_stride %lld, out_stride %lld (multiples of %lld elements, rows of %lld)", who,
                    (long long)a.q_stride, (long long)a.out_stride, (long long)unit, (long long)width);
    if (a.n_rows < 1 || a.max_blocks < 1 || a.table_stride < a.max_blocks || (int64_t)a.max_blocks * p.page > 1 << 30)
        return fail(SXQ_ERR_INVALID, "%s: a table of %d rows of %d blocks, stride %lld", who, a.n_rows, a.max_blocks, (long long)a.table_stride);
    if ((int64_t)a.n_q * a.max_blocks * p.page > (int64_t)1 << 35)
        return fail(SXQ_ERR_INVALID, "%s: %d queries of up to %lld positions", who, a.n_q, (long long)a.max_blocks * p.page);
    if (!(a.scale - a.scale == 0.0f)) return fail(SXQ_ERR_INVALID, "%s: scale is not finite", who);
    if (a.n_q == 0) return SXQ_OK;
    if (!a.q || !a.lens || !a.table || !a.out || !a.ws) return fail(SXQ_ERR_INVALID, "%s: null pointer", who);
    if (((uintptr_t)a.q | (uintptr_t)a.out) & 15) return fail(SXQ_ERR_INVALID, "%s: q and out must be 16-byte aligned", who);
    if ((uintptr_t)a.ws & 255) return fail(SXQ_ERR_INVALID, "%s: the workspace must be 256-byte aligned", who);
    if (workspace_bytes < need)
        return fail(SXQ_ERR_INVALID, "%s: a workspace of %zu bytes, %zu needed", who, workspace_bytes, need);
    return SXQ_OK;
}

sxq_status workspace_of(const char* who, const sxq_kv_pages* pages, int n_q, int n_heads, bool prefix, size_t* bytes) {
    if (!bytes) return fail(SXQ_ERR_INVALID, "%s: null output", who);
    KvPool p;
    if (sxq_status st = kv_pool(who, pages, false, &p)) return st;
    if (prefix && !kv_is8(p.dtype)) return fail(SXQ_ERR_DTYPE, "%s: pages of dtype %d (int8 or e4m3)", who, p.dtype);
    if (n_q < 0 || n_q > 1 << 20 || n_heads < 1 || n_heads > 16384 || n_heads % p.nkv)
        return fail(SXQ_ERR_SHAPE, "%s: %d queries of %d heads over %d KV heads", who, n_q, n_heads, p.nkv);
    *bytes = prefix ? kv8_prefix_workspace(p, n_q, n_heads)
             : kv_is8(p.dtype) ? kv8_attend_workspace(p, n_q, n_heads) : kv_attend_workspace(p, n_q, n_heads);
    return SXQ_OK;
}

}  // namespace

extern "C" {

sxq_status sxq_kv_attention_workspace(const sxq_kv_pages* pages, int n_q, int n_heads, size_t* bytes) {
    return workspace_of("kv_attention_workspace", pages, n_q, n_heads, false, bytes);
}

sxq_status sxq_kv_prefix_attention_workspace(const sxq_kv_pages* pages, int n_q, int n_heads, size_t* bytes) {
    return workspace_of("kv_prefix_attention_workspace", pages, n_q, n_heads, true, bytes);
}

sxq_status sxq_kv_attention(int device, const sxq_kv_pages* pages, int q_dtype, const void* q, int64_t q_stride,
                            int n_q, int n_heads, const int32_t* rows, const int32_t* lens, int n_rows,
                            const int32_t* table, int64_t table_stride, int max_blocks, float scale, void* out,
                            int64_t out_stride, void* workspace, size_t workspace_bytes, void* stream) {
    KvPool p;
    if (sxq_status st = kv_pool("kv_attention", pages, n_q > 0, &p)) return st;
    const KvAttend a = {q,      q_stride,     q_dtype, n_q, n_heads,    rows,     lens, table, n_rows, max_blocks,
                        table_stride, scale, out,     out_stride, workspace};
    const bool is8 = kv_is8(p.dtype), sized = n_q > 0 && n_q <= 1 << 20 && n_heads > 0 && n_heads <= 16384 && n_heads % p.nkv == 0;
    const size_t need = !sized ? 0 : is8 ? kv8_attend_workspace(p, n_q, n_heads) : kv_attend_workspace(p, n_q, n_heads);
    if (sxq_status st = check_attend("kv_attention", p, a, need, workspace_bytes)) return st;
    if (!rows && n_q > n_rows) return fail(SXQ_ERR_SHAPE, "kv_attention: %d queries over %d table rows", n_q, n_rows);
    if (n_q == 0) return SXQ_OK;
    DeviceGuard g(device);
    HIP_TRY(g.err, "hipSetDevice");
    HIP_TRY(is8 ? launch_kv8_attend(a, p, (hipStream_t)stream) : launch_kv_attend(a, p, (hipStream_t)stream), "kv_attention");
    return SXQ_OK;
}

sxq_status sxq_kv_prefix_attention(int device, const sxq_kv_pages* pages, int q_dtype, const void* q, int64_t q_stride,
                                   int n_q, int n_heads, const int32_t* rows, const int32_t* pos, const int32_t* lens,
                                   int n_rows, const int32_t* table, int64_t table_stride, int max_blocks, float scale,
                                   void* out, int64_t out_stride, void* workspace, size_t workspace_bytes, void* stream) {
    KvPool p;
    if (sxq_status st = kv_pool("kv_prefix_attention", pages, n_q > 0, &p)) return st;
    if (!kv_is8(p.dtype)) return fail(SXQ_ERR_DTYPE, "kv_prefix_attention: pages of dtype %d (int8 or e4m3)", p.dtype);
    const KvAttend a = {q,      q_stride,     q_dtype, n_q, n_heads,    rows,     lens, table, n_rows, max_blocks,
                        table_stride, scale, out,     out_stride, workspace};
    const bool sized = n_q > 0 && n_q <= 1 << 20 && n_heads > 0 && n_heads <= 16384 && n_heads % p.nkv == 0;
    if (sxq_status st = check_attend("kv_prefix_attention", p, a, sized ? kv8_prefix_workspace(p, n_q, n_heads) : 0, workspace_bytes)) return st;
    if (n_q == 0) return SXQ_OK;
    if (!rows || !pos) return fail(SXQ_ERR_INVALID, "kv_prefix_attention: null pointer");
    DeviceGuard g(device);
    HIP_TRY(g.err, "hipSetDevice");
    HIP_TRY(launch_kv8_prefix(a, pos, p, (hipStream_t)stream), "kv_prefix_attention");
    return SXQ_OK;
}

}  // extern "C"
