// sxq_paged8_attn.hip -- attention of one new token per request over the 8-bit paged cache
// (sxq_kv_attention over SXQ_I8 and SXQ_E4M3; include/sxq.h states it).
#include <hip/hip_runtime.h>

#include <algorithm>

#include "../../include/sxq.h"
#include "sxq_abi.h"
#include "sxq_paged.h"
#include "sxq_paged8_dev.h"
#include "sxq_paged_split.h"

using namespace sxq;
using namespace sxq::abi;

namespace {

SXQ_DEV v4f mfma(v8bf a, v8bf b, v4f c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
SXQ_DEV v4f mfma(v8h a, v8h b, v4f c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }

constexpr int kHalves = 2;  // 16-position halves of a wave's tile
constexpr int kTile = 16 * kHalves;
inline int attend_places(int hd) { return hd <= 64 ? 1024 : hd <= 128 ? 512 : 256; }

// One item of 16 query heads (or fewer) of one KV head, as k_kv_attend: one pass over its keys and
// values, four waves each with its own running maximum, sum and weighted values in registers.
// Scores: A = 16 keys x 32 head elements, B = the queries' elements x 16 heads; the sum over
// elements may take them in any order, so lane (r = lane % 16, g = lane / 16) loads 16 codes of key r
// and makes two operands of them.  A half tile of 16 positions has one scale of keys and one of
// values, the same for all lanes: the first goes into the factor of the scores, the second into the
// weights before these are cut into bf16 parts (three under f32 queries, else two).  Lane (r, g) of the result holds head r at
// positions 4 g + i; the weights are used in those registers, so the lane loads HDP / 16 columns of
// the values 4 g + i, two of a column meeting in a register by byte permutes before they are widened.
// What bounds it: the keys' and values' bytes, 64 requests of 1000 to 16384 positions, 32 / 8 heads of 128
// in 153 us, 4.7 TB/s (two workgroups a CU for the registers; three are 151 there and 17.8 against 16 us for
// 16 requests of 256 to 2045; tiles of 64 positions a wave instead of 32: 153 and 18.5); 16 requests in
// 16 us, of which 6 are the bytes and the rest the launch, the first loads one after another and the join.
template <typename TQ, typename C, int HDP, bool FULL>
__global__ __launch_bounds__(256, HDP <= 64 ? 4 : HDP <= 128 ? 2 : 1) void k_kv8_attend(const KvAttend A, const KvPool P,
                                                                                         int target) {
    typedef typename Query<TQ>::M M;
    typedef typename Vec8<M>::T V8;
    typedef Operand<C, M> KeyOp;
    typedef Operand<C, __bf16> ValueOp;
    constexpr int H = kHalves, KS = HDP / 64, D = HDP / 16, VD = D / 4;  // VD: dwords of a lane's columns
    constexpr int QP = Query<TQ>::kQP, WP = sizeof(TQ) == 4 ? 3 : 2;  // parts of a query, of a weight
    __shared__ EndShared<HDP> end;

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r = lane & 15, g = lane >> 4;
    const int hd = FULL ? HDP : P.hd, G = A.nh / P.nkv;
    const int ht = attend_head_tiles(A.nh, P.nkv);
    const int kh = blockIdx.y / ht, h0 = kh * G + (blockIdx.y - kh * ht) * 16;
    const int heads = min(16, (kh + 1) * G - h0);
    const float scale2 = A.scale * 1.44269504088896340736f;
    const uint32_t ps = (uint32_t)P.pos_stride;
    const uint32_t kcol = 16 * g, koff = r * ps, vcol = D * r;
    const bool vin = FULL || (int)vcol < hd;
    uint32_t voff[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) voff[i] = (4 * g + i) * ps + (vin ? vcol : 0);
    const char* kpool = (const char*)P.k + (int64_t)kh * P.head_stride;
    const char* vpool = (const char*)P.v + (int64_t)kh * P.head_stride;
    const float* kscale = P.k_scale + (int64_t)kh * P.scale_head_stride;
    const float* vscale = P.v_scale + (int64_t)kh * P.scale_head_stride;

    Item it;
    if (!(A.n_q > kScanMax ? planned_item<kTile>(A, P, blockIdx.x, it) : find_item<kTile>(A, P, target, blockIdx.x, it))) return;

    // the queries: B operands, in the element order of the key loads
    const TQ* qrow = (const TQ*)A.q + (int64_t)it.b * A.q_stride + (int64_t)(h0 + min(r, heads - 1)) * hd;
    V8 qreg[QP][2 * KS];
    int qcol[2 * KS];
    bool qin[2 * KS];
#pragma unroll
    for (int s = 0; s < 2 * KS; ++s) {
        qcol[s] = 64 * (s >> 1) + 16 * g + 8 * (s & 1);
        qin[s] = FULL || qcol[s] < hd;
    }
    const float row_scale = scale2 * load_query<TQ>(qrow, qcol, qin, qreg, [](float v) { return head_max(v); });

    const int32_t* table = A.table + (int64_t)it.row * A.table_stride;
    const int t_last = (it.len + 15) / 16 - 1;  // the last half tile (16 positions) with a position
    const int t_end = min((it.first + it.tiles) * H, t_last + 1);
    // Wave w takes the tiles w, w + 4, ... of the segment.  Lane j holds the page (-1: absent) and the
    // scales of the wave's half tile j of a batch of 64, so that a tile waits for no load of theirs;
    // the next batch's pages are loaded when one begins, its scales two tiles later.
    const int t0 = it.first * H + wave * H, log_p = P.shift - 4, block_mask = (P.page >> kScaleShift) - 1;
    auto tile_of = [&](int batch) { return t0 + (batch * 64 + lane) / H * (kWaves * H) + (lane & (H - 1)); };
    auto page_batch = [&](int batch) {
        const int t = tile_of(batch);
        int id = -1;
        if (t < t_end) id = table[t >> log_p];
        return kv_page_ok(id, P.n_pages) ? id : -1;
    };
    auto scale_batch = [&](const float* scales, int batch, int id) {
        float s = 0.0f;
        if (id >= 0) s = scales[(int64_t)id * P.scale_page_stride + (tile_of(batch) & block_mask)];
        return s;
    };
    int pages = page_batch(0), pages_next = -1;
    float ks_lane = scale_batch(kscale, 0, pages), vs_lane = scale_batch(vscale, 0, pages), ks_next = 0.0f, vs_next = 0.0f;

    v4f acc[D];
#pragma unroll
    for (int d = 0; d < D; ++d) acc[d] = (v4f){0.f, 0.f, 0.f, 0.f};
    float m = -INFINITY, l = 0.0f;

    uint32_t kreg[H][KS][4], vreg[H][4][VD];
    int id[H];
    float ks[H], vs[H];
    int64_t at[H];
    auto place = [&](int t) {
#pragma unroll
        for (int h = 0; h < H; ++h)
            at[h] = max(id[h], 0) * P.page_stride + (int64_t)((uint32_t)(((t + h) * 16) & (P.page - 1)) * (uint64_t)ps);
    };
    auto load_k = [&]() {
#pragma unroll
        for (int h = 0; h < H; ++h)
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                v4u v;
                if constexpr (FULL) v = *(const v4u*)(kpool + at[h] + 64 * s + (koff + kcol));
                else v = *(const v4u*)(kpool + at[h] + (koff + ((int)(64 * s + kcol) < hd ? 64 * s + kcol : 0)));
#pragma unroll
                for (int e = 0; e < 4; ++e) kreg[h][s][e] = v[e];
            }
    };
    auto load_v = [&]() {
#pragma unroll
        for (int h = 0; h < H; ++h)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                typedef uint32_t vec __attribute__((ext_vector_type(VD == 1 ? 2 : VD)));
                const char* src = vpool + at[h] + voff[i];
                if constexpr (VD == 1) vreg[h][i][0] = *(const uint32_t*)src;
                else {
                    const vec v = *(const vec*)src;
#pragma unroll
                    for (int e = 0; e < VD; ++e) vreg[h][i][e] = v[e];
                }
            }
    };

    int t = t0, k = 0;  // the tile's first half, its number in the batch
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
#pragma unroll
        for (int h = 0; h < H; ++h) {
            ks[h] = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(ks_lane), k * H + h));
            vs[h] = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(vs_lane), k * H + h));
        }
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
                    const bool in = (int)(64 * s + kcol) < hd;
#pragma unroll
                    for (int e = 0; e < 4; ++e) kreg[h][s][e] = in ? kreg[h][s][e] : 0;
                }
#pragma unroll
                for (int f = 0; f < 2; ++f) {
                    const V8 key = __builtin_bit_cast(V8, KeyOp::eight(kreg[h][s][2 * f], kreg[h][s][2 * f + 1]));
#pragma unroll
                    for (int q = QP - 1; q >= 0; --q) c = mfma(key, qreg[q][2 * s + f], c);  // the small parts first
                }
            }
            const float factor = score_factor<TQ>(row_scale, ks[h]);
#pragma unroll
            for (int i = 0; i < 4; ++i) x[h][i] = c[i] * factor;
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
                ks_lane = ks_next;
                vs_lane = vs_next;
                pages_next = page_batch(++batch);
            } else if (k == 2) {
                ks_next = scale_batch(kscale, batch, pages_next);
                vs_next = scale_batch(vscale, batch, pages_next);
            }
#pragma unroll
            for (int h = 0; h < H; ++h) id[h] = __builtin_amdgcn_readlane(pages, k * H + h);
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
        const float base = m > -INFINITY ? m : 0.0f;
        float w[H][4];
#pragma unroll
        for (int h = 0; h < H; ++h)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                w[h][i] = exp2_fast(x[h][i] - base);
                l += w[h][i];
                w[h][i] *= vs[h];
            }
        // values that no weight belongs to may hold anything: zeros in their place
        if (partial)
#pragma unroll
            for (int h = 0; h < H; ++h)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const bool in = okh[h] && (t + h) * 16 + 4 * g + i < it.len;
#pragma unroll
                    for (int e = 0; e < VD; ++e) vreg[h][i][e] = in ? vreg[h][i][e] : 0;
                }
#pragma unroll
        for (int hh = 0; hh < H; hh += 2) {
            v8bf part[WP];
#pragma unroll
            for (int p = 0; p < WP; ++p)
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    float& v = w[hh + (j >> 2)][j & 3];
                    part[p][j] = (__bf16)v;
                    v -= (float)part[p][j];
                }
#pragma unroll
            for (int q = 0; q < VD; ++q) {
                uint32_t col[4][4];  // [pair of positions][column]
#pragma unroll
                for (int j = 0; j < 4; ++j)  // positions 2 j and 2 j + 1 of the lane's eight
                    ValueOp::columns(vreg[hh + (j >> 1)][2 * (j & 1)][q], vreg[hh + (j >> 1)][2 * (j & 1) + 1][q], col[j]);
#pragma unroll
                for (int p = WP - 1; p >= 0; --p)  // the small parts first
#pragma unroll
                    for (int c = 0; c < 4; ++c)
                        acc[4 * q + c] = mfma(__builtin_bit_cast(v8bf, (v4u){col[0][c], col[1][c], col[2][c], col[3][c]}), part[p], acc[4 * q + c]);
            }
        }
        if (more) load_v();
        t = next;
    }
    finish_item<TQ, HDP, D, 1>(A, it, hd, h0, heads, acc, m, l, end);
}

template <typename TQ, typename C>
void attend_by_width(const KvAttend& a, const KvPool& p, dim3 grid, int target, hipStream_t s) {
#define SXQ_AT(HDP, FULL) hipLaunchKernelGGL((k_kv8_attend<TQ, C, HDP, FULL>), grid, dim3(256), 0, s, a, p, target)
    if (p.hd == 64) SXQ_AT(64, true);
    else if (p.hd == 128) SXQ_AT(128, true);
    else if (p.hd == 256) SXQ_AT(256, true);
    else if (p.hd < 64) SXQ_AT(64, false);
    else if (p.hd < 128) SXQ_AT(128, false);
    else SXQ_AT(256, false);
#undef SXQ_AT
}
template <typename TQ>
void attend_by_code(const KvAttend& a, const KvPool& p, dim3 grid, int target, hipStream_t s) {
    if (p.dtype == kI8) attend_by_width<TQ, I8>(a, p, grid, target, s);
    else attend_by_width<TQ, E4M3>(a, p, grid, target, s);
}

}  // namespace

namespace sxq {

size_t kv8_attend_workspace(const KvPool& p, int n_q, int nh) {
    return kCountBytes + attend_plan_bytes(n_q) +
           2 * (size_t)attend_target_max(nh, p.nkv, attend_places(p.hd)) * nh * attend_part_floats(p.hd) * sizeof(float);
}

hipError_t launch_kv8_attend(const KvAttend& a, const KvPool& p, hipStream_t s) {
    const int target = attend_target(a.n_q, a.nh, p.nkv, attend_places(p.hd));
    // (no more items than the table's width allows: workgroups that find none cost time)
    const int64_t widest = (int64_t)a.n_q * (((int64_t)a.max_blocks * p.page + kTile * kMinTiles - 1) / (kTile * kMinTiles));
    const dim3 grid((unsigned)std::min<int64_t>(target + a.n_q, widest), p.nkv * attend_head_tiles(a.nh, p.nkv));
    if (a.n_q > kScanMax) hipLaunchKernelGGL(k_kv_attend_plan<kTile>, dim3(1), dim3(1024), 0, s, a, p, target);
    if (a.q_dtype == kF32) attend_by_code<float>(a, p, grid, target, s);
    else if (a.q_dtype == kF16) attend_by_code<_Float16>(a, p, grid, target, s);
    else attend_by_code<__bf16>(a, p, grid, target, s);
    return hipGetLastError();
}

}  // namespace sxq
