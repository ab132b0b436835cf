// sxq_paged_split.h -- what the paged attentions of one new token share: how a launch's work is
// divided into items, and how a workgroup's waves and a query's items are joined.
#pragma once
#include <algorithm>

#include "sxq_paged_launch.h"
#include "sxq_quant_dev.h"
#include "sxq_sync_dev.h"

namespace sxq {
namespace {

typedef float v4f __attribute__((ext_vector_type(4)));
typedef uint32_t v4u __attribute__((ext_vector_type(4)));
typedef uint32_t v2u __attribute__((ext_vector_type(2)));
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));

// ---- how the work is split ---------------------------------------------------------------
// Per KV head and 16 of its query heads, a query's tiles of TILE positions are cut evenly into
// items of at most `piece` tiles, one a workgroup, where piece is the total of all queries'
// tiles over attend_target(): the grid, target + n_q, needs no length, and ragged queries
// weigh on the card by their lengths.  Fewer than target queries have more than one item, and
// fewer than 2 * target items belong to those: so many partials and counters have a place.
// The last of a query's items to finish joins them.
// (One equal share of the line of all tiles a workgroup, whole queries and the ends of two,
// measured: 64 queries of 1000..16384 positions 259 us against 264; 16 of 256..2040, where a
// workgroup's second query waits for the end of its first, 32 against 20.)
constexpr int kWaves = 4;
constexpr int kMinTiles = 4;    // of an item: one a wave
constexpr int kMaxItems = 256;  // of one query
// With a card's worth of items this short (or shorter) latency counts: a join (publishing, an
// atomic, two loads in turn) is 3 us, and a CU takes in a tile for each wave in 1.2 us (16-bit,
// head width 128: 56 GB/s, whatever is in flight).  Queries up to kWholeTiles stay whole: one
// of 256 positions 6.7 us against 8.5 split, of 384 8.4 / 8.7 (f32, width 64), of 500 9.0 / 8.6.
constexpr int kFewTiles = 8;
constexpr int kWholeTiles = 12;
constexpr int kCountBytes = SXQ_KV_COUNTER_BYTES;  // 64 bytes a split query, KV head and 16 heads

SXQ_HD int attend_head_tiles(int nh, int nkv) { return (nh / nkv + 15) / 16; }
// Workgroups per KV head and 16 query heads that the card holds at once, of `all` in all.
inline int attend_slots(int nh, int nkv, int all) { return std::max(1, all / (nkv * attend_head_tiles(nh, nkv))); }
// Few queries (up to half the slots): all items (fewer than target + n_q) resident at once, no
// second round for a few.  Many: smaller items, dealt as workgroups finish.  Measured at 32 / 8
// heads of 128, 64 slots (us): 16 queries of 256..2040 positions by 48 / 64 / 256 pieces 19.5 /
// 21.0 / 27.9; 32 of 500..4000 by 33 / 128 / 256 51.1 / 58.2 / 55.7; one of 131071 by 64 / 128 /
// 256 104 / 114 / 122; 64 of 1000..16384 by 64 / 128 / 256 293 / 269 / 270, 256 of 100..3000
// 181 / 180 / 188.
// (never more split queries than counters have a place: kCountBytes)
inline int attend_target_max(int nh, int nkv, int all) {
    const int counters = kCountBytes / 64 / (nkv * attend_head_tiles(nh, nkv));
    return std::max(1, std::min({kMaxItems, 2 * attend_slots(nh, nkv, all), counters}));
}
inline int attend_target(int n_q, int nh, int nkv, int all) {
    const int slots = attend_slots(nh, nkv, all), most = attend_target_max(nh, nkv, all);
    return n_q <= slots / 2 ? std::min(slots - n_q + 1, most) : most;
}
// A partial: {m, l} and the weighted sum of one head.
SXQ_HD size_t attend_part_floats(int hd) { return (size_t)hd + 4; }

template <int TILE>
SXQ_DEV int tiles_of(int len) { return (len + TILE - 1) / TILE; }  // (of -1, no query: 0)

// Inclusive sum over the wave (row shifts, then the rows' last lanes broadcast onwards).
SXQ_DEV int wave_scan(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);
    return v;
}

// ceil(a / b), 0 <= a < 2^30, 0 < b < 2^30, without a branch: the first quotient from a
// reciprocal is off by at most 2^8, the second, of what that leaves, by one either way.
SXQ_DEV int ceil_div(int a, int b) {
    const float inv = __builtin_amdgcn_rcpf((float)b);
    const int q0 = (int)((float)a * inv), r0 = a - q0 * b;
    const int q1 = (int)((float)r0 * inv), r = r0 - q1 * b;
    return q0 + q1 + (r > b ? 2 : r > 0 ? 1 : r <= -b ? -1 : 0);
}

// Lane l's query of the block of 64 from b0: its table row and length (-1: none).
SXQ_DEV void load_query(const KvAttend& A, const KvPool& P, int b0, int& row, int& len) {
    const int b = b0 + (threadIdx.x & 63);
    len = A.lens[min(b, A.n_rows - 1)];  // a guess in flight with the row, which most often is b
    row = b < A.n_q ? (A.rows ? A.rows[b] : b) : -1;
    const bool live = (uint32_t)row < (uint32_t)A.n_rows;
    if (live && row != b) len = A.lens[row];
    len = live ? kv_clamp_len(len, A.max_blocks, P.shift) : -1;
}

struct Item {
    int b, row, len;   // query, its table row, its positions
    int first, tiles;  // this item's tiles
    int index, count;  // which item of the query, of how many
    int part0, slot;   // a split query's first partial and its counter
};

// The cut of every query, from all queries' tiles.
template <int TILE>
struct Cut {
    int piece;
    bool few;
    SXQ_DEV Cut(int total, int target) {
        const int p = ceil_div(total, target);
        few = p <= kFewTiles;
        piece = max(kMinTiles, p);
    }
    // n items (0: no query) of per tiles: the fewest of at most piece tiles, evenly (short ones:
    // as many for each wave)
    SXQ_DEV void operator()(int len, int& n, int& per) const {
        const int tiles = tiles_of<TILE>(len);
        n = max(1, ceil_div(tiles, piece));
        if (few && tiles <= kWholeTiles) n = 1;
        per = ceil_div(tiles, n);
        if (per <= 4 * kWaves) per = (per + kWaves - 1) / kWaves * kWaves;
        n = len < 0 ? 0 : max(1, ceil_div(tiles, max(per, 1)));
    }
};

// Item x of the launch, found by every wave from the lengths: false if there is none.
template <int TILE>
SXQ_DEV bool find_item(const KvAttend& A, const KvPool& P, int target, int x, Item& it) {
    int row, len;
    load_query(A, P, 0, row, len);
    int total = __builtin_amdgcn_readlane(wave_scan(tiles_of<TILE>(len)), 63);
    for (int b0 = 64; b0 < A.n_q; b0 += 64) {
        int r, n;
        load_query(A, P, b0, r, n);
        total += __builtin_amdgcn_readlane(wave_scan(tiles_of<TILE>(n)), 63);
    }
    const Cut<TILE> cut(total, target);
    int items0 = 0, single0 = 0, split0 = 0;  // over the queries before this block of 64
    for (int b0 = 0; b0 < A.n_q; b0 += 64) {
        if (b0) load_query(A, P, b0, row, len);
        int n, per;
        cut(len, n, per);
        const int incl = wave_scan(n);
        const uint64_t single = __ballot(n == 1), split = __ballot(n > 1);
        const uint64_t mine = __ballot(x >= items0 + incl - n && x < items0 + incl);
        if (mine) {
            const int src = __builtin_ctzll(mine);
            const uint64_t below = ((uint64_t)1 << src) - 1;
            it.b = b0 + src;
            it.row = __builtin_amdgcn_readlane(row, src);
            it.len = __builtin_amdgcn_readlane(len, src);
            it.count = __builtin_amdgcn_readlane(n, src);
            const int start = items0 + __builtin_amdgcn_readlane(incl, src) - it.count;
            const int mine_per = __builtin_amdgcn_readlane(per, src);
            it.index = x - start;
            it.first = it.index * mine_per;
            it.tiles = min(mine_per, tiles_of<TILE>(it.len) - it.first);
            it.part0 = start - single0 - __builtin_popcountll(single & below);
            it.slot = split0 + __builtin_popcountll(split & below);
            return true;
        }
        items0 += __builtin_amdgcn_readlane(incl, 63);
        single0 += __builtin_popcountll(single);
        split0 += __builtin_popcountll(split);
    }
    return false;
}

// Beyond kScanMax queries a launch of its own finds every query's items once (each workgroup's
// walk over all lengths would be n_q^2): in the workspace, first item [n_q + 1] and, of each
// query, {tiles an item, first partial, counter, -}.  us at 32 / 8 heads of 128: 300 queries of
// 200..1000 positions 145 -> 123, 1024 of 100..600 370 -> 228, 4096 of 50..200 2798 -> 480; at 64
// the launch and its hand-over (4) would cost more than the walk (0.2 a block of 64).
constexpr int kScanMax = 256;
SXQ_HD size_t attend_plan_bytes(int n_q) { return n_q <= kScanMax ? 0 : (((size_t)n_q + 1) * 4 + 255) / 256 * 256 + (size_t)n_q * 16; }
struct Plan {
    int* first;
    int4* info;
    SXQ_HD Plan(void* ws, int n_q)
        : first((int*)((char*)ws + kCountBytes)), info((int4*)((char*)ws + kCountBytes + (((size_t)n_q + 1) * 4 + 255) / 256 * 256)) {}
};

template <int TILE>
__global__ __launch_bounds__(1024) void k_kv_attend_plan(const KvAttend A, const KvPool P, int target) {
    __shared__ int red[3][16];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const Plan plan(A.ws, A.n_q);
    // Sums of a, b, c over the workgroup's threads up to this one, and of all.
    auto scan = [&](int (&v)[3], int (&all)[3]) {
#pragma unroll
        for (int k = 0; k < 3; ++k) v[k] = wave_scan(v[k]);
        __syncthreads();
        if (lane == 63)
#pragma unroll
            for (int k = 0; k < 3; ++k) red[k][wave] = v[k];
        __syncthreads();
#pragma unroll
        for (int k = 0; k < 3; ++k) {
            all[k] = 0;
            int before = 0;
            for (int w = 0; w < 16; ++w) {
                if (w == wave) before = all[k];
                all[k] += red[k][w];
            }
            v[k] += before;
        }
    };
    int row, len, total = 0;
    for (int b0 = 0; b0 < A.n_q; b0 += 1024) {
        load_query(A, P, b0 + 64 * wave, row, len);
        int v[3] = {tiles_of<TILE>(len), 0, 0}, all[3];
        scan(v, all);
        total += all[0];
    }
    const Cut<TILE> cut(total, target);
    int done[3] = {0, 0, 0};  // items, items of split queries, split queries
    for (int b0 = 0; b0 < A.n_q; b0 += 1024) {
        load_query(A, P, b0 + 64 * wave, row, len);
        int n, per;
        cut(len, n, per);
        int v[3] = {n, n > 1 ? n : 0, n > 1 ? 1 : 0}, all[3];
        const int own[3] = {v[0], v[1], v[2]};
        scan(v, all);
        const int b = b0 + tid;
        if (b < A.n_q) {
            plan.first[b] = done[0] + v[0] - own[0];
            plan.info[b] = make_int4(per, done[1] + v[1] - own[1], done[2] + v[2] - own[2], 0);
        }
#pragma unroll
        for (int k = 0; k < 3; ++k) done[k] += all[k];
    }
    if (tid == 0) plan.first[A.n_q] = done[0];
}

template <int TILE>
SXQ_DEV bool planned_item(const KvAttend& A, const KvPool& P, int x, Item& it) {
    const Plan plan(A.ws, A.n_q);
    if (x >= plan.first[A.n_q]) return false;
    const int lane = threadIdx.x & 63;
    int lo = 0, n = A.n_q;  // the last query whose first item is at most x, 64 a step
    while (n > 1) {
        const int step = (n + 63) / 64, at = lane * step;
        const int k = __builtin_popcountll(__ballot(at < n && plan.first[lo + min(at, n - 1)] <= x)) - 1;
        lo += k * step;
        n = min(step, n - k * step);
    }
    lo = __builtin_amdgcn_readfirstlane(lo);
    const int4 info = plan.info[lo];
    const int start = __builtin_amdgcn_readfirstlane(plan.first[lo]);
    it.b = lo;
    it.row = __builtin_amdgcn_readfirstlane(A.rows ? A.rows[lo] : lo);
    it.len = __builtin_amdgcn_readfirstlane(kv_clamp_len(A.lens[it.row], A.max_blocks, P.shift));
    it.count = __builtin_amdgcn_readfirstlane(plan.first[lo + 1]) - start;
    it.index = x - start;
    const int per = __builtin_amdgcn_readfirstlane(info.x);
    it.first = it.index * per;
    it.tiles = min(per, tiles_of<TILE>(it.len) - it.first);
    it.part0 = __builtin_amdgcn_readfirstlane(info.y);
    it.slot = __builtin_amdgcn_readfirstlane(info.z);
    return true;
}

// Exchanges lanes 32..63 of a with lanes 0..31 of b; odd 16-lane rows of a with even ones of b.
SXQ_DEV void swap32(float& a, float& b) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(a), __float_as_uint(b), false, false);
    a = __uint_as_float(r[0]);
    b = __uint_as_float(r[1]);
}
SXQ_DEV void swap16(float& a, float& b) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(a), __float_as_uint(b), false, false);
    a = __uint_as_float(r[0]);
    b = __uint_as_float(r[1]);
}
// Over the four lanes of one head (lane % 16).
SXQ_DEV float head_max(float v) {
    float a = v, b = v;
    swap32(a, b);
    v = a = b = fmaxf(a, b);
    swap16(a, b);
    return fmaxf(a, b);
}
SXQ_DEV float head_sum(float v) {
    float a = v, b = v;
    swap32(a, b);
    v = a + b;
    a = b = v;
    swap16(a, b);
    return a + b;
}
// 8 bytes coherent at agent scope, as load16_coherent.
SXQ_DEV float2 load8_coherent(__amdgpu_buffer_rsrc_t r, uint32_t off) {
    typedef float f2 __attribute__((ext_vector_type(2)));
    const f2 v = __builtin_bit_cast(f2, __builtin_amdgcn_raw_buffer_load_b64(r, off, 0, 16));
    return make_float2(v.x, v.y);
}
SXQ_DEV float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// Four columns of an output row: the weighted sum over the weights' sum, zeros without any.
template <typename TQ>
SXQ_DEV void store_out(const KvAttend& A, int b, int64_t at, v4f v, float l, TQ*) {
    typedef TQ v4 __attribute__((ext_vector_type(4)));
    v4 o;
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = from_f32<TQ>(v[e] * inv);
    *(v4*)((TQ*)A.out + (int64_t)b * A.out_stride + at) = o;
}

// What a workgroup's waves hold at an item's end: per wave the running maximum m and sum l of its
// 16 heads, and the weighted values acc[b * VW + e][i] of head lane % 16, column b * 16 VW + (4 g +
// i) VW + e (g = lane / 16).  Added up, and written out, or published as the item's partial, which
// the last of the query's items joins with the others.
template <int HDP>
struct EndShared {
    float m[kWaves][16], l[kWaves][16];
    __attribute__((aligned(16))) float acc[kWaves][16][HDP + 4];
    v4f red[256];
    bool last;
};
template <typename TQ, int HDP, int VW, int BLK>
SXQ_DEV void finish_item(const KvAttend& A, const Item& it, int hd, int h0, int heads, v4f (&acc)[BLK * VW], float m, float l,
                         EndShared<HDP>& S) {
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r = lane & 15, g = lane >> 4;
    l = head_sum(l);

    // the four waves' sums
    if (g == 0) {
        S.m[wave][r] = m;
        S.l[wave][r] = l;
    }
    __syncthreads();
    float M = S.m[0][r];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) M = fmaxf(M, S.m[w][r]);
    {
        const float f = m > -INFINITY ? exp2_fast(m - M) : 1.0f;  // (no weights, or NaN: as they are)
#pragma unroll
        for (int b = 0; b < BLK; ++b)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int e = 0; e < VW; ++e)
                    S.acc[wave][r][b * 16 * VW + (4 * g + i) * VW + e] = acc[b * VW + e][i] * f;
    }
    __syncthreads();
    const int per = hd / 4, n_out = heads * per;  // four columns a thread
    // a partial's bytes; from item to item (all items of a query: below 2^27)
    const uint32_t pf = (uint32_t)(attend_part_floats(hd) * sizeof(float)), step = (uint32_t)A.nh * pf;
    char* parts = (char*)A.ws + kCountBytes + attend_plan_bytes(A.n_q) + (size_t)h0 * pf;
    const bool split = it.count > 1;
    const __amdgpu_buffer_rsrc_t mine =
        coherent_rsrc(parts + (size_t)(it.part0 + it.index) * step, heads * pf);
    for (int o = tid; o < n_out; o += 256) {
        const int h = o / per, c = 4 * (o - h * per);
        float Mh = S.m[0][h], L = 0.0f;
#pragma unroll
        for (int w = 1; w < kWaves; ++w) Mh = fmaxf(Mh, S.m[w][h]);
        v4f v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            const float mw = S.m[w][h];
            L += S.l[w][h] * (mw > -INFINITY ? exp2_fast(mw - Mh) : 1.0f);
            v += *(const v4f*)&S.acc[w][h][c];
        }
        if (!split) {
            store_out(A, it.b, (h0 + h) * hd + c, v, L, (TQ*)nullptr);
        } else {
            store16_coherent(mine, h * pf + 16 + 4 * c, make_float4(v[0], v[1], v[2], v[3]));
            if (c == 0) store16_coherent(mine, h * pf, make_float4(Mh, L, 0.f, 0.f));
        }
    }
    if (!split) return;
    // The last of the query's items to arrive joins them, in their order.  The loads go out
    // first -- up to kFetch partials of four columns a thread (the items dealt over the threads
    // that share them), then {m, l} of the wave's heads, every fourth, over all items -- and the
    // latter give the items' factors, through LDS, while the partials are in flight.
    unsigned* counter = (unsigned*)A.ws + ((size_t)it.slot * gridDim.y + blockIdx.y) * 16;
    const int sub = n_out < 256 ? 256 / n_out : 1;  // threads that share four columns
    const int k0 = n_out < 256 ? tid / n_out : 0, o_first = tid - k0 * n_out;
    const int h_first = min(o_first, n_out - 1) / per;
    if (!publish_and_count(counter, it.count, &S.last)) return;
    if (tid == 0) __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    constexpr int kFetch = 8;
    const int count = it.count;
    const __amdgpu_buffer_rsrc_t all = coherent_rsrc(parts + (size_t)it.part0 * step, 0xFFFFFFFFu);
    float* factor = &S.acc[0][0][0];  // [heads][kMaxItems]
    static_assert(sizeof(S.acc) >= 16 * kMaxItems * sizeof(float), "the factors fit the waves' sums");
    bool first = true;
    for (int o0 = 0; o0 < n_out; o0 += 256) {
        const int o = o_first + o0, oc = min(o, n_out - 1), h = o0 ? oc / per : h_first;
        const uint32_t from = h * pf + 16 + 16 * (oc - h * per);
        v4f v = {0.f, 0.f, 0.f, 0.f};
        for (int i0 = 0; i0 < count; i0 += kFetch * sub) {
            float4 p[kFetch];  // (past the last item it repeats, without effect)
#pragma unroll
            for (int u = 0; u < kFetch; ++u) p[u] = load16_coherent(all, from + min(i0 + k0 + u * sub, count - 1) * step);
            if (first) {
                first = false;
                float mx[4], sum[4];
#pragma unroll
                for (int q = 0; q < 4; ++q) mx[q] = -INFINITY, sum[q] = 0.0f;
                for (int i = lane; i < count; i += 64) {
                    float2 ml[4];
#pragma unroll
                    for (int q = 0; q < 4; ++q) ml[q] = load8_coherent(all, min(wave + kWaves * q, heads - 1) * pf + i * step);
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        factor[(wave + kWaves * q) * kMaxItems + i] = ml[q].x;
                        const float mn = fmaxf(mx[q], ml[q].x);
                        const float up = mx[q] > -INFINITY ? exp2_fast(mx[q] - mn) : 1.0f;
                        sum[q] = sum[q] * up + ml[q].y * (ml[q].x > -INFINITY ? exp2_fast(ml[q].x - mn) : 1.0f);
                        mx[q] = mn;
                    }
                }
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const float Mh = wave_max_rows(mx[q]);
                    const float L = wave_sum_rows(sum[q] * (mx[q] > -INFINITY ? exp2_fast(mx[q] - Mh) : 1.0f));
                    if (lane == 0) S.l[q][wave] = L;
                    mx[q] = Mh;
                }
                for (int i = lane; i < count; i += 64)
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        float* f = factor + (wave + kWaves * q) * kMaxItems + i;
                        *f = *f > -INFINITY ? exp2_fast(*f - mx[q]) : 1.0f;
                    }
                __syncthreads();
            }
#pragma unroll
            for (int u = 0; u < kFetch; ++u) {
                const int n = i0 + k0 + u * sub;
                const float f = factor[h * kMaxItems + min(n, count - 1)];
                if (n < count) v += (v4f){p[u].x * f, p[u].y * f, p[u].z * f, p[u].w * f};
            }
        }
        if (sub > 1) {
            S.red[tid] = v;
            __syncthreads();
            if (k0 == 0)
                for (int u = 1; u < sub; ++u) v += S.red[u * n_out + o];
        }
        if (k0 == 0 && o < n_out) store_out(A, it.b, (h0 + h) * hd + 4 * (o - h * per), v, S.l[h >> 2][h & 3], (TQ*)nullptr);
    }
}


}  // namespace
}  // namespace sxq
