// sxq_paged_attn.hip -- attention of one new token per request over a paged cache
// (sxq_kv_attention; include/sxq.h states it).
#include <hip/hip_runtime.h>

#include <algorithm>

#include "../../include/sxq.h"
#include "sxq_abi.h"
#include "sxq_paged.h"
#include "sxq_paged_launch.h"
#include "sxq_quant_dev.h"
#include "sxq_sync_dev.h"

using namespace sxq;
using namespace sxq::abi;

namespace {

typedef float v4f __attribute__((ext_vector_type(4)));
typedef uint32_t v4u __attribute__((ext_vector_type(4)));
typedef uint32_t v2u __attribute__((ext_vector_type(2)));
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));

// ---- how the work is split ---------------------------------------------------------------
// Per KV head and 16 of its query heads, a query's tiles of 32 positions are cut evenly into
// items of at most `piece` tiles, one a workgroup, where piece is the total of all queries'
// tiles over attend_target(): the grid, target + n_q, needs no length, and ragged queries
// weigh on the card by their lengths.  Fewer than target queries have more than one item, and
// fewer than 2 * target items belong to those: so many partials and counters have a place.
// The last of a query's items to finish joins them.
// (One equal share of the line of all tiles a workgroup, whole queries and the ends of two,
// measured: 64 queries of 1000..16384 positions 259 us against 264; 16 of 256..2040, where a
// workgroup's second query waits for the end of its first, 32 against 20.)
constexpr int kTile = 32;
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
// Workgroups per KV head and 16 query heads that the card holds at once (four a CU at head
// widths up to 64, two up to 128, one above, by their registers).
inline int attend_slots(int nh, int nkv, int hd) {
    const int all = hd <= 64 ? 1024 : hd <= 128 ? 512 : 256;
    return std::max(1, all / (nkv * attend_head_tiles(nh, nkv)));
}
// Few queries (up to half the slots): all items (fewer than target + n_q) resident at once, no
// second round for a few.  Many: smaller items, dealt as workgroups finish.  Measured at 32 / 8
// heads of 128, 64 slots (us): 16 queries of 256..2040 positions by 48 / 64 / 256 pieces 19.5 /
// 21.0 / 27.9; 32 of 500..4000 by 33 / 128 / 256 51.1 / 58.2 / 55.7; one of 131071 by 64 / 128 /
// 256 104 / 114 / 122; 64 of 1000..16384 by 64 / 128 / 256 293 / 269 / 270, 256 of 100..3000
// 181 / 180 / 188.
// (never more split queries than counters have a place: kCountBytes)
inline int attend_target_max(int nh, int nkv, int hd) {
    const int counters = kCountBytes / 64 / (nkv * attend_head_tiles(nh, nkv));
    return std::max(1, std::min({kMaxItems, 2 * attend_slots(nh, nkv, hd), counters}));
}
inline int attend_target(int n_q, int nh, int nkv, int hd) {
    const int slots = attend_slots(nh, nkv, hd), most = attend_target_max(nh, nkv, hd);
    return n_q <= slots / 2 ? std::min(slots - n_q + 1, most) : most;
}
// A partial: {m, l} and the weighted sum of one head.
SXQ_HD size_t attend_part_floats(int hd) { return (size_t)hd + 4; }

SXQ_DEV int tiles_of(int len) { return (len + kTile - 1) / kTile; }  // (of -1, no query: 0)

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
    int first, tiles;  // this item's tiles of 32 positions
    int index, count;  // which item of the query, of how many
    int part0, slot;   // a split query's first partial and its counter
};

// The cut of every query, from all queries' tiles.
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
        const int tiles = tiles_of(len);
        n = max(1, ceil_div(tiles, piece));
        if (few && tiles <= kWholeTiles) n = 1;
        per = ceil_div(tiles, n);
        if (per <= 4 * kWaves) per = (per + kWaves - 1) / kWaves * kWaves;
        n = len < 0 ? 0 : max(1, ceil_div(tiles, max(per, 1)));
    }
};

// Item x of the launch, found by every wave from the lengths: false if there is none.
SXQ_DEV bool find_item(const KvAttend& A, const KvPool& P, int target, int x, Item& it) {
    int row, len;
    load_query(A, P, 0, row, len);
    int total = __builtin_amdgcn_readlane(wave_scan(tiles_of(len)), 63);
    for (int b0 = 64; b0 < A.n_q; b0 += 64) {
        int r, n;
        load_query(A, P, b0, r, n);
        total += __builtin_amdgcn_readlane(wave_scan(tiles_of(n)), 63);
    }
    const Cut cut(total, target);
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
            it.tiles = min(mine_per, tiles_of(it.len) - it.first);
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
        int v[3] = {tiles_of(len), 0, 0}, all[3];
        scan(v, all);
        total += all[0];
    }
    const Cut cut(total, target);
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
    it.tiles = min(per, tiles_of(it.len) - it.first);
    it.part0 = __builtin_amdgcn_readfirstlane(info.y);
    it.slot = __builtin_amdgcn_readfirstlane(info.z);
    return true;
}

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
    __shared__ float s_m[kWaves][16], s_l[kWaves][16];
    __shared__ __attribute__((aligned(16))) float s_acc[kWaves][16][HDP + 4];
    __shared__ v4f s_red[256];
    __shared__ bool s_last;

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
    if (!(A.n_q > kScanMax ? planned_item(A, P, blockIdx.x, it) : find_item(A, P, target, blockIdx.x, it))) return;

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
    l = head_sum(l);

    // the four waves' sums
    if (g == 0) {
        s_m[wave][r] = m;
        s_l[wave][r] = l;
    }
    __syncthreads();
    float M = s_m[0][r];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) M = fmaxf(M, s_m[w][r]);
    {
        const float f = m > -INFINITY ? exp2_fast(m - M) : 1.0f;  // (no weights, or NaN: as they are)
#pragma unroll
        for (int b = 0; b < BLK; ++b)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int e = 0; e < VW; ++e)
                    s_acc[wave][r][b * 16 * VW + (4 * g + i) * VW + e] = acc[b * VW + e][i] * f;
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
        float Mh = s_m[0][h], L = 0.0f;
#pragma unroll
        for (int w = 1; w < kWaves; ++w) Mh = fmaxf(Mh, s_m[w][h]);
        v4f v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            const float mw = s_m[w][h];
            L += s_l[w][h] * (mw > -INFINITY ? exp2_fast(mw - Mh) : 1.0f);
            v += *(const v4f*)&s_acc[w][h][c];
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
    if (!publish_and_count(counter, it.count, &s_last)) return;
    if (tid == 0) __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    constexpr int kFetch = 8;
    const int count = it.count;
    const __amdgpu_buffer_rsrc_t all = coherent_rsrc(parts + (size_t)it.part0 * step, 0xFFFFFFFFu);
    float* factor = &s_acc[0][0][0];  // [heads][kMaxItems]
    static_assert(sizeof s_acc >= 16 * kMaxItems * sizeof(float), "the factors fit the waves' sums");
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
                    if (lane == 0) s_l[q][wave] = L;
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
            s_red[tid] = v;
            __syncthreads();
            if (k0 == 0)
                for (int u = 1; u < sub; ++u) v += s_red[u * n_out + o];
        }
        if (k0 == 0 && o < n_out) store_out(A, it.b, (h0 + h) * hd + 4 * (o - h * per), v, s_l[h >> 2][h & 3], (TQ*)nullptr);
    }
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
    return kCountBytes + attend_plan_bytes(n_q) + 2 * (size_t)attend_target_max(nh, p.nkv, p.hd) * nh * attend_part_floats(p.hd) * sizeof(float);
}

hipError_t launch_kv_attend(const KvAttend& a, const KvPool& p, hipStream_t s) {
    const int target = attend_target(a.n_q, a.nh, p.nkv, p.hd);
    // (no more items than the table's width allows: workgroups that find none cost 1.4 us at
    // one query of 500 positions)
    const int64_t widest = (int64_t)a.n_q * (((int64_t)a.max_blocks * p.page + kTile * kMinTiles - 1) / (kTile * kMinTiles));
    const dim3 grid((unsigned)std::min<int64_t>(target + a.n_q, widest), p.nkv * attend_head_tiles(a.nh, p.nkv));
    if (a.n_q > kScanMax) hipLaunchKernelGGL(k_kv_attend_plan, dim3(1), dim3(1024), 0, s, a, p, target);
    if (p.dtype == kF32) attend_by_width<float, float>(a, p, grid, target, s);
    else if (p.dtype == kF16) attend_by_width<_Float16, _Float16>(a, p, grid, target, s);
    else if (a.q_dtype == kF32) attend_by_width<float, __bf16>(a, p, grid, target, s);
    else attend_by_width<__bf16, __bf16>(a, p, grid, target, s);
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
    if (n_rows < 1 || max_blocks < 1 || table_stride < max_blocks || (int64_t)max_blocks * p.page > 1 << 30)
        return fail(SXQ_ERR_INVALID, "kv_attention: a table of %d rows of %d blocks, stride %lld", n_rows, max_blocks, (long long)table_stride);
    if ((int64_t)n_q * max_blocks * p.page > (int64_t)1 << 35)
        return fail(SXQ_ERR_INVALID, "kv_attention: %d queries of up to %lld positions", n_q, (long long)max_blocks * p.page);
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
