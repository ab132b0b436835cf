// sxq_paged8_prefix.hip -- attention of several new tokens per request over the 8-bit paged cache,
// each over its own prefix (sxq_kv_prefix_attention; include/sxq.h states it).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "../../include/sxq.h"
#include "sxq_abi.h"
#include "sxq_paged.h"
#include "sxq_paged8_dev.h"
#include "sxq_paged_split.h"

using namespace sxq;
using namespace sxq::abi;

namespace {

typedef float v16f __attribute__((ext_vector_type(16)));

// ---- how the work is split ---------------------------------------------------------------
// Consecutive queries of one request make tiles of whole tokens, `rows` rows (a token and a head of the
// KV head's group) or fewer; a group of more heads than that is cut into parts of so many heads, a
// token a tile.  A unit is a KV head and such a part.  A tile's keys are taken `keys` at a time; tiles
// longer than one place's share of the card, of all tiles' keys, are cut along their keys, into
// pieces whose results a launch of its own joins.  A launch of one workgroup writes the tiles and
// pieces ("items") down, from the map's live entries alone, and the attention's workgroups go through them.
// Two kernels: `wide` tiles of 128 rows, whose waves share the keys through LDS, and `few` of 32, whose
// waves share the rows and divide the keys.
constexpr int kWideRows = 128, kFewRows = 32;
constexpr int kFewKeys = 128;  // a tile of keys: 32 a wave
SXQ_HD constexpr int keys_a_tile(int hd) { return hd <= 128 ? 64 : 32; }  // wide (registers)

struct Geometry {
    int rows, keys;                   // of a tile
    int group, parts, units, tokens;  // heads a KV head; parts of a group; units; tokens a tile
    int places, min_piece;            // items of one unit that the card holds at once; tiles of keys
    SXQ_HD Geometry(int nh, int nkv, int hd, bool few) {
        rows = few ? kFewRows : kWideRows;
        keys = few ? kFewKeys : keys_a_tile(hd);
        group = nh / nkv;
        parts = (group + rows - 1) / rows;
        units = nkv * parts;
        tokens = group < rows ? rows / group : 1;
        const int all = hd <= 128 ? 512 : 256;
        places = units < all ? all / units : 1;
        min_piece = few ? 1 : 4;
    }
};

struct TileItem {
    int token, count, row;  // first query, queries, table row
    int limit;              // the most positions that one of them sees
    int first, end;         // this piece's tiles of keys
    int part, pieces;       // where its result goes, of how many pieces (1: out)
};

struct CutTile {
    int token, count;  // as its items'
    int part, pieces;  // its first partial, how many
};

// The workspace: counts {items, tiles that are cut, their pieces, the first item's place}; items; the
// tiles that are cut; partials: per part and unit, {m, l} of each row, then the weighted sums.
struct PrefixPlan {
    int* counts;
    TileItem* item;
    CutTile* cut;
    float* partial;
    size_t bytes;
    SXQ_HD static size_t up(size_t v) { return (v + 255) / 256 * 256; }
    SXQ_HD PrefixPlan(void* ws, int n_q, int hd, const Geometry& g) {
        char* p = (char*)ws;
        const int most = item_room(n_q, g);
        counts = (int*)p;
        p += 256;
        item = (TileItem*)p;
        p += up(sizeof(TileItem) * (size_t)most);
        cut = (CutTile*)p;
        p += up(sizeof(CutTile) * (size_t)g.places);
        partial = (float*)p;
        p += 2 * (size_t)g.places * g.units * part_floats(g.rows, hd) * sizeof(float);
        bytes = (size_t)(p - (char*)ws);
    }
    // a tile each, and the pieces of cut ones (fewer than 2 * places, of fewer than `places` tiles: a tile of x
    // > 5/4 shares makes ceil(x) <= 8/5 x pieces, and all tiles are `places` shares)
    SXQ_HD static int item_room(int n_q, const Geometry& g) { return n_q + 2 * g.places; }
    SXQ_HD static size_t part_floats(int rows, int hd) { return (size_t)rows * (hd + 2); }
};

// The positions that a query sees, of its request's length and its position.
SXQ_DEV int seen_of(int len, int pos, int max_blocks, int shift) { return min(kv_clamp_len(len, max_blocks, shift) - 1, max(pos, -1)) + 1; }
SXQ_DEV int seen(const KvAttend& A, const int32_t* pos, const KvPool& P, int t, int row) {
    return seen_of(A.lens[row], pos[t], A.max_blocks, P.shift);
}

// A thousand queries at a time, a thread each (the next chunk's under way): where its run began and
// which tile it is in by ballots, the last two thousand tiles in LDS.  While there are no more than a
// thousand tiles they stay there until all queries are seen, so that a short call's tiles are cut where
// they are, and are written once, the last tile first.  More go to the end of the items' room, the last
// first too, and are cut from there a thousand at a time: the items of any number of them end before the
// tiles behind them begin.  80 queries 5.3 us, 1412 7.1: an empty launch and the loads of rows, lengths and
// positions, which wait for each other.  (Cut by what the map holds, not by its size: 4 tokens after 30000 in a
// map of 8192 entries take 46 us in all, whole 790.)
constexpr int kTilesKept = 1024, kTileRing = 2 * kTilesKept;
__global__ __launch_bounds__(1024) void k_kv8_prefix_plan(const KvAttend A, const int32_t* pos, const KvPool P, const Geometry g) {
    __shared__ __attribute__((aligned(16))) int s_wave[2][16];
    __shared__ int s_limit[kTileRing], s_end[kTileRing], s_token[kTileRing], s_row[kTileRing], s_cut;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const PrefixPlan plan(A.ws, A.n_q, P.hd, g);
    const int room = PrefixPlan::item_room(A.n_q, g);
    const uint64_t upto = ~(uint64_t)0 >> (63 - lane);
    auto tile = [&](int i) {
        const int k = i & (kTileRing - 1), limit = s_limit[k];
        return TileItem{s_token[k], s_end[k] - s_token[k], s_row[k], limit, 0, (limit + g.keys - 1) / g.keys, 0, 1};
    };
    if (tid == 0) s_cut = 0;
    bool kept = true;        // no tile is written yet
    int tiles = 0, run = 0;  // so far; where the run that reaches into the chunk began
    int row_next = tid < A.n_q ? A.rows[tid] : -1, before_next = tid > 0 && tid < A.n_q ? A.rows[tid - 1] : -1;
    int after_next = tid + 1 < A.n_q ? A.rows[tid + 1] : -1, pos_next = tid < A.n_q ? pos[tid] : -1;
    for (int c0 = 0; c0 < A.n_q; c0 += 1024) {
        const int t = c0 + tid, row = row_next, before = before_next, after = after_next, at_pos = pos_next;
        const bool live = (uint32_t)row < (uint32_t)A.n_rows;
        const int len = live ? A.lens[row] : 0;
        const int t2 = t + 1024;
        row_next = t2 < A.n_q ? A.rows[t2] : -1;
        before_next = t2 < A.n_q ? A.rows[t2 - 1] : -1;
        after_next = t2 + 1 < A.n_q ? A.rows[t2 + 1] : -1;
        pos_next = t2 < A.n_q ? pos[t2] : -1;
        s_limit[(tiles + tid) & (kTileRing - 1)] = 0;
        const uint64_t begins = __ballot(t < A.n_q && (t == 0 || before != row));
        if (lane == 0) s_wave[0][wave] = begins ? c0 + 64 * wave + 63 - __builtin_clzll(begins) : -1;
        __syncthreads();
        int start = run;
#pragma unroll
        for (int w = 0; w < 16; ++w) {
            const int begin = s_wave[0][w];
            start = max(start, w < wave ? begin : -1);
            run = max(run, begin);
        }
        if (begins & upto) start = c0 + 64 * wave + 63 - __builtin_clzll(begins & upto);
        const int in_tile = (t - start) % g.tokens;
        const bool first = live && in_tile == 0;
        const uint64_t firsts = __ballot(first);
        if (lane == 0) s_wave[1][wave] = __builtin_popcountll(firsts);
        __syncthreads();
        int at = tiles - 1 + __builtin_popcountll(firsts & upto), count = 0;  // this query's tile (tiles - 1: the last chunk's last)
#pragma unroll
        for (int w = 0; w < 16; ++w) {
            const int here = s_wave[1][w];
            at += w < wave ? here : 0;
            count += here;
        }
        at = live ? at & (kTileRing - 1) : -1;
        // the tile's most: a query less than the next one, as most are, need not say its own
        const int sees = live ? seen_of(len, at_pos, A.max_blocks, P.shift) : 0;
        const int next_at = __shfl_down(at, 1, 64), next_sees = __shfl_down(sees, 1, 64);
        if (live && (lane == 63 || next_at != at || sees > next_sees)) atomicMax(&s_limit[at], sees);
        if (live && (t + 1 == A.n_q || after != row || in_tile == g.tokens - 1)) s_end[at] = t + 1;
        if (first) {
            s_token[at] = t;
            s_row[at] = row;
        }
        __syncthreads();
        const int new_tiles = tiles + count;
        if (new_tiles > kTilesKept) {
            for (int i = (kept ? 0 : tiles - 1) + tid; i < new_tiles; i += 1024) plan.item[room - 1 - i] = tile(i);
            kept = false;
            __syncthreads();
        }
        tiles = new_tiles;
    }
    // Pieces: tiles longer than a place's share of all keys are cut into such shares (a tile a thread).
    auto scan = [&](int v, int turn, int& all) {  // the sum over the threads up to this one
        v = wave_scan(v);
        if (lane == 63) s_wave[turn][wave] = v;
        __syncthreads();
        int lower = 0;
        all = 0;
#pragma unroll
        for (int w = 0; w < 16; ++w) {
            const int here = s_wave[turn][w];
            lower += w < wave ? here : 0;
            all += here;
        }
        return v + lower;
    };
    int items = 0, pieces = 0, base = 0;
    // The items of `here` tiles, which lie in LDS from the ring's begin on; mine: tile here - 1 - tid.
    auto cut = [&](int here, const TileItem& mine, int piece) {
        const int n = tid < here ? kv_pieces(mine.end, piece) : 0;
        int both;
        const int upto_me = scan(n + (n > 1 ? n << 16 : 0), 1, both);  // items, and those of cut tiles
        const int part = pieces + (upto_me >> 16) - n, count = both & 0xFFFF;
        if (n > 1) plan.cut[atomicAdd(&s_cut, 1)] = CutTile{mine.token, mine.count, part, n};
        // (in the ring's second half: the items before the tile's, its first part, its pieces)
        int *const s_before = s_limit + kTilesKept, *const s_part = s_token + kTilesKept, *const s_pieces = s_end + kTilesKept;
        s_before[tid] = (upto_me & 0xFFFF) - n;
        s_part[tid] = part;
        s_pieces[tid] = n;
        __syncthreads();
        for (int i = tid; i < count; i += 1024) {  // an item a thread
            const int o = owner(s_before, here, i), j = i - s_before[o];
            TileItem it = tile(here - 1 - o);
            const int64_t all = it.end;
            it.pieces = s_pieces[o];
            it.part = it.pieces > 1 ? s_part[o] + j : 0;
            it.first = (int)(all * j / it.pieces);
            it.end = (int)(all * (j + 1) / it.pieces);
            plan.item[items + i] = it;
        }
        items += count;
        pieces += both >> 16;
    };
    // (2^30 positions a tile at most, 2^35 of all: 2^30 tiles of 32 keys, and one a tile for its last)
    int work;
    if (kept) {
        const TileItem none{}, mine = tid < tiles ? tile(tiles - 1 - tid) : none;
        scan(mine.end, 0, work);
        cut(tiles, mine, max(g.min_piece, (work + g.places - 1) / g.places));
    } else {
        int keys = 0, longest = 0;
        for (int i = tid; i < tiles; i += 1024) {
            const int k = plan.item[room - tiles + i].end;
            keys += k;
            longest = max(longest, k);
        }
        scan(keys, 0, work);
        const int piece = max(g.min_piece, (work + g.places - 1) / g.places);
        if (!__syncthreads_or(kv_pieces(longest, piece) > 1)) {
            items = tiles;
            base = room - tiles;
        } else {
            for (int r0 = 0; r0 < tiles; r0 += 1024) {  // from the last tile back
                const int here = min(1024, tiles - r0);
                TileItem mine{};
                __syncthreads();  // (the readers of the tiles before these are done)
                if (tid < here) {
                    mine = plan.item[room - tiles + r0 + tid];
                    const int k = here - 1 - tid;
                    s_token[k] = mine.token;
                    s_end[k] = mine.token + mine.count;
                    s_row[k] = mine.row;
                    s_limit[k] = mine.limit;
                }
                __syncthreads();
                cut(here, mine, piece);
            }
        }
    }
    if (tid == 0) *(int4*)plan.counts = make_int4(items, s_cut, pieces, base);
}

// Item w of units * items, those of the last tile first (of one request the last queries see the most).
// The count and the item it most often is are loaded together.
SXQ_DEV bool item_of(const PrefixPlan& plan, int n_q, const Geometry& g, int64_t w, TileItem& it) {
    const int k = (int)(w / g.units);
    it = plan.item[min(k, PrefixPlan::item_room(n_q, g) - 1)];
    const int4 counts = *(const int4*)plan.counts;
    if (k >= counts.x) return false;
    if (counts.w) it = plan.item[counts.w + k];
    return true;
}

// ---- the attention -----------------------------------------------------------------------
SXQ_DEV v16f mfma32(v8bf a, v8bf b, v16f c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
SXQ_DEV v16f mfma32(v8h a, v8h b, v16f c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }

SXQ_DEV v4f mfma16(v8bf a, v8bf b, v4f c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
SXQ_DEV v4f mfma16(v8h a, v8h b, v4f c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }

// The other half of the wave's value.
SXQ_DEV float other_half(float v) {
    float a = v, b = v;
    swap32(a, b);
    return (threadIdx.x & 32) ? a : b;
}

// Into how many bf16 parts a weight is cut.  Tiles of few rows as the attention of one token does it; those
// of many rows into one under bf16 queries, off by 2^-8 of the weight, half a step of the output's own type:
// a chunk of 2048 after 30720 takes 1310 us so and 1730 by two, its outputs 1.81e-3 and 1.65e-3 off (of
// which the outputs' rounding is 1.65e-3).  (Few rows by one: 24.5 against 25.1 us for 16 drafts of 5.)
template <typename TQ, bool MANY>
constexpr int kWeightParts = sizeof(TQ) == 4 ? 3 : MANY && std::is_same_v<TQ, __bf16> ? 1 : 2;

// A tile of keys and values in LDS, 16-bit: keys [key][element], values [column][key], the 16-byte pieces of
// a row exchanged so that those of neighbouring rows lie on different banks.
template <int HDP>
struct Stage {
    static constexpr int kKeys = keys_a_tile(HDP), kBlocks = kKeys / kScaleBlock;
    __attribute__((aligned(16))) uint16_t k[kKeys * HDP], v[HDP * kKeys];
};
template <int HDP>
SXQ_DEV int k_swap(int key) {
    return HDP == 64 ? key >> 1 & 7 : key & 15;
}
template <int HDP>
SXQ_DEV int v_swap(int col) {
    return keys_a_tile(HDP) == 64 ? (col >> 1 & 7) ^ (col >> 4 & 1) : col >> 2 & 3;
}

// Whether a value scale goes into its weights' exponents, or multiplies the weights.  An exponent near the
// scale's is rounded twice, by up to 2^-18 of the weight each time: below what one bf16 part is off by, not
// below what two or three leave out.
template <typename TQ>
constexpr bool kScaleInExponent = kWeightParts<TQ, true> == 1;
// Whether a scale may do so: the weights then stay above what is flushed to zero down to 2^-66 of the
// largest, and below infinity.  Any other multiplies the values, where it takes nothing from the weights.
SXQ_DEV bool plain_scale(float s) { return s >= 0x1p-60f && s < 0x1p100f; }

// The first key of each column whose value is NaN.
template <int HDP>
struct Nans {
    int first[HDP], any;
};

// Tiles of 128 rows: a wave has 32 of them, its queries and weighted values in registers; the keys and
// values of a tile of keys are widened to 16 bits once for all of them, through LDS, two stages in turn,
// the next tile's codes under way in registers meanwhile.  Scores: A = 32 keys x 16 elements, B = the
// queries' elements x 32 rows, so that a lane has one row's scores for half of the keys (8 (i / 4) +
// 4 (lane / 32) + i % 4) and the softmax of a row is two lanes'; weighted values: A = 32 columns x 16 keys,
// B = the weights in the registers that the scores came in, the values' keys laid out in LDS to match.
// What bounds it: the matrix cores' products and the lanes' work on the weights (an exponential, the
// maximum, the sum, the rounding, the widening of the codes) take turns on a SIMD's two waves.  A chunk of 2048
// bf16 queries after 30720 positions, 32 / 8 heads of 128, takes 1290 us, 825 TFLOP/s (a large matrix product: 1217;
// 1415 on another card); f16 queries, weights in two parts, 1700; f32 ones, in two parts, weights in
// three, 2460.  Of a short prompt much is the beginning
// (tile, pages, scales, codes and queries, loads that wait for each other): a call of one tile of keys
// takes 9.5 us (f32 14.7), each further one of that item 2.1 (3.5).
template <typename TQ, typename C, int HDP, bool FULL>
__global__ __launch_bounds__(256, HDP <= 128 ? 2 : 1) void k_kv8_prefix(const KvAttend A, const int32_t* pos,
                                                                                                 const KvPool P, const Geometry geo) {
    typedef typename Query<TQ>::M M;
    typedef typename Vec8<M>::T V8;
    constexpr int QP = Query<TQ>::kQP, WP = kWeightParts<TQ, true>;
    constexpr bool kLift = kScaleInExponent<TQ>;
    constexpr int KS = HDP / 16, CT = HDP / 32;  // steps over the head's elements, tiles of 32 columns
    constexpr int kKeys = Stage<HDP>::kKeys, NB = Stage<HDP>::kBlocks, KT = kKeys / 32;
    constexpr int kRowPieces = HDP / 16, KP = kKeys * kRowPieces / 256;  // pieces of 16 codes a key; a thread's
    constexpr int VE = HDP == 64 ? 4 : 8;                                // keys of a thread's piece of values (by 4 columns)
    __shared__ Stage<HDP> stage[2];
    __shared__ Nans<HDP> s_nans[2];  // of this item and the last

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int col32 = lane & 31, hf = lane >> 5;
    const int hd = FULL ? HDP : P.hd;
    const PrefixPlan plan(A.ws, A.n_q, hd, geo);
    // (a negative scale is the positive one over negated queries: the running maximum wants factors
    // of 0 or more)
    const float scale2 = fabsf(A.scale) * 1.44269504088896340736f;
    const uint32_t flip = A.scale < 0.0f ? 0x80008000u : 0;  // (an operand's parts are of 16 bits)
    const uint32_t ps = (uint32_t)P.pos_stride;
    const int log_p = P.shift - kScaleShift, block_mask = (P.page >> kScaleShift) - 1;

    // What this thread stages.  Keys: 16 codes of keys kkey + 32 j (256 threads to 64, 32 or 16 keys at
    // once), of a block of 16 keys that is the wave's; values: 4 columns of VE keys of one block, those of
    // an operand's piece (16 u + 4 f + {0..3, 8..11}) or half of it.
    const int kkey = tid / kRowPieces, kc = 16 * (tid % kRowPieces);
    constexpr int kStep = 256 / kRowPieces;  // keys between a thread's pieces
    const int kblock = wave * (64 / kRowPieces) / 16;
    const int vu = HDP == 256 ? wave >> 1 : wave, vf = HDP == 256 ? wave & 1 : HDP == 128 ? hf : lane >> 4 & 1;
    const int vc = 4 * (HDP == 256 ? lane : HDP == 128 ? col32 : lane & 15), vhalf = HDP == 64 ? hf : 0;
    const bool kin = FULL || kc < hd, vin = FULL || vc < hd;
    const uint32_t koff = (uint32_t)(kkey & 15) * ps + (kin ? kc : 0), voff = (uint32_t)(4 * vf + 8 * vhalf) * ps + (vin ? vc : 0);

    int turn = 0;
    TileItem it;
    for (int64_t w = blockIdx.x; item_of(plan, A.n_q, geo, w, it); w += gridDim.x) {
        Nans<HDP>* const nans = &s_nans[turn++ & 1];
        if constexpr (C::kNan) {  // (its readers were done before the last item's first barrier)
            if (tid < HDP) nans->first[tid] = INT32_MAX;
            if (tid == 0) nans->any = 0;
        }
        const int unit = (int)(w % geo.units), kh = unit / geo.parts, h0 = kh * geo.group + (unit - kh * geo.parts) * geo.rows;
        const int heads = min(min(geo.rows, geo.group), (kh + 1) * geo.group - h0);
        it.row = __builtin_amdgcn_readfirstlane(it.row);
        it.limit = __builtin_amdgcn_readfirstlane(it.limit);
        it.first = __builtin_amdgcn_readfirstlane(it.first);
        it.end = __builtin_amdgcn_readfirstlane(it.end);
        const int n_rows = __builtin_amdgcn_readfirstlane(it.count) * heads;
        const int32_t* table = A.table + (int64_t)it.row * A.table_stride;
        const char* kpool = (const char*)P.k + (int64_t)kh * P.head_stride;
        const char* vpool = (const char*)P.v + (int64_t)kh * P.head_stride;
        const float* kscale = P.k_scale + (int64_t)kh * P.scale_head_stride;
        const float* vscale = P.v_scale + (int64_t)kh * P.scale_head_stride;

        // Lane j: the page (-1: absent) and scales of block j of a batch of 64 blocks of 16 keys, so that a
        // tile's addresses are scalar and wait for no load; the next batch is loaded when one begins.
        const int blocks = (it.limit + kScaleBlock - 1) >> kScaleShift, b0 = it.first * NB;
        auto page_batch = [&](int batch) {
            const int b = b0 + 64 * batch + lane;
            int id = -1;
            if (b < blocks) id = table[b >> log_p];
            return kv_page_ok(id, P.n_pages) ? id : -1;
        };
        auto scale_batch = [&](const float* scales, int batch, int id) {
            float s = 1.0f;
            if (id >= 0) s = scales[(int64_t)id * P.scale_page_stride + ((b0 + 64 * batch + lane) & block_mask)];
            return s;
        };
        // (loads that wait for each other first, so that the others are under way with them)
        int pages = page_batch(0), pages_next = -1, batch = 0, at = 0;  // at: the next tile's first block in the batch
        float ks_lane = scale_batch(kscale, 0, pages), vs_lane = scale_batch(vscale, 0, pages), ks_next = 1.0f, vs_next = 1.0f;
        // what a value scale makes of its weights: the exponent that it puts on them, and what takes it out of
        // their sum; or (kLift unset) what multiplies them
        float lift_lane = kLift ? 0.0f : 1.0f, back_lane = 1.0f;
        bool odd_scales = false;
        auto scales_at_hand = [&]() {
            const bool plain = plain_scale(vs_lane);
            if constexpr (kLift) {
                lift_lane = plain ? __builtin_amdgcn_logf(vs_lane) : 0.0f;
                back_lane = plain ? __builtin_amdgcn_rcpf(vs_lane) : 1.0f;
            } else {
                lift_lane = plain ? vs_lane : 1.0f;
            }
            odd_scales = __any(!plain);
        };
        if (blocks > b0 + 64) pages_next = page_batch(1);  // (later ones: -1 past the last block)

        uint32_t kcode[KP][4], vcode[VE];
        float ks[NB], lift[NB], back[NB], ks_load[NB], lift_load[NB], back_load[NB];  // of the tile at hand, and of the one that is loaded
        float value_scale = 1.0f;  // what the values that this thread stages are to be multiplied by
        int absent = 0, absent_load = 0;
        // Codes of a tile under way.  Absent blocks' keys are masked, their values have to be zeros.
        auto load_codes = [&](int tile) {
            if (at == 64) {
                at = 0;
                ++batch;
                pages = pages_next;
                ks_lane = ks_next;
                vs_lane = vs_next;
                pages_next = page_batch(batch + 1);
                scales_at_hand();
            } else if (at == 2 * NB) {
                ks_next = scale_batch(kscale, batch + 1, pages_next);
                vs_next = scale_batch(vscale, batch + 1, pages_next);
            }
            auto page = [&](int b) { return __builtin_amdgcn_readlane(pages, at + b); };
            auto offset = [&](int b, int id) {
                return (int64_t)max(id, 0) * P.page_stride + (int64_t)((uint32_t)((tile * NB + b) & block_mask) * (uint64_t)(kScaleBlock * ps));
            };
#pragma unroll
            for (int j = 0; j < KP; ++j) {
                const int b = kblock + j * kStep / 16;
                const v4u v = *(const v4u*)(kpool + offset(b, page(b)) + koff);
#pragma unroll
                for (int e = 0; e < 4; ++e) kcode[j][e] = v[e];
            }
            const int id = page(vu);
            const char* src = vpool + offset(vu, id);
#pragma unroll
            for (int e = 0; e < VE; ++e) vcode[e] = *(const uint32_t*)(src + ((e & 3) + 8 * (e >> 2)) * ps + voff);
            absent_load = 0;
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                ks_load[b] = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(ks_lane), at + b));
                lift_load[b] = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(lift_lane), at + b));
                if constexpr (kLift) back_load[b] = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(back_lane), at + b));
                absent_load |= page(b) < 0 ? 1 << b : 0;
            }
            value_scale = 1.0f;
            if (odd_scales) {
                const float v = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(vs_lane), at + vu));
                if (!plain_scale(v)) value_scale = v;
            }
            at += NB;
        };
        auto store_stage = [&](Stage<HDP>& S, int tile) {
#pragma unroll
            for (int j = 0; j < KP; ++j) {
                const int key = kkey + kStep * j;
                if constexpr (!FULL)
#pragma unroll
                    for (int e = 0; e < 4; ++e) kcode[j][e] = kin ? kcode[j][e] : 0;
                const int piece = kc / 8;
                *(v4u*)(S.k + key * HDP + 8 * (piece ^ k_swap<HDP>(key))) = Operand<C, M>::eight(kcode[j][0], kcode[j][1]);
                *(v4u*)(S.k + key * HDP + 8 * ((piece + 1) ^ k_swap<HDP>(key))) = Operand<C, M>::eight(kcode[j][2], kcode[j][3]);
            }
            if (absent_load >> vu & 1 || !vin)
#pragma unroll
                for (int e = 0; e < VE; ++e) vcode[e] = 0;
            if constexpr (C::kNan) {
                // A NaN belongs to the rows that see its key, and a weight of zero would not keep it
                // from the others: a zero in its place, and its column's first such key noted.
                uint32_t found = 0;  // (0x7F is the only byte that one more takes to 0x80)
#pragma unroll
                for (int e = 0; e < VE; ++e) found |= (vcode[e] & 0x7F7F7F7Fu) + 0x01010101u;
                if (found & 0x80808080u) {
#pragma unroll
                    for (int e = 0; e < VE; ++e)
#pragma unroll
                        for (int b = 0; b < 4; ++b)
                            if ((vcode[e] >> (8 * b) & 0x7F) == 0x7F) {
                                vcode[e] &= ~(0xFFu << (8 * b));
                                atomicMin(&nans->first[vc + b], tile * kKeys + 16 * vu + 4 * vf + 8 * vhalf + (e & 3) + 8 * (e >> 2));
                                nans->any = 1;
                            }
                }
            }
            uint32_t out[VE / 2][4];  // [pair of keys][column]
#pragma unroll
            for (int e = 0; e < VE / 2; ++e) Operand<C, __bf16>::columns(vcode[2 * e], vcode[2 * e + 1], out[e]);
            if (value_scale != 1.0f)
#pragma unroll
                for (int e = 0; e < VE / 2; ++e)
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        const float lo = __uint_as_float(out[e][c] << 16) * value_scale, hi = __uint_as_float(out[e][c] & 0xFFFF0000u) * value_scale;
                        out[e][c] = __builtin_amdgcn_perm(__float_as_uint(hi), __float_as_uint(lo), 0x07060302);
                    }
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                uint16_t* to = S.v + (vc + c) * kKeys + 8 * ((2 * vu + vf) ^ v_swap<HDP>(vc + c)) + 4 * vhalf;
                if constexpr (VE == 8) *(v4u*)to = (v4u){out[0][c], out[1][c], out[2][c], out[3][c]};
                else *(v2u*)to = (v2u){out[0][c], out[1][c]};
            }
        };

        scales_at_hand();
        if (it.first < it.end) load_codes(it.first);
        // this lane's row of the wave's 32: its query, head and limit
        const int rho = min(wave * 32 + col32, n_rows - 1), tok = it.token + rho / heads, head = h0 + rho % heads;
        V8 qreg[QP][KS];
        float row_scale;
        {
            int qcol[KS];
            bool qin[KS];
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                qcol[s] = 16 * s + 8 * hf;
                qin[s] = FULL || qcol[s] < hd;
            }
            row_scale = scale2 * load_query<TQ>((const TQ*)A.q + (int64_t)tok * A.q_stride + (int64_t)head * hd, qcol, qin, qreg,
                                                [](float v) { return fmaxf(v, other_half(v)); });
#pragma unroll
            for (int p = 0; p < QP; ++p)
#pragma unroll
                for (int s = 0; s < KS; ++s) qreg[p][s] = __builtin_bit_cast(V8, __builtin_bit_cast(v4u, qreg[p][s]) ^ flip);
        }

        const int limit = seen(A, pos, P, tok, it.row);
        int least = limit, most = limit;
#pragma unroll
        for (int o = 16; o >= 1; o >>= 1) {
            least = min(least, __shfl_xor(least, o, 64));
            most = max(most, __shfl_xor(most, o, 64));
        }
        least = __builtin_amdgcn_readfirstlane(least);
        most = __builtin_amdgcn_readfirstlane(most);
        const bool idle = wave * 32 >= n_rows;


        v16f acc[CT];
#pragma unroll
        for (int d = 0; d < CT; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[d][i] = 0.0f;
        float m = -INFINITY, l = 0.0f;

        auto take = [&]() {  // the tile that was loaded is the one at hand
            absent = absent_load;
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                ks[b] = ks_load[b], lift[b] = lift_load[b];
                if constexpr (kLift) back[b] = back_load[b];
            }
        };
        auto compute = [&](const Stage<HDP>& S, int key0) {
            v16f c[KT];
#pragma unroll
            for (int kt = 0; kt < KT; ++kt)
#pragma unroll
                for (int i = 0; i < 16; ++i) c[kt][i] = 0.0f;
            const uint16_t* krow = S.k + col32 * HDP;  // (32 keys on, the same exchange)
            const int kx = k_swap<HDP>(col32) ^ hf;
            {
                // operands four ahead and no further: the scheduler would take them all at once, and spill
                V8 a[2][4];
                auto fetch = [&](int n) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const int s = (4 * n + j) / KT, kt = (4 * n + j) % KT;
                        a[n & 1][j] = *(const V8*)(krow + 32 * kt * HDP + 8 * (kx ^ (2 * s)));
                    }
                };
                fetch(0);
#pragma unroll
                for (int n = 0; n < KS * KT / 4; ++n) {
                    if (n + 1 < KS * KT / 4) fetch(n + 1);
#pragma unroll
                    for (int p = QP - 1; p >= 0; --p)  // the small part first
#pragma unroll
                        for (int j = 0; j < 4; ++j) c[(4 * n + j) % KT] = mfma32(a[n & 1][j], qreg[p][(4 * n + j) / KT], c[(4 * n + j) % KT]);
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
            float factor[NB];
#pragma unroll
            for (int b = 0; b < NB; ++b) factor[b] = score_factor<TQ>(row_scale, ks[b]);
            float mx = -INFINITY;
            if (key0 + kKeys > least || absent) {
#pragma unroll
                for (int b = 0; b < NB; ++b)
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const int key = key0 + 16 * b + 8 * (i >> 2) + 4 * hf + (i & 3);
                        const float x = c[b >> 1][8 * (b & 1) + i] * factor[b];
                        c[b >> 1][8 * (b & 1) + i] = key < limit && !(absent >> b & 1) ? x : -INFINITY;
                        mx = fmaxf(mx, c[b >> 1][8 * (b & 1) + i]);
                    }
#pragma unroll
                for (int b = 0; b < NB; ++b) factor[b] = 1.0f;
            } else {
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    float top = c[b >> 1][8 * (b & 1)];
#pragma unroll
                    for (int i = 1; i < 8; ++i) top = fmaxf(top, c[b >> 1][8 * (b & 1) + i]);
                    mx = fmaxf(mx, top * factor[b]);
                }
            }
            // the running maximum moves only where a score passes it
            if (__any(mx > m)) {
                const float mn = fmaxf(m, fmaxf(mx, other_half(mx)));
                const float al = m > -INFINITY ? exp2_fast(m - mn) : 1.0f;  // nothing but zeros before
                l *= al;
#pragma unroll
                for (int d = 0; d < CT; ++d) acc[d] *= al;
                m = mn;
            }
            const float base = m > -INFINITY ? m : 0.0f;
            const uint16_t* vrow = S.v + col32 * kKeys;  // (32 columns on, the same exchange)
            const int vx = v_swap<HDP>(col32) ^ hf;
            v8bf a[2][CT];
            auto fetch = [&](int u) {
#pragma unroll
                for (int d = 0; d < CT; ++d) a[u & 1][d] = *(const v8bf*)(vrow + 32 * d * kKeys + 8 * (vx ^ (2 * u)));
            };
            fetch(0);
#pragma unroll
            for (int u = 0; u < NB; ++u) {
                if (u + 1 < NB) fetch(u + 1);
                // the weights of a block of 16 keys times its values' scale, and their sum without it
                const float down = kLift ? base - lift[u] : base;
                v8bf part[WP];
                float sum = 0.0f;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    float x = exp2_fast(fmaf(c[u >> 1][8 * (u & 1) + j], factor[u], -down));
                    sum += x;
                    if constexpr (!kLift) x *= lift[u];
#pragma unroll
                    for (int p = 0; p < WP; ++p) {
                        part[p][j] = (__bf16)x;
                        x -= (float)part[p][j];
                    }
                }
                if constexpr (kLift) l = fmaf(sum, back[u], l);
                else l += sum;
#pragma unroll
                for (int p = WP - 1; p >= 0; --p)
#pragma unroll
                    for (int d = 0; d < CT; ++d) acc[d] = mfma32(a[u & 1][d], part[p], acc[d]);
                __builtin_amdgcn_sched_barrier(0);
            }
        };

        __syncthreads();  // the last item's readers are done with the stages
        if (it.first < it.end) store_stage(stage[0], it.first);
        take();
        __syncthreads();
        auto step = [&](const Stage<HDP>& S, Stage<HDP>& next, int tile) {
            const bool more = tile + 1 < it.end;
            if (more) load_codes(tile + 1);
            if (!idle && tile * kKeys < most) compute(S, tile * kKeys);
            if (more) {
                store_stage(next, tile + 1);
                take();
            }
            __syncthreads();
        };
        for (int tile = it.first; tile < it.end; tile += 2) {
            step(stage[0], stage[1], tile);
            if (tile + 1 < it.end) step(stage[1], stage[0], tile + 1);
        }
        l += other_half(l);
        if constexpr (C::kNan)
            if (nans->any)
#pragma unroll
                for (int d = 0; d < CT; ++d)
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        if (nans->first[32 * d + 8 * (i >> 2) + 4 * hf + (i & 3)] < limit) acc[d][i] = NAN;
        if (idle || wave * 32 + col32 >= n_rows) continue;
        const bool alone = it.pieces == 1;
        const float inv = alone ? (l == 0.0f ? 0.0f : 1.0f / l) : 1.0f;
        float* part = plan.partial + ((size_t)it.part * geo.units + unit) * PrefixPlan::part_floats(geo.rows, hd);
        if (!alone && hf == 0) *(float2*)(part + 2 * rho) = make_float2(m, l);
        float* sums = part + 2 * geo.rows + (size_t)rho * hd;
        TQ* out = (TQ*)A.out + (int64_t)tok * A.out_stride + (int64_t)head * hd;
#pragma unroll
        for (int d = 0; d < CT; ++d)
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
                const int col = 32 * d + 2 * i + 4 * hf;
                if (!FULL && col >= hd) continue;
                float f[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) f[e] = acc[d][i + e] * inv;
                if (alone) store4(out + col, f);
                else *(v4f*)(sums + col) = *(const v4f*)f;
            }
    }
}

// ---- few rows ------------------------------------------------------------------------------
// One item of up to 32 rows: the waves go through the keys as those of k_kv8_attend do, 32 each of every
// 128, keys and values straight into registers, two tiles of 16 rows on each operand; then the four
// waves' sums are added up through LDS.  What bounds it is the keys' bytes, or latency: 16 requests' 5 drafted
// tokens over 256 to 2040 positions in 15 us, of which 4.3 are the bytes.
template <typename TQ, typename C, int HDP, bool FULL>
__global__ __launch_bounds__(256, HDP <= 128 ? 2 : 1) void k_kv8_prefix_few(const KvAttend A, const int32_t* pos, const KvPool P,
                                                                          const Geometry geo) {
    typedef typename Query<TQ>::M M;
    typedef typename Vec8<M>::T V8;
    constexpr int H = 2, NR = 2, KS = HDP / 64, D = HDP / 16, VD = D / 4;
    constexpr int QP = Query<TQ>::kQP, WP = kWeightParts<TQ, false>;
    __shared__ float s_m[4][16], s_l[4][16];
    __shared__ __attribute__((aligned(16))) float s_acc[4][16][HDP + 4];
    __shared__ Nans<HDP> nans;

    const int hd = FULL ? HDP : P.hd;
    const PrefixPlan plan(A.ws, A.n_q, hd, geo);
    TileItem it;
    for (int64_t w = blockIdx.x; item_of(plan, A.n_q, geo, w, it); w += gridDim.x) {
        int tid = threadIdx.x;
        asm volatile("" : "+v"(tid));  // (the lane's offsets anew for each item: kept over the loop they spill)
        const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), r = lane & 15, g = lane >> 4;
        const int unit = (int)(w % geo.units);
        const int kh = unit / geo.parts, h0 = kh * geo.group + (unit - kh * geo.parts) * geo.rows;
        const int heads = min(min(geo.rows, geo.group), (kh + 1) * geo.group - h0), n_rows = it.count * heads;
        const float scale2 = A.scale * 1.44269504088896340736f;
        if constexpr (C::kNan) {
            if (tid < HDP) nans.first[tid] = INT32_MAX;
            if (tid == 0) nans.any = 0;
            __syncthreads();
        }

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

        const int32_t* table = A.table + (int64_t)it.row * A.table_stride;
        const int t_last = (it.limit + 15) / 16 - 1;  // the last half tile (16 positions) with a position
        const int t_end = min(it.end * (kFewKeys / 16), t_last + 1);
        // lane j: the page (-1: absent) and scales of the wave's half tile j of a batch of 64
        const int t0 = it.first * (kFewKeys / 16) + wave * H, log_p = P.shift - kScaleShift, block_mask = (P.page >> kScaleShift) - 1;
        auto tile_of = [&](int batch) { return t0 + (batch * 64 + lane) / H * (4 * H) + (lane & (H - 1)); };
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

        v4f acc[NR][D];
        float m[NR], l[NR];
#pragma unroll
        for (int n = 0; n < NR; ++n) {
            m[n] = -INFINITY;
            l[n] = 0.0f;
#pragma unroll
            for (int d = 0; d < D; ++d) acc[n][d] = (v4f){0.f, 0.f, 0.f, 0.f};
        }
        uint32_t kreg[H][KS][4], vreg[H][4][VD];
        int id[H];
        int64_t at[H];
        auto place = [&](int t, int k) {
#pragma unroll
            for (int h = 0; h < H; ++h) {
                id[h] = __builtin_amdgcn_readlane(pages, k * H + h);
                at[h] = max(id[h], 0) * P.page_stride + (int64_t)((uint32_t)(((t + h) * 16) & (P.page - 1)) * (uint64_t)ps);
            }
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
            place(t, 0);
            load_k();
            load_v();
            if (t + 64 / H * (4 * H) < t_end) pages_next = page_batch(1);
        }
        // this lane's rows (those past the last repeat it)
        int limit[NR], least = INT32_MAX, qcol[2 * KS];
        bool qin[2 * KS];
#pragma unroll
        for (int s = 0; s < 2 * KS; ++s) {
            qcol[s] = 64 * (s >> 1) + 16 * g + 8 * (s & 1);
            qin[s] = FULL || qcol[s] < hd;
        }
        V8 qreg[NR][QP][2 * KS];
        float row_scale[NR];
#pragma unroll
        for (int n = 0; n < NR; ++n) {
            const int rho = min(16 * n + r, n_rows - 1), tok = it.token + rho / heads, head = h0 + rho % heads;
            limit[n] = seen(A, pos, P, tok, it.row);
            least = min(least, limit[n]);
            row_scale[n] = scale2 * load_query<TQ>((const TQ*)A.q + (int64_t)tok * A.q_stride + (int64_t)head * hd, qcol, qin, qreg[n],
                                                   [](float v) { return head_max(v); });
        }
#pragma unroll
        for (int o = 8; o >= 1; o >>= 1) least = min(least, __shfl_xor(least, o, 64));
        least = __builtin_amdgcn_readfirstlane(least);

        int batch = 1;
        while (t < t_end) {
            const int next = t + 4 * H;
            const bool more = next < t_end;
            float ks[H], vs[H];
            bool okh[H], absent = false;
#pragma unroll
            for (int h = 0; h < H; ++h) {
                ks[h] = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(ks_lane), k * H + h));
                vs[h] = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(vs_lane), k * H + h));
                okh[h] = id[h] >= 0;
                absent |= !okh[h];
            }
            const bool partial = (t + H) * 16 > least || absent;  // some row does not see some position
            float x[NR][H][4];
#pragma unroll
            for (int h = 0; h < H; ++h) {
                v4f c[NR];
#pragma unroll
                for (int n = 0; n < NR; ++n) c[n] = (v4f){0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int s = 0; s < KS; ++s) {
                    if constexpr (!FULL) {
                        const bool in = (int)(64 * s + kcol) < hd;
#pragma unroll
                        for (int e = 0; e < 4; ++e) kreg[h][s][e] = in ? kreg[h][s][e] : 0;
                    }
#pragma unroll
                    for (int f = 0; f < 2; ++f) {
                        const V8 key = __builtin_bit_cast(V8, Operand<C, M>::eight(kreg[h][s][2 * f], kreg[h][s][2 * f + 1]));
#pragma unroll
                        for (int p = QP - 1; p >= 0; --p)  // the small parts first
#pragma unroll
                            for (int n = 0; n < NR; ++n) c[n] = mfma16(key, qreg[n][p][2 * s + f], c[n]);
                    }
                }
#pragma unroll
                for (int n = 0; n < NR; ++n) {
                    const float factor = score_factor<TQ>(row_scale[n], ks[h]);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        x[n][h][i] = c[n][i] * factor;
                        if (partial && (!okh[h] || (t + h) * 16 + 4 * g + i >= limit[n])) x[n][h][i] = -INFINITY;
                    }
                }
            }
            const int t_now = t;
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
                place(next, k);
                load_k();
            }
            // values that no row of the item sees may hold anything, and a NaN belongs to the rows that see
            // its position (a weight of zero would not keep it from the others): zeros in their place, and
            // a column's first NaN noted
            if (partial)
#pragma unroll
                for (int h = 0; h < H; ++h)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int p = (t_now + h) * 16 + 4 * g + i;
                        const bool in = okh[h] && p < it.limit && vin;
#pragma unroll
                        for (int e = 0; e < VD; ++e) {
                            uint32_t& v = vreg[h][i][e];
                            v = in ? v : 0;
                            if constexpr (C::kNan)
                                if (((v & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u)
                                    for (int b = 0; b < 32; b += 8)
                                        if ((v >> b & 0x7F) == 0x7F) {
                                            v &= ~(0xFFu << b);
                                            atomicMin(&nans.first[vcol + 4 * e + b / 8], p);
                                            nans.any = 1;
                                        }
                        }
                    }
            v8bf part[NR][WP];
#pragma unroll
            for (int n = 0; n < NR; ++n) {
                float mx = x[n][0][0];
#pragma unroll
                for (int h = 0; h < H; ++h)
#pragma unroll
                    for (int i = 0; i < 4; ++i) mx = fmaxf(mx, x[n][h][i]);
                if (__any(mx > m[n])) {
                    const float mn = fmaxf(m[n], head_max(mx));
                    const float al = m[n] > -INFINITY ? exp2_fast(m[n] - mn) : 1.0f;  // nothing but zeros before
                    l[n] *= al;
#pragma unroll
                    for (int d = 0; d < D; ++d) acc[n][d] *= al;
                    m[n] = mn;
                }
                const float base = m[n] > -INFINITY ? m[n] : 0.0f;
#pragma unroll
                for (int h = 0; h < H; ++h)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        float v = exp2_fast(x[n][h][i] - base);
                        l[n] += v;
                        v *= vs[h];
#pragma unroll
                        for (int p = 0; p < WP; ++p) {
                            part[n][p][4 * h + i] = (__bf16)v;
                            v -= (float)part[n][p][4 * h + i];
                        }
                    }
            }
#pragma unroll
            for (int q = 0; q < VD; ++q) {
                uint32_t col[4][4];  // [pair of positions][column]
#pragma unroll
                for (int j = 0; j < 4; ++j)  // positions 2 j and 2 j + 1 of the lane's eight
                    Operand<C, __bf16>::columns(vreg[j >> 1][2 * (j & 1)][q], vreg[j >> 1][2 * (j & 1) + 1][q], col[j]);
#pragma unroll
                for (int p = WP - 1; p >= 0; --p)
#pragma unroll
                    for (int c = 0; c < 4; ++c)
#pragma unroll
                        for (int n = 0; n < NR; ++n)
                            acc[n][4 * q + c] = mfma16(__builtin_bit_cast(v8bf, (v4u){col[0][c], col[1][c], col[2][c], col[3][c]}), part[n][p], acc[n][4 * q + c]);
            }
            if (more) load_v();
            t = next;
        }

        // the four waves' sums, 16 rows at a time
        const bool alone = it.pieces == 1;
        float* to = plan.partial + ((size_t)it.part * geo.units + unit) * PrefixPlan::part_floats(geo.rows, hd);
#pragma unroll
        for (int n = 0; n < NR; ++n) {
            if (16 * n >= n_rows) break;
            if (n) __syncthreads();
            l[n] = head_sum(l[n]);
            if (g == 0) {
                s_m[wave][r] = m[n];
                s_l[wave][r] = l[n];
            }
            __syncthreads();
            float M = s_m[0][r];
#pragma unroll
            for (int w2 = 1; w2 < 4; ++w2) M = fmaxf(M, s_m[w2][r]);
            const float f = m[n] > -INFINITY ? exp2_fast(m[n] - M) : 1.0f;  // (no weights, or NaN: as they are)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int e = 0; e < D; ++e) s_acc[wave][r][(4 * g + i) * D + e] = acc[n][e][i] * f;
            __syncthreads();
            const int per = hd / 4;
            for (int o = tid; o < min(16, n_rows - 16 * n) * per; o += 256) {
                const int row = o / per, c = 4 * (o - row * per), rho = 16 * n + row, tok = it.token + rho / heads;
                float top = s_m[0][row], sum = 0.0f;
#pragma unroll
                for (int w2 = 1; w2 < 4; ++w2) top = fmaxf(top, s_m[w2][row]);
                v4f v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int w2 = 0; w2 < 4; ++w2) {
                    sum += s_l[w2][row] * (s_m[w2][row] > -INFINITY ? exp2_fast(s_m[w2][row] - top) : 1.0f);
                    v += *(const v4f*)&s_acc[w2][row][c];
                }
                if constexpr (C::kNan)
                    if (nans.any) {
                        const int lim = seen(A, pos, P, tok, it.row);
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (nans.first[c + e] < lim) v[e] = NAN;
                    }
                if (alone) {
                    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
                    const float out[4] = {v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv};
                    store4((TQ*)A.out + (int64_t)tok * A.out_stride + (int64_t)(h0 + rho % heads) * hd + c, out);
                } else {
                    *(v4f*)(to + 2 * geo.rows + (size_t)rho * hd + c) = v;
                    if (c == 0) *(float2*)(to + 2 * rho) = make_float2(top, sum);
                }
            }
        }
        __syncthreads();  // (the sums' readers are done)
    }
}

// ---- the join ------------------------------------------------------------------------------
// Running maximum, sum and weighted values of four columns, and those of further keys added to them.
struct Joined {
    float m, l;
    v4f v;
    SXQ_DEV void add(float m2, float l2, v4f v2) {
        const float mn = fmaxf(m, m2);
        const float up = m > -INFINITY ? exp2_fast(m - mn) : 1.0f;  // (no weights, or NaN: as they are)
        const float f = m2 > -INFINITY ? exp2_fast(m2 - mn) : 1.0f;
        l = l * up + l2 * f;
        v = v * up + v2 * f;
        m = mn;
    }
};

// The pieces of each cut tile, four columns of a row a thread, four pieces' loads at a time.  Where there
// are many pieces a tile, `share` threads take a row's in turn and the first joins what they have, in order:
// one request's 8 tokens after 30000 are 2 tiles of 128 pieces (heads of 64), 5 us so and 50 in one chain.
template <typename TQ>
__global__ __launch_bounds__(256) void k_kv8_prefix_join(const KvAttend A, const KvPool P, const Geometry geo) {
    __shared__ Joined s_part[256];
    const PrefixPlan plan(A.ws, A.n_q, P.hd, geo);
    const int4 counts = *(const int4*)plan.counts;
    const int tid = threadIdx.x, hd = P.hd, per = hd / 4, most = 256 / per;
    const int share = max(1, min(most, counts.z / max(4 * counts.y, 1))), at_once = most / share;  // rows a workgroup takes at once
    const int steps = (geo.rows + at_once - 1) / at_once;
    const int sub = tid / per, col = 4 * (tid - sub * per), k_first = sub / at_once;
    for (int w = blockIdx.x; w < counts.y * geo.units * steps; w += gridDim.x) {
        const int step = w % steps, unit = w / steps % geo.units, row = step * at_once + sub % at_once;
        const CutTile cut = plan.cut[w / steps / geo.units];
        const int kh = unit / geo.parts, h0 = kh * geo.group + (unit - kh * geo.parts) * geo.rows;
        const int heads = min(min(geo.rows, geo.group), (kh + 1) * geo.group - h0);
        const bool live = k_first < share && row < cut.count * heads;
        const float* part = plan.partial + ((size_t)cut.part * geo.units + unit) * PrefixPlan::part_floats(geo.rows, hd);
        const size_t stride = (size_t)geo.units * PrefixPlan::part_floats(geo.rows, hd);
        Joined sum{-INFINITY, 0.0f, {0.f, 0.f, 0.f, 0.f}};
        for (int k0 = k_first; live && k0 < cut.pieces; k0 += 4 * share) {
            float2 ml[4];
            v4f x[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const float* p = part + min(k0 + u * share, cut.pieces - 1) * stride;
                ml[u] = *(const float2*)(p + 2 * row);
                x[u] = *(const v4f*)(p + 2 * geo.rows + (size_t)row * hd + col);
            }
#pragma unroll
            for (int u = 0; u < 4; ++u)
                if (k0 + u * share < cut.pieces) sum.add(ml[u].x, ml[u].y, x[u]);
        }
        if (share > 1) {
            if (live && k_first) s_part[tid] = sum;
            __syncthreads();
            if (live && !k_first)
                for (int i = 1; i < share; ++i) {
                    const Joined o = s_part[tid + i * at_once * per];
                    sum.add(o.m, o.l, o.v);
                }
            __syncthreads();
        }
        if (!live || k_first) continue;
        const float inv = sum.l == 0.0f ? 0.0f : 1.0f / sum.l;
        const float f[4] = {sum.v[0] * inv, sum.v[1] * inv, sum.v[2] * inv, sum.v[3] * inv};
        store4((TQ*)A.out + (int64_t)(cut.token + row / heads) * A.out_stride + (int64_t)(h0 + row % heads) * hd + col, f);
    }
}

template <typename TQ, typename C, int HDP, bool FULL>
hipError_t prefix_launch(const KvAttend& a, const int32_t* pos, const KvPool& p, const Geometry& g, hipStream_t s) {
    const int64_t most = ((int64_t)a.n_q + 2 * g.places) * g.units;
    if (g.rows == kFewRows) {
        // (as many as a map's tiles and pieces, were each row of the table in it, but not tens of
        // thousands that find nothing)
        const int64_t tiles = (a.n_q + g.tokens - 1) / g.tokens + std::min(a.n_rows, a.n_q) + 2 * (int64_t)g.places;
        const int grid = (int)std::min<int64_t>(most, std::min<int64_t>(tiles * g.units, 8192));
        hipLaunchKernelGGL((k_kv8_prefix_few<TQ, C, HDP, FULL>), dim3(grid), dim3(256), 0, s, a, pos, p, g);
    } else {
        const int grid = (int)std::min<int64_t>(most, HDP <= 128 ? 512 : 256);
        hipLaunchKernelGGL((k_kv8_prefix<TQ, C, HDP, FULL>), dim3(grid), dim3(256), 0, s, a, pos, p, g);
    }
    return hipGetLastError();
}
template <typename TQ, typename C>
hipError_t prefix_by_width(const KvAttend& a, const int32_t* pos, const KvPool& p, const Geometry& g, hipStream_t s) {
    if (p.hd == 64) return prefix_launch<TQ, C, 64, true>(a, pos, p, g, s);
    if (p.hd == 128) return prefix_launch<TQ, C, 128, true>(a, pos, p, g, s);
    if (p.hd == 256) return prefix_launch<TQ, C, 256, true>(a, pos, p, g, s);
    if (p.hd < 64) return prefix_launch<TQ, C, 64, false>(a, pos, p, g, s);
    if (p.hd < 128) return prefix_launch<TQ, C, 128, false>(a, pos, p, g, s);
    return prefix_launch<TQ, C, 256, false>(a, pos, p, g, s);
}
template <typename TQ>
hipError_t prefix_by_code(const KvAttend& a, const int32_t* pos, const KvPool& p, const Geometry& g, hipStream_t s) {
    const hipError_t e = p.dtype == kI8 ? prefix_by_width<TQ, I8>(a, pos, p, g, s) : prefix_by_width<TQ, E4M3>(a, pos, p, g, s);
    if (e != hipSuccess) return e;
    // (what is cut is known on the device alone: a map's entries may be anyone's or nobody's)
    const int64_t all = (int64_t)g.places * g.units * g.rows;
    hipLaunchKernelGGL((k_kv8_prefix_join<TQ>), dim3((unsigned)std::min<int64_t>(1024, all)), dim3(256), 0, s, a, p, g);
    return hipGetLastError();
}

// Few rows (drafted tokens, short prompts): the kernel of 32-row tiles.  Few / wide, us: 16 requests of
// 1000 positions and 5 new tokens, 32 / 8 heads of 128, bf16 26 / 30, f32 30 / 41; 64 of 16 bf16 67 / 58,
// f32 82 / 101; 512 after 4000 92 / 87 and 118 / 149, 1024 172 / 143 and 219 / 254, 2048 353 / 232 and 451 /
// 438; three prompts of 1412 tokens 47 / 38 and 62 / 57; 500 requests of 200 positions and 2 tokens 91 / 110 and
// 117 / 203; 16 / 4 heads of 256, 512 after 4000 bf16 109 / 174, 64 of 32 152 / 102; 14 / 2 heads of 64, 256
// after 4000 32 / 29, 512 53 / 36.  (Entries of no request count as rows here: the host does not see them.)
inline bool few_rows(int n_q, int nh, int hd, int q_dtype) {
    return (int64_t)n_q * nh <= (hd <= 64 ? 4096 : q_dtype == kF32 && hd <= 128 ? 32768 : 16384);
}

}  // namespace

namespace sxq {

size_t kv8_prefix_workspace(const KvPool& p, int n_q, int nh) {
    size_t most = 0;  // over the kernels that queries of one type or another take
    for (int dtype : {kF32, kBF16}) most = std::max(most, PrefixPlan(nullptr, n_q, p.hd, Geometry(nh, p.nkv, p.hd, few_rows(n_q, nh, p.hd, dtype))).bytes);
    return most;
}

hipError_t launch_kv8_prefix(const KvAttend& a, const int32_t* pos, const KvPool& p, hipStream_t s) {
    const Geometry g(a.nh, p.nkv, p.hd, few_rows(a.n_q, a.nh, p.hd, a.q_dtype));
    hipLaunchKernelGGL(k_kv8_prefix_plan, dim3(1), dim3(1024), 0, s, a, pos, p, g);
    if (const hipError_t e = hipGetLastError(); e != hipSuccess) return e;
    if (a.q_dtype == kF32) return prefix_by_code<float>(a, pos, p, g, s);
    if (a.q_dtype == kF16) return prefix_by_code<_Float16>(a, pos, p, g, s);
    return prefix_by_code<__bf16>(a, pos, p, g, s);
}

}  // namespace sxq
