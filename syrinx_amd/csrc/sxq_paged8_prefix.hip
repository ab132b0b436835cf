// sxq_paged8_prefix.hip -- attention of several new tokens per request over the 8-bit paged cache,
// each over its own prefix (sxq_kv_prefix_attention; include/sxq.h states it).
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

typedef float v16f __attribute__((ext_vector_type(16)));

// ---- how the work is split ---------------------------------------------------------------
// Consecutive queries of one request make tiles of whole tokens, kRows rows (a token and a head of
// the KV head's group) or fewer; a group of more heads than that is cut into parts of kRows heads,
// a token a tile.  A unit is a KV head and such a part.  A tile's keys are taken kKeys at a time;
// where there are fewer tiles than the card has places, the longer ones are cut along their keys,
// into pieces whose results a launch of its own joins.  A launch of one workgroup writes the tiles
// and pieces ("items") down, and the attention's workgroups go through them.
constexpr int kRows = 128;
constexpr int kKeys = 64;
constexpr int kMinPiece = 4;  // tiles of keys

struct Geometry {
    int group, parts, units, tokens;  // heads a KV head; parts of a group; units; tokens a tile
    int places;                       // items of one unit that the card holds at once
    SXQ_HD Geometry(int nh, int nkv, int hd) {
        group = nh / nkv;
        parts = (group + kRows - 1) / kRows;
        units = nkv * parts;
        tokens = group < kRows ? kRows / group : 1;
        const int all = hd <= 128 ? 512 : 256;
        places = units < all ? all / units : 1;
    }
};

struct TileItem {
    int token, count, row;  // first query, queries, table row
    int limit;              // the most positions that one of them sees
    int first, end;         // this piece's tiles of keys
    int part, pieces;       // where its result goes, of how many pieces (1: out)
};

// The workspace: counts {tiles, items}; the tiles' first queries; items; the tiles that are cut
// {first item, pieces}; partials: per part and unit, {m, l} of each row, then the weighted sums.
struct PrefixPlan {
    int* counts;
    int* tile;
    TileItem* item;
    int2* cut;
    float* partial;
    size_t bytes;
    SXQ_HD static size_t up(size_t v) { return (v + 255) / 256 * 256; }
    SXQ_HD PrefixPlan(void* ws, int n_q, int hd, const Geometry& g) {
        char* p = (char*)ws;
        const int most = n_q + g.places;  // items: a tile each, and pieces up to the places
        counts = (int*)p;
        p += 256;
        tile = (int*)p;
        p += up(sizeof(int) * (size_t)n_q);
        item = (TileItem*)p;
        p += up(sizeof(TileItem) * (size_t)most);
        cut = (int2*)p;
        p += up(sizeof(int2) * (size_t)g.places);
        partial = (float*)p;
        p += (size_t)g.places * g.units * part_floats(hd) * sizeof(float);
        bytes = (size_t)(p - (char*)ws);
    }
    SXQ_HD static size_t part_floats(int hd) { return (size_t)kRows * (hd + 2); }
};

// The positions that query t sees, and whether it has a request.
SXQ_DEV int seen(const KvAttend& A, const int32_t* pos, const KvPool& P, int t, int row) {
    const int len = kv_clamp_len(A.lens[row], A.max_blocks, P.shift);
    return min(len, max(pos[t], -1) + 1);
}

__global__ __launch_bounds__(1024) void k_kv8_prefix_plan(const KvAttend A, const int32_t* pos, const KvPool P, const Geometry g,
                                                          bool may_cut) {
    __shared__ int red[16], s_cut;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const PrefixPlan plan(A.ws, A.n_q, P.hd, g);
    // Over the workgroup's threads up to this one: the sum, or the largest.
    auto scan = [&](int v, bool largest, int& all) {
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int u = __shfl_up(v, o, 64);
            if (lane >= o) v = largest ? max(v, u) : v + u;
        }
        __syncthreads();
        if (lane == 63) red[wave] = v;
        __syncthreads();
        int before = largest ? INT32_MIN : 0;
        all = before;
        for (int w = 0; w < 16; ++w) {
            if (w == wave) before = all;
            all = largest ? max(all, red[w]) : all + red[w];
        }
        return largest ? max(v, before) : v + before;
    };
    // 1. the tiles' first queries
    int tiles = 0, run = 0;  // so far; where the run that reaches into the chunk began
    for (int c0 = 0; c0 < A.n_q; c0 += 1024) {
        const int t = c0 + tid;
        const int row = t < A.n_q ? A.rows[t] : -1;
        const bool live = (uint32_t)row < (uint32_t)A.n_rows;
        const bool begins = t < A.n_q && (t == 0 || A.rows[t - 1] != row);
        int last, count;
        const int start = max(run, scan(begins ? t : -1, true, last));
        const bool first = live && (t - start) % g.tokens == 0;
        const int at = scan(first ? 1 : 0, false, count);
        if (first) plan.tile[tiles + at - 1] = t;
        tiles += count;
        run = max(run, last);
    }
    __syncthreads();
    // 2. each tile's queries and keys
    int work = 0;
    for (int i0 = 0; i0 < tiles; i0 += 1024) {
        const int i = i0 + tid;
        int keys = 0, all;
        if (i < tiles) {
            const int t = plan.tile[i], row = A.rows[t];
            int n = 1, limit = seen(A, pos, P, t, row);
            while (n < g.tokens && t + n < A.n_q && A.rows[t + n] == row) limit = max(limit, seen(A, pos, P, t + n, row)), ++n;
            keys = (limit + kKeys - 1) / kKeys;
            plan.item[i] = TileItem{t, n, row, limit, 0, keys, 0, 1};
        }
        scan(keys, false, all);
        work += all;
    }
    if (tid == 0) s_cut = 0;
    __syncthreads();
    // 3. pieces: at most g.places items in all where there are fewer tiles than that
    const bool cutting = may_cut && tiles < g.places;
    int items = tiles;
    if (cutting) {
        const int piece = max(kMinPiece, (work + g.places - tiles - 1) / (g.places - tiles));
        TileItem mine{};  // (tiles < 1024: one a thread)
        int n = 0, all;
        if (tid < tiles) {
            mine = plan.item[tid];
            n = max(1, (mine.end + piece - 1) / piece);
        }
        const int at = scan(n, false, all) - n;
        items = all;
        __syncthreads();
        if (n > 1) plan.cut[atomicAdd(&s_cut, 1)] = make_int2(at, n);
        const int keys = mine.end;
        for (int k = 0; k < n; ++k) {
            mine.first = (int)((int64_t)keys * k / n);
            mine.end = (int)((int64_t)keys * (k + 1) / n);
            mine.part = at + k;
            mine.pieces = n;
            plan.item[at + k] = mine;
        }
        __syncthreads();
    }
    if (tid == 0) {
        plan.counts[0] = items;
        plan.counts[1] = s_cut;
    }
}

// ---- the attention -----------------------------------------------------------------------
SXQ_DEV v16f mfma32(v8bf a, v8bf b, v16f c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
SXQ_DEV v16f mfma32(v8h a, v8h b, v16f c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }

// The other half of the wave's value.
SXQ_DEV float other_half(float v) {
    float a = v, b = v;
    swap32(a, b);
    return (threadIdx.x & 32) ? a : b;
}

// Into how many bf16 parts a weight is cut.
template <typename TQ>
constexpr int kWeightParts = 1;
template <>
constexpr int kWeightParts<_Float16> = 2;
template <>
constexpr int kWeightParts<float> = 3;

template <int HDP>
struct Stage {
    __attribute__((aligned(16))) uint16_t k[kKeys * HDP];  // [key][element], 16-byte pieces exchanged within a row
    __attribute__((aligned(16))) uint16_t v[HDP * kKeys];  // [column][key], the same
    float ks[4], vs[4];                                     // scales of the four blocks of 16 keys
    int absent[4];                                          // whether each block is
};

// The first key of each column whose value is NaN.
template <int HDP>
struct Nans {
    int first[HDP], any;
};

// Where a 16-byte piece of a row lies: the pieces of neighbouring rows on different banks.
template <int HDP>
SXQ_DEV int k_piece(int key, int piece) {
    return HDP == 64 ? piece ^ ((key >> 1) & 7) : piece ^ (key & 15);
}
SXQ_DEV int v_piece(int col, int piece) { return piece ^ ((col >> 1) & 7) ^ ((col >> 4) & 1); }

template <typename TQ, typename C, int HDP, bool FULL>
__global__ __launch_bounds__(256, HDP <= 128 ? 2 : 1) void k_kv8_prefix(const KvAttend A, const int32_t* pos, const KvPool P,
                                                                       const Geometry geo) {
    typedef typename Query<TQ>::M M;
    typedef typename Vec8<M>::T V8;
    constexpr int QP = Query<TQ>::kQP, WP = kWeightParts<TQ>;
    constexpr int KS = HDP / 16, CT = HDP / 32;             // steps over the head's elements, tiles of 32 columns
    constexpr int KP = kKeys * HDP / 16 / 256;              // 16-code pieces of keys a thread stages
    constexpr int VP = 8 * (HDP / 4) / 256 > 0 ? 8 * (HDP / 4) / 256 : 1;  // 8-key x 4-column pieces of values a thread
    constexpr bool VALL = 8 * (HDP / 4) >= 256;
    __shared__ Stage<HDP> stage[2];
    __shared__ Nans<HDP> s_nans[2];  // of this item and the last

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int col32 = lane & 31, hf = lane >> 5;
    const int hd = FULL ? HDP : P.hd;
    const PrefixPlan plan(A.ws, A.n_q, hd, geo);
    const int items = plan.counts[0];
    // (a negative scale is the positive one over negated queries: the running maximum wants factors
    // of 0 or more)
    const float scale2 = fabsf(A.scale) * 1.44269504088896340736f;
    const uint32_t flip = A.scale < 0.0f ? 0x80008000u : 0;  // (an operand's parts are of 16 bits)
    const uint32_t ps = (uint32_t)P.pos_stride;
    const int log_p = P.shift - kScaleShift, block_mask = (P.page >> kScaleShift) - 1;

    // long items first: of one request the last queries see the most
    int turn = 0;
    for (int64_t w = blockIdx.x; w < (int64_t)items * geo.units; w += gridDim.x) {
        Nans<HDP>* const nans = &s_nans[turn++ & 1];
        if constexpr (C::kNan) {  // (its readers were done before the last item's first barrier)
            if (tid < HDP) nans->first[tid] = INT32_MAX;
            if (tid == 0) nans->any = 0;
        }
        const int unit = (int)(w % geo.units), kh = unit / geo.parts, h0 = kh * geo.group + (unit - kh * geo.parts) * kRows;
        const int heads = min(min(kRows, geo.group), (kh + 1) * geo.group - h0);
        const TileItem it = plan.item[items - 1 - (int)(w / geo.units)];
        const int n_rows = it.count * heads;
        const int32_t* table = A.table + (int64_t)it.row * A.table_stride;
        const char* kpool = (const char*)P.k + (int64_t)kh * P.head_stride;
        const char* vpool = (const char*)P.v + (int64_t)kh * P.head_stride;

        // this lane's row of the wave's 32: its query, head and limit
        const int rho = min(wave * 32 + col32, n_rows - 1), tok = it.token + rho / heads, head = h0 + rho % heads;
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

        V8 qreg[QP][KS];
        {
            const TQ* q = (const TQ*)A.q + (int64_t)tok * A.q_stride + (int64_t)head * hd;
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                const int col = 16 * s + 8 * hf;
                const bool in = FULL || col < hd;
                v4u parts[QP];
                query_parts<TQ, QP>(q + (in ? col : 0), in, parts);
#pragma unroll
                for (int p = 0; p < QP; ++p) {
                    parts[p] ^= flip;
                    qreg[p][s] = __builtin_bit_cast(V8, parts[p]);
                }
            }
        }

        // what this thread stages of a tile of keys: pieces of 16 codes of one key, and of 4 columns
        // by the 8 keys of one operand piece (keys 16 u + 4 f + {0..3, 8..11})
        uint32_t kcode[KP][4], vcode[VP][8];
        float sc = 0.0f;
        int block_id = -1;
        auto page_of = [&](int block) {  // of a block of 16 keys
            int id = -1;
            if (block * 16 < it.limit) id = table[block >> log_p];
            return kv_page_ok(id, P.n_pages) ? id : -1;
        };
        int kid[KP], vid[VP], sid = -1;  // pages of the next tile to load
        auto load_ids = [&](int tile) {
#pragma unroll
            for (int j = 0; j < KP; ++j) kid[j] = page_of(tile * 4 + (tid + 256 * j) / (HDP / 16) / 16);
#pragma unroll
            for (int j = 0; j < VP; ++j) vid[j] = page_of(tile * 4 + ((tid + 256 * j) / (HDP / 4) & 7) / 2);
            if (tid < 8) sid = page_of(tile * 4 + (tid & 3));
        };
        auto load_codes = [&](int tile) {
            const int key0 = tile * kKeys;
#pragma unroll
            for (int j = 0; j < KP; ++j) {
                const int piece = tid + 256 * j, key = piece / (HDP / 16), c = 16 * (piece % (HDP / 16));
                const int off = (key0 + key) & (P.page - 1);
                v4u v = {0, 0, 0, 0};
                if (kid[j] >= 0 && (FULL || c < hd)) v = *(const v4u*)(kpool + (int64_t)kid[j] * P.page_stride + (uint64_t)off * ps + c);
#pragma unroll
                for (int e = 0; e < 4; ++e) kcode[j][e] = v[e];
            }
#pragma unroll
            for (int j = 0; j < VP; ++j) {
                const int piece = tid + 256 * j, c = 4 * (piece % (HDP / 4)), o = piece / (HDP / 4) & 7;  // o = 2 u + f
                const int key = 16 * (o >> 1) + 4 * (o & 1), off = (key0 + key) & (P.page - 1);
                const bool in = vid[j] >= 0 && (FULL || c < hd);
                const char* src = vpool + (int64_t)max(vid[j], 0) * P.page_stride + (uint64_t)off * ps + (in ? c : 0);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const int d = (e & 3) + 8 * (e >> 2);
                    // what no query of the item sees may hold anything: zeros
                    vcode[j][e] = in && key0 + key + d < it.limit ? *(const uint32_t*)(src + d * ps) : 0;
                }
            }
            block_id = sid;
            if (tid < 8 && sid >= 0)
                sc = (tid < 4 ? P.k_scale : P.v_scale)[(int64_t)sid * P.scale_page_stride + (int64_t)kh * P.scale_head_stride +
                                                       ((tile * 4 + (tid & 3)) & block_mask)];
        };
        auto store_stage = [&](Stage<HDP>& S, int tile) {
#pragma unroll
            for (int j = 0; j < KP; ++j) {
                const int piece = tid + 256 * j, key = piece / (HDP / 16), c = 2 * (piece % (HDP / 16));
                uint16_t* row = S.k + key * HDP;
                *(v4u*)(row + 8 * k_piece<HDP>(key, c)) = Operand<C, M>::eight(kcode[j][0], kcode[j][1]);
                *(v4u*)(row + 8 * k_piece<HDP>(key, c + 1)) = Operand<C, M>::eight(kcode[j][2], kcode[j][3]);
            }
            if constexpr (C::kNan) {
                // A NaN belongs to the rows that see its key, and a weight of zero would not keep it
                // from the others: a zero in its place, and its column's first such key noted.
                uint32_t found = 0;  // (0x7F is the only byte that one more takes to 0x80)
#pragma unroll
                for (int j = 0; j < VP; ++j)
#pragma unroll
                    for (int e = 0; e < 8; ++e) found |= (vcode[j][e] & 0x7F7F7F7Fu) + 0x01010101u;
                if (found & 0x80808080u) {
#pragma unroll
                    for (int j = 0; j < VP; ++j) {
                        const int piece = tid + 256 * j, c = 4 * (piece % (HDP / 4)), o = piece / (HDP / 4) & 7;
#pragma unroll
                        for (int e = 0; e < 8; ++e)
#pragma unroll
                            for (int b = 0; b < 4; ++b)
                                if ((vcode[j][e] >> (8 * b) & 0x7F) == 0x7F) {
                                    vcode[j][e] &= ~(0xFFu << (8 * b));
                                    atomicMin(&nans->first[c + b], tile * kKeys + 16 * (o >> 1) + 4 * (o & 1) + (e & 3) + 8 * (e >> 2));
                                    nans->any = 1;
                                }
                    }
                }
            }
#pragma unroll
            for (int j = 0; j < VP; ++j) {
                const int piece = tid + 256 * j, c = 4 * (piece % (HDP / 4)), o = piece / (HDP / 4);
                if (!VALL && o >= 8) break;
                uint32_t out[4][4];  // [pair of keys][column]
#pragma unroll
                for (int e = 0; e < 4; ++e) Operand<C, __bf16>::columns(vcode[j][2 * e], vcode[j][2 * e + 1], out[e]);
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    *(v4u*)(S.v + (c + e) * kKeys + 8 * v_piece(c + e, o)) = (v4u){out[0][e], out[1][e], out[2][e], out[3][e]};
            }
            if (tid < 4) {
                S.ks[tid] = block_id >= 0 ? sc : 0.0f;
                S.absent[tid] = block_id < 0;
            } else if (tid < 8) {
                S.vs[tid - 4] = block_id >= 0 ? sc : 0.0f;
            }
        };

        v16f acc[CT];
#pragma unroll
        for (int d = 0; d < CT; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[d][i] = 0.0f;
        float m = -INFINITY, l = 0.0f;

        if (it.first < it.end) {
            load_ids(it.first);
            load_codes(it.first);
            if (it.first + 1 < it.end) load_ids(it.first + 1);
        }
        __syncthreads();  // the last item's readers are done with the stages
        if (it.first < it.end) store_stage(stage[0], it.first);
        __syncthreads();
        for (int tile = it.first; tile < it.end; ++tile) {
            const Stage<HDP>& S = stage[(tile - it.first) & 1];
            const bool more = tile + 1 < it.end;
            if (more) {
                load_codes(tile + 1);
                if (tile + 2 < it.end) load_ids(tile + 2);
            }
            const int key0 = tile * kKeys;
            if (!idle && key0 < most) {
                v16f c[2];
#pragma unroll
                for (int kt = 0; kt < 2; ++kt) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) c[kt][i] = 0.0f;
                    const int key = 32 * kt + col32;
                    const uint16_t* row = S.k + key * HDP;
#pragma unroll
                    for (int s = 0; s < KS; ++s) {
                        const V8 a = *(const V8*)(row + 8 * k_piece<HDP>(key, 2 * s + hf));
#pragma unroll
                        for (int p = QP - 1; p >= 0; --p) c[kt] = mfma32(a, qreg[p][s], c[kt]);  // the small parts first
                    }
                }
                float factor[4], vs[4];
                int absent = 0;
#pragma unroll
                for (int b = 0; b < 4; ++b) {
                    factor[b] = scale2 * S.ks[b];
                    vs[b] = S.vs[b];
                    absent |= S.absent[b];
                }
                float mx = -INFINITY;
                if (key0 + kKeys > least || __builtin_amdgcn_readfirstlane(absent)) {
#pragma unroll
                    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                        for (int i = 0; i < 16; ++i) {
                            const int key = key0 + 32 * kt + 8 * (i >> 2) + 4 * hf + (i & 3);
                            const float x = c[kt][i] * factor[2 * kt + (i >> 3)];
                            c[kt][i] = key < limit && !S.absent[2 * kt + (i >> 3)] ? x : -INFINITY;
                            mx = fmaxf(mx, c[kt][i]);
                        }
#pragma unroll
                    for (int b = 0; b < 4; ++b) factor[b] = 1.0f;
                } else {
#pragma unroll
                    for (int b = 0; b < 4; ++b) {
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
                v8bf part[WP][4];
#pragma unroll
                for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const int b = 2 * kt + (i >> 3);
                        float w = exp2_fast(fmaf(c[kt][i], factor[b], -base));
                        l += w;
                        w *= vs[b];
#pragma unroll
                        for (int p = 0; p < WP; ++p) {
                            part[p][b][i & 7] = (__bf16)w;
                            w -= (float)part[p][b][i & 7];
                        }
                    }
#pragma unroll
                for (int d = 0; d < CT; ++d) {
                    const int col = 32 * d + col32;
                    const uint16_t* row = S.v + col * kKeys;
#pragma unroll
                    for (int u = 0; u < 4; ++u) {
                        const v8bf a = *(const v8bf*)(row + 8 * v_piece(col, 2 * u + hf));
#pragma unroll
                        for (int p = WP - 1; p >= 0; --p) acc[d] = mfma32(a, part[p][u], acc[d]);
                    }
                }
            }
            if (more) store_stage(stage[(tile + 1 - it.first) & 1], tile + 1);
            __syncthreads();
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
        float* part = plan.partial + ((size_t)it.part * geo.units + unit) * PrefixPlan::part_floats(hd);
        if (!alone && hf == 0) *(float2*)(part + 2 * rho) = make_float2(m, l);
        float* sums = part + 2 * kRows + (size_t)rho * hd;
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

// The pieces of each cut tile, joined: a wave a row and unit at a time, four columns a lane.
template <typename TQ>
__global__ __launch_bounds__(256) void k_kv8_prefix_join(const KvAttend A, const KvPool P, const Geometry geo) {
    const PrefixPlan plan(A.ws, A.n_q, P.hd, geo);
    const int cuts = plan.counts[1], lane = threadIdx.x & 63, hd = P.hd;
    const int waves = gridDim.x * 4, mine = blockIdx.x * 4 + (threadIdx.x >> 6);
    for (int64_t w = mine; w < (int64_t)cuts * geo.units * kRows; w += waves) {
        const int row = (int)(w % kRows), unit = (int)(w / kRows % geo.units);
        const int2 cut = plan.cut[w / kRows / geo.units];
        const TileItem it = plan.item[cut.x];
        const int kh = unit / geo.parts, h0 = kh * geo.group + (unit - kh * geo.parts) * kRows;
        const int heads = min(min(kRows, geo.group), (kh + 1) * geo.group - h0);
        if (row >= it.count * heads) continue;
        const float* part = plan.partial + ((size_t)cut.x * geo.units + unit) * PrefixPlan::part_floats(hd);
        const size_t step = (size_t)geo.units * PrefixPlan::part_floats(hd);
        float m = -INFINITY;
        for (int k = lane; k < cut.y; k += 64) m = fmaxf(m, part[k * step + 2 * row]);
        for (int o = 32; o >= 1; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
        float l = 0.0f;
        v4f v = {0.f, 0.f, 0.f, 0.f};
        const int col = 4 * lane;
        for (int k = 0; k < cut.y; ++k) {
            const float2 ml = *(const float2*)(part + k * step + 2 * row);
            const float f = ml.x > -INFINITY ? exp2_fast(ml.x - m) : 1.0f;  // (no weights, or NaN: as they are)
            l += ml.y * f;
            if (col < hd) v += *(const v4f*)(part + k * step + 2 * kRows + (size_t)row * hd + col) * f;
        }
        if (col >= hd) continue;
        float f[4];
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
        for (int e = 0; e < 4; ++e) f[e] = v[e] * inv;
        store4((TQ*)A.out + (int64_t)(it.token + row / heads) * A.out_stride + (int64_t)(h0 + row % heads) * hd + col, f);
    }
}

template <typename TQ, typename C, int HDP, bool FULL>
hipError_t prefix_launch(const KvAttend& a, const int32_t* pos, const KvPool& p, const Geometry& g, hipStream_t s) {
    const int64_t most = ((int64_t)a.n_q + g.places) * g.units;
    const int grid = (int)std::min<int64_t>(most, HDP <= 128 ? 512 : 256);
    hipLaunchKernelGGL((k_kv8_prefix<TQ, C, HDP, FULL>), dim3(grid), dim3(256), 0, s, a, pos, p, g);
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
hipError_t prefix_by_code(const KvAttend& a, const int32_t* pos, const KvPool& p, const Geometry& g, bool may_cut, hipStream_t s) {
    const hipError_t e = p.dtype == kI8 ? prefix_by_width<TQ, I8>(a, pos, p, g, s) : prefix_by_width<TQ, E4M3>(a, pos, p, g, s);
    if (e != hipSuccess || !may_cut) return e;
    const int64_t waves = (int64_t)g.places * g.units * kRows;
    hipLaunchKernelGGL((k_kv8_prefix_join<TQ>), dim3((unsigned)std::min<int64_t>(1024, (waves + 3) / 4)), dim3(256), 0, s, a, p, g);
    return hipGetLastError();
}

}  // namespace

namespace sxq {

size_t kv8_prefix_workspace(const KvPool& p, int n_q, int nh) {
    return PrefixPlan(nullptr, n_q, p.hd, Geometry(nh, p.nkv, p.hd)).bytes;
}

hipError_t launch_kv8_prefix(const KvAttend& a, const int32_t* pos, const KvPool& p, hipStream_t s) {
    const Geometry g(a.nh, p.nkv, p.hd);
    // (as many tiles as places, whatever the map: nothing is cut)
    const bool may_cut = (a.n_q + g.tokens - 1) / g.tokens < g.places;
    hipLaunchKernelGGL(k_kv8_prefix_plan, dim3(1), dim3(1024), 0, s, a, pos, p, g, may_cut);
    if (const hipError_t e = hipGetLastError(); e != hipSuccess) return e;
    if (a.q_dtype == kF32) return prefix_by_code<float>(a, pos, p, g, may_cut, s);
    if (a.q_dtype == kF16) return prefix_by_code<_Float16>(a, pos, p, g, may_cut, s);
    return prefix_by_code<__bf16>(a, pos, p, g, may_cut, s);
}

}  // namespace sxq
