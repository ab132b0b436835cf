// sxq_paged.hip -- the paged key/value cache: page allocation with block tables and slot maps
// (sxq_kv_reserve), and new tokens into the pages (sxq_kv_append).  include/sxq.h states both.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "../../include/sxq.h"
#include "sxq_abi.h"
#include "sxq_decoder.h"
#include "sxq_paged.h"
#include "sxq_paged_launch.h"

using namespace sxq;
using namespace sxq::abi;

namespace {

// ---------------------------------------------------------------------------- reserve
// Sums of pages fit 31 bits (n_rows * max_blocks < 2^31); sums of tokens saturate at
// 2^31 - 1 (the capacity they are compared with is at most that).
SXQ_DEV int sat_add(int a, int b) { return (int)min((uint32_t)a + (uint32_t)b, 0x7FFFFFFFu); }

struct Sums {
    int freed, pages, tokens;
};
SXQ_DEV Sums operator+(Sums a, Sums b) { return {a.freed + b.freed, a.pages + b.pages, sat_add(a.tokens, b.tokens)}; }

// Sum over the workgroup's threads before this one; `total` gets the sum of all.  red: NT / 64.
template <int NT>
SXQ_DEV Sums block_scan(Sums mine, Sums* red, Sums& total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    Sums v = mine;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const Sums u = {__shfl_up(v.freed, o, 64), __shfl_up(v.pages, o, 64), __shfl_up(v.tokens, o, 64)};
        if (lane >= o) v = u + v;
    }
    Sums before = {__shfl_up(v.freed, 1, 64), __shfl_up(v.pages, 1, 64), __shfl_up(v.tokens, 1, 64)};
    if (lane == 0) before = {0, 0, 0};
    if (NT == 64) {
        total = {__shfl(v.freed, 63, 64), __shfl(v.pages, 63, 64), __shfl(v.tokens, 63, 64)};
        return before;
    }
    __syncthreads();  // the last scan's readers are done with red
    if (lane == 63) red[wave] = v;
    __syncthreads();
    Sums lower = {0, 0, 0}, sum = {0, 0, 0};
#pragma unroll
    for (int w = 0; w < NT / 64; ++w) {
        if (w == wave) lower = sum;
        sum = sum + red[w];
    }
    total = sum;
    return lower + before;
}

// The last i with first[i] <= j, over n ascending firsts (first[0] <= j); for U values of j at
// once, so that the steps' LDS (or L2) reads overlap.
template <int U>
SXQ_DEV void owners(const int* first, int n, const int (&j)[U], int (&i)[U]) {
#pragma unroll
    for (int u = 0; u < U; ++u) i[u] = 0;
    for (int step = n > 1 ? 1 << (31 - __builtin_clz(n - 1)) : 0; step; step >>= 1)
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (i[u] + step < n && first[i[u] + step] <= j[u]) i[u] += step;
}
SXQ_DEV int owner(const int* first, int n, int j) {
    const int jj[1] = {j};
    int i[1];
    owners(first, n, jj, i);
    return i[0];
}

// The same by a whole wave for one j: 64 offsets a step.
SXQ_DEV int wave_owner(const int* first, int n, int j) {
    const int lane = threadIdx.x & 63;
    int lo = 0;
    while (n > 1) {
        const int step = (n + 63) / 64, at = lane * step;
        const int k = __builtin_popcountll(__ballot(at < n && first[lo + min(at, n - 1)] <= j)) - 1;
        lo += k * step;
        n = min(step, n - k * step);
    }
    return lo;
}

// How much of a call one workgroup does by itself.
enum ReserveMode {
    kAllInline = 0,  // everything
    kMapApart = 1,   // the token map by k_kv_map
    kPagesApart = 2  // the pages by k_kv_pages too, from the offsets left in the (unwritten) map
};

// One workgroup, NT * R requests at a time, R a thread: the sums that order the requests are
// prefix sums, and the pages and tokens of a chunk are dealt over the threads, each finding its
// request in the chunk's offsets.  A step is latency: lengths in, one scan (a second if a
// request is refused), results out.  16 requests 2.4 us of which an empty launch is about 2;
// 512 4.8; 4096 12.2.  By itself it also moves pages and tokens, four at a time a thread, which
// for many is the address rate of one CU (4096 requests, 12.8 thousand pages and 400 thousand
// tokens each way: 404 us): beyond 256 (one wave) or 2048 mapped tokens those go to the kernels
// below, 12.2 + 6.8 + 8.9 us.  A call that only gives back has no map and stays here: 16384
// pages of 4096 requests 33 us, 8192 of 16 requests (one wave) 59.
template <int NT, int R>
__global__ __launch_bounds__(NT) void k_kv_reserve(const KvReserve A, int mode) {
    constexpr int CH = NT * R, U = 4;
    __shared__ Sums red[NT / 64];
    __shared__ int s_push[CH], s_keep[CH], s_pop[CH], s_have[CH], s_tok[CH], s_old[CH];
    __shared__ int s_refused;
    const int tid = threadIdx.x, n = A.n_rows;
    const int64_t top = (int64_t)A.max_blocks << A.shift;
    const int count = min(max(A.free_count[0], 0), A.n_pages);

    int a[R], old[R];
    auto load = [&](int c0) {
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const int r = c0 + tid * R + i;
            a[i] = r < n ? A.add[r] : 0;
            old[i] = r < n ? kv_clamp_len(A.lens[r], A.max_blocks, A.shift) : 0;
        }
    };
    auto shrunk = [&](int i) { return (int)max((int64_t)old[i] + a[i], (int64_t)0); };
    // what request i of the thread gives back and asks for
    auto sums = [&](int i) -> Sums {
        const int have = kv_blocks(old[i], A.shift);
        if (a[i] < 0) return {have - kv_blocks(shrunk(i), A.shift), 0, 0};
        const int64_t grown = (int64_t)old[i] + a[i];
        if (grown > top) return {0, 0, 0};  // too long for its table row
        return {0, kv_blocks((int)grown, A.shift) - have, a[i]};
    };
    auto thread_sum = [&]() {
        Sums v = {0, 0, 0};
#pragma unroll
        for (int i = 0; i < R; ++i) v = v + sums(i);
        return v;
    };
    // the chunk's pages given back, `done` before them of `freed` in all
    auto push = [&](int c0, Sums before, int total, int done, int freed) {
#pragma unroll
        for (int i = 0; i < R; ++i) {
            s_push[tid * R + i] = before.freed;
            s_keep[tid * R + i] = kv_blocks(a[i] < 0 ? shrunk(i) : old[i], A.shift);
            before.freed += sums(i).freed;
        }
        __syncthreads();
        const int rows = min(CH, n - c0);
        for (int j0 = tid; j0 < total; j0 += U * NT) {
            int j[U], i[U], id[U];
#pragma unroll
            for (int u = 0; u < U; ++u) j[u] = min(j0 + u * NT, total - 1);
            owners(s_push, rows, j, i);
            auto entry = [&](int u) { return A.table + (int64_t)(c0 + i[u]) * A.table_stride + s_keep[i[u]] + (j[u] - s_push[i[u]]); };
#pragma unroll
            for (int u = 0; u < U; ++u) id[u] = j0 + u * NT < total ? *entry(u) : 0;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int at = count + freed - 1 - (done + j[u]);
                if (j0 + u * NT >= total) continue;
                if (at < A.n_pages) A.free_list[at] = id[u];
                *entry(u) = -1;
            }
        }
        __syncthreads();  // before the pops read the stack, and the next chunk's offsets
    };

    // 1. requests beyond one chunk: every page given back is on the stack before one is taken
    const bool chunks = n > CH;
    int freed = 0;
    if (chunks) {
        Sums total;
        for (int c0 = 0; c0 < n; c0 += CH) {
            load(c0);
            block_scan<NT>(thread_sum(), red, total);
            freed += total.freed;
        }
        int done = 0;
        for (int c0 = 0; c0 < n && freed && mode != kPagesApart; c0 += CH) {
            load(c0);
            const Sums before = block_scan<NT>(thread_sum(), red, total);
            push(c0, before, total.freed, done, freed);
            done += total.freed;
        }
    }

    // 2. pages and tokens handed out
    Sums asked = {0, 0, 0}, given = {0, 0, 0};
    int avail = 0, pushed = 0;
    if (tid == 0) A.cu[0] = 0;
    for (int c0 = 0; c0 < n; c0 += CH) {
        load(c0);
        Sums total;
        Sums before = block_scan<NT>(thread_sum(), red, total);
        if (!chunks) {
            freed = total.freed;
            if (freed && mode != kPagesApart) push(c0, before, freed, 0, freed);
        }
        Sums back = before;
        avail = min(count + freed, A.n_pages);
        if (tid == 0) s_refused = 0;
        __syncthreads();
        int status[R];
        bool refused = false;
        Sums upto = asked + before, want = {0, 0, 0};
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const Sums s = sums(i);
            upto = upto + s;
            status[i] = a[i] >= 0 && (int64_t)old[i] + a[i] > top ? 2 : s.pages > 0 && upto.pages > avail ? 1
                        : s.tokens > 0 && upto.tokens > A.limit ? 3 : 0;
            if (status[i] == 0) want = want + s;
            refused |= status[i] == 1 || status[i] == 3;
        }
        asked = asked + total;
        const int chunk_freed = total.freed;
        if (refused) s_refused = 1;
        __syncthreads();
        if (s_refused) before = block_scan<NT>(want, red, total);  // else all that was asked for is given
        Sums at = before;
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const int r = c0 + tid * R + i, k = tid * R + i;
            Sums s = sums(i);
            if (status[i]) s = {0, 0, 0};
            if (mode == kPagesApart && r < n) {
                A.slots[r] = pushed + back.freed;
                A.pos[r] = given.pages + at.pages;
                A.rows[r] = kv_blocks(a[i] < 0 ? shrunk(i) : old[i], A.shift);
                back.freed += sums(i).freed;
            }
            s_pop[k] = at.pages;
            s_tok[k] = at.tokens;
            s_have[k] = kv_blocks(old[i], A.shift);
            s_old[k] = old[i];
            at = at + s;
            if (r < n) {
                A.cu[r + 1] = given.tokens + at.tokens;
                A.status[r] = status[i];
                A.lens[r] = a[i] < 0 ? shrunk(i) : status[i] ? old[i] : old[i] + a[i];
            }
        }
        __syncthreads();
        const int rows = min(CH, n - c0);
        pushed += chunk_freed;
        for (int j0 = tid; j0 < total.pages && mode != kPagesApart; j0 += U * NT) {
            int j[U], i[U], id[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                j[u] = min(j0 + u * NT, total.pages - 1);
                id[u] = A.free_list[avail - 1 - (given.pages + j[u])];
            }
            owners(s_pop, rows, j, i);
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (j0 + u * NT < total.pages)
                    A.table[(int64_t)(c0 + i[u]) * A.table_stride + s_have[i[u]] + (j[u] - s_pop[i[u]])] = id[u];
        }
        __syncthreads();  // the new table entries are read by the tokens' threads
        const int mapped = min(total.tokens, A.capacity - min(given.tokens, A.capacity));
        for (int j = tid; mode == kAllInline && j < mapped; j += NT) {
            const int i = owner(s_tok, rows, j);
            const int pos = s_old[i] + (j - s_tok[i]), t = given.tokens + j;
            A.slots[t] = kv_slot(A.table[(int64_t)(c0 + i) * A.table_stride + (pos >> A.shift)], pos, A.shift, A.n_pages);
            A.pos[t] = pos;
            A.rows[t] = c0 + i;
        }
        given = given + total;
        __syncthreads();
    }
    for (int t = given.tokens + tid; mode == kAllInline && t < A.capacity; t += NT) A.slots[t] = A.pos[t] = A.rows[t] = -1;
    if (tid == 0) {
        A.free_count[0] = avail - given.pages;
        if (mode == kPagesApart) {
            A.slots[n] = pushed;
            A.pos[n] = given.pages;
            A.rows[n] = avail;
        }
    }
}

// The pages of many requests, from k_kv_reserve's offsets: the j-th page given back goes to
// the stack's place for it and is the j-th page handed out, so one thread does both and no
// other touches its table entries; beyond those the pages come off the old stack.  A workgroup
// finds the requests of its first and last page, a thread its own between those.  12.8 thousand
// pages given back or taken, of 4096 requests: 6.8 us, launch and two searches in turn.
constexpr int kPagesPer = 256;
__global__ __launch_bounds__(kPagesPer) void k_kv_pages(const KvReserve A) {
    const int n = A.n_rows;
    const int *push = A.slots, *pop = A.pos, *base = A.rows;
    const int freed = push[n], given = pop[n], avail = base[n];
    for (int j0 = blockIdx.x * kPagesPer; j0 < max(freed, given); j0 += gridDim.x * kPagesPer) {
        const int j = j0 + threadIdx.x;
        int id = -1;
        if (j0 < freed) {
            const int lo = wave_owner(push, n, j0), hi = wave_owner(push, n, min(j0 + kPagesPer, freed) - 1);
            if (j < freed) {
                const int i = lo + owner(push + lo, hi + 1 - lo, j), at = avail - 1 - j;
                int32_t* e = A.table + (int64_t)i * A.table_stride + base[i] + (j - push[i]);
                id = *e;
                *e = -1;
                if (at >= 0) A.free_list[at] = id;
            }
        }
        if (j0 < given) {
            const int lo = wave_owner(pop, n, j0), hi = wave_owner(pop, n, min(j0 + kPagesPer, given) - 1);
            if (j < given) {
                const int i = lo + owner(pop + lo, hi + 1 - lo, j);
                if (j >= freed) id = A.free_list[avail - 1 - j];
                A.table[(int64_t)i * A.table_stride + base[i] + (j - pop[i])] = id;
            }
        }
    }
}

// The map of many tokens, from the offsets, lengths and tables: as above by tokens.  400
// thousand: 8.9 us (4.8 MB written; the searches' and table's loads in turn); 50 thousand 6.5.
constexpr int kMapTokens = 1024;
__global__ __launch_bounds__(256) void k_kv_map(const KvReserve A) {
    const int t0 = blockIdx.x * kMapTokens, total = A.cu[A.n_rows];
    const int t_end = min(t0 + kMapTokens, total);
    int lo = 0, n = 0;
    if (t0 < total) {
        lo = wave_owner(A.cu, A.n_rows, t0);
        n = wave_owner(A.cu, A.n_rows, t_end - 1) + 1 - lo;
    }
    for (int t = t0 + threadIdx.x; t < min(t0 + kMapTokens, A.capacity); t += 256) {
        int slot = -1, pos = -1, row = -1;
        if (t < t_end) {
            row = lo + owner(A.cu + lo, n, t);
            pos = A.lens[row] - (A.cu[row + 1] - t);
            slot = kv_slot(A.table[(int64_t)row * A.table_stride + (pos >> A.shift)], pos, A.shift, A.n_pages);
        }
        A.slots[t] = slot;
        A.pos[t] = pos;
        A.rows[t] = row;
    }
}

// ---------------------------------------------------------------------------- append
// Four consecutive elements as f32, at any element's alignment, and back.
template <typename T>
SXQ_DEV void load4(const T* p, float* f) {
    typedef T v4 __attribute__((ext_vector_type(4), aligned(sizeof(T))));
    const v4 v = *(const v4*)p;
#pragma unroll
    for (int e = 0; e < 4; ++e) f[e] = to_f32(v[e]);
}
template <typename T>
SXQ_DEV void store4(T* p, const float* f) {
    typedef T v4 __attribute__((ext_vector_type(4), aligned(sizeof(T))));
    v4 v;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = from_f32<T>(f[e]);
    *(v4*)p = v;
}

// Eight elements of a head a lane -- four RoPE pairs, as two vectors of four: (8 j, 8 j + 4)
// interleaved, (4 j, hd / 2 + 4 j) in halves -- so that a head takes hd / 8 lanes (rounded up
// to a power of two, LH), a wave 64 / LH heads of one token, the norm's sum stays among
// neighbouring lanes and no element changes lanes.  Bound by HBM: 8192 bf16 tokens of 32 + 16
// heads of 128 (206 MB) 48 us, 4.3 TB/s where a copy reaches 4.8; 1412 f32 ones into bf16 pages
// 13.6 (a wave a head, an element a lane at a time: 137 and 22).  Few tokens are latency, 3 us.
template <typename TI, typename TC>
__global__ __launch_bounds__(256) void k_kv_append(const KvAppend A, const KvPool P, int log_lh) {
    const int t = blockIdx.x, hd = P.hd, half = hd / 2, lh = 1 << log_lh;
    const int hid = blockIdx.y * (256 >> log_lh) + (threadIdx.x >> log_lh), j = threadIdx.x & (lh - 1);
    const int heads = A.nh + 2 * P.nkv;
    const bool live = hid < heads && 8 * j < hd;
    const int slot = A.slots[t];
    if (slot < 0 || slot >= P.n_pages << P.shift) return;
    const bool is_q = hid < A.nh, is_k = !is_q && hid < A.nh + P.nkv;
    const float* w = is_q ? A.q_norm : is_k ? A.k_norm : nullptr;
    const int o1 = A.interleaved ? 8 * j : 4 * j, o2 = A.interleaved ? 8 * j + 4 : half + 4 * j;
    float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (live) {
        const TI* src = (const TI*)A.qkv + (int64_t)t * A.row_stride + (int64_t)hid * hd;
        load4(src + o1, x);
        load4(src + o2, x + 4);
    }
    float c[4], s[4];
    const bool rot = A.cos && (is_q || is_k);
    if (live && rot) {
        const int p = min(max(A.pos[t], 0), A.max_pos - 1);
        load4(A.cos + (int64_t)p * half + 4 * j, c);
        load4(A.sin + (int64_t)p * half + 4 * j, s);
    }
    float ss = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) ss += x[e] * x[e];
    for (int o = lh >> 1; o >= 1; o >>= 1) ss += __shfl_xor(ss, o, 64);
    if (!live || (is_q && !A.q_out)) return;
    if (w) {
        const float inv = 1.0f / sqrtf(ss / (float)hd + A.eps);
        float g[8];
        load4(w + o1, g);
        load4(w + o2, g + 4);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = x[e] * inv * g[e];
    }
    if (rot) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {  // pair e of the lane
            float &a = A.interleaved ? x[2 * e] : x[e], &b = A.interleaved ? x[2 * e + 1] : x[4 + e];
            const float u = a * c[e] - b * s[e];
            b = b * c[e] + a * s[e];
            a = u;
        }
    }
    if (is_q) {
        TI* dst = (TI*)A.q_out + ((int64_t)t * A.nh + hid) * hd;
        store4(dst + o1, x);
        store4(dst + o2, x + 4);
    } else {
        TC* dst = (TC*)(is_k ? P.k : P.v) + kv_slot_base(P, slot, hid - A.nh - (is_k ? 0 : P.nkv));
        store4(dst + o1, x);
        store4(dst + o2, x + 4);
    }
}

template <typename TI>
void append_by_cache(const KvAppend& a, const KvPool& p, hipStream_t s) {
    int log_lh = 0;
    while (8 << log_lh < p.hd) ++log_lh;
    const int per = 256 >> log_lh;  // heads a workgroup
    const dim3 grid(a.n_tokens, (a.nh + 2 * p.nkv + per - 1) / per);
    if (p.dtype == kF32) hipLaunchKernelGGL((k_kv_append<TI, float>), grid, dim3(256), 0, s, a, p, log_lh);
    else if (p.dtype == kF16) hipLaunchKernelGGL((k_kv_append<TI, _Float16>), grid, dim3(256), 0, s, a, p, log_lh);
    else hipLaunchKernelGGL((k_kv_append<TI, __bf16>), grid, dim3(256), 0, s, a, p, log_lh);
}

// ---------------------------------------------------------------------------- gather
// Eight elements of K and of V a thread.
template <typename TC>
__global__ __launch_bounds__(256) void k_kv_gather(const KvPool P, const int32_t* __restrict__ table, int64_t table_stride,
                                                   int max_blocks, const KvSpans S, int r0, int h0, int p0,
                                                   float* __restrict__ k, float* __restrict__ v) {
    const int per = P.hd / 8, i = blockIdx.x * 256 + threadIdx.x, q = i / per, d = 8 * (i - q * per);
    const int total = S.start[S.n];
    if (q >= total) return;
    int row = 0, first = 0;
#pragma unroll
    for (int z = 1; z < 16; ++z)
        if (z < S.n && q >= S.start[z]) row = z, first = S.start[z];
    const int h = blockIdx.y, p = p0 + q - first, b = p >> P.shift;
    const int slot = b < max_blocks ? kv_slot(table[(r0 + row) * table_stride + b], p, P.shift, P.n_pages) : -1;
    const int64_t from = slot < 0 ? 0 : kv_slot_base(P, slot, h0 + h) + d;
    const int64_t to = ((int64_t)h * total + q) * P.hd + d;
#pragma unroll
    for (int o = 0; o < 8; o += 4) {
        float f[4] = {0.f, 0.f, 0.f, 0.f};
        if (k) {
            if (slot >= 0) load4((const TC*)P.k + from + o, f);
            store4(k + to + o, f);
        }
        if (v) {
            if (slot >= 0) load4((const TC*)P.v + from + o, f);
            store4(v + to + o, f);
        }
    }
}

// Every page free, page 0 on top.
__global__ __launch_bounds__(256) void k_kv_stack(int32_t* __restrict__ free_list, int n) {
    const int i = blockIdx.x * 256 + threadIdx.x;
    if (i < n) free_list[i] = n - 1 - i;
}

__global__ __launch_bounds__(64) void k_kv_growths(const KvGrowths g, int32_t* __restrict__ add) {
    if ((int)threadIdx.x < g.n) add[threadIdx.x] = g.add[threadIdx.x];
}

__global__ __launch_bounds__(64) void k_kv_by_row(const int32_t* __restrict__ cu, const int32_t* __restrict__ map_slots,
                                                  const int32_t* __restrict__ map_pos, int rows, int32_t* __restrict__ slots,
                                                  int32_t* __restrict__ pos) {
    const int r = threadIdx.x;
    if (r >= rows) return;
    const int t = cu[r];
    const bool has = cu[r + 1] > t;
    slots[r] = has ? map_slots[t] : -1;
    pos[r] = has ? map_pos[t] : 0;
}

__global__ __launch_bounds__(256) void k_f32_to_bf16(const float* __restrict__ x, int64_t n, __bf16* __restrict__ y) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i < n) y[i] = (__bf16)x[i];
}

bool kv_dtype(int dt) { return dt == kF32 || dt == kF16 || dt == kBF16; }
bool pow2_page(int p) { return p >= 16 && p <= 1024 && (p & (p - 1)) == 0; }

}  // namespace

namespace sxq {

hipError_t launch_kv_reserve(const KvReserve& a, hipStream_t s, bool* moved) {
    const bool wave = a.n_rows <= 64;
    int mode = a.capacity <= (wave ? 256 : 2048) ? kAllInline : wave || a.capacity <= a.n_rows ? kMapApart : kPagesApart;
    // (each launch's own result: `moved` may not depend on an error that an earlier call left)
    auto launch = [&](const void* kernel, int grid, int block, void** args) {
        return hipLaunchKernel(kernel, dim3(grid), dim3(block), args, 0, s);
    };
    void *both[] = {(void*)&a, &mode}, *one[] = {(void*)&a};
    hipError_t e = wave ? launch((const void*)k_kv_reserve<64, 1>, 1, 64, both)
                        : launch(a.n_rows <= 1024 ? (const void*)k_kv_reserve<1024, 1> : (const void*)k_kv_reserve<1024, 4>, 1, 1024, both);
    if (e == hipSuccess && moved) *moved = true;
    if (e == hipSuccess && mode == kPagesApart)
        e = launch((const void*)k_kv_pages, std::min(256, (a.n_pages + kPagesPer - 1) / kPagesPer), kPagesPer, one);
    if (e == hipSuccess && mode != kAllInline) e = launch((const void*)k_kv_map, (a.capacity + kMapTokens - 1) / kMapTokens, 256, one);
    return e;
}

hipError_t launch_kv_append(const KvAppend& all, const KvPool& p, hipStream_t s) {
    constexpr int kMost = 1 << 23;  // tokens a launch: its grid may not pass 2^32 threads
    const size_t e = type_size(all.dtype);
    for (int64_t t0 = 0; t0 < all.n_tokens; t0 += kMost) {
        KvAppend a = all;
        a.n_tokens = (int)std::min<int64_t>(kMost, all.n_tokens - t0);
        a.qkv = (const char*)all.qkv + t0 * all.row_stride * e;
        if (all.pos) a.pos = all.pos + t0;
        a.slots = all.slots + t0;
        if (all.q_out) a.q_out = (char*)all.q_out + t0 * all.nh * p.hd * e;
        if (a.dtype == kF32) append_by_cache<float>(a, p, s);
        else if (a.dtype == kF16) append_by_cache<_Float16>(a, p, s);
        else append_by_cache<__bf16>(a, p, s);
        if (const hipError_t err = hipGetLastError(); err != hipSuccess) return err;
    }
    return hipSuccess;
}

hipError_t launch_kv_gather(const KvPool& p, const int32_t* table, int64_t table_stride, int max_blocks, const KvSpans& spans,
                            int r0, int h0, int heads, int p0, float* k, float* v, hipStream_t s) {
    const dim3 grid((unsigned)(((int64_t)spans.start[spans.n] * (p.hd / 8) + 255) / 256), heads);
#define SXQ_GA(T) hipLaunchKernelGGL(k_kv_gather<T>, grid, dim3(256), 0, s, p, table, table_stride, max_blocks, spans, r0, h0, p0, k, v)
    if (p.dtype == kF32) SXQ_GA(float);
    else SXQ_GA(__bf16);  // (an engine's pages are f32 or bf16)
#undef SXQ_GA
    return hipGetLastError();
}

hipError_t launch_kv_stack(int32_t* free_list, int n, hipStream_t s) {
    hipLaunchKernelGGL(k_kv_stack, dim3((n + 255) / 256), dim3(256), 0, s, free_list, n);
    return hipGetLastError();
}

hipError_t launch_kv_growths(const KvGrowths& g, int32_t* add, hipStream_t s) {
    hipLaunchKernelGGL(k_kv_growths, dim3(1), dim3(64), 0, s, g, add);
    return hipGetLastError();
}

hipError_t launch_kv_by_row(const int32_t* cu, const int32_t* map_slots, const int32_t* map_pos, int rows, int32_t* slots,
                            int32_t* pos, hipStream_t s) {
    hipLaunchKernelGGL(k_kv_by_row, dim3(1), dim3(64), 0, s, cu, map_slots, map_pos, rows, slots, pos);
    return hipGetLastError();
}

hipError_t launch_f32_to_bf16(const float* x, int64_t n, uint16_t* y, hipStream_t s) {
    hipLaunchKernelGGL(k_f32_to_bf16, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, s, x, n, (__bf16*)y);
    return hipGetLastError();
}

namespace abi {

sxq_status kv_pool(const char* who, const sxq_kv_pages* g, bool pointers, KvPool* out) {
    if (!g) return fail(SXQ_ERR_INVALID, "%s: null pages", who);
    if (!kv_dtype(g->dtype)) return fail(SXQ_ERR_DTYPE, "%s: page dtype %d (f32, f16 or bf16)", who, g->dtype);
    if (!pow2_page(g->page_size))
        return fail(SXQ_ERR_INVALID, "%s: page_size %d is not a power of two in 16..1024", who, g->page_size);
    if (g->n_pages < 1 || (int64_t)g->n_pages * g->page_size > 0x7FFFFFFF)
        return fail(SXQ_ERR_INVALID, "%s: n_pages %d (1 or more, n_pages * page_size below 2^31)", who, g->n_pages);
    if (g->n_kv_heads < 1 || g->n_kv_heads > 1024)
        return fail(SXQ_ERR_INVALID, "%s: n_kv_heads %d", who, g->n_kv_heads);
    if (g->head_dim < 8 || g->head_dim > 256 || g->head_dim % 8)
        return fail(SXQ_ERR_SHAPE, "%s: head_dim %d is not a multiple of 8 in 8..256", who, g->head_dim);
    const int64_t unit = 16 / type_size(g->dtype), most = (int64_t)1 << 50;
    for (int64_t st : {g->page_stride, g->head_stride, g->pos_stride})
        if (st < g->head_dim || st % unit || st > most)
            return fail(SXQ_ERR_SHAPE, "%s: page strides (%lld, %lld, %lld) must be multiples of %lld elements, at least head_dim",
                        who, (long long)g->page_stride, (long long)g->head_stride, (long long)g->pos_stride, (long long)unit);
    if (g->pos_stride > 1 << 24) return fail(SXQ_ERR_SHAPE, "%s: pos_stride %lld above 2^24 elements", who, (long long)g->pos_stride);
    if (pointers && (!g->k || !g->v)) return fail(SXQ_ERR_INVALID, "%s: null page pool", who);
    if (((uintptr_t)g->k | (uintptr_t)g->v) & 15) return fail(SXQ_ERR_INVALID, "%s: the page pools must be 16-byte aligned", who);
    out->k = g->k;
    out->v = g->v;
    out->page_stride = g->page_stride;
    out->head_stride = g->head_stride;
    out->pos_stride = g->pos_stride;
    out->dtype = g->dtype;
    out->nkv = g->n_kv_heads;
    out->hd = g->head_dim;
    out->page = g->page_size;
    out->shift = __builtin_ctz((unsigned)g->page_size);
    out->n_pages = g->n_pages;
    return SXQ_OK;
}

}  // namespace abi
}  // namespace sxq

extern "C" {

sxq_status sxq_kv_reserve(int device, int page_size, int n_pages, int n_rows, int max_blocks, const int32_t* add,
                          int32_t* lens, int32_t* table, int64_t table_stride, int32_t* free_list,
                          int32_t* free_count, int capacity, int32_t* cu, int32_t* slots, int32_t* pos,
                          int32_t* rows, int32_t* status, void* stream) {
    if (!pow2_page(page_size))
        return fail(SXQ_ERR_INVALID, "kv_reserve: page_size %d is not a power of two in 16..1024", page_size);
    if (n_pages < 1 || (int64_t)n_pages * page_size > 0x7FFFFFFF)
        return fail(SXQ_ERR_INVALID, "kv_reserve: n_pages %d (1 or more, n_pages * page_size below 2^31)", n_pages);
    if (n_rows < 1 || max_blocks < 1 || (int64_t)n_rows * max_blocks > 0x7FFFFFFF ||
        (int64_t)max_blocks * page_size > 0x7FFFFFFF)
        return fail(SXQ_ERR_INVALID, "kv_reserve: a table of %d rows of %d blocks", n_rows, max_blocks);
    if (table_stride < max_blocks) return fail(SXQ_ERR_SHAPE, "kv_reserve: table_stride %lld below max_blocks %d", (long long)table_stride, max_blocks);
    if (capacity < 0 || capacity > 1 << 30) return fail(SXQ_ERR_INVALID, "kv_reserve: capacity %d (0..2^30)", capacity);
    if (!add || !lens || !table || !free_list || !free_count || !cu || !status || (capacity > 0 && (!slots || !pos || !rows)))
        return fail(SXQ_ERR_INVALID, "kv_reserve: null pointer");
    DeviceGuard g(device);
    HIP_TRY(g.err, "hipSetDevice");
    KvReserve a;
    a.shift = __builtin_ctz((unsigned)page_size);
    a.n_pages = n_pages;
    a.n_rows = n_rows;
    a.max_blocks = max_blocks;
    a.capacity = a.limit = capacity;
    a.table_stride = table_stride;
    a.add = add;
    a.lens = lens;
    a.table = table;
    a.free_list = free_list;
    a.free_count = free_count;
    a.cu = cu;
    a.slots = slots;
    a.pos = pos;
    a.rows = rows;
    a.status = status;
    HIP_TRY(launch_kv_reserve(a, (hipStream_t)stream), "kv_reserve");
    return SXQ_OK;
}

sxq_status sxq_kv_append(int device, const sxq_kv_pages* pages, int in_dtype, const void* qkv, int64_t row_stride,
                         int n_tokens, int n_heads, const float* q_norm, const float* k_norm, float eps,
                         const float* cos, const float* sin, int max_pos, int interleaved, const int32_t* pos,
                         const int32_t* slots, void* q_out, void* stream) {
    KvPool p;
    if (sxq_status st = kv_pool("kv_append", pages, n_tokens > 0, &p)) return st;
    if (!kv_dtype(in_dtype)) return fail(SXQ_ERR_DTYPE, "kv_append: qkv dtype %d (f32, f16 or bf16)", in_dtype);
    if (n_tokens < 0 || n_heads < 1 || n_heads > 16384) return fail(SXQ_ERR_INVALID, "kv_append: %d tokens of %d heads", n_tokens, n_heads);
    const int64_t width = ((int64_t)n_heads + 2 * p.nkv) * p.hd;
    if (row_stride < width) return fail(SXQ_ERR_SHAPE, "kv_append: row_stride %lld below the row's %lld elements", (long long)row_stride, (long long)width);
    if ((cos == nullptr) != (sin == nullptr) || (cos && max_pos < 1))
        return fail(SXQ_ERR_INVALID, "kv_append: RoPE takes both tables and max_pos >= 1");
    if (n_tokens == 0) return SXQ_OK;
    if (!qkv || !slots || (cos && !pos)) return fail(SXQ_ERR_INVALID, "kv_append: null pointer");
    DeviceGuard g(device);
    HIP_TRY(g.err, "hipSetDevice");
    KvAppend a;
    a.qkv = qkv;
    a.row_stride = row_stride;
    a.dtype = in_dtype;
    a.n_tokens = n_tokens;
    a.nh = n_heads;
    a.q_norm = q_norm;
    a.k_norm = k_norm;
    a.eps = eps;
    a.cos = cos;
    a.sin = sin;
    a.max_pos = max_pos;
    a.interleaved = interleaved != 0;
    a.pos = pos;
    a.slots = slots;
    a.q_out = q_out;
    HIP_TRY(launch_kv_append(a, p, (hipStream_t)stream), "kv_append");
    return SXQ_OK;
}

}  // extern "C"
