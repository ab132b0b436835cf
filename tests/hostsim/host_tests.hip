// host_tests.hip -- the decode engine's host side on the simulated runtime: what a call does
// to lengths, pages and workspaces when another call fails or runs beside it.
//   host_tests NAME      runs one test, prints "ok"
#include <hip/hip_runtime.h>

#include <atomic>
#include <chrono>
#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <map>
#include <new>
#include <thread>

#include "../../include/sxq.h"
#include "sim_hip.h"
#include "sxq_decoder.h"
#include "sxq_paged.h"
#include "sxq_paged_launch.h"

using namespace sxq;

// Host allocations that still succeed before one fails (-1: all do).
thread_local int allocations = -1;
void* operator new(size_t n) {
    if (allocations == 0) {
        allocations = -1;
        throw std::bad_alloc();
    }
    if (allocations > 0) --allocations;
    return std::malloc(n ? n : 1);
}
void operator delete(void* p) noexcept { std::free(p); }
void operator delete(void* p, size_t) noexcept { std::free(p); }

#define EXPECT(c)                                                                                            \
    do {                                                                                                     \
        if (!(c)) {                                                                                          \
            std::fprintf(stderr, "failed: %s (line %d; last error: %s)\n", #c, __LINE__, sxq_last_error()); \
            std::exit(1);                                                                                    \
        }                                                                                                    \
    } while (0)

namespace {

// What the engine's last reserve worked on: its device lengths, table and free stack.
KvReserve seen{};

void reserve_rows(const KvReserve& a) {
    seen = a;
    auto blocks = [&](int64_t n) { return (int)((n + (1 << a.shift) - 1) >> a.shift); };
    std::vector<int> back;
    for (int r = 0; r < a.n_rows; ++r) {
        if (a.add[r] >= 0) continue;
        const int keep = (int)std::max<int64_t>(0, (int64_t)a.lens[r] + a.add[r]);
        for (int b = blocks(keep); b < blocks(a.lens[r]); ++b) {
            back.push_back(a.table[r * a.table_stride + b]);
            a.table[r * a.table_stride + b] = -1;
        }
        a.lens[r] = keep;
    }
    for (auto it = back.rbegin(); it != back.rend(); ++it) a.free_list[a.free_count[0]++] = *it;
    const int avail = a.free_count[0];
    int64_t asked = 0, room = 0;
    int t = 0;
    a.cu[0] = 0;
    for (int r = 0; r < a.n_rows; ++r) {
        a.status[r] = 0;
        if (a.add[r] >= 0) {
            const int64_t grown = (int64_t)a.lens[r] + a.add[r];
            const int have = blocks(a.lens[r]), need = blocks(grown) - have;
            if (grown > (int64_t)a.max_blocks << a.shift) a.status[r] = 2;
            else {
                asked += need;
                room += a.add[r];
                if (need && asked > avail) a.status[r] = 1;
                else if (a.add[r] && room > a.limit) a.status[r] = 3;
                else {
                    for (int b = have; b < have + need; ++b) a.table[r * a.table_stride + b] = a.free_list[--a.free_count[0]];
                    for (int64_t p = a.lens[r]; p < grown; ++p, ++t)
                        if (t < a.capacity) {
                            a.slots[t] = kv_slot(a.table[r * a.table_stride + (p >> a.shift)], (int)p, a.shift, a.n_pages);
                            a.pos[t] = (int)p;
                            a.rows[t] = r;
                        }
                    a.lens[r] = (int)grown;
                }
            }
        }
        a.cu[r + 1] = t;
    }
    for (; t < a.capacity; ++t) a.slots[t] = a.pos[t] = a.rows[t] = -1;
}

std::vector<int> stored;  // the slots of the last append, by row
std::vector<KvAppend> appends;

// Bodies of the kernels that keep an engine's lengths and pages.
void page_kernels() {
    sim::kernel("k_kv_reserve", [](void** args) {
        const KvReserve a = *(const KvReserve*)args[0];
        return [a] { reserve_rows(a); };
    });
    sim::kernel("k_kv_by_row", [](void** args) {
        const int32_t *cu = *(int32_t**)args[0], *ms = *(int32_t**)args[1], *mp = *(int32_t**)args[2];
        const int rows = *(int*)args[3];
        int32_t *slots = *(int32_t**)args[4], *pos = *(int32_t**)args[5];
        return [=] {
            for (int r = 0; r < rows; ++r) {
                const bool has = cu[r + 1] > cu[r];
                slots[r] = has ? ms[cu[r]] : -1;
                pos[r] = has ? mp[cu[r]] : 0;
            }
        };
    });
    sim::kernel("k_kv_append", [](void** args) {
        const KvAppend a = *(const KvAppend*)args[0];
        return [a] {
            appends.push_back(a);
            stored.assign(a.slots, a.slots + a.n_tokens);
        };
    });
    sim::kernel("k_kv_stack", [](void** args) {
        int32_t* list = *(int32_t**)args[0];
        const int n = *(int*)args[1];
        return [=] { for (int i = 0; i < n; ++i) list[i] = n - 1 - i; };
    });
    sim::kernel("k_fill_int", [](void** args) {
        int* y = *(int**)args[0];
        const int n = *(int*)args[1], v = *(int*)args[2];
        return [=] { for (int i = 0; i < n; ++i) y[i] = v; };
    });
    sim::kernel("k_kv_growths", [](void** args) {
        const KvGrowths g = *(const KvGrowths*)args[0];
        int32_t* add = *(int32_t**)args[1];
        return [=] { for (int i = 0; i < g.n; ++i) add[i] = g.add[i]; };
    });
}

sxq_lm_config config(int max_seq, int max_batch) {
    sxq_lm_config c{};
    c.n_layers = 1;
    c.dim = 256;
    c.n_heads = 4;
    c.n_kv_heads = 2;
    c.head_dim = 64;
    c.intermediate = 256;
    c.vocab = 64;
    c.max_seq = max_seq;
    c.max_batch = max_batch;
    c.weight_dtype = SXQ_Q8_0;
    c.norm_eps = 1e-6f;
    c.rope_theta = 1e6f;
    return c;
}

struct Engine {
    sxq_lm* lm = nullptr;
    int n, pages;
    std::vector<float> embeds, logits;
    Engine(int pages_, int max_seq = 20000, int batch = 4, int page = 16) : n(batch), pages(pages_) {
        const sxq_lm_config c = config(max_seq, batch);
        EXPECT(sxq_lm_create_paged(0, &c, SXQ_F32, page, pages, &lm) == SXQ_OK);
        embeds.resize((size_t)c.dim * 70000);
        logits.resize((size_t)c.vocab * batch);
    }
    ~Engine() { sxq_lm_destroy(lm); }
    sxq_status step(int streams, unsigned flags = 0) {
        return sxq_lm_step(lm, streams, nullptr, embeds.data(), logits.data(), nullptr, nullptr, flags, nullptr);
    }
    sxq_status prefill(std::vector<int32_t> counts) {
        return sxq_lm_prefill(lm, (int)counts.size(), counts.data(), nullptr, embeds.data(), logits.data(), nullptr, nullptr,
                              0, nullptr, 0, nullptr);
    }
    std::vector<int32_t> lengths() {
        std::vector<int32_t> v(n);
        EXPECT(sxq_lm_get_lengths(lm, v.data(), n) == SXQ_OK);
        return v;
    }
    int free_pages() {
        int f = -1;
        EXPECT(sxq_lm_free_pages(lm, &f) == SXQ_OK);
        return f;
    }
    // The device's lengths are the host's, every page is held once or free once.
    void consistent() {
        EXPECT(seen.lens);
        const std::vector<int32_t> host = lengths();
        std::vector<int> times(pages, 0);
        for (int s = 0; s < n; ++s) {
            EXPECT(seen.lens[s] == host[s]);
            for (int b = 0; b < kv_blocks(host[s], seen.shift); ++b) {
                const int id = seen.table[s * seen.table_stride + b];
                EXPECT(id >= 0 && id < pages);
                ++times[id];
            }
        }
        EXPECT(seen.free_count[0] == free_pages());
        for (int i = 0; i < seen.free_count[0]; ++i) ++times[seen.free_list[i]];
        for (int id = 0; id < pages; ++id) EXPECT(times[id] == 1);
    }
};

// A call that fails leaves no error behind for the next one to report.
void error_of_one_call() {
    Engine e(100);
    EXPECT(e.prefill({5, 20}) == SXQ_OK);
    e.consistent();
    sim::state().malloc_limit = 1 << 16;
    EXPECT(e.prefill({900, 3}) == SXQ_ERR_OOM && std::strstr(sxq_last_error(), "workspace"));
    sim::state().malloc_limit = (size_t)-1;
    EXPECT(hipGetLastError() == hipSuccess);  // nor for the caller's own next launch
    e.consistent();
    EXPECT(e.step(2) == SXQ_OK);
    e.consistent();
    EXPECT((e.lengths() == std::vector<int32_t>{6, 21, 0, 0}));
}

// Whichever of a call's launches and copies fails, the call can be made again: lengths, pages
// and the map stay as the host has them.  Steps (eager, captured, replayed) and prompts.
void failed_calls() {
    for (const char* kind : {"step", "graph", "replay", "prompt"}) {
        const std::string k = kind;
        for (int at = 0;; ++at) {
            Engine e(60, 2000);
            EXPECT(e.prefill({15, 33, 1}) == SXQ_OK && e.step(3) == SXQ_OK);
            if (k == "replay") EXPECT(e.step(3, SXQ_LM_GRAPH) == SXQ_OK);
            e.consistent();
            const std::vector<int32_t> before = e.lengths();
            auto call = [&] { return k == "prompt" ? e.prefill({300, 2, 17}) : e.step(3, k == "step" ? 0 : SXQ_LM_GRAPH); };
            sim::state().fail_in = at;
            const sxq_status st = call();
            const bool all_passed = sim::state().fail_in >= 0;  // fewer calls than that: nothing failed
            sim::state().fail_in = -1;
            e.consistent();
            if (all_passed) {
                EXPECT(st == SXQ_OK && at > (k == "replay" ? 1 : 9));
                break;
            }
            EXPECT(st == SXQ_ERR_DEVICE);
            if (e.lengths() != before) continue;  // what failed was a copy out, after the work
            EXPECT(call() == SXQ_OK);
            e.consistent();
            for (int s = 0; s < 3; ++s) EXPECT(e.lengths()[s] == before[s] + (k == "prompt" ? (int[]){300, 2, 17}[s] : 1));
        }
    }
}

// Where the pages cannot be put back either (the device is lost, say), later calls say so
// instead of running on lengths that the host does not know, until the streams are emptied.
void failed_undo() {
    Engine e(60, 2000);
    EXPECT(e.prefill({15, 33, 1}) == SXQ_OK);
    sim::State& s = sim::state();
    const int before = s.calls;
    EXPECT(e.step(3) == SXQ_OK);
    const int per_step = s.calls - before;
    s.fail_in = per_step / 2;
    s.fail_times = 100;
    EXPECT(e.step(3) == SXQ_ERR_DEVICE);
    s.fail_in = -1;
    s.fail_times = 1;
    for (int again = 0; again < 2; ++again) {
        EXPECT(e.step(3) == SXQ_ERR_INVALID && std::strstr(sxq_last_error(), "reset"));
        EXPECT(e.prefill({4}) == SXQ_ERR_INVALID);
        const int32_t one = 3;
        EXPECT(sxq_lm_set_lengths(e.lm, &one, 1) == SXQ_ERR_INVALID);
        EXPECT(sxq_lm_reset(e.lm, 2, nullptr) == SXQ_ERR_INVALID);  // not all of them
    }
    EXPECT(sxq_lm_reset(e.lm, e.n, nullptr) == SXQ_OK);
    e.consistent();
    EXPECT(e.free_pages() == 60 && e.prefill({15, 33, 1}) == SXQ_OK && e.step(3) == SXQ_OK);
    e.consistent();
}

// A thread that asks for the free pages or the lengths waits for a call that is changing them.
void lengths_are_read_under_the_lock() {
    Engine e(60, 2000);
    const int32_t lens[2] = {40, 3}, more[2] = {100, 90};
    EXPECT(sxq_lm_set_lengths(e.lm, lens, 2) == SXQ_OK);
    for (int what = 0; what < 2; ++what) {
        std::atomic<bool> returned{false}, during{false};
        std::thread reader;
        sim::state().on_sync = [&] {
            if (reader.joinable()) return;
            reader = std::thread([&] {
                int32_t v[2] = {0, 0};
                int pages = 0;
                if (what) EXPECT(sxq_lm_get_lengths(e.lm, v, 2) == SXQ_OK);
                else EXPECT(sxq_lm_free_pages(e.lm, &pages) == SXQ_OK);
                returned = true;
            });
            for (int i = 0; i < 200 && !returned; ++i) std::this_thread::sleep_for(std::chrono::milliseconds(1));
            during = returned.load();
        };
        EXPECT(sxq_lm_set_lengths(e.lm, what ? lens : more, 2) == SXQ_OK);
        reader.join();
        sim::state().on_sync = nullptr;
        EXPECT(!during && returned);
    }
}

// What a step or a prompt checks before its first HIP call takes no host memory: an exception
// would leave through the C entry.
void checks_allocate_nothing() {
    Engine e(10, 2000);
    EXPECT(e.prefill({30, 50}) == SXQ_OK);
    sim::state().on_call = [] { allocations = -1; };
    allocations = 0;
    EXPECT(e.step(2) == SXQ_OK);
    const int32_t big[2] = {300, 5};
    for (int i = 0; i < 2; ++i) {
        allocations = 0;
        EXPECT(i ? e.step(2) == SXQ_OK
                 : sxq_lm_prefill(e.lm, 2, big, nullptr, e.embeds.data(), nullptr, nullptr, nullptr, 0, nullptr, 0, nullptr) == SXQ_ERR_OOM);
    }
    allocations = -1;
    sim::state().on_call = nullptr;
    e.consistent();
}

// Creation runs out of host memory at each of its allocations in turn: an error, every device
// allocation given back.
void creation_out_of_host_memory() {
    const sxq_lm_config c = config(3000, 4);
    for (int paged = 0; paged < 2; ++paged)
        for (int at = 0;; ++at) {
            sxq_lm* lm = nullptr;
            const int held = sim::state().held;
            allocations = at;
            const sxq_status st = paged ? sxq_lm_create_paged(0, &c, SXQ_F32, 16, 100, &lm) : sxq_lm_create(0, &c, &lm);
            const bool enough = allocations > 0;
            allocations = -1;
            EXPECT(st == (lm ? SXQ_OK : SXQ_ERR_OOM) && (lm || sim::state().held == held));
            if (lm) {
                sxq_lm_destroy(lm);
                EXPECT(sim::state().held == held);
            }
            if (enough) break;
        }
}

// Steps in which some streams sit out: those keep lengths and pages, the others' rows get their
// own slots; eager, captured and replayed, each failing at each of its calls.
void streams_that_sit_out() {
    for (unsigned flags : {0u, (unsigned)SXQ_LM_GRAPH}) {
        Engine e(40, 2000);
        EXPECT(e.prefill({15, 31, 7, 64}) == SXQ_OK);
        auto some = [&](std::vector<int32_t> active) {
            return sxq_lm_step_active(e.lm, 4, active.data(), nullptr, e.embeds.data(), e.logits.data(), nullptr, nullptr, flags, nullptr);
        };
        std::vector<int32_t> want = e.lengths();
        for (int turn = 0; turn < 40; ++turn) {
            std::vector<int32_t> active(4);
            for (int s = 0; s < 4; ++s) active[s] = (turn >> s & 1) * (turn + 3);  // any value but 0
            EXPECT(some(active) == SXQ_OK);
            for (int s = 0; s < 4; ++s) {
                want[s] += active[s] != 0;
                const int p = want[s] - 1;
                EXPECT(stored[s] == (active[s] ? seen.table[s * seen.table_stride + (p >> 4)] * 16 + (p & 15) : -1));
            }
            EXPECT(e.lengths() == want);
            e.consistent();
            if (turn % 7 == 3) {
                EXPECT(e.step(4, flags) == SXQ_OK);
                for (int& v : want) ++v;
                e.consistent();
            }
        }
        for (int at = 0;; ++at) {
            sim::state().fail_in = at;
            const sxq_status st = some({1, 0, 1, 0});
            const bool all_passed = sim::state().fail_in >= 0;
            sim::state().fail_in = -1;
            e.consistent();
            if (all_passed) break;
            EXPECT(st == SXQ_ERR_DEVICE);
        }
    }
    // the pool counts only those that take part
    Engine e(4, 2000, 2);
    EXPECT(e.prefill({32, 32}) == SXQ_OK);
    const int32_t one[2] = {0, 1}, none[2] = {0, 0}, small[2] = {16, 32};
    EXPECT(sxq_lm_step_active(e.lm, 2, one, nullptr, e.embeds.data(), nullptr, nullptr, nullptr, 0, nullptr) == SXQ_ERR_OOM);
    EXPECT(sxq_lm_step_active(e.lm, 2, none, nullptr, e.embeds.data(), nullptr, nullptr, nullptr, 0, nullptr) == SXQ_OK);
    EXPECT(sxq_lm_set_lengths(e.lm, small, 2) == SXQ_OK && e.step(2) == SXQ_ERR_OOM);
    EXPECT(sxq_lm_step_active(e.lm, 2, one, nullptr, e.embeds.data(), nullptr, nullptr, nullptr, 0, nullptr) == SXQ_OK);
    e.consistent();
    // nor does a full stream that sits out stop the others
    Engine f(20, 64, 2);
    EXPECT(f.prefill({64, 3}) == SXQ_OK && f.step(2) == SXQ_ERR_INVALID);
    EXPECT(sxq_lm_step_active(f.lm, 2, one, nullptr, f.embeds.data(), nullptr, nullptr, nullptr, 0, nullptr) == SXQ_OK);
    // a contiguous engine's streams cannot
    const sxq_lm_config c = config(64, 2);
    sxq_lm* lm = nullptr;
    EXPECT(sxq_lm_create(0, &c, &lm) == SXQ_OK);
    const int32_t all[2] = {1, 1};
    EXPECT(sxq_lm_step_active(lm, 2, one, nullptr, e.embeds.data(), nullptr, nullptr, nullptr, 0, nullptr) == SXQ_ERR_INVALID);
    EXPECT(sxq_lm_step_active(lm, 2, all, nullptr, e.embeds.data(), nullptr, nullptr, nullptr, 0, nullptr) == SXQ_OK);
    EXPECT(sxq_lm_destroy(lm) == SXQ_OK);
}

// A prompt's workspace holds f32 keys and values of the positions there are, not of streams times
// the longest; and a conversation that grows chunk by chunk allocates it a few times, not at
// every chunk.  Where the headroom does not fit, the bare size does.
void prompt_workspace() {
    const size_t row = 2 * 2 * 64 * sizeof(float);  // K and V of a position, two heads of 64
    const size_t token = 64 << 10;                  // more than the other buffers take for a token
    {
        Engine e(16000 / 16 + 40, 20000, 16);
        std::vector<int32_t> counts(16, 10);
        counts[3] = 16000;
        std::vector<size_t>& m = sim::state().mallocs;
        const size_t before = m.size();
        EXPECT(e.prefill(counts) == SXQ_OK);
        std::vector<int32_t> few(16, 1);
        EXPECT(e.prefill(few) == SXQ_OK);
        EXPECT(m.size() == before + 1 && m.back() < 1.5 * (16150 + 16) * row + 16150 * token);
    }
    {
        Engine e(1250, 20000, 16);
        std::vector<size_t>& m = sim::state().mallocs;
        std::vector<int32_t> small(16, 1), lens(16, 10);
        lens[3] = 16000;
        EXPECT(sxq_lm_set_lengths(e.lm, lens.data(), 16) == SXQ_OK);
        const size_t before = m.size();
        EXPECT(e.prefill(small) == SXQ_OK && m.size() == before + 1);
        EXPECT(m.back() < 1.5 * 16200 * row + 16 * token);  // (streams times the longest: 16 * 16001 * row)
    }
    {
        Engine e(1250, 20000, 2);
        std::vector<size_t>& m = sim::state().mallocs;
        const size_t before = m.size();
        int calls = 0;
        for (; e.lengths()[0] < 19000; ++calls) EXPECT(e.prefill({64, 2}) == SXQ_OK);
        EXPECT(calls > 290 && m.size() - before <= 16);
        const size_t last = m.back();
        const int32_t lens[2] = {0, 10};
        EXPECT(last <= 1250 * 16 * row + 66 * token);  // never for more positions than the pool has
        EXPECT(sxq_lm_set_lengths(e.lm, lens, 2) == SXQ_OK && e.prefill({64, 2}) == SXQ_OK && m.back() == last);
    }
    {
        Engine e(1250, 20000, 2);
        const int32_t lens[2] = {9000, 9000};
        EXPECT(sxq_lm_set_lengths(e.lm, lens, 2) == SXQ_OK);
        sim::state().malloc_limit = 18200 * row + 10 * token;  // no room for more
        EXPECT(e.prefill({4, 4}) == SXQ_OK);
        EXPECT(e.step(2) == SXQ_OK);
        e.consistent();
        sim::state().malloc_limit = (size_t)-1;
    }
}

// Tokens beyond what one launch's grid may hold (2^32 threads): in parts, each at its own rows.
void append_of_many_tokens() {
    const int n = (1 << 24) + 5, width = 3 * 8;
    sxq_kv_pages p{};
    p.dtype = SXQ_F16;
    p.n_kv_heads = 1;
    p.head_dim = 8;
    p.page_size = 16;
    p.n_pages = 4;
    p.k = p.v = (void*)4096;
    p.pos_stride = 8;
    p.head_stride = 128;
    p.page_stride = 128;
    std::vector<int32_t> slots(n, -1), pos(n, 0);
    uint16_t* const qkv = (uint16_t*)(uintptr_t)(1 << 20);
    uint16_t* const out = (uint16_t*)((uintptr_t)1 << 40);
    float tables[8] = {};
    EXPECT(sxq_kv_append(0, &p, SXQ_F16, qkv, width + 8, n, 1, nullptr, nullptr, 1e-6f, tables, tables, 2, 0, pos.data(),
                         slots.data(), out, nullptr) == SXQ_OK);
    int64_t at = 0;
    size_t i = sim::state().launches.size() - appends.size();
    for (const KvAppend& a : appends) {
        EXPECT(a.slots == slots.data() + at && a.pos == pos.data() + at && a.qkv == qkv + at * (width + 8) && a.q_out == out + at * 8);
        EXPECT(a.n_tokens > 0 && sim::state().launches[i++].grid[0] == (unsigned)a.n_tokens);
        at += a.n_tokens;
    }
    EXPECT(at == n && appends.size() > 1);
}

const std::map<std::string, void (*)()> kTests = {
    {"append_of_many_tokens", append_of_many_tokens},
    {"checks_allocate_nothing", checks_allocate_nothing},
    {"creation_out_of_host_memory", creation_out_of_host_memory},
    {"error_of_one_call", error_of_one_call},
    {"failed_calls", failed_calls},
    {"failed_undo", failed_undo},
    {"lengths_are_read_under_the_lock", lengths_are_read_under_the_lock},
    {"prompt_workspace", prompt_workspace},
    {"streams_that_sit_out", streams_that_sit_out},
};

}  // namespace

int main(int argc, char** argv) {
    const auto it = kTests.find(argc > 1 ? argv[1] : "");
    if (it == kTests.end()) {
        for (auto& t : kTests) std::puts(t.first.c_str());
        return argc > 1;
    }
    page_kernels();
    it->second();
    std::puts("ok");
}
