// sim_hip.hip -- see sim_hip.h.
#include <hip/hip_runtime.h>

#include <cstdlib>
#include <cstring>
#include <map>
#include <memory>

#include "sim_hip.h"

extern thread_local int allocations;  // host_tests.hip

namespace {

using Work = std::function<void()>;

std::map<const void*, std::string>& names() {
    static std::map<const void*, std::string> m;
    return m;
}
std::vector<std::pair<std::string, sim::Body>> bodies;
thread_local hipError_t last = hipSuccess;
std::vector<Work>* capture = nullptr;  // the one stream being captured
hipStream_t captured_stream = nullptr;

hipError_t ret(hipError_t e) {
    if (e != hipSuccess) last = e;
    return e;
}
bool fails() {
    sim::State& s = sim::state();
    ++s.calls;
    if (s.fail_in < 0) return false;
    if (s.fail_in > 0) return --s.fail_in, false;
    if (--s.fail_times == 0) s.fail_in = -1, s.fail_times = 1;
    return true;
}
void enqueue(hipStream_t s, Work w) {
    if (capture && s == captured_stream) capture->push_back(std::move(w));
    else w();
}

struct Config {
    dim3 grid, block;
    size_t shared;
    hipStream_t stream;
};
thread_local Config config;

}  // namespace

namespace sim {
State& state() {
    static State s;
    return s;
}
void kernel(const char* name_part, Body body) { bodies.emplace_back(name_part, std::move(body)); }
}  // namespace sim

extern "C" {

void** __hipRegisterFatBinary(const void*) {
    static void* one;
    return &one;
}
void __hipUnregisterFatBinary(void**) {}
void __hipRegisterFunction(void**, const void* host, char*, const char* name, unsigned, void*, void*, void*, void*, int*) {
    names()[host] = name;
}
void __hipRegisterVar(void**, void*, char*, char*, int, size_t, int, int) {}
hipError_t __hipPushCallConfiguration(dim3 grid, dim3 block, size_t shared, hipStream_t stream) {
    config = {grid, block, shared, stream};
    return hipSuccess;
}
hipError_t __hipPopCallConfiguration(dim3* grid, dim3* block, size_t* shared, hipStream_t* stream) {
    *grid = config.grid;
    *block = config.block;
    *shared = config.shared;
    *stream = config.stream;
    return hipSuccess;
}

hipError_t hipLaunchKernel(const void* f, dim3 grid, dim3 block, void** args, size_t, hipStream_t stream) {
    if (fails()) return ret(hipErrorLaunchFailure);
    const unsigned g[3] = {grid.x, grid.y, grid.z}, b[3] = {block.x, block.y, block.z};
    for (int d = 0; d < 3; ++d)
        if (!g[d] || (uint64_t)g[d] * b[d] > 0xFFFFFFFFull || (d && g[d] > 65535)) return ret(hipErrorInvalidConfiguration);
    struct Free {  // the records take no part in a test's count
        int all = allocations;
        Free() { allocations = -1; }
        ~Free() { allocations = all; }
    } records;
    const std::string& name = names()[f];
    sim::state().launches.push_back({name, {g[0], g[1], g[2]}, {b[0], b[1], b[2]}});
    for (auto& k : bodies)
        if (name.find(k.first) != std::string::npos) {
            enqueue(stream, k.second(args));
            break;
        }
    return hipSuccess;
}
hipError_t hipFuncSetAttribute(const void*, hipFuncAttribute, int) { return hipSuccess; }
hipError_t hipGetLastError() {
    const hipError_t e = last;
    last = hipSuccess;
    return e;
}
const char* hipGetErrorString(hipError_t e) { return e == hipErrorOutOfMemory ? "out of memory" : e == hipSuccess ? "no error" : "simulated"; }

hipError_t hipGetDeviceCount(int* n) {
    *n = 1;
    return hipSuccess;
}
hipError_t hipGetDevice(int* d) {
    if (sim::state().on_call) sim::state().on_call();
    *d = 0;
    return hipSuccess;
}
hipError_t hipSetDevice(int) { return hipSuccess; }
hipError_t hipDeviceGetAttribute(int* v, hipDeviceAttribute_t, int) {
    *v = 256;
    return hipSuccess;
}
hipError_t hipDeviceSynchronize() {
    if (sim::state().on_sync) sim::state().on_sync();
    return hipSuccess;
}

hipError_t hipMalloc(void** p, size_t n) {
    if (n > sim::state().malloc_limit) return ret(hipErrorOutOfMemory);
    // (zero pages on demand: 256-byte aligned within a block of its own)
    char* raw = (char*)calloc(1, n + 512);
    if (!raw) return ret(hipErrorOutOfMemory);
    char* at = (char*)(((uintptr_t)raw + 256 + sizeof(void*)) & ~(uintptr_t)255);
    ((void**)at)[-1] = raw;
    *p = at;
    ++sim::state().held;
    const int all = allocations;
    allocations = -1;  // (the records' own memory)
    sim::state().mallocs.push_back(n);
    allocations = all;
    return hipSuccess;
}
hipError_t hipFree(void* p) {
    if (p) free(((void**)p)[-1]), --sim::state().held;
    return hipSuccess;
}
hipError_t hipMallocAsync(void** p, size_t n, hipStream_t) { return hipMalloc(p, n); }
hipError_t hipFreeAsync(void* p, hipStream_t) { return hipFree(p); }
hipError_t hipMemcpy(void* d, const void* s, size_t n, hipMemcpyKind) {
    memcpy(d, s, n);
    return hipSuccess;
}
hipError_t hipMemcpyAsync(void* d, const void* s, size_t n, hipMemcpyKind, hipStream_t stream) {
    if (fails()) return ret(hipErrorInvalidValue);
    enqueue(stream, [=] { memcpy(d, s, n); });
    return hipSuccess;
}
hipError_t hipMemset(void* d, int v, size_t n) {
    memset(d, v, n);
    return hipSuccess;
}
hipError_t hipMemsetAsync(void* d, int v, size_t n, hipStream_t stream) {
    if (fails()) return ret(hipErrorInvalidValue);
    enqueue(stream, [=] { memset(d, v, n); });
    return hipSuccess;
}
hipError_t hipGetSymbolAddress(void** p, const void*) {
    static char image[4096];
    *p = image;
    return hipSuccess;
}

hipError_t hipStreamCreateWithFlags(hipStream_t* s, unsigned) {
    *s = (hipStream_t)calloc(1, 16);
    return hipSuccess;
}
hipError_t hipStreamDestroy(hipStream_t s) {
    free(s);
    return hipSuccess;
}
hipError_t hipStreamSynchronize(hipStream_t) { return hipSuccess; }
hipError_t hipStreamWaitEvent(hipStream_t, hipEvent_t, unsigned) { return hipSuccess; }
hipError_t hipStreamIsCapturing(hipStream_t, hipStreamCaptureStatus* st) {
    *st = hipStreamCaptureStatusNone;
    return hipSuccess;
}
hipError_t hipEventCreateWithFlags(hipEvent_t* e, unsigned) {
    *e = (hipEvent_t)8;
    return hipSuccess;
}
hipError_t hipEventRecord(hipEvent_t, hipStream_t) { return hipSuccess; }
hipError_t hipStreamBeginCapture(hipStream_t s, hipStreamCaptureMode) {
    capture = new std::vector<Work>();
    captured_stream = s;
    return hipSuccess;
}
hipError_t hipStreamEndCapture(hipStream_t, hipGraph_t* g) {
    *g = (hipGraph_t)capture;
    capture = nullptr;
    return hipSuccess;
}
hipError_t hipGraphInstantiate(hipGraphExec_t* e, hipGraph_t g, hipGraphNode_t*, char*, size_t) {
    *e = (hipGraphExec_t) new std::vector<Work>(*(std::vector<Work>*)g);
    return hipSuccess;
}
hipError_t hipGraphDestroy(hipGraph_t g) {
    delete (std::vector<Work>*)g;
    return hipSuccess;
}
hipError_t hipGraphExecDestroy(hipGraphExec_t e) {
    delete (std::vector<Work>*)e;
    return hipSuccess;
}
hipError_t hipGraphLaunch(hipGraphExec_t e, hipStream_t) {
    if (fails()) return ret(hipErrorLaunchFailure);
    for (Work& w : *(std::vector<Work>*)e) w();
    return hipSuccess;
}

}  // extern "C"
