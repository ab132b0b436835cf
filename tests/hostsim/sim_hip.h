// sim_hip.h -- the simulated HIP runtime's controls.  Device memory is host memory; a kernel
// runs only if a test has given it a body (by a part of its name), in the order of the calls;
// the nth call that a test picks fails as the runtime would, with the error left for
// hipGetLastError.  Test infrastructure only.
#pragma once
#include <cstddef>
#include <functional>
#include <string>
#include <vector>

namespace sim {

// The arguments of a launch as it was made -> what to run when the stream gets to it.
using Body = std::function<std::function<void()>(void** args)>;
void kernel(const char* name_part, Body body);

struct Launch {
    std::string name;
    unsigned grid[3], block[3];
};
struct State {
    int fail_in = -1;             // this many more calls of the kinds below succeed, then one fails (-1: none)
    int fail_times = 1;           // and as many after it
    int calls = 0;                // kernel launches, async copies, graph launches
    size_t malloc_limit = (size_t)-1;  // a larger hipMalloc is out of memory
    int held = 0;                 // allocations not yet freed
    std::vector<size_t> mallocs;  // sizes, in order
    std::vector<Launch> launches;
    std::function<void()> on_call;  // in hipGetDevice, the first HIP call of an entry point
    std::function<void()> on_sync;  // in hipDeviceSynchronize
};
State& state();

}  // namespace sim
