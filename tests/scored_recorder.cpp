// Stands in for the HIP runtime's launch entry points in a process without a GPU, as paged_recorder.cpp does, for the launches of flash_forward_paged with other
// scores: their kernels, and what the order of their work-groups goes by.  Nothing runs (tests/scored_launches.py).
#include "paged_kernel.h"

#include <cstring>

namespace {
constexpr int kMaxKernels = 4096;
const void* handles[kMaxKernels];
const char* names[kMaxKernels];
int kernels;
struct {
    const char* name;
    long long groups;
    int order[4];  // direct, ordered, pieces, num_splits
} scored;
}  // namespace

#define SEEN extern "C" __attribute__((visibility("default")))

SEEN void __hipRegisterFunction(void**, const void* handle, char*, const char* name, unsigned, void*, void*, void*, void*, int*)
{
    if (kernels < kMaxKernels) handles[kernels] = handle, names[kernels++] = name;
}
SEEN hipError_t hipLaunchKernel(const void* handle, dim3 grid, dim3, void** args, size_t, hipStream_t)
{
    for (int i = 0; i < kernels; ++i)
        if (handles[i] == handle && std::strstr(names[i], "scored_")) {
            const fa::ScoredArgs& a = *static_cast<const fa::ScoredArgs*>(args[0]);
            scored = {names[i], grid.x, {a.direct, a.ordered, a.pieces, a.num_splits}};
        }
    return hipSuccess;
}
SEEN hipError_t hipGetDevice(int* device)
{
    *device = 0;
    return hipSuccess;
}
SEEN hipError_t hipGetDeviceProperties(hipDeviceProp_t* prop, int)
{
    std::memset(prop, 0, sizeof(*prop));
    std::strcpy(prop->gcnArchName, "gfx950");
    return hipSuccess;
}
SEEN hipError_t hipFuncSetAttribute(const void*, hipFuncAttribute, int) { return hipSuccess; }

SEEN void recorder_clear() { scored = {"", 0, {0, 0, 0, 0}}; }
SEEN const char* recorder_name() { return scored.name; }
SEEN long long recorder_groups() { return scored.groups; }
SEEN int recorder_order(int which) { return scored.order[which]; }
