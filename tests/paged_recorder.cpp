// Stands in for the HIP runtime's launch entry points in a process without a GPU, as launch_recorder.c does, for the launches of
// flash_forward_paged: kernel name, grid and what the order of their work-groups goes by.  Nothing runs.  Loaded with RTLD_GLOBAL in front of the library
// (tests/paged_launches.py).
#include "paged_kernel.h"

#include <cstring>

namespace {
constexpr int kMaxKernels = 4096, kMaxLaunches = 16;
const void* handles[kMaxKernels];
const char* names[kMaxKernels];
int kernels;

struct Launch {
    const char* name;
    long long groups;
    int order[4];  // direct, ordered, pieces, num_splits
} launches[kMaxLaunches];
int launched;
}  // namespace

#define SEEN extern "C" __attribute__((visibility("default")))

SEEN void __hipRegisterFunction(void**, const void* handle, char*, const char* name, unsigned, void*, void*, void*, void*, int*)
{
    if (kernels < kMaxKernels) handles[kernels] = handle, names[kernels++] = name;
}
SEEN hipError_t hipLaunchKernel(const void* handle, dim3 grid, dim3, void** args, size_t, hipStream_t)
{
    Launch l = {"?", grid.x, {0, 0, 0, 0}};
    for (int i = 0; i < kernels; ++i)
        if (handles[i] == handle) l.name = names[i];
    if (std::strstr(l.name, "paged_few_kernel") || std::strstr(l.name, "paged_tall_kernel")) {
        const fa::PagedArgs& a = *static_cast<const fa::PagedArgs*>(args[0]);
        l.order[0] = a.direct, l.order[1] = a.ordered, l.order[2] = a.pieces, l.order[3] = a.num_splits;
    }
    if (launched < kMaxLaunches) launches[launched++] = l;
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

SEEN void recorder_clear() { launched = 0; }
SEEN int recorder_count() { return launched; }
SEEN const char* recorder_name(int i) { return launches[i].name; }
SEEN long long recorder_groups(int i) { return launches[i].groups; }
SEEN int recorder_order(int i, int which) { return launches[i].order[which]; }
