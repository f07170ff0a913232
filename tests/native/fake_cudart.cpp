// Stands in front of the CUDA runtime (LD_PRELOAD) on a machine without a GPU, so that host code's answer to a
// failing call can be tested: cluster queries fail as often as fake_fail_queries says, launches are counted
// and run nothing, everything else succeeds.
#include <cstddef>
#include <cstdint>

namespace
{
int g_fail = 0, g_launches = 0, g_word = 0;
int encode(...) { return 0; }
} // namespace

extern "C"
{
void fake_fail_queries(int n) { g_fail = n; }
int fake_launches() { return g_launches; }

int cudaGetDevice(int* device)
{
    *device = 0;
    return 0;
}
int cudaDeviceGetAttribute(int* value, int, int)
{
    *value = 148;
    return 0;
}
int cudaFuncSetAttribute(const void*, int, int) { return 0; }
int cudaGetLastError() { return 0; }
int cudaGetSymbolAddress(void** p, const void*)
{
    *p = &g_word;
    return 0;
}
int cudaGetDriverEntryPointByVersion(const char*, void** fn, unsigned, unsigned long long, int* found)
{
    *fn = reinterpret_cast<void*>(&encode);
    *found = 0;
    return 0;
}
int cudaOccupancyMaxActiveClusters(int* n, const void*, const void*)
{
    if (g_fail > 0)
    {
        --g_fail;
        return 2;   // out of memory
    }
    *n = 74;
    return 0;
}
int cudaLaunchKernelExC(const void*, const void*, void**)
{
    ++g_launches;
    return 0;
}
}
