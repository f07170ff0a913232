// Stands in front of the CUDA runtime (LD_PRELOAD) on a machine without a GPU, so that host code's answer to a
// failing call can be tested: cluster queries fail as often as fake_fail_queries says, launches are counted
// and run nothing, everything else succeeds.
#include <cstddef>
#include <cstdint>

namespace
{
int g_fail = 0, g_launches = 0, g_word = 0;
// cudaLaunchConfig_t and cudaLaunchAttribute, as far as they are looked at
struct Attribute
{
    int id;
    char pad[4];
    char value[64];
};
struct Config
{
    unsigned grid[3], block[3];
    size_t smem;
    void* stream;
    const Attribute* attrs;
    unsigned count;
};
constexpr int kKept = 4096;
struct Launch
{
    int smem, overlapped, cooperative;
};
Launch g_kept[kKept];
int encode(...) { return 0; }
} // namespace

extern "C"
{
void fake_fail_queries(int n) { g_fail = n; }
int fake_launches() { return g_launches; }
// Launch i: its dynamic shared memory, and whether it may overlap the one before it or is cooperative.
void fake_launch(int i, int* smem, int* overlapped, int* cooperative)
{
    *smem = g_kept[i % kKept].smem;
    *overlapped = g_kept[i % kKept].overlapped;
    *cooperative = g_kept[i % kKept].cooperative;
}

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
int cudaLaunchKernelExC(const Config* c, const void*, void**)
{
    Launch& l = g_kept[g_launches++ % kKept];
    l = {static_cast<int>(c->smem), 0, 0};
    for (unsigned k = 0; k < c->count; ++k)
    {
        l.cooperative |= c->attrs[k].id == 2;
        l.overlapped |= c->attrs[k].id == 6;   // programmatic stream serialization
    }
    return 0;
}
}
