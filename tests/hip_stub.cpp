// hip_stub.cpp -- the HIP calls of attn_ops.cpp on the CPU: device memory is what a test
// names, and a launch is noted, never run.  Built with attn_ops.cpp into one library, it
// shows which calls are refused and what the others would enqueue.
#include <hip/hip_runtime_api.h>
#include <stdarg.h>
#include <stdio.h>
#include <string.h>

#include <string>
#include <vector>

struct Range {
    uintptr_t at, bytes;
    int device;
};
struct Launch {
    std::string name;
    uint32_t grid[3], block;
    std::vector<uint8_t> args;
};
static std::vector<Range> g_ranges;
static std::vector<std::string *> g_functions;
static std::vector<Launch> g_launches;
static char g_error[512];
static size_t g_args_bytes;
static int g_refuse; // which call fails: 1 hipModuleLoad, 2 hipModuleGetFunction, 3 hipModuleLaunchKernel
static hipError_t g_left; // what the runtime would report next

static hipError_t answer(int call)
{
    if (g_refuse == call)
        g_left = hipErrorUnknown;
    return g_refuse == call ? hipErrorUnknown : hipSuccess;
}
extern "C" void stub_refuse(int call) { g_refuse = call; }
extern "C" int stub_left() { return (int)g_left; }

extern "C" void stub_reset(size_t args_bytes)
{
    g_ranges.clear();
    g_launches.clear();
    g_args_bytes = args_bytes; // read of every launch's first argument
}
extern "C" void stub_memory(uintptr_t at, uintptr_t bytes, int device) { g_ranges.push_back({at, bytes, device}); }
extern "C" int stub_launches() { return (int)g_launches.size(); }
extern "C" const char *stub_launch(int i, uint32_t *grid, uint32_t *block)
{
    memcpy(grid, g_launches[i].grid, sizeof(g_launches[i].grid));
    *block = g_launches[i].block;
    return g_launches[i].name.c_str();
}
extern "C" const void *stub_args(int i) { return g_launches[i].args.data(); }
extern "C" const char *stub_error() { return g_error; }

int lfm_vfail(int code, const char *fmt, va_list ap)
{
    vsnprintf(g_error, sizeof(g_error), fmt, ap);
    return code;
}
std::string lfm_beside_code_object(const char *file) { return file; }

hipError_t hipGetDevice(int *d)
{
    *d = 0;
    return hipSuccess;
}
hipError_t hipStreamGetDevice(hipStream_t, hipDevice_t *d)
{
    *d = 0;
    return hipSuccess;
}
hipError_t hipGetLastError()
{
    const hipError_t e = g_left;
    g_left = hipSuccess;
    return e;
}
const char *hipGetErrorString(hipError_t) { return "stub"; }
hipError_t hipPointerGetAttributes(hipPointerAttribute_t *a, const void *p)
{
    for (const Range &r : g_ranges)
        if ((uintptr_t)p >= r.at && (uintptr_t)p < r.at + r.bytes) {
            a->type = hipMemoryTypeDevice;
            a->device = r.device;
            return hipSuccess;
        }
    return g_left = hipErrorInvalidValue;
}
hipError_t hipModuleLoad(hipModule_t *m, const char *)
{
    *m = (hipModule_t)&g_functions;
    return answer(1);
}
hipError_t hipModuleUnload(hipModule_t) { return hipSuccess; }
hipError_t hipModuleGetFunction(hipFunction_t *f, hipModule_t, const char *name)
{
    g_functions.push_back(new std::string(name));
    *f = (hipFunction_t)g_functions.back();
    return answer(2);
}
hipError_t hipModuleLaunchKernel(hipFunction_t f, unsigned gx, unsigned gy, unsigned gz, unsigned bx, unsigned,
                                 unsigned, unsigned, hipStream_t, void **params, void **)
{
    if (answer(3) != hipSuccess)
        return hipErrorUnknown;
    Launch l;
    l.name = *(const std::string *)f;
    l.grid[0] = gx, l.grid[1] = gy, l.grid[2] = gz, l.block = bx;
    if (g_args_bytes)
        l.args.assign((const uint8_t *)params[0], (const uint8_t *)params[0] + g_args_bytes);
    g_launches.push_back(l);
    return hipSuccess;
}
