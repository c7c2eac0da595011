// A HIP runtime that does nothing but keep a log, for tests of the host side of
// libaigpu.so where no GPU is: one gfx950 device of 256 compute units, memory
// that is only addresses, launches that are only names. Loaded ahead of the
// backend with global symbols, it takes the place of the runtime's.
#include <hip/hip_runtime.h>

#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <map>
#include <mutex>
#include <string>

namespace {
std::recursive_mutex gate;
std::string entries;                    // one call a line
std::map<std::string, int> failing;     // calls of a name still to fail
std::map<const void*, std::string> kernels;
uintptr_t next = uintptr_t(1) << 32;
dim3 grid, block;
hipStream_t stream;

hipError_t called(const char* name, const std::string& what = "") {
    std::lock_guard<std::recursive_mutex> lock(gate);
    const bool fails = failing[name] > 0 && failing[name]--;
    entries += std::string(name) + (what.empty() ? "" : " " + what) + (fails ? " failed" : "") + "\n";
    return fails ? hipErrorStreamCaptureUnsupported : hipSuccess;
}

std::string text(const void* p) { return std::to_string(reinterpret_cast<uintptr_t>(p)); }
} // namespace

#define FAKE extern "C" __attribute__((visibility("default")))

FAKE const char* fake_log() {
    static std::string out;
    std::lock_guard<std::recursive_mutex> lock(gate);
    out = entries;
    entries.clear();
    return out.c_str();
}
FAKE void fake_fail(const char* name, int times) { failing[name] = times; }

FAKE void** __hipRegisterFatBinary(const void*) { static void* module; return &module; }
FAKE void __hipUnregisterFatBinary(void**) {}
FAKE void __hipRegisterFunction(void**, const void* host, char*, const char* device, unsigned, void*, void*, dim3*,
                                dim3*, int*) { kernels[host] = device; }
FAKE void __hipRegisterVar(void**, void*, char*, char*, int, size_t, int, int) {}
FAKE hipError_t __hipPushCallConfiguration(dim3 g, dim3 b, size_t, hipStream_t s) {
    grid = g, block = b, stream = s;
    return hipSuccess;
}
FAKE hipError_t __hipPopCallConfiguration(dim3* g, dim3* b, size_t* lds, hipStream_t* s) {
    *g = grid, *b = block, *lds = 0, *s = stream;
    return hipSuccess;
}
FAKE hipError_t hipLaunchKernel(const void* host, dim3 g, dim3, void**, size_t, hipStream_t s) {
    return called("launch", text(s) + " " + std::to_string(g.x) + " " + kernels[host]);
}

FAKE hipError_t hipGetDeviceCount(int* n) { *n = 1; return hipSuccess; }
FAKE hipError_t hipGetDevice(int* d) { *d = 0; return hipSuccess; }
FAKE hipError_t hipSetDevice(int) { return hipSuccess; }
FAKE hipError_t hipGetDevicePropertiesR0600(hipDeviceProp_tR0600* p, int) {
    std::memset(p, 0, sizeof *p);
    std::strcpy(p->name, "none");
    std::strcpy(p->gcnArchName, "gfx950");
    p->multiProcessorCount = 256;
    return hipSuccess;
}
FAKE hipError_t hipGetLastError() { return hipSuccess; }
FAKE const char* hipGetErrorString(hipError_t) { return "refused"; }
FAKE hipError_t hipDeviceSynchronize() { return called("hipDeviceSynchronize"); }
FAKE hipError_t hipHostMalloc(void** p, size_t n, unsigned) { *p = std::calloc(1, n); return hipSuccess; }
FAKE hipError_t hipHostGetDevicePointer(void** d, void* h, unsigned) { *d = h; return hipSuccess; }
FAKE hipError_t hipMalloc(void** p, size_t n) {
    std::lock_guard<std::recursive_mutex> lock(gate);
    *p = reinterpret_cast<void*>(next);
    next += (n + 4095) & ~size_t(4095);
    return called("hipMalloc", std::to_string(n) + " at " + text(*p));
}
FAKE hipError_t hipFree(void* p) { return called("hipFree", text(p)); }
FAKE hipError_t hipMemset(void* p, int, size_t n) { return called("hipMemset", text(p) + " " + std::to_string(n)); }
FAKE hipError_t hipStreamIsCapturing(hipStream_t, hipStreamCaptureStatus* s) {
    *s = hipStreamCaptureStatusNone;
    return hipSuccess;
}
FAKE hipError_t hipEventCreate(hipEvent_t* e) { *e = nullptr; return hipSuccess; }
FAKE hipError_t hipEventCreateWithFlags(hipEvent_t* e, unsigned) { *e = nullptr; return hipSuccess; }
FAKE hipError_t hipEventRecord(hipEvent_t, hipStream_t s) { return called("record", text(s)); }
FAKE hipError_t hipEventSynchronize(hipEvent_t) { return called("finish"); }
FAKE hipError_t hipStreamSynchronize(hipStream_t s) { return called("finish", text(s)); }
FAKE hipError_t hipStreamWaitEvent(hipStream_t s, hipEvent_t, unsigned) { return called("wait", text(s)); }
