// A HIP runtime without a GPU, for tests of what the library's host code asks
// of it: launches are written down, not run, and allocations are address space
// alone.  Loaded before the library (RTLD_GLOBAL), it takes the runtime's place.
#include <hip/hip_runtime_api.h>
#include <sys/mman.h>
#include <unistd.h>

#include <cstring>
#include <map>
#include <mutex>
#include <string>

namespace {

std::mutex mu;
std::map<const void *, std::string> names;
std::map<void *, size_t> memory;
std::string written;
size_t most = SIZE_MAX, pinned_most = SIZE_MAX;   // larger allocations fail
bool capturing = false;
thread_local hipError_t last = hipSuccess;        // as the runtime keeps it, until it is read
struct Config {
    dim3 grid, block;
    size_t shared;
    hipStream_t stream;
};
thread_local Config config;

hipError_t failed(hipError_t e) {
    last = e;
    return e;
}
hipError_t allocate(void **p, size_t bytes, size_t limit) {
    if (bytes > limit) return failed(hipErrorOutOfMemory);
    *p = mmap(nullptr, bytes + 4096, PROT_READ | PROT_WRITE, MAP_PRIVATE | MAP_ANONYMOUS | MAP_NORESERVE, -1, 0);
    if (*p == MAP_FAILED) return failed(hipErrorOutOfMemory);
    std::lock_guard<std::mutex> lock(mu);
    memory[*p] = bytes;
    return hipSuccess;
}
hipError_t release(void *p) {
    std::lock_guard<std::mutex> lock(mu);
    auto it = memory.find(p);
    if (it != memory.end()) {
        munmap(p, it->second + 4096);
        memory.erase(it);
    }
    return hipSuccess;
}

}  // namespace

extern "C" {

// -- for the test ---------------------------------------------------------
void stand_in_limits(size_t device, size_t pinned) { most = device, pinned_most = pinned; }
void stand_in_capturing(int on) { capturing = on; }
size_t stand_in_bytes() {                          // allocated on the device now
    std::lock_guard<std::mutex> lock(mu);
    size_t n = 0;
    for (auto &m : memory) n += m.second;
    return n;
}
// The launches since the last call: "<stream> <grid x> <grid y> <block x> <mangled name>" each.
size_t stand_in_launches(char *to, size_t room) {
    std::lock_guard<std::mutex> lock(mu);
    const size_t n = written.size();
    if (n < room) {
        std::memcpy(to, written.c_str(), n + 1);
        written.clear();
    }
    return n;
}

// -- the runtime ----------------------------------------------------------
void **__hipRegisterFatBinary(const void *) {
    static void *module;
    return &module;
}
void __hipUnregisterFatBinary(void **) {}
void __hipRegisterFunction(void **, const void *f, char *, const char *name, unsigned, void *, void *, void *, void *,
                           int *) {
    names[f] = name;
}
void __hipRegisterVar(void **, void *, char *, char *, int, size_t, int, int) {}
hipError_t __hipPushCallConfiguration(dim3 grid, dim3 block, size_t shared, hipStream_t s) {
    config = {grid, block, shared, s};
    return hipSuccess;
}
hipError_t __hipPopCallConfiguration(dim3 *grid, dim3 *block, size_t *shared, hipStream_t *s) {
    *grid = config.grid, *block = config.block, *shared = config.shared, *s = config.stream;
    return hipSuccess;
}
hipError_t hipLaunchKernel(const void *f, dim3 grid, dim3 block, void **, size_t, hipStream_t s) {
    if (!grid.x || !grid.y || !grid.z || (uint64_t)grid.x * block.x > UINT32_MAX || grid.y > 65535 || grid.z > 65535)
        return failed(hipErrorInvalidConfiguration);
    {
        std::lock_guard<std::mutex> lock(mu);
        written += std::to_string((uintptr_t)s) + ' ' + std::to_string(grid.x) + ' ' + std::to_string(grid.y) + ' ' +
                   std::to_string(block.x) + ' ' + names[f] + '\n';
    }
    usleep(200);   // another thread's turn
    return hipSuccess;
}
hipError_t hipGetLastError() {
    const hipError_t e = last;
    last = hipSuccess;
    return e;
}
const char *hipGetErrorString(hipError_t e) { return e == hipErrorOutOfMemory ? "out of memory" : "stand-in error"; }
hipError_t hipGetDeviceCount(int *n) {
    *n = 1;
    return hipSuccess;
}
hipError_t hipGetDevice(int *d) {
    *d = 0;
    return hipSuccess;
}
hipError_t hipSetDevice(int) { return hipSuccess; }
hipError_t hipGetDevicePropertiesR0600(hipDeviceProp_tR0600 *p, int) {
    std::memset(p, 0, sizeof *p);
    std::strcpy(p->gcnArchName, "gfx950");
    p->multiProcessorCount = 256;
    return hipSuccess;
}
hipError_t hipGetSymbolAddress(void **p, const void *) {
    static char scratch[64];
    *p = scratch;
    return hipSuccess;
}
hipError_t hipStreamCreateWithFlags(hipStream_t *s, unsigned) {
    *s = (hipStream_t)0x1000;
    return hipSuccess;
}
hipError_t hipStreamDestroy(hipStream_t) { return hipSuccess; }
hipError_t hipStreamSynchronize(hipStream_t) { return hipSuccess; }
hipError_t hipDeviceSynchronize() { return hipSuccess; }
hipError_t hipStreamIsCapturing(hipStream_t, hipStreamCaptureStatus *s) {
    *s = capturing ? hipStreamCaptureStatusActive : hipStreamCaptureStatusNone;
    return hipSuccess;
}
hipError_t hipMalloc(void **p, size_t bytes) { return allocate(p, bytes, most); }
hipError_t hipFree(void *p) { return release(p); }
hipError_t hipHostMalloc(void **p, size_t bytes, unsigned) { return allocate(p, bytes, pinned_most); }
hipError_t hipHostFree(void *p) { return release(p); }
hipError_t hipHostGetDevicePointer(void **d, void *p, unsigned) {
    *d = p;
    return hipSuccess;
}
hipError_t hipMemcpy(void *to, const void *from, size_t n, hipMemcpyKind) {
    std::memcpy(to, from, n);
    return hipSuccess;
}
hipError_t hipMemcpyAsync(void *to, const void *from, size_t n, hipMemcpyKind, hipStream_t) {
    std::memcpy(to, from, n);
    return hipSuccess;
}
hipError_t hipMemcpy2DAsync(void *to, size_t tp, const void *from, size_t fp, size_t width, size_t rows, hipMemcpyKind,
                            hipStream_t) {
    for (size_t r = 0; r < rows; ++r) std::memcpy((char *)to + r * tp, (const char *)from + r * fp, width);
    return hipSuccess;
}
hipError_t hipMemsetAsync(void *p, int v, size_t n, hipStream_t) {
    std::memset(p, v, n);
    return hipSuccess;
}
hipError_t hipMemset(void *p, int v, size_t n) {
    std::memset(p, v, n);
    return hipSuccess;
}

}  // extern "C"
