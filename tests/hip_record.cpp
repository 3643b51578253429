// A HIP runtime that runs nothing and records launches: which thread made each, on which stream. Loaded into a process
// ahead of the library under test, whose calls then bind to these, so that what a call enqueues can be checked off the
// GPU. A launch of a numbered thread takes a while, so that threads that may come between two launches of a call do.
#include <chrono>
#include <cstdint>
#include <cstdlib>
#include <map>
#include <mutex>
#include <string>
#include <thread>
#include <vector>

namespace {
struct Grid {
    uint32_t x, y, z;
};
struct Call {
    Grid grid, block;
    size_t shmem;
    void* stream;
};
struct Launch {
    int64_t thread, stream;
    const void* kernel;
    Grid grid;
};
thread_local Call call;
thread_local int64_t number = 0;
std::mutex mu;
std::vector<Launch> launches;
std::map<const void*, std::string>& kernels() {  // (libraries register theirs before main)
    static std::map<const void*, std::string> k;
    return k;
}
std::vector<int64_t> events;  // of memory and streams, in order: kind, address
void note(int64_t kind, void* p) {
    std::lock_guard<std::mutex> lock(mu);
    events.push_back(kind);
    events.push_back((int64_t)p);
}
}  // namespace

extern "C" {
// --- what a test asks for
void record_thread(int64_t n) { number = n; }
void record_clear() {
    std::lock_guard<std::mutex> lock(mu);
    launches.clear();
    events.clear();
}
int64_t record_launches(int64_t* out, int64_t most) {  // pairs of thread and stream
    std::lock_guard<std::mutex> lock(mu);
    for (int64_t i = 0; i < (int64_t)launches.size() && i < most; i++)
        out[2 * i] = launches[i].thread, out[2 * i + 1] = launches[i].stream;
    return (int64_t)launches.size();
}
// the mangled name of launch i's kernel; of kernel i of all that are registered
const char* record_kernel(int64_t i) { return i < (int64_t)launches.size() ? kernels()[launches[i].kernel].c_str() : ""; }
int64_t record_workgroups(int64_t i) {  // of launch i
    const Grid g = i < (int64_t)launches.size() ? launches[i].grid : Grid{0, 0, 0};
    return (int64_t)g.x * g.y * g.z;
}
const char* record_registered(int64_t i) {
    for (const auto& k : kernels())
        if (i-- == 0) return k.second.c_str();
    return "";
}
// pairs: 1 memory given, 2 memory freed, 3 a stream waited for, 4 a stream destroyed
int64_t record_events(int64_t* out, int64_t most) {
    std::lock_guard<std::mutex> lock(mu);
    for (int64_t i = 0; i < (int64_t)events.size() && i < 2 * most; i++) out[i] = events[i];
    return (int64_t)events.size() / 2;
}

// --- the runtime
void** __hipRegisterFatBinary(const void*) {
    static void* none;
    return &none;
}
void __hipUnregisterFatBinary(void**) {}
void __hipRegisterFunction(void**, const void* host, char*, const char* name, unsigned, void*, void*, void*, void*, int*) {
    kernels()[host] = name;
}
void __hipRegisterVar(void**, void*, char*, const char*, int, size_t, int, int) {}
int __hipPushCallConfiguration(Grid grid, Grid block, size_t shmem, void* stream) {
    call = {grid, block, shmem, stream};
    return 0;
}
int __hipPopCallConfiguration(Grid* grid, Grid* block, size_t* shmem, void** stream) {
    *grid = call.grid, *block = call.block, *shmem = call.shmem, *stream = call.stream;
    return 0;
}
int hipLaunchKernel(const void* kernel, Grid grid, Grid, void**, size_t, void* stream) {
    {
        std::lock_guard<std::mutex> lock(mu);
        launches.push_back({number, (int64_t)stream, kernel, grid});
    }
    if (number) std::this_thread::sleep_for(std::chrono::microseconds(100));
    return 0;
}
int hipGetLastError() { return 0; }
int hipGetDevice(int* d) { return *d = 0; }
int hipGetDeviceCount(int* n) { return *n = 1, 0; }
int hipSetDevice(int) { return 0; }
int hipDeviceGetAttribute(int* v, int, int) { return *v = 256, 0; }
int hipOccupancyMaxActiveBlocksPerMultiprocessor(int* n, const void*, int, size_t) { return *n = 2, 0; }
int hipMalloc(void** p, size_t bytes) {
    *p = std::aligned_alloc(256, (bytes + 255) / 256 * 256 + 256);
    note(1, *p);
    return 0;
}
int hipFree(void* p) {
    note(2, p);
    std::free(p);
    return 0;
}
int hipGetSymbolAddress(void** p, const void*) { return *p = (void*)(1 << 20), 0; }
int hipMemcpy(void*, const void*, size_t, int) { return 0; }
int hipMemcpyAsync(void*, const void*, size_t, int, void*) { return 0; }
int hipMemsetAsync(void*, int, size_t, void*) { return 0; }
int hipStreamCreateWithFlags(void** s, unsigned) { return *s = std::malloc(16), 0; }
int hipStreamDestroy(void* s) {
    note(4, s);
    std::free(s);
    return 0;
}
int hipStreamSynchronize(void* s) {
    note(3, s);
    return 0;
}
int hipStreamIsCapturing(void*, int* status) { return *status = 0; }
int hipDeviceSynchronize() { return 0; }
}
