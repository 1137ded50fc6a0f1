// A stand-in for the HIP runtime on a machine without a GPU, for tests of what the library does on the host: device memory is host memory, copies copy,
// kernels do nothing.  Allocations (hipMalloc and operator new) and copies can be told to fail; launches are counted by name, with their first argument kept.
#include <cstdlib>
#include <cstring>
#include <map>
#include <new>
#include <string>
#include <vector>

namespace {
struct Dim3 { unsigned x, y, z; };
struct Launch { std::string name; char arg[512]; };
std::map<const void*, std::string>& names() { static std::map<const void*, std::string> m; return m; }
std::vector<Launch>& launches() { static std::vector<Launch> v; return v; }
std::map<void*, size_t>& blocks() { static std::map<void*, size_t> m; return m; }
std::vector<size_t>& sizes() { static std::vector<size_t> v; return v; }
Dim3 grid, block;
size_t shared;
void* stream;
long fail_malloc = -1, fail_new = -1, fail_copy = -1;   // how many succeed before one fails; -1: all do
int capturing = 0, last_error = 0;
bool due(long& n) { return n >= 0 && n-- == 0; }
int handle;
std::map<const void*, std::vector<char>>& variables() { static std::map<const void*, std::vector<char>> m; return m; }
}  // namespace

void* operator new(size_t n) {
    if (due(fail_new)) throw std::bad_alloc();
    void* p = std::malloc(n ? n : 1);
    if (!p) throw std::bad_alloc();
    return p;
}
void operator delete(void* p) noexcept { std::free(p); }
void operator delete(void* p, size_t) noexcept { std::free(p); }

extern "C" {
// what the tests call
void hostrt_fail_malloc(long after) { fail_malloc = after; }
void hostrt_fail_new(long after) { fail_new = after; }
void hostrt_fail_copy(long after) { fail_copy = after; }
void hostrt_forget() { launches().clear(); sizes().clear(); }
long hostrt_launches(const char* part) {
    long n = 0;
    for (const Launch& l : launches()) n += l.name.find(part) != std::string::npos;
    return n;
}
int hostrt_last(const char* part, void* out, size_t n) {
    for (size_t i = launches().size(); i-- > 0;)
        if (launches()[i].name.find(part) != std::string::npos) {
            std::memcpy(out, launches()[i].arg, n < sizeof(Launch::arg) ? n : sizeof(Launch::arg));
            return 1;
        }
    return 0;
}
long hostrt_sizes(size_t* out, long cap) {
    long n = 0;
    for (size_t s : sizes())
        if (n < cap) out[n++] = s;
    return n;
}
size_t hostrt_held() {
    size_t n = 0;
    for (const auto& b : blocks()) n += b.second;
    return n;
}

// the runtime
void** __hipRegisterFatBinary(const void*) { static void* h; return &h; }
void __hipUnregisterFatBinary(void**) {}
void __hipRegisterFunction(void**, const void* f, char*, const char* name, unsigned, void*, void*, void*, void*, int*) { names()[f] = name; }
void __hipRegisterVar(void**, void* var, char*, char*, int, size_t size, int, int) { variables()[var].resize(size); }
int __hipPushCallConfiguration(Dim3 g, Dim3 b, size_t sh, void* st) { grid = g; block = b; shared = sh; stream = st; return 0; }
int __hipPopCallConfiguration(Dim3* g, Dim3* b, size_t* sh, void** st) { *g = grid; *b = block; *sh = shared; *st = stream; return 0; }
int hipLaunchKernel(const void* f, Dim3, Dim3, void** args, size_t, void*) {
    Launch l;
    l.name = names()[f];
    if (args && args[0]) std::memcpy(l.arg, args[0], sizeof(l.arg));
    launches().push_back(l);
    return 0;
}
int hipMalloc(void** p, size_t n) {
    *p = nullptr;
    if (due(fail_malloc)) return last_error = 2;
    sizes().push_back(n);
    *p = std::calloc(n ? n : 1, 1);
    if (!*p) return last_error = 2;
    blocks()[*p] = n;
    return 0;
}
int hipFree(void* p) {
    if (p && !blocks().erase(p)) return 1;
    std::free(p);
    return 0;
}
int hipMemcpy(void* d, const void* s, size_t n, int) {
    if (due(fail_copy)) return last_error = 1;
    std::memmove(d, s, n);
    return 0;
}
int hipMemcpyAsync(void* d, const void* s, size_t n, int kind, void*) { return hipMemcpy(d, s, n, kind); }
int hipMemset(void* d, int v, size_t n) { std::memset(d, v, n); return 0; }
int hipMemsetAsync(void* d, int v, size_t n, void*) { std::memset(d, v, n); return 0; }
int hipMemsetD32Async(void* d, int v, size_t n, void*) { for (size_t i = 0; i < n; ++i) static_cast<int*>(d)[i] = v; return 0; }
int hipGetSymbolAddress(void** p, const void* var) { *p = variables()[var].data(); return 0; }
int hipPointerGetAttributes(void*, const void*) { return 1; }
int hipGetDevice(int* d) { *d = 0; return 0; }
int hipSetDevice(int d) { return d == 0 ? 0 : 101; }
int hipGetDeviceCount(int* n) { *n = 1; return 0; }
int hipDeviceSynchronize() { return 0; }
int hipFuncSetAttribute(const void*, int, int) { return 0; }
int hipGetLastError() { const int e = last_error; last_error = 0; return e; }
const char* hipGetErrorString(int e) { return e == 2 ? "out of memory" : e ? "error" : "no error"; }
int hipStreamCreateWithFlags(void** s, unsigned) { *s = &handle; return 0; }
int hipStreamDestroy(void*) { return 0; }
int hipStreamSynchronize(void*) { return 0; }
int hipStreamBeginCapture(void*, int) { capturing = 1; return 0; }
int hipStreamEndCapture(void*, void** g) { capturing = 0; *g = &handle; return 0; }
int hipGraphInstantiate(void** e, void*, void*, char*, size_t) { *e = &handle; return 0; }
int hipGraphLaunch(void*, void*) { return 0; }
int hipGraphDestroy(void*) { return 0; }
int hipGraphExecDestroy(void*) { return 0; }
int hipEventCreate(void** e) { *e = &handle; return 0; }
int hipEventDestroy(void*) { return 0; }
int hipEventRecord(void*, void*) { return 0; }
int hipEventSynchronize(void*) { return 0; }
int hipEventElapsedTime(float* ms, void*, void*) { *ms = 0.f; return 0; }
}
