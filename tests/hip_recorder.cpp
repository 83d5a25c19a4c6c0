// A stand-in for the HIP runtime, for tests of the library's host side on a
// machine without a GPU: device memory is host memory (committed when touched),
// kernels are counted and not run, allocations can be made to fail.  Loaded
// with RTLD_GLOBAL before libqnn_hip.so, whose HIP symbols then resolve here.
#include <sys/mman.h>

#include <cstdint>
#include <cstdlib>
#include <cstring>
#include <map>
#include <string>
#include <vector>

namespace {
struct Dim3 {
  uint32_t x, y, z;
};
constexpr int kOutOfMemory = 2, kInvalidConfiguration = 9;
int last_error = 0;
std::map<void *, size_t> live;
std::map<const void *, std::string> names;
std::string launched;  // names of the kernels launched, a line each
uint64_t allocations = 0, live_bytes = 0, largest = 0;
int64_t fail_at = -1;  // allocations until one fails (0: the next)
struct Config {
  Dim3 grid, block;
  size_t shared;
  void *stream;
};
std::vector<Config> configs;
void *map_bytes(size_t n) {
  void *p = mmap(nullptr, n, PROT_READ | PROT_WRITE, MAP_PRIVATE | MAP_ANONYMOUS | MAP_NORESERVE, -1, 0);
  return p == MAP_FAILED ? nullptr : p;
}
}  // namespace

extern "C" {
// ---- what a test asks and sets
uint64_t rec_allocations() { return allocations; }
uint64_t rec_live_bytes() { return live_bytes; }
uint64_t rec_largest() { return largest; }
void rec_forget_largest() { largest = 0; }
void rec_fail_at(int64_t n) { fail_at = n; }
const char *rec_launched() { return launched.c_str(); }
void rec_forget_launched() { launched.clear(); }

// ---- the runtime
int hipGetLastError() {
  const int e = last_error;
  last_error = 0;
  return e;
}
const char *hipGetErrorString(int e) { 
  return e == kOutOfMemory ? "out of memory" : e == kInvalidConfiguration ? "invalid configuration" : "no error";
}
int hipGetDeviceCount(int *n) { return *n = 1, 0; }
int hipSetDevice(int) { return 0; }
int hipDeviceGetAttribute(int *v, int, int) { return *v = 256, 0; }
int hipMemGetInfo(size_t *f, size_t *t) { return *f = *t = size_t(288) << 30, 0; }
int hipMalloc(void **p, size_t n) {
  if (fail_at >= 0 && fail_at-- == 0) return last_error = kOutOfMemory;
  if (!(*p = map_bytes(n))) return last_error = kOutOfMemory;
  live[*p] = n;
  live_bytes += n;
  ++allocations;
  if (n > largest) largest = n;
  return 0;
}
int hipFree(void *p) {
  const auto it = live.find(p);
  if (it == live.end()) return 0;
  munmap(p, it->second);
  live_bytes -= it->second;
  live.erase(it);
  return 0;
}
int hipHostMalloc(void **p, size_t n, unsigned) { return (*p = map_bytes(n)) ? 0 : (last_error = kOutOfMemory); }
int hipHostFree(void *) { return 0; }
int hipMemcpyAsync(void *d, const void *s, size_t n, int, void *) { return std::memcpy(d, s, n), 0; }
int hipMemsetAsync(void *d, int v, size_t n, void *) { return std::memset(d, v, n), 0; }
int hipStreamCreateWithFlags(void **s, unsigned) { return *s = std::malloc(1), 0; }
int hipStreamDestroy(void *s) { return std::free(s), 0; }
int hipStreamSynchronize(void *) { return 0; }
int hipStreamWaitEvent(void *, void *, unsigned) { return 0; }
int hipStreamBeginCapture(void *, int) { return 0; }
int hipStreamEndCapture(void *, void **g) { return *g = std::malloc(1), 0; }
int hipGraphInstantiate(void **e, void *, void **, char *, size_t) { return *e = std::malloc(1), 0; }
int hipGraphLaunch(void *, void *) { return 0; }
int hipGraphDestroy(void *g) { return std::free(g), 0; }
int hipGraphExecDestroy(void *g) { return std::free(g), 0; }
int hipEventCreate(void **e) { return *e = std::malloc(1), 0; }
int hipEventCreateWithFlags(void **e, unsigned) { return *e = std::malloc(1), 0; }
int hipEventDestroy(void *e) { return std::free(e), 0; }
int hipEventRecord(void *, void *) { return 0; }
int hipEventSynchronize(void *) { return 0; }
int hipEventElapsedTime(float *ms, void *, void *) { return *ms = 0, 0; }
int hipFuncSetAttribute(const void *, int, int) { return 0; }
int hipOccupancyMaxActiveBlocksPerMultiprocessor(int *n, const void *, int, size_t) { return *n = 1, 0; }
int hipGetSymbolAddress(void **p, const void *) { return (*p = map_bytes(size_t(64) << 20)) ? 0 : kOutOfMemory; }
int hipLaunchKernel(const void *f, Dim3 grid, Dim3 block, void **, size_t, void *) {
  // Threads along a dimension are counted in 32 bits; y and z take 65535 workgroups.
  if (!grid.x || !grid.y || !grid.z || uint64_t(grid.x) * block.x > 0xffffffffull || grid.y > 65535 || grid.z > 65535)
    return last_error = kInvalidConfiguration;
  launched += names[f] + "\n";
  return 0;
}
int __hipPushCallConfiguration(Dim3 grid, Dim3 block, size_t shared, void *stream) {
  configs.push_back({grid, block, shared, stream});
  return 0;
}
int __hipPopCallConfiguration(Dim3 *grid, Dim3 *block, size_t *shared, void **stream) {
  const Config c = configs.back();
  configs.pop_back();
  *grid = c.grid, *block = c.block, *shared = c.shared, *stream = c.stream;
  return 0;
}
void **__hipRegisterFatBinary(const void *) {
  static void *handle;
  return &handle;
}
void __hipRegisterFunction(void **, const void *host, char *, const char *name, unsigned, void *, void *, void *, void *,
                           int *) {
  names[host] = name;
}
void __hipRegisterVar(void **, void *, char *, char *, int, size_t, int, int) {}
void __hipUnregisterFatBinary(void **) {}
}
