// Two devices of host memory behind the few HIP runtime calls that a context and
// its dense tensors make, so that their lifetimes can be followed without a GPU.
// Loaded before libmoldq.so with global symbols, it is what the library finds.
#include <hip/hip_runtime_api.h>

#include <cstdlib>
#include <cstring>
#include <set>

namespace {
int current = 0, bad_devices = 0, bad_frees = 0;
std::set<void *> live;
char symbol[256];
}  // namespace

extern "C" {
int host_hip_bad_devices() { return bad_devices; }
int host_hip_bad_frees() { return bad_frees; }
int host_hip_live() { return (int)live.size(); }

hipError_t hipGetDeviceCount(int *n) { return *n = 2, hipSuccess; }
hipError_t hipGetDevice(int *d) { return *d = current, hipSuccess; }
hipError_t hipSetDevice(int d) {
  if (d < 0 || d > 1) return ++bad_devices, hipErrorInvalidDevice;
  return current = d, hipSuccess;
}
hipError_t hipGetDeviceProperties(hipDeviceProp_t *p, int) {  // by its versioned name
  memset(p, 0, sizeof *p);
  strcpy(p->gcnArchName, "gfx950");
  p->multiProcessorCount = 256;
  return hipSuccess;
}
hipError_t hipGetSymbolAddress(void **p, const void *) { return *p = symbol, hipSuccess; }
hipError_t hipMalloc(void **p, size_t n) { return *p = malloc(n), live.insert(*p), hipSuccess; }
hipError_t hipFree(void *p) {
  if (p && !live.erase(p)) return ++bad_frees, hipErrorInvalidValue;
  return free(p), hipSuccess;
}
hipError_t hipMemcpyAsync(void *to, const void *from, size_t n, hipMemcpyKind, hipStream_t) {
  return memcpy(to, from, n), hipSuccess;
}
hipError_t hipDeviceSynchronize() { return hipSuccess; }
hipError_t hipStreamIsCapturing(hipStream_t, hipStreamCaptureStatus *s) { return *s = hipStreamCaptureStatusNone, hipSuccess; }
}
