// A stand-in for the HIP runtime calls that libqmm.so's host side makes: one device of 256 CUs whose memory is
// addresses only, and a list of the launches in place of kernels. Loaded before the library (RTLD_GLOBAL) it lets a
// process without a GPU follow a call's checks, workspaces and launches.
#include <hip/hip_runtime_api.h>

#include <cstdint>
#include <cstring>
#include <deque>
#include <string>
#include <vector>

static std::deque<std::string> names;
static std::vector<const std::string*> launched;
static std::deque<std::vector<char>> kept;  // the first argument of each launch
static size_t keep_bytes = 0;
static uintptr_t next_address = (uintptr_t)1 << 44;

extern "C" {
int host_launches() { return (int)launched.size(); }
const char* host_launch(int i) { return launched[i]->c_str(); }
// From here on the first argument of each launch is kept, which has `bytes` bytes in all of them.
void host_keep(size_t bytes) { keep_bytes = bytes; }
const void* host_argument(int i) { return kept[i].data(); }
void host_clear() { launched.clear(), kept.clear(); }

hipError_t hipGetDevice(int* dev) { return *dev = 0, hipSuccess; }
hipError_t hipSetDevice(int dev) { return dev ? hipErrorInvalidDevice : hipSuccess; }
const char* hipGetErrorString(hipError_t e) { return e == hipSuccess ? "no error" : "error"; }
hipError_t hipGetLastError() { return hipSuccess; }
hipError_t hipStreamSynchronize(hipStream_t) { return hipSuccess; }
hipError_t hipModuleUnload(hipModule_t) { return hipSuccess; }
hipError_t hipModuleLoadData(hipModule_t* m, const void*) { return *m = nullptr, hipSuccess; }
hipError_t hipFree(void*) { return hipSuccess; }
hipError_t hipMemcpyAsync(void*, const void*, size_t, hipMemcpyKind, hipStream_t) { return hipSuccess; }

hipError_t hipDeviceGetAttribute(int* v, hipDeviceAttribute_t a, int) {
  *v = a == hipDeviceAttributeMaxSharedMemoryPerBlock ? 160 * 1024 : 256;  // the library asks for this and the CUs
  return hipSuccess;
}

hipError_t hipMalloc(void** p, size_t n) {
  *p = (void*)next_address;
  next_address += (n + 4095) & ~(size_t)4095;
  return hipSuccess;
}

hipError_t hipModuleGetFunction(hipFunction_t* f, hipModule_t, const char* name) {
  names.push_back(name);
  *f = (hipFunction_t)&names.back();
  return hipSuccess;
}

hipError_t hipModuleLaunchKernel(hipFunction_t f, unsigned, unsigned, unsigned, unsigned, unsigned, unsigned, unsigned,
                                 hipStream_t, void** args, void**) {
  kept.emplace_back(keep_bytes);
  if (keep_bytes) memcpy(kept.back().data(), args[0], keep_bytes);
  launched.push_back((const std::string*)f);
  return hipSuccess;
}
}
