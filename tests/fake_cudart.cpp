// A CUDA runtime without a GPU, for tests of the host side: it is linked with the library's own objects in the real
// runtime's place. It keeps what the real one keeps for each device (the shared memory that a kernel was granted),
// refuses what the real one refuses (empty grids, more shared memory than granted), and counts.
#include <cstring>
#include <map>
#include <utility>
#include <vector>

#include <driver_types.h>
#include <vector_types.h>

namespace {

constexpr size_t kDefaultSmem = 48 * 1024;
constexpr int kInvalidValue = 1, kInvalidConfiguration = 9, kNotSupported = 801;

struct Launch {
  int device, grid[3], smem, result;
};
int device = 0, devices = 4, to_fail = 0, attribute_calls = 0, sms[64];
std::map<std::pair<int, const void*>, size_t> granted;
std::vector<Launch> launches;

int launch(const void* kernel, const dim3& grid, size_t smem) {
  int result = 0;
  const auto it = granted.find({device, kernel});
  if (grid.x == 0 || grid.y == 0 || grid.z == 0) result = kInvalidConfiguration;
  else if (smem > (it == granted.end() ? kDefaultSmem : it->second)) result = kInvalidValue;
  launches.push_back({device, {(int)grid.x, (int)grid.y, (int)grid.z}, (int)smem, result});
  return result;
}

int encode_nothing() { return 0; }

}  // namespace

extern "C" {

// ---- the test's side ----
void fake_reset(int sm_count) {  // but for what kernels were granted, which lasts as long as the process
  device = to_fail = attribute_calls = 0;
  for (int& n : sms) n = sm_count;
  launches.clear();
}
void fake_device(int d) { device = d; }
void fake_sms(int d, int n) { sms[d] = n; }
void fake_fail(int calls) { to_fail = calls; }  // the next settings of an attribute fail
int fake_attribute_calls() { return attribute_calls; }
int fake_launches() { return (int)launches.size(); }
void fake_launch(int i, int* out) { std::memcpy(out, &launches[i], sizeof(Launch)); }

// ---- the runtime's ----
int cudaGetDevice(int* d) {
  *d = device;
  return 0;
}
int cudaGetDeviceCount(int* n) {
  *n = devices;
  return 0;
}
int cudaDeviceGetAttribute(int* v, int, int d) {
  *v = sms[d];
  return 0;
}
int cudaFuncSetAttribute(const void* f, int attribute, int value) {
  ++attribute_calls;
  if (to_fail > 0) {
    --to_fail;
    return 2;
  }
  if (attribute == 8) granted[{device, f}] = (size_t)value;  // the largest dynamic shared memory
  return 0;
}
int cudaLaunchKernelExC(const cudaLaunchConfig_t* c, const void* f, void**) { return launch(f, c->gridDim, c->dynamicSmemBytes); }
int cudaLaunchKernel(const void* f, dim3 grid, dim3, void**, size_t smem, cudaStream_t) { return launch(f, grid, smem); }
int cudaGetDriverEntryPoint(const char*, void** f, unsigned long long, int* found) {
  *f = reinterpret_cast<void*>(&encode_nothing);
  if (found != nullptr) *found = 0;
  return 0;
}
int cudaOccupancyMaxActiveClusters(int* n, const void*, const cudaLaunchConfig_t*) {
  *n = 64;
  return 0;
}
int cudaOccupancyMaxActiveBlocksPerMultiprocessorWithFlags(int* n, const void*, int, size_t, unsigned) {
  *n = 1;
  return 0;
}
int cudaGetLastError() { return 0; }
const char* cudaGetErrorString(int) { return "an error of the fake runtime"; }
int cudaDeviceSynchronize() { return 0; }
int cudaFree(void*) { return 0; }
int cudaMalloc(void**, size_t) { return kNotSupported; }
int cudaMemset(void*, int, size_t) { return kNotSupported; }
int cudaGetSymbolAddress(void**, const void*) { return kNotSupported; }
int cudaIpcCloseMemHandle(void*) { return kNotSupported; }
int cudaIpcGetMemHandle(void*, void*) { return kNotSupported; }
int cudaIpcOpenMemHandle(void**, cudaIpcMemHandle_t, unsigned) { return kNotSupported; }
unsigned __cudaPopCallConfiguration(dim3*, dim3*, size_t*, void*) { return 0; }
void** __cudaRegisterFatBinary(void*) {
  static void* handle;
  return &handle;
}
void __cudaRegisterFatBinaryEnd(void**) {}
void __cudaUnregisterFatBinary(void**) {}
void __cudaRegisterFunction(void**, const char*, char*, const char*, int, void*, void*, void*, void*, int*) {}
void __cudaRegisterVar(void**, char*, char*, const char*, int, size_t, int, int) {}
}
