// Stands in for the CUDA runtime calls that launchers make, on host memory: 148 SMs, kernels of as many registers as the test says, tensor maps that are accepted.
// Remembers the launches, with the kernels' names.  Preloaded in front of the real runtime.
#include <dlfcn.h>
#include <stdint.h>
#include <string.h>

#include <map>
#include <string>
#include <vector>

#include <cuda_runtime_api.h>

namespace {
std::map<const void*, std::string>& names() {
  static std::map<const void*, std::string> all;
  return all;
}
std::vector<std::string>& launches() {
  static std::vector<std::string> all;
  return all;
}
int g_registers = 255;
int encode(void*, int, unsigned, void*, const uint64_t*, const uint64_t*, const unsigned*, const unsigned*, int, int, int, int) { return 0; }
}  // namespace

extern "C" {
void fake_registers(int n) { g_registers = n; }
int fake_launches() { return (int)launches().size(); }
const char* fake_name(int i) { return launches()[i].c_str(); }
void fake_clear() { launches().clear(); }

void __cudaRegisterFunction(void** handle, const char* host, char* device, const char* name, int limit, uint3* a, uint3* b, dim3* c, dim3* d, int* e) {
  names()[host] = name;
  using Fn = void (*)(void**, const char*, char*, const char*, int, uint3*, uint3*, dim3*, dim3*, int*);
  reinterpret_cast<Fn>(dlsym(RTLD_NEXT, "__cudaRegisterFunction"))(handle, host, device, name, limit, a, b, c, d, e);
}
cudaError_t cudaGetDevice(int* d) { return *d = 0, cudaSuccess; }
cudaError_t cudaDeviceGetAttribute(int* v, cudaDeviceAttr, int) { return *v = 148, cudaSuccess; }
cudaError_t cudaFuncSetAttribute(const void*, cudaFuncAttribute, int) { return cudaSuccess; }
cudaError_t cudaFuncGetAttributes(cudaFuncAttributes* a, const void*) {
  memset(a, 0, sizeof(*a));
  a->numRegs = g_registers;
  return cudaSuccess;
}
cudaError_t cudaOccupancyMaxActiveBlocksPerMultiprocessorWithFlags(int* n, const void*, int, size_t, unsigned) { return *n = 2, cudaSuccess; }
cudaError_t cudaGetDriverEntryPoint(const char*, void** f, unsigned long long, cudaDriverEntryPointQueryResult* q) {
  *f = reinterpret_cast<void*>(&encode);
  if (q) *q = cudaDriverEntryPointSuccess;
  return cudaSuccess;
}
cudaError_t cudaMemsetAsync(void*, int, size_t, cudaStream_t) { return cudaSuccess; }
cudaError_t cudaMemset2DAsync(void*, size_t, int, size_t, size_t, cudaStream_t) { return cudaSuccess; }
cudaError_t cudaGetLastError() { return cudaSuccess; }
cudaError_t cudaLaunchKernel(const void* f, dim3, dim3, void**, size_t, cudaStream_t) { return launches().push_back(names()[f]), cudaSuccess; }
cudaError_t cudaLaunchKernelExC(const cudaLaunchConfig_t*, const void* f, void**) { return launches().push_back(names()[f]), cudaSuccess; }
}
