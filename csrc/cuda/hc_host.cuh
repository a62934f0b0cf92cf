// Host-side pieces that the launchers share: tensor maps, grid sizes, launches with programmatic serialisation.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>
#include <string.h>

#include "hc_kernels.cuh"

namespace hc {

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

inline EncodeTiledFn encode_tiled_fn() {
  static EncodeTiledFn fn = [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      f = nullptr;
    return reinterpret_cast<EncodeTiledFn>(f);
  }();
  return fn;
}

// A tensor map.  The call needs the device's context to be current, which it is not in a thread that has called nothing of the runtime yet that needs one
// (torch's autograd thread, with its memory from the cache): made current then, and tried again.
template <typename... Args>
bool encode_tiled(Args... args) {
  EncodeTiledFn fn = encode_tiled_fn();
  if (!fn) return false;
  CUresult r = fn(args...);
  if (r == CUDA_ERROR_INVALID_CONTEXT) {
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || cudaSetDevice(dev) != cudaSuccess) return false;
    r = fn(args...);
  }
  return r == CUDA_SUCCESS;
}

// 2-D view {32, rows} of a 4-byte-element array, box {32, box_rows}, 128-byte swizzle
inline bool make_rows_map(CUtensorMap* map, const void* base, uint64_t rows, int box_rows) {
  if (rows == 0 || (reinterpret_cast<uintptr_t>(base) & 15u)) return false;
  cuuint64_t dims[2] = {(cuuint64_t)kBlock, (cuuint64_t)rows};
  cuuint64_t strides[1] = {(cuuint64_t)kBlock * 4};
  cuuint32_t box[2] = {(cuuint32_t)kBlock, (cuuint32_t)box_rows};
  cuuint32_t estr[2] = {1, 1};
  return encode_tiled(map, CU_TENSOR_MAP_DATA_TYPE_UINT32, 2, const_cast<void*>(base), dims, strides, box, estr,
                      CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                      CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
}

struct DeviceInfo {
  int sms = 0;
  bool ready = false;
};
inline DeviceInfo& device_info() {
  static thread_local DeviceInfo info[64];
  int dev = 0;
  cudaGetDevice(&dev);
  DeviceInfo& d = info[dev & 63];
  if (!d.ready) {
    cudaDeviceGetAttribute(&d.sms, cudaDevAttrMultiProcessorCount, dev);
    d.ready = true;
  }
  return d;
}

// A launch of clusters of `size` CTAs.  beside: the kernel may begin while the one before it in the stream runs, once all of that one's CTAs have allowed it or ended (griddepcontrol.launch_dependents),
// and waits for the end of that one where it needs its results (griddepcontrol.wait); some thread of each CTA does, so that it does not end first.
template <typename... Params, typename... Args>
cudaError_t launch_with(void (*kernel)(Params...), int64_t ctas, int size, int threads, int smem, cudaStream_t stream, bool beside, const Args&... args) {
  cudaLaunchConfig_t cfg;
  memset(&cfg, 0, sizeof(cfg));
  cfg.gridDim = dim3((unsigned)ctas);
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = (size_t)smem;
  cfg.stream = stream;
  cudaLaunchAttribute attrs[2];
  memset(attrs, 0, sizeof(attrs));
  cfg.attrs = attrs;
  if (size > 1) {
    attrs[0].id = cudaLaunchAttributeClusterDimension;
    attrs[0].val.clusterDim.x = (unsigned)size;
    attrs[0].val.clusterDim.y = attrs[0].val.clusterDim.z = 1;
    cfg.numAttrs = 1;
  }
  if (beside) {
    attrs[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attrs[cfg.numAttrs].val.programmaticStreamSerializationAllowed = 1;
    ++cfg.numAttrs;
  }
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

template <typename K>
cudaError_t set_smem(K kernel, int bytes) {
  return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
}

// Launch with programmatic stream serialisation: the kernel may start while the one before it drains.  The steps of a
// collective order their data by arrival flags; every other kernel launched this way executes griddepcontrol.wait
// before it touches global memory, and only its launch and set-up overlap (a 4 KB compress back to back: 6.1 us a call
// without).
template <typename... Params, typename... Args>
cudaError_t launch_overlapped(void (*kernel)(Params...), int grid, int block, int smem, cudaStream_t stream,
                              const Args&... args) {
  cudaLaunchConfig_t cfg;
  memset(&cfg, 0, sizeof(cfg));
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3((unsigned)block);
  cfg.dynamicSmemBytes = (size_t)smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr;
  memset(&attr, 0, sizeof(attr));
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

// The same, asked once for each device: `done` is the kernel's own, one bit a device.  All sizes up to the most that a block may
// have are allowed then.  `registers`: what the kernel counts on having a thread; one that was built with fewer is refused.
template <typename K>
cudaError_t allow_smem(K kernel, int most, unsigned long long* done, int registers = 0) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const unsigned long long bit = 1ull << (dev & 63);
  if (__atomic_load_n(done, __ATOMIC_ACQUIRE) & bit) return cudaSuccess;
  if (registers > 0) {
    cudaFuncAttributes a;
    e = cudaFuncGetAttributes(&a, kernel);
    if (e != cudaSuccess) return e;
    if ((a.numRegs + 7) / 8 * 8 < registers) return cudaErrorInvalidConfiguration;
  }
  e = set_smem(kernel, most);
  if (e == cudaSuccess) __atomic_fetch_or(done, bit, __ATOMIC_RELEASE);
  return e;
}

// CTAs of `kernel` that one GPU holds at the same time, asked of the runtime once per device.  The
// kernels are written for a grid that is resident as a whole (CTA i owns tile i, and every look-back
// waits for tiles held by other CTAs of the grid), so the grid is cut to this number, never assumed.
template <typename K>
int resident_ctas(K kernel, int threads, int smem, int* cache) {
  int dev = 0;
  cudaGetDevice(&dev);
  int& c = cache[dev & 63];
  if (c == 0) {
    if (set_smem(kernel, smem) != cudaSuccess) return 0;
    int per_sm = 0;
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kernel, threads, (size_t)smem) != cudaSuccess) return 0;
    c = per_sm * device_info().sms;
  }
  return c;
}

}  // namespace hc
