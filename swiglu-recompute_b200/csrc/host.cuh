// Host-side helpers shared by the translation units of the C ABI: error
// reporting, the current device, TMA map encoding, argument checks and kernel
// launches. Defined in api.cu unless inline here.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cstdint>

#include "swiglu_b200.h"

namespace swiglu {

// Record the message behind swiglu_b200_last_error_message; return the status.
int fail(int code, const char* fmt, ...);
int cuda_fail(cudaError_t e, const char* what);

constexpr int kMaxDevices = 64;

struct DeviceInfo {
  std::atomic<bool> ready{false};
  int sms = 0;
  int major = 0;
  uint32_t* status = nullptr;
};

// The device of the calling thread's context, checked to be a B200.
int current_device(DeviceInfo** out);

// SMs the persistent launches leave free (swiglu_b200_set_sm_reserve).
int sm_reserve();

using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                   const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                   CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

int get_encode_fn(EncodeTiledFn* out);
// 8-bit operand map: row-major [rows, K] bytes, row pitch `ld` bytes; 128-byte
// swizzled boxes of {128 bytes of K, box_rows rows}.
int make_map_bytes(CUtensorMap* m, const void* ptr, uint64_t K, uint64_t rows, uint64_t ld, uint32_t box_rows,
                   const char* what);
int make_store_map(CUtensorMap* m, void* ptr, uint64_t N, uint64_t M, uint64_t ld, bool f32);

inline bool fits_int(int64_t v) { return v >= 0 && v <= 0x7fffffffLL; }
int check_dtype(int dtype);
int check_dims(const char* what, int64_t a, int64_t b, int64_t c);
int check_mult8(const char* what, int64_t v);

// Launches a kernel that begins with wait_for_previous(): its blocks may be
// placed while the stream's previous kernel drains (programmatic dependent
// launch), which hides the 1-2 us between two kernels of a stream.
template <class... Params, class... Args>
cudaError_t launch_after(void (*kern)(Params...), dim3 grid, dim3 block, size_t smem, cudaStream_t st, Args... args) {
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, static_cast<Params>(args)...);
}

// Per-kernel launch state: dynamic shared memory opt-in done (bit per device)
// and, for cluster kernels, how many CTA pairs fit at once on each device.
struct KernelState {
  std::atomic<uint64_t> ready{0};
  int max_clusters[kMaxDevices] = {};
};

template <auto Kernel>
KernelState& kernel_state() {
  static KernelState s;  // one per kernel function
  return s;
}

// Lets a kernel have `bytes` of dynamic shared memory, once per device.
template <auto kern>
int opt_in_smem(int bytes, const char* what) {
  KernelState& ks = kernel_state<kern>();
  int dev = 0;
  cudaGetDevice(&dev);
  if (!(ks.ready.load() & (1ull << dev))) {
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != cudaSuccess) return cuda_fail(e, what);
    ks.ready.fetch_or(1ull << dev);
  }
  return SWIGLU_OK;
}

// Persistent single-CTA launch: one CTA per SM (at most one per tile).
template <auto kern, class Params>
int launch_single(const Params& p, int tiles, int threads, int smem, const DeviceInfo& d, cudaStream_t st,
                  const char* what) {
  if (int rc = opt_in_smem<kern>(smem, what)) return rc;
  int sms = d.sms - sm_reserve();
  if (sms < 1) sms = 1;
  const int grid = tiles < sms ? tiles : sms;
  kern<<<grid, threads, smem, st>>>(p);
  cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? SWIGLU_OK : cuda_fail(e, what);
}

inline cudaLaunchConfig_t pair_launch_config(cudaLaunchAttribute* attr, int threads, int smem, cudaStream_t st) {
  cudaLaunchConfig_t cfg = {};
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cfg;
}

// How many CTA pairs of `kern` fit on the current device at once (queried
// once per device).
template <auto kern>
int pair_capacity(int threads, int smem, const DeviceInfo& d, int* out, const char* what) {
  KernelState& ks = kernel_state<kern>();
  int dev = 0;
  cudaGetDevice(&dev);
  if (!(ks.ready.load() & (1ull << dev))) {
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return cuda_fail(e, what);
    cudaLaunchAttribute attr[1];
    cudaLaunchConfig_t cfg = pair_launch_config(attr, threads, smem, nullptr);
    cfg.gridDim = dim3(2 * (d.sms / 2));
    int n = 0;
    e = cudaOccupancyMaxActiveClusters(&n, kern, &cfg);
    if (e != cudaSuccess) return cuda_fail(e, what);
    if (n < 1) return fail(SWIGLU_ERR_CUDA, "%s: no CTA pair fits on device %d", what, dev);
    ks.max_clusters[dev] = n;
    ks.ready.fetch_or(1ull << dev);
  }
  const int keep = ks.max_clusters[dev] - (sm_reserve() + 1) / 2;
  *out = keep < 1 ? 1 : keep;
  return SWIGLU_OK;
}

// Persistent CTA-pair launch (clusters of 2): as many pairs as fit at once,
// at most one per work unit.
template <auto kern, class Params>
int launch_pair(const Params& p, int units, int threads, int smem, const DeviceInfo& d, cudaStream_t st,
                const char* what) {
  int cap = 0;
  if (int rc = pair_capacity<kern>(threads, smem, d, &cap, what)) return rc;
  cudaLaunchAttribute attr[1];
  cudaLaunchConfig_t cfg = pair_launch_config(attr, threads, smem, st);
  cfg.gridDim = dim3(2 * (units < cap ? units : cap));
  cudaError_t e = cudaLaunchKernelEx(&cfg, kern, p);
  return e == cudaSuccess ? SWIGLU_OK : cuda_fail(e, what);
}

}  // namespace swiglu
