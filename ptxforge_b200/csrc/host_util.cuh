// host_util.cuh -- host-side helpers shared by the library's translation units: the driver's tensor-map encoder,
// programmatic launches and a current-device guard.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

#include <cstdio>
#include <cstdlib>
#include <utility>

#include "pf_b200.h"

namespace pf {

typedef CUresult (*EncodeTiledFn)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *,
                                  const cuuint64_t *, const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// Programmatic dependent launch for the tensor-core kernels: each launch may be scheduled while the previous
// kernel in the stream finishes; the kernel sets up its barriers and TMEM, then waits (griddepcontrol.wait)
// for that kernel's completion before any global memory access, so the result is the same as a plain launch.
// PF_PDL=0 in the environment turns it off (plain launches).
inline bool pdl_enabled() {
  static const bool on = [] {
    const char *e = std::getenv("PF_PDL");
    return !(e && e[0] == '0');
  }();
  return on;
}

// A launch with clusters of `cluster` CTAs along x where that is above 0 (otherwise as the kernel says).
template <class... Params, class... Args>
void launch_cluster(void (*kernel)(Params...), dim3 grid, dim3 block, int smem, int cluster, cudaStream_t s, Args &&...args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  cfg.numAttrs = 0;
  if (pdl_enabled()) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[cfg.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (cluster > 0) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
    attr[cfg.numAttrs].val.clusterDim.x = cluster;
    attr[cfg.numAttrs].val.clusterDim.y = 1;
    attr[cfg.numAttrs++].val.clusterDim.z = 1;
  }
  cfg.attrs = attr;
  cudaLaunchKernelEx(&cfg, kernel, std::forward<Args>(args)...);  // errors surface through cudaGetLastError
}
template <class... Params, class... Args>
void launch_pdl(void (*kernel)(Params...), dim3 grid, dim3 block, int smem, cudaStream_t s, Args &&...args) {
  launch_cluster(kernel, grid, block, smem, 0, s, std::forward<Args>(args)...);
}

// The driver's cuTensorMapEncodeTiled.  A function-local static is initialised exactly once, and threads
// whose first calls race all wait for that one initialisation (C++11 guarantees it), so none can see a
// half-initialised value.
inline EncodeTiledFn get_encode_fn() {
  static const EncodeTiledFn fn = [] {
    void *p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &q) ==
            cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      return reinterpret_cast<EncodeTiledFn>(p);
    return static_cast<EncodeTiledFn>(nullptr);
  }();
  return fn;
}

struct DeviceGuard {
  int prev = -1;
  explicit DeviceGuard(int dev) {
    cudaGetDevice(&prev);
    if (prev != dev) cudaSetDevice(dev);
  }
  ~DeviceGuard() {
    int cur = -1;
    cudaGetDevice(&cur);
    if (prev >= 0 && cur != prev) cudaSetDevice(prev);
  }
};

// A 2-D tiled TMA map; on failure a message goes to msg[0..len) (no heap: the no-allocation entry point
// uses it too).
inline int encode_2d_msg(char *msg, size_t len, CUtensorMap *map, CUtensorMapDataType dt, const void *base,
                         uint64_t inner, uint64_t outer, uint64_t row_bytes, uint32_t box_inner, uint32_t box_outer,
                         CUtensorMapSwizzle swz) {
  EncodeTiledFn enc = get_encode_fn();
  if (!enc) {
    if (msg && len) snprintf(msg, len, "cuTensorMapEncodeTiled unavailable from the CUDA driver");
    return PF_ECUDA;
  }
  cuuint64_t dims[2] = {inner, outer};
  cuuint64_t strides[1] = {row_bytes};
  cuuint32_t box[2] = {box_inner, box_outer};
  cuuint32_t estr[2] = {1, 1};
  CUresult r = enc(map, dt, 2, const_cast<void *>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, swz,
                   CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    if (msg && len)
      snprintf(msg, len, "cuTensorMapEncodeTiled failed (%d) for a %llux%llu tensor, box %ux%u", (int)r,
               (unsigned long long)outer, (unsigned long long)inner, box_outer, box_inner);
    return PF_ECUDA;
  }
  return PF_OK;
}

inline bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

}  // namespace pf
