// Host-side helpers shared by the translation units of the library: the
// error message, the launch counter, the tensor-map encoder, launches with
// programmatic dependent launch, per-device limits.
#pragma once

#include <atomic>
#include <cstdarg>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <mutex>
#include <set>
#include <utility>

#include "common.cuh"

namespace fvb_host {

inline thread_local char g_err[512] = "";
inline std::atomic<long long> g_launches{0};

inline int fail(int code, const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(g_err, sizeof(g_err), fmt, ap);
  va_end(ap);
  return code;
}

inline int check_launch(const char* what) {
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess)
    return fail(FVB_ERR_CUDA, "%s: launch failed: %s", what,
                cudaGetErrorString(e));
  g_launches.fetch_add(1, std::memory_order_relaxed);
  return FVB_OK;
}

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t,
                                  void*, const cuuint64_t*, const cuuint64_t*,
                                  const cuuint32_t*, const cuuint32_t*,
                                  CUtensorMapInterleave, CUtensorMapSwizzle,
                                  CUtensorMapL2promotion,
                                  CUtensorMapFloatOOBfill);

inline EncodeTiledFn get_encode() {
  static EncodeTiledFn fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p,
                                cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<EncodeTiledFn>(p);
  });
  return fn;
}

// Programmatic dependent launch is on unless FVB_PDL=0: each kernel may
// start its prologue (and the GEMMs their weight prefetch) while the
// previous kernel in the stream drains; every kernel executes
// griddepcontrol.wait before touching data produced upstream.
inline bool pdl_enabled() {
  static const int v = [] {
    const char* e = getenv("FVB_PDL");
    return e ? atoi(e) : 1;
  }();
  return v != 0;
}

template <typename... KArgs, typename... Args>
int launch_k(const char* what, void (*kern)(KArgs...), dim3 grid, dim3 block,
             size_t smem, cudaStream_t st, Args&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_enabled() ? 1 : 0;
  cudaError_t e = cudaLaunchKernelEx(&cfg, kern, std::forward<Args>(args)...);
  if (e != cudaSuccess)
    return fail(FVB_ERR_CUDA, "%s: launch failed: %s", what,
                cudaGetErrorString(e));
  return check_launch(what);
}

inline int sm_count() {
  static int counts[128] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 128) return 148;
  if (!counts[dev]) {
    int n = 0;
    cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
    counts[dev] = n > 0 ? n : 148;
  }
  return counts[dev];
}


// cudaFuncSetAttribute applies to the current device only, so the raised
// dynamic shared memory limit is remembered per (kernel, device): a process
// that drives several GPUs through this library sets it on each of them.
inline int ensure_smem(const void* kern, int bytes, const char* what) {
  static std::mutex mu;
  static std::set<std::pair<const void*, int>> done;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess)
    return fail(FVB_ERR_CUDA, "%s: cudaGetDevice: %s", what, cudaGetErrorString(e));
  std::lock_guard<std::mutex> lk(mu);
  if (done.count({kern, dev})) return FVB_OK;
  e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e != cudaSuccess)
    return fail(FVB_ERR_CUDA, "%s: shared memory attribute: %s", what,
                cudaGetErrorString(e));
  done.insert({kern, dev});
  return FVB_OK;
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace fvb_host
