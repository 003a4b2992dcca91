// Host-side helpers shared by the library's translation units: error text, launches with
// programmatic stream serialization, workspaces, tensor maps and the device status word.
#pragma once

#include <cstdarg>
#include <cstdio>
#include <cstring>
#include <mutex>
#include <string>
#include <type_traits>
#include <utility>

#include "dk_common.cuh"

namespace dk {
namespace host {

inline thread_local std::string g_last_error;

inline int fail(int code, const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  g_last_error = buf;
  return code;
}

inline int check_launch(const char* what) {
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return fail(DK_ERR_CUDA, "%s: launch failed: %s", what, cudaGetErrorString(e));
  return DK_OK;
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// Launch with programmatic stream serialization: the kernel may begin (and run
// its preamble) while the previous kernel on the stream finishes; every kernel
// of this library waits for its predecessor (griddepcontrol.wait) before it
// touches global memory that the predecessor may write.  One reads other memory
// first: own::own_kernel its lengths, tiles, queries, keys and values, which is
// safe behind prefix_kernel alone, whose CTAs let it begin only once they have
// themselves waited for whatever wrote those.  Every kernel waits before it ends,
// so that a kernel's end always means the end of all before it.
template <typename... KArgs, typename... Args>
cudaError_t launch_pdl(void (*kernel)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t st,
                       Args&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, std::forward<Args>(args)...);
}

constexpr int kMaxDevices = 64;

// Every workspace starts with a fixed area of arrival counters shared by all
// ops.  It must be zero when the workspace is first used; every call leaves it
// zero again.  Non-counter scratch always lives after it, so calls with
// different shapes never see each other's data in a counter.
constexpr size_t kCounterBytes = DK_WORKSPACE_COUNTER_BYTES;
constexpr int64_t kMaxCounters = static_cast<int64_t>(kCounterBytes / sizeof(int32_t));
inline uint8_t* ws_data(void* ws) { return static_cast<uint8_t*>(ws) + kCounterBytes; }

inline int current_device() {
  int d = 0;
  cudaGetDevice(&d);
  return d;
}

inline int sm_count(int device) {
  static int cache[kMaxDevices] = {0};
  if (device < 0 || device >= kMaxDevices) return 148;
  if (cache[device] == 0) {
    int n = 0;
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, device) != cudaSuccess || n <= 0) n = 148;
    cache[device] = n;
  }
  return cache[device];
}

// Raise the dynamic shared-memory limit of `fn` once per device.
template <typename F>
int ensure_smem(F fn, int bytes, bool (&done)[kMaxDevices]) {
  const int dev = current_device();
  if (dev >= 0 && dev < kMaxDevices && done[dev]) return DK_OK;
  cudaError_t e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e != cudaSuccess) return fail(DK_ERR_CUDA, "cudaFuncSetAttribute: %s", cudaGetErrorString(e));
  if (dev >= 0 && dev < kMaxDevices) done[dev] = true;
  return DK_OK;
}

// ---- TMA tensor maps through the driver entry point (no link-time libcuda dependency) ----
typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

inline EncodeTiledFn encode_fn() {
  static EncodeTiledFn fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &ptr, 12000, cudaEnableDefault, &q) ==
            cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<EncodeTiledFn>(ptr);
  });
  return fn;
}

inline int encode_map(CUtensorMap* map, CUtensorMapDataType dt, int rank, const void* base, const uint64_t* dims,
               const uint64_t* strides_bytes, const uint32_t* box, CUtensorMapSwizzle swz, const char* what) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return fail(DK_ERR_CUDA, "%s: cuTensorMapEncodeTiled unavailable", what);
  cuuint64_t gd[5], gs[4];
  cuuint32_t bx[5], es[5];
  for (int i = 0; i < rank; ++i) {
    gd[i] = dims[i];
    bx[i] = box[i];
    es[i] = 1;
    if (i + 1 < rank) gs[i] = strides_bytes[i];
  }
  CUresult r = fn(map, dt, rank, const_cast<void*>(base), gd, gs, bx, es, CU_TENSOR_MAP_INTERLEAVE_NONE, swz,
                  CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(DK_ERR_INVALID_ARGUMENT, "%s: cuTensorMapEncodeTiled failed (%d)", what, (int)r);
  return DK_OK;
}

inline bool valid_dtype(int d) { return d == DK_F32 || d == DK_F16 || d == DK_BF16; }

inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// The device status word of the including translation unit (each unit's kernels set their own copy;
// dk_device_status reads them all).  Reads, and with `clear` resets, the current device's word.
static inline cudaError_t unit_status(int clear, int* code, int* detail) {
  cudaError_t e = cudaMemcpyFromSymbol(code, dk::g_status_code, sizeof(int));
  if (e == cudaSuccess) e = cudaMemcpyFromSymbol(detail, dk::g_status_detail, sizeof(int));
  if (e == cudaSuccess && clear) {
    const int z = 0;
    e = cudaMemcpyToSymbol(dk::g_status_code, &z, sizeof(int));
    if (e == cudaSuccess) e = cudaMemcpyToSymbol(dk::g_status_detail, &z, sizeof(int));
  }
  return e;
}

// Status words of dk_serving.cu, dk_drafts.cu and dk_tree.cu (same contract as unit_status).
cudaError_t serving_status(int clear, int* code, int* detail);
cudaError_t drafts_status(int clear, int* code, int* detail);
cudaError_t tree_status(int clear, int* code, int* detail);

}  // namespace host
}  // namespace dk
