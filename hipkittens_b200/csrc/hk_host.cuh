// What the translation units of libhk_attn share on the host: the state of a device, errors, launch counts, and tensor maps.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cstdio>
#include <mutex>

#include "../../include/hk_attn.h"
#include "attn_bwd_sm100.cuh"
#include "attn_fwd_sm100.cuh"
#include "dependent_launch.cuh"
#include "paged_decode_common.cuh"

#pragma GCC visibility push(hidden)
namespace hk_host {

constexpr int kMaxDevices = 64;

inline thread_local char g_cuda_err[256] = "";
inline std::atomic<unsigned long long> g_launches{0};

inline int cuda_fail(cudaError_t e, const char* what) {
  cudaGetLastError();  // reported here, and not once more by the caller's next check
  snprintf(g_cuda_err, sizeof(g_cuda_err), "%s: %s", what, cudaGetErrorString(e));
  return HK_ECUDA;
}
#define HK_CUDA(call)                                   \
  do {                                                  \
    cudaError_t e__ = (call);                           \
    if (e__ != cudaSuccess) return cuda_fail(e__, #call); \
  } while (0)

using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                   const cuuint64_t*, const cuuint32_t*, const cuuint32_t*,
                                   CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion,
                                   CUtensorMapFloatOOBfill);

inline EncodeTiledFn get_encode() {
  static EncodeTiledFn fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess) p = nullptr;
    return reinterpret_cast<EncodeTiledFn>(p);
  }();
  return fn;
}

// Per-device state: SM count, the device status word, one-time kernel attribute set-up.
struct DeviceState {
  std::mutex mu;
  bool ready = false;     // set once init_device succeeded; a failed attempt is retried by the next call
  bool window_ready = false;  // the kernels of calls with a window, which have attributes of their own to set
  int sm_count = 0;
  int cc_major = 0;
  hk::DecodeLimits decode;
  bool decode_fp8_ready = false;  // the decode over 8-bit pages, set up by its first call
  hk::DecodeLimits decode_fp8;
  bool ragged_ready = false;  // the kernels of ragged batches, as well
  int bwd_clusters[hk::kMaxDkdvSplit + 1] = {};  // clusters of so many dK/dV CTAs that the device holds at once
  int* status = nullptr;       // the status word, device address (kernels write it only when something went wrong)
  int* status_host = nullptr;  // ... and host address: mapped memory, so that reading it needs no copy
};
inline DeviceState g_dev[kMaxDevices];

// The first call on a device, and the first with a window there (hk_attn_api.cu).
int init_device(int device);
int init_windows();

template <int D, auto KIND, bool DEP>
int prepare_fwd_kernel() {
  auto* fn = hk::attn_fwd_kernel<D, KIND, DEP>;
  HK_CUDA(cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, hk::FwdSmem<D, int(KIND) != hk::kMaskNone>::kDynBytes));
  cudaFuncAttributes attr;
  HK_CUDA(cudaFuncGetAttributes(&attr, fn));
  // The kernel re-balances registers between warpgroups (208 per softmax thread, 88 per producer thread);
  // that only adds up if it was compiled to exactly kFwdRegsAtLaunch registers per thread at launch.
  // Refuse to launch otherwise: a register pool that is too small would block the re-allocation forever.
  if (attr.numRegs != hk::kFwdRegsAtLaunch) {
    snprintf(g_cuda_err, sizeof(g_cuda_err), "attn_fwd_kernel<%d,%d,%d> compiled to %d registers, expected %d", D,
             int(KIND), int(DEP), attr.numRegs, hk::kFwdRegsAtLaunch);
    return HK_EUNSUPPORTED;
  }
  return HK_OK;
}

template <int D, auto KIND>
int prepare_fwd_kernels() {
  const int rc = prepare_fwd_kernel<D, KIND, true>();
  if (rc != HK_OK) return rc;
  return prepare_fwd_kernel<D, KIND, hk::kLongFwdDependent<D, KIND>>();
}

template <typename Kernel>
int prepare_bwd_kernel(Kernel* fn, int dyn_bytes, const char* name) {
  HK_CUDA(cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, dyn_bytes));
  cudaFuncAttributes attr;
  HK_CUDA(cudaFuncGetAttributes(&attr, fn));
  // the count at launch has to be exact, as for the forward kernel: refuse to launch a build it would not add up in
  if (attr.numRegs != hk::kBwdRegsAtLaunch) {
    snprintf(g_cuda_err, sizeof(g_cuda_err), "%s compiled to %d registers, expected %d", name, attr.numRegs,
             hk::kBwdRegsAtLaunch);
    return HK_EUNSUPPORTED;
  }
  if (attr.sharedSizeBytes != 0) {  // the kernels assume their dynamic shared memory starts the CTA's window
    snprintf(g_cuda_err, sizeof(g_cuda_err), "%s has %zu bytes of static shared memory, expected none", name,
             attr.sharedSizeBytes);
    return HK_EUNSUPPORTED;
  }
  return HK_OK;
}

template <int D, auto KIND>
int prepare_bwd_kernels() {
  int rc = prepare_bwd_kernel(hk::attn_bwd_dkdv_kernel<D, KIND, false>, hk::BwdSmem<D>::kDynBytes, "attn_bwd_dkdv_kernel");
  if (rc != HK_OK) return rc;
  if constexpr (int(KIND) != hk::kMaskWindow && int(KIND) != hk::kMaskRagged) {
    rc = prepare_bwd_kernel(hk::attn_bwd_dkdv_kernel<D, KIND, true>, hk::BwdSmem<D>::kDynBytes, "attn_bwd_dkdv_kernel");
    if (rc != HK_OK) return rc;
  }
  return prepare_bwd_kernel(hk::attn_bwd_dq_kernel<D, KIND>, hk::BwdSmem<D>::kDynBytes, "attn_bwd_dq_kernel");
}

// Makes a device current for the duration of one entry point and puts the caller's current device back when the
// entry point returns (the reference launcher never touches the current device; a torch program whose current
// device is another GPU must not find it changed).
class DeviceScope {
 public:
  DeviceScope() = default;
  DeviceScope(const DeviceScope&) = delete;
  DeviceScope& operator=(const DeviceScope&) = delete;
  ~DeviceScope() {
    if (prev_ >= 0 && prev_ != cur_) cudaSetDevice(prev_);
  }
  // Switches to `device` (< 0: stay on the current one) and reports the index in use through *resolved.
  int enter_raw(int device, int* resolved) {
    HK_CUDA(cudaGetDevice(&prev_));
    if (device < 0) device = prev_;
    if (device >= kMaxDevices) return HK_EINVAL;
    if (device != prev_) HK_CUDA(cudaSetDevice(device));
    cur_ = device;
    *resolved = device;
    return HK_OK;
  }
  // enter_raw plus the device's state, initialised on first use (with `window`, for calls with one as well). A failed initialisation is
  // not remembered: the next call tries again (the failing thread finds the reason in hk_last_cuda_error()).
  int enter(int device, DeviceState** out, bool window = false) {
    int rc = enter_raw(device, &device);
    if (rc != HK_OK) return rc;
    DeviceState& st = g_dev[device];
    {
      std::lock_guard<std::mutex> lock(st.mu);
      if (!st.ready) {
        rc = init_device(device);
        if (rc != HK_OK) return rc;
        st.ready = true;
      }
      if (window && !st.window_ready) {
        rc = init_windows();
        if (rc != HK_OK) return rc;
        st.window_ready = true;
      }
    }
    *out = &st;
    return HK_OK;
  }

 private:
  int prev_ = -1, cur_ = -1;
};

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// Device status word -> HK_* code.
inline int status_to_code(int word) {
  switch (word) {
    case hk::kStatusOk: return HK_OK;
    case hk::kStatusSmemAlign: return HK_EUNSUPPORTED;
    case hk::kStatusBadPage: return HK_EBADPAGE;
    case hk::kStatusBadLen: return HK_EBADLEN;
    case hk::kStatusBadPos: return HK_EBADPOS;
    default: return HK_ETIMEOUT;
  }
}

// A tensor map by `encode`, called with the driver's function.
template <typename Encode>
int make_map(const Encode& encode) {
  EncodeTiledFn enc = get_encode();
  if (!enc) {
    snprintf(g_cuda_err, sizeof(g_cuda_err), "cuTensorMapEncodeTiled not available from the driver");
    return HK_ECUDA;
  }
  CUresult r = encode(enc);
  if (r == CUDA_ERROR_INVALID_CONTEXT) {
    // a thread that has made no runtime call yet (autograd's) has no current context: let the runtime bind the
    // device's own and try again. cudaSetDevice does that and, unlike cudaFree(nullptr), leaves a graph alone that
    // some thread is capturing at the time.
    int device = 0;
    HK_CUDA(cudaGetDevice(&device));
    HK_CUDA(cudaSetDevice(device));
    r = encode(enc);
  }
  if (r != CUDA_SUCCESS) {
    snprintf(g_cuda_err, sizeof(g_cuda_err), "cuTensorMapEncodeTiled failed with CUresult %d", int(r));
    return HK_ECUDA;
  }
  return HK_OK;
}

// 4-D map over a contiguous bf16 [B, N, heads, D] tensor, box = 64 columns x 1 head x 128 rows,
// 128-byte swizzle (rows of the box are 128 B, the layout tcgen05 descriptors expect).
// `st` = element strides of the batch, sequence and head dimensions (the D dimension is contiguous); every
// stride must be a multiple of 8 elements (16 bytes), which TMA requires.
inline int make_bnhd_map(CUtensorMap* map, const void* base, int B, int N, int heads, int D, const long long* st,
                  int box_rows = hk::kBlockM) {
  cuuint64_t dims[4] = {cuuint64_t(D), cuuint64_t(heads), cuuint64_t(N), cuuint64_t(B)};
  cuuint64_t strides[3] = {cuuint64_t(st[2]) * 2, cuuint64_t(st[1]) * 2, cuuint64_t(st[0]) * 2};
  cuuint32_t box[4] = {64, 1, cuuint32_t(box_rows), 1};
  cuuint32_t estr[4] = {1, 1, 1, 1};
  return make_map([&](EncodeTiledFn enc) {
    return enc(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(base), dims, strides, box, estr,
               CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  });
}

// 3-D map over the codes of a pool of 8-bit pages, [num_pages * 16 rows, heads, D] bytes, box = one page of one head, its rows of 64 or
// 128 bytes swizzled over as many.
inline int make_code_map(CUtensorMap* map, const void* base, int num_pages, int heads, int D) {
  cuuint64_t dims[3] = {cuuint64_t(D), cuuint64_t(heads), cuuint64_t(num_pages) * hk::kPageTokens};
  cuuint64_t strides[2] = {cuuint64_t(D), cuuint64_t(heads) * D};
  cuuint32_t box[3] = {cuuint32_t(D), 1, hk::kPageTokens};
  cuuint32_t estr[3] = {1, 1, 1};
  return make_map([&](EncodeTiledFn enc) {
    return enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
               D == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  });
}

// Whether an attention kernel is launched so that it may start under the tail of the one before it: up to 100 tiles per CTA
// (two heads x 128 x 128 in the forward, one in the backward), where a launch and a prologue are a visible share of it.
// The tiles are counted as if nothing were masked. A causal call has about half of them, and a paged one those of its
// contexts, which the host does not know, and not of its block table's width: such calls are launched the ordinary way
// from half the time on, or earlier.
// us per call in a loop, dependent / ordinary, at 28, 111, 221 and 443 tiles per CTA (H32/8 D128, B1 N2048, N4096,
// B2 and B4 N4096): non-causal 65.8 / 67.9, 232.0 / 233.7, 415.7 / 417.0, 830.7 / 830.1; causal
// 39.0 / 40.3, 117.7 / 120.4, 230.7 / 229.8, 456.6 / 452.8. Append and paged chunk, 8 x 512 tokens on contexts
// of 4096 (221 tiles): 487.8 / 479.2, and so the line is no higher.
inline bool short_kernel(long long tiles, int grid) { return tiles <= 100ll * grid; }

// The addresses from the first byte of an input or output to behind its last, and whether two of them may share memory.
struct Span {
  uintptr_t begin, end;
  Span(const void* p, long long bytes) : begin(reinterpret_cast<uintptr_t>(p)), end(begin + uintptr_t(bytes)) {}
  // of a [B, N, H, D] tensor of 16-bit elements with these strides
  Span(const void* p, const long long* strides, int B, int N, int H, int D)
      : Span(p, 2 * ((B - 1) * strides[0] + (N - 1) * strides[1] + (H - 1) * strides[2] + D)) {}
  bool meets(const Span& o) const { return begin < o.end && o.begin < end; }
};

}  // namespace hk_host
#pragma GCC visibility pop
