// lk_common.cu — status codes, the device status word, device queries and TMA descriptor
// encoding shared by every entry point.
#include <cudaTypedefs.h>

#include <map>
#include <mutex>
#include <utility>

#include "gemm_split.h"
#include "lk_abi.h"
#include "lk_sm100.cuh"

namespace lk {

__device__ int g_status[4];
__device__ int g_bad_index[4];
__device__ unsigned long long g_wait_limit_ns = 1000000000ull;

namespace {
thread_local int t_last_cuda_error = 0;
thread_local ThreadDevice t_device;

constexpr int kMaxDevices = 64;
int g_sm_count[kMaxDevices];
std::mutex g_mu;

PFN_cuTensorMapEncodeTiled_v12000 g_encode = nullptr;

PFN_cuTensorMapEncodeTiled_v12000 encoder() {
  std::lock_guard<std::mutex> lock(g_mu);
  if (!g_encode) {
    void* fn = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess) {
      g_encode = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(fn);
    }
  }
  return g_encode;
}
}  // namespace

int cuda_status(cudaError_t err) {
  if (err == cudaSuccess) return LK_OK;
  t_last_cuda_error = (int)err;
  return LK_ERR_CUDA;
}

namespace {
struct ContextCalls {
  PFN_cuCtxGetDevice_v2000 device = nullptr;
  PFN_cuCtxGetCurrent_v4000 get = nullptr;
  PFN_cuCtxSetCurrent_v4000 set = nullptr;
  ContextCalls() {
    load("cuCtxGetDevice", device);
    load("cuCtxGetCurrent", get);
    load("cuCtxSetCurrent", set);
  }
  template <class F>
  static void load(const char* name, F& f) {
    void* fn = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint(name, &fn, cudaEnableDefault, &q) == cudaSuccess && q == cudaDriverEntryPointSuccess)
      f = reinterpret_cast<F>(fn);
    else
      cudaGetLastError();
  }
};
const ContextCalls& context_calls() {
  static const ContextCalls c;
  return c;
}
}  // namespace

// The driver is asked: the runtime's cudaGetDevice reports device 0 on a thread without a context.
int CudaApi::current_device(int* dev) {
  CUdevice d = -1;
  const auto f = context_calls().device;
  const int st = f ? (int)f(&d) : (int)CUDA_ERROR_NOT_FOUND;
  *dev = (int)d;
  return st;
}
int CudaApi::current_context(void** ctx) {
  const auto f = context_calls().get;
  return f ? (int)f(reinterpret_cast<CUcontext*>(ctx)) : (int)CUDA_ERROR_NOT_FOUND;
}
int CudaApi::set_context(void* ctx) {
  const auto f = context_calls().set;
  return f ? (int)f(static_cast<CUcontext>(ctx)) : (int)CUDA_ERROR_NOT_FOUND;
}
int CudaApi::set_device(int dev) { return cuda_status(cudaSetDevice(dev)); }

DeviceScope::DeviceScope(int device) : status_(switch_.to(device, t_device)) {}

DeviceScope::DeviceScope() : status_(switch_.to(t_device.for_status(DeviceSwitch<CudaApi>::now()), t_device)) {}

DeviceScope::DeviceScope(cudaStream_t stream) {
  int dev = t_device.for_null_stream();
  if (stream != nullptr) {
    // A capturing stream may not be asked for its device (the query ends the capture with an
    // error): the device that lk_set_device or an earlier call bound is taken, or the current one.
    cudaStreamCaptureStatus cap = cudaStreamCaptureStatusNone;
    if (cudaStreamIsCapturing(stream, &cap) == cudaSuccess && cap != cudaStreamCaptureStatusNone) {
      const int now = DeviceSwitch<CudaApi>::now();
      if (t_device.device < 0 && now >= 0) dev = now;
    } else if ((status_ = cuda_status(cudaStreamGetDevice(stream, &dev))) != LK_OK) {
      return;
    }
  }
  status_ = switch_.to(dev, t_device);
}

int sm_count() {
  int dev = t_device.device;
  if (dev < 0 && cudaGetDevice(&dev) != cudaSuccess) return 148;
  if (dev < 0 || dev >= kMaxDevices) return 148;
  {
    std::lock_guard<std::mutex> lock(g_mu);
    if (g_sm_count[dev] > 0) return g_sm_count[dev];
  }
  int n = 0;
  if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) n = 148;
  std::lock_guard<std::mutex> lock(g_mu);
  g_sm_count[dev] = n;
  return n;
}

int make_tmap(CUtensorMap* map, CUtensorMapDataType dtype, int rank, const void* base, const uint64_t* dims,
              const uint64_t* strides_bytes, const uint32_t* box, CUtensorMapSwizzle swizzle,
              CUtensorMapL2promotion promo) {
  if (!aligned16(base)) return LK_ERR_ALIGNMENT;
  for (int i = 0; i + 1 < rank; ++i)
    if (strides_bytes[i] % 16 != 0) return LK_ERR_ALIGNMENT;
  auto enc = encoder();
  if (!enc) return cuda_status(cudaErrorNotSupported);
  cuuint64_t gdim[5];
  cuuint64_t gstride[4];
  cuuint32_t bdim[5];
  cuuint32_t estride[5];
  for (int i = 0; i < rank; ++i) {
    gdim[i] = dims[i];
    bdim[i] = box[i];
    estride[i] = 1;
  }
  for (int i = 0; i + 1 < rank; ++i) gstride[i] = strides_bytes[i];
  CUresult r = enc(map, dtype, (cuuint32_t)rank, const_cast<void*>(base), gdim, gstride, bdim, estride,
                   CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, promo, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    t_last_cuda_error = 10000 + (int)r;  // driver error codes are offset to tell them apart
    return LK_ERR_CUDA;
  }
  return LK_OK;
}

namespace {
std::mutex g_inject_mu;
Injection g_inject = {LK_INJECT_NONE, -1, -1};
}  // namespace

Injection take_injection(int kind) {
  std::lock_guard<std::mutex> lock(g_inject_mu);
  if (g_inject.kind != kind || kind == LK_INJECT_NONE) return Injection{LK_INJECT_NONE, -1, -1};
  const Injection r = g_inject;
  g_inject = Injection{LK_INJECT_NONE, -1, -1};
  return r;
}

namespace gemm {
namespace {
std::mutex g_ws_mu;
std::map<std::pair<int, uintptr_t>, SplitWorkspace> g_ws_table;  // (device, stream) -> workspace
}  // namespace

bool split_workspace(cudaStream_t stream, int npairs, SplitWorkspace* out) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return false;
  const auto key = std::make_pair(dev, reinterpret_cast<uintptr_t>(stream));
  std::lock_guard<std::mutex> lock(g_ws_mu);
  auto it = g_ws_table.find(key);
  if (it != g_ws_table.end()) {
    *out = it->second;
    return true;
  }
  cudaStreamCaptureStatus cap = cudaStreamCaptureStatusNone;
  if (cudaStreamIsCapturing(stream, &cap) != cudaSuccess || cap != cudaStreamCaptureStatusNone) {
    cudaGetLastError();
    return false;
  }
  SplitWorkspace ws;
  const size_t partial_bytes = (size_t)npairs * 8 * 8 * 256 * sizeof(uint4);
  ws.flag_bytes = (size_t)npairs * 16 * sizeof(int);
  if (cudaMalloc(&ws.partial, partial_bytes) != cudaSuccess) {
    cudaGetLastError();
    return false;
  }
  if (cudaMalloc(&ws.flags, ws.flag_bytes) != cudaSuccess ||
      cudaMemsetAsync(ws.flags, 0, ws.flag_bytes, stream) != cudaSuccess) {
    cudaGetLastError();
    cudaFree(ws.partial);
    if (ws.flags) cudaFree(ws.flags);
    return false;
  }
  g_ws_table[key] = ws;
  *out = ws;
  return true;
}

int reset_split_workspaces() {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return (int)e;
  std::lock_guard<std::mutex> lock(g_ws_mu);
  for (auto& kv : g_ws_table) {
    if (kv.first.first != dev) continue;
    e = cudaMemset(kv.second.flags, 0, kv.second.flag_bytes);
    if (e != cudaSuccess) return (int)e;
  }
  return (int)cudaDeviceSynchronize();
}
}  // namespace gemm

}  // namespace lk

extern "C" {

const char* lk_status_string(int status) {
  switch (status) {
    case LK_OK:
      return "ok";
    case LK_ERR_INVALID_ARG:
      return "invalid argument";
    case LK_ERR_UNSUPPORTED:
      return "unsupported dtype, head dim or layout";
    case LK_ERR_CUDA:
      return "CUDA error";
    case LK_ERR_TIMEOUT:
      return "device pipeline wait timed out";
    case LK_ERR_ALIGNMENT:
      return "pointer or stride not 16-byte aligned";
    case LK_ERR_SCRATCH_LIMIT:
      return "problem exceeds the fixed scratch of a no-allocation entry point (rows > 65536)";
    default:
      return "unknown status";
  }
}

int lk_last_cuda_error(void) { return lk::t_last_cuda_error; }

int lk_version(void) { return (1 << 16) | 0; }

int lk_set_device(int device) {
  using namespace lk;
  if (device >= 0 && device == t_device.device) return LK_OK;
  int n = 0;
  if (int st = cuda_status(cudaGetDeviceCount(&n))) return st;
  if (device < 0 || device >= n) return cuda_status(cudaErrorInvalidDevice);
  t_device.device = device;
  t_device.seen = DeviceSwitch<CudaApi>::now();
  return LK_OK;
}

int lk_device_status(int* out4) {
  int h[4] = {0, 0, 0, 0};
  const lk::DeviceScope scope;
  int st = scope.status();
  if (st == LK_OK) st = lk::cuda_status(cudaDeviceSynchronize());
  if (st != LK_OK) return st;
  st = lk::cuda_status(cudaMemcpyFromSymbol(h, lk::g_status, sizeof(h)));
  if (st != LK_OK) return st;
  if (h[0] == 0) {
    st = lk::cuda_status(cudaMemcpyFromSymbol(h, lk::g_bad_index, sizeof(h)));
    if (st != LK_OK) return st;
  }
  if (out4)
    for (int i = 0; i < 4; ++i) out4[i] = h[i];
  return h[0];
}

int lk_debug_set_wait_limit(int64_t ns) {
  const unsigned long long v = ns > 0 ? (unsigned long long)ns : 1000000000ull;
  const lk::DeviceScope scope;
  int st = scope.status();
  if (st == LK_OK) st = lk::cuda_status(cudaDeviceSynchronize());
  if (st != LK_OK) return st;
  return lk::cuda_status(cudaMemcpyToSymbol(lk::g_wait_limit_ns, &v, sizeof(v)));
}

int lk_debug_inject(int kind, int block, int item) {
  if (kind < LK_INJECT_NONE || kind > LK_INJECT_PAGED_DROP_LOAD) return LK_ERR_INVALID_ARG;
  if (kind != LK_INJECT_NONE && (block < 0 || item < 0)) return LK_ERR_INVALID_ARG;
  std::lock_guard<std::mutex> lock(lk::g_inject_mu);
  lk::g_inject = lk::Injection{kind, block, item};
  return LK_OK;
}

int lk_clear_device_status(void) {
  int z[4] = {0, 0, 0, 0};
  const lk::DeviceScope scope;
  int st = scope.status();
  if (st == LK_OK) st = lk::cuda_status(cudaDeviceSynchronize());
  if (st != LK_OK) return st;
  // A split GEMM launch that gave up may have left its tail counters non-zero.
  st = lk::cuda_status((cudaError_t)lk::gemm::reset_split_workspaces());
  if (st != LK_OK) return st;
  st = lk::cuda_status(cudaMemcpyToSymbol(lk::g_bad_index, z, sizeof(z)));
  if (st != LK_OK) return st;
  return lk::cuda_status(cudaMemcpyToSymbol(lk::g_status, z, sizeof(z)));
}

}  // extern "C"
