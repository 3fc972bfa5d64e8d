// A stand-in for libcuda.so.1 that runs nothing: device memory is host memory, streams do their
// copies at once, and a launch only looks at its arguments. It lets the host side of the library
// (workspaces, limits, threads) be tested on a machine without a GPU, and sees what a GPU
// would fault on: a launch that names freed memory, or more shared memory than was asked for.
#include <cuda.h>

#include <atomic>
#include <chrono>
#include <cstdlib>
#include <cstring>
#include <map>
#include <mutex>
#include <set>
#include <string>
#include <thread>
#include <vector>

namespace {

struct Function {
  std::string name;
  int dynamic_limit;  // bytes; what is not asked for shares 48 KB with the static ones
};

// What a launch names: the kernel and its scratch memory, if it takes any.
struct Launch {
  std::string name;
  CUdeviceptr scratch;
};
using Graph = std::vector<Launch>;

std::mutex mu;
std::map<CUdeviceptr, size_t> live;
std::map<CUstream, Graph> capturing;
std::vector<std::string> log;  // "launch NAME STREAM FIRST-POINTER", "error TEXT"
std::atomic<uintptr_t> next_handle{0x1000};
std::atomic<int> slow_ms{0};

template <typename T>
T handle() {
  return reinterpret_cast<T>(next_handle.fetch_add(16));
}

void pause_if_slow() {
  if (const int ms = slow_ms.load()) std::this_thread::sleep_for(std::chrono::milliseconds(ms));
}

bool inside_live(CUdeviceptr p) {  // (with mu held)
  auto it = live.upper_bound(p);
  return it != live.begin() && p < (--it)->first + it->second;
}

// Which parameter of a kernel points to a stream's scratch memory (-1: none).
int scratch_parameter(const std::string& name) {
  if (name == "gemm_bf16_tn_splitk") return 2;
  if (name == "splitk_reduce_bf16") return 0;
  if (name == "sdpa_fwd_bf16_d128_persist") return 9;
  if (name == "stage_bf16_pad_rows") return 1;
  return -1;
}

int static_bytes(const std::string& name) { return name.rfind("kv_plan_", 0) == 0 ? 272 : 0; }

void run(const Launch& l, CUstream stream) {
  if (l.scratch && !inside_live(l.scratch)) log.push_back("error " + l.name + " launched on freed memory");
  log.push_back("launch " + l.name + " " + std::to_string((uintptr_t)stream) + " " + std::to_string(l.scratch));
}

CUresult launch(const Function* f, unsigned shared, CUstream stream, void** params) {
  pause_if_slow();
  std::lock_guard<std::mutex> lock(mu);
  const int fixed = static_bytes(f->name);
  if ((int)shared > f->dynamic_limit && (int)shared + fixed > 48 * 1024) return CUDA_ERROR_INVALID_VALUE;
  Launch l{f->name, 0};
  if (const int at = scratch_parameter(f->name); at >= 0) memcpy(&l.scratch, params[at], sizeof l.scratch);
  if (auto it = capturing.find(stream); it != capturing.end()) it->second.push_back(l);
  else run(l, stream);
  return CUDA_SUCCESS;
}

}  // namespace

extern "C" {

// ---- what the tests ask ----
void fake_slow(int ms) { slow_ms = ms; }
int fake_log(char* to, int size) {
  std::lock_guard<std::mutex> lock(mu);
  std::string all;
  for (const std::string& line : log) all += line + "\n";
  log.clear();
  if ((int)all.size() + 1 > size) return -1;
  memcpy(to, all.c_str(), all.size() + 1);
  return (int)all.size();
}

// ---- the driver's entry points ----
CUresult cuInit(unsigned) { return CUDA_SUCCESS; }
CUresult cuDriverGetVersion(int* v) { return *v = 12090, CUDA_SUCCESS; }
CUresult cuDeviceGetCount(int* n) { return *n = 1, CUDA_SUCCESS; }
CUresult cuDeviceGet(CUdevice* d, int) { return *d = 0, CUDA_SUCCESS; }
CUresult cuDeviceGetName(char* to, int size, CUdevice) { return strncpy(to, "stand-in", size), CUDA_SUCCESS; }
CUresult cuDeviceGetAttribute(int* v, CUdevice_attribute a, CUdevice) {
  *v = a == CU_DEVICE_ATTRIBUTE_MULTIPROCESSOR_COUNT               ? 148
       : a == CU_DEVICE_ATTRIBUTE_COMPUTE_CAPABILITY_MAJOR         ? 10
       : a == CU_DEVICE_ATTRIBUTE_MAX_SHARED_MEMORY_PER_BLOCK_OPTIN ? 232448
                                                                    : 0;
  return CUDA_SUCCESS;
}
CUresult cuDeviceTotalMem(size_t* n, CUdevice) { return *n = 180ull << 30, CUDA_SUCCESS; }
CUresult cuDevicePrimaryCtxRetain(CUcontext* c, CUdevice) { return *c = handle<CUcontext>(), CUDA_SUCCESS; }
CUresult cuDevicePrimaryCtxRelease(CUdevice) { return CUDA_SUCCESS; }
CUresult cuCtxSetCurrent(CUcontext) { return CUDA_SUCCESS; }
CUresult cuCtxGetCurrent(CUcontext* c) { return *c = nullptr, CUDA_SUCCESS; }
CUresult cuCtxSynchronize() { return CUDA_SUCCESS; }
CUresult cuMemAlloc(CUdeviceptr* p, size_t bytes) {
  void* m = aligned_alloc(256, (bytes + 255) & ~size_t(255));
  if (!m) return CUDA_ERROR_OUT_OF_MEMORY;
  memset(m, 0xab, bytes);  // (what an earlier owner left)
  std::lock_guard<std::mutex> lock(mu);
  live[*p = (CUdeviceptr)m] = bytes;
  return CUDA_SUCCESS;
}
CUresult cuMemFree(CUdeviceptr p) {  // (never given back, so that no address means two blocks)
  std::lock_guard<std::mutex> lock(mu);
  if (!live.erase(p)) log.push_back("error memory freed twice");
  return CUDA_SUCCESS;
}
CUresult cuMemGetInfo(size_t* a, size_t* b) { return *a = *b = 180ull << 30, CUDA_SUCCESS; }
CUresult cuMemHostAlloc(void** p, size_t bytes, unsigned) {
  return (*p = calloc(1, bytes)) ? CUDA_SUCCESS : CUDA_ERROR_OUT_OF_MEMORY;
}
CUresult cuMemFreeHost(void* p) { return free(p), CUDA_SUCCESS; }
CUresult cuMemHostGetDevicePointer(CUdeviceptr* p, void* m, unsigned) { return *p = (CUdeviceptr)m, CUDA_SUCCESS; }
CUresult cuMemcpyHtoDAsync(CUdeviceptr to, const void* from, size_t n, CUstream) {
  return memcpy((void*)to, from, n), CUDA_SUCCESS;
}
CUresult cuMemcpyDtoHAsync(void* to, CUdeviceptr from, size_t n, CUstream) {
  return memcpy(to, (void*)from, n), CUDA_SUCCESS;
}
CUresult cuMemcpyDtoDAsync(CUdeviceptr to, CUdeviceptr from, size_t n, CUstream) {
  return memcpy((void*)to, (void*)from, n), CUDA_SUCCESS;
}
CUresult cuMemsetD8Async(CUdeviceptr p, unsigned char x, size_t n, CUstream) {
  return memset((void*)p, x, n), CUDA_SUCCESS;
}
CUresult cuMemsetD32Async(CUdeviceptr p, unsigned x, size_t n, CUstream) {
  for (size_t i = 0; i < n; ++i) ((unsigned*)p)[i] = x;
  return CUDA_SUCCESS;
}
CUresult cuStreamCreate(CUstream* s, unsigned) { return *s = handle<CUstream>(), CUDA_SUCCESS; }
CUresult cuStreamDestroy(CUstream) { return CUDA_SUCCESS; }
CUresult cuStreamSynchronize(CUstream) { return CUDA_SUCCESS; }
CUresult cuStreamWaitEvent(CUstream, CUevent, unsigned) { return CUDA_SUCCESS; }
CUresult cuStreamBeginCapture(CUstream s, CUstreamCaptureMode) {
  std::lock_guard<std::mutex> lock(mu);
  return capturing.emplace(s, Graph()).second ? CUDA_SUCCESS : CUDA_ERROR_ILLEGAL_STATE;
}
CUresult cuStreamIsCapturing(CUstream stream, CUstreamCaptureStatus* s) {
  std::lock_guard<std::mutex> lock(mu);
  *s = capturing.count(stream) ? CU_STREAM_CAPTURE_STATUS_ACTIVE : CU_STREAM_CAPTURE_STATUS_NONE;
  return CUDA_SUCCESS;
}
CUresult cuStreamEndCapture(CUstream s, CUgraph* g) {
  std::lock_guard<std::mutex> lock(mu);
  auto it = capturing.find(s);
  if (it == capturing.end()) return CUDA_ERROR_ILLEGAL_STATE;
  *g = reinterpret_cast<CUgraph>(new Graph(it->second));
  capturing.erase(it);
  return CUDA_SUCCESS;
}
CUresult cuStreamGetCaptureInfo_v2(CUstream stream, CUstreamCaptureStatus* s, cuuint64_t* id, CUgraph*,
                                   const CUgraphNode**, size_t*) {
  cuStreamIsCapturing(stream, s);
  if (id) *id = (cuuint64_t)(uintptr_t)stream;
  return CUDA_SUCCESS;
}
CUresult cuThreadExchangeStreamCaptureMode(CUstreamCaptureMode*) { return CUDA_SUCCESS; }
CUresult cuGraphInstantiateWithFlags(CUgraphExec* e, CUgraph g, unsigned long long) {
  *e = reinterpret_cast<CUgraphExec>(new Graph(*reinterpret_cast<Graph*>(g)));
  return CUDA_SUCCESS;
}
CUresult cuGraphLaunch(CUgraphExec e, CUstream stream) {
  std::lock_guard<std::mutex> lock(mu);
  for (const Launch& l : *reinterpret_cast<Graph*>(e)) run(l, stream);
  return CUDA_SUCCESS;
}
CUresult cuGraphExecDestroy(CUgraphExec) { return CUDA_SUCCESS; }
CUresult cuGraphDestroy(CUgraph) { return CUDA_SUCCESS; }
CUresult cuEventCreate(CUevent* e, unsigned) { return *e = handle<CUevent>(), CUDA_SUCCESS; }
CUresult cuEventDestroy(CUevent) { return CUDA_SUCCESS; }
CUresult cuEventRecord(CUevent, CUstream) { return CUDA_SUCCESS; }
CUresult cuEventQuery(CUevent) { return CUDA_SUCCESS; }
CUresult cuEventSynchronize(CUevent) { return CUDA_SUCCESS; }
CUresult cuEventElapsedTime(float* ms, CUevent, CUevent) { return *ms = 1.f, CUDA_SUCCESS; }
CUresult cuModuleLoadData(CUmodule* m, const void*) { return *m = handle<CUmodule>(), CUDA_SUCCESS; }
CUresult cuModuleUnload(CUmodule) { return CUDA_SUCCESS; }
CUresult cuModuleGetFunction(CUfunction* f, CUmodule, const char* name) {
  *f = reinterpret_cast<CUfunction>(new Function{name, 0});
  return CUDA_SUCCESS;
}
CUresult cuFuncSetAttribute(CUfunction f, CUfunction_attribute a, int v) {
  pause_if_slow();
  std::lock_guard<std::mutex> lock(mu);
  if (a == CU_FUNC_ATTRIBUTE_MAX_DYNAMIC_SHARED_SIZE_BYTES) reinterpret_cast<Function*>(f)->dynamic_limit = v;
  return CUDA_SUCCESS;
}
CUresult cuFuncGetAttribute(int* v, CUfunction_attribute a, CUfunction f) {
  *v = a == CU_FUNC_ATTRIBUTE_NUM_REGS            ? 255
       : a == CU_FUNC_ATTRIBUTE_SHARED_SIZE_BYTES ? static_bytes(reinterpret_cast<Function*>(f)->name)
                                                  : 0;
  return CUDA_SUCCESS;
}
CUresult cuLaunchKernel(CUfunction f, unsigned, unsigned, unsigned, unsigned, unsigned, unsigned, unsigned shared,
                        CUstream stream, void** params, void**) {
  return launch(reinterpret_cast<Function*>(f), shared, stream, params);
}
CUresult cuLaunchKernelEx(const CUlaunchConfig* c, CUfunction f, void** params, void**) {
  return launch(reinterpret_cast<Function*>(f), c->sharedMemBytes, c->hStream, params);
}
CUresult cuOccupancyMaxActiveClusters(int* n, CUfunction, const CUlaunchConfig*) { return *n = 74, CUDA_SUCCESS; }
CUresult cuTensorMapEncodeTiled(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill) {
  return CUDA_SUCCESS;
}
CUresult cuGetErrorString(CUresult, const char** s) { return *s = "an error", CUDA_SUCCESS; }
CUresult cuGetErrorName(CUresult r, const char** s) {
  return *s = r == CUDA_ERROR_INVALID_VALUE ? "CUDA_ERROR_INVALID_VALUE" : "CUDA_ERROR", CUDA_SUCCESS;
}
CUresult cuPointerGetAttribute(void*, CUpointer_attribute, CUdeviceptr) { return CUDA_ERROR_NOT_SUPPORTED; }
CUresult cuMemGetAddressRange(CUdeviceptr* base, size_t* n, CUdeviceptr p) {
  std::lock_guard<std::mutex> lock(mu);
  auto it = live.upper_bound(p);
  if (it == live.begin()) return CUDA_ERROR_INVALID_VALUE;
  --it;
  return *base = it->first, *n = it->second, CUDA_SUCCESS;
}
CUresult cuIpcGetMemHandle(CUipcMemHandle*, CUdeviceptr) { return CUDA_ERROR_NOT_SUPPORTED; }
CUresult cuIpcOpenMemHandle(CUdeviceptr*, CUipcMemHandle, unsigned) { return CUDA_ERROR_NOT_SUPPORTED; }
CUresult cuIpcCloseMemHandle(CUdeviceptr) { return CUDA_ERROR_NOT_SUPPORTED; }

}  // extern "C"
