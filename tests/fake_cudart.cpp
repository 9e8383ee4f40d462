// A CUDA runtime for host-side tests: device memory is host memory, kernels do
// not run, and every call that orders work is written to a log.  Linked with
// the library's own objects in place of the CUDA runtime.
#include <cuda_runtime_api.h>

#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <map>
#include <string>

namespace {
std::map<const void*, std::string>& kernels() {
  static std::map<const void*, std::string> k;
  return k;
}
std::string g_log;
void note(const char* what, const void* stream) {
  char line[512];
  std::snprintf(line, sizeof(line), "%s %llu\n", what,
                static_cast<unsigned long long>(reinterpret_cast<uintptr_t>(stream)));
  g_log += line;
}
struct Launch {
  dim3 grid, block;
  size_t shared;
  void* stream;
};
thread_local Launch g_launch;
char g_handles[64];
int g_next_handle = 0;
}  // namespace

extern "C" {

// The log so far, one "what stream" a line; `clear` empties it.
const char* fake_log() { return g_log.c_str(); }
void fake_clear() { g_log.clear(); }

void** __cudaRegisterFatBinary(void*) { return reinterpret_cast<void**>(g_handles); }
void __cudaRegisterFatBinaryEnd(void**) {}
void __cudaUnregisterFatBinary(void**) {}
void __cudaRegisterFunction(void**, const char* host, char*, const char* name, int, void*, void*,
                            void*, void*, int*) {
  kernels()[host] = name;
}
void __cudaRegisterVar(void**, char*, char*, const char*, int, size_t, int, int) {}
unsigned __cudaPushCallConfiguration(dim3 grid, dim3 block, size_t shared, void* stream) {
  g_launch = {grid, block, shared, stream};
  return 0;
}
cudaError_t __cudaPopCallConfiguration(dim3* grid, dim3* block, size_t* shared, void* stream) {
  *grid = g_launch.grid;
  *block = g_launch.block;
  *shared = g_launch.shared;
  *static_cast<void**>(stream) = g_launch.stream;
  return cudaSuccess;
}
cudaError_t cudaLaunchKernel(const void* fn, dim3, dim3, void** args, size_t, cudaStream_t s) {
  const std::string& name = kernels()[fn];
  note(("launch " + name).c_str(), s);
  // The wait that runs out: its error word is its first argument.
  if (name.find("k_wait_selftest") != std::string::npos) **static_cast<unsigned**>(args[0]) = 4;
  return cudaSuccess;
}

cudaError_t cudaMalloc(void** p, size_t n) {
  *p = std::aligned_alloc(256, (n + 255) / 256 * 256);
  return cudaSuccess;
}
cudaError_t cudaFree(void* p) {
  std::free(p);
  return cudaSuccess;
}
cudaError_t cudaMallocHost(void** p, size_t n) { return cudaMalloc(p, n); }
cudaError_t cudaFreeHost(void* p) { return cudaFree(p); }
cudaError_t cudaMemcpy(void* d, const void* s, size_t n, cudaMemcpyKind) {
  std::memcpy(d, s, n);
  return cudaSuccess;
}
cudaError_t cudaMemcpyAsync(void* d, const void* s, size_t n, cudaMemcpyKind, cudaStream_t) {
  std::memcpy(d, s, n);
  return cudaSuccess;
}
cudaError_t cudaMemsetAsync(void* d, int v, size_t n, cudaStream_t s) {
  note("memset", s);
  std::memset(d, v, n);
  return cudaSuccess;
}
cudaError_t cudaMemcpyToSymbol(const void*, const void*, size_t, size_t, cudaMemcpyKind) {
  return cudaErrorNotSupported;
}
cudaError_t cudaMemcpyFromSymbol(void*, const void*, size_t, size_t, cudaMemcpyKind) {
  return cudaErrorNotSupported;
}
cudaError_t cudaGetSymbolAddress(void**, const void*) { return cudaErrorNotSupported; }

cudaError_t cudaEventCreate(cudaEvent_t* e) {
  *e = reinterpret_cast<cudaEvent_t>(g_handles + ++g_next_handle % 64);
  return cudaSuccess;
}
cudaError_t cudaEventCreateWithFlags(cudaEvent_t* e, unsigned) { return cudaEventCreate(e); }
cudaError_t cudaEventDestroy(cudaEvent_t) { return cudaSuccess; }
cudaError_t cudaEventQuery(cudaEvent_t) { return cudaSuccess; }
cudaError_t cudaEventElapsedTime(float* ms, cudaEvent_t, cudaEvent_t) {
  *ms = 0.0f;
  return cudaSuccess;
}
cudaError_t cudaEventRecord(cudaEvent_t, cudaStream_t s) {
  note("record", s);
  return cudaSuccess;
}
cudaError_t cudaEventSynchronize(cudaEvent_t) {
  note("synchronize event", nullptr);
  return cudaSuccess;
}
cudaError_t cudaStreamWaitEvent(cudaStream_t s, cudaEvent_t, unsigned) {
  note("wait", s);
  return cudaSuccess;
}
cudaError_t cudaStreamCreateWithFlags(cudaStream_t* s, unsigned) {
  *s = reinterpret_cast<cudaStream_t>(g_handles + ++g_next_handle % 64);
  return cudaSuccess;
}
cudaError_t cudaStreamDestroy(cudaStream_t) { return cudaSuccess; }
cudaError_t cudaStreamSynchronize(cudaStream_t s) {
  note("synchronize", s);
  return cudaSuccess;
}
cudaError_t cudaDeviceSynchronize() {
  note("synchronize device", nullptr);
  return cudaSuccess;
}
cudaError_t cudaStreamIsCapturing(cudaStream_t, cudaStreamCaptureStatus* c) {
  *c = cudaStreamCaptureStatusNone;
  return cudaSuccess;
}

cudaError_t cudaSetDevice(int) { return cudaSuccess; }
cudaError_t cudaGetDevice(int* d) {
  *d = 0;
  return cudaSuccess;
}
cudaError_t cudaGetDeviceCount(int* n) {
  *n = 1;
  return cudaSuccess;
}
cudaError_t cudaGetDeviceProperties_v2(cudaDeviceProp* p, int) {
  std::memset(p, 0, sizeof(*p));
  p->major = 10;
  p->multiProcessorCount = 148;
  return cudaSuccess;
}
cudaError_t cudaDeviceGetAttribute(int* v, cudaDeviceAttr, int) {
  *v = 0;
  return cudaSuccess;
}
cudaError_t cudaFuncSetAttribute(const void*, cudaFuncAttribute, int) { return cudaSuccess; }
cudaError_t cudaFuncGetAttributes(cudaFuncAttributes* a, const void*) {
  std::memset(a, 0, sizeof(*a));
  return cudaSuccess;
}
cudaError_t cudaGetDriverEntryPoint(const char*, void** fn, unsigned long long,
                                    cudaDriverEntryPointQueryResult* q) {
  // cuTensorMapEncodeTiled: its result is never read here.
  *fn = reinterpret_cast<void*>(+[]() -> int { return 0; });
  *q = cudaDriverEntryPointSuccess;
  return cudaSuccess;
}
cudaError_t cudaGetLastError() { return cudaSuccess; }
const char* cudaGetErrorString(cudaError_t) { return "fake"; }

}  // extern "C"
