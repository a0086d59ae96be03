// CUDA's runtime as host memory, for programs that link the library's host code without a GPU: copies and fills are done at once, kernels are not run, the
// `fail_at`-th call that can fail does.  Counts what is allocated, and frees of what is not.
#pragma once
#include <cuda_runtime.h>
#include <stdarg.h>
#include <stdio.h>
#include <stdlib.h>
#include <string.h>

#include <set>
#include <string>

#include "dc_internal.h"

namespace fake {
inline std::set<void*> live;
inline int calls = 0, fail_at = 0, bad_frees = 0, launches = 0;
inline bool capturing = false;
inline std::string last_error;
inline bool fails() { return ++calls == fail_at; }
inline cudaError_t take(void** p, size_t n) {
    if (fails()) return cudaErrorMemoryAllocation;
    *p = n < (size_t(1) << 32) ? malloc(n ? n : 1) : nullptr;
    if (!*p) return cudaErrorMemoryAllocation;
    live.insert(*p);
    return cudaSuccess;
}
inline cudaError_t give(void* p) {
    if (p && !live.erase(p)) ++bad_frees;
    else free(p);
    return cudaSuccess;
}
inline cudaError_t done() { return fails() ? cudaErrorUnknown : cudaSuccess; }
}  // namespace fake

extern "C" {
void** __cudaRegisterFatBinary(void*) {
    static void* h;
    return &h;
}
void __cudaRegisterFatBinaryEnd(void**) {}
void __cudaUnregisterFatBinary(void**) {}
void __cudaRegisterFunction(void**, const char*, char*, const char*, int, uint3*, uint3*, dim3*, dim3*, int*) {}
void __cudaRegisterVar(void**, char*, char*, const char*, int, size_t, int, int) {}
char __cudaInitModule(void**) { return 1; }
unsigned __cudaPushCallConfiguration(dim3, dim3, size_t, cudaStream_t) { return 0; }
cudaError_t __cudaPopCallConfiguration(dim3*, dim3*, size_t*, void*) { return cudaSuccess; }
cudaError_t cudaLaunchKernel(const void*, dim3, dim3, void**, size_t, cudaStream_t) { return ++fake::launches, fake::done(); }
cudaError_t cudaLaunchKernelExC(const cudaLaunchConfig_t*, const void*, void**) { return ++fake::launches, fake::done(); }
cudaError_t cudaMalloc(void** p, size_t n) { return fake::take(p, n); }
cudaError_t cudaFree(void* p) { return fake::give(p); }
cudaError_t cudaHostAlloc(void** p, size_t n, unsigned) { return fake::take(p, n); }
cudaError_t cudaFreeHost(void* p) { return fake::give(p); }
cudaError_t cudaMemcpy(void* to, const void* from, size_t n, cudaMemcpyKind) {
    if (fake::fails()) return cudaErrorUnknown;
    memcpy(to, from, n);
    return cudaSuccess;
}
cudaError_t cudaMemcpyAsync(void* to, const void* from, size_t n, cudaMemcpyKind k, cudaStream_t) { return cudaMemcpy(to, from, n, k); }
cudaError_t cudaMemsetAsync(void* at, int v, size_t n, cudaStream_t) {
    if (fake::fails()) return cudaErrorUnknown;
    memset(at, v, n);
    return cudaSuccess;
}
cudaError_t cudaEventCreateWithFlags(cudaEvent_t* e, unsigned) { return fake::take((void**)e, 1); }
cudaError_t cudaEventDestroy(cudaEvent_t e) { return fake::give(e); }
cudaError_t cudaEventRecord(cudaEvent_t, cudaStream_t) { return fake::done(); }
cudaError_t cudaEventSynchronize(cudaEvent_t) { return fake::done(); }
cudaError_t cudaStreamSynchronize(cudaStream_t) { return cudaSuccess; }
cudaError_t cudaStreamIsCapturing(cudaStream_t, cudaStreamCaptureStatus* s) {
    *s = fake::capturing ? cudaStreamCaptureStatusActive : cudaStreamCaptureStatusNone;
    return cudaSuccess;
}
cudaError_t cudaSetDevice(int) { return cudaSuccess; }
cudaError_t cudaGetLastError() { return cudaSuccess; }
}

int dc_fail(dc_ctx*, int status, const char* fmt, ...) {
    char text[256];
    va_list a;
    va_start(a, fmt);
    vsnprintf(text, sizeof(text), fmt, a);
    va_end(a);
    fake::last_error = text;
    return status;
}
int dc_check_cuda(dc_ctx* ctx, cudaError_t e, const char* what) {
    return e == cudaSuccess ? DC_B200_OK : dc_fail(ctx, e == cudaErrorMemoryAllocation ? DC_B200_OUT_OF_MEMORY : DC_B200_BACKEND_ERROR, "%s", what);
}
int dc_kernel_setup(dc_ctx*, const void*, int, const char*) { return DC_B200_OK; }
uint8_t* dc_scratch(dc_ctx*, size_t) { return nullptr; }
void* dc_pinned(dc_ctx* ctx, size_t n) {
    static char room[1 << 17];
    return n <= sizeof(room) ? room : nullptr;
}
extern "C" int dc_b200_synchronize(dc_ctx*) { return DC_B200_OK; }
