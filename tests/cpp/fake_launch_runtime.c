/* Stands in for the calls that a launcher makes: nothing is launched, a launch with more dynamic shared memory or a larger cluster than its kernel has been allowed on the current device is
 * refused as the runtime refuses it (tests/test_launch_devices_cpu.py). */
#include <cuda_runtime_api.h>
#include <stdlib.h>
#include <string.h>

enum { kKernels = 64, kDevices = 4, kPlain = 48 * 1024 };
static const void* kernels[kKernels];
static int allowed[kKernels][kDevices], wide[kKernels][kDevices], sets, launches, device;
static cudaError_t last;
static int at(const void* f) {
    int i = 0;
    while (i < kKernels - 1 && kernels[i] && kernels[i] != f) ++i;
    kernels[i] = f;
    return i;
}
static cudaError_t done(cudaError_t e) { return e == cudaSuccess ? e : (last = e); }
int fake_sets(void) { return sets; }
int fake_launches(void) { return launches; }

cudaError_t cudaSetDevice(int d) { device = d; return cudaSuccess; }
cudaError_t cudaGetDevice(int* d) { *d = device; return cudaSuccess; }
cudaError_t cudaDeviceGetAttribute(int* v, enum cudaDeviceAttr a, int d) {
    (void)d;
    *v = a == cudaDevAttrMultiProcessorCount ? 148 : 227 * 1024;
    return cudaSuccess;
}
cudaError_t cudaFuncSetAttribute(const void* f, enum cudaFuncAttribute a, int v) {
    ++sets;
    if (a == cudaFuncAttributeMaxDynamicSharedMemorySize) allowed[at(f)][device] = v;
    else wide[at(f)][device] = v;
    return cudaSuccess;
}
static cudaError_t launch(const void* f, size_t smem, unsigned cluster) {
    const int i = at(f);
    if (smem > kPlain && smem > (size_t)allowed[i][device]) return done(cudaErrorInvalidValue);
    if (cluster > 8 && !wide[i][device]) return done(cudaErrorInvalidClusterSize);
    ++launches;
    return cudaSuccess;
}
cudaError_t cudaLaunchKernel(const void* f, dim3 grid, dim3 block, void** args, size_t smem, cudaStream_t st) {
    (void)grid; (void)block; (void)args; (void)st;
    return launch(f, smem, 1);
}
cudaError_t cudaLaunchKernelExC(const cudaLaunchConfig_t* c, const void* f, void** args) {
    unsigned cluster = 1;
    (void)args;
    for (unsigned i = 0; i < c->numAttrs; ++i)
        if (c->attrs[i].id == cudaLaunchAttributeClusterDimension) cluster = c->attrs[i].val.clusterDim.x;
    return launch(f, c->dynamicSmemBytes, cluster);
}
static struct { dim3 grid, block; size_t smem; cudaStream_t st; } pushed;
unsigned __cudaPushCallConfiguration(dim3 grid, dim3 block, size_t smem, cudaStream_t st) {
    pushed.grid = grid; pushed.block = block; pushed.smem = smem; pushed.st = st;
    return 0;
}
cudaError_t __cudaPopCallConfiguration(dim3* grid, dim3* block, size_t* smem, void* st) {
    *grid = pushed.grid; *block = pushed.block; *smem = pushed.smem; *(cudaStream_t*)st = pushed.st;
    return cudaSuccess;
}
cudaError_t cudaGetLastError(void) { const cudaError_t e = last; last = cudaSuccess; return e; }
cudaError_t cudaHostAlloc(void** p, size_t n, unsigned flags) { (void)flags; *p = calloc(1, n); return cudaSuccess; }
cudaError_t cudaThreadExchangeStreamCaptureMode(enum cudaStreamCaptureMode* m) { (void)m; return cudaSuccess; }
static int encode(void) { return 0; }
cudaError_t cudaGetDriverEntryPoint(const char* name, void** p, unsigned long long flags, enum cudaDriverEntryPointQueryResult* r) {
    (void)name; (void)flags;
    *p = (void*)encode;
    *r = cudaDriverEntryPointSuccess;
    return cudaSuccess;
}
