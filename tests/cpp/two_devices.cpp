// Two devices without any hardware: the few runtime calls that opening the
// library and launching a kernel make, answered on the host.  Loaded ahead of
// the library; every LDS opt-in and launch is printed with its device.
#include <hip/hip_runtime_api.h>

#include <cstdio>
#include <cstdlib>
#include <cstring>

static int device = 0;
static dim3 grid, block;
static size_t lds;
static hipStream_t stream;

extern "C" {
hipError_t hipGetDeviceCount(int *n) { return *n = 2, hipSuccess; }
hipError_t hipSetDevice(int d) { return device = d, hipSuccess; }
hipError_t hipGetDevice(int *d) { return *d = device, hipSuccess; }
#undef hipGetDeviceProperties
hipError_t hipGetDevicePropertiesR0600(hipDeviceProp_tR0600 *p, int) {
    memset(p, 0, sizeof(*p));
    strcpy(p->gcnArchName, "gfx950:sramecc+:xnack-");
    return hipSuccess;
}
hipError_t hipMalloc(void **p, size_t n) { return *p = aligned_alloc(256, (n + 255) & ~size_t{255}), hipSuccess; }
hipError_t hipFree(void *p) { return free(p), hipSuccess; }
hipError_t hipGetLastError(void) { return hipSuccess; }
hipError_t hipStreamSynchronize(hipStream_t) { return hipSuccess; }
hipError_t hipDeviceSynchronize(void) { return hipSuccess; }
hipError_t hipFuncSetAttribute(const void *f, hipFuncAttribute, int bytes) {
    printf("optin %d %p %d\n", device, f, bytes);
    return hipSuccess;
}
hipError_t __hipPushCallConfiguration(dim3 g, dim3 b, size_t n, hipStream_t s) {
    return grid = g, block = b, lds = n, stream = s, hipSuccess;
}
hipError_t __hipPopCallConfiguration(dim3 *g, dim3 *b, size_t *n, hipStream_t *s) {
    return *g = grid, *b = block, *n = lds, *s = stream, hipSuccess;
}
hipError_t hipLaunchKernel(const void *f, dim3, dim3, void **, size_t n, hipStream_t) {
    printf("launch %d %p %zu\n", device, f, n);
    fflush(stdout);
    return hipSuccess;
}
}
