// fake_cuda.cu — a CUDA runtime of counters, for tests of the speculative-
// decoding entry points' host side without a GPU: linked with the objects of
// csrc/spec_attn.cu and csrc/spec_verify.cu in the place of cudart. Nothing is
// launched; what a call did is kept in `fake`.
#include <cstdarg>
#include <cstdio>
#include <cstring>

#include "ctx.h"

struct Fake {
    int device;           // the thread's current device
    int devices;          // how many there are
    int launches;         // since the last fake_new
    int launch_device;    // the current device at the last of them
    unsigned word;        // what a copy from the device finds
    int error;            // what the next launch answers
    int cluster;          // CTAs of a cluster at the last launch that named it
    int room[17];         // clusters of so many CTAs that the GPU holds at once
};
static Fake fake;
static cudaError_t last;

extern "C" {
ds_cuda_ctx *fake_new(int device, int sms) {
    fake = Fake();
    fake.devices = 4;
    fake.launch_device = -1;
    for (int n = 1; n <= 16; n++) fake.room[n] = sms / n;
    ds_cuda_ctx *c = new ds_cuda_ctx;
    c->device = device;
    c->sm_count = sms;
    c->ok = true;
    c->stream = (cudaStream_t)16;
    c->d_spec_err = (unsigned *)256;
    return c;
}
void fake_free(ds_cuda_ctx *c) { delete c; }
Fake *fake_state() { return &fake; }
const char *fake_message(ds_cuda_ctx *c) { return c->err.c_str(); }

static cudaError_t launched() {
    fake.launches++;
    fake.launch_device = fake.device;
    const cudaError_t e = (cudaError_t)fake.error;
    fake.error = 0;
    return last = e;
}
#ifndef __CUDA_ARCH__
cudaError_t cudaGetDevice(int *d) { return *d = fake.device, cudaSuccess; }
cudaError_t cudaSetDevice(int d) {
    if (d < 0 || d >= fake.devices) return cudaErrorInvalidDevice;
    return fake.device = d, cudaSuccess;
}
cudaError_t cudaGetLastError() {
    const cudaError_t e = last;
    return last = cudaSuccess, e;
}
cudaError_t cudaFuncSetAttribute(const void *, cudaFuncAttribute, int) { return cudaSuccess; }
cudaError_t cudaLaunchKernel(const void *, dim3, dim3, void **, size_t, cudaStream_t) { return launched(); }
cudaError_t cudaLaunchKernelExC(const cudaLaunchConfig_t *c, const void *, void **) {
    for (unsigned i = 0; i < c->numAttrs; i++)
        if (c->attrs[i].id == cudaLaunchAttributeClusterDimension) fake.cluster = c->attrs[i].val.clusterDim.x;
    return launched();
}
cudaError_t cudaOccupancyMaxActiveClusters(int *n, const void *, const cudaLaunchConfig_t *c) {
    return *n = fake.room[c->attrs[0].val.clusterDim.x], cudaSuccess;
}
cudaError_t cudaGetDriverEntryPoint(const char *, void **, unsigned long long, cudaDriverEntryPointQueryResult *) {
    return cudaErrorNotSupported;
}
cudaError_t cudaMemcpyAsync(void *dst, const void *, size_t n, cudaMemcpyKind, cudaStream_t) {
    return memcpy(dst, &fake.word, n < sizeof fake.word ? n : sizeof fake.word), cudaSuccess;
}
cudaError_t cudaStreamSynchronize(cudaStream_t) { return cudaSuccess; }
unsigned __cudaPushCallConfiguration(dim3, dim3, size_t, CUstream_st *) { return 0; }
cudaError_t __cudaPopCallConfiguration(dim3 *, dim3 *, size_t *, void *) { return cudaSuccess; }
void **__cudaRegisterFatBinary(void *) { return nullptr; }
void __cudaRegisterFatBinaryEnd(void **) {}
void __cudaUnregisterFatBinary(void **) {}
void __cudaRegisterFunction(void **, const char *, char *, const char *, int, uint3 *, uint3 *, dim3 *, dim3 *, int *) {}
void __cudaRegisterVar(void **, char *, char *, const char *, int, size_t, int, int) {}
#endif
}

int ctx_fail(ds_cuda_ctx *c, int code, const char *fmt, ...) {
    if (c) {
        char buf[512];
        va_list ap;
        va_start(ap, fmt);
        vsnprintf(buf, sizeof buf, fmt, ap);
        va_end(ap);
        c->err = buf;
    }
    return code;
}
int ctx_cuda(ds_cuda_ctx *c, cudaError_t e, const char *what) {
    return e == cudaSuccess ? DS_CUDA_OK : ctx_fail(c, DS_CUDA_ECUDA, "%s: %d", what, (int)e);
}
namespace ds {
cudaError_t launch_ex(const void *, dim3, dim3, size_t, cudaStream_t, bool, void **) { return launched(); }
}  // namespace ds
