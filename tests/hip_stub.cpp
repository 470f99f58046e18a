// A HIP runtime without a device, for tests of the host runtime's checks on the CPU: memory is
// host memory, copies happen at once, kernels are counted and not run. Linked with the host
// runtime's own sources into a test library (test_batch_host.py).
#include <hip/hip_ext.h>
#include <hip/hip_runtime.h>

#include <cstdlib>
#include <cstring>

extern "C" {
extern const unsigned char slm_code_object[1] = {0};
extern const size_t slm_code_object_size = 1;
extern const unsigned char slm_batch_object[1] = {0};
extern const size_t slm_batch_object_size = 1;

static long launches = 0;
static int capturing = 0;
long stub_launches() { return launches; }
void stub_set_capturing(int on) { capturing = on; }

static hipError_t grab(void** p, size_t n) {
    if (n > (size_t)4 << 30) return hipErrorOutOfMemory;
    return posix_memalign(p, 4096, n ? n : 1) ? hipErrorOutOfMemory : hipSuccess;
}
hipError_t hipEventCreate(hipEvent_t* e) { return *e = (hipEvent_t)malloc(1), hipSuccess; }
hipError_t hipEventCreateWithFlags(hipEvent_t* e, unsigned) { return hipEventCreate(e); }
hipError_t hipEventDestroy(hipEvent_t e) { return free((void*)e), hipSuccess; }
hipError_t hipEventElapsedTime(float* ms, hipEvent_t, hipEvent_t) { return *ms = 0, hipSuccess; }
hipError_t hipEventQuery(hipEvent_t) { return hipSuccess; }
hipError_t hipEventRecord(hipEvent_t, hipStream_t) { return hipSuccess; }
hipError_t hipEventSynchronize(hipEvent_t) { return hipSuccess; }
hipError_t hipExtModuleLaunchKernel(hipFunction_t, uint32_t, uint32_t, uint32_t, uint32_t, uint32_t, uint32_t, size_t,
                                    hipStream_t, void**, void**, hipEvent_t, hipEvent_t, uint32_t) {
    return launches++, hipSuccess;
}
hipError_t hipFree(void* p) { return free(p), hipSuccess; }
hipError_t hipFuncGetAttribute(int* v, hipFunction_attribute, hipFunction_t) { return *v = 0, hipSuccess; }
hipError_t hipGetDevice(int* d) { return *d = 0, hipSuccess; }
hipError_t hipGetDeviceCount(int* n) { return *n = 1, hipSuccess; }
hipError_t hipGetDevicePropertiesR0600(hipDeviceProp_tR0600* p, int) {
    memset(p, 0, sizeof *p);
    strcpy(p->gcnArchName, "gfx950");
    p->multiProcessorCount = 256;
    return hipSuccess;
}
const char* hipGetErrorString(hipError_t) { return "stub error"; }
hipError_t hipGetLastError() { return hipSuccess; }
hipError_t hipGraphDestroy(hipGraph_t) { return hipSuccess; }
hipError_t hipGraphExecDestroy(hipGraphExec_t) { return hipSuccess; }
hipError_t hipGraphInstantiate(hipGraphExec_t*, hipGraph_t, hipGraphNode_t*, char*, size_t) { return hipErrorUnknown; }
hipError_t hipGraphLaunch(hipGraphExec_t, hipStream_t) { return hipSuccess; }
hipError_t hipHostFree(void* p) { return free(p), hipSuccess; }
hipError_t hipHostGetDevicePointer(void** d, void* h, unsigned) { return *d = h, hipSuccess; }
hipError_t hipHostMalloc(void** p, size_t n, unsigned) { return grab(p, n); }
hipError_t hipMalloc(void** p, size_t n) { return grab(p, n); }
hipError_t hipMemGetInfo(size_t* f, size_t* t) { return *f = *t = (size_t)1 << 38, hipSuccess; }
hipError_t hipMemcpy(void* d, const void* s, size_t n, hipMemcpyKind) { return memcpy(d, s, n), hipSuccess; }
hipError_t hipMemcpyAsync(void* d, const void* s, size_t n, hipMemcpyKind, hipStream_t) { return memcpy(d, s, n), hipSuccess; }
hipError_t hipMemset(void* d, int v, size_t n) { return memset(d, v, n), hipSuccess; }
hipError_t hipMemsetAsync(void* d, int v, size_t n, hipStream_t) { return memset(d, v, n), hipSuccess; }
hipError_t hipModuleGetFunction(hipFunction_t* f, hipModule_t, const char* name) {
    return *f = (hipFunction_t)strdup(name), hipSuccess;
}
hipError_t hipModuleGetGlobal(hipDeviceptr_t* p, size_t* n, hipModule_t, const char*) {
    static int word;
    return *p = &word, *n = sizeof word, hipSuccess;
}
hipError_t hipModuleLaunchKernel(hipFunction_t, unsigned, unsigned, unsigned, unsigned, unsigned, unsigned, unsigned,
                                 hipStream_t, void**, void**) {
    return launches++, hipSuccess;
}
hipError_t hipModuleLoadData(hipModule_t* m, const void*) { return *m = (hipModule_t)1, hipSuccess; }
hipError_t hipModuleOccupancyMaxActiveBlocksPerMultiprocessor(int* n, hipFunction_t, int, size_t) { return *n = 1, hipSuccess; }
hipError_t hipModuleUnload(hipModule_t) { return hipSuccess; }
hipError_t hipSetDevice(int) { return hipSuccess; }
hipError_t hipStreamBeginCapture(hipStream_t, hipStreamCaptureMode) { return hipErrorUnknown; }
hipError_t hipStreamCreateWithFlags(hipStream_t* s, unsigned) { return *s = (hipStream_t)malloc(1), hipSuccess; }
hipError_t hipStreamDestroy(hipStream_t s) { return free((void*)s), hipSuccess; }
hipError_t hipStreamEndCapture(hipStream_t, hipGraph_t*) { return hipErrorUnknown; }
hipError_t hipStreamIsCapturing(hipStream_t, hipStreamCaptureStatus* s) {
    *s = capturing ? hipStreamCaptureStatusActive : hipStreamCaptureStatusNone;
    return hipSuccess;
}
hipError_t hipStreamSynchronize(hipStream_t) { return hipSuccess; }
hipError_t hipStreamWaitEvent(hipStream_t, hipEvent_t, unsigned) { return hipSuccess; }
}

__attribute__((visibility("hidden"))) hipError_t slm_scratch_address(void** out) {
    static char word[64];
    return *out = word, hipSuccess;
}
