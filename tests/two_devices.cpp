// Set-up calls of the block-scaled cache in a process with two devices, on the host: pretend devices
// and streams that note what runs where. Prints the first rule broken and exits with 1.
#include <hip/hip_runtime.h>

#include <cstdio>
#include <cstdlib>

#include "eb_internal.h"

static int line = 0;
#define RULE(x) do { if (!(x) && !line) { line = __LINE__; std::printf("line %d: %s\n", line, #x); } } while (0)

// ---- the pretend runtime: a stream is its device's number + 1 -----------------------------------

static int current = 0;
static int fills = 0;
static int misplaced = 0;  // launches on a stream of a device that is not current

static int device_of(hipStream_t st) { return (int)(reinterpret_cast<uintptr_t>(st) - 1); }

hipError_t hipGetDeviceCount(int *n) { return *n = 2, hipSuccess; }
hipError_t hipSetDevice(int d) { return current = d, hipSuccess; }
hipError_t hipGetDevice(int *d) { return *d = current, hipSuccess; }
hipError_t hipDeviceGetAttribute(int *v, hipDeviceAttribute_t, int) { return *v = 256, hipSuccess; }
hipError_t hipStreamCreateWithFlags(hipStream_t *st, unsigned) {
    return *st = reinterpret_cast<hipStream_t>((uintptr_t)current + 1), hipSuccess;
}
hipError_t hipStreamDestroy(hipStream_t) { return hipSuccess; }
hipError_t hipStreamSynchronize(hipStream_t) { return hipSuccess; }
hipError_t hipStreamIsCapturing(hipStream_t, hipStreamCaptureStatus *s) {
    return *s = hipStreamCaptureStatusNone, hipSuccess;
}
hipError_t hipMalloc(void **p, size_t n) { return (*p = std::malloc(n)) ? hipSuccess : hipErrorOutOfMemory; }
hipError_t hipFree(void *p) { return std::free(p), hipSuccess; }
hipError_t hipGetLastError() { return hipSuccess; }
const char *hipGetErrorName(hipError_t) { return ""; }
const char *hipGetErrorString(hipError_t) { return ""; }

namespace eb {
eb_status noalloc_scratch_of_current_device(float **) { return EB_OTHER; }
eb_status launch_fill_u8(hipStream_t st, uint8_t *, uint8_t, size_t) {
    ++fills;
    misplaced += device_of(st) != current;
    return EB_OK;
}
}  // namespace eb

int main() {
    eb_device *a = nullptr, *b = nullptr;
    RULE(eb_device_new(0, &a) == EB_OK && eb_device_new(1, &b) == EB_OK && current == 1);
    const size_t dims[3] = {64, 128, 64};
    // the second cache's tensors come from the pool, where the first one's went
    for (int i = 0; i < 2; ++i) {
        eb_kv_cache *kv = nullptr;
        current = 1;
        RULE(eb_kv_cache_new_i8(a, dims, 3, 256, 2, 32, &kv) == EB_OK && kv);
        RULE(fills == 6 * (i + 1) && misplaced == 0);
        eb_kv_cache_release(kv);
    }
    eb_device_release(a);
    eb_device_release(b);
    return line != 0;
}
