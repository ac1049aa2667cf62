// The witness calls' status word on the runtime of fake_hip.cpp, where no memory can be allocated (as while a stream of another
// thread is captured) and no stream be waited for: grape_init and the first witness call of each device take neither.
#include <hip/hip_runtime_api.h>
#include <cstdio>
#include "../../include/grape_hip.h"

extern "C" {
void fake_set_device(int device);
unsigned long fake_waits();
unsigned long fake_bytes();
// in front of the fake runtime's and HIP's own
hipError_t hipMalloc(void**, size_t) { return hipErrorStreamCaptureUnsupported; }
hipError_t hipStreamIsCapturing(hipStream_t, hipStreamCaptureStatus* s) {
    *s = hipStreamCaptureStatusNone;          // of the default stream; the captured one is not asked
    return hipSuccess;
}
}

static int failures = 0;
static void expect(bool ok, int device, const char* what) {
    if (!ok) {
        std::printf("device %d: does not hold: %s (%s)\n", device, what, grape_last_error());
        failures++;
    }
}

int main() {
    int32_t* p = reinterpret_cast<int32_t*>(4096);          // nothing is read
    for (int device : {0, 1, 15, 16, 17, 63}) {
        const unsigned long waits = fake_waits();
        expect(grape_init(device) == GRAPE_OK, device, "grape_init takes the device");
        expect(grape_wit_elemul_rescale(p, p, p, p, 1, 65536, nullptr) == GRAPE_OK, device, "a witness call is queued");
        expect(fake_waits() == waits && fake_bytes() == 0, device, "nothing is waited for or allocated");
    }
    // a first witness call on a device that grape_init has not seen
    fake_set_device(40);
    const unsigned long waits = fake_waits();
    expect(grape_wit_elemul_rescale(p, p, p, p, 1, 65536, nullptr) == GRAPE_OK, 40, "a witness call is queued");
    expect(fake_waits() == waits, 40, "nothing is waited for");
    return failures ? 1 : 0;
}
