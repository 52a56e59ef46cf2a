// What every translation unit with entry points of the C ABI shares: the handle behind the void* of a caller, the
// status a HIP error becomes, and the switch to the handle's device.
#pragma once
#include "../../include/sharpnet_hip.h"

#include <hip/hip_runtime.h>
#include <stddef.h>

namespace snhip {

struct Handle {
    int device = 0;
    hipStream_t stream = nullptr;
    float* ws = nullptr;      // split-K partial sums
    size_t ws_bytes = 0;
    int* counters = nullptr;  // split-K arrival counters, zero whenever no GEMM is in flight
    size_t n_counters = 0;
    int splitk_mode = 0;      // 0: automatic, 1: always reduce in a second kernel, 2: always reduce in the GEMM kernel
    int num_cu = 256;
    int math_mode = 0;  // 0: fp32 MFMA, 1: bf16-input MFMA for every GEMM on this handle
    int force_cfg = -1;
    int force_splitk = 0;
    int last_cfg = -1;
    int last_splitk = 0;
    int rnn_step_mode = 0;  // 0: recurrent forward steps as one launch when the shape allows, 1: always GEMM + cell kernel
    unsigned long long rnn_dropout_seed = 0;   // the reference seeds cuDNN's dropout states with 0 (GPUWrapper.cs:472)
    unsigned long long rnn_dropout_calls = 0;  // training-mode forward calls that drew masks so far
    float* static_scratch = nullptr;  // this device's copy of `scratch` (kStaticScratchBytes), never freed
    char last_error[192] = {0};       // text of the last refusal that has more to say than its status code
};

inline int hip_to_status(hipError_t e) {
    switch (e) {
        case hipSuccess:
            return SNHIP_STATUS_SUCCESS;
        case hipErrorOutOfMemory:
            return SNHIP_STATUS_ALLOC_FAILED;
        case hipErrorInvalidValue:
        case hipErrorInvalidDevicePointer:
            return SNHIP_STATUS_INVALID_VALUE;
        case hipErrorNotInitialized:
        case hipErrorNoDevice:
            return SNHIP_STATUS_NOT_INITIALIZED;
        default:
            return SNHIP_STATUS_EXECUTION_FAILED;
    }
}

inline int ceil_div(int a, int b) { return (a + b - 1) / b; }

// Makes a handle's device the current one for the length of a call and the caller's device current again afterwards.
class DeviceScope {
  public:
    explicit DeviceScope(int device) {
        ok_ = hipGetDevice(&before_) == hipSuccess;
        if (ok_ && before_ != device) {
            ok_ = hipSetDevice(device) == hipSuccess;
            moved_ = ok_;
        }
    }
    ~DeviceScope() {
        if (moved_) (void)hipSetDevice(before_);
    }
    DeviceScope(const DeviceScope&) = delete;
    DeviceScope& operator=(const DeviceScope&) = delete;
    bool ok() const { return ok_; }

  private:
    int before_ = -1;
    bool ok_ = false, moved_ = false;
};

}  // namespace snhip
