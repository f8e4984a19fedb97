// What the files of the PyTorch binding share: types, sizes, statuses and the stream of a call.
#pragma once

#include <torch/types.h>
#include <c10/hip/HIPStream.h>

#include <cstdint>

#include "cc1d.h"

#define CHECK_SHAPE(x, ...) \
    TORCH_CHECK(x.sizes() == torch::IntArrayRef({__VA_ARGS__}), #x " must have shape (" #__VA_ARGS__ ")")

namespace {

inline int to_cc1d_dtype(at::ScalarType t, const char *what) {
    switch (t) {
        case at::ScalarType::Float: return CC1D_F32;
        case at::ScalarType::Half: return CC1D_F16;
        case at::ScalarType::BFloat16: return CC1D_BF16;
        default: TORCH_CHECK(false, what, " must be float32, float16 or bfloat16, got ", toString(t));
    }
    return -1;
}

// Sizes travel as int32 in the C ABI; strides and offsets are 64-bit.
inline int32_t size32(int64_t v, const char *what) {
    TORCH_CHECK(v >= 0 && v <= INT32_MAX, what, " = ", v, " does not fit the 32-bit sizes of the kernel library");
    return static_cast<int32_t>(v);
}

inline void check_status(int st, const char *op) {
    TORCH_CHECK(st == CC1D_OK, op, ": ", cc1d_strerror(st));
}

// The stream the launches go to: torch's current one.  A stream that is being captured into a
// HIP graph is refused.  Nothing on the launch path allocates, clears memory or synchronises the
// host, so capture ought to work, but it is not verified: the two capture runs of these operators
// (a decode loop, and a forward + backward, under torch.cuda.graph on a side stream) ended in a
// segmentation fault on the host whose cause was never established, and an error that says so
// is better than a crash in a serving process.
inline cc1d_stream_t current_stream() {
    hipStream_t stream = c10::hip::getCurrentHIPStream().stream();
    if (stream != nullptr) {
        hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
        const hipError_t err = hipStreamIsCapturing(stream, &status);
        TORCH_CHECK(err == hipSuccess && status == hipStreamCaptureStatusNone,
                    "causal_conv1d: the current stream is being captured into a HIP graph; graph capture of "
                    "these operators is not verified in this build and is refused");
    }
    return static_cast<cc1d_stream_t>(stream);
}

}  // namespace
