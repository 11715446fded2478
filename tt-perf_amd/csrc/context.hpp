// context.hpp — what the operators' files (losses.hip, checkpoint8.hip, linear_grad8.hip) use of
// a context, whose state and checks are ttperf.hip's.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <new>
#include <string>

#include "ttperf/ttperf.h"

namespace ttpi {

// Records the message ttp_last_error() returns; gives `code` back.
__attribute__((visibility("hidden"))) int fail(int code, const std::string& msg);

// A failed HIP call's status and message (its error is reset).
__attribute__((visibility("hidden"))) int hip_failed(hipError_t e, const char* what);

struct Op {
    hipStream_t stream;
    int num_cus;
    const float* loss_scale;  // the context's, on the device; null while loss scaling is off
    uint32_t* tickets;        // is_last_block's counters
};

// A call's start: checks the context, makes its device current.
__attribute__((visibility("hidden"))) int begin(ttp_ctx* c, Op* op);

// [p, p + bytes) is device (or managed) memory of the context's device, inside one allocation.
// `seen`: of a call's buffers, the allocation the last one lies in (it answers for the next one
// there without asking the runtime again, about a microsecond).
struct SeenAlloc {
    uintptr_t lo = 0, end = 0;
};
__attribute__((visibility("hidden"))) int device_buffer(const ttp_ctx* c, const void* p,
                                                        uint64_t bytes, const char* what,
                                                        SeenAlloc* seen);

// The context's scratch memory: at least `bytes`, for one call's launches (the next call's reuse
// it, behind them on the stream).  Growing allocates and waits for the stream, which is refused
// while it is captured.  Memory that a capture has seen is kept until the context goes.
__attribute__((visibility("hidden"))) int workspace(ttp_ctx* c, uint64_t bytes,
                                                    void** p);

// Tensor `index`'s gradients, for a kernel that assigns them (no gradient yet) or adds to them.
struct GradTarget {
    void* data;
    uint64_t numel;
    bool bf16;   // the gradients' type: bf16 or fp32
    bool first;  // no gradient yet: assign
};
// Its checks are an accumulate's (the rule for captured calls among them); nothing changes.
__attribute__((visibility("hidden"))) int grad_target(ttp_ctx* c, uint32_t index, GradTarget* out);
// The kernel that writes them is queued: the tensor has a gradient, its sum is not current.
__attribute__((visibility("hidden"))) void grad_written(ttp_ctx* c, uint32_t index);

// Runs an entry point's body: no exception crosses the C ABI.
template <class F>
int guarded(F&& body) {
    try {
        return body();
    } catch (const std::bad_alloc&) {
        return fail(TTP_ERR_OOM, "out of host memory");
    } catch (...) {
        return fail(TTP_ERR_INVALID, "unexpected exception");
    }
}

}  // namespace ttpi

#define TTPI_HIP(expr)                                          \
    do {                                                        \
        hipError_t e_ = (expr);                                 \
        if (e_ != hipSuccess) return ttpi::hip_failed(e_, #expr); \
    } while (0)
