// staging.h -- pinned host buffers for uploads that must not be overwritten while they run.
#pragma once

#include <cuda_runtime.h>
#include <stddef.h>

#include <algorithm>

namespace satori {

// Two pinned buffers used in turn; a buffer is handed out again only after the copy that read it has run.
class Staging {
  public:
    // A buffer of at least `bytes`, or an error.
    cudaError_t take(size_t bytes, void **out)
    {
        turn_ ^= 1;
        Slot &s = slots_[turn_];
        cudaError_t e = cudaSuccess;
        if (!s.done && (e = cudaEventCreateWithFlags(&s.done, cudaEventDisableTiming)) != cudaSuccess) return e;
        if ((e = cudaEventSynchronize(s.done)) != cudaSuccess) return e;
        if (bytes > s.bytes) {
            cudaFreeHost(s.data);
            s.data = nullptr;
            s.bytes = 0;
            const size_t n = std::max<size_t>(2 * bytes, 1 << 16);
            if ((e = cudaHostAlloc(&s.data, n, cudaHostAllocDefault)) != cudaSuccess) return e;
            s.bytes = n;
        }
        *out = s.data;
        return cudaSuccess;
    }
    // Copies the buffer's first `bytes` to the device.
    cudaError_t send(void *to, size_t bytes, cudaStream_t stream)
    {
        Slot &s = slots_[turn_];
        cudaError_t e = cudaMemcpyAsync(to, s.data, bytes, cudaMemcpyHostToDevice, stream);
        return e == cudaSuccess ? cudaEventRecord(s.done, stream) : e;
    }
    void release()
    {
        for (Slot &s : slots_) {
            if (s.done) {
                cudaEventSynchronize(s.done);
                cudaEventDestroy(s.done);
            }
            cudaFreeHost(s.data);
            s = Slot();
        }
    }

  private:
    struct Slot {
        void *data = nullptr;
        size_t bytes = 0;
        cudaEvent_t done = nullptr;
    } slots_[2];
    int turn_ = 0;
};

}  // namespace satori
