// tqk_stream_key.h -- which library-owned buffers a call uses (host only).
#pragma once

#include <cuda_runtime_api.h>

#include <atomic>
#include <tuple>

namespace tqk {

// A stream of a device.  cudaStreamPerThread is one handle for a different stream in every host thread, so there the
// thread belongs to the key: by a number of its own, since the ids of ended threads are given out again.
struct StreamKey {
    int device;
    cudaStream_t stream;
    unsigned long long thread;
    bool operator<(const StreamKey &o) const {
        return std::tie(device, stream, thread) < std::tie(o.device, o.stream, o.thread);
    }
};

inline StreamKey stream_key(int device, cudaStream_t stream) {
    if (stream != cudaStreamPerThread) return StreamKey{device, stream, 0};
    static std::atomic<unsigned long long> next{1};
    thread_local const unsigned long long mine = next.fetch_add(1);
    return StreamKey{device, stream, mine};
}

}  // namespace tqk
