// scratch.cuh — device buffers that a context grows on demand, and CUDA graphs.
//
// A captured graph names the buffers of the call that was captured.  When a
// later, larger call needs larger ones, those buffers stay until the context
// is destroyed: the graph may be replayed at any time.  Buffers that no
// capture has seen are freed.  (A graph and an eager call of one context do
// not overlap on the GPU, so it does not matter that they use different
// buffers: nothing in them outlives a call.)
#pragma once

#include <cuda_runtime.h>

#include <initializer_list>
#include <vector>

namespace m1 {

struct Scratch {
    bool captured = false;     // a capture has seen the present buffers
    std::vector<void *> kept;  // earlier ones that a graph names

    // Call on every use: true if `st` is being captured now.
    bool capturing(cudaStream_t st) {
        cudaStreamCaptureStatus s = cudaStreamCaptureStatusNone;
        if (cudaStreamIsCapturing(st, &s) != cudaSuccess) {
            cudaGetLastError();
            return false;
        }
        captured = captured || s != cudaStreamCaptureStatusNone;
        return s != cudaStreamCaptureStatusNone;
    }
    // The present buffers give way to larger ones.
    void retire(std::initializer_list<void *> old) {
        for (void *p : old) {
            if (!captured || !p) {
                cudaFree(p);
                continue;
            }
            try {
                kept.push_back(p);
            } catch (...) {  // no memory for the list: better lost than freed under a graph
            }
        }
        captured = false;
    }
    void release() {
        for (void *p : kept) cudaFree(p);
        kept.clear();
    }
};

}  // namespace m1
