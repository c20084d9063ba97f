// The driver's tensor-map encoder, looked up once.
#pragma once
#include <cudaTypedefs.h>
#include <cuda_runtime.h>

namespace tb200 {

// Makes the current device's context current in this thread.  The encoder is a driver call and looks for one; a thread that has
// made no runtime call that needs a context yet (torch's backward thread, when the first kernel it launches is one of these) has none.
inline void bind_context() {
    static thread_local int bound = -1;
    int dev = -1;
    if (cudaGetDevice(&dev) == cudaSuccess && dev != bound && cudaSetDevice(dev) == cudaSuccess) bound = dev;
}

// NULL: the driver does not have it.  The first calls of several threads are in order (initialisation of a local static).
inline PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
    bind_context();
    static const PFN_cuTensorMapEncodeTiled_v12000 fn = []() -> PFN_cuTensorMapEncodeTiled_v12000 {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult res;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &res) == cudaSuccess && res == cudaDriverEntryPointSuccess)
            return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
        cudaGetLastError();
        return nullptr;
    }();
    return fn;
}

}  // namespace tb200
