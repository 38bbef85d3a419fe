// What the torch custom operators share: element types, error statuses and streams at the C ABI.
#pragma once
#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/library.h>

#include "p2p_b200.h"

namespace {

inline int dtype_code(const at::Tensor& t) {
    switch (t.scalar_type()) {
        case at::kBFloat16: return P2P_BF16;
        case at::kHalf: return P2P_F16;
        case at::kFloat: return P2P_F32;
        default: TORCH_CHECK(false, "p2p_b200: bfloat16, float16 or float32, got ", t.scalar_type());
    }
    return -1;
}

inline void check(int status, const char* what) {
    TORCH_CHECK(status == P2P_OK, what, ": ", p2p_last_error(), " (status ", status, ")");
}

inline void* stream_of(const at::Tensor& t) {
    return reinterpret_cast<void*>(c10::cuda::getCurrentCUDAStream(t.device().index()).stream());
}

}  // namespace
