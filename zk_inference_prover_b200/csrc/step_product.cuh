// Products of codes: what their kernels share.
#pragma once
#include "step_attention.cuh"

namespace zk {

__device__ __forceinline__ void store_value(void* out, int64_t at, uint32_t type, float y) {
    if (type == ZKB_VALUE_BF16) static_cast<uint16_t*>(out)[at] = round_bf16(y);
    else if (type == ZKB_VALUE_WORD) static_cast<uint32_t*>(out)[at] = round_bf16(y);
    else static_cast<float*>(out)[at] = y;
}

}  // namespace zk
