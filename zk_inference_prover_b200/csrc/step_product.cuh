// Products of codes: what their kernels share.
#pragma once
#include "step_attention.cuh"

namespace zk {

__device__ __forceinline__ void store_value(void* out, int64_t at, uint32_t type, float y) {
    if (type == ZKB_VALUE_BF16) static_cast<uint16_t*>(out)[at] = round_bf16(y);
    else if (type == ZKB_VALUE_WORD) static_cast<uint32_t*>(out)[at] = round_bf16(y);
    else static_cast<float*>(out)[at] = y;
}

// 16 bytes from p on, of which the first `valid` are there; the others are zero. VEC: p is on a 16-byte boundary. `inner`: there are 4 more bytes on both sides.
template <bool VEC>
__device__ __forceinline__ uint4 load16(const int8_t* p, int valid, bool inner) {
    if (valid >= 16 && VEC) return *reinterpret_cast<const uint4*>(p);
    uint32_t w[4] = {};
    if (valid >= 16 && inner) {
        const uint32_t off = (uint32_t)(uintptr_t)p & 3;
        const uint32_t* q = reinterpret_cast<const uint32_t*>(p - off);
        uint32_t v[5];
#pragma unroll
        for (int i = 0; i < 5; i++) v[i] = q[i];
#pragma unroll
        for (int i = 0; i < 4; i++) w[i] = __funnelshift_r(v[i], v[i + 1], 8 * off);
    } else {
#pragma unroll
        for (int i = 0; i < 16; i++)
            if (i < valid) w[i / 4] |= (uint32_t)(uint8_t)p[i] << (8 * (i % 4));
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

template <bool INT4>
cudaError_t launch_tiles(zkb_ctx* ctx, const zkb_step_product_args& a);  // step_product_tiles.cu

}  // namespace zk
