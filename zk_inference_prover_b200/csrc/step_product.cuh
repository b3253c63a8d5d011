// Products of codes: what their kernels share.
#pragma once
#include "product_shapes.hpp"
#include "step_attention.cuh"

namespace zk {

__device__ __forceinline__ void store_value(void* out, int64_t at, uint32_t type, float y) {
    if (type == ZKB_VALUE_BF16) static_cast<uint16_t*>(out)[at] = round_bf16(y);
    else if (type == ZKB_VALUE_WORD) static_cast<uint32_t*>(out)[at] = round_bf16(y);
    else static_cast<float*>(out)[at] = y;
}

// The first n (of up to 16) bytes from p on, byte by byte, zeros behind them.
__device__ __forceinline__ uint4 some_bytes(const int8_t* p, int n) {
    uint32_t w[4] = {};
#pragma unroll
    for (int i = 0; i < 16; i++) w[i / 4] |= i < n ? (uint32_t)(uint8_t)p[i] << (8 * (i % 4)) : 0u;
    return make_uint4(w[0], w[1], w[2], w[3]);
}
// 16 bytes of codes wherever they start. `lo`, `hi`: the array's first byte and the one behind its last. Fetched as the two whole 16-byte blocks of memory that they lie in, where the
// array has those, so that several fetches can be on their way; then turned into place, or, at the array's ends, read byte by byte (bytes outside of it: zeros).
struct Fetched {
    uint4 a, b;
};
__device__ __forceinline__ bool fetch_reaches_out(const int8_t* p, const int8_t* lo, const int8_t* hi) { return blocks_reach_out((uintptr_t)p, (uintptr_t)lo, (uintptr_t)hi); }
__device__ __forceinline__ Fetched fetch16(const int8_t* p, const int8_t* lo, const int8_t* hi) {
    Fetched r{make_uint4(0u, 0u, 0u, 0u), make_uint4(0u, 0u, 0u, 0u)};
    if (!fetch_reaches_out(p, lo, hi)) {
        const uint4* q = reinterpret_cast<const uint4*>(p - ((uint32_t)(uintptr_t)p & 15));
        r.a = q[0], r.b = q[1];
    }
    return r;
}
__device__ __forceinline__ uint4 fetched16(const Fetched& r, const int8_t* p, const int8_t* lo, const int8_t* hi) {
    if (fetch_reaches_out(p, lo, hi)) {
        uint32_t w[4] = {};
#pragma unroll
        for (int i = 0; i < 16; i++) w[i / 4] |= p + i >= lo && p + i < hi ? (uint32_t)(uint8_t)p[i] << (8 * (i % 4)) : 0u;
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
    const uint32_t m = (uint32_t)(uintptr_t)p & 15, v[8] = {r.a.x, r.a.y, r.a.z, r.a.w, r.b.x, r.b.y, r.b.z, r.b.w};
    uint32_t two[6], one[5];
#pragma unroll
    for (int i = 0; i < 6; i++) two[i] = m & 8 ? v[i + 2] : v[i];
#pragma unroll
    for (int i = 0; i < 5; i++) one[i] = m & 4 ? two[i + 1] : two[i];
    return make_uint4(__funnelshift_r(one[0], one[1], 8 * (m & 3)), __funnelshift_r(one[1], one[2], 8 * (m & 3)), __funnelshift_r(one[2], one[3], 8 * (m & 3)), __funnelshift_r(one[3], one[4], 8 * (m & 3)));
}
// The first n bytes, zeros behind them.
__device__ __forceinline__ uint4 first_bytes(uint4 v, int n) {
    auto keep = [&](uint32_t w, int left) { return left >= 4 ? w : left <= 0 ? 0u : w & ((1u << (8 * left)) - 1u); };
    return n >= 16 ? v : make_uint4(keep(v.x, n), keep(v.y, n - 4), keep(v.z, n - 8), keep(v.w, n - 12));
}

template <bool INT4>
cudaError_t launch_tiles(zkb_ctx* ctx, const zkb_step_product_args& a);  // step_product_tiles.cu

}  // namespace zk
