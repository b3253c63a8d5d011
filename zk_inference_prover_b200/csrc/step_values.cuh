// The values of a decode step (zkb_step_*): what its three operators share.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cmath>

#include "common.cuh"

namespace zk {

__device__ __forceinline__ float bf16_low(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float bf16_high(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }
// Two values rounded to bf16, to nearest even, the first in the low half.
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ uint16_t round_bf16(float x) { return __bfloat16_as_ushort(__float2bfloat16_rn(x)); }

// Eight values rounded to bf16 at a multiple of 16 bytes, WORD: their patterns in words.
template <bool WORD>
__device__ __forceinline__ void store8(void* p, int64_t at, const float (&x)[8]) {
    uint32_t v[4];
#pragma unroll
    for (int i = 0; i < 4; i++) v[i] = pack_bf16(x[2 * i], x[2 * i + 1]);
    if constexpr (WORD) {
        uint4* w = reinterpret_cast<uint4*>(static_cast<uint32_t*>(p) + at);
        w[0] = make_uint4(v[0] & 0xffffu, v[0] >> 16, v[1] & 0xffffu, v[1] >> 16);
        w[1] = make_uint4(v[2] & 0xffffu, v[2] >> 16, v[3] & 0xffffu, v[3] >> 16);
    } else {
        *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p) + at) = make_uint4(v[0], v[1], v[2], v[3]);
    }
}

// The sequence that row t belongs to, or -1; by a whole warp. 32 borders are looked at side by side: a round trip to memory for 32
// sequences, two for 1024. Whatever the array holds, it ends and stays inside it.
__device__ __forceinline__ int sequence_of(const int32_t* first, int n_seqs, int t) {
    const int lane = threadIdx.x & 31;
    int lo = 0, hi = n_seqs;
    while (hi - lo > 1) {
        const int step = (hi - lo + 31) / 32, at = lo + (lane + 1) * step;
        const bool before = at < hi && first[at] <= t;
        lo += __popc(__ballot_sync(0xffffffffu, before)) * step;
        hi = min(hi, lo + step);
    }
    return first[lo] <= t && t < first[lo + 1] ? lo : -1;
}

inline bool aligned_to(const void* p, size_t bytes) { return ((uintptr_t)p & (bytes - 1)) == 0; }

// What every call checks of the cache and the rows; the message is the caller's.
inline const char* step_problem(const zkb_kv_cache& c, const zkb_step_rows& r, uint32_t q_heads) {
    if (c.type != ZKB_VALUE_BF16 && c.type != ZKB_VALUE_INT8) return "cache.type is neither BF16 nor INT8";
    if (c.head_dim != 32 && c.head_dim != 64 && c.head_dim != 128) return "cache.head_dim is not 32, 64 or 128";
    if (!c.k || !c.v) return "cache.k or cache.v is NULL";
    if (c.type == ZKB_VALUE_INT8 && (!c.k_scale || !c.v_scale)) return "an INT8 cache needs k_scale and v_scale";
    if (c.type == ZKB_VALUE_BF16 && (!aligned_to(c.k, 2) || !aligned_to(c.v, 2))) return "cache.k or cache.v is not on a 2-byte boundary";
    if (c.type == ZKB_VALUE_INT8 && (!aligned_to(c.k_scale, 4) || !aligned_to(c.v_scale, 4))) return "k_scale or v_scale is not on a 4-byte boundary";
    if (c.n_seqs < 1 || c.n_seqs > 65535) return "cache.n_seqs is not in 1 .. 65535";
    if (c.n_heads < 1 || c.n_heads > 1024) return "cache.n_heads is not in 1 .. 1024";
    if (c.capacity < 1 || c.capacity > (1u << 30)) return "cache.capacity is not in 1 .. 2^30";
    if (c.capacity > 1 && std::llabs(c.token_stride) < (long long)c.head_dim) return "cache.token_stride is shorter than a row";
    if (std::llabs(c.token_stride) > (1ll << 29)) return "cache.token_stride exceeds 2^29";
    if (!r.first || !r.kv_len) return "rows.first or rows.kv_len is NULL";
    if (!aligned_to(r.first, 4) || !aligned_to(r.kv_len, 4)) return "rows.first or rows.kv_len is not on a 4-byte boundary";
    if (r.n_rows > (1u << 30)) return "rows.n_rows exceeds 2^30";
    if (q_heads < 1 || q_heads % c.n_heads != 0 || q_heads / c.n_heads > 64) return "q_heads is not 1 to 64 times cache.n_heads";
    return nullptr;
}

}  // namespace zk
