// Attention over the key-value cache: what its kernels share.
#pragma once
#include "step_values.cuh"

namespace zk {

__device__ __forceinline__ uint32_t cluster_rank() { uint32_t r; asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r)); return r; }
__device__ __forceinline__ uint32_t cluster_ranks() { uint32_t r; asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(r)); return r; }
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// A word at this thread block's place in the shared memory of another one of the cluster.
__device__ __forceinline__ uint32_t peer_word(const void* p, int rank) {
    uint32_t at = (uint32_t)__cvta_generic_to_shared(p), there, w;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(at), "r"(rank));
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(w) : "r"(there) : "memory");
    return w;
}
__device__ __forceinline__ float peer_load(const float* p, int rank) { return __uint_as_float(peer_word(p, rank)); }
__device__ __forceinline__ int peer_load(const int* p, int rank) { return (int)peer_word(p, rank); }

// What is read once: past L1.
__device__ __forceinline__ uint4 ld_stream(const uint4* p) {
    uint4 a;
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(a.x), "=r"(a.y), "=r"(a.z), "=r"(a.w) : "l"(p));
    return a;
}

// c += a b, sixteen rows of a and eight columns of b, over sixteen.
__device__ __forceinline__ void mma_bf16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// An 8 x 8 matrix of 16-bit values, row g's values 2t and 2t + 1 in lane 4g + t, transposed.
__device__ __forceinline__ uint32_t transpose8(uint32_t a) {
    uint32_t b;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(b) : "r"(a));
    return b;
}

__device__ __forceinline__ uint32_t bf16_sub2(uint32_t a, uint32_t b) {
    const __nv_bfloat162 r = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
}
// Two 8-bit codes, in the low bytes of the halves of w, as bf16 (exactly): the low seven bits under 2^7's exponent are 128 + those bits, the sign bit
// in that pattern's last exponent bit makes 256 of 128, and the code is their difference.
__device__ __forceinline__ uint32_t code_halves(uint32_t w) { return bf16_sub2((w & 0x007f007fu) | 0x43004300u, (w & 0x00800080u) | 0x43004300u); }
// Four adjacent codes: the first two, the last two.
__device__ __forceinline__ void codes_to_bf16(uint32_t w, uint32_t& lo, uint32_t& hi) {
    lo = code_halves(__byte_perm(w, 0, 0x4140));
    hi = code_halves(__byte_perm(w, 0, 0x4342));
}
// Two keys' codes of adjacent dimensions, bytes 2 * upper and 2 * upper + 1 of a word apiece: the keys' pair for the one, and for the other.
__device__ __forceinline__ void pair_codes_to_bf16(uint32_t a, uint32_t b, int upper, uint32_t& first, uint32_t& second) {
    first = code_halves(__byte_perm(a, b, upper ? 0x0602 : 0x0400));
    second = code_halves(__byte_perm(a, b, upper ? 0x0703 : 0x0501));
}

// 0 * x + test in both halves: stays zero while all values are numbers.
__device__ __forceinline__ uint32_t zero_or_nan(uint32_t x, uint32_t test) {
    const __nv_bfloat162 r = __hfma2(*reinterpret_cast<const __nv_bfloat162*>(&x), __floats2bfloat162_rn(0.f, 0.f), *reinterpret_cast<const __nv_bfloat162*>(&test));
    return *reinterpret_cast<const uint32_t*>(&r);
}
// x with infinities and NaN as zero.
__device__ __forceinline__ uint32_t numbers_only(uint32_t x) {
    if ((x & 0x7f80u) == 0x7f80u) x &= 0xffff0000u;
    if ((x & 0x7f800000u) == 0x7f800000u) x &= 0xffffu;
    return x;
}
// The sum of what is no number among the values of dimension d that the row at position p sees (bf16 caches): the products are made without
// those values, because a matrix product has no way to keep 0 * NaN from the rows that do not see the key. Slow, and only for caches that hold such values.
__device__ __noinline__ float what_is_no_number(const char* v, int64_t row_bytes, int d, int64_t p, uint32_t capacity, uint32_t window, uint32_t sinks) {
    float y = 0.f;
    const int64_t end = min(p + 1, (int64_t)capacity), near = window ? max((int64_t)0, p - (int64_t)window + 1) : 0;
    for (int64_t j = 0; j < end; j++) {
        if (j >= (int64_t)sinks && j < near) j = near;
        if (j >= end) break;
        const float x = bf16_low(*reinterpret_cast<const uint16_t*>(v + j * row_bytes + 2 * d));
        if (!isfinite(x)) y += x;
    }
    return y;
}

// The rows of a sequence: the first of them, how many, and the first one's position. Whatever the arrays hold, the rows are within n_rows.
struct StepSequence {
    int first, rows;
    int64_t pos;
};
__device__ __forceinline__ StepSequence step_sequence(const zkb_step_rows& r, int seq) {
    const int from = r.first[seq], to = r.first[seq + 1], n = (int)r.n_rows;
    const int first = min(max(from, 0), n), rows = max(0, min(to, n) - first);
    return {first, rows, (int64_t)r.kv_len[seq] - ((int64_t)to - from) + (first - (int64_t)from)};
}

// The blocks of SIZE keys that hold what some row at positions low .. high sees: the first `near` of them from the first token on, the others from `from` on.
struct KeyBlocks {
    int n, sinks, from, end, size;
    __device__ __forceinline__ int base(int i) const { return i < sinks ? i * size : from + (i - sinks) * size; }
};
template <int SIZE>
__device__ __forceinline__ KeyBlocks key_blocks(int64_t low, int64_t high, uint32_t capacity, uint32_t window, uint32_t sinks) {
    KeyBlocks b{0, 0, 0, (int)max((int64_t)0, min(high + 1, (int64_t)capacity)), SIZE};
    if (window) {
        const int64_t near = min(max((int64_t)0, low - (int64_t)window + 1), (int64_t)b.end);
        b.from = (int)(near / SIZE) * SIZE;
        b.sinks = (int)min(((int64_t)min(sinks, capacity) + SIZE - 1) / SIZE, (int64_t)b.from / SIZE);
    }
    b.n = b.sinks + (b.end - b.from + SIZE - 1) / SIZE;
    return b;
}

}  // namespace zk
