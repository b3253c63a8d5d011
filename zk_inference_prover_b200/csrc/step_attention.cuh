// Attention over the key-value cache: what its kernels share.
#pragma once
#include <cuda.h>

#include <algorithm>
#include <cstdlib>

#include "step_values.cuh"

namespace zk {

__device__ __forceinline__ uint32_t cluster_rank() { uint32_t r; asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r)); return r; }
__device__ __forceinline__ uint32_t cluster_ranks() { uint32_t r; asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(r)); return r; }
__device__ __forceinline__ void cluster_arrive() {
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
// To this thread block's place in the shared memory of another one of the cluster.
__device__ __forceinline__ void peer_store_word(const void* p, int rank, uint32_t w) {
    const uint32_t at = (uint32_t)__cvta_generic_to_shared(p);
    uint32_t there;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(at), "r"(rank));
    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(there), "r"(w) : "memory");
}
__device__ __forceinline__ void peer_store(float* p, int rank, float x) { peer_store_word(p, rank, __float_as_uint(x)); }
__device__ __forceinline__ void peer_store(int* p, int rank, int x) { peer_store_word(p, rank, (uint32_t)x); }
__device__ __forceinline__ void peer_store4(uint32_t at, int rank, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    uint32_t there;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(at), "r"(rank));
    asm volatile("st.shared::cluster.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(there), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
// A barrier of some of the thread block's warps.
__device__ __forceinline__ void named_sync(int id, int threads) {
    __syncwarp();
    asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}
__device__ __forceinline__ bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }
__device__ __forceinline__ uint32_t ld_shared(uint32_t p) {
    uint32_t w;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w) : "r"(p) : "memory");
    return w;
}
__device__ __forceinline__ void ld_shared2(uint32_t p, uint32_t& a, uint32_t& b) { asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(a), "=r"(b) : "r"(p) : "memory"); }
__device__ __forceinline__ void ld_shared4(uint32_t p, uint32_t& a, uint32_t& b, uint32_t& c, uint32_t& d) {
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(a), "=r"(b), "=r"(c), "=r"(d) : "r"(p) : "memory");
}
__device__ __forceinline__ void st_shared4(uint32_t p, uint32_t a, uint32_t b, uint32_t c, uint32_t d) { asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(p), "r"(a), "r"(b), "r"(c), "r"(d) : "memory"); }
__device__ __forceinline__ void st_shared(uint32_t p, uint32_t w) { asm volatile("st.shared.u32 [%0], %1;" ::"r"(p), "r"(w) : "memory"); }

// ---- copies by the tensor memory unit --------------------------------------------------------------------------------------------------
__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count) { asm volatile("mbarrier.init.shared.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory"); }
__device__ __forceinline__ void mbar_expect(uint32_t bar, uint32_t bytes) { asm volatile("mbarrier.arrive.expect_tx.shared.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory"); }
__device__ __forceinline__ void mbar_arrive(uint32_t bar) { asm volatile("mbarrier.arrive.shared.b64 _, [%0];" ::"r"(bar) : "memory"); }
// Whether the phase of this parity has ended, or does within a moment.
__device__ __forceinline__ bool mbar_test(uint32_t bar, uint32_t parity) {
    uint32_t done;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(done) : "r"(bar), "r"(parity) : "memory");
    return done;
}
// Waits for it to end; false when the limit of tries (seconds) ran out.
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity) {
    if (mbar_test(bar, parity)) return true;
#pragma unroll 1
    for (int tries = 0; tries < (1 << 20); tries++)
        if (mbar_test(bar, parity)) return true;
    return false;
}
// The box of a cache's map from (value, token, head, sequence) on.
__device__ __forceinline__ void tma_load(uint32_t to, const CUtensorMap* map, int value, int token, int head, int seq, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.4d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(to), "l"(map), "r"(value), "r"(token), "r"(head), "r"(seq), "r"(bar)
                 : "memory");
}
// Where byte `at` of a box's row lies, boxes as wide as BOX bytes.
template <int BOX>
__device__ __forceinline__ uint32_t box_place(int row, int at) {
    return row * BOX + (BOX == 128 ? at ^ ((row & 7) << 4) : BOX == 64 ? at ^ (((row >> 1) & 3) << 4) : at);
}
constexpr unsigned WAIT_RAN_OUT = 0x57e9;  // what zkb_sync reports

// The driver's call that makes a tensor's map, or NULL.
typedef CUresult (*TensorMapEncode)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                    CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
TensorMapEncode tensor_map_encode();

// Maps of a cache's K and V (boxes of `tokens` tokens by up to 128 bytes, swizzled by their own width), or false where the layout has none: the unit wants
// 16-byte boundaries and strides that ascend.
struct CacheMaps {
    CUtensorMap k, v;
};
bool cache_maps(CacheMaps& maps, const zkb_kv_cache& c, uint32_t tokens);

// How many clusters of 1, 2, 4, 8 or 16 thread blocks the GPU holds at a time with one thread block an SM (cudaOccupancyMaxActiveClusters): a cluster lies in one of
// the GPU's eight groups of 16 to 20 SMs. Clusters that have to wait for others double the time: eight of 16 take 38 us where eight of 8 take 25.
inline uint32_t clusters_at_once(uint32_t ranks) { return ranks <= 1 ? 148 : ranks == 2 ? 74 : ranks == 4 ? 33 : ranks == 8 ? 15 : 7; }

// Launches clusters of `ranks` (a power of two) thread blocks, or of fewer where the device, or the share of it that this process has, does not take as many.
// ZKB_STEP_CLUSTERS: as though it took that many at most, to try these ways.
template <class Launch>
inline cudaError_t launch_clusters(uint32_t ranks, Launch launch) {
    const char* const env = getenv("ZKB_STEP_CLUSTERS");
    const uint32_t most = env ? (uint32_t)std::max(1, atoi(env)) : ranks;
    for (;; ranks /= 2) {
        const cudaError_t e = ranks <= most ? launch(ranks) : cudaErrorInvalidClusterSize;
        if (ranks == 1 || (e != cudaErrorInvalidClusterSize && e != cudaErrorInvalidConfiguration && e != cudaErrorLaunchOutOfResources && e != cudaErrorNotSupported)) return e;
        (void)cudaGetLastError();
    }
}

template <int D, bool INT8>
cudaError_t launch_many(zkb_ctx* ctx, const zkb_step_attention_args& a);  // step_attention_many.cu

// 2^x, to 2^-22 of it; below 2^-126 it is 0.
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// c += a b, sixteen rows of a and eight columns of b, over sixteen.
__device__ __forceinline__ void mma_bf16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// An 8 x 8 matrix of 16-bit values, row g's values 2t and 2t + 1 in lane 4g + t, transposed.
__device__ __forceinline__ uint32_t transpose8(uint32_t a) {
    uint32_t b;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(b) : "r"(a));
    return b;
}

__device__ __forceinline__ uint32_t bf16_sub2(uint32_t a, uint32_t b) {
    const __nv_bfloat162 r = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
}
// (w & mask) | bits in one instruction: `bits` in a register that the compiler does not know the value of, or it would write two constants anew each time.
template <uint32_t MASK>
__device__ __forceinline__ uint32_t mask_or(uint32_t w, uint32_t bits) {
    uint32_t r;
    asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(r) : "r"(w), "n"(MASK), "r"(bits));
    return r;
}
__device__ __forceinline__ uint32_t bf16_128() {
    uint32_t c;
    asm volatile("mov.u32 %0, 0x43004300;" : "=r"(c));
    return c;
}
// Two 8-bit codes, in the low bytes of the halves of w, as bf16 (exactly): the low seven bits under 2^7's exponent are 128 + those bits, the sign bit
// in that pattern's last exponent bit makes 256 of 128, and the code is their difference. c128: bf16_128().
__device__ __forceinline__ uint32_t code_halves(uint32_t w, uint32_t c128) { return bf16_sub2(mask_or<0x007f007fu>(w, c128), mask_or<0x00800080u>(w, c128)); }
// Four adjacent codes as fp16 (exactly): the first and the third, the second and the fourth. A code's byte with its sign bit turned is code + 128; under 2^10's
// exponent it is 1152 + code. c1152: f16_1152(). An instruction a pair less than in bf16, whose seven bits do not hold eight.
__device__ __forceinline__ uint32_t f16_1152() {
    uint32_t c;
    asm volatile("mov.u32 %0, 0x64806480;" : "=r"(c));
    return c;
}
__device__ __forceinline__ uint32_t code_halves_f16(uint32_t w, uint32_t c1152) {
    uint32_t r;
    asm("lop3.b32 %0, %1, 0x00ff00ff, %2, 0x6a;\n\tsub.f16x2 %0, %0, %2;" : "=&r"(r) : "r"(w), "r"(c1152));
    return r;
}
__device__ __forceinline__ void codes_to_f16(uint32_t w, uint32_t c1152, uint32_t& even, uint32_t& odd) {
    even = code_halves_f16(w, c1152);
    odd = code_halves_f16(w >> 8, c1152);
}
// Two keys' codes of adjacent dimensions, bytes 2 * upper and 2 * upper + 1 of a word apiece: the keys' pair for the one, and for the other.
__device__ __forceinline__ void pair_codes_to_bf16(uint32_t a, uint32_t b, int upper, uint32_t c128, uint32_t& first, uint32_t& second) {
    const uint32_t pair = __byte_perm(a, b, upper ? 0x7632 : 0x5410);  // a's two bytes, b's two bytes
    first = code_halves(pair, c128);
    second = code_halves(pair >> 8, c128);
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
// An output once more, of the row at position p, that is no number or (`odd`) was made without some that are none: where the row sees values of that dimension that are no numbers, it
// is their sum. The products cannot have it right: 0 * NaN is not kept from the rows that do not see a key (bf16 values are taken out where there are such rows; 8-bit codes are
// numbers, and their scales a part of each row's own weights), and a weight too small for a float makes NaN of an infinity. Slow, and only for caches that hold such values.
template <bool INT8>
static __device__ __noinline__ void put_what_is_no_number(const zkb_step_attention_args& a, int64_t at, bool odd, int seq, int kv_head, int d, int64_t p) {
    const zkb_kv_cache& c = a.cache;
    const bool word = a.out_type == ZKB_VALUE_WORD;
    const uint32_t now = word ? static_cast<const uint32_t*>(a.out)[at] : static_cast<const uint16_t*>(a.out)[at];
    if (!odd && (now & 0x7f80u) != 0x7f80u) return;
    const int64_t from = seq * c.seq_stride + kv_head * c.head_stride + d, end = min(p + 1, (int64_t)c.capacity), near = a.window ? max((int64_t)0, p - (int64_t)a.window + 1) : 0;
    const float* const scale = INT8 ? c.v_scale + seq * c.scale_seq_stride + kv_head * c.scale_head_stride : nullptr;
    float y = 0.f;
    for (int part = 0; part < 2; part++) {  // first tokens, window; several loads on their way; a NaN stays one
        const int64_t to = part ? end : min(min((int64_t)a.sinks, near), end);
        for (int64_t j0 = part ? near : 0; j0 < to && y == y; j0 += 64) {
            const int64_t stop = min(j0 + 64, to);
#pragma unroll 8
            for (int64_t j = j0; j < stop; j++) {
                float x;
                if constexpr (INT8) x = (float)static_cast<const int8_t*>(c.v)[from + j * c.token_stride] * scale[j];
                else x = bf16_low(static_cast<const uint16_t*>(c.v)[from + j * c.token_stride]);
                y += isfinite(x) ? 0.f : x;
            }
        }
    }
    if (y == 0.f) return;
    if (word) static_cast<uint32_t*>(a.out)[at] = round_bf16(y);
    else static_cast<uint16_t*>(a.out)[at] = round_bf16(y);
}

// The rows of a sequence: the first of them, how many, and the first one's position. Whatever the arrays hold, the rows are within n_rows.
struct StepSequence {
    int first, rows;
    int64_t pos;
};
__device__ __forceinline__ StepSequence step_sequence(const zkb_step_rows& r, int seq) {
    const int from = r.first[seq], to = r.first[seq + 1], n = (int)r.n_rows;
    const int first = min(max(from, 0), n), rows = max(min(to, n), first) - first;
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
