// Attention of many rows: 128 query rows a tile on the tensor cores' own memory.
#include <algorithm>

#include "step_attention.cuh"

namespace zk {

// Two tiles of 128 query rows (the heads of a kv head's group, token after token) share each block of 128 keys: S = Q K^T and O += P V are tcgen05
// products whose sums lie in tensor memory, P in bf16 where S was. A thread has a row: its maximum, sum and weights need no other thread. While one tile's
// rows are in the softmax the other's products run: per block and pair, 128 x 128 head dimensions take the tensor cores 2,048 cycles and the exponentials, 16 a
// clock, as many. Warps: 0-3 and 4-7 the tiles' rows, 8 the copies, 9 the products, 10 and on what has to be done to keys and values before
// a product may read them: 8-bit codes become fp16 (K) and bf16 (V), exactly; bf16 values behind the last token or that are no numbers are zeroed where some row does not see them.
// With too few tiles for the GPU the keys are spread over a cluster's thread blocks, which add up through each other's shared memory.
constexpr int MANY_KEYS = 128, MANY_RANKS = 16;

template <int D, bool INT8>
struct Many {
    static constexpr int SIZE = INT8 ? 1 : 2;
    static constexpr int BOX = D * 2 < 128 ? D * 2 : 128, PANELS = D * 2 / BOX;  // bytes of a panel's row of 16-bit values
    static constexpr int TILE = 128 * D * 2;  // bytes of 128 rows of 16-bit values
    static constexpr int RAW_BOX = D * SIZE < 128 ? D * SIZE : 128, RAW_BOXES = D * SIZE / RAW_BOX, RAW = 128 * D * SIZE;  // as the cache has them
    static constexpr int READIERS = INT8 ? 128 : 64, THREADS = 320 + READIERS;  // threads that make ready, all
    static constexpr int STAGES = INT8 ? 3 : 5, RAWS = INT8 ? 3 : 0;
    static constexpr int RING = STAGES * TILE, RAW_RING = RAWS * RAW;
    static_assert(256 * (D + 2) * 4 <= 2 * TILE + RING + RAW_RING, "the cluster's sums lie where Q and the keys were");
    static constexpr int SMEM_USED = 2 * TILE + RING + RAW_RING;
    static constexpr int SMEM = 1024 + (SMEM_USED > 120 * 1024 ? SMEM_USED : 120 * 1024);  // one thread block an SM: it takes all of the tensor memory
    static constexpr int SWIZZLE_KIND = BOX == 128 ? 2 : 4, GROUP = 8 * BOX;  // eight rows
};

// ---- tcgen05 -----------------------------------------------------------------------------------------------------------------------------
// A matrix in shared memory for a product: its start, the strides between panels and between groups of eight rows, its swizzle.
__device__ __forceinline__ uint64_t matrix_desc(uint32_t at, int panel, int group, int swizzle_kind) {
    return (uint64_t)((at >> 4) & 0x3fff) | (uint64_t)((panel >> 4) & 0x3fff) << 16 | (uint64_t)((group >> 4) & 0x3fff) << 32 | (uint64_t)1 << 46 | (uint64_t)swizzle_kind << 61;
}
// kind::f16, sums in 32-bit floats, 128 rows: B type and A type 0 fp16, 1 bf16; b_along_n: B's rows run along N.
__host__ __device__ constexpr uint32_t product_desc(int type, int n, bool b_along_n) { return 1u << 4 | (uint32_t)type << 7 | (uint32_t)type << 10 | (uint32_t)b_along_n << 16 | (uint32_t)(n / 8) << 17 | (128u / 16) << 24; }
__device__ __forceinline__ void product_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t desc, bool add) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(desc), "r"((uint32_t)add) : "memory");
}
__device__ __forceinline__ void product_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t desc, bool add) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(desc), "r"((uint32_t)add) : "memory");
}
// The barrier gets an arrival when the products issued so far are done.
__device__ __forceinline__ void products_done(uint32_t bar) { asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory"); }
__device__ __forceinline__ void tmem_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tmem_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tmem_stored() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
#define R8(x, o) "=r"(x[o]), "=r"(x[o + 1]), "=r"(x[o + 2]), "=r"(x[o + 3]), "=r"(x[o + 4]), "=r"(x[o + 5]), "=r"(x[o + 6]), "=r"(x[o + 7])
#define W8(x, o) "r"(x[o]), "r"(x[o + 1]), "r"(x[o + 2]), "r"(x[o + 3]), "r"(x[o + 4]), "r"(x[o + 5]), "r"(x[o + 6]), "r"(x[o + 7])
// 32 columns of this thread's row; they are there after tmem_loaded, which names them so that nothing that uses them is moved before it.
#define RW8(x, o) "+r"(x[o]), "+r"(x[o + 1]), "+r"(x[o + 2]), "+r"(x[o + 3]), "+r"(x[o + 4]), "+r"(x[o + 5]), "+r"(x[o + 6]), "+r"(x[o + 7])
__device__ __forceinline__ void tmem_loaded(uint32_t (&x)[32]) { asm volatile("tcgen05.wait::ld.sync.aligned;" : RW8(x, 0), RW8(x, 8), RW8(x, 16), RW8(x, 24)::"memory"); }
__device__ __forceinline__ void tmem_loaded(uint32_t (&x)[8]) { asm volatile("tcgen05.wait::ld.sync.aligned;" : RW8(x, 0)::"memory"); }
#undef RW8
__device__ __forceinline__ void tmem_load32(uint32_t at, uint32_t* x) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
                 : R8(x, 0), R8(x, 8), R8(x, 16), R8(x, 24) : "r"(at));
}
__device__ __forceinline__ void tmem_load8(uint32_t at, uint32_t* x) { asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];" : R8(x, 0) : "r"(at)); }
__device__ __forceinline__ void tmem_store16(uint32_t at, const uint32_t* x) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(at), W8(x, 0), W8(x, 8) : "memory");
}
__device__ __forceinline__ void tmem_store8(uint32_t at, const uint32_t* x) { asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(at), W8(x, 0) : "memory"); }
#undef R8
#undef W8


// Two 32-bit floats at once, kept as their words.
__device__ __forceinline__ uint64_t two_words(uint32_t a, uint32_t b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "r"(a), "r"(b));
    return r;
}
__device__ __forceinline__ uint64_t two_floats(float a, float b) { return two_words(__float_as_uint(a), __float_as_uint(b)); }
__device__ __forceinline__ void mul2(uint32_t& x, uint32_t& y, float a, float b) {
    asm("{\n\t.reg .b64 p;\n\tmul.rn.f32x2 p, %2, %3;\n\tmov.b64 {%0, %1}, p;\n\t}" : "=r"(x), "=r"(y) : "l"(two_words(x, y)), "l"(two_floats(a, b)));
}
__device__ __forceinline__ void fma2(uint32_t& x, uint32_t& y, float by, float plus) {
    asm("{\n\t.reg .b64 p;\n\tfma.rn.f32x2 p, %2, %3, %4;\n\tmov.b64 {%0, %1}, p;\n\t}" : "=r"(x), "=r"(y) : "l"(two_words(x, y)), "l"(two_floats(by, by)), "l"(two_floats(plus, plus)));
}
__device__ __forceinline__ void add2(uint32_t& x, uint32_t& y, float a, float b) {
    asm("{\n\t.reg .b64 p;\n\tadd.rn.f32x2 p, %2, %3;\n\tmov.b64 {%0, %1}, p;\n\t}" : "=r"(x), "=r"(y) : "l"(two_words(x, y)), "l"(two_floats(a, b)));
}

struct ManyBars {
    unsigned long long full[5], ready[5], empty[5], raw_full[4], raw_empty[4], s_ready[2], p_ready[2], o_ready[2], q_ready;
};
__device__ __forceinline__ uint32_t bar_of(const unsigned long long& b) { return (uint32_t)__cvta_generic_to_shared(&b); }

// Where 16 bytes from byte `at` of row `row` of a 16-bit tile lie: panels of up to 128 bytes, each of 128 rows.
template <int D, bool INT8>
__device__ __forceinline__ uint32_t tile_place(int row, int at) {
    using M = Many<D, INT8>;
    return at / M::BOX * (128 * M::BOX) + box_place<M::BOX>(row, at % M::BOX);
}

template <int D, bool INT8, bool TMA>
__global__ void __launch_bounds__((Many<D, INT8>::THREADS), 1)
    attention_many_kernel(const __grid_constant__ zkb_step_attention_args a, const __grid_constant__ CacheMaps maps, unsigned* dev_err) {
    using M = Many<D, INT8>;
    extern __shared__ unsigned char many_sm[];
    __shared__ __align__(8) ManyBars bars;
    __shared__ __align__(16) float k_scale_sm[2][INT8 ? 128 : 1];
    __shared__ __align__(16) float v_scale_sm[2][INT8 ? 128 : 1];
    __shared__ int in_odd[MANY_RANKS];
    __shared__ int odd_sm;
    __shared__ uint32_t tmem_sm;
    unsigned char* const sm = many_sm + (-(uint32_t)__cvta_generic_to_shared(many_sm) & 1023);
    float *const in_top = reinterpret_cast<float*>(sm + 256 * D * 4), *const in_sum = in_top + 256;  // behind the sums that the cluster's thread blocks write here
    const uint32_t q_at = (uint32_t)__cvta_generic_to_shared(sm), ring = q_at + 2 * M::TILE, raw_ring = ring + M::RING;
    const zkb_kv_cache& c = a.cache;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int rank = (int)cluster_rank(), ranks = (int)cluster_ranks();
    const int seq = blockIdx.y, kv_head = (int)blockIdx.x / ranks, group = (int)(a.q_heads / c.n_heads);
    const StepSequence s = step_sequence(a.rows, seq);
    const int64_t n_m = (int64_t)s.rows * group;
    const int n_pairs = (int)((n_m + 255) / 256);
    if ((int)blockIdx.z >= n_pairs) return;  // the same for all of a cluster
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"((uint32_t)__cvta_generic_to_shared(&tmem_sm)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    } else if (warp == 1 && lane == 0) {
        for (int i = 0; i < 5; i++) mbar_init(bar_of(bars.full[i]), 1), mbar_init(bar_of(bars.ready[i]), M::READIERS), mbar_init(bar_of(bars.empty[i]), 1);
        for (int i = 0; i < 4; i++) mbar_init(bar_of(bars.raw_full[i]), 1), mbar_init(bar_of(bars.raw_empty[i]), M::READIERS);
        for (int i = 0; i < 2; i++) mbar_init(bar_of(bars.s_ready[i]), 2), mbar_init(bar_of(bars.p_ready[i]), 128), mbar_init(bar_of(bars.o_ready[i]), 1);
        mbar_init(bar_of(bars.q_ready), 256);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    const char* const k = static_cast<const char*>(c.k) + (seq * c.seq_stride + kv_head * c.head_stride) * M::SIZE;
    const char* const v = static_cast<const char*>(c.v) + (seq * c.seq_stride + kv_head * c.head_stride) * M::SIZE;
    const int64_t row_bytes = c.token_stride * M::SIZE;
    const float by = fmaxf(fabsf(a.scale) * 1.44269504f, 1.2e-38f);  // not zero: what is hidden is -inf times this
    uint32_t items = 0, blocks_done = 0, pairs_done = 0;  // of the pairs so far: what the barriers' phases count
    bool failed = false;                  // a wait ran out: what follows is not valid, and nothing more is waited for
    auto wait = [&](const unsigned long long& b, uint32_t parity) {
        if (!failed) failed = !mbar_wait(bar_of(b), parity & 1);
    };

    tmem_fence_before();
    __syncthreads();
    tmem_fence_after();
    const uint32_t tmem = tmem_sm;
    for (int pair = n_pairs - 1 - (int)blockIdx.z; pair >= 0; pair -= (int)gridDim.z) {  // the pair with the most keys first
        if (pairs_done) {  // the last pair's Q, sums and flag have been read
            tmem_fence_before();
            __syncthreads();
            tmem_fence_after();
        }
        const int64_t m0 = (int64_t)pair * 256;
        const bool two = m0 + 128 < n_m;
        const int64_t pos_low = s.pos + m0 / group, pos_high = s.pos + (min(m0 + 256, n_m) - 1) / group;
        const KeyBlocks blocks = key_blocks<MANY_KEYS>(pos_low, pos_high, c.capacity, a.window, a.sinks);
        const int last = blocks.end - 1, n = blocks.n > rank ? (blocks.n - rank + ranks - 1) / ranks : 0;  // this thread block's
        auto base_of = [&](int j) { return blocks.base(rank + j * ranks); };
        // blocks of which every row sees every key
        const int whole_to = (int)min(pos_low, (int64_t)last) - (MANY_KEYS - 1), whole_from = a.window ? (int)max((int64_t)0, pos_high - (int64_t)a.window + 1) : 0;
        const int64_t m = m0 + threadIdx.x;  // warps 0-7: this thread's row
        const bool live = warp < 8 && m < n_m;

        if (warp < 8) {  // ---- the rows: softmax
            const int tile = warp >> 2;
            const uint32_t lanes = (uint32_t)(warp & 3) << 21, s_at = tmem + tile * 128 + lanes, o_at = tmem + 256 + tile * D + lanes;
            const int p = live ? (int)(s.pos + m / group) : -1;
            const int low = a.window ? max(0, p - (int)min(a.window, 1u << 30) + 1) : 0, high = min(p, last), sinks = a.window ? (int)min(a.sinks, c.capacity) : 0;
            float top = -INFINITY, less = 0.f, sum = 0.f, by_row = by;
            {
                // Q into shared memory, its sign that of the scale; for fp16 each row times the power of two that brings its largest value to 2^13: exact
                // down to 2^-27 of that value, and below it off by 2^-38 of it.
                uint32_t w[D / 2];
                const uint16_t* from = static_cast<const uint16_t*>(a.q) + (live ? (s.first + m / group) * a.q_stride + (kv_head * group + m % group) * a.q_head_stride : 0);
                const uint32_t turn = a.scale < 0.f ? 0x80008000u : 0u;
                if (!live) {
#pragma unroll
                    for (int i = 0; i < D / 2; i++) w[i] = 0;
                } else if (aligned16(from)) {
#pragma unroll
                    for (int i = 0; i < D / 2; i += 4) {
                        const uint4 x = *reinterpret_cast<const uint4*>(from + 2 * i);
                        w[i] = x.x, w[i + 1] = x.y, w[i + 2] = x.z, w[i + 3] = x.w;
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < D / 2; i++) w[i] = (uint32_t)from[2 * i] | (uint32_t)from[2 * i + 1] << 16;
                }
                float f = 1.f;
                if constexpr (INT8) {
                    float most = 0.f;
#pragma unroll
                    for (int i = 0; i < D / 2; i++) most = fmaxf(most, fmaxf(fabsf(bf16_low(w[i])), fabsf(bf16_high(w[i]))));
                    const int e = (int)(__float_as_uint(most) >> 23), up = e == 0 || e == 255 ? 0 : min(13 + 127 - e, 126);
                    f = __uint_as_float((uint32_t)(up + 127) << 23);
                    by_row = fmaxf(ldexpf(by, -up), 1.2e-38f);
                }
#pragma unroll
                for (int i = 0; i < D / 2; i++) w[i] = (INT8 ? pack_f16(bf16_low(w[i]) * f, bf16_high(w[i]) * f) : w[i]) ^ turn;
#pragma unroll
                for (int i = 0; i < D / 2; i += 4) st_shared4(q_at + tile * M::TILE + tile_place<D, INT8>(threadIdx.x & 127, i * 4), w[i], w[i + 1], w[i + 2], w[i + 3]);
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                mbar_arrive(bar_of(bars.q_ready));
            }
            if (tile == 0 || two) {
                for (int j = 0; j < n; j++) {
                    const int base = base_of(j);
                    const uint32_t phase = blocks_done + j;
                    wait(bars.s_ready[tile], phase);
                    tmem_fence_after();
                    const bool whole = base >= whole_from && base <= whole_to;
                    // 32 scores of the row, still without the factor by_row
                    auto scores = [&](int i, uint32_t (&x)[32]) {
                        if constexpr (INT8) {
#pragma unroll
                            for (int y = 0; y < 32; y += 4) {
                                const float4 ks = *reinterpret_cast<const float4*>(&k_scale_sm[phase & 1][i + y]);
                                mul2(x[y], x[y + 1], ks.x, ks.y), mul2(x[y + 2], x[y + 3], ks.z, ks.w);
                            }
                        }
                        if (!whole) {
#pragma unroll
                            for (int y = 0; y < 32; y++)
                                if (base + i + y > high || (base + i + y < low && base + i + y >= sinks)) x[y] = 0xff800000u;  // -inf
                        }
                    };
                    uint32_t x[2][32];  // 32 scores are on their way while the 32 before them are worked on
                    float most[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
                    tmem_load32(s_at, x[0]);
#pragma unroll
                    for (int i = 0; i < 128; i += 32) {
                        tmem_loaded(x[(i / 32) & 1]);
                        tmem_load32(s_at + (i + 32) % 128, x[(i / 32 + 1) & 1]);
                        uint32_t(&y)[32] = x[(i / 32) & 1];
                        scores(i, y);
#pragma unroll
                        for (int z = 0; z < 32; z++) most[z & 3] = fmaxf(most[z & 3], __uint_as_float(y[z]));
                    }
                    const float higher = fmaxf(fmaxf(most[0], most[1]), fmaxf(most[2], most[3])) * by_row;
                    // The weights' common factor is 2^-top. It need not be the largest score's, only within 2^8 of it, so O is seldom read back for it.
                    const bool need = higher > top + 8.f;
                    if (__any_sync(0xffffffffu, need)) {
                        const float keep = need ? exp2_fast(top - higher) : 1.f;
                        if (need) top = higher, less = higher, sum *= keep;
                        if (j > 0) {
                            wait(bars.o_ready[tile], phase - 1);
                            tmem_fence_after();
#pragma unroll 1
                            for (int i = 0; i < D; i += 8) {  // few at a time: the scores keep their registers
                                uint32_t o[8];
                                tmem_load8(o_at + i, o);
                                tmem_loaded(o);
#pragma unroll
                                for (int y = 0; y < 8; y++) o[y] = __float_as_uint(__uint_as_float(o[y]) * keep);
                                tmem_store8(o_at + i, o);
                            }
                            tmem_stored();
                        }
                    }
                    uint32_t part[4] = {0u, 0u, 0u, 0u};
#pragma unroll
                    for (int i = 0; i < 128; i += 32) {  // the weights of 32 scores go where 16 scores were that have been read
                        tmem_loaded(x[(i / 32) & 1]);
                        if (i < 96) tmem_load32(s_at + i + 32, x[(i / 32 + 1) & 1]);
                        uint32_t(&y)[32] = x[(i / 32) & 1];
                        scores(i, y);
#pragma unroll
                        for (int z = 0; z < 32; z += 4) {
                            float w[4];
#pragma unroll
                            for (int e = 0; e < 4; e += 2) {
                                uint32_t u = y[z + e], v2 = y[z + e + 1];
                                fma2(u, v2, by_row, -less);
                                w[e] = exp2_fast(__uint_as_float(u)), w[e + 1] = exp2_fast(__uint_as_float(v2));
                                add2(part[e], part[e + 1], w[e], w[e + 1]);
                            }
                            if constexpr (INT8) {
                                const float4 vs = *reinterpret_cast<const float4*>(&v_scale_sm[phase & 1][i + z]);
                                w[0] *= vs.x, w[1] *= vs.y, w[2] *= vs.z, w[3] *= vs.w;
                                if (!whole)
#pragma unroll
                                    for (int e = 0; e < 4; e++)
                                        if (y[z + e] == 0xff800000u) w[e] = 0.f;  // a hidden token's scale may be anything
                            }
                            y[z / 2] = pack_bf16(w[0], w[1]), y[z / 2 + 1] = pack_bf16(w[2], w[3]);
                        }
                        tmem_store16(s_at + i / 2, y);
                    }
                    sum += (__uint_as_float(part[0]) + __uint_as_float(part[1])) + (__uint_as_float(part[2]) + __uint_as_float(part[3]));
                    tmem_stored();
                    tmem_fence_before();
                    mbar_arrive(bar_of(bars.p_ready[tile]));
                }
                if (n > 0) {
                    wait(bars.o_ready[tile], blocks_done + n - 1);
                    tmem_fence_after();
                }
            }
            // the outputs
            if (ranks == 1) {
                named_sync(1, 256 + M::READIERS);  // odd_sm: the warps that look at the values are done
                if (tile == 0 || two) {
                    const int set_aside = INT8 ? 0 : odd_sm;
                    const float inverse = sum == 0.f ? 0.f : 1.f / sum;
                    const int64_t to = live ? (s.first + m / group) * a.out_stride + (kv_head * group + m % group) * a.out_head_stride : 0;
                    const bool word = a.out_type == ZKB_VALUE_WORD, vec = aligned16(static_cast<char*>(a.out) + to * (word ? 4 : 2));
#pragma unroll 1
                    for (int i = 0; i < D; i += 8) {
                        uint32_t o[8];
                        if (n > 0) tmem_load8(o_at + i, o), tmem_loaded(o);
                        if (!live) continue;
                        float z[8];
#pragma unroll
                        for (int e = 0; e < 8; e++) z[e] = sum == 0.f || n == 0 ? 0.f : __uint_as_float(o[e]) * inverse;
                        if (set_aside)
#pragma unroll
                            for (int e = 0; e < 8; e++) z[e] += what_is_no_number(v, row_bytes, i + e, p, c.capacity, a.window, a.sinks);
                        if (word) vec ? store8<true, true>(a.out, to + i, z) : store8<true, false>(a.out, to + i, z);
                        else vec ? store8<false, true>(a.out, to + i, z) : store8<false, false>(a.out, to + i, z);
                    }
                }
            } else {
                // Each thread block finishes `part` of the rows: theirs go to [rank][four dimensions][row] of its shared memory, where Q and the keys were.
                cluster_arrive(), cluster_wait();
                const int rows_here = two ? 256 : 128, part = rows_here / ranks, row = threadIdx.x;
                if (row < rows_here) {
                    const int owner = row / part, at = row % part;
                    peer_store(&in_top[rank * part + at], owner, top);
                    peer_store(&in_sum[rank * part + at], owner, sum);
                    if (at == 0) peer_store(&in_odd[rank], owner, odd_sm);
#pragma unroll 1
                    for (int i = 0; i < D; i += 32) {
                        uint32_t o[32];
                        if (n > 0) tmem_load32(o_at + i, o), tmem_loaded(o);
#pragma unroll
                        for (int y = 0; y < 32; y += 4)
                            peer_store4(q_at + ((rank * (D / 4) + (i + y) / 4) * part + at) * 16, owner, n > 0 ? o[y] : 0u, n > 0 ? o[y + 1] : 0u, n > 0 ? o[y + 2] : 0u, n > 0 ? o[y + 3] : 0u);
                    }
                }
                cluster_arrive(), cluster_wait();
                for (int i = threadIdx.x; i < part * (D / 4); i += 256) {
                    const int at = i % part, d = i / part * 4;
                    const int64_t mm = m0 + rank * part + at;
                    if (mm >= n_m) continue;
                    float most = -INFINITY, all = 0.f, z[4] = {0.f, 0.f, 0.f, 0.f};
                    int set_aside = 0;
                    for (int x = 0; x < ranks; x++) most = fmaxf(most, in_top[x * part + at]);
                    const float least = most == -INFINITY ? 0.f : most;
                    for (int x = 0; x < ranks; x++) {
                        const float f = exp2_fast(in_top[x * part + at] - least);
                        const float4 o = *reinterpret_cast<const float4*>(sm + ((x * (D / 4) + d / 4) * part + at) * 16);
                        z[0] += o.x * f, z[1] += o.y * f, z[2] += o.z * f, z[3] += o.w * f;
                        all += in_sum[x * part + at] * f;
                        set_aside |= INT8 ? 0 : in_odd[x];
                    }
                    const int64_t to = (s.first + mm / group) * a.out_stride + (kv_head * group + mm % group) * a.out_head_stride + d;
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        z[e] = all == 0.f ? 0.f : z[e] / all;
                        if (set_aside) z[e] += what_is_no_number(v, row_bytes, d + e, s.pos + mm / group, c.capacity, a.window, a.sinks);
                        if (a.out_type == ZKB_VALUE_WORD) static_cast<uint32_t*>(a.out)[to + e] = round_bf16(z[e]);
                        else static_cast<uint16_t*>(a.out)[to + e] = round_bf16(z[e]);
                    }
                }
            }
        } else {
            if (warp == 8) {  // ---- the copies
                if (TMA && lane == 0) {
                    for (int i = 0; i < 2 * n; i++) {
                        const uint32_t item = items + i;
                        const CUtensorMap* map = i & 1 ? &maps.v : &maps.k;
                        const int base = base_of(i >> 1);
                        if constexpr (INT8) {
                            const uint32_t st = item % M::RAWS, bar = bar_of(bars.raw_full[st]);
                            wait(bars.raw_empty[st], item / M::RAWS + 1);
                            if (failed) break;
                            mbar_expect(bar, M::RAW);
#pragma unroll
                            for (int x = 0; x < M::RAW_BOXES; x++) tma_load(raw_ring + st * M::RAW + x * 128 * M::RAW_BOX, map, x * M::RAW_BOX, base, kv_head, seq, bar);
                        } else {
                            const uint32_t st = item % M::STAGES, bar = bar_of(bars.full[st]);
                            wait(bars.empty[st], item / M::STAGES + 1);
                            if (failed) break;
                            mbar_expect(bar, M::TILE);
#pragma unroll
                            for (int x = 0; x < M::PANELS; x++) tma_load(ring + st * M::TILE + x * 128 * M::BOX, map, x * (M::BOX / 2), base, kv_head, seq, bar);
                        }
                    }
                }
            } else if (warp == 9) {  // ---- the products
                // One tile's after the other's, so that one tile's rows are in the softmax while the other's products run. (Each tile's from a warp of its
                // own, both were in the softmax and then in their products at the same time: 6,100 cycles a block and pair.)
                if (lane == 0) {
                    constexpr uint32_t qk = product_desc(INT8 ? 0 : 1, MANY_KEYS, false), pv = product_desc(1, D, true);
                    auto scores = [&](int tile, uint32_t st) {
#pragma unroll
                        for (int i = 0; i < D / 16; i++) {
                            const uint32_t at = i / (M::BOX / 32) * (128 * M::BOX) + i % (M::BOX / 32) * 32;
                            product_ss(tmem + tile * 128, matrix_desc(q_at + tile * M::TILE + at, 16, M::GROUP, M::SWIZZLE_KIND), matrix_desc(ring + st * M::TILE + at, 16, M::GROUP, M::SWIZZLE_KIND), qk, i > 0);
                        }
                        products_done(bar_of(bars.s_ready[tile]));
                        mbar_arrive(bar_of(bars.s_ready[tile]));
                    };
                    const int tiles = two ? 2 : 1;
                    wait(bars.q_ready, pairs_done);
                    for (int j = -1; j < n && !failed; j++) {
                        const uint32_t v_item = items + 2 * j + 1, vs = v_item % M::STAGES, k_item = v_item + 1, ks = k_item % M::STAGES, phase = blocks_done + j;
                        for (int tile = 0; tile < tiles; tile++) {
                            if (j >= 0) {
                                wait(bars.p_ready[tile], phase);
                                if (tile == 0) wait(bars.ready[vs], v_item / M::STAGES);
                                if (failed) break;
                                tmem_fence_after();
#pragma unroll
                                for (int i = 0; i < MANY_KEYS / 16; i++)
                                    product_ts(tmem + 256 + tile * D, tmem + tile * 128 + 8 * i, matrix_desc(ring + vs * M::TILE + i * 2 * M::GROUP, 128 * M::BOX, M::GROUP, M::SWIZZLE_KIND), pv, j > 0 || i > 0);
                                products_done(bar_of(bars.o_ready[tile]));
                                if (tile == tiles - 1) products_done(bar_of(bars.empty[vs]));
                            }
                            if (j + 1 < n) {
                                if (tile == 0) wait(bars.ready[ks], k_item / M::STAGES);
                                if (j >= 0) wait(bars.o_ready[tile], phase);  // P has been read where S goes
                                if (failed) break;
                                tmem_fence_after();
                                scores(tile, ks);
                                if (tile == tiles - 1) products_done(bar_of(bars.empty[ks]));
                            }
                        }
                    }
                }
            } else {  // ---- what the products read is made ready
                const int th = threadIdx.x - 320;
                const uint32_t c128 = bf16_128(), c1152 = f16_1152();
                bool odd = false;
                if (th == 0) odd_sm = 0;
                named_sync(2, M::READIERS);
                for (int i = 0; i < 2 * n; i++) {
                    const uint32_t item = items + i, st = item % M::STAGES, to = ring + st * M::TILE;
                    const int base = base_of(i >> 1), kv = i & 1;
                    const bool whole = base >= whole_from && base <= whole_to;
                    if constexpr (INT8) {
                        wait(bars.empty[st], item / M::STAGES + 1);
                        if (kv == 0) {  // both of the block's scales: of the block before the last, nothing is needed any more when this place is free
                            const int key = min(base + th, last), slot = (blocks_done + (i >> 1)) & 1;
                            k_scale_sm[slot][th] = c.k_scale[seq * c.scale_seq_stride + kv_head * c.scale_head_stride + key];
                            v_scale_sm[slot][th] = c.v_scale[seq * c.scale_seq_stride + kv_head * c.scale_head_stride + key];
                        }
                        const uint32_t rs = item % M::RAWS, raw = raw_ring + rs * M::RAW;
                        if constexpr (TMA) wait(bars.raw_full[rs], item / M::RAWS);
#pragma unroll 2
                        for (int x = th; x < M::RAW / 16; x += M::READIERS) {
                            const int row = x / (D / 16), at = x % (D / 16) * 16;
                            uint32_t w[4], h[8];
                            if constexpr (TMA) {
                                ld_shared4(raw + box_place<M::RAW_BOX>(row, at), w[0], w[1], w[2], w[3]);
                            } else {
                                const uint8_t* from = reinterpret_cast<const uint8_t*>((kv ? v : k) + min(base + row, last) * row_bytes + at);
#pragma unroll
                                for (int y = 0; y < 4; y++) w[y] = (uint32_t)from[4 * y] | (uint32_t)from[4 * y + 1] << 8 | (uint32_t)from[4 * y + 2] << 16 | (uint32_t)from[4 * y + 3] << 24;
                            }
#pragma unroll
                            for (int y = 0; y < 4; y++) {
                                if (kv) h[2 * y] = code_halves(__byte_perm(w[y], 0, 0x4140), c128), h[2 * y + 1] = code_halves(__byte_perm(w[y], 0, 0x4342), c128);
                                else h[2 * y] = code_halves_f16(__byte_perm(w[y], 0, 0x4140), c1152), h[2 * y + 1] = code_halves_f16(__byte_perm(w[y], 0, 0x4342), c1152);
                            }
                            st_shared4(to + tile_place<D, INT8>(row, 2 * at), h[0], h[1], h[2], h[3]);
                            st_shared4(to + tile_place<D, INT8>(row, 2 * at + 16), h[4], h[5], h[6], h[7]);
                        }
                        if constexpr (TMA) mbar_arrive(bar_of(bars.raw_empty[rs]));
                        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    } else {
                        if constexpr (TMA) wait(bars.full[st], item / M::STAGES);
                        else wait(bars.empty[st], item / M::STAGES + 1);
                        if (!TMA || (kv && !whole)) {
                            for (int x = th; x < M::TILE / 16; x += M::READIERS) {
                                const int row = x / (D / 8), at = x % (D / 8) * 16;
                                const uint32_t place = to + tile_place<D, INT8>(row, at);
                                uint32_t w[4], test = 0;
                                if constexpr (TMA) {
                                    ld_shared4(place, w[0], w[1], w[2], w[3]);
                                } else {
                                    const uint16_t* from = reinterpret_cast<const uint16_t*>((kv ? v : k) + min(base + row, last) * row_bytes + at);
#pragma unroll
                                    for (int y = 0; y < 4; y++) w[y] = (uint32_t)from[2 * y] | (uint32_t)from[2 * y + 1] << 16;
                                }
                                if (kv && !whole) {
                                    if (base + row > last) {  // behind the last token the cache may hold anything
                                        w[0] = w[1] = w[2] = w[3] = 0;
                                        if (TMA) st_shared4(place, 0u, 0u, 0u, 0u);
                                    }
#pragma unroll
                                    for (int y = 0; y < 4; y++) test = zero_or_nan(w[y], test);
                                    if (test & 0x7fff7fffu) {  // what is no number would reach the rows that do not see its key: it is set aside (what_is_no_number)
                                        odd = true;
#pragma unroll
                                        for (int y = 0; y < 4; y++) w[y] = numbers_only(w[y]);
                                        if (TMA) st_shared4(place, w[0], w[1], w[2], w[3]);
                                    }
                                }
                                if (!TMA) st_shared4(place, w[0], w[1], w[2], w[3]);
                            }
                            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                        }
                    }
                    mbar_arrive(bar_of(bars.ready[st]));
                }
                if (odd) odd_sm = 1;
                if (ranks == 1) named_sync(1, 256 + M::READIERS);
            }
            __syncwarp();
            if (ranks > 1) {
                cluster_arrive(), cluster_wait();
                cluster_arrive(), cluster_wait();
            }
        }
        items += 2 * n;
        blocks_done += n;
        pairs_done++;
        if (failed && lane == 0) *dev_err = WAIT_RAN_OUT;
        if (ranks > 1 && pair >= (int)gridDim.z) {  // the next pair's Q goes where the sums came
            __syncwarp();
            cluster_arrive(), cluster_wait();
        }
    }
    tmem_fence_before();
    __syncthreads();
    if (warp == 0) {
        tmem_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem_sm));
    }
}

template <int D, bool INT8>
cudaError_t launch_many(zkb_ctx* ctx, const zkb_step_attention_args& a) {
    using M = Many<D, INT8>;
    const zkb_kv_cache& c = a.cache;
    const uint32_t group = a.q_heads / c.n_heads, most = a.rows.max_rows ? std::min(a.rows.max_rows, a.rows.n_rows) : a.rows.n_rows;
    const uint32_t pairs = (uint32_t)std::min<uint64_t>(((uint64_t)most * group + 255) / 256, 65535);
    uint64_t len = a.rows.max_len ? std::min(a.rows.max_len, c.capacity) : c.capacity;
    if (a.window) len = std::min<uint64_t>(len, (uint64_t)a.window + a.sinks + 2 * MANY_KEYS);
    // Spread the keys over clusters of as many thread blocks as still are on the GPU all at once.
    const uint64_t units = (uint64_t)c.n_seqs * c.n_heads * pairs;
    uint32_t ranks = 1;
    while (ranks < MANY_RANKS && units <= clusters_at_once(2 * ranks) && len > (uint64_t)ranks * MANY_KEYS) ranks *= 2;
    CacheMaps maps;
    const bool tma = cache_maps(maps, c, MANY_KEYS);
    auto kernel = tma ? attention_many_kernel<D, INT8, true> : attention_many_kernel<D, INT8, false>;
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, M::SMEM);
    if (e != cudaSuccess) return e;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim = {ranks, 1, 1};
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(c.n_heads * ranks, c.n_seqs, pairs);
    cfg.blockDim = dim3(M::THREADS);
    cfg.dynamicSmemBytes = M::SMEM;
    cfg.stream = ctx->stream;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, a, maps, ctx->dev_err);
}
template cudaError_t launch_many<32, false>(zkb_ctx*, const zkb_step_attention_args&);
template cudaError_t launch_many<64, false>(zkb_ctx*, const zkb_step_attention_args&);
template cudaError_t launch_many<128, false>(zkb_ctx*, const zkb_step_attention_args&);
template cudaError_t launch_many<32, true>(zkb_ctx*, const zkb_step_attention_args&);
template cudaError_t launch_many<64, true>(zkb_ctx*, const zkb_step_attention_args&);
template cudaError_t launch_many<128, true>(zkb_ctx*, const zkb_step_attention_args&);

}  // namespace zk
