// Attention of many rows: 128 query rows a tile on the tensor cores' own memory.
#include <algorithm>

#include "step_attention.cuh"

namespace zk {

// Two tiles of 128 query rows (the heads of a kv head's group, token after token) share each block of 128 keys: S = Q K^T and O += P V are tcgen05
// products whose sums lie in tensor memory, P in bf16 where S was. A thread has a row: its maximum, sum and weights need no other thread. While one tile's
// rows are in the softmax the other's products run: per block and pair the tensor cores need 2,048 cycles for 128 head dimensions and the exponentials, 16 a clock, as many.
// Warps: 0-3 and 4-7 the tiles' rows, 8 the copies, 9 the products, 10 and on what has to be done to keys and values before a product may read them: 8-bit codes become
// fp16 (K) and bf16 (V), exactly; bf16 values behind the last token or that are no numbers are zeroed where some row does not see them.
// A thread block takes one pair of tiles after the other; with too few of them for the GPU the keys are spread over a cluster's thread blocks, which add up through
// each other's shared memory, and one tile alone is two, of each block's two halves.
// The weights are rounded to bf16 for the product (2^-8, as the result's own rounding): a second bf16 number for what that leaves, as the few rows' kernel has it, took 15 to 28 % longer.
// 32 heads on 8 of 128, causal, call after call: 8,192 rows of one sequence, bf16, 513 us, 1,070 TFLOP/s of visible pairs; 1,290 to 2,048 rows of four sequences 150 us, int8 245 us; 8,192 rows
// with a window of 1,024, bf16 200 us, int8 320 us: a block's products and its softmax take turns, 1,500 and 2,200 cycles, int8 scales another 2,000 of shared memory's. The three bf16 times
// are 2 us for each block of 128 keys and pair of tiles, and some 10 us for each pair whatever its keys (its Q, the first scores, the rows written), which nothing hides: both tiles are at it at once.
constexpr int MANY_KEYS = 128, MANY_RANKS = 16;

template <int D, bool INT8>
struct Many {
    static constexpr int SIZE = INT8 ? 1 : 2;
    static constexpr int BOX = D * 2 < 128 ? D * 2 : 128, PANELS = D * 2 / BOX;  // bytes of a panel's row of 16-bit values
    static constexpr int TILE = 128 * D * 2;  // bytes of 128 rows of 16-bit values
    static constexpr int RAW_BOX = D * SIZE < 128 ? D * SIZE : 128, RAW_BOXES = D * SIZE / RAW_BOX, RAW = 128 * D * SIZE;  // as the cache has them
    static constexpr int READIERS = INT8 ? 192 : 64, THREADS = 320 + READIERS;  // threads that make ready, all
    static constexpr int STAGES = INT8 ? 3 : 4, RAWS = INT8 ? 3 : 0;
    static constexpr int RING = STAGES * TILE, RAW_RING = RAWS * RAW;
    static_assert(256 * (D + 2) * 4 <= 2 * TILE + RING + RAW_RING, "the cluster's sums lie where Q and the keys were");
    static constexpr int SMEM_USED = 2 * TILE + RING + RAW_RING;
    static constexpr int SMEM = 1024 + (SMEM_USED > 120 * 1024 ? SMEM_USED : 120 * 1024);  // one thread block an SM: it takes all of the tensor memory
    static constexpr int SWIZZLE_KIND = BOX == 128 ? 2 : 4, GROUP = 8 * BOX;  // eight rows
};

// ---- tcgen05 -----------------------------------------------------------------------------------------------------------------------------
// A matrix in shared memory is described by 64 bits: its start and the stride between panels in the lower half, in 16 bytes; the stride between groups of eight rows and
// its swizzle (2: 128 bytes, 4: 64) in the upper.
// kind::f16, sums in 32-bit floats, 128 rows: B type and A type 0 fp16, 1 bf16; b_along_n: B's rows run along N.
__host__ __device__ constexpr uint32_t product_desc(int type, int n, bool b_along_n) { return 1u << 4 | (uint32_t)type << 7 | (uint32_t)type << 10 | (uint32_t)b_along_n << 16 | (uint32_t)(n / 8) << 17 | (128u / 16) << 24; }
// (Called by a whole warp; one lane issues. What the lanes have in common is then in uniform registers, where the instruction wants it.)
__device__ __forceinline__ void product_ss(bool one, uint32_t d, uint64_t a, uint64_t b, uint32_t desc, bool add) {
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(desc), "r"((uint32_t)add),
                 "r"((uint32_t)one)
                 : "memory");
}
__device__ __forceinline__ void product_ts(bool one, uint32_t d, uint32_t a, uint64_t b, uint32_t desc, bool add) {
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(desc), "r"((uint32_t)add),
                 "r"((uint32_t)one)
                 : "memory");
}
// The barrier gets an arrival when the products issued so far are done.
__device__ __forceinline__ void products_done(uint32_t bar) { asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory"); }
__device__ __forceinline__ bool elect_one() {
    uint32_t one;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(one));
    return one;
}
__device__ __forceinline__ void tmem_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tmem_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tmem_stored() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
#define R8(x, o) "=r"(x[o]), "=r"(x[o + 1]), "=r"(x[o + 2]), "=r"(x[o + 3]), "=r"(x[o + 4]), "=r"(x[o + 5]), "=r"(x[o + 6]), "=r"(x[o + 7])
#define W8(x, o) "r"(x[o]), "r"(x[o + 1]), "r"(x[o + 2]), "r"(x[o + 3]), "r"(x[o + 4]), "r"(x[o + 5]), "r"(x[o + 6]), "r"(x[o + 7])
// 32 or 8 columns of this thread's row; they are there after tmem_loaded, which names them so that nothing that uses them is moved before it.
#define RW8(x, o) "+r"(x[o]), "+r"(x[o + 1]), "+r"(x[o + 2]), "+r"(x[o + 3]), "+r"(x[o + 4]), "+r"(x[o + 5]), "+r"(x[o + 6]), "+r"(x[o + 7])
__device__ __forceinline__ void tmem_loaded(uint32_t (&x)[32]) { asm volatile("tcgen05.wait::ld.sync.aligned;" : RW8(x, 0), RW8(x, 8), RW8(x, 16), RW8(x, 24)::"memory"); }
__device__ __forceinline__ void tmem_loaded(uint32_t (&x)[8]) { asm volatile("tcgen05.wait::ld.sync.aligned;" : RW8(x, 0)::"memory"); }
#undef RW8
__device__ __forceinline__ void tmem_load32(uint32_t at, uint32_t* x) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
                 : R8(x, 0), R8(x, 8), R8(x, 16), R8(x, 24) : "r"(at));
}
__device__ __forceinline__ void tmem_load8(uint32_t at, uint32_t* x) { asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];" : R8(x, 0) : "r"(at)); }
__device__ __forceinline__ void tmem_store32(uint32_t at, const uint32_t* x) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(at),
                 W8(x, 0), W8(x, 8), W8(x, 16), W8(x, 24) : "memory");
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
__device__ __forceinline__ void scale2(float& x, float& y, float a, float b) {
    uint32_t u = __float_as_uint(x), v = __float_as_uint(y);
    mul2(u, v, a, b);
    x = __uint_as_float(u), y = __uint_as_float(v);
}
__device__ __forceinline__ void fma2(uint32_t& x, uint32_t& y, float by, float plus) {
    asm("{\n\t.reg .b64 p;\n\tfma.rn.f32x2 p, %2, %3, %4;\n\tmov.b64 {%0, %1}, p;\n\t}" : "=r"(x), "=r"(y) : "l"(two_words(x, y)), "l"(two_floats(by, by)), "l"(two_floats(plus, plus)));
}
__device__ __forceinline__ void add2(uint32_t& x, uint32_t& y, float a, float b) {
    asm("{\n\t.reg .b64 p;\n\tadd.rn.f32x2 p, %2, %3;\n\tmov.b64 {%0, %1}, p;\n\t}" : "=r"(x), "=r"(y) : "l"(two_words(x, y)), "l"(two_floats(a, b)));
}

// 32 bytes, on a 32-byte boundary: a whole sector at once.
__device__ __forceinline__ void store32(void* to, const uint32_t (&x)[8]) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(to), "r"(x[0]), "r"(x[1]), "r"(x[2]), "r"(x[3]), "r"(x[4]), "r"(x[5]), "r"(x[6]), "r"(x[7]) : "memory");
}
// 2^n of a whole number n up to zero, exactly; below 2^-126 it is 0.
__device__ __forceinline__ float power_of_2(float n) { return n < -126.f ? 0.f : __uint_as_float((uint32_t)((int)n + 127) << 23); }
// The lowest n bits.
__device__ __forceinline__ uint32_t bits_below(int n) { return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1u; }

struct ManyBars {
    unsigned long long full[5], ready[5], empty[5], raw_full[4], raw_empty[4], s_ready[2], p_ready[2], o_ready[2], q_ready[2];
};
__device__ __forceinline__ uint32_t bar_of(const unsigned long long& b) { return (uint32_t)__cvta_generic_to_shared(&b); }

// Where 16 bytes from byte `at` of row `row` of a 16-bit tile lie: panels of up to 128 bytes, each of 128 rows.
template <int D, bool INT8>
__device__ __forceinline__ uint32_t tile_place(int row, int at) {
    using M = Many<D, INT8>;
    return at / M::BOX * (128 * M::BOX) + box_place<M::BOX>(row, at % M::BOX);
}

// Two tiles of one sequence's rows and one kv head, and the blocks of keys that this thread block has for them. With one tile only, both can work on it, each on a
// half of every block (split): their sums are joined as those of a cluster's thread blocks are.
struct Unit {
    StepSequence s;
    KeyBlocks blocks;
    int seq, kv_head, n_m, m0, last, n, whole_from, whole_to;
    bool two, split;
};
// All units of a thread block, the ones with the most keys first: pair after pair from the last tokens on, in each all sequences and heads.
struct Units {
    const zkb_step_attention_args& a;
    uint32_t turn, all, depth;  // `depth`: pairs of a sequence that are units of their own
    int rank, ranks, pair;
    uint32_t one;  // sequence and head whose pairs are in turn: the next unit may be another pair of the same
    __device__ Units(const zkb_step_attention_args& args, uint32_t pairs)
        : a(args), turn(0), all(pairs * args.cache.n_seqs * args.cache.n_heads), depth(pairs), rank((int)cluster_rank()),
          ranks((int)cluster_ranks()), pair(-1), one(0) {}
    __device__ bool next(Unit& u) {
        const zkb_kv_cache& c = a.cache;
        const int group = (int)(a.q_heads / c.n_heads);
        auto take = [&] {
            u.seq = (int)(one / c.n_heads), u.kv_head = (int)(one % c.n_heads);
            u.s = step_sequence(a.rows, u.seq);
            u.n_m = u.s.rows * group;
        };
        pair -= (int)depth;
        if (pair >= 0) take();  // sequences of more pairs than the host knew of
        while (pair < 0) {
            // there and back, so that all get as much
            const uint32_t who = blockIdx.x / ranks, step = gridDim.x / ranks, at = turn * step + (turn & 1 ? step - 1 - who : who);
            if (turn * step >= all) return false;
            turn++;
            if (at >= all) continue;
            one = at % (c.n_seqs * c.n_heads);
            take();
            pair = (u.n_m + 255) / 256 - 1 - (int)(at / (c.n_seqs * c.n_heads));
        }
        u.m0 = pair * 256;
        u.two = u.m0 + 128 < u.n_m;
        const int64_t low = u.s.pos + (uint32_t)u.m0 / (uint32_t)group, high = u.s.pos + (uint32_t)(min(u.m0 + 256, u.n_m) - 1) / (uint32_t)group;
        u.blocks = key_blocks<MANY_KEYS>(low, high, c.capacity, a.window, a.sinks);
        u.last = u.blocks.end - 1;
        u.n = u.blocks.n > rank ? (u.blocks.n - rank + ranks - 1) / ranks : 0;
        u.split = !u.two && (ranks > 1 || u.blocks.n > 2);
        // keys that every row sees
        u.whole_to = (int)min(low, (int64_t)u.last), u.whole_from = a.window ? (int)max((int64_t)0, high - (int64_t)a.window + 1) : 0;
        return true;
    }
    __device__ __forceinline__ int base(const Unit& u, int j) const { return u.blocks.base(rank + j * ranks); }
    __device__ __forceinline__ bool whole(const Unit& u, int base, int keys) const { return base >= u.whole_from && base + keys - 1 <= u.whole_to; }
    __device__ __forceinline__ bool joined(const Unit& u) const { return ranks > 1 || u.split; }
};

template <int D, bool INT8, bool TMA>
__global__ void __launch_bounds__((Many<D, INT8>::THREADS), 1)
    attention_many_kernel(const __grid_constant__ zkb_step_attention_args a, const __grid_constant__ CacheMaps maps, uint32_t pairs, unsigned* dev_err) {
    using M = Many<D, INT8>;
    extern __shared__ unsigned char many_sm[];
    __shared__ __align__(8) ManyBars bars;
    __shared__ __align__(16) float k_scale_sm[2][INT8 ? 128 : 1];
    __shared__ __align__(16) float v_scale_sm[2][INT8 ? 128 : 1];
    __shared__ int in_odd[MANY_RANKS];
    __shared__ int odd_sm[8];  // some value was no number: of the units in turn (what makes ready runs a few units ahead)
    __shared__ int slow_sm;  // threads that add up what is no number, which takes as long as the cache is
    __shared__ uint32_t tmem_sm;
    unsigned char* const sm = many_sm + (-(uint32_t)__cvta_generic_to_shared(many_sm) & 1023);
    float *const in_top = reinterpret_cast<float*>(sm + 256 * D * 4), *const in_sum = in_top + 256;  // behind the sums that are joined, where Q and the keys were
    const uint32_t q_at = (uint32_t)__cvta_generic_to_shared(sm), ring = q_at + 2 * M::TILE, raw_ring = ring + M::RING;
    const zkb_kv_cache& c = a.cache;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, group = (int)(a.q_heads / c.n_heads);
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"((uint32_t)__cvta_generic_to_shared(&tmem_sm)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    } else if (warp == 1 && lane == 0) {
        for (int i = 0; i < 5; i++) mbar_init(bar_of(bars.full[i]), 1), mbar_init(bar_of(bars.ready[i]), M::READIERS), mbar_init(bar_of(bars.empty[i]), 1);
        for (int i = 0; i < 4; i++) mbar_init(bar_of(bars.raw_full[i]), 1), mbar_init(bar_of(bars.raw_empty[i]), M::READIERS);
        for (int i = 0; i < 2; i++) mbar_init(bar_of(bars.s_ready[i]), 2), mbar_init(bar_of(bars.p_ready[i]), 128), mbar_init(bar_of(bars.o_ready[i]), 1), mbar_init(bar_of(bars.q_ready[i]), 128);
        slow_sm = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    const int64_t row_bytes = c.token_stride * M::SIZE;
    bool failed = false;  // a wait ran out: what follows is not valid, and nothing more is waited for
    auto wait_one = [&](const unsigned long long& b, uint32_t parity) {
        if (!failed && !mbar_test(bar_of(b), parity & 1)) {
            int tries = 0;
#pragma unroll 1
            do tries = *static_cast<volatile int*>(&slow_sm) ? 0 : tries + 1;  // counted while there is no reason to wait
            while (!mbar_test(bar_of(b), parity & 1) && tries < (1 << 20));
            failed = tries >= 1 << 20;
        }
    };
    auto wait = [&](const unsigned long long& b, uint32_t parity) {  // a whole warp: what follows may be an instruction that wants its lanes together
        wait_one(b, parity);
        failed = __any_sync(0xffffffffu, failed);
    };
    tmem_fence_before();
    __syncthreads();
    tmem_fence_after();
    const uint32_t tmem = tmem_sm;
    Units units(a, pairs);
    auto meet = [&] {  // all of this thread block's threads, or the cluster's
        tmem_fence_before();
        if (units.ranks > 1) cluster_arrive(), cluster_wait();
        else __syncthreads();
        tmem_fence_after();
    };
    Unit u, after;
    bool more = units.next(u);

    if (warp < 8) {  // ---- the rows: softmax
        // An int8 cache takes more threads than leave a row the registers for 64 scores: they get some of those of the other warps (256 * 184 + 256 * 72 = 512 * 128, what the
        // launch has). 8192 rows, window of 1024, int8: 367 -> 331 us when it was
        // tried. -Xptxas -v: the int8 variants keep 72 to 88 bytes of stack and 288 to 354 of spill stores, the bf16 ones (168 registers) 32 to 40 and 42 to 56.
        if constexpr (INT8) asm volatile("setmaxnreg.inc.sync.aligned.u32 184;");
        const int tile = warp >> 2, row = threadIdx.x & 127;
        const uint32_t lanes = (uint32_t)(warp & 3) << 21, s_at = tmem + tile * 128 + lanes, o_at = tmem + 256 + tile * D + lanes;
        const float by = fmaxf(fabsf(a.scale) * 1.44269504f, 1.4e-45f);  // not zero, but the smallest float: what is hidden is -inf times this
        uint32_t done = 0, passed = 0, odd_at = 0;  // steps of this tile, blocks, units with blocks: what the barriers' phases, the scales' places and the flags go by
        auto row_of = [&](const Unit& n) { return n.m0 + (n.split ? row : tile * 128 + row); };
        auto q_of = [&](const Unit& n, int m) {
            const uint32_t i = (uint32_t)m / (uint32_t)group;
            return static_cast<const uint16_t*>(a.q) + (n.s.first + (int)i) * a.q_stride + (n.kv_head * group + m - (int)i * group) * a.q_head_stride;
        };
        // This thread's row of Q into shared memory, its sign that of the scale; for fp16 each row times the power of two that brings its largest value
        // to 2^13: exact down to 2^-27 of that value, and below it off by 2^-38 of it. The factor that is left for the row's scores.
        auto load_q = [&](const Unit& n) {
            const int m = row_of(n);
            const bool live = m < n.n_m;
            const uint16_t* from = q_of(n, live ? m : 0);
            const bool vec = aligned16(from);
            uint4 x[D / 8];  // all loads on their way at once
#pragma unroll
            for (int i = 0; i < D / 8; i++) {
                x[i] = make_uint4(0u, 0u, 0u, 0u);
                const uint16_t* const p = from + 8 * i;
                if (live && vec) x[i] = *reinterpret_cast<const uint4*>(p);
                else if (live) x[i] = make_uint4((uint32_t)p[0] | (uint32_t)p[1] << 16, (uint32_t)p[2] | (uint32_t)p[3] << 16, (uint32_t)p[4] | (uint32_t)p[5] << 16, (uint32_t)p[6] | (uint32_t)p[7] << 16);
            }
            float f = 1.f, left = by;
            if constexpr (INT8) {
                float most = 0.f;
#pragma unroll
                for (int i = 0; i < D / 8; i++)
                    for (uint32_t w : {x[i].x, x[i].y, x[i].z, x[i].w}) most = fmaxf(most, fmaxf(fabsf(bf16_low(w)), fabsf(bf16_high(w))));
                const int e = (int)(__float_as_uint(most) >> 23), up = e == 0 || e == 255 ? 0 : min(13 + 127 - e, 126);
                f = __uint_as_float((uint32_t)(up + 127) << 23);
                left = fmaxf(ldexpf(by, -up), 1.4e-45f);
            }
            const uint32_t turn = a.scale < 0.f ? 0x80008000u : 0u;
            auto word = [&](uint32_t w) { return (INT8 ? pack_f16(bf16_low(w) * f, bf16_high(w) * f) : w) ^ turn; };
#pragma unroll
            for (int i = 0; i < D / 8; i++)
                st_shared4(q_at + tile * M::TILE + tile_place<D, INT8>(row, i * 16), word(x[i].x), word(x[i].y), word(x[i].z), word(x[i].w));
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            mbar_arrive(bar_of(bars.q_ready[tile]));
            return left;
        };
        auto sums_place = [](int row, int four) { return (row * (D / 4) + (four ^ (row & 7))) * 16; };
        // Q of a unit that this tile has products in: no other keeps it from announcing the next one's too soon.
        auto works = [&](const Unit& n) { return n.n > 0 && (tile == 0 || n.two || n.split); };
        float by_row = more && works(u) ? load_q(u) : 0.f;
        while (more) {
            const int m = row_of(u);  // this thread's row
            const bool live = m < u.n_m;
            const int p = live ? (int)u.s.pos + (int)((uint32_t)m / (uint32_t)group) : -1;
            const int low = a.window ? (int)max((int64_t)0, (int64_t)p - (int64_t)a.window + 1) : 0, high = min(p, u.last), sinks = a.window ? (int)min(a.sinks, c.capacity) : 0;
            const bool again = units.next(after);
            if (again) {  // the next unit's Q comes nearer
                const int mm = row_of(after);
                if (mm < after.n_m)
                    for (int i = 0; i < D; i += 64) asm volatile("prefetch.global.L2 [%0];" ::"l"(q_of(after, mm) + i));
            }
            float top = -INFINITY, less = 0.f, sum = 0.f;
            const int steps = u.split || tile == 0 || u.two ? u.n : 0, half = u.split ? 64 * tile : 0, keys = u.split ? 64 : 128;
            for (int j = 0; j < steps; j++, done++) {
                const int base = units.base(u, j) + half, slot = (passed + j) & 1;
                const bool whole = units.whole(u, base, keys);
                wait(bars.s_ready[tile], done);
                tmem_fence_after();
                uint32_t part[4] = {0u, 0u, 0u, 0u};
                // 64 scores at a time become weights that go where scores were that have been read. The weights' common factor is 2^-top, which need not be the largest
                // score's: it is left as it is until a score exceeds it by 2^8, so that one pass over the scores will do. Where weights of this block have
                // been rounded already it changes by a whole power of two, so that they are not rounded again, and else to the largest score, whose weight then is exact.
                // (Weights added up after their rounding would be exact relative to their sum wherever one score is far above: 4 to 9 % slower, the error of such rows 2^-9.4 instead of 2^-9.)
#pragma unroll 1
                for (int at = 0; at < keys; at += 64) {
                    uint32_t x[64];
                    uint32_t(&x0)[32] = *reinterpret_cast<uint32_t(*)[32]>(&x[0]), (&x1)[32] = *reinterpret_cast<uint32_t(*)[32]>(&x[32]);
                    tmem_load32(s_at + at, x0);
                    tmem_load32(s_at + at + 32, x1);
                    tmem_loaded(x0);
                    tmem_loaded(x1);
                    if constexpr (INT8) {
#pragma unroll
                        for (int y = 0; y < 64; y += 4) {
                            const float4 ks = *reinterpret_cast<const float4*>(&k_scale_sm[slot][half + at + y]);
                            mul2(x[y], x[y + 1], ks.x, ks.y), mul2(x[y + 2], x[y + 3], ks.z, ks.w);
                        }
                    }
                    uint32_t seen[2] = {0xffffffffu, 0xffffffffu};
                    if (!whole) {
#pragma unroll
                        for (int i = 0; i < 2; i++) {
                            const int first = base + at + 32 * i;
                            seen[i] = bits_below(high + 1 - first) & (~bits_below(low - first) | bits_below(sinks - first));
#pragma unroll
                            for (int y = 0; y < 32; y++) x[32 * i + y] = seen[i] >> y & 1 ? x[32 * i + y] : 0xff800000u;  // -inf
                        }
                    }
                    float most[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                    for (int z = 0; z < 64; z++) most[z & 3] = fmaxf(most[z & 3], __uint_as_float(x[z]));
                    const float higher = fmaxf(fmaxf(most[0], most[1]), fmaxf(most[2], most[3])) * by_row;
                    const bool need = higher > top + 8.f;
                    if (__any_sync(0xffffffffu, need)) {
                        const bool steps = at != 0 && top > -INFINITY;
                        const float up = steps ? ceilf(higher - top) : higher - top, keep = need ? at ? power_of_2(-up) : exp2_fast(-up) : 1.f;
                        if (need) top = steps ? top + up : higher, less = top, sum *= keep;
#pragma unroll
                        for (int e = 0; e < 4; e++) part[e] = __float_as_uint(__uint_as_float(part[e]) * keep);
                        __syncwarp();
                        tmem_stored();
#pragma unroll 1
                        for (int i = 0; i < at / 2; i += 8) {  // this block's weights so far
                            uint32_t w[8];
                            tmem_load8(s_at + i, w);
                            tmem_loaded(w);
#pragma unroll
                            for (int y = 0; y < 8; y++) w[y] = pack_bf16(bf16_low(w[y]) * keep, bf16_high(w[y]) * keep);
                            tmem_store8(s_at + i, w);
                        }
                        if (j > 0) {
                            wait(bars.o_ready[tile], done - 1);
                            tmem_fence_after();
#pragma unroll 1
                            for (int i = 0; i < D; i += 8) {
                                uint32_t o[8];
                                tmem_load8(o_at + i, o);
                                tmem_loaded(o);
#pragma unroll
                                for (int y = 0; y < 8; y++) o[y] = __float_as_uint(__uint_as_float(o[y]) * keep);
                                tmem_store8(o_at + i, o);
                            }
                        }
                    }
#pragma unroll
                    for (int z = 0; z < 64; z += 4) {
                        float w[4];
#pragma unroll
                        for (int e = 0; e < 4; e += 2) {
                            uint32_t f0 = x[z + e], f1 = x[z + e + 1];
                            fma2(f0, f1, by_row, -less);
                            w[e] = exp2_fast(__uint_as_float(f0)), w[e + 1] = exp2_fast(__uint_as_float(f1));
                            add2(part[e], part[e + 1], w[e], w[e + 1]);
                        }
                        if constexpr (INT8) {
                            const float4 vs = *reinterpret_cast<const float4*>(&v_scale_sm[slot][half + at + z]);
                            scale2(w[0], w[1], vs.x, vs.y), scale2(w[2], w[3], vs.z, vs.w);
                            if (!whole)
#pragma unroll
                                for (int e = 0; e < 4; e++) w[e] = seen[z / 32] >> (z % 32 + e) & 1 ? w[e] : 0.f;  // a hidden token's scale may be anything
                        }
                        x[z / 2] = pack_bf16(w[0], w[1]), x[z / 2 + 1] = pack_bf16(w[2], w[3]);
                    }
                    tmem_store32(s_at + at / 2, x);
                }
                sum += (__uint_as_float(part[0]) + __uint_as_float(part[1])) + (__uint_as_float(part[2]) + __uint_as_float(part[3]));
                tmem_stored();
                tmem_fence_before();
                mbar_arrive(bar_of(bars.p_ready[tile]));
            }
            const bool any = steps > 0, join = units.joined(u);
            float by_next = by_row;
            if (again && !join && works(after)) by_next = load_q(after);  // its products begin while this unit's rows are written
            if (any) {
                wait(bars.o_ready[tile], done - 1);
                tmem_fence_after();
            }
            auto odd_values = [&] { return !INT8 && u.n ? odd_sm[odd_at & 7] : 0; };
            if (!join) {
                const int odd = odd_values();
                if (tile == 0 || u.two) {
                    const float inverse = sum == 0.f ? 0.f : 1.f / sum;
                    const int i0 = (int)((uint32_t)m / (uint32_t)group);
                    const int64_t to = live ? (u.s.first + i0) * a.out_stride + (u.kv_head * group + m - i0 * group) * a.out_head_stride : 0;
                    const bool word = a.out_type == ZKB_VALUE_WORD, vec = ((uintptr_t)(static_cast<char*>(a.out) + to * (word ? 4 : 2)) & 31) == 0;
                    bool slow = odd;
#pragma unroll 1
                    for (int i = 0; i < D; i += 16) {
                        uint32_t o[2][8];
                        __syncwarp();  // rows part ways below: not all are live, written alike or slow
                        if (any) tmem_load8(o_at + i, o[0]), tmem_load8(o_at + i + 8, o[1]), tmem_loaded(o[0]), tmem_loaded(o[1]);
                        if (live) {
                            const int d = i;
                            float z[16];
#pragma unroll
                            for (int e = 0; e < 16; e++) z[e] = sum == 0.f || !any ? 0.f : __uint_as_float(o[e / 8][e & 7]) * inverse;
                            uint32_t w[8], test = 0;
#pragma unroll
                            for (int e = 0; e < 8; e++) w[e] = pack_bf16(z[2 * e], z[2 * e + 1]), test = zero_or_nan(w[e], test);
                            slow |= (test & 0x7fff7fffu) != 0;
                            if (word) {
                                uint32_t* const at = static_cast<uint32_t*>(a.out) + to + d;
#pragma unroll
                                for (int y = 0; y < 2; y++) {
                                    uint32_t x[8];
#pragma unroll
                                    for (int e = 0; e < 8; e++) x[e] = w[4 * y + e / 2] >> 16 * (e & 1) & 0xffffu;
                                    if (vec) store32(at + 8 * y, x);
                                    else
#pragma unroll
                                        for (int e = 0; e < 8; e++) at[8 * y + e] = x[e];
                                }
                            } else {
                                uint16_t* const at = static_cast<uint16_t*>(a.out) + to + d;
                                if (vec) store32(at, w);
                                else
#pragma unroll
                                    for (int e = 0; e < 16; e++) at[e] = (uint16_t)(w[e / 2] >> 16 * (e & 1));
                            }
                        }
                    }
                    // visible values that are no numbers: taken out (bf16) where some row does not see their key, else lost where a weight or a factor of nothing met them
                    if (slow && live && sum > 0.f) {
                        atomicAdd(&slow_sm, 1);
#pragma unroll 1
                        for (int d = 0; d < D; d++) put_what_is_no_number<INT8>(a, to + d, odd, u.seq, u.kv_head, d, p);
                        atomicAdd(&slow_sm, -1);
                    }
                }
            } else {
                // Each thread block finishes `part` of the rows: their sums go to [whose][row][four dimensions] of its shared memory, where Q and the keys were
                // (turned by the row's number, so that a warp's stores, a row a lane, and loads, a row after the other, each meet all banks).
                meet();
                const int odd = odd_values();
                const int rows_here = u.two ? 256 : 128, part = rows_here / units.ranks, one = u.split ? row : tile * 128 + row;
                const int whose = u.split ? 2 * units.rank + tile : units.rank, of = u.split ? 2 * units.ranks : units.ranks;
                if (one < rows_here) {
                    const int owner = one / part, at = one % part;
                    peer_store(&in_top[whose * part + at], owner, top);
                    peer_store(&in_sum[whose * part + at], owner, sum);
                    if (at == 0 && !(u.split && tile)) peer_store(&in_odd[units.rank], owner, odd);
                    __syncwarp();
#pragma unroll 1
                    for (int i = 0; i < D; i += 32) {
                        uint32_t o[32];
                        if (any) tmem_load32(o_at + i, o), tmem_loaded(o);
#pragma unroll
                        for (int y = 0; y < 32; y += 4)
                            peer_store4(q_at + sums_place(whose * part + at, (i + y) / 4), owner, any ? o[y] : 0u, any ? o[y + 1] : 0u, any ? o[y + 2] : 0u, any ? o[y + 3] : 0u);
                    }
                }
                meet();
                int set_aside = 0;
                if (!INT8)
                    for (int x = 0; x < units.ranks; x++) set_aside |= in_odd[x];
                if ((int)threadIdx.x < part) {  // a row's factors, its sum among them, where its maxima were
                    const int at = threadIdx.x;
                    float most = -INFINITY, all = 0.f;
#pragma unroll 4
                    for (int x = 0; x < of; x++) most = fmaxf(most, in_top[x * part + at]);
                    const float least = most == -INFINITY ? 0.f : most;
#pragma unroll 4
                    for (int x = 0; x < of; x++) {
                        const float f = exp2_fast(in_top[x * part + at] - least);
                        all += in_sum[x * part + at] * f;
                        in_top[x * part + at] = f;
                    }
                    in_sum[at] = all == 0.f ? 0.f : 1.f / all;  // (this thread alone has read that place)
                }
                named_sync(4, 256);
                bool slow = false;
#pragma unroll 1
                for (int i = threadIdx.x; i < part * (D / 4); i += 256) {
                    const int at = i / (D / 4), d = i % (D / 4) * 4;
                    const int mm = u.m0 + units.rank * part + at;
                    if (mm >= u.n_m) continue;
                    float z[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
                    for (int x = 0; x < of; x++) {
                        const float f = in_top[x * part + at];
                        const float4 o = *reinterpret_cast<const float4*>(sm + sums_place(x * part + at, d / 4));
                        z[0] += o.x * f, z[1] += o.y * f, z[2] += o.z * f, z[3] += o.w * f;
                    }
                    const float inverse = in_sum[at];
                    const int i0 = (int)((uint32_t)mm / (uint32_t)group);
                    const int64_t to = (u.s.first + i0) * a.out_stride + (u.kv_head * group + mm - i0 * group) * a.out_head_stride + d;
#pragma unroll
                    for (int e = 0; e < 4; e++) z[e] = inverse == 0.f ? 0.f : z[e] * inverse;
                    const bool word = a.out_type == ZKB_VALUE_WORD;
                    char* const out = static_cast<char*>(a.out) + to * (word ? 4 : 2);
                    const uint32_t w0 = pack_bf16(z[0], z[1]), w1 = pack_bf16(z[2], z[3]);
                    if (inverse > 0.f) slow |= set_aside || (zero_or_nan(w1, zero_or_nan(w0, 0)) & 0x7fff7fffu);
                    if (((uintptr_t)out & (word ? 15 : 7)) == 0) {
                        if (word) *reinterpret_cast<uint4*>(out) = make_uint4(w0 & 0xffffu, w0 >> 16, w1 & 0xffffu, w1 >> 16);
                        else *reinterpret_cast<uint2*>(out) = make_uint2(w0, w1);
                    } else {
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            const uint32_t h = (e < 2 ? w0 : w1) >> 16 * (e & 1) & 0xffffu;
                            if (word) reinterpret_cast<uint32_t*>(out)[e] = h;
                            else reinterpret_cast<uint16_t*>(out)[e] = (uint16_t)h;
                        }
                    }
                }
                if (slow) {  // as above
#pragma unroll 1
                    for (int i = threadIdx.x; i < part * (D / 4); i += 256) {
                        const int at = i / (D / 4), d = i % (D / 4) * 4, mm = u.m0 + units.rank * part + at;
                        if (mm >= u.n_m || !(in_sum[at] > 0.f)) continue;
                        const int i0 = (int)((uint32_t)mm / (uint32_t)group);
                        const int64_t to = (u.s.first + i0) * a.out_stride + (u.kv_head * group + mm - i0 * group) * a.out_head_stride + d;
#pragma unroll 1
                        for (int e = 0; e < 4; e++) put_what_is_no_number<INT8>(a, to + e, set_aside, u.seq, u.kv_head, d + e, u.s.pos + i0);
                    }
                }
                if (again) {
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // the next unit's copies go where these sums are
                    meet();
                    if (works(after)) by_next = load_q(after);
                }
            }
            passed += u.n;
            odd_at += u.n > 0;
            by_row = by_next;
            more = again;
            u = after;
        }
    } else {
        uint32_t items = 0, odd_at = 0, q_done[2] = {0, 0}, tile_done[2] = {0, 0};
        bool odd = false;
        const int th = threadIdx.x - 320;
        if constexpr (INT8) asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
        const uint32_t c128 = bf16_128(), c1152 = f16_1152();
        auto landed = [&](uint32_t sent) {  // the last copies of that many
            constexpr uint32_t RING = INT8 ? M::RAWS : M::STAGES;
            for (uint32_t item = sent > RING ? sent - RING : 0; item < sent; item++) mbar_wait(bar_of(INT8 ? bars.raw_full[item % RING] : bars.full[item % RING]), item / RING & 1);
        };
        while (more) {
            if (warp == 8) {  // ---- the copies
                if (TMA && lane == 0 && !failed) {
                    for (int i = 0; i < 2 * u.n; i++) {
                        const uint32_t item = items + i;
                        const CUtensorMap* map = i & 1 ? &maps.v : &maps.k;
                        const int base = units.base(u, i >> 1);
                        if constexpr (INT8) {
                            const uint32_t st = item % M::RAWS, bar = bar_of(bars.raw_full[st]);
                            wait_one(bars.raw_empty[st], item / M::RAWS + 1);
                            if (failed) {
                                landed(item);
                                break;
                            }
                            mbar_expect(bar, M::RAW);
#pragma unroll
                            for (int x = 0; x < M::RAW_BOXES; x++) tma_load(raw_ring + st * M::RAW + x * 128 * M::RAW_BOX, map, x * M::RAW_BOX, base, u.kv_head, u.seq, bar);
                        } else {
                            const uint32_t st = item % M::STAGES, bar = bar_of(bars.full[st]);
                            wait_one(bars.empty[st], item / M::STAGES + 1);
                            if (failed) {
                                landed(item);
                                break;
                            }
                            mbar_expect(bar, M::TILE);
#pragma unroll
                            for (int x = 0; x < M::PANELS; x++) tma_load(ring + st * M::TILE + x * 128 * M::BOX, map, x * (M::BOX / 2), base, u.kv_head, u.seq, bar);
                        }
                    }
                }
            } else if (warp == 9) {  // ---- the products
                // The whole warp goes along, so that what it works out is the same for all lanes and needs no vector registers; one lane issues. (As one lane's own work
                // it took longer than the products.)
                constexpr uint32_t qk = product_desc(INT8 ? 0 : 1, MANY_KEYS, false), qk_half = product_desc(INT8 ? 0 : 1, 64, false), pv = product_desc(1, D, true);
                constexpr uint32_t high = (uint32_t)(M::GROUP >> 4) | 1u << 14 | (uint32_t)M::SWIZZLE_KIND << 29;  // the upper half of every matrix's description
                // (an address in shared memory names the thread block of the cluster in bits that have no place there)
                const uint32_t q_low = (q_at >> 4 & 0x3fff) | 1u << 16, k_low = (ring >> 4 & 0x3fff) | 1u << 16, v_low = (ring >> 4 & 0x3fff) | (uint32_t)(128 * M::BOX >> 4) << 16;
                auto desc = [](uint32_t low) { return two_words(low, high); };
                const uint32_t tmem_u = __shfl_sync(0xffffffffu, tmem, 0);
                const bool one = elect_one();
                const int tiles = u.two || u.split ? 2 : 1;
                auto scores = [&](int tile, int j, uint32_t count) {  // count: the tile's steps before this one
                    const uint32_t item = items + 2 * j, st = item % M::STAGES;
                    if (tile == 0) wait(bars.ready[st], item / M::STAGES);
                    if (count) wait(bars.o_ready[tile], count - 1);  // P has been read where S goes
                    if (failed) return;
                    tmem_fence_after();
                    const uint32_t to = tmem_u + tile * 128, from_q = q_low + tile * (M::TILE >> 4), from_k = k_low + st * (M::TILE >> 4) + (u.split ? tile * (64 * M::BOX >> 4) : 0);
#pragma unroll
                    for (int i = 0; i < D / 16; i++) {
                        const uint32_t at = (i / (M::BOX / 32) * (128 * M::BOX) + i % (M::BOX / 32) * 32) >> 4;
                        product_ss(one, to, desc(from_q + at), desc(from_k + at), u.split ? qk_half : qk, i > 0);
                    }
                    if (one) {
                        products_done(bar_of(bars.s_ready[tile]));
                        if (tile == tiles - 1) products_done(bar_of(bars.empty[st]));
                        mbar_arrive(bar_of(bars.s_ready[tile]));
                    }
                    __syncwarp();
                };
                auto values = [&](int tile, int j, uint32_t count) {
                    const uint32_t item = items + 2 * j + 1, st = item % M::STAGES;
                    if (tile == 0) wait(bars.ready[st], item / M::STAGES);
                    wait(bars.p_ready[tile], count);
                    if (failed) return;
                    tmem_fence_after();
                    const uint32_t to = tmem_u + 256 + tile * D, from_p = tmem_u + tile * 128, from_v = v_low + st * (M::TILE >> 4) + (u.split ? tile * (64 * M::BOX >> 4) : 0);
#pragma unroll
                    for (int i = 0; i < 4; i++) product_ts(one, to, from_p + 8 * i, desc(from_v + i * (2 * M::GROUP >> 4)), pv, j > 0 || i > 0);
                    if (!u.split)
#pragma unroll
                        for (int i = 4; i < 8; i++) product_ts(one, to, from_p + 8 * i, desc(from_v + i * (2 * M::GROUP >> 4)), pv, true);
                    if (one) {
                        products_done(bar_of(bars.o_ready[tile]));
                        if (tile == tiles - 1) products_done(bar_of(bars.empty[st]));
                    }
                    __syncwarp();
                };
                if (u.n) {
                    wait(bars.q_ready[0], q_done[0]++);
                    if (tiles == 2) wait(bars.q_ready[1], q_done[1]++);
                }
#pragma unroll 1
                for (int j = -1; j < u.n; j++)
#pragma unroll
                    for (int tile = 0; tile < 2; tile++)
                        if (tile < tiles) {
                            if (j >= 0) values(tile, j, tile_done[tile] + j);
                            if (j + 1 < u.n) scores(tile, j + 1, tile_done[tile] + j + 1);
                        }
                tile_done[0] += u.n;
                if (tiles == 2) tile_done[1] += u.n;
            } else {  // ---- what the products read is made ready
                const char* const k = static_cast<const char*>(c.k) + (u.seq * c.seq_stride + u.kv_head * c.head_stride) * M::SIZE;
                const char* const v = static_cast<const char*>(c.v) + (u.seq * c.seq_stride + u.kv_head * c.head_stride) * M::SIZE;
                if (!INT8 && u.n) {
                    odd = false;
                    if (th == 0) odd_sm[odd_at & 7] = 0;
                    named_sync(3, M::READIERS);
                }
                for (int i = 0; i < 2 * u.n; i++) {
                    const uint32_t item = items + i, st = item % M::STAGES, to = ring + st * M::TILE;
                    const int base = units.base(u, i >> 1), kv = i & 1, last = u.last;
                    const bool whole = units.whole(u, base, MANY_KEYS);
                    if constexpr (INT8) {
                        wait(bars.empty[st], item / M::STAGES + 1);
                        if (kv == 0 && th < 128) {  // both of the block's scales: of the block before the last, nothing is needed any more when this place is free
                            const int key = min(base + th, last), slot = (item >> 1) & 1;
                            k_scale_sm[slot][th] = c.k_scale[u.seq * c.scale_seq_stride + u.kv_head * c.scale_head_stride + key];
                            v_scale_sm[slot][th] = c.v_scale[u.seq * c.scale_seq_stride + u.kv_head * c.scale_head_stride + key];
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
                                    if (test & 0x7fff7fffu) {  // what is no number would reach the rows that do not see its key: it is set aside (put_what_is_no_number)
                                        odd = true;
#pragma unroll
                                        for (int y = 0; y < 4; y++) w[y] = numbers_only(w[y]);
                                        if (TMA) st_shared4(place, w[0], w[1], w[2], w[3]);
                                    }
                                }
                                if (!TMA) st_shared4(place, w[0], w[1], w[2], w[3]);
                            }
                            if (odd) odd_sm[odd_at & 7] = 1;
                            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                        }
                    }
                    mbar_arrive(bar_of(bars.ready[st]));
                }
                odd_at += u.n > 0;
            }
            items += 2 * u.n;
            const bool join = units.joined(u);
            more = units.next(after);
            __syncwarp();
            if (join) {
                meet();
                meet();
                if (more) meet();
            }
            u = after;
        }
        // Nothing is on its way to shared memory or at work in tensor memory when the thread block gives them up, though a wait may have run out.
        if (TMA && warp == 8 && lane == 0 && !failed) {
            landed(items);
        } else if (warp == 9) {
            if (elect_one()) products_done(bar_of(bars.full[4]));  // (no stage has that one)
            mbar_wait(bar_of(bars.full[4]), 0);
        }
        __syncwarp();
    }
    if (failed && lane == 0) *dev_err = WAIT_RAN_OUT;
    tmem_fence_before();
    __syncthreads();
    if (warp == 0) {
        tmem_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
    }
}

template <int D, bool INT8>
cudaError_t launch_many(zkb_ctx* ctx, const zkb_step_attention_args& a) {
    using M = Many<D, INT8>;
    const zkb_kv_cache& c = a.cache;
    const uint32_t group = a.q_heads / c.n_heads, most = a.rows.max_rows ? std::min(a.rows.max_rows, a.rows.n_rows) : a.rows.n_rows;
    const uint32_t pairs = (uint32_t)std::min<uint64_t>(((uint64_t)most * group + 255) / 256, std::max(1u, (1u << 30) / (c.n_seqs * c.n_heads)));
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
    return launch_clusters(ranks, [&](uint32_t n) {
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim = {n, 1, 1};
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3((uint32_t)std::min<uint64_t>(units, clusters_at_once(n)) * n);
        cfg.blockDim = dim3(M::THREADS);
        cfg.dynamicSmemBytes = M::SMEM;
        cfg.stream = ctx->stream;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        return cudaLaunchKernelEx(&cfg, kernel, a, maps, pairs, ctx->dev_err);
    });
}
template cudaError_t launch_many<32, false>(zkb_ctx*, const zkb_step_attention_args&);
template cudaError_t launch_many<64, false>(zkb_ctx*, const zkb_step_attention_args&);
template cudaError_t launch_many<128, false>(zkb_ctx*, const zkb_step_attention_args&);
template cudaError_t launch_many<32, true>(zkb_ctx*, const zkb_step_attention_args&);
template cudaError_t launch_many<64, true>(zkb_ctx*, const zkb_step_attention_args&);
template cudaError_t launch_many<128, true>(zkb_ctx*, const zkb_step_attention_args&);

}  // namespace zk
