// Products of codes, many rows: tiles on the tensor cores' own memory.
#include <algorithm>

#include "step_product.cuh"
#include "tensor_memory.cuh"

namespace zk {

// A tile is 128 outputs (M, the weights' rows) by N rows of x: tcgen05 products of 8-bit codes with 32-bit sums in tensor memory, a thread an output. The weights come
// in steps of 128 codes:
//   8-bit weights and x by the tensor memory unit, where their rows start on 16-byte boundaries; the sums of a whole row are exact and read once.
//   4-bit weights by warps that turn them into 8-bit codes (16 times the code: the upper half of a byte in place) on their way to shared memory; each group's sum is a product of its own,
//   read from tensor memory, scaled and added up in registers while the next groups' products run.
//   Rows on other boundaries by the same warps.
// Few rows leave the tensor cores idle and are bound by the weights' bytes: N is as small as the rows allow, two thread blocks share an SM, and the steps are spread over the thread
// blocks of a cluster, which add up through each other's shared memory, each a share of the rows.
// Measured: 4096 rows of 4096 x 14336 8-bit weights 174 to 213 us on different GPUs, 2.7 to 2.3 PFLOP/s (a tile's sums are read while the next tile's products run); 32 rows of 4096 x 28672 24 to 25 us, 4.8 TB/s; 2001 rows
// of 4096 x 6144 4-bit weights with groups of 128 118 us, 850 TFLOP/s: there each group's 128 x 128 sums pass through registers, some 2700 warp instructions an SM and group of a tile
// against 256 cycles of the tensor cores, so the rate of instructions bounds it (59 % of all cycles issue one). By the source the sums are some 750 of them and the codes 480; the others, among them
// waits that try again and moves into pairs of registers, have not been told apart.
struct ProductMaps {
    CUtensorMap w, x;
};

// kind::i8, signed codes, 32-bit sums, 128 outputs.
__host__ __device__ constexpr uint32_t codes_desc(int n) { return 2u << 4 | 1u << 7 | 1u << 10 | (uint32_t)(n / 8) << 17 | (128u / 16) << 24; }
__device__ __forceinline__ void product_codes(bool one, uint32_t d, uint64_t a, uint64_t b, uint32_t desc, bool add) {
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t@q tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(desc), "r"((uint32_t)add),
                 "r"((uint32_t)one)
                 : "memory");
}
__device__ __forceinline__ void tma_load_2d(uint32_t to, const CUtensorMap* map, int code, int row, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(to), "l"(map), "r"(code), "r"(row), "r"(bar) : "memory");
}

// Sums of 4-bit weights' groups, below 2^22, begin with the pattern of 1.5 * 2^23: what is read is that float plus the sum, and a subtraction is the whole conversion (the instruction for it
// has an eighth of the rate of additions). Tensor memory is filled with it again as it is read.
constexpr uint32_t SUM_ZERO = 0x4b400000u;

struct TileBars {
    unsigned long long full[6], empty[6], done[32], x_full[8], raw_full[8], raw_empty[8], scale_full[4], scale_empty[4], sum_full[4], sum_empty[4], last;
};


template <int TYPE, bool INT4>
__device__ __forceinline__ void put(const zkb_step_product_args& a, uint32_t t, uint32_t c, uint32_t word, float by, float x_scale) {
    const int64_t at = (int64_t)t * a.out_stride + c;
    if constexpr (TYPE == ZKB_VALUE_INT32) static_cast<uint32_t*>(a.out)[at] = word;
    else store_value(a.out, at, TYPE, INT4 ? __uint_as_float(word) * x_scale : (float)(int)word * (x_scale * by));
}
template <int TYPE, bool INT4>
__device__ __forceinline__ void put(const zkb_step_product_args& a, uint32_t t, uint32_t c, uint32_t word, float by) {
    put<TYPE, INT4>(a, t, c, word, by, TYPE == ZKB_VALUE_INT32 ? 0.f : a.x_scale[t]);
}
// f(type as a constant)
template <bool INT4, class F>
__device__ __forceinline__ void by_type(uint32_t type, F f) {
    if (type == ZKB_VALUE_BF16) f(std::integral_constant<int, ZKB_VALUE_BF16>());
    else if (type == ZKB_VALUE_WORD) f(std::integral_constant<int, ZKB_VALUE_WORD>());
    else if (INT4 || type == ZKB_VALUE_F32) f(std::integral_constant<int, ZKB_VALUE_F32>());
    else f(std::integral_constant<int, ZKB_VALUE_INT32>());
}

// A place in a ring that is gone round, and the parity of its barriers' phase.
template <int SIZE>
struct Ring {
    uint32_t at = 0, parity = 0;
    __device__ __forceinline__ void next() {
        if (++at == SIZE) at = 0, parity ^= 1;
    }
};

template <bool INT4, int N, bool TMA>
__global__ void __launch_bounds__((Tile<INT4, N, TMA>::THREADS), (Tile<INT4, N, TMA>::BLOCKS))
    product_tiles_kernel(const __grid_constant__ zkb_step_product_args a, const __grid_constant__ ProductMaps maps, uint32_t row_tiles, uint32_t all_tiles, unsigned* dev_err) {
    using T = Tile<INT4, N, TMA>;
    extern __shared__ unsigned char tiles_sm[];
    __shared__ __align__(8) TileBars bars;
    __shared__ uint32_t tmem_sm;
    __shared__ float x_scale_sm[T::JOIN > 0 ? N : 1];
    unsigned char* const sm = tiles_sm + (-(uint32_t)__cvta_generic_to_shared(tiles_sm) & 1023);
    const uint32_t ring = (uint32_t)__cvta_generic_to_shared(sm), raw_ring = ring + T::STAGES * T::STAGE, x_ring = raw_ring + T::RAWS * T::RAW_BYTES, scale_ring = x_ring + T::XS * T::B;
    const uint32_t join_at = scale_ring + T::SCALES * T::SCALE_BYTES;
    uint32_t* const join = reinterpret_cast<uint32_t*>(sm + (join_at - ring));
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint32_t rank = cluster_rank(), ranks = cluster_ranks();
    if (warp == T::EPI + 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"((uint32_t)__cvta_generic_to_shared(&tmem_sm)), "n"(T::COLUMNS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    } else if (warp == 0 && lane == 0) {
        for (int i = 0; i < 6; i++) mbar_init(bar_of(bars.full[i]), (TMA && !T::RAW ? 1 : 0) + (T::FILLED ? 4 : 0)), mbar_init(bar_of(bars.empty[i]), 1);
        for (int i = 0; i < 8; i++) mbar_init(bar_of(bars.raw_full[i]), 1), mbar_init(bar_of(bars.raw_empty[i]), 4), mbar_init(bar_of(bars.x_full[i]), 1);
        for (int i = 0; i < 32; i++) mbar_init(bar_of(bars.done[i]), 1);
        for (int i = 0; i < 4; i++) mbar_init(bar_of(bars.sum_full[i]), 1), mbar_init(bar_of(bars.sum_empty[i]), T::EPI), mbar_init(bar_of(bars.scale_full[i]), 1), mbar_init(bar_of(bars.scale_empty[i]), T::EPI);
        mbar_init(bar_of(bars.last), 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    bool failed = false;  // a wait ran out: what follows is not valid, and nothing more is waited for
    auto wait = [&](const unsigned long long& b, uint32_t parity) {
        if (!failed) failed = !mbar_wait(bar_of(b), parity & 1);
        failed = __any_sync(0xffffffffu, failed);
    };
    auto arrive = [&](const unsigned long long& b) {  // once for the whole warp: arrivals at one barrier take turns
        __syncwarp();
        if (lane == 0) mbar_arrive(bar_of(b));
    };
    if constexpr (TMA) {
        if (warp == T::EPI && lane < 2) asm volatile("prefetch.tensormap [%0];" ::"l"(lane ? &maps.w : &maps.x) : "memory");
    }
    // What the last factors are is known now; a cluster has one tile.
    float out_scale = 1.f;
    if (T::JOIN > 0 && ranks > 1 && warp < T::EPI) {
        const uint32_t tile = blockIdx.x / ranks, of = N / ranks, c = tile / row_tiles * 128 + (threadIdx.x & 127), t = tile % row_tiles * N + rank * of + threadIdx.x;
        if (!INT4 && a.w_scale && c < a.n_out) out_scale = static_cast<const float*>(a.w_scale)[c];
        if (threadIdx.x < of) x_scale_sm[threadIdx.x] = a.x_scale && t < a.n_rows ? a.x_scale[t] : 0.f;
    }
    tmem_fence_before();
    __syncthreads();
    tmem_fence_after();
    if (ranks > 1) cluster_arrive();
    const uint32_t tmem = tmem_sm;
    const uint32_t all_steps = (a.n_in + T::CODES - 1) / T::CODES, who = blockIdx.x / ranks, every = gridDim.x / ranks;
    const uint32_t first_step = rank * all_steps / ranks, steps = (rank + 1) * all_steps / ranks - first_step;
    const uint32_t n_tiles = who < all_tiles ? (all_tiles - who + every - 1) / every : 0, items = n_tiles * steps;
    // The steps of all of this thread block's tiles, one after the other.
    struct Walk {
        uint32_t tile, step, row_tile, out_tile;
    };
    auto enter = [&](Walk& w) { w.row_tile = w.tile % row_tiles, w.out_tile = w.tile / row_tiles; };
    auto first = [&] {
        Walk w{who, 0, 0, 0};
        enter(w);
        return w;
    };
    auto next = [&](Walk& w) {
        if (++w.step == steps) w.step = 0, w.tile += every, enter(w);
    };
    const uint32_t log_group = INT4 ? 31 - __clz(a.group) : 7, per_step = T::CODES >> log_group, groups = (a.n_in + (1u << log_group) - 1) >> log_group;
    auto groups_in = [&](uint32_t step) { return min(per_step, groups - (first_step + step) * per_step); };
    // What the products announce. Of 4-bit weights, each read that ends, a step's or a group's: the sums are there then, and with a step's last one its codes and x are done with. There are more
    // barriers than reads under way, so none is gone past before all have seen it. Of 8-bit weights: a step's end, and a tile's sums.
    auto ends_in = [&](uint32_t step) { return !INT4 ? 0u : T::BY_STEP ? 1u : groups_in(step); };
    auto wait_end = [&](uint32_t n) { wait(bars.done[n % 32], n / 32); };  // of read n

    if (warp < T::EPI) {  // ---- the sums: a thread has an output, and half of the rows where two threads share it
        constexpr int MINE = N / (T::EPI / 4), CHUNK = MINE < 32 ? 16 : 32;
        const uint32_t c128 = (uint32_t)(warp & 3) * 32 + lane, half = (uint32_t)(warp >> 2) * MINE, at_lanes = tmem + ((uint32_t)(warp & 3) << 21) + half;
        Ring<T::SUMS> sums;
        Ring<(T::SCALES > 0 ? T::SCALES : 1)> scale;
        uint32_t read_ends = 0;
        if constexpr (INT4) {
#pragma unroll 1
            for (int b = 0; b < T::SUMS; b++) {
#pragma unroll 1
                for (int k = 0; k < T::SUM; k += N)
#pragma unroll
                    for (int j = 0; j < MINE; j += 16) tmem_fill16(at_lanes + b * T::SUM + k + j, SUM_ZERO);
                tmem_stored();
                tmem_fence_before();
                arrive(bars.sum_empty[b]);
            }
        }
        Walk w = first();
        for (uint32_t i = 0; i < n_tiles; i++, w.tile += every, enter(w)) {
            const uint32_t c = w.out_tile * 128 + c128, t0 = w.row_tile * N + half;
            const bool live = c < a.n_out;
            // CHUNK columns at a time of the sums at `at`, to `use`
            auto read = [&](uint32_t at, bool last, auto use) {
#pragma unroll
                for (int j = 0; j < MINE; j += CHUNK) {
                    uint32_t x[CHUNK];
                    if constexpr (CHUNK == 32) tmem_load32(at + j, x);
                    else tmem_load16(at + j, x);
                    tmem_loaded(x);
                    if constexpr (INT4) {
#pragma unroll
                        for (int y = 0; y < CHUNK; y += 16) tmem_fill16(at + j + y, SUM_ZERO);
                    }
                    if (last && j + CHUNK == MINE) {
                        if constexpr (INT4) tmem_stored();
                        tmem_fence_before();
                        arrive(bars.sum_empty[sums.at]);
                    }
                    use(j, x);
                }
            };
            auto arrived = [&] {
                if constexpr (INT4) wait_end(read_ends++);
                else wait(bars.sum_full[sums.at], sums.parity);
                tmem_fence_after();
            };
            // The sums of columns j .. j + COUNT - 1 to the thread blocks that add up those rows, side by side there.
            auto share = [&](int j, const uint32_t(&x)[CHUNK]) {
                const uint32_t log_of = 31 - __clz(N / ranks);
                if (log_of >= 2) {
#pragma unroll
                    for (int y = 0; y < CHUNK; y += 4) {
                        const uint32_t column = half + j + y;
                        peer_store4(join_at + (((rank * 128 + c128) << log_of) + (column & ((1u << log_of) - 1))) * 4, (int)(column >> log_of), x[y], x[y + 1], x[y + 2], x[y + 3]);
                    }
                } else {
#pragma unroll
                    for (int y = 0; y < CHUNK; y++) {
                        const uint32_t column = half + j + y;
                        peer_store_word(join + (((rank * 128 + c128) << log_of) + (column & ((1u << log_of) - 1))), (int)(column >> log_of), x[y]);
                    }
                }
            };
            if constexpr (INT4) {
                uint64_t acc[MINE / 2];
#pragma unroll
                for (int j = 0; j < MINE / 2; j++) acc[j] = 0;
                uint32_t now[4], k8 = 8;  // eight groups' scales
                auto next_scale = [&] {
                    if (k8 == 8) {
                        k8 = 0;
                        wait(bars.scale_full[scale.at], scale.parity);
                        ld_shared4(scale_ring + scale.at * T::SCALE_BYTES + c128 * 16, now[0], now[1], now[2], now[3]);
                        arrive(bars.scale_empty[scale.at]);
                        scale.next();
                    }
                    const uint32_t two = k8 < 4 ? (k8 < 2 ? now[0] : now[1]) : (k8 < 6 ? now[2] : now[3]);
                    const float s = __uint_as_float(k8 & 1 ? two & 0xffff0000u : two << 16);
                    k8++;
                    return s * 0.0625f;  // (the codes are 16 times themselves)
                };
                const uint64_t less = both(-12582912.f, -12582912.f);
                if constexpr (T::BY_STEP) {
#pragma unroll 1
                    for (uint32_t s = 0; s < steps; s++) {
                        const uint32_t n = groups_in(s);
                        arrived();
#pragma unroll 1
                        for (uint32_t k = 0; k < n; k++) {
                            const float by = next_scale();
                            read(at_lanes + sums.at * T::SUM + k * N, k + 1 == n, [&](int j, const uint32_t(&x)[CHUNK]) {
#pragma unroll
                                for (int y = 0; y < CHUNK; y += 2) acc[(j + y) / 2] = fma_both(add_both(two_words(x[y], x[y + 1]), less), both(by, by), acc[(j + y) / 2]);
                            });
                        }
                        sums.next();
                    }
                } else {  // (sixteen columns at a time: more wait in registers)
                    const uint32_t all = min((first_step + steps) * per_step, groups) - first_step * per_step;
#pragma unroll 1
                    for (uint32_t g = 0; g < all; g++) {
                        const float by = next_scale();
                        arrived();
                        const uint32_t at = at_lanes + sums.at * T::SUM;
#pragma unroll
                        for (int j = 0; j < MINE; j += 16) {
                            uint32_t x[16];
                            tmem_load16(at + j, x);
                            tmem_loaded(x);
                            tmem_fill16(at + j, SUM_ZERO);
                            if (j + 16 == MINE) {
                                tmem_stored();
                                tmem_fence_before();
                                arrive(bars.sum_empty[sums.at]);
                            }
#pragma unroll
                            for (int y = 0; y < 16; y += 2) acc[(j + y) / 2] = fma_both(add_both(two_words(x[y], x[y + 1]), less), both(by, by), acc[(j + y) / 2]);
                        }
                        sums.next();
                    }
                }
                if (ranks == 1) {
                    if (live)
                        by_type<INT4>(a.out_type, [&](auto type) {
#pragma unroll
                            for (int j = 0; j < MINE; j++)
                                if (t0 + j < a.n_rows) put<decltype(type)::value, INT4>(a, t0 + j, c, (uint32_t)(acc[j / 2] >> (32 * (j % 2))), 1.f);
                        });
                } else if constexpr (T::JOIN > 0) {
                    cluster_wait();
#pragma unroll
                    for (int j = 0; j < MINE; j += CHUNK) {
                        uint32_t x[CHUNK];
#pragma unroll
                        for (int y = 0; y < CHUNK; y++) x[y] = (uint32_t)(acc[(j + y) / 2] >> (32 * (y % 2)));
                        share(j, x);
                    }
                }
            } else {
                const float by = live && a.w_scale ? static_cast<const float*>(a.w_scale)[c] : 1.f;
                if (ranks > 1) {
                    if constexpr (T::JOIN > 0) cluster_wait();
                }
                arrived();
                if (ranks == 1) {
                    read(at_lanes + sums.at * T::SUM, true, [&](int j, const uint32_t(&x)[CHUNK]) {
                        if (live)
                            by_type<INT4>(a.out_type, [&](auto type) {
#pragma unroll
                                for (int y = 0; y < CHUNK; y++)
                                    if (t0 + j + y < a.n_rows) put<decltype(type)::value, INT4>(a, t0 + j + y, c, x[y], by);
                            });
                    });
                } else if constexpr (T::JOIN > 0) {
                    read(at_lanes + sums.at * T::SUM, true, share);
                }
                sums.next();
            }
        }
    } else if (warp == T::EPI) {  // ---- copies
        if constexpr (TMA) {  // x and 8-bit weights into the stages, or x into its own ring
            constexpr int SIZE = T::RAW ? T::XS : T::STAGES;
            const unsigned long long* const full = T::RAW ? bars.x_full : bars.full;
            uint32_t sent = 0;
            Ring<SIZE> st;
            Walk w = first(), old = first();  // `old`: the step whose place is taken
            uint32_t ends = 0;
            for (; sent < items; sent++, st.next(), next(w)) {
                if constexpr (T::RAW) {
                    if (sent >= SIZE) ends += ends_in(old.step), next(old), wait_end(ends - 1);
                } else {
                    wait(bars.empty[st.at], st.parity ^ 1);
                }
                if (failed) break;
                if (lane == 0) {
                    const uint32_t to = T::RAW ? x_ring + st.at * T::B : ring + st.at * T::STAGE + T::A, bar = bar_of(full[st.at]);
                    mbar_expect(bar, T::RAW ? T::B : T::STAGE);
                    if constexpr (!INT4) tma_load_2d(to - T::A, &maps.w, (first_step + w.step) * 128, w.out_tile * 128, bar);
#pragma unroll
                    for (int h = 0; h < T::HALVES; h++) tma_load_2d(to + h * T::B_HALF, &maps.x, (first_step + w.step) * T::CODES + h * 128, w.row_tile * N, bar);
                }
                __syncwarp();
            }
            // Whatever is on its way comes to its place before the thread block ends, though a wait may have run out.
            for (uint32_t j = sent < SIZE ? 0 : sent - SIZE; j < sent; j++) mbar_wait(bar_of(full[j % SIZE]), (j / SIZE) & 1);
        }
    } else if (warp == T::EPI + 1) {  // ---- products
        constexpr uint32_t high = (1024u >> 4) | 1u << 14 | 2u << 29, desc = codes_desc(N);
        const uint32_t a_low = (ring >> 4 & 0x3fff) | 1u << 16, x_low = (x_ring >> 4 & 0x3fff) | 1u << 16, tmem_u = __shfl_sync(0xffffffffu, tmem, 0);
        const bool one = elect_one();
        Ring<T::STAGES> st;
        Ring<(T::XS > 0 ? T::XS : 1)> xs;
        Ring<T::SUMS> sums;
        const uint32_t parts = (1u << log_group) / 32;
        uint32_t step = 0, ends = 0;
#pragma unroll 1
        for (uint32_t i = 0; i < items; i++, st.next()) {
            const uint32_t from_a = a_low + st.at * (T::STAGE >> 4), from_b = T::RAW ? x_low + xs.at * (T::B >> 4) : from_a + (T::A >> 4);
            if constexpr (!INT4) {
                if (step == 0) wait(bars.sum_empty[sums.at], sums.parity ^ 1);
            }
            if constexpr (T::RAW) wait(bars.x_full[xs.at], xs.parity);
            wait(bars.full[st.at], st.parity);
            if (failed) break;
            tmem_fence_after();
            if constexpr (INT4) {
                const uint32_t n = groups_in(step);
                for (uint32_t g = 0; g < n; g++) {
                    if (!T::BY_STEP || g == 0) {
                        wait(bars.sum_empty[sums.at], sums.parity);  // (filled to begin with: its first arrivals)
                        if (failed) break;
                        tmem_fence_after();
                    }
                    const uint32_t half = g << log_group >> 7, from = 2 * (g * parts & 3), group_a = from_a + half * (T::A_HALF >> 4) + from, group_b = from_b + half * (T::B_HALF >> 4) + from;
                    for (uint32_t k = 0; k < parts; k++)
                        product_codes(one, tmem_u + sums.at * T::SUM + (T::BY_STEP ? g * N : 0), two_words(group_a + 2 * k, high), two_words(group_b + 2 * k, high), desc, true);
                    if (!T::BY_STEP || g + 1 == n) {
                        if (one) products_done(bar_of(bars.done[ends % 32]));
                        ends++;
                        sums.next();
                    }
                }
                if constexpr (T::RAW) xs.next();
            } else {
#pragma unroll
                for (uint32_t k = 0; k < 4; k++)
                    product_codes(one, tmem_u + sums.at * T::SUM, two_words(from_a + 2 * k, high), two_words(from_b + 2 * k, high), desc, step > 0 || k > 0);
                if (one) {
                    products_done(bar_of(bars.empty[st.at]));
                    if (step + 1 == steps) products_done(bar_of(bars.sum_full[sums.at]));
                }
                if (step + 1 == steps) sums.next();
            }
            if (++step == steps) step = 0;
            __syncwarp();
        }
        // Nothing is at work in tensor memory when the thread block gives it up, though a wait may have run out.
        if (one) products_done(bar_of(bars.last));
        __syncwarp();
        mbar_wait(bar_of(bars.last), 0);
    } else if constexpr (T::FILLED) {
        if (warp == T::EPI + 2) {  // ---- copies of 4-bit weights
            if constexpr (T::RAW) {
                uint32_t sent = 0;
                Ring<T::RAWS> rs;
                Walk w = first();
                for (; sent < items; sent++, rs.next(), next(w)) {
                    wait(bars.raw_empty[rs.at], rs.parity ^ 1);
                    if (failed) break;
                    if (lane == 0) {
                        mbar_expect(bar_of(bars.raw_full[rs.at]), T::RAW_BYTES);
                        tma_load_2d(raw_ring + rs.at * T::RAW_BYTES, &maps.w, (first_step + w.step) * (T::CODES / 2), w.out_tile * 128, bar_of(bars.raw_full[rs.at]));
                    }
                    __syncwarp();
                }
                for (uint32_t j = sent < T::RAWS ? 0 : sent - T::RAWS; j < sent; j++) mbar_wait(bar_of(bars.raw_full[j % T::RAWS]), (j / T::RAWS) & 1);
            }
        } else if (INT4 && warp == T::EPI + 3) {  // ---- scales, eight groups of the tile's 128 outputs at a time, four outputs a lane; the next ones on their way
            Ring<(T::SCALES > 0 ? T::SCALES : 1)> scale;
            const uint32_t g0 = first_step * per_step, g1 = min((first_step + steps) * per_step, groups), blocks = (g1 - g0 + 7) / 8;
            const uint16_t* const scales = static_cast<const uint16_t*>(a.w_scale);
            auto each = [&](auto load) {  // load(first scale, how many are there): eight
                uint32_t out_tile = who / row_tiles, block = 0, tile = who;
                uint4 ahead[4];
                auto fetch = [&] {
#pragma unroll
                    for (int j = 0; j < 4; j++) ahead[j] = load(scales + (int64_t)min(out_tile * 128 + j * 32 + lane, a.n_out - 1) * a.w_scale_stride + g0 + block * 8, groups - (g0 + block * 8));
                    if (++block == blocks) block = 0, tile += every, out_tile = tile / row_tiles;
                };
                const uint32_t all = n_tiles * blocks;
                if (all) fetch();
                for (uint32_t i = 0; i < all; i++) {
                    uint4 now[4];
#pragma unroll
                    for (int j = 0; j < 4; j++) now[j] = ahead[j];
                    if (i + 1 < all) fetch();
                    wait(bars.scale_empty[scale.at], scale.parity ^ 1);
                    if (failed) break;
#pragma unroll
                    for (int j = 0; j < 4; j++) st_shared4(scale_ring + scale.at * T::SCALE_BYTES + (j * 32 + lane) * 16, now[j].x, now[j].y, now[j].z, now[j].w);
                    arrive(bars.scale_full[scale.at]);
                    scale.next();
                }
            };
            auto one_by_one = [](const uint16_t* p, uint32_t n) {
                uint32_t v[8];
#pragma unroll
                for (int y = 0; y < 8; y++) v[y] = y < n ? p[y] : 0u;
                return make_uint4(v[0] | v[1] << 16, v[2] | v[3] << 16, v[4] | v[5] << 16, v[6] | v[7] << 16);
            };
            if (scales_by_eights((uintptr_t)(scales + g0), g0, groups, a.w_scale_stride, a.n_out)) each([](const uint16_t* p, uint32_t) { return *reinterpret_cast<const uint4*>(p); });
            else each(one_by_one);
        } else {  // ---- codes into shared memory: each set of four warps every SETS-th step
            const int f = threadIdx.x - 32 * T::FIRST_FILLER, th = f & 127, set = f >> 7;
            const int64_t w_row = INT4 ? a.w_stride / 2 : a.w_stride;
            const int bytes = INT4 ? (int)(a.n_in + 1) / 2 : (int)a.n_in;
            constexpr int STEP = 128, ROW = STEP / 16, MINE = ROW;  // bytes of a row's step, 16s of them, a thread's
            auto put_codes = [&](uint32_t to, int row, int b, const uint4& v) {  // 16 bytes from byte b of a row's step on
                if constexpr (INT4) {
                    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
                    uint32_t u[8];
#pragma unroll
                    for (int y = 0; y < 4; y++) {
                        const uint32_t even = w[y] << 4 & 0xf0f0f0f0u, odd = w[y] & 0xf0f0f0f0u;
                        u[2 * y] = __byte_perm(even, odd, 0x5140), u[2 * y + 1] = __byte_perm(even, odd, 0x7362);
                    }
                    // (the second half's first: the lanes of a row write to different banks)
                    const bool second = b >= 64;
                    const uint32_t place = to + (second ? T::A_HALF : 0), at = 2 * b & 127, x = second ? 16 : 0;
                    st_shared4(place + box_place<128>(row, at + x), second ? u[4] : u[0], second ? u[5] : u[1], second ? u[6] : u[2], second ? u[7] : u[3]);
                    st_shared4(place + box_place<128>(row, at + 16 - x), second ? u[0] : u[4], second ? u[1] : u[5], second ? u[2] : u[6], second ? u[3] : u[7]);
                } else {
                    st_shared4(to + box_place<128>(row, b), v.x, v.y, v.z, v.w);
                }
            };
            Ring<T::STAGES> st;
            Ring<(T::RAWS > 0 ? T::RAWS : 1)> rs;
            Walk w = first(), old = first();
            uint32_t ends = 0, passed = 0;  // reads that have ended with the step that was in this stage before, steps so far
            auto stage_free = [&] {
                if constexpr (!INT4) wait(bars.empty[st.at], st.parity ^ 1);
                else if (passed >= T::STAGES) wait_end(ends + ends_in(old.step) - 1);
            };
            auto skip = [&] {
                if (INT4 && passed >= T::STAGES) ends += ends_in(old.step), next(old);
                passed++;
                st.next(), next(w);
                if constexpr (T::RAW) rs.next();
            };
            for (int i = 0; i < set; i++) skip();
#pragma unroll 1
            for (uint32_t i = set; i < items; i += T::SETS) {
                const uint32_t to = ring + st.at * T::STAGE;
                if constexpr (T::RAW) {
                    before_codes(stage_free, [&] { wait(bars.raw_full[rs.at], rs.parity); });
                    if (failed) break;
#pragma unroll
                    for (int j0 = 0; j0 < MINE; j0 += 4) {
                        uint4 v[4];
#pragma unroll
                        for (int j = 0; j < 4; j++) ld_shared4(raw_ring + rs.at * T::RAW_BYTES + (th + (j0 + j) * 128) * 16, v[j].x, v[j].y, v[j].z, v[j].w);
#pragma unroll
                        for (int j = 0; j < 4; j++) put_codes(to, (th + (j0 + j) * 128) / ROW, (th + (j0 + j) * 128) % ROW * 16, v[j]);
                    }
                    arrive(bars.raw_empty[rs.at]);
                } else {
                    const int step = (int)(first_step + w.step);
                    const int8_t *const w_lo = static_cast<const int8_t*>(a.w), *const w_hi = w_lo + (a.n_out - 1) * w_row + bytes, *const x_hi = a.x + (int64_t)(a.n_rows - 1) * a.x_stride + a.n_in;
                    // Four 16s at a time: their loads, and then, into a stage that is free, their codes. What lies behind a row's codes counts for nothing where x is zero there (`cut`).
                    auto four = [&](int q0, int n, auto from_of, const int8_t* lo, const int8_t* hi, int row_bytes, int at, auto to_place, bool cut) {
                        Fetched r[4];
                        const int8_t* p[4];
#pragma unroll
                        for (int j = 0; j < 4; j++) {
                            const int q = q0 + j * 128;
                            p[j] = from_of(q);
                            if (q < n) r[j] = fetch16(p[j], lo, hi);
                        }
                        stage_free();
#pragma unroll
                        for (int j = 0; j < 4; j++) {
                            const int q = q0 + j * 128;
                            if (q < n) {
                                const uint4 v = fetched16(r[j], p[j], lo, hi);
                                to_place(q, cut ? first_bytes(v, row_bytes - at - q % 8 * 16) : v);
                            }
                        }
                    };
#pragma unroll 1
                    for (int q = th; q < 128 * ROW; q += 512)
                        four(q, 128 * ROW, [&](int q) { return w_lo + (int64_t)min(w.out_tile * 128 + q / ROW, a.n_out - 1) * w_row + step * STEP + q % ROW * 16; }, w_lo, w_hi, bytes, 0,
                             [&](int q, const uint4& v) { put_codes(to, q / ROW, q % ROW * 16, v); }, false);
#pragma unroll 1
                    for (int h = 0; h < T::HALVES; h++)
#pragma unroll 1
                        for (int q = th; q < N * 8; q += 512)
                            four(q, N * 8, [&](int q) { return a.x + (int64_t)min(w.row_tile * N + q / 8, a.n_rows - 1) * a.x_stride + step * T::CODES + h * 128 + q % 8 * 16; }, a.x, x_hi, (int)a.n_in,
                                 step * T::CODES + h * 128, [&](int q, const uint4& v) { st_shared4(to + T::A + h * T::B_HALF + box_place<128>(q / 8, q % 8 * 16), v.x, v.y, v.z, v.w); }, true);
                    if (failed) break;
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                arrive(bars.full[st.at]);
#pragma unroll
                for (int j = 0; j < T::SETS; j++) skip();
            }
        }
    }
    __syncwarp();
    if (ranks > 1) {
        if (warp >= T::EPI || n_tiles == 0) cluster_wait();
        cluster_arrive(), cluster_wait();
        if constexpr (T::JOIN > 0) {
            const Walk w = first();
            const uint32_t c128 = threadIdx.x & 127, c = w.out_tile * 128 + c128, of = N / ranks, first_row = w.row_tile * N + rank * of;
            if (warp < T::EPI && c < a.n_out) {
                by_type<INT4>(a.out_type, [&](auto type) {
#pragma unroll 4
                    for (uint32_t j = threadIdx.x >> 7; j < of; j += T::EPI / 4) {
                        if (first_row + j >= a.n_rows) break;
                        uint32_t word = join[c128 * of + j];
                        for (uint32_t r = 1; r < ranks; r++) {
                            const uint32_t more = join[(r * 128 + c128) * of + j];
                            word = INT4 ? __float_as_uint(__uint_as_float(word) + __uint_as_float(more)) : word + more;
                        }
                        put<decltype(type)::value, INT4>(a, first_row + j, c, word, out_scale, x_scale_sm[j]);
                    }
                });
            }
        }
    }
    if (failed && lane == 0) *dev_err = WAIT_RAN_OUT;
    tmem_fence_before();
    __syncthreads();
    if (warp == T::EPI + 1) {
        tmem_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(T::COLUMNS));
    }
}

// A map of rows of `bytes` bytes in boxes of `rows` rows by `box` bytes, or false where the layout has none: the unit wants 16-byte boundaries.
static bool rows_map(CUtensorMap& map, const void* p, uint32_t bytes, uint32_t n_rows, int64_t stride, uint32_t rows, uint32_t box, bool swizzled) {
    const TensorMapEncode encode = tensor_map_encode();
    if (n_rows == 1) stride = (bytes + 15) / 16 * 16;
    if (!encode || !aligned_to(p, 16) || stride % 16 != 0 || stride >= (1ll << 40)) return false;
    const cuuint64_t dims[2] = {bytes, n_rows}, strides[1] = {(cuuint64_t)stride};
    const cuuint32_t boxes[2] = {box, rows}, ones[2] = {1, 1};
    return encode(&map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(p), dims, strides, boxes, ones, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzled ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_NONE,
                  CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <bool INT4, int N, bool TMA>
static cudaError_t launch_variant(zkb_ctx* ctx, const zkb_step_product_args& a, const ProductMaps& maps) {
    using T = Tile<INT4, N, TMA>;
    auto kernel = product_tiles_kernel<INT4, N, TMA>;
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, T::SMEM);
    if (e != cudaSuccess) return e;
    const uint32_t row_tiles = (a.n_rows + N - 1) / N, tiles = row_tiles * ((a.n_out + 127) / 128), steps = (a.n_in + T::CODES - 1) / T::CODES;
    // Few tiles are spread over clusters, while all of them are on the GPU at once, with an SM for each thread block where a share is short: a cluster costs some 4 us, as much as 6 steps of 4-bit
    // weights or 12 of 8-bit ones. By 1, 2, 4 and 8 thread blocks a tile, in us: 20 rows of 8192 x 1024 8-bit (4-bit) weights 22, 16, 12, 9 (29, 21, 15, 11.5), 17 of 4096 x 4096 14.1, 13.1, 10.8
    // (18.6, 15.9, 13.0); by 1 and 2, 128 rows of 14336 x 4096 35 and 27, of 4096 x 4096 14.3 and 14.9; 64 rows of 1024 x 4096 8.2 by 1 and 10.2 by 4.
    uint32_t ranks = 1;
    if (T::JOIN > 0 && steps >= (INT4 ? 12 : 24))
        while (ranks < 16 && ranks < N && tiles <= (!INT4 && steps > 32 * ranks ? 2 : 1) * clusters_at_once(2 * ranks) && steps >= (INT4 ? 2 : 4) * ranks) ranks *= 2;
    return launch_clusters(ranks, [&](uint32_t n) {
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim = {n, 1, 1};
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(n > 1 ? tiles * n : std::min(tiles, 148u * T::BLOCKS));
        cfg.blockDim = dim3(T::THREADS);
        cfg.dynamicSmemBytes = T::SMEM;
        cfg.stream = ctx->stream;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        return cudaLaunchKernelEx(&cfg, kernel, a, maps, row_tiles, tiles, ctx->dev_err);
    });
}

template <bool INT4, int N>
static cudaError_t launch_rows_of(zkb_ctx* ctx, const zkb_step_product_args& a) {
    ProductMaps maps{};
    const bool tma = rows_map(maps.x, a.x, a.n_in, a.n_rows, a.x_stride, N, 128, true) && (INT4 ? rows_map(maps.w, a.w, (a.n_in + 1) / 2, a.n_out, a.w_stride / 2, 128, 128, false) : rows_map(maps.w, a.w, a.n_in, a.n_out, a.w_stride, 128, 128, true));
    return tma ? launch_variant<INT4, N, true>(ctx, a, maps) : launch_variant<INT4, N, false>(ctx, a, maps);
}

template <bool INT4>
cudaError_t launch_tiles(zkb_ctx* ctx, const zkb_step_product_args& a) {
    // Rows a tile: the fewest that leave no more tiles than are on the GPU at once, of those that the rows need and the kernels have (a group's sums of 4-bit weights are kept in registers: up to
    // 128). Of 8-bit weights that is two tiles an SM: they share it up to 64 rows, and of 128 rows two take less than one of 256. In us:
    //   8-bit, n_in 4096, rows x n_out       32     64    128    256       4-bit, groups of 128     32     64    128
    //      256 x 4096                      16.3   18.3   16.5   23.2          33 x 14336          31.8   21.0
    //      128 x 14336                     25.1   21.5   18.8                128 x 8192           31.6   20.8   24.4
    //      256 x 14336                     39.9   30.9   25.2   27.5         128 x 14336          56.7   34.4   25.1
    //      512 x 14336                     63.7   49.5   40.3   35.6         160 x 8192           44.4   34.4   24.7
    // 32 rows of more than 32 are not taken of 4-bit weights: the best by a tenth at 128 x 1024 (12.4 and 14.1), the worst by a fifth at 64 x 4096 with groups of 32 (25.3 and 20.1). 64 of 8-bit
    // weights are for up to 64 rows only (64 x 28672: 29.0, 26.2 and 28.3 by 32, 64 and 128). On odd boundaries an SM has one tile of each size (700 x 4097 x 4095: 104 by 128, 84 by 256).
    const uint64_t out_tiles = (a.n_out + 127) / 128;
    const bool pairs = !INT4 && aligned_to(a.x, 16) && aligned_to(a.w, 16) && a.x_stride % 16 == 0 && a.w_stride % 16 == 0;
    auto at_once = [&](uint32_t n) { return (a.n_rows + n - 1) / n * out_tiles <= (pairs ? 296 : 148); };
    uint32_t n = INT4 ? 128 : 256;
    if (!INT4 && a.n_rows <= 16) n = 16;  // (4-bit weights of up to sixteen rows come another way)
    else if (a.n_rows <= 32 || (!INT4 && at_once(32))) n = 32;
    else if (a.n_rows <= 64 || (INT4 && at_once(64))) n = 64;
    else if (a.n_rows <= 128 || at_once(128)) n = 128;
    if constexpr (!INT4)
        if (n == 16) return launch_rows_of<INT4, 16>(ctx, a);
    if (n == 32) return launch_rows_of<INT4, 32>(ctx, a);
    if (n == 64) return launch_rows_of<INT4, 64>(ctx, a);
    if constexpr (!INT4)
        if (n == 256) return launch_rows_of<INT4, 256>(ctx, a);
    return launch_rows_of<INT4, 128>(ctx, a);
}
template cudaError_t launch_tiles<true>(zkb_ctx*, const zkb_step_product_args&);
template cudaError_t launch_tiles<false>(zkb_ctx*, const zkb_step_product_args&);

}  // namespace zk
