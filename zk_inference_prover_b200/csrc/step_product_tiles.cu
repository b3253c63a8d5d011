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
struct ProductMaps {
    CUtensorMap w, x;
};

template <bool INT4, int N, bool TMA>
struct Tile {
    static constexpr bool FILLED = INT4 || !TMA;                       // the weights' part of a stage is written by warps
    static constexpr int EPI = N >= 128 ? 8 : 4, FILL = FILLED ? 8 : 0;  // warps that read the sums, and that write codes
    static constexpr int THREADS = 32 * (EPI + 2 + FILL), FILLERS = 32 * FILL;
    static constexpr int A = 128 * 128, B = N * 128, STAGE = A + B;
    static constexpr int BLOCKS = N <= 32 || (N == 64 && !FILLED) ? 2 : 1;  // thread blocks an SM
    static constexpr int JOIN = N <= 64 ? N * 512 : 0;                  // a cluster's sums
    static constexpr int ROOM = BLOCKS == 2 ? 112 * 1024 : 208 * 1024;
    static constexpr int STAGES = (ROOM - JOIN) / STAGE < 6 ? (ROOM - JOIN) / STAGE : 6;
    static constexpr int SUMS = INT4 ? 4 : 2;                           // tiles' or groups' sums in tensor memory at a time
    static constexpr int COLUMNS = SUMS * N < 32 ? 32 : SUMS * N;
    // A thread block never waits for tensor memory: those that fit an SM's shared memory together (this kernel's variants and attention's, which take all columns and 121 KB) fit its
    // 512 columns. Clusters that each hold what another waits for would wait forever.
    static constexpr int LEAST = BLOCKS == 2 ? 108 * 1024 : 121 * 1024;
    static constexpr int SMEM = 1024 + (STAGES * STAGE + JOIN > LEAST ? STAGES * STAGE + JOIN : LEAST);
    static_assert(COLUMNS * BLOCKS <= 512 && (COLUMNS & (COLUMNS - 1)) == 0, "");
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

struct TileBars {
    unsigned long long full[6], empty[6], sum_full[4], sum_empty[4], last;
};


template <int TYPE, bool INT4>
__device__ __forceinline__ void put(const zkb_step_product_args& a, uint32_t t, uint32_t c, uint32_t word, float by) {
    const int64_t at = (int64_t)t * a.out_stride + c;
    if constexpr (TYPE == ZKB_VALUE_INT32) static_cast<uint32_t*>(a.out)[at] = word;
    else store_value(a.out, at, TYPE, INT4 ? __uint_as_float(word) * a.x_scale[t] : (float)(int)word * (a.x_scale[t] * by));
}
// f(type as a constant)
template <bool INT4, class F>
__device__ __forceinline__ void by_type(uint32_t type, F f) {
    if (type == ZKB_VALUE_BF16) f(std::integral_constant<int, ZKB_VALUE_BF16>());
    else if (type == ZKB_VALUE_WORD) f(std::integral_constant<int, ZKB_VALUE_WORD>());
    else if (INT4 || type == ZKB_VALUE_F32) f(std::integral_constant<int, ZKB_VALUE_F32>());
    else f(std::integral_constant<int, ZKB_VALUE_INT32>());
}

// VEC: 4-bit weights whose rows start on 16-byte boundaries.
template <bool INT4, int N, bool TMA, bool VEC>
__global__ void __launch_bounds__((Tile<INT4, N, TMA>::THREADS), (Tile<INT4, N, TMA>::BLOCKS))
    product_tiles_kernel(const __grid_constant__ zkb_step_product_args a, const __grid_constant__ ProductMaps maps, uint32_t row_tiles, uint32_t all_tiles, unsigned* dev_err) {
    using T = Tile<INT4, N, TMA>;
    extern __shared__ unsigned char tiles_sm[];
    __shared__ __align__(8) TileBars bars;
    __shared__ uint32_t tmem_sm;
    unsigned char* const sm = tiles_sm + (-(uint32_t)__cvta_generic_to_shared(tiles_sm) & 1023);
    const uint32_t ring = (uint32_t)__cvta_generic_to_shared(sm);
    uint32_t* const join = reinterpret_cast<uint32_t*>(sm + T::STAGES * T::STAGE);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint32_t rank = cluster_rank(), ranks = cluster_ranks();
    if (warp == T::EPI + 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"((uint32_t)__cvta_generic_to_shared(&tmem_sm)), "n"(T::COLUMNS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    } else if (warp == 0 && lane == 0) {
        for (int i = 0; i < 6; i++) mbar_init(bar_of(bars.full[i]), (TMA ? 1 : 0) + T::FILLERS), mbar_init(bar_of(bars.empty[i]), 1);
        for (int i = 0; i < 4; i++) mbar_init(bar_of(bars.sum_full[i]), 1), mbar_init(bar_of(bars.sum_empty[i]), 32 * T::EPI);
        mbar_init(bar_of(bars.last), 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    bool failed = false;  // a wait ran out: what follows is not valid, and nothing more is waited for
    auto wait = [&](const unsigned long long& b, uint32_t parity) {
        if (!failed) failed = !mbar_wait(bar_of(b), parity & 1);
        failed = __any_sync(0xffffffffu, failed);
    };
    tmem_fence_before();
    __syncthreads();
    tmem_fence_after();
    if (ranks > 1) cluster_arrive();
    const uint32_t tmem = tmem_sm;
    const uint32_t all_steps = (a.n_in + 127) / 128, who = blockIdx.x / ranks, every = gridDim.x / ranks;
    const uint32_t first_step = rank * all_steps / ranks, steps = (rank + 1) * all_steps / ranks - first_step;
    const uint32_t n_tiles = who < all_tiles ? (all_tiles - who + every - 1) / every : 0, items = n_tiles * steps;
    auto tile_at = [&](uint32_t i, uint32_t& row_tile, uint32_t& out_tile) {
        const uint32_t tile = who + i * every;
        row_tile = tile % row_tiles, out_tile = tile / row_tiles;
    };

    if (warp < T::EPI) {  // ---- the sums: a thread has an output, and half of the rows where two threads share it
        constexpr int MINE = N / (T::EPI / 4), CHUNK = MINE < 32 ? 8 : 32;
        const uint32_t c128 = (uint32_t)(warp & 3) * 32 + lane, half = (uint32_t)(warp >> 2) * MINE, at_lanes = tmem + ((uint32_t)(warp & 3) << 21) + half;
        uint32_t done = 0;  // sums read
        for (uint32_t i = 0; i < n_tiles; i++) {
            uint32_t row_tile, out_tile;
            tile_at(i, row_tile, out_tile);
            const uint32_t c = out_tile * 128 + c128, t0 = row_tile * N + half;
            const bool live = c < a.n_out;
            uint32_t x[CHUNK];
            // the sums of columns `from` on, CHUNK at a time, to `use`
            auto read = [&](auto use) {
                const uint32_t buf = done % T::SUMS;
                wait(bars.sum_full[buf], done / T::SUMS);
                tmem_fence_after();
#pragma unroll
                for (int j = 0; j < MINE; j += CHUNK) {
                    if constexpr (CHUNK == 32) tmem_load32(at_lanes + buf * N + j, x);
                    else tmem_load8(at_lanes + buf * N + j, x);
                    tmem_loaded(x);
                    if (j + CHUNK == MINE) {
                        tmem_fence_before();
                        mbar_arrive(bar_of(bars.sum_empty[buf]));
                    }
                    use(j);
                }
                done++;
            };
            auto share = [&](int column, uint32_t word) {  // to the thread block that adds up this row
                const uint32_t of = N / ranks, to = column / of;
                peer_store_word(join + (rank * of + column % of) * 128 + c128, (int)to, word);
            };
            if constexpr (INT4) {
                float acc[MINE];
#pragma unroll
                for (int j = 0; j < MINE; j++) acc[j] = 0.f;
                const uint32_t groups = (a.n_in + a.group - 1) / a.group, per = 128 / a.group;
                const uint16_t* const scales = static_cast<const uint16_t*>(a.w_scale) + (int64_t)min(c, a.n_out - 1) * a.w_scale_stride;
                const uint32_t g0 = first_step * per, g1 = min((first_step + steps) * per, groups);
                uint32_t scale = g0 < g1 ? scales[g0] : 0u;
#pragma unroll 1
                for (uint32_t g = g0; g < g1; g++) {
                    const float by = __uint_as_float(scale << 16) * 0.0625f;  // (the codes are 16 times themselves)
                    scale = g + 1 < g1 ? scales[g + 1] : 0u;
                    read([&](int j) {
#pragma unroll
                        for (int y = 0; y < CHUNK; y++) acc[j + y] = fmaf((float)(int)x[y], by, acc[j + y]);
                    });
                }
                if (ranks == 1) {
                    if (live)
                        by_type<INT4>(a.out_type, [&](auto type) {
#pragma unroll
                            for (int j = 0; j < MINE; j++)
                                if (t0 + j < a.n_rows) put<decltype(type)::value, INT4>(a, t0 + j, c, __float_as_uint(acc[j]), 1.f);
                        });
                } else if constexpr (T::JOIN > 0) {
                    cluster_wait();
#pragma unroll
                    for (int j = 0; j < MINE; j++) share(j, __float_as_uint(acc[j]));
                }
            } else {
                const float by = live && a.w_scale ? static_cast<const float*>(a.w_scale)[c] : 1.f;
                if (ranks == 1) {
                    read([&](int j) {
                        if (live)
                            by_type<INT4>(a.out_type, [&](auto type) {
#pragma unroll
                                for (int y = 0; y < CHUNK; y++)
                                    if (t0 + j + y < a.n_rows) put<decltype(type)::value, INT4>(a, t0 + j + y, c, x[y], by);
                            });
                    });
                } else if constexpr (T::JOIN > 0) {
                    cluster_wait();
                    read([&](int j) {
#pragma unroll
                        for (int y = 0; y < CHUNK; y++) share(j + y, x[y]);
                    });
                }
            }
        }
    } else if (warp == T::EPI) {  // ---- copies
        if constexpr (TMA) {
            uint32_t sent = 0;
            for (uint32_t i = 0; i < items; i++) {
                const uint32_t st = i % T::STAGES, step = first_step + i % steps;
                uint32_t row_tile, out_tile;
                tile_at(i / steps, row_tile, out_tile);
                wait(bars.empty[st], i / T::STAGES + 1);
                if (failed) break;
                sent = i + 1;
                if (lane == 0) {
                    const uint32_t to = ring + st * T::STAGE, bar = bar_of(bars.full[st]);
                    mbar_expect(bar, INT4 ? T::B : T::STAGE);
                    if constexpr (!INT4) tma_load_2d(to, &maps.w, step * 128, out_tile * 128, bar);
                    tma_load_2d(to + T::A, &maps.x, step * 128, row_tile * N, bar);
                }
                __syncwarp();
            }
            // Whatever is on its way comes to its place before the thread block ends, though a wait may have run out.
            for (uint32_t j = sent < T::STAGES ? 0 : sent - T::STAGES; j < sent; j++) mbar_wait(bar_of(bars.full[j % T::STAGES]), (j / T::STAGES) & 1);
        }
    } else if (warp == T::EPI + 1) {  // ---- products
        constexpr uint32_t high = (1024u >> 4) | 1u << 14 | 2u << 29, desc = codes_desc(N);
        const uint32_t a_low = (ring >> 4 & 0x3fff) | 1u << 16, tmem_u = __shfl_sync(0xffffffffu, tmem, 0);
        const bool one = elect_one();
        uint32_t done = 0;
#pragma unroll 1
        for (uint32_t i = 0; i < items; i++) {
            const uint32_t st = i % T::STAGES, in_tile = i % steps;
            const uint32_t from_a = a_low + st * (T::STAGE >> 4), from_b = from_a + (T::A >> 4);
            if constexpr (!INT4) {
                if (in_tile == 0) wait(bars.sum_empty[done % T::SUMS], done / T::SUMS + 1);
            }
            wait(bars.full[st], i / T::STAGES);
            if (failed) break;
            tmem_fence_after();
            if constexpr (INT4) {
                const uint32_t left = min(128u, a.n_in - (first_step + in_tile) * 128), groups = (left + a.group - 1) / a.group, parts = a.group / 32;
                for (uint32_t g = 0; g < groups; g++) {
                    wait(bars.sum_empty[done % T::SUMS], done / T::SUMS + 1);
                    if (failed) break;
                    tmem_fence_after();
                    for (uint32_t k = 0; k < parts; k++) {
                        const uint32_t at = 2 * (g * parts + k);
                        product_codes(one, tmem_u + done % T::SUMS * N, two_words(from_a + at, high), two_words(from_b + at, high), desc, k > 0);
                    }
                    if (one) products_done(bar_of(bars.sum_full[done % T::SUMS]));
                    done++;
                }
                if (one) products_done(bar_of(bars.empty[st]));
            } else {
#pragma unroll
                for (uint32_t k = 0; k < 4; k++)
                    product_codes(one, tmem_u + done % T::SUMS * N, two_words(from_a + 2 * k, high), two_words(from_b + 2 * k, high), desc, in_tile > 0 || k > 0);
                if (one) {
                    products_done(bar_of(bars.empty[st]));
                    if (in_tile + 1 == steps) products_done(bar_of(bars.sum_full[done % T::SUMS]));
                }
                if (in_tile + 1 == steps) done++;
            }
            __syncwarp();
        }
        // Nothing is at work in tensor memory when the thread block gives it up, though a wait may have run out.
        if (one) products_done(bar_of(bars.last));
        __syncwarp();
        mbar_wait(bar_of(bars.last), 0);
    } else if constexpr (T::FILLED) {  // ---- codes into shared memory
        const int f = threadIdx.x - 32 * (T::EPI + 2);
        const int64_t w_row = INT4 ? a.w_stride / 2 : a.w_stride;
        const int bytes = INT4 ? (int)(a.n_in + 1) / 2 : (int)a.n_in;
        constexpr int STEP = INT4 ? 64 : 128, ROW = STEP / 16, MINE = 128 * ROW / T::FILLERS;  // bytes of a row's step, 16s of them, a thread's
        constexpr int AHEAD = VEC ? 4 : 1;
        auto load_w = [&](uint32_t i, uint4 (&v)[MINE]) {
            uint32_t row_tile, out_tile;
            tile_at(i / steps, row_tile, out_tile);
            const int step = (int)(first_step + i % steps);
#pragma unroll
            for (int j = 0; j < MINE; j++) {
                const int q = f + j * T::FILLERS, row = q / ROW, b = step * STEP + q % ROW * 16;
                const int8_t* const from = static_cast<const int8_t*>(a.w) + (int64_t)min(out_tile * 128 + row, a.n_out - 1) * w_row + b;
                v[j] = b < bytes ? load16<VEC>(from, bytes - b, b >= 4 && b + 20 <= bytes) : make_uint4(0u, 0u, 0u, 0u);
            }
        };
        uint4 v[AHEAD][MINE];
        if constexpr (VEC) {
#pragma unroll
            for (int j = 0; j < AHEAD; j++)
                if (j < (int)items) load_w(j, v[j]);
        }
#pragma unroll 1
        for (uint32_t i0 = 0; i0 < items; i0 += AHEAD) {
#pragma unroll
            for (int k = 0; k < AHEAD; k++) {
                const uint32_t i = i0 + k, st = i % T::STAGES;
                if (i >= items) break;
                if constexpr (!VEC) load_w(i, v[0]);
                wait(bars.empty[st], i / T::STAGES + 1);
                if (failed) break;
                const uint32_t to = ring + st * T::STAGE;
#pragma unroll
                for (int j = 0; j < MINE; j++) {
                    const int q = f + j * T::FILLERS, row = q / ROW, b = q % ROW * 16;
                    if constexpr (INT4) {
                        const uint32_t w[4] = {v[k][j].x, v[k][j].y, v[k][j].z, v[k][j].w};
                        uint32_t u[8];
#pragma unroll
                        for (int y = 0; y < 4; y++) {
                            const uint32_t even = w[y] << 4 & 0xf0f0f0f0u, odd = w[y] & 0xf0f0f0f0u;
                            u[2 * y] = __byte_perm(even, odd, 0x5140), u[2 * y + 1] = __byte_perm(even, odd, 0x7362);
                        }
                        st_shared4(to + box_place<128>(row, 2 * b), u[0], u[1], u[2], u[3]);
                        st_shared4(to + box_place<128>(row, 2 * b + 16), u[4], u[5], u[6], u[7]);
                    } else {
                        st_shared4(to + box_place<128>(row, b), v[k][j].x, v[k][j].y, v[k][j].z, v[k][j].w);
                    }
                }
                if constexpr (!TMA) {
                    uint32_t row_tile, out_tile;
                    tile_at(i / steps, row_tile, out_tile);
                    const int step = (int)(first_step + i % steps);
#pragma unroll 4
                    for (int q = f; q < N * 8; q += T::FILLERS) {
                        const int row = q / 8, b = q % 8 * 16, at = step * 128 + b;
                        const int8_t* const from = a.x + (int64_t)min(row_tile * N + row, a.n_rows - 1) * a.x_stride + at;
                        const uint4 u = at < (int)a.n_in ? load16<false>(from, (int)a.n_in - at, at >= 4 && at + 20 <= (int)a.n_in) : make_uint4(0u, 0u, 0u, 0u);
                        st_shared4(to + T::A + box_place<128>(row, b), u.x, u.y, u.z, u.w);
                    }
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                mbar_arrive(bar_of(bars.full[st]));
                if constexpr (VEC) {
                    if (i + AHEAD < items) load_w(i + AHEAD, v[k]);
                }
            }
            if (failed) break;
        }
    }
    __syncwarp();
    if (ranks > 1) {
        if (warp >= T::EPI || n_tiles == 0) cluster_wait();
        cluster_arrive(), cluster_wait();
        if constexpr (T::JOIN > 0) {
            uint32_t row_tile, out_tile;
            tile_at(0, row_tile, out_tile);
            const uint32_t c128 = threadIdx.x, c = out_tile * 128 + c128, of = N / ranks;
            if (warp < T::EPI && c < a.n_out) {
                const float by = !INT4 && a.w_scale ? static_cast<const float*>(a.w_scale)[c] : 1.f;
                by_type<INT4>(a.out_type, [&](auto type) {
                    for (uint32_t j = 0; j < of; j++) {
                        const uint32_t t = row_tile * N + rank * of + j;
                        if (t >= a.n_rows) break;
                        uint32_t word = join[j * 128 + c128];
                        for (uint32_t r = 1; r < ranks; r++) {
                            const uint32_t more = join[(r * of + j) * 128 + c128];
                            word = INT4 ? __float_as_uint(__uint_as_float(word) + __uint_as_float(more)) : word + more;
                        }
                        put<decltype(type)::value, INT4>(a, t, c, word, by);
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

// A map of rows of codes in boxes of `rows` rows by 128, or false where the layout has none: the unit wants 16-byte boundaries.
static bool rows_map(CUtensorMap& map, const void* p, uint32_t codes, uint32_t n_rows, int64_t stride, uint32_t rows) {
    const TensorMapEncode encode = tensor_map_encode();
    if (n_rows == 1) stride = (codes + 15) / 16 * 16;
    if (!encode || !aligned_to(p, 16) || stride % 16 != 0 || stride >= (1ll << 40)) return false;
    const cuuint64_t dims[2] = {codes, n_rows}, strides[1] = {(cuuint64_t)stride};
    const cuuint32_t boxes[2] = {128, rows}, ones[2] = {1, 1};
    return encode(&map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(p), dims, strides, boxes, ones, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <bool INT4, int N, bool TMA, bool VEC>
static cudaError_t launch_variant(zkb_ctx* ctx, const zkb_step_product_args& a, const ProductMaps& maps) {
    using T = Tile<INT4, N, TMA>;
    auto kernel = product_tiles_kernel<INT4, N, TMA, VEC>;
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, T::SMEM);
    if (e != cudaSuccess) return e;
    const uint32_t row_tiles = (a.n_rows + N - 1) / N, tiles = row_tiles * ((a.n_out + 127) / 128), steps = (a.n_in + 127) / 128;
    // Few tiles are spread over clusters, while all of them are on the GPU at once and each thread block has two steps.
    uint32_t ranks = 1;
    if (T::JOIN > 0)
        while (ranks < 16 && ranks < N && tiles <= T::BLOCKS * clusters_at_once(2 * ranks) && steps >= 4 * ranks) ranks *= 2;
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
    const bool x = rows_map(maps.x, a.x, a.n_in, a.n_rows, a.x_stride, N);
    if constexpr (INT4) {
        const bool vec = aligned_to(a.w, 16) && (a.n_out == 1 || a.w_stride % 32 == 0);
        return x && vec ? launch_variant<true, N, true, true>(ctx, a, maps) : launch_variant<true, N, false, false>(ctx, a, maps);
    } else {
        return x && rows_map(maps.w, a.w, a.n_in, a.n_out, a.w_stride, 128) ? launch_variant<false, N, true, true>(ctx, a, maps) : launch_variant<false, N, false, false>(ctx, a, maps);
    }
}

template <bool INT4>
cudaError_t launch_tiles(zkb_ctx* ctx, const zkb_step_product_args& a) {
    // As many rows a tile as there are, up to 256 (4-bit weights 128: a group's sums are kept in registers); fewer while that leaves SMs without a tile.
    uint32_t n = 16;
    while (n < (INT4 ? 128u : 256u) && n < a.n_rows) n *= 2;
    while (n > 32 && (uint64_t)((a.n_rows + n - 1) / n) * ((a.n_out + 127) / 128) < 120) n /= 2;
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
