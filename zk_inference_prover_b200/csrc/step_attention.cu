// Attention of a step's rows over the key-value cache.
#include <algorithm>
#include <cmath>
#include <cstdlib>

#include "step_attention.cuh"

namespace zk {

TensorMapEncode tensor_map_encode() {
    static const TensorMapEncode encode = [] {
        void* f = nullptr;
        cudaDriverEntryPointQueryResult found;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &found) != cudaSuccess || found != cudaDriverEntryPointSuccess) f = nullptr;
        return (TensorMapEncode)f;
    }();
    return encode;
}

bool cache_maps(CacheMaps& maps, const zkb_kv_cache& c, uint32_t tokens) {
    const TensorMapEncode encode = tensor_map_encode();
    const bool int8 = c.type == ZKB_VALUE_INT8;
    const int64_t size = int8 ? 1 : 2, row = c.head_dim * size, box = std::min<int64_t>(row, 128);
    // a dimension of one entry has no stride to speak of
    const int64_t token = c.capacity > 1 ? c.token_stride * size : row, head = c.n_heads > 1 ? c.head_stride * size : row, seq = c.n_seqs > 1 ? c.seq_stride * size : row;
    for (int64_t s : {token, head, seq})
        if (s <= 0 || s % 16 != 0 || s >= (1ll << 40)) return false;
    if (!encode || !aligned_to(c.k, 16) || !aligned_to(c.v, 16)) return false;
    const cuuint64_t dims[4] = {c.head_dim, c.capacity, c.n_heads, c.n_seqs}, strides[3] = {(cuuint64_t)token, (cuuint64_t)head, (cuuint64_t)seq};
    const cuuint32_t boxes[4] = {(cuuint32_t)(box / size), tokens, 1, 1}, ones[4] = {1, 1, 1, 1};
    const CUtensorMapSwizzle swizzle = box == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : box == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_NONE;
    for (int i = 0; i < 2; i++)
        if (encode(i ? &maps.v : &maps.k, int8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, i ? c.v : c.k, dims, strides, boxes, ones, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle,
                   CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
            return false;
    return true;
}

// ---- few rows: one token, or a few, of each sequence -----------------------------------------------------------------------------------
// The cache is read once and everything else is small, so this is bound by the cache's bytes. Eight query rows (the heads of a kv head's
// group, of one token or several) are the N of mma.m16n8k16 and sixteen keys its M, S^T = K Q^T, O^T = V^T P^T:
//   K: lane (g, t) takes keys g and g + 8 and a quarter of their dimensions; which dimension is which k of the product is free as long as Q agrees.
//   V: lane (g, t) takes keys 2t, 2t + 1, 2t + 8, 2t + 9, and an eighth of their dimensions; two keys' values make a register of the product.
// P^T is S^T's registers transposed eight by eight (movmatrix). Each warp takes every W-th block of sixteen keys, with its own running maximum and
// sum, and its own ring in shared memory that the tensor memory unit fills two blocks ahead (copies by the lanes themselves came to 26 bytes a clock
// and SM): nothing waits for other warps. Warps join through shared memory, thread blocks of a cluster by writing into each other's, so that
// a long sequence is spread over up to 16 SMs without a workspace or a second launch.
// 64 sequences of 4,096 to 8,192 bf16 tokens, 32 heads on 8 of 128, call after call: 243 us, 6.6 TB/s, a copy's rate; int8 tokens 171 us, 4.9 TB/s: each of the two products for a warp's sixteen keys
// waits for the conversion of its codes, which take turns in one warp, and issue slots are busy to 57 %. One sequence of 2,048 int8 tokens: 8.9 us, most of it the launch and the joining.
constexpr int FEW_WARPS = 8, FEW_RANKS = 16;
constexpr float NO_SCORE = -3.40282346e38f;  // of a hidden key, the lowest number: a visible one's may be -inf; both weigh nothing

// T: how many times eight rows a thread block has for the keys that it reads.
template <int D, bool INT8, int T>
struct Few {
    static constexpr int ROWS = 8 * T;
    static constexpr int SIZE = INT8 ? 1 : 2;
    static constexpr int ROW = D * SIZE, BOX = ROW < 128 ? ROW : 128, BOXES = ROW / BOX;  // bytes of a token and head, and of a box's row
    static constexpr int KW = ROW / 16, VW = ROW / 32, KB = KW / BOXES, VB = VW / BOXES;  // words a lane and key, in all and in a box
    static constexpr int TILE = 16 * ROW;  // bytes of sixteen keys of K or of V
    static constexpr int THREAD_BLOCKS = TILE <= 2048 && T == 1 ? 2 : 1;  // an SM
    static constexpr int STAGES = 3;
    static constexpr int JOIN = FEW_WARPS * ROWS * (D + 4) * 4;  // the warps' sums, after the rings are done with
    static constexpr int RING = FEW_WARPS * STAGES * 2 * TILE;
    static constexpr int SMEM = 1024 + (RING > JOIN ? RING : JOIN);  // boxes start on 1024 bytes
};

// WORDS words from byte `at` of a row on.
template <int BOX, int WORDS>
__device__ __forceinline__ void read_row(uint32_t box, int row, int at, uint32_t* w) {
    if constexpr (WORDS >= 4) {
#pragma unroll
        for (int x = 0; x < WORDS; x += 4) ld_shared4(box + box_place<BOX>(row, at + 4 * x), w[x], w[x + 1], w[x + 2], w[x + 3]);
    } else if constexpr (WORDS == 2) {
        ld_shared2(box + box_place<BOX>(row, at), w[0], w[1]);
    } else {
        w[0] = ld_shared(box + box_place<BOX>(row, at));
    }
}

template <int D, bool INT8, int T, bool TMA>
__global__ void __launch_bounds__(FEW_WARPS * 32, (Few<D, INT8, T>::THREAD_BLOCKS))
    attention_few_kernel(const __grid_constant__ zkb_step_attention_args a, const __grid_constant__ CacheMaps maps, unsigned* dev_err) {
    using F = Few<D, INT8, T>;
    constexpr int STEPS = D / 16, STRIDE = D + 4, ROWS = F::ROWS;
    extern __shared__ unsigned char few_sm[];
    __shared__ float top_sm[FEW_WARPS][ROWS], sum_sm[FEW_WARPS][ROWS], all_top[ROWS], all_sum[ROWS];
    __shared__ float in_o[ROWS * D], in_top[FEW_RANKS][ROWS], in_sum[FEW_RANKS][ROWS];  // what the cluster's thread blocks write here: [rank][this one's part]
    __shared__ int in_odd[FEW_RANKS];  // some value of V was no number
    __shared__ __align__(8) unsigned long long full[FEW_WARPS][F::STAGES];
    __shared__ float scale_sm[INT8 ? FEW_WARPS * F::STAGES * 32 : 1];
    float* const o_sm = reinterpret_cast<float*>(few_sm + (-(uintptr_t)__cvta_generic_to_shared(few_sm) & 1023));  // [warp][row][dimension], where the rings were
    const zkb_kv_cache& c = a.cache;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    const int seq = blockIdx.z, kv_head = blockIdx.y, group = (int)(a.q_heads / c.n_heads);
    const int rank = (int)cluster_rank(), ranks = (int)cluster_ranks();
    if (ranks > 1) cluster_arrive();  // "I have begun": waited for before the first word goes to another thread block
    const uint32_t ring = (uint32_t)__cvta_generic_to_shared(o_sm) + warp * F::STAGES * 2 * F::TILE, bars = (uint32_t)__cvta_generic_to_shared(&full[warp][0]);
    const uint32_t scale_ring = (uint32_t)__cvta_generic_to_shared(&scale_sm[0]) + warp * F::STAGES * 128;
    if (TMA && lane == 0) {
#pragma unroll
        for (int i = 0; i < F::STAGES; i++) mbar_init(bars + 8 * i, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    __syncwarp();
    const StepSequence s = step_sequence(a.rows, seq);
    const char* const k = static_cast<const char*>(c.k) + (seq * c.seq_stride + kv_head * c.head_stride) * F::SIZE;
    const char* const v = static_cast<const char*>(c.v) + (seq * c.seq_stride + kv_head * c.head_stride) * F::SIZE;
    const float* const scales = INT8 ? (lane < 16 ? c.k_scale : c.v_scale) + seq * c.scale_seq_stride + kv_head * c.scale_head_stride : nullptr;
    const int row_bytes = (int)c.token_stride * F::SIZE;
    const int64_t n_m = (int64_t)s.rows * group, m_step = (int64_t)(gridDim.x / ranks) * ROWS;  // below 2^31, so that rows are found by 32-bit divisions
    auto token = [&](int64_t m) { return (int)((uint32_t)m / (uint32_t)group); };
    const float by = a.scale * 1.44269504f;
    const uint32_t c128 = bf16_128(), c1152 = f16_1152();
    int stage = 0;
    uint32_t parity = 0;
    bool failed = false;  // a copy never came: what follows is not valid, and nothing more is waited for
    // Sixteen keys from `base` on into a stage of the ring. Tokens behind the last one are whatever the cache holds, or zeros behind its capacity: they are masked.
    auto copy = [&](int st, int base, int last) {
        const uint32_t to = ring + st * 2 * F::TILE;
        if constexpr (TMA) {
            if (lane == 0) {
                mbar_expect(bars + 8 * st, 2 * F::TILE);
#pragma unroll
                for (int x = 0; x < F::BOXES; x++) {
                    tma_load(to + x * 16 * F::BOX, &maps.k, x * (F::BOX / F::SIZE), base, kv_head, seq, bars + 8 * st);
                    tma_load(to + F::TILE + x * 16 * F::BOX, &maps.v, x * (F::BOX / F::SIZE), base, kv_head, seq, bars + 8 * st);
                }
            }
        } else {
            for (int i = lane; i < 2 * F::TILE / 4; i += 32) {  // any layout: a word from its bytes
                const int kv = i / (F::TILE / 4), row = i % (F::TILE / 4) / (F::ROW / 4), at = i % (F::ROW / 4) * 4;
                const uint8_t* b = reinterpret_cast<const uint8_t*>((kv ? v : k) + (int64_t)min(base + row, last) * row_bytes + at);
                st_shared(to + kv * F::TILE + at / F::BOX * 16 * F::BOX + box_place<F::BOX>(row, at % F::BOX), (uint32_t)b[0] | (uint32_t)b[1] << 8 | (uint32_t)b[2] << 16 | (uint32_t)b[3] << 24);
            }
        }
        if constexpr (INT8) asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(scale_ring + st * 128 + 4 * lane), "l"(scales + min(base + (lane & 15), last)) : "memory");
    };
    bool begun = ranks == 1;
    for (int64_t m0 = (int64_t)(blockIdx.x / ranks) * ROWS; m0 < n_m; m0 += m_step) {
        const int64_t pos_low = s.pos + token(m0), pos_high = s.pos + token(min(m0 + ROWS, n_m) - 1);
        const KeyBlocks blocks = key_blocks<16>(pos_low, pos_high, c.capacity, a.window, a.sinks);
        const int stride = ranks * FEW_WARPS, last = (int)blocks.end - 1, n_blocks = failed ? 0 : blocks.n;
        const int at0 = rank * FEW_WARPS + warp;
#pragma unroll
        for (int i = 0; i < F::STAGES - 1; i++) {
            if (at0 + i * stride < n_blocks) copy(stage + i < F::STAGES ? stage + i : stage + i - F::STAGES, blocks.base(at0 + i * stride), last);
            asm volatile("cp.async.commit_group;" ::: "memory");
        }
        // Q: lane (g, t) has row g's dimensions (of each eight rows) in the order in which its K quarter comes
        uint32_t q[T][STEPS][2];
        float by_row[T][2];
#pragma unroll
        for (int n = 0; n < T; n++) {
            constexpr int BOX_DIMS = F::BOX / F::SIZE, LANE_DIMS = BOX_DIMS / 4;
            const int64_t m = m0 + 8 * n + g;
            const int i0 = m < n_m ? token(m) : 0;
            const uint16_t* from = static_cast<const uint16_t*>(a.q) + (m < n_m ? (s.first + i0) * a.q_stride + (kv_head * group + (int)m - i0 * group) * a.q_head_stride : 0);
            const bool quads = ((uintptr_t)from & 7) == 0;
#pragma unroll
            for (int i = 0; i < STEPS; i++) {
                const int d = (4 * i / LANE_DIMS) * BOX_DIMS + t * LANE_DIMS + 4 * i % LANE_DIMS;
                uint2 w = make_uint2(0u, 0u);
                if (m < n_m) {
                    if (quads) w = *reinterpret_cast<const uint2*>(from + d);
                    else w = make_uint2((uint32_t)from[d] | (uint32_t)from[d + 1] << 16, (uint32_t)from[d + 2] | (uint32_t)from[d + 3] << 16);
                }
                q[n][i][0] = INT8 ? __byte_perm(w.x, w.y, 0x5410) : w.x;  // codes_to_f16's order
                q[n][i][1] = INT8 ? __byte_perm(w.x, w.y, 0x7632) : w.y;
            }
            by_row[n][0] = by_row[n][1] = by;
            if constexpr (INT8) {
                // Codes are cheaper to have in fp16, so Q is taken there too, each row times the power of two that brings its largest value to 2^13: exact down to
                // 2^-27 of that value, and below it off by 2^-38 of it.
                float most = 0.f;
#pragma unroll
                for (int i = 0; i < 2 * STEPS; i++) most = fmaxf(most, fmaxf(fabsf(bf16_low(q[n][i / 2][i & 1])), fabsf(bf16_high(q[n][i / 2][i & 1]))));
                most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
                most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
                const int e = (int)(__float_as_uint(most) >> 23);  // 0: all zero or nearly; 255: an infinity, which stays one
                const int up = e == 0 || e == 255 ? 0 : min(13 + 127 - e, 126);
                const float f = __uint_as_float((uint32_t)(up + 127) << 23);
#pragma unroll
                for (int i = 0; i < 2 * STEPS; i++) q[n][i / 2][i & 1] = pack_f16(bf16_low(q[n][i / 2][i & 1]) * f, bf16_high(q[n][i / 2][i & 1]) * f);
#pragma unroll
                for (int r = 0; r < 2; r++) by_row[n][r] = by * __uint_as_float((uint32_t)(127 - __shfl_sync(0xffffffffu, up, (2 * t + r) * 4)) << 23);
            }
        }
        // rows 2t and 2t + 1 (of each eight): their positions, running maxima and this lane's part of their sums
        int p[T][2];
        float top[T][2], less[T][2], sum[T][2], o[T][STEPS][4];
#pragma unroll
        for (int n = 0; n < T; n++) {
#pragma unroll
            for (int r = 0; r < 2; r++) {
                const int64_t m = m0 + 8 * n + 2 * t + r;
                p[n][r] = m < n_m ? (int)s.pos + token(m) : -1;
                top[n][r] = NO_SCORE, less[n][r] = 0.f, sum[n][r] = 0.f;
            }
#pragma unroll
            for (int i = 0; i < STEPS; i++)
#pragma unroll
                for (int x = 0; x < 4; x++) o[n][i][x] = 0.f;
        }
        bool odd = false;
        const int whole_to = (int)min(pos_low, (int64_t)last) - 15, whole_from = a.window ? (int)max((int64_t)0, pos_high - (int64_t)a.window + 1) : 0;  // blocks that all rows see
        for (int at = at0; at < n_blocks; at += stride) {
            const int base = blocks.base(at), ahead = at + (F::STAGES - 1) * stride;
            const uint32_t here = ring + stage * 2 * F::TILE, scales_here = scale_ring + stage * 128 + 4 * g;
            if (ahead < n_blocks) copy(stage == 0 ? F::STAGES - 1 : stage - 1, blocks.base(ahead), last);
            asm volatile("cp.async.commit_group;" ::: "memory");
            asm volatile("cp.async.wait_group %0;" ::"n"(F::STAGES - 1) : "memory");
            __syncwarp();
            if (TMA && __any_sync(0xffffffffu, !mbar_wait(bars + 8 * stage, parity))) {
                failed = true;  // the copies that are still on their way come first (a stage that has none takes the wait's limit)
                for (int i = 0; i < F::STAGES; i++) mbar_wait(bars + 8 * i, i < stage ? parity ^ 1 : parity);
                break;
            }
            if (++stage == F::STAGES) stage = 0, parity ^= 1;
            float sc[T][4] = {}, sc2[T][4] = {};
            {
                uint32_t k0[F::KW], k1[F::KW];
#pragma unroll
                for (int x = 0; x < F::BOXES; x++) {
                    read_row<F::BOX, F::KB>(here + x * 16 * F::BOX, g, t * F::KB * 4, k0 + x * F::KB);
                    read_row<F::BOX, F::KB>(here + x * 16 * F::BOX, g + 8, t * F::KB * 4, k1 + x * F::KB);
                }
#pragma unroll
                for (int i = 0; i < STEPS; i++) {
                    uint32_t f[4];
                    if constexpr (INT8) {
                        codes_to_f16(k0[i], c1152, f[0], f[2]);
                        codes_to_f16(k1[i], c1152, f[1], f[3]);
#pragma unroll
                        for (int n = 0; n < T; n++) mma_f16(i & 1 ? sc2[n] : sc[n], f, q[n][i][0], q[n][i][1]);
                    } else {
                        f[0] = k0[2 * i], f[1] = k1[2 * i], f[2] = k0[2 * i + 1], f[3] = k1[2 * i + 1];
#pragma unroll
                        for (int n = 0; n < T; n++) mma_bf16(i & 1 ? sc2[n] : sc[n], f, q[n][i][0], q[n][i][1]);
                    }
                }
            }
            float k_by[2] = {1.f, 1.f}, v_by[2] = {1.f, 1.f};  // keys g and g + 8
            if constexpr (INT8) {
                k_by[0] = __uint_as_float(ld_shared(scales_here)), k_by[1] = __uint_as_float(ld_shared(scales_here + 32));
                v_by[0] = __uint_as_float(ld_shared(scales_here + 64)), v_by[1] = __uint_as_float(ld_shared(scales_here + 96));
            }
            uint32_t w[T][2], left[T][2];
#pragma unroll
            for (int n = 0; n < T; n++) {
                // z: key g with rows 2t, 2t + 1, then key g + 8
                float z[4];
#pragma unroll
                for (int i = 0; i < 4; i++) z[i] = (sc[n][i] + sc2[n][i]) * (INT8 ? by_row[n][i & 1] * k_by[i >> 1] : by);
                if (base < whole_from || base > whole_to) {
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const int key = base + g + 8 * (i >> 1), gap = p[n][i & 1] - key;
                        if (gap < 0 || key > last || (a.window != 0 && (uint32_t)gap >= a.window && (uint32_t)key >= a.sinks)) z[i] = NO_SCORE;
                    }
                }
                // The weights' common factor is 2^-top. It need not be the largest score's, only within 2^8 of it, so it is seldom that it changes.
                if (__any_sync(0xffffffffu, fmaxf(z[0], z[2]) > top[n][0] + 8.f || fmaxf(z[1], z[3]) > top[n][1] + 8.f)) {
#pragma unroll
                    for (int r = 0; r < 2; r++) {
                        float higher = fmaxf(top[n][r], fmaxf(z[r], z[r + 2]));
#pragma unroll
                        for (int x = 4; x < 32; x <<= 1) higher = fmaxf(higher, __shfl_xor_sync(0xffffffffu, higher, x));
                        const float keep = higher > top[n][r] ? exp2_fast(top[n][r] - higher) : 1.f;
                        sum[n][r] *= keep, top[n][r] = higher, less[n][r] = higher == NO_SCORE ? 0.f : higher;
#pragma unroll
                        for (int i = 0; i < STEPS; i++) o[n][i][r] *= keep, o[n][i][r + 2] *= keep;
                    }
                }
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float e = exp2_fast(z[i] - less[n][i & 1]);
                    sum[n][i & 1] += e;
                    z[i] = INT8 ? (z[i] == NO_SCORE ? 0.f : e * v_by[i >> 1]) : e;  // a hidden token's scale may be anything; a visible one's reaches the row whatever its score
                }
                // A weight is two bf16 numbers, its rounding and what that leaves: off by 2^-16 where the result's own rounding takes 2^-8. (One number alone, when it was timed: 64 sequences of
                // 8,192 int8 tokens in 164 us instead of 174, bf16 240 instead of 243, and results up to 1.6 times as far off.)
                const uint32_t high[2] = {pack_bf16(z[0], z[1]), pack_bf16(z[2], z[3])};
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    z[i] -= i & 1 ? bf16_high(high[i >> 1]) : bf16_low(high[i >> 1]);
                    if (INT8) z[i] = z[i] == z[i] ? z[i] : 0.f;  // an infinity leaves nothing
                }
#pragma unroll
                for (int i = 0; i < 2; i++) w[n][i] = transpose8(high[i]), left[n][i] = transpose8(pack_bf16(z[2 * i], z[2 * i + 1]));
            }
            uint32_t vw[4][F::VW];
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int x = 0; x < F::BOXES; x++) read_row<F::BOX, F::VB>(here + F::TILE + x * 16 * F::BOX, 2 * t + (i & 1) + 8 * (i >> 1), g * F::VB * 4, vw[i] + x * F::VB);
            if constexpr (!INT8) {
                if (base + 15 > last) {  // behind the last token the cache may hold anything
#pragma unroll
                    for (int i = 0; i < 4; i++)
#pragma unroll
                        for (int x = 0; x < F::VW; x++) vw[i][x] = base + 2 * t + (i & 1) + 8 * (i >> 1) > last ? 0u : vw[i][x];
                }
                // a value that is no number would reach the rows that do not see its key: it is set aside (put_what_is_no_number)
                uint32_t test = 0;
#pragma unroll
                for (int i = 0; i < 4; i++)
#pragma unroll
                    for (int x = 0; x < F::VW; x++) test = zero_or_nan(vw[i][x], test);
                if (__any_sync(0xffffffffu, (test & 0x7fff7fffu) != 0)) {
                    odd = true;
#pragma unroll
                    for (int i = 0; i < 4; i++)
#pragma unroll
                        for (int x = 0; x < F::VW; x++) vw[i][x] = numbers_only(vw[i][x]);
                }
            }
#pragma unroll
            for (int i = 0; i < STEPS; i++) {
                uint32_t f[4];  // dimensions 2i and 2i + 1 of the lane's, keys 2t and 2t + 1, then 2t + 8 and 2t + 9
                if constexpr (INT8) {
                    pair_codes_to_bf16(vw[0][i / 2], vw[1][i / 2], i & 1, c128, f[0], f[1]);
                    pair_codes_to_bf16(vw[2][i / 2], vw[3][i / 2], i & 1, c128, f[2], f[3]);
                } else {
                    f[0] = __byte_perm(vw[0][i], vw[1][i], 0x5410), f[1] = __byte_perm(vw[0][i], vw[1][i], 0x7632);
                    f[2] = __byte_perm(vw[2][i], vw[3][i], 0x5410), f[3] = __byte_perm(vw[2][i], vw[3][i], 0x7632);
                }
#pragma unroll
                for (int n = 0; n < T; n++) mma_bf16(o[n][i], f, w[n][0], w[n][1]), mma_bf16(o[n][i], f, left[n][0], left[n][1]);
            }
            __syncwarp();  // all lanes have read the block that the next copies go to
        }
        // join the warps
        asm volatile("cp.async.wait_all;" ::: "memory");
        if (failed && lane == 0) *dev_err = WAIT_RAN_OUT;
        const int any_odd = __syncthreads_or(odd);  // and the rings are done with
#pragma unroll
        for (int n = 0; n < T; n++) {
            constexpr int BOX_DIMS = F::BOX / F::SIZE, LANE_DIMS = BOX_DIMS / 8;
#pragma unroll
            for (int r = 0; r < 2; r++) {
#pragma unroll
                for (int x = 4; x < 32; x <<= 1) sum[n][r] += __shfl_xor_sync(0xffffffffu, sum[n][r], x);
                if (g == 0) top_sm[warp][8 * n + 2 * t + r] = top[n][r], sum_sm[warp][8 * n + 2 * t + r] = sum[n][r];
            }
#pragma unroll
            for (int i = 0; i < STEPS; i++)
#pragma unroll
                for (int x = 0; x < 4; x++) {
                    const int e = 2 * i + (x >> 1);
                    o_sm[(warp * ROWS + 8 * n + 2 * t + (x & 1)) * STRIDE + e / LANE_DIMS * BOX_DIMS + g * LANE_DIMS + e % LANE_DIMS] = o[n][i][x];
                }
        }
        __syncthreads();
        if (!begun) {
            __syncwarp();
            cluster_wait();
            begun = true;
        }
        // the warps' factors, and the row's sum
        if (threadIdx.x < ROWS) {
            const int r = threadIdx.x;
            float most = top_sm[0][r], all = 0.f, f[FEW_WARPS];
#pragma unroll
            for (int w = 1; w < FEW_WARPS; w++) most = fmaxf(most, top_sm[w][r]);
            const float base = most == NO_SCORE ? 0.f : most;
#pragma unroll
            for (int w = 0; w < FEW_WARPS; w++) f[w] = exp2_fast(top_sm[w][r] - base), all += sum_sm[w][r] * f[w];
#pragma unroll
            for (int w = 0; w < FEW_WARPS; w++) sum_sm[w][r] = f[w];
            all_top[r] = most, all_sum[r] = all;
        }
        __syncthreads();
        // this thread block's sums to whoever finishes them: outputs part, part + 1, ... of them all go to the thread block of that rank (ranks: a power of two)
        const int part_log = 31 - __clz(ROWS * D / ranks), part = 1 << part_log;
#pragma unroll
        for (int x = 0; x < ROWS * D; x += FEW_WARPS * 32) {
            const int i = x + threadIdx.x, r = i / D, d = i % D;
            float y = 0.f;
#pragma unroll
            for (int w = 0; w < FEW_WARPS; w++) y += o_sm[(w * ROWS + r) * STRIDE + d] * sum_sm[w][r];
            float* const to = &in_o[rank * part + (i & (part - 1))];
            if (ranks > 1) peer_store(to, i >> part_log, y);
            else *to = y;
        }
        for (int i = threadIdx.x; i < ROWS * ranks; i += FEW_WARPS * 32) {
            const int r = i % ROWS, to = i / ROWS;
            peer_store(&in_top[rank][r], to, all_top[r]);
            peer_store(&in_sum[rank][r], to, all_sum[r]);
            if (r == 0) peer_store(&in_odd[rank], to, any_odd);
        }
        if (TMA) asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // the next rows' copies go where the warps' sums are
        if (ranks > 1) cluster_arrive(), cluster_wait();
        else __syncthreads();
        for (int i = threadIdx.x; i < part; i += FEW_WARPS * 32) {
            const int r = (rank * part + i) / D, d = (rank * part + i) % D;
            const int64_t m = m0 + r;
            if (m >= n_m) continue;
            float most = NO_SCORE, y = 0.f, all = 0.f;
            int set_aside = 0;
            for (int x = 0; x < ranks; x++) most = fmaxf(most, in_top[x][r]);
            const float base = most == NO_SCORE ? 0.f : most;
            for (int x = 0; x < ranks; x++) {
                const float f = exp2_fast(in_top[x][r] - base);
                y += in_o[x * part + i] * f;
                all += in_sum[x][r] * f;
                set_aside |= in_odd[x];
            }
            y = all == 0.f ? 0.f : y / all;
            const int i0 = token(m);
            const int64_t to = (s.first + i0) * a.out_stride + (kv_head * group + (int)m - i0 * group) * a.out_head_stride + d;
            if (a.out_type == ZKB_VALUE_WORD) static_cast<uint32_t*>(a.out)[to] = round_bf16(y);
            else static_cast<uint16_t*>(a.out)[to] = round_bf16(y);
            if ((INT8 ? !isfinite(y) : set_aside) && all > 0.f) put_what_is_no_number<INT8>(a, to, set_aside, seq, kv_head, d, s.pos + i0);
        }
        if (m0 + m_step < n_m) {  // the next rows' sums come to the same places
            if (ranks > 1) cluster_arrive(), cluster_wait();
            else __syncthreads();
        }
    }
    if (!begun) cluster_wait();
}

// How a call is laid out: `tiles` of T times eight rows a kv head of the longest sequence, each spread over `ranks` thread blocks.
struct FewPlan {
    uint64_t len, units;
    uint32_t tiles, ranks;
};
template <int D, bool INT8, int T>
static FewPlan plan_few(const zkb_step_attention_args& a) {
    const zkb_kv_cache& c = a.cache;
    const uint32_t group = a.q_heads / c.n_heads, most = a.rows.max_rows ? std::min(a.rows.max_rows, a.rows.n_rows) : a.rows.n_rows;
    using F = Few<D, INT8, T>;
    FewPlan p;
    p.tiles = (uint32_t)std::min<uint64_t>(((uint64_t)most * group + F::ROWS - 1) / F::ROWS, 1u << 20);
    p.len = a.rows.max_len ? std::min(a.rows.max_len, c.capacity) : c.capacity;
    if (a.window) p.len = std::min<uint64_t>(p.len, (uint64_t)a.window + a.sinks + 32);
    // Split a sequence over more thread blocks while all of them are on the GPU at once and each warp keeps two blocks of keys: 16 sequences of 1,028 visible
    // bf16 tokens take 14.6 us in 128 thread blocks and 22.8 in 256, one of 2,048 int8 tokens 23.2 in 8 and 10.6 in 64.
    p.units = (uint64_t)c.n_seqs * c.n_heads * p.tiles;
    p.ranks = 1;
    while (p.ranks < FEW_RANKS && p.units <= clusters_at_once(2 * p.ranks) * F::THREAD_BLOCKS && p.len > (uint64_t)p.ranks * FEW_WARPS * 16 * 2) p.ranks *= 2;
    return p;
}

template <int D, bool INT8, int T>
static cudaError_t launch_few(zkb_ctx* ctx, const zkb_step_attention_args& a) {
    const zkb_kv_cache& c = a.cache;
    using F = Few<D, INT8, T>;
    const FewPlan plan = plan_few<D, INT8, T>(a);
    CacheMaps maps;
    const bool tma = cache_maps(maps, c, 16);
    auto kernel = tma ? attention_few_kernel<D, INT8, T, true> : attention_few_kernel<D, INT8, T, false>;
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, F::SMEM);
    if (e != cudaSuccess) return e;
    return launch_clusters(plan.ranks, [&](uint32_t n) {
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim = {n, 1, 1};
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(plan.tiles * n, c.n_heads, c.n_seqs);
        cfg.blockDim = dim3(FEW_WARPS * 32);
        cfg.dynamicSmemBytes = F::SMEM;
        cfg.stream = ctx->stream;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        return cudaLaunchKernelEx(&cfg, kernel, a, maps, ctx->dev_err);
    });
}

template <int D>
static cudaError_t launch_attention(zkb_ctx* ctx, const zkb_step_attention_args& a) {
    const zkb_kv_cache& c = a.cache;
    // Eight rows a product or 128, by what each was measured to take when the GPU is full: the first kernel 40 ns for each eight rows of a kv head and 0.04 ns for each key that they are
    // shown, the second, which starts some 12 us later, 80 ns (bf16 caches: 40) for each 256 rows and 0.2 ns (0.12) a key. The figures are those of 128 head dimensions; with fewer both kernels get
    // faster alike: over 306 batches of 128 and 153 each of 64 and 32 the rule's choice is within 1 % of the better one on the average, within 1.4 times at the worst. Eight kv heads of 128, one
    // sequence of 1,032 int8 tokens against 32 rows a head: 12.6 us and 25.5, of 8,032 against 128 rows: 60 and 46; 16 sequences of 32 bf16 tokens against 128 rows: 79 and 13; 1,024
    // sequences of 64 int8 tokens against 16 rows: 419 and 673.
    const uint32_t group = a.q_heads / c.n_heads;
    const uint64_t rows = (uint64_t)(a.rows.max_rows ? std::min(a.rows.max_rows, a.rows.n_rows) : a.rows.n_rows) * group, len = a.rows.max_len ? std::min(a.rows.max_len, c.capacity) : c.capacity;
    auto shown = [&](uint32_t tile, uint32_t block) { return a.window ? (double)std::min<uint64_t>(len, (uint64_t)a.window + a.sinks + tile / group + block) : (double)len; };
    const double of_8 = 0.04 * shown(8, 16) + 40., of_256 = c.type == ZKB_VALUE_INT8 ? 0.2 * shown(256, 128) + 80. : 0.12 * shown(256, 128) + 40.;
    const bool few = ((double)((rows + 7) / 8) * of_8 - (double)((rows + 255) / 256) * of_256) * c.n_seqs * c.n_heads < 12000.;
    if (!few) return c.type == ZKB_VALUE_INT8 ? launch_many<D, true>(ctx, a) : launch_many<D, false>(ctx, a);
    if (c.type != ZKB_VALUE_INT8) return launch_few<D, false, 1>(ctx, a);
    // Sixteen rows for each code that is turned into a 16-bit value instead of eight, with half the warps on an SM. That gains where eight rows would have thread blocks share SMs, over caches
    // long enough, and loses where half as many units spread over no more thread blocks. Eight kv heads of 128: 16 sequences of 8,008 tokens against 32 rows a head 164 us instead of 206, one of
    // 2,048 against 128 rows 20.9 instead of 23.2; but one of 8,008 against 32 rows 29.2 instead of 23.3, 48 of 1,600 against 24 rows 138 instead of 105. (675 batches of head dimensions 32 to 128:
    // within 0.4 % of the better one on the average, within 13 % at the worst.)
    const FewPlan of8 = plan_few<D, true, 1>(a), of16 = plan_few<D, true, 2>(a);
    const bool sixteen = rows > 8 && of8.len >= std::max(1500u, 256 * of8.ranks) && of8.units > clusters_at_once(of8.ranks) && of16.ranks >= of8.ranks &&
                         (of8.units <= 512 || (D == 128 && 8 * (uint64_t)of16.tiles < 5 * (uint64_t)of8.tiles));
    return sixteen ? launch_few<D, true, 2>(ctx, a) : launch_few<D, true, 1>(ctx, a);
}

}  // namespace zk

using namespace zk;

extern "C" int zkb_step_attention(zkb_ctx* ctx, const zkb_step_attention_args* args) {
    if (!ctx) return ZKB_EINVAL;
    ZKB_CHECK_ARG(ctx, args);
    const zkb_step_attention_args& a = *args;
    const zkb_kv_cache& c = a.cache;
    if (const char* why = step_problem(c, a.rows, a.q_heads)) return set_error(ctx, ZKB_EINVAL, "zkb_step_attention: %s", why);
    ZKB_CHECK_ARG(ctx, a.out_type == ZKB_VALUE_BF16 || a.out_type == ZKB_VALUE_WORD);
    ZKB_CHECK_ARG(ctx, std::isfinite(a.scale) && (uint64_t)a.rows.n_rows * a.q_heads <= 0x7fffffffu && (uint64_t)a.rows.n_rows * (a.q_heads / c.n_heads) <= 0x7fffff00u);
    if (a.rows.n_rows == 0) return ZKB_OK;
    ZKB_CHECK_ARG(ctx, a.q && a.out && aligned_to(a.q, 2) && aligned_to(a.out, a.out_type == ZKB_VALUE_WORD ? 4 : 2));
    ZKB_CHECK_ARG(ctx, a.q_heads == 1 || std::llabs(a.out_head_stride) >= (long long)c.head_dim);
    ZKB_CHECK_ARG(ctx, a.rows.n_rows == 1 || std::llabs(a.out_stride) >= (long long)c.head_dim);
    DeviceGuard g(ctx);
    ProfScope prof(ctx, "step_attention_kernel");
    ZKB_CUDA(ctx, c.head_dim == 128 ? launch_attention<128>(ctx, a) : c.head_dim == 64 ? launch_attention<64>(ctx, a) : launch_attention<32>(ctx, a));
    return ZKB_OK;
}
