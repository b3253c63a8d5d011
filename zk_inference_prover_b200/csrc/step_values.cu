// The values of a decode step: embedding rows, norms and rotation of queries and keys with the cache that they fill.
#include <algorithm>
#include <cmath>
#include <cstdlib>
#include <type_traits>

#include "step_values.cuh"

namespace zk {

// ---- embedding rows ------------------------------------------------------------------------------------------------------------------
// A row of the table is scaled, rounded and written: bound by its bytes. Eight values a thread; blockIdx.y names the run of the row, blockIdx.x the tokens, whose ids and then
// whose values are asked for together: EMBED_TOKENS loads on their way, where a load at a time left the memory waiting (16384 tokens of 4096 bf16: 40 us -> 35 us, 5.7 TB/s).
constexpr int EMBED_TOKENS = 4;
struct EmbedArgs {
    zkb_step_embed_args a;
    uint32_t tokens_a_block;  // <= EMBED_TOKENS
};

template <bool INT8, bool WORD>
__global__ void __launch_bounds__(256) embed_kernel(const __grid_constant__ EmbedArgs e) {
    const zkb_step_embed_args& a = e.a;
    const uint32_t col = (blockIdx.y * 256u + threadIdx.x) * 8u;
    const uint32_t t0 = blockIdx.x * e.tokens_a_block, t1 = min(a.n_tokens, t0 + e.tokens_a_block);
    if (col >= a.width) return;
    const int64_t at = a.segment ? (int64_t)(col / a.segment) * a.segment_stride + col % a.segment : (int64_t)col;
    int32_t id[EMBED_TOKENS];
#pragma unroll
    for (int i = 0; i < EMBED_TOKENS; i++) id[i] = t0 + i < t1 ? a.ids[t0 + i] : -1;
    uint32_t raw[EMBED_TOKENS][INT8 ? 2 : 4];
    float by[EMBED_TOKENS];
#pragma unroll
    for (int i = 0; i < EMBED_TOKENS; i++) {
        const bool inside = id[i] >= 0 && (uint32_t)id[i] < a.vocab;
        const int64_t from = (int64_t)id[i] * a.table_stride + col;
        if constexpr (INT8) {
            const uint2 w = inside ? *reinterpret_cast<const uint2*>(static_cast<const int8_t*>(a.table) + from) : make_uint2(0u, 0u);
            raw[i][0] = w.x, raw[i][1] = w.y;
            by[i] = inside ? a.row_scale[id[i]] * a.scale : 0.f;
        } else {
            const uint4 w = inside ? *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.table) + from) : make_uint4(0u, 0u, 0u, 0u);
            raw[i][0] = w.x, raw[i][1] = w.y, raw[i][2] = w.z, raw[i][3] = w.w;
            by[i] = inside ? a.scale : 0.f;
        }
    }
#pragma unroll
    for (int i = 0; i < EMBED_TOKENS; i++) {
        if (t0 + i >= t1) break;
        if ((id[i] < 0 || (uint32_t)id[i] >= a.vocab) && col == 0 && a.off_table) atomicAdd(reinterpret_cast<unsigned long long*>(a.off_table), 1ull);
        float x[8];
#pragma unroll
        for (int y = 0; y < 8; y++) {
            if constexpr (INT8) x[y] = (float)(int8_t)(raw[i][y / 4] >> (8 * (y % 4))) * by[i];
            else x[y] = (y % 2 ? bf16_high(raw[i][y / 2]) : bf16_low(raw[i][y / 2])) * by[i];
        }
        store8<WORD>(a.out, (int64_t)(t0 + i) * a.out_stride + at, x);
    }
}

// Any width, stride and alignment: a value a thread.
template <bool INT8, bool WORD>
__global__ void __launch_bounds__(256) embed_ragged_kernel(const __grid_constant__ EmbedArgs e) {
    const zkb_step_embed_args& a = e.a;
    const uint32_t col = blockIdx.y * 256u + threadIdx.x;
    const uint32_t t0 = blockIdx.x * e.tokens_a_block, t1 = min(a.n_tokens, t0 + e.tokens_a_block);
    if (col >= a.width) return;
    const int64_t at = a.segment ? (int64_t)(col / a.segment) * a.segment_stride + col % a.segment : (int64_t)col;
    for (uint32_t t = t0; t < t1; t++) {
        const int32_t id = a.ids[t];
        const bool inside = id >= 0 && (uint32_t)id < a.vocab;
        if (!inside && col == 0 && a.off_table) atomicAdd(reinterpret_cast<unsigned long long*>(a.off_table), 1ull);
        float x = 0.f;
        if (inside) {
            const int64_t from = (int64_t)id * a.table_stride + col;
            if constexpr (INT8) x = (float)static_cast<const int8_t*>(a.table)[from] * (a.row_scale[id] * a.scale);
            else x = bf16_low(static_cast<const uint16_t*>(a.table)[from]) * a.scale;
        }
        const int64_t to = (int64_t)t * a.out_stride + at;
        if constexpr (WORD) static_cast<uint32_t*>(a.out)[to] = round_bf16(x);
        else static_cast<uint16_t*>(a.out)[to] = round_bf16(x);
    }
}

// ---- norms, rotation, the cache's new tokens -------------------------------------------------------------------------------------------
struct NormRopeArgs {
    zkb_step_norm_rope_args a;
    uint32_t parts;   // warps a row
    double turns[64]; // h_inv_freq / (2 pi): turns a position
};

// The value n values of SIZE bytes behind p.
template <int SIZE>
__device__ __forceinline__ void* value_at(const void* p, int64_t n) {
    return static_cast<char*>(const_cast<void*>(p)) + n * SIZE;
}

// Four adjacent values as they lie in memory, and as floats. VEC: the address is a multiple of their size.
template <bool WORD, bool VEC>
__device__ __forceinline__ void load4(const void* p, int64_t at, uint32_t* x) {
    if constexpr (WORD) {
        const uint32_t* w = static_cast<const uint32_t*>(p) + at;
        if constexpr (VEC) {
            const uint4 v = *reinterpret_cast<const uint4*>(w);
            x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++) x[i] = w[i];
        }
    } else {
        const uint16_t* h = static_cast<const uint16_t*>(p) + at;
        if constexpr (VEC) {
            const uint2 v = *reinterpret_cast<const uint2*>(h);
            x[0] = v.x, x[1] = v.y;
        } else {
            x[0] = h[0] | (uint32_t)h[1] << 16, x[1] = h[2] | (uint32_t)h[3] << 16;
        }
    }
}
template <bool WORD>
__device__ __forceinline__ void floats4(const uint32_t* w, float* x) {
    if constexpr (WORD) {
#pragma unroll
        for (int i = 0; i < 4; i++) x[i] = bf16_low(w[i]);
    } else {
        x[0] = bf16_low(w[0]), x[1] = bf16_high(w[0]), x[2] = bf16_low(w[1]), x[3] = bf16_high(w[1]);
    }
}
template <bool VEC>
__device__ __forceinline__ void store4(void* p, int64_t at, const float* x) {
    uint16_t* h = static_cast<uint16_t*>(p) + at;
    if constexpr (VEC) *reinterpret_cast<uint2*>(h) = make_uint2(pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]));
    else
#pragma unroll
        for (int i = 0; i < 4; i++) h[i] = round_bf16(x[i]);
}

// A warp takes the heads of one row (or one part of them), D / 8 lanes a head, the loads of four passes over them (words: two) on their way at a time. A lane has the values that
// turn together: four of the first half of the rotary dimensions and the four they are paired with (interleaved, and behind the rotary dimensions: eight adjacent ones), so nothing
// of the rotation crosses lanes. The row's angles are worked out once, two a lane: position times turns in 64 bits, what is left of whole turns in 32. Bound by the bytes: a value
// is read and written once. 4 x 2048 rows of 32 + 2 x 8 heads of 128 into a bf16 cache: 37 us, 4.6 TB/s; int8 42 us; with registers for eight
// blocks a multiprocessor instead of six, which spills a few, 42 us, with eight passes' loads at a time for four blocks, 49 us.
template <int D, bool WORD, bool INT8, bool VEC>
__global__ void __launch_bounds__(128, 6) norm_rope_kernel(const __grid_constant__ NormRopeArgs n) {
    constexpr int LANES = D / 8, HEADS = 32 / LANES, AHEAD = WORD ? 2 : 4, FOUR = WORD ? 4 : 2;  // lanes a head, heads a warp, their loads at a time, words of four values
    __shared__ float2 turn_sm[4][64];
    const zkb_step_norm_rope_args& a = n.a;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint64_t unit = (uint64_t)blockIdx.x * 4 + warp;
    const int t = (int)(unit / n.parts), part = (int)(unit % n.parts);
    if ((uint32_t)t >= a.rows.n_rows) return;
    const int rotary = (int)a.rotary_dim, half = rotary / 2;
    const int l = lane % LANES, mine = lane / LANES;
    const bool turned = 8 * l < rotary, pairs = turned && !a.interleaved;
    const int d0 = pairs ? 4 * l : 8 * l, d1 = pairs ? half + 4 * l : 8 * l + 4;
    const int seq = sequence_of(a.rows.first, (int)a.cache.n_seqs, t);
    if (seq < 0) return;
    const int64_t first = a.rows.first[seq];
    const int64_t pos = (int64_t)a.rows.kv_len[seq] - ((int64_t)a.rows.first[seq + 1] - first) + (t - first);
    for (int i = lane; i < half; i += 32) {
        const double turn = (double)pos * n.turns[i];
        float2 v;
        sincospif(2.f * (float)(turn - rint(turn)), &v.y, &v.x);
        turn_sm[warp][i] = v;
    }
    __syncwarp();
    const bool cached = pos >= 0 && pos < (int64_t)a.cache.capacity;
    float c[4], s[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float2 v = turned ? turn_sm[warp][4 * l + i] : make_float2(0.f, 0.f);
        c[i] = v.x, s[i] = v.y;
    }
    auto weight_of = [&](const uint16_t* w, uint32_t (&v)[4]) {
        if (!w) return;
        v[0] = w[d0] | (uint32_t)w[d0 + 1] << 16, v[1] = w[d0 + 2] | (uint32_t)w[d0 + 3] << 16, v[2] = w[d1] | (uint32_t)w[d1 + 1] << 16, v[3] = w[d1 + 2] | (uint32_t)w[d1 + 3] << 16;
    };
    // Heads part * HEADS + mine, ... of queries (0), keys (1) or values (2).
    auto heads = [&](auto kind, const void* from, int64_t at, int count, const uint16_t* weight) {
        constexpr int KIND = decltype(kind)::value;
        uint32_t w[4] = {};
        weight_of(weight, w);
        const int stride = (int)n.parts * HEADS, h_first = part * HEADS + mine;
        // where this lane's next head is read and written: heads are `stride` apart
        const void* in = value_at<WORD ? 4 : 2>(from, at + h_first * a.head_stride + d0);
        const int64_t in_step = stride * a.head_stride;
        void* out = KIND == 0 ? value_at<2>(a.q_out, t * a.q_out_stride + h_first * a.q_out_head_stride + d0)
                              : value_at<INT8 ? 1 : 2>(KIND == 2 ? a.cache.v : a.cache.k, seq * a.cache.seq_stride + h_first * a.cache.head_stride + pos * a.cache.token_stride + d0);
        const int64_t out_step = stride * (KIND == 0 ? a.q_out_head_stride : a.cache.head_stride);
        float* scale = (KIND == 2 ? a.cache.v_scale : a.cache.k_scale) + (INT8 ? seq * a.cache.scale_seq_stride + h_first * a.cache.scale_head_stride + pos : 0);
#pragma unroll 1
        for (int h0 = part * HEADS; h0 < count; h0 += stride * AHEAD) {
            uint32_t raw[AHEAD][2 * FOUR] = {};
#pragma unroll
            for (int i = 0; i < AHEAD; i++) {
                if (h0 + i * stride + mine < count) load4<WORD, VEC>(in, 0, raw[i]), load4<WORD, VEC>(in, d1 - d0, raw[i] + FOUR);
                in = value_at<WORD ? 4 : 2>(in, in_step);
            }
#pragma unroll
            for (int i = 0; i < AHEAD; i++) {
                if (h0 + i * stride >= count) break;  // the same for the whole warp
                const bool has = h0 + i * stride + mine < count;
                float x[8];
                floats4<WORD>(raw[i], x), floats4<WORD>(raw[i] + FOUR, x + 4);
                if (KIND < 2 && weight) {
                    float ss = 0.f;
#pragma unroll
                    for (int y = 0; y < 8; y++) ss = fmaf(x[y], x[y], ss);
#pragma unroll
                    for (int o = LANES / 2; o; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
                    const float by = rsqrtf(ss * (1.f / D) + a.eps);
#pragma unroll
                    for (int y = 0; y < 4; y++) x[2 * y] *= by * bf16_low(w[y]), x[2 * y + 1] *= by * bf16_high(w[y]);
                }
                if (KIND < 2) {  // (what lies behind the rotary dimensions is left, not turned by nothing: 0 times an infinity is NaN; a branch took a tenth longer)
                    if (a.interleaved) {
#pragma unroll
                        for (int y = 0; y < 4; y++) {
                            const float u = x[2 * y], v = x[2 * y + 1], r = u * c[y] - v * s[y], t = u * s[y] + v * c[y];
                            x[2 * y] = turned ? r : u, x[2 * y + 1] = turned ? t : v;
                        }
                    } else {
#pragma unroll
                        for (int y = 0; y < 4; y++) {
                            const float u = x[y], v = x[y + 4], r = u * c[y] - v * s[y], t = u * s[y] + v * c[y];
                            x[y] = turned ? r : u, x[y + 4] = turned ? t : v;
                        }
                    }
                }
                if (KIND == 0) {
                    if (has) store4<VEC>(out, 0, x), store4<VEC>(out, d1 - d0, x + 4);
                } else if (INT8) {
                    float most = 0.f;
                    bool nan = false;
#pragma unroll
                    for (int y = 0; y < 8; y++) most = fmaxf(most, fabsf(x[y])), nan |= x[y] != x[y];
#pragma unroll
                    for (int o = LANES / 2; o; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
                    if (__ballot_sync(0xffffffffu, nan) >> (mine * LANES) & (LANES == 32 ? 0xffffffffu : (1u << LANES % 32) - 1u)) most = __int_as_float(0x7fc00000);
                    if (has && cached) {
                        float top = most;
                        if (most < 0x1p-64f) {  // (127 over less than 2^-121 is no float)
                            top *= 0x1p64f;
#pragma unroll
                            for (int y = 0; y < 8; y++) x[y] *= 0x1p64f;
                        }
                        const float up = top > 0x1.fcp-80f ? 127.f / top : 0.f;  // codes are 0 where the scale is (up to 127 x 2^-150), and where it is NaN or infinite
                        uint32_t q[2] = {0, 0};
#pragma unroll
                        for (int y = 0; y < 8; y++) q[y / 4] |= (uint32_t)(max(-127, min(127, __float2int_rn(x[y] * up))) & 255) << (8 * (y % 4));
                        int8_t* to = static_cast<int8_t*>(out);
                        if constexpr (VEC) {
                            *reinterpret_cast<uint32_t*>(to) = q[0], *reinterpret_cast<uint32_t*>(to + d1 - d0) = q[1];
                        } else {
#pragma unroll
                            for (int y = 0; y < 4; y++) to[y] = (int8_t)(q[0] >> (8 * y)), to[d1 - d0 + y] = (int8_t)(q[1] >> (8 * y));
                        }
                        if (l == 0) *scale = most / 127.f;
                    }
                } else if (has && cached) {
                    store4<VEC>(out, 0, x), store4<VEC>(out, d1 - d0, x + 4);
                }
                out = value_at<KIND && INT8 ? 1 : 2>(out, out_step);
                if (KIND && INT8) scale += stride * a.cache.scale_head_stride;
            }
        }
    };
    heads(std::integral_constant<int, 0>(), a.q, t * a.q_stride, (int)a.q_heads, a.q_weight);
    heads(std::integral_constant<int, 1>(), a.k, t * a.k_stride, (int)a.cache.n_heads, a.k_weight);
    heads(std::integral_constant<int, 2>(), a.v, t * a.v_stride, (int)a.cache.n_heads, nullptr);
}

template <int D, bool WORD, bool INT8>
static cudaError_t launch_norm_rope(zkb_ctx* ctx, const NormRopeArgs& n, bool vec) {
    const unsigned grid = (unsigned)(((uint64_t)n.a.rows.n_rows * n.parts + 3) / 4);
    if (vec) norm_rope_kernel<D, WORD, INT8, true><<<grid, 128, 0, ctx->stream>>>(n);
    else norm_rope_kernel<D, WORD, INT8, false><<<grid, 128, 0, ctx->stream>>>(n);
    return cudaGetLastError();
}
template <int D>
static cudaError_t launch_norm_rope(zkb_ctx* ctx, const NormRopeArgs& n, bool vec) {
    const bool word = n.a.type == ZKB_VALUE_WORD, int8 = n.a.cache.type == ZKB_VALUE_INT8;
    return word ? (int8 ? launch_norm_rope<D, true, true>(ctx, n, vec) : launch_norm_rope<D, true, false>(ctx, n, vec))
                : (int8 ? launch_norm_rope<D, false, true>(ctx, n, vec) : launch_norm_rope<D, false, false>(ctx, n, vec));
}

}  // namespace zk

using namespace zk;

extern "C" {

int zkb_step_embed(zkb_ctx* ctx, const zkb_step_embed_args* args) {
    if (!ctx) return ZKB_EINVAL;
    ZKB_CHECK_ARG(ctx, args);
    const zkb_step_embed_args& a = *args;
    ZKB_CHECK_ARG(ctx, a.table_type == ZKB_VALUE_BF16 || a.table_type == ZKB_VALUE_INT8);
    ZKB_CHECK_ARG(ctx, a.out_type == ZKB_VALUE_BF16 || a.out_type == ZKB_VALUE_WORD);
    ZKB_CHECK_ARG(ctx, a.width >= 1 && a.width <= (1u << 23) && a.vocab <= 0x7fffffffu && a.n_tokens <= 0x7fffffffu && std::isfinite(a.scale));
    if (a.n_tokens == 0) return ZKB_OK;
    const bool int8 = a.table_type == ZKB_VALUE_INT8, word = a.out_type == ZKB_VALUE_WORD;
    const size_t in_size = int8 ? 1 : 2, out_size = word ? 4 : 2;
    ZKB_CHECK_ARG(ctx, a.ids && a.out && (a.vocab == 0 || a.table) && (int8 ? (a.vocab == 0 || a.row_scale) : !a.row_scale));
    ZKB_CHECK_ARG(ctx, aligned_to(a.table, in_size) && aligned_to(a.out, out_size) && aligned_to(a.ids, 4) && aligned_to(a.row_scale, 4) && aligned_to(a.off_table, 8));
    ZKB_CHECK_ARG(ctx, a.segment == 0 || a.segment >= a.width || std::llabs(a.segment_stride) >= (long long)a.segment);
    ZKB_CHECK_ARG(ctx, a.n_tokens == 1 || std::llabs(a.out_stride) >= (long long)(a.segment && a.segment < a.width ? a.segment : a.width));
    DeviceGuard g(ctx);
    const bool vec = a.width % 8 == 0 && a.table_stride % 8 == 0 && aligned_to(a.table, 8 * in_size) && aligned_to(a.out, 16) && a.out_stride * (int64_t)out_size % 16 == 0 &&
                     (a.segment == 0 || (a.segment % 8 == 0 && a.segment_stride * (int64_t)out_size % 16 == 0));
    const uint32_t per_block = vec ? 2048 : 256, runs = (a.width + per_block - 1) / per_block;
    EmbedArgs e{a, 1};
    while (e.tokens_a_block < EMBED_TOKENS && (uint64_t)a.n_tokens * runs / e.tokens_a_block > 148 * 16) e.tokens_a_block *= 2;
    const dim3 grid((a.n_tokens + e.tokens_a_block - 1) / e.tokens_a_block, runs);
    ProfScope prof(ctx, "step_embed_kernel");
    auto launch = [&](auto kernel) { kernel<<<grid, 256, 0, ctx->stream>>>(e); };
    if (vec) int8 ? (word ? launch(embed_kernel<true, true>) : launch(embed_kernel<true, false>)) : (word ? launch(embed_kernel<false, true>) : launch(embed_kernel<false, false>));
    else int8 ? (word ? launch(embed_ragged_kernel<true, true>) : launch(embed_ragged_kernel<true, false>)) : (word ? launch(embed_ragged_kernel<false, true>) : launch(embed_ragged_kernel<false, false>));
    ZKB_LAUNCH_CHECK(ctx);
    return ZKB_OK;
}

int zkb_step_norm_rope(zkb_ctx* ctx, const zkb_step_norm_rope_args* args) {
    if (!ctx) return ZKB_EINVAL;
    ZKB_CHECK_ARG(ctx, args);
    const zkb_step_norm_rope_args& a = *args;
    const zkb_kv_cache& c = a.cache;
    if (const char* why = step_problem(c, a.rows, a.q_heads)) return set_error(ctx, ZKB_EINVAL, "zkb_step_norm_rope: %s", why);
    ZKB_CHECK_ARG(ctx, a.type == ZKB_VALUE_BF16 || a.type == ZKB_VALUE_WORD);
    ZKB_CHECK_ARG(ctx, a.rotary_dim % 16 == 0 && a.rotary_dim <= c.head_dim && a.interleaved <= 1 && (a.rotary_dim == 0 || a.h_inv_freq));
    ZKB_CHECK_ARG(ctx, std::isfinite(a.eps) && a.eps >= 0.f);
    if (a.rows.n_rows == 0) return ZKB_OK;
    const bool word = a.type == ZKB_VALUE_WORD, int8 = c.type == ZKB_VALUE_INT8;
    const size_t in_size = word ? 4 : 2, kv_size = int8 ? 1 : 2;
    ZKB_CHECK_ARG(ctx, a.q && a.k && a.v && a.q_out);
    ZKB_CHECK_ARG(ctx, aligned_to(a.q, in_size) && aligned_to(a.k, in_size) && aligned_to(a.v, in_size) && aligned_to(a.q_out, 2) && aligned_to(a.q_weight, 2) && aligned_to(a.k_weight, 2));
    ZKB_CHECK_ARG(ctx, a.q_heads == 1 || std::llabs(a.q_out_head_stride) >= (long long)c.head_dim);
    ZKB_CHECK_ARG(ctx, a.rows.n_rows == 1 || std::llabs(a.q_out_stride) >= (long long)c.head_dim);
    NormRopeArgs n{};
    n.a = a;
    for (uint32_t i = 0; i < a.rotary_dim / 2; i++) {
        ZKB_CHECK_ARG(ctx, std::isfinite(a.h_inv_freq[i]));
        n.turns[i] = a.h_inv_freq[i] / 6.283185307179586476925;
    }
    n.a.h_inv_freq = nullptr;
    // four values at a time where all rows start on such a boundary
    const bool vec = aligned_to(a.q, 4 * in_size) && aligned_to(a.k, 4 * in_size) && aligned_to(a.v, 4 * in_size) && aligned_to(a.q_out, 8) && aligned_to(c.k, 4 * kv_size) && aligned_to(c.v, 4 * kv_size) &&
                     a.q_stride % 4 == 0 && a.k_stride % 4 == 0 && a.v_stride % 4 == 0 && a.head_stride % 4 == 0 && a.q_out_stride % 4 == 0 && a.q_out_head_stride % 4 == 0 && c.seq_stride % 4 == 0 &&
                     c.head_stride % 4 == 0 && c.token_stride % 4 == 0;
    // A warp a row; few rows are spread over more, down to a warp for each of its passes over the query heads.
    const uint32_t passes = (a.q_heads + 256 / c.head_dim - 1) / (256 / c.head_dim);
    n.parts = std::max(1u, std::min(passes, 148u * 16u / a.rows.n_rows));
    DeviceGuard g(ctx);
    ProfScope prof(ctx, "step_norm_rope_kernel");
    ZKB_CUDA(ctx, c.head_dim == 128 ? launch_norm_rope<128>(ctx, n, vec) : c.head_dim == 64 ? launch_norm_rope<64>(ctx, n, vec) : launch_norm_rope<32>(ctx, n, vec));
    return ZKB_OK;
}

}  // extern "C"
