// The values of a decode step: embedding rows, norms and rotation of queries and keys with the cache that they fill.
#include <algorithm>
#include <cmath>
#include <cstdlib>

#include "step_values.cuh"

namespace zk {

// ---- embedding rows ------------------------------------------------------------------------------------------------------------------
struct EmbedArgs {
    zkb_step_embed_args a;
    uint32_t tokens_a_block;
};

// Eight values a thread; blockIdx.y names the run of the row, blockIdx.x the tokens.
template <bool INT8, bool WORD>
__global__ void __launch_bounds__(256) embed_kernel(const __grid_constant__ EmbedArgs e) {
    const zkb_step_embed_args& a = e.a;
    const uint32_t col = (blockIdx.y * 256u + threadIdx.x) * 8u;
    const uint32_t t0 = blockIdx.x * e.tokens_a_block, t1 = min(a.n_tokens, t0 + e.tokens_a_block);
    if (col >= a.width) return;
    const int64_t at = a.segment ? (int64_t)(col / a.segment) * a.segment_stride + col % a.segment : (int64_t)col;
    for (uint32_t t = t0; t < t1; t++) {
        const int32_t id = a.ids[t];
        const bool inside = id >= 0 && (uint32_t)id < a.vocab;
        if (!inside && col == 0 && a.off_table) atomicAdd(reinterpret_cast<unsigned long long*>(a.off_table), 1ull);
        float x[8] = {0, 0, 0, 0, 0, 0, 0, 0};
        if (inside) {
            const int64_t from = (int64_t)id * a.table_stride + col;
            if constexpr (INT8) {
                const uint2 w = *reinterpret_cast<const uint2*>(static_cast<const int8_t*>(a.table) + from);
                const float by = a.row_scale[id] * a.scale;
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    x[i] = (float)(int8_t)(w.x >> (8 * i)) * by;
                    x[4 + i] = (float)(int8_t)(w.y >> (8 * i)) * by;
                }
            } else {
                load8<false, true>(a.table, from, x);
#pragma unroll
                for (int i = 0; i < 8; i++) x[i] *= a.scale;
            }
        }
        store8<WORD, true>(a.out, (int64_t)t * a.out_stride + at, x);
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
    uint32_t parts;   // thread blocks a row
    double turns[64]; // h_inv_freq / (2 pi): turns a position
};

// A thread block takes the heads of one row (or one part of them); D / 8 lanes take a head, eight values each. The row's angles are worked
// out once, by half a rotary dimension's threads, and read by all: position times turns in 64 bits, what is left of whole turns in 32.
template <int D, bool WORD, bool INT8, bool VEC>
__global__ void __launch_bounds__(128) norm_rope_kernel(const __grid_constant__ NormRopeArgs n) {
    constexpr int LANES = D / 8, HEADS = 32 / LANES;  // lanes a head, heads a warp
    __shared__ float cos_sm[64], sin_sm[64];
    const zkb_step_norm_rope_args& a = n.a;
    const int t = (int)(blockIdx.x / n.parts), part = (int)(blockIdx.x % n.parts);
    const int seq = sequence_of(a.rows.first, (int)a.cache.n_seqs, t);
    if (seq < 0) return;
    const int64_t first = a.rows.first[seq];
    const int64_t pos = (int64_t)a.rows.kv_len[seq] - ((int64_t)a.rows.first[seq + 1] - first) + (t - first);
    const int half = (int)a.rotary_dim / 2;
    if ((int)threadIdx.x < half) {
        const double turn = (double)pos * n.turns[threadIdx.x];
        sincospif(2.f * (float)(turn - rint(turn)), &sin_sm[threadIdx.x], &cos_sm[threadIdx.x]);
    }
    __syncthreads();
    const bool cached = pos >= 0 && pos < (int64_t)a.cache.capacity;
    const int lane = threadIdx.x & 31, l = lane % LANES, d0 = 8 * l;
    const int heads = (int)(a.q_heads + 2 * a.cache.n_heads), q_heads = (int)a.q_heads, kv_heads = (int)a.cache.n_heads;
    for (int h0 = (part * 4 + (int)(threadIdx.x >> 5)) * HEADS; h0 < heads; h0 += (int)n.parts * 4 * HEADS) {
        const int hh = h0 + lane / LANES;
        const bool live = hh < heads, is_q = hh < q_heads, is_v = hh >= q_heads + kv_heads;
        const int h = is_q ? hh : is_v ? hh - q_heads - kv_heads : hh - q_heads;
        float x[8] = {0, 0, 0, 0, 0, 0, 0, 0};
        if (live) {
            const void* from = is_q ? a.q : is_v ? a.v : a.k;
            load8<WORD, VEC>(from, t * (is_q ? a.q_stride : is_v ? a.v_stride : a.k_stride) + h * a.head_stride + d0, x);
        }
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < 8; i++) ss = fmaf(x[i], x[i], ss);
#pragma unroll
        for (int o = LANES / 2; o; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        const uint16_t* weight = is_v ? nullptr : is_q ? a.q_weight : a.k_weight;
        if (weight) {
            const float by = rsqrtf(ss * (1.f / D) + a.eps);
#pragma unroll
            for (int i = 0; i < 8; i++) x[i] = x[i] * by * bf16_low(weight[d0 + i]);
        }
        if (half) {
            if (a.interleaved) {
                if (d0 < 2 * half && !is_v) {
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const float c = cos_sm[d0 / 2 + i], s = sin_sm[d0 / 2 + i], u = x[2 * i], v = x[2 * i + 1];
                        x[2 * i] = u * c - v * s;
                        x[2 * i + 1] = v * c + u * s;
                    }
                }
            } else {
                // half is a multiple of eight: the other value of each pair lies with one lane
                const bool low = d0 < half, turned = d0 < 2 * half && !is_v;
                const int other = lane + (d0 >= 2 * half ? 0 : low ? half / 8 : -(half / 8)), at = low ? d0 : d0 - half;
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const float y = __shfl_sync(0xffffffffu, x[i], other);
                    if (turned) x[i] = fmaf(x[i], cos_sm[at + i], (low ? -y : y) * sin_sm[at + i]);
                }
            }
        }
        if (is_q && live) store8<false, VEC>(a.q_out, t * a.q_out_stride + h * a.q_out_head_stride + d0, x);
        if constexpr (INT8) {
            float most = 0.f;
            bool nan = false;
#pragma unroll
            for (int i = 0; i < 8; i++) most = fmaxf(most, fabsf(x[i])), nan |= x[i] != x[i];
            if (nan) most = __int_as_float(0x7fc00000);
#pragma unroll
            for (int o = LANES / 2; o; o >>= 1) {
                const float m = __shfl_xor_sync(0xffffffffu, most, o);
                most = m != m || most != most ? m + most : fmaxf(most, m);
            }
            if (!is_q && live && cached) {
                const float scale = __fdiv_rn(most, 127.f);
                uint32_t w[2] = {0, 0};
                if (scale > 0.f)
#pragma unroll
                    for (int i = 0; i < 8; i++) w[i / 4] |= (uint32_t)(max(-127, min(127, __float2int_rn(__fdiv_rn(x[i], scale)))) & 255) << (8 * (i % 4));
                int8_t* to = static_cast<int8_t*>(is_v ? a.cache.v : a.cache.k) + seq * a.cache.seq_stride + h * a.cache.head_stride + pos * a.cache.token_stride + d0;
                if constexpr (VEC) *reinterpret_cast<uint2*>(to) = make_uint2(w[0], w[1]);
                else
#pragma unroll
                    for (int i = 0; i < 8; i++) to[i] = (int8_t)(w[i / 4] >> (8 * (i % 4)));
                if (l == 0) (is_v ? a.cache.v_scale : a.cache.k_scale)[seq * a.cache.scale_seq_stride + h * a.cache.scale_head_stride + pos] = scale;
            }
        } else if (!is_q && live && cached) {
            store8<false, VEC>(is_v ? a.cache.v : a.cache.k, seq * a.cache.seq_stride + h * a.cache.head_stride + pos * a.cache.token_stride + d0, x);
        }
    }
}

template <int D, bool WORD, bool INT8>
static cudaError_t launch_norm_rope(zkb_ctx* ctx, const NormRopeArgs& n, bool vec) {
    const unsigned grid = n.a.rows.n_rows * n.parts;
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
    ZKB_CHECK_ARG(ctx, aligned_to(a.table, in_size) && aligned_to(a.out, out_size));
    ZKB_CHECK_ARG(ctx, a.segment == 0 || a.segment >= a.width || std::llabs(a.segment_stride) >= (long long)a.segment);
    ZKB_CHECK_ARG(ctx, a.n_tokens == 1 || std::llabs(a.out_stride) >= (long long)(a.segment && a.segment < a.width ? a.segment : a.width));
    DeviceGuard g(ctx);
    const bool vec = a.width % 8 == 0 && a.table_stride % 8 == 0 && aligned_to(a.table, 8 * in_size) && aligned_to(a.out, 16) && a.out_stride * (int64_t)out_size % 16 == 0 &&
                     (a.segment == 0 || (a.segment % 8 == 0 && a.segment_stride * (int64_t)out_size % 16 == 0));
    const uint32_t per_block = vec ? 2048 : 256, runs = (a.width + per_block - 1) / per_block;
    EmbedArgs e{a, 1};
    while (e.tokens_a_block < 4 && (uint64_t)a.n_tokens * runs / e.tokens_a_block > 148 * 16) e.tokens_a_block *= 2;
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
    // a head's rows are read and written 16 bytes (INT8 caches: 8) at a time where every row starts on such a boundary
    const int64_t in_step = 16 / (int64_t)in_size;
    const bool vec = aligned_to(a.q, 16) && aligned_to(a.k, 16) && aligned_to(a.v, 16) && aligned_to(a.q_out, 16) && aligned_to(c.k, 8 * kv_size) && aligned_to(c.v, 8 * kv_size) &&
                     a.q_stride % in_step == 0 && a.k_stride % in_step == 0 && a.v_stride % in_step == 0 && a.head_stride % in_step == 0 && a.q_out_stride % 8 == 0 && a.q_out_head_stride % 8 == 0 &&
                     c.seq_stride % 8 == 0 && c.head_stride % 8 == 0 && c.token_stride % 8 == 0;
    // Few rows are spread over the SMs, a pass of four warps each.
    const uint32_t heads = a.q_heads + 2 * c.n_heads, a_pass = 4 * 32 / (c.head_dim / 8), passes = (heads + a_pass - 1) / a_pass;
    n.parts = std::max(1u, std::min(passes, 148u * 4u / a.rows.n_rows));
    DeviceGuard g(ctx);
    ProfScope prof(ctx, "step_norm_rope_kernel");
    ZKB_CUDA(ctx, c.head_dim == 128 ? launch_norm_rope<128>(ctx, n, vec) : c.head_dim == 64 ? launch_norm_rope<64>(ctx, n, vec) : launch_norm_rope<32>(ctx, n, vec));
    return ZKB_OK;
}

}  // extern "C"
