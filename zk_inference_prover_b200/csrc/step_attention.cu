// Attention of a step's rows over the key-value cache.
#include <algorithm>
#include <cmath>
#include <cstdlib>

#include "step_values.cuh"

namespace zk {

// A warp a row and query head: the keys that the row sees one after another, the running maximum and sum of the softmax beside the
// weighted sum of the values, D / 32 of its elements a lane.
template <int D, bool INT8, bool WORD>
__global__ void __launch_bounds__(128) attention_kernel(const __grid_constant__ zkb_step_attention_args a) {
    constexpr int E = D / 32;
    const uint64_t unit = (uint64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
    const int t = (int)(unit / a.q_heads), h = (int)(unit % a.q_heads), lane = threadIdx.x & 31;
    if ((uint32_t)t >= a.rows.n_rows) return;
    const zkb_kv_cache& c = a.cache;
    const int seq = sequence_of(a.rows.first, (int)c.n_seqs, t);
    if (seq < 0) return;
    const int64_t first = a.rows.first[seq], pos = (int64_t)a.rows.kv_len[seq] - ((int64_t)a.rows.first[seq + 1] - first) + (t - first);
    const int64_t end = min(pos + 1, (int64_t)c.capacity), near = a.window ? max((int64_t)0, pos - (int64_t)a.window + 1) : 0;
    const int64_t kv = seq * c.seq_stride + (h / (int)(a.q_heads / c.n_heads)) * c.head_stride;
    const int64_t sc = seq * c.scale_seq_stride + (h / (int)(a.q_heads / c.n_heads)) * c.scale_head_stride;
    float q[E], o[E], top = -INFINITY, sum = 0.f;
    for (int e = 0; e < E; e++) {
        q[e] = bf16_low(static_cast<const uint16_t*>(a.q)[t * a.q_stride + h * a.q_head_stride + lane * E + e]) * a.scale;
        o[e] = 0.f;
    }
    for (int64_t j = 0; j < end; j++) {
        if (j < near && j >= (int64_t)a.sinks) j = near;
        if (j >= end) break;
        const int64_t at = kv + j * c.token_stride + lane * E;
        float k[E], v[E], s = 0.f;
        for (int e = 0; e < E; e++) {
            k[e] = INT8 ? (float)static_cast<const int8_t*>(c.k)[at + e] * c.k_scale[sc + j] : bf16_low(static_cast<const uint16_t*>(c.k)[at + e]);
            v[e] = INT8 ? (float)static_cast<const int8_t*>(c.v)[at + e] * c.v_scale[sc + j] : bf16_low(static_cast<const uint16_t*>(c.v)[at + e]);
            s = fmaf(q[e], k[e], s);
        }
        for (int x = 16; x; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
        const float higher = s != s ? s : fmaxf(top, s), base = higher == -INFINITY ? 0.f : higher;
        const float keep = expf(top - base), p = expf(s - base);
        sum = sum * keep + p;
        for (int e = 0; e < E; e++) o[e] = o[e] * keep + p * v[e];
        top = higher;
    }
    for (int e = 0; e < E; e++) {
        const float y = sum == 0.f ? 0.f : o[e] / sum;
        const int64_t to = t * a.out_stride + h * a.out_head_stride + lane * E + e;
        if (WORD) static_cast<uint32_t*>(a.out)[to] = round_bf16(y);
        else static_cast<uint16_t*>(a.out)[to] = round_bf16(y);
    }
}

template <int D>
static void launch_attention(zkb_ctx* ctx, const zkb_step_attention_args& a) {
    const unsigned grid = (unsigned)(((uint64_t)a.rows.n_rows * a.q_heads + 3) / 4);
    const bool int8 = a.cache.type == ZKB_VALUE_INT8, word = a.out_type == ZKB_VALUE_WORD;
    auto launch = [&](auto kernel) { kernel<<<grid, 128, 0, ctx->stream>>>(a); };
    if (int8) word ? launch(attention_kernel<D, true, true>) : launch(attention_kernel<D, true, false>);
    else word ? launch(attention_kernel<D, false, true>) : launch(attention_kernel<D, false, false>);
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
    ZKB_CHECK_ARG(ctx, std::isfinite(a.scale));
    if (a.rows.n_rows == 0) return ZKB_OK;
    ZKB_CHECK_ARG(ctx, a.q && a.out && aligned_to(a.q, 2) && aligned_to(a.out, a.out_type == ZKB_VALUE_WORD ? 4 : 2));
    ZKB_CHECK_ARG(ctx, a.q_heads == 1 || std::llabs(a.out_head_stride) >= (long long)c.head_dim);
    ZKB_CHECK_ARG(ctx, a.rows.n_rows == 1 || std::llabs(a.out_stride) >= (long long)c.head_dim);
    DeviceGuard g(ctx);
    ProfScope prof(ctx, "step_attention_kernel");
    c.head_dim == 128 ? launch_attention<128>(ctx, a) : c.head_dim == 64 ? launch_attention<64>(ctx, a) : launch_attention<32>(ctx, a);
    ZKB_LAUNCH_CHECK(ctx);
    return ZKB_OK;
}
