// Attention of a step's rows over the key-value cache.
#include <algorithm>
#include <cmath>
#include <cstdlib>

#include "step_attention.cuh"

namespace zk {

// ---- few rows: one token, or a few, of each sequence -----------------------------------------------------------------------------------
// The cache is read once and everything else is small, so this is bound by the cache's bytes. Eight query rows (the heads of a kv head's
// group, of one token or several) are the N of mma.m16n8k16 and sixteen keys its M, S^T = K Q^T, O^T = V^T P^T: every value of K and V goes
// from memory into the register of the lane that multiplies it, 16 bytes at a time, with no shared memory between:
//   K: lane (g, t) holds keys g and g + 8 and a quarter of their dimensions; which dimension is which k of the product is free as long as Q agrees.
//   V: lane (g, t) holds keys 2t, 2t + 1, 2t + 8, 2t + 9, and an eighth of their dimensions; two keys' bytes make a register of the product.
// P^T is S^T's registers transposed eight by eight (movmatrix). A warp takes every W-th block of sixteen keys with its own running maximum and
// sum; warps join through shared memory, thread blocks of a cluster through each other's, so that a long sequence is spread over up to 16 SMs
// without a workspace or a second launch.
constexpr int FEW_WARPS = 8;

template <int D, bool INT8>
struct FewBlock {  // sixteen keys of K and V as they came from memory
    static constexpr int KW = D * (INT8 ? 1 : 2) / 16, VW = D * (INT8 ? 1 : 2) / 32;  // words a lane and key
    uint32_t k[2][KW], v[4][VW];
    float ks[2], vs[2];
};

// `words` words of a row from byte `at` on, in pieces of up to 16 bytes `apart` bytes apart.
template <int WORDS, bool VEC>
__device__ __forceinline__ void load_row(const char* p, int apart, uint32_t (&w)[WORDS]) {
    constexpr int PIECE = WORDS < 4 ? WORDS : 4;
#pragma unroll
    for (int i = 0; i < WORDS; i += PIECE) {
        const char* from = p + (i / PIECE) * apart;
        if constexpr (!VEC) {
#pragma unroll
            for (int x = 0; x < PIECE; x++) {
                const uint8_t* b = reinterpret_cast<const uint8_t*>(from) + 4 * x;
                w[i + x] = (uint32_t)b[0] | (uint32_t)b[1] << 8 | (uint32_t)b[2] << 16 | (uint32_t)b[3] << 24;
            }
        } else if constexpr (PIECE == 4) {
            const uint4 a = ld_stream(reinterpret_cast<const uint4*>(from));
            w[i] = a.x, w[i + 1] = a.y, w[i + 2] = a.z, w[i + 3] = a.w;
        } else if constexpr (PIECE == 2) {
            const uint2 a = *reinterpret_cast<const uint2*>(from);
            w[i] = a.x, w[i + 1] = a.y;
        } else {
            w[i] = *reinterpret_cast<const uint32_t*>(from);
        }
    }
}

template <int D, bool INT8, bool VEC>
__device__ __forceinline__ void few_load(FewBlock<D, INT8>& b, const char* k, const char* v, const float* ks, const float* vs, int64_t row_bytes, int base, int last) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    constexpr int KW = FewBlock<D, INT8>::KW, VW = FewBlock<D, INT8>::VW, KP = KW < 4 ? KW * 4 : 16, VP = VW < 4 ? VW * 4 : 16;
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const int key = min(base + 8 * i + g, last);
        load_row<KW, VEC>(k + key * row_bytes + t * KP, 4 * KP, b.k[i]);
        if constexpr (INT8) b.ks[i] = __ldg(ks + key), b.vs[i] = __ldg(vs + key);
    }
#pragma unroll
    for (int i = 0; i < 4; i++) load_row<VW, VEC>(v + min(base + 8 * (i >> 1) + 2 * t + (i & 1), last) * row_bytes + g * VP, 8 * VP, b.v[i]);
}

template <int D, bool INT8, bool VEC>
__global__ void __launch_bounds__(FEW_WARPS * 32) attention_few_kernel(const __grid_constant__ zkb_step_attention_args a) {
    constexpr int STEPS = D / 16, KW = FewBlock<D, INT8>::KW, VW = FewBlock<D, INT8>::VW;
    __shared__ float o_sm[FEW_WARPS][8][D + 4], top_sm[FEW_WARPS][8], sum_sm[FEW_WARPS][8];
    __shared__ float cta_top[8], cta_sum[8];
    __shared__ int odd_sm;  // some value of V was no number
    const zkb_kv_cache& c = a.cache;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    const int seq = blockIdx.z, kv_head = blockIdx.y, group = (int)(a.q_heads / c.n_heads);
    const int rank = (int)cluster_rank(), ranks = (int)cluster_ranks();
    const StepSequence s = step_sequence(a.rows, seq);
    const int size = INT8 ? 1 : 2;
    const char* const k = static_cast<const char*>(c.k) + (seq * c.seq_stride + kv_head * c.head_stride) * size;
    const char* const v = static_cast<const char*>(c.v) + (seq * c.seq_stride + kv_head * c.head_stride) * size;
    const float* const ks = INT8 ? c.k_scale + seq * c.scale_seq_stride + kv_head * c.scale_head_stride : nullptr;
    const float* const vs = INT8 ? c.v_scale + seq * c.scale_seq_stride + kv_head * c.scale_head_stride : nullptr;
    const int64_t row_bytes = c.token_stride * size;
    const int64_t n_m = (int64_t)s.rows * group;
    const float by = a.scale * 1.44269504f;
    for (int64_t m0 = (int64_t)(blockIdx.x / ranks) * 8; m0 < n_m; m0 += (int64_t)(gridDim.x / ranks) * 8) {
        const int64_t pos_low = s.pos + m0 / group, pos_high = s.pos + (min(m0 + 8, n_m) - 1) / group;
        const KeyBlocks blocks = key_blocks<16>(pos_low, pos_high, c.capacity, a.window, a.sinks);
        // Q: lane (g, t) has row g's dimensions in the order in which its K quarter comes
        uint32_t q[STEPS][2];
        {
            constexpr int PIECE = (KW < 4 ? KW : 4) * (INT8 ? 4 : 2);  // dimensions in a piece
            const int64_t m = m0 + g;
            const uint16_t* from = static_cast<const uint16_t*>(a.q) + (m < n_m ? (s.first + m / group) * a.q_stride + (kv_head * group + m % group) * a.q_head_stride : 0);
#pragma unroll
            for (int i = 0; i < STEPS; i++)
#pragma unroll
                for (int x = 0; x < 2; x++) {
                    const int e = 4 * i + 2 * x, d = (e / PIECE) * 4 * PIECE + t * PIECE + e % PIECE;
                    q[i][x] = m < n_m ? (uint32_t)from[d] | (uint32_t)from[d + 1] << 16 : 0u;
                }
        }
        // rows 2t and 2t + 1: their positions, running maxima and this lane's part of their sums
        int64_t p[2];
        float top[2] = {-INFINITY, -INFINITY}, sum[2] = {0.f, 0.f}, o[STEPS][4];
#pragma unroll
        for (int r = 0; r < 2; r++) p[r] = m0 + 2 * t + r < n_m ? s.pos + (m0 + 2 * t + r) / group : -1;
#pragma unroll
        for (int i = 0; i < STEPS; i++)
#pragma unroll
            for (int x = 0; x < 4; x++) o[i][x] = 0.f;
        bool odd = false;
        if (threadIdx.x == 0) odd_sm = 0;
        const int stride = ranks * FEW_WARPS, last = (int)blocks.end - 1;
        FewBlock<D, INT8> next;
        int at = rank * FEW_WARPS + warp;
        if (at < blocks.n) few_load<D, INT8, VEC>(next, k, v, ks, vs, row_bytes, blocks.base(at), last);
        for (; at < blocks.n; at += stride) {
            const int base = blocks.base(at);
            FewBlock<D, INT8> b = next;
            if (at + stride < blocks.n) few_load<D, INT8, VEC>(next, k, v, ks, vs, row_bytes, blocks.base(at + stride), last);
            float sc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < STEPS; i++) {
                uint32_t f[4];
                if constexpr (INT8) {
                    codes_to_bf16(b.k[0][i], f[0], f[2]);
                    codes_to_bf16(b.k[1][i], f[1], f[3]);
                } else {
                    f[0] = b.k[0][2 * i], f[1] = b.k[1][2 * i], f[2] = b.k[0][2 * i + 1], f[3] = b.k[1][2 * i + 1];
                }
                mma_bf16(sc, f, q[i][0], q[i][1]);
            }
            // sc: key g with rows 2t, 2t + 1, then key g + 8
            float higher[2] = {top[0], top[1]};
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int64_t key = base + g + 8 * (i >> 1), gap = p[i & 1] - key;
                const bool seen = gap >= 0 && key <= last && (a.window == 0 || gap < (int64_t)a.window || key < (int64_t)a.sinks);
                sc[i] = seen ? sc[i] * (INT8 ? b.ks[i >> 1] * by : by) : -INFINITY;
                higher[i & 1] = fmaxf(higher[i & 1], sc[i]);
            }
#pragma unroll
            for (int r = 0; r < 2; r++)
#pragma unroll
                for (int x = 4; x < 32; x <<= 1) higher[r] = fmaxf(higher[r], __shfl_xor_sync(0xffffffffu, higher[r], x));
            if (__any_sync(0xffffffffu, higher[0] > top[0] || higher[1] > top[1])) {
                const float keep[2] = {higher[0] > top[0] ? exp2f(top[0] - higher[0]) : 1.f, higher[1] > top[1] ? exp2f(top[1] - higher[1]) : 1.f};
#pragma unroll
                for (int r = 0; r < 2; r++) sum[r] *= keep[r], top[r] = higher[r];
#pragma unroll
                for (int i = 0; i < STEPS; i++)
#pragma unroll
                    for (int x = 0; x < 4; x++) o[i][x] *= keep[x & 1];
            }
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float w = exp2f(sc[i] - (top[i & 1] == -INFINITY ? 0.f : top[i & 1]));
                sum[i & 1] += w;
                sc[i] = INT8 ? (sc[i] == -INFINITY ? 0.f : w * b.vs[i >> 1]) : w;  // a hidden token's scale may be anything
            }
            const uint32_t w0 = transpose8(pack_bf16(sc[0], sc[1])), w1 = transpose8(pack_bf16(sc[2], sc[3]));
            if constexpr (!INT8) {
                // a value that is no number would reach the rows that do not see its key: it is set aside (below)
                uint32_t test = 0;
#pragma unroll
                for (int i = 0; i < 4; i++)
#pragma unroll
                    for (int x = 0; x < VW; x++) test = zero_or_nan(b.v[i][x], test);
                if (__any_sync(0xffffffffu, (test & 0x7fff7fffu) != 0)) {
                    odd = true;
#pragma unroll
                    for (int i = 0; i < 4; i++)
#pragma unroll
                        for (int x = 0; x < VW; x++) b.v[i][x] = numbers_only(b.v[i][x]);
                }
            }
#pragma unroll
            for (int i = 0; i < STEPS; i++) {
                uint32_t f[4];  // dimensions 2i and 2i + 1 of the lane's, keys 2t and 2t + 1, then 2t + 8 and 2t + 9
                if constexpr (INT8) {
                    pair_codes_to_bf16(b.v[0][i / 2], b.v[1][i / 2], i & 1, f[0], f[1]);
                    pair_codes_to_bf16(b.v[2][i / 2], b.v[3][i / 2], i & 1, f[2], f[3]);
                } else {
                    f[0] = __byte_perm(b.v[0][i], b.v[1][i], 0x5410), f[1] = __byte_perm(b.v[0][i], b.v[1][i], 0x7632);
                    f[2] = __byte_perm(b.v[2][i], b.v[3][i], 0x5410), f[3] = __byte_perm(b.v[2][i], b.v[3][i], 0x7632);
                }
                mma_bf16(o[i], f, w0, w1);
            }
        }
        // join the warps
        __syncthreads();  // odd_sm is cleared; the last tile's o_sm has been read
        if (odd && lane == 0) odd_sm = 1;
#pragma unroll
        for (int r = 0; r < 2; r++) {
#pragma unroll
            for (int x = 4; x < 32; x <<= 1) sum[r] += __shfl_xor_sync(0xffffffffu, sum[r], x);
            if (g == 0) top_sm[warp][2 * t + r] = top[r], sum_sm[warp][2 * t + r] = sum[r];
        }
        {
            constexpr int PIECE = (VW < 4 ? VW : 4) * (INT8 ? 4 : 2);
#pragma unroll
            for (int i = 0; i < STEPS; i++)
#pragma unroll
                for (int x = 0; x < 4; x++) {
                    const int e = 2 * i + (x >> 1);
                    o_sm[warp][2 * t + (x & 1)][(e / PIECE) * 8 * PIECE + g * PIECE + e % PIECE] = o[i][x];
                }
        }
        __syncthreads();
        if (warp == 0 && lane < 8) {
            float most = -INFINITY, all = 0.f;
            for (int w = 0; w < FEW_WARPS; w++) most = fmaxf(most, top_sm[w][lane]);
            const float base = most == -INFINITY ? 0.f : most;
            for (int w = 0; w < FEW_WARPS; w++) {
                const float f = exp2f(top_sm[w][lane] - base);
                all += sum_sm[w][lane] * f;
                top_sm[w][lane] = f;
            }
            cta_top[lane] = most, cta_sum[lane] = all;
        }
        __syncthreads();
        for (int i = threadIdx.x; i < 8 * D; i += FEW_WARPS * 32) {
            const int r = i / D, d = i % D;
            float y = 0.f;
#pragma unroll
            for (int w = 0; w < FEW_WARPS; w++) y += o_sm[w][r][d] * top_sm[w][r];
            o_sm[0][r][d] = y;
        }
        // join the cluster: each thread block takes a part of the outputs
        if (ranks > 1) cluster_sync();
        else __syncthreads();
        int any_odd = 0;
        for (int k2 = 0; k2 < ranks; k2++) any_odd |= ranks > 1 ? peer_load(&odd_sm, k2) : odd_sm;
        for (int i = threadIdx.x + rank * FEW_WARPS * 32; i < 8 * D; i += ranks * FEW_WARPS * 32) {
            const int r = i / D, d = i % D;
            const int64_t m = m0 + r;
            if (m >= n_m) continue;
            float y, all;
            if (ranks == 1) {
                y = o_sm[0][r][d], all = cta_sum[r];
            } else {
                float most = -INFINITY;
                for (int k2 = 0; k2 < ranks; k2++) most = fmaxf(most, peer_load(&cta_top[r], k2));
                const float base = most == -INFINITY ? 0.f : most;
                y = all = 0.f;
                for (int k2 = 0; k2 < ranks; k2++) {
                    const float f = exp2f(peer_load(&cta_top[r], k2) - base);
                    y += peer_load(&o_sm[0][r][d], k2) * f;
                    all += peer_load(&cta_sum[r], k2) * f;
                }
            }
            y = all == 0.f ? 0.f : y / all;
            if (!INT8 && any_odd) y += what_is_no_number(v, row_bytes, d, s.pos + m / group, c.capacity, a.window, a.sinks);
            const int64_t to = (s.first + m / group) * a.out_stride + (kv_head * group + m % group) * a.out_head_stride + d;
            if (a.out_type == ZKB_VALUE_WORD) static_cast<uint32_t*>(a.out)[to] = round_bf16(y);
            else static_cast<uint16_t*>(a.out)[to] = round_bf16(y);
        }
        if (ranks > 1) cluster_sync();  // nobody leaves, or starts the next rows, while others read its part
        else __syncthreads();
    }
}

template <int D, bool INT8>
static cudaError_t launch_few(zkb_ctx* ctx, const zkb_step_attention_args& a, bool vec) {
    const zkb_kv_cache& c = a.cache;
    const uint32_t group = a.q_heads / c.n_heads, most = a.rows.max_rows ? std::min(a.rows.max_rows, a.rows.n_rows) : a.rows.n_rows;
    const uint32_t tiles = (uint32_t)std::min<uint64_t>(((uint64_t)most * group + 7) / 8, 1u << 20);
    uint64_t len = a.rows.max_len ? std::min(a.rows.max_len, c.capacity) : c.capacity;
    if (a.window) len = std::min<uint64_t>(len, (uint64_t)a.window + a.sinks + 32);
    // Split a sequence over more thread blocks while the GPU has room for them and each warp keeps two blocks of keys.
    const uint64_t units = (uint64_t)c.n_seqs * c.n_heads * tiles;
    uint32_t ranks = 1;
    while (ranks < 16 && units * ranks * 2 <= 148 * 4 && len > (uint64_t)ranks * FEW_WARPS * 16 * 2) ranks *= 2;
    auto kernel = vec ? attention_few_kernel<D, INT8, true> : attention_few_kernel<D, INT8, false>;
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) return e;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim = {ranks, 1, 1};
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(tiles * ranks, c.n_heads, c.n_seqs);
    cfg.blockDim = dim3(FEW_WARPS * 32);
    cfg.stream = ctx->stream;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, a);
}

template <int D>
static cudaError_t launch_attention(zkb_ctx* ctx, const zkb_step_attention_args& a) {
    const zkb_kv_cache& c = a.cache;
    const int64_t step = c.type == ZKB_VALUE_INT8 ? 16 : 8;
    const bool vec = aligned_to(c.k, 16) && aligned_to(c.v, 16) && c.seq_stride % step == 0 && c.head_stride % step == 0 && c.token_stride % step == 0;
    return c.type == ZKB_VALUE_INT8 ? launch_few<D, true>(ctx, a, vec) : launch_few<D, false>(ctx, a, vec);
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
    ZKB_CUDA(ctx, c.head_dim == 128 ? launch_attention<128>(ctx, a) : c.head_dim == 64 ? launch_attention<64>(ctx, a) : launch_attention<32>(ctx, a));
    return ZKB_OK;
}
