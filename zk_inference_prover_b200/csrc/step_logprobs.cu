// What a model answers with: log probabilities of given tokens, the entropy, and the likeliest tokens of rows of logits.
#include <algorithm>
#include <cmath>
#include <cstdlib>

#include "step_attention.cuh"

namespace zk {

// A row (a piece of it where rows are few: the thread blocks of a cluster have one each, and the first joins) stays in registers, so its logits are read once; longer pieces are
// taken in parts. With the part's largest value m, a second pass over the registers sums w = exp(z - m) and w (z - m):
//   lse = m + log(S),  entropy = log(S) - sum(w (z - m)) / S,  S = 1 + what the others leave, so that log1p has all of its bits where one token is nearly certain.
// The n_top largest: the n_top-th largest of the maxima of groups of lanes is no larger than the n_top-th largest value, so the values that reach it, a few more
// than n_top, are listed, and each one's rank among them is counted; where too many tie for the list, they are found one after the other.
constexpr int LP_VECTORS = 8, LP_TOP = 32, LP_LIST = 1024, LP_PARTS = 64, LP_RANKS = 16;

// What is left of a part: the largest logit, how many have it, the sums over the others, the largest n_top with their places.
struct LpPart {
    float most, rest, lean;  // rest: sum of w; lean: sum of w * d, d = log2(w)
    uint32_t equal;
    uint64_t top[LP_TOP];  // value_word << 32 | ~index, 0: none
};

__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
// Ordered as the value, 0 and -0 alike; -infinity and below: up to 0x007fffff.
__device__ __forceinline__ uint32_t value_word(float x) {
    const uint32_t u = __float_as_uint(x + 0.f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float word_value(uint32_t u) { return __uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~u); }
constexpr uint32_t WORD_NONE = 0x007fffffu;  // -infinity's

struct LogprobArgs {
    zkb_step_logprobs_args a;
    uint32_t piece, part, lanes;  // logits of a thread block, of a part; lanes of a group
    float log2_scale;
};

// TYPE: ZKB_VALUE_*; N: 16-byte vectors a thread.
template <int TYPE, int N>
__global__ void __launch_bounds__(512, N == 8 ? 2 : 1) logprobs_kernel(const __grid_constant__ LogprobArgs p) {
    constexpr int PER = TYPE == ZKB_VALUE_BF16 ? 8 : 4, SIZE = 16 / PER;
    __shared__ LpPart parts[LP_PARTS];
    __shared__ uint64_t list[LP_LIST];
    __shared__ uint32_t groups[64];
    __shared__ float sums[3][16];
    __shared__ uint32_t n_list;
    __shared__ uint64_t best[16];
    const zkb_step_logprobs_args& a = p.a;
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5, rank = cluster_rank(), ranks = cluster_ranks(), n_top = a.n_top;
    const uint32_t t = blockIdx.x / ranks;
    const char* const row = static_cast<const char*>(a.logits) + (int64_t)t * a.logits_stride * SIZE;
    const uint32_t begin = min(rank * p.piece, a.vocab), end = min(begin + p.piece, a.vocab), n_parts = (p.piece + p.part - 1) / p.part;
    if (threadIdx.x == 0) n_list = 0;
    for (uint32_t q = 0; q < n_parts; q++) {
        const uint32_t from = min(begin + q * p.part, end), to = min(from + p.part, end);
        // Vectors lie on 16-byte boundaries: the first one may reach before `from`, and values outside the part are -infinity.
        const char* const base = row + (int64_t)from * SIZE;
        const uint32_t ahead = (uint32_t)((uintptr_t)base & 15) / SIZE;
        auto place = [&](int i, int y) { return ((uint32_t)i * blockDim.x + threadIdx.x) * PER + y - ahead; };  // from `from` on (wraps below it)
        const uint32_t n = to - from;
        uint32_t raw[N][4];
#pragma unroll
        for (int i = 0; i < N; i++) {
            const uint32_t at = place(i, 0);
            constexpr uint32_t NONE = TYPE == ZKB_VALUE_BF16 ? 0xff80ff80u : TYPE == ZKB_VALUE_WORD ? 0xff80u : 0xff800000u;
            raw[i][0] = raw[i][1] = raw[i][2] = raw[i][3] = NONE;
            if (at < n && n - at >= PER) {
                const uint4 w = __ldcs(reinterpret_cast<const uint4*>(base + (int64_t)at * SIZE));
                raw[i][0] = w.x, raw[i][1] = w.y, raw[i][2] = w.z, raw[i][3] = w.w;
            } else if (at + (PER - 1) < n + (PER - 1)) {  // a part of the vector is inside
#pragma unroll
                for (int y = 0; y < PER; y++)
                    if (at + y < n) {
                        if constexpr (TYPE == ZKB_VALUE_BF16) {
                            const uint32_t h = *reinterpret_cast<const uint16_t*>(base + (int64_t)(int32_t)(at + y) * SIZE);
                            raw[i][y / 2] = y % 2 ? (raw[i][y / 2] & 0xffffu) | h << 16 : (raw[i][y / 2] & 0xffff0000u) | h;
                        } else {
                            raw[i][y] = *reinterpret_cast<const uint32_t*>(base + (int64_t)(int32_t)(at + y) * SIZE);
                        }
                    }
            }
        }
        auto value = [&](int i, int y) {
            if constexpr (TYPE == ZKB_VALUE_BF16) return y % 2 ? bf16_high(raw[i][y / 2]) : bf16_low(raw[i][y / 2]);
            else if constexpr (TYPE == ZKB_VALUE_WORD) return bf16_low(raw[i][y]);
            else return __uint_as_float(raw[i][y]);
        };
        float mine = -INFINITY;
#pragma unroll
        for (int i = 0; i < N; i++)
#pragma unroll
            for (int y = 0; y < PER; y++) mine = max_nan(mine, value(i, y));
        // NaN and +infinity are the largest word
        uint32_t word = mine < INFINITY ? value_word(mine) : 0xffffffffu, group = word;
        const uint32_t mine_word = word;
        for (uint32_t o = 1; o < p.lanes; o <<= 1) group = max(group, __shfl_xor_sync(0xffffffffu, group, o));
        const uint32_t a_warp = 32 / p.lanes, n_groups = warps * a_warp;
        if (lane % p.lanes == 0) groups[warp * a_warp + lane / p.lanes] = group;
        __syncthreads();
        // every warp finds the largest and the n_top-th largest of the groups
        uint32_t one = lane < n_groups ? groups[lane] : 0u, two = lane + 32 < n_groups ? groups[lane + 32] : 0u;
        if (two > one) { const uint32_t s = one; one = two, two = s; }
        uint32_t most_word = __reduce_max_sync(0xffffffffu, one), threshold = most_word;
        for (uint32_t k = 1; k < n_top; k++) {
            const uint32_t who = __ballot_sync(0xffffffffu, one == threshold);
            if ((int)lane == __ffs(who) - 1) one = two, two = 0u;
            threshold = __reduce_max_sync(0xffffffffu, one);
        }
        threshold = max(threshold, WORD_NONE + 1);
        const float most = most_word == 0xffffffffu ? __int_as_float(0x7fc00000) : word_value(most_word);
        const float less = most_word <= WORD_NONE || most_word == 0xffffffffu ? 0.f : most;
        float rest = 0.f, lean = 0.f;
        uint32_t equal = 0;
#pragma unroll
        for (int i = 0; i < N; i++)
#pragma unroll
            for (int y = 0; y < PER; y++) {
                const float d = fmaxf((value(i, y) - less) * p.log2_scale, -300.f), w = exp2_fast(d);  // below 2^-126 nothing counts
                if (d < 0.f) rest += w;
                else equal++;
                lean = fmaf(w, d, lean);
            }
        if (most_word <= WORD_NONE) equal = 0;
        if (n_top && mine_word >= threshold) {
#pragma unroll
            for (int i = 0; i < N; i++)
#pragma unroll
                for (int y = 0; y < PER; y++) {
                    const uint32_t w = value_word(value(i, y));
                    if (w >= threshold && place(i, y) < n) {
                        const uint32_t at = atomicAdd(&n_list, 1u);
                        if (at < LP_LIST) list[at] = (uint64_t)w << 32 | (0xffffffffu - (from + place(i, y)));
                    }
                }
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) rest += __shfl_xor_sync(0xffffffffu, rest, o), lean += __shfl_xor_sync(0xffffffffu, lean, o);
        equal = __reduce_add_sync(0xffffffffu, equal);
        if (lane == 0) sums[0][warp] = rest, sums[1][warp] = lean, sums[2][warp] = __uint_as_float(equal);
        __syncthreads();
        LpPart& part = parts[q];
        const uint32_t listed = n_list;
        if (warp == 0) {
            float r = lane < warps ? sums[0][lane] : 0.f, l = lane < warps ? sums[1][lane] : 0.f;
            uint32_t e = lane < warps ? __float_as_uint(sums[2][lane]) : 0u;
#pragma unroll
            for (int o = 16; o; o >>= 1) r += __shfl_xor_sync(0xffffffffu, r, o), l += __shfl_xor_sync(0xffffffffu, l, o);
            e = __reduce_add_sync(0xffffffffu, e);
            if (lane == 0) part.most = most, part.rest = r, part.lean = l, part.equal = e;
        }
        if (listed <= LP_LIST) {
            for (uint32_t i = threadIdx.x; i < listed; i += blockDim.x) {
                const uint64_t key = list[i];
                uint32_t above = 0;
                for (uint32_t j = 0; j < listed; j++) above += list[j] > key;
                if (above < n_top) part.top[above] = key;
            }
            for (uint32_t i = listed + threadIdx.x; i < n_top; i += blockDim.x) part.top[i] = 0;
            __syncthreads();
        } else {
            uint64_t last = ~0ull;
            for (uint32_t k = 0; k < n_top; k++) {
                uint64_t key = 0;
#pragma unroll
                for (int i = 0; i < N; i++)
#pragma unroll
                    for (int y = 0; y < PER; y++) {
                        const uint32_t w = value_word(value(i, y));
                        const uint64_t x = (uint64_t)w << 32 | (0xffffffffu - (from + place(i, y)));
                        if (w > WORD_NONE && place(i, y) < n && x < last && x > key) key = x;
                    }
#pragma unroll
                for (int o = 16; o; o >>= 1) {
                    const uint64_t other = __shfl_xor_sync(0xffffffffu, key, o);
                    key = key > other ? key : other;
                }
                if (lane == 0) best[warp] = key;
                __syncthreads();
                key = 0;
                for (uint32_t i = 0; i < warps; i++) key = best[i] > key ? best[i] : key;
                if (threadIdx.x == 0) part.top[k] = key;
                last = key;
                __syncthreads();
            }
        }
        if (threadIdx.x == 0) n_list = 0;
    }
    // The thread blocks' parts go to the first one's shared memory, behind its own.
    if (ranks > 1) {
        cluster_arrive(), cluster_wait();
        if (rank) {
            for (uint32_t q = 0; q < n_parts; q++) {
                LpPart& to = parts[rank * n_parts + q];
                const LpPart& mine = parts[q];
                const uint32_t words = 4 + 2 * n_top;
                for (uint32_t i = threadIdx.x; i < words; i += blockDim.x) peer_store_word(reinterpret_cast<uint32_t*>(&to) + i, 0, reinterpret_cast<const uint32_t*>(&mine)[i]);
            }
        }
        cluster_arrive(), cluster_wait();
        if (rank) return;
    } else {
        __syncthreads();
    }
    const uint32_t all = ranks * n_parts;
    // every thread joins the sums: they are a few
    float most = -INFINITY;
    for (uint32_t i = 0; i < all; i++) most = max_nan(most, parts[i].most);
    float rest = 0.f, lean = 0.f;
    uint32_t equal = 0;
    for (uint32_t i = 0; i < all; i++) {
        const LpPart& x = parts[i];
        if (!(x.most > -INFINITY)) continue;
        const float d = fmaxf((x.most - most) * p.log2_scale, -300.f), w = exp2_fast(d);
        if (d == 0.f) equal += x.equal, rest += x.rest, lean += x.lean;
        else rest += w * (x.rest + (float)x.equal), lean += w * (x.lean + d * (x.rest + (float)x.equal));
    }
    constexpr float LN2 = 0.693147181f;
    const bool odd = most != most, none = most == -INFINITY;
    const float nan = __int_as_float(0x7fc00000);
    const float total = (float)equal + rest;
    const float log_total = none ? 0.f : equal == 1 ? log1pf(rest) : logf(total);
    auto log_probability = [&](float x) { return odd ? nan : none || x == -INFINITY ? -INFINITY : (x - most) * a.scale - log_total; };
    if (threadIdx.x == 0 && a.entropy) a.entropy[t] = odd ? nan : none ? 0.f : log_total - lean * LN2 / total;
    for (uint32_t i = threadIdx.x; i < a.n_given; i += blockDim.x) {
        const int32_t id = a.ids[(int64_t)t * a.n_given + i];
        float y = 0.f;
        if (id >= 0 && (uint32_t)id < a.vocab) {
            const char* at = row + (int64_t)id * SIZE;
            y = log_probability(TYPE == ZKB_VALUE_F32 ? *reinterpret_cast<const float*>(at) : bf16_low(TYPE == ZKB_VALUE_BF16 ? *reinterpret_cast<const uint16_t*>(at) : *reinterpret_cast<const uint32_t*>(at)));
        } else if (a.off_table) {
            atomicAdd(reinterpret_cast<unsigned long long*>(a.off_table), 1ull);
        }
        a.logprobs[(int64_t)t * a.n_given + i] = y;
    }
    for (uint32_t i = threadIdx.x; i < all * n_top; i += blockDim.x) {
        const uint64_t key = parts[i / n_top].top[i % n_top];
        uint32_t above = 0;
        for (uint32_t j = 0; j < all; j++)
            for (uint32_t k = 0; k < n_top; k++) {
                const uint64_t other = parts[j].top[k];
                if (other < key || (other == key && (key || j * n_top + k >= i))) break;  // (in order; places without a token behind those with one, among themselves by their number)
                above++;
            }
        if (above < n_top) {
            const bool is = key && !odd;
            a.top_ids[(int64_t)t * n_top + above] = is ? (int32_t)(0xffffffffu - (uint32_t)key) : -1;
            a.top_logprobs[(int64_t)t * n_top + above] = is ? log_probability(word_value((uint32_t)(key >> 32))) : odd ? nan : -INFINITY;
        }
    }
}

template <int TYPE>
static cudaError_t launch_logprobs(zkb_ctx* ctx, const zkb_step_logprobs_args& a) {
    constexpr uint32_t PER = TYPE == ZKB_VALUE_BF16 ? 8 : 4;
    // Few rows are spread over clusters of as many thread blocks as are on the GPU at once, 2048 logits each at least.
    uint32_t ranks = 1;
    while (ranks < LP_RANKS && a.n_rows <= clusters_at_once(2 * ranks) && a.vocab >= ranks * 4096) ranks *= 2;
    return launch_clusters(ranks, [&](uint32_t n) {
        LogprobArgs p{a, 0, 0, 32, a.scale * 1.44269504f};
        p.piece = ((a.vocab + n - 1) / n + PER - 1) / PER * PER;
        const uint32_t at_most = 512 * LP_VECTORS * PER - PER;  // (less one vector: the first may begin before the piece)
        const uint32_t n_parts = (p.piece + at_most - 1) / at_most;
        p.part = ((p.piece + n_parts - 1) / n_parts + PER - 1) / PER * PER;
        const uint32_t vectors = p.part / PER + 1;
        uint32_t threads = 64;
        while (threads < 512 && vectors > threads) threads *= 2;
        uint32_t each = 1;
        while (each * threads < vectors) each *= 2;
        while (a.n_top > threads / p.lanes) p.lanes /= 2;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim = {n, 1, 1};
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(a.n_rows * n);
        cfg.blockDim = dim3(threads);
        cfg.stream = ctx->stream;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        auto kernel = each == 1 ? logprobs_kernel<TYPE, 1> : each == 2 ? logprobs_kernel<TYPE, 2> : each == 4 ? logprobs_kernel<TYPE, 4> : logprobs_kernel<TYPE, 8>;
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        return e == cudaSuccess ? cudaLaunchKernelEx(&cfg, kernel, p) : e;
    });
}

}  // namespace zk

using namespace zk;

extern "C" int zkb_step_logprobs(zkb_ctx* ctx, const zkb_step_logprobs_args* args) {
    if (!ctx) return ZKB_EINVAL;
    ZKB_CHECK_ARG(ctx, args);
    const zkb_step_logprobs_args& a = *args;
    ZKB_CHECK_ARG(ctx, a.type == ZKB_VALUE_BF16 || a.type == ZKB_VALUE_WORD || a.type == ZKB_VALUE_F32);
    ZKB_CHECK_ARG(ctx, a.vocab >= 1 && a.vocab <= (1u << 19) && a.n_rows <= (1u << 26) && a.n_top <= LP_TOP && a.n_given <= (1u << 19) && std::isfinite(a.scale) && a.scale > 0.f);
    if (a.n_rows == 0) return ZKB_OK;
    ZKB_CHECK_ARG(ctx, a.logits && aligned_to(a.logits, a.type == ZKB_VALUE_BF16 ? 2 : 4));
    ZKB_CHECK_ARG(ctx, a.n_given == 0 || (a.ids && a.logprobs && aligned_to(a.ids, 4) && aligned_to(a.logprobs, 4)));
    ZKB_CHECK_ARG(ctx, a.n_top == 0 || (a.top_ids && a.top_logprobs && aligned_to(a.top_ids, 4) && aligned_to(a.top_logprobs, 4)));
    ZKB_CHECK_ARG(ctx, aligned_to(a.entropy, 4) && aligned_to(a.off_table, 8));
    DeviceGuard g(ctx);
    ProfScope prof(ctx, "step_logprobs_kernel");
    ZKB_CUDA(ctx, a.type == ZKB_VALUE_BF16 ? launch_logprobs<ZKB_VALUE_BF16>(ctx, a) : a.type == ZKB_VALUE_WORD ? launch_logprobs<ZKB_VALUE_WORD>(ctx, a) : launch_logprobs<ZKB_VALUE_F32>(ctx, a));
    return ZKB_OK;
}
