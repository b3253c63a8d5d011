// What a model answers with: log probabilities of given tokens, the entropy, and the likeliest tokens of rows of logits.
#include <algorithm>
#include <cmath>
#include <cstdlib>

#include "step_attention.cuh"
#include "tensor_memory.cuh"

namespace zk {

// A row (a piece of it where rows are few: the thread blocks of a cluster have one each, and the first joins) stays in registers, so its logits are read once; longer pieces are
// taken in parts. With the part's largest value m, a second pass over the registers sums w = exp(z - m) and w (z - m):
//   lse = m + log(S),  entropy = log(S) - sum(w (z - m)) / S,  S = 1 + what the others leave, so that log1p has all of its bits where one token is nearly certain.
// The n_top largest: as many values reach the n_top-th largest of the maxima of groups of lanes, so the n_top largest do. Those that reach
// it, a few more than n_top, are listed, and each one's rank among them is counted; where too many tie for the list, they are found one after the other.
constexpr int LP_VECTORS = 8, LP_TOP = 32, LP_LIST = 1024, LP_PARTS = 64, LP_RANKS = 16;

// What is left of a part: the largest logit, how many have it, the sums over the others, the largest n_top with their places.
struct LpPart {
    float most, rest, lean;  // rest: sum of w, of all but `equal` ones with the largest logit; lean: sum of w * d, d = log2(w)
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

__device__ __forceinline__ uint32_t max_nan_bf16(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
__device__ __forceinline__ uint32_t max_bf16(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("max.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}

template <int TYPE>
__device__ __forceinline__ float logit_at(const char* row, uint32_t i) {
    if constexpr (TYPE == ZKB_VALUE_F32) return reinterpret_cast<const float*>(row)[i];
    else return bf16_low(TYPE == ZKB_VALUE_BF16 ? reinterpret_cast<const uint16_t*>(row)[i] : reinterpret_cast<const uint32_t*>(row)[i]);
}

// The whole 16-byte blocks of a row, into shared memory; how many bytes.
__device__ __forceinline__ uint32_t copy_row(uint32_t to, const char* row, uint32_t bytes, uint32_t bar) {
    const uint32_t ahead = -(uint32_t)(uintptr_t)row & 15, size = bytes > ahead ? (bytes - ahead) & ~15u : 0u;
    mbar_expect(bar, size);
    if (ahead) to += 16;  // (where the row's first block is)
    if (size) asm volatile("cp.async.bulk.shared::cta.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(to), "l"(row + ahead), "r"(size), "r"(bar) : "memory");
    return size;
}

// TYPE: ZKB_VALUE_*; N: 16-byte vectors a thread. STAGED: a thread block has row after row, and the next one comes to shared memory while this one is summed.
template <int TYPE, int N, bool STAGED>
__global__ void __launch_bounds__(512, 2) logprobs_kernel(const __grid_constant__ LogprobArgs p, unsigned* dev_err) {
    extern __shared__ __align__(16) unsigned char row_sm[];
    __shared__ __align__(8) unsigned long long row_bar;
    constexpr int PER = TYPE == ZKB_VALUE_BF16 ? 8 : 4, SIZE = 16 / PER;
    __shared__ LpPart parts[LP_PARTS];
    __shared__ uint64_t list[LP_LIST];
    __shared__ __align__(16) uint32_t groups[64];
    __shared__ float sums[3][16];
    __shared__ uint32_t n_list;
    __shared__ uint64_t best[16];
    const zkb_step_logprobs_args& a = p.a;
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5, rank = cluster_rank(), ranks = cluster_ranks(), n_top = a.n_top;
    const uint32_t begin = min(rank * p.piece, a.vocab), end = min(begin + p.piece, a.vocab), n_parts = (p.piece + p.part - 1) / p.part;
    const bool alone = ranks == 1 && n_parts == 1;
    if (threadIdx.x == 0) n_list = 0;
    if (threadIdx.x < 64 && threadIdx.x >= warps * (32 / p.lanes)) groups[threadIdx.x] = 0;
    if (ranks > 1) cluster_arrive();
    const uint32_t stage = (uint32_t)__cvta_generic_to_shared(row_sm);
    bool failed = false;
    uint32_t turn = 0;
    if constexpr (STAGED) {
        if (threadIdx.x == 0) {
            mbar_init(bar_of(row_bar), 1);
            asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            copy_row(stage, static_cast<const char*>(a.logits) + (int64_t)blockIdx.x * a.logits_stride * SIZE, a.vocab * SIZE, bar_of(row_bar));
        }
        __syncthreads();
    }
    for (uint32_t t = blockIdx.x / ranks; t < a.n_rows; t += gridDim.x / ranks) {  // (one row only where a cluster has it)
    const char* const row = static_cast<const char*>(a.logits) + (int64_t)t * a.logits_stride * SIZE;
    // what is asked of the row is on its way meanwhile
    const int32_t id_first = threadIdx.x < a.n_given && (!alone || warp == 0) ? a.ids[(int64_t)t * a.n_given + threadIdx.x] : -1;
    const float given_first = id_first >= 0 && (uint32_t)id_first < a.vocab ? logit_at<TYPE>(row, (uint32_t)id_first) : 0.f;
    for (uint32_t q = 0; q < n_parts; q++) {
        const uint32_t from = min(begin + q * p.part, end), to = min(from + p.part, end);
        // Vectors lie on 16-byte boundaries: the first one may reach before `from`, and values outside the part are -infinity.
        const char* const base = row + (int64_t)from * SIZE;
        const uint32_t ahead = (uint32_t)((uintptr_t)base & 15) / SIZE;
        auto place = [&](int i, int y) { return ((uint32_t)i * blockDim.x + threadIdx.x) * PER + y - ahead; };  // from `from` on (wraps below it)
        const uint32_t n = to - from;
        uint32_t raw[N][4];
        constexpr uint32_t NONE = TYPE == ZKB_VALUE_BF16 ? 0xff80ff80u : TYPE == ZKB_VALUE_WORD ? 0xff80u : 0xff800000u;
        auto load_some = [&](int i) {  // a vector of which a part, or nothing, is inside
            const uint32_t at = place(i, 0);
            raw[i][0] = raw[i][1] = raw[i][2] = raw[i][3] = NONE;
            if (at + (PER - 1) < n + (PER - 1)) {
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
        };
        if constexpr (STAGED) {
            if (!failed) failed = !mbar_wait(bar_of(row_bar), turn++ & 1);
            const uint32_t whole = (n + ahead) / PER;  // vectors up to the first that does not end inside
#pragma unroll
            for (int i = 0; i < N; i++) ld_shared4(stage + ((uint32_t)i * blockDim.x + threadIdx.x) * 16, raw[i][0], raw[i][1], raw[i][2], raw[i][3]);
            if (threadIdx.x == 0 && ahead) load_some(0);
#pragma unroll
            for (int i = 0; i < N; i++)
                if ((uint32_t)i * blockDim.x + threadIdx.x >= whole) load_some(i);
        } else {
#pragma unroll
            for (int i = 0; i < N; i++) {
                const uint32_t at = place(i, 0);
                if (at < n && n - at >= PER) {
                    const uint4 w = __ldcs(reinterpret_cast<const uint4*>(base + (int64_t)at * SIZE));
                    raw[i][0] = w.x, raw[i][1] = w.y, raw[i][2] = w.z, raw[i][3] = w.w;
                } else {
                    load_some(i);
                }
            }
        }
        auto value = [&](int i, int y) {
            if constexpr (TYPE == ZKB_VALUE_BF16) return y % 2 ? bf16_high(raw[i][y / 2]) : bf16_low(raw[i][y / 2]);
            else if constexpr (TYPE == ZKB_VALUE_WORD) return bf16_low(raw[i][y]);
            else return __uint_as_float(raw[i][y]);
        };
        auto largest_of = [&](int i, float m) {
            if constexpr (TYPE == ZKB_VALUE_BF16) {
                const uint32_t w = max_nan_bf16(max_nan_bf16(raw[i][0], raw[i][1]), max_nan_bf16(raw[i][2], raw[i][3]));
                return max_nan(m, max_nan(bf16_low(w), bf16_high(w)));
            } else {
                return max_nan(m, max_nan(max_nan(value(i, 0), value(i, 1)), max_nan(value(i, 2), value(i, 3))));
            }
        };
        float mine = -INFINITY;
        if constexpr (TYPE == ZKB_VALUE_BF16) {
            uint32_t w = 0xff80ff80u;
#pragma unroll
            for (int i = 0; i < N; i++) w = max_nan_bf16(w, max_nan_bf16(max_nan_bf16(raw[i][0], raw[i][1]), max_nan_bf16(raw[i][2], raw[i][3])));
            mine = max_nan(bf16_low(w), bf16_high(w));
        } else {
#pragma unroll
            for (int i = 0; i < N; i++) mine = largest_of(i, mine);
        }
        // NaN and +infinity are the largest word
        const uint32_t mine_word = mine < INFINITY ? value_word(mine) : 0xffffffffu;
        uint32_t group = mine_word;
        if (p.lanes == 32) group = __reduce_max_sync(0xffffffffu, group);
        else
            for (uint32_t o = 1; o < p.lanes; o <<= 1) group = max(group, __shfl_xor_sync(0xffffffffu, group, o));
        const uint32_t a_warp = 32 / p.lanes, n_groups = warps * a_warp;
        if (lane % p.lanes == 0) groups[warp * a_warp + lane / p.lanes] = group;
        __syncthreads();
        if constexpr (STAGED) {  // all have their logits in registers
            if (threadIdx.x == blockDim.x - 1 && !failed && t + gridDim.x < a.n_rows) copy_row(stage, row + (int64_t)gridDim.x * a.logits_stride * SIZE, a.vocab * SIZE, bar_of(row_bar));
        }
        // Every warp finds the largest of the groups' maxima, and the n_top-th largest, where that is a token's: as many values reach it.
        const uint32_t one = lane < n_groups ? groups[lane] : 0u, two = lane + 32 < n_groups ? groups[lane + 32] : 0u;
        const uint32_t most_word = __reduce_max_sync(0xffffffffu, max(one, two));
        uint32_t threshold = most_word;
        if (n_top > 1) {
            uint32_t above_one = 0, above_two = 0;
            for (uint32_t g = 0; g < n_groups; g += 4) {
                const uint4 o = *reinterpret_cast<const uint4*>(&groups[g]);
                above_one += (o.x > one) + (o.y > one) + (o.z > one) + (o.w > one);
                if (n_groups > 32) above_two += (o.x > two) + (o.y > two) + (o.z > two) + (o.w > two);
            }
            // the smallest that fewer than n_top are above: of equal ones any may be the n_top-th
            threshold = __reduce_min_sync(0xffffffffu, min(lane < n_groups && above_one < n_top ? one : 0xffffffffu, lane + 32 < n_groups && above_two < n_top ? two : 0xffffffffu));
            if (n_top > n_groups) threshold = 0;
        }
        threshold = max(threshold, WORD_NONE + 1);
        const float most = most_word == 0xffffffffu ? __int_as_float(0x7fc00000) : word_value(most_word);
        const float less = most_word <= WORD_NONE || most_word == 0xffffffffu ? 0.f : most;
        // What is further below is taken for that: its weight is zero, and so is its product with a number.
        const float low = fminf(less, fmaxf(less - 300.f / p.log2_scale, -3.38953139e38f));  // (bf16 has none below)
        const uint32_t low_bf16 = (uint32_t)__bfloat16_as_ushort(__float2bfloat16_rd(low)) * 0x10001u;
        const uint64_t minus = both(-less, -less), by = both(p.log2_scale, p.log2_scale);
        uint64_t rests = 0, leans = 0;  // (zero is a pair of zeros)
#pragma unroll
        for (int i = 0; i < N; i++)
#pragma unroll
            for (int y = 0; y < PER; y += 2) {
                float u, v;
                if constexpr (TYPE == ZKB_VALUE_BF16) {
                    const uint32_t w = max_bf16(raw[i][y / 2], low_bf16);
                    u = bf16_low(w), v = bf16_high(w);
                } else {
                    u = fmaxf(value(i, y), low), v = fmaxf(value(i, y + 1), low);
                }
                const uint64_t d = mul_both(add_both(both(u, v), minus), by), w = both(exp2_fast(first_of(d)), exp2_fast(second_of(d)));
                rests = add_both(rests, w);
                leans = fma_both(w, d, leans);
            }
        float rest = first_of(rests) + second_of(rests), lean = first_of(leans) + second_of(leans);
        if (most_word > WORD_NONE && (less - low) * p.log2_scale < 200.f) {  // there is no number that far below: -infinity is told from the lowest one
            rest = lean = 0.f;
#pragma unroll
            for (int i = 0; i < N; i++)
#pragma unroll
                for (int y = 0; y < PER; y++) {
                    const float x = value(i, y), d = (fmaxf(x, low) - less) * p.log2_scale, w = x > -INFINITY ? exp2_fast(d) : 0.f;
                    rest += w, lean = fmaf(w, d, lean);
                }
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) rest += __shfl_xor_sync(0xffffffffu, rest, o), lean += __shfl_xor_sync(0xffffffffu, lean, o);
        if (lane == 0) sums[0][warp] = rest, sums[1][warp] = lean;
        if (n_top) {
            uint64_t found = 0;  // which of this thread's values reach the threshold
            float first = 0.f;   // the last one of those, first written
            if (mine_word >= threshold) {
                const float reach = word_value(threshold);
#pragma unroll
                for (int i = 0; i < N; i++)
                    if (largest_of(i, -INFINITY) >= reach) {  // (few do)
#pragma unroll
                        for (int y = 0; y < PER; y++)
                            if (value(i, y) >= reach) found |= 1ull << (i * PER + y), first = value(i, y);
                    }
            }
            if (__any_sync(0xffffffffu, found != 0)) {
                const uint32_t n_mine = __popcll(found);
                uint32_t before = n_mine;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const uint32_t x = __shfl_up_sync(0xffffffffu, before, o);
                    if (lane >= o) before += x;
                }
                uint32_t at = 0;
                if (lane == 31) at = atomicAdd(&n_list, before);
                at = __shfl_sync(0xffffffffu, at, 31) + before - n_mine;
                if (found) {
                    const uint32_t top_bit = 63 - __clzll(found);
                    for (bool again = false; found && at < LP_LIST; at++, again = true) {  // the others are fetched once more
                        const uint32_t bit = again ? __ffsll(found) - 1 : top_bit, where = place((int)(bit / PER), (int)(bit % PER));
                        list[at] = (uint64_t)value_word(again ? logit_at<TYPE>(base, where) : first) << 32 | (0xffffffffu - (from + where));
                        found &= ~(1ull << bit);
                    }
                }
            }
        }
        __syncthreads();
        LpPart& part = parts[q];
        const uint32_t listed = n_list;
        auto over_warps = [&](const float* x) {
            float y = lane < warps ? x[lane] : 0.f;
#pragma unroll
            for (int o = 8; o; o >>= 1) y += __shfl_xor_sync(0xffffffffu, y, o);
            return __shfl_sync(0xffffffffu, y, 0);
        };
        rest = over_warps(sums[0]);
        lean = over_warps(sums[1]);
        uint32_t equal = 0;
        if (rest < 1.25f && most_word > WORD_NONE && most_word != 0xffffffffu) {  // one token is likely: the sum without it, for all of its bits
            equal = 1;
            rest = 0.f;
#pragma unroll
            for (int i = 0; i < N; i++)
#pragma unroll
                for (int y = 0; y < PER; y++) {
                    const float x = value(i, y), d = (fmaxf(x, low) - less) * p.log2_scale;
                    rest += x > -INFINITY && x != less ? exp2_fast(d) : 0.f;
                }
#pragma unroll
            for (int o = 16; o; o >>= 1) rest += __shfl_xor_sync(0xffffffffu, rest, o);
            if (lane == 0) sums[2][warp] = rest;
            __syncthreads();
            rest = over_warps(sums[2]);
        }
        if (threadIdx.x == 0) part.most = most, part.rest = rest, part.lean = lean, part.equal = equal;
        if (listed <= LP_LIST) {
            // a short list is the first warp's, while the others begin with the next row
            const uint32_t by_threads = alone && listed <= 64 ? 32u : blockDim.x;
            for (uint32_t i = threadIdx.x; i < listed && threadIdx.x < by_threads; i += by_threads) {
                const uint64_t key = list[i];
                uint32_t above = 0;
#pragma unroll 4
                for (uint32_t j = 0; j < listed; j++) above += list[j] > key;
                if (above < n_top) part.top[above] = key;
            }
            if (threadIdx.x < by_threads)
                for (uint32_t i = listed + threadIdx.x; i < n_top; i += by_threads) part.top[i] = 0;
            if (by_threads > 32) __syncthreads();
            else __syncwarp();
        } else {
            uint64_t last = ~0ull;
            for (uint32_t k = 0; k < n_top; k++) {
                uint64_t key = 0;
#pragma unroll 4
                for (uint32_t i = threadIdx.x; i < n; i += blockDim.x) {  // (from memory: registers for this would be missed above)
                    const uint32_t w = value_word(logit_at<TYPE>(base, i));
                    const uint64_t x = (uint64_t)w << 32 | (0xffffffffu - (from + i));
                    if (w > WORD_NONE && x < last && x > key) key = x;
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
        __syncwarp();
    }
    if (alone && warp) continue;  // the first warp has the rest of the row
    // The thread blocks' parts go to the first one's shared memory, behind its own.
    if (ranks > 1) {
        __syncthreads();
        cluster_wait();
        if (rank) {
            const uint32_t words = 4 + 2 * n_top;
            for (uint32_t i = threadIdx.x; i < words * n_parts; i += blockDim.x) {
                const uint32_t q = i / words;
                peer_store_word(reinterpret_cast<uint32_t*>(&parts[rank * n_parts + q]) + i % words, 0, reinterpret_cast<const uint32_t*>(&parts[q])[i % words]);
            }
        }
        cluster_arrive(), cluster_wait();
        if (rank) return;
    }
    const uint32_t all = ranks * n_parts, joiners = alone ? 32u : blockDim.x;
    // every warp joins the sums, a part a lane
    float most = -INFINITY;
    for (uint32_t i = lane; i < all; i += 32) most = max_nan(most, parts[i].most);
    if (all > 1)
#pragma unroll
        for (int o = 16; o; o >>= 1) most = max_nan(most, __shfl_xor_sync(0xffffffffu, most, o));
    else most = parts[0].most;
    float rest = 0.f, lean = 0.f;
    uint32_t equal = 0;
    for (uint32_t i = lane; i < all; i += 32) {
        const LpPart& x = parts[i];
        if (!(x.most > -INFINITY)) continue;
        const float d = fmaxf((x.most - most) * p.log2_scale, -300.f), w = exp2_fast(d);
        if (d == 0.f) equal += x.equal, rest += x.rest, lean += x.lean;
        else rest += w * (x.rest + (float)x.equal), lean += w * (x.lean + d * (x.rest + (float)x.equal));
    }
    if (all > 1) {
#pragma unroll
        for (int o = 16; o; o >>= 1) rest += __shfl_xor_sync(0xffffffffu, rest, o), lean += __shfl_xor_sync(0xffffffffu, lean, o);
        equal = __reduce_add_sync(0xffffffffu, equal);
    } else {
        rest = __shfl_sync(0xffffffffu, rest, 0), lean = __shfl_sync(0xffffffffu, lean, 0), equal = __shfl_sync(0xffffffffu, equal, 0);
    }
    constexpr float LN2 = 0.693147181f;
    const bool odd = most != most, none = most == -INFINITY;
    const float nan = __int_as_float(0x7fc00000);
    const float total = (float)equal + rest;
    const float log_total = none ? 0.f : equal == 1 ? log1pf(rest) : logf(total);
    auto log_probability = [&](float x) { return odd ? nan : none || x == -INFINITY ? -INFINITY : (x - most) * a.scale - log_total; };
    if (threadIdx.x == 0 && a.entropy) a.entropy[t] = odd ? nan : none ? 0.f : log_total - lean * LN2 / total;
    for (uint32_t i = threadIdx.x; i < a.n_given; i += joiners) {
        const int32_t id = i == threadIdx.x ? id_first : a.ids[(int64_t)t * a.n_given + i];
        float y = 0.f;
        if (id >= 0 && (uint32_t)id < a.vocab) {
            y = log_probability(i == threadIdx.x ? given_first : logit_at<TYPE>(row, (uint32_t)id));
        } else if (a.off_table) {
            atomicAdd(reinterpret_cast<unsigned long long*>(a.off_table), 1ull);
        }
        a.logprobs[(int64_t)t * a.n_given + i] = y;
    }
    // (a key's place is how many others are larger: the parts' keys are in order; places without a token lie behind those with one)
    for (uint32_t i = threadIdx.x; i < all * n_top; i += joiners) {
        const uint32_t mine = i / n_top, place = i - mine * n_top;
        const uint64_t key = parts[mine].top[place];
        uint32_t above = place;
        if (key || place == 0)
            for (uint32_t j = 0; j < all && above < n_top; j++)
                for (uint32_t k = 0; j != mine && k < n_top && parts[j].top[k] > key; k++) above++;
        if (key && above < n_top) {
            a.top_ids[(int64_t)t * n_top + above] = odd ? -1 : (int32_t)(0xffffffffu - (uint32_t)key);
            a.top_logprobs[(int64_t)t * n_top + above] = log_probability(word_value((uint32_t)(key >> 32)));
        }
    }
    if (n_top) {  // what is left without a token
        uint32_t found = 0;
        for (uint32_t i = lane; i < all; i += 32) {
            uint32_t k = n_top;
            while (k > 0 && !parts[i].top[k - 1]) k--;
            found += k;
        }
        found = __reduce_add_sync(0xffffffffu, found);
        for (uint32_t i = found + threadIdx.x; i < n_top; i += joiners) a.top_ids[(int64_t)t * n_top + i] = -1, a.top_logprobs[(int64_t)t * n_top + i] = odd ? nan : -INFINITY;
    }
    }
    if (STAGED && failed) {  // nothing is on its way to shared memory when the thread block gives it up
        *dev_err = WAIT_RAN_OUT;
        mbar_wait(bar_of(row_bar), (turn - 1) & 1);
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
        // A vector a thread where that fills the GPU no more than once, up to eight where there are rows enough.
        uint32_t threads = 64, each = 1;
        while (threads < 512 && threads < vectors && (threads * LP_VECTORS < vectors || (uint64_t)threads * n * a.n_rows < 148 * 512)) threads *= 2;
        while (each * threads < vectors) each *= 2;
        // The groups that look for the n_top largest, by lanes of a warp or by the whole of it: twice as many of those that have logits, where there are so many threads.
        while (p.lanes > 1 && threads / p.lanes < 64 && 2 * a.n_top > std::min(threads, vectors) / p.lanes) p.lanes /= 2;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim = {n, 1, 1};
        cudaLaunchConfig_t cfg = {};
        const uint32_t at_once = 148u * (1024 / threads);
        const bool staged = n == 1 && n_parts == 1 && each == 8 && a.n_rows > at_once;
        cfg.gridDim = dim3(n > 1 ? a.n_rows * n : std::min(a.n_rows, at_once));
        cfg.dynamicSmemBytes = staged ? threads * LP_VECTORS * 16 : 0;
        cfg.blockDim = dim3(threads);
        cfg.stream = ctx->stream;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        auto kernel = staged ? logprobs_kernel<TYPE, 8, true> : each == 1 ? logprobs_kernel<TYPE, 1, false> : each == 2 ? logprobs_kernel<TYPE, 2, false> : each == 4 ? logprobs_kernel<TYPE, 4, false> : logprobs_kernel<TYPE, 8, false>;
        cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        if (e == cudaSuccess && staged) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 512 * LP_VECTORS * 16);
        return e == cudaSuccess ? cudaLaunchKernelEx(&cfg, kernel, p, ctx->dev_err) : e;
    });
}

}  // namespace zk

using namespace zk;

extern "C" int zkb_step_logprobs(zkb_ctx* ctx, const zkb_step_logprobs_args* args) {
    if (!ctx) return ZKB_EINVAL;
    ZKB_CHECK_ARG(ctx, args);
    const zkb_step_logprobs_args& a = *args;
    ZKB_CHECK_ARG(ctx, a.type == ZKB_VALUE_BF16 || a.type == ZKB_VALUE_WORD || a.type == ZKB_VALUE_F32);
    ZKB_CHECK_ARG(ctx, a.vocab >= 1 && a.vocab <= (1u << 19) && a.n_rows <= (1u << 26) && a.n_top <= LP_TOP && a.n_given <= (1u << 19) && a.scale >= 0x1p-100f && a.scale <= 0x1p100f);
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
