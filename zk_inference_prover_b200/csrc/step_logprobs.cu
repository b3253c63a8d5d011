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
// Measured: 4096 rows of 32003 bf16 logits 70 to 74 us without and 90 to 94 with the likeliest 5 (40 is the bytes' time): 14.7 warp instructions for 32 logits, and 60 % of all cycles issue one. By the
// source the sums are five of them, an exp2 and a half of every packed operation; the others have not been told apart. One row of 32000 floats 4.3 us without and 9 to 10 with the likeliest 8: trips to
// memory, barriers and a cluster's joining, one after the other.
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

// A thread's logits of a part: N 16-byte vectors on 16-byte boundaries, `threads` apart. The first one may reach before the part; values outside it are -infinity.
template <int TYPE, int N>
struct Logits {
    static constexpr int PER = TYPE == ZKB_VALUE_BF16 ? 8 : 4, SIZE = 16 / PER;
    static constexpr uint32_t NONE = TYPE == ZKB_VALUE_BF16 ? 0xff80ff80u : TYPE == ZKB_VALUE_WORD ? 0xff80u : 0xff800000u;
    uint32_t raw[N][4];
    const char* base;  // the part's first logit
    uint32_t n, ahead, threads, thread;
    __device__ __forceinline__ Logits(const char* first, uint32_t count, uint32_t all, uint32_t mine) : base(first), n(count), ahead((uint32_t)((uintptr_t)first & 15) / SIZE), threads(all), thread(mine) {}
    __device__ __forceinline__ uint32_t place(int i, int y) const { return ((uint32_t)i * threads + thread) * PER + y - ahead; }  // in the part (wraps before it)
    __device__ __forceinline__ void load_some(int i) {  // a vector of which a part, or nothing, is inside
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
    }
    __device__ __forceinline__ void load() {
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
    // From shared memory, where copy_row has put the whole ones.
    __device__ __forceinline__ void load_copied(uint32_t stage) {
        const uint32_t whole = (n + ahead) / PER;  // vectors up to the first that does not end inside
#pragma unroll
        for (int i = 0; i < N; i++) ld_shared4(stage + ((uint32_t)i * threads + thread) * 16, raw[i][0], raw[i][1], raw[i][2], raw[i][3]);
        if (thread == 0 && ahead) load_some(0);
#pragma unroll
        for (int i = 0; i < N; i++)
            if ((uint32_t)i * threads + thread >= whole) load_some(i);
    }
    __device__ __forceinline__ float value(int i, int y) const {
        if constexpr (TYPE == ZKB_VALUE_BF16) return y % 2 ? bf16_high(raw[i][y / 2]) : bf16_low(raw[i][y / 2]);
        else if constexpr (TYPE == ZKB_VALUE_WORD) return bf16_low(raw[i][y]);
        else return __uint_as_float(raw[i][y]);
    }
    __device__ __forceinline__ float largest_of(int i, float m) const {
        if constexpr (TYPE == ZKB_VALUE_BF16) {
            const uint32_t w = max_nan_bf16(max_nan_bf16(raw[i][0], raw[i][1]), max_nan_bf16(raw[i][2], raw[i][3]));
            return max_nan(m, max_nan(bf16_low(w), bf16_high(w)));
        } else {
            return max_nan(m, max_nan(max_nan(value(i, 0), value(i, 1)), max_nan(value(i, 2), value(i, 3))));
        }
    }
    // The largest one's word; NaN and +infinity are the largest word.
    __device__ __forceinline__ uint32_t largest() const {
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
        return mine < INFINITY ? value_word(mine) : 0xffffffffu;
    }
    // Sums of w = exp2(d) and of w d over this thread's logits x, d = (x - less) * log2_scale. What is below `low` is taken for that: its weight is zero, and so is its product with a number.
    __device__ __forceinline__ void weigh(float less, float low, float log2_scale, bool tokens, float& rest, float& lean) const {
        const uint32_t low_bf16 = (uint32_t)__bfloat16_as_ushort(__float2bfloat16_rd(low)) * 0x10001u;
        const uint64_t minus = both(-less, -less), by = both(log2_scale, log2_scale);
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
        rest = first_of(rests) + second_of(rests), lean = first_of(leans) + second_of(leans);
        // `low` leaves nothing where it is 200 or more below; it is not where there is no number that far below, where its step from `less` was rounded away, or where the product leaves 32
        // bits. -infinity is then told from the lowest number, and a weight of zero has no product.
        const float below = (less - (TYPE == ZKB_VALUE_BF16 ? bf16_low(low_bf16) : low)) * log2_scale;
        if (tokens && !(below >= 200.f && below < INFINITY)) {
            rest = lean = 0.f;
#pragma unroll
            for (int i = 0; i < N; i++)
#pragma unroll
                for (int y = 0; y < PER; y++) {
                    const float d = (value(i, y) - less) * log2_scale, w = exp2_fast(d);
                    rest += w, lean += w > 0.f ? w * d : 0.f;
                }
        }
    }
    // The sum of w without the largest one's.
    __device__ __forceinline__ float weigh_others(float less, float log2_scale) const {
        float rest = 0.f;
#pragma unroll
        for (int i = 0; i < N; i++)
#pragma unroll
            for (int y = 0; y < PER; y++) {
                const float x = value(i, y);
                rest += x != less ? exp2_fast((x - less) * log2_scale) : 0.f;
            }
        return rest;
    }
    // Those that reach the threshold, to a list shared by the warps (by a whole warp; mine: this thread's largest). `from`: the part's place in the row.
    __device__ __forceinline__ void list_reaching(uint32_t threshold, uint32_t mine, uint32_t from, uint64_t* list, uint32_t* n_list) const {
        uint64_t found = 0;
        float first = 0.f;  // the last one's value: the one that is written first
        if (mine >= threshold) {
            const float reach = word_value(threshold);
#pragma unroll
            for (int i = 0; i < N; i++)
                if (largest_of(i, -INFINITY) >= reach) {  // (few do)
#pragma unroll
                    for (int y = 0; y < PER; y++)
                        if (value(i, y) >= reach) found |= 1ull << (i * PER + y), first = value(i, y);
                }
        }
        if (!__any_sync(0xffffffffu, found != 0)) return;
        const uint32_t lane = threadIdx.x & 31, n_mine = __popcll(found);
        uint32_t before = n_mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t x = __shfl_up_sync(0xffffffffu, before, o);
            if (lane >= o) before += x;
        }
        uint32_t at = 0;
        if (lane == 31) at = atomicAdd(n_list, before);
        at = __shfl_sync(0xffffffffu, at, 31) + before - n_mine;
        if (found) {
            const uint32_t last_bit = 63 - __clzll(found);
            for (bool again = false; found && at < LP_LIST; at++, again = true) {  // the others are fetched once more
                const uint32_t bit = again ? __ffsll(found) - 1 : last_bit, where = place((int)(bit / PER), (int)(bit % PER));
                list[at] = (uint64_t)value_word(again ? logit_at<TYPE>(base, where) : first) << 32 | (0xffffffffu - (from + where));
                found &= ~(1ull << bit);
            }
        }
    }
};

// What a part's sums are relative to, from its largest word.
struct LpScale {
    float most, less, low;
    bool tokens;  // there is one at least, and no NaN or +infinity
    __device__ __forceinline__ LpScale(uint32_t word, float log2_scale) {
        tokens = word > WORD_NONE && word != 0xffffffffu;
        most = word == 0xffffffffu ? __int_as_float(0x7fc00000) : word_value(word);
        less = tokens ? most : 0.f;
        low = fminf(less, fmaxf(less - 300.f / log2_scale, -3.38953139e38f));  // (bf16 has none below)
    }
};

// Groups of `lanes` lanes: their largest words, and the n_top-th largest of those where that is a token's: as many values reach it. By every warp for itself, behind a barrier.
__device__ __forceinline__ void store_group(uint32_t* groups, uint32_t lanes, uint32_t warp, uint32_t lane, uint32_t word) {
    if (lanes == 32) word = __reduce_max_sync(0xffffffffu, word);
    else
        for (uint32_t o = 1; o < lanes; o <<= 1) word = max(word, __shfl_xor_sync(0xffffffffu, word, o));
    if (lane % lanes == 0) groups[warp * (32 / lanes) + lane / lanes] = word;
}
__device__ __forceinline__ uint32_t threshold_of(const uint32_t* groups, uint32_t n_groups, uint32_t lane, uint32_t n_top, uint32_t& most_word) {
    const uint32_t one = lane < n_groups ? groups[lane] : 0u, two = lane + 32 < n_groups ? groups[lane + 32] : 0u;
    most_word = __reduce_max_sync(0xffffffffu, max(one, two));
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
    return max(threshold, WORD_NONE + 1);
}
__device__ __forceinline__ float over_warps(const float* x, uint32_t warps, uint32_t lane) {
    float y = lane < warps ? x[lane] : 0.f;
#pragma unroll
    for (int o = 8; o; o >>= 1) y += __shfl_xor_sync(0xffffffffu, y, o);
    return __shfl_sync(0xffffffffu, y, 0);
}

// What a row's outputs are made of.
struct LpResult {
    float most, scale, log_total, total, lean;
    bool odd, none;
    __device__ __forceinline__ LpResult(float largest, uint32_t equal, float rest, float lean_sum, float by) : most(largest), scale(by), total((float)equal + rest), lean(lean_sum) {
        odd = most != most, none = most == -INFINITY;
        log_total = none ? 0.f : equal == 1 ? log1pf(rest) : logf(total);
    }
    __device__ __forceinline__ float log_probability(float x) const {
        if (odd) return __int_as_float(0x7fc00000);
        if (none || x == -INFINITY) return -INFINITY;
        const float d = x - most;  // (of two numbers that no float holds it is -infinity: scaled, it may be one)
        return (d > -INFINITY ? d * scale : x * scale - most * scale) - log_total;
    }
    __device__ __forceinline__ float entropy() const { return odd ? __int_as_float(0x7fc00000) : none ? 0.f : log_total - lean * 0.693147181f / total; }
    __device__ __forceinline__ void give(const zkb_step_logprobs_args& a, uint32_t t, uint32_t i, int32_t id, float x) const {
        float y = 0.f;
        if (id >= 0 && (uint32_t)id < a.vocab) y = log_probability(x);
        else if (a.off_table) atomicAdd(reinterpret_cast<unsigned long long*>(a.off_table), 1ull);
        a.logprobs[(int64_t)t * a.n_given + i] = y;
    }
    __device__ __forceinline__ void give_top(const zkb_step_logprobs_args& a, uint32_t t, uint32_t place, uint64_t key) const {
        a.top_ids[(int64_t)t * a.n_top + place] = odd || !key ? -1 : (int32_t)(0xffffffffu - (uint32_t)key);
        a.top_logprobs[(int64_t)t * a.n_top + place] = odd ? __int_as_float(0x7fc00000) : !key ? -INFINITY : log_probability(word_value((uint32_t)(key >> 32)));
    }
};

// Few rows, or long ones: a thread block has a row, or a piece of it. TYPE: ZKB_VALUE_*; N: 16-byte vectors a thread.
template <int TYPE, int N>
__global__ void __launch_bounds__(512, 2) logprobs_kernel(const __grid_constant__ LogprobArgs p) {
    constexpr int SIZE = Logits<TYPE, N>::SIZE;
    __shared__ LpPart parts[LP_PARTS];
    __shared__ uint64_t list[LP_LIST];
    __shared__ __align__(16) uint32_t groups[64];
    __shared__ float sums[3][16];
    __shared__ uint32_t n_list;
    __shared__ uint64_t best[16];
    const zkb_step_logprobs_args& a = p.a;
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5, rank = cluster_rank(), ranks = cluster_ranks(), n_top = a.n_top, n_groups = warps * (32 / p.lanes);
    const uint32_t begin = min(rank * p.piece, a.vocab), end = min(begin + p.piece, a.vocab), n_parts = (p.piece + p.part - 1) / p.part, t = blockIdx.x / ranks;
    if (threadIdx.x == 0) n_list = 0;
    if (threadIdx.x < 64 && threadIdx.x >= n_groups) groups[threadIdx.x] = 0;
    if (ranks > 1) cluster_arrive();
    const char* const row = static_cast<const char*>(a.logits) + (int64_t)t * a.logits_stride * SIZE;
    // what is asked of the row is on its way meanwhile
    const int32_t id_first = threadIdx.x < a.n_given && rank == 0 ? a.ids[(int64_t)t * a.n_given + threadIdx.x] : -1;
    const float given_first = id_first >= 0 && (uint32_t)id_first < a.vocab ? logit_at<TYPE>(row, (uint32_t)id_first) : 0.f;
    for (uint32_t q = 0; q < n_parts; q++) {
        const uint32_t from = min(begin + q * p.part, end), to = min(from + p.part, end), n = to - from;
        Logits<TYPE, N> x(row + (int64_t)from * SIZE, n, blockDim.x, threadIdx.x);
        x.load();
        const uint32_t mine = x.largest();
        store_group(groups, p.lanes, warp, lane, mine);
        __syncthreads();
        uint32_t most_word;
        const uint32_t threshold = threshold_of(groups, n_groups, lane, n_top, most_word);
        const LpScale s(most_word, p.log2_scale);
        float rest, lean;
        x.weigh(s.less, s.low, p.log2_scale, s.tokens, rest, lean);
#pragma unroll
        for (int o = 16; o; o >>= 1) rest += __shfl_xor_sync(0xffffffffu, rest, o), lean += __shfl_xor_sync(0xffffffffu, lean, o);
        if (lane == 0) sums[0][warp] = rest, sums[1][warp] = lean;
        if (n_top) x.list_reaching(threshold, mine, from, list, &n_list);
        __syncthreads();
        LpPart& part = parts[q];
        const uint32_t listed = n_list;
        rest = over_warps(sums[0], warps, lane);
        lean = over_warps(sums[1], warps, lane);
        uint32_t equal = 0;
        if (rest < 1.25f && s.tokens) {  // one token is likely: the sum without it, for all of its bits
            equal = 1;
            rest = x.weigh_others(s.less, p.log2_scale);
#pragma unroll
            for (int o = 16; o; o >>= 1) rest += __shfl_xor_sync(0xffffffffu, rest, o);
            if (lane == 0) sums[2][warp] = rest;
            __syncthreads();
            rest = over_warps(sums[2], warps, lane);
        }
        if (threadIdx.x == 0) part.most = s.most, part.rest = rest, part.lean = lean, part.equal = equal;
        if (listed <= LP_LIST) {
            for (uint32_t i = threadIdx.x; i < listed; i += blockDim.x) {
                const uint64_t key = list[i];
                uint32_t above = 0;
#pragma unroll 4
                for (uint32_t j = 0; j < listed; j++) above += list[j] > key;
                if (above < n_top) part.top[above] = key;
            }
            for (uint32_t i = listed + threadIdx.x; i < n_top; i += blockDim.x) part.top[i] = 0;
            __syncthreads();
        } else {
            uint64_t last = ~0ull;
            for (uint32_t k = 0; k < n_top; k++) {
                uint64_t key = 0;
#pragma unroll 4
                for (uint32_t i = threadIdx.x; i < n; i += blockDim.x) {  // (from memory: registers for this would be missed above)
                    const uint32_t w = value_word(logit_at<TYPE>(x.base, i));
                    const uint64_t y = (uint64_t)w << 32 | (0xffffffffu - (from + i));
                    if (w > WORD_NONE && y < last && y > key) key = y;
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
    const uint32_t all = ranks * n_parts;
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
    const LpResult r(most, equal, rest, lean, a.scale);
    if (threadIdx.x == 0 && a.entropy) a.entropy[t] = r.entropy();
    for (uint32_t i = threadIdx.x; i < a.n_given; i += blockDim.x) {
        const int32_t id = i == threadIdx.x ? id_first : a.ids[(int64_t)t * a.n_given + i];
        r.give(a, t, i, id, i == threadIdx.x ? given_first : id >= 0 && (uint32_t)id < a.vocab ? logit_at<TYPE>(row, (uint32_t)id) : 0.f);
    }
    // (a key's place is how many others are larger: the parts' keys are in order; places without a token lie behind those with one)
    for (uint32_t i = threadIdx.x; i < all * n_top; i += blockDim.x) {
        const uint32_t mine = i / n_top, place = i - mine * n_top;
        const uint64_t key = parts[mine].top[place];
        uint32_t above = place;
        if (key)
            for (uint32_t j = 0; j < all && above < n_top; j++)
                for (uint32_t k = 0; j != mine && k < n_top && parts[j].top[k] > key; k++) above++;
        if (key && above < n_top) r.give_top(a, t, above, key);
    }
    if (n_top) {  // what is left without a token
        uint32_t found = 0;
        for (uint32_t i = lane; i < all; i += 32) {
            uint32_t k = n_top;
            while (k > 0 && !parts[i].top[k - 1]) k--;
            found += k;
        }
        found = __reduce_add_sync(0xffffffffu, found);
        for (uint32_t i = found + threadIdx.x; i < n_top; i += blockDim.x) r.give_top(a, t, i, 0);
    }
}

// Many rows: a thread block has row after row. The next one comes to shared memory while this one is summed, and a warp of its own writes a row's outputs while the others are at the next:
// the chain from the last sum to the last store, some 2000 cycles, is hidden.
constexpr int LP_ROWS_N = 8;
template <int TYPE>
__global__ void __launch_bounds__(544, 2) logprobs_rows_kernel(const __grid_constant__ LogprobArgs p, unsigned* dev_err) {
    constexpr int SIZE = Logits<TYPE, LP_ROWS_N>::SIZE;
    extern __shared__ __align__(16) unsigned char row_sm[];
    __shared__ __align__(8) unsigned long long row_bar;
    __shared__ uint64_t list[2][LP_LIST];
    __shared__ __align__(16) uint32_t groups[64];
    __shared__ float sums[3][16], part_sm[2][3];  // most, rest, lean
    __shared__ uint32_t n_list[2], equal_sm[2];
    const zkb_step_logprobs_args& a = p.a;
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = (blockDim.x >> 5) - 1, threads = 32 * warps, n_top = a.n_top, n_groups = warps * (32 / p.lanes);
    const uint32_t stage = (uint32_t)__cvta_generic_to_shared(row_sm);
    auto row_of = [&](uint32_t t) { return static_cast<const char*>(a.logits) + (int64_t)t * a.logits_stride * SIZE; };
    // Barriers: 1 the summing warps', 2 and 3 a row's results are there, 4 and 5 they have been written.
    enum { SUMMING = 1, THERE = 2, WRITTEN = 4 };
    auto arrive = [&](int id) {
        __syncwarp();
        asm volatile("bar.arrive %0, %1;" ::"r"(id), "r"(threads + 32) : "memory");
    };
    if (threadIdx.x == 0) {
        mbar_init(bar_of(row_bar), 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        copy_row(stage, row_of(blockIdx.x), a.vocab * SIZE, bar_of(row_bar));
        n_list[0] = n_list[1] = 0;
    }
    if (threadIdx.x < 64 && threadIdx.x >= n_groups) groups[threadIdx.x] = 0;
    __syncthreads();
    uint32_t turn = 0;
    if (warp == warps) {  // ---- outputs
        for (uint32_t t = blockIdx.x; t < a.n_rows; t += gridDim.x, turn++) {
            const uint32_t buf = turn & 1;
            const char* const row = row_of(t);
            const int32_t id_first = lane < a.n_given ? a.ids[(int64_t)t * a.n_given + lane] : -1;
            const float given_first = id_first >= 0 && (uint32_t)id_first < a.vocab ? logit_at<TYPE>(row, (uint32_t)id_first) : 0.f;
            named_sync(THERE + buf, threads + 32);
            const uint32_t listed = n_list[buf];
            const LpResult r(part_sm[buf][0], equal_sm[buf], part_sm[buf][1], part_sm[buf][2], a.scale);
            if (lane == 0 && a.entropy) a.entropy[t] = r.entropy();
            for (uint32_t i = lane; i < a.n_given; i += 32) {
                const int32_t id = i == lane ? id_first : a.ids[(int64_t)t * a.n_given + i];
                r.give(a, t, i, id, i == lane ? given_first : id >= 0 && (uint32_t)id < a.vocab ? logit_at<TYPE>(row, (uint32_t)id) : 0.f);
            }
            __syncwarp();
            if (n_top) {
                // Lane k holds the k-th largest key so far: a larger one than the n_top-th takes its place and moves those behind it on. (Of equal logits the keys of lower indexes are larger.)
                uint64_t mine = 0, least = 0;
                auto take = [&](uint64_t key) {
                    uint32_t who = __ballot_sync(0xffffffffu, key > least);
                    while (who) {
                        const uint64_t k = __shfl_sync(0xffffffffu, key, __ffs(who) - 1);
                        const uint32_t smaller = __ballot_sync(0xffffffffu, mine < k), at = __ffs(smaller) - 1;  // (some lane's is: the n_top-th)
                        const uint64_t before = __shfl_up_sync(0xffffffffu, mine, 1);
                        if (lane == at) mine = k;
                        else if (lane > at) mine = before;
                        least = __shfl_sync(0xffffffffu, mine, n_top - 1);
                        who &= who - 1;
                        who &= __ballot_sync(0xffffffffu, key > least);
                    }
                };
                if (listed <= LP_LIST) {
                    for (uint32_t i = 0; i < listed; i += 32) take(i + lane < listed ? list[buf][i + lane] : 0);
                } else {
                    for (uint32_t i = 0; i < a.vocab; i += 256) {  // too many tie: from the row itself
                        uint64_t key[8];
#pragma unroll
                        for (int y = 0; y < 8; y++) {
                            const uint32_t at = i + y * 32 + lane, w = at < a.vocab ? value_word(logit_at<TYPE>(row, at)) : 0u;
                            key[y] = w > WORD_NONE ? (uint64_t)w << 32 | (0xffffffffu - at) : 0;
                        }
#pragma unroll
                        for (int y = 0; y < 8; y++) take(key[y]);
                    }
                }
                if (lane < n_top) r.give_top(a, t, lane, mine);
            }
            __syncwarp();
            if (lane == 0) n_list[buf] = 0;
            arrive(WRITTEN + buf);
        }
        return;
    }
    bool failed = false;
    for (uint32_t t = blockIdx.x; t < a.n_rows; t += gridDim.x, turn++) {
        const uint32_t buf = turn & 1;
        if (!failed) failed = !mbar_wait(bar_of(row_bar), turn & 1);
        Logits<TYPE, LP_ROWS_N> x(row_of(t), a.vocab, threads, threadIdx.x);
        x.load_copied(stage);
        const uint32_t mine = x.largest();
        __syncwarp();
        store_group(groups, p.lanes, warp, lane, mine);
        named_sync(SUMMING, threads);
        // all have their logits in registers
        if (threadIdx.x == threads - 1 && !failed && t + gridDim.x < a.n_rows) copy_row(stage, row_of(t + gridDim.x), a.vocab * SIZE, bar_of(row_bar));
        __syncwarp();
        uint32_t most_word;
        const uint32_t threshold = threshold_of(groups, n_groups, lane, n_top, most_word);
        const LpScale s(most_word, p.log2_scale);
        float rest, lean;
        x.weigh(s.less, s.low, p.log2_scale, s.tokens, rest, lean);
#pragma unroll
        for (int o = 16; o; o >>= 1) rest += __shfl_xor_sync(0xffffffffu, rest, o), lean += __shfl_xor_sync(0xffffffffu, lean, o);
        if (lane == 0) sums[0][warp] = rest, sums[1][warp] = lean;
        if (turn >= 2) named_sync(WRITTEN + buf, threads + 32);  // the list is free
        if (n_top) x.list_reaching(threshold, mine, 0, list[buf], &n_list[buf]);
        named_sync(SUMMING, threads);
        rest = over_warps(sums[0], warps, lane);
        uint32_t equal = 0;
        if (rest < 1.25f && s.tokens) {  // one token is likely: the sum without it, for all of its bits
            equal = 1;
            rest = x.weigh_others(s.less, p.log2_scale);
#pragma unroll
            for (int o = 16; o; o >>= 1) rest += __shfl_xor_sync(0xffffffffu, rest, o);
            if (lane == 0) sums[2][warp] = rest;
            named_sync(SUMMING, threads);
            rest = over_warps(sums[2], warps, lane);
        }
        if (warp == 0) {
            lean = over_warps(sums[1], warps, lane);
            if (lane == 0) part_sm[buf][0] = s.most, part_sm[buf][1] = rest, part_sm[buf][2] = lean, equal_sm[buf] = equal;
        }
        arrive(THERE + buf);
    }
    // (every arrival is waited for: the last rows' results have been written)
    for (uint32_t last = turn < 2 ? 0 : turn - 2; last < turn; last++) named_sync(WRITTEN + (last & 1), threads + 32);
    if (failed) {  // nothing is on its way to shared memory when the thread block gives it up
        *dev_err = WAIT_RAN_OUT;
        mbar_wait(bar_of(row_bar), (turn - 1) & 1);
    }
}

template <int TYPE>
static cudaError_t launch_logprobs(zkb_ctx* ctx, const zkb_step_logprobs_args& a) {
    constexpr uint32_t PER = TYPE == ZKB_VALUE_BF16 ? 8 : 4;
    // Few rows are spread over clusters of as many thread blocks as are on the GPU at once, 2048 logits each at least. By 1, 2, 4 and 8 thread blocks, in us: one row of 32000 floats 10.8, 8.1, 7.7,
    // 8.0; sixteen 10.6, 8.2, 7.7, 7.7.
    uint32_t ranks = 1;
    while (ranks < LP_RANKS && a.n_rows <= clusters_at_once(2 * ranks) && a.vocab >= ranks * 4096) ranks *= 2;
    return launch_clusters(ranks, [&](uint32_t n) {
        LogprobArgs p{a, 0, 0, 32, a.scale * 1.44269504f};
        p.piece = ((a.vocab + n - 1) / n + PER - 1) / PER * PER;
        const uint32_t at_most = 512 * LP_VECTORS * PER - PER;  // (less one vector: the first may begin before the piece)
        const uint32_t n_parts = (p.piece + at_most - 1) / at_most;
        p.part = ((p.piece + n_parts - 1) / n_parts + PER - 1) / PER * PER;
        const uint32_t vectors = p.part / PER + 1;
        // A vector a thread where that fills the GPU no more than once, up to eight where there are rows enough. By 64, 128, 256 and 512 threads: 64 rows of 4000 bf16 7.1, 6.0, 5.9, 5.9 us, 4096 rows
        // of them 28.3, 27.1, 42, 76.
        uint32_t threads = 64, each = 1;
        while (threads < 512 && threads < vectors && (threads * LP_VECTORS < vectors || (uint64_t)threads * n * a.n_rows < 148 * 512)) threads *= 2;
        while (each * threads < vectors) each *= 2;
        // The groups that look for the n_top largest, by lanes of a warp or by the whole of it: twice as many of those that have logits, where there are so many threads.
        while (p.lanes > 1 && threads / p.lanes < 64 && 2 * a.n_top > std::min(threads, vectors) / p.lanes) p.lanes /= 2;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim = {n, 1, 1};
        cudaLaunchConfig_t cfg = {};
        const uint32_t at_once = 148u * std::min(1024 / threads, 216 * 1024 / (threads * LP_ROWS_N * 16 + 18 * 1024));  // of the kernel for many rows
        // (4096 rows of 32003 bf16 logits 92 us, by a thread block a row 124; of 12000, 256 threads, 53 and 60; of 8000, 128 threads, 46 and 36: a warp for the outputs is too many there)
        const bool rows = n == 1 && n_parts == 1 && threads >= 256 && each == LP_ROWS_N && a.n_rows > at_once;
        cfg.gridDim = dim3(rows ? at_once : a.n_rows * n);
        cfg.blockDim = dim3(rows ? threads + 32 : threads);
        cfg.stream = ctx->stream;
        if (rows) {
            cfg.dynamicSmemBytes = threads * LP_ROWS_N * 16;
            const cudaError_t e = cudaFuncSetAttribute(logprobs_rows_kernel<TYPE>, cudaFuncAttributeMaxDynamicSharedMemorySize, 512 * LP_ROWS_N * 16);
            return e == cudaSuccess ? cudaLaunchKernelEx(&cfg, logprobs_rows_kernel<TYPE>, p, ctx->dev_err) : e;
        }
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
