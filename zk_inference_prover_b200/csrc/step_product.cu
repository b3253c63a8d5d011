// Products of 8-bit codes with weights held as 8-bit or 4-bit codes.
#include <algorithm>
#include <cmath>
#include <cstdlib>

#include "step_product.cuh"

namespace zk {

// ---- few rows ------------------------------------------------------------------------------------------------------------------------
// The weights are read once and everything else is small, so this is bound by the weights' bytes. A thread block has CHANNELS outputs of R rows; its warps' lanes take turns in
// the weights, 16 bytes each, and multiply four codes an instruction (dp4a). Of 4-bit codes the two halves of the bytes are taken apart in place, as 16 times the code, against
// the even and the odd codes of x; 16 bytes are 32 codes of one group, whose sum is exact and then scaled. One row of 4096 x 32000 8-bit codes: 22.7 to 24.6 us, 5.3 to 5.8 TB/s, its loads' latency
// between a thread block's start and its end is what is left; of 4096 x 4096 4-bit codes 3.5 to 4.1 us, where a launch and three trips to memory are most of it.
constexpr int CHANNELS = 4, FEW_WARPS = 4;

// VEC: all rows of x and of the weights start on 16-byte boundaries.
template <bool INT4, int R, bool VEC>
__global__ void __launch_bounds__(32 * FEW_WARPS, R == 1 ? 8 : 6) product_few_kernel(const __grid_constant__ zkb_step_product_args a) {
    __shared__ uint32_t joined[FEW_WARPS][R][CHANNELS];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint32_t c0 = blockIdx.x * CHANNELS;
    constexpr int CODES = INT4 ? 32 : 16, XS = CODES / 16;  // codes of 16 bytes; 16s of x to them
    const int n_in = (int)a.n_in, bytes = INT4 ? (n_in + 1) / 2 : n_in;
    const int64_t w_row = INT4 ? a.w_stride / 2 : a.w_stride;
    const int8_t *const w_lo = static_cast<const int8_t*>(a.w), *const w_hi = w_lo + (a.n_out - 1) * w_row + bytes, *const x_hi = a.x + (int64_t)(a.n_rows - 1) * a.x_stride + n_in;
    auto w_of = [&](int c) { return w_lo + (int64_t)min(c0 + c, a.n_out - 1) * w_row; };
    auto x_of = [&](int r) { return a.x + (int64_t)min((uint32_t)r, a.n_rows - 1) * a.x_stride; };
    const uint32_t log_group = INT4 ? 31 - __clz(a.group) : 0;
    int sum[CHANNELS][R] = {};
    float part[CHANNELS][R] = {};
    // 16 bytes of each output's weights, from byte b of its row on, times x_at(row, which 16 codes)
    auto multiply = [&](int b, const uint4 (&v)[CHANNELS], auto x_at) {
        float by[CHANNELS];
#pragma unroll
        for (int c = 0; c < CHANNELS; c++)
            if constexpr (INT4)
                by[c] = bf16_low(static_cast<const uint16_t*>(a.w_scale)[(int64_t)min(c0 + c, a.n_out - 1) * a.w_scale_stride + ((uint32_t)(b * 2) >> log_group)]) * 0.0625f;
#pragma unroll
        for (int r = 0; r < R; r++) {
            uint32_t xs[4 * XS];
#pragma unroll
            for (int i = 0; i < XS; i++) {
                const uint4 u = x_at(r, i);
                xs[4 * i] = u.x, xs[4 * i + 1] = u.y, xs[4 * i + 2] = u.z, xs[4 * i + 3] = u.w;
            }
            if constexpr (INT4) {
                uint32_t even[4], odd[4];
#pragma unroll
                for (int i = 0; i < 4; i++) even[i] = __byte_perm(xs[2 * i], xs[2 * i + 1], 0x6420), odd[i] = __byte_perm(xs[2 * i], xs[2 * i + 1], 0x7531);
#pragma unroll
                for (int c = 0; c < CHANNELS; c++) {
                    const uint32_t w[4] = {v[c].x, v[c].y, v[c].z, v[c].w};
                    int d = 0;
#pragma unroll
                    for (int i = 0; i < 4; i++) d = __dp4a((int)(w[i] << 4 & 0xf0f0f0f0u), (int)even[i], d), d = __dp4a((int)(w[i] & 0xf0f0f0f0u), (int)odd[i], d);
                    part[c][r] = fmaf((float)d, by[c], part[c][r]);
                }
            } else {
#pragma unroll
                for (int c = 0; c < CHANNELS; c++) {
                    const uint32_t w[4] = {v[c].x, v[c].y, v[c].z, v[c].w};
#pragma unroll
                    for (int i = 0; i < 4; i++) sum[c][r] = __dp4a((int)w[i], (int)xs[i], sum[c][r]);
                }
            }
        }
    };
    const int whole = n_in / CODES * 16;  // bytes of a row's weights in whole 16s of codes
    if constexpr (VEC) {
#pragma unroll(R == 1 ? 2 : 1)
        for (int b = threadIdx.x * 16; b < whole; b += 512 * FEW_WARPS) {
            uint4 v[CHANNELS];
#pragma unroll
            for (int c = 0; c < CHANNELS; c++) v[c] = __ldg(reinterpret_cast<const uint4*>(w_of(c) + b));
            multiply(b, v, [&](int r, int i) { return __ldg(reinterpret_cast<const uint4*>(x_of(r) + b * XS + 16 * i)); });
        }
    } else {
#pragma unroll 1
        for (int b = threadIdx.x * 16; b < whole; b += 512 * FEW_WARPS) {
            Fetched f[CHANNELS];
            uint4 v[CHANNELS];
#pragma unroll
            for (int c = 0; c < CHANNELS; c++) f[c] = fetch16(w_of(c) + b, w_lo, w_hi);
#pragma unroll
            for (int c = 0; c < CHANNELS; c++) v[c] = fetched16(f[c], w_of(c) + b, w_lo, w_hi);
            multiply(b, v, [&](int r, int i) {
                const int8_t* const from = x_of(r) + b * XS + 16 * i;
                return fetched16(fetch16(from, a.x, x_hi), from, a.x, x_hi);
            });
        }
    }
    if (whole < bytes && threadIdx.x == whole / 16 % (32 * FEW_WARPS)) {  // the last codes: what lies behind them counts for nothing
        uint4 v[CHANNELS];
#pragma unroll
        for (int c = 0; c < CHANNELS; c++) v[c] = some_bytes(w_of(c) + whole, bytes - whole);
        multiply(whole, v, [&](int r, int i) { return some_bytes(x_of(r) + whole * XS + 16 * i, n_in - whole * XS - 16 * i); });
    }
#pragma unroll
    for (int r = 0; r < R; r++)
#pragma unroll
        for (int c = 0; c < CHANNELS; c++) {
            uint32_t y;
            if constexpr (INT4) {
                float f = part[c][r];
#pragma unroll
                for (int o = 16; o; o >>= 1) f += __shfl_xor_sync(0xffffffffu, f, o);
                y = __float_as_uint(f);
            } else {
                y = (uint32_t)__reduce_add_sync(0xffffffffu, sum[c][r]);
            }
            if (lane == 0) joined[warp][r][c] = y;
        }
    __syncthreads();
    const uint32_t c = threadIdx.x % CHANNELS, r = threadIdx.x / CHANNELS;
    if (r < R && c0 + c < a.n_out && r < a.n_rows) {
        uint32_t y = joined[0][r][c];
#pragma unroll
        for (int w = 1; w < FEW_WARPS; w++) y = INT4 ? __float_as_uint(__uint_as_float(y) + __uint_as_float(joined[w][r][c])) : y + joined[w][r][c];
        const int64_t at = (int64_t)r * a.out_stride + c0 + c;
        if (a.out_type == ZKB_VALUE_INT32) static_cast<uint32_t*>(a.out)[at] = y;
        else store_value(a.out, at, a.out_type, INT4 ? __uint_as_float(y) * a.x_scale[r] : (float)(int)y * (a.x_scale[r] * static_cast<const float*>(a.w_scale)[c0 + c]));
    }
}

template <bool INT4>
static cudaError_t launch_few(zkb_ctx* ctx, const zkb_step_product_args& a, bool vec) {
    const uint32_t grid = (a.n_out + CHANNELS - 1) / CHANNELS;
    if (a.n_rows == 2) product_few_kernel<INT4, 2, true><<<grid, 32 * FEW_WARPS, 0, ctx->stream>>>(a);  // (on other boundaries: below)
    else if (vec) product_few_kernel<INT4, 1, true><<<grid, 32 * FEW_WARPS, 0, ctx->stream>>>(a);
    else product_few_kernel<INT4, 1, false><<<grid, 32 * FEW_WARPS, 0, ctx->stream>>>(a);
    return cudaGetLastError();
}

// ---- up to sixteen rows ----------------------------------------------------------------------------------------------------------------
// Codes from memory into the registers that multiply them: m16n8k32 with 16 outputs of the weights as its long side and eight rows of x as the short one. Which code is which k of a product
// is free as long as both sides agree, so a lane takes the 16 bytes that it loads side by side; low and high halves of 4-bit codes' bytes are 16 times the even and the odd codes. A warp has 32
// outputs and every so manieth run of codes; a thread block's warps add up through shared memory. Nothing waits for anything but its own loads, two or three runs of which are under way.
// Sixteen rows of 14336 x 4096 4-bit codes in groups of 128 (64, 32): 12.9 us (14.4, 19.2), of 4096 x 4096 8-bit ones, eight rows, 6.6 (more weights go to the tiles: 17.6 and 15.5): what bounds it is the first cache, whose lines the eight rows of a load take one
// after the other, x's among them in every thread block (with 8 bytes of 4-bit weights a lane 17.6), and registers: more runs under way go to memory.
__device__ __forceinline__ void mma_s8(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
constexpr int SOME_OUTPUTS = 32;  // of a warp

// T: eights of rows. GROUP: of 4-bit codes; 0: 8-bit ones. The groups of a run are products of their own. Of 64 codes: lanes exchange halves of their codes, so that each has a quarter
// of either group. Of 32: each lane's codes are one group's, and the others' are zeros in its product.
template <int GROUP, int T, bool VEC>
__global__ void __launch_bounds__(512, 1) product_some_kernel(const __grid_constant__ zkb_step_product_args a) {
    extern __shared__ uint32_t some_sm[];  // [warp][row][output]
    constexpr bool INT4 = GROUP > 0, LONG = GROUP >= 64;
    constexpr int RUN = LONG ? 128 : 64, W = INT4 ? RUN / 32 : 4, XS = RUN / 64, PARTS = !INT4 || GROUP == 128 ? 1 : 2;  // codes of a run, of which a lane has W words of weights and XS sixteens of x
    constexpr int D = LONG ? 2 : 3;  // runs on their way
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5, g = lane >> 2, q = lane & 3;
    const uint32_t c0 = blockIdx.x * SOME_OUTPUTS, n_in = a.n_in, whole = n_in / RUN;
    const int64_t w_row = INT4 ? a.w_stride / 2 : a.w_stride;
    const int8_t* w[2][2];
    const int8_t* x[T];
#pragma unroll
    for (int m = 0; m < 2; m++)
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const int64_t c = min(c0 + m * 16 + h * 8 + g, a.n_out - 1);
            w[m][h] = static_cast<const int8_t*>(a.w) + c * w_row + q * (4 * W);
        }
    constexpr int X_NEXT = GROUP == 128 ? 16 : 64;  // from a lane's first sixteen of x to its second
    const int x_first = GROUP == 128 ? q * 32 : GROUP == 64 ? (q & 1) * 32 + (q >> 1) * 16 : q * 16;
#pragma unroll
    for (int n = 0; n < T; n++) x[n] = a.x + (int64_t)min((uint32_t)(n * 8 + g), a.n_rows - 1) * a.x_stride + x_first;
    struct Run {
        uint32_t w[2][2][W], x[T][4 * XS], s;
    };
    // A lane has the scales of a run of one output, and asks the others for those that it needs.
    const uint16_t* const s = static_cast<const uint16_t*>(a.w_scale) + (INT4 ? (int64_t)min(c0 + lane, a.n_out - 1) * a.w_scale_stride : 0);
    const bool pairs = PARTS == 2 && (reinterpret_cast<uintptr_t>(a.w_scale) & 3) == 0 && (a.n_out == 1 || a.w_scale_stride % 2 == 0);
    auto scales = [&](uint32_t run) {
        if (PARTS == 1) return (uint32_t)s[run];
        if (pairs && run * RUN + RUN <= n_in) return *reinterpret_cast<const uint32_t*>(s + run * 2);
        return (uint32_t)s[run * 2] | (run * RUN + RUN / 2 < n_in ? (uint32_t)s[run * 2 + 1] << 16 : 0u);
    };
    auto put4 = [](uint32_t* to, const uint4& v) { to[0] = v.x, to[1] = v.y, to[2] = v.z, to[3] = v.w; };
    auto put_w = [&](uint32_t (&to)[W], const uint4& v) {
        to[0] = v.x, to[1] = v.y;
        if constexpr (W == 4) to[2] = v.z, to[3] = v.w;
    };
    auto load = [&](uint32_t run, Run& r) {
#pragma unroll
        for (int m = 0; m < 2; m++)
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const int8_t* const p = w[m][h] + run * (16 * W);
                if constexpr (!VEC) {
                    const int8_t *const lo = static_cast<const int8_t*>(a.w), *const hi = lo + (a.n_out - 1) * w_row + (INT4 ? (n_in + 1) / 2 : n_in);
                    put_w(r.w[m][h], fetched16(fetch16(p, lo, hi), p, lo, hi));
                } else if constexpr (W == 4) {
                    put_w(r.w[m][h], __ldg(reinterpret_cast<const uint4*>(p)));
                } else {
                    const uint2 v = __ldg(reinterpret_cast<const uint2*>(p));
                    r.w[m][h][0] = v.x, r.w[m][h][1] = v.y;
                }
            }
#pragma unroll
        for (int n = 0; n < T; n++)
#pragma unroll
            for (int k = 0; k < XS; k++) {
                const int8_t *const p = x[n] + run * RUN + k * X_NEXT, *const hi = a.x + (int64_t)(a.n_rows - 1) * a.x_stride + n_in;
                put4(&r.x[n][4 * k], VEC ? __ldg(reinterpret_cast<const uint4*>(p)) : fetched16(fetch16(p, a.x, hi), p, a.x, hi));
            }
        if constexpr (INT4) r.s = scales(run);
    };
    float acc[2][T][4] = {};
    int sum[2][T][4] = {};
    auto multiply = [&](Run& r) {
        uint32_t by[2][2];
        if constexpr (INT4) {
#pragma unroll
            for (int m = 0; m < 2; m++)
#pragma unroll
                for (int h = 0; h < 2; h++) by[m][h] = __shfl_sync(0xffffffffu, r.s, m * 16 + h * 8 + g);
        }
        if constexpr (GROUP == 64) {  // lanes 0 and 1 have the first group's codes, 2 and 3 the second's
#pragma unroll
            for (int m = 0; m < 2; m++)
#pragma unroll
                for (int h = 0; h < 2; h++)
#pragma unroll
                    for (int y = 0; y < 2; y++) {
                        uint32_t &lo = r.w[m][h][y], &hi = r.w[m][h][2 + y];
                        const uint32_t got = __shfl_xor_sync(0xffffffffu, q < 2 ? hi : lo, 2);
                        if (q < 2) hi = got;
                        else lo = got;
                    }
        }
#pragma unroll
        for (int n = 0; n < T; n++) {
            uint32_t b[4 * XS];
#pragma unroll
            for (int i = 0; i < 4 * XS; i += 2) {
                b[i] = INT4 ? __byte_perm(r.x[n][i], r.x[n][i + 1], 0x6420) : r.x[n][i];
                b[i + 1] = INT4 ? __byte_perm(r.x[n][i], r.x[n][i + 1], 0x7531) : r.x[n][i + 1];
            }
#pragma unroll
            for (int m = 0; m < 2; m++) {
                if constexpr (INT4) {
#pragma unroll
                    for (int p = 0; p < PARTS; p++) {
                        const uint32_t mine = GROUP != 32 || q / 2 == p ? 0xffffffffu : 0u;
                        constexpr int WORDS = GROUP == 64 ? 2 : W;  // of a part
                        int c[4] = {};
#pragma unroll
                        for (int y = 0; y < WORDS; y++) {
                            const int i = (GROUP == 64 ? 2 * p : 0) + y;
                            mma_s8(c, r.w[m][0][i] << 4 & 0xf0f0f0f0u, r.w[m][1][i] << 4 & 0xf0f0f0f0u, r.w[m][0][i] & 0xf0f0f0f0u, r.w[m][1][i] & 0xf0f0f0f0u, b[2 * i] & mine, b[2 * i + 1] & mine);
                        }
                        const float lo = (p ? bf16_high(by[m][0]) : bf16_low(by[m][0])) * 0.0625f, hi = (p ? bf16_high(by[m][1]) : bf16_low(by[m][1])) * 0.0625f;
#pragma unroll
                        for (int i = 0; i < 4; i++) acc[m][n][i] = fmaf((float)c[i], i < 2 ? lo : hi, acc[m][n][i]);
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < W; i += 2) mma_s8(sum[m][n], r.w[m][0][i], r.w[m][1][i], r.w[m][0][i + 1], r.w[m][1][i + 1], b[i], b[i + 1]);
                }
            }
        }
    };
    Run r[D];
#pragma unroll
    for (int k = 0; k < D; k++)
        if (warp + k * warps < whole) load(warp + k * warps, r[k]);
#pragma unroll 1
    for (uint32_t run = warp; run < whole; run += D * warps)
#pragma unroll
        for (int k = 0; k < D; k++)
            if (run + k * warps < whole) {
                multiply(r[k]);
                if (run + (k + D) * warps < whole) load(run + (k + D) * warps, r[k]);
            }
    if (whole * RUN < n_in && warp == whole % warps) {  // the last codes: what lies behind them counts for nothing
        const int left = (int)(n_in - whole * RUN);
#pragma unroll
        for (int m = 0; m < 2; m++)
#pragma unroll
            for (int h = 0; h < 2; h++) put_w(r[0].w[m][h], some_bytes(w[m][h] + whole * (16 * W), (INT4 ? (left + 1) / 2 : left) - q * (4 * W)));
#pragma unroll
        for (int n = 0; n < T; n++)
#pragma unroll
            for (int k = 0; k < XS; k++) put4(&r[0].x[n][4 * k], some_bytes(x[n] + whole * RUN + k * X_NEXT, left - x_first - k * X_NEXT));
        if constexpr (INT4) r[0].s = scales(whole);
        multiply(r[0]);
    }
#pragma unroll
    for (int n = 0; n < T; n++)
#pragma unroll
        for (int m = 0; m < 2; m++)
#pragma unroll
            for (int i = 0; i < 4; i++)
                some_sm[(warp * (8 * T) + n * 8 + 2 * q + (i & 1)) * SOME_OUTPUTS + m * 16 + (i >> 1) * 8 + g] = INT4 ? __float_as_uint(acc[m][n][i]) : (uint32_t)sum[m][n][i];
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < 8 * T * SOME_OUTPUTS; i += blockDim.x) {
        const uint32_t t = i / SOME_OUTPUTS, c = c0 + i % SOME_OUTPUTS;
        if (t >= a.n_rows || c >= a.n_out) continue;
        uint32_t y = some_sm[i];
        for (int w = 1; w < warps; w++) {
            const uint32_t more = some_sm[w * (8 * T * SOME_OUTPUTS) + i];
            y = INT4 ? __float_as_uint(__uint_as_float(y) + __uint_as_float(more)) : y + more;
        }
        const int64_t at = (int64_t)t * a.out_stride + c;
        if (a.out_type == ZKB_VALUE_INT32) static_cast<uint32_t*>(a.out)[at] = y;
        else store_value(a.out, at, a.out_type, INT4 ? __uint_as_float(y) * a.x_scale[t] : (float)(int)y * (a.x_scale[t] * static_cast<const float*>(a.w_scale)[c]));
    }
}

template <int GROUP, int T>
static cudaError_t launch_some(zkb_ctx* ctx, const zkb_step_product_args& a, bool vec) {
    // Eight warps let two thread blocks share an SM; where there is one for each, it has sixteen. Eight rows of 4096 x 4096 codes: 8.7 us by 8 and 6.7 by 16; of 4096 x 6144 9.7 and 10.7.
    const uint32_t grid = (a.n_out + SOME_OUTPUTS - 1) / SOME_OUTPUTS, warps = grid <= 148 ? 16 : 8;
    const size_t room = (size_t)warps * 8 * T * SOME_OUTPUTS * 4;
    if (vec) product_some_kernel<GROUP, T, true><<<grid, 32 * warps, room, ctx->stream>>>(a);
    else product_some_kernel<GROUP, T, false><<<grid, 32 * warps, room, ctx->stream>>>(a);
    return cudaGetLastError();
}
template <int GROUP>
static cudaError_t launch_some(zkb_ctx* ctx, const zkb_step_product_args& a, bool vec) {
    return a.n_rows <= 8 ? launch_some<GROUP, 1>(ctx, a, vec) : launch_some<GROUP, 2>(ctx, a, vec);
}

}  // namespace zk

using namespace zk;

extern "C" int zkb_step_product(zkb_ctx* ctx, const zkb_step_product_args* args) {
    if (!ctx) return ZKB_EINVAL;
    ZKB_CHECK_ARG(ctx, args);
    const zkb_step_product_args& a = *args;
    const bool int4 = a.w_type == ZKB_VALUE_INT4;
    ZKB_CHECK_ARG(ctx, a.w_type == ZKB_VALUE_INT8 || a.w_type == ZKB_VALUE_INT4);
    ZKB_CHECK_ARG(ctx, a.out_type == ZKB_VALUE_BF16 || a.out_type == ZKB_VALUE_WORD || a.out_type == ZKB_VALUE_F32 || (a.out_type == ZKB_VALUE_INT32 && !int4));
    ZKB_CHECK_ARG(ctx, int4 ? a.group == 32 || a.group == 64 || a.group == 128 : a.group == 0);
    ZKB_CHECK_ARG(ctx, a.n_in >= 1 && a.n_in <= 131071 && a.n_out >= 1 && a.n_out <= (1u << 24) && a.n_rows <= (1u << 18));
    if (a.n_rows == 0) return ZKB_OK;
    ZKB_CHECK_ARG(ctx, a.x && a.w && a.out && (a.out_type == ZKB_VALUE_INT32 ? !a.x_scale && !a.w_scale : a.x_scale && a.w_scale));
    ZKB_CHECK_ARG(ctx, aligned_to(a.out, a.out_type == ZKB_VALUE_BF16 ? 2 : 4) && aligned_to(a.x_scale, 4) && aligned_to(a.w_scale, int4 ? 2 : 4));
    ZKB_CHECK_ARG(ctx, (a.n_out == 1 || a.w_stride >= (int64_t)a.n_in) && (!int4 || a.w_stride % 2 == 0));
    ZKB_CHECK_ARG(ctx, !int4 || a.n_out == 1 || a.w_scale_stride >= (int64_t)((a.n_in + a.group - 1) / a.group));
    ZKB_CHECK_ARG(ctx, a.n_rows == 1 || (a.x_stride >= (int64_t)a.n_in && a.out_stride >= (int64_t)a.n_out));
    DeviceGuard g(ctx);
    ProfScope prof(ctx, "step_product_kernel");
    const int64_t w_row = int4 ? a.w_stride / 2 : a.w_stride;
    const bool vec = aligned_to(a.x, 16) && aligned_to(a.w, 16) && (a.n_rows == 1 || a.x_stride % 16 == 0) && (a.n_out == 1 || w_row % 16 == 0);
    // By what each was measured to take, in us, calls of a graph on inputs in turn that the L2 does not hold (4-bit codes in groups of 128, of 64, of 32; 8-bit ones):
    //                                   dp4a                     a warp's products          tiles
    //   1 row of 4096 x 4096            3.5  3.9  4.0  5.0       4.6  5.7  6.9  6.5
    //   1 row of 14336 x 4096           7.3  7.5  7.6  11.0      10.7 11.2 16.8 16.3
    //   2 rows of 4096 x 4096           5.0  5.0  5.0  6.3       5.0  5.7  6.9  6.5
    //   2 rows of 14336 x 4096          10.4 10.6 10.7 14.2      10.6 11.3 16.9 16.3
    //   1 of 1637 x 9144, odd rows      11.8 11.8 11.9 11.1      9.3  9.8  12.9 13.4
    //   1 of 10344 x 6512, odd rows     19.3 19.7 20.0 25.0      38.4 41.4 68.4 61.5
    //   8 rows of 4096 x 4096                                    5.1  5.7  7.0  6.6         12.1 13.6 17.0 8.6
    //   16 rows of 14336 x 4096                                  12.9 14.4 19.2 17.6        19.7 24.4 35.1 15.5
    //   16 rows of 4096 x 14336                                  15.0 17.5 22.3 19.1        18.7 24.7 36.6 14.9
    //   16 rows of 4096 x 32000                                  28.2 32.3 42.4 36.2        31.5 43.3 67.1 24.5
    // (One short row on odd boundaries with long groups would take a fifth less the other way, a long one twice as much. Two rows on odd boundaries have no dp4a: it took twice as long at 1637 x 9144.)
    const uint64_t bytes = (uint64_t)a.n_out * a.n_in;
    const bool some = a.n_rows > 2 ? a.n_rows <= 16 && (int4 || bytes <= (32u << 20)) : a.n_rows == 2 && !vec;
    if (some) {
        ZKB_CUDA(ctx, (!int4 ? launch_some<0>(ctx, a, vec) : a.group == 32 ? launch_some<32>(ctx, a, vec) : a.group == 64 ? launch_some<64>(ctx, a, vec) : launch_some<128>(ctx, a, vec)));
        return ZKB_OK;
    }
    if (a.n_rows > 2) {
        ZKB_CUDA(ctx, int4 ? launch_tiles<true>(ctx, a) : launch_tiles<false>(ctx, a));
        return ZKB_OK;
    }
    ZKB_CUDA(ctx, int4 ? launch_few<true>(ctx, a, vec) : launch_few<false>(ctx, a, vec));
    return ZKB_OK;
}
