// Products of 8-bit codes with weights held as 8-bit or 4-bit codes.
#include <algorithm>
#include <cmath>
#include <cstdlib>

#include "step_product.cuh"

namespace zk {

// ---- few rows ------------------------------------------------------------------------------------------------------------------------
// The weights are read once and everything else is small, so this is bound by the weights' bytes. A thread block has CHANNELS outputs of R rows; its warps' lanes take turns in
// the weights, 16 bytes each, and multiply four codes an instruction (dp4a). Of 4-bit codes the two halves of the bytes are taken apart in place, as 16 times the code, against
// the even and the odd codes of x; 16 bytes are 32 codes of one group, whose sum is exact and then scaled. One row of 4096 x 32000 8-bit codes: 23.3 us, 5.6 TB/s, its loads' latency
// between a thread block's start and its end is what is left; of 4096 x 4096 4-bit codes 4.4 us, where a launch and three trips to memory are most of it.
constexpr int CHANNELS = 4, FEW_WARPS = 4;

// VEC: all rows of x and of the weights start on 16-byte boundaries.
template <bool INT4, int R, bool VEC>
__global__ void __launch_bounds__(32 * FEW_WARPS, R == 1 ? 8 : 6) product_few_kernel(const __grid_constant__ zkb_step_product_args a) {
    __shared__ uint32_t joined[FEW_WARPS][R][CHANNELS];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint32_t c0 = blockIdx.x * CHANNELS, t0 = blockIdx.y * R;
    constexpr int CODES = INT4 ? 32 : 16, XS = CODES / 16;  // codes of 16 bytes; 16s of x to them
    const int n_in = (int)a.n_in, bytes = INT4 ? (n_in + 1) / 2 : n_in;
    const int64_t w_row = INT4 ? a.w_stride / 2 : a.w_stride;
    const int8_t *const w_lo = static_cast<const int8_t*>(a.w), *const w_hi = w_lo + (a.n_out - 1) * w_row + bytes, *const x_hi = a.x + (int64_t)(a.n_rows - 1) * a.x_stride + n_in;
    auto w_of = [&](int c) { return w_lo + (int64_t)min(c0 + c, a.n_out - 1) * w_row; };
    auto x_of = [&](int r) { return a.x + (int64_t)min(t0 + r, a.n_rows - 1) * a.x_stride; };
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
    if (r < R && c0 + c < a.n_out && t0 + r < a.n_rows) {
        uint32_t y = joined[0][r][c];
#pragma unroll
        for (int w = 1; w < FEW_WARPS; w++) y = INT4 ? __float_as_uint(__uint_as_float(y) + __uint_as_float(joined[w][r][c])) : y + joined[w][r][c];
        const int64_t at = (int64_t)(t0 + r) * a.out_stride + c0 + c;
        if (a.out_type == ZKB_VALUE_INT32) static_cast<uint32_t*>(a.out)[at] = y;
        else store_value(a.out, at, a.out_type, INT4 ? __uint_as_float(y) * a.x_scale[t0 + r] : (float)(int)y * (a.x_scale[t0 + r] * static_cast<const float*>(a.w_scale)[c0 + c]));
    }
}

template <bool INT4, bool VEC>
static cudaError_t launch_few(zkb_ctx* ctx, const zkb_step_product_args& a) {
    const uint32_t grid = (a.n_out + CHANNELS - 1) / CHANNELS;
    auto launch = [&](auto kernel, uint32_t r) { kernel<<<dim3(grid, (a.n_rows + r - 1) / r), 32 * FEW_WARPS, 0, ctx->stream>>>(a); };
    if (a.n_rows == 1) launch(product_few_kernel<INT4, 1, VEC>, 1);
    else launch(product_few_kernel<INT4, 2, VEC>, 2);
    return cudaGetLastError();
}

// ---- up to sixteen rows ----------------------------------------------------------------------------------------------------------------
// Codes from memory into the registers that multiply them: m16n8k32 with 16 outputs of the weights as its long side and eight rows of x as the short one. Which code is which k of a product
// is free as long as both sides agree, so a lane takes the codes that it loads side by side: of 8-bit weights 16 of an output's 64, of 4-bit ones a quarter of a group, whose low and high
// halves of bytes are 16 times the even and the odd codes. A warp has 32 outputs and every so manieth run of codes; a thread block's warps add up through shared memory. Nothing waits
// for anything but its own loads, three runs of which are under way. Sixteen rows of 14336 x 4096 4-bit (8-bit) codes: 17.5 (16.1) us, 1.8 (3.7) TB/s: loads of 8 bytes, x's among them, by a lane
// take turns in the first cache (62 % of its rate). Sixteen-byte loads of 4-bit weights leave no registers for the runs under way: 21 to 23 us.
__device__ __forceinline__ void mma_s8(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
constexpr int SOME_OUTPUTS = 32;  // of a warp

// T: eights of rows. PARTS: groups in a run of 4-bit codes: each is a product of its own, with zeros for the codes of the lanes that have the others.
template <bool INT4, int T, int PARTS, bool VEC>
__global__ void __launch_bounds__(512, 1) product_some_kernel(const __grid_constant__ zkb_step_product_args a) {
    extern __shared__ uint32_t some_sm[];  // [warp][row][output]
    constexpr int RUN = 64, W = INT4 ? 2 : 4, D = 3;  // codes of a run, of which a lane has W words of weights and four of x; runs on their way
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5, g = lane >> 2, q = lane & 3;
    const uint32_t c0 = blockIdx.x * SOME_OUTPUTS, n_in = a.n_in, whole = n_in / RUN;
    const int64_t w_row = INT4 ? a.w_stride / 2 : a.w_stride;
    const int8_t* w[2][2];
    const int8_t* x[T];
    const uint16_t* s[2][2];
#pragma unroll
    for (int m = 0; m < 2; m++)
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const int64_t c = min(c0 + m * 16 + h * 8 + g, a.n_out - 1);
            w[m][h] = static_cast<const int8_t*>(a.w) + c * w_row + q * (4 * W);
            s[m][h] = static_cast<const uint16_t*>(a.w_scale) + (INT4 ? c * a.w_scale_stride : 0);
        }
#pragma unroll
    for (int n = 0; n < T; n++) x[n] = a.x + (int64_t)min((uint32_t)(n * 8 + g), a.n_rows - 1) * a.x_stride + q * 16;
    const uint32_t log_group = INT4 ? 31 - __clz(a.group) : 0;
    struct Run {
        uint32_t w[2][2][W], x[T][4], s[2][2];
    };
    auto scales = [&](uint32_t run, Run& r) {
        if constexpr (INT4) {
#pragma unroll
            for (int m = 0; m < 2; m++)
#pragma unroll
                for (int h = 0; h < 2; h++) {
#pragma unroll
                    for (int p = 0; p < PARTS; p++) {
                        const uint32_t v = run * RUN + p * (RUN / PARTS) < n_in ? s[m][h][(run * RUN >> log_group) + p] : 0u;
                        r.s[m][h] = p ? r.s[m][h] | v << 16 : v;
                    }
                }
        }
    };
    auto put4 = [](uint32_t (&to)[4], const uint4& v) { to[0] = v.x, to[1] = v.y, to[2] = v.z, to[3] = v.w; };
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
        for (int n = 0; n < T; n++) {
            const int8_t *const p = x[n] + run * RUN, *const hi = a.x + (int64_t)(a.n_rows - 1) * a.x_stride + n_in;
            put4(r.x[n], VEC ? __ldg(reinterpret_cast<const uint4*>(p)) : fetched16(fetch16(p, a.x, hi), p, a.x, hi));
        }
        scales(run, r);
    };
    float acc[2][T][4] = {};
    int sum[2][T][4] = {};
    auto multiply = [&](const Run& r) {
#pragma unroll
        for (int n = 0; n < T; n++) {
            uint32_t b[4];
#pragma unroll
            for (int i = 0; i < 4; i += 2) {
                b[i] = INT4 ? __byte_perm(r.x[n][i], r.x[n][i + 1], 0x6420) : r.x[n][i];
                b[i + 1] = INT4 ? __byte_perm(r.x[n][i], r.x[n][i + 1], 0x7531) : r.x[n][i + 1];
            }
#pragma unroll
            for (int m = 0; m < 2; m++) {
                if constexpr (INT4) {
#pragma unroll
                    for (int p = 0; p < PARTS; p++) {
                        const uint32_t mine = PARTS == 1 || q / (4 / PARTS) == p ? 0xffffffffu : 0u;
                        int c[4] = {};
#pragma unroll
                        for (int i = 0; i < W; i++)
                            mma_s8(c, r.w[m][0][i] << 4 & 0xf0f0f0f0u, r.w[m][1][i] << 4 & 0xf0f0f0f0u, r.w[m][0][i] & 0xf0f0f0f0u, r.w[m][1][i] & 0xf0f0f0f0u, b[2 * i] & mine, b[2 * i + 1] & mine);
                        const float lo = (p ? bf16_high(r.s[m][0]) : bf16_low(r.s[m][0])) * 0.0625f, hi = (p ? bf16_high(r.s[m][1]) : bf16_low(r.s[m][1])) * 0.0625f;
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
        for (int n = 0; n < T; n++) put4(r[0].x[n], some_bytes(x[n] + whole * RUN, left - q * 16));
        scales(whole, r[0]);
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

template <bool INT4, int T, int PARTS>
static cudaError_t launch_some(zkb_ctx* ctx, const zkb_step_product_args& a, bool vec) {
    // Eight warps let two thread blocks share an SM; where there is one for each, it has sixteen. Eight rows of 4096 x 4096 codes: 8.7 us by 8 and 6.7 by 16; of 4096 x 6144 9.7 and 10.7.
    const uint32_t grid = (a.n_out + SOME_OUTPUTS - 1) / SOME_OUTPUTS, warps = grid <= 148 ? 16 : 8;
    const size_t room = (size_t)warps * 8 * T * SOME_OUTPUTS * 4;
    if (vec) product_some_kernel<INT4, T, PARTS, true><<<grid, 32 * warps, room, ctx->stream>>>(a);
    else product_some_kernel<INT4, T, PARTS, false><<<grid, 32 * warps, room, ctx->stream>>>(a);
    return cudaGetLastError();
}
template <bool INT4, int PARTS>
static cudaError_t launch_some(zkb_ctx* ctx, const zkb_step_product_args& a, bool vec) {
    return a.n_rows <= 8 ? launch_some<INT4, 1, PARTS>(ctx, a, vec) : launch_some<INT4, 2, PARTS>(ctx, a, vec);
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
    // By what each was measured to take, in us: one row of 4096 x 4096 4-bit (8-bit) codes 4.4 (5.3) by dp4a and 6.4 (6.8) by a warp's products, two rows 6.2 (6.6) and 6.4 (6.9), four 6.9 (7.2) and
    // 6.5 (6.8). Eight of 4096 x 4096 5 to 7 by a warp's products and 11 (9) by tiles, sixteen of 14336 x 4096 17 (18) and 18 to 22 (16), of 4096 x 32000 35 (37) and 29 (25): tiles are
    // better at more than 32 MB of weights. Rows on odd boundaries: 7 of 1637 x 9144 13 (14) and 14 (15), 12 of 10344 x 6512 69 (70) and 37 (46).
    const uint64_t bytes = (uint64_t)a.n_out * (int4 ? a.n_in / 2 : a.n_in);
    if (a.n_rows > 2 && a.n_rows <= 16 && bytes <= (32u << 20)) {
        ZKB_CUDA(ctx, (!int4 ? launch_some<false, 1>(ctx, a, vec) : a.group > 32 ? launch_some<true, 1>(ctx, a, vec) : launch_some<true, 2>(ctx, a, vec)));
        return ZKB_OK;
    }
    if (a.n_rows > 2) {
        ZKB_CUDA(ctx, int4 ? launch_tiles<true>(ctx, a) : launch_tiles<false>(ctx, a));
        return ZKB_OK;
    }
    ZKB_CUDA(ctx, int4 ? (vec ? launch_few<true, true>(ctx, a) : launch_few<true, false>(ctx, a)) : (vec ? launch_few<false, true>(ctx, a) : launch_few<false, false>(ctx, a)));
    return ZKB_OK;
}
