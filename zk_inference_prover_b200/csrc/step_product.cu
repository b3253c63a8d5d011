// Products of 8-bit codes with weights held as 8-bit or 4-bit codes.
#include <algorithm>
#include <cmath>
#include <cstdlib>

#include "step_product.cuh"

namespace zk {

// ---- few rows ------------------------------------------------------------------------------------------------------------------------
// The weights are read once and everything else is small, so this is bound by the weights' bytes. A thread block has CHANNELS outputs of R rows; its warps' lanes take turns in
// the weights, 16 bytes each, and multiply four codes an instruction (dp4a). Of 4-bit codes the two halves of the bytes are taken apart in place, as 16 times the code, against
// the even and the odd codes of x; 16 bytes are 32 codes of one group, whose sum is exact and then scaled.
constexpr int CHANNELS = 4, FEW_WARPS = 4;

// VEC: all rows of x and of the weights start on 16-byte boundaries.
template <bool INT4, int R, bool VEC>
__global__ void __launch_bounds__(32 * FEW_WARPS, R == 1 ? 8 : R == 2 ? 6 : 4) product_few_kernel(const __grid_constant__ zkb_step_product_args a) {
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
        if constexpr (INT4)
#pragma unroll
            for (int c = 0; c < CHANNELS; c++)
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
    else if (a.n_rows == 2) launch(product_few_kernel<INT4, 2, VEC>, 2);
    else launch(product_few_kernel<INT4, 4, VEC>, 4);
    return cudaGetLastError();
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
    if (getenv("FEW") ? (int)a.n_rows > atoi(getenv("FEW")) : a.n_rows > 4) {
        ZKB_CUDA(ctx, int4 ? launch_tiles<true>(ctx, a) : launch_tiles<false>(ctx, a));
        return ZKB_OK;
    }
    ZKB_CUDA(ctx, int4 ? (vec ? launch_few<true, true>(ctx, a) : launch_few<true, false>(ctx, a)) : (vec ? launch_few<false, true>(ctx, a) : launch_few<false, false>(ctx, a)));
    return ZKB_OK;
}
