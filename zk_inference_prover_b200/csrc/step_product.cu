// Products of 8-bit codes with weights held as 8-bit or 4-bit codes.
#include <algorithm>
#include <cmath>
#include <cstdlib>

#include "step_product.cuh"

namespace zk {

// ---- few rows ------------------------------------------------------------------------------------------------------------------------
// The weights are read once and everything else is small, so this is bound by the weights' bytes. A warp has CHANNELS outputs and R rows; its lanes take turns in the
// weights, 16 bytes each, and multiply four codes an instruction (dp4a). Of 4-bit codes the two halves of the bytes are taken apart in place, as 16 times the code, against
// the even and the odd codes of x; 16 bytes are 32 codes of one group, whose sum is exact and then scaled.
constexpr int CHANNELS = 4;

template <bool INT4, int R, bool VEC>
__global__ void __launch_bounds__(128) product_few_kernel(const __grid_constant__ zkb_step_product_args a) {
    const int lane = threadIdx.x & 31;
    const uint32_t c0 = (blockIdx.x * 4u + (threadIdx.x >> 5)) * CHANNELS, t0 = blockIdx.y * R;
    if (c0 >= a.n_out) return;
    const int codes = INT4 ? 32 : 16;  // of 16 bytes
    const int bytes = INT4 ? (int)(a.n_in + 1) / 2 : (int)a.n_in;
    const int64_t w_row = INT4 ? a.w_stride / 2 : a.w_stride;
    const int8_t* w[CHANNELS];
    const uint16_t* s[CHANNELS];
    const int8_t* x[R];
#pragma unroll
    for (int c = 0; c < CHANNELS; c++) {
        const int64_t at = min(c0 + c, a.n_out - 1);
        w[c] = static_cast<const int8_t*>(a.w) + at * w_row;
        s[c] = static_cast<const uint16_t*>(a.w_scale) + (INT4 ? at * a.w_scale_stride : 0);
    }
#pragma unroll
    for (int r = 0; r < R; r++) x[r] = a.x + (int64_t)min(t0 + r, a.n_rows - 1) * a.x_stride;
    int sum[CHANNELS][R] = {};
    float part[CHANNELS][R] = {};
#pragma unroll(INT4 ? 2 : 4)
    for (int b = lane * 16; b < bytes; b += 512) {
        const bool inner = b >= 4 && b + 20 <= bytes;
        uint4 v[CHANNELS];
#pragma unroll
        for (int c = 0; c < CHANNELS; c++) v[c] = load16<VEC>(w[c] + b, bytes - b, inner);
        const int at = b / 16 * codes, left = (int)a.n_in - at;
        if constexpr (INT4) {
            float by[CHANNELS];
#pragma unroll
            for (int c = 0; c < CHANNELS; c++) by[c] = bf16_low(s[c][(uint32_t)at / a.group]) * 0.0625f;
#pragma unroll
            for (int r = 0; r < R; r++) {
                const bool x_inner = at >= 4 && left >= 36;
                const uint4 lo = load16<VEC>(x[r] + at, left, x_inner), hi = load16<VEC>(x[r] + at + 16, left - 16, x_inner);
                const uint32_t xs[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
#pragma unroll
                for (int c = 0; c < CHANNELS; c++) {
                    const uint32_t ws[4] = {v[c].x, v[c].y, v[c].z, v[c].w};
                    int d = 0;
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        d = __dp4a((int)(ws[i] << 4 & 0xf0f0f0f0u), (int)__byte_perm(xs[2 * i], xs[2 * i + 1], 0x6420), d);
                        d = __dp4a((int)(ws[i] & 0xf0f0f0f0u), (int)__byte_perm(xs[2 * i], xs[2 * i + 1], 0x7531), d);
                    }
                    part[c][r] = fmaf((float)d, by[c], part[c][r]);
                }
            }
        } else {
#pragma unroll
            for (int r = 0; r < R; r++) {
                const uint4 u = load16<VEC>(x[r] + at, left, inner);
#pragma unroll
                for (int c = 0; c < CHANNELS; c++) {
                    sum[c][r] = __dp4a((int)v[c].x, (int)u.x, sum[c][r]), sum[c][r] = __dp4a((int)v[c].y, (int)u.y, sum[c][r]);
                    sum[c][r] = __dp4a((int)v[c].z, (int)u.z, sum[c][r]), sum[c][r] = __dp4a((int)v[c].w, (int)u.w, sum[c][r]);
                }
            }
        }
    }
#pragma unroll
    for (int r = 0; r < R; r++) {
        uint32_t mine = 0;  // lane c keeps output c
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
            if (lane == c) mine = y;
        }
        if (lane < CHANNELS && c0 + lane < a.n_out && t0 + r < a.n_rows) {
            const int64_t at = (int64_t)(t0 + r) * a.out_stride + c0 + lane;
            if (a.out_type == ZKB_VALUE_INT32) static_cast<uint32_t*>(a.out)[at] = mine;
            else store_value(a.out, at, a.out_type, INT4 ? __uint_as_float(mine) * a.x_scale[t0 + r] : (float)(int)mine * (a.x_scale[t0 + r] * static_cast<const float*>(a.w_scale)[c0 + lane]));
        }
    }
}

template <bool INT4, bool VEC>
static cudaError_t launch_few(zkb_ctx* ctx, const zkb_step_product_args& a) {
    const uint32_t grid = (a.n_out + 4 * CHANNELS - 1) / (4 * CHANNELS);
    auto launch = [&](auto kernel, uint32_t r) { kernel<<<dim3(grid, (a.n_rows + r - 1) / r), 128, 0, ctx->stream>>>(a); };
    if (a.n_rows == 1) launch(product_few_kernel<INT4, 1, VEC>, 1);
    else if (a.n_rows == 2) launch(product_few_kernel<INT4, 2, VEC>, 2);
    else if (a.n_rows <= 4) launch(product_few_kernel<INT4, 4, VEC>, 4);
    else launch(product_few_kernel<INT4, 8, VEC>, 8);
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
    if (a.n_rows > 8) {
        ZKB_CUDA(ctx, int4 ? launch_tiles<true>(ctx, a) : launch_tiles<false>(ctx, a));
        return ZKB_OK;
    }
    ZKB_CUDA(ctx, int4 ? (vec ? launch_few<true, true>(ctx, a) : launch_few<true, false>(ctx, a)) : (vec ? launch_few<false, true>(ctx, a) : launch_few<false, false>(ctx, a)));
    return ZKB_OK;
}
