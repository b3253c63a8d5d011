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

// VEC: all rows of x and of the weights start on 16-byte boundaries.
template <bool INT4, int R, bool VEC>
__global__ void __launch_bounds__(128) product_few_kernel(const __grid_constant__ zkb_step_product_args a) {
    const int lane = threadIdx.x & 31;
    const uint32_t c0 = (blockIdx.x * 4u + (threadIdx.x >> 5)) * CHANNELS, t0 = blockIdx.y * R;
    if (c0 >= a.n_out) return;
    constexpr int CODES = INT4 ? 32 : 16, XS = CODES / 16, AHEAD = R == 1 ? (INT4 ? 2 : 4) : R == 2 ? 2 : 1;  // codes of 16 bytes; 16s of x to them; rounds whose weights are on their way at a time
    const int bytes = INT4 ? (int)(a.n_in + 1) / 2 : (int)a.n_in;
    const int64_t w_row = INT4 ? a.w_stride / 2 : a.w_stride;
    const int8_t *const w_lo = static_cast<const int8_t*>(a.w), *const w_hi = w_lo + (a.n_out - 1) * w_row + bytes, *const x_hi = a.x + (int64_t)(a.n_rows - 1) * a.x_stride + a.n_in;
    const int8_t* w[CHANNELS];
    const uint16_t* s[CHANNELS];
    const int8_t* x[R];
#pragma unroll
    for (int c = 0; c < CHANNELS; c++) {
        const int64_t at = min(c0 + c, a.n_out - 1);
        w[c] = w_lo + at * w_row;
        s[c] = static_cast<const uint16_t*>(a.w_scale) + (INT4 ? at * a.w_scale_stride : 0);
    }
#pragma unroll
    for (int r = 0; r < R; r++) x[r] = a.x + (int64_t)min(t0 + r, a.n_rows - 1) * a.x_stride;
    const uint32_t log_group = INT4 ? 31 - __clz(a.group) : 0;
    int sum[CHANNELS][R] = {};
    float part[CHANNELS][R] = {};
#pragma unroll 1
    for (int b0 = lane * 16; b0 < bytes; b0 += 512 * AHEAD) {
        Fetched<VEC> v[AHEAD][CHANNELS];
        uint32_t by[AHEAD][CHANNELS];
#pragma unroll
        for (int h = 0; h < AHEAD; h++) {
            const int b = b0 + h * 512;
#pragma unroll
            for (int c = 0; c < CHANNELS; c++) {
                if (b < bytes) v[h][c] = fetch16<VEC>(w[c] + b, w_lo, w_hi);
                if (INT4 && b < bytes) by[h][c] = s[c][(uint32_t)(b * 2) >> log_group];
            }
        }
#pragma unroll
        for (int h = 0; h < AHEAD; h++) {
            const int b = b0 + h * 512, at = b / 16 * CODES, left = (int)a.n_in - at;
            if (b >= bytes) break;
            uint32_t ws[CHANNELS][4];
#pragma unroll
            for (int c = 0; c < CHANNELS; c++) {
                const uint4 u = fetched16<VEC>(v[h][c], w[c] + b, w_lo, w_hi);
                ws[c][0] = u.x, ws[c][1] = u.y, ws[c][2] = u.z, ws[c][3] = u.w;
            }
#pragma unroll
            for (int r = 0; r < R; r++) {
                uint32_t xs[4 * XS];
#pragma unroll
                for (int i = 0; i < XS; i++) {
                    uint4 u = make_uint4(0u, 0u, 0u, 0u);
                    const int8_t* const from = x[r] + at + 16 * i;
                    if (left > 16 * i) u = first_bytes(fetched16<VEC>(fetch16<VEC>(from, a.x, x_hi), from, a.x, x_hi), left - 16 * i);  // what lies behind a row's codes, of x's or of the weights', counts for nothing
                    xs[4 * i] = u.x, xs[4 * i + 1] = u.y, xs[4 * i + 2] = u.z, xs[4 * i + 3] = u.w;
                }
                if constexpr (INT4) {
                    uint32_t even[4], odd[4];
#pragma unroll
                    for (int i = 0; i < 4; i++) even[i] = __byte_perm(xs[2 * i], xs[2 * i + 1], 0x6420), odd[i] = __byte_perm(xs[2 * i], xs[2 * i + 1], 0x7531);
#pragma unroll
                    for (int c = 0; c < CHANNELS; c++) {
                        int d = 0;
#pragma unroll
                        for (int i = 0; i < 4; i++) d = __dp4a((int)(ws[c][i] << 4 & 0xf0f0f0f0u), (int)even[i], d), d = __dp4a((int)(ws[c][i] & 0xf0f0f0f0u), (int)odd[i], d);
                        part[c][r] = fmaf((float)d, __uint_as_float(by[h][c] << 16) * 0.0625f, part[c][r]);
                    }
                } else {
#pragma unroll
                    for (int c = 0; c < CHANNELS; c++)
#pragma unroll
                        for (int i = 0; i < 4; i++) sum[c][r] = __dp4a((int)ws[c][i], (int)xs[i], sum[c][r]);
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
