// Rows of the residual stream: its next values with their norms, and the gate between a feed-forward layer's products, as values or as 8-bit codes.
#include <algorithm>
#include <cmath>
#include <cstdlib>

#include "step_values.cuh"

namespace zk {

// Both calls are a pass over rows: values in, one number of the whole row (the mean of squares, the largest value), values out. A row stays in registers between
// its reading and its writing, V times eight values a thread, so nothing is read twice: bound by the bytes, and by a row's one barrier, which two thread blocks an SM cover for one another.
// Measured: the norm of 8191 rows of 4096 with the residual's sum and codes 38 us, 6.15 TB/s; of one row 2.1 to 2.9, a launch and two trips to memory; the gate of 4096 rows of 14336 to codes 58 us,
// 5.0 TB/s (two sixteens of bytes of each input and thread are as much as its registers hold under way).
struct RowsArgs {
    const void* x;
    const void* other;  // the residual stream, or the gate
    const uint16_t* weight;
    void* sum;
    void* out;
    float* scale;
    int64_t x_stride, segment_stride, other_stride, sum_stride, out_stride;
    uint32_t n_rows, width, segment, out_type;
    bool other_word, sum_word;
    float eps;
    uint32_t warps;  // a row's
};

// This thread's values of a row, in pairs as bf16: VEC eight adjacent ones at a time, on 16-byte boundaries; else a value at a time, adjacent ones in adjacent lanes.
template <bool VEC>
__device__ __forceinline__ uint32_t column_of(uint32_t v, uint32_t y, uint32_t threads, uint32_t th) {
    return VEC ? (v * threads + th) * 8 + y : (v * 8 + y) * threads + th;
}
template <int V, bool VEC>
__device__ __forceinline__ void load_row(const void* p, int64_t row, uint32_t segment, int64_t segment_stride, bool word, uint32_t width, uint32_t threads, uint32_t th, uint32_t (&x)[V][4]) {
    auto place = [&](uint32_t col) { return row + (segment ? (int64_t)(col / segment) * segment_stride + col % segment : (int64_t)col); };
    if constexpr (VEC) {
        if (word) {
            uint4 a[V], b[V];
#pragma unroll
            for (int v = 0; v < V; v++) {
                const uint32_t col = column_of<VEC>(v, 0, threads, th);
                a[v] = b[v] = make_uint4(0u, 0u, 0u, 0u);
                if (col < width) {
                    const uint4* w = reinterpret_cast<const uint4*>(static_cast<const uint32_t*>(p) + place(col));
                    a[v] = w[0], b[v] = w[1];
                }
            }
#pragma unroll
            for (int v = 0; v < V; v++) {
                x[v][0] = __byte_perm(a[v].x, a[v].y, 0x5410), x[v][1] = __byte_perm(a[v].z, a[v].w, 0x5410);
                x[v][2] = __byte_perm(b[v].x, b[v].y, 0x5410), x[v][3] = __byte_perm(b[v].z, b[v].w, 0x5410);
            }
        } else {
#pragma unroll
            for (int v = 0; v < V; v++) {
                const uint32_t col = column_of<VEC>(v, 0, threads, th);
                uint4 a = make_uint4(0u, 0u, 0u, 0u);
                if (col < width) a = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p) + place(col));
                x[v][0] = a.x, x[v][1] = a.y, x[v][2] = a.z, x[v][3] = a.w;
            }
        }
    } else {
#pragma unroll
        for (int v = 0; v < V; v++) {
            uint32_t h[8];
#pragma unroll
            for (int y = 0; y < 8; y++) {
                const uint32_t col = column_of<VEC>(v, y, threads, th);
                h[y] = 0;
                if (col < width) h[y] = word ? static_cast<const uint32_t*>(p)[place(col)] : static_cast<const uint16_t*>(p)[place(col)];
            }
#pragma unroll
            for (int y = 0; y < 4; y++) x[v][y] = __byte_perm(h[2 * y], h[2 * y + 1], 0x5410);
        }
    }
}
template <int V, bool VEC>
__device__ __forceinline__ void store_row(void* p, int64_t row, bool word, uint32_t width, uint32_t threads, uint32_t th, const uint32_t (&x)[V][4]) {
#pragma unroll
    for (int v = 0; v < V; v++) {
        if constexpr (VEC) {
            const uint32_t col = column_of<VEC>(v, 0, threads, th);
            if (col >= width) continue;
            if (word) {
                uint4* const to = reinterpret_cast<uint4*>(static_cast<uint32_t*>(p) + row + col);
                to[0] = make_uint4(x[v][0] & 0xffffu, x[v][0] >> 16, x[v][1] & 0xffffu, x[v][1] >> 16);
                to[1] = make_uint4(x[v][2] & 0xffffu, x[v][2] >> 16, x[v][3] & 0xffffu, x[v][3] >> 16);
            } else {
                *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p) + row + col) = make_uint4(x[v][0], x[v][1], x[v][2], x[v][3]);
            }
        } else {
#pragma unroll
            for (int y = 0; y < 8; y++) {
                const uint32_t col = column_of<VEC>(v, y, threads, th), h = y % 2 ? x[v][y / 2] >> 16 : x[v][y / 2] & 0xffffu;
                if (col >= width) continue;
                if (word) static_cast<uint32_t*>(p)[row + col] = h;
                else static_cast<uint16_t*>(p)[row + col] = (uint16_t)h;
            }
        }
    }
}

// A sum and a largest word over a row's warps. `room`: the warps' own words, another one for each use within a row.
struct RowRoom {
    float sum[32];
    uint32_t most[32];
};
__device__ __forceinline__ void over_row(RowRoom& room, uint32_t warps, float& sum, float& largest) {
    uint32_t most = __float_as_uint(largest);  // sizes are ordered as their words, NaN above all
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    most = __reduce_max_sync(0xffffffffu, most);
    largest = __uint_as_float(most);
    if (warps == 1) return;
    if (lane == 0) room.sum[warp] = sum, room.most[warp] = most;
    __syncthreads();
    sum = lane < warps ? room.sum[lane] : 0.f;
    largest = __uint_as_float(__reduce_max_sync(0xffffffffu, lane < warps ? room.most[lane] : 0u));
#pragma unroll
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
}
// The larger of a and |b|, NaN where one of them is.
__device__ __forceinline__ float larger_size(float a, float b) {
    float r;
    asm("{\n\t.reg .f32 t;\n\tabs.f32 t, %2;\n\tmax.NaN.f32 %0, %1, t;\n\t}" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
// Two bf16 values, -infinity as the lowest number: its factor, zero, then has a product.
__device__ __forceinline__ uint32_t numbers_from_below(uint32_t w) {
    uint32_t r;
    asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(w), "r"(0xff7fff7fu));
    return r;
}
// g / (1 + exp(-g)): the exponent's rounding, which is 2^-17 of the result at |g| near 87 and less in proportion, two approximations (2^-22 and 2^-23 of their results), and the products.
__device__ __forceinline__ float gated(float g) {
    float e, r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(g * -1.44269504f));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + e));
    return g * r;
}

constexpr int ROW_GROUP = 4;  // rows a thread block has where a row is a warp's

template <int V, bool GATE, bool VEC>
__global__ void __launch_bounds__(V >= 4 ? 512 : 1024, V == 4 ? 2 : 1) rows_kernel(const __grid_constant__ RowsArgs a, bool x_word) {
    __shared__ RowRoom room[2];
    const uint32_t threads = a.warps * 32, th = a.warps == 1 ? threadIdx.x & 31 : threadIdx.x;
    const int64_t t = a.warps == 1 ? (int64_t)blockIdx.x * ROW_GROUP + (threadIdx.x >> 5) : (int64_t)blockIdx.x;
    if (t >= a.n_rows) return;  // (a whole warp)
    uint32_t s[V][4];  // what came in: the residual stream's values
    float y[V][8];     // what goes out, but for the norm's factor
    float by = 1.f, most = 0.f;
    load_row<V, VEC>(a.x, t * a.x_stride, a.segment, a.segment_stride, x_word, a.width, threads, th, s);
    if constexpr (GATE) {
        if (a.other) {
            uint32_t g[V][4];
            load_row<V, VEC>(a.other, t * a.other_stride, a.segment, a.segment_stride, x_word, a.width, threads, th, g);
#pragma unroll
            for (int v = 0; v < V; v++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const uint32_t two = numbers_from_below(g[v][i]);
                    y[v][2 * i] = gated(bf16_low(two)) * bf16_low(s[v][i]), y[v][2 * i + 1] = gated(bf16_high(two)) * bf16_high(s[v][i]);
                }
        } else {
#pragma unroll
            for (int v = 0; v < V; v++)
#pragma unroll
                for (int i = 0; i < 4; i++) y[v][2 * i] = bf16_low(s[v][i]), y[v][2 * i + 1] = bf16_high(s[v][i]);
        }
        if (a.out_type == ZKB_VALUE_INT8) {
#pragma unroll
            for (int v = 0; v < V; v++)
#pragma unroll
                for (int i = 0; i < 8; i++) most = larger_size(most, y[v][i]);
            float none = 0.f;
            over_row(room[0], a.warps, none, most);
        }
    } else {
        uint32_t w[V][4];
        {
            uint32_t h[V][4];
            if (a.other) load_row<V, VEC>(a.other, t * a.other_stride, 0, 0, a.other_word, a.width, threads, th, h);
            if (a.weight) load_row<V, VEC>(a.weight, 0, 0, 0, false, a.width, threads, th, w);
            if (a.other) {
#pragma unroll
                for (int v = 0; v < V; v++)
#pragma unroll
                    for (int i = 0; i < 4; i++) s[v][i] = pack_bf16(bf16_low(s[v][i]) + bf16_low(h[v][i]), bf16_high(s[v][i]) + bf16_high(h[v][i]));
            }
        }
        if (a.sum) store_row<V, VEC>(a.sum, t * a.sum_stride, a.sum_word, a.width, threads, th, s);
        float ss = 0.f;
#pragma unroll
        for (int v = 0; v < V; v++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float lo = bf16_low(s[v][i]), hi = bf16_high(s[v][i]);
                ss = fmaf(lo, lo, ss), ss = fmaf(hi, hi, ss);
                y[v][2 * i] = a.weight ? lo * bf16_low(w[v][i]) : lo, y[v][2 * i + 1] = a.weight ? hi * bf16_high(w[v][i]) : hi;
                most = larger_size(larger_size(most, y[v][2 * i]), y[v][2 * i + 1]);
            }
        over_row(room[0], a.warps, ss, most);
        const float mean = ss / (float)a.width + a.eps;
        by = rsqrtf(mean);
        // Squares or products that 32 bits do not hold, or values that are no numbers: the same for the whole row. A product, y before the norm's factor, is off by up to 2^-150, whatever its size. To codes
        // that is nothing beside the largest one; of values it is 2^-7 of bf16's least step, 2^-133, where the factor is less than 2^10 (with an eps of 10^-6 it always is).
        const float least = a.out_type == ZKB_VALUE_INT8 ? 0x1p-90f : 0x1p-20f;
        if (!(mean > least && mean < 0x1p120f && most > 0x1p-80f && most < INFINITY)) {
            double wide = 0.;
#pragma unroll
            for (int v = 0; v < V; v++)
#pragma unroll
                for (int i = 0; i < 4; i++) wide += (double)bf16_low(s[v][i]) * bf16_low(s[v][i]) + (double)bf16_high(s[v][i]) * bf16_high(s[v][i]);
#pragma unroll
            for (int o = 16; o; o >>= 1) wide += __shfl_xor_sync(0xffffffffu, wide, o);
            __shared__ double wide_sm[32];
            if (a.warps > 1) {
                if ((threadIdx.x & 31) == 0) wide_sm[threadIdx.x >> 5] = wide;
                __syncthreads();
                wide = 0.;
                for (uint32_t i = 0; i < a.warps; i++) wide += wide_sm[i];
            }
            if (wide != 0.) {  // (a row of zeros is as it was)
                const double root = rsqrt(wide / a.width + (double)a.eps);
                most = 0.f, by = 1.f;
#pragma unroll
                for (int v = 0; v < V; v++)
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        const uint32_t col = column_of<VEC>(v, i, threads, th);
                        const double by_weight = a.weight && col < a.width ? (double)bf16_low(a.weight[col]) : 1.;
                        y[v][i] = (float)((double)(i % 2 ? bf16_high(s[v][i / 2]) : bf16_low(s[v][i / 2])) * by_weight * root);
                        if (col < a.width) most = larger_size(most, y[v][i]);
                    }
                float none = 0.f;
                over_row(room[1], a.warps, none, most);
            }
        }
    }
    if (a.out_type != ZKB_VALUE_INT8) {
#pragma unroll
        for (int v = 0; v < V; v++)
#pragma unroll
            for (int i = 0; i < 4; i++) s[v][i] = pack_bf16(y[v][2 * i] * by, y[v][2 * i + 1] * by);
        store_row<V, VEC>(a.out, t * a.out_stride, a.out_type == ZKB_VALUE_WORD, a.width, threads, th, s);
        return;
    }
    // The codes of y * by: y times 127 over the largest of y, which 1.5 * 2^23 added rounds to the last bits of a float. Halfway between two codes, exactly, lies half the largest value, at 63.5, whose even code is
    // the upper one: the factor is the float not below 127 over the largest. Others, y / most = odd / 254, are there only where 127 divides the largest one's bits (then the factor, of eight bits, is exact;
    // of sixteen, a product's, the code by the float below is another one, and the even one of both is it).
    if (th == 0) a.scale[t] = most * by / 127.f;
    const bool numbers = most < INFINITY;  // else codes are 0
    if (most < 0x1p-64f) {                 // 127 over less than 2^-121 is no float
        most *= 0x1p64f;
#pragma unroll
        for (int v = 0; v < V; v++)
#pragma unroll
            for (int i = 0; i < 8; i++) y[v][i] *= 0x1p64f;
    }
    float to_code = 0.f, below = 0.f;
    if (numbers && most > 0x1.fcp-80f) {  // codes are 0 where the scale is (up to 127 x 2^-150)
        const float near = 127.f / most, left = fmaf(-near, most, 127.f);
        to_code = __uint_as_float(__float_as_uint(near) + (left > 0.f)), below = __uint_as_float(__float_as_uint(near) - (left < 0.f));
    }
    const bool halves = !GATE && ((__float_as_uint(most) & 0x7fffffu) | 0x800000u) % 127 == 0;
    int8_t* const to = static_cast<int8_t*>(a.out) + t * a.out_stride;
#pragma unroll
    for (int v = 0; v < V; v++) {
        uint32_t q[8];
#pragma unroll
        for (int i = 0; i < 8; i++) q[i] = numbers ? __float_as_uint(fmaf(y[v][i], to_code, 12582912.f)) : 0u;
        if (halves) {
#pragma unroll
            for (int i = 0; i < 8; i++)
                if (q[i] & 1) q[i] = __float_as_uint(fmaf(y[v][i], below, 12582912.f));
        }
        const uint32_t lo = __byte_perm(__byte_perm(q[0], q[1], 0x0040), __byte_perm(q[2], q[3], 0x0040), 0x5410), hi = __byte_perm(__byte_perm(q[4], q[5], 0x0040), __byte_perm(q[6], q[7], 0x0040), 0x5410);
        if constexpr (VEC) {
            const uint32_t col = column_of<VEC>(v, 0, threads, th);
            if (col < a.width) *reinterpret_cast<uint2*>(to + col) = make_uint2(lo, hi);
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const uint32_t col = column_of<VEC>(v, i, threads, th);
                if (col < a.width) to[col] = (int8_t)q[i];
            }
        }
    }
}

template <bool GATE>
static cudaError_t launch_rows(zkb_ctx* ctx, RowsArgs a, bool x_word, bool vec) {
    // Few rows: a row over many warps, for the time of one; many: four times eight values a thread, for the bytes under way; a row of up to 512 values to each warp. In us by 1, 2, 4 and 8 times
    // eight values a thread: norms of 1 x 4096 2.9, 2.8, 3.4; of 592 x 4096 7.3, 5.8, 6.3; of 8191 x 4096 63, 45, 38; of 8191 x 512 10, 8.5, 9.9; gates of 32 x 14336 -, 4.1, 4.3, 4.7, of
    // 4096 x 14336 -, 83, 58, 67, of 4096 x 16384 -, 93, 63, 68.
    const uint32_t eights = (a.width + 7) / 8;
    uint32_t v = 4;
    if (eights <= 32 || (a.n_rows < 148 * 4 && eights <= 1024)) v = 1;
    else if (eights <= 64 || (a.n_rows < 148 * 4 && eights <= 2048)) v = 2;
    a.warps = (eights + 32 * v - 1) / (32 * v);
    if (v == 4 && a.warps > 16) v = 8, a.warps = (eights + 255) / 256;
    const uint32_t block = a.warps == 1 ? 32 * ROW_GROUP : 32 * a.warps, grid = a.warps == 1 ? (a.n_rows + ROW_GROUP - 1) / ROW_GROUP : a.n_rows;
    auto launch = [&](auto one, auto two, auto four, auto eight) {
        if (v == 1) one<<<grid, block, 0, ctx->stream>>>(a, x_word);
        else if (v == 2) two<<<grid, block, 0, ctx->stream>>>(a, x_word);
        else if (v == 4) four<<<grid, block, 0, ctx->stream>>>(a, x_word);
        else eight<<<grid, block, 0, ctx->stream>>>(a, x_word);
    };
    if (vec) launch(rows_kernel<1, GATE, true>, rows_kernel<2, GATE, true>, rows_kernel<4, GATE, true>, rows_kernel<8, GATE, true>);
    else launch(rows_kernel<1, GATE, false>, rows_kernel<2, GATE, false>, rows_kernel<4, GATE, false>, rows_kernel<8, GATE, false>);
    return cudaGetLastError();
}

static size_t value_size(uint32_t type) { return type == ZKB_VALUE_WORD ? 4 : type == ZKB_VALUE_INT8 ? 1 : 2; }
static bool is_values(uint32_t type) { return type == ZKB_VALUE_BF16 || type == ZKB_VALUE_WORD; }

}  // namespace zk

using namespace zk;

extern "C" {

int zkb_step_residual_norm(zkb_ctx* ctx, const zkb_step_residual_norm_args* args) {
    if (!ctx) return ZKB_EINVAL;
    ZKB_CHECK_ARG(ctx, args);
    const zkb_step_residual_norm_args& a = *args;
    ZKB_CHECK_ARG(ctx, is_values(a.x_type) && is_values(a.residual_type) && is_values(a.sum_type) && (is_values(a.out_type) || a.out_type == ZKB_VALUE_INT8));
    ZKB_CHECK_ARG(ctx, a.width >= 1 && a.width <= 32768 && a.n_rows <= 0x7fffffffu && std::isfinite(a.eps) && a.eps >= 0.f);
    if (a.n_rows == 0) return ZKB_OK;
    const size_t xs = value_size(a.x_type), rs = value_size(a.residual_type), ss = value_size(a.sum_type), os = value_size(a.out_type);
    ZKB_CHECK_ARG(ctx, a.x && a.out && (a.out_type == ZKB_VALUE_INT8 ? a.out_scale != nullptr : !a.out_scale));
    ZKB_CHECK_ARG(ctx, aligned_to(a.x, xs) && aligned_to(a.residual, rs) && aligned_to(a.weight, 2) && aligned_to(a.sum_out, ss) && aligned_to(a.out, os) && aligned_to(a.out_scale, 4));
    ZKB_CHECK_ARG(ctx, a.n_rows == 1 || std::llabs(a.out_stride) >= (long long)a.width);
    ZKB_CHECK_ARG(ctx, a.n_rows == 1 || !a.sum_out || std::llabs(a.sum_stride) >= (long long)a.width);
    ZKB_CHECK_ARG(ctx, a.sum_out == nullptr || a.sum_out != a.residual || (a.sum_type == a.residual_type && (a.n_rows == 1 || a.sum_stride == a.residual_stride)));
    const bool split = a.x_segment && a.x_segment < a.width;
    auto wide = [](const void* p, size_t size, int64_t stride) { return aligned_to(p, size == 1 ? 8 : 16) && (size == 1 ? stride % 8 == 0 : stride * (int64_t)size % 16 == 0); };
    const bool vec = a.width % 8 == 0 && wide(a.x, xs, a.x_stride) && wide(a.residual, rs, a.residual ? a.residual_stride : 0) && aligned_to(a.weight, 16) && wide(a.sum_out, ss, a.sum_out ? a.sum_stride : 0) &&
                     wide(a.out, os, a.out_stride) && (!split || (a.x_segment % 8 == 0 && a.x_segment_stride * (int64_t)xs % 16 == 0));
    DeviceGuard g(ctx);
    ProfScope prof(ctx, "step_residual_norm_kernel");
    const RowsArgs r{a.x, a.residual, a.weight, a.sum_out, a.out, a.out_scale, a.x_stride, a.x_segment_stride, a.residual_stride, a.sum_stride, a.out_stride, a.n_rows, a.width, split ? a.x_segment : 0u,
                     a.out_type, a.residual_type == ZKB_VALUE_WORD, a.sum_type == ZKB_VALUE_WORD, a.eps, 0};
    ZKB_CUDA(ctx, launch_rows<false>(ctx, r, a.x_type == ZKB_VALUE_WORD, vec));
    return ZKB_OK;
}

int zkb_step_gate(zkb_ctx* ctx, const zkb_step_gate_args* args) {
    if (!ctx) return ZKB_EINVAL;
    ZKB_CHECK_ARG(ctx, args);
    const zkb_step_gate_args& a = *args;
    ZKB_CHECK_ARG(ctx, is_values(a.x_type) && (is_values(a.out_type) || a.out_type == ZKB_VALUE_INT8));
    ZKB_CHECK_ARG(ctx, a.width >= 1 && a.width <= 32768 && a.n_rows <= 0x7fffffffu);
    if (a.n_rows == 0) return ZKB_OK;
    const size_t xs = value_size(a.x_type), os = value_size(a.out_type);
    ZKB_CHECK_ARG(ctx, a.x && a.out && (a.out_type == ZKB_VALUE_INT8 ? a.out_scale != nullptr : !a.out_scale));
    ZKB_CHECK_ARG(ctx, aligned_to(a.x, xs) && aligned_to(a.gate, xs) && aligned_to(a.out, os) && aligned_to(a.out_scale, 4));
    ZKB_CHECK_ARG(ctx, a.n_rows == 1 || std::llabs(a.out_stride) >= (long long)a.width);
    const bool split = a.segment && a.segment < a.width;
    auto wide = [](const void* p, size_t size, int64_t stride) { return aligned_to(p, size == 1 ? 8 : 16) && (size == 1 ? stride % 8 == 0 : stride * (int64_t)size % 16 == 0); };
    const bool vec = a.width % 8 == 0 && wide(a.x, xs, a.x_stride) && wide(a.gate, xs, a.gate ? a.gate_stride : 0) && wide(a.out, os, a.out_stride) &&
                     (!split || (a.segment % 8 == 0 && a.segment_stride * (int64_t)xs % 16 == 0));
    DeviceGuard g(ctx);
    ProfScope prof(ctx, "step_gate_kernel");
    const RowsArgs r{a.x, a.gate, nullptr, nullptr, a.out, a.out_scale, a.x_stride, a.segment_stride, a.gate_stride, 0, a.out_stride, a.n_rows, a.width, split ? a.segment : 0u, a.out_type, false, false, 0.f, 0};
    ZKB_CUDA(ctx, launch_rows<true>(ctx, r, a.x_type == ZKB_VALUE_WORD, vec));
    return ZKB_OK;
}

}  // extern "C"
