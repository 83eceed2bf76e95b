// Root-mean-square norm of rows of features with the addition of the residual stream, its output in the stream's types or
// in 8 bits with a scale a row, its gradient, and rows of any matrix in 8 bits.
//
//     h = x + r;  s = 1 / sqrt(mean(h^2) + eps);  y = h s w
//     8 bits: t = h w, a = max|t| of the row: q = round(t (T / a)), scale = a s / T, T = 448 (e4m3) or 127 (int8)
//     gradient, g = dy w, c = s^2 / D sum(g h):  dh = s (g - h c) + dh_in;  dw = sum over rows of dy h s
//
// The 8-bit form needs no second look at a row: the row's maximum of |h w| is found in the pass that sums h^2, s
// stands in the scale alone and q does not depend on its rounding.
//
// All of it is bound by memory (5 to 12 operations an element against 2 to 16 bytes), so a row is read once and stays in registers:
// G neighbouring threads hold a row, 8 C elements each, in pieces of eight that are 16 bytes of a 16-bit type.  G and C follow
// from the row's length alone; workgroups walk over the rows with the weight in registers.  Sums are in 32 bits, added in a fixed
// order; the weight's gradient leaves one partial row per workgroup, which a second kernel adds up, also in a fixed order.
// Squares of a row that leave the range of 32 bits - elements beyond 1.8e19, or all so small that eps does not hold them up - are summed again
// from the row times a power of two (rescale), which y, the scale and dw do not notice.
// A row of a length that is no multiple of eight ends in a piece that reaches back into the piece before it: its elements
// are read and written twice, with the same values, and summed once.
//
// Measured, against a copy of 1 GiB at 5.04 TB/s: float32 170k x 128 with a float32 stream 70 us (5.0 TB/s), bfloat16 16k x 4096 into e4m3 86 (5.5),
// gradient of bfloat16 32k x 2048 103 (5.2), of float16 5003 x 1001 in odd rows 12 + 4 (two launches); one row of 4096 features 4.
#include "lf_rows.h"

namespace {

using namespace lf;

struct NormArgs {
    const void* x; const void* res; const void* w; void* y; void* h; float* scale;
    int64_t ldx, ldr, ldy, ldh;
    int64_t rows;
    int32_t dim, w_dtype, y_dtype, norm;                    // norm 0: rows as they are (quantize_rows)
    int32_t stream;                                         // outputs past the caches
    float eps, inv_dim;
};

template <typename XT, typename RT, int G, int C>
__global__ void __launch_bounds__(G < 256 ? 256 : G)
rms_norm_kernel(NormArgs a) {
    constexpr int T = G < 256 ? 256 : G, R = T / G;
    __shared__ float s_red[2 * (G > 64 ? G / 64 : 1)];
    const int lane = threadIdx.x % G, group = threadIdx.x / G, dim = a.dim;
    const bool q8 = a.scale != nullptr;
    float8_t w[C];
#pragma unroll
    for (int c = 0; c < C; ++c) {
        w[c] = float8_t{1.f, 1.f, 1.f, 1.f, 1.f, 1.f, 1.f, 1.f};
        if (a.w) w[c] = load_piece(a.w, 0, a.w_dtype, piece_of((c * G + lane) * 8, dim), dim);
    }
    for (int64_t row = (int64_t)blockIdx.x * R + group; row < a.rows; row += (int64_t)gridDim.x * R) {
        float8_t h[C];
        const XT* x = (const XT*)a.x + row * a.ldx;
#pragma unroll
        for (int c = 0; c < C; ++c) h[c] = load_piece(x, piece_of((c * G + lane) * 8, dim), dim);
        if (a.res) {
            const RT* r = (const RT*)a.res + row * a.ldr;
            float8_t v[C];
#pragma unroll
            for (int c = 0; c < C; ++c) v[c] = load_piece(r, piece_of((c * G + lane) * 8, dim), dim);
#pragma unroll
            for (int c = 0; c < C; ++c) h[c] += v[c];
        }
        float sum, none = 0.f;
        uint32_t top;
        auto reduce = [&](float up) {
            sum = 0.f;
            top = 0;
#pragma unroll
            for (int c = 0; c < C; ++c) {
                const Piece p = piece_of((c * G + lane) * 8, dim);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float t = h[c][i] * up, v = i >= p.first ? t : 0.f;
                    sum = fmaf(v, v, sum);
                    if (q8) top = max(top, __float_as_uint(p.first < 8 ? t * w[c][i] : 0.f) & 0x7fffffffu);
                }
            }
            row_reduce<G, true>(sum, none, top, s_red);
        };
        reduce(1.f);
        float s = 1.f, up = 1.f;
        if (a.norm) {
            float ms = fmaf(sum, a.inv_dim, a.eps);
            up = rescale(ms);
            if (__builtin_expect(up != 1.f, 0)) {                        // (the same for all threads of the row)
                reduce(up);
                ms = fmaf(sum, a.inv_dim, a.eps * up * up);
            }
            s = 1.f / sqrtf(ms);
        }
        if (a.res) {
            RT* hr = (RT*)a.h + row * a.ldh;
#pragma unroll
            for (int c = 0; c < C; ++c) {
                const Piece p = piece_of((c * G + lane) * 8, dim);
                if (p.first < 8) store_piece(hr, p, dim, h[c], a.stream);
            }
        }
        if (__builtin_expect(up != 1.f, 0))
#pragma unroll
            for (int c = 0; c < C; ++c) h[c] *= up;
        if (!q8) {
#pragma unroll
            for (int c = 0; c < C; ++c) {
                const Piece p = piece_of((c * G + lane) * 8, dim);
                if (p.first < 8) store_piece(a.y, row * a.ldy, a.y_dtype, p, dim, h[c] * s * w[c], a.stream);
            }
            continue;
        }
        const Eighth q(top, a.y_dtype);
        if (lane == 0) a.scale[row] = q.scale(s);
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const Piece p = piece_of((c * G + lane) * 8, dim);
            if (p.first < 8) q.store((uint8_t*)a.y + row * a.ldy + p.at, h[c] * w[c], dim, a.stream);
        }
    }
}

// Rows that no workgroup holds in its registers: read once for the sums and once more, out of the caches, for the output.
template <typename XT, typename RT>
__global__ void __launch_bounds__(1024)
rms_norm_long_kernel(NormArgs a) {
    __shared__ float s_red[32];
    const int dim = a.dim;
    const bool q8 = a.scale != nullptr;
    auto weight = [&](int col, int n) {
        return a.w ? load_upto8(a.w, col, a.w_dtype, n) : float8_t{1.f, 1.f, 1.f, 1.f, 1.f, 1.f, 1.f, 1.f};
    };
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const XT* x = (const XT*)a.x + row * a.ldx;
        const RT* r = (const RT*)a.res + row * a.ldr;
        auto sum8 = [&](int col, int n) {
            float8_t h = load_upto8(x + col, n);
            if (a.res) h += load_upto8(r + col, n);
            return h;
        };
        float sum, none = 0.f, up = 1.f, s = 1.f;
        uint32_t top;
        auto reduce = [&] {
            sum = 0.f;
            top = 0;
            for (int col = threadIdx.x * 8; col < dim; col += 8192) {
                const int n = min(8, dim - col);
                const float8_t h = sum8(col, n) * up;
#pragma unroll
                for (int i = 0; i < 8; ++i) sum = fmaf(h[i], h[i], sum);
                if (q8) {
                    const float8_t t = h * weight(col, n);
#pragma unroll
                    for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(i < n ? t[i] : 0.f) & 0x7fffffffu);
                }
            }
            row_reduce<1024, true>(sum, none, top, s_red);
        };
        reduce();
        if (a.norm) {
            up = rescale(fmaf(sum, a.inv_dim, a.eps));
            if (up != 1.f) reduce();
            s = 1.f / sqrtf(fmaf(sum, a.inv_dim, a.eps * up * up));
        }
        const Eighth q(top, a.y_dtype);
        if (q8 && threadIdx.x == 0) a.scale[row] = q.scale(s);
        for (int col = threadIdx.x * 8; col < dim; col += 8192) {
            const int n = min(8, dim - col);
            const float8_t h = sum8(col, n), w = weight(col, n);
            if (a.res) store_upto8((RT*)a.h + row * a.ldh + col, h, n);
            if (!q8) {
                store_upto8(a.y, row * a.ldy + col, a.y_dtype, h * up * s * w, n);
            } else {
                q.store((uint8_t*)a.y + row * a.ldy + col, h * up * w, n, a.stream);
            }
        }
    }
}

struct GradArgs {
    const void* dy; const void* h; const void* w; const void* dh; void* dx; float* part;
    void* dw;                                               // of a single workgroup, which needs no partial sums
    int64_t ldy, ldh, ldd, ldx;
    int64_t rows;
    int32_t dim, w_dtype;
    int32_t stream;
    float eps, inv_dim;
};

template <typename DT, typename HT, int G, int C>
__global__ void __launch_bounds__(G < 256 ? 256 : G)
rms_norm_grad_kernel(GradArgs a) {
    constexpr int T = G < 256 ? 256 : G, R = T / G;
    __shared__ float s_red[2 * (G > 64 ? G / 64 : 1)];
    __shared__ float s_dw[R > 1 ? T * 8 * C : 1];
    const int lane = threadIdx.x % G, group = threadIdx.x / G, dim = a.dim;
    float8_t w[C], dw[C];
#pragma unroll
    for (int c = 0; c < C; ++c) {
        w[c] = float8_t{1.f, 1.f, 1.f, 1.f, 1.f, 1.f, 1.f, 1.f};
        dw[c] = float8_t{0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        if (a.w) w[c] = load_piece(a.w, 0, a.w_dtype, piece_of((c * G + lane) * 8, dim), dim);
    }
    for (int64_t row = (int64_t)blockIdx.x * R + group; row < a.rows; row += (int64_t)gridDim.x * R) {
        float8_t h[C], dy[C];
        const HT* hr = (const HT*)a.h + row * a.ldh;
        const DT* dr = (const DT*)a.dy + row * a.ldy;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const Piece p = piece_of((c * G + lane) * 8, dim);
            h[c] = load_piece(hr, p, dim);
            dy[c] = load_piece(dr, p, dim);
        }
        float sum, dot, up = 1.f;
        uint32_t none = 0;
        auto reduce = [&] {
            sum = dot = 0.f;
#pragma unroll
            for (int c = 0; c < C; ++c) {
                const Piece p = piece_of((c * G + lane) * 8, dim);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float v = i >= p.first ? h[c][i] : 0.f;
                    sum = fmaf(v, v, sum);
                    // (a 0 for h in its place must not meet an infinite gradient)
                    dot = i >= p.first ? fmaf(dy[c][i] * w[c][i], v, dot) : dot;
                }
            }
            row_reduce<G, false>(sum, dot, none, s_red);
        };
        reduce();
        float ms = fmaf(sum, a.inv_dim, a.eps);
        up = rescale(ms);
        if (__builtin_expect(up != 1.f, 0)) {                            // (the same for all threads of the row)
#pragma unroll
            for (int c = 0; c < C; ++c) h[c] *= up;
            reduce();
            ms = fmaf(sum, a.inv_dim, a.eps * up * up);
        }
        const float s = 1.f / sqrtf(ms);                                 // (of h as it is now: up times less than of the row itself)
        const float k = dot * a.inv_dim * s * s, s_row = s * up;
        HT* dx = (HT*)a.dx + row * a.ldx;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const Piece p = piece_of((c * G + lane) * 8, dim);
            float8_t d = (dy[c] * w[c] - h[c] * k) * s_row;
            if (a.dh) d += load_piece((const HT*)a.dh + row * a.ldd, p, dim);
            dw[c] += dy[c] * h[c] * s;
            if (p.first < 8) store_piece(dx, p, dim, d, a.stream);
        }
    }
    if (!a.part && !a.dw) return;
    auto leave = [&](int col, float v) {
        if (a.part) a.part[(int64_t)blockIdx.x * dim + col] = v;
        else store_one(a.dw, col, a.w_dtype, v);
    };
    if constexpr (R > 1) {
        // the sums of a workgroup's row groups, column by column
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int i = 0; i < 8; ++i) s_dw[(group * C + c) * 8 * G + lane * 8 + i] = dw[c][i];
        __syncthreads();
        for (int j = threadIdx.x; j < 8 * C * G; j += T) {
            const Piece p = piece_of(j & ~7, dim);
            if ((j & 7) < p.first || p.at + (j & 7) >= dim) continue;
            float v = 0.f;
#pragma unroll
            for (int g = 0; g < R; ++g) v += s_dw[g * 8 * C * G + j];
            leave(p.at + (j & 7), v);
        }
    } else {
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const Piece p = piece_of((c * G + lane) * 8, dim);
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (i >= p.first && p.at + i < dim) leave(p.at + i, dw[c][i]);
        }
    }
}

template <typename DT, typename HT>
__global__ void __launch_bounds__(1024)
rms_norm_grad_long_kernel(GradArgs a) {
    __shared__ float s_red[32];
    const int dim = a.dim;
    float* part = a.part ? a.part + (int64_t)blockIdx.x * dim : nullptr;      // (a thread's own columns of it, from row to row)
    auto weighted = [&](float8_t dy, int col, int n) { return a.w ? dy * load_upto8(a.w, col, a.w_dtype, n) : dy; };
    bool first = true;
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const HT* hr = (const HT*)a.h + row * a.ldh;
        const DT* dr = (const DT*)a.dy + row * a.ldy;
        float sum, dot, up = 1.f;
        uint32_t none = 0;
        auto reduce = [&] {
            sum = dot = 0.f;
            for (int col = threadIdx.x * 8; col < dim; col += 8192) {
                const int n = min(8, dim - col);
                const float8_t h = load_upto8(hr + col, n) * up, g = weighted(load_upto8(dr + col, n), col, n);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    sum = fmaf(h[i], h[i], sum);
                    dot = fmaf(g[i], h[i], dot);
                }
            }
            row_reduce<1024, false>(sum, dot, none, s_red);
        };
        reduce();
        up = rescale(fmaf(sum, a.inv_dim, a.eps));
        if (up != 1.f) reduce();
        const float s = 1.f / sqrtf(fmaf(sum, a.inv_dim, a.eps * up * up));
        const float k = dot * a.inv_dim * s * s, s_row = s * up;
        for (int col = threadIdx.x * 8; col < dim; col += 8192) {
            const int n = min(8, dim - col);
            const float8_t h = load_upto8(hr + col, n) * up, dy = load_upto8(dr + col, n);
            float8_t d = (weighted(dy, col, n) - h * k) * s_row;
            if (a.dh) d += load_upto8((const HT*)a.dh + row * a.ldd + col, n);
            store_upto8((HT*)a.dx + row * a.ldx + col, d, n);
            if (part) {
                float8_t w = dy * h * s;
                if (!first) w += load_upto8(part + col, n);
                store_upto8(part + col, w, n);
            }
        }
        first = false;
    }
}

// Columns of [n][dim] partial sums: 16 columns to a workgroup, every 64th row to a thread, then the threads in order.
__global__ void __launch_bounds__(1024) column_sums_kernel(const float* part, int64_t n, int32_t dim, void* out, int32_t dtype) {
    __shared__ float s[64][17];
    const int col = blockIdx.x * 16 + (threadIdx.x & 15), slice = threadIdx.x >> 4;
    const float* src = part + min(col, dim - 1);
    float v = 0.f;
#pragma unroll 8
    for (int64_t r = slice; r < n; r += 64) v += src[r * dim];
    s[slice][threadIdx.x & 15] = v;
    __syncthreads();
    if (slice || col >= dim) return;
    v = 0.f;
#pragma unroll
    for (int i = 0; i < 64; ++i) v += s[i][threadIdx.x];
    store_one(out, col, dtype, v);
}

template <typename A, typename B> struct Kernels {
    using Norm = void (*)(NormArgs);
    using Grad = void (*)(GradArgs);
    static Norm norm(Shape s) {
        switch (s.group) {
            case 8: return rms_norm_kernel<A, B, 8, 1>;
            case 16: return rms_norm_kernel<A, B, 16, 1>;
            case 32: return rms_norm_kernel<A, B, 32, 1>;
            case 64: return s.pieces == 1 ? rms_norm_kernel<A, B, 64, 1> : rms_norm_kernel<A, B, 64, 2>;
            case 256: return s.pieces == 1 ? rms_norm_kernel<A, B, 256, 1> : rms_norm_kernel<A, B, 256, 2>;
            case 512: return rms_norm_kernel<A, B, 512, 2>;
            default: return s.pieces == 2 ? rms_norm_kernel<A, B, 1024, 2> : rms_norm_long_kernel<A, B>;
        }
    }
    static Grad grad(Shape s) {
        switch (s.group) {
            case 8: return rms_norm_grad_kernel<A, B, 8, 1>;
            case 16: return rms_norm_grad_kernel<A, B, 16, 1>;
            case 32: return rms_norm_grad_kernel<A, B, 32, 1>;
            case 64: return s.pieces == 1 ? rms_norm_grad_kernel<A, B, 64, 1> : rms_norm_grad_kernel<A, B, 64, 2>;
            case 256: return s.pieces == 1 ? rms_norm_grad_kernel<A, B, 256, 1> : rms_norm_grad_kernel<A, B, 256, 2>;
            case 512: return rms_norm_grad_kernel<A, B, 512, 2>;
            default: return s.pieces == 2 ? rms_norm_grad_kernel<A, B, 1024, 2> : rms_norm_grad_long_kernel<A, B>;
        }
    }
};
template <typename F> auto of_types(int32_t a, int32_t b, F f) {
    auto second = [&](auto x) {
        using X = decltype(x);
        return b == LF_DTYPE_F32 ? f(Kernels<X, float>{}) : b == LF_DTYPE_BF16 ? f(Kernels<X, __bf16>{}) : f(Kernels<X, _Float16>{});
    };
    return a == LF_DTYPE_F32 ? second(0.f) : a == LF_DTYPE_BF16 ? second((__bf16)0.f) : second((_Float16)0.f);
}

// Workgroups of 256 threads.  Of the norm twice what fills the GPU, so that its last ones are few (bf16 16k x 4096 into e4m3 with 2048 / 3072 / 4096 75.8 / 71.9 / 71.1 us,
// 170k x 47 9.2 / 8.9 / 9.6); of the gradient only as many as fill it, as each leaves a partial row of dw.
constexpr int kNormGroups = 3072, kGradGroups = 1024;
unsigned grad_groups(int64_t rows, int64_t dim) {
    return std::min(workgroups(rows, shape_of(dim), kGradGroups), (unsigned)std::max<int64_t>(1, (1ll << 26) / dim));
}
// Whether a launch of one workgroup leaves dw itself, which saves the second launch's 4 us (long rows keep it in memory meanwhile).
bool alone(int64_t rows, int64_t dim) { return shape_of(dim).pieces <= 2 && grad_groups(rows, dim) == 1; }

}  // namespace

namespace lf {
int column_sums(const float* part, int64_t n, int64_t dim, void* out, int32_t dtype, hipStream_t stream) {
    column_sums_kernel<<<(unsigned)ceil_div(dim, 16), 1024, 0, stream>>>(part, n, (int32_t)dim, out, dtype);
    LF_HIP(hipGetLastError());
    return LF_OK;
}
}  // namespace lf

extern "C" {

int lf_rms_norm(const void* d_x, int64_t ld_x, int32_t x_dtype, const void* d_residual, int64_t ld_residual, int32_t residual_dtype,
                const void* d_weight, int32_t weight_dtype, int64_t rows, int64_t dim, float eps, void* d_y, int64_t ld_y, int32_t y_dtype,
                float* d_scale, void* d_h, int64_t ld_h, lf_stream_t stream) {
    LF_TRY(check_shape(rows, dim));
    LF_REQUIRE(is_float_dtype(x_dtype) && (!d_residual || is_float_dtype(residual_dtype)) && (!d_weight || is_float_dtype(weight_dtype)),
               LF_ERR_UNSUPPORTED, "x, residual and weight are float32, bfloat16 or float16");
    LF_REQUIRE(is_float_dtype(y_dtype) || is_8bit_dtype(y_dtype), LF_ERR_UNSUPPORTED, "unknown type of y");
    LF_REQUIRE(is_8bit_dtype(y_dtype) == (d_scale != nullptr) || rows == 0, LF_ERR_INVALID, "8-bit rows, and only they, come with scales");
    LF_REQUIRE(eps >= 0.f, LF_ERR_INVALID, "eps must not be negative");
    LF_REQUIRE(!d_residual == !d_h || rows == 0, LF_ERR_INVALID, "the residual and h = x + residual come together");
    if (rows == 0) return LF_OK;
    LF_TRY(check_rows("x", rows, dim, d_x, ld_x, x_dtype));
    LF_TRY(check_rows("y", rows, dim, d_y, ld_y, y_dtype));
    if (d_residual) {
        LF_TRY(check_rows("residual", rows, dim, d_residual, ld_residual, residual_dtype));
        LF_TRY(check_rows("h", rows, dim, d_h, ld_h, residual_dtype));
    }
    if (d_weight) LF_TRY(check_rows("weight", 1, dim, d_weight, dim, weight_dtype));
    const NormArgs a{d_x, d_residual, d_weight, d_y, d_h, d_scale, ld_x, ld_residual, ld_y, ld_h, rows, (int32_t)dim, weight_dtype, y_dtype, 1,
                     rows * dim * (dtype_bytes(y_dtype) + (d_h ? dtype_bytes(residual_dtype) : 0)) >= kStreamBytes, eps, (float)(1.0 / (double)dim)};
    const Shape s = shape_of(dim);
    auto kernel = of_types(x_dtype, d_residual ? residual_dtype : x_dtype, [&](auto k) { return decltype(k)::norm(s); });
    kernel<<<workgroups(rows, s, kNormGroups), std::max(s.group, 256), 0, (hipStream_t)stream>>>(a);
    LF_HIP(hipGetLastError());
    return LF_OK;
}

int lf_quantize_rows(const void* d_x, int64_t ld_x, int32_t x_dtype, int64_t rows, int64_t dim, void* d_q, int64_t ld_q, int32_t q_dtype,
                     float* d_scale, lf_stream_t stream) {
    LF_TRY(check_shape(rows, dim));
    LF_REQUIRE(is_float_dtype(x_dtype), LF_ERR_UNSUPPORTED, "x is float32, bfloat16 or float16");
    LF_REQUIRE(is_8bit_dtype(q_dtype), LF_ERR_UNSUPPORTED, "q is e4m3 or int8");
    if (rows == 0) return LF_OK;
    LF_REQUIRE(d_scale, LF_ERR_INVALID, "null pointer");
    LF_TRY(check_rows("x", rows, dim, d_x, ld_x, x_dtype));
    LF_TRY(check_rows("q", rows, dim, d_q, ld_q, q_dtype));
    const NormArgs a{d_x, nullptr, nullptr, d_q, nullptr, d_scale, ld_x, 0, ld_q, 0, rows, (int32_t)dim, LF_DTYPE_F32, q_dtype, 0,
                     rows * dim >= kStreamBytes, 0.f, 0.f};
    const Shape s = shape_of(dim);
    auto kernel = of_types(x_dtype, x_dtype, [&](auto k) { return decltype(k)::norm(s); });
    kernel<<<workgroups(rows, s, kNormGroups), std::max(s.group, 256), 0, (hipStream_t)stream>>>(a);
    LF_HIP(hipGetLastError());
    return LF_OK;
}

size_t lf_rms_norm_grad_work_bytes(int64_t rows, int64_t dim) {
    if (rows <= 0 || dim < 1 || dim > kMaxDim || alone(rows, dim)) return 0;
    return (size_t)grad_groups(rows, dim) * (size_t)dim * sizeof(float);
}

int lf_rms_norm_grad(const void* d_dy, int64_t ld_dy, int32_t dy_dtype, const void* d_h, int64_t ld_h, int32_t h_dtype, const void* d_weight,
                     int32_t weight_dtype, const void* d_dh, int64_t ld_dh, int64_t rows, int64_t dim, float eps, void* d_dx, int64_t ld_dx,
                     void* d_dw, void* d_work, size_t work_bytes, lf_stream_t stream) {
    LF_TRY(check_shape(rows, dim));
    LF_REQUIRE(is_float_dtype(dy_dtype) && is_float_dtype(h_dtype) && ((!d_weight && !d_dw) || is_float_dtype(weight_dtype)), LF_ERR_UNSUPPORTED,
               "dy, h and weight are float32, bfloat16 or float16");
    LF_REQUIRE(eps >= 0.f, LF_ERR_INVALID, "eps must not be negative");
    const Shape s = shape_of(dim);
    const unsigned groups = rows ? grad_groups(rows, dim) : 0;
    if (d_dw) {
        LF_TRY(check_rows("dw", 1, dim, d_dw, dim, weight_dtype));
        LF_REQUIRE(rows == 0 || alone(rows, dim) || (d_work && (uintptr_t)d_work % 16 == 0), LF_ERR_INVALID, "null or unaligned workspace");
        LF_REQUIRE(work_bytes >= lf_rms_norm_grad_work_bytes(rows, dim), LF_ERR_WORKSPACE, "workspace of %zu bytes, %zu are needed", work_bytes,
                   lf_rms_norm_grad_work_bytes(rows, dim));
    }
    hipStream_t st = (hipStream_t)stream;
    if (rows) {
        LF_TRY(check_rows("dy", rows, dim, d_dy, ld_dy, dy_dtype));
        LF_TRY(check_rows("h", rows, dim, d_h, ld_h, h_dtype));
        LF_TRY(check_rows("dx", rows, dim, d_dx, ld_dx, h_dtype));
        if (d_dh) LF_TRY(check_rows("dh", rows, dim, d_dh, ld_dh, h_dtype));
        if (d_weight) LF_TRY(check_rows("weight", 1, dim, d_weight, dim, weight_dtype));
        const bool one = alone(rows, dim);
        const GradArgs a{d_dy, d_h, d_weight, d_dh, d_dx, d_dw && !one ? (float*)d_work : nullptr, one ? d_dw : nullptr, ld_dy, ld_h, ld_dh, ld_dx, rows, (int32_t)dim, weight_dtype,
                         rows * dim * dtype_bytes(h_dtype) >= kStreamBytes, eps, (float)(1.0 / (double)dim)};
        auto kernel = of_types(dy_dtype, h_dtype, [&](auto k) { return decltype(k)::grad(s); });
        kernel<<<groups, std::max(s.group, 256), 0, st>>>(a);
        LF_HIP(hipGetLastError());
    }
    if (d_dw && !(rows && alone(rows, dim))) LF_TRY(lf::column_sums((const float*)d_work, groups, dim, d_dw, weight_dtype, st));
    return LF_OK;
}

}  // extern "C"
