// Layer norm of rows of features with the addition of the residual stream, its output in the stream's types or in 8 bits with a
// scale a row, and its gradient.
//
//     h = x + r;  mu = mean(h);  s = 1 / sqrt(mean((h - mu)^2) + eps);  t = (h - mu) s;  y = t w + b
//     8 bits: a = max|y| of the row: q = round(y (T / a)), scale = a / T, T = 448 (e4m3) or 127 (int8)
//     gradient, g = dy w:  dh = s (g - mean(g) - t mean(g t)) + dh_in;  dw = sum over rows of dy t;  db = sum over rows of dy
//
// Bound by memory, as the norms of lf_norm.hip and in their layout: a row is read once and stays in the registers of G neighbouring threads, workgroups
// walk over the rows with weight and bias in registers, partial rows of dw and db are added up by a second kernel in a fixed order.
// Two sums over the row one after the other: that of h, then those of d = h - mu and d^2 (and, in the gradient, of g and g d).  The second
// look at the mean takes off what the rounding of the first has left, so that rows far from zero keep their digits: mu is off by less than
// a rounding of the largest |h - mu|, not of |mu|.
// Measured with inputs that no cache holds, against a copy of 1 GiB at 4.96 TB/s: float32 170k x 128 with a float32 stream 69 us (5.0 TB/s), bfloat16 16k x 4096
// with its stream 99 (5.4), gradient of bfloat16 32k x 2048 108 + 5 (5.0); one row of 4096 features 4.6.
// The gradient has five sums over a row and four barriers where a workgroup shares one.  Two barriers, or products and sums in one operation, made no difference; rows of 2048
// in one wavefront, without barriers, took 139 us.
// Rows whose sums overflow are taken times 2^-100 and summed again, those whose squares vanish after the subtraction times 2^100.  Where the variance is less than
// what the correction takes off - equal elements, or such as differ in their last places - the mean is corrected first and the squares are summed once more.
#include "lf_rows.h"

namespace {

// Sums of N numbers over the G threads of a row; `s` holds N G / 64 words where G > 64.
template <int G, int N> __device__ __forceinline__ void row_sums(float (&v)[N], float* s) {
#pragma unroll
    for (int n = 0; n < N; ++n) v[n] = dpp_add<(G < 64 ? G : 64)>(v[n]);
    if constexpr (G > 64) {
        constexpr int W = G / 64;
        __syncthreads();                                   // what was there before has been read
        if ((threadIdx.x & 63) == 0)
#pragma unroll
            for (int n = 0; n < N; ++n) s[n * W + (threadIdx.x >> 6)] = v[n];
        __syncthreads();
#pragma unroll
        for (int n = 0; n < N; ++n) {
            v[n] = 0.f;
#pragma unroll
            for (int w = 0; w < W; ++w) v[n] += s[n * W + w];
        }
    }
}
template <int G> __device__ __forceinline__ uint32_t row_max(uint32_t m, uint32_t* s) {
    m = lanes_max<G>(m);
    if constexpr (G > 64) {
        constexpr int W = G / 64;
        __syncthreads();
        if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = m;
        __syncthreads();
        m = 0;
#pragma unroll
        for (int w = 0; w < W; ++w) m = max(m, s[w]);
    }
    return m;
}

__device__ __forceinline__ bool counts(const Piece& p, int i, int dim) { return i >= p.first && p.at + i < dim; }

struct LayerArgs {
    const void* x; const void* res; const void* w; const void* b; void* y; void* h; float* scale;
    int64_t ldx, ldr, ldy, ldh;
    int64_t rows;
    int32_t dim, w_dtype, b_dtype, y_dtype;
    int32_t stream;                                         // outputs past the caches
    float eps, inv_dim;
};

// What changes a row.
struct Change {
    float off, by;
    template <typename V> __device__ __forceinline__ V operator()(V x) const { return (x - off) * by; }
};

// A row's statistics: t = (h - mean - less) inv.  Where sums overflow or squares vanish the row is changed first, h -> (h - off) by, and what is said here is of
// the row as it is then; by: the power of two.
struct Centre {
    float mean, less, inv, by;
    // sum: of h.  first(f): that of f(h).  second(f, d, dd): d, dd <- sums of f(h) - mean and of its squares.  change(f): h <- f(h)
    template <typename FIRST, typename SECOND, typename CHANGE>
    __device__ __forceinline__ void find(float eps, float inv_dim, float sum, FIRST first, SECOND second, CHANGE change) {
        by = 1.f;
        float var, more = eps;                              // mean((h - mean)^2) - less^2, and what is added to it
        auto look = [&](auto f) {
            float d, dd;
            second(f, d, dd);
            less = d * inv_dim;
            const float v = fmaf(dd, inv_dim, -(less * less));
            var = (v < 0.f ? 0.f : v) + more;                            // (a NaN stays)
        };
        mean = sum * inv_dim;
        look([](float x) { return x; });
        if (__builtin_expect(!(var >= fmaxf(kTiny, less * less) && var < __builtin_inff()), 0)) {      // (the same for all threads of the row)
            // Where the variance is less than what was taken off - rows far from zero that differ in their last places, or not at all - the mean moves to the float
            // nearest to the true one, beside which such differences are not small; equal elements then leave 0.
            Change f{0.f, 1.f};
#pragma unroll 1
            for (int moves = 0;;) {
                if (less * less > var && moves < 3) {
                    ++moves;
                    mean += less;
                } else if (f.by == 1.f && !(var >= kTiny && var < __builtin_inff())) {
                    moves = 0;
                    f = var < kTiny ? Change{mean, 1.f / kTiny} : Change{0.f, kTiny};
                    more = eps * f.by * f.by;
                    mean = first(f) * inv_dim;
                } else {
                    break;
                }
                look(f);
            }
            change(f);
            by = f.by;
            if (by < 1.f && var == 0.f && eps > 0.f) {                   // (equal elements: eps alone, which the power of two has taken away)
                by = 1.f;
                var = eps;
            }
        }
        inv = 1.f / sqrtf(var);
    }
    template <typename V> __device__ __forceinline__ V of(V h) const { return (h - mean - less) * inv; }
};

template <typename XT, typename RT, int G, int C>
__global__ void __launch_bounds__(G < 256 ? 256 : G)
layer_norm_kernel(LayerArgs a) {
    constexpr int T = G < 256 ? 256 : G, R = T / G;
    __shared__ float s_red[2 * (G > 64 ? G / 64 : 1)];
    const int lane = threadIdx.x % G, group = threadIdx.x / G, dim = a.dim;
    const bool q8 = a.scale != nullptr;
    float8_t w[C], b[C];
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const Piece p = piece_of((c * G + lane) * 8, dim);
        w[c] = float8_t{1.f, 1.f, 1.f, 1.f, 1.f, 1.f, 1.f, 1.f};
        b[c] = float8_t{0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        if (a.w) w[c] = load_piece(a.w, 0, a.w_dtype, p, dim);
        if (a.b) b[c] = load_piece(a.b, 0, a.b_dtype, p, dim);
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
        const bool whole = dim % 8 == 0;                                 // (then no element needs to be looked at by itself)
        auto each_of = [&](auto f) {
#pragma unroll
            for (int c = 0; c < C; ++c) {
                const Piece p = piece_of((c * G + lane) * 8, dim);
                if (whole) {
                    if (p.first == 0)
#pragma unroll
                        for (int i = 0; i < 8; ++i) f(h[c][i]);
                } else {
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        if (counts(p, i, dim)) f(h[c][i]);
                }
            }
        };
        auto first = [&](auto f) {
            float v[1] = {0.f};
            each_of([&](float x) { v[0] += f(x); });
            row_sums<G>(v, s_red);
            return v[0];
        };
        const float sum = first([](float x) { return x; });
        // (behind the sum's barriers: h may be the residual itself, and the end of a row reaches back into what another wavefront reads)
        if (a.res) {
            RT* hr = (RT*)a.h + row * a.ldh;
#pragma unroll
            for (int c = 0; c < C; ++c) {
                const Piece p = piece_of((c * G + lane) * 8, dim);
                if (p.first < 8) store_piece(hr, p, dim, h[c], a.stream);
            }
        }
        Centre m;
        m.find(a.eps, a.inv_dim, sum, first,
               [&](auto f, float& d, float& dd) {
                   float v[2] = {0.f, 0.f};
                   each_of([&](float x) {
                       const float t = f(x) - m.mean;
                       v[0] += t;
                       v[1] = fmaf(t, t, v[1]);
                   });
                   row_sums<G>(v, s_red);
                   d = v[0];
                   dd = v[1];
               },
               [&](auto f) {
#pragma unroll
                   for (int c = 0; c < C; ++c) h[c] = f(h[c]);
               });
#pragma unroll
        for (int c = 0; c < C; ++c) h[c] = m.of(h[c]) * w[c] + b[c];
        if (!q8) {
#pragma unroll
            for (int c = 0; c < C; ++c) {
                const Piece p = piece_of((c * G + lane) * 8, dim);
                if (p.first < 8) store_piece(a.y, row * a.ldy, a.y_dtype, p, dim, h[c], a.stream);
            }
            continue;
        }
        uint32_t top = 0;
        each_of([&](float x) { top = max(top, __float_as_uint(x) & 0x7fffffffu); });
        const Eighth q(row_max<G>(top, (uint32_t*)s_red), a.y_dtype);
        if (lane == 0) a.scale[row] = q.scale(1.f);
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const Piece p = piece_of((c * G + lane) * 8, dim);
            if (p.first < 8) q.store((uint8_t*)a.y + row * a.ldy + p.at, h[c], dim, a.stream);
        }
    }
}

// Rows that no workgroup holds in its registers: read for the sum, for the squares, in 8 bits for the largest, and for the output.
template <typename XT, typename RT>
__global__ void __launch_bounds__(1024)
layer_norm_long_kernel(LayerArgs a) {
    __shared__ float s_red[32];
    const int dim = a.dim;
    const bool q8 = a.scale != nullptr;
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const XT* x = (const XT*)a.x + row * a.ldx;
        const RT* r = (const RT*)a.res + row * a.ldr;
        auto sum8 = [&](int col, int n) {
            float8_t h = load_upto8(x + col, n);
            if (a.res) h += load_upto8(r + col, n);
            return h;
        };
        auto pieces = [&](auto f) {
            for (int col = threadIdx.x * 8; col < dim; col += 8192) {
                const int n = min(8, dim - col);
                f(col, n, sum8(col, n));
            }
        };
        float off = 0.f, by = 1.f;                                       // (read again, the row is changed again)
        auto first = [&](auto f) {
            float v[1] = {0.f};
            pieces([&](int, int n, float8_t h) {
#pragma unroll
                for (int i = 0; i < 8; ++i) v[0] += i < n ? f(h[i]) : 0.f;
            });
            row_sums<1024>(v, s_red);
            return v[0];
        };
        const float sum = first([](float x) { return x; });
        Centre m;
        m.find(a.eps, a.inv_dim, sum, first,
               [&](auto f, float& d, float& dd) {
                   float v[2] = {0.f, 0.f};
                   pieces([&](int, int n, float8_t h) {
#pragma unroll
                       for (int i = 0; i < 8; ++i) {
                           const float t = i < n ? f(h[i]) - m.mean : 0.f;
                           v[0] += t;
                           v[1] = fmaf(t, t, v[1]);
                       }
                   });
                   row_sums<1024>(v, s_red);
                   d = v[0];
                   dd = v[1];
               },
               [&](auto f) {
                   off = f.off;
                   by = f.by;
               });
        auto out = [&](int col, int n, float8_t h) {
            float8_t y = m.of((h - off) * by);
            if (a.w) y *= load_upto8(a.w, col, a.w_dtype, n);
            if (a.b) y += load_upto8(a.b, col, a.b_dtype, n);
            return y;
        };
        uint32_t top = 0;
        if (q8) {
            pieces([&](int col, int n, float8_t h) {
                const float8_t y = out(col, n, h);
#pragma unroll
                for (int i = 0; i < 8; ++i) top = max(top, i < n ? __float_as_uint(y[i]) & 0x7fffffffu : 0u);
            });
            top = row_max<1024>(top, (uint32_t*)s_red);
        }
        const Eighth q(top, a.y_dtype);
        if (q8 && threadIdx.x == 0) a.scale[row] = q.scale(1.f);
        pieces([&](int col, int n, float8_t h) {
            const float8_t y = out(col, n, h);
            if (a.res) store_upto8((RT*)a.h + row * a.ldh + col, h, n);
            if (q8) q.store((uint8_t*)a.y + row * a.ldy + col, y, n, a.stream);
            else store_upto8(a.y, row * a.ldy + col, a.y_dtype, y, n);
        });
    }
}

struct LayerGradArgs {
    const void* dy; const void* h; const void* w; const void* dh; void* dx;
    float* part;                                            // [workgroups][2][dim]: of dw and db
    void* dw; void* db;
    int64_t ldy, ldh, ldd, ldx;
    int64_t rows;
    int32_t dim, w_dtype, db_dtype;
    int32_t stream;
    float eps, inv_dim;
    // `which` 0: dw, 1: db
    __device__ __forceinline__ bool wants(int which) const { return which ? db != nullptr : dw != nullptr; }
    __device__ __forceinline__ void leave(int which, int col, float v) const {
        if (part) part[((int64_t)blockIdx.x * 2 + which) * dim + col] = v;
        else if (which) store_one(db, col, db_dtype, v);
        else store_one(dw, col, w_dtype, v);
    }
};

// A piece as it lies in memory: what is loaded a row ahead takes no more registers than that.
template <typename T> __device__ __forceinline__ typename Eight<T>::vec load_raw(const T* row, const Piece& p, int dim) {
    return dim >= 8 ? reinterpret_cast<const typename Eight<T>::Any*>(row + p.at)->v : __builtin_convertvector(load_upto8(row, dim), typename Eight<T>::vec);
}

// A workgroup's next row is loaded before the sums of this one, whose barriers it fills (bf16 32k x 2048: 117 us without).  Not where the registers for it would
// take the place of other wavefronts.
template <typename DT, typename HT, int G, int C>
__global__ void __launch_bounds__(G < 256 ? 256 : G)
layer_norm_grad_kernel(LayerGradArgs a) {
    constexpr int T = G < 256 ? 256 : G, R = T / G;
    __shared__ float s_red[4 * (G > 64 ? G / 64 : 1)];
    __shared__ float s_sum[R > 1 ? T * 8 * C : 1];
    const int lane = threadIdx.x % G, group = threadIdx.x / G, dim = a.dim;
    // A workgroup of 1024 threads has 128 registers a thread.  With a stream of float32 the weight exceeds them by 11 words: read again from the caches it takes 80 us for
    // 900 x 16,384, not 84; with one of 16 bits by 3, and there 57 us become 61.
    constexpr bool HELD = G < 1024 || sizeof(HT) == 2;
    float8_t w[C], sums[2][C];
    auto weight = [&](int c) {
        uintptr_t at = (uintptr_t)a.w;
        if (!HELD) asm volatile("" : "+s"(at));            // (for every row, not once before them all)
        const void* p = (const void*)(const __attribute__((address_space(1))) char*)at;
        return at ? load_piece(p, 0, a.w_dtype, piece_of((c * G + lane) * 8, dim), dim) : float8_t{1.f, 1.f, 1.f, 1.f, 1.f, 1.f, 1.f, 1.f};
    };
#pragma unroll
    for (int c = 0; c < C; ++c) {
        if (HELD) w[c] = weight(c);
        sums[0][c] = sums[1][c] = float8_t{0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    }
    constexpr bool AHEAD = G < 1024 && C * (sizeof(DT) + 2 * sizeof(HT)) <= 12;
    typename Eight<HT>::vec raw_h[C], raw_dh[C];
    typename Eight<DT>::vec raw_dy[C];
    auto load = [&](int64_t row) {
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const Piece p = piece_of((c * G + lane) * 8, dim);
            raw_h[c] = load_raw((const HT*)a.h + row * a.ldh, p, dim);
            raw_dy[c] = load_raw((const DT*)a.dy + row * a.ldy, p, dim);
            if (a.dh && AHEAD) raw_dh[c] = load_raw((const HT*)a.dh + row * a.ldd, p, dim);
        }
    };
    const int64_t step = (int64_t)gridDim.x * R;
    int64_t row = (int64_t)blockIdx.x * R + group;
    if (AHEAD && row < a.rows) load(row);
    for (; row < a.rows; row += step) {
        if (!AHEAD) load(row);
        float8_t h[C], dy[C], dh[C];
#pragma unroll
        for (int c = 0; c < C; ++c) {
            h[c] = __builtin_convertvector(raw_h[c], float8_t);
            dy[c] = __builtin_convertvector(raw_dy[c], float8_t);
            if (AHEAD) dh[c] = __builtin_convertvector(raw_dh[c], float8_t);
        }
        if (AHEAD && row + step < a.rows) load(row + step);
        const bool whole = dim % 8 == 0;
        auto each_of = [&](auto f) {
#pragma unroll
            for (int c = 0; c < C; ++c) {
                const Piece p = piece_of((c * G + lane) * 8, dim);
                if (!HELD) w[c] = weight(c);
                if (whole) {
                    if (p.first == 0)
#pragma unroll
                        for (int i = 0; i < 8; ++i) f(h[c][i], dy[c][i] * w[c][i]);
                } else {
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        if (counts(p, i, dim)) f(h[c][i], dy[c][i] * w[c][i]);
                }
            }
        };
        Centre m;
        float g_sum, g_dot;                                              // of g and g (h - mean)
        auto first = [&](auto f) {
            float v[1] = {0.f};
            each_of([&](float x, float) { v[0] += f(x); });
            row_sums<G>(v, s_red);
            return v[0];
        };
        const float sum = first([](float x) { return x; });
        m.find(a.eps, a.inv_dim, sum, first,
               [&](auto f, float& d, float& dd) {
                   float v[4] = {0.f, 0.f, 0.f, 0.f};
                   each_of([&](float x, float g) {
                       const float t = f(x) - m.mean;
                       v[0] += t;
                       v[1] = fmaf(t, t, v[1]);
                       v[2] += g;
                       v[3] = fmaf(g, t, v[3]);
                   });
                   row_sums<G>(v, s_red);
                   d = v[0];
                   dd = v[1];
                   g_sum = v[2];
                   g_dot = v[3];
               },
               [&](auto f) {
#pragma unroll
                   for (int c = 0; c < C; ++c) h[c] = f(h[c]);
               });
        const float g_mean = g_sum * a.inv_dim, along = fmaf(-m.less, g_sum, g_dot) * m.inv * a.inv_dim, s = m.inv * m.by;
        HT* dx = (HT*)a.dx + row * a.ldx;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const Piece p = piece_of((c * G + lane) * 8, dim);
            if (!HELD) w[c] = weight(c);
            const float8_t t = m.of(h[c]);
            float8_t d = (dy[c] * w[c] - g_mean - t * along) * s;
            if (a.dh) d += AHEAD ? dh[c] : load_piece((const HT*)a.dh + row * a.ldd, p, dim);
            sums[0][c] += dy[c] * t;
            sums[1][c] += dy[c];
            if (p.first < 8) store_piece(dx, p, dim, d, a.stream);
        }
    }
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        if (!a.wants(which)) continue;
        if constexpr (R > 1) {
            // the sums of a workgroup's row groups, column by column
            __syncthreads();
#pragma unroll
            for (int c = 0; c < C; ++c)
#pragma unroll
                for (int i = 0; i < 8; ++i) s_sum[(group * C + c) * 8 * G + lane * 8 + i] = sums[which][c][i];
            __syncthreads();
            for (int j = threadIdx.x; j < 8 * C * G; j += T) {
                const Piece p = piece_of(j & ~7, dim);
                if (!counts(p, j & 7, dim)) continue;
                float v = 0.f;
#pragma unroll
                for (int g = 0; g < R; ++g) v += s_sum[g * 8 * C * G + j];
                a.leave(which, p.at + (j & 7), v);
            }
        } else {
#pragma unroll
            for (int c = 0; c < C; ++c) {
                const Piece p = piece_of((c * G + lane) * 8, dim);
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (counts(p, i, dim)) a.leave(which, p.at + i, sums[which][c][i]);
            }
        }
    }
}

template <typename DT, typename HT>
__global__ void __launch_bounds__(1024)
layer_norm_grad_long_kernel(LayerGradArgs a) {
    __shared__ float s_red[64];
    const int dim = a.dim;
    bool first_row = true;
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const HT* hr = (const HT*)a.h + row * a.ldh;
        const DT* dr = (const DT*)a.dy + row * a.ldy;
        auto pieces = [&](auto f) {
            for (int col = threadIdx.x * 8; col < dim; col += 8192) {
                const int n = min(8, dim - col);
                f(col, n, load_upto8(hr + col, n), load_upto8(dr + col, n));
            }
        };
        auto weighted = [&](float8_t dy, int col, int n) { return a.w ? dy * load_upto8(a.w, col, a.w_dtype, n) : dy; };
        float off = 0.f, by = 1.f;
        Centre m;
        float g_sum, g_dot;
        auto first = [&](auto f) {
            float v[1] = {0.f};
            pieces([&](int, int n, float8_t h, float8_t) {
#pragma unroll
                for (int i = 0; i < 8; ++i) v[0] += i < n ? f(h[i]) : 0.f;
            });
            row_sums<1024>(v, s_red);
            return v[0];
        };
        const float sum = first([](float x) { return x; });
        m.find(a.eps, a.inv_dim, sum, first,
               [&](auto f, float& d, float& dd) {
                   float v[4] = {0.f, 0.f, 0.f, 0.f};
                   pieces([&](int col, int n, float8_t h, float8_t dy) {
                       const float8_t g = weighted(dy, col, n);
#pragma unroll
                       for (int i = 0; i < 8; ++i) {
                           if (i >= n) continue;
                           const float t = f(h[i]) - m.mean;
                           v[0] += t;
                           v[1] = fmaf(t, t, v[1]);
                           v[2] += g[i];
                           v[3] = fmaf(g[i], t, v[3]);
                       }
                   });
                   row_sums<1024>(v, s_red);
                   d = v[0];
                   dd = v[1];
                   g_sum = v[2];
                   g_dot = v[3];
               },
               [&](auto f) {
                   off = f.off;
                   by = f.by;
               });
        const float g_mean = g_sum * a.inv_dim, along = fmaf(-m.less, g_sum, g_dot) * m.inv * a.inv_dim, s = m.inv * m.by;
        pieces([&](int col, int n, float8_t h, float8_t dy) {
            const float8_t t = m.of((h - off) * by);
            float8_t d = (weighted(dy, col, n) - g_mean - t * along) * s;
            if (a.dh) d += load_upto8((const HT*)a.dh + row * a.ldd + col, n);
            store_upto8((HT*)a.dx + row * a.ldx + col, d, n);
            if (!a.part) return;
            // (a thread's own columns of the partial rows, from row to row)
            float* part = a.part + (int64_t)blockIdx.x * 2 * dim + col;
            float8_t dw = dy * t, db = dy;
            if (!first_row) {
                dw += load_upto8(part, n);
                db += load_upto8(part + dim, n);
            }
            store_upto8(part, dw, n);
            store_upto8(part + dim, db, n);
        });
        first_row = false;
    }
}

// Columns of [n][2][dim] partial sums into dw and db (blockIdx.y): 32 columns to a workgroup, two to a thread (a line of 128 bytes of a row), every 64th row,
// then the threads in order.
__global__ void __launch_bounds__(1024) layer_norm_sums_kernel(const float* part, int64_t n, int32_t dim, void* dw, int32_t w_dtype, void* db, int32_t db_dtype) {
    typedef float any2_t __attribute__((ext_vector_type(2), aligned(4)));
    __shared__ float s[64][33];
    void* out = blockIdx.y ? db : dw;
    if (!out) return;
    const int col0 = blockIdx.x * 32, col = col0 + (threadIdx.x & 15) * 2, slice = threadIdx.x >> 4;
    const float* src = part + (int64_t)blockIdx.y * dim;
    float a = 0.f, b = 0.f;
    if (col + 1 < dim) {
#pragma unroll 8
        for (int64_t r = slice; r < n; r += 64) {
            const any2_t v = *reinterpret_cast<const any2_t*>(src + r * 2 * dim + col);
            a += v[0];
            b += v[1];
        }
    } else if (col < dim) {
#pragma unroll 8
        for (int64_t r = slice; r < n; r += 64) a += src[r * 2 * dim + col];
    }
    s[slice][(threadIdx.x & 15) * 2] = a;
    s[slice][(threadIdx.x & 15) * 2 + 1] = b;
    __syncthreads();
    if (threadIdx.x >= 32 || col0 + (int)threadIdx.x >= dim) return;
    float v = 0.f;
#pragma unroll
    for (int i = 0; i < 64; ++i) v += s[i][threadIdx.x];
    store_one(out, col0 + threadIdx.x, blockIdx.y ? db_dtype : w_dtype, v);
}

template <typename A, typename B> struct Kernels {
    using Norm = void (*)(LayerArgs);
    using Grad = void (*)(LayerGradArgs);
    static Norm norm(Shape s) {
        switch (s.group) {
            case 8: return layer_norm_kernel<A, B, 8, 1>;
            case 16: return layer_norm_kernel<A, B, 16, 1>;
            case 32: return layer_norm_kernel<A, B, 32, 1>;
            case 64: return s.pieces == 1 ? layer_norm_kernel<A, B, 64, 1> : layer_norm_kernel<A, B, 64, 2>;
            case 256: return s.pieces == 1 ? layer_norm_kernel<A, B, 256, 1> : layer_norm_kernel<A, B, 256, 2>;
            case 512: return layer_norm_kernel<A, B, 512, 2>;
            default: return s.pieces == 2 ? layer_norm_kernel<A, B, 1024, 2> : layer_norm_long_kernel<A, B>;
        }
    }
    static Grad grad(Shape s) {
        switch (s.group) {
            case 8: return layer_norm_grad_kernel<A, B, 8, 1>;
            case 16: return layer_norm_grad_kernel<A, B, 16, 1>;
            case 32: return layer_norm_grad_kernel<A, B, 32, 1>;
            case 64: return s.pieces == 1 ? layer_norm_grad_kernel<A, B, 64, 1> : layer_norm_grad_kernel<A, B, 64, 2>;
            case 256: return s.pieces == 1 ? layer_norm_grad_kernel<A, B, 256, 1> : layer_norm_grad_kernel<A, B, 256, 2>;
            case 512: return layer_norm_grad_kernel<A, B, 512, 2>;
            default: return s.pieces == 2 ? layer_norm_grad_kernel<A, B, 1024, 2> : layer_norm_grad_long_kernel<A, B>;
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

// Workgroups of 256 threads, as many as for the norms of lf_norm.hip; in the gradient each leaves two partial rows, where theirs leaves one.
constexpr int kNormGroups = 12 * 256, kGradGroups = 4 * 256;
unsigned grad_groups(int64_t rows, int64_t dim) {
    return std::min(workgroups(rows, shape_of(dim), kGradGroups), (unsigned)std::max<int64_t>(1, (1ll << 25) / dim));
}
// Whether a launch of one workgroup leaves dw and db itself (long rows keep them in memory meanwhile).
bool alone(int64_t rows, int64_t dim) { return shape_of(dim).pieces <= 2 && grad_groups(rows, dim) == 1; }

}  // namespace

extern "C" {

int lf_layer_norm(const lf_layer_norm_args* h_args, lf_stream_t stream) {
    LF_REQUIRE(h_args, LF_ERR_INVALID, "null argument");
    const lf_layer_norm_args& a = *h_args;
    LF_TRY(check_shape(a.rows, a.dim));
    LF_REQUIRE(is_float_dtype(a.x_dtype) && (!a.d_residual || is_float_dtype(a.residual_dtype)) && (!a.d_weight || is_float_dtype(a.weight_dtype)) &&
                   (!a.d_bias || is_float_dtype(a.bias_dtype)), LF_ERR_UNSUPPORTED, "x, residual, weight and bias are float32, bfloat16 or float16");
    LF_REQUIRE(is_float_dtype(a.y_dtype) || is_8bit_dtype(a.y_dtype), LF_ERR_UNSUPPORTED, "unknown type of y");
    LF_REQUIRE(is_8bit_dtype(a.y_dtype) == (a.d_scale != nullptr) || a.rows == 0, LF_ERR_INVALID, "8-bit rows, and only they, come with scales");
    LF_REQUIRE(a.eps >= 0.f, LF_ERR_INVALID, "eps must not be negative");
    LF_REQUIRE(!a.d_residual == !a.d_h || a.rows == 0, LF_ERR_INVALID, "the residual and h = x + residual come together");
    if (a.rows == 0) return LF_OK;
    LF_TRY(check_rows("x", a.rows, a.dim, a.d_x, a.ld_x, a.x_dtype));
    LF_TRY(check_rows("y", a.rows, a.dim, a.d_y, a.ld_y, a.y_dtype));
    if (a.d_residual) {
        LF_TRY(check_rows("residual", a.rows, a.dim, a.d_residual, a.ld_residual, a.residual_dtype));
        LF_TRY(check_rows("h", a.rows, a.dim, a.d_h, a.ld_h, a.residual_dtype));
    }
    if (a.d_weight) LF_TRY(check_rows("weight", 1, a.dim, a.d_weight, a.dim, a.weight_dtype));
    if (a.d_bias) LF_TRY(check_rows("bias", 1, a.dim, a.d_bias, a.dim, a.bias_dtype));
    const LayerArgs k{a.d_x, a.d_residual, a.d_weight, a.d_bias, a.d_y, a.d_h, a.d_scale, a.ld_x, a.ld_residual, a.ld_y, a.ld_h, a.rows, (int32_t)a.dim, a.weight_dtype,
                      a.bias_dtype, a.y_dtype, a.rows * a.dim * (dtype_bytes(a.y_dtype) + (a.d_h ? dtype_bytes(a.residual_dtype) : 0)) >= kStreamBytes, a.eps,
                      (float)(1.0 / (double)a.dim)};
    const Shape s = shape_of(a.dim);
    auto kernel = of_types(a.x_dtype, a.d_residual ? a.residual_dtype : a.x_dtype, [&](auto t) { return decltype(t)::norm(s); });
    kernel<<<workgroups(a.rows, s, kNormGroups), std::max(s.group, 256), 0, (hipStream_t)stream>>>(k);
    LF_HIP(hipGetLastError());
    return LF_OK;
}

size_t lf_layer_norm_grad_work_bytes(int64_t rows, int64_t dim) {
    if (rows <= 0 || dim < 1 || dim > kMaxDim || alone(rows, dim)) return 0;
    return (size_t)grad_groups(rows, dim) * 2 * (size_t)dim * sizeof(float);
}

int lf_layer_norm_grad(const lf_layer_norm_grad_args* h_args, void* d_work, size_t work_bytes, lf_stream_t stream) {
    LF_REQUIRE(h_args, LF_ERR_INVALID, "null argument");
    const lf_layer_norm_grad_args& a = *h_args;
    LF_TRY(check_shape(a.rows, a.dim));
    LF_REQUIRE(is_float_dtype(a.dy_dtype) && is_float_dtype(a.h_dtype) && ((!a.d_weight && !a.d_dw) || is_float_dtype(a.weight_dtype)) &&
                   (!a.d_db || is_float_dtype(a.db_dtype)), LF_ERR_UNSUPPORTED, "dy, h, weight and db are float32, bfloat16 or float16");
    LF_REQUIRE(a.eps >= 0.f, LF_ERR_INVALID, "eps must not be negative");
    const Shape s = shape_of(a.dim);
    const unsigned groups = a.rows ? grad_groups(a.rows, a.dim) : 0;
    const bool sums = a.d_dw || a.d_db, one = a.rows && alone(a.rows, a.dim);
    if (a.d_dw) LF_TRY(check_rows("dw", 1, a.dim, a.d_dw, a.dim, a.weight_dtype));
    if (a.d_db) LF_TRY(check_rows("db", 1, a.dim, a.d_db, a.dim, a.db_dtype));
    if (sums) {
        LF_REQUIRE(a.rows == 0 || one || (d_work && (uintptr_t)d_work % 16 == 0), LF_ERR_INVALID, "null or unaligned workspace");
        LF_REQUIRE(work_bytes >= lf_layer_norm_grad_work_bytes(a.rows, a.dim), LF_ERR_WORKSPACE, "workspace of %zu bytes, %zu are needed", work_bytes,
                   lf_layer_norm_grad_work_bytes(a.rows, a.dim));
    }
    hipStream_t st = (hipStream_t)stream;
    if (a.rows) {
        LF_TRY(check_rows("dy", a.rows, a.dim, a.d_dy, a.ld_dy, a.dy_dtype));
        LF_TRY(check_rows("h", a.rows, a.dim, a.d_h, a.ld_h, a.h_dtype));
        LF_TRY(check_rows("dx", a.rows, a.dim, a.d_dx, a.ld_dx, a.h_dtype));
        if (a.d_dh) LF_TRY(check_rows("dh", a.rows, a.dim, a.d_dh, a.ld_dh, a.h_dtype));
        if (a.d_weight) LF_TRY(check_rows("weight", 1, a.dim, a.d_weight, a.dim, a.weight_dtype));
        const LayerGradArgs k{a.d_dy, a.d_h, a.d_weight, a.d_dh, a.d_dx, sums && !one ? (float*)d_work : nullptr, a.d_dw, a.d_db, a.ld_dy, a.ld_h, a.ld_dh, a.ld_dx, a.rows,
                              (int32_t)a.dim, a.weight_dtype, a.db_dtype, a.rows * a.dim * dtype_bytes(a.h_dtype) >= kStreamBytes, a.eps, (float)(1.0 / (double)a.dim)};
        auto kernel = of_types(a.dy_dtype, a.h_dtype, [&](auto t) { return decltype(t)::grad(s); });
        kernel<<<groups, std::max(s.group, 256), 0, st>>>(k);
        LF_HIP(hipGetLastError());
    }
    if (sums && !one) {
        layer_norm_sums_kernel<<<dim3((unsigned)ceil_div(a.dim, 32), 2), 1024, 0, st>>>((const float*)d_work, groups, (int32_t)a.dim, a.d_dw, a.weight_dtype, a.d_db,
                                                                                        a.db_dtype);
        LF_HIP(hipGetLastError());
    }
    return LF_OK;
}

}  // extern "C"
