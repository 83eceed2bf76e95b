// lf_linear and lf_linear_grad: what is launched for a product, and the kernels around the tiled ones of lf_product.h - few rows,
// the joining of partial sums, the gradient of the activation.
#include "lf_product.h"

namespace {

// The splits' partial sums in order, and the epilogue: SLICES threads share the splits of eight outputs, and their sums are added in order.
template <typename A, int SLICES>
__global__ void __launch_bounds__(256) join_kernel(const A* part, int64_t m, int64_t n, int32_t splits, Epilogue e) {
    constexpr int UNITS = 256 / SLICES;
    __shared__ A s_sum[SLICES][UNITS][9];
    const int64_t across = (n + 7) / 8, u = (int64_t)blockIdx.x * UNITS + threadIdx.x % UNITS;
    const int slice = threadIdx.x / UNITS;
    const int64_t row = u / across, col = (u % across) * 8;
    const int count = row < m ? (int)min((int64_t)8, n - col) : 0;
    A sum[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    struct __attribute__((packed, aligned(4))) Any { A v[8]; };
    const A* src = part + row * n + col;
    if (count == 8) {
#pragma unroll 4
        for (int s = slice; s < splits; s += SLICES) {
            const Any v = *reinterpret_cast<const Any*>(src + (int64_t)s * m * n);
#pragma unroll
            for (int i = 0; i < 8; ++i) sum[i] += v.v[i];
        }
    } else if (count > 0) {
#pragma unroll 2
        for (int s = slice; s < splits; s += SLICES)
#pragma unroll
            for (int i = 0; i < 8; ++i) sum[i] += src[(int64_t)s * m * n + min(i, count - 1)];
    }
    if constexpr (SLICES > 1) {
#pragma unroll
        for (int i = 0; i < 8; ++i) s_sum[slice][threadIdx.x % UNITS][i] = sum[i];
        __syncthreads();
        // all threads add up some slices of an output, then the first ones their sums
        constexpr int OUT = UNITS * 8, PARTS = 256 / OUT, EACH = SLICES / PARTS;
        const int o = threadIdx.x % OUT, first = threadIdx.x / OUT * EACH;
        A t = s_sum[first][o / 8][o % 8];
#pragma unroll
        for (int i = 1; i < EACH; ++i) t += s_sum[first + i][o / 8][o % 8];
        __syncthreads();
        s_sum[first][o / 8][o % 8] = t;
        __syncthreads();
        if (slice) return;
#pragma unroll
        for (int i = 0; i < 8; ++i) sum[i] = s_sum[0][threadIdx.x][i];
#pragma unroll
        for (int p = 1; p < PARTS; ++p)
#pragma unroll
            for (int i = 0; i < 8; ++i) sum[i] += s_sum[p * EACH][threadIdx.x][i];
    }
    if (count == 0) return;
    float8_t v;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = (float)sum[i];
    finish(e, row, col, count, v);
}
template <typename A> int launch_join(const Product& g, hipStream_t st) {
    const int slices = g.splits <= 4 ? 1 : g.splits <= 32 ? 8 : g.splits <= 128 ? 32 : 64;
    const int64_t groups = ceil_div(g.m * ceil_div(g.n, 8), 256 / slices);
    LF_REQUIRE(groups < (1ll << 31), LF_ERR_UNSUPPORTED, "too many outputs");
    auto kernel = slices == 1 ? join_kernel<A, 1> : slices == 8 ? join_kernel<A, 8> : slices == 32 ? join_kernel<A, 32> : join_kernel<A, 64>;
    kernel<<<(unsigned)groups, 256, 0, st>>>((const A*)g.part, g.m, g.n, g.splits, g.e);
    LF_HIP(hipGetLastError());
    return LF_OK;
}

// ---------------------------------------------------------------------------- few rows

// Up to 16 rows of X: a workgroup takes 16 rows of W, its wavefronts the 128-byte steps of k in turn, and their sums
// meet in LDS.  W goes from memory into the matrix instructions' registers, 32 consecutive bytes a lane and step.  Bound by the
// read of W, small ones by the launch: one row, bf16 W of 8192^2 29 us (4.6 TB/s), of 4096^2 9.4 (3.6); 13 rows, int8 W of 1001 x 4000 6.
// Gated: eight rows of each half, so that a workgroup reads as much as one of 16 outputs does; one row, bf16 of 2 x 8192 x 4096 from memory 26 - 28 us (4.8 - 5.2 TB/s),
// with 16 rows of each half, half as many workgroups of more registers, 31.  16 rows take 39 (36 so): X comes from L2 for every workgroup.
template <typename T, int WAVES, bool GATED>
__global__ void __launch_bounds__(64 * WAVES)
few_rows_kernel(Product g) {
    constexpr int KS = 128 / sizeof(T), MINE = 32 / sizeof(T), E = 16 / sizeof(T), OUT = GATED ? 8 : 16;
    using Acc = typename Elem<T>::Acc;
    using S = std::conditional_t<std::is_same_v<Acc, int4v>, int32_t, float>;
    __shared__ S s_sum[WAVES][16][17];
    const int lane = threadIdx.x & 63, li = lane & 15, lg = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t n0 = (int64_t)blockIdx.x * OUT, row = GATED ? (li >> 3) * g.n + min(n0 + (li & 7), g.n - 1) : min(n0 + li, g.n - 1);
    const T* w = (const T*)g.q + row * g.ld_q + lg * MINE;
    const bool on = li < g.m;
    const T* x = (const T*)g.p + (on ? li : 0) * g.ld_p + lg * MINE;
    Acc acc = {0, 0, 0, 0};
    auto multiply = [&](const uint4_t (&a)[2], const uint4_t (&b)[2]) {
        if constexpr (std::is_same_v<T, float>) {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                acc = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a[i >> 2][i & 3]), __uint_as_float(b[i >> 2][i & 3]), acc, 0, 0, 0);
        } else if constexpr (std::is_same_v<T, e4m3_t>) {
            acc = mma_e4m3(a[0], a[1], b[0], b[1], acc);
        } else {
            acc = mma(a[0], b[0], acc, T{});
            acc = mma(a[1], b[1], acc, T{});
        }
    };
    constexpr int U = 4;                                        // steps under way at once
    const int64_t steps = g.k / KS;
    int64_t s = wave;
    for (; s + (U - 1) * WAVES < steps; s += U * WAVES) {
        uint4_t a[U][2], b[U][2];
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                a[u][h] = load16(w + (s + u * WAVES) * KS + h * E);
                b[u][h] = uint4_t{0u, 0u, 0u, 0u};
                if (on) b[u][h] = load16(x + (s + u * WAVES) * KS + h * E);
            }
#pragma unroll
        for (int u = 0; u < U; ++u) multiply(a[u], b[u]);
    }
    for (; s < steps + (g.k % KS != 0); s += WAVES) {
        uint4_t a[2], b[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int left = (int)min((int64_t)E, g.k - s * KS - lg * MINE - h * E);
            a[h] = load16_each(w + s * KS + h * E, left);
            b[h] = load16_each(x + s * KS + h * E, on ? left : 0);
        }
        multiply(a, b);
    }
#pragma unroll
    for (int v = 0; v < 4; ++v) s_sum[wave][li][lg * 4 + v] = acc[v];
    __syncthreads();
    const int m = threadIdx.x >> 1, half = threadIdx.x & 1;
    if (m >= g.m || (!GATED && n0 + half * 8 >= g.n)) return;
    float8_t out[2];                                            // (gated: the gate's, from the first of the two threads, and the other half's)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        S t = 0;
#pragma unroll
        for (int u = 0; u < WAVES; ++u) t += s_sum[u][m][half * 8 + i];
        out[0][i] = (float)t;
        if constexpr (GATED) out[1][i] = __shfl_xor(out[0][i], 1);
    }
    if constexpr (GATED) {
        if (!half) finish_gated(g.e, m, n0, g.n, (int)min((int64_t)8, g.n - n0), out);
    } else {
        finish(g.e, m, n0 + half * 8, (int)min((int64_t)8, g.n - n0 - half * 8), out[0]);
    }
}

// ---------------------------------------------------------------------------- gradient of the activation

// dz = dy act'(z), in rows of `ld_dz` elements, and the column sums of a slab of rows (before rounding): ACROSS threads of eight columns
// each, the others take further rows.  A single slab's sums are db.
template <typename T, int ACROSS>
__global__ void __launch_bounds__(256)
activation_grad_kernel(const T* dy, int64_t ld_dy, const T* z, int64_t ld_z, T* dz, int64_t ld_dz, float* part, void* db, int32_t db_dtype, int64_t m, int64_t n,
                       int32_t act, int64_t slab) {
    constexpr int DOWN = 256 / ACROSS;
    __shared__ float s[DOWN][ACROSS][9];
    const int lx = threadIdx.x % ACROSS, ly = threadIdx.x / ACROSS;
    const int64_t col = ((int64_t)blockIdx.x * ACROSS + lx) * 8;
    const int count = (int)min((int64_t)8, n - col);
    const int64_t r1 = min(m, ((int64_t)blockIdx.y + 1) * slab);
    float8_t sum = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (count > 0)
#pragma unroll 2
        for (int64_t r = (int64_t)blockIdx.y * slab + ly; r < r1; r += DOWN) {
            float8_t d = load_upto8(dy + r * ld_dy + col, count);
            if (act != LF_ACT_NONE) {
                const float8_t v = load_upto8(z + r * ld_z + col, count);
#pragma unroll
                for (int i = 0; i < 8; ++i) d[i] *= activate_grad<std::is_same_v<T, float>>(v[i], act);
            }
            if (dz) store_upto8(dz + r * ld_dz + col, d, count);
            sum += d;
        }
    if (!part && !db) return;
#pragma unroll
    for (int i = 0; i < 8; ++i) s[ly][lx][i] = sum[i];
    __syncthreads();
    const int64_t c = (int64_t)blockIdx.x * ACROSS * 8 + threadIdx.x;
    if (threadIdx.x >= ACROSS * 8 || c >= n) return;
    float t = 0.f;
#pragma unroll
    for (int i = 0; i < DOWN; ++i) t += s[i][threadIdx.x >> 3][threadIdx.x & 7];
    if (part) part[(int64_t)blockIdx.y * n + c] = t;
    else store_one(db, c, db_dtype, t);
}

// ---------------------------------------------------------------------------- gate

// join_kernel of a gated product: the splits' partial sums [splits][m][2 n] in order, and its epilogue.
template <typename A, int SLICES>
__global__ void __launch_bounds__(256) gated_join_kernel(const A* part, int64_t m, int64_t n, int32_t splits, Epilogue e) {
    constexpr int UNITS = 256 / SLICES;
    __shared__ A s_sum[2][SLICES][UNITS][9];
    const int64_t across = (n + 7) / 8, u = (int64_t)blockIdx.x * UNITS + threadIdx.x % UNITS;
    const int slice = threadIdx.x / UNITS;
    const int64_t row = u / across, col = (u % across) * 8;
    const int count = row < m ? (int)min((int64_t)8, n - col) : 0;
    A sum[2][8] = {};
    struct __attribute__((packed, aligned(4))) Any { A v[8]; };
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const A* src = part + row * 2 * n + h * n + col;
        if (count == 8) {
#pragma unroll 4
            for (int s = slice; s < splits; s += SLICES) {
                const Any v = *reinterpret_cast<const Any*>(src + (int64_t)s * m * 2 * n);
#pragma unroll
                for (int i = 0; i < 8; ++i) sum[h][i] += v.v[i];
            }
        } else if (count > 0) {
#pragma unroll 2
            for (int s = slice; s < splits; s += SLICES)
#pragma unroll
                for (int i = 0; i < 8; ++i) sum[h][i] += src[(int64_t)s * m * 2 * n + min(i, count - 1)];
        }
    }
    if constexpr (SLICES > 1) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < 8; ++i) s_sum[h][slice][threadIdx.x % UNITS][i] = sum[h][i];
        __syncthreads();
        // a thread adds up the slices of some outputs
        constexpr int OUT = 2 * UNITS * 8;
        for (int o = threadIdx.x; o < OUT; o += 256) {
            const int h = o / (UNITS * 8), unit = o / 8 % UNITS, i = o % 8;
            A t = s_sum[h][0][unit][i];
#pragma unroll
            for (int v = 1; v < SLICES; ++v) t += s_sum[h][v][unit][i];
            s_sum[h][0][unit][i] = t;
        }
        __syncthreads();
        if (slice) return;
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < 8; ++i) sum[h][i] = s_sum[h][0][threadIdx.x][i];
    }
    if (count == 0) return;
    float8_t v[2];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 8; ++i) v[h][i] = (float)sum[h][i];
    finish_gated(e, row, col, n, count, v);
}
template <typename A> int launch_gated_join(const Product& g, hipStream_t st) {
    const int slices = g.splits <= 4 ? 1 : g.splits <= 32 ? 8 : 32;
    const int64_t groups = ceil_div(g.m * ceil_div(g.n, 8), 256 / slices);
    LF_REQUIRE(groups < (1ll << 31), LF_ERR_UNSUPPORTED, "too many outputs");
    auto kernel = slices == 1 ? gated_join_kernel<A, 1> : slices == 8 ? gated_join_kernel<A, 8> : gated_join_kernel<A, 32>;
    kernel<<<(unsigned)groups, 256, 0, st>>>((const A*)g.part, g.m, g.n, g.splits, g.e);
    LF_HIP(hipGetLastError());
    return LF_OK;
}

// dz = [dy u act'(g) | dy act(g)] of z = [g | u], in rows of `ld_dz`, and the column sums of a slab of rows, as activation_grad_kernel has them.
// Bound by memory: bf16 8192 x 4096 67 us (335 MB at 5.0 TB/s), float32 57,001 x 200 50 (228 MB at 4.6).  dz is rounded to the operands' type, since the products
// take it so.
template <typename T, int ACROSS>
__global__ void __launch_bounds__(256)
gate_grad_kernel(const T* dy, int64_t ld_dy, const T* z, int64_t ld_z, T* dz, int64_t ld_dz, float* part, void* db, int32_t db_dtype, int64_t m, int64_t n, int32_t act,
                 int64_t slab) {
    constexpr int DOWN = 256 / ACROSS;
    constexpr bool FINE = std::is_same_v<T, float>;
    __shared__ float s[DOWN][ACROSS][9];
    const int lx = threadIdx.x % ACROSS, ly = threadIdx.x / ACROSS;
    const int64_t col = ((int64_t)blockIdx.x * ACROSS + lx) * 8;
    const int count = (int)min((int64_t)8, n - col);
    const int64_t r1 = min(m, ((int64_t)blockIdx.y + 1) * slab);
    float8_t sum[2];
    sum[0] = sum[1] = float8_t{0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (count > 0)
#pragma unroll 2
        for (int64_t r = (int64_t)blockIdx.y * slab + ly; r < r1; r += DOWN) {
            const float8_t d = load_upto8(dy + r * ld_dy + col, count), g = load_upto8(z + r * ld_z + col, count), u = load_upto8(z + r * ld_z + n + col, count);
            const float8_t du = d * activate(g, activation_of(act, FINE ? LF_DTYPE_F32 : LF_DTYPE_BF16));
            float8_t dg = d * u;
#pragma unroll
            for (int i = 0; i < 8; ++i) dg[i] *= activate_grad<FINE>(g[i], act);
            store_upto8(dz + r * ld_dz + col, dg, count);
            store_upto8(dz + r * ld_dz + n + col, du, count);
            sum[0] += dg;
            sum[1] += du;
        }
    if (!part && !db) return;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 8; ++i) s[ly][lx][i] = sum[h][i];
        __syncthreads();
        const int64_t c = (int64_t)blockIdx.x * ACROSS * 8 + threadIdx.x;
        if (threadIdx.x >= ACROSS * 8 || c >= n) continue;
        float t = 0.f;
#pragma unroll
        for (int i = 0; i < DOWN; ++i) t += s[i][threadIdx.x >> 3][threadIdx.x & 7];
        if (part) part[((int64_t)blockIdx.y * 2 + h) * n + c] = t;
        else store_one(db, h * n + c, db_dtype, t);
    }
}

// ---------------------------------------------------------------------------- launches

ProductFn product_of(int32_t dtype, bool px, bool qx, int tile, bool aligned, bool deep) {
    switch (dtype) {
        case LF_DTYPE_F32: return product_f32(px, qx, tile, aligned, deep);
        case LF_DTYPE_BF16: return product_bf16(px, qx, tile, aligned, deep);
        case LF_DTYPE_F16: return product_f16(px, qx, tile, aligned, deep);
        case LF_DTYPE_E4M3: return product_e4m3(px, qx, tile, aligned, deep);
        default: return product_i8(px, qx, tile, aligned, deep);
    }
}
ProductFn gated_of(int32_t dtype, int tile, bool aligned, bool deep) {
    switch (dtype) {
        case LF_DTYPE_F32: return gated_f32(tile, aligned, deep);
        case LF_DTYPE_BF16: return gated_bf16(tile, aligned, deep);
        case LF_DTYPE_F16: return gated_f16(tile, aligned, deep);
        case LF_DTYPE_E4M3: return gated_e4m3(tile, aligned, deep);
        default: return gated_i8(tile, aligned, deep);
    }
}
template <int WAVES, bool GATED> ProductFn few_rows_of(int32_t dtype) {
    switch (dtype) {
        case LF_DTYPE_F32: return few_rows_kernel<float, WAVES, GATED>;
        case LF_DTYPE_BF16: return few_rows_kernel<__bf16, WAVES, GATED>;
        case LF_DTYPE_F16: return few_rows_kernel<_Float16, WAVES, GATED>;
        case LF_DTYPE_E4M3: return few_rows_kernel<e4m3_t, WAVES, GATED>;
        default: return few_rows_kernel<int8_t, WAVES, GATED>;
    }
}

// gated: g.n outputs, of 2 g.n rows of Q
int launch_product(Product g, int32_t dtype, bool px, bool qx, void* work, hipStream_t st, bool gated = false) {
    if (g.m == 0 || g.n == 0) return LF_OK;
    const int64_t q_rows = gated ? 2 * g.n : g.n;
    g.e.stream = g.m * (g.n * dtype_bytes(g.e.y_dtype) + (gated && g.e.z ? q_rows * dtype_bytes(g.e.z_dtype) : 0)) >= kStreamBytes;
    const Path path = path_of(dtype_bytes(dtype), {g.p, g.ld_p, g.m, px}, {g.q, g.ld_q, q_rows, qx}, g.k);
    if (path.kernel == kPathFewRows) {
        const int64_t groups = ceil_div(g.n, gated ? 8 : 16);
        LF_REQUIRE(groups < (1ll << 31), LF_ERR_UNSUPPORTED, "too many columns");
        // few workgroups take 16 wavefronts each
        if (groups <= 256) (gated ? few_rows_of<16, true>(dtype) : few_rows_of<16, false>(dtype))<<<(unsigned)groups, 1024, 0, st>>>(g);
        else (gated ? few_rows_of<8, true>(dtype) : few_rows_of<8, false>(dtype))<<<(unsigned)groups, 512, 0, st>>>(g);
        LF_HIP(hipGetLastError());
        return LF_OK;
    }
    const Cut& c = path.cut;
    const int64_t tm = ceil_div(g.m, c.tile), tn = ceil_div(q_rows, c.tile);
    LF_REQUIRE(tm < (1ll << 27) && tn < (1ll << 27) && tm * tn < (1ll << 31), LF_ERR_UNSUPPORTED, "too many tiles");
    g.tiles_m = (int32_t)tm;
    g.tiles_n = (int32_t)tn;
    g.splits = c.splits;
    g.k_split = c.k_split;
    g.part = c.splits > 1 ? work : nullptr;
    const bool aligned = path.kernel != kPathProduct;
    (gated ? gated_of(dtype, c.tile, aligned, path.deep) : product_of(dtype, px, qx, c.tile, aligned, path.deep))<<<dim3((unsigned)(tm * tn), (unsigned)c.splits), 256, 0, st>>>(g);
    LF_HIP(hipGetLastError());
    if (c.splits == 1) return LF_OK;
    if (gated) return dtype == LF_DTYPE_I8 ? launch_gated_join<int32_t>(g, st) : launch_gated_join<float>(g, st);
    return dtype == LF_DTYPE_I8 ? launch_join<int32_t>(g, st) : launch_join<float>(g, st);
}

constexpr int64_t kMostRows = 1ll << 40, kMostFeatures = 1ll << 24;

int check_matrix(const char* what, const void* p, int64_t rows, int64_t cols, int64_t ld, int32_t dtype) {
    LF_REQUIRE(p || rows == 0 || cols == 0, LF_ERR_INVALID, "%s: null pointer", what);
    LF_REQUIRE(ld >= cols || rows <= 1, LF_ERR_INVALID, "%s: rows of %lld elements, %lld apart", what, (long long)cols, (long long)ld);
    LF_REQUIRE((uintptr_t)p % dtype_bytes(dtype) == 0, LF_ERR_INVALID, "%s: not aligned to its elements", what);
    return LF_OK;
}
int check_sizes(int64_t m, int64_t n, int64_t k, int32_t dtype, int32_t act) {
    LF_REQUIRE(m >= 0 && n >= 0 && k >= 0, LF_ERR_INVALID, "negative size");
    LF_REQUIRE(m < kMostRows && n <= kMostFeatures && k <= kMostFeatures, LF_ERR_UNSUPPORTED, "a product of %lld x %lld x %lld", (long long)m, (long long)n,
               (long long)k);
    LF_REQUIRE(is_float_dtype(dtype) || is_8bit_dtype(dtype), LF_ERR_UNSUPPORTED, "unknown type");
    LF_REQUIRE(act >= LF_ACT_NONE && act <= LF_ACT_SILU, LF_ERR_UNSUPPORTED, "unknown activation");
    LF_REQUIRE(dtype != LF_DTYPE_I8 || k < (1 << 17), LF_ERR_UNSUPPORTED, "int8 sums of %lld products do not fit 32 bits", (long long)k);
    return LF_OK;
}

// Rows of a gated weight; sizes that are refused stay as they are (twice INT64_MIN would be 0).
int64_t both_halves(int64_t n) { return n < 0 || n > kMostFeatures ? n : 2 * n; }

// Rows of dz are padded to a multiple of 16 bytes.
int64_t ld_dz(int64_t n) { return ceil_div(n, 8) * 8; }
size_t padded(size_t bytes) { return (bytes + 255) / 256 * 256; }
// Threads across a row (of eight columns each), and slabs of rows whose column sums are kept apart: enough workgroups to fill the GPU.
int threads_across(int64_t n) { return n <= 64 ? 8 : n <= 128 ? 16 : 32; }
int64_t slabs_of(int64_t m, int64_t n) {
    return std::max<int64_t>(1, std::min(ceil_div(m, 64), ceil_div(512, std::clamp<int64_t>(ceil_div(n, 256), 1, 4))));
}

struct GradWork { size_t dz, sums, parts, total; };
GradWork grad_work(int64_t m, int64_t n, int64_t k, int32_t dtype, int32_t act, bool dx, bool dw, bool db) {
    GradWork w{0, 0, 0, 0};
    if (act != LF_ACT_NONE) w.dz = padded((size_t)m * (size_t)ld_dz(n) * dtype_bytes(dtype));
    if (db && slabs_of(m, n) > 1) w.sums = padded((size_t)slabs_of(m, n) * (size_t)n * 4);
    if (dx && m && k) w.parts = cut_product(dtype_bytes(dtype), m, k, n).bytes;
    if (dw && n && k) w.parts = std::max(w.parts, cut_product(dtype_bytes(dtype), n, k, m).bytes);
    w.total = w.dz + w.sums + w.parts;
    return w;
}

// Of the gated product, whose dz has 2 n columns.
GradWork gated_work(int64_t m, int64_t n, int64_t k, int32_t dtype, bool dx, bool dw, bool db) {
    GradWork w = grad_work(m, 2 * n, k, dtype, LF_ACT_SILU, dx, dw, false);
    if (db && slabs_of(m, n) > 1) w.sums = padded((size_t)slabs_of(m, n) * 2 * (size_t)n * 4);
    w.total += w.sums;
    return w;
}

// dx = dz w and dw = dz^T x for dz of `n` columns.
int two_products(const lf_linear_grad_args& a, int64_t n, const void* dz, int64_t ld, void* parts, hipStream_t st) {
    if (a.d_dx) {
        Product g{};
        g.p = dz; g.ld_p = ld; g.q = a.d_w; g.ld_q = a.ld_w; g.m = a.m; g.n = a.k; g.k = n;
        g.e.y = a.d_dx; g.e.ld_y = a.ld_dx; g.e.y_dtype = a.dtype;
        LF_TRY(launch_product(g, a.dtype, false, true, parts, st));
    }
    if (a.d_dw) {
        Product g{};
        g.p = dz; g.ld_p = ld; g.q = a.d_x; g.ld_q = a.ld_x; g.m = n; g.n = a.k; g.k = a.m;
        g.e.y = a.d_dw; g.e.ld_y = a.ld_dw; g.e.y_dtype = a.dtype;
        LF_TRY(launch_product(g, a.dtype, true, true, parts, st));
    }
    return LF_OK;
}

}  // namespace

extern "C" {

size_t lf_linear_work_bytes(int64_t m, int64_t n, int64_t k, int32_t dtype) {
    if (m <= kFewRows || n <= 0 || k <= 0 || !(is_float_dtype(dtype) || is_8bit_dtype(dtype))) return 0;
    return cut_product(dtype_bytes(dtype), m, n, k).bytes;
}

int lf_linear(const lf_linear_args* h_args, void* d_work, size_t work_bytes, lf_stream_t stream) {
    LF_REQUIRE(h_args, LF_ERR_INVALID, "null argument");
    const lf_linear_args& a = *h_args;
    LF_TRY(check_sizes(a.m, a.n, a.k, a.dtype, a.activation));
    LF_REQUIRE(is_float_dtype(a.y_dtype) && (!a.d_bias || is_float_dtype(a.bias_dtype)) && (!a.d_residual || is_float_dtype(a.residual_dtype)) &&
                   (!a.d_z || is_float_dtype(a.z_dtype)), LF_ERR_UNSUPPORTED, "y, z, bias and residual are float32, bfloat16 or float16");
    if (a.m == 0 || a.n == 0) return LF_OK;
    LF_TRY(check_matrix("x", a.d_x, a.m, a.k, a.ld_x, a.dtype));
    LF_TRY(check_matrix("w", a.d_w, a.n, a.k, a.ld_w, a.dtype));
    LF_TRY(check_matrix("y", a.d_y, a.m, a.n, a.ld_y, a.y_dtype));
    if (a.d_residual) LF_TRY(check_matrix("residual", a.d_residual, a.m, a.n, a.ld_residual, a.residual_dtype));
    if (a.d_z) LF_TRY(check_matrix("z", a.d_z, a.m, a.n, a.ld_z, a.z_dtype));
    if (a.d_bias) LF_TRY(check_matrix("bias", a.d_bias, 1, a.n, a.n, a.bias_dtype));
    LF_REQUIRE(!a.d_x_scale == !a.d_w_scale && is_8bit_dtype(a.dtype) == (a.d_x_scale != nullptr), LF_ERR_INVALID, "8-bit operands, and only they, come with scales");
    const size_t need = lf_linear_work_bytes(a.m, a.n, a.k, a.dtype);
    LF_REQUIRE(need == 0 || (d_work && (uintptr_t)d_work % 16 == 0), LF_ERR_INVALID, "null or unaligned workspace");
    LF_REQUIRE(work_bytes >= need, LF_ERR_WORKSPACE, "workspace of %zu bytes, %zu are needed", work_bytes, need);
    Product g{};
    g.p = a.d_x; g.q = a.d_w; g.ld_p = a.ld_x; g.ld_q = a.ld_w; g.m = a.m; g.n = a.n; g.k = a.k;
    g.e = Epilogue{a.d_y, a.d_residual, a.d_z, a.d_bias, a.d_x_scale, a.d_w_scale, a.ld_y, a.ld_residual, a.ld_z, a.y_dtype, a.residual_dtype, a.z_dtype,
                   a.bias_dtype, activation_of(a.activation, a.y_dtype)};
    return launch_product(g, a.dtype, false, false, d_work, (hipStream_t)stream);
}

size_t lf_linear_grad_work_bytes(int64_t m, int64_t n, int64_t k, int32_t dtype, int32_t activation, int32_t want_dx, int32_t want_dw, int32_t want_db) {
    if (m < 0 || n < 0 || k < 0 || !is_float_dtype(dtype)) return 0;
    return grad_work(m, n, k, dtype, activation, want_dx, want_dw, want_db).total;
}

int lf_linear_grad(const lf_linear_grad_args* h_args, void* d_work, size_t work_bytes, lf_stream_t stream) {
    LF_REQUIRE(h_args, LF_ERR_INVALID, "null argument");
    const lf_linear_grad_args& a = *h_args;
    LF_TRY(check_sizes(a.m, a.n, a.k, a.dtype, a.activation));
    LF_REQUIRE(is_float_dtype(a.dtype) && (!a.d_db || is_float_dtype(a.db_dtype)), LF_ERR_UNSUPPORTED, "gradients are of float32, bfloat16 or float16");
    LF_REQUIRE((a.activation == LF_ACT_NONE) || a.d_z || a.m == 0 || a.n == 0, LF_ERR_INVALID, "the activation's gradient needs z");
    LF_TRY(check_matrix("dy", a.d_dy, a.m, a.n, a.ld_dy, a.dtype));
    if (a.activation != LF_ACT_NONE) LF_TRY(check_matrix("z", a.d_z, a.m, a.n, a.ld_z, a.dtype));
    if (a.d_dw) {
        LF_TRY(check_matrix("x", a.d_x, a.m, a.k, a.ld_x, a.dtype));
        LF_TRY(check_matrix("dw", a.d_dw, a.n, a.k, a.ld_dw, a.dtype));
    }
    if (a.d_dx) {
        LF_TRY(check_matrix("w", a.d_w, a.n, a.k, a.ld_w, a.dtype));
        LF_TRY(check_matrix("dx", a.d_dx, a.m, a.k, a.ld_dx, a.dtype));
    }
    if (a.d_db) LF_TRY(check_matrix("db", a.d_db, 1, a.n, a.n, a.db_dtype));
    if (a.n == 0 && a.k == 0) return LF_OK;
    const GradWork w = grad_work(a.m, a.n, a.k, a.dtype, a.activation, a.d_dx, a.d_dw, a.d_db);
    LF_REQUIRE(w.total == 0 || (d_work && (uintptr_t)d_work % 16 == 0), LF_ERR_INVALID, "null or unaligned workspace");
    LF_REQUIRE(work_bytes >= w.total, LF_ERR_WORKSPACE, "workspace of %zu bytes, %zu are needed", work_bytes, w.total);
    hipStream_t st = (hipStream_t)stream;
    char* at = (char*)d_work;
    void* dz = w.dz ? at : nullptr;
    float* sums = w.sums ? (float*)(at + w.dz) : nullptr;
    void* parts = at + w.dz + w.sums;
    const int64_t slabs = slabs_of(a.m, a.n), slab = ceil_div(std::max<int64_t>(a.m, 1), slabs);
    if ((dz || a.d_db) && a.n > 0) {
        const int across = threads_across(a.n);
        const dim3 grid((unsigned)ceil_div(a.n, 8 * across), (unsigned)slabs);
        auto go = [&](auto t) {
            using T = decltype(t);
            auto kernel = across == 8 ? activation_grad_kernel<T, 8> : across == 16 ? activation_grad_kernel<T, 16> : activation_grad_kernel<T, 32>;
            kernel<<<grid, 256, 0, st>>>((const T*)a.d_dy, a.ld_dy, (const T*)a.d_z, a.ld_z, (T*)dz, ld_dz(a.n), sums, sums ? nullptr : a.d_db, a.db_dtype, a.m, a.n, a.activation, slab);
        };
        if (a.dtype == LF_DTYPE_F32) go(0.f); else if (a.dtype == LF_DTYPE_BF16) go((__bf16)0.f); else go((_Float16)0.f);
        LF_HIP(hipGetLastError());
        if (sums) LF_TRY(lf::column_sums(sums, slabs, a.n, a.d_db, a.db_dtype, st));
    }
    return two_products(a, a.n, dz ? dz : a.d_dy, dz ? ld_dz(a.n) : a.ld_dy, parts, st);
}

size_t lf_gated_linear_work_bytes(int64_t m, int64_t n, int64_t k, int32_t dtype) {
    return n > kMostFeatures ? 0 : lf_linear_work_bytes(m, both_halves(n), k, dtype);
}

int lf_gated_linear(const lf_linear_args* h_args, void* d_work, size_t work_bytes, lf_stream_t stream) {
    LF_REQUIRE(h_args, LF_ERR_INVALID, "null argument");
    const lf_linear_args& a = *h_args;
    LF_TRY(check_sizes(a.m, both_halves(a.n), a.k, a.dtype, a.activation));
    LF_REQUIRE(is_float_dtype(a.y_dtype) && (!a.d_bias || is_float_dtype(a.bias_dtype)) && (!a.d_z || is_float_dtype(a.z_dtype)), LF_ERR_UNSUPPORTED,
               "y, z and bias are float32, bfloat16 or float16");
    LF_REQUIRE(!a.d_residual, LF_ERR_INVALID, "a gated product has no residual");
    if (a.m == 0 || a.n == 0) return LF_OK;
    LF_TRY(check_matrix("x", a.d_x, a.m, a.k, a.ld_x, a.dtype));
    LF_TRY(check_matrix("w", a.d_w, 2 * a.n, a.k, a.ld_w, a.dtype));
    LF_TRY(check_matrix("y", a.d_y, a.m, a.n, a.ld_y, a.y_dtype));
    if (a.d_z) LF_TRY(check_matrix("z", a.d_z, a.m, 2 * a.n, a.ld_z, a.z_dtype));
    if (a.d_bias) LF_TRY(check_matrix("bias", a.d_bias, 1, 2 * a.n, 2 * a.n, a.bias_dtype));
    LF_REQUIRE(!a.d_x_scale == !a.d_w_scale && is_8bit_dtype(a.dtype) == (a.d_x_scale != nullptr), LF_ERR_INVALID, "8-bit operands, and only they, come with scales");
    const size_t need = lf_gated_linear_work_bytes(a.m, a.n, a.k, a.dtype);
    LF_REQUIRE(need == 0 || (d_work && (uintptr_t)d_work % 16 == 0), LF_ERR_INVALID, "null or unaligned workspace");
    LF_REQUIRE(work_bytes >= need, LF_ERR_WORKSPACE, "workspace of %zu bytes, %zu are needed", work_bytes, need);
    Product g{};
    g.p = a.d_x; g.q = a.d_w; g.ld_p = a.ld_x; g.ld_q = a.ld_w; g.m = a.m; g.n = a.n; g.k = a.k;
    g.e = Epilogue{a.d_y, nullptr, a.d_z, a.d_bias, a.d_x_scale, a.d_w_scale, a.ld_y, 0, a.ld_z, a.y_dtype, 0, a.z_dtype, a.bias_dtype, activation_of(a.activation, a.y_dtype)};
    return launch_product(g, a.dtype, false, false, d_work, (hipStream_t)stream, true);
}

size_t lf_gated_linear_grad_work_bytes(int64_t m, int64_t n, int64_t k, int32_t dtype, int32_t want_dx, int32_t want_dw, int32_t want_db) {
    if (m <= 0 || n <= 0 || n > kMostFeatures || k < 0 || !is_float_dtype(dtype)) return 0;
    return gated_work(m, n, k, dtype, want_dx, want_dw, want_db).total;
}

int lf_gated_linear_grad(const lf_linear_grad_args* h_args, void* d_work, size_t work_bytes, lf_stream_t stream) {
    LF_REQUIRE(h_args, LF_ERR_INVALID, "null argument");
    const lf_linear_grad_args& a = *h_args;
    LF_TRY(check_sizes(a.m, both_halves(a.n), a.k, a.dtype, a.activation));
    LF_REQUIRE(is_float_dtype(a.dtype) && (!a.d_db || is_float_dtype(a.db_dtype)), LF_ERR_UNSUPPORTED, "gradients are of float32, bfloat16 or float16");
    LF_TRY(check_matrix("dy", a.d_dy, a.m, a.n, a.ld_dy, a.dtype));
    LF_TRY(check_matrix("z", a.d_z, a.m, 2 * a.n, a.ld_z, a.dtype));
    if (a.d_dw) {
        LF_TRY(check_matrix("x", a.d_x, a.m, a.k, a.ld_x, a.dtype));
        LF_TRY(check_matrix("dw", a.d_dw, 2 * a.n, a.k, a.ld_dw, a.dtype));
    }
    if (a.d_dx) {
        LF_TRY(check_matrix("w", a.d_w, 2 * a.n, a.k, a.ld_w, a.dtype));
        LF_TRY(check_matrix("dx", a.d_dx, a.m, a.k, a.ld_dx, a.dtype));
    }
    if (a.d_db) LF_TRY(check_matrix("db", a.d_db, 1, 2 * a.n, 2 * a.n, a.db_dtype));
    if (a.n == 0 && a.k == 0) return LF_OK;
    const GradWork w = gated_work(a.m, a.n, a.k, a.dtype, a.d_dx, a.d_dw, a.d_db);
    LF_REQUIRE(w.total == 0 || (d_work && (uintptr_t)d_work % 16 == 0), LF_ERR_INVALID, "null or unaligned workspace");
    LF_REQUIRE(work_bytes >= w.total, LF_ERR_WORKSPACE, "workspace of %zu bytes, %zu are needed", work_bytes, w.total);
    hipStream_t st = (hipStream_t)stream;
    char* at = (char*)d_work;
    void* dz = at;
    float* sums = w.sums ? (float*)(at + w.dz) : nullptr;
    void* parts = at + w.dz + w.sums;
    const int64_t slabs = slabs_of(a.m, a.n), slab = ceil_div(std::max<int64_t>(a.m, 1), slabs);
    if (a.n > 0) {
        const int across = threads_across(a.n);
        const dim3 grid((unsigned)ceil_div(a.n, 8 * across), (unsigned)slabs);
        auto go = [&](auto t) {
            using T = decltype(t);
            auto kernel = across == 8 ? gate_grad_kernel<T, 8> : across == 16 ? gate_grad_kernel<T, 16> : gate_grad_kernel<T, 32>;
            kernel<<<grid, 256, 0, st>>>((const T*)a.d_dy, a.ld_dy, (const T*)a.d_z, a.ld_z, (T*)dz, ld_dz(2 * a.n), sums, sums ? nullptr : a.d_db, a.db_dtype, a.m, a.n, a.activation,
                                         slab);
        };
        if (a.dtype == LF_DTYPE_F32) go(0.f); else if (a.dtype == LF_DTYPE_BF16) go((__bf16)0.f); else go((_Float16)0.f);
        LF_HIP(hipGetLastError());
        if (sums && a.d_db) LF_TRY(lf::column_sums(sums, slabs, 2 * a.n, a.d_db, a.db_dtype, st));
    }
    return two_products(a, 2 * a.n, dz, ld_dz(2 * a.n), parts, st);
}

}  // extern "C"
