// Products of dense rows of features with a weight, on the matrix cores:
//
//     Y = act(X W^T + b) + R          X [m][k], W [n][k] of float32, bfloat16, float16, or 8 bits with a scale a row
//     dZ = dY act'(Z);  dX = dZ W;  dW = dZ^T X;  db = column sums of dZ
//
// One tiled kernel makes all of them.  It computes D[m][n] = sum over k of P[m][k] Q[n][k]; either operand may be
// stored with k along its rows (X, W of the forward product) or across them (W of dX, both of dW).
//   * A tile of TM x TN outputs belongs to a workgroup; a step stages 128 bytes of k (float32: 32 elements) of its
//     TM + TN rows in LDS, in two buffers, so that one step is read while the next is on its way: global loads into registers
//     a step ahead, LDS stores after the products, one barrier a step.
//   * In LDS both operands have k along the rows, in pieces of 16 bytes that are swapped about by a key of the row, so
//     that the 16 rows that a matrix instruction reads at once lie in different banks.  Operands stored across k are turned in
//     registers on their way there, four k at a time.
//   * Q gives the rows of a matrix instruction and P its columns, and neighbouring instructions take the rows of Q in fours: a lane
//     then holds eight consecutive outputs of a row, which the epilogue (scales, bias, activation, residual) reads and writes at once.
//   * float32 has no fast matrix instruction.  A value is cut into three bfloat16 of 8 bits each (exactly: by truncation), and
//     six of the nine products - all but those below 2^-24 of the largest - go through the bfloat16 one, which is 16 times as fast
//     as the float32 one.  Inf and NaN do not survive the cut; outputs that are not finite are computed again from the operands.
//   * Few tiles are cut along k as well: partial sums in 32 bits, added up in a fixed order by a second kernel with the epilogue.
// Up to 16 rows of X are another problem - W is read once, nothing is shared - and have a kernel of their own.
#include <algorithm>

#include "lf_dense.h"

namespace {

using namespace lf;

typedef float float4_t __attribute__((ext_vector_type(4)));
typedef int int4v __attribute__((ext_vector_type(4)));
typedef int int8v __attribute__((ext_vector_type(8)));

struct e4m3_t { uint8_t b; };

// ---------------------------------------------------------------------------- element types

template <typename T> struct Elem;
template <> struct Elem<__bf16> { static constexpr int kPlanes = 1; using Acc = float4_t; };
template <> struct Elem<_Float16> { static constexpr int kPlanes = 1; using Acc = float4_t; };
template <> struct Elem<e4m3_t> { static constexpr int kPlanes = 1; using Acc = float4_t; };
template <> struct Elem<int8_t> { static constexpr int kPlanes = 1; using Acc = int4v; };
template <> struct Elem<float> { static constexpr int kPlanes = 3; using Acc = float4_t; };

__device__ __forceinline__ float4_t mma(uint4_t a, uint4_t b, float4_t c, __bf16) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
}
__device__ __forceinline__ float4_t mma(uint4_t a, uint4_t b, float4_t c, _Float16) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
}
__device__ __forceinline__ int4v mma(uint4_t a, uint4_t b, int4v c, int8_t) {
    return __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(int4v, a), __builtin_bit_cast(int4v, b), c, 0, 0, 0);
}
// Two pieces of each at once: which k a byte stands for is free, as long as it is the same one on both sides.
__device__ __forceinline__ float4_t mma_e4m3(uint4_t a0, uint4_t a1, uint4_t b0, uint4_t b1, float4_t c) {
    const int8v a = {(int)a0[0], (int)a0[1], (int)a0[2], (int)a0[3], (int)a1[0], (int)a1[1], (int)a1[2], (int)a1[3]};
    const int8v b = {(int)b0[0], (int)b0[1], (int)b0[2], (int)b0[3], (int)b1[0], (int)b1[1], (int)b1[2], (int)b1[3]};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 0, 0, 0, 0, 0, 0);
}

// 16 bytes at any address that suits the type
template <typename T> __device__ __forceinline__ uint4_t load16(const T* p) {
    struct __attribute__((packed, aligned(sizeof(T)))) Any { uint4_t v; };
    return reinterpret_cast<const Any*>(p)->v;
}
// the first n elements of them, zeros behind
template <typename T> __device__ __forceinline__ uint4_t load16_upto(const T* p, int n) {
    constexpr int E = 16 / sizeof(T);
    if (n >= E) return load16(p);
    uint4_t r = {0u, 0u, 0u, 0u};
    for (int i = 0; i < E; ++i)
        if (i < n) {
            if constexpr (sizeof(T) == 4) r[i] = __builtin_bit_cast(uint32_t, p[i]);
            else if constexpr (sizeof(T) == 2) r[i >> 1] |= (uint32_t)__builtin_bit_cast(uint16_t, p[i]) << (16 * (i & 1));
            else r[i >> 2] |= (uint32_t)__builtin_bit_cast(uint8_t, p[i]) << (8 * (i & 3));
        }
    return r;
}

// Two floats as the halves of three words: 8 bits of each per word, which together are the floats exactly.
__device__ __forceinline__ void cut(float a, float b, uint32_t (&w)[3]) {
    const uint32_t top = 0xffff0000u;
#pragma unroll
    for (int p = 0; p < 3; ++p) {
        const uint32_t ua = __float_as_uint(a), ub = __float_as_uint(b);
        w[p] = __builtin_amdgcn_perm(ub, ua, 0x07060302u);
        a -= __uint_as_float(ua & top);
        b -= __uint_as_float(ub & top);
    }
}

// ---------------------------------------------------------------------------- the epilogue

struct Epilogue {
    void* y; const void* res; void* z; const void* bias; const float* x_scale; const float* w_scale;
    int64_t ld_y, ld_res, ld_z;
    int32_t y_dtype, res_dtype, z_dtype, bias_dtype, act;
};

// `count` outputs (at most eight) of row m from column n on
__device__ __forceinline__ void finish(const Epilogue& e, int64_t m, int64_t n, int count, float8_t v) {
    if (e.x_scale) v = v * e.x_scale[m] * load_upto8(e.w_scale + n, count);
    if (e.bias) v += load_upto8(e.bias, n, e.bias_dtype, count);
    if (e.z) store_upto8(e.z, m * e.ld_z + n, e.z_dtype, v, count);
    if (e.act != LF_ACT_NONE)
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = activate(v[i], e.act);
    if (e.res) v += load_upto8(e.res, m * e.ld_res + n, e.res_dtype, count);
    store_upto8(e.y, m * e.ld_y + n, e.y_dtype, v, count);
}

// ---------------------------------------------------------------------------- the tiled product

struct Product {
    const void* p; const void* q;
    int64_t ld_p, ld_q;
    int64_t m, n, k;
    int64_t k_split;                // elements of k to a split, a multiple of a step's
    int32_t tiles_m, tiles_n, splits;
    void* part;                     // [splits][m][n] partial sums, or NULL: the epilogue follows at once
    Epilogue e;
};

// Where 16-byte piece c of a row stands among the row's pieces.  Matrix instructions read 16 rows at one c (P: 16
// consecutive ones, Q: 8 a + 4 i + b for a, b < 4), turned operands are stored at rows 8 apart.
template <bool Q, int PIECES> __device__ __forceinline__ int slot(int row, int c) {
    if constexpr (PIECES == 8) {
        const int key = Q ? ((row & 3) | ((row >> 3 & 1) << 2)) ^ (row >> 4 & 7) : (row ^ row >> 3) & 7;
        return row * 8 + (c ^ key);
    } else {
        const int key = Q ? ((row >> 1 & 1) | ((row >> 3 & 1) << 1)) ^ (row >> 4 & 3) : (row >> 1 ^ row >> 3) & 3;
        return row * 4 + (c ^ key);
    }
}

// One operand's tile of ROWS x (a step of k): global memory -> registers -> LDS.
template <typename T, bool Q, bool ACROSS, int ROWS, int THREADS> struct Stage {
    static constexpr int kPlanes = Elem<T>::kPlanes;
    static constexpr int kStep = sizeof(T) == 4 ? 32 : 128 / sizeof(T);   // elements of k
    static constexpr int kPieces = sizeof(T) == 4 ? 4 : 8;                // pieces of a row in LDS (of each plane)
    static constexpr int kElems = kStep / kPieces;                        // elements of a piece
    static constexpr int kSlots = ROWS * kPieces;                         // 16-byte slots of a plane
    // along k: a unit is a piece (float32: 32 bytes).  Across: 4 k of 16 bytes of neighbouring rows.
    static constexpr int kWide = 16 / sizeof(T);                          // rows of a unit across
    static constexpr int kUnits = ACROSS ? (ROWS / kWide) * (kStep / 4) : ROWS * kPieces;
    static constexpr int kMine = (kUnits + THREADS - 1) / THREADS;
    static constexpr int kRegs = ACROSS ? 4 : kPlanes == 3 ? 2 : 1;       // 16-byte registers of a unit
    uint4_t r[kMine][kRegs];

    // `left`: elements of k from this step on (more than a step: the fast way)
    __device__ __forceinline__ void load(const T* base, int64_t ld, int64_t row0, int64_t rows, int64_t k0, int64_t left, int tid) {
        const bool whole = left >= kStep;
#pragma unroll
        for (int i = 0; i < kMine; ++i) {
            const int u = tid + i * THREADS;
            if (kUnits % THREADS && u >= kUnits) continue;
            if constexpr (!ACROSS) {
                const int64_t row = min(row0 + u / kPieces, rows - 1);    // (rows past the end are read for the last one and not used)
                const int at = (u % kPieces) * kElems;
                const T* src = base + row * ld + k0 + at;
#pragma unroll
                for (int h = 0; h < kRegs; ++h) {
                    if (whole) r[i][h] = load16(src + h * kWide);
                    else r[i][h] = load16_upto(src + h * kWide, (int)left - at - h * kWide);
                }
            } else {
                const Across a(u);
                const int64_t row = row0 + a.row;
                const int n = (int)min((int64_t)kWide, rows - row);
#pragma unroll
                for (int h = 0; h < 4; ++h) {
                    const T* src = base + (k0 + a.k + h) * ld + row;
                    const bool in = whole || a.k + h < left;
                    if (in && n == kWide) r[i][h] = load16(src);
                    else r[i][h] = load16_upto(src, in ? n : 0);
                }
            }
        }
    }
    struct Across {
        int row, k;                                                       // of the unit in the tile
        __device__ __forceinline__ explicit Across(int u) {
            // eight neighbouring units along k, then along the rows: 128 bytes of a row of the operand to a load instruction
            constexpr int KU = kStep / 4, RU = ROWS / kWide;
            static_assert(KU % 8 == 0 && RU % 8 == 0, "");
            const int kl = u & 7, rl = u >> 3 & 7, rest = u >> 6;
            row = (rl + 8 * (rest % (RU / 8))) * kWide;
            k = (kl + 8 * (rest / (RU / 8))) * 4;
        }
    };
    __device__ __forceinline__ void store(uint4_t* lds, int tid) const {
#pragma unroll
        for (int i = 0; i < kMine; ++i) {
            const int u = tid + i * THREADS;
            if (kUnits % THREADS && u >= kUnits) continue;
            if constexpr (!ACROSS && kPlanes == 1) {
                lds[slot<Q, kPieces>(u / kPieces, u % kPieces)] = r[i][0];
            } else if constexpr (!ACROSS) {
                uint4_t out[3];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    uint32_t w[3];
                    cut(__uint_as_float(r[i][j >> 1][2 * (j & 1)]), __uint_as_float(r[i][j >> 1][2 * (j & 1) + 1]), w);
                    out[0][j] = w[0]; out[1][j] = w[1]; out[2][j] = w[2];
                }
#pragma unroll
                for (int p = 0; p < 3; ++p) lds[p * kSlots + slot<Q, kPieces>(u / kPieces, u % kPieces)] = out[p];
            } else {
                const Across a(u);
                uint2_t* half = reinterpret_cast<uint2_t*>(lds);
#pragma unroll
                for (int j = 0; j < kWide; ++j) {
                    const int at = 2 * slot<Q, kPieces>(a.row + j, a.k / kElems) + (a.k / 4 & 1);
                    if constexpr (kPlanes == 1) {
                        const uint32_t sel = j & 1 ? 0x07060302u : 0x05040100u;
                        half[at] = uint2_t{__builtin_amdgcn_perm(r[i][1][j >> 1], r[i][0][j >> 1], sel), __builtin_amdgcn_perm(r[i][3][j >> 1], r[i][2][j >> 1], sel)};
                    } else {
                        uint32_t lo[3], hi[3];
                        cut(__uint_as_float(r[i][0][j]), __uint_as_float(r[i][1][j]), lo);
                        cut(__uint_as_float(r[i][2][j]), __uint_as_float(r[i][3][j]), hi);
#pragma unroll
                        for (int p = 0; p < 3; ++p) half[2 * p * kSlots + at] = uint2_t{lo[p], hi[p]};
                    }
                }
            }
        }
    }
};

// One output of a float32 product from the operands themselves.
template <bool PX, bool QX> __device__ __noinline__ float dot_f32(const Product& g, int64_t m, int64_t n, int64_t k0, int64_t k1) {
    const float* p = (const float*)g.p;
    const float* q = (const float*)g.q;
    float s = 0.f;
    for (int64_t k = k0; k < k1; ++k) s = fmaf(PX ? p[k * g.ld_p + m] : p[m * g.ld_p + k], QX ? q[k * g.ld_q + n] : q[n * g.ld_q + k], s);
    return s;
}

// The tile of a workgroup.  Workgroups go to the eight XCDs in turn: each XCD gets a run of neighbouring tiles, eight rows of
// tiles deep, so that what its L2 holds of both operands is used by its 32 CUs at once.
__device__ __forceinline__ void tile_of(const Product& g, unsigned id, int& tm, int& tn) {
    const unsigned n = (unsigned)g.tiles_m * g.tiles_n, xcd = id % 8, each = n / 8, more = n % 8;
    unsigned t = xcd * each + min(xcd, more) + id / 8;
    constexpr unsigned kDeep = 8;
    const unsigned band = t / (kDeep * g.tiles_n), first = band * kDeep, deep = min(kDeep, (unsigned)g.tiles_m - first);
    t -= band * kDeep * g.tiles_n;
    tm = (int)(first + t % deep);
    tn = (int)(t / deep);
}

template <typename T, bool PX, bool QX, int TM, int TN, int WM, int WN>
__global__ void __launch_bounds__(64 * WM * WN)
product_kernel(Product g) {
    constexpr int THREADS = 64 * WM * WN, FM = TM / WM / 16, FN = TN / WN / 16;
    static_assert(FN % 2 == 0, "");
    using Acc = typename Elem<T>::Acc;
    using StageP = Stage<T, false, PX, TM, THREADS>;
    using StageQ = Stage<T, true, QX, TN, THREADS>;
    constexpr int PL = StageP::kPlanes, PC = StageP::kPieces, KS = StageP::kStep;
    __shared__ uint4_t s_p[2][PL * StageP::kSlots];
    __shared__ uint4_t s_q[2][PL * StageQ::kSlots];
    const int tid = threadIdx.x, lane = tid & 63, li = lane & 15, lg = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), wm = wave % WM, wn = wave / WM;
    int tm, tn;
    tile_of(g, blockIdx.x, tm, tn);
    const int64_t m0 = (int64_t)tm * TM, n0 = (int64_t)tn * TN;
    const int64_t k_first = (int64_t)blockIdx.y * g.k_split, k_last = min(g.k, k_first + g.k_split);

    Acc acc[FM][FN];
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j) acc[i][j] = Acc{0, 0, 0, 0};

    // rows of the matrix instructions' operands in the tile
    const int row_p = wm * (TM / WM) + li, row_q = wn * (TN / WN) + (li >> 2) * 8 + (li & 3);
    auto multiply = [&](const uint4_t* sp, const uint4_t* sq) {
        if constexpr (PL == 3) {
            // a step is one 32-deep instruction, for six pairs of planes
            uint4_t a[3][FN];
#pragma unroll
            for (int p = 0; p < 3; ++p)
#pragma unroll
                for (int j = 0; j < FN; ++j) a[p][j] = sq[p * StageQ::kSlots + slot<true, PC>(row_q + (j >> 1) * 32 + (j & 1) * 4, lg)];
#pragma unroll
            for (int i = 0; i < FM; ++i) {
                uint4_t b[3];
#pragma unroll
                for (int p = 0; p < 3; ++p) b[p] = sp[p * StageP::kSlots + slot<false, PC>(row_p + i * 16, lg)];
#pragma unroll
                for (int p = 2; p >= 0; --p)                              // the smallest products first
#pragma unroll
                    for (int q = 2 - p; q >= 0; --q)
#pragma unroll
                        for (int j = 0; j < FN; ++j) acc[i][j] = mma(a[q][j], b[p], acc[i][j], (__bf16)0.f);
            }
        } else if constexpr (sizeof(T) == 1 && !std::is_same_v<T, int8_t>) {
            uint4_t a[FN][2];
#pragma unroll
            for (int j = 0; j < FN; ++j)
#pragma unroll
                for (int h = 0; h < 2; ++h) a[j][h] = sq[slot<true, PC>(row_q + (j >> 1) * 32 + (j & 1) * 4, 4 * h + lg)];
#pragma unroll
            for (int i = 0; i < FM; ++i) {
                uint4_t b[2];
#pragma unroll
                for (int h = 0; h < 2; ++h) b[h] = sp[slot<false, PC>(row_p + i * 16, 4 * h + lg)];
#pragma unroll
                for (int j = 0; j < FN; ++j) acc[i][j] = mma_e4m3(a[j][0], a[j][1], b[0], b[1], acc[i][j]);
            }
        } else {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                uint4_t a[FN];
#pragma unroll
                for (int j = 0; j < FN; ++j) a[j] = sq[slot<true, PC>(row_q + (j >> 1) * 32 + (j & 1) * 4, 4 * h + lg)];
#pragma unroll
                for (int i = 0; i < FM; ++i) {
                    const uint4_t b = sp[slot<false, PC>(row_p + i * 16, 4 * h + lg)];
#pragma unroll
                    for (int j = 0; j < FN; ++j) acc[i][j] = mma(a[j], b, acc[i][j], T{});
                }
            }
        }
    };

    const int64_t steps = k_last > k_first ? (k_last - k_first + KS - 1) / KS : 0;
    if (steps > 0) {
        StageP p;
        StageQ q;
        auto load = [&](int64_t s) {
            const int64_t k = k_first + s * KS;
            p.load((const T*)g.p, g.ld_p, m0, g.m, k, k_last - k, tid);
            q.load((const T*)g.q, g.ld_q, n0, g.n, k, k_last - k, tid);
        };
        load(0);
        p.store(s_p[0], tid);
        q.store(s_q[0], tid);
        if (steps > 1) load(1);
        __syncthreads();
        for (int64_t s = 0; s < steps; ++s) {
            const int now = (int)(s & 1);
            multiply(s_p[now], s_q[now]);
            if (s + 1 < steps) {
                p.store(s_p[now ^ 1], tid);
                q.store(s_q[now ^ 1], tid);
                if (s + 2 < steps) load(s + 2);
            }
            __syncthreads();
        }
    }

#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; j += 2) {
            const int64_t m = m0 + wm * (TM / WM) + i * 16 + li, n = n0 + wn * (TN / WN) + j * 16 + lg * 8;
            if (m >= g.m || n >= g.n) continue;
            const int count = (int)min((int64_t)8, g.n - n);
            if constexpr (std::is_same_v<Acc, int4v>) {
                if (g.part) {
                    int32_t* to = (int32_t*)g.part + ((int64_t)blockIdx.y * g.m + m) * g.n + n;
#pragma unroll
                    for (int v = 0; v < 8; ++v)
                        if (v < count) to[v] = acc[i][j + (v >> 2)][v & 3];
                    continue;
                }
            }
            float8_t v;
#pragma unroll
            for (int r = 0; r < 8; ++r) v[r] = (float)acc[i][j + (r >> 2)][r & 3];
            if constexpr (PL == 3) {
#pragma unroll
                for (int r = 0; r < 8; ++r)
                    if (r < count && !(fabsf(v[r]) < __builtin_inff())) v[r] = dot_f32<PX, QX>(g, m, n + r, k_first, k_last);
            }
            if (g.part) store_upto8((float*)g.part + ((int64_t)blockIdx.y * g.m + m) * g.n + n, v, count);
            else finish(g.e, m, n, count, v);
        }
}

// The splits' partial sums in order, and the epilogue.
template <typename A>
__global__ void __launch_bounds__(256) join_kernel(const A* part, int64_t m, int64_t n, int32_t splits, Epilogue e) {
    const int64_t across = (n + 7) / 8, u = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (u >= m * across) return;
    const int64_t row = u / across, col = (u % across) * 8;
    const int count = (int)min((int64_t)8, n - col);
    A sum[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    for (int s = 0; s < splits; ++s) {
        const A* src = part + ((int64_t)s * m + row) * n + col;
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < count) sum[i] += src[i];
    }
    float8_t v;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = (float)sum[i];
    finish(e, row, col, count, v);
}

// ---------------------------------------------------------------------------- few rows

// Up to 16 rows of X: a workgroup takes 16 rows of W, its wavefronts the 128-byte steps of k in turn, and their sums
// meet in LDS.  W goes from memory into the matrix instructions' registers, 32 consecutive bytes a lane and step.
template <typename T, int WAVES>
__global__ void __launch_bounds__(64 * WAVES)
few_rows_kernel(Product g) {
    constexpr int KS = 128 / sizeof(T), MINE = 32 / sizeof(T), E = 16 / sizeof(T);
    using Acc = typename Elem<T>::Acc;
    using S = std::conditional_t<std::is_same_v<Acc, int4v>, int32_t, float>;
    __shared__ S s_sum[WAVES][16][17];
    const int lane = threadIdx.x & 63, li = lane & 15, lg = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t n0 = (int64_t)blockIdx.x * 16;
    const T* w = (const T*)g.q + min(n0 + li, g.n - 1) * g.ld_q + lg * MINE;
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
            a[h] = load16_upto(w + s * KS + h * E, left);
            b[h] = load16_upto(x + s * KS + h * E, on ? left : 0);
        }
        multiply(a, b);
    }
#pragma unroll
    for (int v = 0; v < 4; ++v) s_sum[wave][li][lg * 4 + v] = acc[v];
    __syncthreads();
    const int m = threadIdx.x >> 1, at = (threadIdx.x & 1) * 8;
    if (m >= g.m || n0 + at >= g.n) return;
    float8_t out;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        S t = 0;
#pragma unroll
        for (int u = 0; u < WAVES; ++u) t += s_sum[u][m][at + i];
        out[i] = (float)t;
    }
    finish(g.e, m, n0 + at, (int)min((int64_t)8, g.n - n0 - at), out);
}

// ---------------------------------------------------------------------------- gradient of the activation

// dz = dy act'(z), in rows of `ld_dz` elements, and the column sums of a slab of rows (before rounding).
template <typename T>
__global__ void __launch_bounds__(256)
activation_grad_kernel(const T* dy, int64_t ld_dy, const T* z, int64_t ld_z, T* dz, int64_t ld_dz, float* part, int64_t m, int64_t n, int32_t act,
                       int64_t slab) {
    __shared__ float s[8][32][9];
    const int lx = threadIdx.x & 31, ly = threadIdx.x >> 5;
    const int64_t col = ((int64_t)blockIdx.x * 32 + lx) * 8;
    const int count = (int)min((int64_t)8, n - col);
    const int64_t r1 = min(m, ((int64_t)blockIdx.y + 1) * slab);
    float8_t sum = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (count > 0)
        for (int64_t r = (int64_t)blockIdx.y * slab + ly; r < r1; r += 8) {
            float8_t d = load_upto8(dy + r * ld_dy + col, count);
            if (act != LF_ACT_NONE) {
                const float8_t v = load_upto8(z + r * ld_z + col, count);
#pragma unroll
                for (int i = 0; i < 8; ++i) d[i] *= activate_grad(v[i], act);
            }
            if (dz) store_upto8(dz + r * ld_dz + col, d, count);
            sum += d;
        }
    if (!part) return;
#pragma unroll
    for (int i = 0; i < 8; ++i) s[ly][lx][i] = sum[i];
    __syncthreads();
    const int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (c >= n) return;
    float t = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) t += s[i][threadIdx.x >> 3][threadIdx.x & 7];
    part[(int64_t)blockIdx.y * n + c] = t;
}

// ---------------------------------------------------------------------------- launches

// How a product is cut up: tile, splits of k, bytes of partial sums.
struct Cut { int tile; int splits; int64_t k_split; size_t bytes; };

Cut cut_product(int32_t dtype, int64_t m, int64_t n, int64_t k) {
    const int step = dtype == LF_DTYPE_F32 ? 32 : 128 / dtype_bytes(dtype);
    auto tiles = [&](int t) { return ceil_div(m, t) * ceil_div(n, t); };
    const int tile = dtype != LF_DTYPE_F32 && tiles(256) >= 200 ? 256 : tiles(128) >= 200 || (m > 64 && n > 64) ? 128 : 64;
    const int64_t t = tiles(tile), steps = ceil_div(k, step);
    int64_t splits = 1;
    if (t < 200 && steps >= 16) splits = std::min<int64_t>(ceil_div(512, t), steps / 8);
    const int64_t each = std::max<int64_t>(1, ceil_div(steps, splits));
    splits = std::max<int64_t>(1, ceil_div(steps, each));
    return {tile, (int)splits, each * step, splits > 1 ? (size_t)splits * (size_t)m * (size_t)n * 4 : 0};
}

using ProductFn = void (*)(Product);
template <typename T, bool PX, bool QX> ProductFn product_of(int tile) {
    if constexpr (!std::is_same_v<T, float>)
        if (tile == 256) return product_kernel<T, PX, QX, 256, 256, 2, 4>;
    return tile == 128 ? product_kernel<T, PX, QX, 128, 128, 2, 2> : product_kernel<T, PX, QX, 64, 64, 2, 2>;
}
template <bool PX, bool QX> ProductFn product_of(int32_t dtype, int tile) {
    if constexpr (!PX && !QX) {
        if (dtype == LF_DTYPE_E4M3) return product_of<e4m3_t, PX, QX>(tile);
        if (dtype == LF_DTYPE_I8) return product_of<int8_t, PX, QX>(tile);
    }
    return dtype == LF_DTYPE_F32 ? product_of<float, PX, QX>(tile) : dtype == LF_DTYPE_BF16 ? product_of<__bf16, PX, QX>(tile) : product_of<_Float16, PX, QX>(tile);
}
template <int WAVES> ProductFn few_rows_of(int32_t dtype) {
    switch (dtype) {
        case LF_DTYPE_F32: return few_rows_kernel<float, WAVES>;
        case LF_DTYPE_BF16: return few_rows_kernel<__bf16, WAVES>;
        case LF_DTYPE_F16: return few_rows_kernel<_Float16, WAVES>;
        case LF_DTYPE_E4M3: return few_rows_kernel<e4m3_t, WAVES>;
        default: return few_rows_kernel<int8_t, WAVES>;
    }
}

constexpr int64_t kFewRows = 16;

int launch_product(Product g, int32_t dtype, bool px, bool qx, void* work, hipStream_t st) {
    if (g.m == 0 || g.n == 0) return LF_OK;
    if (!px && !qx && g.m <= kFewRows) {
        const int64_t groups = ceil_div(g.n, 16);
        LF_REQUIRE(groups < (1ll << 31), LF_ERR_UNSUPPORTED, "too many columns");
        // few workgroups take 16 wavefronts each
        if (groups <= 256) few_rows_of<16>(dtype)<<<(unsigned)groups, 1024, 0, st>>>(g);
        else few_rows_of<8>(dtype)<<<(unsigned)groups, 512, 0, st>>>(g);
        LF_HIP(hipGetLastError());
        return LF_OK;
    }
    const Cut c = cut_product(dtype, g.m, g.n, g.k);
    const int64_t tm = ceil_div(g.m, c.tile), tn = ceil_div(g.n, c.tile);
    LF_REQUIRE(tm < (1ll << 27) && tn < (1ll << 27) && tm * tn < (1ll << 31), LF_ERR_UNSUPPORTED, "too many tiles");
    g.tiles_m = (int32_t)tm;
    g.tiles_n = (int32_t)tn;
    g.splits = c.splits;
    g.k_split = c.k_split;
    g.part = c.splits > 1 ? work : nullptr;
    const ProductFn f = px ? product_of<true, true>(dtype, c.tile) : qx ? product_of<false, true>(dtype, c.tile) : product_of<false, false>(dtype, c.tile);
    f<<<dim3((unsigned)(tm * tn), (unsigned)c.splits), c.tile == 256 ? 512 : 256, 0, st>>>(g);
    LF_HIP(hipGetLastError());
    if (c.splits > 1) {
        const int64_t groups = ceil_div(g.m * ceil_div(g.n, 8), 256);
        LF_REQUIRE(groups < (1ll << 31), LF_ERR_UNSUPPORTED, "too many outputs");
        if (dtype == LF_DTYPE_I8) join_kernel<int32_t><<<(unsigned)groups, 256, 0, st>>>((const int32_t*)work, g.m, g.n, c.splits, g.e);
        else join_kernel<float><<<(unsigned)groups, 256, 0, st>>>((const float*)work, g.m, g.n, c.splits, g.e);
        LF_HIP(hipGetLastError());
    }
    return LF_OK;
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

// Rows of dz are padded to a multiple of 16 bytes.
int64_t ld_dz(int64_t n) { return ceil_div(n, 8) * 8; }
size_t padded(size_t bytes) { return (bytes + 255) / 256 * 256; }
// Slabs of rows whose column sums are kept apart: enough workgroups to fill the GPU.
int64_t slabs_of(int64_t m, int64_t n) { return std::max<int64_t>(1, std::min(ceil_div(m, 64), ceil_div(2048, ceil_div(n, 256)))); }

struct GradWork { size_t dz, sums, parts, total; };
GradWork grad_work(int64_t m, int64_t n, int64_t k, int32_t dtype, int32_t act, bool dx, bool dw, bool db) {
    GradWork w{0, 0, 0, 0};
    if (act != LF_ACT_NONE) w.dz = padded((size_t)m * (size_t)ld_dz(n) * dtype_bytes(dtype));
    if (db) w.sums = padded((size_t)slabs_of(m, n) * (size_t)n * 4);
    if (dx && m && k) w.parts = cut_product(dtype, m, k, n).bytes;
    if (dw && n && k) w.parts = std::max(w.parts, cut_product(dtype, n, k, m).bytes);
    w.total = w.dz + w.sums + w.parts;
    return w;
}

}  // namespace

extern "C" {

size_t lf_linear_work_bytes(int64_t m, int64_t n, int64_t k, int32_t dtype) {
    if (m <= kFewRows || n <= 0 || k <= 0 || !(is_float_dtype(dtype) || is_8bit_dtype(dtype))) return 0;
    return cut_product(dtype, m, n, k).bytes;
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
                   a.bias_dtype, a.activation};
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
    if ((dz || sums) && a.n > 0) {
        const dim3 grid((unsigned)ceil_div(a.n, 256), (unsigned)slabs);
        auto go = [&](auto t) {
            using T = decltype(t);
            activation_grad_kernel<T><<<grid, 256, 0, st>>>((const T*)a.d_dy, a.ld_dy, (const T*)a.d_z, a.ld_z, (T*)dz, ld_dz(a.n), sums, a.m, a.n, a.activation, slab);
        };
        if (a.dtype == LF_DTYPE_F32) go(0.f); else if (a.dtype == LF_DTYPE_BF16) go((__bf16)0.f); else go((_Float16)0.f);
        LF_HIP(hipGetLastError());
        if (a.d_db) LF_TRY(lf::column_sums(sums, slabs, a.n, a.d_db, a.db_dtype, st));
    }
    const void* d = dz ? dz : a.d_dy;
    const int64_t ld = dz ? ld_dz(a.n) : a.ld_dy;
    if (a.d_dx) {
        Product g{};
        g.p = d; g.ld_p = ld; g.q = a.d_w; g.ld_q = a.ld_w; g.m = a.m; g.n = a.k; g.k = a.n;
        g.e.y = a.d_dx; g.e.ld_y = a.ld_dx; g.e.y_dtype = a.dtype;
        LF_TRY(launch_product(g, a.dtype, false, true, parts, st));
    }
    if (a.d_dw) {
        Product g{};
        g.p = d; g.ld_p = ld; g.q = a.d_x; g.ld_q = a.ld_x; g.m = a.n; g.n = a.k; g.k = a.m;
        g.e.y = a.d_dw; g.e.ld_y = a.ld_dw; g.e.y_dtype = a.dtype;
        LF_TRY(launch_product(g, a.dtype, true, true, parts, st));
    }
    return LF_OK;
}

}  // extern "C"
