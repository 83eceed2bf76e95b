// The tiled products behind lf_linear and lf_linear_grad: dense rows of features with a weight, on the matrix cores:
//
//     Y = act(X W^T + b) + R          X [m][k], W [n][k] of float32, bfloat16, float16, or 8 bits with a scale a row
//     dZ = dY act'(Z);  dX = dZ W;  dW = dZ^T X;  db = column sums of dZ
//
// Each is D[m][n] = sum over k of P[m][k] Q[n][k]; either operand may be stored with k along its rows (X, W of the forward
// product) or across them (W of dX, both of dW).  Three tiled kernels: this one, for any operands, and two for aligned ones of 8 and 16 bits, further down.
//   * A tile of TM x TN outputs belongs to a workgroup; a step stages 128 bytes of k (float32: 32 elements) of its
//     TM + TN rows in LDS, in two buffers, so that one step is read while the next is on its way: global loads into registers
//     a step ahead, LDS stores after the products, one barrier a step.
//   * In LDS both operands have k along the rows, in pieces of 16 bytes that are swapped about by a key of the row, so
//     that the 16 rows that a matrix instruction reads at once lie in different banks.  Operands stored across k are turned in
//     registers on their way there, four k at a time.
//   * Q gives the rows of a matrix instruction and P its columns: a lane holds four consecutive outputs of a row.  They go through LDS into
//     whole rows, in which the epilogue (scales, bias, activation, residual) reads and writes.
//   * float32 has no fast matrix instruction.  A value is cut into three bfloat16 of 8 bits each (exactly: by truncation), and
//     six of the nine products - all but those below 2^-24 of the largest - go through the bfloat16 one, which is 16 times as fast
//     as the float32 one: 4096^3 695 us (198 TFLOP/s), the library's float32 product 940.  Bound by the matrix cores there, by memory where
//     k is short (170k x 128 by 256 116 us, 3.8 TB/s).  Inf and NaN do not survive the cut; outputs that are not finite are computed again from the operands (repair).
//     What a cut leaves below 2^-126 is lost to the instruction: values below 2^-110 have fewer digits than a float.
//   * Few tiles are cut along k as well: partial sums in 32 bits, added up in a fixed order by a second kernel with the epilogue.
// Up to 16 rows of X are another problem - W is read once, nothing is shared - and have a kernel of their own.
#pragma once
#include <algorithm>
#include <type_traits>

#include "lf_cut.h"
#include "lf_dense.h"

namespace lf {

typedef float float4_t __attribute__((ext_vector_type(4)));
typedef int int4v __attribute__((ext_vector_type(4)));
typedef int int8v __attribute__((ext_vector_type(8)));

struct e4m3_t { uint8_t b; };

// ---------------------------------------------------------------------------- the epilogue

struct Epilogue {
    void* y; const void* res; void* z; const void* bias; const float* x_scale; const float* w_scale;
    int64_t ld_y, ld_res, ld_z;
    int32_t y_dtype, res_dtype, z_dtype, bias_dtype, act;
    int32_t stream;                 // y past the caches
};

struct Product {
    const void* p; const void* q;
    int64_t ld_p, ld_q;
    int64_t m, n, k;
    int64_t k_split;                // elements of k to a split, a multiple of a step's
    int32_t tiles_m, tiles_n, splits;
    void* part;                     // [splits][m][n] partial sums, or NULL: the epilogue follows at once
    Epilogue e;
};
using ProductFn = void (*)(Product);

// The kernel for operands of a type: px, qx: P, Q stored across k; tile: 64, 128 or, aligned and not float32, 256 (kWideTile); aligned: pieces of
// 16 bytes of the operands are, and across k they are whole; deep: few workgroups.
ProductFn product_f32(bool px, bool qx, int tile, bool aligned, bool deep);
ProductFn product_bf16(bool px, bool qx, int tile, bool aligned, bool deep);
ProductFn product_f16(bool px, bool qx, int tile, bool aligned, bool deep);
ProductFn product_e4m3(bool px, bool qx, int tile, bool aligned, bool deep);
ProductFn product_i8(bool px, bool qx, int tile, bool aligned, bool deep);

}  // namespace lf

namespace {

using namespace lf;

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

// `count` outputs (at most eight) of row m from column n on
__device__ __forceinline__ void finish(const Epilogue& e, int64_t m, int64_t n, int count, float8_t v) {
    if (e.x_scale) v = v * e.x_scale[m] * load_upto8(e.w_scale + n, count);
    if (e.bias) v += load_upto8(e.bias, n, e.bias_dtype, count);
    if (e.z) store_upto8(e.z, m * e.ld_z + n, e.z_dtype, v, count);
    v = activate(v, e.act);
    if (e.res) v += load_upto8(e.res, m * e.ld_res + n, e.res_dtype, count);
    store_upto8(e.y, m * e.ld_y + n, e.y_dtype, v, count);
}

template <typename F> __device__ __forceinline__ void with_type(int32_t dtype, F f) {
    if (dtype == LF_DTYPE_F32) f(0.f);
    else if (dtype == LF_DTYPE_BF16) f((__bf16)0.f);
    else f((_Float16)0.f);
}

// ---------------------------------------------------------------------------- the tiled product

// Where 16-byte piece c of a row stands among the row's pieces: matrix instructions read 16 consecutive rows at one c, operands across k are
// stored at rows 8 apart.
template <int PIECES> __device__ __forceinline__ int slot(int row, int c) {
    return PIECES == 8 ? row * 8 + (c ^ ((row ^ row >> 3) & 7)) : row * 4 + (c ^ ((row >> 1 ^ row >> 3) & 3));
}

// One operand's tile of ROWS x (a step of k): global memory -> registers -> LDS.
template <typename T, bool ACROSS, int ROWS, int THREADS> struct Stage {
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

    // `left`: elements of k from this step on, to the end of the product's part; `k`: of the matrix.
    // Along k rows past the end are read for the last one and not used.
    // Across, every piece is loaded whole: what stands behind a row in memory comes along, as rows of the tile that are never left.  In the last steps a
    // piece that would pass the end of the matrix is loaded from its last 16 bytes instead, and store() moves its elements to their places and
    // clears those of k past the end.  (Loaded by their size, in branches of each lane, pieces of bf16 4279 x 3514 by 4279 x 224 waited
    // for each other at every step: dw 124 us, now 60.  Along k, where branches are of whole wavefronts but in a last step, the same costs 4 %.)
    // A matrix of less than a piece, which has one step, is loaded one by one.
    static __device__ __forceinline__ int64_t last_piece(int64_t ld, int64_t rows, int64_t k) { return (k - 1) * ld + rows - kWide; }
    static __device__ __forceinline__ int64_t across_at(int u, int h, int64_t ld, int64_t row0, int64_t k0, int64_t rows) {
        const Across a(u);
        return max((int64_t)0, (k0 + a.k + h) * ld + min(row0 + a.row, rows - 1));   // (one row: ld is any number)
    }
    template <bool FIRST> __device__ __forceinline__ void load(const T* base, int64_t ld, int64_t row0, int64_t rows, int64_t k0, int64_t k, int64_t left, int tid) {
        if constexpr (!ACROSS) {
            const bool whole = left >= kStep;
#pragma unroll
            for (int i = 0; i < kMine; ++i) {
                const int u = tid + i * THREADS;
                if (kUnits % THREADS && u >= kUnits) continue;
                const int at = (u % kPieces) * kElems;
                const T* src = base + min(row0 + u / kPieces, rows - 1) * ld + k0 + at;
#pragma unroll
                for (int h = 0; h < kRegs; ++h) {
                    if (whole) r[i][h] = load16(src + h * kWide);
                    else r[i][h] = part16(src + h * kWide, (int)left - at - h * kWide);
                }
            }
        } else {
            // (a piece reaches up to kWide - 1 elements past its row, as many rows of k behind it hold at least; offsets in 32 bits)
            if (k - k0 >= kStep + kWide && ld < (1 << 20)) {
                const T* step = base + k0 * ld + row0;
                const uint32_t last_row = (uint32_t)min((int64_t)ROWS, rows - 1 - row0);
#pragma unroll
                for (int i = 0; i < kMine; ++i) {
                    const int u = tid + i * THREADS;
                    if (kUnits % THREADS && u >= kUnits) continue;
                    const Across a(u);
                    const uint32_t off = (a.k * (uint32_t)ld + min((uint32_t)a.row, last_row)) * (uint32_t)sizeof(T);
#pragma unroll
                    for (int h = 0; h < kRegs; ++h) r[i][h] = load16((const T*)((const char*)(step + h * ld) + off));
                }
                return;
            }
            asm volatile("" : "+s"(ld));             // (or the addresses of these few steps would stay in registers through all)
            const int64_t last = last_piece(ld, rows, k);
#pragma unroll
            for (int i = 0; i < kMine; ++i) {
                const int u = tid + i * THREADS;
                if (kUnits % THREADS && u >= kUnits) continue;
                if constexpr (FIRST)
                    if (last < 0) {
#pragma unroll
                        for (int h = 0; h < kRegs; ++h) {
                            const int64_t o = across_at(u, h, ld, row0, k0, rows);
                            r[i][h] = load16_each(base + min(o, last + kWide), (int)max((int64_t)0, last + kWide - o));
                        }
                        continue;
                    }
#pragma unroll
                for (int h = 0; h < kRegs; ++h) r[i][h] = load16(base + min(across_at(u, h, ld, row0, k0, rows), last));
            }
        }
    }
    // (as it was loaded)
    __device__ __forceinline__ void store(uint4_t* lds, int64_t ld, int64_t row0, int64_t rows, int64_t k0, int64_t k, int64_t left, int tid) {
        if constexpr (!ACROSS) {
            if (left < kStep)
#pragma unroll
                for (int i = 0; i < kMine; ++i)
#pragma unroll
                    for (int h = 0; h < kRegs; ++h) r[i][h] = join16<T>(r[i][h], (int)left - (tid + i * THREADS) % kPieces * kElems - h * kWide);
        } else if (left < kStep + kWide) {
            asm volatile("" : "+s"(ld));
            const int64_t last = last_piece(ld, rows, k);
#pragma unroll
            for (int i = 0; i < kMine; ++i) {
                const int u = tid + i * THREADS;
                if (kUnits % THREADS && u >= kUnits) continue;
#pragma unroll
                for (int h = 0; h < kRegs; ++h) {
                    const int64_t o = across_at(u, h, ld, row0, k0, rows);
                    r[i][h] = move16<T>(r[i][h], last < 0 ? 0 : (int)min((int64_t)kWide, max((int64_t)0, o - last)), Across(u).k + h < left ? kWide : 0);
                }
            }
        }
#pragma unroll
        for (int i = 0; i < kMine; ++i) {
            const int u = tid + i * THREADS;
            if (kUnits % THREADS && u >= kUnits) continue;
            if constexpr (!ACROSS && kPlanes == 1) {
                lds[slot<kPieces>(u / kPieces, u % kPieces)] = r[i][0];
            } else if constexpr (!ACROSS) {
                uint4_t out[3];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    uint32_t w[3];
                    cut(__uint_as_float(r[i][j >> 1][2 * (j & 1)]), __uint_as_float(r[i][j >> 1][2 * (j & 1) + 1]), w);
                    out[0][j] = w[0]; out[1][j] = w[1]; out[2][j] = w[2];
                }
#pragma unroll
                for (int p = 0; p < 3; ++p) lds[p * kSlots + slot<kPieces>(u / kPieces, u % kPieces)] = out[p];
            } else {
                const Across a(u);
                uint2_t* half = reinterpret_cast<uint2_t*>(lds);
#pragma unroll
                for (int j = 0; j < kWide; ++j) {
                    const int at = 2 * slot<kPieces>(a.row + j, a.k / kElems) + (a.k / 4 & 1);
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

// Sums of planes that are not finite: infinities, NaN and values near the ends of the exponents' range do not survive the cut, or leave the range on the
// way.  Sixteen rows of P with such an output are multiplied again by float32 matrix instructions, operands from memory; finite sums stay as they
// are.  (Each output by a lane of its own, along k: a NaN in 1024^3 took 525 us where 40 are usual, an operand of NaN in 4096^3 73 ms for 0.7; now 58 us
// and 2.8 ms.)
template <bool ACROSS> __device__ __forceinline__ uint4_t four_of(const float* p, int64_t ld, int64_t row, int64_t k, int64_t end) {
    if constexpr (!ACROSS) return load16_each(p + row * ld + k, (int)max((int64_t)0, min((int64_t)4, end - k)));
    uint4_t r = {0u, 0u, 0u, 0u};
#pragma unroll
    for (int c = 0; c < 4; ++c)
        if (k + c < end) r[c] = __float_as_uint(p[(k + c) * ld + row]);
    return r;
}
template <bool PX, bool QX, int FM, int FN>
__device__ __forceinline__ void repair(const Product& g, float4_t (&acc)[FM][FN], int64_t m, int64_t n, int64_t k_first, int64_t k_last) {
    const int li = threadIdx.x & 15, lg = threadIdx.x >> 4 & 3;
#pragma unroll
    for (int i = 0; i < FM; ++i) {
        float none = 0.f;                                                // NaN where a sum is not finite
#pragma unroll
        for (int j = 0; j < FN; ++j)
#pragma unroll
            for (int v = 0; v < 4; ++v) none = fmaf(acc[i][j][v], 0.f, none);
        if (__builtin_expect(__all(none == 0.f), 1)) continue;
        bool fine = true;                                                // ... in rows and columns that there are
#pragma unroll
        for (int j = 0; j < FN; ++j)
#pragma unroll
            for (int v = 0; v < 4; ++v) fine = fine && (fabsf(acc[i][j][v]) < __builtin_inff() || n + 16 * j + 4 * lg + v >= g.n);
        if (__all(fine || m + 16 * i + li >= g.m)) continue;
        float4_t again[FN];
#pragma unroll
        for (int j = 0; j < FN; ++j) again[j] = float4_t{0.f, 0.f, 0.f, 0.f};
        uint4_t p, q[FN];
        auto load = [&](int64_t k) {                                     // (sixteen k: four of a lane, the same ones of both operands)
            p = four_of<PX>((const float*)g.p, g.ld_p, min(m + 16 * i + li, g.m - 1), k + 4 * lg, k_last);
#pragma unroll
            for (int j = 0; j < FN; ++j) q[j] = four_of<QX>((const float*)g.q, g.ld_q, min(n + 16 * j + li, g.n - 1), k + 4 * lg, k_last);
        };
        load(k_first);
#pragma unroll 1
        for (int64_t k = k_first; k < k_last; k += 16) {
            const uint4_t b = p;
            uint4_t a[FN];
#pragma unroll
            for (int j = 0; j < FN; ++j) a[j] = q[j];
            load(k + 16);
#pragma unroll
            for (int c = 0; c < 4; ++c)
#pragma unroll
                for (int j = 0; j < FN; ++j) again[j] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a[j][c]), __uint_as_float(b[c]), again[j], 0, 0, 0);
        }
#pragma unroll
        for (int j = 0; j < FN; ++j)
#pragma unroll
            for (int v = 0; v < 4; ++v) acc[i][j][v] = fabsf(acc[i][j][v]) < __builtin_inff() ? acc[i][j][v] : again[j][v];
    }
}

// What a wavefront does with its WC columns of sums from (m, n) on: partial ones go to the work space, others through the epilogue.
// They pass through its part of LDS (`lds`, room for PR rows), from the matrix instructions' order into rows, so that the
// residual is read and the output written in whole lines.  The residual of PR rows is under way while their sums are turned: one after the
// other, its pieces would wait for memory each (bf16 8192^3, four rows at a time: 889 us).  Wavefronts at the last
// columns, with pieces of less than eight, take them one by one.
template <int N> __device__ __forceinline__ void activate_all(float8_t (&v)[N], int32_t act) {
    auto all = [&](auto f) {
#pragma unroll
        for (int u = 0; u < N; ++u) v[u] = each(v[u], f);
    };
    if (act == LF_ACT_RELU) all([](float z) { return relu(z); });
    else if (act == LF_ACT_GELU) all([](float z) { return gelu<false>(z); });
    else if (act == LF_ACT_SILU) all([](float z) { return silu<false>(z); });
}
// Where four columns, from 4 c on, of a row of WC turned sums stand: even c first, then odd ones, so that lanes that read every second one lie in
// different banks, as do those that write one c of eight rows.
template <int WC> __device__ __forceinline__ int turned(int row, int c) { return row * (WC / 4) + (((c & 1) * (WC / 8) + (c >> 1)) ^ (row & 7)); }
// What the epilogue needs of a tile's rows and columns, loaded before the first operands and kept in LDS: at the end each would be a wait.
template <int TM, int TN> struct Vectors {
    float bias[TN], w_scale[TN], x_scale[TM];
    struct Loaded { float b, w, x; };
    // (by 256 threads)
    static __device__ __forceinline__ Loaded load(const Product& g, int64_t m0, int64_t n0) {
        const int t = threadIdx.x;
        Loaded l{0.f, 1.f, 1.f};
        if (g.part) return l;
        if (t < TN && n0 + t < g.n) {
            if (g.e.bias) {
                if (g.e.bias_dtype == LF_DTYPE_F32) l.b = ((const float*)g.e.bias)[n0 + t];
                else if (g.e.bias_dtype == LF_DTYPE_BF16) l.b = (float)((const __bf16*)g.e.bias)[n0 + t];
                else l.b = (float)((const _Float16*)g.e.bias)[n0 + t];
            }
            if (g.e.w_scale) l.w = g.e.w_scale[n0 + t];
        }
        if (g.e.x_scale && t < TM && m0 + t < g.m) l.x = g.e.x_scale[m0 + t];
        return l;
    }
    __device__ __forceinline__ void keep(const Loaded& l) {
        const int t = threadIdx.x;
        if (t < TN) {
            bias[t] = l.b;
            w_scale[t] = l.w;
        }
        if (t < TM) x_scale[t] = l.x;
    }
};
// (m0, n0): of the tile that `vec` is of
template <int FM, int FN, int PR, typename Acc, typename Vec>
__device__ __forceinline__ void leave(const Product& g, const Acc (&acc)[FM][FN], uint4_t* lds, const Vec& vec, int64_t m0, int64_t n0, int row0, int col0) {
    constexpr int WC = 16 * FN, LANES = WC / 8, AT_ONCE = 64 / LANES, U = PR / AT_ONCE, PHASES = FM * 16 / PR;
    constexpr bool INT = std::is_same_v<Acc, int4v>;
    static_assert(FM * 16 % PR == 0 && PR % AT_ONCE == 0 && PHASES <= 4, "");
    const int lane = threadIdx.x & 63, li = lane & 15, lg = lane >> 4;
    const int mine = lane / LANES, piece = lane % LANES;
    const int64_t m = m0 + row0, n = n0 + col0 + piece * 8;
    const int count = (int)max((int64_t)0, min((int64_t)8, g.n - n));
    const Epilogue& e = g.e;
    const bool whole = __all(count == 0 || count == 8) && !g.part;
    float8_t bias, ws;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        bias[i] = vec.bias[col0 + piece * 8 + i];
        ws[i] = vec.w_scale[col0 + piece * 8 + i];
    }
    auto place = [&](int row, int h) { return lds + turned<WC>(row, 2 * piece + h); };
    auto sums = [&](int row) {
        const uint4_t a = *place(row, 0), b = *place(row, 1);
        const uint32_t w[8] = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
        float8_t v;
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(w[i]);
        return v;
    };
    auto phase = [&](auto number) {
        constexpr int FIRST = decltype(number)::value * PR;
        const int64_t top = m + FIRST + mine;                                     // the lane's first row
        uint4_t raw[U][2];
        if (whole && e.res && count) {
            const int size = e.res_dtype == LF_DTYPE_F32 ? 4 : 2;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const char* src = (const char*)e.res + (min(top + u * AT_ONCE, g.m - 1) * e.ld_res + n) * size;
                raw[u][0] = load16((const uint16_t*)src);
                if (size == 4) raw[u][1] = load16((const uint16_t*)src + 8);
            }
        }
#pragma unroll
        for (int i = 0; i < PR / 16; ++i)
#pragma unroll
            for (int j = 0; j < FN; ++j) {
                const int row = 16 * i + li, c = 4 * j + lg;
                lds[turned<WC>(row, c)] = __builtin_bit_cast(uint4_t, acc[FIRST / 16 + i][j]);
            }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        if (__builtin_expect(g.part != nullptr, 0)) {
#pragma unroll 2
            for (int row = mine; row < PR; row += AT_ONCE)
                if (m + FIRST + row < g.m && count) store_upto8((float*)g.part + ((int64_t)blockIdx.y * g.m + m + FIRST + row) * g.n + n, sums(row), count);
        } else if (__builtin_expect(whole, 1)) {
            // What follows the sums and comes before the residual, in a lane's own places of LDS: a loop, since its code is long and would be read
            // from memory for every tile if it stood there sixteen times (gelu: 44 us of the 285 of an e4m3 product of 16k x 4k x 4k, 25 as a loop)
            constexpr int H = U < 4 ? U : 4;
            const bool first_pass = INT || e.x_scale || e.z || e.act != LF_ACT_NONE;
            auto pass = [&](auto rows, auto act) {
                constexpr int N = decltype(rows)::value;
#pragma unroll 1
                for (int r0 = mine; r0 < PR; r0 += N * AT_ONCE) {
                    float8_t v[N];
#pragma unroll
                    for (int u = 0; u < N; ++u) {
                        v[u] = sums(r0 + u * AT_ONCE);
                        if constexpr (INT)
#pragma unroll
                            for (int i = 0; i < 8; ++i) v[u][i] = (float)__float_as_int(v[u][i]);
                        if (e.x_scale) v[u] = v[u] * vec.x_scale[row0 + FIRST + r0 + u * AT_ONCE] * ws;
                        v[u] += bias;
                        const int64_t row = m + FIRST + r0 + u * AT_ONCE;
                        if (e.z && row < g.m && count) store_upto8(e.z, row * e.ld_z + n, e.z_dtype, v[u], 8);
                    }
                    act(v);
#pragma unroll
                    for (int u = 0; u < N; ++u) {
                        *place(r0 + u * AT_ONCE, 0) = __builtin_bit_cast(uint4_t, float4_t{v[u][0], v[u][1], v[u][2], v[u][3]});
                        *place(r0 + u * AT_ONCE, 1) = __builtin_bit_cast(uint4_t, float4_t{v[u][4], v[u][5], v[u][6], v[u][7]});
                    }
                }
            };
            // (gelu and silu of float32 outputs are longer still: a row at a time.  What is expected, here and above, is for the order in memory: the
            // code that large products run has to stay in the instruction cache; with this pass in its midst e4m3 16k x 4k x 4k took 10 to 20 us more)
            if (__builtin_expect(e.act & kActFine, 0)) pass(std::integral_constant<int, 1>{}, [&](float8_t (&v)[1]) { v[0] = activate_fine(v[0], e.act); });
            else if (first_pass) pass(std::integral_constant<int, H>{}, [&](float8_t (&v)[H]) { activate_all(v, e.act); });
#pragma unroll
            for (int u0 = 0; u0 < U; u0 += H) {
                float8_t v[H];
#pragma unroll
                for (int u = 0; u < H; ++u) {
                    v[u] = sums(mine + (u0 + u) * AT_ONCE);
                    if (!first_pass) v[u] += bias;
                }
                if (e.res)
                    with_type(e.res_dtype, [&](auto t) {
                        using R = decltype(t);
#pragma unroll
                        for (int u = 0; u < H; ++u) {
                            if constexpr (sizeof(R) == 4) {
                                const float4_t a = __builtin_bit_cast(float4_t, raw[u0 + u][0]), b = __builtin_bit_cast(float4_t, raw[u0 + u][1]);
                                v[u] += float8_t{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
                            } else {
                                v[u] += __builtin_convertvector(__builtin_bit_cast(typename Eight<R>::vec, raw[u0 + u][0]), float8_t);
                            }
                        }
                    });
                if (count)
                    with_type(e.y_dtype, [&](auto t) {
                        using Y = decltype(t);
#pragma unroll
                        for (int u = 0; u < H; ++u)
                            if (top + (u0 + u) * AT_ONCE < g.m) store8((Y*)e.y + (top + (u0 + u) * AT_ONCE) * e.ld_y + n, v[u], e.stream);
                    });
            }
        } else {
#pragma unroll 1
            for (int row = mine; row < PR; row += AT_ONCE) {
                float8_t v = sums(row);
                if constexpr (INT)
#pragma unroll
                    for (int i = 0; i < 8; ++i) v[i] = (float)__float_as_int(v[i]);
                if (m + FIRST + row < g.m && count) finish(e, m + FIRST + row, n, count, v);
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    };
    phase(std::integral_constant<int, 0>{});
    if constexpr (PHASES > 1) phase(std::integral_constant<int, 1>{});
    if constexpr (PHASES > 2) phase(std::integral_constant<int, 2>{});
    if constexpr (PHASES > 3) phase(std::integral_constant<int, 3>{});
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
__global__ void __launch_bounds__(64 * WM * WN, TM == 128 ? 2 : 4)
product_kernel(Product g) {
    constexpr int THREADS = 64 * WM * WN, FM = TM / WM / 16, FN = TN / WN / 16;
    using Acc = typename Elem<T>::Acc;
    using StageP = Stage<T, PX, TM, THREADS>;
    using StageQ = Stage<T, QX, TN, THREADS>;
    constexpr int PL = StageP::kPlanes, PC = StageP::kPieces, KS = StageP::kStep;
    // float32 takes three planes: one buffer, so that a CU holds two workgroups, one of which multiplies while the other stores
    constexpr int NB = PL == 3 ? 1 : 2;
    constexpr int SP = PL * StageP::kSlots, SQ = PL * StageQ::kSlots;
    __shared__ uint4_t s_all[NB * (SP + SQ)];
    uint4_t *const s_p = s_all, *const s_q = s_all + NB * SP;
    __shared__ Vectors<TM, TN> s_vec;
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
    const int row_p = wm * (TM / WM) + li, row_q = wn * (TN / WN) + li;
    auto multiply = [&](const uint4_t* sp, const uint4_t* sq) {
        if constexpr (PL == 3) {
            // a step is one 32-deep instruction, for six pairs of planes
            uint4_t a[3][FN];
#pragma unroll
            for (int p = 0; p < 3; ++p)
#pragma unroll
                for (int j = 0; j < FN; ++j) a[p][j] = sq[p * StageQ::kSlots + slot<PC>(row_q + j * 16, lg)];
#pragma unroll
            for (int i = 0; i < FM; ++i) {
                uint4_t b[3];
#pragma unroll
                for (int p = 0; p < 3; ++p) b[p] = sp[p * StageP::kSlots + slot<PC>(row_p + i * 16, lg)];
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
                for (int h = 0; h < 2; ++h) a[j][h] = sq[slot<PC>(row_q + j * 16, 4 * h + lg)];
#pragma unroll
            for (int i = 0; i < FM; ++i) {
                uint4_t b[2];
#pragma unroll
                for (int h = 0; h < 2; ++h) b[h] = sp[slot<PC>(row_p + i * 16, 4 * h + lg)];
#pragma unroll
                for (int j = 0; j < FN; ++j) acc[i][j] = mma_e4m3(a[j][0], a[j][1], b[0], b[1], acc[i][j]);
            }
        } else {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                uint4_t a[FN];
#pragma unroll
                for (int j = 0; j < FN; ++j) a[j] = sq[slot<PC>(row_q + j * 16, 4 * h + lg)];
#pragma unroll
                for (int i = 0; i < FM; ++i) {
                    const uint4_t b = sp[slot<PC>(row_p + i * 16, 4 * h + lg)];
#pragma unroll
                    for (int j = 0; j < FN; ++j) acc[i][j] = mma(a[j], b, acc[i][j], T{});
                }
            }
        }
    };

    const int64_t steps = k_last > k_first ? (k_last - k_first + KS - 1) / KS : 0;
    const auto vectors = s_vec.load(g, m0, n0);
    if (steps > 0) {
        StageP p;
        StageQ q;
        auto load = [&](int64_t s) {
            const int64_t k = k_first + s * KS;
            p.template load<false>((const T*)g.p, g.ld_p, m0, g.m, k, g.k, k_last - k, tid);
            q.template load<false>((const T*)g.q, g.ld_q, n0, g.n, k, g.k, k_last - k, tid);
        };
        auto store = [&](int64_t s, int buffer) {
            const int64_t k = k_first + s * KS;
            p.store(s_p + buffer * SP, g.ld_p, m0, g.m, k, g.k, k_last - k, tid);
            q.store(s_q + buffer * SQ, g.ld_q, n0, g.n, k, g.k, k_last - k, tid);
        };
        p.template load<true>((const T*)g.p, g.ld_p, m0, g.m, k_first, g.k, k_last - k_first, tid);
        q.template load<true>((const T*)g.q, g.ld_q, n0, g.n, k_first, g.k, k_last - k_first, tid);
        s_vec.keep(vectors);
        if constexpr (NB == 1) {
            for (int64_t s = 0; s < steps; ++s) {
                store(s, 0);
                __syncthreads();
                if (s + 1 < steps) load(s + 1);
                multiply(s_p, s_q);
                __syncthreads();
            }
        } else {
            store(0, 0);
            if (steps > 1) load(1);
            __syncthreads();
            for (int64_t s = 0; s < steps; ++s) {
                const int now = (int)(s & 1);
                multiply(s_p + now * SP, s_q + now * SQ);
                if (s + 1 < steps) {
                    store(s + 1, now ^ 1);
                    if (s + 2 < steps) load(s + 2);
                }
                __syncthreads();
            }
        }
    }

    if (steps <= 0) {
        s_vec.keep(vectors);
        __syncthreads();
    }
    // (the last step is behind a barrier: LDS is free)
    constexpr int SLOTS = NB * PL * (StageP::kSlots + StageQ::kSlots) / (WM * WN), WHOLE = FM * 16, FIT = SLOTS / (FN * 4);
    constexpr int PR = 32;                       // (64 would take the registers of the CU's second workgroup)
    static_assert(PR <= FIT && WHOLE % PR == 0, "");
    uint4_t* mine = s_all + wave * SLOTS;
    const int row0 = wm * (TM / WM), col0 = wn * (TN / WN);
    if constexpr (PL == 3) repair<PX, QX>(g, acc, m0 + row0, n0 + col0, k_first, k_last);
    leave<FM, FN, PR>(g, acc, mine, s_vec, m0, n0, row0, col0);
}

// ---------------------------------------------------------------------------- the tiled product, large tiles

// A tile of 256 x 256 for operands whose pieces of 16 bytes are aligned: four wavefronts of 128 x 128 outputs, which read 32 KB of LDS for
// 4 x 2 MB of products a step, half of what eight of 128 x 64 read.  Operands go from memory into LDS without registers in between (64 lanes
// x 16 bytes to consecutive addresses; the order of the pieces there follows from the addresses they are read from).  Operands across k
// lie in LDS as they do in memory and are turned by the transposing LDS load.
// A step: three quarters of P are read during the products of the first quarter; then - behind the only barrier, when the next buffer has
// arrived and this one is read - the next step's Q and first quarter are read, and the step after it is loaded, during the products of the
// others.  The order of the instructions is the one written here: one of these beside every product or two.  (Left to the compiler's scheduler, reads stood
// together and products waited for them: bf16 8192^3 999 us.)
// A last step of less than 128 bytes of k goes through registers, with zeros behind the end.
// Measured: bf16 8192^3 with bias, silu and residual 800 - 850 us by the clock (1290 - 1370 TFLOP/s; a library product without them 802), matrix cores busy for 70 % of the cycles at
// a clock of 1.7 GHz; e4m3 16k x 4k x 4k with gelu and residual 285 - 301, 60 - 80 of them epilogue; bf16 across k 4096 x 4096 x 8192 207 - 242.

template <typename T> struct Frag { uint4_t c[2]; };                      // 64 bytes of k of a row: two pieces of a lane

// The sums fill the 256 accumulation registers of a lane to the last one.  The compiler's own matrix instructions write to other
// registers than they add to and would need spare ones: with none left it moves 400 registers about a step (half the
// speed).  These add in place.  What the compiler knows about its own it does not know about them, so two idle cycles keep
// a move into an operand away from its use, and settle() the last instruction from the reading of its sums.
template <typename T> __device__ __forceinline__ void add_product(typename Elem<T>::Acc& c, const Frag<T>& a, const Frag<T>& b, int half) {
    if constexpr (std::is_same_v<T, e4m3_t>) {
        const int8v x = __builtin_shufflevector(__builtin_bit_cast(int4v, a.c[0]), __builtin_bit_cast(int4v, a.c[1]), 0, 1, 2, 3, 4, 5, 6, 7);
        const int8v y = __builtin_shufflevector(__builtin_bit_cast(int4v, b.c[0]), __builtin_bit_cast(int4v, b.c[1]), 0, 1, 2, 3, 4, 5, 6, 7);
        asm("s_nop 1\n\tv_mfma_f32_16x16x128_f8f6f4 %0, %1, %2, %0" : "+a"(c) : "v"(x), "v"(y));
    } else if constexpr (std::is_same_v<T, int8_t>) {
        asm("s_nop 1\n\tv_mfma_i32_16x16x64_i8 %0, %1, %2, %0" : "+a"(c) : "v"(a.c[half]), "v"(b.c[half]));
    } else if constexpr (std::is_same_v<T, __bf16>) {
        asm("s_nop 1\n\tv_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+a"(c) : "v"(a.c[half]), "v"(b.c[half]));
    } else {
        asm("s_nop 1\n\tv_mfma_f32_16x16x32_f16 %0, %1, %2, %0" : "+a"(c) : "v"(a.c[half]), "v"(b.c[half]));
    }
}
template <typename Acc> __device__ __forceinline__ void settle(Acc (&c)[8]) {
    asm volatile("s_nop 15\n\ts_nop 15" : "+a"(c[0]), "+a"(c[1]), "+a"(c[2]), "+a"(c[3]), "+a"(c[4]), "+a"(c[5]), "+a"(c[6]), "+a"(c[7]));
}

typedef short short4_t __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) short4_t lds_short4;
typedef __attribute__((address_space(3))) uint32_t lds_word;
template <int N> __device__ __forceinline__ uint32_t lds_address(uint4_t (&s)[N]) { return (uint32_t)(uintptr_t)(lds_word*)&s[0]; }

// One operand's tile of ROWS x (a step of k: 128 bytes) on its way from memory to the matrix instructions, for four wavefronts.
template <typename T, bool ACROSS, int ROWS> struct Direct {
    static constexpr int kStep = 128 / sizeof(T), kElems = 16 / sizeof(T);
    static constexpr int kLoads = ROWS / 32;                              // instructions of a wavefront for a step
    // LDS slots from a load instruction to the next.  Across k, 64 bytes more than what it loads: four k read at once lie in different banks
    static constexpr int kLoad = ACROSS ? 68 : 64, kSlots = 4 * kLoads * kLoad;
    static constexpr int kPair = ROWS / 4, kPairs = 64 / kPair;           // across: slots of two k, pairs of a load instruction
    const char* base;                  // of the tile at the step that is loaded next
    int64_t step_bytes;                // from step to step
    uint32_t off[kLoads];              // bytes from there to what this lane reads by the load instructions of its wavefront
    int wave, lane, li, lg;

    // A load instruction reads eight rows (along) or some pairs of k (across); the wavefronts take them in turn.  Along, piece c of row r stands
    // at place c ^ (r & 7) of the row; across, piece c of k stands at place 2 c + (k & 1) of the pair, and pairs that are read at once
    // (see read) are neighbours.  Rows past the end are read for the last ones, and not used.
    // Element of k (along), k (across) that this lane reads by load instruction i.
    __device__ __forceinline__ int at(int i) const {
        if constexpr (!ACROSS) return ((lane & 7) ^ (lane >> 3)) * kElems;
        const int n = kPairs * (wave + 4 * i) + lane / kPair;
        return 2 * ((n & 16) | (n >> 1 & 3) * 4 | (n >> 3 & 1) * 2 | (n & 1)) + (lane & 1);
    }
    __device__ __forceinline__ Direct(const void* p, int64_t ld, int64_t row0, int64_t rows, int64_t k0) {
        lane = threadIdx.x & 63;
        li = lane & 15;
        lg = lane >> 4;
        wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        const uint32_t ld_bytes = (uint32_t)(ld * sizeof(T));
        if constexpr (!ACROSS) {
            base = (const char*)p + (row0 * ld + k0) * sizeof(T);
            step_bytes = 128;
#pragma unroll
            for (int i = 0; i < kLoads; ++i) off[i] = (uint32_t)min((int64_t)(8 * (wave + 4 * i) + (lane >> 3)), rows - 1 - row0) * ld_bytes + at(i) * (int)sizeof(T);
        } else {
            base = (const char*)p + (k0 * ld + row0) * sizeof(T);
            step_bytes = kStep * ld * sizeof(T);
            const uint32_t c = (uint32_t)min((int64_t)(lane % kPair / 2 * 8), rows - 8 - row0) * (int)sizeof(T);
#pragma unroll
            for (int i = 0; i < kLoads; ++i) off[i] = at(i) * ld_bytes + c;
        }
    }
    // Load instruction i of a step, into the array of LDS that begins at `lds`.  (In assembly, since the compiler would have every transposing
    // read wait for all loads.  It has no output in registers; arrived() waits for it.)
    // m0 is declared as written (nothing else here uses it, an access of the compiler's own might); that it belongs to the compiler is known.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
    __device__ __forceinline__ void load(uint32_t lds, int i) const {
        asm volatile("s_add_u32 m0, %2, %3\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off[i]), "s"(base), "s"(wave * (kLoad * 16)), "s"(lds + i * (4 * kLoad * 16))
                     : "memory", "m0", "scc");
    }
#pragma clang diagnostic pop
    __device__ __forceinline__ void load_last(uint4_t* lds, int left) const {
        uint4_t r[kLoads];
        auto count = [&](int i) { return ACROSS ? (at(i) < left ? kElems : 0) : left - at(i); };
#pragma unroll
        for (int i = 0; i < kLoads; ++i) r[i] = part16((const T*)(base + off[i]), count(i));
#pragma unroll
        for (int i = 0; i < kLoads; ++i) lds[(wave + 4 * i) * kLoad + lane] = join16<T>(r[i], count(i));
    }
    // half h of rows `row` .. + 15 of the tile as an operand of the matrix instructions
    __device__ __forceinline__ void read(Frag<T>& f, const uint4_t* lds, int row, int h) const {
        if constexpr (!ACROSS) {
            f.c[h] = lds[(row + li) * 8 + ((4 * h + lg) ^ (li & 7))];
        } else {
            // 16 lanes read 16 rows of four k, lane 4 r + s rows 4 s .. of the r-th, and receive four k of a row each.  The k of a lane are the eight
            // from 8 lg on, as along; the two pairs that a group of lanes reads at once lie beside those of the next group, in other banks.
            auto pair = [&](int n) { return (n / kPairs * kLoad + n % kPairs * kPair) * 16; };
            const char* src = (const char*)lds + pair(2 * lg) + (li & 2) * 16 + (li >> 2 & 1) * 16 + (li & 1) * 8 + (kPairs > 1 ? (li >> 3) * (kPair * 16) : (li >> 3) * (kLoad * 16));
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const uint2_t v = __builtin_bit_cast(uint2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4*)(src + pair(16 * h + 8 * t) + row * 4)));
                f.c[h][2 * t] = v[0];
                f.c[h][2 * t + 1] = v[1];
            }
        }
    }
};
// No load and no access to LDS of this wavefront is under way, and none of the others'.
__device__ __forceinline__ void arrived() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0x70);
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

template <typename T, bool PX, bool QX>
__global__ void __launch_bounds__(256)
wide_kernel(Product g) {
    using Acc = typename Elem<T>::Acc;
    using F = Frag<T>;
    constexpr int KS = 128 / sizeof(T);
    // (arrays of their own: what is read from one must not wait for what is on its way into another)
    __shared__ uint4_t s_p0[Direct<T, PX, 256>::kSlots], s_q0[Direct<T, QX, 256>::kSlots], s_p1[Direct<T, PX, 256>::kSlots], s_q1[Direct<T, QX, 256>::kSlots];
    __shared__ Vectors<256, 256> s_vec;
    int tm, tn;
    tile_of(g, blockIdx.x, tm, tn);
    const int64_t m0 = (int64_t)tm * 256, n0 = (int64_t)tn * 256;
    const int64_t k_first = (int64_t)blockIdx.y * g.k_split, k_last = min(g.k, k_first + g.k_split);
    using DP = Direct<T, PX, 256>;
    using DQ = Direct<T, QX, 256>;
    DP P(g.p, g.ld_p, m0, g.m, k_first);
    DQ Q(g.q, g.ld_q, n0, g.n, k_first);
    const int wm = P.wave & 1, wn = P.wave >> 1, row_p = wm * 128, row_q = wn * 128;

    Acc acc[8][8];
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) acc[i][j] = Acc{0, 0, 0, 0};

    constexpr int ROW = std::is_same_v<T, e4m3_t> ? 8 : 16;              // products of a row of instructions: eight, or twice eight
    F p[8], q0[8], q1[8];
    auto product = [&](int n, const F (&q)[8]) {                          // the n-th of a step
        const int i = n / ROW, h = n % ROW / 8, j = n % 8;
        add_product<T>(acc[i][j], q[j], p[i], h);
    };
    auto read_p = [&](const uint4_t* s, int n) { P.read(p[n / 2], s, row_p + n / 2 * 16, n % 2); };
    auto read_q = [&](const uint4_t* s, F (&q)[8], int n) { Q.read(q[n / 2], s, row_q + n / 2 * 16, n % 2); };
    auto load = [&](uint32_t sp, uint32_t sq, int n) {
        if (n < 8) P.load(sp, n); else Q.load(sq, n - 8);
    };
    const uint32_t at_p0 = lds_address(s_p0), at_q0 = lds_address(s_q0), at_p1 = lds_address(s_p1), at_q1 = lds_address(s_q1);

    const int64_t length = k_last > k_first ? k_last - k_first : 0, steps = length / KS;
    const int left = (int)(length - steps * KS);
    const char *const p_first = P.base, *const q_first = Q.base;
    auto go_to = [&](int64_t s) {
        P.base = p_first + s * P.step_bytes;
        Q.base = q_first + s * Q.step_bytes;
    };
    const auto vectors = s_vec.load(g, m0, n0);
    if (steps <= 0) s_vec.keep(vectors);
    if (steps > 0) {
        // (a load past the last step loads that one again, where nobody reads it)
        auto both = [&](uint32_t sp, uint32_t sq) {
#pragma unroll
            for (int n = 0; n < 16; ++n) load(sp, sq, n);
        };
        both(at_p0, at_q0);
        s_vec.keep(vectors);
        arrived();
        go_to(min((int64_t)1, steps - 1));
        both(at_p1, at_q1);
        go_to(min((int64_t)2, steps - 1));
#pragma unroll
        for (int n = 0; n < 16; ++n) read_q(s_q0, q0, n);
#pragma unroll
        for (int n = 0; n < 4; ++n) read_p(s_p0, n);
        auto step = [&](int64_t s, const uint4_t* sp, uint32_t at_p, uint32_t at_q, const uint4_t* next_p, const uint4_t* next_q, const F (&q)[8], F (&next)[8]) {
#pragma unroll
            for (int n = 0; n < 2 * ROW; ++n) {
                product(n, q);
                if (n % (ROW / 8) == 0 && n / (ROW / 8) < 12) read_p(sp, 4 + n / (ROW / 8));
                __builtin_amdgcn_sched_barrier(0);
            }
            arrived();
#pragma unroll
            for (int n = 0; n < 6 * ROW; ++n) {
                product(2 * ROW + n, q);
                // 16 loads in two thirds of the time: closer, they queue up and products wait (791 -> 761 us, 8192^3 without residual), later they arrive late
                if (n < 4 * ROW && n % (ROW / 4) == 0) load(at_p, at_q, n / (ROW / 4));
                if (n % (ROW / 4) == 1) {
                    const int r = n / (ROW / 4);
                    if (r < 16) read_q(next_q, next, r);
                    else if (r < 20) read_p(next_p, r - 16);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
            if (s + 3 < steps) {
                P.base += P.step_bytes;
                Q.base += Q.step_bytes;
            }
        };
        int64_t s = 0;
        for (; s + 1 < steps; s += 2) {
            step(s, s_p0, at_p0, at_q0, s_p1, s_q1, q0, q1);
            step(s + 1, s_p1, at_p1, at_q1, s_p0, s_q0, q1, q0);
        }
        if (s < steps) step(s, s_p0, at_p0, at_q0, s_p1, s_q1, q0, q1);
        arrived();
    }
    if (left > 0) {
        go_to(steps);
        P.load_last(s_p0, left);
        Q.load_last(s_q0, left);
        __syncthreads();
#pragma unroll
        for (int n = 0; n < 16; ++n) {
            read_q(s_q0, q0, n);
            read_p(s_p0, n);
        }
#pragma unroll
        for (int n = 0; n < 8 * ROW; ++n) product(n, q0);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) settle(acc[i]);
    __syncthreads();
    uint4_t* mine = P.wave == 0 ? s_p0 : P.wave == 1 ? s_q0 : P.wave == 2 ? s_p1 : s_q1;
    leave<8, 8, 64>(g, acc, mine, s_vec, m0, n0, row_p, row_q);
}

// ---------------------------------------------------------------------------- the tiled product, aligned operands, small tiles

// The same way into LDS for tiles of 128 x 128 and 64 x 64: a barrier a step, the operands of the next one read during the products
// of this one, the order of the instructions left to the compiler.  With two buffers a CU holds two (four) workgroups, whose wavefronts
// cover one another's waits; where there are too few workgroups for that, four buffers have more steps on their way.
// bf16 2000^3 28 us, through registers (rows at odd addresses) 40; the tile of 64 and that of 128: see step_us().
template <typename T, bool PX, bool QX, int TILE, int BUFFERS>
__global__ void __launch_bounds__(256, BUFFERS == 4 ? 1 : TILE == 128 ? 2 : 4)
direct_kernel(Product g) {
    using Acc = typename Elem<T>::Acc;
    using DP = Direct<T, PX, TILE>;
    using DQ = Direct<T, QX, TILE>;
    constexpr int KS = 128 / sizeof(T), FR = TILE / 32, SB = DP::kSlots + DQ::kSlots;
    __shared__ uint4_t s[BUFFERS * SB];
    __shared__ Vectors<TILE, TILE> s_vec;
    int tm, tn;
    tile_of(g, blockIdx.x, tm, tn);
    const int64_t m0 = (int64_t)tm * TILE, n0 = (int64_t)tn * TILE;
    const int64_t k_first = (int64_t)blockIdx.y * g.k_split, k_last = min(g.k, k_first + g.k_split);
    DP P(g.p, g.ld_p, m0, g.m, k_first);
    DQ Q(g.q, g.ld_q, n0, g.n, k_first);
    const int row_p = (P.wave & 1) * (TILE / 2), row_q = (P.wave >> 1) * (TILE / 2);
    Acc acc[FR][FR];
#pragma unroll
    for (int i = 0; i < FR; ++i)
#pragma unroll
        for (int j = 0; j < FR; ++j) acc[i][j] = Acc{0, 0, 0, 0};
    struct Operands { Frag<T> p[FR], q[FR]; };
    auto read = [&](Operands& o, const uint4_t* tile) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < FR; ++i) {
                Q.read(o.q[i], tile + DP::kSlots, row_q + i * 16, h);
                P.read(o.p[i], tile, row_p + i * 16, h);
            }
    };
    auto multiply = [&](const Operands& o) {
#pragma unroll
        for (int h = 0; h < (std::is_same_v<T, e4m3_t> ? 1 : 2); ++h)
#pragma unroll
            for (int i = 0; i < FR; ++i)
#pragma unroll
                for (int j = 0; j < FR; ++j) {
                    if constexpr (std::is_same_v<T, e4m3_t>) acc[i][j] = mma_e4m3(o.q[j].c[0], o.q[j].c[1], o.p[i].c[0], o.p[i].c[1], acc[i][j]);
                    else acc[i][j] = mma(o.q[j].c[h], o.p[i].c[h], acc[i][j], T{});
                }
    };
    const uint32_t at = lds_address(s);
    auto load = [&](uint32_t buffer) {
#pragma unroll
        for (int i = 0; i < DP::kLoads; ++i) P.load(at + buffer, i);
#pragma unroll
        for (int i = 0; i < DQ::kLoads; ++i) Q.load(at + buffer + DP::kSlots * 16, i);
    };
    const int64_t length = k_last > k_first ? k_last - k_first : 0, steps = length / KS;
    const int left = (int)(length - steps * KS);
    constexpr int ON_THE_WAY = (BUFFERS - 2) * (DP::kLoads + DQ::kLoads), SIZE = SB * 16;
    static_assert(ON_THE_WAY < 64, "");
    const char *const p_first = P.base, *const q_first = Q.base;
    const auto vectors = s_vec.load(g, m0, n0);
    if (steps <= 0) s_vec.keep(vectors);
    if (steps > 0) {
        // (a load past the last step loads that one again, where nobody reads it: the number under way is always the same)
        auto advance = [&](int64_t next) {
            if (next < steps) {
                P.base += P.step_bytes;
                Q.base += Q.step_bytes;
            }
        };
        auto wait = [] {
            asm volatile("" ::: "memory");
            __builtin_amdgcn_s_waitcnt((ON_THE_WAY & 15) | (ON_THE_WAY >> 4) << 14 | 0x70);
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
        };
#pragma unroll
        for (int b = 0; b < BUFFERS - 1; ++b) {
            load(b * SIZE);
            advance(b + 1);
        }
        s_vec.keep(vectors);
        wait();
        load((BUFFERS - 1) * SIZE);
        advance(BUFFERS);
        Operands even, odd;
        read(even, s);
        uint32_t now = 0;                                                 // bytes to the buffer of the step whose operands are in registers
        auto step = [&](int64_t t, const Operands& o, Operands& next) {
            const uint32_t then = now == (BUFFERS - 1) * SIZE ? 0 : now + SIZE;
            wait();                                                       // the next step's buffer has arrived, this one's has been read
            load(now);
            advance(t + BUFFERS + 1);
            read(next, s + then / 16);
            multiply(o);
            now = then;
        };
        int64_t t = 0;
        for (; t + 1 < steps; t += 2) {
            step(t, even, odd);
            step(t + 1, odd, even);
        }
        if (t < steps) multiply(even);
    }
    if (left > 0) {
        P.base = p_first + steps * P.step_bytes;
        Q.base = q_first + steps * Q.step_bytes;
        arrived();
        P.load_last(s, left);
        Q.load_last(s + DP::kSlots, left);
        arrived();
        Operands o;
        read(o, s);
        multiply(o);
    }
    arrived();
    leave<FR, FR, TILE / 2 < 32 ? TILE / 2 : 32>(g, acc, s + P.wave * (SB / 2), s_vec, m0, n0, row_p, row_q);
}

template <typename T, bool PX, bool QX> ProductFn kernel_of(int tile, bool aligned, bool deep) {
    if constexpr (!std::is_same_v<T, float>)
        if (tile == kWideTile) return wide_kernel<T, PX, QX>;
    if constexpr (!std::is_same_v<T, float>)
        if (aligned) return tile == 128 ? (deep ? direct_kernel<T, PX, QX, 128, 4> : direct_kernel<T, PX, QX, 128, 2>)
                               : deep ? direct_kernel<T, PX, QX, 64, 4> : direct_kernel<T, PX, QX, 64, 2>;
    return tile == 128 ? product_kernel<T, PX, QX, 128, 128, 2, 2> : product_kernel<T, PX, QX, 64, 64, 2, 2>;
}
template <typename T> ProductFn kernel_of(bool px, bool qx, int tile, bool aligned, bool deep) {
    return px ? kernel_of<T, true, true>(tile, aligned, deep) : qx ? kernel_of<T, false, true>(tile, aligned, deep) : kernel_of<T, false, false>(tile, aligned, deep);
}

}  // namespace
