// What the norms of rows of features (lf_norm.hip, lf_layer_norm.hip) share: how a row lies in the registers of some threads, sums over them,
// its way into 8 bits.
#pragma once
#include <algorithm>

#include "lf_dense.h"

namespace {

using namespace lf;

constexpr int64_t kMaxDim = 1 << 24;

template <int G> __device__ __forceinline__ float dpp_add(float v) {
    // within 16 lanes by moves of the ALU, beyond that through the permute network
    auto mov = [](float x, auto ctrl) { return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), decltype(ctrl)::value, 0xf, 0xf, true)); };
    if constexpr (G >= 2) v += mov(v, std::integral_constant<int, 0xB1>{});     // lane ^ 1
    if constexpr (G >= 4) v += mov(v, std::integral_constant<int, 0x4E>{});     // lane ^ 2
    if constexpr (G >= 8) v += mov(v, std::integral_constant<int, 0x141>{});    // the other half of 8
    if constexpr (G >= 16) v += mov(v, std::integral_constant<int, 0x140>{});   // the other half of 16
    if constexpr (G >= 32) v += __shfl_xor(v, 16);
    if constexpr (G >= 64) v += __shfl_xor(v, 32);
    return v;
}
// The largest of non-negative floats, by their bits: a NaN is larger than infinity and stays.
template <int G> __device__ __forceinline__ uint32_t lanes_max(uint32_t v) {
#pragma unroll
    for (int o = 1; o < (G < 64 ? G : 64); o *= 2) v = max(v, (uint32_t)__shfl_xor((int)v, o));
    return v;
}

// Sums (and maximum) over the G threads of a row; `s` holds 2 G / 64 words where G > 64.
template <int G, bool MAX> __device__ __forceinline__ void row_reduce(float& a, float& b, uint32_t& m, float* s) {
    a = dpp_add<(G < 64 ? G : 64)>(a);
    if constexpr (MAX) m = lanes_max<G>(m); else b = dpp_add<(G < 64 ? G : 64)>(b);
    if constexpr (G > 64) {
        constexpr int W = G / 64;
        __syncthreads();                                   // the row before has been read
        if ((threadIdx.x & 63) == 0) {
            s[threadIdx.x >> 6] = a;
            s[W + (threadIdx.x >> 6)] = MAX ? __uint_as_float(m) : b;
        }
        __syncthreads();
        a = 0.f;
        if constexpr (MAX) m = 0; else b = 0.f;
#pragma unroll
        for (int w = 0; w < W; ++w) {
            a += s[w];
            if constexpr (MAX) m = max(m, __float_as_uint(s[W + w])); else b += s[W + w];
        }
    }
}

// Where a thread's piece c of a row stands, and from which of its elements on it counts.
struct Piece {
    int at, first;                                          // first = 8: the piece lies past the row
    __device__ __forceinline__ Piece(int col, int dim) : at(min(col, dim - 8)), first(col < dim ? col - min(col, dim - 8) : 8) {}
};
template <typename T> __device__ __forceinline__ float8_t load_piece(const T* row, const Piece& p, int dim) {
    return dim >= 8 ? load8(row + p.at) : load_upto8(row, dim);
}
template <typename T> __device__ __forceinline__ void store_piece(T* row, const Piece& p, int dim, float8_t v, bool stream) {
    if (dim >= 8) store8(row + p.at, v, stream); else store_upto8(row, v, dim);
}
__device__ __forceinline__ float8_t load_piece(const void* base, int64_t at, int32_t dtype, const Piece& p, int dim) {
    return dim >= 8 ? load_upto8(base, at + p.at, dtype, 8) : load_upto8(base, at, dtype, dim);
}
__device__ __forceinline__ void store_piece(void* base, int64_t at, int32_t dtype, const Piece& p, int dim, float8_t v, bool stream) {
    if (dim >= 8) store_upto8(base, at + p.at, dtype, v, 8, stream); else store_upto8(base, at, dtype, v, dim);
}
// For rows shorter than eight the one piece counts from 0, and its elements past the row are zeros.
__device__ __forceinline__ Piece piece_of(int col, int dim) {
    Piece p(col, dim);
    if (dim < 8) { p.at = 0; p.first = col == 0 ? 0 : 8; }
    return p;
}

// The power of two that a row is to be multiplied by, from the mean of its squares plus eps; 1: as it is.
constexpr float kTiny = 0x1p-100f;
__device__ __forceinline__ float rescale(float ms) { return ms >= kTiny && ms < __builtin_inff() ? 1.f : ms < kTiny ? 1.f / kTiny : kTiny; }

// A row's way into 8 bits, from the largest magnitude of t.  A maximum whose reciprocal would overflow is scaled up with its row;
// Inf and NaN leave a scale of NaN.
struct Eighth {
    float top8, amax, up, to;
    bool fine, e4m3;
    __device__ __forceinline__ Eighth(uint32_t top, int32_t dtype) {
        e4m3 = dtype == LF_DTYPE_E4M3;
        top8 = e4m3 ? 448.f : 127.f;
        amax = __uint_as_float(top);
        up = amax < 1e-30f ? 0x1p64f : 1.f;
        fine = top < 0x7f800000u;
        to = top == 0 || !fine ? 0.f : top8 / (amax * up);
    }
    __device__ __forceinline__ float scale(float s) const { return !fine ? __uint_as_float(0x7fc00000u) : amax == 0.f ? 0.f : amax * s / top8; }
    __device__ __forceinline__ void store(uint8_t* q, float8_t t, int n, bool stream) const {
#pragma unroll
        for (int i = 0; i < 8; ++i) t[i] = fminf(fmaxf(t[i] * up * to, -top8), top8);        // (NaN goes to -top8)
        const uint2_t b = e4m3 ? to_e4m3(t) : to_int8(t);
        if (n >= 8) {
            typedef uint32_t any2_t __attribute__((ext_vector_type(2), aligned(1)));
            if (stream) __builtin_nontemporal_store(b, reinterpret_cast<any2_t __attribute__((address_space(1)))*>(reinterpret_cast<uintptr_t>(q)));
            else *reinterpret_cast<any2_t*>(q) = b;
        } else {
            for (int i = 0; i < n; ++i) q[i] = (uint8_t)(b[i >> 2] >> (8 * (i & 3)));
        }
    }
};

// Threads that hold a row, and pieces of eight of each (more than two: the kernels for long rows).
struct Shape { int group, pieces; };
inline Shape shape_of(int64_t dim) {
    const int g = dim <= 64 ? 8 : dim <= 128 ? 16 : dim <= 256 ? 32 : dim <= 1024 ? 64 : dim <= 4096 ? 256 : dim <= 8192 ? 512 : 1024;
    return {g, (int)ceil_div(dim, 8 * g)};
}
inline unsigned workgroups(int64_t rows, Shape s, int most) {
    const int threads = std::max(s.group, 256);
    return (unsigned)std::min<int64_t>(ceil_div(rows, threads / s.group), (int64_t)most * 256 / threads);
}

int check_rows(const char* what, int64_t rows, int64_t dim, const void* p, int64_t ld, int32_t dtype) {
    LF_REQUIRE(p || rows == 0, LF_ERR_INVALID, "%s: null pointer", what);
    LF_REQUIRE(ld >= dim || rows <= 1, LF_ERR_INVALID, "%s: rows of %lld elements, %lld apart", what, (long long)dim, (long long)ld);
    LF_REQUIRE((uintptr_t)p % dtype_bytes(dtype) == 0, LF_ERR_INVALID, "%s: not aligned to its elements", what);
    return LF_OK;
}
int check_shape(int64_t rows, int64_t dim) {
    LF_REQUIRE(rows >= 0 && dim >= 1, LF_ERR_INVALID, "bad shape %lld x %lld", (long long)rows, (long long)dim);
    LF_REQUIRE(dim <= kMaxDim, LF_ERR_UNSUPPORTED, "rows of at most %lld elements are supported (got %lld)", (long long)kMaxDim, (long long)dim);
    LF_REQUIRE(rows < (1ll << 40), LF_ERR_UNSUPPORTED, "too many rows");
    return LF_OK;
}

}  // namespace
