// What the kernels for dense rows of features (lf_norm.hip, lf_linear.hip) share: element types, loads and
// stores of eight elements at any alignment, activations.
#pragma once
#include <hip/hip_runtime.h>
#include <cstdint>

#include "lf_internal.h"

namespace lf {

typedef float float8_t __attribute__((ext_vector_type(8)));
typedef uint32_t uint4_t __attribute__((ext_vector_type(4)));
typedef uint32_t uint2_t __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));

constexpr bool is_float_dtype(int32_t t) { return t == LF_DTYPE_F32 || t == LF_DTYPE_BF16 || t == LF_DTYPE_F16; }
constexpr bool is_8bit_dtype(int32_t t) { return t == LF_DTYPE_E4M3 || t == LF_DTYPE_I8; }
constexpr int dtype_bytes(int32_t t) { return t == LF_DTYPE_F32 ? 4 : is_8bit_dtype(t) ? 1 : 2; }

// Eight elements at any address that is a multiple of the element's size: the hardware takes 16-byte accesses there, and a
// row of an odd number of 2-byte elements, or a row inside a wider buffer, needs no code of its own.
template <typename T> struct Eight {
    typedef T vec __attribute__((ext_vector_type(8)));
    struct __attribute__((packed, aligned(sizeof(T)))) Any { vec v; };
};
template <typename T> __device__ __forceinline__ float8_t load8(const T* p) {
    return __builtin_convertvector(reinterpret_cast<const typename Eight<T>::Any*>(p)->v, float8_t);
}
// stream: past the caches, which leaves them to what is read again.  Pieces of 32 bytes (float32) would go there in halves, which is
// slower (170k x 128 117 -> 120 us) than through the caches.
template <typename T> __device__ __forceinline__ void store8(T* p, float8_t f, bool stream = false) {
    const typename Eight<T>::vec v = __builtin_convertvector(f, typename Eight<T>::vec);
    if constexpr (sizeof(T) == 2) {
        if (stream) {
            // (through an integer, or the compiler folds the two stores into an ordinary one)
            typedef uint32_t any4_t __attribute__((ext_vector_type(4), aligned(2)));
            __builtin_nontemporal_store(__builtin_bit_cast(uint4_t, v), reinterpret_cast<any4_t __attribute__((address_space(1)))*>(reinterpret_cast<uintptr_t>(p)));
            return;
        }
    }
    reinterpret_cast<typename Eight<T>::Any*>(p)->v = v;
}
// Outputs of this many bytes are stored past the caches: norm of 16k x 4096 into e4m3 90.9 -> 86.2 us, its gradient at 32k x 2048 105.1 -> 102.7,
// e4m3 product of 16k x 4k x 4k 293.5 -> 285.7 (bf16 8192^3: less than its runs differ by).  Smaller ones the next operation may find there.
constexpr int64_t kStreamBytes = 64ll << 20;
// 16 bytes at any address that suits the type
template <typename T> __device__ __forceinline__ uint4_t load16(const T* p) {
    struct __attribute__((packed, aligned(sizeof(T)))) Any { uint4_t v; };
    return reinterpret_cast<const Any*>(p)->v;
}
// The first n elements of them, zeros behind, one by one: loads that nothing waits for.
template <typename T> __device__ __forceinline__ uint4_t load16_each(const T* p, int n) {
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
// The same as eight, four, two bytes and one, where their number has that bit.  In two steps, so that several
// such loads can be under way: part16 leaves what it loads beside each other, join16 puts it together.
template <typename T> __device__ __forceinline__ uint4_t part16(const T* p, int n) {
    constexpr int S = sizeof(T);
    uint4_t r = {0u, 0u, 0u, 0u};
    if (n >= 16 / S) {
        r = load16(p);
    } else if (n > 0) {
        const char* src = (const char*)p;
        const int bytes = n * S;
        struct __attribute__((packed, aligned(S))) Any8 { uint2_t v; };
        struct __attribute__((packed, aligned(S))) Any4 { uint32_t v; };
        struct __attribute__((packed, aligned(S < 2 ? S : 2))) Any2 { uint16_t v; };
        if (bytes & 8) {
            const uint2_t a = reinterpret_cast<const Any8*>(src)->v;
            r[0] = a[0];
            r[1] = a[1];
        }
        if (bytes & 4) r[2] = reinterpret_cast<const Any4*>(src + (bytes & 8))->v;
        if constexpr (S < 4)
            if (bytes & 2) r[3] = reinterpret_cast<const Any2*>(src + (bytes & 12))->v;
        if constexpr (S == 1)
            if (bytes & 1) r[3] |= (uint32_t)(uint8_t)src[bytes & 14] << (bytes & 2 ? 16 : 0);
    }
    return r;
}
template <typename T> __device__ __forceinline__ uint4_t join16(uint4_t r, int n) {
    if (n >= 16 / (int)sizeof(T)) return r;
    const int bytes = n > 0 ? n * (int)sizeof(T) : 0;
    const uint32_t x = bytes & 4 ? r[2] : r[3], y = bytes & 4 ? r[3] : 0;
    return bytes & 8 ? uint4_t{r[0], r[1], x, y} : uint4_t{x, y, 0u, 0u};
}

// 16 bytes without their first d elements, and zeros from the n-th of what is left (any n).
template <typename T> __device__ __forceinline__ uint4_t move16(uint4_t r, int d, int n) {
    constexpr int E = 16 / sizeof(T), BITS = 8 * sizeof(T);
    unsigned __int128 v = __builtin_bit_cast(unsigned __int128, r);
    v = d >= E ? 0 : v >> (d * BITS);
    if (n < E) v = n <= 0 ? 0 : v & (((unsigned __int128)1 << (n * BITS)) - 1);
    return __builtin_bit_cast(uint4_t, v);
}

// The first `n` of eight elements (any n; others read as zero).
template <typename T> __device__ __forceinline__ float8_t load_upto8(const T* p, int n) {
    if constexpr (sizeof(T) == 2) return __builtin_convertvector(__builtin_bit_cast(typename Eight<T>::vec, join16<T>(part16(p, n), n)), float8_t);
    if (n >= 8) return load8(p);
    float8_t f = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (i < n) f[i] = (float)p[i];
    return f;
}
template <typename T> __device__ __forceinline__ void store_upto8(T* p, float8_t f, int n, bool stream = false) {
    if (n >= 8) return store8(p, f, stream);
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (i < n) p[i] = (T)f[i];
}
// The same of a type that is known at run time (one for the whole launch).
__device__ __forceinline__ float8_t load_upto8(const void* p, int64_t at, int32_t dtype, int n) {
    if (dtype == LF_DTYPE_F32) return load_upto8((const float*)p + at, n);
    if (dtype == LF_DTYPE_BF16) return load_upto8((const __bf16*)p + at, n);
    return load_upto8((const _Float16*)p + at, n);
}
__device__ __forceinline__ void store_upto8(void* p, int64_t at, int32_t dtype, float8_t f, int n, bool stream = false) {
    if (dtype == LF_DTYPE_F32) return store_upto8((float*)p + at, f, n);
    if (dtype == LF_DTYPE_BF16) return store_upto8((__bf16*)p + at, f, n, stream);
    return store_upto8((_Float16*)p + at, f, n, stream);
}

__device__ __forceinline__ void store_one(void* p, int64_t at, int32_t dtype, float v) {
    if (dtype == LF_DTYPE_F32) ((float*)p)[at] = v;
    else if (dtype == LF_DTYPE_BF16) ((__bf16*)p)[at] = (__bf16)v;
    else ((_Float16*)p)[at] = (_Float16)v;
}

// Eight values as e4m3 (nearest, ties to even; |v| <= 448 is the caller's, NaN stays NaN).
__device__ __forceinline__ uint2_t to_e4m3(float8_t v) {
    uint2_t r = {0u, 0u};
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        int w = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * h], v[4 * h + 1], 0, false);
        r[h] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(v[4 * h + 2], v[4 * h + 3], w, true);
    }
    return r;
}
// ... and as int8.
__device__ __forceinline__ uint2_t to_int8(float8_t v) {
    uint2_t r = {0u, 0u};
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i >> 2] |= ((uint32_t)(int)rintf(v[i]) & 0xffu) << (8 * (i & 3));
    return r;
}

// exp(c (x + x2)), c x of -128 to 0, c a power of two and x2 less than the last place of x: 2^(c x / ln 2) with what the product's rounding, 1 / ln 2 in 32
// bits and x2 leave, in one more term of exp's series.
__device__ __forceinline__ float exp_of(float x, float x2, float c) {
    const float t = x * (c * 1.44269502f);
    const float rest = fmaf(x2, c * 1.44269502f, fmaf(x, c * 1.92596299e-8f, fmaf(x, c * 1.44269502f, -t)));
    const float e = __builtin_amdgcn_exp2f(t);
    return fmaf(e, rest * 0.693147181f, e);
}
// 1 - Phi(a) for a = |z|, at most 16, and exp(-a^2 / 2) with it.  Their ratio goes from 1/2 at 0 as 0.4 / a: a quotient of polynomials in a, fitted over
// 0 .. 14.5 for the least relative error, so that what gelu leaves of a negative z has its digits too.
// FINE, for float32: degrees 4 and 5, off by 6e-9, at most 20 roundings of 32 bits with those of its evaluation, among them that of a^2,
// which exp would take times a^2 / 2.  For 16 bits: degrees 3 and 4, off by 4e-7, and by up to a^2 2^-24 in exp's argument.
template <bool FINE> __device__ __forceinline__ float normal_tail(float a, float& e) {
    if constexpr (FINE) {
        const float sq = a * a;
        e = exp_of(sq, fmaf(a, a, -sq), -0.5f);
        const float p = fmaf(fmaf(fmaf(fmaf(4.116355848e-3f, a, 4.063350893e-2f), a, 0.1832359274f), a, 0.4382959418f), a, 0.5f);
        const float q = fmaf(fmaf(fmaf(fmaf(fmaf(1.031805421e-2f, a, 0.1018595493f), a, 0.4694727291f), a, 1.202506301f), a, 1.674476865f), a, 1.f);
        return p * __builtin_amdgcn_rcpf(q) * e;
    } else {
        e = __builtin_amdgcn_exp2f(a * a * -0.72134752f);
        const float p = fmaf(fmaf(fmaf(1.717115205e-2f, a, 0.1200515037f), a, 0.3628747862f), a, 0.4999998005f);
        const float q = fmaf(fmaf(fmaf(fmaf(4.304641672e-2f, a, 0.3007297552f), a, 0.9559268397f), a, 1.523614424f), a, 1.f);
        return p * __builtin_amdgcn_rcpf(q) * e;
    }
}
// What the kernels take for an activation: for float32 outputs gelu and silu to their last places (kActFine), for 16 bits with fewer instructions.
// e4m3 16k x 4k x 4k with gelu into float32: 333 us, 312 with those of 16 bits; float32 170k x 128 by 256 138, 129.
constexpr int32_t kActFine = 8;
constexpr int32_t activation_of(int32_t act, int32_t dtype) { return dtype == LF_DTYPE_F32 && (act == LF_ACT_GELU || act == LF_ACT_SILU) ? act | kActFine : act; }
// act(z) and act'(z).  gelu is z Phi(z) with the normal distribution's Phi.
__device__ __forceinline__ float relu(float z) { return __builtin_elementwise_maximum(z, 0.f); }     // (NaN stays)
template <bool FINE> __device__ __forceinline__ float gelu(float z) {
    float e;
    const float a = fminf(fabsf(z), 16.f);                               // (beyond, the tail is 0 in 32 bits, and Inf has none)
    return fmaf(-a, normal_tail<FINE>(a, e), relu(z));
}
// z s(z), FINE likewise from what is left at -|z|: s(-a) = e / (1 + e), e = exp(-a)
template <bool FINE> __device__ __forceinline__ float silu(float z) {
    if constexpr (!FINE) return z * __builtin_amdgcn_rcpf(1.f + __expf(-z));
    const float a = fminf(fabsf(z), 128.f), e = exp_of(a, 0.f, -1.f);
    return fmaf(-a, e * __builtin_amdgcn_rcpf(1.f + e), relu(z));
}
template <typename V, typename F> __device__ __forceinline__ V each(V z, F f) {
#pragma unroll
    for (int i = 0; i < (int)(sizeof(V) / sizeof(float)); ++i) z[i] = f(z[i]);
    return z;
}
template <typename V> __device__ __forceinline__ V activate_fine(V z, int32_t act) {
    return act == (LF_ACT_GELU | kActFine) ? each(z, [](float v) { return gelu<true>(v); }) : each(z, [](float v) { return silu<true>(v); });
}
__device__ __forceinline__ float8_t activate(float8_t z, int32_t act) {
    if (act == LF_ACT_RELU) return each(z, [](float v) { return relu(v); });
    if (act == LF_ACT_GELU) return each(z, [](float v) { return gelu<false>(v); });
    if (act == LF_ACT_SILU) return each(z, [](float v) { return silu<false>(v); });
    return act & kActFine ? activate_fine(z, act) : z;
}
// FINE: of float32 z
template <bool FINE> __device__ __forceinline__ float activate_grad(float z, int32_t act) {
    if (act == LF_ACT_RELU) return z > 0.f ? 1.f : 0.f;
    if (act == LF_ACT_GELU) {
        float e;
        const float a = fminf(fabsf(z), 16.f), tail = normal_tail<FINE>(a, e), d = fmaf(a * 0.39894228f, e, -tail);
        return z != z ? z : z < 0.f ? -d : 1.f + d;                      // Phi(z) + z phi(z)
    }
    if (act == LF_ACT_SILU) {
        if constexpr (!FINE) {
            const float s = 1.f / (1.f + __expf(-z));
            return s * (1.f + z * (1.f - s));
        }
        const float e = exp_of(fminf(fabsf(z), 128.f), 0.f, -1.f), more = __builtin_amdgcn_rcpf(1.f + e), less = e * more;
        return z < 0.f ? less * fmaf(z, more, 1.f) : more * fmaf(z, less, 1.f);      // s(z) and 1 - s(z) = s(-z), neither as a difference
    }
    return 1.f;
}

// Columns of [n][dim] partial sums, added up in order (lf_norm.hip).
int column_sums(const float* part, int64_t n, int64_t dim, void* out, int32_t dtype, hipStream_t stream);

}  // namespace lf

#define LF_TRY(call)                  \
    do {                              \
        if (int rc_ = (call)) return rc_; \
    } while (0)
