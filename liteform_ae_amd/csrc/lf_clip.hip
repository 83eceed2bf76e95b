// The norm of the gradients of all parameters together, and the gradients cut to a largest norm:
//
//     norm = sqrt(sum over all elements of all tensors of g^2);  out = g min(1, most / (norm + eps))
//
// Squares are added in 64 bits: none overflows or vanishes, whatever the type, and the sum is good to the last place of the norm's 32.
// Tensors are handed to the kernels as arguments, a few dozen to a launch, so that nothing is copied to the GPU.
//
// Bound by memory, three passes of it: the norm has to be known before the first output.  403M elements of bfloat16 141 + 297 us (5.7 and 5.4 TB/s; with one piece of
// eight elements under way a thread, not eight, the norm took 215); 150k of float32 5 + 8.
#include <algorithm>
#include <new>
#include <vector>

#include "lf_dense.h"

namespace {

using namespace lf;

constexpr int kTensors = 64;                                // to a launch
constexpr int64_t kChunk = 16384;                           // elements to a workgroup
constexpr int kMostParts = 2048;                            // partial sums of a launch
constexpr int64_t kMostElements = 1ll << 40;                // of all tensors: chunks are counted in 32 bits

struct Tensor { const void* src; void* dst; int64_t rows, cols, ld_src, ld_dst; };
struct List {
    Tensor t[kTensors];
    int32_t first[kTensors + 1];                            // workgroup-chunk that a tensor begins with
    int8_t dtype[kTensors];
    int32_t n;
};

__device__ __forceinline__ int tensor_of(const List& l, int chunk) {
    int lo = 0, hi = l.n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (l.first[mid] <= chunk) lo = mid; else hi = mid;
    }
    return lo;
}
// Eight pieces of eight elements to a thread, all under way at once: f(piece, element of src, of dst, count) for each.
constexpr int kMine = (int)(kChunk / 8 / 256);
template <typename F> __device__ __forceinline__ void pieces_of(const Tensor& t, int64_t chunk, F f) {
    const int64_t u0 = chunk * (kChunk / 8) + threadIdx.x;
    if (t.rows == 1) {
#pragma unroll
        for (int i = 0; i < kMine; ++i) {
            const int64_t col = (u0 + i * 256) * 8;
            f(i, col, col, (int)max((int64_t)0, min((int64_t)8, t.cols - col)));
        }
        return;
    }
    const int64_t across = (t.cols + 7) / 8, end = across * t.rows;
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
        const int64_t u = u0 + i * 256, row = u / across, col = (u - row * across) * 8;
        f(i, row * t.ld_src + col, row * t.ld_dst + col, u < end ? (int)min((int64_t)8, t.cols - col) : 0);
    }
}
template <typename F> __device__ __forceinline__ void of_type(int32_t dtype, F f) {
    if (dtype == LF_DTYPE_F32) f(0.f); else if (dtype == LF_DTYPE_BF16) f((__bf16)0.f); else f((_Float16)0.f);
}
template <typename T> using Raw = typename Eight<T>::vec;
template <typename T> __device__ __forceinline__ Raw<T> load_raw(const T* p, int n) {
    return n >= 8 ? reinterpret_cast<const typename Eight<T>::Any*>(p)->v : __builtin_convertvector(load_upto8(p, n), Raw<T>);
}
__device__ __forceinline__ double sum_of_workgroup(double v) {
    __shared__ double s[4];
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
    __syncthreads();
    return (s[0] + s[1]) + (s[2] + s[3]);
}

__global__ void __launch_bounds__(256) squares_kernel(List l, double* part) {
    double sum = 0.0;
    for (int chunk = blockIdx.x; chunk < l.first[l.n]; chunk += gridDim.x) {
        const int i = tensor_of(l, chunk);
        const Tensor& t = l.t[i];
        of_type(l.dtype[i], [&](auto z) {
            using T = decltype(z);
            Raw<T> raw[kMine];
            pieces_of(t, chunk - l.first[i], [&](int u, int64_t at, int64_t, int n) { raw[u] = load_raw((const T*)t.src + at, n); });
            double mine[kMine];
#pragma unroll
            for (int u = 0; u < kMine; ++u) {
                mine[u] = 0.0;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const double v = (double)(float)raw[u][j];
                    mine[u] = fma(v, v, mine[u]);
                }
            }
#pragma unroll
            for (int u = 0; u < kMine; ++u) sum += mine[u];
        });
    }
    sum = sum_of_workgroup(sum);
    if (threadIdx.x == 0) part[blockIdx.x] = sum;
}

// (every workgroup adds up the partial sums, all in one order)
__global__ void __launch_bounds__(256) clip_kernel(List l, const double* part, int32_t parts, float most, float eps, float* norm, int32_t write_norm, int32_t stream) {
    double sum = 0.0;
    for (int i = threadIdx.x; i < parts; i += 256) sum += part[i];
    const float total = (float)sqrt(sum_of_workgroup(sum));
    if (write_norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = total;
    // (a norm of NaN leaves NaN; a limit that is infinite cuts nothing, not even an infinite norm)
    const float by = most / (total + eps), c = by > 1.f || total == 0.f || (most == __builtin_inff() && total == total) ? 1.f : by;
    for (int chunk = blockIdx.x; chunk < l.first[l.n]; chunk += gridDim.x) {
        const int i = tensor_of(l, chunk);
        const Tensor& t = l.t[i];
        if (c == 1.f && t.src == t.dst) continue;
        of_type(l.dtype[i], [&](auto z) {
            using T = decltype(z);
            Raw<T> raw[kMine];
            pieces_of(t, chunk - l.first[i], [&](int u, int64_t at, int64_t, int n) { raw[u] = load_raw((const T*)t.src + at, n); });
            pieces_of(t, chunk - l.first[i], [&](int u, int64_t, int64_t at, int n) {
                store_upto8((T*)t.dst + at, __builtin_convertvector(raw[u], float8_t) * c, n, stream);
            });
        });
    }
}

// Bytes that a tensor's rows take: `width` of every `pitch` from `at` on.
struct Span {
    uintptr_t at, end, width, pitch;
    int32_t tensor;
    bool written;
};
Span span_of(const void* p, int64_t rows, int64_t cols, int64_t ld, int32_t dtype, int32_t tensor, bool written) {
    const uintptr_t e = dtype_bytes(dtype), at = (uintptr_t)p;
    return {at, at + (rows - 1) * ld * e + cols * e, cols * e, rows > 1 ? ld * e : 0, tensor, written};
}
// Columns of one wider matrix, side by side
bool side_by_side(const Span& a, const Span& b) {
    const uintptr_t pitch = a.pitch ? a.pitch : b.pitch;
    if (!pitch || (a.pitch && b.pitch && a.pitch != b.pitch)) return false;
    const uintptr_t off = b.at >= a.at ? (b.at - a.at) % pitch : (pitch - (a.at - b.at) % pitch) % pitch;
    return a.width <= off && off + b.width <= pitch;
}
// Whether an output lies on another tensor's elements, or on its own in other places.
bool overlapping(const lf_tensor_desc* t, int32_t n) {
    std::vector<Span> all;
    all.reserve(2 * (size_t)n);
    for (int32_t i = 0; i < n; ++i) {
        if (!t[i].rows || !t[i].cols) continue;
        all.push_back(span_of(t[i].d_dst, t[i].rows, t[i].cols, t[i].ld_dst, (int32_t)t[i].dtype, i, true));
        if (t[i].d_src != t[i].d_dst || (t[i].rows > 1 && t[i].ld_src != t[i].ld_dst)) all.push_back(span_of(t[i].d_src, t[i].rows, t[i].cols, t[i].ld_src, (int32_t)t[i].dtype, i, false));
    }
    std::sort(all.begin(), all.end(), [](const Span& a, const Span& b) { return a.at < b.at; });
    std::vector<const Span*> open;                          // those that may reach beyond where we are
    for (const Span& s : all) {
        open.erase(std::remove_if(open.begin(), open.end(), [&](const Span* o) { return o->end <= s.at; }), open.end());
        for (const Span* o : open)
            if ((o->written || s.written) && !side_by_side(*o, s)) return true;
        open.push_back(&s);
    }
    return false;
}

struct Call { std::vector<List> lists; };
void add(Call& c, const lf_tensor_desc& d, int64_t chunks) {
    if (c.lists.empty() || c.lists.back().n == kTensors) {
        c.lists.emplace_back();
        c.lists.back().n = 0;
        c.lists.back().first[0] = 0;
    }
    List& l = c.lists.back();
    const bool flat = d.rows == 1 || (d.ld_src == d.cols && (!d.d_dst || d.ld_dst == d.cols));
    l.t[l.n] = {d.d_src, d.d_dst, flat ? 1 : d.rows, flat ? d.rows * d.cols : d.cols, d.ld_src, d.ld_dst};
    l.dtype[l.n] = (int8_t)d.dtype;
    l.first[l.n + 1] = l.first[l.n] + (int32_t)chunks;
    ++l.n;
}

int clip(const lf_tensor_desc* t, int32_t n, float most, float eps, float* d_norm, void* d_work, size_t work_bytes, hipStream_t st) {
    bool out = false, any = false;
    int64_t elements = 0;
    for (int32_t i = 0; i < n; ++i) {
        const lf_tensor_desc& d = t[i];
        LF_REQUIRE(is_float_dtype((int32_t)d.dtype), LF_ERR_UNSUPPORTED, "tensor %d: gradients are of float32, bfloat16 or float16", i);
        LF_REQUIRE(d.rows >= 0 && d.cols >= 0, LF_ERR_INVALID, "tensor %d: %lld x %lld", i, (long long)d.rows, (long long)d.cols);
        if (!d.rows || !d.cols) continue;
        LF_REQUIRE(d.cols <= kMostElements && d.rows <= kMostElements / (ceil_div(d.cols, 8) * 8) && d.ld_src <= kMostElements && d.ld_dst <= kMostElements, LF_ERR_UNSUPPORTED,
                   "tensor %d: %lld x %lld", i, (long long)d.rows, (long long)d.cols);
        elements += d.rows * d.cols;
        LF_REQUIRE(d.d_src, LF_ERR_INVALID, "tensor %d: null pointer", i);
        LF_REQUIRE((uintptr_t)d.d_src % dtype_bytes((int32_t)d.dtype) == 0 && (uintptr_t)d.d_dst % dtype_bytes((int32_t)d.dtype) == 0, LF_ERR_INVALID, "tensor %d: not aligned to its elements", i);
        LF_REQUIRE(d.rows <= 1 || (d.ld_src >= d.cols && (!d.d_dst || d.ld_dst >= d.cols)), LF_ERR_INVALID, "tensor %d: rows of %lld elements overlap", i, (long long)d.cols);
        LF_REQUIRE(!any || out == (d.d_dst != nullptr), LF_ERR_INVALID, "outputs are for all tensors or for none");
        any = true;
        out = d.d_dst != nullptr;
        LF_REQUIRE(elements <= kMostElements, LF_ERR_UNSUPPORTED, "more elements than any GPU holds");
    }
    const size_t need = lf_clip_work_bytes(n);
    LF_REQUIRE(need == 0 || (d_work && (uintptr_t)d_work % 16 == 0), LF_ERR_INVALID, "null or unaligned workspace");
    LF_REQUIRE(work_bytes >= need, LF_ERR_WORKSPACE, "workspace of %zu bytes, %zu are needed", work_bytes, need);
    LF_REQUIRE(!out || !overlapping(t, n), LF_ERR_INVALID, "an output lies on another tensor");
    Call c;
    for (int32_t i = 0; i < n; ++i) {
        const int64_t pieces = t[i].rows == 0 || t[i].cols == 0 ? 0
                               : t[i].rows == 1 || (t[i].ld_src == t[i].cols && (!t[i].d_dst || t[i].ld_dst == t[i].cols)) ? ceil_div(t[i].rows * t[i].cols, 8)
                                                                                                                              : t[i].rows * ceil_div(t[i].cols, 8);
        if (pieces) add(c, t[i], ceil_div(pieces, kChunk / 8));
    }
    int64_t bytes = 0;
    for (int32_t i = 0; i < n; ++i) bytes += t[i].rows * t[i].cols * dtype_bytes((int32_t)t[i].dtype);
    const int32_t stream = bytes >= kStreamBytes;
    double* part = (double*)d_work;
    int32_t parts = 0;
    for (const List& l : c.lists) {
        const int groups = std::min(l.first[l.n], kMostParts);
        squares_kernel<<<(unsigned)groups, 256, 0, st>>>(l, part + parts);
        LF_HIP(hipGetLastError());
        parts += groups;
    }
    if (c.lists.empty() || !out) {
        List none{};
        clip_kernel<<<1, 256, 0, st>>>(none, part, parts, most, eps, d_norm, 1, 0);
        LF_HIP(hipGetLastError());
        return LF_OK;
    }
    for (size_t i = 0; i < c.lists.size(); ++i) {
        const List& l = c.lists[i];
        clip_kernel<<<(unsigned)std::min(l.first[l.n], 4096), 256, 0, st>>>(l, part, parts, most, eps, d_norm, i == 0, stream);
        LF_HIP(hipGetLastError());
    }
    return LF_OK;
}

}  // namespace

extern "C" {

size_t lf_clip_work_bytes(int32_t n) { return n <= 0 ? 0 : (size_t)ceil_div(n, kTensors) * kMostParts * sizeof(double); }

int lf_clip_gradients(const lf_tensor_desc* h_tensors, int32_t n, float most, float eps, float* d_norm, void* d_work, size_t work_bytes, lf_stream_t stream) {
    LF_REQUIRE(n >= 0 && (h_tensors || n == 0) && d_norm, LF_ERR_INVALID, "null argument");
    LF_REQUIRE(most >= 0.f && eps >= 0.f, LF_ERR_INVALID, "the largest norm and eps must not be negative");
    try {
        return clip(h_tensors, n, most, eps, d_norm, d_work, work_bytes, (hipStream_t)stream);
    } catch (const std::bad_alloc&) {
        return fail(LF_ERR_HIP, "out of host memory for %d tensors", n);
    }
}

}  // extern "C"
