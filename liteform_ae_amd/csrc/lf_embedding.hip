// Rows of a table by id, and the gradient of the table.
//
//     y_i = c W[id_i]          dW_v = c sum over i with id_i = v of dy_i
//
// An id outside 0 .. rows - 1 (padding) stands for a row of zeros, and has no gradient.
//
// The gradient sorts the ids, by digits of up to 11 bits and stably, so that a row's terms are added in the order in which they were
// looked up, whatever the scheduling; no two threads add to one address.
#include <algorithm>

#include "lf_dense.h"

namespace {

using namespace lf;

// ---------------------------------------------------------------------------- lookup

struct Ids {
    const void* p;
    int64_t stride, n, rows;
    int32_t wide;                                           // 64 bits each
    // of entry i; rows: none of the table's
    __device__ __forceinline__ int64_t at(int64_t i) const {
        const int64_t v = wide ? ((const int64_t*)p)[i * stride] : (int64_t)((const int32_t*)p)[i * stride];
        return v >= 0 && v < rows ? v : rows;
    }
};

// Threads of eight columns each to a row, and how many times they go over it.
inline int group_of(int64_t dim) { return dim <= 64 ? 8 : dim <= 128 ? 16 : dim <= 256 ? 32 : 64; }

template <typename WT, int G>
__global__ void __launch_bounds__(256)
embedding_kernel(Ids ids, const WT* w, int64_t ld_w, int64_t dim, float scale, void* y, int64_t ld_y, int32_t y_dtype, int32_t stream) {
    const int lane = threadIdx.x % G;
    const int64_t i = (int64_t)blockIdx.x * (256 / G) + threadIdx.x / G;
    if (i >= ids.n) return;
    const int64_t id = ids.at(i);
    for (int64_t col = lane * 8; col < dim; col += G * 8) {
        const int count = (int)min((int64_t)8, dim - col);
        float8_t v = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        if (id < ids.rows) v = load_upto8(w + id * ld_w + col, count) * scale;
        store_upto8(y, i * ld_y + col, y_dtype, v, count, stream);
    }
}

// ---------------------------------------------------------------------------- sorting

struct Entry { uint32_t key, at; };                         // id and position
constexpr int kMostBits = 11, kMostDigits = 1 << kMostBits, kTile = 4096;

struct Passes { int passes, bits; };
// of keys 0 .. rows
inline Passes passes_of(int64_t rows) {
    const int all = ilog2(std::max<int64_t>(rows, 1)) + 1, n = (int)ceil_div(all, kMostBits);
    return {n, (int)ceil_div(all, n)};
}
// Workgroups of a pass: each takes some tiles one after the other.
inline int64_t tiles_each(int64_t n) { return std::max<int64_t>(1, ceil_div(n, (int64_t)kTile * 1024)); }
inline int64_t sort_groups(int64_t n) { return ceil_div(n, kTile * tiles_each(n)); }

struct SortArgs {
    Ids ids;                                                // of the first pass
    const Entry* from; Entry* to;
    uint32_t* counts;                                       // [workgroup][digit]: entries, then the entries of that digit before them
    uint32_t* totals;                                       // [digit]
    int64_t n, each;                                        // entries; to a workgroup
    int32_t bits, shift, groups;
    __device__ __forceinline__ Entry entry(int64_t i) const { return from ? from[i] : Entry{(uint32_t)ids.at(i), (uint32_t)i}; }
    __device__ __forceinline__ uint32_t digit(uint32_t key) const { return key >> shift & ((1u << bits) - 1); }
};

__global__ void __launch_bounds__(256) sort_count_kernel(SortArgs a) {
    __shared__ uint32_t s_count[kMostDigits];
    const int digits = 1 << a.bits;
    for (int d = threadIdx.x; d < digits; d += 256) s_count[d] = 0;
    __syncthreads();
    const int64_t first = (int64_t)blockIdx.x * a.each, last = min(a.n, first + a.each);
#pragma unroll 4
    for (int64_t i = first + threadIdx.x; i < last; i += 256) atomicAdd(&s_count[a.digit(a.entry(i).key)], 1u);
    __syncthreads();
    for (int d = threadIdx.x; d < digits; d += 256) a.counts[(int64_t)blockIdx.x * digits + d] = s_count[d];
}

// 16 digits to a workgroup; 64 threads share the workgroups' counts of one.
__global__ void __launch_bounds__(1024) sort_offsets_kernel(SortArgs a) {
    __shared__ uint32_t s[64][17];
    const int digits = 1 << a.bits, d = blockIdx.x * 16 + (threadIdx.x & 15), slice = threadIdx.x >> 4;
    const int each = (a.groups + 63) / 64, first = slice * each, last = min(a.groups, first + each);
    uint32_t sum = 0;
    if (d < digits)
#pragma unroll 8
        for (int g = first; g < last; ++g) sum += a.counts[(int64_t)g * digits + d];
    s[slice][threadIdx.x & 15] = sum;
    __syncthreads();
    uint32_t before = 0;
    for (int i = 0; i < slice; ++i) before += s[i][threadIdx.x & 15];
    if (d >= digits) return;
    if (slice == 63) a.totals[d] = before + sum;
    for (int g = first; g < last; ++g) {
        uint32_t* c = a.counts + (int64_t)g * digits + d;
        const uint32_t v = *c;
        *c = before;
        before += v;
    }
}

// The lanes of the wavefront with this lane's digit (of those that are `on`).
__device__ __forceinline__ uint64_t same_digit(uint32_t digit, int bits, bool on) {
    uint64_t mask = __ballot(on);
    for (int b = 0; b < bits; ++b) {
        const uint64_t set = __ballot(digit >> b & 1);
        mask &= digit >> b & 1 ? set : ~set;
    }
    return mask;
}

__global__ void __launch_bounds__(256) sort_move_kernel(SortArgs a) {
    constexpr int WAVES = 4, ROUNDS = kTile / 256;
    __shared__ uint32_t s_base[kMostDigits], s_count[WAVES][kMostDigits], s_wave[WAVES];
    const int digits = 1 << a.bits, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    // where each digit begins: the digits below it, and this digit's entries of the workgroups before
    {
        const int each = (digits + 255) / 256, first = threadIdx.x * each;
        uint32_t sum = 0;
        for (int d = first; d < min(digits, first + each); ++d) sum += a.totals[d];
        uint32_t upto = sum;
        for (int o = 1; o < 64; o *= 2) {
            const uint32_t v = __shfl_up((int)upto, o);
            if (lane >= o) upto += v;
        }
        if (lane == 63) s_wave[wave] = upto;
        __syncthreads();
        uint32_t before = upto - sum;
        for (int w = 0; w < wave; ++w) before += s_wave[w];
        for (int d = first; d < min(digits, first + each); ++d) {
            s_base[d] = before + a.counts[(int64_t)blockIdx.x * digits + d];
            before += a.totals[d];
        }
    }
    const int64_t end = min(a.n, ((int64_t)blockIdx.x + 1) * a.each);
    for (int64_t tile = (int64_t)blockIdx.x * a.each; tile < end; tile += kTile) {
        for (int w = 0; w < WAVES; ++w)
            for (int d = threadIdx.x; d < digits; d += 256) s_count[w][d] = 0;
        Entry e[ROUNDS];
        uint32_t rank[ROUNDS];
        const int64_t mine = tile + wave * (64 * ROUNDS) + lane;
#pragma unroll
        for (int r = 0; r < ROUNDS; ++r)
            if (mine + r * 64 < end) e[r] = a.entry(mine + r * 64);
        __syncthreads();
        // a wavefront's entries in order, 64 at a time: those of the digit before, and among the 64
#pragma unroll
        for (int r = 0; r < ROUNDS; ++r) {
            const bool on = mine + r * 64 < end;
            const uint32_t d = on ? a.digit(e[r].key) : 0;
            const uint64_t same = same_digit(d, a.bits, on);
            const int before = __popcll(same & ((1ull << lane) - 1));
            const uint32_t seen = on ? s_count[wave][d] : 0;
            rank[r] = seen + before;
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
            if (on && before == 0) s_count[wave][d] = seen + __popcll(same);
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
        }
        __syncthreads();
        for (int d = threadIdx.x; d < digits; d += 256) {
            uint32_t at = s_base[d];
#pragma unroll
            for (int w = 0; w < WAVES; ++w) {
                const uint32_t v = s_count[w][d];
                s_count[w][d] = at;
                at += v;
            }
            s_base[d] = at;
        }
        __syncthreads();
#pragma unroll
        for (int r = 0; r < ROUNDS; ++r)
            if (mine + r * 64 < end) a.to[s_count[wave][a.digit(e[r].key)] + rank[r]] = e[r];
        __syncthreads();
    }
}

// ---------------------------------------------------------------------------- sums

// The first of n sorted entries whose key is `key` or more.
__device__ __forceinline__ int64_t first_of(const Entry* e, int64_t n, uint32_t key) {
    int64_t lo = 0, hi = n;
    while (lo < hi) {
        const int64_t mid = (lo + hi) >> 1;
        if (e[mid].key < key) lo = mid + 1; else hi = mid;
    }
    return lo;
}

template <typename DT, int G>
__global__ void __launch_bounds__(256)
embedding_sums_kernel(const Entry* e, int64_t n, const DT* dy, int64_t ld_dy, int64_t rows, int64_t dim, float scale, void* dw, int64_t ld_dw, int32_t dw_dtype) {
    const int lane = threadIdx.x % G;
    const int64_t row = (int64_t)blockIdx.x * (256 / G) + threadIdx.x / G;
    if (row >= rows) return;
    const int64_t first = first_of(e, n, (uint32_t)row);
    for (int64_t col = lane * 8; col < dim; col += G * 8) {
        const int count = (int)min((int64_t)8, dim - col);
        float8_t v = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        for (int64_t i = first; i < n && e[i].key == (uint32_t)row; ++i) v += load_upto8(dy + (int64_t)e[i].at * ld_dy + col, count);
        store_upto8(dw, row * ld_dw + col, dw_dtype, v * scale, count);
    }
}

template <typename F> void of_type(int32_t t, F f) {
    if (t == LF_DTYPE_F32) f(0.f); else if (t == LF_DTYPE_BF16) f((__bf16)0.f); else f((_Float16)0.f);
}

struct GradWork { size_t entries, counts, totals, total; };
inline size_t padded(size_t bytes) { return (bytes + 255) / 256 * 256; }
GradWork grad_work(int64_t n, int64_t rows) {
    const Passes p = passes_of(rows);
    GradWork w{padded((size_t)n * sizeof(Entry)), padded(((size_t)sort_groups(n) << p.bits) * 4), padded(4 << p.bits), 0};
    w.total = 2 * w.entries + w.counts + w.totals;
    return w;
}

constexpr int64_t kMost = 1ll << 31;
int check_ids(const void* ids, int64_t stride, int32_t bits, int64_t n, int64_t rows, int64_t dim) {
    LF_REQUIRE(n >= 0 && rows >= 0 && dim >= 1, LF_ERR_INVALID, "bad sizes: %lld ids, %lld rows of %lld", (long long)n, (long long)rows, (long long)dim);
    LF_REQUIRE(n < kMost && rows < kMost && dim <= (1 << 24), LF_ERR_UNSUPPORTED, "%lld ids, %lld rows of %lld", (long long)n, (long long)rows, (long long)dim);
    LF_REQUIRE(bits == 32 || bits == 64, LF_ERR_UNSUPPORTED, "ids have 32 or 64 bits");
    LF_REQUIRE(ids || n == 0, LF_ERR_INVALID, "ids: null pointer");
    LF_REQUIRE(stride >= 0, LF_ERR_INVALID, "ids: negative stride");
    LF_REQUIRE((uintptr_t)ids % (bits / 8) == 0, LF_ERR_INVALID, "ids: not aligned to its elements");
    return LF_OK;
}
int check_table(const char* what, const void* p, int64_t rows, int64_t dim, int64_t ld, int32_t dtype) {
    LF_REQUIRE(is_float_dtype(dtype), LF_ERR_UNSUPPORTED, "%s is of float32, bfloat16 or float16", what);
    LF_REQUIRE(p || rows == 0, LF_ERR_INVALID, "%s: null pointer", what);
    LF_REQUIRE(ld >= dim || rows <= 1, LF_ERR_INVALID, "%s: rows of %lld elements, %lld apart", what, (long long)dim, (long long)ld);
    LF_REQUIRE((uintptr_t)p % dtype_bytes(dtype) == 0, LF_ERR_INVALID, "%s: not aligned to its elements", what);
    return LF_OK;
}

}  // namespace

extern "C" {

int lf_embedding(const lf_embedding_args* h_args, lf_stream_t stream) {
    LF_REQUIRE(h_args, LF_ERR_INVALID, "null argument");
    const lf_embedding_args& a = *h_args;
    LF_TRY(check_ids(a.d_ids, a.ids_stride, a.ids_bits, a.n, a.rows, a.dim));
    LF_TRY(check_table("the table", a.d_table, a.rows, a.dim, a.ld_table, a.table_dtype));
    LF_TRY(check_table("y", a.d_y, a.n, a.dim, a.ld_y, a.y_dtype));
    if (a.n == 0) return LF_OK;
    const Ids ids{a.d_ids, a.ids_stride, a.n, a.rows, a.ids_bits == 64};
    const int group = group_of(a.dim);
    const int32_t stream_out = a.n * a.dim * dtype_bytes(a.y_dtype) >= kStreamBytes;
    of_type(a.table_dtype, [&](auto t) {
        using T = decltype(t);
        auto kernel = group == 8 ? embedding_kernel<T, 8> : group == 16 ? embedding_kernel<T, 16> : group == 32 ? embedding_kernel<T, 32> : embedding_kernel<T, 64>;
        kernel<<<(unsigned)ceil_div(a.n, 256 / group), 256, 0, (hipStream_t)stream>>>(ids, (const T*)a.d_table, a.ld_table, a.dim, a.scale, a.d_y, a.ld_y, a.y_dtype, stream_out);
    });
    LF_HIP(hipGetLastError());
    return LF_OK;
}

size_t lf_embedding_grad_work_bytes(int64_t n, int64_t rows, int64_t dim) {
    if (n <= 0 || rows <= 0 || dim < 1 || n >= kMost || rows >= kMost) return 0;
    return grad_work(n, rows).total;
}

int lf_embedding_grad(const lf_embedding_grad_args* h_args, void* d_work, size_t work_bytes, lf_stream_t stream) {
    LF_REQUIRE(h_args, LF_ERR_INVALID, "null argument");
    const lf_embedding_grad_args& a = *h_args;
    LF_TRY(check_ids(a.d_ids, a.ids_stride, a.ids_bits, a.n, a.rows, a.dim));
    LF_TRY(check_table("dy", a.d_dy, a.n, a.dim, a.ld_dy, a.dy_dtype));
    LF_TRY(check_table("the gradient", a.d_grad, a.rows, a.dim, a.ld_grad, a.grad_dtype));
    if (a.rows == 0) return LF_OK;
    const size_t need = lf_embedding_grad_work_bytes(a.n, a.rows, a.dim);
    LF_REQUIRE(need == 0 || (d_work && (uintptr_t)d_work % 16 == 0), LF_ERR_INVALID, "null or unaligned workspace");
    LF_REQUIRE(work_bytes >= need, LF_ERR_WORKSPACE, "workspace of %zu bytes, %zu are needed", work_bytes, need);
    hipStream_t st = (hipStream_t)stream;
    const Entry* sorted = nullptr;
    if (a.n) {
        const GradWork w = grad_work(a.n, a.rows);
        const Passes p = passes_of(a.rows);
        char* at = (char*)d_work;
        Entry* turn[2] = {(Entry*)at, (Entry*)(at + w.entries)};
        SortArgs s{{a.d_ids, a.ids_stride, a.n, a.rows, a.ids_bits == 64}, nullptr, nullptr, (uint32_t*)(at + 2 * w.entries), (uint32_t*)(at + 2 * w.entries + w.counts), a.n,
                   kTile * tiles_each(a.n), p.bits, 0, (int32_t)sort_groups(a.n)};
        for (int pass = 0; pass < p.passes; ++pass) {
            s.from = sorted;
            s.to = turn[pass & 1];
            s.shift = pass * p.bits;
            sort_count_kernel<<<s.groups, 256, 0, st>>>(s);
            LF_HIP(hipGetLastError());
            sort_offsets_kernel<<<(unsigned)ceil_div(1 << p.bits, 16), 1024, 0, st>>>(s);
            LF_HIP(hipGetLastError());
            sort_move_kernel<<<s.groups, 256, 0, st>>>(s);
            LF_HIP(hipGetLastError());
            sorted = s.to;
        }
    }
    const int group = group_of(a.dim);
    of_type(a.dy_dtype, [&](auto t) {
        using T = decltype(t);
        auto kernel = group == 8 ? embedding_sums_kernel<T, 8> : group == 16 ? embedding_sums_kernel<T, 16> : group == 32 ? embedding_sums_kernel<T, 32> : embedding_sums_kernel<T, 64>;
        kernel<<<(unsigned)ceil_div(a.rows, 256 / group), 256, 0, st>>>(sorted, a.n, (const T*)a.d_dy, a.ld_dy, a.rows, a.dim, a.scale, a.d_grad, a.ld_grad, a.grad_dtype);
    });
    LF_HIP(hipGetLastError());
    return LF_OK;
}

}  // extern "C"
