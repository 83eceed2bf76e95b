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
    for (int64_t i = (int64_t)blockIdx.x * (256 / G) + threadIdx.x / G; i < ids.n; i += (int64_t)gridDim.x * (256 / G)) {
        const int64_t id = ids.at(i);
        for (int64_t col = lane * 8; col < dim; col += G * 8) {
            const int count = (int)min((int64_t)8, dim - col);
            float8_t v = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
            if (id < ids.rows) v = load_upto8(w + id * ld_w + col, count) * scale;
            store_upto8(y, i * ld_y + col, y_dtype, v, count, stream);
        }
    }
}

// ---------------------------------------------------------------------------- sorting

struct Entry { uint32_t key, at; };                         // id and position
constexpr int kMostBits = 11, kMostDigits = 1 << kMostBits, kTile = 4096;

struct Passes { int passes, bits; };
// of keys 0 .. rows
inline Passes passes_of(int64_t rows, int most) {
    const int all = ilog2(std::max<int64_t>(rows, 1)) + 1, n = (int)ceil_div(all, most);
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

// How many of the wavefront's entries with this lane's digit come before it: those counted so far, and of the lanes before.  They are counted, too.
template <typename C> __device__ __forceinline__ uint32_t rank_in_wave(C* count, uint32_t digit, int bits, bool on) {
    const uint64_t same = same_digit(digit, bits, on);
    const int before = __popcll(same & ((1ull << (threadIdx.x & 63)) - 1));
    const uint32_t seen = on ? count[digit] : 0;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    if (on && before == 0) count[digit] = (C)(seen + __popcll(same));
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    return seen + before;
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
            rank[r] = rank_in_wave(s_count[wave], d, a.bits, on);
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

// Up to kSmall entries: all passes in one workgroup, the entries in its LDS from pass to pass.
constexpr int kSmall = 8192, kSmallBits = 10;
template <int ROUNDS>
__global__ void __launch_bounds__(1024) sort_small_kernel(SortArgs a, int32_t passes) {
    constexpr int WAVES = 16;
    __shared__ uint16_t s_count[WAVES][1 << kSmallBits];
    __shared__ uint32_t s_key[1024 * ROUNDS];
    __shared__ uint16_t s_at[1024 * ROUNDS];
    __shared__ uint32_t s_wave[WAVES];
    const int digits = 1 << a.bits, lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n = (int)a.n;
    const int mine = wave * (64 * ROUNDS) + lane;
    uint32_t key[ROUNDS];
    uint16_t at[ROUNDS];
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r)
        if (mine + r * 64 < n) {
            key[r] = (uint32_t)a.ids.at(mine + r * 64);
            at[r] = (uint16_t)(mine + r * 64);
        }
    for (int pass = 0; pass < passes; ++pass) {
        a.shift = pass * a.bits;
        for (int w = 0; w < WAVES; ++w)
            if ((int)threadIdx.x < digits) s_count[w][threadIdx.x] = 0;
        __syncthreads();
        uint16_t rank[ROUNDS];
#pragma unroll
        for (int r = 0; r < ROUNDS; ++r) {
            const bool on = mine + r * 64 < n;
            rank[r] = (uint16_t)rank_in_wave(s_count[wave], on ? a.digit(key[r]) : 0, a.bits, on);
        }
        __syncthreads();
        // a digit's entries of all wavefronts, and those of the digits below it
        uint32_t sum = 0;
        if ((int)threadIdx.x < digits)
#pragma unroll
            for (int w = 0; w < WAVES; ++w) sum += s_count[w][threadIdx.x];
        uint32_t upto = sum;
#pragma unroll
        for (int o = 1; o < 64; o *= 2) {
            const uint32_t v = __shfl_up((int)upto, o);
            if (lane >= o) upto += v;
        }
        if (lane == 63) s_wave[wave] = upto;
        __syncthreads();
        uint32_t before = upto - sum;
        for (int w = 0; w < wave; ++w) before += s_wave[w];
        if ((int)threadIdx.x < digits)
#pragma unroll
            for (int w = 0; w < WAVES; ++w) {
                const uint32_t v = s_count[w][threadIdx.x];
                s_count[w][threadIdx.x] = (uint16_t)before;
                before += v;
            }
        __syncthreads();
#pragma unroll
        for (int r = 0; r < ROUNDS; ++r)
            if (mine + r * 64 < n) {
                const uint32_t to = s_count[wave][a.digit(key[r])] + rank[r];
                if (pass == passes - 1) {
                    a.to[to] = {key[r], at[r]};
                } else {
                    s_key[to] = key[r];
                    s_at[to] = at[r];
                }
            }
        if (pass == passes - 1) return;
        __syncthreads();
#pragma unroll
        for (int r = 0; r < ROUNDS; ++r)
            if (mine + r * 64 < n) {
                key[r] = s_key[mine + r * 64];
                at[r] = s_at[mine + r * 64];
            }
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

// G threads take `each` sorted entries one after the other, eight columns a thread.  An id that begins and ends among them is done there; of one that does not
// they leave what they have of it: `head` where it begins before them, `tail` where it begins among them.
template <typename S> struct Sums {
    const Entry* e;
    const void* dy; void* dw;
    S* part;                                                // [chunk][head, tail][ld_part]
    int64_t n, ld_dy, rows, dim, ld_dw, ld_part, chunks;
    int32_t dw_dtype, each, sum_groups;
    float scale;
    __device__ __forceinline__ S* head(int64_t chunk) const { return part + chunk * 2 * ld_part; }
    __device__ __forceinline__ S* tail(int64_t chunk) const { return head(chunk) + ld_part; }
};
template <typename S> struct Eight8 { typedef S vec __attribute__((ext_vector_type(8))); };

template <typename S> __device__ __forceinline__ float8_t scaled(typename Eight8<S>::vec v, float scale) {
    return __builtin_convertvector(v * (S)scale, float8_t);
}

template <typename DT, typename S, int G>
__global__ void __launch_bounds__(256) embedding_sums_kernel(Sums<S> a) {
    using V = typename Eight8<S>::vec;
    constexpr int U = 8;
    const int lane = threadIdx.x % G, team = threadIdx.x / G;
    const int64_t col = ((int64_t)blockIdx.y * G + lane) * 8;
    const int count = (int)min((int64_t)8, a.dim - col);
    if ((int)blockIdx.x >= a.sum_groups) {
        // Rows of ids that do not occur: 64 to a wavefront, each looked for by a lane.
        const int64_t base = ((int64_t)(blockIdx.x - a.sum_groups) * 4 + (threadIdx.x >> 6)) * 64;
        const int64_t row = base + (threadIdx.x & 63);
        bool absent = false;
        if (row < a.rows) {
            const int64_t at = first_of(a.e, a.n, (uint32_t)row);
            absent = at >= a.n || a.e[at].key != (uint32_t)row;
        }
        const uint64_t zeros = __ballot(absent);
        constexpr int AT_ONCE = 64 / G;
        const int mine = (threadIdx.x & 63) / G;
        if (count > 0)
            for (int r = mine; r < 64; r += AT_ONCE)
                if (zeros >> r & 1) store_upto8(a.dw, (base + r) * a.ld_dw + col, a.dw_dtype, float8_t{0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}, count);
        return;
    }
    const int64_t chunk = (int64_t)blockIdx.x * (256 / G) + team, first = chunk * a.each, last = min(a.n, first + a.each);
    if (first >= a.n || count <= 0) return;
    const uint32_t none = (uint32_t)a.rows, before = first > 0 ? a.e[first - 1].key : none, after = last < a.n ? a.e[last].key : none;
    uint32_t key = a.e[first].key;
    V sum = V{0, 0, 0, 0, 0, 0, 0, 0};
    auto leave = [&](bool end) {
        if (key == none) return;
        S* part = key == before ? a.head(chunk) : end && key == after ? a.tail(chunk) : nullptr;     // (sorted: `before` is the key of the chunk's first id or of none)
        if (part) *reinterpret_cast<V*>(part + col) = sum;
        else store_upto8(a.dw, (int64_t)key * a.ld_dw + col, a.dw_dtype, scaled<S>(sum, a.scale), count);
    };
    for (int64_t i = first; i < last; i += U) {
        Entry e[U];
        float8_t v[U];
#pragma unroll
        for (int u = 0; u < U; ++u) e[u] = i + u < last ? a.e[i + u] : Entry{none, 0};
#pragma unroll
        for (int u = 0; u < U; ++u) v[u] = e[u].key != none ? load_upto8((const DT*)a.dy + (int64_t)e[u].at * a.ld_dy + col, count) : float8_t{0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (i + u < last && e[u].key != key) {
                leave(false);
                key = e[u].key;
                sum = V{0, 0, 0, 0, 0, 0, 0, 0};
            }
            sum += __builtin_convertvector(v[u], V);
        }
    }
    leave(true);
}

// What the chunks left of ids that go on from one to the next: G threads look after the end of a chunk; where an id begins in it that goes on, they add
// up its parts, in order.  Ids of more than kFewParts parts are left to all threads of the workgroup.
constexpr int kFewParts = 64;
template <typename S, int G>
__global__ void __launch_bounds__(1024) embedding_join_kernel(Sums<S> a) {
    using V = typename Eight8<S>::vec;
    typedef double D8 __attribute__((ext_vector_type(8)));
    constexpr int TEAMS = 1024 / G;
    __shared__ int s_parts[TEAMS];
    __shared__ double s_sum[TEAMS][G][8];
    const int lane = threadIdx.x % G, team = threadIdx.x / G;
    const int64_t col = ((int64_t)blockIdx.y * G + lane) * 8;
    const int count = (int)min((int64_t)8, a.dim - col);
    const int64_t chunk0 = (int64_t)blockIdx.x * TEAMS;
    auto key_at = [&](int64_t i) { return a.e[i].key; };
    // parts behind the tail of the chunk's last id; 0: it does not go on, or begins before
    auto parts_of = [&](int64_t chunk) -> int {
        const int64_t first = chunk * a.each, next = first + a.each;
        if (next >= a.n) return 0;
        const uint32_t key = key_at(next - 1);
        if (key >= (uint32_t)a.rows || key_at(next) != key || (first > 0 && key_at(first - 1) == key)) return 0;
        // the last chunk whose first entry is of this id: by steps of 1, 2, 4 .., then between
        int64_t lo = chunk + 1, step = 1;
        while (lo + step < a.chunks && key_at((lo + step) * a.each) == key) {
            lo += step;
            step *= 2;
        }
        int64_t hi = min(lo + step, a.chunks);
        while (hi - lo > 1) {
            const int64_t mid = (lo + hi) >> 1;
            if (key_at(mid * a.each) == key) lo = mid; else hi = mid;
        }
        return (int)(lo - chunk);
    };
    auto add_heads = [&](D8& sum, int64_t from, int64_t to) {
        if (count <= 0) return;
#pragma unroll 8
        for (int64_t c = from; c < to; ++c) sum += __builtin_convertvector(*reinterpret_cast<const V*>(a.head(c) + col), D8);
    };
    auto leave = [&](int64_t chunk, D8 sum) {
        if (count > 0)
            store_upto8(a.dw, (int64_t)key_at((chunk + 1) * a.each) * a.ld_dw + col, a.dw_dtype, __builtin_convertvector(sum * (double)a.scale, float8_t), count);
    };
    auto tail_of = [&](int64_t chunk) {
        D8 sum = D8{0, 0, 0, 0, 0, 0, 0, 0};
        if (count > 0) sum = __builtin_convertvector(*reinterpret_cast<const V*>(a.tail(chunk) + col), D8);
        return sum;
    };
    const int64_t chunk = chunk0 + team;
    const int parts = chunk < a.chunks ? parts_of(chunk) : 0;
    if (lane == 0) s_parts[team] = parts;
    if (parts > 0 && parts <= kFewParts) {
        D8 sum = tail_of(chunk);
        add_heads(sum, chunk + 1, chunk + 1 + parts);
        leave(chunk, sum);
    }
    __syncthreads();
    for (int t = 0; t < TEAMS; ++t) {
        const int n = s_parts[t];                           // (the same for all threads)
        if (n <= kFewParts) continue;
        const int64_t c = chunk0 + t;
        const int each = (n + TEAMS - 1) / TEAMS, from = min(n, team * each), to = min(n, from + each);
        D8 sum = D8{0, 0, 0, 0, 0, 0, 0, 0};
        if (team == 0) sum = tail_of(c);
        add_heads(sum, c + 1 + from, c + 1 + to);
#pragma unroll
        for (int i = 0; i < 8; ++i) s_sum[team][lane][i] = sum[i];
        __syncthreads();
        if (team == 0) {
#pragma unroll 4
            for (int o = 1; o < TEAMS; ++o)
#pragma unroll
                for (int i = 0; i < 8; ++i) sum[i] += s_sum[o][lane][i];
            leave(c, sum);
        }
        __syncthreads();
    }
}

template <typename F> void of_type(int32_t t, F f) {
    if (t == LF_DTYPE_F32) f(0.f); else if (t == LF_DTYPE_BF16) f((__bf16)0.f); else f((_Float16)0.f);
}

inline size_t padded(size_t bytes) { return (bytes + 255) / 256 * 256; }
// Entries that some threads take one after the other: enough of them for 8192 wavefronts.
int64_t entries_each(int64_t n, int64_t dim) {
    const int64_t waves = n * ceil_div(dim, 8 * group_of(dim)) * group_of(dim) / 64;
    return waves <= 16 * 8192 ? 16 : waves <= 32 * 8192 ? 32 : 64;
}
inline int sum_bytes(int32_t dtype) { return dtype == LF_DTYPE_F32 ? 8 : 4; }
struct GradWork { size_t entries, counts, totals, parts, total; };
GradWork grad_work(int64_t n, int64_t rows, int64_t dim, int32_t dtype) {
    const Passes p = passes_of(rows, kMostBits);
    const int64_t chunks = ceil_div(n, entries_each(n, dim));
    GradWork w{padded((size_t)n * sizeof(Entry)), 0, 0, 0, 0};
    if (n > kSmall) {
        w.counts = padded(((size_t)sort_groups(n) << p.bits) * 4);
        w.totals = padded(4 << p.bits);
    }
    if (chunks > 1) w.parts = (size_t)chunks * 2 * (size_t)(ceil_div(dim, 8) * 8) * sum_bytes(dtype);
    w.total = (n > kSmall ? 2 : 1) * w.entries + w.counts + w.totals + w.parts;
    return w;
}
template <typename DT, typename S, int G> int launch_sums(const Sums<S>& a, hipStream_t st) {
    const unsigned slices = (unsigned)ceil_div(a.dim, 8 * G);
    embedding_sums_kernel<DT, S, G><<<dim3((unsigned)(a.sum_groups + ceil_div(a.rows, 256)), slices), 256, 0, st>>>(a);
    LF_HIP(hipGetLastError());
    if (a.chunks > 1) {
        embedding_join_kernel<S, G><<<dim3((unsigned)ceil_div(a.chunks, 1024 / G), slices), 1024, 0, st>>>(a);
        LF_HIP(hipGetLastError());
    }
    return LF_OK;
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
        kernel<<<(unsigned)std::min<int64_t>(ceil_div(a.n, 256 / group), 1 << 20), 256, 0, (hipStream_t)stream>>>(ids, (const T*)a.d_table, a.ld_table, a.dim, a.scale, a.d_y, a.ld_y, a.y_dtype, stream_out);
    });
    LF_HIP(hipGetLastError());
    return LF_OK;
}

size_t lf_embedding_grad_work_bytes(int64_t n, int64_t rows, int64_t dim, int32_t dy_dtype) {
    if (n <= 0 || rows <= 0 || dim < 1 || n >= kMost || rows >= kMost || dim > (1 << 24) || !is_float_dtype(dy_dtype)) return 0;
    return grad_work(n, rows, dim, dy_dtype).total;
}

int lf_embedding_grad(const lf_embedding_grad_args* h_args, void* d_work, size_t work_bytes, lf_stream_t stream) {
    LF_REQUIRE(h_args, LF_ERR_INVALID, "null argument");
    const lf_embedding_grad_args& a = *h_args;
    LF_TRY(check_ids(a.d_ids, a.ids_stride, a.ids_bits, a.n, a.rows, a.dim));
    LF_TRY(check_table("dy", a.d_dy, a.n, a.dim, a.ld_dy, a.dy_dtype));
    LF_TRY(check_table("the gradient", a.d_grad, a.rows, a.dim, a.ld_grad, a.grad_dtype));
    if (a.rows == 0) return LF_OK;
    const size_t need = lf_embedding_grad_work_bytes(a.n, a.rows, a.dim, a.dy_dtype);
    LF_REQUIRE(need == 0 || (d_work && (uintptr_t)d_work % 16 == 0), LF_ERR_INVALID, "null or unaligned workspace");
    LF_REQUIRE(work_bytes >= need, LF_ERR_WORKSPACE, "workspace of %zu bytes, %zu are needed", work_bytes, need);
    hipStream_t st = (hipStream_t)stream;
    const Entry* sorted = nullptr;
    char* at = (char*)d_work;
    if (a.n) {
        const GradWork w = grad_work(a.n, a.rows, a.dim, a.dy_dtype);
        SortArgs s{{a.d_ids, a.ids_stride, a.n, a.rows, a.ids_bits == 64}, nullptr, (Entry*)at, nullptr, nullptr, a.n, kTile * tiles_each(a.n), 0, 0, (int32_t)sort_groups(a.n)};
        if (a.n <= kSmall) {
            const Passes p = passes_of(a.rows, kSmallBits);
            s.bits = p.bits;
            auto kernel = a.n <= 1024 ? sort_small_kernel<1> : a.n <= 2048 ? sort_small_kernel<2> : a.n <= 4096 ? sort_small_kernel<4> : sort_small_kernel<8>;
            kernel<<<1, 1024, 0, st>>>(s, p.passes);
            LF_HIP(hipGetLastError());
            sorted = s.to;
            at += w.entries;
        } else {
            const Passes p = passes_of(a.rows, kMostBits);
            Entry* turn[2] = {(Entry*)at, (Entry*)(at + w.entries)};
            s.counts = (uint32_t*)(at + 2 * w.entries);
            s.totals = (uint32_t*)(at + 2 * w.entries + w.counts);
            s.bits = p.bits;
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
            at += 2 * w.entries + w.counts + w.totals;
        }
    }
    const int group = group_of(a.dim);
    const int64_t each = entries_each(a.n, a.dim), chunks = ceil_div(a.n, each);
    int rc = LF_OK;
    of_type(a.dy_dtype, [&](auto t) {
        using T = decltype(t);
        using S = std::conditional_t<std::is_same_v<T, float>, double, float>;
        const Sums<S> k{sorted, a.d_dy, a.d_grad, (S*)at, a.n, a.ld_dy, a.rows, a.dim, a.ld_grad, ceil_div(a.dim, 8) * 8, chunks, a.grad_dtype, (int32_t)each,
                        (int32_t)ceil_div(chunks, 256 / group), a.scale};
        rc = group == 8 ? launch_sums<T, S, 8>(k, st) : group == 16 ? launch_sums<T, S, 16>(k, st) : group == 32 ? launch_sums<T, S, 32>(k, st) : launch_sums<T, S, 64>(k, st);
    });
    return rc;
}

}  // extern "C"
