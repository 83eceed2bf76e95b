// Rows of a table by id, and the gradient of the table.
//
//     y_i = c W[id_i]          dW_v = c sum over i with id_i = v of dy_i
//
// An id outside 0 .. rows - 1 (padding) stands for a row of zeros, and has no gradient.
//
// The gradient sorts the ids, by digits of up to 11 bits and stably, so that a row's terms are added in the order in which they were
// looked up, whatever the scheduling; no two threads add to one address.  Then equal parts of the sorted entries are added up, whatever ids they are of, and what
// parts have of one id is put together, in LDS and (from a workgroup to the next) through memory.  Sums of float32 are in 64 bits, of 16-bit types in 32, and
// in 64 from part to part: an id may have all rows.
//
// Measured with inputs that no cache holds: 57,001 rows of 2.45M x 128 f16 8 us; gradient of 16,384 ids of 32,000 x 4096 bf16, most of them a few ids, 104 us: sort
// 25 in four launches, sums and rows of zeros 75 (396 MB: 5.3 TB/s), join 6.  Bound by memory where rows are long; else by launches and by
// the latency of each pass (100,000 ids of 45,000 x 16 f32: 51 us).  Counts of the next digit made with atomic additions while the entries move, a launch less: 94 us
// became 110, 72 (432k ids of 82) became 95.
#include <algorithm>

#include "lf_dense.h"
#include "lf_rules.h"

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
constexpr int kMostBits = 11, kMostDigits = 1 << kMostBits, kTile = 2048, kSortThreads = 512;

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
    uint8_t* present;                                       // [row]: the first pass clears it, the last one marks the ids that occur
    int64_t n, each;                                        // entries; to a workgroup
    int32_t bits, shift, groups, first, last;
    __device__ __forceinline__ Entry entry(int64_t i) const { return from ? from[i] : Entry{(uint32_t)ids.at(i), (uint32_t)i}; }
    __device__ __forceinline__ uint32_t digit(uint32_t key) const { return key >> shift & ((1u << bits) - 1); }
};

__global__ void __launch_bounds__(kSortThreads) sort_count_kernel(SortArgs a) {
    __shared__ uint32_t s_count[kMostDigits];
    const int digits = 1 << a.bits;
    for (int d = threadIdx.x; d < digits; d += kSortThreads) s_count[d] = 0;
    if (a.first)                                            // (in pieces of 16 bytes, which there is room for)
        for (int64_t i = (int64_t)blockIdx.x * kSortThreads + threadIdx.x; i * 16 < a.ids.rows; i += (int64_t)gridDim.x * kSortThreads)
            reinterpret_cast<uint4_t*>(a.present)[i] = uint4_t{0u, 0u, 0u, 0u};
    __syncthreads();
    const int64_t first = (int64_t)blockIdx.x * a.each, last = min(a.n, first + a.each);
    for (int64_t tile = first; tile < last; tile += kTile) {
        uint32_t d[kTile / kSortThreads];
#pragma unroll
        for (int r = 0; r < kTile / kSortThreads; ++r) {
            const int64_t i = tile + threadIdx.x + r * kSortThreads;
            d[r] = i < last ? a.digit(a.entry(i).key) : ~0u;
        }
#pragma unroll
        for (int r = 0; r < kTile / kSortThreads; ++r)
            if (d[r] != ~0u) atomicAdd(&s_count[d[r]], 1u);
    }
    __syncthreads();
    for (int d = threadIdx.x; d < digits; d += kSortThreads) a.counts[(int64_t)blockIdx.x * digits + d] = s_count[d];
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
    for (int g0 = first; g0 < last; g0 += 8) {
        uint32_t v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = g0 + i < last ? a.counts[(int64_t)(g0 + i) * digits + d] : 0;
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (g0 + i < last) {
                a.counts[(int64_t)(g0 + i) * digits + d] = before;
                before += v[i];
            }
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

// FEW: `counts` is what sort_count_kernel left, and each workgroup adds up those of all (sort_adds_counts)
template <bool FEW>
__global__ void __launch_bounds__(kSortThreads) sort_move_kernel(SortArgs a) {
    constexpr int WAVES = kSortThreads / 64, ROUNDS = kTile / kSortThreads, MINE = kMostDigits / kSortThreads;
    __shared__ uint32_t s_base[kMostDigits], s_count[WAVES][kMostDigits], s_wave[WAVES];
    const int digits = 1 << a.bits, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t end = min(a.n, ((int64_t)blockIdx.x + 1) * a.each);
    int64_t mine = (int64_t)blockIdx.x * a.each + wave * (64 * ROUNDS) + lane;
    Entry e[ROUNDS];
    auto load = [&] {
#pragma unroll
        for (int r = 0; r < ROUNDS; ++r)
            if (mine + r * 64 < end) e[r] = a.entry(mine + r * 64);
    };
    load();
    // where each digit begins: the digits below it, and this digit's entries of the workgroups before
    {
        uint32_t total[MINE], sum = 0;
#pragma unroll
        for (int i = 0; i < MINE; ++i) {
            const int d = threadIdx.x * MINE + i;
            total[i] = 0;
            if (d >= digits) continue;
            if constexpr (FEW) {
                uint32_t before = 0;
#pragma unroll 8
                for (int g = 0; g < a.groups; ++g) {
                    const uint32_t v = a.counts[g * digits + d];
                    before += g < (int)blockIdx.x ? v : 0;
                    total[i] += v;
                }
                s_base[d] = before;
            } else {
                total[i] = a.totals[d];
                s_base[d] = a.counts[(int64_t)blockIdx.x * digits + d];
            }
        }
#pragma unroll
        for (int i = 0; i < MINE; ++i) sum += total[i];
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
#pragma unroll
        for (int i = 0; i < MINE; ++i) {
            const int d = threadIdx.x * MINE + i;
            if (d < digits) s_base[d] += before;
            before += total[i];
        }
    }
    for (int64_t tile = (int64_t)blockIdx.x * a.each;;) {
        for (int w = 0; w < WAVES; ++w)
            for (int d = threadIdx.x; d < digits; d += kSortThreads) s_count[w][d] = 0;
        __syncthreads();
        // a wavefront's entries in order, 64 at a time: those of the digit before, and among the 64
        uint32_t rank[ROUNDS];
#pragma unroll
        for (int r = 0; r < ROUNDS; ++r) {
            const bool on = mine + r * 64 < end;
            rank[r] = rank_in_wave(s_count[wave], on ? a.digit(e[r].key) : 0, a.bits, on);
        }
        __syncthreads();
        for (int d = threadIdx.x; d < digits; d += kSortThreads) {
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
            if (mine + r * 64 < end) {
                a.to[s_count[wave][a.digit(e[r].key)] + rank[r]] = e[r];
                if (a.last && e[r].key < (uint32_t)a.ids.rows) a.present[e[r].key] = 1;
            }
        tile += kTile;
        if (tile >= end) return;
        mine += kTile;
        load();
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

// The first entry before `hi` that is not of the id that entry `lo` has, or hi.
__device__ __forceinline__ int end_of(const Entry* e, int lo, int hi, uint32_t key) {
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (e[mid].key == key) lo = mid; else hi = mid;
    }
    return hi;
}

// A workgroup takes a span of sorted entries, G threads of it `each` one after the other, eight columns a thread.  Ids that go on from these G threads to the next are
// put together in LDS; of one that goes on from a workgroup to the next, `tail` is what the one that it begins in has of it, `head` what each of the others has.
constexpr int kSumThreads = 256, kMostEach = 64;
template <typename S> struct Sums {
    const Entry* e;
    const uint8_t* present;                                 // of each row, whether its id occurs; NULL: it is looked for
    const void* dy; void* dw;
    S* part;                                                // [workgroup][head, tail][ld_part]
    int64_t n, ld_dy, rows, dim, ld_dw, ld_part;
    int32_t dw_dtype, each, sum_groups, fill_rows, stream;
    uint32_t slices, groups;                                // of a row's columns; of all that adds up and fills
    int32_t by_slice;                                       // one slice after the other
    float scale;
    __device__ __forceinline__ S* head(int64_t group) const { return part + group * 2 * ld_part; }
    __device__ __forceinline__ S* tail(int64_t group) const { return head(group) + ld_part; }
};
template <typename S> struct Eight8 { typedef S vec __attribute__((ext_vector_type(8))); };

// A thread's eight columns.  The last ones of a row whose length is no multiple of eight reach back into those before, which two threads then
// compute and write, alike; rows of less than eight have `count` columns.
struct Columns {
    int64_t col;
    int count;
    bool on;
    __device__ __forceinline__ Columns(int64_t first, int64_t dim) : col(dim < 8 ? 0 : min(first, dim - 8)), count((int)min(dim, (int64_t)8)), on(first < dim) {}
};
template <typename S> struct AnyEight { struct __attribute__((packed, aligned(sizeof(S)))) type { typename Eight8<S>::vec v; }; };

template <typename S> __device__ __forceinline__ float8_t scaled(typename Eight8<S>::vec v, float scale) {
    return __builtin_convertvector(v * (S)scale, float8_t);
}

// Rows of ids that do not occur: `fill_rows` to a wavefront, a row's id to a lane.
template <typename S, int G> __device__ __forceinline__ void fill_rows(const Sums<S>& a, int group, const Columns& at) {
    const int64_t base = ((int64_t)group * (kSumThreads / 64) + (threadIdx.x >> 6)) * a.fill_rows;
    const int64_t row = base + (threadIdx.x & 63);
    bool absent = false;
    if (row < min(a.rows, base + a.fill_rows)) {
        if (a.present) {
            absent = !a.present[row];
        } else {
            const int64_t at = first_of(a.e, a.n, (uint32_t)row);
            absent = at >= a.n || a.e[at].key != (uint32_t)row;
        }
    }
    const uint64_t zeros = __ballot(absent);
    if (!at.on) return;
    for (int r = (threadIdx.x & 63) / G; r < a.fill_rows; r += 64 / G)
        if (zeros >> r & 1) store_upto8(a.dw, (base + r) * a.ld_dw + at.col, a.dw_dtype, float8_t{0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}, at.count, a.stream);
}

template <typename DT, typename S, int G>
__global__ void __launch_bounds__(kSumThreads) embedding_sums_kernel(Sums<S> a) {
    using V = typename Eight8<S>::vec;
    using R = typename Eight<DT>::vec;                      // (eight elements as they lie in memory: floats of them would take twice the registers)
    constexpr int U = sizeof(DT) == 4 ? 4 : 8, TEAMS = kSumThreads / G;
    const int lane = threadIdx.x % G, team = threadIdx.x / G;
    const uint32_t slice = a.by_slice ? blockIdx.x / a.groups : blockIdx.x % a.slices;
    const int group = (int)(a.by_slice ? blockIdx.x % a.groups : blockIdx.x / a.slices);
    const Columns at(((int64_t)slice * G + lane) * 8, a.dim);
    if (group >= a.sum_groups) return fill_rows<S, G>(a, group - a.sum_groups, at);
    extern __shared__ Entry s_e[];                          // [TEAMS * each + 2]: with the entry before, and that behind
    __shared__ S s_head[TEAMS][8][G];                       // what G threads have of an id that begins before theirs
    const uint32_t none = (uint32_t)a.rows;
    const int64_t from0 = (int64_t)group * TEAMS * a.each - 1;
    for (int j = threadIdx.x; j < TEAMS * a.each + 2; j += kSumThreads) s_e[j] = from0 + j >= 0 && from0 + j < a.n ? a.e[from0 + j] : Entry{none, 0};
    __syncthreads();
    auto key_at = [&](int i) { return s_e[i].key; };
    // rows of dy of the entries `from` to `to` of s_e; between(key, sum) before each is added
    auto add = [&](int from, int to, auto between) {
        V sum = V{0, 0, 0, 0, 0, 0, 0, 0};
        if (!at.on) return sum;
        auto row = [&](const Entry& e) { return (const DT*)a.dy + (int64_t)e.at * a.ld_dy + at.col; };
        if (a.dim < 8) {
#pragma unroll 1
            for (int i = from; i < to; ++i) {
                const Entry e = s_e[i];
                between(e.key, sum);
                if (e.key != none)
#pragma unroll
                    for (int c = 0; c < 7; ++c)
                        if (c < at.count) sum[c] += (S)(float)row(e)[c];
            }
            return sum;
        }
#pragma unroll 1
        for (int i = from; i < to; i += U) {
            R v[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const Entry e = i + u < to ? s_e[i + u] : Entry{none, 0};
                v[u] = R{};
                if (e.key != none) v[u] = reinterpret_cast<const typename Eight<DT>::Any*>(row(e))->v;
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (i + u < to) between(key_at(i + u), sum);
                sum += __builtin_convertvector(__builtin_convertvector(v[u], float8_t), V);
            }
        }
        return sum;
    };
    auto leave = [&](uint32_t key, V sum) {
        if (key != none && at.on) store_upto8(a.dw, (int64_t)key * a.ld_dw + at.col, a.dw_dtype, scaled<S>(sum, a.scale), at.count, a.stream);
    };
    int first = 1 + team * a.each;
    const int last = first + a.each;                        // (entries past the end have no id)
    const uint32_t key0 = key_at(first), key1 = key_at(last - 1);
    const bool from_before = key0 != none && key_at(first - 1) == key0, goes_on = key1 != none && key_at(last) == key1;
    if (from_before) {
        const int end = end_of(s_e, first, last, key0);
        const V sum = add(first, end, [](uint32_t, V&) {});
#pragma unroll
        for (int i = 0; i < 8; ++i) s_head[team][i][lane] = sum[i];
        first = end;
    }
    V rest = V{0, 0, 0, 0, 0, 0, 0, 0};
    const bool begins = first < last;
    if (begins) {
        uint32_t key = key_at(first);
        rest = add(first, last, [&](uint32_t next, V& sum) {
            if (next == key) return;
            leave(key, sum);
            key = next;
            sum = V{0, 0, 0, 0, 0, 0, 0, 0};
        });
        if (!goes_on) leave(key, rest);
    }
    __syncthreads();
    // adds what the threads from `t` on have of the id `key`; true: it goes on behind the workgroup's entries
    auto follow = [&](V& sum, uint32_t key, int t) {
        for (;; ++t) {
            if (t == TEAMS) return true;
#pragma unroll
            for (int i = 0; i < 8; ++i) sum[i] += s_head[t][i][lane];
            const int next = 1 + (t + 1) * a.each;
            if (key_at(next - 1) != key || key_at(next) != key) return false;
        }
    };
    auto keep = [&](S* part, V sum) {
        if (at.on) reinterpret_cast<typename AnyEight<S>::type*>(part + at.col)->v = sum;
    };
    if (begins && goes_on) {
        if (follow(rest, key1, team + 1)) keep(a.tail(group), rest);
        else leave(key1, rest);
    }
    if (team == 0 && from_before) {
        V sum = V{0, 0, 0, 0, 0, 0, 0, 0};
        follow(sum, key0, 0);
        keep(a.head(group), sum);
    }
}

// What the workgroups left of ids that go on from one to the next: G threads look after the end of one; where an id begins in it that goes on, they add up its
// parts, in order.  Ids of more than kFewParts parts are left to all threads of the workgroup.
constexpr int kFewParts = 16;
template <typename S, int G>
__global__ void __launch_bounds__(1024) embedding_join_kernel(Sums<S> a) {
    typedef double D8 __attribute__((ext_vector_type(8)));
    constexpr int TEAMS = 1024 / G;
    __shared__ int s_parts[TEAMS];
    __shared__ double s_sum[TEAMS][8][G];
    const int lane = threadIdx.x % G, team = threadIdx.x / G;
    const Columns at(((int64_t)blockIdx.y * G + lane) * 8, a.dim);
    const int64_t span = kSumThreads / G * a.each;
    const int group0 = blockIdx.x * TEAMS;
    auto key_at = [&](int64_t i) { return a.e[i].key; };
    // parts behind the tail of the group's last id; 0: it does not go on, or begins before
    auto parts_of = [&](int group) -> int {
        const int64_t first = group * span, next = first + span;
        if (next >= a.n) return 0;
        const uint32_t key = key_at(next - 1), behind = key_at(next), own = key_at(first), before = key_at(max(first, (int64_t)1) - 1);
        if (key >= (uint32_t)a.rows || behind != key || (first > 0 && before == key && own == key)) return 0;
        // the last group whose first entry is of this id: G at a time, then in steps of G, G * G ..
        int64_t lo = group + 1, step = 1;
        for (;;) {
            const int64_t c = lo + (lane + 1) * step;
            const bool same = c < a.sum_groups && key_at(c * span) == key;
            const uint64_t all = __ballot(same) >> (threadIdx.x & 63 & ~(G - 1));
            const int those = __popcll(G < 64 ? all & ((1ull << (G & 63)) - 1) : all);
            lo += those * step;
            if (those == G) step *= G;
            else if (step == 1) break;
            else step /= G;
        }
        return (int)(lo - group);
    };
    auto add_heads = [&](D8& sum, int from, int to) {
        if (!at.on) return;
#pragma unroll 4
        for (int c = from; c < to; ++c) sum += __builtin_convertvector(reinterpret_cast<const typename AnyEight<S>::type*>(a.head(c) + at.col)->v, D8);
    };
    auto leave = [&](int group, D8 sum) {
        if (at.on) store_upto8(a.dw, (int64_t)key_at((group + 1) * span) * a.ld_dw + at.col, a.dw_dtype, __builtin_convertvector(sum * (double)a.scale, float8_t), at.count);
    };
    auto tail_of = [&](int group) {
        D8 sum = D8{0, 0, 0, 0, 0, 0, 0, 0};
        if (at.on) sum = __builtin_convertvector(reinterpret_cast<const typename AnyEight<S>::type*>(a.tail(group) + at.col)->v, D8);
        return sum;
    };
    const int group = group0 + team, parts = group < a.sum_groups ? parts_of(group) : 0;
    if (lane == 0) s_parts[team] = parts;
    if (parts > 0 && parts <= kFewParts) {
        D8 sum = tail_of(group);
        add_heads(sum, group + 1, group + 1 + parts);
        leave(group, sum);
    }
    if (!__syncthreads_or(parts > kFewParts)) return;
    for (int t = 0; t < TEAMS; ++t) {
        const int n = s_parts[t];                           // (the same for all threads)
        if (n <= kFewParts) continue;
        const int c = group0 + t, each = (n + TEAMS - 1) / TEAMS, from = min(n, team * each), to = min(n, from + each);
        D8 sum = D8{0, 0, 0, 0, 0, 0, 0, 0};
        if (team == 0) sum = tail_of(c);
        add_heads(sum, c + 1 + from, c + 1 + to);
#pragma unroll
        for (int i = 0; i < 8; ++i) s_sum[team][i][lane] = sum[i];
        __syncthreads();
#pragma unroll
        for (int half = TEAMS / 2; half > 0; half /= 2) {
            if (team < half)
#pragma unroll
                for (int i = 0; i < 8; ++i) s_sum[team][i][lane] += s_sum[team + half][i][lane];
            __syncthreads();
        }
        if (team == 0) {
#pragma unroll
            for (int i = 0; i < 8; ++i) sum[i] = s_sum[0][i][lane];
            leave(c, sum);
        }
        __syncthreads();
    }
}

template <typename F> void of_type(int32_t t, F f) {
    if (t == LF_DTYPE_F32) f(0.f); else if (t == LF_DTYPE_BF16) f((__bf16)0.f); else f((_Float16)0.f);
}

inline size_t padded(size_t bytes) { return (bytes + 255) / 256 * 256; }
// Entries that some threads take one after the other: eight up to 1024 wavefronts of eights (1440 ids of 16 columns 17 us, in sixteens 22), then as many as leave up to 8192
// wavefronts, and 64 for more.
int entries_each(int64_t n, int64_t dim) {
    const int64_t waves = n * ceil_div(dim, 8 * group_of(dim)) * group_of(dim) / 64;
    return waves <= 8 * 1024 ? 8 : waves <= 16 * 8192 ? 16 : waves <= 32 * 8192 ? 32 : kMostEach;
}
int64_t sum_groups(int64_t n, int64_t dim) { return ceil_div(n, (int64_t)entries_each(n, dim) * (kSumThreads / group_of(dim))); }
inline int sum_bytes(int32_t dtype) { return dtype == LF_DTYPE_F32 ? 8 : 4; }
struct GradWork { size_t entries, counts, totals, present, parts, total; };
GradWork grad_work(int64_t n, int64_t rows, int64_t dim, int32_t dtype) {
    const Passes p = passes_of(rows, kMostBits);
    const int64_t groups = sum_groups(n, dim);
    GradWork w{padded((size_t)n * sizeof(Entry)), 0, 0, 0, 0, 0};
    if (n > kSmall) {
        w.counts = padded(((size_t)sort_groups(n) << p.bits) * 4);
        w.totals = padded(4 << p.bits);
        w.present = padded(rows);
    }
    if (groups > 1) w.parts = (size_t)groups * 2 * (size_t)(ceil_div(dim, 8) * 8) * sum_bytes(dtype);
    w.total = (n > kSmall ? 2 : 1) * w.entries + w.counts + w.totals + w.present + w.parts;
    return w;
}
template <typename DT, typename S, int G> int launch_sums(Sums<S> a, hipStream_t st) {
    const int64_t slices = ceil_div(a.dim, 8 * G);
    // rows to a wavefront: 64, or fewer for enough of them
    a.fill_rows = a.rows * slices >= 64 * 4096 ? 64 : 16;
    const int64_t fill = ceil_div(a.rows, (int64_t)a.fill_rows * (kSumThreads / 64));
    a.slices = (uint32_t)slices;
    a.groups = (uint32_t)(a.sum_groups + fill);
    // Neighbouring workgroups take the slices of a row, so that it is read and written whole by what is on the GPU at once (16,384 ids of 32,000 x 4096
    // bf16 104 us, one slice after the other 128), but for some sizes of float32.
    a.by_slice = sizeof(DT) == 4 && sums_by_slice(a.n, a.rows, a.dim);
    LF_REQUIRE((a.sum_groups + fill) * slices < (1ll << 32) / kSumThreads, LF_ERR_UNSUPPORTED, "too many rows");
    embedding_sums_kernel<DT, S, G><<<(unsigned)((a.sum_groups + fill) * slices), kSumThreads, (kSumThreads / G * a.each + 2) * sizeof(Entry), st>>>(a);
    LF_HIP(hipGetLastError());
    if (a.sum_groups > 1) {
        embedding_join_kernel<S, G><<<dim3((unsigned)ceil_div(a.sum_groups, 1024 / G), (unsigned)slices), 1024, 0, st>>>(a);
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
    const uint8_t* present = nullptr;
    char* at = (char*)d_work;
    if (a.n) {
        const GradWork w = grad_work(a.n, a.rows, a.dim, a.dy_dtype);
        SortArgs s{{a.d_ids, a.ids_stride, a.n, a.rows, a.ids_bits == 64}, nullptr, (Entry*)at, nullptr, nullptr, nullptr, a.n, kTile * tiles_each(a.n), 0, 0, (int32_t)sort_groups(a.n), 0, 0};
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
            present = s.present = (uint8_t*)(at + 2 * w.entries + w.counts + w.totals);
            s.bits = p.bits;
            for (int pass = 0; pass < p.passes; ++pass) {
                s.from = sorted;
                s.to = turn[pass & 1];
                s.shift = pass * p.bits;
                s.first = pass == 0;
                s.last = pass == p.passes - 1;
                sort_count_kernel<<<s.groups, kSortThreads, 0, st>>>(s);
                LF_HIP(hipGetLastError());
                const bool few = sort_adds_counts(s.groups, p.bits);
                if (!few) {
                    sort_offsets_kernel<<<(unsigned)ceil_div(1 << p.bits, 16), 1024, 0, st>>>(s);
                    LF_HIP(hipGetLastError());
                }
                (few ? sort_move_kernel<true> : sort_move_kernel<false>)<<<s.groups, kSortThreads, 0, st>>>(s);
                LF_HIP(hipGetLastError());
                sorted = s.to;
            }
            at += 2 * w.entries + w.counts + w.totals + w.present;
        }
    }
    const int group = group_of(a.dim);
    int rc = LF_OK;
    of_type(a.dy_dtype, [&](auto t) {
        using T = decltype(t);
        using S = std::conditional_t<std::is_same_v<T, float>, double, float>;
        const Sums<S> k{sorted, present, a.d_dy, a.d_grad, (S*)at, a.n, a.ld_dy, a.rows, a.dim, a.ld_grad, ceil_div(a.dim, 8) * 8, a.grad_dtype, entries_each(a.n, a.dim),
                        (int32_t)sum_groups(a.n, a.dim), 0, a.rows * a.dim * dtype_bytes(a.grad_dtype) >= kStreamBytes, 0, 0, 0, a.scale};
        rc = group == 8 ? launch_sums<T, S, 8>(k, st) : group == 16 ? launch_sums<T, S, 16>(k, st) : group == 32 ? launch_sums<T, S, 32>(k, st) : launch_sums<T, S, 64>(k, st);
    });
    return rc;
}

}  // extern "C"
