// Which kernel a dense product takes (lf_linear.hip), by its sizes, the size of its elements and the alignment of its operands.  Plain functions, which a
// host program may call as well.
#ifndef LF_CUT_H
#define LF_CUT_H
#include <algorithm>
#include <cstddef>
#include <cstdint>

namespace lf {

constexpr int kWideTile = 256;
constexpr int64_t kFewRows = 16;

// How a product is cut up: tile, splits of k, bytes of partial sums.
struct Cut { int tile; int splits; int64_t k_split; size_t bytes; };

// Microseconds of a step (128 bytes of k; float32 32 elements) of all workgroups that are on the GPU at once, `each` of them to a CU, as
// measured with products of 64 .. 4096 rows and columns on 256 CUs.  Large tiles do the most to an operand's byte, small ones are more: bf16
// 1024 x 2048 x 2048 in tiles of 128 / 64 takes 25 / 14 us, 4096 x 2048 x 1024 21 / 28, 3000^3 in tiles of 256 / 128 82 / 102.
inline double step_us(bool f32, int tile, int64_t each) {
    static const double k16[2][4] = {{0.23, 0.30, 0.52, 0.80}, {0.65, 1.15, 0, 0}}, k32[2][4] = {{0.70, 1.08, 1.40, 1.74}, {1.80, 2.60, 0, 0}};
    return tile == kWideTile ? 1.5 : (f32 ? k32 : k16)[tile == 128][each - 1];
}
// Of a launch, of an epilogue of a large tile, and of the second kernel where k is split, which reads what the first one wrote at 4 TB/s.
constexpr double kLaunchUs = 4.0, kWideUs = 8.0, kJoinUs = 5.0, kJoinBytesPerUs = 4e6;
constexpr int kCus = 256;

// `bytes` of an element; those of 4 are float32.
inline Cut cut_product(int bytes_each, int64_t m, int64_t n, int64_t k) {
    const bool f32 = bytes_each == 4;
    const int step = f32 ? 32 : 128 / bytes_each;
    auto up = [](int64_t a, int64_t b) { return (a + b - 1) / b; };
    const int64_t steps = std::max<int64_t>(1, up(k, step));
    Cut best{64, 1, steps * step, 0};
    double best_us = 1e300;
    for (const int tile : {64, 128, kWideTile}) {
        if (tile == kWideTile && f32) continue;
        const int64_t tiles = up(m, tile) * up(n, tile), most = (tile == 64 ? 4 : tile == 128 ? 2 : 1) * kCus;
        for (int64_t want = 1; want <= 512 && want * 2 <= steps + 1; want += std::max<int64_t>(1, want / 2)) {
            const int64_t each = up(steps, want), splits = up(steps, each);
            const int64_t groups = tiles * splits, rest = groups % most;
            if (splits > 1 && groups > 2 * most) break;
            const double bytes = splits > 1 ? 4.0 * (double)splits * (double)m * (double)n : 0.0;
            const double us = (double)each * ((double)(groups / most) * step_us(f32, tile, most / kCus) + (rest ? step_us(f32, tile, up(rest, kCus)) : 0.0)) + kLaunchUs +
                              (tile == kWideTile ? kWideUs * (double)up(groups, most) : 0.0) + (splits > 1 ? kJoinUs + 2 * bytes / kJoinBytesPerUs : 0.0);
            if (us < best_us) {
                best_us = us;
                best = {tile, (int)splits, each * step, (size_t)bytes};
            }
        }
    }
    return best;
}

// An operand: rows of a product, k along them or across.
struct Operand { const void* p; int64_t ld, rows; bool across; };
// Whether it can go straight into LDS: pieces of 16 bytes that are aligned (across k whole ones, too), and the rows of a tile within
// 32-bit offsets.
inline bool aligned_operand(const Operand& o, int bytes) {
    return (uintptr_t)o.p % 16 == 0 && o.ld * bytes % 16 == 0 && (o.across ? 64 : 256) * o.ld * bytes < (1ll << 31) && (!o.across || o.rows % 8 == 0);
}

// The kernel: few rows of P; tiles through registers (product_kernel), straight into LDS (direct_kernel), large ones (wide_kernel); deep: few workgroups.
enum { kPathFewRows, kPathProduct, kPathDirect, kPathWide };
struct Path { int kernel; bool deep; Cut cut; };
inline Path path_of(int bytes, const Operand& p, const Operand& q, int64_t k) {
    if (!p.across && !q.across && p.rows <= kFewRows) return {kPathFewRows, false, Cut{}};
    Cut c = cut_product(bytes, p.rows, q.rows, k);
    const bool aligned = bytes < 4 && aligned_operand(p, bytes) && aligned_operand(q, bytes);
    if (c.tile == kWideTile && !aligned) c.tile = 128;
    const int64_t tiles = (p.rows + c.tile - 1) / c.tile * ((q.rows + c.tile - 1) / c.tile);
    return {c.tile == kWideTile ? kPathWide : aligned ? kPathDirect : kPathProduct, tiles * c.splits <= kCus, c};
}

}  // namespace lf
#endif
