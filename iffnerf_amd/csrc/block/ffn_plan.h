// ffn_plan.h -- which tiles the products of the gated feed-forward block are cut into (ffn_kernels.hip).  Host code without HIP: a function of
// sizes and types alone, so that a size query and a call, and a test on a machine without a GPU, get the same answer.
#pragma once
#include <stdint.h>

#include <algorithm>

namespace {

constexpr int64_t pad8(int64_t n) { return (n + 7) / 8 * 8; }

// ---- which tiles, and how many shares of the k loop.  A round is one tile on every CU (two of the 128 x 128 ones); its time is modelled as
// the k loop at the rate measured on full rounds (1.8 us per 64 k of a 256 x 256 tile; the smaller tiles move more operand bytes per
// product: 5 % and 20 % on top) plus the epilogue's traffic at 4.5 GB/ms.  Two things decide between the shapes: how full the last round is
// (a weight gradient of 8192 x 1536: one round of 256 x 192 tiles in 369 us, 0.75 rounds of 256 x 256 ones in 447 us), and the rows behind the last whole
// tile (257 tokens per image leave 64 of them): as tiles of 256 they can cost a whole round, as a second launch of 128 x 128 tiles
// about 6 us and their k loop.
// A product with few tiles is bound by the latency of its steps instead: 0.85 us per 64 k of a 128 x 128 tile alone on its CU with two buffers,
// less with four (then the tile has the CU to itself), and 64 x 64 tiles bring four times the workgroups.
enum { SHAPE_256 = 0, SHAPE_192, SHAPE_128, SHAPE_128_DEEP, SHAPE_64, SHAPES };
constexpr struct Shape { int bm, bn, slots_log2; double step; } kShape[SHAPES] = {     // step: us per 64 k of a round
    {256, 256, 8, 1.8}, {256, 192, 8, 1.42}, {128, 128, 9, 1.08}, {128, 128, 8, 0.60}, {64, 64, 9, 0.45}};
struct Plan { int shape, splits; int64_t main_rows; int rest_shape, rest_splits; };      // the rows behind main_rows go to a launch of their own

// rows x N of C in one launch of `shape`, us (this runs at every call: nothing but the tile counts is divided per shape)
struct Cost {
    int64_t tiles[SHAPES]; double elements, traffic;
    Cost(int64_t rows, int64_t N, double out_bytes) : elements((double)rows * N), traffic((double)rows * N * out_bytes / 4.5e6) {
        for (int i = 0; i < SHAPES; ++i) tiles[i] = (rows + kShape[i].bm - 1) / kShape[i].bm * ((N + kShape[i].bn - 1) / kShape[i].bn);
    }
    double of(int shape, int splits, double steps) const {
        const Shape& s = kShape[shape];
        const int64_t rounds = (tiles[shape] * splits + (1 << s.slots_log2) - 1) >> s.slots_log2;
        return (double)rounds * (steps * s.step + 3.0) + traffic + (splits > 1 ? 5.0 + elements * 4 * (splits + 1) / 4.5e6 : 0.0);
    }
};
// out_bytes: what the epilogue moves per element of C; most: shares of the k loop that may be taken, each at least 256 deep
inline Plan plan_tiles(int64_t M, int64_t N, int64_t K, double out_bytes, bool may_192, int most, bool may_rest = true) {
    Plan best{SHAPE_128, 1, M, SHAPE_128, 1};
    double least = 1e300, rest = 1e300;
    const int64_t whole = may_rest && M % 256 ? M / 256 * 256 : 0;
    const Cost all(M, N, out_bytes), behind(M - whole, N, out_bytes), front(whole, N, out_bytes);
    const double steps_1 = (double)((K + 63) / 64);
    int rest_shape = SHAPE_128, rest_splits = 1;
    for (int z = 1; z <= most && (z == 1 || K >= 256 * (int64_t)z); z += z < 8 ? 1 : z < 16 ? 2 : 8) {      // 1 .. 8, 10 .. 16, 24 .. 64
        const double steps = z == 1 ? steps_1 : (double)((K + 64 * z - 1) / (64 * z));
        for (int shape = SHAPE_256; shape < SHAPES; ++shape) {
            if (shape == SHAPE_192 && !may_192) continue;
            const double t = all.of(shape, z, steps);
            if (t < least) { least = t; best = {shape, z, M, SHAPE_128, 1}; }
            if (!whole || shape < SHAPE_128 || z > 16) continue;
            const double r = 6.0 + behind.of(shape, z, steps);
            if (r < rest) { rest = r; rest_shape = shape; rest_splits = z; }
        }
    }
    for (int shape = SHAPE_256; whole && shape <= SHAPE_192; ++shape) {
        if (shape == SHAPE_192 && !may_192) continue;
        const double two = front.of(shape, 1, steps_1) + rest;
        if (two < least) { least = two; best = {shape, 1, whole, rest_shape, rest_splits}; }
    }
    return best;
}

// The plans of a call's products.  es: bytes of the type; pairs: products of planes per product (fp32 6, else 1).
// [g | u] of M rows over K, HP gate and HP up columns; keeps: p and q are written too
inline Plan gate_plan(int64_t M, int64_t HP, int64_t K, int es, int pairs, bool keeps) {
    return plan_tiles(M, 2 * HP, K * pairs, (es + (keeps ? 8 : 0)) / 2.0, false, 1);
}
// dh, with p and q read and [dg | du] written
inline Plan dh_plan(int64_t M, int64_t HP, int64_t K, int es, int pairs) {
    Plan p = plan_tiles(M, HP, K * pairs, 8 + 2 * es, false, 1);
    if (p.rest_shape == SHAPE_64) p.rest_shape = SHAPE_128_DEEP;     // (one height of the waves' rows, that of the sums, per product)
    return p;
}
// y and dx
inline Plan rows_plan(int64_t M, int64_t N, int64_t K, int es, int pairs) {
    return plan_tiles(M, N, K * pairs, es, false, (int)std::max<int64_t>(1, std::min<int64_t>(16, K / 64)));
}
// a weight gradient of M x N over K rows of the batch
inline Plan weight_plan(int64_t M, int64_t N, int64_t K, int es, int pairs) {
    return plan_tiles(M, N, K * pairs, es, true, (int)std::max<int64_t>(1, std::min<int64_t>(64, K / 256)), false);
}

}  // namespace
