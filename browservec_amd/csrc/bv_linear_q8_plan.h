// Which tiles a product of codes goes by (bv_linear_q8.hip): the shapes that there
// are, what each takes, and the choice.  Plain C++.
#pragma once

#include <stdint.h>

namespace bvk {

// Shapes of tiles, and when one is done with m rows: `fix` and rounds of the tiles that
// the card holds at a time, each a + b k and what its activations take; the last round
// of fewer tiles is `part` hundredths of one and their share of the rest (ns, fitted to
// 40..32768 x 384..4096 x 384..4096 without an activation, within 3 to 7%: the shapes
// chosen take 1.3% more than each size's best).  32768 x 1024, k 1024: 50.5 us in the last,
// the others 53.4, 59.2, 60.8, 75.4, 113, 107 and 141; 2037 x 768, k 768: 17.6, 12.6, 14.7,
// 11.8, 8.8, 7.5, 7.6 and 10.7; 200 x 1024, k 4096: 51, 39, 43, 35, 26, 18, 14 and 11.
struct Q8Shape {
    uint32_t bm, bn, bk;                      // a tile's rows, columns, and codes of a step
    uint32_t cus, part, fix, a, b, gelu;      // cus: tiles of a compute unit
};
constexpr int Q8_SHAPES = 8;
constexpr Q8Shape q8_shapes[Q8_SHAPES] = {
    {64, 64, 512, 1, 80, 2150, 2906, 163, 470},    {64, 64, 256, 2, 55, 2391, 2494, 375, 750},
    {64, 128, 256, 1, 80, 2116, 3082, 361, 940},   {128, 128, 128, 1, 85, 1883, 2968, 585, 1880},
    {128, 256, 128, 1, 80, 1815, 5220, 845, 3760}, {192, 256, 128, 1, 75, 1829, 7617, 1105, 4400},
    {128, 256, 64, 2, 45, 2504, 7446, 1590, 3000}, {256, 256, 128, 1, 70, 2947, 7700, 1389, 7500}};

inline uint64_t q8_done_in(uint64_t m, uint32_t n, uint32_t k, int act, const Q8Shape &t) {
    const uint64_t tiles = ((m + t.bm - 1) / t.bm) * (((uint64_t)n + t.bn - 1) / t.bn), at_a_time = 256 * t.cus, rest = tiles % at_a_time;
    const uint64_t rounds = tiles / at_a_time * 100 + (rest ? t.part + (100 - t.part) * rest / at_a_time : 0);
    return t.fix + rounds * (t.a + (uint64_t)t.b * k / 100 + (act > 1 ? t.gelu : 0)) / 100;
}
inline uint64_t q8_done_in(uint64_t m, uint32_t n, uint32_t k, int act, int *shape) {
    uint64_t least = ~0ull;
    for (int i = 0; i < Q8_SHAPES; i++) {
        const uint64_t ns = q8_done_in(m, n, k, act, q8_shapes[i]);
        if (ns < least) least = ns, *shape = i;
    }
    return least;
}

// Whole rounds of tiles in one shape, and the rows that are left in another, where
// that is done first.  20011 x 1024, k 4096: 16384 rows in 256 x 256 tiles and 3627 in 128 x
// 128, 135 -> 125 us; 16492 x 1024, k 1024, GELU: 42.3 -> 37.9.  2 us: what the second launch adds.
struct Q8Plan {
    int shape;      // of the first `rows` rows
    uint64_t rows;
    int then;       // of the others, where there are any
};
inline Q8Plan q8_plan(uint64_t m, uint32_t n, uint32_t k, int act) {
    Q8Plan p{0, m, 0};
    uint64_t least = q8_done_in(m, n, k, act, &p.shape);
    for (int i = 0; i < Q8_SHAPES; i++) {
        const Q8Shape &t = q8_shapes[i];
        const uint64_t tiles_n = ((uint64_t)n + t.bn - 1) / t.bn, at_a_time = 256 * t.cus;
        const uint64_t whole = (m + t.bm - 1) / t.bm * tiles_n / at_a_time * at_a_time / tiles_n * t.bm;
        if (whole == 0 || whole >= m) continue;
        int j = 0;
        const uint64_t ns = q8_done_in(whole, n, k, act, t) + q8_done_in(m - whole, n, k, act, &j) + 2000;
        if (ns < least) least = ns, p = {i, whole, j};
    }
    return p;
}

}  // namespace bvk
