// int8_slices.h -- how the rows that become 8-bit integers are shared out over
// launches: plain C++ (tests/test_int8_slices.py builds it on its own).
#pragma once
#include <stdint.h>

namespace chimere {

// Columns of a row: a thread counts them in int, four waves of up to eight
// elements a lane, 4096 and a step of 2048 past its last ones.
constexpr int I8_MAX_ROW = 0x7FFFFFFF - 8191;

// A row goes to one wave up to 1024 columns, to four above.
constexpr int I8_WAVE_ROW = 1024;
template <int THREADS>
constexpr int i8_rows_per_group(int ncols) { return THREADS / 64 / (ncols <= I8_WAVE_ROW ? 1 : 4); }

// f(first row, rows, work-groups of THREADS threads) per launch: 2^22
// work-groups at most, since a grid has less than 2^32 threads.
template <int THREADS, typename F>
void i8_slices(int64_t nrows, int ncols, F f) {
    const int per = i8_rows_per_group<THREADS>(ncols);
    const int64_t at_once = ((int64_t)1 << 22) * per;
    for (int64_t r = 0; r < nrows; r += at_once) {
        const int64_t n = nrows - r < at_once ? nrows - r : at_once;
        f(r, n, (n + per - 1) / per);
    }
}

}  // namespace chimere
