// Rows in a buffer: `rows` of `width` floats, `ld` >= width apart. Host only; no product of a caller's numbers is taken before it is known to fit 64 bits.
#pragma once
#include <stddef.h>
#include <stdint.h>

#include <algorithm>

namespace alice {

inline bool rows_fit(size_t len, size_t rows, size_t ld, size_t width) {
    return rows == 0 || (len >= width && (rows == 1 || (len - width) / (rows - 1) >= ld));
}
// floats that rows which fit span
inline size_t rows_span(size_t rows, size_t ld, size_t width) { return rows ? (rows - 1) * ld + width : 0; }
// rows, up to `most`, of x and as many of y none of which meets one of the other's: all where they lie side by side in rows as wide for both, else those of the first
// that end before the other's begin. Rows of which `most` fit.
inline size_t rows_apart(const float* x, size_t x_ld, size_t x_width, const float* y, size_t y_ld, size_t y_width, size_t most) {
    if (reinterpret_cast<uintptr_t>(x) > reinterpret_cast<uintptr_t>(y)) return rows_apart(y, y_ld, y_width, x, x_ld, x_width, most);
    const size_t off = (reinterpret_cast<uintptr_t>(y) - reinterpret_cast<uintptr_t>(x)) / sizeof(float);
    if (x_ld == y_ld && off % x_ld >= x_width && off % x_ld + y_width <= x_ld) return most;
    return off < x_width ? 0 : std::min(most, (off - x_width) / x_ld + 1);
}

}  // namespace alice
