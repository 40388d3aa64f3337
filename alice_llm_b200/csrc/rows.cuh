// Rows in a buffer: `rows` of `width` floats, `ld` >= width apart. Host only; no product of a caller's numbers is taken before it is known to fit 64 bits.
#pragma once
#include <stddef.h>

namespace alice {

inline bool rows_fit(size_t len, size_t rows, size_t ld, size_t width) {
    return rows == 0 || (len >= width && (rows == 1 || (len - width) / (rows - 1) >= ld));
}
// floats that rows which fit span
inline size_t rows_span(size_t rows, size_t ld, size_t width) { return rows ? (rows - 1) * ld + width : 0; }

}  // namespace alice
