// ft_overlap.hpp -- whether two sets of rows in memory have a byte in common:
// what an entry point refuses of its inputs and outputs. Host code without the
// GPU runtime, so that a test compiles it alone.
#pragma once

#include <stdint.h>

namespace ft {

// `n` rows of `bytes` bytes, each `stride` bytes after the one before (stride >= bytes). None where at is null.
struct Span {
    const void* at;
    int64_t n, stride, bytes;
};

// Exact, so that rows beside rows in one buffer (columns of a wider matrix) are none of each other's. Rows of one
// stride, and a single row beside any, are decided at once; rows of two strides whose extents meet, row by row.
inline bool overlap(const Span& a, const Span& b) {
    using wide = __int128;
    if (!a.at || !b.at || a.n <= 0 || b.n <= 0 || a.bytes <= 0 || b.bytes <= 0) return false;
    const wide d = (wide)(uintptr_t)a.at - (wide)(uintptr_t)b.at;  // a's first byte past b's
    const wide a_len = (wide)(a.n - 1) * a.stride + a.bytes, b_len = (wide)(b.n - 1) * b.stride + b.bytes;
    if (d >= b_len || -d >= a_len) return false;
    // whether any of n rows at base + k * stride, each `bytes` long, meets [at, at + len)
    const auto meets = [](wide base, int64_t n, int64_t stride, int64_t bytes, wide at, wide len) {
        wide k = at - bytes - base;  // the first row that ends past `at`
        k = k < 0 ? 0 : k / stride + 1;
        return k < n && base + k * stride < at + len;
    };
    if (b.n == 1) return meets(d, a.n, a.stride, a.bytes, 0, b.bytes);
    if (a.n == 1) return meets(0, b.n, b.stride, b.bytes, d, a.bytes);
    if (a.stride == b.stride)  // row i of a lies to row j of b as i - j says
        return meets(d - (wide)(b.n - 1) * a.stride, a.n + b.n - 1, a.stride, a.bytes, 0, b.bytes);
    for (int64_t i = 0; i < a.n; ++i)
        if (meets(0, b.n, b.stride, b.bytes, d + (wide)i * a.stride, a.bytes)) return true;
    return false;
}

}  // namespace ft
