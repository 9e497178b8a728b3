// Whether two sets of rows share memory: what the calls on packed batches refuse (api.cu, binding.cc).
#pragma once
#include <stddef.h>
#include <stdint.h>

namespace smeg {

struct RowsAt {
    const uint16_t* at;       // null: none
    size_t stride, width;     // in elements; rows of one set do not overlap
};
inline bool same_rows(const RowsAt& a, const RowsAt& b, size_t rows) { return a.at == b.at && a.width == b.width && (rows == 1 || a.stride == b.stride); }
// `rows` rows each.  Rows of one buffer that lie side by side (slices of [q | k | v] rows) share nothing.
inline bool rows_share(const RowsAt& a, const RowsAt& b, size_t rows) {
    if (!a.at || !b.at || rows == 0) return false;
    const intptr_t a0 = (intptr_t)a.at, b0 = (intptr_t)b.at, wa = 2 * (intptr_t)a.width, wb = 2 * (intptr_t)b.width, sa = 2 * (intptr_t)a.stride, sb = 2 * (intptr_t)b.stride,
                   last = (intptr_t)rows - 1;
    if (a0 + last * sa + wa <= b0 || b0 + last * sb + wb <= a0) return false;
    if (rows == 1) return true;
    if (sa == sb) {
        // row i of a and row j of b: -wb < (b0 - a0) + (j - i) s < wa, for one of the two j - i next to (a0 - b0) / s
        const intptr_t d = b0 - a0;
        intptr_t q = d / sa, r = d - q * sa;
        if (r < 0) { r += sa; --q; }
        return (r < wa && -q <= last && q <= last) || (sa - r < wb && -q - 1 <= last && q + 1 <= last);
    }
    for (intptr_t i = 0; i <= last; ++i) {
        // the first row of b that ends behind this one's start
        const intptr_t lo = a0 + i * sa - wb - b0;
        const intptr_t j = lo < 0 ? 0 : lo / sb + 1;
        if (j <= last && b0 + j * sb < a0 + i * sa + wa) return true;
    }
    return false;
}

}  // namespace smeg
