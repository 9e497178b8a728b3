// rows_share against the bytes themselves, rows of every small size, stride and distance.
#include <cstdio>
#include <set>
#include <vector>

#include "../../sme_gemm_b200/csrc/rows.h"

using namespace smeg;

int main() {
    long n = 0, shared = 0;
    const uintptr_t base = 1 << 20;
    for (int rows : {0, 1, 2, 3, 5})
        for (int wa : {1, 2, 5})
            for (int wb : {1, 3, 4})
                for (int sa = wa; sa <= wa + 6; ++sa)
                    for (int sb = wb; sb <= wb + 8; ++sb)
                        for (int d = -70; d <= 70; ++d) {
                            std::set<uintptr_t> bytes;
                            const uintptr_t at = base + d;
                            for (int i = 0; i < rows; ++i)
                                for (int x = 0; x < 2 * wa; ++x) bytes.insert(base + 2 * i * sa + x);
                            bool want = false;
                            for (int i = 0; i < rows; ++i)
                                for (int x = 0; x < 2 * wb; ++x) want = want || bytes.count(at + 2 * i * sb + x);
                            const RowsAt a = {(const uint16_t*)base, (size_t)sa, (size_t)wa}, b = {(const uint16_t*)at, (size_t)sb, (size_t)wb};
                            if (rows_share(a, b, rows) != want || rows_share(b, a, rows) != want)
                                return std::printf("rows %d widths %d %d strides %d %d distance %d: %d\n", rows, wa, wb, sa, sb, d, want), 1;
                            ++n;
                            shared += want;
                        }
    const RowsAt none = {nullptr, 8, 8}, some = {(const uint16_t*)base, 8, 8};
    if (rows_share(none, some, 3) || rows_share(some, none, 3) || !same_rows(some, some, 3)) return 1;
    std::printf("ok %ld %ld\n", n, shared);
    return 0;
}
