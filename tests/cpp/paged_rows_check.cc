// keys_of_row and beyond_table of paged.h at starts of every size, against 128-bit arithmetic.
#include <cstdio>
#include <cstdlib>
#include <random>

#include "../../sme_gemm_b200/csrc/paged.h"

using namespace smeg;

int main() {
    std::mt19937_64 rng(7);
    const int starts[] = {-2147483647 - 1, -5, -1, 0, 1, 15, 16, 63, 64, 1000, 1 << 20, 2147483647 - 70, 2147483647 - 1, 2147483647};
    long n = 0;
    for (int start : starts)
        for (int cols : {0, 1, 4, 100, 1 << 22, 0x7fffffff / 16})
            for (int rows : {0, 1, 3, 70, 1 << 20, 2147483647}) {
                const int cu[2] = {0, rows}, table[1] = {0};
                const PackedSeqs p = {cu, &start, table, 1, cols, rows, 1, 4};
                const SeqUnits u = seq_units(p, 0, 1, 1, 8);
                const __int128 room = (__int128)cols * 16, end = (__int128)start + rows;
                if (beyond_table(u) != (start >= 0 && end > room)) return std::printf("beyond: start %d cols %d rows %d\n", start, cols, rows), 1;
                for (int k = 0; k < 20 && rows; ++k) {
                    const int i = k == 0 ? 0 : (k == 1 ? rows - 1 : (int)(rng() % (unsigned long long)rows));
                    __int128 want = (__int128)start + i + 1;
                    if (want > room) want = room;
                    if (want > end) want = end;
                    if (start < 0) want = 0;
                    if (keys_of_row(u, i) != (int)want) return std::printf("keys: start %d cols %d rows %d row %d\n", start, cols, rows, i), 1;
                    ++n;
                }
            }
    std::printf("ok %ld\n", n);
    return 0;
}
