// The index arithmetic of sme_gemm_b200/csrc/paged.h on sound batches (it has to be exact) and on batches of any values (it has to stay inside the
// buffers).  Prints "ok <checks>"; "sizes" prints the sizes of the argument structures.
#include <cstdio>
#include <cstring>
#include <random>
#include <set>
#include <vector>

#include "../../include/smeg_api.h"
#include "../../sme_gemm_b200/csrc/paged.h"

using namespace smeg;
static long checks = 0;
#define REQUIRE(x)                                                                  \
    do {                                                                            \
        ++checks;                                                                   \
        if (!(x)) { std::printf("line %d: %s\n", __LINE__, #x); return 1; }         \
    } while (0)

struct Batch {
    std::vector<int> cu, starts, table;
    PackedSeqs p;
    void bind(int rows, int cols, int pages, int page_log2) {
        p = {cu.data(), starts.data(), table.data(), (int)starts.size(), cols, rows, pages, page_log2};
    }
};

static int count_upto(const PackedSeqs& p, long long x, int log2_len, int extra, int group) {
    int n = 0;
    for (int s = 0; s < p.seqs; ++s) {
        int f;
        seq_rows(p, s, &f);
        n += first_slot((long long)f * group, s, log2_len, extra) <= x;
    }
    return n;
}

// Every slot of the grid, as the kernels resolve it: what it covers, within the buffers.  Returns the rows covered (with their multiplicity).
static int walk(Batch& b, int log2_len, int extra, int group, std::vector<int>* seen) {
    const PackedSeqs& p = b.p;
    const long long slots = ((long long)p.rows * group >> log2_len) + (long long)extra * p.seqs;
    for (long long j = 0; j < slots; ++j) {
        const int s = count_upto(p, j, log2_len, extra, group) - 1;
        if (s < 0) continue;
        REQUIRE(s < p.seqs);
        int first;
        const int rows = seq_rows(p, s, &first);
        REQUIRE(first >= 0 && rows >= 0 && first + rows <= p.rows);
        const long long piece = j - first_slot((long long)first * group, s, log2_len, extra);
        if (piece < 0) continue;                                       // (offsets that go back)
        const int start = extra == 2 ? p.starts[s] : 0;
        if (start < 0) continue;
        const long long d = extra == 2 ? start & ((1 << log2_len) - 1) : 0, n = (long long)rows * group;
        if (piece >= pieces(n, d, log2_len)) continue;
        const long long len = 1ll << log2_len, r0 = piece == 0 ? 0 : piece * len - d, r1 = std::min(n, (piece + 1) * len - d);
        REQUIRE(0 <= r0 && r0 < r1 && r1 <= n);
        if (extra == 2) {
            const long long pos = (long long)start + r0;
            const int id = page_of(p, s, pos);
            REQUIRE(id >= -1 && id < p.pages);
            const int at = piece == 0 ? (int)d : 0;
            REQUIRE(at + (r1 - r0) <= len && ((pos & (len - 1)) == at));
        }
        if (seen)
            for (long long r = r0; r < r1; ++r) (*seen)[(size_t)first * group + r]++;
    }
    return 0;
}

static int shares(Batch& b, int group, int kv, int tile, int workers) {
    long long total = 0;
    for (int s = 0; s < b.p.seqs; ++s) {
        const SeqUnits u = seq_units(b.p, s, group, kv, tile);
        REQUIRE(u.keys >= 0 && u.keys <= ((long long)b.p.cols << b.p.page_log2));
        REQUIRE(u.tiles >= 1 && u.items >= 0 && u.first >= 0 && u.first + u.rows <= b.p.rows);
        REQUIRE((long long)u.tiles * kUnitKeys >= u.keys && (u.keys == 0 || (long long)(u.tiles - 1) * kUnitKeys < u.keys));
        total += u.items * u.tiles;
    }
    REQUIRE(share_begin(total, workers, 0) == 0 && share_begin(total, workers, workers) == total);
    for (int w = 0; w < workers; ++w) {
        const long long a = share_begin(total, workers, w), e = share_begin(total, workers, w + 1);
        REQUIRE(a <= e && e - a <= total / workers + 1);
        if (a < e) REQUIRE(share_of(total, workers, a) == w && share_of(total, workers, e - 1) == w);
    }
    return 0;
}

int main(int argc, char** argv) {
    if (argc > 1 && !std::strcmp(argv[1], "sizes")) {
        std::printf("%zu %zu %zu %zu %zu %zu\n", sizeof(smeg_rotate_args), offsetof(smeg_rotate_args, start), sizeof(smeg_paged_attend_args),
                    offsetof(smeg_paged_attend_args, workspace_bytes), sizeof(smeg_attn_packed_args), sizeof(smeg_paged_read_args));
        return 0;
    }
    for (uint32_t d : {1u, 2u, 3u, 5u, 7u, 8u, 12u, 24u, 63u, 64u, 100u, 641u, 65535u})
        for (uint64_t n : {0ull, 1ull, 2ull, 6ull, 7ull, 8ull, 65535ull, 1000003ull, 2147483646ull, 2147483647ull})
            for (int e = -2; e <= 2; ++e) {
                const long long x = (long long)(n / d * d) + e;
                if (x >= 0 && x <= 2147483647) REQUIRE(div_by((int)x, fast_div(d)) == (int)(x / d));
            }
    for (long long total : {0ll, 5ll, 443ll, 444ll, 4294967295ll, 4294967296ll, 1234567890123ll})
        for (int n : {1, 7, 444}) {
            for (int w = 0; w <= n; ++w) REQUIRE(share_begin(total, n, w) == total / n * w + std::min<long long>(w, total % n));
            for (int w = 0; w < n; ++w) {
                const long long a = share_begin(total, n, w), e = share_begin(total, n, w + 1);
                if (a < e) REQUIRE(share_of(total, n, a) == w && share_of(total, n, e - 1) == w);
            }
        }
    std::mt19937_64 rng(7);
    auto pick = [&](long long lo, long long hi) { return lo + (long long)(rng() % (unsigned long long)(hi - lo + 1)); };
    for (int round = 0; round < 3000; ++round) {
        const bool sound = round % 2 == 0;
        const int seqs = (int)pick(1, 12), page_log2 = (int)pick(4, 8), cols = (int)pick(0, 6), pages = (int)pick(0, 9), group = (int)pick(1, 9);
        Batch b;
        b.cu.push_back(0);
        for (int s = 0; s < seqs; ++s) b.cu.push_back(b.cu.back() + (int)(pick(0, 3) == 0 ? 0 : pick(0, 3) == 0 ? pick(0, 700) : pick(1, 5)));
        const int rows = b.cu.back() + (int)pick(0, 3);
        for (int s = 0; s < seqs; ++s) b.starts.push_back((int)(pick(0, 5) == 0 ? -1 : pick(0, 900)));
        for (int i = 0; i < seqs * cols; ++i) b.table.push_back((int)pick(0, pages > 0 ? pages - 1 : 0));
        if (!sound) {
            const int any[] = {-2147483647 - 1, 2147483647, -1, 0, 1, 1000000, -77, rows, rows + 1};
            for (auto* v : {&b.cu, &b.starts, &b.table})
                for (int& x : *v)
                    if (pick(0, 2) == 0) x = pick(0, 1) ? any[pick(0, 8)] : (int)rng();
        }
        b.table.push_back(0);
        b.bind(rows, cols, pages, page_log2);
        for (int extra = 1; extra <= 2; ++extra) {
            const int g = extra == 1 ? group : 1, log2_len = extra == 1 ? (int)pick(6, 8) : page_log2;
            std::vector<int> seen((size_t)rows * g + 1, 0);
            if (walk(b, log2_len, extra, g, sound ? &seen : nullptr)) return 1;
            if (sound)
                for (int s = 0; s < seqs; ++s)
                    for (int r = b.cu[s] * g; r < b.cu[s + 1] * g; ++r) REQUIRE(seen[r] == (extra == 2 && b.starts[s] < 0 ? 0 : 1));
        }
        {                                                          // pieces of any length
            const int len = (int)pick(1, 300);
            std::vector<int> seen((size_t)rows + 1, 0);
            for (long long j = 0; j < rows / len + b.p.seqs; ++j) {
                int n = 0, first = 0;
                for (int s = 0; s < b.p.seqs; ++s) n += (seq_rows(b.p, s, &first), first_slot_of(first, s, len) <= j);
                if (!n) continue;
                const int mine = seq_rows(b.p, n - 1, &first);
                const long long piece = j - first_slot_of(first, n - 1, len);
                if (piece < 0 || piece >= pieces_of(mine, len)) continue;
                for (long long r = piece * len; r < std::min<long long>(mine, (piece + 1) * len); ++r) {
                    REQUIRE(first + r >= 0 && first + r < rows);
                    seen[first + r]++;
                }
            }
            if (sound)
                for (int r = 0; r < b.cu[seqs]; ++r) REQUIRE(seen[r] == 1);
        }
        for (int tile : {8, 16})
            if (shares(b, group, (int)pick(1, 5), tile, (int)pick(1, 500))) return 1;
    }
    std::printf("ok %ld\n", checks);
    return 0;
}
