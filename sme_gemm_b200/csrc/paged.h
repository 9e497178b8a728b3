// Packed batches of sequences and the pages of the 8-bit key/value cache: the index arithmetic of rotary.cu, paged.cu and prompt.cu, on the
// device and on the host (tests/cpp/paged_index_check.cc runs it on values of every kind, sound and not).
//
// Everything here that comes from device memory -- row offsets, starts, page numbers -- may hold anything: it is bounded before it is used, so
// that a wrong table costs its own rows their results (and raises STATUS_PAGE) but no access leaves the buffers.
#pragma once
#include <stddef.h>
#include <stdint.h>

#ifdef __CUDACC__
#define SMEG_HD __host__ __device__ __forceinline__
#else
#define SMEG_HD inline
#endif

namespace smeg {

// Rows cu[s] .. cu[s + 1] of the packed batch belong to sequence s; its first is position starts[s] (below zero: the sequence is idle).  Page
// table[s * cols + i] of the pool holds its positions i * page ...
struct PackedSeqs {
    const int* cu;
    const int* starts;        // null: every sequence starts at position 0
    const int* table;         // null: no cache
    int seqs, cols, rows;
    int pages, page_log2;
};

// Sequence s's rows: the first one, and how many.
SMEG_HD int seq_rows(const PackedSeqs& p, int s, int* first) {
    int a = p.cu[s], b = p.cu[s + 1];
    a = a < 0 ? 0 : (a > p.rows ? p.rows : a);
    b = b < a ? a : (b > p.rows ? p.rows : b);
    *first = a;
    return b - a;
}

// Pieces of `len` things that n things from the d-th on of a run of len touch.
SMEG_HD long long pieces(long long n, long long d, int log2_len) {
    return n <= 0 ? 0 : ((d + n - 1) >> log2_len) + 1;
}

// Work slots: sequence s, whose things (rows, or rows x heads of a group) begin at the packed index `first`, has the slots from
// (first >> log2_len) + extra * s on.  With pieces of 2^log2_len things that start where the sequence does (extra = 1), or anywhere (extra = 2), no two
// sequences share a slot, and there are (total >> log2_len) + extra * seqs of them: the grid needs neither the lengths nor a prefix sum.
SMEG_HD long long first_slot(long long first, int s, int log2_len, int extra) { return (first >> log2_len) + (long long)extra * s; }

// The same for pieces of any length that start where their sequence does.
SMEG_HD long long first_slot_of(long long first, int s, int len) { return first / len + s; }
SMEG_HD long long pieces_of(long long n, int len) { return (n + len - 1) / len; }

// The pool's page that holds position pos of sequence s; -1: none.
SMEG_HD int page_of(const PackedSeqs& p, int s, long long pos) {
    const long long col = pos >> p.page_log2;
    if (pos < 0 || col >= p.cols) return -1;
    const int id = p.table[(size_t)s * p.cols + (size_t)col];
    return id < 0 || id >= p.pages ? -1 : id;
}

// ---- shares of the attention over the cache ----
// A unit is kUnitKeys keys of one (sequence, row tile, KV head); a sequence's units are row tile by row tile, head by head, key by key.
constexpr int kUnitKeys = 128;
struct SeqUnits {
    int first, rows;          // packed rows
    int start;                // position of the first row (below zero: idle)
    int keys;                 // positions up to its last row's, no more than the table has room for
    int tiles;                // units along the keys, at least one
    long long items;          // row tiles x KV heads
};
SMEG_HD SeqUnits seq_units(const PackedSeqs& p, int s, int group, int kv_heads, int tile_rows) {
    SeqUnits u;
    u.rows = seq_rows(p, s, &u.first);
    u.start = p.starts[s];
    const long long room = (long long)p.cols << p.page_log2;
    long long keys = u.start < 0 ? 0 : (long long)u.start + u.rows;
    if (keys > room) keys = room;
    u.keys = (int)keys;
    u.tiles = keys > 0 ? (int)((keys + kUnitKeys - 1) / kUnitKeys) : 1;
    u.items = ((long long)u.rows * group + tile_rows - 1) / tile_rows * kv_heads;
    return u;
}
// Keys that the sequence's row i attends to: positions up to its own that the table has room for.
SMEG_HD int keys_of_row(const SeqUnits& u, int i) {
    const uint32_t own = (uint32_t)u.start + (uint32_t)i + 1;      // (below 2^32: a start and a row are below 2^31)
    return u.start < 0 ? 0 : (own < (uint32_t)u.keys ? (int)own : u.keys);
}
// Whether some row's own position lies behind what the table has room for.
SMEG_HD bool beyond_table(const SeqUnits& u) { return u.start >= 0 && (uint32_t)u.start + (uint32_t)u.rows > (uint32_t)u.keys; }
// x / y for x not below zero, in 32 bits where that will do (a 64-bit quotient is a hundred instructions).
SMEG_HD long long quotient(long long x, int y) { return x <= 0xffffffffll ? (long long)((uint32_t)x / (uint32_t)y) : x / y; }
// Worker w of n takes the units from share_begin(w) to share_begin(w + 1); unit u is worker share_of(u)'s.
SMEG_HD long long share_begin(long long total, int n, int w) {
    const long long q = quotient(total, n), r = total - q * n;   // the first r workers have one more
    return q * w + (w < r ? w : r);
}
SMEG_HD int share_of(long long total, int n, long long u) {
    const long long q = quotient(total, n), r = total - q * n, cut = (q + 1) * r;
    if (u < cut) return (int)(q < 0x7fffffff ? quotient(u, (int)q + 1) : u / (q + 1));
    return q ? (int)(r + (q <= 0x7fffffff ? quotient(u - cut, (int)q) : (u - cut) / q)) : n - 1;
}
// n / d for n below 2^31 by a product.
struct FastDiv {
    uint32_t mul, shift;
};
inline FastDiv fast_div(uint32_t d) {
    FastDiv f = {1, 0};
    while ((1ull << f.shift) < d) ++f.shift;
    if (d > 1) f.mul = (uint32_t)(((1ull << 32) * ((1ull << f.shift) - d)) / d + 1);
    return f;
}
SMEG_HD int div_by(int n, FastDiv f) {
#ifdef __CUDA_ARCH__
    return (int)((__umulhi((uint32_t)n, f.mul) + (uint32_t)n) >> f.shift);
#else
    return (int)(((uint32_t)(((uint64_t)(uint32_t)n * f.mul) >> 32) + (uint32_t)n) >> f.shift);
#endif
}

}  // namespace smeg
