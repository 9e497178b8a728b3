// Attention of a batch's new rows against the pages of the 8-bit key/value cache (sm_100a).
//
//   out = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale * q . k_j - max),  j up to the row's own position;  k, v = (byte - 128) * scale of the
//   page's block.  One pass over the keys with the running maximum and sum, 32-bit sums.
//
// What bounds it is the cache: 2 bytes per position, KV head and depth, each read once for all query rows of a tile (a tile: 8 or 16 rows x heads
// of a group).  The keys of all (sequence, row tile, KV head) are one line of units of 128 keys, cut into equal shares for as many CTAs as the GPU
// holds, whatever the lengths; an item that a cut goes through is joined by a second kernel from the shares' unnormalised sums (few short items: by a cluster each, in
// distributed shared memory).  Within a unit a
// warp has 32 keys and needs no other warp until its share of an item is done.
//
// Both products are mma.m16n8k16 with the cache as the 16-row operand, so that up to eight query rows cost one column tile:
//   S^T (keys x rows) = K Q^T,   O^T (depths x rows) += V^T P^T
// A byte is not converted: as the low byte of a half word it is the f16 subnormal u * 2^-24, two masks for four codes, and the 128 of its offset
// comes off through the accumulators' start values (-128 * 2^-24 * the sum of the other operand, formed by the same instruction on a constant).
// Keys and values come by tiled copies into a ring of each warp's own (32 keys a stage, the copies' swizzle, and an order of the keys that
// keeps the operand loads off each other's banks); a lane then takes 16 consecutive depths of a key as four steps of the first product, and 16
// depths of its four keys as eight row tiles of the second.  The ring runs ahead over the ends of items, so that the next item's keys are on their way
// while the warps' shares of this one meet.  A query row is scaled by a power of two into f16's range (so bf16 queries are exact too); the
// probabilities are f16 at 2^7, and a page's product is multiplied by its scale in 32 bits; the reference of a row's exponentials follows
// its maximum when that is 2^8 above it; each 32 keys' sums are folded into 32-bit registers, since the tensor core cuts its sums off.
//
// Measured: a long context streams at 6.8 TB/s beside 12 to 15 us that do not depend on its length (launches, the first bytes, the warps' meeting, the join): one token over
// 131071 positions of 8 KV heads of 128 50.7 us (5.3 TB/s), 64 sequences of 500 to 5000 positions 76.5 us (5.0 TB/s); 901 positions by clusters 6.9 us.  With several rows of
// eight query heads each it is bound by the unpacking and the exponentials (64 x 5 rows of 3000 positions, 24 / 3 heads of 64: 77 us).
#include "common.cuh"
#include "kernels.h"
#include "paged.h"
#include "tc_common.cuh"

#include <string.h>

#include <atomic>

namespace smeg {
namespace {

constexpr int kPaThreads = 128, kPaWarps = 4;
constexpr uint32_t kOffset = 0x00800080u;           // two f16 subnormals of 128 * 2^-24
constexpr float kPScale = 128.0f;
constexpr float kLazy = 8.0f;                       // a row's reference follows its maximum when that is 2^8 above it

// d = a b + c
__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1, const float (&c)[4]) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
                 : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
}
__device__ __forceinline__ uint32_t mov_trans(uint32_t x) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
    return r;
}
__device__ __forceinline__ uint32_t even_bytes(uint32_t w) { return w & 0x00ff00ffu; }
__device__ __forceinline__ uint32_t odd_bytes(uint32_t w) { return __byte_perm(w, 0, 0x4341); }
__device__ __forceinline__ uint4 lds16(uint32_t a) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ uint4 lds8(uint32_t a) {
    uint4 v = make_uint4(0, 0, 0, 0);
    asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ void tma_3d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
                 ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar)) : "memory");
}
// (x, y) += (a, b) * s in one instruction
__device__ __forceinline__ void fma2(float& x, float& y, float a, float b, float s) {
    asm("{\n\t.reg .b64 u, v, w;\n\tmov.b64 u, {%0, %1};\n\tmov.b64 v, {%2, %3};\n\tmov.b64 w, {%4, %4};\n\tfma.rn.f32x2 u, v, w, u;\n\tmov.b64 {%0, %1}, u;\n\t}"
        : "+f"(x), "+f"(y) : "f"(a), "f"(b), "f"(s));
}
__device__ __forceinline__ float ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// First sequence whose units reach beyond unit u0, and u0's place in it; `total`: of all sequences.  The block's threads together.
struct Place {
    int s;
    long long off;
};
template <int THREADS>
__device__ __forceinline__ long long block_scan(long long x, long long* warp_sums, long long* all) {   // inclusive
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    __syncthreads();                                               // (the sums of a scan before have been read)
    if (lane == 31) warp_sums[warp] = x;
    __syncthreads();
    long long before = 0, sum = 0;
#pragma unroll
    for (int w = 0; w < THREADS / 32; ++w) {
        if (w < warp) before += warp_sums[w];
        sum += warp_sums[w];
    }
    *all = sum;
    return x + before;
}
__device__ __forceinline__ long long units_of(const PagedAttendArgs& p, int s, int tile_rows) {
    if (s >= p.seqs.seqs) return 0;
    const SeqUnits u = seq_units(p.seqs, s, p.heads / p.kv_heads, p.kv_heads, tile_rows);
    return u.items * u.tiles;
}
// The total of all units, and (find) the place of unit `at(total)`; false where there is none.
template <int THREADS, class At>
__device__ __forceinline__ bool find_unit(const PagedAttendArgs& p, int tile_rows, At at, long long* total_out, Place* out) {
    __shared__ long long warp_sums[THREADS / 32], s_off;
    __shared__ int s_seq;
    const int tid = threadIdx.x, n = p.seqs.seqs;
    const bool once = n <= THREADS;
    if (tid == 0) s_seq = -1;
    long long total = 0, mine = 0, incl = 0, all = 0;
    for (int s0 = 0; s0 < n; s0 += THREADS) {
        mine = units_of(p, s0 + tid, tile_rows);
        incl = block_scan<THREADS>(mine, warp_sums, &all);
        total += all;
    }
    *total_out = total;
    const long long u = at(total);
    if (u < 0 || u >= total) return false;                         // (uniform: the whole block)
    long long base = 0;
    for (int s0 = 0; s0 < n; s0 += THREADS) {
        if (!once) {
            mine = units_of(p, s0 + tid, tile_rows);
            incl = block_scan<THREADS>(mine, warp_sums, &all);
        }
        const long long end = base + incl;
        if (u >= end - mine && u < end) {
            s_seq = s0 + tid;
            s_off = u - (end - mine);
        }
        base += all;
    }
    __syncthreads();
    out->s = s_seq;
    out->off = s_off;
    return out->s >= 0;
}

// The sequence of item `item` of all sequences': its first item and its first unit, and the total of all units.
template <int THREADS>
__device__ __forceinline__ bool find_item(const PagedAttendArgs& p, int tile_rows, int item, long long* total_out, int* seq, long long* first_item, long long* first_unit) {
    __shared__ long long warp_sums[THREADS / 32], s_item, s_unit;
    __shared__ int s_seq;
    const int tid = threadIdx.x, n = p.seqs.seqs;
    if (tid == 0) s_seq = -1;
    long long items = 0, units = 0;
    for (int s0 = 0; s0 < n; s0 += THREADS) {
        long long mine = 0, all_items, all_units, tiles = 0;
        if (s0 + tid < n) {
            const SeqUnits u = seq_units(p.seqs, s0 + tid, p.heads / p.kv_heads, p.kv_heads, tile_rows);
            mine = u.items;
            tiles = u.tiles;
        }
        const long long upto = items + block_scan<THREADS>(mine, warp_sums, &all_items);
        const long long end = units + block_scan<THREADS>(mine * tiles, warp_sums, &all_units);
        if (item >= upto - mine && item < upto) {
            s_seq = s0 + tid;
            s_item = upto - mine;
            s_unit = end - mine * tiles;
        }
        items += all_items;
        units += all_units;
    }
    __syncthreads();
    *total_out = units;
    *seq = s_seq;
    *first_item = s_item;
    *first_unit = s_unit;
    return s_seq >= 0;
}

// Unnormalised sums of a share of an item: maxima, sums of the probabilities, then rows x depths.
__host__ __device__ constexpr size_t part_floats(int tile_rows, int hd) { return (size_t)tile_rows * (hd + 2); }

template <int BF16>
__device__ __forceinline__ void store_row4(const PagedAttendArgs& p, int row, int head, int d, float4 v) {
    uint16_t* o = p.out + (size_t)row * p.out_stride + (size_t)head * p.head_dim + d;
    const uint32_t lo = pack2_t<BF16>(v.x, v.y), hi = pack2_t<BF16>(v.z, v.w);
    if (p.out_vec) {
        *reinterpret_cast<uint2*>(o) = make_uint2(lo, hi);
    } else {
        o[0] = (uint16_t)lo; o[1] = (uint16_t)(lo >> 16); o[2] = (uint16_t)hi; o[3] = (uint16_t)(hi >> 16);
    }
}

// Where a worker is: sequence, its item (row tile, KV head) and unit.
struct Walk {
    int s, tile, kvh, row_tile;
    long long left;                                  // units to go
    SeqUnits U;
};
__device__ __forceinline__ void walk_to(const PagedAttendArgs& p, Walk& w, int tile_rows) {   // the sequence's sizes; sequences without units are passed over
    while (w.s < p.seqs.seqs) {
        w.U = seq_units(p.seqs, w.s, p.heads / p.kv_heads, p.kv_heads, tile_rows);
        if (w.U.items > 0) return;
        ++w.s;
    }
    w.left = 0;
}
__device__ __forceinline__ void walk_on(const PagedAttendArgs& p, Walk& w, int units, int tile_rows) {   // units: no more than the item has left
    w.left -= units;
    w.tile += units;
    if (w.tile < w.U.tiles) return;
    w.tile = 0;
    if (++w.kvh < p.kv_heads) return;
    w.kvh = 0;
    if ((long long)++w.row_tile * p.kv_heads < w.U.items) return;
    w.row_tile = 0;
    ++w.s;
    if (w.left > 0) walk_to(p, w, tile_rows);
}

struct PagedMaps {
    CUtensorMap codes;                               // [block][position][depth], swizzled boxes of 64 or 128 depths x 16 or 32 positions
};

// CTAs of an SM and stages of a warp's ring.  HC: depths in units of 64 (1, 2 or 4); NT: tiles of eight query rows.
// (Heads of 64 have little work behind a load, so more warps serve them better than deeper rings.  us with three CTAs of four stages and as it is: 128
// sequences of 2000, 32 / 4 heads, 50.2 and 42.6; 512 rows behind 3500, 24 / 3 heads, 119.6 and 113.9; 64 x 5 rows of 3000 80.6 and 78.9.  Heads of 128 with three
// CTAs of two stages: no faster than two of three.)
__host__ __device__ constexpr int ctas_of(int hc, int nt) { return hc == 4 ? 1 : (hc == 2 ? 2 : (nt == 1 ? 5 : 4)); }
__host__ __device__ constexpr int stages_of(int hc) { return hc == 1 ? 2 : 3; }

__device__ __forceinline__ float ld_dsmem(uint32_t cluster_addr) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(cluster_addr) : "memory");
    return v;
}
__device__ __forceinline__ float4 ld_dsmem4(uint32_t cluster_addr) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(cluster_addr) : "memory");
    return v;
}

template <int N>
struct Int {
    static constexpr int value = N;
};
// P16: pages of 16 positions, two of which make a piece; else a piece lies in one.  CL: the CTAs of a cluster (2^cluster_log2 of them) share one item's units and meet in distributed shared memory, without a second kernel: for few items of few units.
template <int BF16, int HC, int NT, int CL, int P16>
__global__ void __launch_bounds__(kPaThreads, ctas_of(HC, NT)) paged_attend_kernel(const __grid_constant__ PagedMaps maps, const __grid_constant__ PagedAttendArgs p) {
    constexpr int MT = 4 * HC;                       // tiles of 16 depths
    constexpr int NR = 8 * NT;
    constexpr int kStages = stages_of(HC);
    constexpr int kPitch = HC == 1 ? 64 : 128, kPanel = 32 * kPitch, kPanels = HC == 4 ? 2 : 1;   // bytes of a key, of 32 keys; panels of 128 depths
    constexpr int kHalf = kPanels * kPanel, kStage = 2 * kHalf;                                   // keys, then values
    extern __shared__ unsigned char smem_dyn[];
    unsigned char* smem = smem_dyn + ((1024u - (smem_u32(smem_dyn) & 1023u)) & 1023u);
    __shared__ __align__(8) uint64_t full[kPaWarps][kStages];
    __shared__ int s_block[kPaWarps][kStages][2];    // of each group of 16 keys, below zero: none
    __shared__ float s_m[kPaWarps][NR], s_l[kPaWarps][NR];
    __shared__ int abort_word;
    volatile int* abort_flag = &abort_word;
    const int tid = threadIdx.x, warp = warp_index(), lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int hd = p.head_dim, group = p.heads / p.kv_heads, page = P16 ? 16 : 1 << p.seqs.page_log2;
    if (tid == 0) {
        abort_word = 0;
        for (int w = 0; w < kPaWarps; ++w)
            for (int i = 0; i < kStages; ++i) mbar_init(&full[w][i], 1);
        fence_barrier_init();
    }
    pdl_wait();
    pdl_launch_dependents();                         // (behind the wait: what ran before this kernel is there for the next one's index work, too)
    long long total;
    Walk now;
    if (CL) {
        const int item = blockIdx.x >> p.cluster_log2, rank = blockIdx.x & ((1 << p.cluster_log2) - 1);
        long long first_item, first_unit;
        if (!find_item<kPaThreads>(p, NR, item, &total, &now.s, &first_item, &first_unit)) return;   // (the whole cluster)
        walk_to(p, now, NR);
        const long long mine = item - first_item;
        now.row_tile = (int)quotient(mine, p.kv_heads);
        now.kvh = (int)(mine - (long long)now.row_tile * p.kv_heads);
        now.tile = (int)((long long)now.U.tiles * rank >> p.cluster_log2);
        now.left = ((long long)now.U.tiles * (rank + 1) >> p.cluster_log2) - now.tile;
    } else {
        Place at;
        if (!find_unit<kPaThreads>(p, NR, [&](long long n) { return share_begin(n, gridDim.x, blockIdx.x); }, &total, &at)) return;   // (with barriers: the mbarriers are set up)
        now.s = at.s;
        now.left = share_begin(total, gridDim.x, blockIdx.x + 1) - share_begin(total, gridDim.x, blockIdx.x);
        walk_to(p, now, NR);
        const long long item = quotient(at.off, now.U.tiles);
        now.tile = (int)(at.off - item * now.U.tiles);
        now.row_tile = (int)quotient(item, p.kv_heads);
        now.kvh = (int)(item - (long long)now.row_tile * p.kv_heads);
    }
    const Walk whose = now;
    __shared__ float part_m[NR], part_l[NR];         // CL: this CTA's share of the item (part_l below zero: it had none), its sums behind the ring
    float* part_o = reinterpret_cast<float*>(smem + kPaWarps * kStages * kStage);
    if (CL && now.left == 0 && tid < NR) { part_m[tid] = -INFINITY; part_l[tid] = -1.0f; }
    // ---- this warp's ring ----
    Walk ahead = now;
    const uint32_t ring = smem_u32(smem) + warp * kStages * kStage;
    int put = 0, issued = 0;
    auto issue = [&]() {                             // the next piece (32 keys) that this warp has
        while (ahead.left > 0) {
            const int key0 = ahead.tile * kUnitKeys + 32 * warp;
            const bool has = key0 < ahead.U.keys;
            if (has) {
                // (positions below U.keys are within the table)
                const int* row = p.seqs.table + (size_t)ahead.s * p.seqs.cols + (key0 >> p.seqs.page_log2);
                int id[2];
                id[0] = (unsigned)row[0] < (unsigned)p.seqs.pages ? row[0] : -1;
                id[1] = key0 + 16 >= ahead.U.keys ? -2 : id[0];
                if (P16 && id[1] != -2) id[1] = (unsigned)row[1] < (unsigned)p.seqs.pages ? row[1] : -1;
                if (lane == 0) {
                    if ((id[0] == -1 || id[1] == -1) && p.status) atomicOr(p.status, STATUS_PAGE);
                    const int z0 = 2 * (id[0] * p.kv_heads + ahead.kvh), z1 = 2 * (id[1] * p.kv_heads + ahead.kvh);
                    s_block[warp][put][0] = id[0] < 0 ? -1 : z0;
                    s_block[warp][put][1] = id[1] < 0 ? -1 : z1;
                    const uint32_t dst = ring + put * kStage;
                    uint64_t* bar = &full[warp][put];
                    const int y = key0 & (page - 1);
                    if (!P16) {
                        mbar_expect_tx(bar, id[0] < 0 ? 0 : kStage);
                        if (id[0] >= 0)
#pragma unroll
                            for (int c = 0; c < kPanels; ++c) {
                                tma_3d(dst + c * kPanel, &maps.codes, 128 * c, y, z0, bar);
                                tma_3d(dst + kHalf + c * kPanel, &maps.codes, 128 * c, y, z0 + 1, bar);
                            }
                    } else {
                        mbar_expect_tx(bar, ((id[0] >= 0) + (id[1] >= 0)) * (kStage / 2));
#pragma unroll
                        for (int b = 0; b < 2; ++b)
                            if (id[b] >= 0)
#pragma unroll
                                for (int c = 0; c < kPanels; ++c) {
                                    tma_3d(dst + c * kPanel + b * 16 * kPitch, &maps.codes, 128 * c, 0, b ? z1 : z0, bar);
                                    tma_3d(dst + kHalf + c * kPanel + b * 16 * kPitch, &maps.codes, 128 * c, 0, (b ? z1 : z0) + 1, bar);
                                }
                    }
                }
                __syncwarp();
                ++issued;
                if (++put == kStages) put = 0;
            }
            walk_on(p, ahead, 1, NR);
            if (has) return;
        }
    };
#pragma unroll
    for (int i = 0; i < kStages; ++i) issue();

    // Key order: row g of a group's A operand is key pi(g), so that the lanes of a quarter warp meet different banks in both products
    const int pi_g = g & 1 ? g ^ 4 : g, pi_t = (2 * t + 1) ^ 4;
    const uint32_t k_at = HC == 1 ? pi_g * 64 + ((t ^ ((pi_g >> 1) & 3)) << 4) : pi_g * 128 + ((t ^ pi_g) << 4);
    const uint32_t v_even = HC == 1 ? 2 * t * 64 + (((g >> 1) ^ t) << 4) + 8 * (g & 1) : 2 * t * 128 + ((g ^ (2 * t)) << 4);
    const uint32_t v_odd = HC == 1 ? pi_t * 64 + (((g >> 1) ^ ((pi_t >> 1) & 3)) << 4) + 8 * (g & 1) : pi_t * 128 + ((g ^ pi_t) << 4);
    const float zero4[4] = {0.f, 0.f, 0.f, 0.f};
    int get = 0, parity = 0, taken = 0;
    bool first_piece = true, ok = true;
    float sk_n[2] = {0.f, 0.f}, sv_n[2] = {0.f, 0.f};
    auto fetch_scales = [&](int stage) {             // of the piece in `stage`, whose pages are known since it was issued
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            const int z = s_block[warp][stage][b];
            const float2 x = z >= 0 ? *reinterpret_cast<const float2*>(p.scales + z) : make_float2(0.f, 0.f);
            sk_n[b] = x.x;
            sv_n[b] = x.y;
        }
    };
    if (issued > 0) fetch_scales(0);

    while (now.left > 0) {
        const SeqUnits U = now.U;
        const int kvh = now.kvh, tile0 = now.tile, tile1 = (int)min((long long)U.tiles, tile0 + now.left);
        const int n0 = now.row_tile * NR, nrow = (int)min((long long)NR, (long long)U.rows * group - n0);   // packed rows x heads of the tile

        if (tid == 0 && p.status && beyond_table(U)) atomicOr(p.status, STATUS_PAGE);

        // ---- queries: B fragments, a power of two to each row ----
        uint32_t qf[NT][4 * HC][2];
        float row_scale[NT][2], start0[NT][4];
        int limit[NT][2];                            // keys that rows 2 t and 2 t + 1 of a tile attend to
        const int low = keys_of_row(U, div_by(n0, p.by_group));                                   // keys that every row of the tile attends to
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            const int n = n0 + 8 * j + g, i = div_by(n, p.by_group), head = kvh * group + (n - i * group);
            const bool in = 8 * j + g < nrow;
            const uint16_t* q = p.q + (size_t)(U.first + i) * p.q_stride + (size_t)head * hd;
            float x[HC][16];
            float mx = 0.0f;
#pragma unroll
            for (int c = 0; c < HC; ++c) {
                const int d = 16 * (t + 4 * c);
#pragma unroll
                for (int e = 0; e < 16; ++e) x[c][e] = 0.0f;
                if (in && d < hd) {
                    if (p.q_vec) {
                        const uint4 u0 = *reinterpret_cast<const uint4*>(q + d), u1 = *reinterpret_cast<const uint4*>(q + d + 8);
                        const uint32_t w[8] = {u0.x, u0.y, u0.z, u0.w, u1.x, u1.y, u1.z, u1.w};
#pragma unroll
                        for (int e = 0; e < 16; ++e) x[c][e] = t_to_f32<BF16>((uint16_t)(w[e / 2] >> (16 * (e & 1))));
                    } else {
#pragma unroll
                        for (int e = 0; e < 16; ++e) x[c][e] = t_to_f32<BF16>(q[d + e]);
                    }
                }
#pragma unroll
                for (int e = 0; e < 16; ++e) mx = fmaxf(mx, fabsf(x[c][e]));
            }
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
            // largest magnitude to 2^14 .. 2^15: exact but for depths 2^-28 below it (f16's own range needs no more than that)
            const int ex = (int)(__float_as_uint(mx) >> 23) - 127;
            const int up = mx > 0.0f && ex < 128 && ex > -110 ? 14 - ex : 0;
            const float f = __uint_as_float((uint32_t)(127 + up) << 23);
            // (from 2^100 on the scores come out 2^(ex - 99) too small, which leaves a softmax of such scores as it is: their products with 2^24 stay numbers)
            const float back = __uint_as_float((uint32_t)(127 - max(up, 14 - 99)) << 23) * (p.scale_log2e * 16777216.0f);
#pragma unroll
            for (int c = 0; c < HC; ++c)
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    qf[j][4 * c + w][0] = pack2_t<0>(x[c][4 * w] * f, x[c][4 * w + 2] * f);
                    qf[j][4 * c + w][1] = pack2_t<0>(x[c][4 * w + 1] * f, x[c][4 * w + 3] * f);
                }
            float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int k = 0; k < 4 * HC; ++k) mma_f16(sum, kOffset, kOffset, kOffset, kOffset, qf[j][k][0], qf[j][k][1], sum);
#pragma unroll
            for (int e = 0; e < 4; ++e) start0[j][e] = -sum[e & 1];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                row_scale[j][e] = __shfl_sync(0xffffffffu, back, 4 * (2 * t + e));
                const int m = n0 + 8 * j + 2 * t + e;
                limit[j][e] = 8 * j + 2 * t + e < nrow ? keys_of_row(U, div_by(m, p.by_group)) : 0;
            }
        }

        // ---- this warp's pieces of the units ----
        float o[NT][MT][4], m_run[NT][2], l_run[NT][2];
#pragma unroll
        for (int j = 0; j < NT; ++j) {
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[j][m][e] = 0.0f;
#pragma unroll
            for (int e = 0; e < 2; ++e) { m_run[j][e] = -INFINITY; l_run[j][e] = 0.0f; }
        }
        const int end = min(tile1 * kUnitKeys, U.keys);
        int last = -1;                                                 // the stage consumed last
        for (int key0 = tile0 * kUnitKeys + 32 * warp; key0 < end; key0 += kUnitKeys) {
            if (last >= 0) issue();                                    // (into the stage that the piece before has left)
            const float sk[2] = {sk_n[0], sk_n[1]}, sv[2] = {sv_n[0], sv_n[1]};
            const bool here0 = s_block[warp][get][0] >= 0, here1 = s_block[warp][get][1] >= 0;
            ++taken;
            if (taken < issued) fetch_scales(get + 1 == kStages ? 0 : get + 1);
            ok = ok && __all_sync(0xffffffffu, mbar_wait(&full[warp][get], parity, abort_flag, p.status));
            const uint32_t stage = ring + get * kStage;
            // scores
            float sc[NT][2][4];
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int c = 0; c < HC; ++c) {
                    const uint32_t a = stage + (c >> 1) * kPanel + b * 16 * kPitch + (k_at ^ (64 * (c & 1)));
                    const uint4 x = lds16(a), y = lds16(a + 8 * kPitch);
                    const uint32_t lo[4] = {x.x, x.y, x.z, x.w}, hi[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
                    for (int w = 0; w < 4; ++w) {
                        const uint32_t a0 = even_bytes(lo[w]), a1 = even_bytes(hi[w]), a2 = odd_bytes(lo[w]), a3 = odd_bytes(hi[w]);
#pragma unroll
                        for (int j = 0; j < NT; ++j)
                            mma_f16(sc[j][b], a0, a1, a2, a3, qf[j][4 * c + w][0], qf[j][4 * c + w][1], c + w == 0 ? start0[j] : sc[j][b]);
                    }
                }
            // Probabilities at 2^7, NaN under a scale that is NaN: it stays with the rows that attend to it.  Two pages of 16 have a product each, with their own scale.  (With a common factor for
            // both, the smaller scale's probabilities have few bits or none left in f16 where the scales are far apart, whatever the weight of the larger one's keys is for a row: none, where
            // the row does not attend to them.)
            float one[2];
#pragma unroll
            for (int b = 0; b < 2; ++b) one[b] = fmaf(sv[P16 ? b : 0], 0.0f, kPScale);
            const bool whole = key0 + 32 <= low && here0 && here1;
            uint32_t pf[NT][2][2];
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                float f[2][2];
#pragma unroll
                for (int b = 0; b < 2; ++b)
#pragma unroll
                    for (int e = 0; e < 2; ++e) f[b][e] = row_scale[j][e] * sk[b];
                float mx[2] = {-INFINITY, -INFINITY};
                unsigned on = 0xffu;                                   // bit 4 b + e: element e of group b counts
                if (!whole) {
#pragma unroll
                    for (int b = 0; b < 2; ++b)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const int key = key0 + 16 * b + pi_g + 8 * (e >> 1);
                            if (!((b ? here1 : here0) && key < limit[j][e & 1])) on &= ~(1u << (4 * b + e));
                        }
                }
#pragma unroll
                for (int b = 0; b < 2; ++b)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        sc[j][b][e] *= f[b][e & 1];
                        if (!whole && !(on >> (4 * b + e) & 1)) sc[j][b][e] = -INFINITY;
                        mx[e & 1] = fmaxf(mx[e & 1], sc[j][b][e]);
                    }
                bool far = false;
#pragma unroll
                for (int e = 0; e < 2; ++e) {
#pragma unroll
                    for (int w = 4; w < 32; w <<= 1) mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], w));
                    far = far || mx[e] > m_run[j][e] + kLazy;          // (from -inf: whatever there is)
                }
                if (__any_sync(0xffffffffu, far)) {
                    float alpha[2];
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const float to = fmaxf(m_run[j][e], mx[e]);
                        alpha[e] = ex2(m_run[j][e] - (to == -INFINITY ? 0.0f : to));
                        m_run[j][e] = to;
                        l_run[j][e] *= alpha[e];
                    }
#pragma unroll
                    for (int m = 0; m < MT; ++m)
#pragma unroll
                        for (int e = 0; e < 4; ++e) o[j][m][e] *= alpha[e & 1];
                }
                const float ref[2] = {m_run[j][0] == -INFINITY ? 0.0f : m_run[j][0], m_run[j][1] == -INFINITY ? 0.0f : m_run[j][1]};
#pragma unroll
                for (int b = 0; b < 2; ++b) {
                    float w[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float x = ex2(sc[j][b][e] - ref[e & 1]);
                        l_run[j][e & 1] += x;
                        w[e] = x * one[b];
                        if (!whole && !(on >> (4 * b + e) & 1)) w[e] = 0.0f;          // (not 0 * the NaN of a page that the row does not attend to)
                    }
                    pf[j][b][0] = mov_trans(pack2_t<0>(w[0], w[1]));
                    pf[j][b][1] = mov_trans(pack2_t<0>(w[2], w[3]));
                }
            }
            // values: += the products of groups FIRST .. FIRST + COUNT times their scale
            auto add_values = [&](auto from, auto count, float scale) {
                constexpr int FIRST = decltype(from)::value, LAST = FIRST + decltype(count)::value - 1;
                float off0[NT][4];
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                    mma_f16(off0[j], kOffset, kOffset, kOffset, kOffset, pf[j][FIRST][0], pf[j][FIRST][1], zero4);
                    if (LAST > FIRST) mma_f16(off0[j], kOffset, kOffset, kOffset, kOffset, pf[j][LAST][0], pf[j][LAST][1], off0[j]);
#pragma unroll
                    for (int e = 0; e < 4; ++e) off0[j][e] = -off0[j][e];
                }
#pragma unroll
                for (int c = 0; c < (HC == 4 ? 2 : 1); ++c) {
                    uint32_t vw[2][4][4];                              // group, key, word
#pragma unroll
                    for (int b = FIRST; b <= LAST; ++b)
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            const uint32_t a = stage + kHalf + c * kPanel + (16 * b + 8 * (r >> 1)) * kPitch + (r & 1 ? v_odd : v_even);
                            const uint4 v = HC == 1 ? lds8(a) : lds16(a);
                            vw[b][r][0] = v.x; vw[b][r][1] = v.y; vw[b][r][2] = v.z; vw[b][r][3] = v.w;
                        }
#pragma unroll
                    for (int w = 0; w < (HC == 1 ? 2 : 4); ++w)
#pragma unroll
                        for (int h = 0; h < 2; ++h) {                  // depths 4 w + 2 h and the next: row tile m
                            const int m = 8 * c + 2 * w + h;
                            float acc[NT][4];
#pragma unroll
                            for (int b = FIRST; b <= LAST; ++b) {
                                const uint32_t x = __byte_perm(vw[b][0][w], vw[b][1][w], h ? 0x7632 : 0x5410), y = __byte_perm(vw[b][2][w], vw[b][3][w], h ? 0x7632 : 0x5410);
                                const uint32_t a0 = even_bytes(x), a1 = odd_bytes(x), a2 = even_bytes(y), a3 = odd_bytes(y);
#pragma unroll
                                for (int j = 0; j < NT; ++j) mma_f16(acc[j], a0, a1, a2, a3, pf[j][b][0], pf[j][b][1], b > FIRST ? acc[j] : off0[j]);
                            }
#pragma unroll
                            for (int j = 0; j < NT; ++j) {
                                fma2(o[j][m][0], o[j][m][1], acc[j][0], acc[j][1], scale);
                                fma2(o[j][m][2], o[j][m][3], acc[j][2], acc[j][3], scale);
                            }
                        }
                }
            };
            if (P16) {
                add_values(Int<0>(), Int<1>(), fmaxf(sv[0], 0.0f));    // (fmaxf drops a NaN)
                add_values(Int<1>(), Int<1>(), fmaxf(sv[1], 0.0f));
            } else {
                add_values(Int<0>(), Int<2>(), fmaxf(sv[0], 0.0f));
            }
            last = get;
            if (++get == kStages) { get = 0; parity ^= 1; }
            __syncwarp();                                              // (every lane has read the stage)
        }

        // ---- the warps' shares meet in the stages they have left, then the item's ----
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                float l = l_run[j][e];
#pragma unroll
                for (int w = 4; w < 32; w <<= 1) l += __shfl_xor_sync(0xffffffffu, l, w);
                if (g == 0) {
                    s_m[warp][8 * j + 2 * t + e] = m_run[j][e];
                    s_l[warp][8 * j + 2 * t + e] = last < 0 ? -1.0f : l;               // below zero: this warp had no keys
                }
            }
        // (rows one after the other where stages are as large as NR x 64 HC numbers: kStage = 4096 HC = 16 * 64 HC * 4)
        static_assert(kStage >= NR * 64 * HC * 4, "a stage holds a warp's share");
        __shared__ int s_last[kPaWarps];
        if (lane == 0) s_last[warp] = last;
        if (last >= 0) {
            float* mine = reinterpret_cast<float*>(smem + (size_t)(warp * kStages + last) * kStage);
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int m = 0; m < MT; ++m)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        // row tile m's rows g and g + 8 are depths 2 m and 2 m + 1 of the lane's run
                        const int d = HC == 1 ? 8 * g + 2 * m + (e >> 1) : 16 * g + 128 * (m / 8) + 2 * (m % 8) + (e >> 1);
                        mine[(8 * j + 2 * t + (e & 1)) * 64 * HC + d] = o[j][m][e];
                    }
        }
        __syncthreads();
        const bool all_of_it = tile0 == 0 && tile1 == U.tiles;
        float* ws = p.ws + (2 * (size_t)blockIdx.x + (first_piece ? 0 : 1)) * part_floats(NR, hd);
        first_piece = false;
        for (int it = tid; it < nrow * (hd / 4); it += kPaThreads) {
            const int n = div_by(it, p.by_quads), d = (it - n * (hd / 4)) * 4;
            float mx = -INFINITY;
#pragma unroll
            for (int w = 0; w < kPaWarps; ++w) mx = fmaxf(mx, s_m[w][n]);
            const float ref = mx == -INFINITY ? 0.0f : mx;
            float l = 0.0f;
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < kPaWarps; ++w) {
                if (s_l[w][n] < 0.0f) continue;
                const float f = ex2(s_m[w][n] - ref);
                const float4 x = *reinterpret_cast<const float4*>(smem + (size_t)(w * kStages + s_last[w]) * kStage + (n * 64 * HC + d) * 4);
                l = fmaf(f, s_l[w][n], l);
                v.x = fmaf(f, x.x, v.x); v.y = fmaf(f, x.y, v.y); v.z = fmaf(f, x.z, v.z); v.w = fmaf(f, x.w, v.w);
            }
            if (CL) {
                if (d == 0) { part_m[n] = mx; part_l[n] = l; }
                *reinterpret_cast<float4*>(part_o + n * 64 * HC + d) = v;
            } else if (all_of_it) {
                const float r = l == 0.0f ? 0.0f : __fdiv_rn(16777216.0f / kPScale, l);   // (a row that attends to nothing is zero)
                const int i = div_by(n0 + n, p.by_group), head = kvh * group + (n0 + n) - i * group;
                store_row4<BF16>(p, U.first + i, head, d, make_float4(v.x * r, v.y * r, v.z * r, v.w * r));
            } else {
                if (d == 0) { ws[n] = mx; ws[NR + n] = l; }
                *reinterpret_cast<float4*>(ws + 2 * NR + n * hd + d) = v;
            }
        }
        walk_on(p, now, tile1 - tile0, NR);
        if (now.left > 0) {
            fence_proxy_async();                                       // (the shares' place is the ring's again)
            __syncthreads();
            if (last >= 0) issue();
        }
    }
    if (CL) {
        cluster_sync_all();
        const int ranks = 1 << p.cluster_log2, rank = blockIdx.x & (ranks - 1), n0 = whose.row_tile * NR;
        const int nrow = (int)min((long long)NR, (long long)whose.U.rows * group - n0);
        const uint32_t m_a = smem_u32(part_m), l_a = smem_u32(part_l), o_a = smem_u32(part_o);
        for (int it = rank * kPaThreads + tid; it < nrow * (hd / 4); it += ranks * kPaThreads) {
            const int n = div_by(it, p.by_quads), d = (it - n * (hd / 4)) * 4;
            float m[8], s[8], mx = -INFINITY, l = 0.0f;
            float4 x[8], v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int from = min(e, ranks - 1);
                m[e] = ld_dsmem(mapa_shared(m_a + n * 4, from));
                s[e] = ld_dsmem(mapa_shared(l_a + n * 4, from));
                x[e] = ld_dsmem4(mapa_shared(o_a + (n * 64 * HC + d) * 4, from));
            }
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (e < ranks) mx = fmaxf(mx, m[e]);
            const float ref = mx == -INFINITY ? 0.0f : mx;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                if (e >= ranks || s[e] < 0.0f) continue;           // (a NaN of a share is no number below zero)
                const float f = ex2(m[e] - ref);
                l = fmaf(f, s[e], l);
                v.x = fmaf(f, x[e].x, v.x); v.y = fmaf(f, x[e].y, v.y); v.z = fmaf(f, x[e].z, v.z); v.w = fmaf(f, x[e].w, v.w);
            }
            const float r = l == 0.0f ? 0.0f : __fdiv_rn(16777216.0f / kPScale, l);
            const int i = div_by(n0 + n, p.by_group), head = whose.kvh * group + (n0 + n) - i * group;
            store_row4<BF16>(p, whose.U.first + i, head, d, make_float4(v.x * r, v.y * r, v.z * r, v.w * r));
        }
        cluster_sync_all();                                        // (nobody leaves while its shared memory is read)
    }
}

// The items that were cut are joined by a kernel of their own, whose search for them runs while the shares are still being made.
// (A grid whose CTAs all left without waiting could end before the grid that it depends on, and the next one would not wait for that.)
__device__ __forceinline__ void leave() {
    if (blockIdx.x == 0) pdl_wait();
}
// Many items of few shares: CTA b has the item that the cut before worker b + 1 goes through, if that is the first one through it.  A cut item is the last of its first worker's
// and the first of the others'.
template <int BF16>
__global__ void __launch_bounds__(kPaThreads) paged_join_cuts_kernel(const __grid_constant__ PagedAttendArgs p, int workers, int tile_rows) {
    const int tid = threadIdx.x, hd = p.head_dim, group = p.heads / p.kv_heads;
    // (the batch is there: paged_attend_kernel lets this grid go behind its own wait)
    const int cut = blockIdx.x + 1;
    long long total;
    Place at;
    if (!find_unit<kPaThreads>(p, tile_rows, [&](long long n) { return share_begin(n, workers, cut); }, &total, &at)) return leave();
    const SeqUnits U = seq_units(p.seqs, at.s, group, p.kv_heads, tile_rows);
    const long long item = quotient(at.off, U.tiles), u = share_begin(total, workers, cut);
    const long long begin = u - (at.off - item * U.tiles), end = begin + U.tiles;
    if (begin == u) return leave();                                            // the cut is between two items
    const int w0 = share_of(total, workers, begin), w1 = share_of(total, workers, end - 1);
    if (w0 != cut - 1) return leave();
    const int row_tile = (int)quotient(item, p.kv_heads), kvh = (int)(item - (long long)row_tile * p.kv_heads), n0 = row_tile * tile_rows;
    const int nrow = (int)min((long long)tile_rows, (long long)U.rows * group - n0);
    pdl_wait();
    pdl_launch_dependents();
    const size_t pf = part_floats(tile_rows, hd);
    const size_t slot0 = 2 * (size_t)w0 + (begin > share_begin(total, workers, w0) ? 1 : 0);
    for (int it = tid; it < nrow * (hd / 4); it += kPaThreads) {
        const int n = div_by(it, p.by_quads), d = (it - n * (hd / 4)) * 4;
        float mx = -INFINITY, l = 0.0f;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int w = w0; w <= w1; w += 4) {                            // four shares' loads at a time
            float m[4], s[4];
            float4 x[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float* ws = p.ws + (w + e == w0 ? slot0 : 2 * (size_t)min(w + e, w1)) * pf;
                m[e] = w + e <= w1 ? ws[n] : -INFINITY;
                s[e] = ws[tile_rows + n];
                x[e] = *reinterpret_cast<const float4*>(ws + 2 * tile_rows + n * hd + d);
            }
            float now = mx;
#pragma unroll
            for (int e = 0; e < 4; ++e) now = fmaxf(now, m[e]);
            const float ref = now == -INFINITY ? 0.0f : now, f0 = ex2(mx - ref);
            l *= f0;
            v.x *= f0; v.y *= f0; v.z *= f0; v.w *= f0;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (w + e > w1) break;
                const float f = ex2(m[e] - ref);
                l = fmaf(f, s[e], l);
                v.x = fmaf(f, x[e].x, v.x); v.y = fmaf(f, x[e].y, v.y); v.z = fmaf(f, x[e].z, v.z); v.w = fmaf(f, x[e].w, v.w);
            }
            mx = now;
        }
        const float r = l == 0.0f ? 0.0f : __fdiv_rn(16777216.0f / kPScale, l);
        const int i = div_by(n0 + n, p.by_group), head = kvh * group + (n0 + n) - i * group;
        store_row4<BF16>(p, U.first + i, head, d, make_float4(v.x * r, v.y * r, v.z * r, v.w * r));
    }
}

// Fewer items than workers, so that an item has many shares: CTAs (b, y) take `par` rows at a time of item b.  A thread takes four depths of a row and every
// so many shares; the threads of the same depths meet in shared memory.  (131071 keys of one sequence in 37 shares an item, us in all: by cuts 61, so 51.
// 64 sequences of 2900 in two or three shares: by cuts 71.5, with this kernel's inner part by cuts 75.)
constexpr int kPjThreads = 256;
template <int BF16>
__global__ void __launch_bounds__(kPjThreads) paged_join_items_kernel(const __grid_constant__ PagedAttendArgs p, int workers, int tile_rows, int par) {
    __shared__ float4 s_v[kPjThreads];
    __shared__ float s_m[kPjThreads / 4], s_l[kPjThreads / 4];
    const int tid = threadIdx.x, hd = p.head_dim, group = p.heads / p.kv_heads;
    // (the batch is there: paged_attend_kernel lets this grid go behind its own wait)
    long long total, first_item, begin;
    int s;
    if (!find_item<kPjThreads>(p, tile_rows, blockIdx.x, &total, &s, &first_item, &begin)) return leave();
    const long long item = blockIdx.x - first_item;
    const SeqUnits U = seq_units(p.seqs, s, group, p.kv_heads, tile_rows);
    begin += item * U.tiles;
    const int w0 = share_of(total, workers, begin), w1 = share_of(total, workers, begin + U.tiles - 1);
    if (w0 == w1) return leave();                                                          // (not cut)
    const int row_tile = (int)quotient(item, p.kv_heads), kvh = (int)(item - (long long)row_tile * p.kv_heads), n0 = row_tile * tile_rows;
    const int nrow = (int)min((long long)tile_rows, (long long)U.rows * group - n0);
    const size_t pf = part_floats(tile_rows, hd);
    const size_t slot0 = 2 * (size_t)w0 + (begin > share_begin(total, workers, w0) ? 1 : 0);
    const int quads = hd / 4, lane = div_by(tid, p.by_quads), d = (tid - lane * quads) * 4;
    const int lanes = div_by(div_by(kPjThreads, p.by_quads), p.by_par), pg = div_by(lane, p.by_par), r = lane - pg * par;    // share, row of this thread
    pdl_wait();
    pdl_launch_dependents();                         // (not before: the next kernel's CTAs would take the room that this grid's wait for)
    for (int nb = blockIdx.y * par; nb < nrow; nb += gridDim.y * par) {
        const int n = nb + r;
        const bool in = pg < lanes && n < nrow;
        float mx = -INFINITY, l = 0.0f;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        if (in)
            for (int w = w0 + pg; w <= w1; w += 4 * lanes) {           // four shares' loads at a time
                float m[4], q[4];
                float4 x[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int k = w + e * lanes;
                    const float* ws = p.ws + (k == w0 ? slot0 : 2 * (size_t)min(k, w1)) * pf;
                    m[e] = k <= w1 ? ws[n] : -INFINITY;
                    q[e] = k <= w1 ? ws[tile_rows + n] : 0.0f;
                    x[e] = k <= w1 ? *reinterpret_cast<const float4*>(ws + 2 * tile_rows + n * hd + d) : make_float4(0.f, 0.f, 0.f, 0.f);
                }
                const float now = fmaxf(fmaxf(fmaxf(mx, m[0]), fmaxf(m[1], m[2])), m[3]);
                const float ref = now == -INFINITY ? 0.0f : now, f0 = ex2(mx - ref);
                l *= f0;
                v.x *= f0; v.y *= f0; v.z *= f0; v.w *= f0;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float f = ex2(m[e] - ref);
                    l = fmaf(f, q[e], l);
                    v.x = fmaf(f, x[e].x, v.x); v.y = fmaf(f, x[e].y, v.y); v.z = fmaf(f, x[e].z, v.z); v.w = fmaf(f, x[e].w, v.w);
                }
                mx = now;
            }
        s_v[tid] = v;
        if (d == 0 && in) { s_m[lane] = mx; s_l[lane] = l; }
        __syncthreads();
        if (pg == 0 && in) {
            float top = -INFINITY;
            for (int e = 0; e < lanes; ++e) top = fmaxf(top, s_m[e * par + r]);
            const float ref = top == -INFINITY ? 0.0f : top;
            l = 0.0f;
            v = make_float4(0.f, 0.f, 0.f, 0.f);
            for (int e = 0; e < lanes; ++e) {
                const float f = ex2(s_m[e * par + r] - ref);
                const float4 x = s_v[e * par * quads + tid];
                l = fmaf(f, s_l[e * par + r], l);
                v.x = fmaf(f, x.x, v.x); v.y = fmaf(f, x.y, v.y); v.z = fmaf(f, x.z, v.z); v.w = fmaf(f, x.w, v.w);
            }
            const float scale = l == 0.0f ? 0.0f : __fdiv_rn(16777216.0f / kPScale, l);
            const int i = div_by(n0 + n, p.by_group), head = kvh * group + (n0 + n) - i * group;
            store_row4<BF16>(p, U.first + i, head, d, make_float4(v.x * scale, v.y * scale, v.z * scale, v.w * scale));
        }
        __syncthreads();
    }
}

// Query rows of a tile: 16 share the unpacking of the codes, and 8 leave fewer rows empty.  A tile of 8 costs three fifths of one of 16 (512 rows behind 3500, heads of 64, us:
// 16 119, 8 139; of 128: 73 and 90), so 8 win for up to 8, 17 to 24 and 33 to 40 rows of a sequence and KV head (12 x 5 rows x 8 heads of 64: 20.6 and 19.4).
int tile_rows_of(int group, int max_rows) {
    const long long n = (long long)group * max_rows, by8 = (n + 7) / 8, by16 = (n + 15) / 16;
    return 3 * by8 <= 5 * by16 ? 8 : 16;
}

long long items_bound(const PagedAttendArgs& a, int tile_rows) {
    return ((long long)a.seqs.rows * (a.heads / a.kv_heads) / tile_rows + a.seqs.seqs) * a.kv_heads;
}
// The same, tight for sequences of a row each: r rows have ceil(r * group / tile_rows) tiles and never more than r * ceil(group / tile_rows).  (Which join is taken was measured
// over the looser one.)
long long items_most(const PagedAttendArgs& a, int tile_rows) {
    const long long by_row = (long long)(a.heads / a.kv_heads + tile_rows - 1) / tile_rows * a.seqs.rows * a.kv_heads, bound = items_bound(a, tile_rows);
    return by_row < bound ? by_row : bound;
}

// CTAs: as many as the GPU holds at a time (the occupancy of the variant), no more than there can be units.
int workers_of(const PagedAttendArgs& a, int tile_rows, int sm_count) {
    const int hc = a.head_dim <= 64 ? 1 : (a.head_dim <= 128 ? 2 : 4);
    const int per_sm = ctas_of(hc, tile_rows / 8);
    const long long room = ((long long)a.seqs.cols << a.seqs.page_log2), tiles = (room + kUnitKeys - 1) / kUnitKeys;
    const long long items = items_bound(a, tile_rows);
    const long long most = (long long)sm_count * per_sm, units = items * (tiles > 0 ? tiles : 1);
    return (int)(units < most ? (units > 0 ? units : 1) : most);
}

// CTAs of an item (log2) where a cluster each takes the place of shares and join; 0: it does not.  It does where all clusters are on the machine at a time and no CTA has
// more than three units, which is little beside the join whatever the lengths are, nor more than one above its equal share.  (us by shares and by clusters, heads of 128: 901
// positions of 8 KV heads 7.6 and 6.9, four sequences of 1800 12.1 and 9.3, sixteen of 500 12.3 and 9.7, 2500 positions of 32 KV heads 12.6 and 10.0; two above: 3000 positions
// of 8 KV heads 8.7 and 9.3; seven units: 12 x 5 rows of 800 to 3200 positions, heads of 64, 18.7 and 22.4.)
int cluster_of(const PagedAttendArgs& a, int tile_rows, int sm_count) {
    const int hc = a.head_dim <= 64 ? 1 : (a.head_dim <= 128 ? 2 : 4);
    const long long room = ((long long)a.seqs.cols << a.seqs.page_log2), tiles = (room + kUnitKeys - 1) / kUnitKeys, items = items_most(a, tile_rows);
    const long long most = (long long)sm_count * ctas_of(hc, tile_rows / 8);
    if (tiles <= 1) return 0;
    for (int c = 3; c > 0; --c)
        if (items << c <= most) {
            const long long units = (tiles + (1 << c) - 1) >> c;
            return units <= 3 && units <= (items * tiles + most - 1) / most + 1 ? c : 0;
        }
    return 0;
}

template <int BF16, int HC, int NT, int CL, int P16>
cudaError_t attend_launch(const PagedAttendArgs& a, int workers, cudaStream_t stream) {
    auto kern = paged_attend_kernel<BF16, HC, NT, CL, P16>;
    TensorMapEncodeFn enc = tensor_map_encoder();
    if (!enc) return cudaErrorNotSupported;
    const int page = 1 << a.seqs.page_log2;
    PagedMaps m;
    const cuuint64_t dim[3] = {(cuuint64_t)a.head_dim, (cuuint64_t)page, (cuuint64_t)a.seqs.pages * a.kv_heads * 2};
    const cuuint64_t stride[2] = {(cuuint64_t)a.head_dim, (cuuint64_t)page * a.head_dim};
    const cuuint32_t box[3] = {HC == 1 ? 64u : 128u, page >= 32 ? 32u : 16u, 1}, ones[3] = {1, 1, 1};
    if (dim[2] == 0) return cudaErrorInvalidValue;
    if (enc(&m.codes, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, (void*)a.codes, dim, stride, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
            HC == 1 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
        return cudaErrorInvalidValue;
    const size_t smem = 1024 + (size_t)kPaWarps * stages_of(HC) * 4096 * HC + (CL ? 8 * NT * 64 * HC * 4 : 0);
    static std::atomic<int> attr_dev{-1};          // the opt-in is per device
    int dev = 0;
    cudaGetDevice(&dev);
    if (attr_dev.load() != dev) {
        const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) return e;
        attr_dev.store(dev);
    }
    if (!CL) return launch_pdl(kern, dim3((unsigned)workers), dim3(kPaThreads), smem, stream, m, a);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)workers);
    cfg.blockDim = dim3(kPaThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = 1u << a.cluster_log2;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, kern, m, a);
}

}  // namespace

// Floats of workspace for any batch of these sizes: two partial sums a worker.
size_t paged_attend_ws_floats(const PagedAttendArgs& a, int sm_count) {
    const int tr = tile_rows_of(a.heads / a.kv_heads, a.max_rows), w = workers_of(a, tr, sm_count);
    return w > 1 && !cluster_of(a, tr, sm_count) ? 2 * (size_t)w * part_floats(tr, a.head_dim) : 0;
}

cudaError_t paged_attend_launch(PagedAttendArgs a, int bf16, int sm_count, cudaStream_t stream) {
    if (a.seqs.rows == 0 || a.seqs.seqs == 0) return cudaSuccess;
    a.q_vec = a.q_stride % 8 == 0 && ((uintptr_t)a.q & 15) == 0;
    a.by_group = fast_div((uint32_t)(a.heads / a.kv_heads));
    a.by_quads = fast_div((uint32_t)(a.head_dim / 4));
    a.out_vec = a.out_stride % 4 == 0 && ((uintptr_t)a.out & 7) == 0;
    const int tr = tile_rows_of(a.heads / a.kv_heads, a.max_rows);
    a.cluster_log2 = cluster_of(a, tr, sm_count);
    const int workers = a.cluster_log2 ? (int)(items_most(a, tr) << a.cluster_log2) : workers_of(a, tr, sm_count);
    const int hc = a.head_dim <= 64 ? 1 : (a.head_dim <= 128 ? 2 : 4);
    cudaError_t e;
#define SMEG_PA2(B, H, N, C) (a.seqs.page_log2 == 4 ? attend_launch<B, H, N, C, 1>(a, workers, stream) : attend_launch<B, H, N, C, 0>(a, workers, stream))
#define SMEG_PA(B, H, N) (a.cluster_log2 ? SMEG_PA2(B, H, N, 1) : SMEG_PA2(B, H, N, 0))
    if (bf16) {
        if (tr == 8) e = hc == 1 ? SMEG_PA(1, 1, 1) : (hc == 2 ? SMEG_PA(1, 2, 1) : SMEG_PA(1, 4, 1));
        else e = hc == 1 ? SMEG_PA(1, 1, 2) : (hc == 2 ? SMEG_PA(1, 2, 2) : SMEG_PA(1, 4, 2));
    } else {
        if (tr == 8) e = hc == 1 ? SMEG_PA(0, 1, 1) : (hc == 2 ? SMEG_PA(0, 2, 1) : SMEG_PA(0, 4, 1));
        else e = hc == 1 ? SMEG_PA(0, 1, 2) : (hc == 2 ? SMEG_PA(0, 2, 2) : SMEG_PA(0, 4, 2));
    }
#undef SMEG_PA
#undef SMEG_PA2
    if (e != cudaSuccess || workers == 1 || a.cluster_log2) return e;
    const long long items = items_bound(a, tr);
    if (items >= workers)
        return bf16 ? launch_pdl(paged_join_cuts_kernel<1>, dim3((unsigned)workers - 1), dim3(kPaThreads), 0, stream, a, workers, tr)
                    : launch_pdl(paged_join_cuts_kernel<0>, dim3((unsigned)workers - 1), dim3(kPaThreads), 0, stream, a, workers, tr);
    // a row a CTA while that is no more than two CTAs an SM
    const int lanes = kPjThreads / (a.head_dim / 4), rows = (int)min((long long)tr, (long long)a.max_rows * (a.heads / a.kv_heads));
    int par = 1;
    while (par * 2 <= lanes && par < rows && items * ((rows + par - 1) / par) > 2 * sm_count) par *= 2;
    a.by_par = fast_div((uint32_t)par);
    const dim3 grid((unsigned)items, (unsigned)((rows + par - 1) / par));
    return bf16 ? launch_pdl(paged_join_items_kernel<1>, grid, dim3(kPjThreads), 0, stream, a, workers, tr, par)
                : launch_pdl(paged_join_items_kernel<0>, grid, dim3(kPjThreads), 0, stream, a, workers, tr, par);
}

}  // namespace smeg
