// Attention of a batch's new rows against the pages of the 8-bit key/value cache (sm_100a).
//
//   out = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale * q . k_j - max),  j up to the row's own position;  k, v = (byte - 128) * scale of the
//   page's block.  One pass over the keys with the running maximum and sum, 32-bit sums.
//
// What bounds it is the cache: 2 bytes per position, KV head and depth, each read once for all query rows of a tile (a tile: 8 or 16 rows x heads
// of a group).  The keys of all (sequence, row tile, KV head) are one line of units of 128 keys, cut into equal shares for as many CTAs as the GPU
// holds, whatever the lengths; an item that a cut goes through is joined by a second kernel from the shares' unnormalised sums.  Within a unit a
// warp has 32 keys and needs no other warp until its share of an item is done.
//
// Both products are mma.m16n8k16 with the cache as the 16-row operand, so that up to eight query rows cost one column tile:
//   S^T (keys x rows) = K Q^T,   O^T (depths x rows) += V^T P^T
// A byte is not converted: as the low byte of a half word it is the f16 subnormal u * 2^-24, two masks for four codes, and the 128 of its offset
// comes off through the accumulators' start values (-128 * 2^-24 * the sum of the other operand, formed by the same instruction on a constant).
// Operands go from global memory to the registers they are used from: a lane takes 16 consecutive depths of a key as four steps of the first product, and
// 16 depths of its four keys as eight row tiles of the second.  A query row is scaled by a power of two into f16's range (so bf16 queries are
// exact too); the probabilities are f16 at 2^14, a group's scaled by its page's scale over the larger of the warp's two, and each 32 keys' sums are
// folded into 32-bit registers, since the tensor core cuts its sums off.
#include "common.cuh"
#include "kernels.h"
#include "paged.h"

namespace smeg {
namespace {

constexpr int kPaThreads = 128, kPaWarps = 4;
constexpr uint32_t kOffset = 0x00800080u;           // two f16 subnormals of 128 * 2^-24
constexpr float kPScale = 16384.0f;

__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t mov_trans(uint32_t x) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
    return r;
}
__device__ __forceinline__ uint32_t even_bytes(uint32_t w) { return w & 0x00ff00ffu; }
__device__ __forceinline__ uint32_t odd_bytes(uint32_t w) { return __byte_perm(w, 0, 0x4341); }
__device__ __forceinline__ uint4 ld_stream(const uint8_t* p) {
    uint4 v;
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}
__device__ __forceinline__ uint2 ld_stream2(const uint8_t* p) {
    uint2 v;
    asm volatile("ld.global.L1::no_allocate.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p));
    return v;
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
__device__ __forceinline__ long long block_scan(long long x, long long* warp_sums, long long* all) {   // inclusive; 128 threads
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    __syncthreads();                                               // (the sums of a scan before have been read)
    if (lane == 31) warp_sums[warp] = x;
    __syncthreads();
    long long before = 0;
#pragma unroll
    for (int w = 0; w < kPaWarps; ++w) {
        if (w < warp) before += warp_sums[w];
    }
    *all = warp_sums[0] + warp_sums[1] + warp_sums[2] + warp_sums[3];
    return x + before;
}
__device__ __forceinline__ long long units_of(const PagedAttendArgs& p, int s, int tile_rows) {
    if (s >= p.seqs.seqs) return 0;
    const SeqUnits u = seq_units(p.seqs, s, p.heads / p.kv_heads, p.kv_heads, tile_rows);
    return u.items * u.tiles;
}
// The total of all units, and (find) the place of unit `at(total)`; false where there is none.
template <class At>
__device__ __forceinline__ bool find_unit(const PagedAttendArgs& p, int tile_rows, At at, long long* total_out, Place* out) {
    __shared__ long long warp_sums[kPaWarps], s_off;
    __shared__ int s_seq;
    const int tid = threadIdx.x, n = p.seqs.seqs;
    const bool once = n <= kPaThreads;
    if (tid == 0) s_seq = -1;
    long long total = 0, mine = 0, incl = 0, all = 0;
    for (int s0 = 0; s0 < n; s0 += kPaThreads) {
        mine = units_of(p, s0 + tid, tile_rows);
        incl = block_scan(mine, warp_sums, &all);
        total += all;
    }
    *total_out = total;
    const long long u = at(total);
    if (u < 0 || u >= total) return false;                         // (uniform: the whole block)
    long long base = 0;
    for (int s0 = 0; s0 < n; s0 += kPaThreads) {
        if (!once) {
            mine = units_of(p, s0 + tid, tile_rows);
            incl = block_scan(mine, warp_sums, &all);
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

// HC: depths in units of 64 (1, 2 or 4); NT: tiles of eight query rows.
template <int BF16, int HC, int NT>
__global__ void __launch_bounds__(kPaThreads, HC == 4 ? (NT == 1 ? 2 : 1) : (NT == 1 ? 3 : 2)) paged_attend_kernel(const __grid_constant__ PagedAttendArgs p) {
    constexpr int G = HC == 4 ? 1 : 2;               // groups of 16 keys that a warp has at a time
    constexpr int kKeys = 16 * G;
    constexpr int MT = 4 * HC;                       // tiles of 16 depths
    constexpr int NR = 8 * NT;
    extern __shared__ __align__(16) float part[];    // [warp][NR maxima, NR sums, NR x depths]
    const int tid = threadIdx.x, warp = warp_index(), lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int hd = p.head_dim, group = p.heads / p.kv_heads, page = 1 << p.seqs.page_log2;
    const size_t block = (size_t)page * hd;
    pdl_launch_dependents();
    pdl_wait();
    long long total;
    Place at;
    if (!find_unit(p, NR, [&](long long n) { return share_begin(n, gridDim.x, blockIdx.x); }, &total, &at)) return;
    long long left = share_begin(total, gridDim.x, blockIdx.x + 1) - share_begin(total, gridDim.x, blockIdx.x);
    bool first_piece = true;
    int s = at.s;
    long long off = at.off;
    while (left > 0 && s < p.seqs.seqs) {
        const SeqUnits U = seq_units(p.seqs, s, group, p.kv_heads, NR);
        if (off >= U.items * U.tiles) { ++s; off = 0; continue; }
        const long long item = off / U.tiles;
        const int tile0 = (int)(off - item * U.tiles), tile1 = (int)min((long long)U.tiles, tile0 + left);
        const int kvh = (int)(item % p.kv_heads);
        const long long row_tile = item / p.kv_heads;
        const int n0 = (int)(row_tile * NR), nrow = (int)min((long long)NR, (long long)U.rows * group - n0);   // packed rows x heads of the tile
        left -= tile1 - tile0;
        off += tile1 - tile0;

        // ---- queries: B fragments, a power of two to each row ----
        uint32_t qf[NT][4 * HC][2];
        float row_scale[NT][2], start0[NT][2];
        int limit[NT][2];                            // keys that rows 2 t and 2 t + 1 of a tile attend to
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            const int n = n0 + 8 * j + g, i = n / group, head = kvh * group + (n - i * group);
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
            const int up = mx > 0.0f && ex < 120 && ex > -110 ? 14 - ex : 0;
            const float f = __uint_as_float((uint32_t)(127 + up) << 23);
            const float back = __uint_as_float((uint32_t)(127 - up) << 23) * (p.scale_log2e * 16777216.0f);
#pragma unroll
            for (int c = 0; c < HC; ++c)
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    qf[j][4 * c + w][0] = pack2_t<0>(x[c][4 * w] * f, x[c][4 * w + 2] * f);
                    qf[j][4 * c + w][1] = pack2_t<0>(x[c][4 * w + 1] * f, x[c][4 * w + 3] * f);
                }
            float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int k = 0; k < 4 * HC; ++k) mma_f16(sum, kOffset, kOffset, kOffset, kOffset, qf[j][k][0], qf[j][k][1]);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                start0[j][e] = -sum[e];
                row_scale[j][e] = __shfl_sync(0xffffffffu, back, 4 * (2 * t + e));
                const int m = n0 + 8 * j + 2 * t + e;
                limit[j][e] = 8 * j + 2 * t + e < nrow && U.start >= 0 ? min(U.start + m / group + 1, U.keys) : 0;
            }
        }

        // ---- this warp's keys of the tiles ----
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
        constexpr int kPer = kUnitKeys / kPaWarps / kKeys;             // pieces of kKeys keys that a warp has of a unit
        const int pieces_all = (tile1 - tile0) * kPer;
        uint4 kq[G][2][HC];                                            // key g and g + 8 of a group, 16 depths a chunk
        uint4 vq[G][4][HC == 4 ? 2 : 1];                               // keys 2 t, 2 t + 1, 2 t + 8, 2 t + 9
        float sk[G], sv[G];
        float sk_n[G], sv_n[G];
        const uint8_t* base[G];
        bool there[G];                                                 // the group's page holds keys that some row attends to
        auto key_of = [&](int i) { return (tile0 + i / kPer) * kUnitKeys + warp * 32 + (i % kPer) * kKeys; };
        auto locate = [&](int i) {
#pragma unroll
            for (int b = 0; b < G; ++b) {
                const int key = key_of(i) + 16 * b;
                int id = -1;
                if (i < pieces_all && key < U.keys) {
                    id = page_of(p.seqs, s, key);
                    if (id < 0 && lane == 0 && p.status) atomicOr(p.status, STATUS_PAGE);
                }
                there[b] = id >= 0;
                const size_t blk = ((size_t)max(id, 0) * p.kv_heads + kvh) * 2;
                base[b] = p.codes + blk * block + (size_t)(key & (page - 1)) * hd;
                sk_n[b] = there[b] ? p.scales[blk] : 0.0f;
                sv_n[b] = there[b] ? p.scales[blk + 1] : 0.0f;
            }
        };
        auto load_k = [&]() {
#pragma unroll
            for (int b = 0; b < G; ++b)
#pragma unroll
                for (int r = 0; r < 2; ++r)
#pragma unroll
                    for (int c = 0; c < HC; ++c) {
                        const int d = 16 * (t + 4 * c);
                        kq[b][r][c] = there[b] && d < hd ? ld_stream(base[b] + (size_t)(g + 8 * r) * hd + d) : make_uint4(0, 0, 0, 0);
                    }
        };
        auto load_v = [&]() {
#pragma unroll
            for (int b = 0; b < G; ++b)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const uint8_t* v = base[b] + block + (size_t)(2 * t + (r & 1) + 8 * (r >> 1)) * hd;
                    if (HC == 1) {
                        const uint2 w = there[b] && 8 * g < hd ? ld_stream2(v + 8 * g) : make_uint2(0, 0);
                        vq[b][r][0] = make_uint4(w.x, w.y, 0, 0);
                    } else {
#pragma unroll
                        for (int c = 0; c < (HC == 4 ? 2 : 1); ++c) {
                            const int d = 16 * g + 128 * c;
                            vq[b][r][c] = there[b] && d < hd ? ld_stream(v + d) : make_uint4(0, 0, 0, 0);
                        }
                    }
                }
        };
        locate(0);
        load_k();
        load_v();
        for (int i = 0; i < pieces_all; ++i) {
            const int key0 = key_of(i);
#pragma unroll
            for (int b = 0; b < G; ++b) { sk[b] = sk_n[b]; sv[b] = sv_n[b]; }
            bool here[G];
#pragma unroll
            for (int b = 0; b < G; ++b) here[b] = there[b];
            // scores
            float sc[NT][G][4];
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int b = 0; b < G; ++b) {
                    sc[j][b][0] = sc[j][b][2] = start0[j][0];
                    sc[j][b][1] = sc[j][b][3] = start0[j][1];
                }
#pragma unroll
            for (int b = 0; b < G; ++b)
#pragma unroll
                for (int c = 0; c < HC; ++c) {
                    const uint32_t lo[4] = {kq[b][0][c].x, kq[b][0][c].y, kq[b][0][c].z, kq[b][0][c].w};
                    const uint32_t hi[4] = {kq[b][1][c].x, kq[b][1][c].y, kq[b][1][c].z, kq[b][1][c].w};
#pragma unroll
                    for (int w = 0; w < 4; ++w) {
                        const uint32_t a0 = even_bytes(lo[w]), a1 = even_bytes(hi[w]), a2 = odd_bytes(lo[w]), a3 = odd_bytes(hi[w]);
#pragma unroll
                        for (int j = 0; j < NT; ++j) mma_f16(sc[j][b], a0, a1, a2, a3, qf[j][4 * c + w][0], qf[j][4 * c + w][1]);
                    }
                }
            // (the next keys are on their way while these are weighed; their values' addresses are kept for after this piece's values)
            locate(i + 1);
            load_k();
            float st = 0.0f;                                           // (fmaxf drops a NaN: it stays with the rows that attend to it)
#pragma unroll
            for (int b = 0; b < G; ++b) st = fmaxf(st, sv[b]);
            uint32_t pf[NT][G][2];
            float alpha[NT][2];
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                float mx[2] = {-INFINITY, -INFINITY};
                bool on[G][4];
#pragma unroll
                for (int b = 0; b < G; ++b)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int key = key0 + 16 * b + g + 8 * (e >> 1);
                        on[b][e] = here[b] && key < limit[j][e & 1];
                        sc[j][b][e] = sc[j][b][e] * (row_scale[j][e & 1] * sk[b]);
                        if (on[b][e]) mx[e & 1] = fmaxf(mx[e & 1], sc[j][b][e]);
                    }
#pragma unroll
                for (int e = 0; e < 2; ++e) {
#pragma unroll
                    for (int w = 4; w < 32; w <<= 1) mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], w));
                    mx[e] = fmaxf(mx[e], m_run[j][e]);
                    const float ref = mx[e] == -INFINITY ? 0.0f : mx[e];
                    alpha[j][e] = ex2(m_run[j][e] - ref);
                    m_run[j][e] = mx[e];
                    mx[e] = ref;
                    l_run[j][e] *= alpha[j][e];
                }
#pragma unroll
                for (int b = 0; b < G; ++b) {
                    const float ratio = (sv[b] == st ? 1.0f : (st > 0.0f ? __fdividef(sv[b], st) : sv[b])) * kPScale;
                    float w[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float x = ex2(sc[j][b][e] - mx[e & 1]);
                        l_run[j][e & 1] += on[b][e] ? x : 0.0f;
                        w[e] = on[b][e] ? x * ratio : 0.0f;
                    }
                    pf[j][b][0] = mov_trans(pack2_t<0>(w[0], w[1]));
                    pf[j][b][1] = mov_trans(pack2_t<0>(w[2], w[3]));
                }
            }
            // values
            float off0[NT][4];
#pragma unroll
            for (int j = 0; j < NT; ++j) {
#pragma unroll
                for (int e = 0; e < 4; ++e) off0[j][e] = 0.0f;
#pragma unroll
                for (int b = 0; b < G; ++b) mma_f16(off0[j], kOffset, kOffset, kOffset, kOffset, pf[j][b][0], pf[j][b][1]);
            }
#pragma unroll
            for (int m = 0; m < MT; m += 2) {                          // a word of four depths: tiles m and m + 1
                float acc[2][NT][4];
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int j = 0; j < NT; ++j)
#pragma unroll
                        for (int e = 0; e < 4; ++e) acc[h][j][e] = -off0[j][e];
#pragma unroll
                for (int b = 0; b < G; ++b) {
                    uint32_t w[4];
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const uint4 v = vq[b][r][HC == 4 ? m / 8 : 0];
                        const uint32_t x[4] = {v.x, v.y, v.z, v.w};
                        w[r] = x[(m / 2) & 3];
                    }
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const uint32_t x = __byte_perm(w[0], w[1], h ? 0x7632 : 0x5410), y = __byte_perm(w[2], w[3], h ? 0x7632 : 0x5410);
#pragma unroll
                        for (int j = 0; j < NT; ++j) mma_f16(acc[h][j], even_bytes(x), odd_bytes(x), even_bytes(y), odd_bytes(y), pf[j][b][0], pf[j][b][1]);
                    }
                }
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int j = 0; j < NT; ++j)
#pragma unroll
                        for (int e = 0; e < 4; ++e) o[j][m + h][e] = fmaf(o[j][m + h][e], alpha[j][e & 1], acc[h][j][e] * st);
            }
            load_v();
        }

        // ---- the warps' shares meet, then the item's ----
        __syncthreads();                                               // (an earlier item's have been read)
        float* mine = part + (size_t)warp * part_floats(NR, hd);
#pragma unroll
        for (int j = 0; j < NT; ++j) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                float l = l_run[j][e];
#pragma unroll
                for (int w = 4; w < 32; w <<= 1) l += __shfl_xor_sync(0xffffffffu, l, w);
                if (g == 0) {
                    mine[8 * j + 2 * t + e] = m_run[j][e];
                    mine[NR + 8 * j + 2 * t + e] = l;
                }
            }
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    // row tile m's rows g and g + 8 are depths 2 m and 2 m + 1 of the lane's run
                    const int d = HC == 1 ? 8 * g + 2 * m + (e >> 1) : 16 * g + 128 * (m / 8) + 2 * (m % 8) + (e >> 1);
                    if (d < hd) mine[2 * NR + (8 * j + 2 * t + (e & 1)) * hd + d] = o[j][m][e];
                }
        }
        __syncthreads();
        const bool whole = tile0 == 0 && tile1 == U.tiles;
        float* ws = p.ws + (2 * (size_t)blockIdx.x + (first_piece ? 0 : 1)) * part_floats(NR, hd);
        first_piece = false;
        for (int it = tid; it < nrow * (hd / 4); it += kPaThreads) {
            const int n = it / (hd / 4), d = (it - n * (hd / 4)) * 4;
            float mx = -INFINITY;
#pragma unroll
            for (int w = 0; w < kPaWarps; ++w) mx = fmaxf(mx, part[(size_t)w * part_floats(NR, hd) + n]);
            const float ref = mx == -INFINITY ? 0.0f : mx;
            float l = 0.0f;
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < kPaWarps; ++w) {
                const float* o_w = part + (size_t)w * part_floats(NR, hd);
                const float f = ex2(o_w[n] - ref);
                const float4 x = *reinterpret_cast<const float4*>(o_w + 2 * NR + n * hd + d);
                l = fmaf(f, o_w[NR + n], l);
                v.x = fmaf(f, x.x, v.x); v.y = fmaf(f, x.y, v.y); v.z = fmaf(f, x.z, v.z); v.w = fmaf(f, x.w, v.w);
            }
            if (whole) {
                const float r = l == 0.0f ? 0.0f : __fdiv_rn(16777216.0f / kPScale, l);   // (a row that attends to nothing is zero)
                const int i = (n0 + n) / group, head = kvh * group + (n0 + n) - i * group;
                store_row4<BF16>(p, U.first + i, head, d, make_float4(v.x * r, v.y * r, v.z * r, v.w * r));
            } else {
                if (d == 0) { ws[n] = mx; ws[NR + n] = l; }
                *reinterpret_cast<float4*>(ws + 2 * NR + n * hd + d) = v;
            }
        }
    }
}

// CTA b: the item that the cut before worker b + 1 goes through, if that is the first one through it.  A cut item is the last of its first worker's
// and the first of the others'.
template <int BF16>
__global__ void __launch_bounds__(kPaThreads) paged_join_kernel(const __grid_constant__ PagedAttendArgs p, int workers, int tile_rows) {
    const int tid = threadIdx.x, hd = p.head_dim, group = p.heads / p.kv_heads;
    pdl_launch_dependents();
    pdl_wait();
    const int cut = blockIdx.x + 1;
    long long total;
    Place at;
    if (!find_unit(p, tile_rows, [&](long long n) { return share_begin(n, workers, cut); }, &total, &at)) return;
    const SeqUnits U = seq_units(p.seqs, at.s, group, p.kv_heads, tile_rows);
    const long long item = at.off / U.tiles, u = share_begin(total, workers, cut);
    const long long begin = u - (at.off - item * U.tiles), end = begin + U.tiles;
    if (begin == u) return;                                            // the cut is between two items
    const int w0 = share_of(total, workers, begin), w1 = share_of(total, workers, end - 1);
    if (w0 != cut - 1) return;
    const int kvh = (int)(item % p.kv_heads), n0 = (int)(item / p.kv_heads * tile_rows);
    const int nrow = (int)min((long long)tile_rows, (long long)U.rows * group - n0);
    const size_t pf = part_floats(tile_rows, hd);
    const size_t slot0 = 2 * (size_t)w0 + (begin > share_begin(total, workers, w0) ? 1 : 0);
    for (int it = tid; it < nrow * (hd / 4); it += kPaThreads) {
        const int n = it / (hd / 4), d = (it - n * (hd / 4)) * 4;
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
        const int i = (n0 + n) / group, head = kvh * group + (n0 + n) - i * group;
        store_row4<BF16>(p, U.first + i, head, d, make_float4(v.x * r, v.y * r, v.z * r, v.w * r));
    }
}

int tile_rows_of(int group, int max_rows) { return (long long)group * max_rows > 8 ? 16 : 8; }

// CTAs: as many as the GPU holds at a time (the occupancy of the variant), no more than there can be units.
int workers_of(const PagedAttendArgs& a, int tile_rows, int sm_count) {
    const int hc = a.head_dim <= 64 ? 1 : (a.head_dim <= 128 ? 2 : 4);
    const int per_sm = hc == 4 ? (tile_rows == 8 ? 2 : 1) : (tile_rows == 8 ? 3 : 2);
    const long long room = ((long long)a.seqs.cols << a.seqs.page_log2), tiles = (room + kUnitKeys - 1) / kUnitKeys;
    const long long items = ((long long)a.seqs.rows * (a.heads / a.kv_heads) / tile_rows + a.seqs.seqs) * a.kv_heads;
    const long long most = (long long)sm_count * per_sm, units = items * (tiles > 0 ? tiles : 1);
    return (int)(units < most ? (units > 0 ? units : 1) : most);
}

template <int BF16, int HC, int NT>
cudaError_t attend_launch(const PagedAttendArgs& a, int workers, cudaStream_t stream) {
    auto kern = paged_attend_kernel<BF16, HC, NT>;
    const size_t smem = kPaWarps * part_floats(8 * NT, a.head_dim) * sizeof(float);
    if (smem > 48 * 1024) {
        const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) return e;
    }
    return launch_pdl(kern, dim3((unsigned)workers), dim3(kPaThreads), smem, stream, a);
}

}  // namespace

// Floats of workspace for any batch of these sizes: two partial sums a worker.
size_t paged_attend_ws_floats(const PagedAttendArgs& a, int sm_count) {
    const int tr = tile_rows_of(a.heads / a.kv_heads, a.max_rows), w = workers_of(a, tr, sm_count);
    return w > 1 ? 2 * (size_t)w * part_floats(tr, a.head_dim) : 0;
}

cudaError_t paged_attend_launch(PagedAttendArgs a, int bf16, int sm_count, cudaStream_t stream) {
    if (a.seqs.rows == 0 || a.seqs.seqs == 0) return cudaSuccess;
    a.q_vec = a.q_stride % 8 == 0 && ((uintptr_t)a.q & 15) == 0;
    a.out_vec = a.out_stride % 4 == 0 && ((uintptr_t)a.out & 7) == 0;
    const int tr = tile_rows_of(a.heads / a.kv_heads, a.max_rows), workers = workers_of(a, tr, sm_count);
    const int hc = a.head_dim <= 64 ? 1 : (a.head_dim <= 128 ? 2 : 4);
    cudaError_t e;
#define SMEG_PA(B, H, N) attend_launch<B, H, N>(a, workers, stream)
    if (bf16) {
        if (tr == 8) e = hc == 1 ? SMEG_PA(1, 1, 1) : (hc == 2 ? SMEG_PA(1, 2, 1) : SMEG_PA(1, 4, 1));
        else e = hc == 1 ? SMEG_PA(1, 1, 2) : (hc == 2 ? SMEG_PA(1, 2, 2) : SMEG_PA(1, 4, 2));
    } else {
        if (tr == 8) e = hc == 1 ? SMEG_PA(0, 1, 1) : (hc == 2 ? SMEG_PA(0, 2, 1) : SMEG_PA(0, 4, 1));
        else e = hc == 1 ? SMEG_PA(0, 1, 2) : (hc == 2 ? SMEG_PA(0, 2, 2) : SMEG_PA(0, 4, 2));
    }
#undef SMEG_PA
    if (e != cudaSuccess || workers == 1) return e;
    return bf16 ? launch_pdl(paged_join_kernel<1>, dim3((unsigned)workers - 1), dim3(kPaThreads), 0, stream, a, workers, tr)
                : launch_pdl(paged_join_kernel<0>, dim3((unsigned)workers - 1), dim3(kPaThreads), 0, stream, a, workers, tr);
}

}  // namespace smeg
