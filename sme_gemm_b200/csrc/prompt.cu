// Causal attention over whole packed prompts, grouped heads (sm_100a): row i of a sequence attends to the sequence's rows 0 .. i.
//
//   out = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale * q . k_j - max), j <= i
// One pass over the keys with the running maximum and sum; sums are 32 bits wide, the probabilities are rounded to the inputs' type for the second
// product.  The query rows of one KV head -- every row times every head of the group -- are the rows of a tile, so that grouped heads share one
// read of the keys and values.
//
// Bound by the tensor cores where prompts are long: 8192 rows, 32 / 8 heads of 128, 480 to 500 us back to back, under the power cap (1100 to 1150 TFLOP/s of causal work; a
// long cuBLAS product holds 1409), 4096 rows of 16 / 2 heads of 256 116 us (1180).  Heads of 64 do a product in half the time and the same exponentials, which bound them
// there: 350 us.  Short prompts are bound by an item's ends -- first scores, last product, results on their way out -- and the masked halves of last blocks: eleven
// prompts of 7001 rows, 32 / 8 heads of 128, 73 to 77 us, 15 of which the results' way out took before it was a bulk store.
#include "common.cuh"
#include "kernels.h"
#include "paged.h"
#include "tc_common.cuh"

#include <string.h>

#include <atomic>

namespace smeg {
namespace {

constexpr float kInf = INFINITY;

__device__ __forceinline__ float ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// ---- rows formed again ----
// A key block's second product multiplies every value of the block by every row's probability, also by the zeros of rows that do not attend to it: an
// infinity or NaN there makes NaNs (0 * inf).  So rows whose results are not finite although their probabilities are get them from what they attend to alone, where the
// blocks that they share with later rows hold such a value.

template <int BF16>
__device__ __forceinline__ void mma_t(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if (BF16)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Eight 16-bit values of a row, from any address, zeros where there are none.
__device__ __forceinline__ uint4 load8(const uint16_t* x, bool in, bool vec) {
    if (!in) return make_uint4(0, 0, 0, 0);
    if (vec) return *reinterpret_cast<const uint4*>(x);
    uint32_t w[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) w[e] = (uint32_t)x[2 * e] | (uint32_t)x[2 * e + 1] << 16;
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// Rows n0 .. n0 + nrow (at most 16 of a sequence's rows x heads of the group) of KV head kvh: those whose bit is set in `which` are formed and written.  A warp.  Keys that
// all rows attend to go through the tensor cores, 32 at a time and PANEL depths a pass; the last few, which only some do, are added value by value, so that nothing is
// multiplied by a zero that stands for "not attended".  (Whole keys are loaded as runs of eight depths: as the depths of a product may come in any order, lane t's
// run of a 32-depth piece is its share of two products, and lane g's run of 64 depths a column of eight.)
// (PANEL: 64 or 128 depths a pass.  VEC: rows on 16-byte boundaries.)  One infinity in the last rows of 8192, 32 / 8 heads of 128: 2.9 ms for 0.42, twice 256 steps of 32 keys;
// infinities at one in a hundred of the values' rows 4.4 ms; a key at a time for each row 16 ms at 1024 rows, where these are 0.31.
template <int BF16, int VEC, int PANEL>
__device__ __forceinline__ void form_again(const PromptArgs& p, int first, int kvh, long long n0, int nrow, unsigned which, int vec) {
    const bool vec_q = VEC || (vec & 1), vec_kv = VEC || (vec >> 1);
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3, hd = p.head_dim, group = p.heads / p.kv_heads;
    const int low = (int)(n0 / group), keys = (int)((n0 + nrow - 1) / group) + 1;                 // keys that every row attends to: low + 1
    const uint16_t *q[2], *k0 = p.k + (size_t)first * p.k_stride + (size_t)kvh * hd, *v0 = p.v + (size_t)first * p.v_stride + (size_t)kvh * hd;
    int tok[2];
    size_t out_at[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        const long long n = n0 + min(g + 8 * e, nrow - 1);
        tok[e] = (int)(n / group);
        const size_t head = (size_t)kvh * group + (size_t)(n - (long long)tok[e] * group);
        q[e] = p.q + (size_t)(first + tok[e]) * p.q_stride + head * hd;
        out_at[e] = (size_t)(first + tok[e]) * p.out_stride + head * hd;
    }
    for (int d0 = 0; d0 < hd; d0 += PANEL) {
        float o[PANEL / 8][4], m[2] = {-kInf, -kInf}, l[2] = {0.0f, 0.0f};
#pragma unroll
        for (int n = 0; n < PANEL / 8; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[n][e] = 0.0f;
        for (int key0 = 0; key0 < keys; key0 += 32) {
            float s[4][4];
#pragma unroll
            for (int n = 0; n < 4; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) s[n][e] = 0.0f;
            for (int c = 0; c < hd; c += 32) {
                const int d = c + 8 * t;
                const uint4 x = load8(q[0] + d, d < hd, vec_q), y = load8(q[1] + d, d < hd, vec_q);
                const uint32_t a0[4] = {x.x, y.x, x.y, y.y}, a1[4] = {x.z, y.z, x.w, y.w};
#pragma unroll
                for (int n = 0; n < 4; ++n) {
                    const uint4 b = load8(k0 + (size_t)min(key0 + 8 * n + g, keys - 1) * p.k_stride + d, d < hd, vec_kv);
                    mma_t<BF16>(s[n], a0, b.x, b.y);
                    mma_t<BF16>(s[n], a1, b.z, b.w);
                }
            }
            float mx[2] = {m[0], m[1]};
#pragma unroll
            for (int n = 0; n < 4; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    s[n][e] = key0 + 8 * n + 2 * t + (e & 1) <= tok[e >> 1] ? s[n][e] * p.scale_log2e : -kInf;
                    mx[e >> 1] = fmaxf(mx[e >> 1], s[n][e]);
                }
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], 1));
                mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], 2));
                const float ref = mx[e] == -kInf ? 0.0f : mx[e], alpha = ex2(m[e] - ref);
                m[e] = mx[e];
                mx[e] = ref;
                l[e] *= alpha;
#pragma unroll
                for (int n = 0; n < PANEL / 8; ++n) {
                    o[n][2 * e] *= alpha;
                    o[n][2 * e + 1] *= alpha;
                }
            }
            bool lost = false;                                         // a weight that f16 has no number for
#pragma unroll
            for (int n = 0; n < 4; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    s[n][e] = ex2(s[n][e] - mx[e >> 1]);
                    l[e >> 1] += s[n][e];
                    lost = lost || (s[n][e] > 0.0f && s[n][e] <= 0x1p-25f);
                }
            bool one_by_one = key0 + 31 > low;
            if (!BF16 && !one_by_one && __any_sync(0xffffffffu, lost)) {   // (a lost weight of an infinity is none of zero)
                bool found = false;
                for (int d = d0 + 8 * t; d < min(hd, d0 + PANEL); d += 32)
#pragma unroll
                    for (int n = 0; n < 4; ++n) {
                        const uint4 b = load8(v0 + (size_t)(key0 + 8 * n + g) * p.v_stride + d, true, vec_kv);
                        const uint32_t w[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
                        for (int i = 0; i < 4; ++i) found = found || (w[i] & 0x7c00u) == 0x7c00u || (w[i] & 0x7c000000u) == 0x7c000000u;
                    }
                one_by_one = __any_sync(0xffffffffu, found);
            }
            if (!one_by_one) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const uint32_t pa[4] = {pack2_t<BF16>(s[2 * h][0], s[2 * h][1]), pack2_t<BF16>(s[2 * h][2], s[2 * h][3]), pack2_t<BF16>(s[2 * h + 1][0], s[2 * h + 1][1]),
                                            pack2_t<BF16>(s[2 * h + 1][2], s[2 * h + 1][3])};
                    const uint16_t* v = v0 + (size_t)(key0 + 16 * h + 2 * t) * p.v_stride;
#pragma unroll
                    for (int c = 0; c < PANEL / 64; ++c) {
                        const int d = d0 + 64 * c + 8 * g;
                        if (c > 0 && d0 + 64 * c >= hd) break;
                        const uint4 w0 = load8(v + d, d < hd, vec_kv), w1 = load8(v + p.v_stride + d, d < hd, vec_kv), w2 = load8(v + 8 * p.v_stride + d, d < hd, vec_kv),
                                    w3 = load8(v + 9 * p.v_stride + d, d < hd, vec_kv);
                        const uint32_t r0[4] = {w0.x, w0.y, w0.z, w0.w}, r1[4] = {w1.x, w1.y, w1.z, w1.w}, r2[4] = {w2.x, w2.y, w2.z, w2.w}, r3[4] = {w3.x, w3.y, w3.z, w3.w};
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            const unsigned pick = i & 1 ? 0x7632 : 0x5410;
                            mma_t<BF16>(o[8 * c + i], pa, __byte_perm(r0[i / 2], r1[i / 2], pick), __byte_perm(r2[i / 2], r3[i / 2], pick));
                        }
                    }
                }
            } else {
#pragma unroll 1
                for (int k = 0; k < 32 && key0 + k < keys; ++k) {
                    float w[2];
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const float a = k & 1 ? (k & 8 ? (k & 16 ? s[3][2 * e + 1] : s[1][2 * e + 1]) : (k & 16 ? s[2][2 * e + 1] : s[0][2 * e + 1]))
                                              : (k & 8 ? (k & 16 ? s[3][2 * e] : s[1][2 * e]) : (k & 16 ? s[2][2 * e] : s[0][2 * e]));
                        w[e] = __shfl_sync(0xffffffffu, a, (lane & ~3) | ((k & 7) >> 1));
                    }
                    const bool on[2] = {key0 + k <= tok[0], key0 + k <= tok[1]};
                    const uint16_t* v = v0 + (size_t)(key0 + k) * p.v_stride;
#pragma unroll
                    for (int c = 0; c < PANEL / 32; ++c) {
                        const int d = d0 + 64 * (c >> 1) + 16 * t + 8 * (c & 1);
                        const uint4 x = load8(v + d, d < hd, vec_kv);
                        const uint32_t r[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            const float f = t_to_f32<BF16>((uint16_t)(r[i / 2] >> (16 * (i & 1))));
#pragma unroll
                            for (int e = 0; e < 2; ++e)
                                if (on[e]) o[8 * (c >> 1) + i][2 * e + (c & 1)] = fmaf(w[e], f, o[8 * (c >> 1) + i][2 * e + (c & 1)]);
                        }
                    }
                }
            }
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            l[e] += __shfl_xor_sync(0xffffffffu, l[e], 1);
            l[e] += __shfl_xor_sync(0xffffffffu, l[e], 2);
            if (!(which >> (g + 8 * e) & 1)) continue;
#pragma unroll
            for (int c = 0; c < PANEL / 32; ++c) {
                const int d = d0 + 64 * (c >> 1) + 16 * t + 8 * (c & 1);
                if (d >= hd) continue;
#pragma unroll
                for (int i = 0; i < 8; ++i) p.out[out_at[e] + d + i] = f32_to_t<BF16>(__fdiv_rn(o[8 * (c >> 1) + i][2 * e + (c & 1)], l[e]));
            }
        }
    }
}

// Which of a run of eight values are NaN, infinite, infinite below zero: a bit a value.
struct Odd {
    unsigned nan, up, down;
    __device__ __forceinline__ unsigned any() const { return nan | up | down; }
    __device__ __forceinline__ unsigned lost() const { return nan | (up & down); }                // a sum of these is a NaN
};
template <int BF16>
__device__ __forceinline__ void note(Odd& o, const uint4 x) {
    constexpr unsigned kExp = BF16 ? 0x7f80u : 0x7c00u;
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const unsigned u = w[e / 2] >> (16 * (e & 1)) & 0xffffu;
        o.nan |= (unsigned)((u & 0x7fffu) > kExp) << e;
        o.up |= (unsigned)(u == kExp) << e;
        o.down |= (unsigned)(u == (kExp | 0x8000u)) << e;
    }
}
// Rows r0 .. of a tile of `rows` that starts at n0 and whose key blocks end before row `to` of the batch: those of `mask` have results that are not finite.  A warp, once what
// it has stored is there.  A depth counts where a key that not all of the warp's rows attend to has a value that is not finite.  Where one that they all attend to has one
// as well, the sum is what these leave -- an infinity, or a NaN -- and is written; else the rows are formed again.  (A depth that is
// infinite at every position is the former: 8192 rows 0.88 ms for 0.42.)
template <int BF16, int VEC, int PANEL>
__device__ __forceinline__ void mend(const PromptArgs& p, int first, int kvh, long long n0, int to, int r0, int rows, unsigned mask, int vec) {
    __syncwarp();
    const int lane = threadIdx.x & 31, hd = p.head_dim, group = p.heads / p.kv_heads, low = first + (int)((n0 + r0) / group);
    const uint16_t* v = p.v + (size_t)kvh * hd;
    const bool in = 8 * lane < hd, vec_kv = VEC || (vec >> 1);
    Odd later = {0, 0, 0}, had = {0, 0, 0};                            // of this lane's depths 8 lane ..
#pragma unroll 4
    for (int j = low + 1; j < to; ++j) note<BF16>(later, load8(v + (size_t)j * p.v_stride + 8 * lane, in, vec_kv));
    const unsigned depths = later.any();
    for (unsigned left = __ballot_sync(0xffffffffu, depths != 0); left; left &= left - 1) {
        const int c = __ffs(left) - 1;                                 // eight depths, a key a lane, from the last one back
        const unsigned want = __shfl_sync(0xffffffffu, depths, c);
        Odd o = {0, 0, 0};
        for (int j0 = low; j0 >= first; j0 -= 128) {
            uint4 x[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int j = j0 - 32 * i - lane;
                x[i] = load8(v + (size_t)max(j, first) * p.v_stride + 8 * c, j >= first, vec_kv);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) note<BF16>(o, x[i]);
            const unsigned u = __reduce_or_sync(0xffffffffu, o.nan | o.up << 8 | o.down << 16);
            o = {u & 0xffu, u >> 8 & 0xffu, u >> 16};
            if ((want & ~o.lost()) == 0) break;                        // (nothing changes a NaN)
        }
        if (lane == c) had = o;
    }
    if (__any_sync(0xffffffffu, (depths & ~had.any()) != 0)) {
        for (int h = 0; h < 32; h += 16)
            if (mask >> h & 0xffffu) form_again<BF16, VEC, PANEL>(p, first, kvh, n0 + r0 + h, min(16, rows - r0 - h), mask >> h & 0xffffu, vec);
        return;
    }
    int at = low;                                                      // keys up to here are in `had`
    for (; mask; mask &= mask - 1) {
        const long long n = n0 + r0 + __ffs(mask) - 1;
        const int tok = (int)(n / group), head = kvh * group + (int)(n - (long long)tok * group);
        for (; at < first + tok; ++at) note<BF16>(had, load8(v + (size_t)(at + 1) * p.v_stride + 8 * lane, in, vec_kv));
        uint16_t* y = p.out + (size_t)(first + tok) * p.out_stride + (size_t)head * hd + 8 * lane;
        for (int e = 0; e < 8; ++e)
            if (depths >> e & 1) y[e] = f32_to_t<BF16>(had.lost() >> e & 1 ? __uint_as_float(0x7fc00000u) : (had.up >> e & 1 ? kInf : -kInf));
    }
}

// ---- any strides, heads of up to 256 depths: warp-level MMAs ----
constexpr int kPwThreads = 128, kPwRows = 64, kPwKeys = 64;

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t a) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ void ldsm4_trans(uint32_t (&r)[4], uint32_t a) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
// Sequence and piece of a work slot: `slot` counts pieces of 2^log2_len packed (row, head of the group) pairs.  The block's threads together.
__device__ __forceinline__ bool find_piece(const PromptArgs& p, int group, long long slot, int log2_len, int threads, int* first, int* rows, long long* piece) {
    int n = 0;
    for (int s0 = 0; s0 < p.seqs.seqs; s0 += threads) {
        const int s = s0 + (int)threadIdx.x;
        int f = 0;
        const bool at = s < p.seqs.seqs && (seq_rows(p.seqs, s, &f), first_slot((long long)f * group, s, log2_len, 1) <= slot);
        n += __syncthreads_count(at);
    }
    if (n == 0) return false;
    *rows = seq_rows(p.seqs, n - 1, first);
    *piece = slot - first_slot((long long)*first * group, n - 1, log2_len, 1);
    return *piece >= 0 && *piece < pieces((long long)*rows * group, 0, log2_len);
}

template <int BF16, int HD>
__global__ void __launch_bounds__(kPwThreads, HD == 64 ? 4 : (HD == 128 ? 3 : 2)) prompt_mma_kernel(const __grid_constant__ PromptArgs p, int vec_q, int vec_kv) {
    constexpr int LD = HD + 8;
    extern __shared__ __align__(16) uint16_t tile[];
    uint16_t *q_s = tile, *k_s = q_s + kPwRows * LD, *v_s = k_s + kPwKeys * LD;
    const int tid = threadIdx.x, warp = warp_index(), lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int hd = p.head_dim, group = p.heads / p.kv_heads, kvh = blockIdx.y;
    pdl_launch_dependents();
    pdl_wait();
    int first, rows;
    long long piece;
    if (!find_piece(p, group, (long long)(gridDim.x - 1 - blockIdx.x), 6, kPwThreads, &first, &rows, &piece)) return;
    const long long n0 = piece * kPwRows;
    const int nrow = (int)min((long long)kPwRows, (long long)rows * group - n0);
    const int keys = (int)((n0 + nrow - 1) / group) + 1;                                   // of the tile's last row
    for (int it = tid; it < kPwRows * (HD / 8); it += kPwThreads) {
        const int r = it / (HD / 8), d = (it - r * (HD / 8)) * 8;
        const int i = (int)((n0 + r) / group), head = kvh * group + (int)(n0 + r - (long long)i * group);
        const uint4 x = load8(p.q + (size_t)(first + i) * p.q_stride + (size_t)head * hd + d, r < nrow && d < hd, vec_q);
        *reinterpret_cast<uint4*>(q_s + r * LD + d) = x;
    }
    float o[HD / 8][4], m[2] = {-kInf, -kInf}, l[2] = {0.0f, 0.0f};
#pragma unroll
    for (int n = 0; n < HD / 8; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[n][e] = 0.0f;
    int row[2];                                                        // this lane's rows of the sequence
#pragma unroll
    for (int e = 0; e < 2; ++e) row[e] = (int)((n0 + min(16 * warp + g + 8 * e, nrow - 1)) / group);
    for (int key0 = 0; key0 < keys; key0 += kPwKeys) {
        __syncthreads();
        for (int it = tid; it < kPwKeys * (HD / 8); it += kPwThreads) {
            const int r = it / (HD / 8), d = (it - r * (HD / 8)) * 8;
            const bool in = key0 + r < keys && d < hd;
            const size_t j = (size_t)(first + key0 + r);
            *reinterpret_cast<uint4*>(k_s + r * LD + d) = load8(p.k + j * p.k_stride + (size_t)kvh * hd + d, in, vec_kv);
            *reinterpret_cast<uint4*>(v_s + r * LD + d) = load8(p.v + j * p.v_stride + (size_t)kvh * hd + d, in, vec_kv);
        }
        __syncthreads();
        float s[8][4];
#pragma unroll
        for (int n = 0; n < 8; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[n][e] = 0.0f;
#pragma unroll
        for (int k = 0; k < HD / 16; ++k) {
            uint32_t a[4];
            ldsm4(a, smem_u32(q_s + (16 * warp + (lane & 15)) * LD + 16 * k + 8 * (lane >> 4)));
#pragma unroll
            for (int n = 0; n < 8; n += 2) {
                uint32_t b[4];
                ldsm4(b, smem_u32(k_s + (8 * n + (lane & 7) + 8 * (lane >> 4)) * LD + 16 * k + 8 * ((lane >> 3) & 1)));
                mma_t<BF16>(s[n], a, b[0], b[1]);
                mma_t<BF16>(s[n + 1], a, b[2], b[3]);
            }
        }
        float mx[2] = {m[0], m[1]}, alpha[2];
#pragma unroll
        for (int n = 0; n < 8; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const bool on = key0 + 8 * n + 2 * t + (e & 1) <= row[e >> 1];
                s[n][e] = on ? s[n][e] * p.scale_log2e : -kInf;        // (a NaN of the scores stays a NaN)
                mx[e >> 1] = fmaxf(mx[e >> 1], s[n][e]);
            }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], 1));
            mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], 2));
            const float ref = mx[e] == -kInf ? 0.0f : mx[e];
            alpha[e] = ex2(m[e] - ref);
            m[e] = mx[e];
            mx[e] = ref;
            l[e] *= alpha[e];
        }
        uint32_t pa[4][4];
#pragma unroll
        for (int n = 0; n < 8; ++n) {
            float w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                w[e] = ex2(s[n][e] - mx[e >> 1]);
                l[e >> 1] += w[e];
            }
            pa[n / 2][(n & 1) * 2] = pack2_t<BF16>(w[0], w[1]);
            pa[n / 2][(n & 1) * 2 + 1] = pack2_t<BF16>(w[2], w[3]);
        }
#pragma unroll
        for (int n = 0; n < HD / 8; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[n][e] *= alpha[e >> 1];
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
            for (int n = 0; n < HD / 8; n += 2) {
                uint32_t b[4];
                ldsm4_trans(b, smem_u32(v_s + (16 * k + (lane & 15)) * LD + 8 * n + 8 * (lane >> 4)));
                mma_t<BF16>(o[n], pa[k], b[0], b[1]);
                mma_t<BF16>(o[n + 1], pa[k], b[2], b[3]);
            }
    }
    bool bad[2] = {false, false};
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        l[e] += __shfl_xor_sync(0xffffffffu, l[e], 1);
        l[e] += __shfl_xor_sync(0xffffffffu, l[e], 2);
        const int r = 16 * warp + g + 8 * e;
        const long long n = n0 + r;
        const int i = (int)(n / group), head = kvh * group + (int)(n - (long long)i * group);
        const float inv = __fdiv_rn(1.0f, l[e]);
#pragma unroll
        for (int c = 0; c < HD / 8; ++c)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const float x = o[c][2 * e + h] * inv;
                if (r < nrow && 8 * c + 2 * t < hd) {
                    bad[e] = bad[e] || (l[e] > 0.0f && !(fabsf(x) <= 3.402823466e38f));
                    p.out[(size_t)(first + i) * p.out_stride + (size_t)head * hd + 8 * c + 2 * t + h] = f32_to_t<BF16>(x);
                }
            }
    }
    unsigned which = 0;                                                // a bit a row
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        const unsigned mask = __ballot_sync(0xffffffffu, bad[e]);
#pragma unroll
        for (int r = 0; r < 8; ++r) which |= (unsigned)((mask >> (4 * r) & 0xfu) != 0) << (r + 8 * e);
    }
    if (which) mend<BF16, 0, HD == 64 ? 64 : 128>(p, first, kvh, n0, first + keys, 16 * warp, nrow, which, vec_q | vec_kv << 1);
}

// ---- rows on 16-byte boundaries: tcgen05 ----
// Up to 128 depths two query tiles take turns: while one's scores are weighed, the other's products run.  Above, tensor memory holds the result of one tile and
// two blocks of its scores: the next block's are formed while this one's are weighed.
constexpr int kPtThreads = 320;                    // warps 0-3 and 4-7: softmax of the two query tiles, 8: TMA, 9: MMA
constexpr int kPtKeys = 128;
constexpr int kPtChunk = 128 * 128;                // bytes of 128 rows x 64 depths
constexpr int kPtStage = 32 * 128;                 // bytes of 32 rows x 64 results, where a softmax warp's turn from a row a lane to rows side by side
constexpr int kPtMaxSlots = 10;
constexpr uint32_t kPtO = 256;                     // tensor memory: scores / probabilities at columns 0 and 128, results behind them
constexpr float kLazy = 8.0f;                      // a row's reference follows its maximum when that is 2^8 above it

__device__ __forceinline__ uint64_t desc_mn(uint32_t smem_addr) {              // [key][64 depths]: 64 MN elements a row, as the values lie
    uint64_t d = 0;
    d |= (uint64_t)((smem_addr >> 4) & 0x3fffu);
    d |= (uint64_t)(kPtChunk >> 4) << 16;
    d |= (uint64_t)(1024 >> 4) << 32;
    d |= (uint64_t)1 << 46;
    d |= (uint64_t)2 << 61;
    return d;
}
__device__ __forceinline__ void tma_3d(void* dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
                 ::"r"(smem_u32(dst)), "l"(map), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void tma_4d(void* dst, const CUtensorMap* map, int x, int y, int z, int w, uint64_t* bar) {
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
                 ::"r"(smem_u32(dst)), "l"(map), "r"(x), "r"(y), "r"(z), "r"(w), "r"(smem_u32(bar)) : "memory");
}
// From shared memory; the thread that issues it commits and waits.
__device__ __forceinline__ void tma_store_4d(const CUtensorMap* map, int x, int y, int z, int w, uint32_t src) {
    asm volatile("cp.async.bulk.tensor.4d.global.shared::cta.bulk_group [%0, {%1, %2, %3, %4}], [%5];\n\tcp.async.bulk.commit_group;"
                 ::"l"(map), "r"(x), "r"(y), "r"(z), "r"(w), "r"(src) : "memory");
}
template <int LEFT>
__device__ __forceinline__ void bulk_wait_read() { asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(LEFT) : "memory"); }
__device__ __forceinline__ void bulk_wait_all() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
__device__ __forceinline__ uint64_t pack64(float x, float y) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
    return r;
}
__device__ __forceinline__ void unpack64(uint64_t v, float& x, float& y) { asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(v)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

// The last items of a CTA: it takes no more once a softmax warp has met rows to mend.  When one warp has done item f, the slowest is at f - 2 (a place of two is free again when
// all have read it) and the loads at f + 3 at most (that CTA may have been asked for).
constexpr int kPtKept = 8;

struct PromptTc {
    CUtensorMap q, k, v, out;
    PromptArgs p;
    int tokens;                                    // of a query tile: 128 / heads of a group
    int slots;                                     // K / V ring
    long long pieces;                              // work slots of a KV head
};
// A work item: rows tok0 .. of a sequence, two query tiles of them, for one KV head.
struct PromptItem {
    int first, rows, tok0, kvh;                    // the sequence; rows below zero: there is no more
};

// The grid has a CTA for every work slot, and a CTA that has finished its own takes over the next one that has not been launched: the barriers and the
// tensor memory are set up once, and the next item's queries and keys are on their way while this one's last blocks are weighed and its results stored.  (A CTA for every
// item alone, timed in turn with this: 8192 rows 532 us against 490, eleven prompts of 7001 88.7 against 63.9.)
__device__ __forceinline__ void take_next_cta(uint32_t answer, uint64_t* bar) {
    asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(answer), "r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ int taken_cta(uint32_t answer) {        // its index, -1: all have been launched or taken
    uint32_t ok, x;
    asm volatile(
        "{\n\t.reg .b128 h;\n\t.reg .pred p;\n\t"
        "ld.shared.b128 h, [%2];\n\t"
        "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, h;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t"
        "mov.u32 %1, 0;\n\t"
        "@p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %1, h;\n\t}"
        : "=r"(ok), "=r"(x) : "r"(answer) : "memory");
    return ok ? (int)x : -1;
}

// The rows of this warp that are left, by item: mend() for each.
template <int BF16, int NCH>
__device__ __forceinline__ void mend_items(const PromptTc& a, const PromptItem* items, const unsigned (*odd)[kPtKept]) {
    const int warp = threadIdx.x >> 5, tt = a.tokens, group = a.p.heads / a.p.kv_heads;
#pragma unroll 1
    for (int k = 0; k < kPtKept; ++k) {
        const unsigned mask = odd[warp][k];
        if (!mask) continue;
        const PromptItem w = items[k];
        const int low = w.tok0 + (warp >> 2) * tt, ntok = min(tt, w.rows - low), n = (low + ntok - 1) / kPtKeys + 1;
        mend<BF16, 1, NCH == 1 ? 64 : 128>(a.p, w.first, w.kvh, (long long)low * group, min(w.first + n * kPtKeys, a.p.rows), (warp & 3) * 32, ntok * group, mask, 3);
    }
}
template <int BF16>
__device__ __noinline__ void mend_items_1(const PromptTc& a, const PromptItem* items, const unsigned (*odd)[kPtKept]) { mend_items<BF16, 1>(a, items, odd); }
// BULK: a softmax warp's 32 rows are whole tokens, out lies on 16-byte boundaries, and full warps' results leave by bulk stores from the warp's stage.
template <int BF16, int NCH, int BULK>
__global__ void __launch_bounds__(kPtThreads, 1) prompt_tc_kernel(const __grid_constant__ PromptTc a) {
    constexpr int kTile = NCH * kPtChunk, kTiles = NCH <= 2 ? 2 : 1;
    const PromptArgs& p = a.p;
    extern __shared__ unsigned char smem_dyn[];
    unsigned char* smem = smem_dyn + ((1024u - (smem_u32(smem_dyn) & 1023u)) & 1023u);
    __shared__ __align__(16) uint4 answer;
    __shared__ __align__(8) uint64_t bars[2 * kPtMaxSlots + 15];
    __shared__ PromptItem items[2], kept[kPtKept];
    __shared__ unsigned odd[8][kPtKept];                           // of a softmax warp's rows of an item, those with results that are not finite
    __shared__ int odd_any;
    __shared__ uint32_t tmem_slot;
    __shared__ int abort_word;
    volatile int* abort_flag = &abort_word;
    uint64_t *full = bars, *empty = full + kPtMaxSlots, *q_full = empty + kPtMaxSlots, *q_empty = q_full + 1, *s_full = q_empty + 1, *p_full = s_full + 2, *o_done = p_full + 2,
             *item_full = o_done + 2, *item_empty = item_full + 2, *taken = item_empty + 2, *p_half = taken + 1;
    const int tid = threadIdx.x, warp = warp_index(), lane = tid & 31;
    const int hd = p.head_dim, hd16 = (hd + 15) & ~15, group = p.heads / p.kv_heads, tt = a.tokens;
    unsigned char *q_s = smem, *out_s = smem + kTiles * kTile, *ring = out_s + kTiles * 4 * kPtStage;

    if (tid < 8 * kPtKept) odd[tid / kPtKept][tid % kPtKept] = 0;
    if (tid == 0) {
        abort_word = 0;
        odd_any = 0;
        for (int i = 0; i < a.slots; ++i) { mbar_init(&full[i], 1); mbar_init(&empty[i], 1); }
        mbar_init(q_full, 1);
        mbar_init(q_empty, 1);
        mbar_init(taken, 1);
        for (int i = 0; i < 2; ++i) {
            mbar_init(&s_full[i], 1); mbar_init(&p_half[i], 4); mbar_init(&p_full[i], 4); mbar_init(&o_done[i], 1);
            mbar_init(&item_full[i], 1); mbar_init(&item_empty[i], 9);
        }
        fence_barrier_init();
    }
    pdl_wait();                                                    // (before the allocation: the kernel ahead may still hold tensor memory)
    if (warp == 9) {
        tmem_alloc(&tmem_slot, 512);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    pdl_launch_dependents();
    const uint32_t tmem = tmem_slot;

    // Item `it` of this CTA, for the warps that work on it: its place is free again once all of them have read it.
    auto next_item = [&](int it, PromptItem& w) {
        const int k = it & 1;
        if (!__all_sync(0xffffffffu, mbar_wait(&item_full[k], (it >> 1) & 1, abort_flag, p.status))) return false;
        w = items[k];
        __syncwarp();
        if (lane == 0) mbar_arrive(&item_empty[k]);
        return w.rows >= 0;
    };
    auto tokens_of = [&](const PromptItem& w, int x) { return kTiles == 1 && x ? 0 : max(0, min(tt, w.rows - w.tok0 - x * tt)); };
    auto blocks_of = [&](const PromptItem& w, int x) {
        const int n = tokens_of(w, x);
        return n ? (w.tok0 + x * tt + n - 1) / kPtKeys + 1 : 0;
    };

    if (warp == 8) {                                               // ---- items and loads ----
        int cta = blockIdx.x, slot = 0, round = 0, it = 0, asked = 0;
        bool ok = true;
        auto load = [&](const CUtensorMap* map, const PromptItem& w, int j) {
            if (round && !__all_sync(0xffffffffu, mbar_wait(&empty[slot], (round - 1) & 1, abort_flag, p.status))) return false;
            if (elect_one()) {
                mbar_expect_tx(&full[slot], kTile);
                for (int c = 0; c < NCH; ++c) tma_3d(ring + (size_t)slot * kTile + c * kPtChunk, map, c * 64, w.kvh, w.first + j * kPtKeys, &full[slot]);
            }
            __syncwarp();
            if (++slot == a.slots) { slot = 0; ++round; }
            return true;
        };
        while (ok) {
            // the slot's sequence and piece; the pieces with the most keys first
            PromptItem w = {0, -1, 0, 0};
            if (cta >= 0) {
                const int q = cta / p.kv_heads;
                const long long slot_id = a.pieces - 1 - q;
                w.kvh = cta - q * p.kv_heads;
                int n = 0;
                for (int s0 = 0; s0 < p.seqs.seqs; s0 += 32) {
                    const int s = s0 + lane;
                    int f = 0;
                    n += __popc(__ballot_sync(0xffffffffu, s < p.seqs.seqs && (seq_rows(p.seqs, s, &f), first_slot_of(f, s, kTiles * tt) <= slot_id)));
                }
                if (n > 0) {
                    const int rows = seq_rows(p.seqs, n - 1, &w.first);
                    const long long piece = slot_id - first_slot_of(w.first, n - 1, kTiles * tt);
                    if (piece >= 0 && piece < pieces_of(rows, kTiles * tt)) {
                        w.rows = rows;
                        w.tok0 = (int)(piece * kTiles * tt);
                    }
                }
            }
            if (cta < 0 || w.rows > 0) {                           // (a slot may be nobody's)
                const int k = it & 1;
                if (it >= 2) ok = __all_sync(0xffffffffu, mbar_wait(&item_empty[k], ((it >> 1) - 1) & 1, abort_flag, p.status));
                if (!ok) break;
                if (lane == 0) {
                    items[k] = w;
                    kept[it % kPtKept] = w;
                    mbar_arrive(&item_full[k]);
                }
                __syncwarp();
                if (cta < 0) break;
                if (it > 0) ok = __all_sync(0xffffffffu, mbar_wait(q_empty, (it - 1) & 1, abort_flag, p.status));
                if (!ok) break;
                ++it;
                const int tiles = tokens_of(w, 1) ? 2 : 1, n = max(blocks_of(w, 0), blocks_of(w, 1));
                if (elect_one()) {
                    mbar_expect_tx(q_full, tiles * NCH * tt * group * 128);
                    for (int x = 0; x < tiles; ++x)
                        for (int c = 0; c < NCH; ++c) tma_4d(q_s + x * kTile + c * kPtChunk, &a.q, c * 64, 0, w.kvh, w.first + w.tok0 + x * tt, q_full);
                }
                __syncwarp();
                if (kTiles == 2) {
                    for (int j = 0; ok && j < n; ++j) ok = load(&a.k, w, j) && load(&a.v, w, j);
                } else {
                    ok = load(&a.k, w, 0);
                    for (int j = 0; ok && j < n; ++j) ok = (j + 1 == n || load(&a.k, w, j + 1)) && load(&a.v, w, j);
                }
                if (!ok) break;
            }
            if (__any_sync(0xffffffffu, *const_cast<volatile int*>(&odd_any))) {
                cta = -1;                                          // (rows to mend: the slots that are left get CTAs of their own)
                continue;
            }
            if (elect_one()) {
                fence_proxy_async();                               // (the last answer has been read)
                mbar_expect_tx(taken, 16);
                take_next_cta(smem_u32(&answer), taken);
            }
            __syncwarp();
            ok = __all_sync(0xffffffffu, mbar_wait(taken, asked & 1, abort_flag, p.status));
            ++asked;
            cta = taken_cta(smem_u32(&answer));
            __syncwarp();
        }
    } else if (warp == 9) {                                        // ---- products: one lane, so that nothing but the waits stands between them ----
        if (elect_one()) {
            const uint32_t idesc_s = umma_idesc(BF16, 128, kPtKeys), idesc_o = umma_idesc(BF16, 128, hd16) | (1u << 16);
            const int ksteps = hd16 >> 4;
            const uint64_t q_d = umma_desc_sw128(smem_u32(q_s)), k_d = umma_desc_sw128(smem_u32(ring)), v_d = desc_mn(smem_u32(ring));   // (an address is its low 14 bits, in 16 bytes)
            int slot = 0, par = 0, done[2] = {0, 0};               // blocks of the two tiles so far
            bool ok = true;
            auto take = [&]() {                                    // the next slot of the ring, filled
                const int at = slot;
                ok = ok && mbar_wait(&full[at], par, abort_flag, p.status);
                if (++slot == a.slots) { slot = 0; par ^= 1; }
                return at;
            };
            auto scores = [&](int x, int buf, int at) {            // of query tile x, into the columns of buffer buf
                const uint64_t q0 = q_d + x * (kTile >> 4), k0 = k_d + at * (kTile >> 4);
                tc_fence_after();
#pragma unroll
                for (int s = 0; s < 4 * NCH; ++s)
                    if (s < ksteps) umma_f16(tmem + 128 * buf, q0 + ((s >> 2) * kPtChunk + (s & 3) * 32) / 16, k0 + ((s >> 2) * kPtChunk + (s & 3) * 32) / 16, idesc_s, s > 0);
                umma_commit(&s_full[buf]);
            };
            // Probabilities of buffer buf times the values, half of the keys at a time: the first half's product runs while the second half is weighed
            auto values = [&](int x, int buf, int at, int half, bool first) {
                const uint64_t v0 = v_d + at * (kTile >> 4);
                tc_fence_after();
#pragma unroll
                for (int i = 0; i < kPtKeys / 32; ++i) {
                    const int s = half * (kPtKeys / 32) + i;
                    umma_f16_ts(tmem + kPtO + 128 * x, tmem + 128 * buf + 8 * s, v0 + s * 128, idesc_o, !first || s > 0);
                }
            };
            for (int it = 0; ok; ++it) {
                ok = mbar_wait(&item_full[it & 1], (it >> 1) & 1, abort_flag, p.status);
                if (!ok) break;
                const PromptItem w = items[it & 1];
                mbar_arrive(&item_empty[it & 1]);
                if (w.rows < 0) break;
                const int nblk[2] = {blocks_of(w, 0), blocks_of(w, 1)}, nmax = max(nblk[0], nblk[1]);
                ok = mbar_wait(q_full, it & 1, abort_flag, p.status);
                int k_at = take(), v_at;
                if (!ok) break;
                scores(0, kTiles == 2 ? 0 : done[0] & 1, k_at);
                if (nblk[1]) scores(1, 1, k_at);
                umma_commit(&empty[k_at]);
                if (nmax == 1) umma_commit(q_empty);
                if (kTiles == 1)
                    for (int j = 0; j < nmax; ++j) {
                        const int buf = done[0] & 1;
                        if (j + 1 < nmax) {
                            k_at = take();
                            if (!ok) break;
                            scores(0, buf ^ 1, k_at);              // (behind the product that read this buffer's probabilities)
                            umma_commit(&empty[k_at]);
                            if (j + 2 == nmax) umma_commit(q_empty);
                        }
                        v_at = take();
                        ok = ok && mbar_wait_poll(&p_half[buf], (done[0] >> 1) & 1, abort_flag, p.status, STATUS_TMEM_TIMEOUT);
                        if (!ok) break;
                        values(0, buf, v_at, 0, j == 0);
                        ok = mbar_wait_poll(&p_full[buf], (done[0] >> 1) & 1, abort_flag, p.status, STATUS_TMEM_TIMEOUT);
                        if (!ok) break;
                        values(0, buf, v_at, 1, false);
                        ++done[0];
                        umma_commit(&empty[v_at]);
                        umma_commit(&o_done[0]);
                    }
                for (int j = 0; kTiles == 2 && ok && j < nmax; ++j) {
                    const bool more = j + 1 < nmax;
                    v_at = take();
                    if (more) k_at = take();
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        if (!ok || j >= nblk[x]) continue;
                        ok = mbar_wait_poll(&p_half[x], done[x] & 1, abort_flag, p.status, STATUS_TMEM_TIMEOUT);
                        if (!ok) break;
                        values(x, x, v_at, 0, j == 0);
                        ok = mbar_wait_poll(&p_full[x], done[x] & 1, abort_flag, p.status, STATUS_TMEM_TIMEOUT);
                        if (!ok) break;
                        values(x, x, v_at, 1, false);
                        ++done[x];
                        if (j + 1 == nblk[x]) umma_commit(&o_done[x]);
                        else scores(x, x, k_at);
                    }
                    if (!ok) break;
                    umma_commit(&empty[v_at]);
                    if (more) umma_commit(&empty[k_at]);
                    if (j + 2 == nmax) umma_commit(q_empty);       // (the last scores have been formed)
                }
            }
        }
        __syncwarp();
    } else {                                                       // ---- softmax ----
        const int x = warp >> 2, row = (warp & 3) * 32 + lane;
        const int t = row / group, g = row - t * group;
        const uint32_t ts0 = tmem + ((uint32_t)((warp & 3) * 32) << 16) + 128 * x, to = ts0 + kPtO;
        const float sc = p.scale_log2e;
        int done = 0, tiles = 0;                                   // blocks and tiles so far
        bool ok = true;
        PromptItem w;
        for (int it = 0; ok && next_item(it, w); ++it) {
            const int ntok = tokens_of(w, x), n = blocks_of(w, x), low = w.tok0 + x * tt;      // low: the tile's first row
            const int tok = low + min(t, max(ntok, 1) - 1), head = w.kvh * group + g;
            const bool in = t < ntok;
            float m = -kInf, l = 0.0f;
            for (int j = 0; j < n; ++j, ++done) {
                // (one tile: the buffers take turns, the blocks before are done with where o_done says so)
                const int buf = kTiles == 2 ? x : done & 1;
                const uint32_t ts = kTiles == 2 ? ts0 : ts0 + 128 * buf;
                ok = __all_sync(0xffffffffu, mbar_wait_poll(&s_full[buf], (kTiles == 2 ? done : done >> 1) & 1, abort_flag, p.status, STATUS_TMEM_TIMEOUT));
                if (!ok) break;
                tc_fence_after();
                uint32_t s[4][32];
#pragma unroll
                for (int c = 0; c < 4; ++c) tmem_ld32(ts + 32 * c, s[c]);
                tmem_ld_wait();
                const int key0 = j * kPtKeys;
                if (key0 + kPtKeys - 1 > low) {                    // keys behind some row's own
                    const int lim = tok - key0;
#pragma unroll
                    for (int c = 0; c < 4; ++c)
#pragma unroll
                        for (int i = 0; i < 32; ++i) s[c][i] = 32 * c + i <= lim ? s[c][i] : 0xff800000u;
                }
                float mx[4] = {m, m, m, m};
#pragma unroll
                for (int c = 0; c < 4; ++c)
#pragma unroll
                    for (int i = 0; i < 32; i += 2) mx[c] = max3(mx[c], __uint_as_float(s[c][i]), __uint_as_float(s[c][i + 1]));
                const float now = fmaxf(max3(mx[0], mx[1], mx[2]), mx[3]);
                const bool far = (now - m) * sc > kLazy;           // (from -inf: inf; -inf to -inf: NaN, no)
                if (j == 0) {
                    m = now;
                } else if (__any_sync(0xffffffffu, far)) {
                    if (kTiles == 1) {                             // (with two tiles the product before was done with when these scores were)
                        ok = __all_sync(0xffffffffu, mbar_wait_poll(&o_done[0], (done - 1) & 1, abort_flag, p.status, STATUS_TMEM_TIMEOUT));
                        if (!ok) break;
                        tc_fence_after();
                    }
                    const float f = far ? ex2((m - now) * sc) : 1.0f;
                    if (far) m = now;
                    l *= f;
                    const uint64_t f2 = pack64(f, f);
                    for (int c = 0; c < hd16; c += 16) {
                        uint32_t o[16];
                        tmem_ld16(to + c, o);
                        tmem_ld_wait();
#pragma unroll
                        for (int i = 0; i < 16; i += 2) {
                            float u, v;
                            unpack64(mul2(pack64(__uint_as_float(o[i]), __uint_as_float(o[i + 1])), f2), u, v);
                            o[i] = __float_as_uint(u);
                            o[i + 1] = __float_as_uint(v);
                        }
                        tmem_st16(to + c, o);
                    }
                }
                const float ref = m == -kInf ? 0.0f : m * sc;
                const uint64_t sc2 = pack64(sc, sc), ref2 = pack64(-ref, -ref);
                uint64_t sum[2] = {0, 0};
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    uint32_t e[16];
#pragma unroll
                    for (int i = 0; i < 32; i += 2) {
                        const uint64_t y = fma2(pack64(__uint_as_float(s[c][i]), __uint_as_float(s[c][i + 1])), sc2, ref2);
                        float u, v;
                        unpack64(y, u, v);
                        u = ex2(u);
                        v = ex2(v);
                        sum[(i >> 1) & 1] = add2(sum[(i >> 1) & 1], pack64(u, v));
                        e[i / 2] = pack2_t<BF16>(u, v);
                    }
                    tmem_st16(ts + 16 * c, e);
                    if (c & 1) {
                        tmem_st_wait();
                        tc_fence_before();
                        // One tile: every phase of o_done in its turn, the last one while the next cannot be over without this warp.  (These scores were formed before the product
                        // before: without the wait a warp that is ahead of the others could take the parity of an earlier phase for that of its last one, and a result
                        // leave before its products are done.)
                        if (kTiles == 1 && c == 3 && done > 0) ok = __all_sync(0xffffffffu, mbar_wait_poll(&o_done[0], (done - 1) & 1, abort_flag, p.status, STATUS_TMEM_TIMEOUT));
                        __syncwarp();
                        if (lane == 0) mbar_arrive(c == 1 ? &p_half[buf] : &p_full[buf]);
                    }
                }
                float u, v;
                unpack64(add2(sum[0], sum[1]), u, v);
                l += u + v;
                if (kTiles == 1 && !ok) break;
            }
            if (!ok || n == 0) continue;
            ok = __all_sync(0xffffffffu, mbar_wait(&o_done[x], (kTiles == 2 ? tiles : done - 1) & 1, abort_flag, p.status, STATUS_TMEM_TIMEOUT));
            ++tiles;
            if (!ok) break;
            tc_fence_after();
            const float inv = __fdiv_rn(1.0f, l);
            const uint64_t inv2 = pack64(inv, inv);
            const bool vec = (((uintptr_t)p.out | (p.out_stride * 2)) & 15) == 0;
            const long long at = (long long)(w.first + tok) * (long long)p.out_stride + (long long)head * hd;
            const unsigned rows_in = __ballot_sync(0xffffffffu, in);
            const uint32_t mine = smem_u32(out_s) + warp * kPtStage;
            uint64_t zero = 0;                                     // 0 * every result: not a number where one of them is not finite
            const bool bulk = BULK && rows_in == 0xffffffffu;
            if (bulk) {
                const int tok_w = w.first + low + (warp & 3) * 32 / group;
                for (int c0 = 0; c0 < hd; c0 += 64) {
                    uint32_t o[2][32], e[32];
                    tmem_ld32(to + c0, o[0]);
                    tmem_ld32(to + c0 + 32, o[1]);
                    tmem_ld_wait();
#pragma unroll
                    for (int i = 0; i < 32; ++i) {
                        const uint64_t y = mul2(pack64(__uint_as_float(o[i / 16][2 * (i % 16)]), __uint_as_float(o[i / 16][2 * (i % 16) + 1])), inv2);
                        if (c0 + 2 * i < hd) zero = fma2(y, 0, zero);
                        float u, v;
                        unpack64(y, u, v);
                        e[i] = pack2_t<BF16>(u, v);
                    }
                    if (lane == 0) bulk_wait_read<0>();            // (the last store has read the stage)
                    __syncwarp();
#pragma unroll
                    for (int c = 0; c < 8; ++c)
                        asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(mine + lane * 128 + ((c ^ (lane & 7)) << 4)), "r"(e[4 * c]), "r"(e[4 * c + 1]), "r"(e[4 * c + 2]), "r"(e[4 * c + 3]) : "memory");
                    fence_proxy_async();
                    __syncwarp();
                    if (lane == 0) tma_store_4d(&a.out, c0, 0, w.kvh, tok_w, mine);
                }
            } else if (BULK && lane == 0) {
                bulk_wait_read<0>();
            }
            if (BULK) __syncwarp();
            for (int c0 = bulk ? hd : 0; c0 < hd; c0 += 64) {
                uint32_t o[2][32];
                tmem_ld32(to + c0, o[0]);                          // (what lies behind the head's depths is not used)
                tmem_ld32(to + c0 + 32, o[1]);
                tmem_ld_wait();
                __syncwarp();                                      // (the stage's last reader is through)
#pragma unroll
                for (int c = 0; c < 8; ++c) {
                    uint32_t e[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const uint64_t y = mul2(pack64(__uint_as_float(o[c / 4][8 * (c % 4) + 2 * i]), __uint_as_float(o[c / 4][8 * (c % 4) + 2 * i + 1])), inv2);
                        if (c0 + 8 * c < hd) zero = fma2(y, 0, zero);
                        float u, v;
                        unpack64(y, u, v);
                        e[i] = pack2_t<BF16>(u, v);
                    }
                    asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(mine + lane * 128 + ((c ^ (lane & 7)) << 4)), "r"(e[0]), "r"(e[1]), "r"(e[2]), "r"(e[3]) : "memory");
                }
                __syncwarp();
                const int c = c0 + 8 * (lane & 7);
#pragma unroll
                for (int i = 0; i < 8; ++i) {                      // four rows of 128 bytes at a time
                    const int r = 4 * i + (lane >> 3);
                    uint4 e;
                    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(e.x), "=r"(e.y), "=r"(e.z), "=r"(e.w) : "r"(mine + r * 128 + (((lane & 7) ^ (r & 7)) << 4)) : "memory");
                    const long long to_row = __shfl_sync(0xffffffffu, at, r);
                    if (!(rows_in >> r & 1) || c >= hd) continue;
                    uint16_t* dst = p.out + to_row + c;
                    if (vec) {
                        *reinterpret_cast<uint4*>(dst) = e;
                    } else {
                        const uint32_t x4[4] = {e.x, e.y, e.z, e.w};
#pragma unroll
                        for (int k = 0; k < 8; ++k) dst[k] = (uint16_t)(x4[k / 2] >> (16 * (k & 1)));
                    }
                }
            }
            float z0, z1;
            unpack64(zero, z0, z1);
            const bool bad = !(z0 + z1 == 0.0f);
            const unsigned mask = __ballot_sync(0xffffffffu, bad && l > 0.0f) & rows_in;
            if (mask) {
                odd[warp][it % kPtKept] = mask;
                *const_cast<volatile int*>(&odd_any) = 1;
            }
        }
        if (BULK) {
            if (lane == 0) bulk_wait_all();                        // (stored, not only read: the grid that waits for this one finds the results)
            __syncwarp();
        }
        tc_fence_before();
    }
    __syncthreads();
    if (warp == 9) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
    // Rows to mend, once nobody waits for this CTA.  (A call within the softmax loop costs its registers there, whatever is behind it: 7001 rows 65.7 us and 71.5, 8192 rows 494 and 521.  Here,
    // inline, 64.1 and 489; heads of 64 are better off with a call, 200 rows 8.5 and 8.7.)
    if (odd_any && warp_index() < 8) {
        if (NCH == 1) mend_items_1<BF16>(a, kept, odd);
        else mend_items<BF16, NCH>(a, kept, odd);
    }
}

template <int BF16, int NCH, int BULK>
cudaError_t tc_launch(const PromptArgs& p, cudaStream_t stream, bool* taken) {
    constexpr int kTiles = NCH <= 2 ? 2 : 1;
    *taken = false;
    TensorMapEncodeFn enc = tensor_map_encoder();
    const int group = p.heads / p.kv_heads;
    if (!enc || group > 128) return cudaSuccess;
    PromptTc a;
    memset(&a, 0, sizeof(a));
    a.p = p;
    a.tokens = 128 / group;
    a.slots = (int)((227 * 1024 - 2048 - kTiles * (NCH * kPtChunk + 4 * kPtStage)) / (NCH * kPtChunk));
    if (a.slots > kPtMaxSlots) a.slots = kPtMaxSlots;
    a.pieces = p.rows / (kTiles * a.tokens) + (long long)p.seqs.seqs;
    if (a.pieces * p.kv_heads > 0x7fffffffll) return cudaErrorInvalidValue;
    const CUtensorMapDataType type = BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    const cuuint64_t hd = (cuuint64_t)p.head_dim;
    const cuuint64_t qd[4] = {hd, (cuuint64_t)group, (cuuint64_t)p.kv_heads, (cuuint64_t)p.rows}, qs[3] = {hd * 2, hd * 2 * group, (cuuint64_t)p.q_stride * 2};
    const cuuint32_t qb[4] = {64, (cuuint32_t)group, 1, (cuuint32_t)a.tokens}, ones[4] = {1, 1, 1, 1};
    if (enc(&a.q, type, 4, (void*)p.q, qd, qs, qb, ones, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS) return cudaSuccess;
    const cuuint64_t kd[3] = {hd, (cuuint64_t)p.kv_heads, (cuuint64_t)p.rows}, ks[2] = {hd * 2, (cuuint64_t)p.k_stride * 2}, vs[2] = {hd * 2, (cuuint64_t)p.v_stride * 2};
    const cuuint32_t kb[3] = {64, 1, (cuuint32_t)kPtKeys};
    if (enc(&a.k, type, 3, (void*)p.k, kd, ks, kb, ones, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS ||
        enc(&a.v, type, 3, (void*)p.v, kd, vs, kb, ones, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
        return cudaSuccess;
    // (us without and with bulk stores, heads of 128: eleven prompts of 7001 rows 83 and 78, four of 1024 47 and 44; nine of 300 rows of 256 31 and 26.  Heads of 64, one chunk
    // a row: 60 prompts of 100 rows 18.9 and 20.5.)
    if (BULK) {
        const cuuint64_t os[3] = {hd * 2, hd * 2 * group, (cuuint64_t)p.out_stride * 2};
        const cuuint32_t ob[4] = {64, (cuuint32_t)group, 1, (cuuint32_t)(32 / group)};
        if (enc(&a.out, type, 4, (void*)p.out, qd, os, ob, ones, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_NONE,
                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS) return cudaSuccess;
    }
    auto kern = prompt_tc_kernel<BF16, NCH, BULK>;
    const size_t smem = 1024 + (size_t)(kTiles + a.slots) * NCH * kPtChunk + kTiles * 4 * kPtStage;
    static std::atomic<int> attr_dev{-1};          // the opt-in is per device
    int dev = 0;
    cudaGetDevice(&dev);
    if (attr_dev.load() != dev) {
        const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) return e;
        attr_dev.store(dev);
    }
    *taken = true;
    return launch_pdl(kern, dim3((unsigned)(a.pieces * p.kv_heads)), dim3(kPtThreads), smem, stream, a);
}

template <int BF16, int HD>
cudaError_t mma_launch(const PromptArgs& a, cudaStream_t stream) {
    auto kern = prompt_mma_kernel<BF16, HD>;
    const size_t smem = (size_t)(kPwRows + 2 * kPwKeys) * (HD + 8) * 2;
    static std::atomic<int> attr_dev{-1};          // the opt-in is per device
    int dev = 0;
    cudaGetDevice(&dev);
    if (attr_dev.load() != dev) {
        const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) return e;
        attr_dev.store(dev);
    }
    const long long slots = ((long long)a.rows * (a.heads / a.kv_heads) >> 6) + a.seqs.seqs;
    if (slots > 0x7fffffffll || a.kv_heads > 65535) return cudaErrorInvalidValue;
    const int vec_q = a.q_stride % 8 == 0 && ((uintptr_t)a.q & 15) == 0;
    const int vec_kv = a.k_stride % 8 == 0 && a.v_stride % 8 == 0 && (((uintptr_t)a.k | (uintptr_t)a.v) & 15) == 0;
    return launch_pdl(kern, dim3((unsigned)slots, (unsigned)a.kv_heads), dim3(kPwThreads), smem, stream, a, vec_q, vec_kv);
}

}  // namespace

cudaError_t prompt_launch(PromptArgs a, int sm_count, cudaStream_t stream) {
    if (a.rows == 0 || a.seqs.seqs == 0) return cudaSuccess;
    // rows and heads on 16-byte boundaries (what a tensor map needs), strides that it can hold, a positive scale (the maximum is taken before it)
    const bool aligned = ((a.q_stride | a.k_stride | a.v_stride) & 7) == 0 && (((uintptr_t)a.q | (uintptr_t)a.k | (uintptr_t)a.v) & 15) == 0 &&
                         ((a.q_stride | a.k_stride | a.v_stride) >> 38) == 0;
    if (aligned && a.scale_log2e > 0.0f && a.scale_log2e < 1e30f) {
        bool taken = false;
        typedef cudaError_t (*Launch)(const PromptArgs&, cudaStream_t, bool*);
        static const Launch launches[2][2][4] = {{{tc_launch<0, 1, 0>, tc_launch<0, 2, 0>, tc_launch<0, 3, 0>, tc_launch<0, 4, 0>},
                                                  {tc_launch<1, 1, 0>, tc_launch<1, 2, 0>, tc_launch<1, 3, 0>, tc_launch<1, 4, 0>}},
                                                 {{tc_launch<0, 1, 0>, tc_launch<0, 2, 1>, tc_launch<0, 3, 1>, tc_launch<0, 4, 1>},
                                                  {tc_launch<1, 1, 0>, tc_launch<1, 2, 1>, tc_launch<1, 3, 1>, tc_launch<1, 4, 1>}}};
        const bool bulk = 32 % (a.heads / a.kv_heads) == 0 && (((uintptr_t)a.out | (a.out_stride * 2)) & 15) == 0 && a.out_stride >> 38 == 0;
        const cudaError_t e = launches[bulk][a.bf16 ? 1 : 0][(a.head_dim + 63) / 64 - 1](a, stream, &taken);
        if (taken || e != cudaSuccess) return e;
    }
    if (a.bf16) return a.head_dim <= 64 ? mma_launch<1, 64>(a, stream) : (a.head_dim <= 128 ? mma_launch<1, 128>(a, stream) : mma_launch<1, 256>(a, stream));
    return a.head_dim <= 64 ? mma_launch<0, 64>(a, stream) : (a.head_dim <= 128 ? mma_launch<0, 128>(a, stream) : mma_launch<0, 256>(a, stream));
}

}  // namespace smeg
