// Causal attention over whole packed prompts, grouped heads (sm_100a): row i of a sequence attends to the sequence's rows 0 .. i.
//
//   out = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale * q . k_j - max), j <= i
// One pass over the keys with the running maximum and sum; sums are 32 bits wide, the probabilities are rounded to the inputs' type for the second
// product.  The query rows of one KV head -- every row times every head of the group -- are the rows of a tile, so that grouped heads share one
// read of the keys and values.
#include "common.cuh"
#include "kernels.h"
#include "paged.h"

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
// infinity or NaN there makes NaNs (0 * inf).  So a row whose result is not finite although its probabilities are is formed again, key by key over
// what it attends to, where the blocks that it shares with later rows hold such a value.

// Whether any value of keys [from, to) of a KV head is an infinity or NaN.  A warp.
__device__ __noinline__ bool any_bad_value(const PromptArgs& p, int kvh, int from, int to) {
    const unsigned expo = p.bf16 ? 0x7f80u : 0x7c00u;
    bool bad = false;
    for (int j = from; j < to; ++j) {
        const uint16_t* v = p.v + (size_t)j * p.v_stride + (size_t)kvh * p.head_dim;
        for (int d = threadIdx.x & 31; d < p.head_dim; d += 32) bad = bad || (v[d] & expo) == expo;
    }
    return __any_sync(0xffffffffu, bad);
}
// Row `row` (of the packed batch) of query head `head` over keys [first, row].  A warp; a lane has eight depths.
template <int BF16>
__device__ __noinline__ void exact_row(const PromptArgs& p, int first, int row, int head) {
    const int lane = threadIdx.x & 31, d = lane * 8, hd = p.head_dim, kvh = head / (p.heads / p.kv_heads);
    const bool in = d < hd;
    float q[8], acc[8], m = -kInf, l = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        q[e] = in ? t_to_f32<BF16>(p.q[(size_t)row * p.q_stride + (size_t)head * hd + d + e]) : 0.0f;
        acc[e] = 0.0f;
    }
    for (int j = first; j <= row; ++j) {
        const uint16_t *k = p.k + (size_t)j * p.k_stride + (size_t)kvh * hd + d, *v = p.v + (size_t)j * p.v_stride + (size_t)kvh * hd + d;
        float s = 0.0f;
        if (in)
#pragma unroll
            for (int e = 0; e < 8; ++e) s = fmaf(q[e], t_to_f32<BF16>(k[e]), s);
#pragma unroll
        for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        s *= p.scale_log2e;
        const float now = fmaxf(m, s), ref = now == -kInf ? 0.0f : now, a = ex2(m - ref), w = ex2(s - ref);
        m = now;
        l = fmaf(l, a, w);
        if (in)
#pragma unroll
            for (int e = 0; e < 8; ++e) acc[e] = fmaf(w, t_to_f32<BF16>(v[e]), acc[e] * a);
    }
    if (in)
#pragma unroll
        for (int e = 0; e < 8; ++e) p.out[(size_t)row * p.out_stride + (size_t)head * hd + d + e] = f32_to_t<BF16>(__fdiv_rn(acc[e], l));
}

// ---- any strides, heads of up to 256 depths: warp-level MMAs ----
constexpr int kPwThreads = 128, kPwRows = 64, kPwKeys = 64;

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
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t a) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ void ldsm4_trans(uint32_t (&r)[4], uint32_t a) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
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
__global__ void __launch_bounds__(kPwThreads) prompt_mma_kernel(const __grid_constant__ PromptArgs p, int vec_q, int vec_kv) {
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
    const int i_first = (int)(n0 / group), keys = (int)((n0 + nrow - 1) / group) + 1;      // rows of the sequence; keys of the tile's last row
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
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        unsigned mask = __ballot_sync(0xffffffffu, bad[e]);
        mask = (mask | mask >> 1 | mask >> 2 | mask >> 3) & 0x11111111u;      // one bit a row
        if (!mask || !any_bad_value(p, kvh, first + i_first + 1, first + keys)) continue;
        for (; mask; mask &= mask - 1) {
            const long long n = n0 + 16 * warp + (__ffs(mask) - 1) / 4 + 8 * e;
            const int i = (int)(n / group);
            __syncwarp();
            exact_row<BF16>(p, first, first + i, kvh * group + (int)(n - (long long)i * group));
        }
    }
}

template <int BF16, int HD>
cudaError_t mma_launch(const PromptArgs& a, cudaStream_t stream) {
    auto kern = prompt_mma_kernel<BF16, HD>;
    const size_t smem = (size_t)(kPwRows + 2 * kPwKeys) * (HD + 8) * 2;
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return e;
    const long long slots = ((long long)a.rows * (a.heads / a.kv_heads) >> 6) + a.seqs.seqs;
    if (slots > 0x7fffffffll || a.kv_heads > 65535) return cudaErrorInvalidValue;
    const int vec_q = a.q_stride % 8 == 0 && ((uintptr_t)a.q & 15) == 0;
    const int vec_kv = a.k_stride % 8 == 0 && a.v_stride % 8 == 0 && (((uintptr_t)a.k | (uintptr_t)a.v) & 15) == 0;
    return launch_pdl(kern, dim3((unsigned)slots, (unsigned)a.kv_heads), dim3(kPwThreads), smem, stream, a, vec_q, vec_kv);
}

}  // namespace

cudaError_t prompt_launch(PromptArgs a, int sm_count, cudaStream_t stream) {
    if (a.rows == 0 || a.seqs.seqs == 0) return cudaSuccess;
    if (a.bf16) return a.head_dim <= 64 ? mma_launch<1, 64>(a, stream) : (a.head_dim <= 128 ? mma_launch<1, 128>(a, stream) : mma_launch<1, 256>(a, stream));
    return a.head_dim <= 64 ? mma_launch<0, 64>(a, stream) : (a.head_dim <= 128 ? mma_launch<0, 128>(a, stream) : mma_launch<0, 256>(a, stream));
}

}  // namespace smeg
