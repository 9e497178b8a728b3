// Norms of query and key heads, their rotation by position, and the append of keys and values to the pages of the 8-bit cache (sm_100a): what lies
// between the fused [q | k | v] projection of a self-attention block and its attention.
//
//   norm      y = x / sqrt(mean(x^2) + eps) * w, per head, 32 bits
//   rotation  of the first `rot` of a head's depths: the pair (a, b) becomes (a c - b s, b c + a s) with c, s the cosine and sine of
//             position * frequency (times a factor); pairs are (i, i + rot / 2), or (2 i, 2 i + 1) interleaved
//   pages     code = rint(x / scale) as a byte code + 128, scale = largest magnitude / 127 for each page, KV head and keys or values; a page's
//             scale starts over with its first position and otherwise only grows, and then the codes that are there are rounded again
// Everything from the loaded 16-bit value to the one rounding at the end (to 16 bits, or to a code) is 32 bits wide.  The angle is not: position *
// (frequency / 2 pi) is formed and reduced to a fraction of a turn in 64 bits, since a position of 10^6 at 32 bits would leave 4 digits of it.
//
// A thread holds four pairs of one head (eight depths), the threads of a head are neighbouring lanes; a row's cosines and sines are formed once
// in shared memory and serve all of its heads.  Rows of queries and the (page, KV heads) of a batch are CTAs of one launch.  A page's CTA reads its rows
// twice -- for the largest magnitude, then for the codes; the second time they come from L2.
#include "common.cuh"
#include "kernels.h"
#include "paged.h"

namespace smeg {
namespace {

constexpr int kRotThreads = 256;
constexpr int kTrigRows = 64;                      // rows whose cosines and sines are in shared memory at a time
constexpr float kLeastScale = 7.703719777548943e-34f;   // 2^-110: a smaller scale has no reciprocal to speak of and counts as zero

struct HeadLay {
    int hd, rot, half, group, inter;               // depths, rotated depths, rot / 2, lanes of a head (a power of two), interleaved pairs
};

// Index of the first (e = 0) or second member of a head's pair p.
__device__ __forceinline__ int pair_at(const HeadLay& L, int p, int e) {
    if (p >= L.half || L.inter) return 2 * p + e;   // (pairs behind the rotated part are neighbours, as 2 p = rot + 2 (p - rot / 2))
    return p + e * L.half;
}

// Pairs 4 c .. 4 c + 3 of a head.  VEC: rot a multiple of 8 and every head on an 8-byte boundary.
template <int BF16, int VEC>
__device__ __forceinline__ void load_pairs(const uint16_t* x, const HeadLay& L, int c, float (&a)[4], float (&b)[4]) {
    if (VEC) {
        const bool split = !L.inter && 4 * c < L.half;
        const uint2 u = *reinterpret_cast<const uint2*>(x + (split ? 4 * c : 8 * c));
        const uint2 w = *reinterpret_cast<const uint2*>(x + (split ? L.half + 4 * c : 8 * c + 4));
        const uint32_t r[4] = {u.x, u.y, w.x, w.y};
        float f[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            f[2 * i] = t_to_f32<BF16>((uint16_t)r[i]);
            f[2 * i + 1] = t_to_f32<BF16>((uint16_t)(r[i] >> 16));
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            a[j] = split ? f[j] : f[2 * j];
            b[j] = split ? f[4 + j] : f[2 * j + 1];
        }
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            a[j] = t_to_f32<BF16>(x[pair_at(L, 4 * c + j, 0)]);
            b[j] = t_to_f32<BF16>(x[pair_at(L, 4 * c + j, 1)]);
        }
    }
}
template <int BF16, int VEC>
__device__ __forceinline__ void store_pairs(uint16_t* x, const HeadLay& L, int c, const float (&a)[4], const float (&b)[4]) {
    if (VEC) {
        const bool split = !L.inter && 4 * c < L.half;
        uint2 u, w;
        u.x = split ? pack2_t<BF16>(a[0], a[1]) : pack2_t<BF16>(a[0], b[0]);
        u.y = split ? pack2_t<BF16>(a[2], a[3]) : pack2_t<BF16>(a[1], b[1]);
        w.x = split ? pack2_t<BF16>(b[0], b[1]) : pack2_t<BF16>(a[2], b[2]);
        w.y = split ? pack2_t<BF16>(b[2], b[3]) : pack2_t<BF16>(a[3], b[3]);
        *reinterpret_cast<uint2*>(x + (split ? 4 * c : 8 * c)) = u;
        *reinterpret_cast<uint2*>(x + (split ? L.half + 4 * c : 8 * c + 4)) = w;
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            x[pair_at(L, 4 * c + j, 0)] = f32_to_t<BF16>(a[j]);
            x[pair_at(L, 4 * c + j, 1)] = f32_to_t<BF16>(b[j]);
        }
    }
}
__device__ __forceinline__ uint32_t to_code(float x, float inv) {
    return (uint32_t)((int)fminf(fmaxf(rintf(x * inv), -127.0f), 127.0f) + 128);
}
// Codes of four pairs: whole words where the pairs lie that way (a cache row starts on a 16-byte boundary), else byte by byte.
__device__ __forceinline__ void store_codes(uint8_t* x, const HeadLay& L, int c, const float (&a)[4], const float (&b)[4], float inv) {
    uint32_t u[4], w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        u[j] = to_code(a[j], inv);
        w[j] = to_code(b[j], inv);
    }
    if (L.half % 4 == 0) {
        const bool split = !L.inter && 4 * c < L.half;
        const uint32_t lo = split ? u[0] | u[1] << 8 | u[2] << 16 | u[3] << 24 : u[0] | w[0] << 8 | u[1] << 16 | w[1] << 24;
        const uint32_t hi = split ? w[0] | w[1] << 8 | w[2] << 16 | w[3] << 24 : u[2] | w[2] << 8 | u[3] << 16 | w[3] << 24;
        *reinterpret_cast<uint32_t*>(x + (split ? 4 * c : 8 * c)) = lo;
        *reinterpret_cast<uint32_t*>(x + (split ? L.half + 4 * c : 8 * c + 4)) = hi;
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            x[pair_at(L, 4 * c + j, 0)] = (uint8_t)u[j];
            x[pair_at(L, 4 * c + j, 1)] = (uint8_t)w[j];
        }
    }
}

// Norm (w0, w1: the weights of the thread's pairs) and rotation (cs: cosine and sine of the row's pairs).  All lanes of the warp.
__device__ __forceinline__ void turn(const HeadLay& L, bool live, bool norm, float eps, const float (&w0)[4], const float (&w1)[4], const float2* cs,
                                     float (&a)[4], float (&b)[4]) {
    if (norm) {
        float sum = 0.0f;
#pragma unroll
        for (int j = 0; j < 4; ++j) sum = fmaf(a[j], a[j], fmaf(b[j], b[j], sum));
        if (!live) sum = 0.0f;
        for (int o = L.group >> 1; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        const float r = __fdiv_rn(1.0f, __fsqrt_rn(__fdiv_rn(sum, (float)L.hd) + eps));
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            a[j] = a[j] * r * w0[j];
            b[j] = b[j] * r * w1[j];
        }
    }
    if (cs) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float2 t = cs[j];
            const float x = a[j], y = b[j];
            a[j] = fmaf(-y, t.y, x * t.x);
            b[j] = fmaf(x, t.y, y * t.x);
        }
    }
}

// Cosines and sines of `rows` rows' pairs (1 and 0 behind the rotated part).
template <class Pos>
__device__ __forceinline__ void fill_trig(const RotateArgs& p, const HeadLay& L, float2* cs, int rows, Pos pos) {
    const int pairs = L.hd / 2;
    for (int i = threadIdx.x; i < rows * pairs; i += kRotThreads) {
        const int r = i / pairs, j = i - r * pairs;
        float2 t = make_float2(1.0f, 0.0f);
        if (j < L.half) {
            const double turns = (double)pos(r) * p.turns[j];
            const float frac = (float)(turns - rint(turns));
            sincospif(2.0f * frac, &t.y, &t.x);
            t.x *= p.factor;
            t.y *= p.factor;
        }
        cs[i] = t;
    }
}

// How many s below n have key(s) <= x: the block's threads together (every thread, the same arguments).
template <class Key>
__device__ __forceinline__ int count_upto(int n, long long x, Key key) {
    int got = 0;
    for (int s0 = 0; s0 < n; s0 += kRotThreads) {
        const int s = s0 + threadIdx.x;
        got += __syncthreads_count(s < n && key(s) <= x);
    }
    return got;
}

// A (page, KV heads) of the batch, keys or values.
template <int BF16, int VEC>
__device__ __forceinline__ void page_unit(const RotateArgs& p, const HeadLay& L, float2* cs, int unit) {
    __shared__ unsigned s_max[32];
    __shared__ float s_inv[32], s_ratio[32];
    const PackedSeqs& B = p.seqs;
    const int tid = threadIdx.x, page = 1 << B.page_log2;
    const int which = unit & 1, hgroups = (p.kv_heads + p.page_heads - 1) / p.page_heads;
    const int hg = (unit >> 1) % hgroups;
    const long long slot = (unit >> 1) / hgroups;
    const int h0 = hg * p.page_heads, nh = min(p.page_heads, p.kv_heads - h0);
    const int s = count_upto(B.seqs, slot, [&](int i) { int f; seq_rows(B, i, &f); return first_slot(f, i, B.page_log2, 2); }) - 1;
    if (s < 0) return;
    int first;
    const int rows = seq_rows(B, s, &first), start = B.starts[s];
    if (start < 0) return;
    const long long piece = slot - first_slot(first, s, B.page_log2, 2);
    const int d = start & (page - 1);                              // slot of the sequence's first row in its page
    if (piece < 0 || piece >= pieces(rows, d, B.page_log2)) return;
    const int r0 = piece == 0 ? 0 : (int)(piece * page - d), r1 = (int)min((long long)rows, (piece + 1) * page - d), n = r1 - r0;
    const int at = piece == 0 ? d : 0;                             // first slot that is written
    const int id = page_of(B, s, (long long)start + r0);
    if (id < 0) {
        if (tid == 0 && p.status) atomicOr(p.status, STATUS_PAGE);
        return;
    }
    const bool keys = which == 0;
    const uint16_t* src = (keys ? p.k : p.v) + (size_t)(first + r0) * (keys ? p.k_stride : p.v_stride) + (size_t)h0 * L.hd;
    const size_t stride = keys ? p.k_stride : p.v_stride;
    const size_t block = (size_t)page * L.hd;                      // bytes of one head's keys or values in a page
    uint8_t* dst = p.codes + (((size_t)id * p.kv_heads + h0) * 2 + which) * block + (size_t)at * L.hd;
    float* scale = p.scales + ((size_t)id * p.kv_heads + h0) * 2 + which;
    if (tid < 32) s_max[tid] = 0;
    const int lane_c = tid & (L.group - 1), per_pass = kRotThreads / L.group, mine = tid / L.group;
    const bool live_c = lane_c * 8 < L.hd, norm = keys && p.k_w != nullptr, rotate = keys && p.turns != nullptr;
    float w0[4] = {}, w1[4] = {};
    if (norm && live_c)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            w0[j] = p.k_w[pair_at(L, 4 * lane_c + j, 0)];
            w1[j] = p.k_w[pair_at(L, 4 * lane_c + j, 1)];
        }
    auto trig = [&](int c0, int m) {
        if (!rotate) return;
        __syncthreads();
        fill_trig(p, L, cs, m, [&](int r) { return (long long)start + r0 + c0 + r; });
        __syncthreads();
    };
    auto pass = [&](int c0, int m, auto done) {                    // rows c0 .. c0 + m of the page's, all heads
        for (int i0 = 0; i0 < m * nh; i0 += per_pass) {
            const int it = i0 + mine;
            const bool live = it < m * nh && live_c;
            const int r = live ? it / nh : 0, h = live ? it - r * nh : 0;
            float a[4] = {}, b[4] = {};
            if (live) load_pairs<BF16, VEC>(src + (size_t)(c0 + r) * stride + (size_t)h * L.hd, L, lane_c, a, b);
            turn(L, live, norm, p.k_eps, w0, w1, rotate && live ? cs + (size_t)r * (L.hd / 2) + 4 * lane_c : nullptr, a, b);
            done(live, c0 + r, h, a, b);
        }
    };
    __syncthreads();
    for (int c0 = 0; c0 < n; c0 += kTrigRows) {
        const int m = min(kTrigRows, n - c0);
        trig(c0, m);
        pass(c0, m, [&](bool live, int, int h, const float (&a)[4], const float (&b)[4]) {
            unsigned mx = 0;                                       // (of the bits: an infinity or NaN is larger than every number)
#pragma unroll
            for (int j = 0; j < 4; ++j) mx = max(mx, max(__float_as_uint(fabsf(a[j])), __float_as_uint(fabsf(b[j]))));
            if (!live) mx = 0;
            for (int o = L.group >> 1; o; o >>= 1) mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, o));
            if (live && lane_c == 0) atomicMax(&s_max[h], mx);
        });
    }
    __syncthreads();
    if (tid < nh) {
        const float old = at == 0 ? 0.0f : scale[2 * tid], mx = __uint_as_float(s_max[tid]);
        float now = mx < __uint_as_float(0x7f800000u) ? __fdiv_rn(mx, 127.0f) : __uint_as_float(0x7fc00000u);
        if (now < kLeastScale) now = 0.0f;
        if (old >= now || old != old) now = old;                   // (a block that holds a NaN or an infinity is NaN until its page starts over)
        scale[2 * tid] = now;
        s_inv[tid] = now > 0.0f ? __fdiv_rn(1.0f, now) : 0.0f;
        s_ratio[tid] = now > old ? __fdiv_rn(old, now) : 1.0f;
    }
    __syncthreads();
    // the codes of earlier calls under a scale that grew
    for (int h = 0; h < nh; ++h) {
        const float ratio = s_ratio[h];
        if (ratio == 1.0f || at == 0) continue;
        uint32_t* old = reinterpret_cast<uint32_t*>(dst - (size_t)at * L.hd + (size_t)h * 2 * block);
        for (int i = tid; i < at * L.hd / 4; i += kRotThreads) {
            const uint32_t w = old[i];
            uint32_t o = 0;
#pragma unroll
            for (int e = 0; e < 4; ++e) o |= to_code((float)((int)(w >> 8 * e & 255u) - 128), ratio) << 8 * e;
            old[i] = o;
        }
    }
    for (int c0 = 0; c0 < n; c0 += kTrigRows) {
        const int m = min(kTrigRows, n - c0);
        if (n > kTrigRows) trig(c0, m);
        pass(c0, m, [&](bool live, int r, int h, const float (&a)[4], const float (&b)[4]) {
            if (!live) return;
            store_codes(dst + (size_t)h * 2 * block + (size_t)r * L.hd, L, lane_c, a, b, s_inv[h]);
            if (keys && p.k_out) store_pairs<BF16, VEC>(p.k_out + (size_t)(first + r0 + r) * p.ko_stride + (size_t)(h0 + h) * L.hd, L, lane_c, a, b);
        });
    }
}

// Rows of heads: queries, or keys that go to no cache.
template <int BF16, int VEC>
__device__ __forceinline__ void row_unit(const RotateArgs& p, const HeadLay& L, float2* cs, int unit) {
    __shared__ long long s_pos[kTrigRows];
    const int tid = threadIdx.x;
    const int tile = unit / p.head_tiles, ht = unit - tile * p.head_tiles;
    const int r0 = tile * p.row_tile, n = min(p.row_tile, p.rows - r0);
    const int all = p.q_heads_here + p.k_heads_here, h0 = ht * p.head_tile, nh = min(p.head_tile, all - h0);
    // positions, -1 for a row that is nobody's
    for (int r = 0; r < n; ++r) {
        if (p.positions) {
            if (tid == 0) s_pos[r] = p.positions[r0 + r];
        } else if (!p.seqs.cu) {
            if (tid == 0) s_pos[r] = p.start + r0 + r;
        } else {
            const PackedSeqs& B = p.seqs;
            const int s = count_upto(B.seqs, r0 + r, [&](int i) { int f; seq_rows(B, i, &f); return (long long)f; }) - 1;
            if (tid == 0) {
                int f = 0;
                const int m = s < 0 ? 0 : seq_rows(B, s, &f), st = s < 0 ? -1 : B.starts[s];
                s_pos[r] = st >= 0 && r0 + r < f + m ? (long long)st + (r0 + r - f) : -1;
            }
        }
    }
    __syncthreads();
    if (p.turns) fill_trig(p, L, cs, n, [&](int r) { return s_pos[r]; });
    __syncthreads();
    const int lane_c = tid & (L.group - 1), per_pass = kRotThreads / L.group, mine = tid / L.group;
    const bool live_c = lane_c * 8 < L.hd;
    float qw[2][4] = {}, kw[2][4] = {};
    if (live_c)
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                if (p.q_w) qw[e][j] = p.q_w[pair_at(L, 4 * lane_c + j, e)];
                if (p.k_w && p.k_heads_here) kw[e][j] = p.k_w[pair_at(L, 4 * lane_c + j, e)];
            }
    for (int i0 = 0; i0 < n * nh; i0 += per_pass) {
        const int it = i0 + mine;
        const bool in = it < n * nh;
        const int r = in ? it / nh : 0, h = h0 + (in ? it - r * nh : 0);
        const bool is_q = h < p.q_heads_here;
        const int hh = is_q ? h : h - p.q_heads_here;
        const bool live = in && live_c && (!p.seqs.cu || s_pos[r] >= 0);
        float a[4] = {}, b[4] = {};
        if (live) load_pairs<BF16, VEC>((is_q ? p.q + (size_t)(r0 + r) * p.q_stride : p.k + (size_t)(r0 + r) * p.k_stride) + (size_t)hh * L.hd, L, lane_c, a, b);
        const float2* t = p.turns && live ? cs + (size_t)r * (L.hd / 2) + 4 * lane_c : nullptr;
        float w0[4], w1[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            w0[j] = is_q ? qw[0][j] : kw[0][j];
            w1[j] = is_q ? qw[1][j] : kw[1][j];
        }
        const bool norm_q = p.q_w != nullptr, norm_k = p.k_w != nullptr;
        float x[4], y[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) { x[j] = a[j]; y[j] = b[j]; }
        if (norm_q || norm_k) {                                    // (the reduction is the whole warp's, whichever heads its lanes have)
            turn(L, live, true, is_q ? p.q_eps : p.k_eps, w0, w1, nullptr, a, b);
            if (!(is_q ? norm_q : norm_k))
#pragma unroll
                for (int j = 0; j < 4; ++j) { a[j] = x[j]; b[j] = y[j]; }
        }
        turn(L, live, false, 0.0f, w0, w1, t, a, b);
        if (live) store_pairs<BF16, VEC>((is_q ? p.q_out + (size_t)(r0 + r) * p.qo_stride : p.k_out + (size_t)(r0 + r) * p.ko_stride) + (size_t)hh * L.hd, L, lane_c, a, b);
    }
}

template <int BF16, int VEC>
__global__ void __launch_bounds__(kRotThreads) rotate_append_kernel(const __grid_constant__ RotateArgs p) {
    extern __shared__ __align__(16) unsigned char smem[];
    float2* cs = reinterpret_cast<float2*>(smem);
    HeadLay L;
    L.hd = p.head_dim; L.rot = p.rot; L.half = p.rot / 2; L.inter = p.interleaved; L.group = p.lanes;
    pdl_launch_dependents();
    pdl_wait();
    if ((int)blockIdx.x < p.page_units) page_unit<BF16, VEC>(p, L, cs, blockIdx.x);
    else row_unit<BF16, VEC>(p, L, cs, blockIdx.x - p.page_units);
}

// The values of whole pages: 16 codes a thread.
template <int BF16>
__global__ void __launch_bounds__(256) paged_read_kernel(uint16_t* __restrict__ out, const uint8_t* __restrict__ codes, const float* __restrict__ scales,
                                                         const int* __restrict__ ids, size_t n, size_t per_page, size_t block, int pages, int out_vec, unsigned* status) {
    pdl_launch_dependents();
    pdl_wait();
    const size_t idx = ((size_t)blockIdx.x * blockDim.x + threadIdx.x) * 16;
    if (idx >= n * per_page) return;
    const size_t i = idx / per_page, off = idx - i * per_page;
    const int id = ids[i];
    uint4 w = make_uint4(0x80808080u, 0x80808080u, 0x80808080u, 0x80808080u);
    float s = 0.0f;
    if (id >= 0 && id < pages) {
        w = *reinterpret_cast<const uint4*>(codes + (size_t)id * per_page + off);
        s = scales[(size_t)id * (per_page / block) + off / block];
    } else if (off == 0) {
        atomicOr(status, STATUS_PAGE);
    }
    const uint32_t r[4] = {w.x, w.y, w.z, w.w};
    uint32_t o[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const uint32_t x = r[e / 2] >> (16 * (e & 1));
        o[e] = pack2_t<BF16>((float)((int)(x & 255u) - 128) * s, (float)((int)(x >> 8 & 255u) - 128) * s);
    }
    if (out_vec) {
        *reinterpret_cast<uint4*>(out + idx) = make_uint4(o[0], o[1], o[2], o[3]);
        *reinterpret_cast<uint4*>(out + idx + 8) = make_uint4(o[4], o[5], o[6], o[7]);
    } else {
#pragma unroll
        for (int e = 0; e < 16; ++e) out[idx + e] = (uint16_t)(o[e / 2] >> (16 * (e & 1)));
    }
}

}  // namespace

cudaError_t rotate_append_launch(RotateArgs a, int bf16, int sm_count, cudaStream_t stream) {
    const bool paged = a.codes != nullptr;
    a.lanes = 1;
    while (a.lanes * 8 < a.head_dim) a.lanes *= 2;
    // row units: all heads of a few rows, so that they share the rows' cosines; of one row, as many heads as the block has at a time, while the
    // machine has room for more CTAs
    a.q_heads_here = a.q ? a.heads : 0;
    a.k_heads_here = a.k && !paged ? a.kv_heads : 0;
    const int all = a.q_heads_here + a.k_heads_here;
    a.row_tile = (size_t)a.rows >= (size_t)sm_count * 16 ? 4 : 1;
    a.head_tile = (size_t)a.rows >= (size_t)sm_count * 4 ? all : kRotThreads / a.lanes;
    if (a.head_tile > all) a.head_tile = all;
    a.head_tiles = all ? (all + a.head_tile - 1) / a.head_tile : 0;
    const long long row_units = (long long)((a.rows + a.row_tile - 1) / a.row_tile) * a.head_tiles;
    long long page_units = 0;
    int trig_rows = a.row_tile;
    if (paged) {
        // as many KV heads to a CTA as make 256 rows of a full page; more share the cosines, fewer share the work
        const int page = 1 << a.seqs.page_log2;
        a.page_heads = page >= 256 ? 1 : 256 / page;
        if (a.page_heads > a.kv_heads) a.page_heads = a.kv_heads;
        const long long most = ((long long)a.rows >> a.seqs.page_log2) + 2ll * a.seqs.seqs;
        page_units = most * ((a.kv_heads + a.page_heads - 1) / a.page_heads) * 2;
        trig_rows = page < kTrigRows ? page : kTrigRows;
    }
    if (row_units + page_units > 0x7fffffffll) return cudaErrorInvalidValue;
    if (row_units + page_units == 0) return cudaSuccess;
    a.page_units = (int)page_units;
    const size_t smem = a.turns ? (size_t)trig_rows * (a.head_dim / 2) * sizeof(float2) : 0;
    const bool vec = a.rot % 8 == 0 && ((a.q_stride | a.k_stride | a.v_stride | a.qo_stride | a.ko_stride) & 3) == 0 &&
                     (((uintptr_t)a.q | (uintptr_t)a.k | (uintptr_t)a.v | (uintptr_t)a.q_out | (uintptr_t)a.k_out) & 7) == 0;
    void (*kern)(RotateArgs) = bf16 ? (vec ? rotate_append_kernel<1, 1> : rotate_append_kernel<1, 0>) : (vec ? rotate_append_kernel<0, 1> : rotate_append_kernel<0, 0>);
    if (smem > 48 * 1024) {
        const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) return e;
    }
    return launch_pdl(kern, dim3((unsigned)(row_units + page_units)), dim3(kRotThreads), smem, stream, a);
}

cudaError_t paged_read_launch(uint16_t* out, const uint8_t* codes, const float* scales, const int* ids, size_t n, int pages, int page, int kv_heads, int head_dim,
                              int bf16, unsigned* status, cudaStream_t stream) {
    const size_t block = (size_t)page * head_dim, per_page = block * kv_heads * 2, threads = n * per_page / 16, grid = (threads + 255) / 256;
    if (grid == 0) return cudaSuccess;
    if (grid > 0x7fffffffu) return cudaErrorInvalidValue;
    const int vec = ((uintptr_t)out & 15) == 0;
    if (bf16) return launch_pdl(paged_read_kernel<1>, dim3((unsigned)grid), dim3(256), 0, stream, out, codes, scales, ids, n, per_page, block, pages, vec, status);
    return launch_pdl(paged_read_kernel<0>, dim3((unsigned)grid), dim3(256), 0, stream, out, codes, scales, ids, n, per_page, block, pages, vec, status);
}

}  // namespace smeg
