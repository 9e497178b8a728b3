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
// A thread holds four pairs of one head (eight depths), the threads of a head are neighbouring lanes.  Rows of queries and the (page, KV heads) of a
// batch are CTAs of one launch.  A row's cosines and sines are formed once in shared memory and serve all of its query heads.  A page's CTA has few
// heads, so there they are formed for its first row alone, and row r takes the sum formulas with the cosines and sines of r frequencies, which the
// caller's table holds.
//
// Bytes bound it from some thousand rows on (each 16-bit value is read and written once, a cached one is read once and leaves as a byte), the instructions next to
// them: 8192 rows of 32 + 8 normalised heads of 128 take 36 us (4.6 TB/s of 6.5 measured), without norms, 28 + 4 heads of 96, 23 (4.4), 2001 of those 7.2 (3.4);
// 4096 rows of five prompts with their pages 31 us, 15 of them the pages', with issue slots 54 % busy at the 20 warps an SM that 96 registers allow.  Short calls are a
// chain of dependent loads -- row offsets, page number, rows, scale -- and a launch: one row 2.1 us, append and read of 48 single rows 6.5.
#include "common.cuh"
#include "kernels.h"
#include "paged.h"

namespace smeg {
namespace {

constexpr int kRotThreads = 128;
constexpr int kRowTile = 8;                        // rows of a CTA of query heads, at most
constexpr int kHeld = 8;                           // runs of eight depths that a thread of a page's CTA keeps
constexpr int kPageHeads = 32;                     // heads of a page's CTA, at most
constexpr int kAhead = 2;                          // and that a thread of a row's CTA has on their way
constexpr float kLeastScale = 7.703719777548943e-34f;   // 2^-110: a smaller scale has no reciprocal to speak of and counts as zero
constexpr float kRound = 12582912.0f;              // 1.5 * 2^23: what is added to it is rounded to an integer, in the low bits of the sum

// How a head's pairs lie.  A thread has the pairs 4 c .. 4 c + 3.
enum { kHalves = 0,                                // (i, i + hd / 2): two runs of four depths
       kNeighbours = 1,                            // (2 i, 2 i + 1): one run of eight
       kMixed = 2,                                 // (i, i + rot / 2) up to rot, neighbours behind: one or the other
       kAny = 3 };                                 // rot no multiple of 8, or heads off the 8-byte grid: depth by depth

struct HeadLay {
    int hd, half, group, log2_group, inter;        // depths, rotated pairs, lanes of a head (a power of two), interleaved pairs
    float inv_hd;
};

// Index of the first (e = 0) or second member of a head's pair p.
__device__ __forceinline__ int pair_at(const HeadLay& L, int p, int e) {
    if (p >= L.half || L.inter) return 2 * p + e;   // (pairs behind the rotated part are neighbours, as 2 p = rot + 2 (p - rot / 2))
    return p + e * L.half;
}
template <int LAY>
__device__ __forceinline__ bool is_split(const HeadLay& L, int c) {
    return LAY == kHalves || (LAY == kMixed && 4 * c < L.half);
}

struct Octet {
    float a[4], b[4];                              // first and second members of four pairs
};
template <int BF16>
__device__ __forceinline__ float2 both(uint32_t w) {
    if (BF16) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
    return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
struct Raw {
    uint2 u, w;                                    // as they lie: halves, four first members, then four second ones; neighbours, eight depths
};
template <int LAY>
__device__ __forceinline__ Raw load_raw(const uint16_t* x, const HeadLay& L, int c) {
    Raw o;
    if (LAY != kAny) {
        const bool split = is_split<LAY>(L, c);
        o.u = *reinterpret_cast<const uint2*>(x + (split ? 4 * c : 8 * c));
        o.w = *reinterpret_cast<const uint2*>(x + (split ? L.half + 4 * c : 8 * c + 4));
    } else {
        uint32_t r[8];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            r[j] = x[pair_at(L, 4 * c + j, 0)];
            r[4 + j] = x[pair_at(L, 4 * c + j, 1)];
        }
        o.u = make_uint2(r[0] | r[1] << 16, r[2] | r[3] << 16);
        o.w = make_uint2(r[4] | r[5] << 16, r[6] | r[7] << 16);
    }
    return o;
}
template <int BF16, int LAY>
__device__ __forceinline__ Octet unpack(const Raw& x, const HeadLay& L, int c) {
    const bool split = LAY == kAny || is_split<LAY>(L, c);
    const float2 f[4] = {both<BF16>(x.u.x), both<BF16>(x.u.y), both<BF16>(x.w.x), both<BF16>(x.w.y)};
    Octet o;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        o.a[j] = split ? (j & 1 ? f[j / 2].y : f[j / 2].x) : f[j].x;
        o.b[j] = split ? (j & 1 ? f[2 + j / 2].y : f[2 + j / 2].x) : f[j].y;
    }
    return o;
}
template <int BF16, int LAY>
__device__ __forceinline__ void store_pairs(uint16_t* x, const HeadLay& L, int c, const Octet& o) {
    if (LAY != kAny) {
        const bool split = is_split<LAY>(L, c);
        uint2 u, w;
        u.x = split ? pack2_t<BF16>(o.a[0], o.a[1]) : pack2_t<BF16>(o.a[0], o.b[0]);
        u.y = split ? pack2_t<BF16>(o.a[2], o.a[3]) : pack2_t<BF16>(o.a[1], o.b[1]);
        w.x = split ? pack2_t<BF16>(o.b[0], o.b[1]) : pack2_t<BF16>(o.a[2], o.b[2]);
        w.y = split ? pack2_t<BF16>(o.b[2], o.b[3]) : pack2_t<BF16>(o.a[3], o.b[3]);
        *reinterpret_cast<uint2*>(x + (split ? 4 * c : 8 * c)) = u;
        *reinterpret_cast<uint2*>(x + (split ? L.half + 4 * c : 8 * c + 4)) = w;
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            x[pair_at(L, 4 * c + j, 0)] = f32_to_t<BF16>(o.a[j]);
            x[pair_at(L, 4 * c + j, 1)] = f32_to_t<BF16>(o.b[j]);
        }
    }
}
// code + 128 in the low byte: |x * inv| is at most 127 and a little (not half a code more), so nothing is clamped.
__device__ __forceinline__ uint32_t code_of(float x, float inv) { return __float_as_uint(fmaf(x, inv, kRound + 128.0f)); }
__device__ __forceinline__ uint32_t four_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}
// Byte e of a word of codes as the code it stands for: 2^23 + byte is a number whose bits end in the byte.
__device__ __forceinline__ float byte_value(uint32_t w, int e) { return __uint_as_float(__byte_perm(w, 0x4b000000u, 0x7440 | e)) - 8388736.0f; }
// Codes of four pairs: whole words where the pairs lie that way (a cache row starts on a 16-byte boundary), else byte by byte.
template <int LAY>
__device__ __forceinline__ void store_codes(uint8_t* x, const HeadLay& L, int c, const Octet& o, float inv) {
    uint32_t u[4], w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        u[j] = code_of(o.a[j], inv);
        w[j] = code_of(o.b[j], inv);
    }
    if (LAY != kAny || L.half % 4 == 0) {
        const bool split = LAY == kAny ? !L.inter && 4 * c < L.half : is_split<LAY>(L, c);
        const uint32_t lo = split ? four_bytes(u[0], u[1], u[2], u[3]) : four_bytes(u[0], w[0], u[1], w[1]);
        const uint32_t hi = split ? four_bytes(w[0], w[1], w[2], w[3]) : four_bytes(u[2], w[2], u[3], w[3]);
        if (LAY == kNeighbours) {
            *reinterpret_cast<uint2*>(x + 8 * c) = make_uint2(lo, hi);
        } else {
            *reinterpret_cast<uint32_t*>(x + (split ? 4 * c : 8 * c)) = lo;
            *reinterpret_cast<uint32_t*>(x + (split ? L.half + 4 * c : 8 * c + 4)) = hi;
        }
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            x[pair_at(L, 4 * c + j, 0)] = (uint8_t)u[j];
            x[pair_at(L, 4 * c + j, 1)] = (uint8_t)w[j];
        }
    }
}

// Sum, or largest, of a head's lanes: every lane of the warp, whichever heads they have.
__device__ __forceinline__ float head_sum(float x, int group) {
#pragma unroll
    for (int s = 16; s; s >>= 1)
        if (s < group) x += __shfl_xor_sync(0xffffffffu, x, s);
    return x;
}
__device__ __forceinline__ unsigned head_max(unsigned x, int group) {
#pragma unroll
    for (int s = 16; s; s >>= 1)
        if (s < group) x = max(x, __shfl_xor_sync(0xffffffffu, x, s));
    return x;
}
// Norm (w: the weights of the thread's pairs).  All lanes of the warp.
__device__ __forceinline__ void normalise(const HeadLay& L, bool live, float eps, const Octet& w, Octet& o) {
    float sum = 0.0f;
#pragma unroll
    for (int j = 0; j < 4; ++j) sum = fmaf(o.a[j], o.a[j], fmaf(o.b[j], o.b[j], sum));
    const float mean = fmaf(head_sum(live ? sum : 0.0f, L.group), L.inv_hd, eps);
    float r;                                                       // (within 2 units of the last place; a mean below 2^-126 counts as zero)
    asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(mean));
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        o.a[j] = o.a[j] * r * w.a[j];
        o.b[j] = o.b[j] * r * w.b[j];
    }
}
// Rotation by the cosines and sines of the four pairs.
__device__ __forceinline__ void rotate4(const float4 c, const float4 s, Octet& o) {
    const float cc[4] = {c.x, c.y, c.z, c.w}, ss[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const float x = o.a[j], y = o.b[j];
        o.a[j] = fmaf(-y, ss[j], x * cc[j]);
        o.b[j] = fmaf(x, ss[j], y * cc[j]);
    }
}
template <int LAY>
__device__ __forceinline__ Octet norm_weights(const float* w, const HeadLay& L, int c, bool live) {
    Octet o = {};
    if (!w || !live) return o;
    if (LAY != kAny) {
        const bool split = is_split<LAY>(L, c);
        const float4 x = *reinterpret_cast<const float4*>(w + (split ? 4 * c : 8 * c)), y = *reinterpret_cast<const float4*>(w + (split ? L.half + 4 * c : 8 * c + 4));
        const float f[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            o.a[j] = split ? f[j] : f[2 * j];
            o.b[j] = split ? f[4 + j] : f[2 * j + 1];
        }
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            o.a[j] = w[pair_at(L, 4 * c + j, 0)];
            o.b[j] = w[pair_at(L, 4 * c + j, 1)];
        }
    }
    return o;
}
__device__ __forceinline__ float2 cos_sin(const RotateArgs& p, long long pos, int pair) {
    const double turns = (double)pos * p.turns[pair];
    const float frac = (float)(turns - rint(turns));
    float2 t;
    sincospif(2.0f * frac, &t.y, &t.x);
    return make_float2(t.x * p.factor, t.y * p.factor);
}
// Cosines and sines of `rows` rows' pairs (1 and 0 behind the rotated part): a row's cosines, then its sines.
template <class Pos>
__device__ __forceinline__ void fill_trig(const RotateArgs& p, const HeadLay& L, float* cs, int rows, Pos pos) {
    const int pairs = L.hd / 2;
    int r = 0, j = threadIdx.x;
    while (j >= pairs) { j -= pairs; ++r; }
    int dr = 0, dj = kRotThreads;
    while (dj >= pairs) { dj -= pairs; ++dr; }
    while (r < rows) {
        const float2 t = j < L.half ? cos_sin(p, pos(r), j) : make_float2(1.0f, 0.0f);
        cs[r * L.hd + j] = t.x;
        cs[r * L.hd + pairs + j] = t.y;
        r += dr;
        j += dj;
        if (j >= pairs) { j -= pairs; ++r; }
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

// The largest of x, |a|, |b|; NaN where one of them is.
__device__ __forceinline__ float max_abs3(float x, float a, float b) {
    float r;
    asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(x), "f"(a), "f"(b));
    return r;
}

// A (page, KV heads) of the batch, keys or values.  A thread keeps what it has -- kHeld runs of eight -- from the search for the largest magnitude to the codes: values
// as they were loaded, keys as they come out of norm and rotation, in 32 bits in shared memory (a place of each thread's own).  A longer page is read, and its keys
// are formed, twice.
template <int BF16, int LAY, int KEYS>
__device__ __forceinline__ void page_unit(const RotateArgs& p, const HeadLay& L, float* cs, int unit) {
    __shared__ unsigned s_max[kPageHeads];
    __shared__ float s_inv[kPageHeads], s_ratio[kPageHeads];
    __shared__ int s_start[kRotThreads];
    const PackedSeqs& B = p.seqs;
    const int tid = threadIdx.x, page = 1 << B.page_log2;
    if (tid < B.seqs) s_start[tid] = B.starts[tid];                // (asked for together with the row offsets, not behind them)
    constexpr int which = KEYS ? 0 : 1;
    const int slot = (unit >> 1) / p.page_groups, hg = (unit >> 1) - slot * p.page_groups;
    const int h0 = hg * p.page_heads, nh = min(p.page_heads, p.kv_heads - h0);
    const int s = count_upto(B.seqs, slot, [&](int i) { int f; seq_rows(B, i, &f); return first_slot(f, i, B.page_log2, 2); }) - 1;
    if (s < 0) return;
    int first;
    const int rows = seq_rows(B, s, &first), start = s < kRotThreads ? s_start[s] : B.starts[s];
    if (start < 0) return;
    const long long piece = slot - first_slot(first, s, B.page_log2, 2);
    const int d = start & (page - 1);                              // slot of the sequence's first row in its page
    if (piece < 0 || piece >= pieces(rows, d, B.page_log2)) return;
    const int r0 = piece == 0 ? 0 : (int)(piece * page - d), r1 = (int)min((long long)rows, (piece + 1) * page - d), n = r1 - r0;
    const int at = piece == 0 ? d : 0;                             // first slot that is written
    // (row, head) of this thread's group of lanes, pairs 4 c ... of it
    const int c = tid & (L.group - 1), mine = tid >> L.log2_group, rpp = p.page_rows, mr = mine * p.page_magic >> 16, mh = mine - mr * p.page_heads;
    const bool mine_ok = 8 * c < L.hd && mr < rpp && mh < nh;
    const bool norm = KEYS && p.k_w != nullptr, rotate = KEYS && p.turns != nullptr;
    const size_t stride = KEYS ? p.k_stride : p.v_stride, step = stride * rpp;
    const uint16_t* src = (KEYS ? p.k : p.v) + (size_t)(first + r0 + mr) * stride + (h0 + mh) * L.hd;
    const int left = mine_ok ? n - mr : 0;                         // rows from this thread's first one on
    Raw held[kHeld];
    auto load = [&](int c0) {                                      // rows c0 + mr, c0 + mr + rpp, ...
        const uint16_t* x = src + (size_t)c0 * stride;
#pragma unroll
        for (int e = 0; e < kHeld; ++e) {
            held[e].u = held[e].w = make_uint2(0, 0);
            if (c0 + e * rpp < left) held[e] = load_raw<LAY>(x, L, c);
            x += step;
        }
    };
    load(0);                                                       // (on their way while the page is looked up)
    const int id = page_of(B, s, (long long)start + r0);
    if (id < 0) {
        if (tid == 0 && p.status) atomicOr(p.status, STATUS_PAGE);
        return;
    }
    const int block = page * L.hd;                                 // bytes of one head's keys or values in a page
    uint8_t* dst = p.codes + (((size_t)id * p.kv_heads + h0) * 2 + which) * block + at * L.hd;
    float* scale = p.scales + ((size_t)id * p.kv_heads + h0) * 2 + which;
    const float old = tid < nh && at > 0 ? scale[2 * tid] : 0.0f;  // (asked for here, used behind the search)
    if (tid < kPageHeads) s_max[tid] = 0;
    const Octet w = norm_weights<LAY>(norm ? p.k_w : nullptr, L, c, mine_ok);
    // The first row's angles are formed here; row r is r steps of the frequencies further, by the sum formulas (steps: [256][cosines, sines], 32 bits)
    if (rotate) fill_trig(p, L, cs, 1, [&](int) { return (long long)start + r0; });
    __syncthreads();
    float4 c_0 = make_float4(1.f, 1.f, 1.f, 1.f), s_0 = make_float4(0.f, 0.f, 0.f, 0.f);
    if (rotate && mine_ok) {
        c_0 = *reinterpret_cast<const float4*>(cs + 4 * c);
        s_0 = *reinterpret_cast<const float4*>(cs + L.hd / 2 + 4 * c);
    }
    auto treat = [&](int e, int r) {                               // run e, row r
        Octet o = unpack<BF16, LAY>(held[e], L, c);
        if (norm) normalise(L, r < left + mr, p.k_eps, w, o);
        if (rotate && r < left + mr) {
            float4 u = make_float4(1.f, 1.f, 1.f, 1.f), v = make_float4(0.f, 0.f, 0.f, 0.f);
            const float* t = p.steps + r * 2 * L.half + 4 * c;
            if (LAY != kAny || L.half % 4 == 0) {
                if (4 * c < L.half && r > 0) {                     // (no load stands before a single row's codes)
                    u = *reinterpret_cast<const float4*>(t);
                    v = *reinterpret_cast<const float4*>(t + L.half);
                }
            } else {
                float x[4], y[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const bool in = 4 * c + j < L.half;
                    x[j] = in ? t[j] : 1.0f;
                    y[j] = in ? t[L.half + j] : 0.0f;
                }
                u = make_float4(x[0], x[1], x[2], x[3]);
                v = make_float4(y[0], y[1], y[2], y[3]);
            }
            const float4 cc = make_float4(fmaf(-s_0.x, v.x, c_0.x * u.x), fmaf(-s_0.y, v.y, c_0.y * u.y), fmaf(-s_0.z, v.z, c_0.z * u.z), fmaf(-s_0.w, v.w, c_0.w * u.w));
            const float4 ss = make_float4(fmaf(c_0.x, v.x, s_0.x * u.x), fmaf(c_0.y, v.y, s_0.y * u.y), fmaf(c_0.z, v.z, s_0.z * u.z), fmaf(c_0.w, v.w, s_0.w * u.w));
            rotate4(cc, ss, o);
        }
        return o;
    };
    float4* kept = reinterpret_cast<float4*>(cs + L.hd) + tid;     // [run][first, second members][thread]
    float top_f = 0.0f;
    unsigned top_16 = 0;                                           // (of the bits of two values: an infinity or NaN is larger than every number)
    const int chunk = kHeld * rpp;
    const bool keep = n <= chunk;
    for (int c0 = 0; c0 < n; c0 += chunk) {
        if (c0) load(c0);
#pragma unroll
        for (int e = 0; e < kHeld; ++e) {
            if (c0 + e * rpp >= n) break;                          // (the same for the whole block)
            if (KEYS) {
                const Octet o = treat(e, c0 + e * rpp + mr);
                if (c0 + e * rpp >= left) continue;                // (no row: zeros, and under a norm with an eps of zero not even those)
#pragma unroll
                for (int j = 0; j < 4; ++j) top_f = max_abs3(top_f, o.a[j], o.b[j]);
                if (keep) {
                    kept[(2 * e) * kRotThreads] = make_float4(o.a[0], o.a[1], o.a[2], o.a[3]);
                    kept[(2 * e + 1) * kRotThreads] = make_float4(o.b[0], o.b[1], o.b[2], o.b[3]);
                }
            } else {
                const unsigned r[4] = {held[e].u.x, held[e].u.y, held[e].w.x, held[e].w.y};
#pragma unroll
                for (int j = 0; j < 4; ++j) top_16 = __vmaxu2(top_16, r[j] & 0x7fff7fffu);
            }
        }
    }
    unsigned mx = __float_as_uint(top_f);
    if (!KEYS) {
        const float2 f = both<BF16>(top_16);
        mx = max(__float_as_uint(f.x), __float_as_uint(f.y));
    }
    mx = head_max(mx, L.group);
    if (mine_ok && c == 0) atomicMax(&s_max[mh], mx);
    __syncthreads();
    if (tid < nh) {
        const float top = __uint_as_float(s_max[tid]);
        float now = top < __uint_as_float(0x7f800000u) ? __fdiv_rn(top, 127.0f) : __uint_as_float(0x7fc00000u);
        if (now < kLeastScale) now = 0.0f;
        if (old >= now || old != old) now = old;                   // (a block that holds a NaN or an infinity is NaN until its page starts over)
        scale[2 * tid] = now;
        s_inv[tid] = now > 0.0f ? __fdiv_rn(1.0f, now) : 0.0f;
        s_ratio[tid] = now > old ? __fdiv_rn(old, now) : 1.0f;
    }
    __syncthreads();
    // the codes of earlier calls under a scale that grew
    if (at > 0)
        for (int h = 0; h < nh; ++h) {
            const float ratio = s_ratio[h];
            if (ratio == 1.0f) continue;
            uint32_t* old = reinterpret_cast<uint32_t*>(dst - at * L.hd + h * 2 * block);
            for (int i = tid; i < at * L.hd / 4; i += kRotThreads) {
                const uint32_t x = old[i];
                uint32_t o[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) o[e] = code_of(byte_value(x, e), ratio);
                old[i] = four_bytes(o[0], o[1], o[2], o[3]);
            }
        }
    const float inv = mine_ok ? s_inv[mh] : 0.0f;
    uint8_t* to = dst + mh * 2 * block + mr * L.hd;
    uint16_t* ko = KEYS && p.k_out ? p.k_out + (size_t)(first + r0 + mr) * p.ko_stride + (h0 + mh) * L.hd : nullptr;
    for (int c0 = 0; c0 < n; c0 += chunk) {
        if (!keep) load(c0);
#pragma unroll
        for (int e = 0; e < kHeld; ++e) {
            const int r = c0 + e * rpp;
            if (r >= n) break;
            Octet o;
            if (KEYS && keep) {
                const float4 u = kept[(2 * e) * kRotThreads], v = kept[(2 * e + 1) * kRotThreads];
                o.a[0] = u.x; o.a[1] = u.y; o.a[2] = u.z; o.a[3] = u.w;
                o.b[0] = v.x; o.b[1] = v.y; o.b[2] = v.z; o.b[3] = v.w;
            } else {
                o = treat(e, r + mr);
            }
            if (r >= left) continue;
            store_codes<LAY>(to + r * L.hd, L, c, o, inv);
            if (ko) store_pairs<BF16, LAY>(ko + (size_t)r * p.ko_stride, L, c, o);
        }
    }
}

// A few rows of some query heads, or of key heads that go to no cache; of all query heads and then all key heads (p.joint), which have the rows' cosines in common.
template <int BF16, int LAY>
__device__ __forceinline__ void row_unit(const RotateArgs& p, const HeadLay& L, float* cs, int unit) {
    __shared__ long long s_pos[kRowTile];
    const int tid = threadIdx.x;
    const int tile = unit / p.head_tiles;
    int ht = unit - tile * p.head_tiles;
    const int r0 = tile * p.row_tile, n = min(p.row_tile, p.rows - r0);
    bool is_q = ht < p.q_tiles;
    if (!is_q) ht -= p.q_tiles;
    const int h0 = ht * p.head_tile;
    int nh = min(p.head_tile, (is_q ? p.heads : p.kv_heads) - h0);
    // (row, head) of this thread's group of lanes: `hpp` heads of `rpp` rows at a time, kAhead times as many rows on their way
    const int hpp = p.row_heads, rpp = p.row_rows;
    const int mine = tid * p.lanes_magic >> 16, c = tid - mine * p.lanes, mr = mine * p.row_magic >> 16, mh = mine - mr * hpp;
    const bool mine_ok = 8 * c < L.hd && mr < rpp;
    size_t si = is_q ? p.q_stride : p.k_stride, so = is_q ? p.qo_stride : p.ko_stride;
    const uint16_t* src = (is_q ? p.q : p.k) + (size_t)(r0 + mr) * si + (h0 + mh) * L.hd;
    uint16_t* dst = (is_q ? p.q_out : p.k_out) + (size_t)(r0 + mr) * so + (h0 + mh) * L.hd;
    Raw next[kAhead];
    int nh_load = nh;                                              // (of the heads that are being loaded)
    auto load = [&](int r, int h) {
        const uint16_t* x = src + (size_t)r * si + h * L.hd;
        const bool ok = mine_ok && h + mh < nh_load;
#pragma unroll
        for (int e = 0; e < kAhead; ++e) {
            next[e].u = next[e].w = make_uint2(0, 0);
            if (ok && r + e * rpp + mr < n) next[e] = load_raw<LAY>(x, L, c);
            x += si * rpp;
        }
    };
    load(0, 0);                                                    // (on their way while the rows' angles are formed)
    // positions, -1 for a row that is nobody's
    __shared__ int s_start[kRotThreads];
    int s = 0;
    if (p.seqs.cu && tid < p.seqs.seqs) s_start[tid] = p.seqs.starts[tid];
    if (p.seqs.cu) s = count_upto(p.seqs.seqs, r0, [&](int i) { int f; seq_rows(p.seqs, i, &f); return (long long)f; }) - 1;
    if (tid < n) {
        long long pos = p.start + r0 + tid;
        if (p.positions) pos = p.positions[r0 + tid];
        if (p.seqs.cu) {
            int f = 0, m = 0;
            if (s < 0) s = 0;
            while (s + 1 < p.seqs.seqs && p.seqs.cu[s + 1] <= r0 + tid) ++s;
            m = seq_rows(p.seqs, s, &f);
            const int st = s < kRotThreads ? s_start[s] : p.seqs.starts[s];
            pos = st >= 0 && r0 + tid >= f && r0 + tid < f + m ? (long long)st + (r0 + tid - f) : -1;
        }
        s_pos[tid] = pos;
    }
    const float* nw = is_q ? p.q_w : p.k_w;
    float eps = is_q ? p.q_eps : p.k_eps;
    Octet w = norm_weights<LAY>(nw, L, c, mine_ok);
    __syncthreads();
    if (p.turns) {
        fill_trig(p, L, cs, n, [&](int r) { return s_pos[r]; });
        __syncthreads();
    }
    const bool any_row = p.seqs.cu == nullptr;
    bool more = p.joint;                                           // the key heads are still to come
    for (int h = 0, r = 0; h < nh;) {
        Raw cur[kAhead];
#pragma unroll
        for (int e = 0; e < kAhead; ++e) cur[e] = next[e];
        const int h_now = h, r_now = r;
        r += kAhead * rpp;
        if (r >= n) { r = 0; h += hpp; }
        const bool turn = more && h >= nh;
        if (turn) {
            src = p.k + (size_t)(r0 + mr) * p.k_stride + mh * L.hd;
            si = p.k_stride;
            nh_load = p.kv_heads;
            h = 0;
        }
        if (turn || h < nh) load(r, h);
        uint16_t* y = dst + (size_t)r_now * so + h_now * L.hd;
        const bool head_ok = mine_ok && h_now + mh < nh;
#pragma unroll
        for (int e = 0; e < kAhead; ++e) {
            if (r_now + e * rpp >= n) break;                       // (the same for the whole block)
            const int row = r_now + e * rpp + mr;
            const bool live = head_ok && row < n && (any_row || s_pos[row] >= 0);
            Octet o = unpack<BF16, LAY>(cur[e], L, c);
            if (nw) normalise(L, live, eps, w, o);
            if (p.turns && live)
                rotate4(*reinterpret_cast<const float4*>(cs + row * L.hd + 4 * c), *reinterpret_cast<const float4*>(cs + row * L.hd + L.hd / 2 + 4 * c), o);
            if (live) store_pairs<BF16, LAY>(y, L, c, o);
            y += so * rpp;
        }
        if (turn) {
            more = false;
            dst = p.k_out + (size_t)(r0 + mr) * p.ko_stride + mh * L.hd;
            so = p.ko_stride;
            nh = nh_load;
            nw = p.k_w;
            eps = p.k_eps;
            w = norm_weights<LAY>(nw, L, c, mine_ok);
        }
    }
}

__device__ __forceinline__ HeadLay head_lay(const RotateArgs& p) {
    HeadLay L;
    L.hd = p.head_dim; L.half = p.rot / 2; L.inter = p.interleaved; L.log2_group = p.lanes_log2; L.group = 1 << p.lanes_log2; L.inv_hd = p.inv_hd;
    return L;
}
// Rows alone, and pages with rows: in one kernel the pages' registers cost the rows 3 to 14 %.  The next grid starts when these CTAs have gone, and not where they begin: its
// CTAs would take the places that are free by then, and gather on a few SMs (rows at the start and so, us: 2001 of 28 / 4 heads of 96 8.2 and 7.7, 300 of 32 / 8 of 128 5.7 and
// 4.4; append and read of 48 rows 7.5 and 6.6).  Rows with two runs a thread on their way and eight CTAs an SM: 800 rows 7.5 -> 5.4, 8192 37.2 -> 36.0 us.
template <int BF16, int LAY>
__global__ void __launch_bounds__(kRotThreads, 8) rotate_rows_kernel(const __grid_constant__ RotateArgs p) {
    extern __shared__ __align__(16) float trig_s[];
    pdl_wait();
    row_unit<BF16, LAY>(p, head_lay(p), trig_s, blockIdx.x);
}
// CTAS: of an SM.  Five where there are that many (4096 rows of prompts, us with four, five, six and seven: 41.1, 38.2, 38.4, 39.2), four, which spill nothing, for the grids of a
// step (48 single rows with four and five: 6.45 and 6.66; 37 rows: 5.63 and 5.84).
template <int BF16, int LAY, int CTAS>
__global__ void __launch_bounds__(kRotThreads, CTAS) rotate_append_kernel(const __grid_constant__ RotateArgs p) {
    extern __shared__ __align__(16) float trig_s[];
    const HeadLay L = head_lay(p);
    pdl_wait();
    if ((int)blockIdx.x >= p.page_units) row_unit<BF16, LAY>(p, L, trig_s, blockIdx.x - p.page_units);
    else if (blockIdx.x & 1) page_unit<BF16, LAY == kAny ? kAny : kNeighbours, 0>(p, L, trig_s, blockIdx.x);
    else page_unit<BF16, LAY, 1>(p, L, trig_s, blockIdx.x);
}

// The values of whole pages: a CTA takes kReadCodes of a page's codes, a thread eight at a time, so that a warp's loads and stores are whole lines.
constexpr int kReadThreads = 256, kReadCodes = 2 * 8 * kReadThreads;
template <int BF16>
__global__ void __launch_bounds__(kReadThreads) paged_read_kernel(uint16_t* __restrict__ out, const uint8_t* __restrict__ codes, const float* __restrict__ scales,
                                                                  const int* __restrict__ ids, unsigned parts, unsigned per_page, unsigned block, int pages, int out_vec,
                                                                  unsigned* status) {
    pdl_wait();
    const unsigned i = blockIdx.x / parts, off0 = (blockIdx.x - i * parts) * kReadCodes + 8 * threadIdx.x;
    const int id = ids[i];
    const bool there = id >= 0 && id < pages;
    if (!there && off0 == 0) atomicOr(status, STATUS_PAGE);
    const uint8_t* x = codes + (size_t)(there ? id : 0) * per_page;
    const float* sc = scales + (size_t)(there ? id : 0) * (per_page / block);
    uint16_t* y = out + (size_t)i * per_page;
    uint2 w[2];
    float s[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const unsigned off = off0 + h * (kReadCodes / 2);
        w[h] = make_uint2(0x80808080u, 0x80808080u);
        s[h] = 0.0f;
        if (there && off < per_page) {
            w[h] = *reinterpret_cast<const uint2*>(x + off);
            s[h] = sc[off / block];
        }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const unsigned off = off0 + h * (kReadCodes / 2);
        if (off >= per_page) break;
        const uint32_t r[2] = {w[h].x, w[h].y};
        uint32_t o[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = pack2_t<BF16>(byte_value(r[e / 2], 2 * (e & 1)) * s[h], byte_value(r[e / 2], 2 * (e & 1) + 1) * s[h]);
        if (out_vec) {
            *reinterpret_cast<uint4*>(y + off) = make_uint4(o[0], o[1], o[2], o[3]);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) y[off + e] = (uint16_t)(o[e / 2] >> (16 * (e & 1)));
        }
    }
}

typedef void (*RotKernel)(RotateArgs);
template <int BF16, int LAY>
RotKernel rot_kernel_of(int kind) {                                // 0: rows alone; else the CTAs of an SM with pages
    return kind == 0 ? rotate_rows_kernel<BF16, LAY> : (kind == 4 ? rotate_append_kernel<BF16, LAY, 4> : rotate_append_kernel<BF16, LAY, 5>);
}
template <int BF16>
RotKernel rot_kernel(int lay, int kind) {
    return lay == kHalves ? rot_kernel_of<BF16, kHalves>(kind) : (lay == kNeighbours ? rot_kernel_of<BF16, kNeighbours>(kind) : (lay == kMixed ? rot_kernel_of<BF16, kMixed>(kind) : rot_kernel_of<BF16, kAny>(kind)));
}

}  // namespace

cudaError_t rotate_append_launch(RotateArgs a, int bf16, int sm_count, cudaStream_t stream) {
    const bool paged = a.codes != nullptr, vec = a.rot % 8 == 0 && ((a.q_stride | a.k_stride | a.v_stride | a.qo_stride | a.ko_stride) & 3) == 0 &&
                     (((uintptr_t)a.q | (uintptr_t)a.k | (uintptr_t)a.v | (uintptr_t)a.q_out | (uintptr_t)a.k_out) & 7) == 0 &&
                     (((uintptr_t)a.q_w | (uintptr_t)a.k_w) & 15) == 0;
    const int lay = !vec ? kAny : (a.interleaved || a.rot == 0 ? kNeighbours : (a.rot == a.head_dim ? kHalves : kMixed));
    a.lanes_log2 = 0;
    while (8 << a.lanes_log2 < a.head_dim) ++a.lanes_log2;
    const int per_pass = kRotThreads >> a.lanes_log2;
    // Lanes of a head in row units: without norms they need not find one another, and heads of 96 or 80 depths leave none idle
    a.lanes = paged || a.q_w || a.k_w ? 1 << a.lanes_log2 : a.head_dim / 8;
    a.lanes_magic = (65536 + a.lanes - 1) / a.lanes;               // tid * magic >> 16 = tid / lanes
    const int row_pass = kRotThreads / a.lanes;
    a.inv_hd = 1.0f / (float)a.head_dim;
    // row units: all heads of a few rows, so that they share the rows' cosines: two, or four where there are CTAs enough, for each row that the block's threads have at a time;
    // of one row, as many heads as the block has at a time, while the machine has room for more CTAs.  (us with tiles of two, four and eight rows: 2001 rows of 28 / 4 heads of 96
    // 7.2, 8.5, 11.9, of 32 / 8 heads of 128 10.9, 12.9, 19.6; 8192 rows 36.9, 36.3, 37.5; 2001 rows of 6 heads of 64, of which there are two rows at a time, 3.8, 3.5, 4.4, 5000 rows
    // 7.7, 6.3, 5.8)
    const int qh = a.q ? a.heads : 0, kh = a.k && !paged ? a.kv_heads : 0, most = qh > kh ? qh : kh;
    a.head_tile = (size_t)a.rows >= (size_t)sm_count * 4 ? most : row_pass;
    if (a.head_tile > most) a.head_tile = most;
    a.q_tiles = qh ? (qh + a.head_tile - 1) / a.head_tile : 0;
    a.joint = qh && kh && a.head_tile == most;
    a.head_tiles = a.joint ? 1 : a.q_tiles + (kh ? (kh + a.head_tile - 1) / a.head_tile : 0);
    a.row_heads = a.head_tile < row_pass ? a.head_tile : row_pass;
    if (a.row_heads < 1) a.row_heads = 1;
    a.row_rows = row_pass / a.row_heads;
    const int tile = ((size_t)a.rows < (size_t)sm_count * 32 ? 2 : 4) * a.row_rows;
    a.row_tile = (size_t)a.rows < (size_t)sm_count * 8 ? 1 : (tile < kRowTile ? tile : kRowTile);
    a.row_magic = (65536 + a.row_heads - 1) / a.row_heads;         // mine * magic >> 16 = mine / row_heads for mine below 256
    const long long row_units = (long long)((a.rows + a.row_tile - 1) / a.row_tile) * a.head_tiles;
    long long page_units = 0;
    if (paged) {
        // KV heads of a CTA: as many as fill its registers with a sequence's rows in a page, and fewer while there is not a CTA an SM
        const int page = 1 << a.seqs.page_log2, mean = (a.rows + a.seqs.seqs - 1) / a.seqs.seqs;
        const long long slots = ((long long)a.rows >> a.seqs.page_log2) + 2ll * a.seqs.seqs;
        a.page_heads = kHeld * per_pass / (mean < page ? mean : page);
        if (a.page_heads > per_pass) a.page_heads = per_pass;
        if (a.page_heads > kPageHeads) a.page_heads = kPageHeads;
        if (a.page_heads > a.kv_heads) a.page_heads = a.kv_heads;
        if (a.page_heads < 1) a.page_heads = 1;
        while (a.page_heads > 1 && slots * ((a.kv_heads + a.page_heads - 1) / a.page_heads) * 2 < sm_count) a.page_heads = (a.page_heads + 1) / 2;
        a.page_rows = per_pass / a.page_heads;
        a.page_magic = (65536 + a.page_heads - 1) / a.page_heads;
        a.page_groups = (a.kv_heads + a.page_heads - 1) / a.page_heads;
        page_units = slots * a.page_groups * 2;
    }
    if (row_units + page_units > 0x7fffffffll) return cudaErrorInvalidValue;
    if (row_units + page_units == 0) return cudaSuccess;
    a.page_units = (int)page_units;
    const size_t rows_smem = a.turns ? (size_t)a.row_tile * a.head_dim * sizeof(float) : 0;
    const size_t page_smem = paged ? a.head_dim * sizeof(float) + (size_t)kHeld * 8 * kRotThreads * sizeof(float) : 0;
    const size_t smem = rows_smem > page_smem ? rows_smem : page_smem;
    const int kind = !paged ? 0 : (row_units + page_units <= 4ll * sm_count ? 4 : 5);
    const RotKernel kern = bf16 ? rot_kernel<1>(lay, kind) : rot_kernel<0>(lay, kind);
    return launch_pdl(kern, dim3((unsigned)(row_units + page_units)), dim3(kRotThreads), smem, stream, a);
}

cudaError_t paged_read_launch(uint16_t* out, const uint8_t* codes, const float* scales, const int* ids, size_t n, int pages, int page, int kv_heads, int head_dim,
                              int bf16, unsigned* status, cudaStream_t stream) {
    const size_t block = (size_t)page * head_dim, per_page = block * kv_heads * 2, parts = (per_page + kReadCodes - 1) / kReadCodes;
    if (n == 0) return cudaSuccess;
    if (per_page > 0xffffffffu - kReadCodes || n > 0x7fffffffu / parts) return cudaErrorInvalidValue;
    const int vec = ((uintptr_t)out & 15) == 0;
    const dim3 grid((unsigned)(n * parts));
    if (bf16)
        return launch_pdl(paged_read_kernel<1>, grid, dim3(kReadThreads), 0, stream, out, codes, scales, ids, (unsigned)parts, (unsigned)per_page, (unsigned)block, pages, vec, status);
    return launch_pdl(paged_read_kernel<0>, grid, dim3(kReadThreads), 0, stream, out, codes, scales, ids, (unsigned)parts, (unsigned)per_page, (unsigned)block, pages, vec, status);
}

}  // namespace smeg
