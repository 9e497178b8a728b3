"""Rotation, the 8-bit paged cache and attention over packed batches on the GPU, against the definitions in 64 bits.

The tolerances are counted: a result is rounded once to 16 bits (half a step, eps / 2 of its value); the 32-bit work before that and the
probabilities' own rounding are bounded beside each check."""
import math

import numpy as np
import pytest
import torch

import sme_gemm_b200 as sg

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


@pytest.fixture(autouse=True)
def _status():
    yield
    if torch.cuda.is_available():
        assert sg.last_status() == 0


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(gen, *shape, dtype=F16, scale=1.0):
    return (torch.randn(shape, generator=gen, device="cuda") * scale).to(dtype)


def _int(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _half_step(dtype):
    return torch.finfo(dtype).eps / 2


def _near(got, want, tol, dtype):
    """|got - want| <= half a step of the value + tol (f64, elementwise), + half the smallest number of the type."""
    err = (got.double() - want).abs()
    room = _half_step(dtype) * (want.abs() + tol) + tol + (2.0 ** -25 if dtype == F16 else 2.0 ** -133)
    bad = ~(err <= room)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off: worst {float((err - room).max()):.3g} over, at {bad.nonzero()[0].tolist()}"


# ------------------------------------------------------------------------------------------------ rotation

def _turned(x, hd, positions, rotary, norm):
    """(heads in 64 bits, bound of the 32-bit error).  The bound: a norm's sum of hd squares in 32 bits, a root, a quotient and two products are off by less than
    2^-19 of a value up to 256 depths (64 additions at most in a chain, 2^-24 each); the angle's fraction is rounded at 2^-25 of a turn and the
    cosine and sine at 2^-22; two products and a sum: 2^-22.  Together under 2^-18 of the pair's length."""
    rows = x.shape[0]
    x = x.double().reshape(rows, -1, hd)
    if norm is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + norm.eps) * norm.weight.double()
    y, size = x.clone(), x.abs()
    if rotary is not None:
        f, rot = torch.tensor(rotary.frequencies(), device="cuda"), rotary.rotary_dim()
        angle = positions.double()[:, None, None] * f
        c, s = torch.cos(angle) * rotary.factor(), torch.sin(angle) * rotary.factor()
        i0 = torch.arange(0, rot, 2, device="cuda") if rotary.interleaved() else torch.arange(rot // 2, device="cuda")
        i1 = i0 + (1 if rotary.interleaved() else rot // 2)
        a, b = x[..., i0], x[..., i1]
        y[..., i0], y[..., i1] = a * c - b * s, b * c + a * s
        length = (a * a + b * b).sqrt() * rotary.factor()
        size[..., i0], size[..., i1] = length, length
    return y.reshape(rows, -1), (size * 2.0 ** -18).reshape(rows, -1)


def _norm(gen, hd):
    return sg.Norm.rms((1.0 + 0.2 * torch.randn(hd, generator=gen, device="cuda")).cpu().numpy(), 1e-6)


@pytest.mark.parametrize("rows,heads,kv,hd,rot,inter,norms,dtype,pad,shift", [
    (1, 32, 8, 128, 128, False, True, F16, 0, 0), (1, 1, 1, 8, 2, False, False, F16, 0, 0), (3, 5, 1, 80, 20, True, True, BF16, 3, 1),
    (37, 6, 6, 64, 64, False, False, F16, 8, 0), (700, 3, 3, 40, 10, False, True, BF16, 0, 0), (2500, 4, 2, 96, 48, True, False, F16, 16, 8),
    (64, 2, 1, 256, 256, True, True, F16, 0, 0), (5, 7, 7, 112, 56, False, True, F16, 1, 0), (2, 40, 2, 16, 16, False, True, BF16, 0, 4)])
def test_rotated_heads(rows, heads, kv, hd, rot, inter, norms, dtype, pad, shift):
    gen = _gen(rows + hd)
    width = (heads + kv) * hd + pad
    buf = _randn(gen, rows * width + shift, dtype=dtype, scale=3.0)
    x = buf[shift:].view(rows, width)
    q, k = x[:, :heads * hd], x[:, heads * hd:(heads + kv) * hd]
    rotary = sg.Rotary(hd, rotary_dim=rot, interleaved=inter)
    pos = torch.randint(0, 1 << 20, (rows,), generator=gen, device="cuda", dtype=torch.int32)
    qn, kn = (_norm(gen, hd), _norm(gen, hd)) if norms else (None, None)
    q_out, k_out = torch.zeros(rows, heads * hd, dtype=dtype, device="cuda"), torch.zeros(rows, kv * hd + 5, dtype=dtype, device="cuda")
    sg.rotate_heads(q, k, pos, rotary, q_out, k_out[:, :kv * hd], q_norm=qn, k_norm=kn)
    for got, src, norm in ((q_out, q, qn), (k_out[:, :kv * hd], k, kn)):
        want, tol = _turned(src, hd, pos, rotary, norm)
        _near(got, want, tol, dtype)
    assert not k_out[:, kv * hd:].any()
    # in place, one kind of heads at a time, and from a first position on
    want, tol = _turned(k, hd, torch.arange(1000, 1000 + rows, device="cuda"), rotary, kn)
    sg.rotate_heads(None, k, 1000, rotary, None, k, k_norm=kn)
    _near(k, want, tol, dtype)


def test_norms_of_one_kind_and_scaled_frequencies():
    gen = _gen(5)
    hd, rows = 64, 9
    for rotary in (sg.Rotary(hd).linear(3.0), sg.Rotary(hd).by_wavelength(8.0, 1.0, 4.0, 8192), sg.Rotary(hd, rotary_dim=32, interleaved=True).yarn(16.0, 4096), None):
        q, k = _randn(gen, rows, 4 * hd), _randn(gen, rows, 2 * hd)
        qn = _norm(gen, hd)
        pos = torch.arange(7, 7 + rows, device="cuda", dtype=torch.int32)
        q_out, k_out = torch.empty_like(q), torch.empty_like(k)
        sg.rotate_heads(q, k, pos, rotary, q_out, k_out, q_norm=qn, head_dim=hd)
        for got, src, norm in ((q_out, q, qn), (k_out, k, None)):
            _near(got, *_turned(src, hd, pos, rotary, norm), F16)


def test_rotation_past_32_bit_offsets():
    """Row offsets of over 2^31 elements."""
    rows, stride, hd = 2200, 1 << 20, 64
    buf = torch.empty(rows * stride, dtype=F16, device="cuda")
    x = buf.view(rows, stride)[:, :2 * hd]
    gen = _gen(1)
    x.copy_(_randn(gen, rows, 2 * hd))
    out = torch.empty(rows, 2 * hd, dtype=F16, device="cuda")
    rotary = sg.Rotary(hd)
    sg.rotate_heads(x, None, 0, rotary, out, None)
    _near(out, *_turned(x, hd, torch.arange(rows, device="cuda"), rotary, None), F16)


# ------------------------------------------------------------------------------------------------ the cache

class Pool:
    """A cache with sequences in it, appended to in steps, and what it should hold: unquantised values in 64 bits."""

    def __init__(self, heads, kv, hd, page, seqs, cols, spare=3, seed=0, dtype=F16, **kw):
        self.gen = _gen(seed)
        self.dtype, self.heads, self.kv, self.hd, self.page, self.cols = dtype, heads, kv, hd, page, cols
        pages = seqs * cols + spare
        self.cache = sg.PagedKvCache(heads, kv, hd, pages, page)
        self.cache.codes.copy_(torch.randint(0, 256, self.cache.codes.shape, generator=self.gen, device="cuda", dtype=torch.uint8))   # what earlier users left
        self.cache.scales.copy_(torch.rand(self.cache.scales.shape, generator=self.gen, device="cuda") * 9)
        self.table = torch.randperm(pages, generator=self.gen, device="cuda")[:seqs * cols].reshape(seqs, cols).to(torch.int32)
        self.have = [0] * seqs
        self.true = [torch.zeros(2, 0, kv, hd, dtype=torch.float64, device="cuda") for _ in range(seqs)]

    def batch(self, rows, idle=(), starts=None):
        starts = [(-1 if s in idle else n) for s, n in enumerate(self.have)] if starts is None else starts
        return sg.PagedBatch(_int([0] + np.cumsum(rows).tolist()), _int(starts), self.table)

    def append(self, rows, idle=(), rotary=None, k_norm=None, scale=1.0, behind=0, pad=0, **kw):
        total = sum(rows) + behind
        row = self.kv * self.hd
        x = _randn(self.gen, total, 2 * row + pad, dtype=self.dtype, scale=scale)
        k, v = x[:, :row], x[:, row:2 * row]
        batch = self.batch(rows, idle)
        self.cache.append(k, v, batch, rotary, k_norm=k_norm, **kw)
        r0 = 0
        for s, r in enumerate(rows):
            if s not in idle and r:
                at = torch.arange(self.have[s], self.have[s] + r, device="cuda")
                kk, _ = _turned(k[r0:r0 + r], self.hd, at, rotary, k_norm)
                new = torch.stack([kk.reshape(r, self.kv, self.hd), v[r0:r0 + r].double().reshape(r, self.kv, self.hd)])
                self.true[s] = torch.cat([self.true[s], new], 1)
                self.have[s] += r
            r0 += r
        return batch, k, v

    def values(self, s):
        """[2, positions, kv heads, head_dim] that the cache holds for sequence s, in 64 bits, and each position's scale."""
        n = self.have[s]
        ids = self.table[s, :-(-n // self.page)].long()
        sc = self.cache.scales[ids].double()[..., None, None]
        x = (self.cache.codes[ids].double() - 128) * sc
        cut = lambda y: y.permute(2, 0, 3, 1, 4).reshape(2, -1, self.kv, y.shape[-1])[:, :n]  # noqa: E731
        return cut(x), cut(sc.expand(-1, -1, -1, self.page, 1))

    def check(self, times=1):
        """A value is off by at most half a code, `times` over (a code is rounded again where its page's scale grew), + the 32-bit error of the
        value, of the scale and of the product with its reciprocal: under 127 * 2^-17 codes."""
        for s, true in enumerate(self.true):
            got, scale = self.values(s)
            assert torch.all((got - true).abs() <= scale * (0.5 * times + 127 * 2.0 ** -17)), f"sequence {s}"
            # and the scale is the largest magnitude of the page so far
            for p in range(0, self.have[s], self.page):
                most = true[:, p:p + self.page].abs().amax((1, 3))
                assert torch.all((scale[:, p, :, 0] * 127 - most).abs() <= most * 2.0 ** -17)


@pytest.mark.parametrize("kv,hd,page,dtype,rot,norm", [(8, 128, 64, F16, 128, True), (1, 16, 16, BF16, 0, False), (3, 80, 32, F16, 20, True), (2, 256, 256, BF16, 256, True),
                                                       (20, 64, 128, F16, 32, False), (6, 112, 16, F16, 112, True)])
def test_appended_rows_stand_in_their_pages(kv, hd, page, dtype, rot, norm):
    seqs = 5
    pool = Pool(kv * 2, kv, hd, page, seqs, 700 // page + 2, seed=hd, dtype=dtype)
    rotary = sg.Rotary(hd, rotary_dim=rot) if rot else None
    k_norm = _norm(pool.gen, hd) if norm else None
    untouched = pool.cache.codes.clone(), pool.cache.scales.clone()
    # prompts of several lengths, one of them empty; a step of one row each with an idle sequence; a chunk; rows behind the last sequence
    for rows, idle, behind, pad in (([1, 0, page, page + 1, 333], (), 0, 0), ([1, 1, 1, 1, 1], (2,), 2, 8), ([0, 2 * page, 3, 0, 40], (0,), 0, 3)):
        pool.append(rows, idle, rotary, k_norm, behind=behind, pad=pad, scale=0.5 if idle else 1.0)
    assert pool.have == [2, 2 * page + 1, page + 3, page + 2, 374]
    pool.check(times=3)
    used = torch.cat([pool.table[s, :-(-n // page)] for s, n in enumerate(pool.have)]).long()
    free = torch.ones(len(untouched[1]), dtype=torch.bool, device="cuda")
    free[used] = False
    assert torch.equal(pool.cache.codes[free], untouched[0][free]) and torch.equal(pool.cache.scales[free], untouched[1][free])


def test_growing_magnitudes_round_the_codes_again_and_a_new_page_starts_over():
    pool = Pool(2, 2, 32, 16, 2, 4, seed=9)
    for i in range(20):
        pool.append([1, 2], scale=0.1 * 1.5 ** i)
    for s in range(2):
        got, scale = pool.values(s)
        # each growth costs a position at most half a code of the scale it grew to, and those are geometric: 0.5 * (1 + 2/3 + ...) = 1.5 of the last, a step more
        # where a draw skips (a row's largest value is within a factor of four of the last one's): 3
        assert torch.all((got - pool.true[s]).abs() <= scale * 3.0)
        assert torch.all(scale[:, 1:16] == scale[:, :1].expand(-1, 15, -1, -1))
    # the same table used by other sequences: position 0 starts the scale over
    pool.have, pool.true = [0, 0], [t[:, :0] for t in pool.true]
    pool.append([5, 16], scale=0.01)
    pool.check()


def test_zeros_tiny_values_and_blocks_with_nan_or_infinity():
    pool = Pool(2, 2, 32, 16, 1, 4, seed=3, dtype=BF16)
    k, v = torch.zeros(4, 64, dtype=BF16, device="cuda"), torch.full((4, 64), 1e-38, dtype=BF16, device="cuda")
    pool.cache.append(k, v, pool.batch([4]))
    page = int(pool.table[0, 0])
    assert torch.all(pool.cache.scales[page] == 0) and torch.all(pool.cache.codes[page, :, :, :4] == 128)
    k[1, 3], v[2, 40] = math.inf, math.nan                      # key head 0, value head 1
    pool.cache.append(k, v, pool.batch([4], starts=[4]))
    assert torch.equal(torch.isnan(pool.cache.scales[page]), torch.tensor([[True, False], [False, True]], device="cuda"))
    pool.cache.append(torch.ones_like(k), torch.ones_like(v), pool.batch([4], starts=[8]))     # sticky ...
    assert torch.equal(torch.isnan(pool.cache.scales[page]), torch.tensor([[True, False], [False, True]], device="cuda"))
    pool.cache.append(torch.ones_like(k), torch.ones_like(v), pool.batch([4], starts=[0]))     # ... until the page starts over
    assert torch.all(pool.cache.codes[page, :, :, :4] == 255) and torch.allclose(pool.cache.scales[page], torch.tensor(1 / 127, device="cuda"))


def test_queries_and_keys_of_the_same_pass():
    gen = _gen(4)
    pool = Pool(6, 2, 64, 32, 3, 8, seed=4)
    pool.append([3, 60, 1])
    rotary, qn, kn = sg.Rotary(64, rotary_dim=32), _norm(gen, 64), _norm(gen, 64)
    rows, idle = [2, 5, 40], (1,)
    x = _randn(gen, 49, 10 * 64)
    q, k, v = x[:, :384], x[:, 384:512], x[:, 512:]
    q_out, k_out = torch.full((49, 384), 7.0, dtype=F16, device="cuda"), torch.full((49, 128), 7.0, dtype=F16, device="cuda")
    batch = pool.batch(rows, idle)
    pool.cache.append(k, v, batch, rotary, k_norm=kn, k_out=k_out, q=q, q_out=q_out, q_norm=qn)
    pos = torch.tensor([3, 4] + [0] * 5 + list(range(1, 41)), device="cuda")
    live = torch.tensor([True] * 2 + [False] * 5 + [True] * 40 + [False] * 2, device="cuda")
    for out, src, norm in ((q_out, q, qn), (k_out, k, kn)):
        want, tol = _turned(src[:47], 64, pos, rotary, norm)
        _near(out[:47][live[:47]], want[live[:47]], tol[live[:47]], F16)
        assert torch.all(out[~live] == 7.0)
    # in place, the same bits
    codes = pool.cache.codes.clone()
    pool.cache.append(k, v, batch, rotary, k_norm=kn, k_out=k, q=q, q_out=q, q_norm=qn)
    assert torch.equal(q[live], q_out[live]) and torch.equal(k[live], k_out[live]) and torch.equal(codes, pool.cache.codes)


@pytest.mark.parametrize("dtype,shift", [(F16, 0), (BF16, 3)])
def test_pages_read_back_are_the_values_they_stand_for(dtype, shift):
    pool = Pool(4, 2, 48, 32, 3, 3, seed=8)
    pool.append([70, 1, 33])
    ids = torch.cat([pool.table.reshape(-1), pool.table[1, :1]])
    out = torch.zeros(ids.numel() * 2 * 2 * 32 * 48 + shift, dtype=dtype, device="cuda")
    pool.cache.read(ids, out[shift:])
    want = (pool.cache.codes[ids.long()].float() - 128) * pool.cache.scales[ids.long()][..., None, None]
    assert torch.equal(out[shift:].view(want.shape), want.to(dtype))


def test_pages_outside_the_pool_are_skipped_and_told():
    pool = Pool(2, 1, 32, 16, 3, 4, seed=2)
    pool.append([20, 20, 20])
    pool.table[1, 1], pool.table[1, 2] = -1, 10 ** 6
    before = pool.cache.codes.clone(), pool.cache.scales.clone()
    x = _randn(pool.gen, 18, 32)
    pool.cache.append(x, x, pool.batch([0, 18, 0]))             # positions 20 .. 37 of sequence 1: pages 1 and 2, neither in the pool
    assert sg.last_status() == 8 and torch.equal(before[0], pool.cache.codes) and torch.equal(before[1], pool.cache.scales)
    out = torch.empty(2, 1, 2, 16, 32, dtype=F16, device="cuda")
    pool.cache.read(pool.table[1, :2].contiguous(), out)
    assert sg.last_status() == 8 and not out[1].any() and out[0].any()
    # attention: the pages that are there count, other sequences are whole
    q, o = _randn(pool.gen, 3, 64), torch.zeros(3, 64, dtype=F16, device="cuda")
    pool.cache.attend(q, pool.batch([1, 1, 1], starts=[19, 19, 19]), o)
    assert sg.last_status() == 8
    pool.have = [20, 16, 20]
    want, tol = _attended(pool, q, [1, 1, 1], [19, 19, 19])
    _near(o, want, tol, F16)
    # positions behind the table's room
    pool.cache.append(x[:2], x[:2], pool.batch([2, 0, 0], starts=[64, 0, 0]))
    assert sg.last_status() == 8


# ------------------------------------------------------------------------------------------------ attention over the cache

def _attended(pool, q, rows, starts, scale=None):
    """(attention in 64 bits over what the cache holds, bound of the error before the last rounding).

    With A the probability-weighted mean of |v|: a probability's rounding to f16 moves the result by 2^-11 A.  A score is a chain of hd / 16 products steps
    over bytes 0..255 (the offset comes off first) in 32 bits, whose additions the tensor core cuts off: (hd / 16 + 4) * 2^-23 of
    sum |q| * 255 * scale_k, and 2^-21 of the score itself for the products with its scales and the exponential; both numerator and sum move by
    twice that.  The values' sums run over bytes too, three steps a fold: 2^-20 * 255 * scale_v.  2^-18 A: folds, joins and the quotient."""
    hd, kv, heads = pool.hd, pool.kv, pool.heads
    group = heads // kv
    scale = pool.cache.scale() if scale is None else scale
    out = torch.zeros(len(q), heads, hd, dtype=torch.float64, device="cuda")
    tol = torch.zeros_like(out)
    r0 = 0
    for s, r in enumerate(rows):
        if starts[s] >= 0 and r:
            x, sc = pool.values(s)
            k, v = x.repeat_interleave(group, 2)
            sk, sv = sc.repeat_interleave(group, 2)[..., 0]
            qq = q[r0:r0 + r].double().reshape(r, heads, hd)
            z = torch.einsum("rhd,nhd->hrn", qq, k) * scale
            on = torch.arange(k.shape[0], device="cuda")[None, :] <= starts[s] + torch.arange(r, device="cuda")[:, None]
            e = (hd / 16 + 4) * 2.0 ** -23 * scale * qq.abs().sum(-1).T * 255 * sk.amax(0)[:, None] + 2.0 ** -21 * z.abs().masked_fill(~on, 0).amax(-1)
            p = torch.softmax(z.masked_fill(~on, -math.inf), -1)
            out[r0:r0 + r] = torch.einsum("hrn,nhd->rhd", p, v)
            a = torch.einsum("hrn,nhd->rhd", p, v.abs())
            tol[r0:r0 + r] = a * (2.0 ** -11 + 2.0 ** -18 + 4 * e.T[..., None]) + 2.0 ** -20 * 255 * sv.amax(0)[:, None]
        r0 += r
    return out.reshape(len(q), -1), tol.reshape(len(q), -1)


@pytest.mark.parametrize("heads,kv,hd,page,lens,rows,dtype,q_scale", [
    (32, 8, 128, 64, [901], [1], F16, 1.0), (8, 1, 128, 16, [1, 16, 17, 700], [1, 1, 1, 1], BF16, 1.0), (6, 6, 64, 32, [130, 2, 128, 129], [1, 2, 1, 1], F16, 3.0),
    (24, 3, 64, 16, [200, 33, 1000], [5, 5, 5], F16, 1.0), (12, 4, 80, 128, [257, 300], [3, 1], BF16, 2.0), (16, 2, 256, 64, [500, 40], [1, 1], F16, 1.0),
    (14, 2, 112, 256, [600, 256, 255], [1, 4, 9], F16, 1.0), (4, 4, 16, 16, [90], [90], F16, 1.0), (3, 1, 32, 32, [64, 1, 3], [7, 1, 0], BF16, 4.0),
    (16, 1, 256, 32, [300], [6], BF16, 1.0), (40, 8, 128, 64, [5000, 20], [1, 1], F16, 6.0)])
def test_attention_over_the_cache(heads, kv, hd, page, lens, rows, dtype, q_scale):
    pool = Pool(heads, kv, hd, page, len(lens), -(-max(lens) // page) + 1, seed=heads + hd, dtype=dtype)
    pool.append(lens)
    starts = [n - r for n, r in zip(lens, rows)]
    total = sum(rows)
    buf = _randn(pool.gen, total + 2, heads * hd + 8, dtype=dtype, scale=q_scale)
    q = buf[:, :heads * hd]
    out = torch.full((total + 2, heads * hd), 5.0, dtype=dtype, device="cuda")
    pool.cache.attend(q, pool.batch(rows, starts=starts), out)
    want, tol = _attended(pool, q[:total], rows, starts)
    _near(out[:total], want, tol, dtype)
    assert torch.all(out[total:] == 5.0)
    # the same from and to rows that start anywhere, bit for bit
    off = torch.empty((total + 2) * (heads * hd + 3) + 1, dtype=dtype, device="cuda")[1:].view(total + 2, -1)
    off.copy_(torch.cat([q, q[:, :3]], 1))
    o2 = torch.full((total + 2, heads * hd + 1), 5.0, dtype=dtype, device="cuda")
    pool.cache.attend(off[:, :heads * hd], pool.batch(rows, starts=starts), o2[:, 1:])
    assert torch.equal(o2[:, 1:], out) and torch.all(o2[:, 0] == 5.0)


def test_many_sequences_of_all_lengths_and_idle_ones():
    rng = np.random.default_rng(0)
    n = 150
    lens = [int(x) for x in np.exp(rng.uniform(0, math.log(1500), n))]
    pool = Pool(8, 2, 64, 16, n, -(-max(lens) // 16), seed=1)
    pool.append(lens)
    idle = set(rng.choice(n, 20, replace=False).tolist())
    starts = [-1 if s in idle else x - 1 for s, x in enumerate(lens)]
    q, out = _randn(pool.gen, n, 512), torch.full((n, 512), 5.0, dtype=F16, device="cuda")
    pool.cache.attend(q, pool.batch([1] * n, starts=starts), out)
    want, tol = _attended(pool, q, [1] * n, starts)
    _near(out, want, tol, F16)
    assert not out[list(idle)].any()


def test_a_chunk_behind_cached_positions():
    pool = Pool(8, 2, 64, 32, 2, 20, seed=6)
    pool.append([300, 40])
    pool.append([150, 77])
    q, out = _randn(pool.gen, 227, 512), torch.empty(227, 512, dtype=F16, device="cuda")
    pool.cache.attend(q, pool.batch([150, 77], starts=[300, 40]), out)
    _near(out, *_attended(pool, q, [150, 77], [300, 40]), F16)


def test_non_finite_blocks_and_queries_stay_with_the_rows_that_attend_to_them():
    pool = Pool(4, 2, 64, 16, 2, 10, seed=7)
    pool.append([100, 50])
    page = int(pool.table[0, 3])                                # positions 48 .. 63 of sequence 0
    pool.cache.scales[page, 0, 1] = math.nan                    # values of KV head 0
    pool.cache.scales[page, 1, 0] = math.nan                    # keys of KV head 1
    rows, starts = [60, 2], [40, 48]
    q, out = _randn(pool.gen, 62, 256), torch.empty(62, 256, dtype=F16, device="cuda")
    q[61, 70] = math.inf                                        # one head of the last row
    pool.cache.attend(q, pool.batch(rows, starts=starts), out)
    bad = torch.isnan(out)
    assert bad[8:60].all() and not bad[:8].any()                # rows from position 48 on
    assert not bad[60].any() and bad[61, 64:128].all() and not bad[61, :64].any() and not bad[61, 128:].any()
    clean = pool.have
    pool.have = [48, 50]
    want, tol = _attended(pool, q[:8], [8, 0], [40, 48])
    _near(out[:8], want, tol, F16)
    pool.have = clean


def test_scales_of_very_different_size_in_one_tile():
    """Pages of 16 whose values differ by 10^6: the larger page's result is not touched by the smaller one's scale, nor by keys of zeros."""
    pool = Pool(2, 1, 64, 16, 1, 4, seed=11)
    for scale in (1e-3, 1e3, 1.0, 0.0):
        pool.append([16], scale=scale)
    q, out = _randn(pool.gen, 1, 128, scale=1e-3), torch.empty(1, 128, dtype=F16, device="cuda")
    pool.cache.attend(q, pool.batch([1], starts=[63]), out)
    _near(out, *_attended(pool, q, [1], [63]), F16)


def test_a_pool_past_32_bit_offsets():
    """Pages whose bytes lie past 2^32 of the pool."""
    kv, hd, page = 8, 128, 256
    pages = (5 << 30) // (kv * 2 * page * hd)
    cache = sg.PagedKvCache(8, kv, hd, pages, page)
    pool = Pool(8, kv, hd, page, 2, 3, seed=12)
    pool.cache = cache
    pool.table = _int([[pages - 1, pages - 2, 0], [1, pages - 4, pages - 3]])
    pool.append([600, 513])
    pool.check()
    q, out = _randn(pool.gen, 2, 1024), torch.empty(2, 1024, dtype=F16, device="cuda")
    cache.attend(q, pool.batch([1, 1], starts=[599, 512]), out)
    _near(out, *_attended(pool, q, [1, 1], [599, 512]), F16)


# ------------------------------------------------------------------------------------------------ packed prompts

def _prompt(q, k, v, rows, heads, kv, scale=None):
    """(causal attention in 64 bits, bound before the last rounding): a probability's rounding to the type moves the result by half a step of A, the weighted
    mean of |v|; a score's chain is hd / 16 steps of 32 bits, cut off, over sum |q| |k|; the values' chain one step per 16 keys; 2^-20 of
    the score for the exponential."""
    hd = q.shape[1] // heads
    scale = hd ** -0.5 if scale is None else scale
    out, tol = torch.zeros(len(q), heads, hd, dtype=torch.float64, device="cuda"), torch.zeros(len(q), heads, hd, dtype=torch.float64, device="cuda")
    r0 = 0
    for r in rows:
        if r:
            qq, kk, vv = (x[r0:r0 + r].double().reshape(r, -1, hd) for x in (q, k, v))
            kk, vv = kk.repeat_interleave(heads // kv, 1), vv.repeat_interleave(heads // kv, 1)
            on = torch.ones(r, r, dtype=torch.bool, device="cuda").tril()
            for h in range(heads):
                z = (qq[:, h] @ kk[:, h].T * scale).masked_fill(~on, -math.inf)
                mag = (qq[:, h].abs() @ kk[:, h].abs().T * scale).masked_fill(~on, 0).amax(-1)
                e = (hd / 16 + 4) * 2.0 ** -23 * mag + 2.0 ** -20 * z.masked_fill(~on, 0).abs().amax(-1)
                p = torch.softmax(z, -1)
                out[r0:r0 + r, h] = p @ vv[:, h]
                tol[r0:r0 + r, h] = (p @ vv[:, h].abs()) * (_half_step(q.dtype) + 4 * e + (r / 16 + 16) * 2.0 ** -23)[:, None]
        r0 += r
    return out.reshape(len(q), -1), tol.reshape(len(q), -1)


PROMPTS = [(6, 6, 64, [200], F16, 1.0), (1, 1, 64, [1], F16, 1.0), (32, 8, 128, [129, 1, 0, 128, 300], BF16, 1.0), (8, 1, 128, [77, 5, 1000], F16, 3.0),
           (3, 3, 8, [64, 65], F16, 1.0), (12, 4, 80, [31, 257], BF16, 2.0), (16, 2, 256, [100, 40], F16, 1.0), (28, 4, 96, [513], F16, 1.0), (5, 5, 40, [3, 2, 1], BF16, 1.0),
           (14, 2, 112, [260, 9], BF16, 1.0), (4, 2, 200, [150], F16, 1.0), (2, 2, 128, [2000, 3], F16, 6.0), (48, 1, 64, [90, 200], F16, 1.0),
           (160, 1, 16, [40], F16, 1.0), (20, 20, 64, [1] * 70, F16, 1.0)]


@pytest.mark.parametrize("heads,kv,hd,rows,dtype,q_scale", PROMPTS)
@pytest.mark.parametrize("pad,shift", [(0, 0), (8, 8), (3, 1)])
def test_packed_prompts(heads, kv, hd, rows, dtype, q_scale, pad, shift):
    gen = _gen(heads + hd + len(rows))
    total, width = sum(rows), (heads + 2 * kv) * hd + pad
    buf = _randn(gen, (total + 2) * width + shift, dtype=dtype)
    x = buf[shift:].view(total + 2, width)
    q, k, v = x[:, :heads * hd], x[:, heads * hd:(heads + kv) * hd], x[:, (heads + kv) * hd:(heads + 2 * kv) * hd]
    q.mul_(q_scale)
    x[total:] = math.nan                                        # rows behind the last sequence
    out = torch.full((total + 2, heads * hd + pad), 5.0, dtype=dtype, device="cuda")
    cu = _int([0] + np.cumsum(rows).tolist())
    sg.attend_packed(q, k, v, cu, out[:, :heads * hd], heads, kv)
    want, tol = _prompt(q[:total], k[:total], v[:total], rows, heads, kv)
    _near(out[:total, :heads * hd], want, tol, dtype)
    assert torch.all(out[total:] == 5.0) and torch.all(out[:, heads * hd:] == 5.0)


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("kind", [math.inf, -math.inf, math.nan])
def test_non_finite_values_keys_and_queries_of_packed_prompts(hd, kind):
    """A row is finite exactly where what it attends to is: an infinity among the values of a later position, or of the next sequence, does not reach it."""
    gen = _gen(hd)
    heads, kv, rows = 4, 2, [200, 60]
    q, k, v = _randn(gen, 260, heads * hd), _randn(gen, 260, kv * hd), _randn(gen, 260, kv * hd)
    v[150, 5] = kind                                            # sequence 0, KV head 0
    v[200, hd + 7] = kind                                       # sequence 1's first row, KV head 1
    out = torch.empty_like(q)
    sg.attend_packed(q, k, v, _int([0, 200, 260]), out, heads, kv)
    clean = v.clone()
    clean[150, 5], clean[200, hd + 7] = 0.0, 0.0
    want, tol = _prompt(q, k, clean, rows, heads, kv)
    hit = torch.zeros(260, heads, hd, dtype=torch.bool, device="cuda")
    hit[150:200, :2, 5] = True
    hit[200:, 2:, 7] = True
    hit = hit.reshape(260, -1)
    assert not torch.isfinite(out[hit]).any()
    if kind == kind:
        assert torch.all(out[hit] == kind)
    _near(out[~hit], want[~hit], tol[~hit], F16)
    # a key that is not finite spoils the rows that attend to it and no other; so does a query its own row
    v, k2, q2 = clean, k.clone(), q.clone()
    k2[150, 3], q2[20, hd + 1] = math.nan, math.nan
    sg.attend_packed(q2, k2, v, _int([0, 200, 260]), out, heads, kv)
    hit = torch.zeros(260, heads, hd, dtype=torch.bool, device="cuda")
    hit[150:200, :2] = True
    hit[20, 1] = True
    hit = hit.reshape(260, -1)
    assert torch.isnan(out[hit]).all()
    _near(out[~hit], want[~hit], tol[~hit], F16)


def test_equal_and_extreme_scores():
    """Zero queries weigh all keys alike; large ones pick the largest; a scale of zero and a negative one are scales too."""
    gen = _gen(2)
    heads, kv, hd, n = 4, 2, 64, 300
    k, v = _randn(gen, n, kv * hd), _randn(gen, n, kv * hd)
    out = torch.empty(n, heads * hd, dtype=F16, device="cuda")
    for q, scale in ((torch.zeros(n, heads * hd, dtype=F16, device="cuda"), None), (_randn(gen, n, heads * hd, scale=2000.0), 1.0), (_randn(gen, n, heads * hd), 0.0),
                     (_randn(gen, n, heads * hd), -0.3)):
        sg.attend_packed(q, k, v, _int([0, n]), out, heads, kv, scale=scale)
        want, tol = _prompt(q, k, v, [n], heads, kv, scale)
        if scale == 1.0:                                        # two scores that the bound cannot tell apart: nothing to say
            keep = tol < 0.05
            assert keep.any()
            _near(out[keep], want[keep], tol[keep], F16)
        else:
            _near(out, want, tol + (2.0 ** -20 if scale is not None and scale < 0 else 0), F16)


# ------------------------------------------------------------------------------------------------ together, as they are used

def test_prompts_then_tokens_one_layer():
    """Prompts through append + attend_packed, then tokens through append + attend, as a server does, against 64 bits over the unquantised values: the cache's own
    half codes are added to the bound."""
    gen = _gen(21)
    heads, kv, hd, page, prompts = 8, 2, 64, 16, [70, 1, 33]
    rotary, qn, kn = sg.Rotary(hd), _norm(gen, hd), _norm(gen, hd)
    pool = Pool(heads, kv, hd, page, 3, 8, seed=21)
    total = sum(prompts)
    x = _randn(gen, total, (heads + 2 * kv) * hd)
    q, k, v = x.split([heads * hd, kv * hd, kv * hd], 1)
    batch = pool.batch(prompts)
    pool.cache.append(k, v, batch, rotary, q=q, q_out=q, k_out=k, q_norm=qn, k_norm=kn)
    out = torch.empty(total, heads * hd, dtype=F16, device="cuda")
    sg.attend_packed(q, k, v, batch.cu_rows, out, heads, kv)
    _near(out, *_prompt(q, k, v, prompts, heads, kv), F16)
    # the same rows over the cache: the same but for the codes
    pool.have = list(prompts)
    again = torch.empty_like(out)
    pool.cache.attend(q, batch, again)
    _near(again, *_attended(pool, q, prompts, [0, 0, 0]), F16)
    assert (again - out).abs().max() < 0.1
    for step in range(20):
        y = _randn(gen, 3, (heads + 2 * kv) * hd)
        q, k, v = y.split([heads * hd, kv * hd, kv * hd], 1)
        batch = pool.batch([1, 1, 1])
        want_q, tol_q = _turned(q, hd, batch.starts, rotary, qn)
        pool.cache.append(k, v, batch, rotary, q=q, q_out=q, q_norm=qn, k_norm=kn)
        _near(q, want_q, tol_q, F16)
        pool.have = [n + 1 for n in pool.have]
        out = torch.empty(3, heads * hd, dtype=F16, device="cuda")
        pool.cache.attend(q, batch, out)
        _near(out, *_attended(pool, q, [1, 1, 1], [n - 1 for n in pool.have]), F16)


def test_a_captured_step_is_replayed_with_other_lengths_pages_and_rows():
    gen = _gen(31)
    heads, kv, hd, page, n = 8, 2, 64, 16, 4
    rotary = sg.Rotary(hd)
    pool = Pool(heads, kv, hd, page, n, 10, seed=31)
    pool.append([3, 90, 16, 40])
    x = torch.zeros(n, (heads + 2 * kv) * hd, dtype=F16, device="cuda")
    q, k, v = x.split([heads * hd, kv * hd, kv * hd], 1)
    batch = pool.batch([1] * n)
    q_out, out = torch.empty(n, heads * hd, dtype=F16, device="cuda"), torch.empty(n, heads * hd, dtype=F16, device="cuda")

    def step():
        pool.cache.append(k, v, batch, rotary, q=q, q_out=q_out)
        pool.cache.attend(q_out, batch, out)

    step()                                                      # (the frequencies are on the device from the first call on)
    graphs = []
    for _ in range(2):                                          # two graphs of the same step: no memory of a call is shared
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            step()
        graphs.append(g)
    for i, idle in enumerate(((), (2,), (), (0, 3), ())):
        x.copy_(_randn(gen, *x.shape))
        starts = [-1 if s in idle else have for s, have in enumerate(pool.have)]
        batch.starts.copy_(_int(starts))
        graphs[i % 2].replay()
        pool.have = [have + (s not in idle) for s, have in enumerate(pool.have)]
        want, tol = _attended(pool, q_out, [1] * n, starts)
        _near(out, want, tol, F16)
        assert all(not out[s].any() for s in idle)


def test_two_streams_at_once_and_a_repeat_give_the_same_bits():
    pool = Pool(32, 8, 128, 64, 4, 60, seed=41)
    pool.append([3000, 100, 1700, 2500])
    q = [_randn(pool.gen, 4, 32 * 128) for _ in range(2)]
    batch = pool.batch([1] * 4, starts=[n - 1 for n in pool.have])
    want = []
    for x in q:
        o = torch.empty_like(x)
        pool.cache.attend(x, batch, o)
        want.append(o)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[torch.empty_like(q[0]) for _ in range(20)] for _ in range(2)]
    for i in range(20):
        for j, s in enumerate(streams):
            with torch.cuda.stream(s):
                pool.cache.attend(q[j], batch, got[j][i])
    torch.cuda.synchronize()
    for j in range(2):
        assert all(torch.equal(o, want[j]) for o in got[j])
    gen = _gen(42)
    x = _randn(gen, 700, 48 * 128)
    qq, k, v = x.split([32 * 128, 8 * 128, 8 * 128], 1)
    outs = [torch.empty(700, 32 * 128, dtype=F16, device="cuda") for _ in range(6)]
    for i, o in enumerate(outs):
        with torch.cuda.stream(streams[i % 2]):
            sg.attend_packed(qq, k, v, _int([0, 300, 700]), o, 32, 8)
    torch.cuda.synchronize()
    assert all(torch.equal(o, outs[0]) for o in outs)


def _layer(gen, d, heads, kv, hd, rotary, norms):
    w = lambda n, k: (torch.randn(n, k, generator=gen, device="cuda") * k ** -0.5).cpu().numpy()  # noqa: E731
    lin = lambda n, k: sg.Linear.quantize(w(n, k), sg.WeightLayout.OutIn, n, k)  # noqa: E731
    attn = sg.SelfAttention.new(lin((heads + 2 * kv) * hd, d), lin(d, heads * hd), heads, kv, hd)
    if rotary is not None or norms:
        attn.with_rotary(rotary, *((_norm(gen, hd), _norm(gen, hd)) if norms else (None, None)))
    n1, n2 = (sg.Norm.rms(np.ones(d, np.float32), 1e-6) for _ in range(2))
    mlp = sg.Mlp.gated(sg.GatedLinear.quantize(w(3 * d // 2, d), w(3 * d // 2, d), sg.WeightLayout.OutIn, 3 * d // 2, d, sg.Gate.Silu), lin(d, 3 * d // 2))
    return sg.Block.new(n1, attn, n2, mlp)


@pytest.mark.parametrize("rotate,norms", [(True, True), (True, False), (False, True), (False, False)])
def test_layer_on_a_packed_batch_is_its_parts(rotate, norms):
    """Block.accumulate_batch: prompts, then a step with an idle sequence and a padded row, the same bits as its parts run in turn."""
    gen = _gen(51)
    d, heads, kv, hd, page = 256, 4, 2, 64, 16
    block = _layer(gen, d, heads, kv, hd, sg.Rotary(hd) if rotate else None, norms)
    attn = block.attn
    cache, parts = attn.paged_cache(40, page), attn.paged_cache(40, page)
    table = torch.randperm(40, generator=gen, device="cuda")[:30].reshape(3, 10).to(torch.int32)
    have = [0, 0, 0]
    for rows, pad, idle, fresh in (([20, 1, 70], 0, (), True), ([1, 1, 1], 1, (1,), False), ([5, 0, 2], 2, (), False)):
        m = sum(rows) + pad
        batch = sg.PagedBatch(_int([0] + np.cumsum(rows).tolist()), _int([-1 if s in idle else n for s, n in enumerate(have)]), table)
        x = torch.randn(m, d, generator=gen, device="cuda")
        y = x.clone()
        block.accumulate_batch(x, cache, batch, m, fresh)
        h = torch.empty(m, d, dtype=F16, device="cuda")
        block.norm1.forward(y, h)
        qkv = torch.empty(m, (heads + 2 * kv) * hd, dtype=F16, device="cuda")
        attn.qkv.forward(h, qkv, m)
        q, k, v = qkv.split([heads * hd, kv * hd, kv * hd], 1)
        q2, k2 = q.clone(), k.clone()
        parts.append(k, v, batch, attn.rotary, q=q, q_out=q2, k_out=k2, q_norm=attn.q_norm, k_norm=attn.k_norm)
        att = torch.zeros(m, heads * hd, dtype=F16, device="cuda")
        if fresh:
            sg.attend_packed(q2, k2, v, batch.cu_rows, att, heads, kv)
        else:
            parts.attend(q2, batch, att)
        attn.out.accumulate(att, y, m)
        block.norm2.forward(y, h)
        block.mlp.accumulate(h, y, m)
        assert torch.equal(x, y) and torch.equal(cache.codes, parts.codes) and torch.equal(cache.scales, parts.scales)
        assert not att[sum(rows):].any()
        have = [n + (0 if s in idle else r) for s, (n, r) in enumerate(zip(have, rows))]


def test_rotated_layer_on_the_f16_cache():
    """SelfAttention.with_rotary on a KvCache: prompt, then tokens, against the packed form of the whole sequence (the same rotated 16-bit rows; the f16 cache's attention is
    within 2e-5 of the packed one's 64-bit result, whose own bound holds), and a Block of it, which runs by its parts."""
    gen = _gen(52)
    d, heads, kv, hd, n = 256, 4, 2, 64, 50
    block = _layer(gen, d, heads, kv, hd, sg.Rotary(hd, rotary_dim=32).linear(2.0), True)
    attn = block.attn
    x = _randn(gen, n, d)
    cache = attn.cache(n)
    got = torch.cat([attn.attend(x[:41], cache, 41)] + [attn.attend(x[i:i + 1], cache, 1) for i in range(41, n)])
    k, v = cache.keys(), cache.values()                          # rotated, as cached
    qkv = torch.cat([torch.empty(0, (heads + 2 * kv) * hd, dtype=F16, device="cuda")] + [_forward(attn.qkv, x[a:b]) for a, b in [(0, 41)] + [(i, i + 1) for i in range(41, n)]])
    pos = torch.arange(n, device="cuda")
    want_k, tol_k = _turned(qkv[:, heads * hd:(heads + kv) * hd], hd, pos, attn.rotary, attn.k_norm)
    _near(k, want_k, tol_k, F16)
    q = torch.empty(n, heads * hd, dtype=F16, device="cuda")
    sg.rotate_heads(qkv[:, :heads * hd], None, 0, attn.rotary, q, None, q_norm=attn.q_norm)
    want, tol = _prompt(q, k, v, [n], heads, kv)
    _near(got, want, tol + 2e-5 * (1 + want.abs()), F16)
    # a whole layer: the native form does not take it, its parts do
    y = torch.randn(9, d, generator=gen, device="cuda")
    z, c1, c2 = y.clone(), block.cache(9), block.cache(9)
    block.accumulate(y, c1, 9)
    h = torch.empty(9, d, dtype=F16, device="cuda")
    block.norm1.forward(z, h)
    attn.accumulate(h, c2, z, 9)
    block.norm2.forward(z, h)
    block.mlp.accumulate(h, z, 9)
    assert torch.equal(y, z)
    with pytest.raises(AssertionError, match="heads of head_dim"):
        attn.with_rotary(sg.Rotary(128))
    with pytest.raises(AssertionError, match="RMS norms"):
        attn.with_rotary(None, sg.Norm.rms(np.ones(32, np.float32), 1e-6))


def _forward(lin, x):
    y = torch.empty(len(x), lin.n(), dtype=F16, device="cuda")
    lin.forward(x.contiguous(), y, len(x))
    return y


def test_refusals_with_tensors_on_the_device():
    cache = sg.PagedKvCache(4, 2, 32, 5, 16)
    assert (cache.heads(), cache.kv_heads(), cache.head_dim(), cache.pages(), cache.page(), cache.row_len(), cache.query_len()) == (4, 2, 32, 5, 16, 64, 128)
    assert cache.with_scale(0.5).scale() == 0.5
    cu, starts, table = _int([0, 2]), _int([0]), _int([[0, 1]])
    batch = sg.PagedBatch(cu, starts, table)
    assert batch.seqs() == 1
    r = lambda rows, width, dtype=F16: torch.zeros(rows, width, dtype=dtype, device="cuda")  # noqa: E731
    for bad, message in [
            (lambda: sg.PagedBatch(cu, _int([0, 1]), table), "one value more"), (lambda: sg.PagedBatch(_int([0, 1, 2]), _int([0, 0]), table), "a row of pages"),
            (lambda: sg.PagedBatch(cu.long(), starts, table), "int32"), (lambda: cache.append(r(2, 64), r(2, 63), batch), "rows of 64"),
            (lambda: cache.append(r(2, 64), r(3, 64), batch), "as many rows"), (lambda: cache.append(r(2, 64), r(2, 64, BF16), batch), "same type"),
            (lambda: cache.append(r(2, 64, torch.float32), r(2, 64, torch.float32), batch), "f16 or bf16"),
            (lambda: cache.append(r(64, 2).T, r(2, 64), batch), "side by side"), (lambda: cache.append(r(2, 64), r(2, 64), batch, q=r(2, 128)), "come together"),
            (lambda: cache.append(r(2, 64), r(2, 64), batch, sg.Rotary(64)), "heads of head_dim"),
            (lambda: cache.append(r(2, 64), r(2, 64), batch, k_norm=sg.Norm.rms(np.ones(16, np.float32), 1e-6)), "head_dim weights"),
            (lambda: cache.append(r(2, 64), r(2, 64), batch, k_norm=sg.Norm.layer(np.ones(32, np.float32), None, 1e-6)), "RMS norm"),
            (lambda: cache.attend(r(2, 64), batch, r(2, 128)), "rows of 128"), (lambda: cache.attend(r(2, 128), batch, r(1, 128)), "as many rows"),
            (lambda: cache.read(_int([0]), r(1, 4)), "n pages"), (lambda: cache.read(table.long(), r(1, 4)), "int32"),
            (lambda: sg.attend_packed(r(2, 128), r(2, 64), r(2, 64), cu.long(), r(2, 128), 4, 2), "int32"),
            (lambda: sg.attend_packed(r(2, 128), r(2, 32), r(2, 64), cu, r(2, 128), 4, 2), "rows of 64"),
            (lambda: sg.rotate_heads(r(2, 128), None, _int([1]), sg.Rotary(32), r(2, 128), None), "one value a row"),
            (lambda: sg.rotate_heads(r(2, 120), None, 0, sg.Rotary(32), r(2, 120), None), "whole heads")]:
        with pytest.raises(AssertionError, match=message):
            bad()
    # nothing to do
    cache.append(r(0, 64), r(0, 64), batch)
    cache.attend(r(0, 128), batch, r(0, 128))
    cache.read(_int([]), r(0, 1))
    sg.attend_packed(r(0, 128), r(0, 64), r(0, 64), _int([0]), r(0, 128), 4, 2)
    sg.rotate_heads(r(0, 128), None, 0, sg.Rotary(32), r(0, 128), None)


# ------------------------------------------------------------------------------------------------ calls at the edges

def test_more_narrow_heads_than_a_warp_has_lanes():
    """Heads of 16 depths are two lanes each: 64 of them in a block at a time, and 40 are more than a page's CTA takes."""
    seqs = 80
    pool = Pool(80, 40, 16, 16, seqs, 3, seed=40)
    rotary, kn = sg.Rotary(16), _norm(pool.gen, 16)
    pool.append([3] * seqs, (), rotary, kn)
    pool.append([1] * seqs, (7,), rotary, kn)
    pool.append([20] * seqs, (), rotary, kn)
    pool.check(times=3)


@pytest.mark.parametrize("hd", [64, 128, 256])
def test_values_that_are_lost_altogether(hd):
    """From position 100 on no value is finite: NaNs, infinities of one sign, of both in turn.  A row has what the sum over what it attends to has."""
    gen = _gen(hd + 1)
    heads, kv, n = 4, 2, 700
    q, k, v0 = _randn(gen, n, heads * hd), _randn(gen, n, kv * hd), _randn(gen, n, kv * hd)
    want, tol = _prompt(q[:100], k[:100], v0[:100], [100], heads, kv)
    for kind in ("nan", "inf", "both"):
        v = v0.clone()
        v[100:] = math.nan if kind == "nan" else math.inf
        if kind == "both":
            v[101::2] = -math.inf
        out = torch.empty_like(q)
        sg.attend_packed(q, k, v, _int([0, n]), out, heads, kv)
        _near(out[:100], want, tol, F16)
        if kind == "inf":
            assert torch.all(out[100:] == math.inf)
        else:
            assert torch.isnan(out[101:]).all() and torch.all(out[100] == math.inf if kind == "both" else torch.isnan(out[100]))


@pytest.mark.parametrize("size", [1e25, 1e31, 1e37])
def test_queries_near_the_largest_numbers(size):
    """bf16 queries so large that a row's best key has all the weight: the result is that key's value, to a rounding and the offset's error."""
    pool = Pool(8, 2, 64, 16, 1, 4, seed=5, dtype=BF16)
    pool.append([50])
    q = _randn(pool.gen, 4, 512, dtype=BF16) * size
    assert torch.isfinite(q).all()
    out = torch.empty_like(q)
    pool.cache.attend(q, pool.batch([4], starts=[46]), out)
    assert torch.isfinite(out).all()
    x, sc = pool.values(0)
    k, v = x.repeat_interleave(4, 2)
    z = torch.einsum("rhd,nhd->rhn", q.double().reshape(4, 8, 64), k)
    z = z.masked_fill(torch.arange(50, device="cuda")[None, None, :] > 46 + torch.arange(4, device="cuda")[:, None, None], -math.inf)
    top = z.topk(2, -1)
    clear = (top.values[..., 0] - top.values[..., 1]) > 2.0 ** -10 * z.masked_fill(z == -math.inf, 0).abs().amax(-1)
    assert clear.sum() > 16
    best = v[top.indices[..., 0], torch.arange(8, device="cuda")[None, :]]
    room = best.abs() * (2.0 ** -8 + 2.0 ** -10) + 2.0 ** -18 * 255 * sc.amax()
    assert torch.all(((out.double().reshape(4, 8, 64) - best).abs() <= room)[clear])


def test_the_first_call_with_a_rotation_is_not_captured():
    rotary, q, out = sg.Rotary(32), torch.ones(2, 64, dtype=F16, device="cuda"), torch.zeros(2, 64, dtype=F16, device="cuda")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        with pytest.raises(AssertionError, match="before a capture"):
            sg.rotate_heads(q, None, 0, rotary, out, None)
        out.add_(1.0)
    g.replay()
    assert torch.all(out == 1.0)
    sg.rotate_heads(q, None, 0, rotary, out, None)
    again, h = torch.zeros_like(out), torch.cuda.CUDAGraph()
    with torch.cuda.graph(h):
        sg.rotate_heads(q, None, 0, rotary, again, None)
    h.replay()
    assert torch.equal(again, out)


def test_refusals_of_overlaps_and_of_tables_without_pages():
    q, k = torch.zeros(4, 128, dtype=F16, device="cuda"), torch.zeros(4, 64, dtype=F16, device="cuda")
    with pytest.raises(AssertionError, match="none of the inputs"):
        sg.attend_packed(q, k, k, _int([0, 4]), q, 4, 2)
    with pytest.raises(AssertionError, match="a page for each"):
        sg.PagedBatch(_int([0, 4]), _int([0]), torch.zeros(1, 0, dtype=torch.int32, device="cuda"))
    assert sg.PagedBatch(_int([0]), torch.zeros(0, dtype=torch.int32, device="cuda"), torch.zeros(0, 3, dtype=torch.int32, device="cuda")).seqs() == 0


@pytest.mark.parametrize("kv,rows", [(3, [3, 1, 9]), (1, [5, 2, 70])])
def test_a_norm_without_an_eps(kv, rows):
    """Lanes without a row have nothing to normalise: no NaN of theirs reaches a scale."""
    pool = Pool(2 * kv, kv, 64, 16, 3, 8, seed=kv)
    norm = sg.Norm.rms(np.ones(64, np.float32), 0.0)
    pool.append(rows, (), sg.Rotary(64), norm)
    pool.append([1, 1, 1], (), sg.Rotary(64), norm)
    pool.check(times=2)


@pytest.mark.parametrize("heads,kv,hd,page,lens,rows,dtype", [
    (32, 8, 128, 64, [9000], [1], F16), (32, 8, 128, 64, [200 + 29 * i for i in range(50)], [1] * 50, BF16), (24, 3, 64, 16, [3000, 2500, 10], [5, 5, 5], F16),
    (6, 6, 64, 32, [7000, 1], [1, 1], F16), (16, 2, 256, 64, [6000, 4000], [2, 1], BF16), (4, 4, 80, 128, [40 * i + 1 for i in range(60)], [1] * 60, F16)])
def test_long_contexts_and_many_sequences(heads, kv, hd, page, lens, rows, dtype):
    """Keys shared out evenly over the machine, the cut items joined afterwards: item by item and cut by cut."""
    pool = Pool(heads, kv, hd, page, len(lens), -(-max(lens) // page) + 1, seed=len(lens) + hd, dtype=dtype)
    pool.append(lens)
    starts = [n - r for n, r in zip(lens, rows)]
    q = _randn(pool.gen, sum(rows), heads * hd, dtype=dtype)
    out = torch.full_like(q, 5.0)
    pool.cache.attend(q, pool.batch(rows, starts=starts), out)
    want, tol = _attended(pool, q, rows, starts)
    _near(out, want, tol, dtype)


@pytest.mark.parametrize("heads,kv,hd,dtype", [(16, 2, 256, F16), (12, 4, 192, BF16), (16, 2, 128, F16), (8, 8, 64, BF16)])
def test_prompts_whose_warps_run_apart(heads, kv, hd, dtype):
    """Sequences that end inside tiles and scores whose maxima move: a warp may be a block ahead of the others, and its results wait for all products all the same.  Every
    run gives the same bits."""
    gen = _gen(hd)
    rows = [289, 245, 272, 261, 250, 277, 266, 255, 283, 244, 271, 260, 303]
    total = sum(rows)
    cu = _int([0] + np.cumsum(rows).tolist())
    first = None
    for run in range(12):
        if run % 4 == 0:
            q, k, v = _randn(gen, total, heads * hd, dtype=dtype, scale=1.5), _randn(gen, total, kv * hd, dtype=dtype), _randn(gen, total, kv * hd, dtype=dtype)
            k += torch.linspace(0, 1, total, device="cuda").to(dtype)[:, None] * k          # later keys are larger: maxima move along
            want, tol = _prompt(q, k, v, rows, heads, kv)
            first = None
        out = torch.full_like(q, 7.0)
        sg.attend_packed(q, k, v, cu, out, heads, kv)
        if first is None:
            first = out
            _near(out, want, tol, dtype)
        assert torch.equal(out, first)


def _lost(v, rows, heads, kv):
    """What the infinities and NaNs among v leave of each result whose weights are all above zero: 0 nothing, +-inf, NaN ([rows, heads * head_dim], 64 bits)."""
    out = []
    r0 = 0
    for r in rows:
        x = v[r0:r0 + r].double().reshape(r, kv, -1)
        nan, up, down = (torch.cummax(y.to(torch.int8), 0).values.bool() for y in (torch.isnan(x), x == math.inf, x == -math.inf))
        y = torch.zeros_like(x)
        y[up], y[down], y[nan | (up & down)] = math.inf, -math.inf, math.nan
        out.append(y.repeat_interleave(heads // kv, 1).reshape(r, -1))
        r0 += r
    return torch.cat(out)


@pytest.mark.parametrize("heads,kv,hd,dtype,shift", [(8, 2, 64, F16, 0), (8, 2, 128, BF16, 0), (4, 2, 256, F16, 0), (6, 1, 80, BF16, 0), (3, 3, 96, F16, 0), (4, 2, 192, BF16, 0),
                                                     (8, 2, 64, BF16, 1), (8, 2, 128, F16, 1), (2, 2, 256, F16, 1), (5, 5, 40, F16, 1),
                                                     (32, 8, 64, F16, 0), (32, 8, 128, BF16, 0)])
@pytest.mark.parametrize("kind", ["channel", "down", "scattered", "late"])
def test_infinities_all_over_the_values_of_packed_prompts(heads, kv, hd, dtype, shift, kind):
    """A depth that is infinite at every position, infinities and NaNs at every hundredth, one at the end of each sequence: each result is the sum over what its row attends to.
    (With 32 heads there are more items of work than SMs.)"""
    gen = _gen(hd + len(kind))
    rows = [1400, 33, 1300] if heads == 32 else [700, 33, 300]
    total = sum(rows)
    width = (heads + 2 * kv) * hd + 8
    x = _randn(gen, total * width + shift, dtype=dtype)[shift:].view(total, width)
    q, k, v = x[:, :heads * hd], x[:, heads * hd:(heads + kv) * hd], x[:, (heads + kv) * hd:(heads + 2 * kv) * hd]
    if kind in ("channel", "down"):
        v[:, 5] = math.inf if kind == "channel" else -math.inf
    elif kind == "late":
        v[[rows[0] - 10, rows[0] + 32, total - 1], hd - 3] = torch.tensor([math.inf, math.nan, -math.inf], device="cuda", dtype=dtype)
    else:
        at = torch.rand(v.shape, generator=gen, device="cuda") < 0.01 / hd
        v[at] = torch.tensor([math.inf, -math.inf, math.nan], device="cuda", dtype=dtype)[torch.randint(0, 3, v.shape, generator=gen, device="cuda")][at]
    out = torch.empty(total, heads * hd, dtype=dtype, device="cuda")
    sg.attend_packed(q, k, v, _int([0] + np.cumsum(rows).tolist()), out, heads, kv)
    lost = _lost(v, rows, heads, kv)
    clean = torch.where(torch.isfinite(v), v, torch.zeros_like(v))
    want, tol = _prompt(q, k, clean, rows, heads, kv)
    whole = lost == 0
    assert whole.any() and not whole.all()
    _near(out[whole], want[whole], tol[whole], dtype)
    assert torch.equal(out[~whole].double().nan_to_num(7.0, posinf=8.0, neginf=9.0), lost[~whole].nan_to_num(7.0, posinf=8.0, neginf=9.0))


def test_an_infinite_channel_costs_no_pass_of_single_values():
    """Every row of such a prompt is formed again.  Warp-level products take some ten times as long as the others, their operands come from the L2 cache piece by piece, which
    doubles that, and a pass comes before: 25 times at most, where a key at a time for each row took hundreds."""
    gen = _gen(77)
    heads, kv, hd, n = 32, 8, 128, 4096
    q, k, v = _randn(gen, n, heads * hd), _randn(gen, n, kv * hd), _randn(gen, n, kv * hd)
    bad = v.clone()
    bad.view(n, kv, hd)[:, :, 9] = math.inf
    out, cu, took = torch.empty_like(q), _int([0, n]), []
    for x in (v, bad):
        times = []
        for _ in range(6):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            sg.attend_packed(q, k, x, cu, out, heads, kv)
            b.record()
            b.synchronize()
            times.append(a.elapsed_time(b))
        took.append(min(times[1:]))
    assert torch.all(out.view(n, heads, hd)[:, :, 9] == math.inf) and torch.isfinite(out.view(n, heads, hd)[:, :, :9]).all()
    assert took[1] < 25 * took[0], took


@pytest.mark.parametrize("heads,kv,hd,dtype,ratio", [(2, 1, 64, F16, 2.0 ** -14), (8, 1, 128, BF16, 2.0 ** -20), (4, 2, 256, BF16, 2.0 ** -40), (24, 1, 64, BF16, 2.0 ** -60), (2, 2, 128, F16, 2.0 ** -9)])
@pytest.mark.parametrize("small_first", [True, False])
def test_pages_of_small_values_beside_pages_of_large_ones(heads, kv, hd, dtype, ratio, small_first):
    """Two pages of 16 of one piece of 32 keys, the values of one far below the other's: rows that attend to the first page alone, and rows whose weights lie on the small one.  The
    bound counts a page's scale with its weight: an error of a product's steps is one of what the product adds."""
    pool = Pool(heads, kv, hd, 16, 1, 6, seed=hd + heads, dtype=dtype)
    group, n = heads // kv, 64
    k, v = (_randn(pool.gen, n, kv * hd, dtype=dtype, scale=s) for s in (0.05, 1.0))
    small = (torch.arange(n, device="cuda") // 16 % 2 == (0 if small_first else 1))
    v[small] *= ratio
    k.view(n, kv, hd)[:, :, 0] = torch.where(small, 8.0, -8.0)[:, None].to(dtype)       # a query's first depth says how much less the large page's keys weigh
    pool.cache.append(k, v, pool.batch([n]))
    pool.have = [n]
    start, rows = 8, n - 8
    q = _randn(pool.gen, rows, heads * hd, dtype=dtype)
    q.view(rows, heads, hd)[:, :, 0] = (torch.arange(rows, device="cuda") % 3 * 1.5 * math.sqrt(hd))[:, None].to(dtype)   # e^0, e^-24, e^-48
    out = torch.empty_like(q)
    pool.cache.attend(q, pool.batch([rows], starts=[start]), out)
    x, sc = pool.values(0)
    kk, vv = x.repeat_interleave(group, 2)
    sk, sv = sc.repeat_interleave(group, 2)[..., 0]
    z = torch.einsum("rhd,nhd->hrn", q.double().reshape(rows, heads, hd), kk) * pool.cache.scale()
    z = z.masked_fill(torch.arange(n, device="cuda")[None, :] > start + torch.arange(rows, device="cuda")[:, None], -math.inf)
    p = torch.softmax(z, -1)
    want, a, step = (torch.einsum("hrn,nhd->rhd", p, y) for y in (vv, vv.abs(), sv[..., None].expand(-1, -1, hd)))
    # A score's chain: (hd / 16 + 4) * 2^-23 of sum |q| * 255 * scale_k and 2^-21 of itself, four times that of the result; a probability's rounding 2^-11 of what it adds, or half
    # of f16's last place (2^-25, of probabilities that stand 2^7 higher, in sums that reach 1 at least) of its page's values, 32 keys a time
    e = (hd / 16 + 4) * 2.0 ** -23 * pool.cache.scale() * q.double().abs().reshape(rows, heads, hd).sum(-1) * 255 * sk.amax() + 2.0 ** -21 * z.masked_fill(z == -math.inf, 0).abs().amax(-1).T
    on = (z > -math.inf).to(torch.float64)
    floor = torch.einsum("hrn,nhd->rhd", on, vv.abs()) * 2.0 ** -32
    tol = a * (2.0 ** -11 + 2.0 ** -18 + 4 * e[..., None]) + 2.0 ** -20 * 255 * step + floor * 2.0
    _near(out.view(rows, heads, hd), want, tol, dtype)
    lone = out.view(rows, heads, hd)[:8]                          # rows of the first page alone
    assert lone.abs().amax() > 0


@pytest.mark.parametrize("cols,seqs", [(2, 3), (40, 3), (60, 70)])
def test_rows_behind_the_table_attend_to_what_it_has_room_for(cols, seqs):
    """By clusters, by shares item by item and cut by cut: such rows attend to all positions of the table, and bit 3 of the status tells."""
    pool = Pool(8, 2, 64, 64, seqs, cols, seed=cols)
    room = cols * 64
    pool.append([room] * seqs)
    q = _randn(pool.gen, 2 * seqs, 512)
    for start in (room - 1, room, room + 100, 2 ** 31 - 2, 2 ** 31 - 1):
        starts = [5] + [start] * (seqs - 1)
        out = torch.full_like(q, 7.0)
        pool.cache.attend(q, pool.batch([2] * seqs, starts=starts), out)
        assert sg.last_status() == 8
        want, tol = _attended(pool, q, [2] * seqs, starts)
        _near(out, want, tol, F16)
    pool.cache.attend(q, pool.batch([2] * seqs, starts=[room - 2] * seqs), out)
    assert sg.last_status() == 0


def test_outputs_that_share_memory_with_other_rows():
    """Refused; slices of the same rows side by side, and an output in its own input's place, are not."""
    cache = sg.PagedKvCache(4, 2, 32, 5, 16)
    batch = sg.PagedBatch(_int([0, 4]), _int([0]), _int([[0, 1]]))
    x = torch.zeros(9, 320, dtype=F16, device="cuda")             # [q | k | v | 64 more]
    q, k, v = x[:4, :128], x[:4, 128:192], x[:4, 192:256]
    turn, cu = sg.Rotary(32), _int([0, 4])
    for bad in (lambda: sg.rotate_heads(q, k, 0, turn, x[1:5, :128], k), lambda: sg.rotate_heads(q, k, 0, turn, x[:4, 64:192], k), lambda: sg.rotate_heads(q, k, 0, turn, q, x[:4, 96:160]),
                lambda: sg.rotate_heads(q, k, 0, turn, x[:8].view(4, 640)[:, :128], k), lambda: sg.rotate_heads(k, v, 0, turn, v, k),
                lambda: cache.append(k, v, batch, turn, k_out=v), lambda: cache.append(k, v, batch, turn, k_out=k, q=q, q_out=x[:4, 192:320]),
                lambda: cache.append(k, v, batch, turn, k_out=x[:4, 100:164]), lambda: cache.attend(q, batch, q), lambda: cache.attend(q, batch, x[3:7, :128]),
                lambda: sg.attend_packed(q, k, v, cu, x[:4, 192:320], 4, 2), lambda: sg.attend_packed(q, k, v, cu, x[:4, 8:136], 4, 2)):
        with pytest.raises(AssertionError, match="no memory with"):
            bad()
    sg.rotate_heads(q, k, 0, turn, q, k)
    sg.rotate_heads(q, None, 0, turn, x[4:8, :128], None)
    cache.append(k, v, batch, turn, k_out=k, q=q, q_out=q)
    cache.append(k, v, batch, turn, k_out=x[:4, 256:])
    cache.attend(q, batch, x[5:9, 192:])
    cache.attend(q, batch, x[:4, 192:])                           # (beside q in the same rows)
    sg.attend_packed(q, k, v, cu, x[4:8, 128:256], 4, 2)


def test_copies_of_caches_batches_and_rotations_stand_by_themselves():
    import copy
    pool = Pool(4, 2, 64, 16, 2, 4, seed=61)
    rotary = sg.Rotary(64)
    pool.append([20, 5], rotary=rotary)
    cache, other, turn = pool.cache.with_scale(0.2), copy.deepcopy(pool.cache), copy.deepcopy(rotary)
    x = _randn(pool.gen, 2, 2 * 128)
    k, v = x.split([128, 128], 1)
    batch = pool.batch([1, 1])
    twin = copy.deepcopy(batch)
    before = cache.codes.clone()
    other.append(k, v, twin, turn)
    assert torch.equal(cache.codes, before) and not torch.equal(other.codes, before) and other.scale() == cache.scale()
    cache.append(k, v, batch, rotary)
    assert torch.equal(cache.codes, other.codes) and torch.equal(cache.scales, other.scales)
    twin.starts.fill_(-1)                                        # the copy's own
    q = _randn(pool.gen, 2, 256)
    out, idle = torch.empty_like(q), torch.full_like(q, 3.0)
    cache.attend(q, batch, out)
    other.attend(q, twin, idle)
    assert out.any(1).all() and not idle.any()
    again = torch.empty_like(q)
    other.attend(q, batch, again)
    assert torch.equal(again, out)


def test_a_layer_over_sharded_heads_has_no_packed_batches():
    from sme_gemm_b200.tp import TpSelfAttention
    gen = _gen(71)
    block = _layer(gen, 256, 4, 2, 64, sg.Rotary(64), True)
    cache, batch = block.attn.paged_cache(8, 16), sg.PagedBatch(_int([0, 3]), _int([0]), _int([[0, 1]]))
    sharded = sg.Block.new(block.norm1, TpSelfAttention(block.attn, 1), block.norm2, block.mlp)
    x = torch.randn(3, 256, generator=gen, device="cuda")
    y = x.clone()
    with pytest.raises(AssertionError, match="TpSelfAttention has no packed batches"):
        sharded.accumulate_batch(x, cache, batch, 3, True)
    assert torch.equal(x, y)


# ------------------------------------------------------------------------------------------------ searches of several passes, threads

@pytest.mark.parametrize("seqs,heads,kv,hd,cols,form", [(129, 4, 1, 64, 8, "clusters"), (200, 4, 1, 64, 8, "clusters"), (250, 8, 1, 16, 10, "clusters"), (300, 4, 1, 64, 30, "shares"),
                                                        (270, 4, 1, 128, 40, "cuts")])
def test_searches_through_more_sequences_than_threads(seqs, heads, kv, hd, cols, form):
    """129 and more sequences are several passes of a CTA's search for its item (257 and more of the join's): lengths of every kind, sequences without rows, idle ones."""
    rng = np.random.default_rng(seqs)
    page = 64
    lens = [int(x) for x in rng.integers(1, cols * page + 1, seqs)]
    pool = Pool(heads, kv, hd, page, seqs, cols, seed=seqs)
    pool.append(lens)
    rows = [0 if i % 17 == 3 else 1 for i in range(seqs)]
    rows[-1] = 1
    idle = set(range(5, seqs, 23))
    starts = [-1 if s in idle else n - 1 for s, n in enumerate(lens)]
    q = _randn(pool.gen, sum(rows) + 1, heads * hd)
    out = torch.full_like(q, 5.0)
    pool.cache.attend(q, pool.batch(rows, starts=starts), out)
    want, tol = _attended(pool, q[:-1], rows, starts)
    _near(out[:-1], want, tol, F16)
    assert torch.all(out[-1] == 5.0)


def test_two_streams_whose_inputs_are_there():
    """As above, with the streams waiting for the inputs and the outputs against 64 bits."""
    gen = _gen(43)
    rows = [300, 400]
    x = _randn(gen, 700, 48 * 128)
    q, k, v = x.split([32 * 128, 8 * 128, 8 * 128], 1)
    cu = _int([0, 300, 700])
    outs = [torch.full((700, 32 * 128), 7.0, dtype=F16, device="cuda") for _ in range(8)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for i, o in enumerate(outs):
        with torch.cuda.stream(streams[i % 2]):
            sg.attend_packed(q, k, v, cu, o, 32, 8)
    torch.cuda.synchronize()
    assert all(torch.equal(o, outs[0]) for o in outs)
    _near(outs[0], *_prompt(q, k, v, rows, 32, 8), F16)


def test_two_host_threads_on_one_rotation_and_one_cache():
    """Each thread on a stream, and in sequences, of its own; the rotation's first call on the device is one of theirs."""
    import threading
    pool = Pool(8, 2, 64, 16, 2, 12, seed=81)
    rotary, steps = sg.Rotary(64), 60
    x = [[_randn(pool.gen, 1, 12 * 64) for _ in range(steps)] for _ in range(2)]
    want = [[torch.empty(1, 512, dtype=F16, device="cuda") for _ in range(steps)] for _ in range(2)]
    got = [[torch.full_like(o, 7.0) for o in w] for w in want]

    def serve(cache, turn, t, out, stream):
        with torch.cuda.stream(stream):
            for i in range(steps):
                q, k, v = x[t][i].split([512, 128, 128], 1)
                batch = batches[t][i]
                turned = torch.empty_like(q)
                cache.append(k, v, batch, turn, q=q, q_out=turned)
                cache.attend(turned, batch, out[t][i])

    batches = [[sg.PagedBatch(_int([0, 1]), _int([i]), pool.table[t:t + 1].contiguous()) for i in range(steps)] for t in range(2)]
    for t in range(2):
        serve(pool.cache, sg.Rotary(64), t, want, torch.cuda.current_stream())
    codes = pool.cache.codes.clone()
    torch.cuda.synchronize()
    failed = []

    def thread(t):
        try:
            serve(pool.cache, rotary, t, got, streams[t])
        except BaseException as e:                                # noqa: BLE001
            failed.append(e)

    streams = [torch.cuda.Stream() for _ in range(2)]
    threads = [threading.Thread(target=thread, args=(t,)) for t in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not failed, failed
    assert all(torch.equal(a, b) for t in range(2) for a, b in zip(got[t], want[t])) and torch.equal(codes, pool.cache.codes)
