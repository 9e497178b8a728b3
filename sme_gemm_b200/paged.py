"""Packed batches of sequences: rotation by position, the 8-bit paged key/value cache, attention.

What a model with rotated, normalised heads and a server with many sequences need around the projections of a self-attention block (the reference
applies no rotation, src/self_attention.rs:66-231, and keeps one f16 buffer a sequence, src/kernels/kv_attention.rs:354-581).  Tensors are CUDA
tensors of f16 or bf16 rows, heads * head_dim values each, at any row stride: slices of the [q | k | v] rows that a fused projection leaves are taken
as they are.  Every call enqueues its work on torch's current stream of the tensors' device; nothing is read back, so that all of them can be
captured into a graph (row offsets, starts and page tables are device memory).
"""
from __future__ import annotations

import math

import numpy as np

from ._lib import ATTN_PACKED_ARGS, PAGED_ATTEND_ARGS, READ_ARGS, ROTATE_ARGS, check, lib
from .host import Norm, torch

_Tensor, _F16, _BF16 = torch.Tensor, torch.float16, torch.bfloat16
_get_device, _raw_stream = getattr(torch._C, "_cuda_getDevice", None), getattr(torch._C, "_cuda_getCurrentRawStream", None)


class _On:
    """The tensors' device as the current one, for a call from elsewhere."""

    def __init__(self, device: int):
        self._device = device

    def __enter__(self):
        self._was = torch.cuda.current_device()
        if self._was != self._device:
            torch.cuda.set_device(self._device)

    def __exit__(self, *exc):
        if self._was != self._device:
            torch.cuda.set_device(self._was)


_FNS: dict = {}                                             # entry points by name


def _enqueue(name: str, device: int, args: bytes) -> None:
    """Calls `name` with the packed arguments on the current stream of `device`."""
    fn = _FNS.get(name)
    if fn is None:
        fn = _FNS[name] = getattr(lib(), name)
    if _get_device() == device:
        rc = fn(args, _raw_stream(device))
    else:
        with _On(device):
            rc = fn(args, _raw_stream(device))
    if rc:
        check(name, rc)


def _first_rows(x, what: str):
    """((type, device index), number, length) of the rows that the other tensors of a call have to be like."""
    if type(x) is _Tensor:
        dtype, shape, device = x.dtype, x.shape, x.get_device()
        if (dtype is _F16 or dtype is _BF16) and device >= 0 and len(shape) == 2:
            return (dtype, device), shape[0], shape[1]
    assert isinstance(x, torch.Tensor) and x.is_cuda, f"{what} is a CUDA tensor"
    assert x.dtype in (_F16, _BF16), f"{what} is f16 or bf16"
    assert x.dim() == 2, f"{what} has rows"
    return (x.dtype, x.get_device()), x.shape[0], x.shape[1]


def _rows(x, what: str, rows: int, width: int, like) -> int:
    """Checks a tensor of rows; their stride in elements.  (A call is some five of these checks, and a small one is over in the time they take: the
    sound case is one condition, what is wrong is found afterwards.)"""
    if type(x) is _Tensor and x.shape == (rows, width) and (x.dtype, x.get_device()) == like:
        stride, one = x.stride()
        if one == 1 and stride >= width:
            return stride
        if rows <= 1 and (one == 1 or width == 1):
            return width
    assert isinstance(x, torch.Tensor) and x.is_cuda, f"{what} is a CUDA tensor"
    assert x.dtype in (_F16, _BF16), f"{what} is f16 or bf16"
    assert x.dim() == 2 and x.shape[1] == width, f"{what} has rows of {width} values"
    assert (x.dtype, x.get_device()) == like, f"{what} has the same type and device as the other rows"
    assert x.shape[0] == rows, f"{what} has as many rows as the others"
    stride, one = x.stride()
    assert rows <= 1 or stride >= width and one == 1 or width == 1, f"{what} has its rows' values side by side"
    assert one == 1 or width == 1 or rows == 0, f"{what} has its rows' values side by side"
    return max(stride, width)


def _ints(x, what: str, device: int) -> None:
    assert isinstance(x, torch.Tensor) and x.is_cuda and x.dtype is torch.int32 and x.is_contiguous(), f"{what} is a contiguous int32 CUDA tensor"
    assert device is None or x.get_device() == device, f"{what} is on the rows' device"


def _head_norm(norm, what: str, head_dim: int, device: int):
    if norm is None:
        return 0, 0.0
    assert isinstance(norm, Norm) and norm.is_rms, f"{what} is an RMS norm"
    w = norm.weight
    assert w.numel() == head_dim, f"{what} has head_dim weights"
    assert w.get_device() == device, f"{what} is on the rows' device"
    return w.data_ptr(), norm.eps


class Rotary:
    """The rotation of heads by position: pair i of the first `rotary_dim` depths turns by position * frequency_i, frequency_i =
    base^(-2 i / rotary_dim).  A pair is (i, i + rotary_dim / 2), or (2 i, 2 i + 1) interleaved; the depths behind rotary_dim stay as they are.
    linear(), by_wavelength() and yarn() give the same rotation with its frequencies scaled for contexts longer than the trained one."""

    def __init__(self, head_dim: int, base: float = 10000.0, rotary_dim: int | None = None, interleaved: bool = False):
        rot = head_dim if rotary_dim is None else rotary_dim
        assert head_dim % 8 == 0 and 8 <= head_dim <= 256, "head_dim must be a multiple of 8 in 8..=256"
        assert rot % 2 == 0 and 2 <= rot <= head_dim, "rotary_dim is even, at least 2 and at most head_dim"
        assert base > 0.0 and math.isfinite(base), "base is positive"
        self._head_dim, self._rot, self._base, self._interleaved = head_dim, rot, float(base), bool(interleaved)
        self._set(self._base ** (-2.0 * np.arange(rot // 2, dtype=np.float64) / rot), 1.0)

    def _set(self, frequencies, factor: float) -> None:
        self._frequencies, self._factor = frequencies, float(factor)
        self._turns = {}                                       # device -> turns per position, and where they are

    def _scaled(self, frequencies, factor: float = 1.0) -> "Rotary":
        r = Rotary(self._head_dim, self._base, self._rot, self._interleaved)
        r._set(frequencies, self._factor * factor)
        return r

    def linear(self, factor: float) -> "Rotary":
        """Positions divided by `factor`."""
        assert factor > 0.0, "factor is positive"
        return self._scaled(self._frequencies / factor)

    def by_wavelength(self, factor: float, low: float, high: float, original: int) -> "Rotary":
        """Frequencies that turn more than `high` times over the `original` context stay, those that turn less than `low` times are divided by
        `factor`, linear in the number of turns between."""
        assert factor > 0.0 and 0.0 < low < high and original > 0, "factor and original are positive, low is below high"
        s = np.clip((original * self._frequencies / (2.0 * math.pi) - low) / (high - low), 0.0, 1.0)
        return self._scaled((1.0 - s) * self._frequencies / factor + s * self._frequencies)

    def yarn(self, factor: float, original: int, fast: float = 32.0, slow: float = 1.0, attention: float | None = None) -> "Rotary":
        """Pairs that turn more than `fast` times over the `original` context stay, those below `slow` are divided by `factor`, linear in the pair's
        index between; cosines and sines are multiplied by `attention` (0.1 ln(factor) + 1)."""
        assert factor > 0.0 and original > 0 and fast > slow > 0.0, "factor and original are positive, fast is above slow"

        def at(turns):
            return self._rot * math.log(original / (turns * 2.0 * math.pi)) / (2.0 * math.log(self._base))

        lo, hi = max(math.floor(at(fast)), 0), min(math.ceil(at(slow)), self._rot - 1)
        r = np.clip((np.arange(self._rot // 2, dtype=np.float64) - lo) / max(hi - lo, 0.001), 0.0, 1.0)
        if attention is None:
            attention = 0.1 * math.log(factor) + 1.0 if factor > 1.0 else 1.0
        return self._scaled(self._frequencies / factor * r + self._frequencies * (1.0 - r), attention)

    def head_dim(self) -> int:
        return self._head_dim

    def rotary_dim(self) -> int:
        return self._rot

    def interleaved(self) -> bool:
        return self._interleaved

    def frequencies(self) -> np.ndarray:
        """Radians per position of each pair (f64)."""
        return self._frequencies.copy()

    def factor(self) -> float:
        """On the cosines and sines."""
        return self._factor

    def _on(self, device: int):
        """(address of the turns per position of each pair, f64; address of the cosines and sines of 0 .. 255 times the frequencies, f32; the tensors).  Made by
        the first call on a device: before a capture, then."""
        t = self._turns.get(device)
        if t is None:
            at = torch.device("cuda", device)
            turns = torch.tensor(self._frequencies / (2.0 * math.pi), dtype=torch.float64, device=at)
            angle = np.arange(256, dtype=np.float64)[:, None] * self._frequencies
            steps = torch.tensor(np.concatenate([np.cos(angle), np.sin(angle)], 1), dtype=torch.float32, device=at)
            t = self._turns[device] = turns.data_ptr(), steps.data_ptr(), turns, steps
        return t


def _rotation(rotary, head_dim: int, device: int):
    if rotary is None:
        return 0, 0, 0, 0, 1.0
    assert isinstance(rotary, Rotary) and rotary._head_dim == head_dim, "the rotation is one of heads of head_dim"
    turns, steps, _, _ = rotary._on(device)
    return turns, steps, rotary._rot, rotary._interleaved, rotary._factor


def rotate_heads(q, k, positions, rotary, q_out, k_out, *, q_norm=None, k_norm=None, head_dim: int | None = None) -> None:
    """q_out, k_out = the heads of the rows q and k (either may be None), each normalised (q_norm, k_norm: RMS norms of head_dim weights) and rotated by
    its row's position, in one pass with one rounding.  positions: an int32 tensor, one a row, or the first row's as a number.  The outputs may be
    the inputs.  rotary None: the norms alone (head_dim is needed then)."""
    assert rotary is not None or head_dim is not None, "without a rotation, head_dim says what a head is"
    hd = rotary._head_dim if rotary is not None else head_dim
    assert head_dim is None or head_dim == hd, "the rotation is one of heads of head_dim"
    assert hd % 8 == 0 and 8 <= hd <= 256, "head_dim must be a multiple of 8 in 8..=256"
    assert q is not None or k is not None, "there are queries or keys"
    assert (q is None) == (q_out is None), "q and q_out come together"
    assert (k is None) == (k_out is None), "k and k_out come together"
    q_ptr = k_ptr = qo_ptr = ko_ptr = qs = ks = qos = kos = heads = kv_heads = 0
    like = None
    if q is not None:
        like, rows, width = _first_rows(q, "q")
        heads = width // hd
        assert heads * hd == width and heads > 0, "q has rows of whole heads"
        qs, qos = _rows(q, "q", rows, width, like), _rows(q_out, "q_out", rows, width, like)
        q_ptr, qo_ptr = q.data_ptr(), q_out.data_ptr()
    if k is not None:
        if like is None:
            like, rows, width = _first_rows(k, "k")
        else:
            width = _first_rows(k, "k")[2]
        kv_heads = width // hd
        assert kv_heads * hd == width and kv_heads > 0, "k has rows of whole heads"
        ks, kos = _rows(k, "k", rows, width, like), _rows(k_out, "k_out", rows, width, like)
        k_ptr, ko_ptr = k.data_ptr(), k_out.data_ptr()
    dtype, device = like
    pos_ptr, start = 0, 0
    if isinstance(positions, torch.Tensor):
        _ints(positions, "positions", device)
        assert positions.numel() == rows, "positions has one value a row"
        pos_ptr = positions.data_ptr()
    else:
        start = int(positions)
    turns, steps, rot, inter, factor = _rotation(rotary, hd, device)
    qn, qe = _head_norm(q_norm, "q_norm", hd, device)
    kn, ke = _head_norm(k_norm, "k_norm", hd, device)
    if rows == 0:
        return
    _enqueue("smeg_rotate_heads_dev", device, ROTATE_ARGS.pack(
        q_ptr, k_ptr, 0, qo_ptr, ko_ptr, qs, ks, 0, qos, kos, qn, kn, turns, steps, qe, ke, factor, inter, dtype is _BF16, 0, rot, rows, heads, kv_heads, hd,
        pos_ptr, start, 0, 0, 0, 0, 0, 0, 0, 0, 0))


class PagedBatch:
    """Which rows of a packed batch are whose, where each sequence stands and which pages it has: rows cu_rows[s] .. cu_rows[s + 1] are sequence s's,
    its first row has position starts[s] (below zero: the sequence is idle in this step), table[s, i] is the page of its positions i * page ...
    int32 CUDA tensors, which the caller may change in place between calls (a captured step reads them anew at every replay)."""

    def __init__(self, cu_rows, starts, table):
        _ints(starts, "starts", None)
        _ints(cu_rows, "cu_rows", starts.get_device())
        _ints(table, "table", starts.get_device())
        n = starts.numel()
        assert cu_rows.numel() == n + 1, "cu_rows has one value more than there are sequences"
        assert table.dim() == 2 and table.shape[0] == n, "table has a row of pages for each sequence"
        self._tensors = cu_rows, starts, table
        self._device = starts.get_device()
        self._fields = cu_rows.data_ptr(), starts.data_ptr(), table.data_ptr(), n, table.shape[1]

    @property
    def cu_rows(self):
        return self._tensors[0]

    @property
    def starts(self):
        return self._tensors[1]

    @property
    def table(self):
        return self._tensors[2]

    def seqs(self) -> int:
        return self._fields[3]


class PagedKvCache:
    """An 8-bit key/value cache of pages for one attention layer, with the attention against it: `pages` pages of `page` positions in one pool, which
    sequences take pages of by their tables (PagedBatch).  codes uint8 [pages, kv_heads, 2, page, head_dim] (keys, values), scales f32
    [pages, kv_heads, 2]; a value is (code - 128) * scale.  The scale of a page's block is its largest magnitude / 127: it starts over with
    the page's first position and otherwise only grows, and then the codes that are there are rounded again.  A block that received a NaN or an
    infinity is NaN until its page starts over.  A page that is appended to belongs to one sequence; any number may read it."""

    def __init__(self, heads: int, kv_heads: int, head_dim: int, pages: int, page: int = 64, device=None):
        assert head_dim % 16 == 0 and 16 <= head_dim <= 256, "head_dim must be a multiple of 16 in 16..=256"
        assert kv_heads > 0 and heads > 0 and heads % kv_heads == 0, "heads must be a positive multiple of kv_heads"
        assert page in (16, 32, 64, 128, 256), "a page holds 16, 32, 64, 128 or 256 positions"
        assert pages > 0, "a cache has pages"
        self._heads, self._kv_heads, self._head_dim, self._pages, self._page = heads, kv_heads, head_dim, pages, page
        device = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
        self._codes = torch.full((pages, kv_heads, 2, page, head_dim), 128, dtype=torch.uint8, device=device)
        self._scales = torch.zeros((pages, kv_heads, 2), dtype=torch.float32, device=device)
        self._device = self._codes.get_device()
        self._at = self._codes.data_ptr(), self._scales.data_ptr()
        self._scale = float(np.float32(1.0) / np.sqrt(np.float32(head_dim)))
        self._ws_bytes = {}

    @property
    def codes(self):
        return self._codes

    @property
    def scales(self):
        return self._scales

    def with_scale(self, scale: float) -> "PagedKvCache":
        self._scale = float(np.float32(scale))
        return self

    def heads(self) -> int:
        return self._heads

    def kv_heads(self) -> int:
        return self._kv_heads

    def head_dim(self) -> int:
        return self._head_dim

    def pages(self) -> int:
        return self._pages

    def page(self) -> int:
        return self._page

    def scale(self) -> float:
        return self._scale

    def row_len(self) -> int:
        return self._kv_heads * self._head_dim

    def query_len(self) -> int:
        return self._heads * self._head_dim

    def _like(self, x, what: str, batch):
        like, rows, _ = _first_rows(x, what)
        assert like[1] == self._device, "the rows are on the cache's device"
        assert isinstance(batch, PagedBatch) and batch._device == self._device, "the batch is on the cache's device"
        return like, rows

    def append(self, k, v, batch: PagedBatch, rotary: Rotary | None = None, *, k_norm=None, k_out=None, q=None, q_out=None, q_norm=None) -> None:
        """The rows k and v (kv_heads * head_dim values) to the pages of their sequences' positions; keys are normalised (k_norm) and rotated on the way.
        k_out: the keys so treated as 16-bit rows as well.  q, q_out: the queries, normalised (q_norm) and rotated, in the same pass.  The outputs
        may be the inputs.  Rows of idle sequences and rows behind the last sequence are left as they are."""
        hd = self._head_dim
        row, device = self._kv_heads * hd, self._device
        like, rows = self._like(k, "k", batch)
        ks, vs = _rows(k, "k", rows, row, like), _rows(v, "v", rows, row, like)
        q_ptr = qo_ptr = ko_ptr = qs = qos = kos = 0
        if k_out is not None:
            kos, ko_ptr = _rows(k_out, "k_out", rows, row, like), k_out.data_ptr()
        assert (q is None) == (q_out is None), "q and q_out come together"
        if q is not None:
            q_len = self._heads * hd
            qs, qos = _rows(q, "q", rows, q_len, like), _rows(q_out, "q_out", rows, q_len, like)
            q_ptr, qo_ptr = q.data_ptr(), q_out.data_ptr()
        turns, steps, rot, inter, factor = _rotation(rotary, hd, device)
        qn, qe = _head_norm(q_norm, "q_norm", hd, device)
        kn, ke = _head_norm(k_norm, "k_norm", hd, device)
        if rows == 0 or batch._fields[3] == 0:
            return
        _enqueue("smeg_paged_append_dev", device, ROTATE_ARGS.pack(
            q_ptr, k.data_ptr(), v.data_ptr(), qo_ptr, ko_ptr, qs, ks, vs, qos, kos, qn, kn, turns, steps, qe, ke, factor, inter, like[0] is _BF16, 0, rot,
            rows, self._heads, self._kv_heads, hd, 0, 0, *batch._fields, *self._at, self._pages, self._page))

    def attend(self, q, batch: PagedBatch, out) -> None:
        """out = the attention of the query rows (heads * head_dim values) against their sequences' cached positions, which already hold the rows' own
        (append, then attend, with the same batch): row i of a sequence attends to positions 0..=start + i.  Rows of idle sequences become
        zeros, rows behind the last sequence stay as they are."""
        like, rows = self._like(q, "q", batch)
        width, device = self._heads * self._head_dim, self._device
        qs, os_ = _rows(q, "q", rows, width, like), _rows(out, "out", rows, width, like)
        cu, starts, table, seqs, cols = batch._fields
        if rows == 0 or seqs == 0:
            return
        size = rows, seqs, cols
        need = self._ws_bytes.get(size)
        if need is None:
            with _On(device):
                need = lib().smeg_paged_attend_workspace(rows, seqs, cols, self._page, self._heads, self._kv_heads, self._head_dim)
            self._ws_bytes[size] = need
        # the call's own memory, from the stream's pool: two streams, or two captured graphs, never share it
        ws = self._codes.new_empty(need) if need else None
        _enqueue("smeg_paged_attend_dev", device, PAGED_ATTEND_ARGS.pack(
            q.data_ptr(), out.data_ptr(), qs, os_, *self._at, cu, starts, table, seqs, cols, self._pages, self._page, rows, self._heads, self._kv_heads,
            self._head_dim, self._scale, like[0] is _BF16, ws.data_ptr() if need else 0, need))

    def read(self, ids, out) -> None:
        """The values of whole pages: out [n, kv_heads, 2, page, head_dim] (keys, values), contiguous f16 or bf16, for the n int32 page ids."""
        _ints(ids, "ids", self._device)
        n = ids.numel()
        assert isinstance(out, torch.Tensor) and out.get_device() == self._device and out.dtype in (_F16, _BF16) and out.is_contiguous(), "out is contiguous f16 or bf16"
        assert out.numel() == n * self._kv_heads * 2 * self._page * self._head_dim, "out holds n pages"
        if n == 0:
            return
        device = self._device
        _enqueue("smeg_paged_read_dev", device, READ_ARGS.pack(out.data_ptr(), *self._at, ids.data_ptr(), n, self._pages, self._page, self._kv_heads, self._head_dim,
                                                               out.dtype is _BF16, 0))


def attend_packed(q, k, v, cu_rows, out, heads: int, kv_heads: int, scale: float | None = None) -> None:
    """out = causal attention over whole packed prompts: rows cu_rows[s] .. cu_rows[s + 1] (int32 CUDA tensor) are a sequence's, row i of it attends to
    its rows 0..=i.  q, out: rows of heads * head_dim values, k, v of kv_heads * head_dim, f16 or bf16, at any row stride; scale 1 / sqrt(head_dim).
    Rows behind the last sequence are left as they are."""
    assert kv_heads > 0 and heads > 0 and heads % kv_heads == 0, "heads must be a positive multiple of kv_heads"
    like, rows, width = _first_rows(q, "q")
    dtype, device = like
    hd = width // heads
    assert hd * heads == width, "q has rows of heads * head_dim values"
    assert hd % 8 == 0 and 8 <= hd <= 256, "head_dim must be a multiple of 8 in 8..=256"
    row = kv_heads * hd
    qs, ks, vs, os_ = _rows(q, "q", rows, width, like), _rows(k, "k", rows, row, like), _rows(v, "v", rows, row, like), _rows(out, "out", rows, width, like)
    _ints(cu_rows, "cu_rows", device)
    seqs = cu_rows.numel() - 1
    assert seqs >= 0, "cu_rows has one value more than there are sequences"
    if rows == 0 or seqs == 0:
        return
    _enqueue("smeg_attn_packed_dev", device, ATTN_PACKED_ARGS.pack(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), qs, ks, vs, os_, cu_rows.data_ptr(), seqs, rows, heads, kv_heads, hd,
        hd ** -0.5 if scale is None else scale, dtype is _BF16))
