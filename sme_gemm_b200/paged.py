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

from ._lib import ATTN_PACKED_ARGS, PAGED_ATTEND_ARGS, ROTATE_ARGS, check, lib
from .host import Norm, torch

_DTYPES = (torch.float16, torch.bfloat16)


class _On:
    """The tensors' device as the current one, for a call from elsewhere."""

    def __init__(self, device):
        self._device = device

    def __enter__(self):
        self._was = torch.cuda.current_device()
        if self._was != self._device:
            torch.cuda.set_device(self._device)

    def __exit__(self, *exc):
        if self._was != self._device:
            torch.cuda.set_device(self._was)


def _enqueue(name: str, device: int, args: bytes) -> None:
    """Calls `name` with the packed arguments on the current stream of `device`."""
    fn = getattr(lib(), name)
    if torch._C._cuda_getDevice() == device:
        rc = fn(args, torch._C._cuda_getCurrentRawStream(device))
    else:
        with _On(device):
            rc = fn(args, torch._C._cuda_getCurrentRawStream(device))
    if rc:
        check(name, rc)


def _rows(x, what: str, width: int, like=None):
    """Checks a tensor of rows; its row stride in elements."""
    assert isinstance(x, torch.Tensor) and x.is_cuda, f"{what} is a CUDA tensor"
    assert x.dtype in _DTYPES, f"{what} is f16 or bf16"
    assert x.dim() == 2 and x.shape[1] == width, f"{what} has rows of {width} values"
    rows = x.shape[0]
    stride = x.stride(0)
    if rows > 1:
        assert x.stride(1) == 1 and stride >= width, f"{what} has its rows' values side by side"
    else:
        assert width == 1 or x.stride(1) == 1, f"{what} has its rows' values side by side"
        stride = width
    if like is not None:
        assert x.dtype == like.dtype and x.device == like.device, f"{what} has the same type and device as the other rows"
        assert rows == like.shape[0], f"{what} has as many rows as the others"
    return stride


def _ints(x, what: str, device) -> None:
    assert isinstance(x, torch.Tensor) and x.is_cuda and x.dtype == torch.int32 and x.is_contiguous(), f"{what} is a contiguous int32 CUDA tensor"
    assert device is None or x.device == device, f"{what} is on the rows' device"


def _head_norm(norm, what: str, head_dim: int, device):
    if norm is None:
        return 0, 0.0
    assert isinstance(norm, Norm) and norm.is_rms, f"{what} is an RMS norm"
    assert norm.width() == head_dim, f"{what} has head_dim weights"
    assert norm.weight.device == device, f"{what} is on the rows' device"
    return norm.weight.data_ptr(), norm.eps


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
        self._turns = {}                                       # device -> turns per position

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

    def turns(self, device):
        """The frequencies as turns per position, on `device` (kept from the first call on: before a capture, then)."""
        t = self._turns.get(device)
        if t is None:
            t = self._turns[device] = torch.tensor(self._frequencies / (2.0 * math.pi), dtype=torch.float64, device=device)
        return t


def _rotation(rotary, head_dim: int, device):
    if rotary is None:
        return 0, 0, 0, 1.0
    assert isinstance(rotary, Rotary) and rotary._head_dim == head_dim, "the rotation is one of heads of head_dim"
    return rotary.turns(device).data_ptr(), rotary._rot, int(rotary._interleaved), rotary._factor


def rotate_heads(q, k, positions, rotary, q_out, k_out, *, q_norm=None, k_norm=None, head_dim: int | None = None) -> None:
    """q_out, k_out = the heads of the rows q and k (either may be None), each normalised (q_norm, k_norm: RMS norms of head_dim weights) and rotated by
    its row's position, in one pass with one rounding.  positions: an int32 tensor, one a row, or the first row's as a number.  The outputs may be
    the inputs.  rotary None: the norms alone (head_dim is needed then)."""
    assert rotary is not None or head_dim is not None, "without a rotation, head_dim says what a head is"
    hd = rotary._head_dim if rotary is not None else head_dim
    assert head_dim is None or head_dim == hd, "the rotation is one of heads of head_dim"
    assert hd % 8 == 0 and 8 <= hd <= 256, "head_dim must be a multiple of 8 in 8..=256"
    one = q if q is not None else k
    assert one is not None, "there are queries or keys"
    ptr, stride, heads = [0, 0, 0, 0], [0, 0, 0, 0], [0, 0]
    for i, (x, out, what) in enumerate(((q, q_out, "q"), (k, k_out, "k"))):
        assert (x is None) == (out is None), f"{what} and {what}_out come together"
        if x is None:
            continue
        assert x.dim() == 2 and x.shape[1] % hd == 0 and x.shape[1] > 0, f"{what} has rows of whole heads"
        stride[i], stride[2 + i] = _rows(x, what, x.shape[1], one), _rows(out, what + "_out", x.shape[1], one)
        ptr[i], ptr[2 + i], heads[i] = x.data_ptr(), out.data_ptr(), x.shape[1] // hd
    rows, device = one.shape[0], one.device
    pos_ptr, start = 0, 0
    if isinstance(positions, torch.Tensor):
        _ints(positions, "positions", device)
        assert positions.numel() == rows, "positions has one value a row"
        pos_ptr = positions.data_ptr()
    else:
        start = int(positions)
    turns, rot, inter, factor = _rotation(rotary, hd, device)
    qn, qe = _head_norm(q_norm, "q_norm", hd, device)
    kn, ke = _head_norm(k_norm, "k_norm", hd, device)
    if rows == 0:
        return
    _enqueue("smeg_rotate_heads_dev", device.index, ROTATE_ARGS.pack(
        ptr[0], ptr[1], 0, ptr[2], ptr[3], stride[0], stride[1], 0, stride[2], stride[3], qn, kn, turns, qe, ke, factor, inter,
        one.dtype == torch.bfloat16, 0, rot, rows, heads[0], heads[1], hd, pos_ptr, start, 0, 0, 0, 0, 0, 0, 0, 0, 0))


class PagedBatch:
    """Which rows of a packed batch are whose, where each sequence stands and which pages it has: rows cu_rows[s] .. cu_rows[s + 1] are sequence s's,
    its first row has position starts[s] (below zero: the sequence is idle in this step), table[s, i] is the page of its positions i * page ...
    int32 CUDA tensors, which the caller may change in place between calls (a captured step reads them anew at every replay)."""

    def __init__(self, cu_rows, starts, table):
        _ints(starts, "starts", None)
        _ints(cu_rows, "cu_rows", starts.device)
        _ints(table, "table", starts.device)
        n = starts.numel()
        assert cu_rows.numel() == n + 1, "cu_rows has one value more than there are sequences"
        assert table.dim() == 2 and table.shape[0] == n, "table has a row of pages for each sequence"
        self.cu_rows, self.starts, self.table = cu_rows, starts, table

    def seqs(self) -> int:
        return self.starts.numel()

    def _fields(self):
        return self.cu_rows.data_ptr(), self.starts.data_ptr(), self.table.data_ptr(), self.starts.numel(), self.table.shape[1]


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
        assert pages >= 0, "pages is a number of pages"
        self._heads, self._kv_heads, self._head_dim, self._pages, self._page = heads, kv_heads, head_dim, pages, page
        device = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
        self.codes = torch.full((max(pages, 1), kv_heads, 2, page, head_dim), 128, dtype=torch.uint8, device=device)
        self.scales = torch.zeros((max(pages, 1), kv_heads, 2), dtype=torch.float32, device=device)
        self._device = self.codes.device
        self._scale = float(np.float32(1.0) / np.sqrt(np.float32(head_dim)))
        self._ws_bytes = {}

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

    def _mine(self, x, batch) -> None:
        assert x.device == self._device, "the rows are on the cache's device"
        assert isinstance(batch, PagedBatch) and batch.starts.device == self._device, "the batch is on the cache's device"

    def append(self, k, v, batch: PagedBatch, rotary: Rotary | None = None, *, k_norm=None, k_out=None, q=None, q_out=None, q_norm=None) -> None:
        """The rows k and v (kv_heads * head_dim values) to the pages of their sequences' positions; keys are normalised (k_norm) and rotated on the way.
        k_out: the keys so treated as 16-bit rows as well.  q, q_out: the queries, normalised (q_norm) and rotated, in the same pass.  The outputs
        may be the inputs.  Rows of idle sequences and rows behind the last sequence are left as they are."""
        row, hd = self.row_len(), self._head_dim
        ks, vs = _rows(k, "k", row), _rows(v, "v", row, k)
        self._mine(k, batch)
        kos = _rows(k_out, "k_out", row, k) if k_out is not None else 0
        assert (q is None) == (q_out is None), "q and q_out come together"
        qs = qos = 0
        if q is not None:
            qs, qos = _rows(q, "q", self.query_len(), k), _rows(q_out, "q_out", self.query_len(), k)
        turns, rot, inter, factor = _rotation(rotary, hd, self._device)
        qn, qe = _head_norm(q_norm, "q_norm", hd, self._device)
        kn, ke = _head_norm(k_norm, "k_norm", hd, self._device)
        cu, starts, table, seqs, cols = batch._fields()
        if k.shape[0] == 0 or seqs == 0:
            return
        _enqueue("smeg_paged_append_dev", self._device.index, ROTATE_ARGS.pack(
            q.data_ptr() if q is not None else 0, k.data_ptr(), v.data_ptr(), q_out.data_ptr() if q is not None else 0,
            k_out.data_ptr() if k_out is not None else 0, qs, ks, vs, qos, kos, qn, kn, turns, qe, ke, factor, inter, k.dtype == torch.bfloat16, 0,
            rot, k.shape[0], self._heads, self._kv_heads, hd, 0, 0, cu, starts, table, seqs, cols, self.codes.data_ptr(), self.scales.data_ptr(),
            self._pages, self._page))

    def attend(self, q, batch: PagedBatch, out) -> None:
        """out = the attention of the query rows (heads * head_dim values) against their sequences' cached positions, which already hold the rows' own
        (append, then attend, with the same batch): row i of a sequence attends to positions 0..=start + i.  Rows of idle sequences become
        zeros, rows behind the last sequence stay as they are."""
        qs, os_ = _rows(q, "q", self.query_len()), _rows(out, "out", self.query_len(), q)
        self._mine(q, batch)
        cu, starts, table, seqs, cols = batch._fields()
        rows = q.shape[0]
        if rows == 0 or seqs == 0:
            return
        size = (rows, seqs, cols)
        need = self._ws_bytes.get(size)
        if need is None:
            with _On(self._device.index):
                need = lib().smeg_paged_attend_workspace(rows, seqs, cols, self._page, self._heads, self._kv_heads, self._head_dim)
            self._ws_bytes[size] = need
        # the call's own memory, from the stream's pool: two streams, or two captured graphs, never share it
        ws = torch.empty(need, dtype=torch.uint8, device=self._device) if need else None
        _enqueue("smeg_paged_attend_dev", self._device.index, PAGED_ATTEND_ARGS.pack(
            q.data_ptr(), out.data_ptr(), qs, os_, self.codes.data_ptr(), self.scales.data_ptr(), cu, starts, table, seqs, cols, self._pages, self._page,
            rows, self._heads, self._kv_heads, self._head_dim, self._scale, q.dtype == torch.bfloat16, ws.data_ptr() if need else 0, need))

    def read(self, ids, out) -> None:
        """The values of whole pages: out [n, kv_heads, 2, page, head_dim] (keys, values), contiguous f16 or bf16, for the n int32 page ids."""
        _ints(ids, "ids", self._device)
        n = ids.numel()
        assert isinstance(out, torch.Tensor) and out.device == self._device and out.dtype in _DTYPES and out.is_contiguous(), "out is contiguous f16 or bf16"
        assert out.numel() == n * self._kv_heads * 2 * self._page * self._head_dim, "out holds n pages"
        if n == 0:
            return
        args = (out.data_ptr(), self.codes.data_ptr(), self.scales.data_ptr(), ids.data_ptr(), n, self._pages, self._page, self._kv_heads, self._head_dim,
                out.dtype == torch.bfloat16)
        with _On(self._device.index):
            check("smeg_paged_read_dev", lib().smeg_paged_read_dev(*args, torch._C._cuda_getCurrentRawStream(self._device.index)))


def attend_packed(q, k, v, cu_rows, out, heads: int, kv_heads: int, scale: float | None = None) -> None:
    """out = causal attention over whole packed prompts: rows cu_rows[s] .. cu_rows[s + 1] (int32 CUDA tensor) are a sequence's, row i of it attends to
    its rows 0..=i.  q, out: rows of heads * head_dim values, k, v of kv_heads * head_dim, f16 or bf16, at any row stride; scale 1 / sqrt(head_dim).
    Rows behind the last sequence are left as they are."""
    assert kv_heads > 0 and heads > 0 and heads % kv_heads == 0, "heads must be a positive multiple of kv_heads"
    assert isinstance(q, torch.Tensor) and q.dim() == 2 and q.shape[1] % heads == 0, "q has rows of heads * head_dim values"
    hd = q.shape[1] // heads
    assert hd % 8 == 0 and 8 <= hd <= 256, "head_dim must be a multiple of 8 in 8..=256"
    qs = _rows(q, "q", heads * hd)
    ks, vs, os_ = _rows(k, "k", kv_heads * hd, q), _rows(v, "v", kv_heads * hd, q), _rows(out, "out", heads * hd, q)
    _ints(cu_rows, "cu_rows", q.device)
    assert cu_rows.numel() >= 1, "cu_rows has one value more than there are sequences"
    rows, seqs = q.shape[0], cu_rows.numel() - 1
    if rows == 0 or seqs == 0:
        return
    scale = float(np.float32(1.0) / np.sqrt(np.float32(hd))) if scale is None else float(scale)
    _enqueue("smeg_attn_packed_dev", q.device.index, ATTN_PACKED_ARGS.pack(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), qs, ks, vs, os_, cu_rows.data_ptr(), seqs, rows, heads, kv_heads, hd, scale,
        q.dtype == torch.bfloat16))
