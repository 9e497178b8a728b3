"""Packed batches of sequences: rotation by position, the 8-bit paged key/value cache, attention.

What a model with rotated, normalised heads and a server with many sequences need around the projections of a self-attention block (the reference
applies no rotation, src/self_attention.rs:66-231, and keeps one f16 buffer a sequence, src/kernels/kv_attention.rs:354-581).  Tensors are CUDA
tensors of f16 or bf16 rows, heads * head_dim values each, at any row stride: slices of the [q | k | v] rows that a fused projection leaves are taken
as they are.  Every call enqueues its work on torch's current stream of the tensors' device; nothing is read back, so that all of them can be
captured into a graph (row offsets, starts and page tables are device memory).
"""
from __future__ import annotations

import ctypes
import importlib
import math
import os

import numpy as np

from ._lib import check, lib
from .host import Norm, torch

_CALLS = None                                                # the compiled side of the calls: reads and checks tensors (csrc/binding.cc)
_NO_ROTATION_YET = -1000                                     # from it: the rotation's table is not on the rows' device


def _calls():
    global _CALLS
    if _CALLS is None:
        L = lib()
        try:
            m = importlib.import_module("._binding", __package__)
        except ImportError as e:
            there = any(f.startswith("_binding.") and f.endswith(".so") for f in os.listdir(os.path.dirname(os.path.abspath(__file__))))
            what = f"does not load ({e})" if there else "is missing"
            raise RuntimeError(f"sme_gemm_b200/_binding {what}: build it with `python -m sme_gemm_b200.build`") from e
        m.bind(*(ctypes.cast(getattr(L, "smeg_" + n), ctypes.c_void_p).value for n in (
            "rotate_heads_dev", "paged_append_dev", "paged_attend_dev", "paged_attend_workspace", "attn_packed_dev", "paged_read_dev")))
        _CALLS = m
    return _CALLS


def _ints(x, what: str, device: int) -> None:
    assert isinstance(x, torch.Tensor) and x.is_cuda and x.dtype is torch.int32 and x.is_contiguous(), f"{what} is a contiguous int32 CUDA tensor"
    assert device is None or x.get_device() == device, f"{what} is on the rows' device"


def _head_norm(norm, what: str):
    """(weights, eps) of a norm of the heads."""
    if norm is None:
        return None, 0.0
    assert isinstance(norm, Norm) and norm.is_rms, f"{what} is an RMS norm"
    return norm.weight, norm.eps


class Rotary:
    """The rotation of heads by position: pair i of the first `rotary_dim` depths turns by position * frequency_i, frequency_i =
    base^(-2 i / rotary_dim).  A pair is (i, i + rotary_dim / 2), or (2 i, 2 i + 1) interleaved; the depths behind rotary_dim stay as they are.
    The first call with it on a device places its tables there, and so cannot be one that a graph captures.
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
        self._call = self._turns, self._rot, self._interleaved, self._factor

    def __getstate__(self):                                    # a copy, or one of another process, has tables of its own
        return self._head_dim, self._rot, self._base, self._interleaved, self._frequencies, self._factor

    def __setstate__(self, state) -> None:
        self._head_dim, self._rot, self._base, self._interleaved, frequencies, factor = state
        self._set(frequencies, factor)

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
        """(address of the turns per position of each pair, f64; address of the cosines and sines of 0 .. 255 times the frequencies, f32; the tensors)."""
        t = self._turns.get(device)
        if t is None:
            with torch.cuda.device(device):
                capturing = torch.cuda.is_current_stream_capturing()
            assert not capturing, "the first call with a rotation on a device lies before a capture"
            at = torch.device("cuda", device)
            turns = torch.tensor(self._frequencies / (2.0 * math.pi), dtype=torch.float64, device=at)
            angle = np.arange(256, dtype=np.float64)[:, None] * self._frequencies
            steps = torch.tensor(np.concatenate([np.cos(angle), np.sin(angle)], 1), dtype=torch.float32, device=at)
            t = self._turns.setdefault(device, (turns.data_ptr(), steps.data_ptr(), turns, steps))     # (another thread's, if that was first)
        return t


def _rotation(rotary, head_dim: int):
    if rotary is None:
        return None
    assert isinstance(rotary, Rotary) and rotary._head_dim == head_dim, "the rotation is one of heads of head_dim"
    return rotary._call


def rotate_heads(q, k, positions, rotary, q_out, k_out, *, q_norm=None, k_norm=None, head_dim: int | None = None) -> None:
    """q_out, k_out = the heads of the rows q and k (either may be None), each normalised (q_norm, k_norm: RMS norms of head_dim weights) and rotated by
    its row's position, in one pass with one rounding.  positions: an int32 tensor, one a row, or the first row's as a number.  q_out may be
    q, and k_out k; else the outputs share no memory with one another or the inputs.  rotary None: the norms alone (head_dim is needed then)."""
    assert rotary is not None or head_dim is not None, "without a rotation, head_dim says what a head is"
    hd = rotary._head_dim if rotary is not None else head_dim
    assert head_dim is None or head_dim == hd, "the rotation is one of heads of head_dim"
    assert hd % 8 == 0 and 8 <= hd <= 256, "head_dim must be a multiple of 8 in 8..=256"
    args = (q, k, positions, q_out, k_out, *_head_norm(q_norm, "q_norm"), *_head_norm(k_norm, "k_norm"), _rotation(rotary, hd), hd)
    rc = (_CALLS or _calls()).rotate(*args)
    if rc == _NO_ROTATION_YET:
        rotary._on((k if q is None else q).get_device())
        rc = _CALLS.rotate(*args)
    if rc:
        check("smeg_rotate_heads_dev", rc)


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
        assert n == 0 or table.shape[1] > 0, "table has a page for each sequence"
        self._tensors = cu_rows, starts, table
        self._device = starts.get_device()
        self._fields = cu_rows.data_ptr(), starts.data_ptr(), table.data_ptr(), n, table.shape[1], self._device

    def __getstate__(self):                                    # (the addresses are the tensors', which a copy has its own of)
        return self._tensors

    def __setstate__(self, tensors) -> None:
        self.__init__(*tensors)

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
        self._set_scale(1.0 / np.sqrt(np.float32(head_dim)))

    def __getstate__(self):                                    # (as PagedBatch)
        return {name: x for name, x in self.__dict__.items() if name not in ("_device", "_fields")}

    def __setstate__(self, state) -> None:
        self.__dict__.update(state)
        self._device = self._codes.get_device()
        self._set_scale(self._scale)

    def _set_scale(self, scale: float) -> None:
        self._scale = float(np.float32(scale))
        self._fields = (self._codes.data_ptr(), self._scales.data_ptr(), self._pages, self._page, self._heads, self._kv_heads, self._head_dim, self._device,
                        self._scale)

    @property
    def codes(self):
        return self._codes

    @property
    def scales(self):
        return self._scales

    def with_scale(self, scale: float) -> "PagedKvCache":
        self._set_scale(scale)
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

    def append(self, k, v, batch: PagedBatch, rotary: Rotary | None = None, *, k_norm=None, k_out=None, q=None, q_out=None, q_norm=None) -> None:
        """The rows k and v (kv_heads * head_dim values) to the pages of their sequences' positions; keys are normalised (k_norm) and rotated on the way.
        k_out: the keys so treated as 16-bit rows as well.  q, q_out: the queries, normalised (q_norm) and rotated, in the same pass.  q_out
        may be q, and k_out k; else they share no memory with one another or the inputs.  Rows of idle sequences and rows behind the last sequence are left as they are."""
        assert isinstance(batch, PagedBatch), "batch is a PagedBatch"
        args = (k, v, k_out, q, q_out, *_head_norm(q_norm, "q_norm"), *_head_norm(k_norm, "k_norm"), _rotation(rotary, self._head_dim), batch._fields, self._fields)
        rc = (_CALLS or _calls()).append(*args)
        if rc == _NO_ROTATION_YET:
            rotary._on(self._device)
            rc = _CALLS.append(*args)
        if rc:
            check("smeg_paged_append_dev", rc)

    def attend(self, q, batch: PagedBatch, out) -> None:
        """out = the attention of the query rows (heads * head_dim values) against their sequences' cached positions, which already hold the rows' own
        (append, then attend, with the same batch): row i of a sequence attends to positions 0..=start + i.  Rows of idle sequences become
        zeros, rows behind the last sequence stay as they are.  Probabilities are f16 in the product with the values.  out shares no memory with q."""
        assert isinstance(batch, PagedBatch), "batch is a PagedBatch"
        rc = (_CALLS or _calls()).attend(q, out, batch._fields, self._fields)
        if rc:
            check("smeg_paged_attend_dev", rc)

    def read(self, ids, out) -> None:
        """The values of whole pages: out [n, kv_heads, 2, page, head_dim] (keys, values), contiguous f16 or bf16, for the n int32 page ids."""
        rc = (_CALLS or _calls()).read(ids, out, self._fields)
        if rc:
            check("smeg_paged_read_dev", rc)


def attend_packed(q, k, v, cu_rows, out, heads: int, kv_heads: int, scale: float | None = None) -> None:
    """out = causal attention over whole packed prompts: rows cu_rows[s] .. cu_rows[s + 1] (int32 CUDA tensor) are a sequence's, row i of it attends to
    its rows 0..=i.  q, out: rows of heads * head_dim values, k, v of kv_heads * head_dim, f16 or bf16, at any row stride; scale 1 / sqrt(head_dim).
    Rows behind the last sequence are left as they are.  Probabilities have the rows' type in the product with the values (KvCache's attention is closer).
    out shares no memory with the inputs."""
    assert kv_heads > 0 and heads > 0 and heads % kv_heads == 0, "heads must be a positive multiple of kv_heads"
    rc = (_CALLS or _calls()).packed(q, k, v, cu_rows, out, heads, kv_heads, scale)
    if rc:
        check("smeg_attn_packed_dev", rc)
