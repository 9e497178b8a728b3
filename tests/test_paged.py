"""Packed batches and the 8-bit paged cache, what needs no GPU: the index arithmetic, the rotation's frequencies, the refusals."""
import math
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

import sme_gemm_b200 as sg
from sme_gemm_b200._lib import ATTN_PACKED_ARGS, PAGED_ATTEND_ARGS, READ_ARGS, ROTATE_ARGS

HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.fixture(scope="module")
def index_check(tmp_path_factory):
    exe = tmp_path_factory.mktemp("paged") / "paged_index_check"
    subprocess.run(["g++", "-O1", "-std=c++17", "-fsanitize=undefined", "-fno-sanitize-recover=all", "-o", str(exe),
                    os.path.join(HERE, "cpp", "paged_index_check.cc")], check=True)
    return str(exe)


def test_index_arithmetic_covers_sound_batches_and_stays_inside_for_any_values(index_check):
    r = subprocess.run([index_check], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and r.stdout.startswith("ok "), r.stdout + r.stderr
    assert int(r.stdout.split()[1]) > 100000


def test_packed_arguments_are_the_structures(index_check):
    got = list(map(int, subprocess.run([index_check, "sizes"], capture_output=True, text=True, check=True).stdout.split()))
    import struct
    start = struct.calcsize("@PPPPPNNNNNPPPPfffiiiNNNNNPq") - 8
    end = PAGED_ATTEND_ARGS.size - 8
    assert got == [ROTATE_ARGS.size, start, PAGED_ATTEND_ARGS.size, end, ATTN_PACKED_ARGS.size, READ_ARGS.size]


def test_frequencies_follow_their_definitions():
    r = sg.Rotary(128, base=10000.0, rotary_dim=96)
    f = r.frequencies()
    assert f.shape == (48,) and f[0] == 1.0 and abs(f[7] - 10000.0 ** (-14 / 96)) < 1e-15
    assert np.array_equal(r.linear(4.0).frequencies(), f / 4.0)
    w = r.by_wavelength(8.0, 1.0, 4.0, 8192).frequencies()
    turns = 8192 * f / (2 * math.pi)
    assert np.array_equal(w[turns > 4], f[turns > 4]) and np.allclose(w[turns < 1], f[turns < 1] / 8, rtol=1e-15)
    mid = (turns >= 1) & (turns <= 4)
    assert mid.any() and np.all((w[mid] <= f[mid]) & (w[mid] >= f[mid] / 8))
    y = r.yarn(16.0, 4096)
    assert abs(y.factor() - (0.1 * math.log(16.0) + 1.0)) < 1e-15 and r.factor() == 1.0
    assert y.frequencies()[0] == f[0] and abs(y.frequencies()[-1] - f[-1] / 16) < 1e-18
    assert r.yarn(16.0, 4096, attention=1.0).factor() == 1.0
    assert r.rotary_dim() == 96 and r.head_dim() == 128 and not r.interleaved()


@pytest.mark.parametrize("bad,message", [
    (lambda: sg.Rotary(12), "multiple of 8"), (lambda: sg.Rotary(264), "multiple of 8"), (lambda: sg.Rotary(64, rotary_dim=33), "even"),
    (lambda: sg.Rotary(64, rotary_dim=66), "at most head_dim"), (lambda: sg.Rotary(64, rotary_dim=0), "at least 2"), (lambda: sg.Rotary(64, base=0.0), "positive"),
    (lambda: sg.Rotary(64).linear(0.0), "positive"), (lambda: sg.Rotary(64).by_wavelength(8.0, 4.0, 4.0, 8192), "below high"),
    (lambda: sg.Rotary(64).yarn(8.0, 4096, fast=1.0, slow=2.0), "above slow"),
    (lambda: sg.PagedKvCache(4, 2, 24, 3), "multiple of 16"), (lambda: sg.PagedKvCache(4, 3, 32, 3), "multiple of kv_heads"),
    (lambda: sg.PagedKvCache(4, 2, 32, 3, page=48), "a page holds"),
    (lambda: sg.PagedBatch(torch.zeros(3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32), torch.zeros(2, 4, dtype=torch.int32)), "CUDA tensor"),
    (lambda: sg.rotate_heads(torch.zeros(2, 64), None, 0, sg.Rotary(64), torch.zeros(2, 64), None), "CUDA tensor"),
    (lambda: sg.rotate_heads(None, None, 0, sg.Rotary(64), None, None), "queries or keys"),
    (lambda: sg.rotate_heads(torch.zeros(2, 64), None, 0, None, torch.zeros(2, 64), None), "head_dim says"),
    (lambda: sg.attend_packed(*[torch.zeros(2, 64)] * 3, None, torch.zeros(2, 64), 3, 2), "multiple of kv_heads"),
    (lambda: sg.attend_packed(*[torch.zeros(2, 24)] * 3, None, torch.zeros(2, 24), 2, 2), "CUDA tensor"),
])
def test_refusals_before_any_device_work(bad, message):
    with pytest.raises(AssertionError, match=message):
        bad()


def _rotate(**kw):
    names = ("q k v q_out k_out q_stride k_stride v_stride q_out_stride k_out_stride q_norm k_norm turns steps q_eps k_eps factor interleaved bf16 reserved rot rows heads "
             "kv_heads head_dim positions start cu_rows starts table seqs table_cols codes scales pages page").split()
    a = dict(q=4096, k=4096, v=0, q_out=4096, k_out=4096, q_stride=256, k_stride=128, v_stride=128, q_out_stride=256, k_out_stride=128, q_norm=0, k_norm=0, turns=0, steps=0,
             q_eps=0.0, k_eps=0.0, factor=1.0, interleaved=0, bf16=0, reserved=0, rot=0, rows=2, heads=4, kv_heads=2, head_dim=64, positions=0, start=0, cu_rows=0,
             starts=0, table=0, seqs=0, table_cols=0, codes=0, scales=0, pages=0, page=0)
    a.update(kw)
    return ROTATE_ARGS.pack(*(a[n] for n in names))


def _paged(**kw):
    return _rotate(**{**dict(v=4096, cu_rows=4096, starts=4096, table=4096, seqs=2, table_cols=3, codes=4096, scales=4096, pages=5, page=64), **kw})


@pytest.mark.parametrize("kw,rc", [(dict(head_dim=60), -4), (dict(head_dim=0), -4), (dict(head_dim=320), -4), (dict(rot=7), -4), (dict(rot=66), -4),
                                   (dict(turns=4096), -4), (dict(q=0, k=0), -4), (dict(q_out=0), -4), (dict(k_out=0), -4), (dict(q_stride=255), -4),
                                   (dict(q_out_stride=255), -4), (dict(k_stride=127), -4), (dict(k_out_stride=127), -4), (dict(rows=1 << 31), -3),
                                   (dict(heads=65536, head_dim=8, q_stride=1 << 30, q_out_stride=1 << 30), -3), (dict(rows=0), 0)])
def test_rotation_refuses_bad_arguments(kw, rc):
    assert sg.lib().smeg_rotate_heads_dev(_rotate(**kw), None) == rc


@pytest.mark.parametrize("kw,rc", [(dict(head_dim=24), -4), (dict(v=0), -4), (dict(codes=0), -4), (dict(scales=0), -4), (dict(cu_rows=0), -4), (dict(starts=0), -4),
                                   (dict(table=0), -4), (dict(page=48), -4), (dict(page=8), -4), (dict(page=512), -4), (dict(v_stride=127), -4),
                                   (dict(codes=4100), -4), (dict(turns=4096, rot=64), -4), (dict(turns=4096, rot=64, steps=4100), -4), (dict(k=0), -4), (dict(table_cols=1 << 26), -3), (dict(pages=1 << 32), -3), (dict(seqs=1 << 25), -3),
                                   (dict(seqs=0), 0), (dict(rows=0), 0)])
def test_append_refuses_bad_arguments(kw, rc):
    assert sg.lib().smeg_paged_append_dev(_paged(**kw), None) == rc


@pytest.mark.parametrize("kw,rc", [(dict(head_dim=40), -4), (dict(heads=5), -4), (dict(kv_heads=0), -4), (dict(page=20), -4), (dict(q=0), -4), (dict(out=0), -4),
                                   (dict(codes=0), -4), (dict(scales=0), -4), (dict(cu=0), -4), (dict(starts=0), -4), (dict(table=0), -4), (dict(codes=4104), -4), (dict(scales=4100), -4), (dict(pages=0), -3),
                                   (dict(q_stride=255), -4), (dict(out_stride=255), -4), (dict(cols=1 << 26), -3), (dict(rows=1 << 31), -3), (dict(rows=0), 0),
                                   (dict(seqs=0), 0)])
def test_cache_attention_refuses_bad_arguments(kw, rc):
    a = dict(q=4096, out=4096, q_stride=256, out_stride=256, codes=4096, scales=4096, cu=4096, starts=4096, table=4096, seqs=2, cols=3, pages=5, page=64, rows=2,
             heads=4, kv_heads=2, head_dim=64, scale=0.125, bf16=0, ws=0, bytes=0)
    a.update(kw)
    assert sg.lib().smeg_paged_attend_dev(PAGED_ATTEND_ARGS.pack(*a.values()), None) == rc


@pytest.mark.parametrize("kw,rc", [(dict(head_dim=12), -4), (dict(heads=5), -4), (dict(q=0), -4), (dict(k=0), -4), (dict(v=0), -4), (dict(out=0), -4), (dict(cu=0), -4),
                                   (dict(q_stride=255), -4), (dict(k_stride=127), -4), (dict(v_stride=127), -4), (dict(out_stride=255), -4),
                                   (dict(rows=1 << 31), -3), (dict(rows=0), 0), (dict(seqs=0), 0)])
def test_prompt_attention_refuses_bad_arguments(kw, rc):
    a = dict(q=4096, k=4096, v=4096, out=4096, q_stride=256, k_stride=128, v_stride=128, out_stride=256, cu=4096, seqs=1, rows=2, heads=4, kv_heads=2, head_dim=64,
             scale=0.125, bf16=0)
    a.update(kw)
    assert sg.lib().smeg_attn_packed_dev(ATTN_PACKED_ARGS.pack(*a.values()), None) == rc


def test_null_argument_structures_are_refused():
    L = sg.lib()
    assert [f(None, None) for f in (L.smeg_rotate_heads_dev, L.smeg_paged_append_dev, L.smeg_paged_attend_dev, L.smeg_attn_packed_dev)] == [-4] * 4
    assert L.smeg_paged_read_dev(None, None) == -4
    read = dict(out=4096, codes=4096, scales=4096, ids=4096, n=1, pages=5, page=64, kv_heads=2, head_dim=64, bf16=0, reserved=0)
    for kw, rc in ((dict(page=24), -4), (dict(n=0), 0), (dict(out=0), -4), (dict(codes=4104), -4), (dict(head_dim=40), -4), (dict(kv_heads=0), -4), (dict(n=1 << 31), -3)):
        assert L.smeg_paged_read_dev(READ_ARGS.pack(*{**read, **kw}.values()), None) == rc


def test_keys_of_a_row_at_starts_of_every_size(tmp_path):
    exe = tmp_path / "paged_rows_check"
    subprocess.run(["g++", "-O1", "-std=c++17", "-fsanitize=undefined", "-fno-sanitize-recover=all", "-o", str(exe), os.path.join(HERE, "cpp", "paged_rows_check.cc")], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0 and r.stdout.startswith("ok "), r.stdout + r.stderr


def test_rows_that_share_memory_are_told_from_rows_side_by_side(tmp_path):
    exe = tmp_path / "rows_share_check"
    subprocess.run(["g++", "-O1", "-std=c++17", "-fsanitize=undefined", "-fno-sanitize-recover=all", "-o", str(exe), os.path.join(HERE, "cpp", "rows_share_check.cc")], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and r.stdout.startswith("ok "), r.stdout + r.stderr
    assert all(int(x) > 10000 for x in r.stdout.split()[1:])


M = 1 << 20                                                   # rows that share nothing
ROWS = dict(q=M, k=2 * M, v=3 * M, q_out=4 * M, k_out=5 * M, rows=4, q_stride=256, k_stride=128, v_stride=128, q_out_stride=256, k_out_stride=128)


@pytest.mark.parametrize("kw", [dict(q_out=M + 2), dict(q_out=M, q_out_stride=264), dict(k_out=2 * M - 254), dict(q_out=2 * M + 256), dict(k_out=M + 512), dict(k_out=4 * M + 1024), dict(q_out=2 * M),
                                dict(q=M, k=M + 512, q_stride=512, k_stride=512, q_out=M + 256, q_out_stride=512)])
def test_outputs_that_share_memory_with_other_rows_are_refused(kw):
    L = sg.lib()
    assert L.smeg_rotate_heads_dev(_rotate(**{**ROWS, **kw}), None) == -4
    assert L.smeg_paged_append_dev(_paged(**{**ROWS, **kw}), None) == -4


def test_outputs_in_place_and_side_by_side_are_not_refused():
    """Past the checks, which without a GPU ends at the device (-5)."""
    if torch.cuda.is_available():
        pytest.skip("would run on made-up addresses")
    L = sg.lib()
    wide = dict(q_stride=512, k_stride=512, v_stride=512, q_out_stride=512, k_out_stride=512)
    for kw in (dict(), dict(q_out=M, k_out=2 * M), {**wide, **dict(q=M, k=M + 512, v=M + 768, q_out=M, k_out=M + 512)}, {**wide, **dict(q=M, k=M + 512, v=M + 768, q_out=2 * M, k_out=2 * M + 512)}):
        assert L.smeg_rotate_heads_dev(_rotate(**{**ROWS, **kw}), None) == -5
        assert L.smeg_paged_append_dev(_paged(**{**ROWS, **kw}), None) == -5
    for kw in (dict(v=M + 512, **wide), dict(k_out=3 * M), dict(q_out=3 * M + 4)):
        assert L.smeg_paged_append_dev(_paged(**{**ROWS, **{**dict(q=M, q_out=M), **kw}}), None) == (-5 if "q_stride" in kw else -4)
    a = dict(q=M, out=M + 256, q_stride=256, out_stride=256, codes=4096, scales=4096, cu=4096, starts=4096, table=4096, seqs=2, cols=3, pages=5, page=64, rows=2,
             heads=2, kv_heads=2, head_dim=64, scale=0.125, bf16=0, ws=0, bytes=0)
    assert L.smeg_paged_attend_dev(PAGED_ATTEND_ARGS.pack(*a.values()), None) == -5
    for at in (M, M + 2, M + 254, M - 2, M + 512):
        assert L.smeg_paged_attend_dev(PAGED_ATTEND_ARGS.pack(*{**a, "out": at}.values()), None) == -4
    a = dict(q=M, k=M + 512, v=M + 768, out=2 * M, q_stride=512, k_stride=512, v_stride=512, out_stride=256, cu=4096, seqs=1, rows=2, heads=4, kv_heads=2, head_dim=64, scale=0.125, bf16=0)
    assert L.smeg_attn_packed_dev(ATTN_PACKED_ARGS.pack(*a.values()), None) == -5
    for at in (M, M + 512, M + 1022, M + 1024 + 768 + 254):
        assert L.smeg_attn_packed_dev(ATTN_PACKED_ARGS.pack(*{**a, "out": at}.values()), None) == -4


def test_a_copied_rotation_has_no_addresses_of_the_first_one():
    import copy
    import pickle
    r = sg.Rotary(64, base=500.0, rotary_dim=32, interleaved=True).yarn(8.0, 4096)
    r._turns[0] = (4096, 8192, None, None)                    # as a call on device 0 leaves it
    for c in (copy.copy(r), copy.deepcopy(r), pickle.loads(pickle.dumps(r))):
        assert c._turns == {} and c._call[0] is c._turns and c._call[1:] == r._call[1:]
        assert np.array_equal(c.frequencies(), r.frequencies()) and c.factor() == r.factor()
        assert (c.head_dim(), c.rotary_dim(), c.interleaved()) == (64, 32, True)
        assert np.array_equal(c.linear(2.0).frequencies(), r.linear(2.0).frequencies())


def test_a_blocks_rotation_is_set_by_with_rotary_alone():
    class Part:                                               # as wide as a projection, without weights
        def __init__(self, n, k):
            self.n, self.k = (lambda: n), (lambda: k)

    attn = sg.SelfAttention(Part(8 * 64, 256), Part(256, 4 * 64), 4, 2, 64)
    assert attn.rotary is None and attn.q_norm is None and attn.k_norm is None and not attn._turns
    for name in ("rotary", "q_norm", "k_norm"):
        with pytest.raises(AttributeError):
            setattr(attn, name, sg.Rotary(64))
    r = sg.Rotary(64)
    assert attn.with_rotary(r) is attn and attn.rotary is r and attn._turns
    assert not attn.with_rotary(None)._turns and attn.rotary is None


def test_the_library_builds_without_torch():
    code = ("import sys; sys.modules['torch'] = None\n"
            "from sme_gemm_b200 import build\nprint(build.build(), build.build_binding())")
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=600, cwd=os.path.dirname(HERE))
    assert r.returncode == 0 and r.stdout.strip().endswith("libsmeg_b200.so None") and "paged.py" in r.stderr, r.stdout + r.stderr


def test_the_binding_is_built_again_for_another_torch(monkeypatch, tmp_path):
    from sme_gemm_b200 import build
    runs = []

    def run(cmd, **kw):
        runs.append(cmd)
        out = cmd[cmd.index("-o") + 1]
        open(out, "w").close()
        return subprocess.CompletedProcess(cmd, 0, "", "")

    monkeypatch.setattr(build, "HERE", str(tmp_path / "pkg"))
    monkeypatch.setattr(build.subprocess, "run", run)
    os.makedirs(tmp_path / "pkg")
    os.makedirs(tmp_path / "include")
    open(tmp_path / "include" / "smeg_api.h", "w").close()
    out = build.build_binding()
    assert len(runs) == 1 and build.build_binding() == out and len(runs) == 1
    monkeypatch.setattr(torch, "__version__", "0.0.other")
    assert build.build_binding() == out and len(runs) == 2 and build.build_binding() == out and len(runs) == 2
    monkeypatch.setattr(torch, "compiled_with_cxx11_abi", lambda: not runs)
    build.build_binding()
    assert len(runs) == 3
    os.remove(out)
    build.build_binding()
    assert len(runs) == 4


def test_a_binding_that_does_not_load_says_why(monkeypatch):
    from sme_gemm_b200 import paged
    monkeypatch.setattr(paged, "_CALLS", None)

    def fails(*a):
        raise ImportError("undefined symbol: of_another_torch")

    monkeypatch.setattr(paged.importlib, "import_module", fails)
    with pytest.raises(RuntimeError, match="does not load .undefined symbol: of_another_torch.*build it"):
        paged._calls()
    monkeypatch.setattr(paged.os, "listdir", lambda d: ["paged.py"])
    with pytest.raises(RuntimeError, match="_binding is missing: build it"):
        paged._calls()
