"""The attention of a serving step, operator by operator: what their speed is measured on.

Queries, keys and values come as the 16-bit rows that a fused [q | k | v] projection leaves, the sequences of a batch packed one behind the other
(`cu_rows[s] .. cu_rows[s + 1]` are sequence s's rows).  Four operators:

  rotate   RMS norms of the query and key heads and the rotation by position, in one pass (`rotate_heads`)
  append   the same, with the keys and values quantised into the pages of an 8-bit cache on the way (`PagedKvCache.append`), and the pages that
           were written read back as the values they stand for (`PagedKvCache.read`)
  paged    attention of new rows against that cache (`PagedKvCache.attend`)
  prompt   causal attention over whole packed prompts, grouped heads (`attend_packed`)

The cache holds a byte code + 128 per value, pages of `page` positions, and a 32-bit scale for each page, KV head and keys or values: scale =
largest magnitude / 127.  A page's scale starts with its first position and only grows; where it does, the codes that are there are rounded again.
"""
import math

import numpy as np
import torch

own = False

F16 = {"f16": torch.float16, "bf16": torch.bfloat16}
BASE = 10000.0


def listed():
    return [
        # one generated token: 32 query and 8 key heads of 128, normalised and rotated in place of two passes each
        {"name": "rotate_1", "kind": "rotate", "rows": 1, "heads": 32, "kv_heads": 8, "hd": 128, "rot": 128, "layout": "half", "scaling": "none",
         "norm": True, "start": 4095, "dtype": "f16"},
        # a prompt of odd length, far along in a long context: half of each head rotated, neighbouring pairs, stretched frequencies, no norms
        {"name": "rotate_2001_part_bf16", "kind": "rotate", "rows": 2001, "heads": 28, "kv_heads": 4, "hd": 96, "rot": 48, "layout": "interleaved",
         "scaling": "yarn", "norm": False, "start": 200000, "dtype": "bf16"},
        # a serving step of 48 sequences, one new token each, small pages
        {"name": "append_decode_48", "kind": "append", "seqs": 48, "rows": 48, "spread": 0.0, "past": 1500, "page": 16, "heads": 32, "kv_heads": 8,
         "hd": 128, "rot": 128, "layout": "half", "scaling": "wavelength", "norm": True, "dtype": "f16"},
        # a short chunk behind 100 positions of a character model's cache
        {"name": "append_chunk_37", "kind": "append", "seqs": 1, "rows": 37, "spread": 0.0, "past": 100, "page": 32, "heads": 6, "kv_heads": 6,
         "hd": 64, "rot": 64, "layout": "half", "scaling": "none", "norm": False, "dtype": "f16"},
        # five prompts of different lengths into an empty cache, with normalised heads
        {"name": "append_prompt_4096_bf16", "kind": "append", "seqs": 5, "rows": 4096, "spread": 0.8, "past": 0, "page": 64, "heads": 32,
         "kv_heads": 8, "hd": 128, "rot": 128, "layout": "half", "scaling": "none", "norm": True, "dtype": "bf16"},
        # one generated token over a short context: the smallest call
        {"name": "paged_decode_1", "kind": "paged", "seqs": 1, "rows": 1, "keys": 901, "spread": 0.0, "page": 64, "heads": 32, "kv_heads": 8,
         "hd": 128, "dtype": "f16"},
        # a serving batch: 64 sequences of 500 to 5000 positions, one token each
        {"name": "paged_decode_64_bf16", "kind": "paged", "seqs": 64, "rows": 1, "keys": 2900, "spread": 0.9, "page": 64, "heads": 32, "kv_heads": 8,
         "hd": 128, "dtype": "bf16"},
        # one token over a very long context: the keys have to be shared out
        {"name": "paged_long_131071", "kind": "paged", "seqs": 1, "rows": 1, "keys": 131071, "spread": 0.0, "page": 128, "heads": 32, "kv_heads": 8,
         "hd": 128, "dtype": "f16"},
        # five drafted tokens to be checked in each of twelve sequences, small pages, eight query heads to a KV head
        {"name": "paged_draft_12x5", "kind": "paged", "seqs": 12, "rows": 5, "keys": 2000, "spread": 0.6, "page": 16, "heads": 24, "kv_heads": 3,
         "hd": 64, "dtype": "f16"},
        # a short prompt through a character model's layer
        {"name": "prompt_1x200", "kind": "prompt", "seqs": 1, "rows": 200, "spread": 0.0, "heads": 6, "kv_heads": 6, "hd": 64, "dtype": "f16"},
        # eleven prompts of different lengths in one call
        {"name": "prompt_11x7001_bf16", "kind": "prompt", "seqs": 11, "rows": 7001, "spread": 0.9, "heads": 32, "kv_heads": 8, "hd": 128,
         "dtype": "bf16"},
        # one long prompt: the largest
        {"name": "prompt_1x8192", "kind": "prompt", "seqs": 1, "rows": 8192, "spread": 0.0, "heads": 32, "kv_heads": 8, "hd": 128, "dtype": "f16"},
    ]


# ------------------------------------------------------------------------------------------------ more of the same ranges

def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


# (query heads, KV heads, depths of a head)
HEADS = [(32, 8, 128), (6, 6, 64), (24, 3, 64), (28, 4, 96), (12, 4, 80), (28, 4, 128), (16, 2, 256), (8, 1, 128), (20, 20, 64), (32, 32, 128),
         (10, 2, 64), (4, 4, 32), (14, 2, 112)]


def draw(rng):
    heads, kv_heads, hd = rng.choice(HEADS)
    shape = {"heads": heads, "kv_heads": kv_heads, "hd": hd, "dtype": rng.choice(["f16", "bf16"])}
    turn = {"rot": max(8, int(hd * rng.choice([1, 1, 0.5, 0.25])) // 2 * 2), "layout": rng.choice(["half", "half", "interleaved"]),
            "scaling": rng.choice(["none", "none", "linear", "wavelength", "yarn"]), "norm": rng.random() < 0.5}
    kind = rng.choice(["rotate", "append", "append", "paged", "paged", "prompt", "prompt"])
    if kind == "rotate":
        return {"kind": kind, "rows": _log(rng, 1, 8192), **shape, **turn, "start": rng.choice([0, _log(rng, 1, 1000000)])}
    if kind == "append":
        seqs = _log(rng, 1, 128)
        rows = seqs if rng.random() < 0.4 else max(seqs, _log(rng, 2, 8192))
        return {"kind": kind, "seqs": seqs, "rows": rows, "spread": round(rng.uniform(0, 0.9), 2), "past": rng.choice([0, _log(rng, 1, 4000)]),
                "page": rng.choice([16, 32, 64, 128, 256]), **shape, **turn}
    if kind == "paged":
        seqs = _log(rng, 1, 128)
        rows = rng.choice([1, 1, 1, 2, 3, 5, 8])
        keys = max(2 * rows, _log(rng, 1, max(2, 131071 * 8 * 128 // (seqs * kv_heads * hd))))
        return {"kind": kind, "seqs": seqs, "rows": rows, "keys": min(keys, 131071), "spread": round(rng.uniform(0, 0.9), 2),
                "page": rng.choice([16, 32, 64, 128, 256]), **shape}
    rows = _log(rng, 1, 8192 if heads * hd <= 4096 else 4096)
    return {"kind": kind, "seqs": max(1, min(rows, _log(rng, 1, 40))), "rows": rows, "spread": round(rng.uniform(0, 0.9), 2), **shape}


def _ragged(total, n, spread):
    """n lengths that add up to total, none below one: the same for every seed, so that the work is the case's."""
    w = [1.0 - spread * ((i * 0.6180339887) % 1.0) for i in range(n)]
    got = [max(1, int(total * x / sum(w))) for x in w]
    i = 0
    while sum(got) != total:                                  # what the rounding left over, one by one
        d = 1 if sum(got) < total else -1
        if got[i % n] + d >= 1:
            got[i % n] += d
        i += 1
    return got


def _rows_of(case):
    if case["kind"] == "rotate":
        return [case["rows"]]
    if case["kind"] == "paged":
        return [case["rows"]] * case["seqs"]
    return _ragged(case["rows"], case["seqs"], case["spread"])


def _starts_of(case):
    """Positions that each sequence has in the cache before the call's rows."""
    n = case["seqs"]
    if case["kind"] == "append":
        return [int(case["past"] * (1.0 - 0.7 * ((i * 0.7548776662) % 1.0))) for i in range(n)]
    return [max(0, x - case["rows"]) for x in _ragged(max(n, case["keys"] * n), n, case["spread"])]


# ------------------------------------------------------------------------------------------------ inputs

def _frequencies(case):
    """Radians per position of each rotated pair, and the factor on the cosines and sines."""
    rot = case["rot"]
    i = np.arange(rot // 2, dtype=np.float64)
    f = BASE ** (-2.0 * i / rot)
    if case["scaling"] == "linear":
        return f / 4.0, 1.0
    if case["scaling"] == "wavelength":                       # factor 8, from an original context of 8192, bounds 1 and 4
        turns = 8192.0 * f / (2.0 * np.pi)
        s = np.clip((turns - 1.0) / (4.0 - 1.0), 0.0, 1.0)
        return (1.0 - s) * f / 8.0 + s * f, 1.0
    if case["scaling"] == "yarn":                             # factor 16, from an original context of 4096, bounds 32 and 1
        at = lambda turns: rot * math.log(4096.0 / (turns * 2.0 * math.pi)) / (2.0 * math.log(BASE))  # noqa: E731
        lo, hi = max(math.floor(at(32.0)), 0), min(math.ceil(at(1.0)), rot - 1)
        r = np.clip((i - lo) / max(hi - lo, 0.001), 0.0, 1.0)
        return f / 16.0 * r + f * (1.0 - r), 0.1 * math.log(16.0) + 1.0
    return f, 1.0


def _rotary(case):
    import sme_gemm_b200 as sg
    r = sg.Rotary(case["hd"], base=BASE, rotary_dim=case["rot"], interleaved=case["layout"] == "interleaved")
    if case["scaling"] == "linear":
        return r.linear(4.0)
    if case["scaling"] == "wavelength":
        return r.by_wavelength(8.0, 1.0, 4.0, 8192)
    if case["scaling"] == "yarn":
        return r.yarn(16.0, 4096)
    return r


def _randn(gen, *shape):
    return torch.randn(shape, generator=gen, device="cuda")


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    kind, heads, kv, hd, dtype = case["kind"], case["heads"], case["kv_heads"], case["hd"], F16[case["dtype"]]
    rows = _rows_of(case)
    total = sum(rows)
    st = {"case": case, "total": total}
    # the rows of a fused projection: queries, keys and values side by side
    qkv = _randn(gen, total, (heads + 2 * kv) * hd)
    if kind == "prompt":
        qkv[:, :heads * hd] *= 1.5                            # scores of some spread
    st["qkv"] = qkv.to(dtype)
    q_len, kv_len = heads * hd, kv * hd
    st["q"], st["k"], st["v"] = st["qkv"][:, :q_len], st["qkv"][:, q_len:q_len + kv_len], st["qkv"][:, q_len + kv_len:]
    st["q_out"] = torch.empty((total, q_len), dtype=dtype, device="cuda")
    cu = np.concatenate([[0], np.cumsum(rows)])
    st["cu"] = torch.tensor(cu, dtype=torch.int32, device="cuda")
    if kind in ("rotate", "append"):
        if case["norm"]:
            st["q_w"], st["k_w"] = 1.0 + 0.1 * _randn(gen, hd), 1.0 + 0.1 * _randn(gen, hd)
        f, factor = _frequencies(case)
        st["freq"], st["factor"] = torch.tensor(f, device="cuda"), factor
        if kind == "rotate" or case["rows"] > case["seqs"]:
            st["k_out"] = torch.empty((total, kv_len), dtype=dtype, device="cuda")
        if own:
            import sme_gemm_b200 as sg
            st["rotary"] = _rotary(case)
            st["norms"] = [sg.Norm.rms(st[w].cpu().numpy(), 1e-6) if case["norm"] else None for w in ("q_w", "k_w")]
    if kind == "rotate":
        st["pos"] = torch.arange(case["start"], case["start"] + total, dtype=torch.int32, device="cuda")
        return st
    st["seq"] = torch.tensor(np.repeat(np.arange(len(rows)), rows), device="cuda")
    if kind == "prompt":
        st["in_seq"] = torch.tensor(np.concatenate([np.arange(r) for r in rows]), device="cuda")
        st["longest"] = max(rows)
        return st
    # the cache: pages of the pool in no order, gaussian values in those that sequences hold
    starts, page = _starts_of(case), case["page"]
    st["starts"] = torch.tensor(starts, dtype=torch.int32, device="cuda")
    st["pos"] = torch.tensor(np.concatenate([a + np.arange(r) for a, r in zip(starts, rows)]), device="cuda")
    held = [-(-(a + r) // page) for a, r in zip(starts, rows)]
    pages = sum(held) + 3
    ids = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
    table = torch.full((len(rows), max(held)), -1, dtype=torch.int32, device="cuda")
    owner = torch.tensor(np.repeat(np.arange(len(rows)), held), device="cuda")
    nth = torch.tensor(np.concatenate([np.arange(h) for h in held]), device="cuda")
    table[owner, nth] = ids[:len(nth)]
    st["table"] = table
    st["codes"] = (_randn(gen, pages, kv, 2, page, hd) * 32 + 128).round_().clamp_(1, 255).to(torch.uint8)
    st["scales"] = 0.015 + 0.02 * torch.rand((pages, kv, 2), generator=gen, device="cuda")
    if kind == "append":
        new = [table[s, n] for s, (a, r) in enumerate(zip(starts, rows)) for n in range(a // page, (a + r - 1) // page + 1)]
        st["touched"] = torch.stack(new)
        st["values"] = torch.empty((len(new), kv, 2, page, hd), dtype=dtype, device="cuda")
    if own:
        import sme_gemm_b200 as sg
        st["cache"] = sg.PagedKvCache(heads, kv, hd, pages, page)
        st["cache"].codes.copy_(st["codes"])
        st["cache"].scales.copy_(st["scales"])
        st["batch"] = sg.PagedBatch(st["cu"], st["starts"], st["table"])
    return st


# ------------------------------------------------------------------------------------------------ one pass

def run(st):
    kind = st["case"]["kind"]
    if own:
        import sme_gemm_b200 as sg
        if kind == "rotate":
            sg.rotate_heads(st["q"], st["k"], st["pos"], st["rotary"], st["q_out"], st["k_out"], q_norm=st["norms"][0], k_norm=st["norms"][1])
            return {"q": st["q_out"], "k": st["k_out"]}
        if kind == "append":
            st["cache"].append(st["k"], st["v"], st["batch"], st["rotary"], q=st["q"], q_out=st["q_out"], k_out=st.get("k_out"),
                               q_norm=st["norms"][0], k_norm=st["norms"][1])
            st["cache"].read(st["touched"], st["values"])
            return {"q": st["q_out"], "k": st.get("k_out"), "pages": st["values"]}
        if kind == "paged":
            st["cache"].attend(st["q"], st["batch"], st["q_out"])
            return st["q_out"]
        c = st["case"]
        sg.attend_packed(st["q"], st["k"], st["v"], st["cu"], st["q_out"], c["heads"], c["kv_heads"])
        return st["q_out"]
    return {"rotate": _rotate, "append": _append, "paged": _paged, "prompt": _prompt}[kind](st)


def _turned(st, x, w):
    """Heads (rows, heads, depths), 32 bits: RMS norm, then the rotation by the row's position."""
    c = st["case"]
    x = x.float().reshape(st["total"], -1, c["hd"])
    if c["norm"]:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * w
    angle = st["pos"].double()[:, None] * st["freq"]          # in 64 bits: far positions turn many times
    cos, sin = (torch.cos(angle) * st["factor"]).float()[:, None], (torch.sin(angle) * st["factor"]).float()[:, None]
    rot = c["rot"]
    out = x.clone()
    if c["layout"] == "half":
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        out[..., :rot // 2], out[..., rot // 2:rot] = a * cos - b * sin, b * cos + a * sin
    else:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        out[..., 0:rot:2], out[..., 1:rot:2] = a * cos - b * sin, b * cos + a * sin
    return out


def _rotate(st):
    dtype = st["qkv"].dtype
    q, k = _turned(st, st["q"], st.get("q_w")), _turned(st, st["k"], st.get("k_w"))
    return {"q": q.reshape(st["total"], -1).to(dtype), "k": k.reshape(st["total"], -1).to(dtype)}


def _append(st):
    c, dtype = st["case"], st["qkv"].dtype
    page, kv, hd = c["page"], c["kv_heads"], c["hd"]
    q, k = _turned(st, st["q"], st.get("q_w")), _turned(st, st["k"], st.get("k_w"))
    new = torch.stack([k, st["v"].float().reshape(st["total"], kv, hd)], 2)                     # rows, KV heads, keys | values, depths
    at, slot = st["table"][st["seq"], st["pos"] // page].long(), st["pos"] % page
    codes, scales, ids = st["codes"], st["scales"], st["touched"].long()
    fresh = torch.zeros(len(scales), dtype=torch.bool, device="cuda")
    fresh[at[slot == 0]] = True                                # pages that begin with this call
    first = torch.full((len(scales),), page, device="cuda").index_reduce_(0, at, slot, "amin")  # the call's first position of each page
    want = torch.zeros_like(scales).index_reduce_(0, at, new.abs().amax(-1), "amax") / 127.0
    old = torch.where(fresh[:, None, None], torch.zeros_like(scales), scales)
    grown = torch.maximum(old, want)[ids]
    ratio = torch.where(grown > old[ids], old[ids] / grown, torch.ones_like(grown))
    there = torch.arange(page, device="cuda")[None, :] < first[ids][:, None]                    # positions of earlier calls
    was = codes[ids].float() - 128.0
    again = torch.round(was * ratio[..., None, None]) + 128.0
    codes[ids] = torch.where(there[:, None, None, :, None], again, was + 128.0).to(torch.uint8)
    scales[ids] = grown
    s = scales[at][..., None]
    codes[at, :, :, slot] = (torch.round(torch.where(s > 0, new / s, torch.zeros_like(new))).clamp(-127, 127) + 128.0).to(torch.uint8)
    values = ((codes[ids].float() - 128.0) * scales[ids][..., None, None]).to(dtype)
    k_out = k.reshape(st["total"], -1).to(dtype) if "k_out" in st else None
    return {"q": q.reshape(st["total"], -1).to(dtype), "k": k_out, "pages": values}


def _paged(st):
    c = st["case"]
    heads, kv, hd, rows, n = c["heads"], c["kv_heads"], c["hd"], c["rows"], c["seqs"]
    ids = st["table"].long().clamp(min=0)
    values = (st["codes"][ids].float() - 128.0) * st["scales"][ids][..., None, None]            # sequences, pages, KV heads, 2, positions, depths
    values = values.permute(3, 0, 2, 1, 4, 5).reshape(2, n, kv, -1, hd)
    q = st["q"].float().reshape(n, rows, kv, heads // kv, hd).permute(0, 2, 1, 3, 4).reshape(n, kv, -1, hd)
    s = q @ values[0].transpose(-1, -2) / math.sqrt(hd)                                         # sequences, KV heads, rows x heads of a group, positions
    last = st["pos"].reshape(n, 1, rows, 1).expand(n, 1, rows, heads // kv).reshape(n, 1, -1, 1)
    s = s.masked_fill_(torch.arange(s.shape[-1], device="cuda") > last, -math.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True))
    o = p @ values[1] / p.sum(-1, keepdim=True)
    return o.reshape(n, kv, rows, heads // kv, hd).permute(0, 2, 1, 3, 4).reshape(n * rows, heads * hd).to(st["qkv"].dtype)


def _prompt(st):
    c, total = st["case"], st["total"]
    heads, kv, hd, n, most = c["heads"], c["kv_heads"], c["hd"], c["seqs"], st["longest"]
    # packed rows to sequences of one length: (sequences, heads, rows, depths)
    x = torch.zeros((n, most, heads + 2 * kv, hd), device="cuda")
    x[st["seq"], st["in_seq"]] = st["qkv"].float().reshape(total, heads + 2 * kv, hd)
    q, k, v = (y.transpose(1, 2) for y in x.split([heads, kv, kv], 2))
    q = q.reshape(n, kv, heads // kv * most, hd)
    s = q @ k.transpose(-1, -2) / math.sqrt(hd)
    i = torch.arange(most, device="cuda")
    s = s.reshape(n, kv, heads // kv, most, most).masked_fill_(i[None, :] > i[:, None], -math.inf)
    p = s.sub_(s.amax(-1, keepdim=True)).exp_()
    p = p.div_(p.sum(-1, keepdim=True)).reshape(n, kv, heads // kv * most, most)
    o = (p @ v).reshape(n, heads, most, hd).transpose(1, 2)
    return o[st["seq"], st["in_seq"]].reshape(total, heads * hd).to(st["qkv"].dtype)


# ------------------------------------------------------------------------------------------------ what a pass cannot do without

def work(case):
    kind, heads, kv, hd = case["kind"], case["heads"], case["kv_heads"], case["hd"]
    rows = _rows_of(case)
    total = sum(rows)
    if kind == "rotate":
        return {"bytes": 2 * 2 * total * (heads + kv) * hd + 4 * total, "flops": 8 * total * (heads + kv) * hd}
    if kind == "append":
        page, starts = case["page"], _starts_of(case)
        touched = sum((a + r - 1) // page - a // page + 1 for a, r in zip(starts, rows))
        read = 2 * total * (heads + 2 * kv) * hd + 4 * (2 * len(rows) + touched)
        wrote = 2 * total * heads * hd + 2 * total * kv * hd + (2 * total * kv * hd if case["rows"] > case["seqs"] else 0)
        values = touched * kv * 2 * page * hd
        return {"bytes": read + wrote + 3 * values + 8 * touched * kv, "flops": 8 * total * (heads + 2 * kv) * hd + values}
    if kind == "paged":
        page, starts = case["page"], _starts_of(case)
        keys = sum(a + case["rows"] for a in starts)
        pages = sum(-(-(a + case["rows"]) // page) for a in starts)
        pairs = sum(case["rows"] * a + case["rows"] * (case["rows"] + 1) // 2 for a in starts)
        return {"bytes": keys * kv * 2 * hd + pages * (8 * kv + 4) + 2 * 2 * total * heads * hd, "flops": 4 * pairs * heads * hd}
    pairs = sum(r * (r + 1) // 2 for r in rows)
    return {"bytes": 2 * total * (2 * heads + 2 * kv) * hd + 4 * len(rows), "flops": 4 * pairs * heads * hd}


# ------------------------------------------------------------------------------------------------ the definitions, in 64 bits

def _exact_head_rows(case, x, w, positions):
    """One tensor of heads (rows, heads, depths) in 64 bits, from the definition, pair by pair."""
    x = x.double()
    if case["norm"]:
        x = x / torch.sqrt(x.pow(2).sum(-1, keepdim=True) / case["hd"] + 1e-6) * w.double()
    y, rot = x.clone(), case["rot"]
    for j in range(rot // 2):
        f, factor = BASE ** (-2.0 * j / rot), 1.0
        if case["scaling"] == "linear":
            f /= 4.0
        elif case["scaling"] == "wavelength":
            wave = 2.0 * math.pi / f
            if wave > 8192.0 / 1.0:
                f /= 8.0
            elif wave >= 8192.0 / 4.0:
                s = (8192.0 / wave - 1.0) / (4.0 - 1.0)
                f = (1.0 - s) * f / 8.0 + s * f
        elif case["scaling"] == "yarn":
            factor = 0.1 * math.log(16.0) + 1.0
            lo = max(math.floor(rot * math.log(4096.0 / (32.0 * 2.0 * math.pi)) / (2.0 * math.log(BASE))), 0)
            hi = min(math.ceil(rot * math.log(4096.0 / (1.0 * 2.0 * math.pi)) / (2.0 * math.log(BASE))), rot - 1)
            r = min(max((j - lo) / max(hi - lo, 0.001), 0.0), 1.0)
            f = f / 16.0 * r + f * (1.0 - r)
        a, b = (j, j + rot // 2) if case["layout"] == "half" else (2 * j, 2 * j + 1)
        z = torch.polar(torch.full_like(positions, factor), positions * f)[:, None] * torch.complex(x[..., a], x[..., b])
        y[..., a], y[..., b] = z.real, z.imag
    return y


def exact(case, seed):
    kind, heads, kv, hd = case["kind"], case["heads"], case["kv_heads"], case["hd"]
    st = prepare(case, seed)
    total, group = st["total"], heads // kv
    if kind in ("rotate", "append"):
        at = st["pos"].double()
        q = _exact_head_rows(case, st["q"].reshape(total, heads, hd), st.get("q_w"), at)
        k = _exact_head_rows(case, st["k"].reshape(total, kv, hd), st.get("k_w"), at)
        got = {"q": q.reshape(total, -1), "k": k.reshape(total, -1) if "k_out" in st else None}
        if kind == "rotate":
            return got
        page, rows, starts = case["page"], _rows_of(case), _starts_of(case)
        new = torch.stack([k, st["v"].reshape(total, kv, hd).double()], 1)                      # rows, keys | values, KV heads, depths
        pages, row, n = [], 0, 0
        for a, r in zip(starts, rows):
            done = 0
            while done < r:                                    # page by page, as the positions come
                slot, here = (a + done) % page, min(r - done, page - (a + done) % page)
                p = int(st["touched"][n])
                part = new[row + done:row + done + here].permute(2, 1, 0, 3)                    # KV heads, 2, positions, depths
                old = st["scales"][p].double() if slot else torch.zeros((kv, 2), dtype=torch.float64, device="cuda")
                scale = torch.maximum(old, part.abs().amax((-1, -2)) / 127.0)
                code = st["codes"][p].double() - 128.0
                grown = scale > old
                code[:, :, :slot] = torch.where(grown[..., None, None], torch.round(code[:, :, :slot] * (old / scale)[..., None, None]), code[:, :, :slot])
                code[:, :, slot:slot + here] = torch.round(part / scale[..., None, None]).clamp(-127, 127)
                pages.append(code * scale[..., None, None])
                done, n = done + here, n + 1
            row += r
        got["pages"] = torch.stack(pages)
        return got
    out = torch.empty((total, heads, hd), dtype=torch.float64, device="cuda")
    row = 0
    for s, r in enumerate(_rows_of(case)):
        if kind == "paged":
            end = _starts_of(case)[s] + r
            mine = st["table"][s, :-(-end // case["page"])].long()
            both = (st["codes"][mine].double() - 128.0) * st["scales"][mine].double()[..., None, None]
            both = both.permute(2, 1, 0, 3, 4).reshape(2, kv, -1, hd)[:, :, :end]               # keys | values, KV heads, positions, depths
        else:
            end = r
            both = torch.stack([st[x][row:row + r].reshape(r, kv, hd).double().transpose(0, 1) for x in ("k", "v")])
        for h in range(heads):
            q = st["q"][row:row + r].reshape(r, heads, hd)[:, h].double()
            for i in range(0, r, 2048):                        # rows i .. of the head, 2048 at a time
                z = q[i:i + 2048] @ both[0, h // group].T * hd ** -0.5
                n = torch.arange(i, i + len(z), device="cuda")[:, None] + end - r
                z = torch.where(torch.arange(end, device="cuda")[None] <= n, z, torch.full_like(z, -math.inf))
                out[row + i:row + i + len(z), h] = torch.softmax(z, -1) @ both[1, h // group]
        row += r
    return out.reshape(total, heads * hd)
