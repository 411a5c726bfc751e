# SPDX-License-Identifier: Unlicense
"""Operators of a transformer layer over a kept sequence, as measurable cases:
a norm that takes the residual's addition along and leaves 8-bit codes for the
next layer, keys and values coded as they are kept and read back, attention
within a window and over the first tokens, of float32 keys and of kept ones.

A case is a dict of plain values with a "kind":

norm    h = x + r, y = h / rms(h) g: y in float32 ("out": "float"), in 8-bit
        codes with a scale per token ("q8"), or in both ("both")
cache   the new tokens' keys and values of several sequences written to their
        pages in 8 bits, a scale per token and head; the last `back` tokens
        of each sequence, the new ones among them, read back
window  attention of the last nq of nk positions: a query at position p sees
        the positions p - left .. p + right and those of the first `sinks`
        that are not behind p + right
attend  the same with right = 0 over the kept 8-bit keys and values, for the
        new tokens of several sequences of unlike lengths; left = -1: every
        earlier token

`run` computes a case with elementary torch operations, or, with `own`, by
the library's entry points. Tensors live in torch memory; the library gets
views of it and queues its work on a stream of its own, which torch's streams
and events know nothing of: what `run` returns then is valid, and a state may
be written by torch or dropped, only after torch.cuda.synchronize().
"""

import ctypes
import importlib.util
import math
import random
import sys
from pathlib import Path

import numpy as np
import torch

ROOT = Path(__file__).resolve().parent.parent
own = False

EPS = float(np.float32(1e-6))
# The smallest row maximum that keeps its codes; rows below it count as zero.
TINY = 2.0 ** -100
# Queries of a piece of the plain form's window.
PIECE = 512
_held = {}


def _package():
    """The package (its folder is no Python identifier)."""
    if "icoreg_amd" not in sys.modules:
        folder = ROOT / "i.coregistration.opencl_amd"
        spec = importlib.util.spec_from_file_location("icoreg_amd", folder / "__init__.py")
        mod = importlib.util.module_from_spec(spec)
        sys.modules["icoreg_amd"] = mod
        spec.loader.exec_module(mod)
    return sys.modules["icoreg_amd"]


def _device():
    if "device" not in _held:
        torch.cuda.init()
        _held["device"] = _package().Device("auto")
    return _held["device"]


# ---- the cases ---------------------------------------------------------------


def listed():
    return [
        # One token between two layers of a ViT-L: latency.
        {"name": "norm_token", "kind": "norm", "rows": 1, "c": 1024, "residual": True, "out": "q8"},
        # The tokens of a 560 x 560 pair in a ViT-L/14, for a float32 layer.
        {"name": "norm_vit_pair", "kind": "norm", "rows": 3202, "c": 1024, "residual": True, "out": "float"},
        # A long batch of tokens in front of an 8-bit layer.
        {"name": "norm_long", "kind": "norm", "rows": 12805, "c": 4096, "residual": True, "out": "q8"},
        # One token of each of 32 sequences kept, the tokens of their last
        # blocks read back for the blocks' index.
        {"name": "cache_step", "kind": "cache", "seqs": 32, "most": 8192, "new": 1, "back": 64, "kv_heads": 4,
         "d": 128, "page": 64},
        # The coarse cells of four large tiles kept, and read back whole.
        {"name": "cache_prompt", "kind": "cache", "seqs": 4, "most": 6400, "new": 6400, "back": 6400, "kv_heads": 8,
         "d": 64, "page": 32},
        # One token that sees the last 4096 and the first four.
        {"name": "window_token", "kind": "window", "nq": 1, "nk": 16380, "heads": 16, "kv_heads": 4, "d": 128,
         "left": 4095, "right": 0, "sinks": 4, "masked": False},
        # A ViT-L/14's attention on a 560 x 560 image: four rows of patches
        # either way and the class token.
        {"name": "window_vit_1601", "kind": "window", "nq": 1601, "nk": 1601, "heads": 16, "kv_heads": 16, "d": 64,
         "left": 160, "right": 160, "sinks": 1, "masked": False},
        # The coarse cells of a 640 x 640 tile, four rows either way, part of
        # it without data.
        {"name": "window_grid_6400", "kind": "window", "nq": 6400, "nk": 6400, "heads": 8, "kv_heads": 8, "d": 32,
         "left": 320, "right": 320, "sinks": 0, "masked": True},
        # A long sequence with shared key heads, each token and the ones before it.
        {"name": "window_long", "kind": "window", "nq": 16380, "nk": 16380, "heads": 16, "kv_heads": 4, "d": 128,
         "left": 2047, "right": 0, "sinks": 4, "masked": False},
        # One token over a long cache, all of it.
        {"name": "attend_token", "kind": "attend", "seqs": 1, "most": 131005, "new": 1, "heads": 16, "kv_heads": 4,
         "d": 128, "page": 64, "left": -1, "sinks": 0},
        # One token of each of 64 sequences, whose pages behind the window are
        # given back.
        {"name": "attend_batch", "kind": "attend", "seqs": 64, "most": 16384, "new": 1, "heads": 16, "kv_heads": 4,
         "d": 128, "page": 32, "left": 4095, "sinks": 4},
        # New stretches of three sequences over what is kept of them.
        {"name": "attend_prompt", "kind": "attend", "seqs": 3, "most": 8192, "new": 4096, "heads": 16, "kv_heads": 4,
         "d": 128, "page": 64, "left": -1, "sinks": 0},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    kind = rng.choice(["norm", "cache", "window", "attend"])
    if kind == "norm":
        c = rng.choice([256, 512, 1024, 2048, 4096]) if rng.random() < 0.5 else _log(rng, 64, 4096)
        return {"kind": kind, "rows": _log(rng, 1, 9600), "c": c, "residual": rng.random() < 0.7,
                "out": rng.choice(["float", "q8", "both"])}
    kv, d = rng.choice([1, 2, 4, 8]), rng.choice([16, 32, 40, 64, 100, 128])
    heads = kv * rng.choice([1, 2, 4]) if kv <= 4 else kv * rng.choice([1, 2])
    page = rng.choice([16, 32, 64, 128])
    if kind == "cache":
        seqs = _log(rng, 1, 64)
        new = 1 if rng.random() < 0.4 else _log(rng, 2, 12800 // seqs)
        most = new + _log(rng, 1, max(2, 65536 // seqs))
        return {"kind": kind, "seqs": seqs, "most": most, "new": new,
                "back": min(most, max(new, _log(rng, 1, 12800 // seqs))), "kv_heads": kv, "d": d, "page": page}
    if kind == "window":
        nk = _log(rng, 64, 16380)
        nq = 1 if rng.random() < 0.2 else nk if rng.random() < 0.5 else _log(rng, 2, nk)
        left = _log(rng, 1, 2047)
        return {"kind": kind, "nq": nq, "nk": nk, "heads": heads, "kv_heads": kv, "d": d, "left": left,
                "right": 0 if rng.random() < 0.5 else rng.randint(0, min(left, 512)),
                "sinks": rng.choice([0, 0, 1, 4, 5, 37]), "masked": rng.random() < 0.3}
    left = -1 if rng.random() < 0.5 else _log(rng, 1, 4095)
    if rng.random() < 0.6:
        seqs, new = _log(rng, 1, 64), rng.choice([1, 1, 1, 4])
        most = new + _log(rng, 64, 131000 if left < 0 and seqs == 1 else 262144 // max(seqs, 8))
    else:
        seqs = rng.randint(1, 3)
        new = _log(rng, 2, 4096)
        most = new + _log(rng, 1, 4096)
    return {"kind": kind, "seqs": seqs, "most": most, "new": new, "heads": heads, "kv_heads": kv, "d": d, "page": page,
            "left": left, "sinks": 0 if left < 0 else rng.choice([0, 1, 4, 20])}


def _lengths(c):
    """(tokens kept after the call, new ones among them) of each sequence:
    the first as long as they come, the others at unlike lengths."""
    rng = random.Random(c["seqs"] * 65537 + c["most"])
    new = [c["new"]] + [rng.randint(max(1, c["new"] // 2), c["new"]) for _ in range(c["seqs"] - 1)]
    kept = [c["most"]] + [rng.randint(max(n, c["most"] // 3), c["most"]) for n in new[1:]]
    return kept, new


def _back(c):
    """Tokens of each sequence that are read back."""
    kept, new = _lengths(c)
    return [max(n, min(k, c["back"])) for k, n in zip(kept, new)]


# ---- inputs --------------------------------------------------------------------


def _pitch(d):
    """Bytes of a kept key: its codes and zeros up to a multiple of 16."""
    return -(-d // 16) * 16


def _starts(n):
    return torch.tensor([0] + list(np.cumsum(n)), dtype=torch.int32, device="cuda")


def _pages(c, g):
    """The page table of the sequences, their pages in no order; -1 for pages
    that no query of this call sees, where a window gives them back."""
    kept, new = _lengths(c)
    page, width = c["page"], -(-c["most"] // c["page"])
    at = torch.arange(width)[None]
    kept_t, new_t = torch.tensor(kept)[:, None], torch.tensor(new)[:, None]
    held = at * page < kept_t
    if c.get("left", -1) >= 0:
        held &= ((at + 1) * page > kept_t - new_t - c["left"]) | (at * page < c["sinks"])
    total = int(held.sum())
    table = torch.full(held.shape, -1, dtype=torch.int32)
    order = torch.randperm(total, generator=torch.Generator().manual_seed(g.initial_seed()))
    table[held] = order.int()
    return table.cuda(), total


def _views(t):
    """The library's views of the state's tensors."""
    lib = _package().lib()
    return {k: lib.ocl_wrap(v.data_ptr(), v.numel() * v.element_size()) for k, v in t.items() if v is not None}


def _handles(c, t, m):
    """The library's descriptions of the cache and of the sequences in it."""
    ic = _package()
    if not hasattr(ic, "Cache") or "table" not in t:
        return {}
    h = {"cache": ic.Cache(m["kc"], m["vc"], m["ks"], m["vs"], t["ks"].shape[0], c["page"], c["kv_heads"], c["d"])}
    h |= {n: ic.Seqs(m[n], m["len"], m["table"], c["seqs"], t["table"].shape[1]) for n in ("start", "bstart") if n in m}
    return {k: ctypes.pointer(v) for k, v in h.items()}


def prepare(case, seed):
    c, dev, lib = case, _device(), _package().lib()
    g = torch.Generator("cuda").manual_seed(int(seed))
    randn = lambda *s, std=1.0: std * torch.randn(s, generator=g, device="cuda")  # noqa: E731
    empty = lambda *s, dtype=torch.float32: torch.empty(s, dtype=dtype, device="cuda")  # noqa: E731
    s = {"case": c, "api": dev.api, "po": dev.po}
    if c["kind"] == "norm":
        # A residual stream with a few large channels, as in trained
        # transformers, and what a layer adds to it.
        n, w = c["rows"], c["c"]
        x, r = randn(n, w, std=0.5), randn(n, w, std=2.0) if c["residual"] else None
        (x if r is None else r)[:, :: max(1, w // 3)] *= 20
        t = {"x": x, "r": r, "g": 1 + randn(w, std=0.2), "h": empty(n, w) if c["residual"] else None,
             "y": empty(n, w) if c["out"] != "q8" else None,
             "q": empty(n, -(-w // 64) * 64, dtype=torch.int8) if c["out"] != "float" else None,
             "s": empty(n) if c["out"] != "float" else None}
    elif c["kind"] == "window":
        h, kv, d, nq, nk = (c[n] for n in ("heads", "kv_heads", "d", "nq", "nk"))
        t = {"q": randn(nq, h, d, std=1.4), "k": randn(nk, kv, d), "v": randn(nk, kv, d), "mask": None,
             "out": empty(nq, h, d)}
        if c["masked"]:
            # Stretches without data, as at the border of a mosaic.
            t["mask"] = (randn(-(-nk // 40)).repeat_interleave(40)[:nk] > -0.7).to(torch.uint8)
        if hasattr(lib, "ops_attention_window_work_bytes"):
            t["work"] = empty(lib.ops_attention_window_work_bytes(nq, h, d), dtype=torch.uint8)
    else:
        kept, new = _lengths(c)
        rows, kv, d = sum(new), c["kv_heads"], c["d"]
        table, pages = _pages(c, g)
        # Kept keys and values of unlike size, as heads and tokens have them.
        kc, ks = _codes(randn(pages, kv, c["page"], d) * torch.exp(randn(pages, kv, c["page"], 1, std=0.3)))
        vc, vs = _codes(randn(pages, kv, c["page"], d) * torch.exp(randn(pages, kv, c["page"], 1, std=0.3)))
        t = {"kc": kc, "ks": ks, "vc": vc, "vs": vs, "table": table, "start": _starts(new),
             "len": torch.tensor(kept, dtype=torch.int32, device="cuda")}
        if c["kind"] == "cache":
            t |= {"k": randn(rows, kv, d), "v": randn(rows, kv, d), "bstart": _starts(_back(c)),
                  "bk": empty(sum(_back(c)), kv, d), "bv": empty(sum(_back(c)), kv, d)}
        else:
            t |= {"q": randn(rows, c["heads"], d, std=1.4), "out": empty(rows, c["heads"], d)}
            if hasattr(lib, "ops_attention_cache_work_bytes"):
                t["work"] = empty(lib.ops_attention_cache_work_bytes(rows, c["heads"], d), dtype=torch.uint8)
        s |= {"kept": kept, "new": new, "rows": rows, "back": _back(c) if c["kind"] == "cache" else None}
    s |= {"t": t, "m": _views(t)}
    s["handles"] = _handles(c, t, s["m"])
    torch.cuda.synchronize()
    return s


# ---- a pass: the plain form ------------------------------------------------------


def _codes(x, pitch=None):
    """8-bit codes (rows padded with zeros to the pitch) and scales of the
    rows of x: scale a / 127 of the row's largest magnitude a, code the
    float32 product x (127 / a) to the nearest integer, ties to even."""
    a = x.abs().amax(-1)
    live = a >= TINY
    # Quotients in 64 bits, so that their rounding to 32 is the nearest one.
    r = torch.where(live, (127.0 / torch.where(live, a, 1.0).double()).float(), 0.0)
    q = torch.zeros(x.shape[:-1] + (pitch or _pitch(x.shape[-1]),), dtype=torch.int8, device=x.device)
    q[..., : x.shape[-1]] = (x * r[..., None]).round_().to(torch.int8)
    return q, torch.where(live, (a.double() / 127.0).float(), 0.0)


def _norm(c, t):
    """The mean of the squares in 64 bits, its root's reciprocal rounded to
    float32, and two products rounded to float32: the codes next to a border
    do not depend on an order of summation."""
    h = t["x"] if t["r"] is None else t["x"] + t["r"]
    inv = (1 / (h.double().square().mean(-1, keepdim=True) + EPS).sqrt()).float()
    y = h * inv * t["g"]
    out = {} if t["r"] is None else {"h": h}
    if c["out"] != "q8":
        out["y"] = y
    if c["out"] != "float":
        out["q"], out["s"] = _codes(y, -(-c["c"] // 64) * 64)
    return out


def _places(c, t, kept, n):
    """(page, place) of the last n[b] tokens of each sequence b, in order."""
    n = torch.tensor(n, device="cuda")
    owner = torch.repeat_interleave(torch.arange(c["seqs"], device="cuda"), n)
    pos = torch.arange(len(owner), device="cuda") - (n.cumsum(0) - n)[owner] + (torch.tensor(kept, device="cuda") - n)[owner]
    return t["table"][owner, pos // c["page"]].long(), pos % c["page"]


def _cache(c, s):
    t, out = s["t"], {}
    page, at = _places(c, t, s["kept"], s["new"])
    bpage, bat = _places(c, t, s["kept"], s["back"])
    for x, codes, scales in (("k", "kc", "ks"), ("v", "vc", "vs")):
        # As the cache has them, (page, head, place, channel).
        t[codes][page, :, at], t[scales][page, :, at] = _codes(t[x])
        out[x] = t[codes][bpage, :, bat][..., : c["d"]].float() * t[scales][bpage, :, bat][..., None]
    return out


def _softmax_rows(s, v):
    """softmax(s) v over the last axis of s; zeros where s is all -inf."""
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s.sub_(torch.where(top > -math.inf, top, 0.0)))
    total = p.sum(-1, keepdim=True)
    return torch.matmul(p, v) / torch.where(total > 0, total, 1.0)


def _attend(q, k, v, keep):
    """q (batch, n, heads, d) over k, v (batch, keys, key heads, d) where
    keep (batch, n, keys): (batch, n, heads, d)."""
    b, n, h, d = q.shape
    kv = k.shape[2]
    q = (q * d ** -0.5).view(b, n, kv, h // kv, d).permute(0, 2, 3, 1, 4).reshape(b, kv, -1, d)
    s = torch.matmul(q, k.permute(0, 2, 3, 1).contiguous()).view(b, kv, h // kv, n, -1)
    s.masked_fill_(~keep[:, None, None], -math.inf)
    o = _softmax_rows(s.view(b, kv, (h // kv) * n, -1), v.permute(0, 2, 1, 3).contiguous())
    return o.view(b, kv, h // kv, n, d).permute(0, 3, 1, 2, 4).reshape(b, n, h, d)


def _window(c, t):
    nq, nk, left, right = c["nq"], c["nk"], c["left"], c["right"]
    # Pieces of queries, each with the keys that it sees: the first tokens,
    # and the window's.
    piece = min(PIECE, nq)
    pieces = -(-nq // piece)
    i = torch.arange(pieces * piece, device="cuda").view(pieces, piece)
    p = nk - nq + i[:, :, None]
    near = (nk - nq - left + piece * torch.arange(pieces, device="cuda"))[:, None] + torch.arange(
        piece + left + right, device="cuda")
    first = torch.arange(min(c["sinks"], nk), device="cuda").expand(pieces, -1)
    inside = (near >= 0) & (near < nk)
    near = near.clamp(0, nk - 1)
    keep = torch.cat([(first[:, None] < p - left) & (first[:, None] <= p + right),
                      (near[:, None] >= p - left) & (near[:, None] <= p + right) & inside[:, None]], -1)
    keys = torch.cat([first, near], 1)
    if t["mask"] is not None:
        keep &= t["mask"][keys][:, None] != 0
    out = _attend(t["q"][i.clamp(max=nq - 1)], t["k"][keys], t["v"][keys], keep)
    return out.flatten(0, 1)[:nq]


def _kept(c, codes, scales, page, at):
    """Float32 keys or values at (page, place): (..., key heads, d)."""
    return codes[page, :, at][..., : c["d"]].float() * scales[page, :, at][..., None]


def _attend_kept(c, s):
    t, page, left = s["t"], c["page"], c["left"]
    new, kept = torch.tensor(s["new"], device="cuda")[:, None], torch.tensor(s["kept"], device="cuda")[:, None]
    most = c["new"]
    if left < 0:
        keys = torch.arange(c["most"], device="cuda").expand(c["seqs"], -1)
    else:
        near = kept - new - left + torch.arange(left + most, device="cuda")
        sinks = torch.arange(min(c["sinks"], c["most"]), device="cuda").expand(c["seqs"], -1)
        keys = torch.cat([sinks, near], 1)
        first = torch.arange(keys.shape[1], device="cuda") < sinks.shape[1]
    i = torch.arange(most, device="cuda")
    p = (kept - new + i)[:, :, None]
    inside = (keys >= 0) & (keys < kept)
    at = keys.clamp(0, c["most"] - 1)
    where = t["table"].gather(1, at // page).long()
    keep = (keys[:, None] <= p) & (inside & (where >= 0))[:, None]
    if left >= 0:
        keep &= torch.where(first, keys[:, None] < p - left, keys[:, None] >= p - left)
    where, at = where.clamp(min=0), at % page
    row = t["start"][:-1, None].long() + torch.minimum(i[None], new - 1)
    out = _attend(t["q"][row], _kept(c, t["kc"], t["ks"], where, at), _kept(c, t["vc"], t["vs"], where, at), keep)
    return out[i[None] < new]


# ---- a pass: the library's calls ---------------------------------------------------


def _operand(s, name, off, ld):
    return _package().Opnd(s["m"].get(name), off, ld, 0, 0)


def _norm_own(c, s):
    w, m, t = c["c"], s["m"], s["t"]
    x, r, h, y = (_operand(s, n, 0, w) for n in ("x", "r", "h", "y"))
    s["api"].ops_rms_norm(s["po"], c["rows"], w, x, r, m["g"], EPS, h, y, m.get("q"), m.get("s"))
    return {k: t[k] for k in ("h", "y", "q", "s") if t[k] is not None}


def _cache_own(c, s):
    h, w = s["handles"], c["kv_heads"] * c["d"]
    a, t = s["api"], s["t"]
    a.ops_cache_write(s["po"], h["cache"], h["start"], s["rows"], _operand(s, "k", 0, w), _operand(s, "v", 0, w))
    a.ops_cache_read(s["po"], h["cache"], h["bstart"], len(t["bk"]), _operand(s, "bk", 0, w), _operand(s, "bv", 0, w))
    return {"k": t["bk"], "v": t["bv"]}


def _window_own(c, s):
    h, kv, d, nq, nk = (c[n] for n in ("heads", "kv_heads", "d", "nq", "nk"))
    q, k, v, o = (_operand(s, n, 0, w * d) for n, w in (("q", h), ("k", kv), ("v", kv), ("out", h)))
    s["api"].ops_attention_window(s["po"], q, k, v, o, nq, nk, h, kv, d, nk - nq, c["left"], c["right"], c["sinks"],
                                  d ** -0.5, s["m"].get("mask"), s["m"]["work"])
    return s["t"]["out"]


def _attend_own(c, s):
    h, d, hd = c["heads"], c["d"], s["handles"]
    s["api"].ops_attention_cache(s["po"], hd["cache"], hd["start"], s["rows"], _operand(s, "q", 0, h * d),
                                 _operand(s, "out", 0, h * d), h, c["left"], c["sinks"], d ** -0.5, s["m"]["work"])
    return s["t"]["out"]


def run(state):
    c, t = state["case"], state["t"]
    if own:
        return {"norm": _norm_own, "cache": _cache_own, "window": _window_own, "attend": _attend_own}[c["kind"]](c, state)
    if c["kind"] == "norm":
        return _norm(c, t)
    if c["kind"] == "window":
        return _window(c, t)
    return (_cache if c["kind"] == "cache" else _attend_kept)(c, state)


# ---- what a pass cannot do without -------------------------------------------------


def _seen(p, nk, left, right, sinks):
    """Positions that queries at positions p see (left, right < 0: no limit)."""
    hi = np.minimum(p + right, nk - 1) if right >= 0 else np.full_like(p, nk - 1)
    lo = np.maximum(p - left, 0) if left >= 0 else np.zeros_like(p)
    return np.maximum(hi - lo + 1, 0) + np.minimum(np.minimum(lo, sinks), np.maximum(hi + 1, 0))


def work(case):
    c = case
    if c["kind"] == "norm":
        n = c["rows"] * c["c"]
        return {"bytes": n * (4 + (8 if c["residual"] else 0) + {"float": 4, "q8": 1, "both": 5}[c["out"]]) + 4 * c["c"] +
                (0 if c["out"] == "float" else 4 * c["rows"]), "flops": 5 * n}
    if c["kind"] == "window":
        p = np.arange(c["nk"] - c["nq"], c["nk"])
        pairs = int(_seen(p, c["nk"], c["left"], c["right"], c["sinks"]).sum()) * c["heads"]
        lo = max(0, c["nk"] - c["nq"] - c["left"])
        keys = c["nk"] - lo + min(lo, c["sinks"])
        return {"bytes": 8 * c["d"] * (c["nq"] * c["heads"] + keys * c["kv_heads"]) + (keys if c["masked"] else 0),
                "flops": 4 * c["d"] * pairs}
    kept, new = _lengths(c)
    row = 2 * c["kv_heads"] * (c["d"] + 4)
    if c["kind"] == "cache":
        wide = 8 * c["kv_heads"] * c["d"]
        return {"bytes": (sum(new) + sum(_back(c))) * (row + wide), "flops": 4 * sum(new) * c["kv_heads"] * c["d"]}
    pairs = keys = 0
    for k, n in zip(kept, new):
        pairs += int(_seen(np.arange(k - n, k), k, c["left"], 0, c["sinks"]).sum())
        lo = max(0, k - n - c["left"]) if c["left"] >= 0 else 0
        keys += k - lo + min(lo, c["sinks"])
    return {"bytes": 8 * sum(new) * c["heads"] * c["d"] + keys * row, "flops": 4 * c["d"] * pairs * c["heads"]}


# ---- the same from the definitions, in 64 bits ---------------------------------------


def _exact_codes(x):
    """The codes as the definition rounds them: the quotient 127 / a and its
    product with x to float32 (both single roundings of a 64-bit result)."""
    x = x.double()
    a = x.abs().amax(-1, keepdim=True)
    r = torch.where(a < TINY, 0.0, (127 / a.clamp(min=TINY)).float().double())
    return (x * r).float().double().round(), torch.where(a < TINY, 0.0, (a / 127).float().double())


def _exact_rows(q, k, v, keep):
    """q (n, d), k, v (keys, d), keep (n, keys), all of one head."""
    s = (q @ k.T) * q.shape[1] ** -0.5
    s[~keep] = -math.inf
    s -= s.amax(1, keepdim=True).clamp(min=-1e300)
    p = s.exp_()
    return (p @ v) / p.sum(1, keepdim=True).clamp(min=1e-300)


def _exact_seen(p, j, c, right):
    inside = (j <= p + right) if right >= 0 else torch.ones_like(j <= p)
    return inside & ((j >= p - c["left"]) | (j < c["sinks"])) if c["left"] >= 0 else inside


def exact(case, seed):
    c, s = case, prepare(case, seed)
    t = s["t"]
    if c["kind"] == "norm":
        h = t["x"].double() if t["r"] is None else t["x"].double() + t["r"].double()
        y = h * torch.rsqrt((h * h).sum(-1, keepdim=True) / c["c"] + EPS) * t["g"].double()
        return {k: {"h": h, "y": y, "q": None, "s": y.abs().amax(-1) / 127}[k] for k in ("h", "y", "q", "s")
                if t[k] is not None}
    if c["kind"] == "window":
        nq, nk, g = c["nq"], c["nk"], c["heads"] // c["kv_heads"]
        p, j = torch.arange(nk - nq, nk, device="cuda")[:, None], torch.arange(nk, device="cuda")[None]
        keep = _exact_seen(p, j, c, c["right"])
        if t["mask"] is not None:
            keep = keep & (t["mask"] != 0)
        return torch.stack([_exact_rows(t["q"][:, i].double(), t["k"][:, i // g].double(), t["v"][:, i // g].double(), keep)
                            for i in range(c["heads"])], 1)
    page, seen = c["page"], {"k": [], "v": []}
    if c["kind"] == "cache":
        at = 0
        for b, (k, n, m) in enumerate(zip(s["kept"], s["new"], s["back"])):
            rows = t["table"][b].long()
            for x, codes, scales in (("k", "kc", "ks"), ("v", "vc", "vs")):
                old = torch.arange(k - m, k - n, device="cuda")
                old = t[codes][rows[old // page], :, old % page][..., : c["d"]].double() * t[scales][
                    rows[old // page], :, old % page][..., None].double()
                code, scale = _exact_codes(t[x][at:at + n])
                seen[x].append(torch.cat([old, code * scale]))
            at += n
        return {x: torch.cat(seen[x]) for x in ("k", "v")}
    out, at, g = [], 0, c["heads"] // c["kv_heads"]
    for b, (k, n) in enumerate(zip(s["kept"], s["new"])):
        j = torch.arange(k, device="cuda")
        row = t["table"][b].long()[j // page]
        keep = _exact_seen(j[k - n:, None], j[None], c, 0)
        j, row, keep = j[row >= 0] % page, row[row >= 0], keep[:, row >= 0]
        key, val = (t[codes][row, :, j][..., : c["d"]].double() * t[scales][row, :, j][..., None].double()
                    for codes, scales in (("kc", "ks"), ("vc", "vs")))
        out.append(torch.stack([_exact_rows(t["q"][at:at + n, i].double(), key[:, i // g], val[:, i // g], keep)
                                for i in range(c["heads"])], 1))
        at += n
    return torch.cat(out)
