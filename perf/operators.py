# SPDX-License-Identifier: Unlicense
"""Operators of a transformer layer for large tiles and long sequences, as
measurable cases: products in 8-bit integers, rotary positions computed from
coordinates, attention over selected blocks of keys.

A case is a dict of plain values with a "kind":

linear  y = act(x W^T + b) (+ y): tokens quantised to 8 bits on the way, a
        scale per token, weights kept in 8 bits with a scale per channel
rope    queries and keys out of packed projection rows, rotated by their
        tokens' coordinates
sparse  the index of the key blocks, each query's selection, the attention
        over the selected blocks; with "refresh" the index is kept and only
        its last block is made again, as after a token was appended

`run` computes a case with elementary torch operations, or, with `own`, by
the library's entry points. Tensors live in torch memory; the library gets
views of it and queues its work on a stream of its own, which torch's streams
and events know nothing of: what `run` returns then is valid, and a state may
be written by torch or dropped, only after torch.cuda.synchronize().
"""

import importlib.util
import math
import sys
from pathlib import Path

import numpy as np
import torch

ROOT = Path(__file__).resolve().parent.parent
own = False

ACT_NONE, ACT_GELU, ACT_RELU = 0, 1, 2
# The smallest row maximum that keeps its codes; rows below it count as zero.
TINY = 2.0 ** -100
KINDS = {"plain": 0, "linear": 1, "base": 2, "parts": 3}
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
        # One token through a ViT-L MLP's first layer: the weights' bytes.
        {"name": "linear_token", "kind": "linear", "rows": 1, "cin": 1024, "cout": 4096, "act": ACT_GELU,
         "bias": True, "residual": False},
        # ELoFTR's projections on the 20 x 20 tokens of a 640 x 640 tile.
        {"name": "linear_agg_400", "kind": "linear", "rows": 400, "cin": 256, "cout": 256, "act": ACT_NONE,
         "bias": False, "residual": False},
        # A ViT-L/14's MLP on the tokens of a 560 x 560 pair: first layer,
        # and second with the residual.
        {"name": "linear_vit_fc1", "kind": "linear", "rows": 3202, "cin": 1024, "cout": 4096, "act": ACT_GELU,
         "bias": True, "residual": False},
        {"name": "linear_vit_fc2", "kind": "linear", "rows": 3202, "cin": 4096, "cout": 1024, "act": ACT_NONE,
         "bias": True, "residual": True},
        # A long batch of tokens through a square layer.
        {"name": "linear_long", "kind": "linear", "rows": 12805, "cin": 4096, "cout": 4096, "act": ACT_NONE,
         "bias": True, "residual": False},
        # One token far behind the trained length: latency.
        {"name": "rope_token", "kind": "rope", "rows": 1, "heads": 16, "kv_heads": 4, "d": 128, "rot": 128,
         "axes": 1, "interleaved": False, "inverse": False, "scaling": "parts", "factor": 8.0, "start": 131071},
        # ELoFTR's 2-D encoding on the coarse grid of a 640 x 640 tile.
        {"name": "rope_grid_80", "kind": "rope", "rows": 6400, "heads": 8, "kv_heads": 8, "d": 32, "rot": 32,
         "axes": 2, "interleaved": True, "inverse": False, "scaling": "linear", "factor": 2.0, "start": 1},
        # A long sequence, half of each head rotated, on the way back.
        {"name": "rope_long_back", "kind": "rope", "rows": 65533, "heads": 16, "kv_heads": 4, "d": 128, "rot": 64,
         "axes": 1, "interleaved": False, "inverse": True, "scaling": "parts", "factor": 16.0, "start": 1000003},
        # One token over a long cache, the index kept beside it.
        {"name": "sparse_token", "kind": "sparse", "nq": 1, "nk": 131005, "heads": 16, "kv_heads": 4, "d": 128,
         "block": 64, "top": 16, "masked": False, "refresh": True},
        # A ViT-L/14's attention on a 560 x 560 image.
        {"name": "sparse_vit_1601", "kind": "sparse", "nq": 1601, "nk": 1601, "heads": 16, "kv_heads": 16, "d": 64,
         "block": 32, "top": 8, "masked": False, "refresh": False},
        # The coarse cells of a 640 x 640 pair, one image's against the
        # other's, part of it without data.
        {"name": "sparse_cross_6400", "kind": "sparse", "nq": 6400, "nk": 6400, "heads": 8, "kv_heads": 8, "d": 32,
         "block": 64, "top": 8, "masked": True, "refresh": False},
        # A long sequence with shared key heads.
        {"name": "sparse_long", "kind": "sparse", "nq": 8192, "nk": 16380, "heads": 8, "kv_heads": 2, "d": 64,
         "block": 64, "top": 16, "masked": False, "refresh": False},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    kind = rng.choice(["linear", "rope", "sparse"])
    if kind == "linear":
        width = lambda: rng.choice([256, 512, 1024, 2048, 4096]) if rng.random() < 0.5 else _log(rng, 64, 4096)  # noqa: E731
        return {"kind": kind, "rows": _log(rng, 1, 12805), "cin": width(), "cout": width(),
                "act": rng.choice([ACT_NONE, ACT_GELU, ACT_RELU]), "bias": rng.random() < 0.7,
                "residual": rng.random() < 0.3}
    if kind == "rope":
        axes, kv = rng.choice([1, 1, 2]), rng.choice([1, 2, 4, 8])
        d = 4 * rng.randint(4, 32)
        return {"kind": kind, "rows": _log(rng, 1, 65533), "heads": kv * rng.choice([1, 2]), "kv_heads": kv, "d": d,
                "rot": d if rng.random() < 0.5 else 4 * rng.randint(1, d // 4), "axes": axes,
                "interleaved": rng.random() < 0.5, "inverse": rng.random() < 0.3,
                "scaling": rng.choice(sorted(KINDS)), "factor": rng.choice([2.0, 4.0, 8.0, 32.0]),
                "start": _log(rng, 1, 1000003)}
    kv, d = rng.choice([1, 2, 4, 8]), rng.choice([16, 32, 48, 64, 100, 128])
    heads = kv * rng.choice([1, 1, 2, 4]) if kv <= 2 else 8
    nq = 1 if rng.random() < 0.25 else _log(rng, 2, 8192)
    # A decoding step has a long cache; a long batch of queries a shorter one.
    nk = _log(rng, 64, 131005) if nq == 1 else _log(rng, 64, 16380)
    block = rng.choice([16, 32, 64, 128])
    top = rng.randint(1, 16)
    if nq > 1024:
        block, top, d = min(block, 64), min(top, 8) if d > 64 else top, d
    return {"kind": kind, "nq": nq, "nk": nk, "heads": heads, "kv_heads": kv, "d": d, "block": block, "top": top,
            "masked": rng.random() < 0.4, "refresh": nq == 1}


# ---- the definitions that inputs, plain form and library share -----------------


def _pitch(c):
    """Bytes of a row of c codes."""
    return -(-c // 64) * 64


def _freqs(c):
    """Radians per position of each pair, in 64 bits: the trained
    frequencies b^(-2 k / n), n = rot / axes channels of a coordinate, k the
    pair's place among them, stretched by `factor` all alike, by another
    base, or only those that turn less than 1 .. 32 times over the trained
    4096 positions."""
    n, base, f = c["rot"] // c["axes"], 10000.0, c["factor"]
    k = (np.arange(c["rot"] // 2) // c["axes"]).astype(np.float64)
    if c["scaling"] == "base":
        base *= f ** (n / (n - 2)) if n > 2 else f
    w = base ** (-2 * k / n)
    if c["scaling"] == "linear":
        return w / f
    if c["scaling"] == "parts":
        g = np.clip((4096 * w / (2 * math.pi) - 1) / (32 - 1), 0, 1)
        return w * (g + (1 - g) / f)
    return w


def _mult(c):
    return float(np.float32(0.1 * math.log(c["factor"]) + 1)) if c["scaling"] == "parts" else 1.0


# ---- inputs --------------------------------------------------------------------


def _views(t):
    """The library's views of the state's tensors."""
    lib = _package().lib()
    return {k: lib.ocl_wrap(v.data_ptr(), v.numel() * v.element_size()) for k, v in t.items() if v is not None}


def prepare(case, seed):
    c, dev, lib = case, _device(), _package().lib()
    g = torch.Generator("cuda").manual_seed(int(seed))
    randn = lambda *s, std=1.0: std * torch.randn(s, generator=g, device="cuda")  # noqa: E731
    empty = lambda *s, dtype=torch.float32: torch.empty(s, dtype=dtype, device="cuda")  # noqa: E731
    if c["kind"] == "linear":
        # Tokens after a norm, a few channels of which are large, as they are
        # in trained transformers; weights that keep the scale, quantised.
        x = randn(c["rows"], c["cin"])
        x[:, :: max(1, c["cin"] // 5)] *= 4
        wc, ws = _codes(randn(c["cout"], c["cin"], std=c["cin"] ** -0.5))
        t = {"x": x, "wc": wc, "ws": ws, "b": randn(c["cout"], std=0.05) if c["bias"] else None,
             "y0": randn(c["rows"], c["cout"]) if c["residual"] else None, "y": empty(c["rows"], c["cout"])}
        if hasattr(lib, "ops_linear_q8_work_bytes"):
            t["work"] = empty(lib.ops_linear_q8_work_bytes(c["rows"], c["cin"]), dtype=torch.uint8)
    elif c["kind"] == "rope":
        n, d = c["rows"], c["d"]
        i = torch.arange(n, device="cuda", dtype=torch.int64)
        if c["axes"] == 1:
            pos = i[:, None] + c["start"]
        else:
            w = max(1, math.isqrt(n))
            pos = torch.stack([i // w, i % w], 1) + c["start"]
        t = {"x": randn(n, (c["heads"] + 2 * c["kv_heads"]) * d), "pos": pos.int(),
             "freq": torch.from_numpy(_freqs(c)).cuda(), "q": empty(n, c["heads"] * d),
             "k": empty(n, c["kv_heads"] * d)}
    else:
        nk, kv, d = c["nk"], c["kv_heads"], c["d"]
        blocks = -(-nk // c["block"])
        # Neighbouring keys are alike, as neighbouring image tokens are.
        near = randn(blocks, kv, d).repeat_interleave(c["block"], 0)[:nk]
        t = {"q": randn(c["nq"], c["heads"], d, std=1.4), "k": (near + randn(nk, kv, d)).contiguous(),
             "v": randn(nk, kv, d), "mask": None, "kc": empty(blocks, kv, _pitch(d), dtype=torch.int8),
             "ks": empty(blocks, kv), "sel": empty(c["nq"], c["heads"], c["top"], dtype=torch.int32),
             "out": empty(c["nq"], c["heads"], d)}
        if c["masked"]:
            # Stretches without data, as at the border of a mosaic.
            t["mask"] = (randn(-(-nk // 40)).repeat_interleave(40)[:nk] > -0.7).to(torch.uint8)
        if c["refresh"]:
            kc, ks = _index(c, t, 0, blocks)
            t["kc"].copy_(kc)
            t["ks"].copy_(ks)
        if hasattr(lib, "ops_attention_blocks_work_bytes"):
            n = max(lib.ops_block_select_work_bytes(c["nq"], c["heads"], blocks, c["top"]),
                    lib.ops_attention_blocks_work_bytes(c["nq"], nk, c["heads"], kv, d, c["block"], c["top"]))
            t["work"] = empty(n, dtype=torch.uint8)
    s = {"case": c, "t": t, "m": _views(t), "api": dev.api, "po": dev.po}
    torch.cuda.synchronize()
    return s


# ---- a pass: the plain form ------------------------------------------------------


def _codes(x):
    """8-bit codes (rows padded with zeros to the pitch) and scales of the
    rows of x: scale a / 127 of the row's largest magnitude a, code the
    float32 product x (127 / a) to the nearest integer, ties to even."""
    a = x.abs().amax(-1)
    live = a >= TINY
    # Quotients in 64 bits, so that their rounding to 32 is the nearest one.
    r = torch.where(live, (127.0 / torch.where(live, a, 1.0).double()).float(), 0.0)
    q = torch.zeros(x.shape[:-1] + (_pitch(x.shape[-1]),), dtype=torch.int8, device=x.device)
    q[..., : x.shape[-1]] = (x * r[..., None]).round_().to(torch.int8)
    return q, torch.where(live, (a.double() / 127.0).float(), 0.0)


def _act(y, act):
    if act == ACT_GELU:
        return 0.5 * y * (1 + torch.erf(y * 0.70710678118654752))
    return y.relu() if act == ACT_RELU else y


def _linear(c, t):
    xc, xs = _codes(t["x"])
    y = (xc.float() @ t["wc"].float().T) * (xs[:, None] * t["ws"])
    if t["b"] is not None:
        y = y + t["b"]
    y = _act(y, c["act"])
    return y if t["y0"] is None else y + t["y0"]


def _turn(c, x, cos, sin):
    """x (rows, heads, d) with the first rot channels rotated."""
    rot, m = c["rot"], _mult(c)
    part = x[..., :rot]
    a, b = (part[..., 0::2], part[..., 1::2]) if c["interleaved"] else (part[..., : rot // 2], part[..., rot // 2:])
    u, v = m * (a * cos - b * sin), m * (a * sin + b * cos)
    y = x.clone()
    y[..., :rot] = torch.stack([u, v], -1).flatten(-2) if c["interleaved"] else torch.cat([u, v], -1)
    return y


def _rope(c, t):
    n, h, kv, d = c["rows"], c["heads"], c["kv_heads"], c["d"]
    axis = torch.arange(c["rot"] // 2, device="cuda") % c["axes"]
    angle = t["pos"].double()[:, axis] * t["freq"]
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    if c["inverse"]:
        sin = -sin
    x = t["x"].view(n, h + 2 * kv, d)
    return {"q": _turn(c, x[:, :h], cos, sin).flatten(1), "k": _turn(c, x[:, h:h + kv], cos, sin).flatten(1)}


def _index(c, t, first, last):
    """Codes and scales of the key blocks first .. last - 1: the means of
    their kept keys; scale -1 where no key is kept."""
    bs, kv, d = c["block"], c["kv_heads"], c["d"]
    k = t["k"][first * bs:last * bs]
    keep = torch.ones(len(k), dtype=torch.uint8, device="cuda") if t["mask"] is None else t["mask"][first * bs:last * bs]
    short = (last - first) * bs - len(k)
    k = torch.cat([k, k.new_zeros(short, kv, d)]).view(-1, bs, kv, d).double()
    keep = torch.cat([keep, keep.new_zeros(short)]).view(-1, bs).double()
    count = keep.sum(1)
    mean = ((k * keep[:, :, None, None]).sum(1) / count.clamp(min=1)[:, None, None]).float()
    kc, ks = _codes(mean)
    return kc, torch.where(count[:, None] > 0, ks, -1.0)


def _select(c, q, kc, ks):
    """Each query and head's best blocks, best first, -1 where there are no
    more: the scale times the whole-number product of the codes, ties to
    the lower block."""
    nq, h, kv, d = c["nq"], c["heads"], c["kv_heads"], c["d"]
    qc = _codes(q)[0][..., :d].float().view(nq, kv, h // kv, d)
    s = torch.matmul(qc.permute(1, 2, 0, 3).reshape(kv, -1, d), kc[..., :d].float().permute(1, 2, 0).contiguous())
    s = s.view(h, nq, -1) * ks.T.repeat_interleave(h // kv, 0)[:, None]
    live = (ks >= 0).T.repeat_interleave(h // kv, 0)[:, None]
    s, at = torch.where(live, s, -math.inf).sort(dim=-1, descending=True, stable=True)
    sel = torch.full((nq, h, c["top"]), -1, dtype=torch.int32, device="cuda")
    n = min(c["top"], s.shape[-1])
    sel[..., :n] = torch.where(s[..., :n] > -math.inf, at[..., :n], -1).transpose(0, 1).int()
    return sel


def _softmax_rows(s, v):
    """softmax(s) v over the last axis of s; zeros where s is all -inf."""
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top > -math.inf, top, 0.0))
    total = p.sum(-1, keepdim=True)
    return torch.matmul(p, v) / torch.where(total > 0, total, 1.0)


def _attend(c, t, sel):
    nq, nk, h, kv, d, bs = c["nq"], c["nk"], c["heads"], c["kv_heads"], c["d"], c["block"]
    blocks = -(-nk // bs)
    q = t["q"].transpose(0, 1) * d ** -0.5
    if nq * c["top"] * bs <= nk:
        # Few queries: the selected keys are gathered.
        key = sel.transpose(0, 1).long()[..., None] * bs + torch.arange(bs, device="cuda")
        keep = ((key >= 0) & (key < nk)).flatten(2)
        key = key.clamp(0, nk - 1).flatten(2)
        head = (torch.arange(h, device="cuda") // (h // kv))[:, None, None]
        if t["mask"] is not None:
            keep &= t["mask"][key] != 0
        s = torch.matmul(t["k"][key, head], q[..., None])[..., 0].masked_fill(~keep, -math.inf)
        return _softmax_rows(s[:, :, None], t["v"][key, head])[:, :, 0].transpose(0, 1)
    # Many: every score, and those of other blocks left out.
    k, v = (t[n].permute(1, 0, 2).repeat_interleave(h // kv, 0) for n in ("k", "v"))
    chosen = torch.zeros(h, nq, blocks + 1, dtype=torch.bool, device="cuda")
    at = sel.transpose(0, 1).long()
    chosen.scatter_(2, torch.where(at < 0, blocks, at), True)
    keep = chosen[..., :blocks].repeat_interleave(bs, -1)[..., :nk]
    if t["mask"] is not None:
        keep = keep & (t["mask"] != 0)
    s = torch.matmul(q, k.transpose(1, 2).contiguous()).masked_fill_(~keep, -math.inf)
    return _softmax_rows(s, v).transpose(0, 1)


def _sparse(c, t):
    blocks = -(-c["nk"] // c["block"])
    first = blocks - 1 if c["refresh"] else 0
    kc, ks = _index(c, t, first, blocks)
    t["kc"][first:], t["ks"][first:] = kc, ks
    sel = _select(c, t["q"], t["kc"], t["ks"])
    return {"ks": t["ks"], "sel": sel, "out": _attend(c, t, sel)}


# ---- a pass: the library's calls ---------------------------------------------------


def _linear_own(c, s):
    a, m, t = s["api"], s["m"], s["t"]
    a.ops_linear_q8(s["po"], c["rows"], c["cin"], c["cout"], m["x"], 0, c["cin"], m["wc"], m["ws"], m.get("b"),
                    m.get("y0"), 0, m["y"], 0, c["cout"], c["act"], 0.0, m["work"])
    return t["y"]


def _rope_own(c, s):
    ic, m, t = _package(), s["m"], s["t"]
    d, row = c["d"], (c["heads"] + 2 * c["kv_heads"]) * c["d"]
    flags = (1 if c["interleaved"] else 0) | (2 if c["inverse"] else 0)
    s["api"].ops_rope_pos(s["po"], c["rows"], d, c["rot"], c["axes"], m["pos"], m["freq"], _mult(c), flags,
                          ic.Opnd(m["x"], 0, row, 0, 0), ic.Opnd(m["q"], 0, c["heads"] * d, 0, 0), c["heads"],
                          ic.Opnd(m["x"], c["heads"] * d, row, 0, 0), ic.Opnd(m["k"], 0, c["kv_heads"] * d, 0, 0),
                          c["kv_heads"])
    return {"q": t["q"], "k": t["k"]}


def _sparse_own(c, s):
    ic, a, po, m, t = _package(), s["api"], s["po"], s["m"], s["t"]
    nq, nk, h, kv, d, bs, top = (c[n] for n in ("nq", "nk", "heads", "kv_heads", "d", "block", "top"))
    blocks = -(-nk // bs)
    first = blocks - 1 if c["refresh"] else 0
    q, k, v, o = (ic.Opnd(m[n], 0, w * d, 0, 0) for n, w in (("q", h), ("k", kv), ("v", kv), ("out", h)))
    a.ops_block_index(po, k, nk, kv, d, bs, m.get("mask"), first, blocks - first, m["kc"], m["ks"])
    a.ops_block_select(po, q, nq, h, kv, d, m["kc"], m["ks"], blocks, top, m["sel"], m["work"])
    a.ops_attention_blocks(po, q, k, v, o, nq, nk, h, kv, d, bs, top, m["sel"], d ** -0.5, m.get("mask"), m["work"])
    return {"ks": t["ks"], "sel": t["sel"], "out": t["out"]}


def run(state):
    c = state["case"]
    if own:
        return {"linear": _linear_own, "rope": _rope_own, "sparse": _sparse_own}[c["kind"]](c, state)
    return {"linear": _linear, "rope": _rope, "sparse": _sparse}[c["kind"]](c, state["t"])


# ---- what a pass cannot do without -------------------------------------------------


def work(case):
    c = case
    if c["kind"] == "linear":
        n, k, m = c["rows"], c["cin"], c["cout"]
        return {"bytes": 4 * n * k + m * k + 4 * m + 4 * n * m * (2 if c["residual"] else 1) + (4 * m if c["bias"] else 0),
                "flops": 2 * n * k * m}
    if c["kind"] == "rope":
        n = c["rows"] * (c["heads"] + c["kv_heads"]) * c["d"]
        return {"bytes": 8 * n + 4 * c["rows"] * c["axes"], "flops": 3 * n * c["rot"] // c["d"]}
    nq, nk, h, kv, d = (c[n] for n in ("nq", "nk", "heads", "kv_heads", "d"))
    blocks = -(-nk // c["block"])
    keys = min(nk, c["top"] * c["block"])
    # Keys and values are read once, or only the selected where those are
    # fewer; the index reads what it makes.
    seen = min(nk * kv, keys * nq * h)
    made = c["block"] if c["refresh"] else nk
    read = max(seen, made * kv) + seen
    return {"bytes": 4 * d * (2 * nq * h + read) + blocks * kv * (d + 4) + 4 * nq * h * c["top"],
            "flops": 4 * nq * h * keys * d + 2 * nq * h * blocks * d}


# ---- the same from the definitions, in 64 bits ---------------------------------------


def _exact_codes(x):
    """The codes as the definition rounds them: the quotient 127 / a and its
    product with x to float32 (both single roundings of a 64-bit result)."""
    x = x.double()
    a = x.abs().amax(-1, keepdim=True)
    r = torch.where(a < TINY, 0.0, (127 / a.clamp(min=TINY)).float().double())
    return (x * r).float().double().round(), torch.where(a < TINY, 0.0, (a / 127).float().double())[..., 0]


def exact(case, seed):
    c, t = case, prepare(case, seed)["t"]
    if c["kind"] == "linear":
        xc, xs = _exact_codes(t["x"])
        y = xc @ t["wc"][:, : c["cin"]].double().T
        y *= xs[:, None]
        y *= t["ws"].double()
        if c["bias"]:
            y += t["b"].double()
        if c["act"] == ACT_GELU:
            y = y * torch.special.ndtr(y)
        elif c["act"] == ACT_RELU:
            y = y.clamp(min=0)
        return y + t["y0"].double() if c["residual"] else y
    if c["kind"] == "rope":
        h, kv, d, rot = c["heads"], c["kv_heads"], c["d"], c["rot"]
        f = torch.from_numpy(_freqs(c)).cuda()
        a = torch.stack([t["pos"][:, p % c["axes"]].double() * f[p] for p in range(rot // 2)], 1)[:, None]
        turn = torch.polar(torch.full_like(a, _mult(c)), -a if c["inverse"] else a)
        out, at = {}, 0
        for name, n in (("q", h), ("k", kv)):
            x = t["x"][:, at * d:(at + n) * d].double().view(-1, n, d)
            at += n
            first = torch.arange(rot // 2, device="cuda") * (2 if c["interleaved"] else 1)
            second = first + (1 if c["interleaved"] else rot // 2)
            z = torch.complex(x[..., first], x[..., second]) * turn
            y = x.clone()
            y[..., first], y[..., second] = z.real, z.imag
            out[name] = y.flatten(1)
        return out
    nq, nk, h, kv, d, bs, top = (c[n] for n in ("nq", "nk", "heads", "kv_heads", "d", "block", "top"))
    blocks, g = -(-nk // bs), h // kv
    keep = torch.ones(nk, dtype=torch.bool, device="cuda") if t["mask"] is None else t["mask"] != 0
    owner = torch.arange(nk, device="cuda") // bs
    count = torch.zeros(blocks, dtype=torch.float64, device="cuda").index_add_(0, owner, keep.double())
    out = torch.zeros(nq, h, d, dtype=torch.float64, device="cuda")
    scales = torch.empty(blocks, kv, dtype=torch.float64, device="cuda")
    for j in range(kv):
        k, v = t["k"][:, j].double(), t["v"][:, j].double()
        total = torch.zeros(blocks, d, dtype=torch.float64, device="cuda").index_add_(0, owner, k * keep[:, None])
        code, scale = _exact_codes((total / count.clamp(min=1)[:, None]).float())
        scales[:, j] = torch.where(count > 0, scale, -1)
        for i in range(j * g, (j + 1) * g):
            q = t["q"][:, i]
            score = ((_exact_codes(q)[0] @ code.T) * scale).float()
            score[:, count == 0] = -math.inf
            at = torch.argsort(score, dim=1, descending=True, stable=True)[:, :top]
            member = torch.zeros(nq, blocks, dtype=torch.bool, device="cuda").scatter_(1, at, True) & (count > 0)
            s = (q.double() @ k.T) * d ** -0.5
            s[~(member[:, owner] & keep)] = -math.inf
            s -= s.amax(1, keepdim=True).clamp(min=-1e300)
            p = s.exp_()
            out[:, i] = (p @ v) / p.sum(1, keepdim=True).clamp(min=1e-300)
    return {"ks": scales, "sel": None, "out": out}
