"""What the operators around packed documents are measured on: the mask built from a batch's document ids, rotary positions given per
token, attention under that mask with capped scores or a distance bias, and the norms between two blocks.

One GPU.  Widths and head counts are those of ``yafsdp_b200.models.llama.CONFIGS``, lengths those of the framework's benchmarks and
tests.  ``run`` takes one pass of one operator, forward or forward and backward, either in its plain form (elementary torch operations
in 32 bits, angles in 64) or, with ``own``, through ``yafsdp_b200.ops.functional``.  Kinds:

* ``mask``       document ids of a packed batch to key ranges, query ranges and positions (whole numbers);
* ``rotary``     queries and keys turned by per-token positions of one or three axes;
* ``attention``  head_dim 128, grouped heads, causal inside documents, with prefixes, windows, padding, a tanh cap and a linear bias;
* ``norm``       norm after a block, gate, residual scale, residual add and the norm before the next block.
"""

from __future__ import annotations

import math
import random
from typing import Any

import numpy as np
import torch

own = False

HEAD_DIM = 128
HEADS = ((4, 2), (32, 32), (40, 40), (32, 8), (64, 8))  # query and key/value heads of the model configurations
WIDTHS = (512, 4096, 5120, 8192)
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed() -> list[dict[str, Any]]:
    return [
        # the masks of a small fine-tuning batch, padded rows
        _mask("mask 3x333 padded", batch=3, seq=333, docs=80, padding=True),
        # the masks of long packed pre-training rows whose documents start with a prefix that is seen from both sides
        _mask("mask 4x32768 prefix", batch=4, seq=32768, docs=700, prefix=True),
        # the prompt of one chat turn, forward only: bound by latency
        _rotary("rotary 1x45", batch=1, seq=45, heads=(32, 32), axes=1, dtype="bf16", backward=False),
        # a training batch of images and text: time, height and width of every token
        _rotary("rotary 2x4096 three axes", batch=2, seq=4096, heads=(64, 8), axes=3, dtype="bf16", backward=True),
        # supervised fine-tuning on short packed conversations, rows padded at the end
        _attention("attention 3x333 packed", batch=3, seq=333, heads=(40, 40), docs=80, padding=True, backward=True),
        # the headline pre-training length, packed documents, grouped heads
        _attention("attention 1x2048 packed capped", batch=1, seq=2048, heads=(32, 8), docs=400, softcap=50.0, backward=True),
        # long packed pre-training rows
        _attention("attention 1x8192 packed", batch=1, seq=8192, heads=(32, 8), docs=1200, backward=True),
        # a whole long document whose scores are capped
        _attention("attention 1x8192 capped", batch=1, seq=8192, heads=(32, 32), softcap=30.0, backward=True),
        # scoring answers to long prompts: prompt seen from both sides, linear distance bias, no gradient
        _attention("attention 2x4096 prefix bias", batch=2, seq=4096, heads=(64, 8), docs=2500, prefix=True, slopes=True, backward=False),
        # the residual step of one chat turn's prompt: bound by latency
        _norm("norm 45x4096", tokens=45, samples=1, width=4096, gate="none", post=False, dtype="bf16", backward=False),
        # ragged fine-tuning batch whose block is gated per sample, residual stream in 32 bits
        _norm("norm 3x333x5120 fp32", tokens=999, samples=3, width=5120, gate="sample", post=True, dtype="fp32", backward=True),
        # the widest model's residual step in pre-training: norms on both sides of the block and a gate per channel
        _norm("norm 8192x8192", tokens=8192, samples=4, width=8192, gate="channel", post=True, dtype="bf16", backward=True),
    ]


def _mask(name: str, *, batch: int, seq: int, docs: int, prefix: bool = False, window: int = 0, padding: bool = False) -> dict[str, Any]:
    return {"name": name, "kind": "mask", "batch": batch, "seq": seq, "docs": docs, "prefix": prefix, "window": window, "padding": padding}


def _rotary(name: str, *, batch: int, seq: int, heads: tuple[int, int], axes: int, dtype: str, backward: bool) -> dict[str, Any]:
    return {"name": name, "kind": "rotary", "batch": batch, "seq": seq, "q_heads": heads[0], "kv_heads": heads[1], "axes": axes, "dtype": dtype,
            "backward": backward}


def _attention(name: str, *, batch: int, seq: int, heads: tuple[int, int], docs: int = 0, prefix: bool = False, window: int = 0,
               padding: bool = False, softcap: float = 0.0, slopes: bool = False, backward: bool) -> dict[str, Any]:
    """``docs``: mean length of a document, 0 for one causal sequence per row."""
    return {"name": name, "kind": "attention", "batch": batch, "seq": seq, "q_heads": heads[0], "kv_heads": heads[1], "docs": docs,
            "prefix": prefix, "window": window, "padding": padding, "softcap": softcap, "slopes": slopes, "backward": backward}


def _norm(name: str, *, tokens: int, samples: int, width: int, gate: str, post: bool, dtype: str, backward: bool) -> dict[str, Any]:
    return {"name": name, "kind": "norm", "tokens": tokens, "samples": samples, "width": width, "gate": gate, "post": post, "dtype": dtype,
            "backward": backward}


def _log_int(rng: Any, lo: int, hi: int) -> int:
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _cost(case: dict[str, Any]) -> float:
    w = work(case)
    full = 0.0
    if case["kind"] == "attention":  # the plain form multiplies whole rows of keys
        full = 4.0 * case["batch"] * case["q_heads"] * case["seq"] ** 2 * HEAD_DIM * (2.5 if case["backward"] else 1.0) / 200.0
    return max(w["bytes"], w["flops"] / 200.0, full)


def draw(rng: Any) -> dict[str, Any]:
    while True:
        kind = rng.choice(("mask", "rotary", "attention", "attention", "attention", "norm", "norm"))
        batch = rng.choice((1, 1, 2, 3, 4, 8))
        if kind == "mask":
            seq = max(1, _log_int(rng, 1, 131072) // batch)
            case = _mask("", batch=batch, seq=seq, docs=_log_int(rng, 1, max(2, seq)), prefix=rng.random() < 0.4,
                         window=rng.choice((0, 0, _log_int(rng, 1, max(2, seq)))), padding=rng.random() < 0.4)
        elif kind == "rotary":
            case = _rotary("", batch=batch, seq=max(1, _log_int(rng, 1, 8192) // batch), heads=rng.choice(HEADS), axes=rng.choice((1, 3)),
                           dtype=rng.choice(("bf16", "bf16", "fp16", "fp32")), backward=rng.random() < 0.5)
        elif kind == "attention":
            seq = max(1, _log_int(rng, 1, 8192) // batch)
            packed = rng.random() < 0.7
            case = _attention("", batch=batch, seq=seq, heads=rng.choice(HEADS), docs=_log_int(rng, 1, max(2, seq)) if packed else 0,
                              prefix=packed and rng.random() < 0.3, window=_log_int(rng, 1, max(2, seq)) if packed and rng.random() < 0.3 else 0,
                              padding=packed and rng.random() < 0.4, softcap=rng.choice((0.0, 0.0, 30.0, 50.0)), slopes=rng.random() < 0.3,
                              backward=rng.random() < 0.7)
        else:
            samples = batch
            case = _norm("", tokens=samples * max(1, _log_int(rng, 1, 8192) // samples), samples=samples,
                         width=rng.choice((*WIDTHS, 8 * _log_int(rng, 8, 1024))), gate=rng.choice(("none", "channel", "sample", "token")),
                         post=rng.random() < 0.6, dtype=rng.choice(("bf16", "bf16", "fp16", "fp32")), backward=rng.random() < 0.6)
        case.pop("name")
        if _cost(case) <= max(_cost(c) for c in listed()):
            return case


# ----------------------------------------------------------------------------------------- documents
def _documents(case: dict[str, Any]) -> list[list[tuple[int, int]]]:
    """(length, prefix) of every document of every row: a property of the case, so that its work is; their order is the seed's."""
    rng = random.Random(f"{case['batch']} {case['seq']} {case['docs']}")
    rows = []
    for _ in range(case["batch"]):
        left = case["seq"] - (rng.randrange(case["seq"] // 2 + 1) if case["padding"] else 0)
        row = []
        while left > 0:
            n = min(left, max(1, int(round(rng.expovariate(1.0 / case["docs"])))))
            row.append((n, int(n * rng.random() * 0.6)))
            left -= n
        rows.append(row)
    return rows


def _layout(case: dict[str, Any], seed: int) -> tuple[torch.Tensor, torch.Tensor | None, list[list[tuple[int, int, int]]]]:
    """Document ids [B, S] (negative: padding), prefix flags or None, and every row's (start, end, prefix) of its documents."""
    rng = random.Random(seed)
    ids = np.full((case["batch"], case["seq"]), -1, dtype=np.int64)
    flags = np.zeros((case["batch"], case["seq"]), dtype=bool)
    where: list[list[tuple[int, int, int]]] = []
    for b, row in enumerate(_documents(case)):
        rng.shuffle(row)
        at, places, base = 0, [], rng.randrange(1000)
        for d, (n, p) in enumerate(row):
            ids[b, at : at + n] = base + d
            if case["prefix"]:
                flags[b, at : at + p] = True
            places.append((at, at + n, p if case["prefix"] else 0))
            at += n
        where.append(places)
    return torch.from_numpy(ids), torch.from_numpy(flags) if case["prefix"] else None, where


def _pairs(case: dict[str, Any]) -> int:
    """Query-key pairs that see each other, over all rows."""
    s, w = case["seq"], case["window"]
    if not case["docs"]:
        return int(case["batch"] * s * (s + 1) // 2)
    total = 0
    for row in _documents(case):
        for n, p in row:
            i = np.arange(n, dtype=np.int64)
            hi = np.maximum(i + 1, p if case["prefix"] else 0)
            total += int((hi - (np.maximum(i - w + 1, 0) if w else 0)).sum())
    return total


def work(case: dict[str, Any]) -> dict[str, float]:
    if case["kind"] == "mask":  # ids of 8 bytes and flags of one in; two ranges and a position out
        tokens = case["batch"] * case["seq"]
        return {"bytes": tokens * (8 + case["prefix"] + 20), "flops": 0}
    size = DTYPES[case["dtype"]].itemsize if "dtype" in case else 2
    if case["kind"] == "rotary":
        tokens, heads = case["batch"] * case["seq"], case["q_heads"] + case["kv_heads"]
        turned = tokens * heads * HEAD_DIM
        once = 2 * turned * size
        times = 2 if case["backward"] else 1
        return {"bytes": times * once + tokens * case["axes"] * 8, "flops": times * turned * 3}
    if case["kind"] == "attention":
        tokens = case["batch"] * case["seq"]
        q, kv = tokens * case["q_heads"] * HEAD_DIM * 2, tokens * case["kv_heads"] * HEAD_DIM * 2
        forward = 2 * q + 2 * kv
        backward = 2 * q + 2 * kv  # dO in, dQ, dK and dV out
        products = 4 + (10 if case["backward"] else 0)
        return {"bytes": forward + (backward if case["backward"] else 0) + (tokens * 16 if case["docs"] else 0),
                "flops": products * HEAD_DIM * case["q_heads"] * _pairs(case)}
    x = case["tokens"] * case["width"] * size
    rows = {"none": 0, "channel": 1, "sample": case["samples"], "token": case["tokens"]}[case["gate"]]
    small = (rows + 1 + case["post"]) * case["width"] * size
    flops = case["tokens"] * case["width"] * (10 + (20 if case["backward"] else 0))
    return {"bytes": (4 + (4 if case["backward"] else 0)) * x + small * (2 if case["backward"] else 1), "flops": flops}


# ----------------------------------------------------------------------------------------- preparation
def prepare(case: dict[str, Any], seed: int) -> dict[str, Any]:
    dev = torch.device("cuda", 0)
    gen = torch.Generator(device=dev).manual_seed(seed)
    state: dict[str, Any] = {"case": case}
    if case["kind"] == "mask":
        ids, flags, _ = _layout(case, seed)
        state.update(ids=ids.to(dev), prefix=None if flags is None else flags.to(dev))
        return state
    if case["kind"] == "norm":
        shape = (case["samples"], case["tokens"] // case["samples"], case["width"])
        dtype = DTYPES[case["dtype"]]

        def tensor(*size: int, scale: float = 1.0, offset: float = 0.0) -> torch.Tensor:
            return (torch.randn(*size, device=dev, generator=gen) * scale + offset).to(dtype).requires_grad_(case["backward"])

        gate = {"none": None, "channel": (case["width"],), "sample": (shape[0], 1, case["width"]), "token": shape}[case["gate"]]
        state.update(x=tensor(*shape, scale=2.0), y=tensor(*shape, scale=0.5), weight=tensor(case["width"], scale=0.1, offset=1.0),
                     post=tensor(case["width"], scale=0.1, offset=1.0) if case["post"] else None,
                     gate=None if gate is None else tensor(*gate, scale=0.3, offset=0.5), scale=0.7,
                     dh=tensor(*shape, scale=0.01).detach(), dn=tensor(*shape, scale=0.01).detach())
        return state
    b, s, hq, hk = case["batch"], case["seq"], case["q_heads"], case["kv_heads"]
    dtype = DTYPES[case["dtype"]] if case["kind"] == "rotary" else torch.bfloat16
    qkv = torch.randn(b, s, hq + 2 * hk, HEAD_DIM, device=dev, generator=gen)
    qkv[:, :, :hq] *= 2.0  # scores with a deviation of two
    q, k, v = (t.requires_grad_(case["backward"]) for t in qkv.to(dtype).detach().split((hq, hk, hk), dim=2))  # of one fused projection
    state.update(q=q, k=k)
    if case["kind"] == "rotary":
        state["dq"], state["dk"] = ((torch.randn(b, s, h, HEAD_DIM, device=dev, generator=gen) * 0.01).to(dtype) for h in (hq, hk))
        state["theta"] = 500000.0
        state["sections"] = (HEAD_DIM // 2,) if case["axes"] == 1 else (16, 24, 24)
        start = torch.randint(0, 100000, (case["axes"], b, 1), device=dev, generator=gen)
        if case["axes"] == 1:
            state["positions"] = start[0] + torch.arange(s, device=dev)
        else:  # rows of image patches: time, height, width
            state["positions"] = start + torch.stack([torch.arange(s, device=dev) // n % m for n, m in ((1024, 1 << 30), (32, 32), (1, 32))])[:, None]
        if own:
            from yafsdp_b200.ops import functional as Fn

            state["axes"] = Fn.RotaryAxes(HEAD_DIM, state["theta"], state["sections"])
        return state
    state["v"] = v
    state["dout"] = (torch.randn(b, s, hq, HEAD_DIM, device=dev, generator=gen) * 0.01).to(dtype)
    state["slopes"] = torch.tensor([2.0 ** (-8.0 * (h + 1) / hq) for h in range(hq)], device=dev) if case["slopes"] else None
    state["mask"] = None
    if case["docs"]:
        ids, flags, _ = _layout(case, seed)
        state["ids"], state["prefix"] = ids.to(dev), None if flags is None else flags.to(dev)
        if own:  # one mask serves all layers of a step
            from yafsdp_b200.ops import functional as Fn

            state["mask"] = Fn.document_mask(state["ids"], state["prefix"], case["window"])
        else:
            state["mask"] = _plain_mask(state["ids"], state["prefix"], case["window"])
    return state


# ----------------------------------------------------------------------------------------- plain forms
def _plain_mask(ids: torch.Tensor, prefix: torch.Tensor | None, window: int) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    s = ids.shape[1]
    at = torch.arange(s, device=ids.device).expand_as(ids)
    new = torch.ones_like(ids, dtype=torch.bool)
    new[:, 1:] = ids[:, 1:] != ids[:, :-1]
    start = torch.where(new, at, 0).cummax(1).values
    last = torch.ones_like(new)
    last[:, :-1] = new[:, 1:]
    end = torch.where(last, at + 1, s).flip(1).cummin(1).values.flip(1)
    lead, run_end = torch.zeros_like(new), end
    if prefix is not None:
        lead = prefix & (torch.where(prefix, -1, at).cummax(1).values < start)
        run_end = torch.minimum(end, torch.where(prefix, s, at).flip(1).cummin(1).values.flip(1))
    lo, hi = start, torch.where(lead, run_end, at + 1)
    first, stop = torch.where(lead, start, at), end
    if window:
        lo, stop = torch.maximum(lo, at - window + 1), torch.minimum(stop, at + window)
    pad = ids < 0
    lo, hi, first, stop = (torch.where(pad, at, t) for t in (lo, hi, first, stop))
    spans, key_spans = torch.stack([lo, hi], -1).int(), torch.stack([first, stop], -1).int()
    return spans, key_spans, torch.where(pad, 0, at - start).int()


def _plain_rotary(state: dict[str, Any]) -> list[torch.Tensor]:
    half = HEAD_DIM // 2
    freq = state["theta"] ** (torch.arange(half, device="cuda", dtype=torch.float64) * -2.0 / HEAD_DIM)
    positions = state["positions"] if state["positions"].dim() == 3 else state["positions"][None]
    axis = torch.repeat_interleave(torch.arange(len(state["sections"]), device="cuda"), torch.tensor(state["sections"], device="cuda"))
    angle = positions.permute(1, 2, 0).double()[..., axis] * freq  # [B, S, half]
    cos, sin = angle.cos().float()[:, :, None], angle.sin().float()[:, :, None]

    def turn(t: torch.Tensor, sign: float) -> torch.Tensor:
        a, b = t.float()[..., :half], t.float()[..., half:]
        return torch.cat([a * cos - b * sin * sign, b * cos + a * sin * sign], -1).to(t.dtype)

    out = [turn(state["q"].detach(), 1.0), turn(state["k"].detach(), 1.0)]
    if state["case"]["backward"]:
        out += [turn(state["dq"], -1.0), turn(state["dk"], -1.0)]
    return out


def _plain_attention(state: dict[str, Any]) -> list[torch.Tensor]:
    case, q, k, v, dout = state["case"], state["q"].detach(), state["k"].detach(), state["v"].detach(), state["dout"]
    b, s, hq, hk = case["batch"], case["seq"], case["q_heads"], case["kv_heads"]
    group, scale, cap = hq // hk, 1.0 / math.sqrt(HEAD_DIM), case["softcap"]
    at = torch.arange(s, device=q.device)
    out = torch.empty(b, s, hq, HEAD_DIM, device=q.device, dtype=q.dtype)
    dq, dk, dv = torch.empty_like(out), torch.empty(k.shape, device=q.device, dtype=q.dtype), torch.empty(v.shape, device=q.device, dtype=q.dtype)
    for i in range(b):
        if state["mask"] is None:
            hidden = at[None, :] > at[:, None]
        else:
            lo, hi = state["mask"][0][i, :, :1], state["mask"][0][i, :, 1:]
            hidden = (at[None, :] < lo) | (at[None, :] >= hi)
        far = (at[:, None] - at[None, :]).abs().float()
        for j in range(hk):
            heads = slice(j * group, (j + 1) * group)
            qf, kf, vf = q[i, :, heads].float().transpose(0, 1), k[i, :, j].float(), v[i, :, j].float()
            score = (qf @ kf.T) * scale
            if cap:
                t = torch.tanh(score / cap)
                score = cap * t
            if state["slopes"] is not None:
                score = score - state["slopes"][heads, None, None] * far
            score = score.masked_fill(hidden, -math.inf)
            top = score.amax(-1, keepdim=True)
            p = torch.exp(score - torch.where(top == -math.inf, 0.0, top))
            total = p.sum(-1, keepdim=True)
            p = p / torch.where(total == 0, 1.0, total)
            o = p @ vf
            out[i, :, heads] = o.transpose(0, 1).to(q.dtype)
            if case["backward"]:
                g = dout[i, :, heads].float().transpose(0, 1)
                dv[i, :, j] = (p.transpose(1, 2) @ g).sum(0).to(q.dtype)
                ds = p * (g @ vf.T - (g * o).sum(-1, keepdim=True))
                if cap:
                    ds = ds * (1.0 - t * t)
                dq[i, :, heads] = ((ds @ kf) * scale).transpose(0, 1).to(q.dtype)
                dk[i, :, j] = ((ds.transpose(1, 2) @ qf) * scale).sum(0).to(q.dtype)
    return [out, dq, dk, dv] if case["backward"] else [out]


def _plain_norm(state: dict[str, Any]) -> list[torch.Tensor | None]:
    x, y, w = (state[n].detach().float() for n in ("x", "y", "weight"))
    post, gate = (None if state[n] is None else state[n].detach().float() for n in ("post", "gate"))
    eps, scale, dtype = 1e-5, state["scale"], state["x"].dtype
    u, yhat, ry = y, None, None
    if post is not None:
        ry = torch.rsqrt((y * y).mean(-1, keepdim=True) + eps)
        yhat = y * ry
        u = yhat * post
    h = x + scale * (u if gate is None else gate * u)
    rh = torch.rsqrt((h * h).mean(-1, keepdim=True) + eps)
    hhat = h * rh
    out: list[torch.Tensor | None] = [h.to(dtype), (hhat * w).to(dtype)]
    if not state["case"]["backward"]:
        return out
    dh, dn = state["dh"].float(), state["dn"].float()
    dw = (dn * hhat).sum((0, 1))
    c = dn * w
    g = dh + rh * (c - hhat * (c * hhat).mean(-1, keepdim=True))
    e = scale * (g if gate is None else g * gate)
    dgate = None
    if gate is not None:
        dgate = scale * g * u
        if state["case"]["gate"] == "channel":
            dgate = dgate.sum((0, 1))
        elif state["case"]["gate"] == "sample":
            dgate = dgate.sum(1, keepdim=True)
    dpost, dy = None, e
    if post is not None:
        dpost = (e * yhat).sum((0, 1))
        c = e * post
        dy = ry * (c - yhat * (c * yhat).mean(-1, keepdim=True))
    return out + [None if t is None else t.to(dtype) for t in (g, dy, dw, dpost, dgate)]


# ----------------------------------------------------------------------------------------- one pass
def _own(state: dict[str, Any]) -> list[torch.Tensor | None]:
    from yafsdp_b200.ops import functional as Fn

    case = state["case"]
    if case["kind"] == "mask":
        mask = Fn.document_mask(state["ids"], state["prefix"], case["window"])
        return [mask.spans, mask.key_spans, mask.positions]
    if case["kind"] == "rotary":
        q, k = Fn.rotary(state["q"], state["k"], state["positions"], state["axes"])
        return [q, k] if not case["backward"] else [q.detach(), k.detach(), *torch.autograd.grad((q, k), (state["q"], state["k"]), (state["dq"], state["dk"]))]
    if case["kind"] == "attention":
        out = Fn.attention(state["q"], state["k"], state["v"], state["mask"], softcap=case["softcap"], slopes=state["slopes"])
        return [out] if not case["backward"] else [out.detach(), *torch.autograd.grad(out, (state["q"], state["k"], state["v"]), state["dout"])]
    h, n = Fn.residual_norm(state["x"], state["y"], state["weight"], post_weight=state["post"], gate=state["gate"], scale=state["scale"], eps=1e-5)
    if not case["backward"]:
        return [h, n]
    names = [t for t in ("x", "y", "weight", "post", "gate") if state[t] is not None]
    grads = dict(zip(names, torch.autograd.grad((h, n), [state[t] for t in names], (state["dh"], state["dn"]))))
    return [h.detach(), n.detach(), *(grads.get(t) for t in ("x", "y", "weight", "post", "gate"))]


def run(state: dict[str, Any]) -> list[torch.Tensor | None]:
    if own:
        return _own(state)
    kind = state["case"]["kind"]
    with torch.no_grad():
        if kind == "mask":
            return list(_plain_mask(state["ids"], state["prefix"], state["case"]["window"]))
        return {"rotary": _plain_rotary, "attention": _plain_attention, "norm": _plain_norm}[kind](state)


# ----------------------------------------------------------------------------------------- the definitions in 64 bits
def exact(case: dict[str, Any], seed: int) -> list[torch.Tensor | None] | None:
    global own
    before, own = own, False  # inputs alone: no plan of the framework
    try:
        state = prepare(case, seed)
    finally:
        own = before
    return {"mask": _exact_mask, "rotary": _exact_rotary, "attention": _exact_attention, "norm": _exact_norm}[case["kind"]](state, seed)


def _exact_mask(state: dict[str, Any], seed: int) -> list[torch.Tensor | None]:
    case = state["case"]
    b, s, w = case["batch"], case["seq"], case["window"] or case["seq"]
    at = np.broadcast_to(np.arange(s), (b, s))
    spans, key_spans, positions = np.stack([at, at], -1).copy(), np.stack([at, at], -1).copy(), np.zeros((b, s), dtype=np.int64)
    for i, places in enumerate(_layout(case, seed)[2]):
        for start, end, prefix in places:
            t = np.arange(start, end)
            ahead = t < start + prefix
            spans[i, start:end, 0] = np.maximum(start, t - w + 1)
            spans[i, start:end, 1] = np.where(ahead, start + prefix, t + 1)
            key_spans[i, start:end, 0] = np.where(ahead, start, t)
            key_spans[i, start:end, 1] = np.minimum(end, t + w)
            positions[i, start:end] = t - start
    return [torch.from_numpy(t).int().cuda() for t in (spans, key_spans, positions)]


def _exact_rotary(state: dict[str, Any], seed: int) -> list[torch.Tensor | None]:
    positions = state["positions"].reshape(-1, *state["positions"].shape[-2:]).double()
    parts, j = [], 0
    for axis, n in enumerate(state["sections"]):
        for _ in range(n):
            parts.append(positions[axis] * math.exp(-math.log(state["theta"]) * j / (HEAD_DIM // 2)))
            j += 1
    angle = torch.stack(parts, -1)[:, :, None]
    unit = torch.polar(torch.ones_like(angle), angle)

    def turn(t: torch.Tensor, by: torch.Tensor) -> torch.Tensor:
        pairs = t.detach().double().unflatten(-1, (2, HEAD_DIM // 2))
        z = torch.complex(pairs[..., 0, :].contiguous(), pairs[..., 1, :].contiguous()) * by
        return torch.cat([z.real, z.imag], -1)

    out: list[torch.Tensor | None] = [turn(state["q"], unit), turn(state["k"], unit)]
    return out + [turn(state["dq"], unit.conj()), turn(state["dk"], unit.conj())] if state["case"]["backward"] else out


def _exact_attention(state: dict[str, Any], seed: int) -> list[torch.Tensor | None] | None:
    """Document by document (a row without documents is one), a few heads at a time, gradients by differentiation."""
    case = state["case"]
    q, k, v, dout = (state[n].detach().double() for n in ("q", "k", "v", "dout"))
    group, cap, w = case["q_heads"] // case["kv_heads"], case["softcap"], case["window"] or case["seq"]
    out, dq, dk, dv = (torch.zeros_like(t) for t in (q, q, k, v))
    places = _layout(case, seed)[2] if case["docs"] else [[(0, case["seq"], 0)]] * case["batch"]
    if sum(len(row) for row in places) > 4000:
        return None  # a launch or more for each: too long
    for b, row in enumerate(places):
        for start, end, prefix in row:
            n = end - start
            t = torch.arange(n, device=q.device)
            delta = t[:, None] - t[None, :]
            seen = ((delta >= 0) | (t[None, :] < prefix) & (t[:, None] < prefix)) & (delta < w)
            step = max(1, min(case["q_heads"], (1 << 26) // (n * n)))
            for h0 in range(0, case["q_heads"], step):
                heads = torch.arange(h0, min(h0 + step, case["q_heads"]), device=q.device)
                qs = q[b, start:end, heads].transpose(0, 1).requires_grad_(case["backward"])
                ks, vs = (x[b, start:end, heads // group].transpose(0, 1).requires_grad_(case["backward"]) for x in (k, v))
                score = qs @ ks.transpose(1, 2) * HEAD_DIM**-0.5
                if cap:
                    score = torch.tanh(score / cap) * cap
                if state["slopes"] is not None:
                    score = score - state["slopes"][heads].double()[:, None, None] * delta.abs()
                o = torch.softmax(score.masked_fill(~seen, -math.inf), -1) @ vs
                out[b, start:end, heads] = o.detach().transpose(0, 1)
                if case["backward"]:
                    gq, gk, gv = torch.autograd.grad(o, (qs, ks, vs), dout[b, start:end, heads].transpose(0, 1))
                    dq[b, start:end, heads] = gq.transpose(0, 1)
                    dk[b, start:end].index_add_(1, heads // group, gk.transpose(0, 1))
                    dv[b, start:end].index_add_(1, heads // group, gv.transpose(0, 1))
    return [out, dq, dk, dv] if case["backward"] else [out]


def _exact_norm(state: dict[str, Any], seed: int) -> list[torch.Tensor | None]:
    names = [n for n in ("x", "y", "weight", "post", "gate") if state[n] is not None]
    t = {n: state[n].detach().double().requires_grad_(state["case"]["backward"]) for n in names}
    block = t["y"]
    if "post" in t:
        block = block / (block.pow(2).mean(-1, keepdim=True) + 1e-5).sqrt() * t["post"]
    if "gate" in t:
        block = block * t["gate"]
    h = t["x"] + state["scale"] * block
    n = h / (h.pow(2).mean(-1, keepdim=True) + 1e-5).sqrt() * t["weight"]
    out: list[torch.Tensor | None] = [h.detach(), n.detach()]
    if not state["case"]["backward"]:
        return out
    grads = dict(zip(names, torch.autograd.grad((h, n), [t[m] for m in names], (state["dh"].double(), state["dn"].double()))))
    return out + [grads.get(m) for m in ("x", "y", "weight", "post", "gate")]
