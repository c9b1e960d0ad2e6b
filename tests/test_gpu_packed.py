"""Kernels around packed documents (mask, rotary positions, attention, residual norm step) against their definitions in 64 bits."""

import math

import packed_oracle as oracle
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"


def _ids(b, s, mean, padding, seed=0):
    """Rows of documents of random lengths around ``mean``; with padding some documents are negative, the last one always."""
    gen = torch.Generator().manual_seed(seed)
    cut = torch.rand(b, s, generator=gen) < 1.0 / mean
    ids = cut.int().cumsum(1) + 3
    if padding:
        ids = torch.where((ids % 3 == 1) | (ids == ids[:, -1:]), -ids, ids)
    return ids


def _done():
    from yafsdp_b200.ops import kernels

    torch.cuda.synchronize()
    kernels.check_status()


# ----------------------------------------------------------------------------------------- mask
@pytest.mark.parametrize("b,s,mean", [(1, 1, 1), (3, 5, 2), (2, 127, 9), (1, 128, 128), (4, 129, 40), (2, 1024, 1), (2, 1025, 300), (1, 5000, 700), (3, 2049, 5000)])
@pytest.mark.parametrize("window", [0, 1, 37])
@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_document_mask(b, s, mean, window, dtype):
    from yafsdp_b200.ops import functional as Fn

    for padding, kind in ((False, None), (True, "random"), (True, "all")):
        ids = _ids(b, s, mean, padding).to(dtype)
        prefix = None if kind is None else torch.ones(b, s, dtype=torch.bool) if kind == "all" else torch.rand(b, s, generator=torch.Generator().manual_seed(1)) < 0.9
        want = Fn._document_mask_ref(ids, prefix, window)
        got = Fn.document_mask(ids.to(DEV), None if prefix is None else prefix.to(DEV), window)
        for name in ("spans", "key_spans", "positions", "padding"):
            assert torch.equal(getattr(got, name).cpu(), getattr(want, name)), name
    for w, o in zip((want.spans, want.key_spans, want.positions), oracle.spans_of(ids, prefix, window)):
        assert torch.equal(w, o)


def test_document_mask_strides_and_nothing():
    from yafsdp_b200.ops import functional as Fn

    ids = _ids(4, 300, 20, True).long()
    wide = torch.zeros(4, 700, dtype=torch.int64, device=DEV)
    for view in (wide[:, 100:400], wide[:, 0:600:2], wide.t()[:300].t()):
        view.copy_(ids)
        assert torch.equal(Fn.document_mask(view).spans.cpu(), Fn.document_mask(ids).spans)
    one = ids[:1].to(DEV).expand(3, 300)  # the same row three times
    assert torch.equal(Fn.document_mask(one, one % 2 == 0).spans.cpu(), Fn.document_mask(ids[:1], ids[:1] % 2 == 0).spans.expand(3, 300, 2))
    for shape in ((0, 5), (3, 0)):
        assert Fn.document_mask(torch.zeros(shape, dtype=torch.int64, device=DEV)).spans.shape == (*shape, 2)


# ----------------------------------------------------------------------------------------- rotary
@pytest.mark.parametrize("b,s,hq,hk,d,sections", [(1, 1, 1, 1, 128, (64,)), (2, 45, 4, 2, 128, (16, 24, 24)), (3, 7, 5, 1, 64, (32,)), (1, 300, 2, 2, 80, (10, 0, 30)),
                                                  (1, 3, 1, 3, 16, (3, 5)), (1, 9, 1, 1, 512, (256,))])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("pos", [torch.int32, torch.int64])
def test_rotary(b, s, hq, hk, d, sections, dtype, pos):
    from yafsdp_b200.ops import functional as Fn

    torch.manual_seed(0)
    axes = Fn.RotaryAxes(d, 500000.0, sections, interleaved=len(sections) == 2)
    qkv = torch.randn(b, s, hq + 2 * hk, d, device=DEV).to(dtype)
    q, k = (t.detach().requires_grad_() for t in (qkv[:, :, :hq], qkv[:, :, hq : hq + hk]))
    positions = torch.randint(-5, 1 << 20, (len(sections), b, s), device=DEV).to(pos)
    out = Fn.rotary(q, k, positions[0] if len(sections) == 1 else positions, axes)
    dout = [torch.randn_like(t) for t in out]
    grads = torch.autograd.grad(out, (q, k), dout)
    _done()
    angle = positions.double()[axes.axis].permute(1, 2, 0) * torch.tensor(axes.frequency, dtype=torch.float64, device=DEV)
    cos, sin = angle.cos()[:, :, None], angle.sin()[:, :, None]
    for sign, pairs in ((1.0, zip((q, k), out)), (-1.0, zip(dout, grads))):
        for x, got in pairs:
            a, z = x.detach().double().chunk(2, -1)
            want = torch.cat([a * cos - z * sin * sign, z * cos + a * sin * sign], -1)
            # cosines and sines to 2^-22 (the turn's fraction to 2^-25, sincospi to two units), two fp32 products and a sum
            off = oracle.HALF_STEP[dtype] * want.abs() + 2.0**-21 * (a.abs() + z.abs()).repeat(1, 1, 1, 2)
            oracle.close(got.detach(), (want, off))


def test_rotary_layouts_and_missing_gradients():
    from yafsdp_b200.ops import functional as Fn

    torch.manual_seed(0)
    axes = Fn.RotaryAxes(64, 1e4)
    q, k = torch.randn(2, 33, 4, 64, device=DEV).bfloat16(), torch.randn(2, 33, 2, 64, device=DEV).bfloat16()
    positions = torch.randint(0, 1000, (2, 33), device=DEV)
    want = Fn.rotary(q, k, positions, axes)
    by_head = q.transpose(1, 2).contiguous().transpose(1, 2)  # [B, H, S, D] in memory
    odd = torch.randn(2, 33, 2 * 64 + 1, device=DEV).bfloat16()[..., 1:].unflatten(-1, (2, 64)).copy_(k)  # rows at odd pitches and addresses
    for a, z in ((by_head, k), (q, odd)):
        for got, w in zip(Fn.rotary(a, z, positions, axes), want):
            assert torch.equal(got, w)
    shared = positions[:, :1].expand(2, 33)
    assert torch.equal(Fn.rotary(q, k, shared, axes)[0], Fn.rotary(q, k, shared.contiguous(), axes)[0])
    wide = k[:, :, :1].expand(2, 33, 5, 64).detach().requires_grad_()  # one head for all
    q.requires_grad_()
    out_q, out_k = Fn.rotary(q, wide, positions, axes)
    assert torch.autograd.grad(out_k.sum(), wide, retain_graph=True)[0].shape == wide.shape
    assert torch.autograd.grad(out_q.sum(), q)[0].shape == q.shape
    for shape in ((0, 3), (2, 0)):
        e = torch.empty(*shape, 4, 64, device=DEV).requires_grad_()
        out = Fn.rotary(e, e, torch.zeros(shape, device=DEV, dtype=torch.int64), axes)[0]
        assert out.shape == e.shape and torch.autograd.grad(out.sum(), e)[0].shape == e.shape


# ----------------------------------------------------------------------------------------- attention
def _seen(mask, b, s):
    at = torch.arange(s, device=DEV)
    if mask is None:
        return (at <= at[:, None]).expand(b, s, s)
    return (at >= mask.spans[..., :1]) & (at < mask.spans[..., 1:])


def _qkv(b, s, hq, hkv, spread=2.0, seed=0):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    qkv = torch.randn(b, s, hq + 2 * hkv, 128, device=DEV, generator=gen)
    qkv[:, :, :hq] *= spread
    return [t.requires_grad_() for t in qkv.bfloat16().split((hq, hkv, hkv), 2)]


def _check(b, s, hq, hkv, mask, softcap=0.0, slopes=None, spread=2.0, scale=None):
    from yafsdp_b200.ops import functional as Fn

    q, k, v = _qkv(b, s, hq, hkv, spread)
    out = Fn.attention(q, k, v, mask, softcap=softcap, slopes=slopes, scale=scale)
    dout = torch.randn(out.shape, device=DEV, generator=torch.Generator(device=DEV).manual_seed(1)).bfloat16()
    grads = torch.autograd.grad(out, (q, k, v), dout)
    with torch.no_grad():
        assert torch.equal(Fn.attention(q, k, v, mask, softcap=softcap, slopes=slopes, scale=scale), out)
    _done()
    want = oracle.attention(q.detach(), k.detach(), v.detach(), _seen(mask, b, s), 128**-0.5 if scale is None else scale, softcap, slopes, dout)
    for name, got, w in zip(("out", "dq", "dk", "dv"), (out, *grads), want):
        oracle.close(got.detach(), w, name)


@pytest.mark.parametrize("b,s,hq,hkv", [(1, 1, 1, 1), (2, 2, 4, 2), (3, 45, 2, 2), (1, 64, 8, 1), (2, 127, 2, 1), (1, 128, 2, 2), (2, 129, 4, 1), (1, 200, 6, 2), (1, 333, 40, 40),
                                        (2, 700, 8, 2), (1, 1100, 4, 4)])
@pytest.mark.parametrize("softcap,biased", [(0.0, False), (30.0, False), (0.0, True), (5.0, True)])
@pytest.mark.parametrize("packed", [False, True])
def test_attention(b, s, hq, hkv, softcap, biased, packed):
    from yafsdp_b200.ops import functional as Fn

    mask = Fn.document_mask(_ids(b, s, max(1, s // 4), False).to(DEV)) if packed else None
    slopes = torch.tensor([2.0 ** (-8.0 * (h + 1) / hq) for h in range(hq)], device=DEV) if biased else None
    _check(b, s, hq, hkv, mask, softcap, slopes)


@pytest.mark.parametrize("mean", [1, 30, 200, 10000])
@pytest.mark.parametrize("padding,prefix,window", [(True, False, 0), (False, True, 0), (True, True, 17), (True, True, 300), (False, False, 1)])
@pytest.mark.parametrize("softcap,biased", [(0.0, False), (20.0, True)])
def test_attention_masks(mean, padding, prefix, window, softcap, biased):
    from yafsdp_b200.ops import functional as Fn

    b, s, hq, hkv = 2, 600, 4, 2
    ids = _ids(b, s, mean, padding, seed=mean).to(DEV)
    flags = torch.rand(b, s, device=DEV, generator=torch.Generator(device=DEV).manual_seed(2)) < 0.97 if prefix else None
    _check(b, s, hq, hkv, Fn.document_mask(ids, flags, window), softcap, torch.rand(hq, device=DEV) if biased else None)


@pytest.mark.parametrize("softcap", [0.05, 1.0, 1000.0, 1e6])
def test_attention_caps(softcap):
    """Scores far beyond the cap, close to it, and a cap that does nothing."""
    _check(2, 260, 4, 2, None, softcap, spread=6.0)


@pytest.mark.parametrize("fill", [math.nan, math.inf, -math.inf, torch.finfo(torch.bfloat16).max])
@pytest.mark.parametrize("softcap,biased", [(0.0, False), (30.0, True)])
def test_attention_ignores_what_padding_holds(fill, softcap, biased):
    from yafsdp_b200.ops import functional as Fn

    b, s, hq, hkv = 2, 700, 4, 2
    ids = _ids(b, s, 90, True, seed=3)
    ids[0, 300:560] = -7  # whole tiles of padding
    ids[1, :140] = -1
    pad = (ids < 0).to(DEV)
    assert pad.any() and not pad.all()
    mask = Fn.document_mask(ids.to(DEV))
    slopes = torch.rand(hq, device=DEV) if biased else None
    results = []
    for value in (0.0, fill):
        q, k, v = (t.detach().clone().masked_fill(pad[..., None, None], value).requires_grad_() for t in _qkv(b, s, hq, hkv))
        dout = torch.randn(b, s, hq, 128, device=DEV, generator=torch.Generator(device=DEV).manual_seed(1)).bfloat16().masked_fill(pad[..., None, None], value)
        out = Fn.attention(q, k, v, mask, softcap=softcap, slopes=slopes)
        results.append([out.detach(), *torch.autograd.grad(out, (q, k, v), dout)])
    _done()
    for name, a, z in zip(("out", "dq", "dk", "dv"), *results):
        assert not torch.isnan(z).any() and not torch.isinf(z).any(), name
        assert (z.masked_select(pad[..., None, None]) == 0).all(), name
        if name == "dq":  # atomic sums: the order may move the last bit before the rounding
            assert torch.allclose(a.float(), z.float(), rtol=2.0**-7, atol=1e-5), name
        else:
            assert torch.equal(a, z), name


def test_attention_nothing_but_padding_and_nothing_at_all():
    from yafsdp_b200.ops import functional as Fn

    mask = Fn.document_mask(torch.full((2, 200), -1, device=DEV))
    q, k, v = _qkv(2, 200, 4, 2)
    out = Fn.attention(q, k, v, mask)
    assert all((t == 0).all() for t in (out, *torch.autograd.grad(out, (q, k, v), torch.ones_like(out))))
    for b, s in ((0, 5), (2, 0)):
        q, k, v = _qkv(b, s, 4, 2)
        out = Fn.attention(q, k, v, Fn.document_mask(torch.zeros(b, s, device=DEV, dtype=torch.int32)))
        assert out.shape == q.shape and [t.shape for t in torch.autograd.grad(out, (q, k, v), torch.ones_like(out))] == [q.shape, k.shape, v.shape]
    _done()


def test_attention_plain_against_the_causal_kernel():
    from yafsdp_b200.ops import functional as Fn
    from yafsdp_b200.ops import kernels

    q, k, v = _qkv(2, 300, 4, 2)
    want, _ = kernels.attn_fwd(*(t.detach().reshape(600, -1) for t in (q, k, v)), 2, 300, 4, 2, 128**-0.5)
    # they split a row's softmax at other keys: both are within o_off of the definition
    _, o_off = oracle.attention(q.detach(), k.detach(), v.detach(), _seen(None, 2, 300), 128**-0.5, 0.0, None)
    oracle.close(Fn.attention(q, k, v).detach(), (want.view(2, 300, 4, 128).double(), 2 * o_off))
    _check(2, 300, 4, 2, None)
    # one document per row is the causal form too
    _check(2, 300, 4, 2, Fn.document_mask(torch.zeros(2, 300, dtype=torch.int64, device=DEV)), scale=0.3)


def test_attention_layouts():
    from yafsdp_b200.ops import functional as Fn

    b, s, hq, hkv = 2, 150, 4, 2
    q, k, v = (t.detach() for t in _qkv(b, s, hq, hkv))
    mask = Fn.document_mask(_ids(b, s, 40, True).to(DEV))
    want = Fn.attention(q, k, v, mask, softcap=9.0)
    by_head = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v)]
    odd = torch.empty(b, s, hq * 128 + 3, device=DEV, dtype=torch.bfloat16)[..., 1 : 1 + hq * 128].unflatten(-1, (hq, 128)).copy_(q)
    padded = torch.empty(b, s + 9, hkv, 128, device=DEV, dtype=torch.bfloat16)[:, 4 : 4 + s].copy_(k)
    for args in (by_head, (odd, k, v), (q, padded, v), (q, k, v.contiguous())):
        assert torch.equal(Fn.attention(*args, mask, softcap=9.0), want)
    # one key head given to all query heads, one sequence to both rows: the gradients of what was broadcast
    k1, v1 = (torch.randn(1, s, 1, 128, device=DEV).bfloat16().requires_grad_() for _ in range(2))
    g = torch.randn_like(q)
    wide = torch.autograd.grad(Fn.attention(q, k1.expand(b, s, 1, 128), v1.expand(b, s, 1, 128), mask), (k1, v1), g)
    each = [torch.autograd.grad(Fn.attention(q[i : i + 1], k1, v1, Fn.document_mask(_ids(b, s, 40, True)[i : i + 1].to(DEV))), (k1, v1), g[i : i + 1]) for i in range(b)]
    for w, e0, e1 in zip(wide, *each):
        assert torch.allclose(w.float(), e0.float() + e1.float(), rtol=3 * 2.0**-8, atol=2.0**-8 * max(e0.abs().max().item(), e1.abs().max().item()))


@pytest.mark.parametrize("hq,hkv", [(8, 2), (8, 1)])
def test_attention_shared_key_tiles(hq, hkv):
    """Several CTAs for a key tile: the same dK and dV but for the order of the sums, also where a tile holds nothing but padding."""
    from yafsdp_b200.ops import functional as Fn
    from yafsdp_b200.ops import kernels

    b, s = 2, 400
    ids = _ids(b, s, 60, True)
    ids[0, 100:300] = -1
    m = Fn.document_mask(ids.to(DEV))
    q, k, v = (t.detach() for t in _qkv(b, s, hq, hkv))
    slopes = torch.rand(hq, device=DEV)
    for cap, sl in ((0.0, None), (9.0, None), (0.0, slopes), (9.0, slopes)):
        out, out_lo, lse = kernels.attn_fwd_mods(q, k, v, 0.1, cap, sl, m.spans, m.padding)
        dout, got = torch.randn_like(out), []
        for parts in [p for p in range(1, hq // hkv + 1) if (hq // hkv) % p == 0]:
            got.append(kernels.attn_bwd_mods(q, k, v, out, out_lo, dout, lse, 0.1, cap, sl, m.spans, m.key_spans, m.padding, head_parts=parts))
        _done()
        for g in got[1:]:
            for a, z in zip(g, got[0]):
                assert torch.allclose(a.float(), z.float(), rtol=2.0**-7, atol=1e-4)


def test_attention_repeats_and_streams():
    """The same bits from run to run (but dQ), on the default stream or another one, and two calls at once."""
    from yafsdp_b200.ops import functional as Fn

    b, s, hq, hkv = 2, 900, 8, 2
    mask = Fn.document_mask(_ids(b, s, 200, True).to(DEV))
    q, k, v = _qkv(b, s, hq, hkv)
    dout = torch.randn(b, s, hq, 128, device=DEV).bfloat16()

    def once():
        out = Fn.attention(q, k, v, mask, softcap=20.0)
        return out.detach(), *torch.autograd.grad(out, (q, k, v), dout)

    want = once()
    torch.cuda.synchronize()
    streams, results = [torch.cuda.Stream() for _ in range(2)], []
    for _ in range(3):
        for st in streams:
            with torch.cuda.stream(st):
                results.append(once())
    _done()
    for r in results:
        for i, (a, z) in enumerate(zip(r, want)):
            assert torch.allclose(a.float(), z.float(), rtol=2.0**-7, atol=1e-4) if i == 1 else torch.equal(a, z)


def test_attention_gradient_against_differences():
    from yafsdp_b200.ops import functional as Fn

    b, s, hq, hkv = 1, 140, 4, 2
    mask = Fn.document_mask(_ids(b, s, 50, True).to(DEV))
    slopes = torch.rand(hq, device=DEV)
    q, k, v = _qkv(b, s, hq, hkv)
    dout = torch.randn(b, s, hq, 128, device=DEV).bfloat16()
    out = Fn.attention(q, k, v, mask, softcap=3.0, slopes=slopes)
    grads = torch.autograd.grad(out, (q, k, v), dout)
    seen = _seen(mask, b, s)
    bounds = oracle.attention(q.detach(), k.detach(), v.detach(), seen, 128**-0.5, 3.0, slopes, dout)[1:]
    for i, (g, (_, off)) in enumerate(zip(grads, bounds)):
        way = torch.randn(g.shape, device=DEV, dtype=torch.float64)
        ends = []
        for sign in (1e-5, -1e-5):
            args = [t.detach().double() for t in (q, k, v)]
            args[i] = args[i] + sign * way
            ends.append((oracle.attention(*args, seen, 128**-0.5, 3.0, slopes)[0] * dout.double()).sum())
        assert abs((ends[0] - ends[1]).item() / 2e-5 - (g.double() * way).sum().item()) <= (off * way.abs()).sum().item() + 1e-4


# ----------------------------------------------------------------------------------------- residual norm
def _norm_case(shape, gate, post, dtype, seed=0):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    make = lambda *size, scale=1.0, offset=0.0: (torch.randn(*size, device=DEV, generator=gen) * scale + offset).to(dtype)  # noqa: E731
    b, s, d = shape
    g = {"none": None, "channel": (d,), "sample": (b, 1, d), "token": shape}[gate]
    return (make(*shape, scale=2.0), make(*shape), make(d, scale=0.1, offset=1.0), make(d, scale=0.1, offset=1.0) if post else None,
            None if g is None else make(*g, offset=0.5), make(*shape), make(*shape))


def _norm_check(x, y, w, post, gate, dh, dn, scale=0.7):
    from yafsdp_b200.ops import functional as Fn

    leaves = {n: t.requires_grad_() for n, t in (("dx", x), ("dy", y), ("dw", w), ("dpost", post), ("dgate", gate)) if t is not None}
    h, n = Fn.residual_norm(x, y, w, post_weight=post, gate=gate, scale=scale)
    grads = dict(zip(leaves, torch.autograd.grad((h, n), list(leaves.values()), (dh, dn))))
    _done()
    plain = [None if t is None else t.detach() for t in (x, y, w, post, gate)]
    want = oracle.residual_norm(*plain, scale, 1e-5, dh, dn)
    for name, got in {"h": h.detach(), "n": n.detach(), **grads}.items():
        oracle.close(got, want[name], name)


@pytest.mark.parametrize("shape", [(1, 1, 8), (2, 3, 64), (3, 111, 512), (2, 45, 1000), (1, 200, 1368), (4, 30, 4096), (3, 50, 5120), (2, 33, 8192), (1, 5, 8184)])
@pytest.mark.parametrize("gate", ["none", "channel", "sample", "token"])
@pytest.mark.parametrize("post", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_residual_norm(shape, gate, post, dtype):
    _norm_check(*_norm_case(shape, gate, post, dtype))


@pytest.mark.parametrize("shape,gate", [((300, 2, 64), "sample"), ((700, 1, 512), "sample"), ((150, 7, 2048), "sample"), ((1, 3000, 512), "channel"), ((1, 2500, 4096), "token")])
def test_residual_norm_many_rows(shape, gate):
    _norm_check(*_norm_case(shape, gate, True, torch.bfloat16))


def test_residual_norm_layouts_and_missing_gradients():
    from yafsdp_b200.ops import functional as Fn

    x, y, w, post, gate, dh, dn = _norm_case((2, 31, 512), "sample", True, torch.bfloat16)
    want = Fn.residual_norm(x, y, w, post_weight=post, gate=gate)
    wide = torch.empty(2, 31, 515, device=DEV, dtype=torch.bfloat16)[..., 1:513].copy_(x)
    turned = y.transpose(0, 1).contiguous().transpose(0, 1)
    odd_w = torch.empty(513, device=DEV, dtype=torch.bfloat16)[1:].copy_(w)
    for got, ref in zip(Fn.residual_norm(wide, turned, odd_w, post_weight=post, gate=gate), want):
        assert torch.equal(got, ref)
    # one gradient alone: the other one is zero
    leaves = [t.requires_grad_() for t in (x, y, w, post, gate)]
    for which in (0, 1):
        outs = Fn.residual_norm(*leaves[:3], post_weight=post, gate=gate)
        one = torch.autograd.grad(outs[which], leaves, (dh, dn)[which], allow_unused=True)
        outs = Fn.residual_norm(*leaves[:3], post_weight=post, gate=gate)
        both = torch.autograd.grad(outs, leaves, (dh, torch.zeros_like(dn)) if which == 0 else (torch.zeros_like(dh), dn))
        for a, z in zip(one, both):
            assert torch.equal(a, z)
    e = torch.empty(2, 0, 512, device=DEV, dtype=torch.bfloat16).requires_grad_()
    h, n = Fn.residual_norm(e, e, w, post_weight=post)
    g = torch.autograd.grad(h.sum() + n.sum(), (e, w, post))
    assert h.shape == e.shape and g[0].shape == e.shape and (g[1] == 0).all() and (g[2] == 0).all()
    # a gate that was broadcast by expand gets the sum of its rows' gradients
    small = gate.detach()[:1].requires_grad_()
    h, n = Fn.residual_norm(x, y, w, gate=small.expand(2, 1, 512))
    (got,) = torch.autograd.grad((h, n), small, (dh, dn))
    rows = gate.detach()[:1].expand(2, 1, 512).contiguous().requires_grad_()
    (each,) = torch.autograd.grad(Fn.residual_norm(x, y, w, gate=rows), rows, (dh, dn))
    assert torch.equal(got, each.sum(0, keepdim=True))


# ----------------------------------------------------------------------------------------- refusals, graphs, a whole layer
def test_refusals():
    from yafsdp_b200.ops import functional as Fn
    from yafsdp_b200.ops import kernels

    q, k, v = (t.detach() for t in _qkv(1, 4, 2, 1))
    with pytest.raises(TypeError):
        Fn.attention(q.half(), k.half(), v.half())
    with pytest.raises(TypeError):
        Fn.attention(q[..., :64], k[..., :64], v[..., :64])
    with pytest.raises(ValueError):
        Fn.attention(q, k, v, Fn.document_mask(torch.zeros(1, 4, dtype=torch.int64)))  # a mask on the CPU
    with pytest.raises(ValueError):
        Fn.rotary(q, k, torch.zeros(1, 4, dtype=torch.int64), Fn.RotaryAxes(128, 1e4))  # positions on the CPU
    with pytest.raises(ValueError):
        Fn.residual_norm(torch.ones(2, 12, device=DEV), torch.ones(2, 12, device=DEV), torch.ones(12, device=DEV))
    with pytest.raises(ValueError):
        Fn.residual_norm(*[torch.ones(2, 8200, device=DEV)] * 2, torch.ones(8200, device=DEV))
    with pytest.raises(ValueError):
        Fn.residual_norm(torch.ones(2, 16, device=DEV), torch.ones(2, 16), torch.ones(16, device=DEV))
    # the C entries refuse what the host can see
    with pytest.raises(RuntimeError):
        kernels.attn_fwd_mods(q, k, v, 0.1, -1.0, None, None, None)
    with pytest.raises(RuntimeError):
        kernels.attn_fwd_mods(q, k, v, 0.1, 0.0, None, torch.zeros(1, 4, 2, device=DEV, dtype=torch.int32), None)
    with pytest.raises(RuntimeError):
        kernels.attn_fwd_mods(q, k.expand(1, 4, 3, 128), v.expand(1, 4, 3, 128), 0.1, 0.0, None, None, None)
    with pytest.raises(RuntimeError):
        kernels.residual_norm_fwd(torch.ones(3, 8, device=DEV), torch.ones(3, 8, device=DEV), torch.ones(8, device=DEV), None, torch.ones(2, 8, device=DEV), 2, 1.0, 1e-5)


def test_captured_and_replayed():
    """A step of all four operators, forward and backward, in a graph: replays give what eager calls give on new inputs.  No eager
    graph of the same leaves may be alive during the capture: PyTorch then ties their gradients to the stream of that graph."""
    from yafsdp_b200.ops import functional as Fn

    b, s, hq, hkv = 2, 300, 4, 2
    axes = Fn.RotaryAxes(128, 1e4)
    ids = _ids(b, s, 60, True).to(DEV)
    q, k, v = (t.detach().clone().requires_grad_() for t in _qkv(b, s, hq, hkv))
    x, _, w, post, gate, dh, dn = _norm_case((b, s, hq * 128), "sample", True, torch.bfloat16)
    leaves = [t.requires_grad_() for t in (q, k, v, x, w, post, gate)]

    def step():
        mask = Fn.document_mask(ids)
        a = Fn.attention(*Fn.rotary(q, k, mask.positions, axes), v, mask, softcap=30.0)
        h, n = Fn.residual_norm(x, a.reshape(b, s, -1), w, post_weight=post, gate=gate)
        return [h.detach(), n.detach(), *torch.autograd.grad((h, n), leaves, (dh, dn))]

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for seed in (3, 4):
        with torch.no_grad():
            ids.copy_(_ids(b, s, 40 * seed, True, seed).to(DEV))
            for t, new in zip((q, k, v), _qkv(b, s, hq, hkv, seed=seed)):
                t.copy_(new)
            x.copy_(torch.randn_like(x))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in captured]
        for i, (a, z) in enumerate(zip(got, step())):
            assert torch.allclose(a.float(), z.float(), rtol=2.0**-7, atol=1e-4) if i == 2 else torch.equal(a, z), i
    _done()


def test_packed_layer_equals_its_documents_alone():
    """Mask, rotary positions, attention, projection and residual norm over a packed row, as a decoder layer uses them: every document's rows are
    those of the same layer on the document alone, and the parameters' gradients are the sums."""
    from yafsdp_b200.ops import functional as Fn

    torch.manual_seed(0)
    hq, hkv, d = 4, 2, 512
    lengths, s = (130, 1, 77, 300), 600
    axes = Fn.RotaryAxes(128, 1e4)
    w_qkv = (torch.randn((hq + 2 * hkv) * 128, d, device=DEV) * d**-0.5).bfloat16().requires_grad_()
    w_o = (torch.randn(d, hq * 128, device=DEV) * d**-0.5).bfloat16().requires_grad_()
    w, post, gate = ((1 + 0.1 * torch.randn(d, device=DEV)).bfloat16().requires_grad_() for _ in range(3))
    params = (w_qkv, w_o, w, post, gate)
    x, dh, dn = (torch.randn(1, s, d, device=DEV).bfloat16() for _ in range(3))

    qkv = torch.nn.functional.linear(x, w_qkv)  # once: a library product of other rows rounds elsewhere

    def layer(x, qkv, ids):
        mask = Fn.document_mask(ids)
        q, k, v = qkv.unflatten(-1, (hq + 2 * hkv, 128)).split((hq, hkv, hkv), 2)
        q, k = Fn.rotary(q, k, mask.positions, axes)
        y = torch.nn.functional.linear(Fn.attention(q, k, v, mask, softcap=50.0).flatten(2), w_o)
        return y, *Fn.residual_norm(x, y, w, post_weight=post, gate=gate), q, k, v

    ids = torch.full((1, s), -1, device=DEV)
    at, total = 0, [torch.zeros(p.shape, device=DEV) for p in params]
    places = []
    for i, n in enumerate(lengths):
        ids[0, at : at + n] = i
        places.append((at, at + n))
        at += n
    live = (ids >= 0)[..., None]
    dh, dn = dh * live, dn * live
    packed = layer(x, qkv, ids)
    grads = torch.autograd.grad(packed[1:3], params, (dh, dn), retain_graph=True)
    u = 2.0**-8
    for a, z in places:
        n = z - a
        y, h, normed, q, k, v = layer(x[:, a:z], qkv[:, a:z], torch.zeros(1, n, dtype=torch.int64, device=DEV))
        assert torch.equal(q, packed[3][:, a:z]) and torch.equal(k, packed[4][:, a:z])
        # The two attentions see the same numbers but split their rows' softmax at other keys: each is within o_off of the definition.  A
        # difference d goes through the projection as |w_o| d plus two roundings, through a norm as r d + |hat| mean(r |hat| d) to first
        # order (a tenth more for what is beyond it), and through the gate as it is.
        tri = torch.ones(1, n, n, dtype=torch.bool, device=DEV).tril()
        _, o_off = oracle.attention(q.detach(), k.detach(), v.detach(), tri, 128**-0.5, 50.0, None)
        d_y = 2 * o_off.flatten(2) @ w_o.detach().double().abs().T + 2.1 * u * y.detach().double().abs()

        def through_norm(t, d, weight):
            r = torch.rsqrt(t.pow(2).mean(-1, keepdim=True) + 1e-5)
            hat = t * r
            return 1.1 * (r * d + hat.abs() * (r * hat.abs() * d).mean(-1, keepdim=True)) * weight.detach().double().abs()

        h64 = h.detach().double()
        d_h = through_norm(y.detach().double(), d_y, post) * gate.detach().double().abs() + 2.1 * u * h64.abs()
        d_n = through_norm(h64, d_h, w) + 2.1 * u * normed.detach().double().abs()
        for got, want, off in ((packed[0], y, d_y), (packed[1], h, d_h), (packed[2], normed, d_n)):
            oracle.close(got[:, a:z].detach(), (want.detach().double(), off))
        for t, g in zip(total, torch.autograd.grad((h, normed), params, (dh[:, a:z], dn[:, a:z]), retain_graph=True)):
            t += g.float()
    _done()
    for g, t in zip(grads, total):
        assert ((g.float() - t).norm() / t.norm()).item() < 2.0**-6


# ----------------------------------------------------------------------------------------- more work than the GPU holds at once, places far apart
def _uneven_rows(s):
    """Rows of nothing but padding, with padding in front, in the middle, behind, of one document and of many."""
    ids = torch.zeros(6, s, dtype=torch.int64)
    ids[0] = -1
    ids[1, : s * 3 // 7] = -2
    ids[2, s // 5 : s * 4 // 7] = -1
    ids[3, s // 2 :] = -1
    ids[5] = _ids(1, s, 30, True)[0]
    return ids


@pytest.mark.parametrize("softcap,biased", [(0.0, False), (30.0, False), (30.0, True)])
def test_attention_of_more_tiles_than_fit(softcap, biased):
    """Blocks that go on with other heads and sequences, of other lengths and without any: what the sequences give alone, to the bit, and the
    definition."""
    from yafsdp_b200.ops import functional as Fn

    b, s, hq, hkv = 6, 700, 32, 8
    ids = _uneven_rows(s).to(DEV)
    mask = Fn.document_mask(ids)
    slopes = torch.tensor([2.0 ** (-8.0 * (h + 1) / hq) for h in range(hq)], device=DEV) if biased else None
    q, k, v = (t.detach() for t in _qkv(b, s, hq, hkv))
    out = Fn.attention(q, k, v, mask, softcap=softcap, slopes=slopes)
    for i in range(b):
        alone = Fn.attention(*(t[i : i + 1] for t in (q, k, v)), Fn.document_mask(ids[i : i + 1]), softcap=softcap, slopes=slopes)
        assert torch.equal(alone[0], out[i]), i
    _check(b, s, hq, hkv, mask, softcap, slopes)


def test_attention_rows_far_apart():
    """A projection's rows at a pitch that takes their offsets past 32 bits: what the same rows give side by side."""
    from yafsdp_b200.ops import functional as Fn
    from yafsdp_b200.ops import kernels

    s, pitch = 33000, 1 << 16
    wide = torch.empty(1, s, pitch, device=DEV, dtype=torch.bfloat16)
    near = _qkv(1, s, 2, 1)
    q, k, v = (wide[..., at : at + t.shape[2] * 128].unflatten(-1, (-1, 128)) for t, at in zip(near, (65024, 128, 4096)))
    for far, t in zip((q, k, v), near):
        far.copy_(t.detach())
    mask = Fn.document_mask(_ids(1, s, 900, True).to(DEV))
    dout = torch.randn(1, s, 2, 128, device=DEV).bfloat16()
    results = []
    for args in ((q, k, v), [t.detach().contiguous() for t in near]):
        out, low, lse = kernels.attn_fwd_mods(*args, 0.1, 0.0, None, mask.spans, mask.padding)
        results.append((out, low, lse, *kernels.attn_bwd_mods(*args, out, low, dout, lse, 0.1, 0.0, None, mask.spans, mask.key_spans, mask.padding)[1:]))
    _done()
    assert all(torch.equal(a, z) for a, z in zip(*results))


def test_rotary_and_residual_norm_past_32_bits():
    """The last tokens of tensors of more than 2^31 elements: what they give alone."""
    from yafsdp_b200.ops import functional as Fn

    t, d = 263000, 8192
    x, y, dh, dn = (torch.empty(t, d, device=DEV, dtype=torch.bfloat16) for _ in range(4))
    for big in (x, y, dh, dn):
        big[:-5].zero_()
        big[-5:] = torch.randn(5, d, device=DEV).bfloat16()
    w = torch.ones(d, device=DEV, dtype=torch.bfloat16)
    ends = []
    for cut in (slice(None), slice(-5, None)):
        leaves = [z[cut].requires_grad_() for z in (x, y)]
        h, n = Fn.residual_norm(*leaves, w)
        grads = torch.autograd.grad((h, n), leaves, (dh[cut], dn[cut]))
        ends.append([z[-5:].clone() for z in (h.detach(), n.detach(), *grads)])
        del h, n, grads
    assert all(torch.equal(a, z) for a, z in zip(*ends))
    axes = Fn.RotaryAxes(128, 1e4)
    positions = torch.arange(t, device=DEV)[None]
    q = x.detach().view(1, t, 64, 128)
    far = Fn.rotary(q, q[:, :, :1], positions, axes)[0][:, -5:].clone()
    assert torch.equal(far, Fn.rotary(q[:, -5:], q[:, -5:, :1], positions[:, -5:], axes)[0])
    _done()


def test_residual_norm_in_a_sharded_module():
    """Weights of a sharded module, one of them used twice, over two backward passes: their fp32 gradients are the sums of what the calls give one by
    one to within the roundings of those, and the norm is theirs."""
    import torch.distributed as dist

    from yafsdp_b200 import MixedPrecisionPolicy, fully_shard
    from yafsdp_b200.ops import functional as Fn
    from yafsdp_b200.optim import clip_grad_norm_

    d = 520

    class Steps(torch.nn.Module):
        def __init__(self):
            super().__init__()
            gen = torch.Generator(device=DEV).manual_seed(0)
            self.w, self.post, self.gate = (torch.nn.Parameter((1 + 0.1 * torch.randn(d, device=DEV, generator=gen)).bfloat16().float()) for _ in range(3))

        def forward(self, x, y):
            h, n = Fn.residual_norm(x, y, self.w, post_weight=self.post, gate=self.gate, scale=0.5)
            return Fn.residual_norm(h, n, self.w)

    torch.cuda.set_device(0)
    created = not dist.is_initialized()
    if created:
        dist.init_process_group("nccl", store=dist.HashStore(), rank=0, world_size=1)
    try:
        model = Steps()
        w, post, gate = (p.detach().bfloat16() for p in (model.w, model.post, model.gate))
        fully_shard(model, mp_policy=MixedPrecisionPolicy(param_dtype=torch.bfloat16, reduce_dtype=torch.float32))
        total = {name: [torch.zeros(d, device=DEV, dtype=torch.float64) for _ in range(2)] for name in ("w", "post", "gate")}
        for step in range(2):
            x, y, dh, dn = (torch.randn(1, 77, d, device=DEV).bfloat16() for _ in range(4))
            torch.autograd.backward(model(x, y), (dh, dn))
            one, two = w.clone().requires_grad_(), w.clone().requires_grad_()
            p, g = post.clone().requires_grad_(), gate.clone().requires_grad_()
            h, n = Fn.residual_norm(x, y, one, post_weight=p, gate=g, scale=0.5)
            for name, grad in zip(("w", "w", "post", "gate"), torch.autograd.grad(Fn.residual_norm(h, n, two), (one, two, p, g), (dh, dn))):
                total[name][0] += grad.double()
                total[name][1] += grad.double().abs()
        _done()
        grads = {name: p.grad._local_tensor for name, p in model.named_parameters()}
        for name, (want, mass) in total.items():
            # each bf16 gradient is off by half a step of its own; where the module adds bf16 gradients (the gate), its sums are fp32
            assert ((grads[name].view(-1).double() - want).abs() <= 1.01 * 2.0**-8 * mass + 1e-12).all(), name
        norm = torch.stack([g.double().norm() for g in grads.values()]).norm()
        assert abs(clip_grad_norm_(model, 1e9).item() / norm.item() - 1.0) < 1e-5
    finally:
        if created:
            dist.destroy_process_group()


def test_attention_refuses_too_many_rows():
    from yafsdp_b200.ops import functional as Fn

    t = torch.empty(65536, 1, 1, 128, device=DEV, dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        Fn.attention(t, t, t)


@pytest.mark.parametrize("s,window,mean", [(1, 0, 1), (1, 1, 1), (300, 1, 50), (300, 0, 1), (300, 0, 3)])
@pytest.mark.parametrize("softcap,biased,hkv", [(0.0, False, 4), (30.0, True, 1)])
def test_tokens_that_see_one_key(s, window, mean, softcap, biased, hkv):
    """The probability of an only key is 1: the output is its value to the bit, and neither q nor a key that nothing else looks at gets a gradient."""
    from yafsdp_b200.ops import functional as Fn

    b, hq = 3, 4
    mask = Fn.document_mask((_ids(b, s, mean, False) if mean > 1 else torch.arange(s).expand(b, s)).to(DEV), window=window)
    slopes = torch.rand(hq, device=DEV) if biased else None
    for m in (mask, None) if s == 1 else (mask,):
        q, k, v = _qkv(b, s, hq, hkv)
        out = Fn.attention(q, k, v, m, softcap=softcap, slopes=slopes)
        dq, dk, dv = torch.autograd.grad(out, (q, k, v), torch.randn_like(out))
        one = mask.spans[..., 1] - mask.spans[..., 0] == 1
        at = mask.spans[..., 0].long()
        values = v.detach().repeat_interleave(hq // hkv, 2).gather(1, at[..., None, None].expand(b, s, hq, 128))
        assert one.any() and torch.equal(out[one], values[one])
        assert (dq[one] == 0).all() and (one.all() or (dq[~one] != 0).any())
        only = (mask.key_spans[..., 1] - mask.key_spans[..., 0] == 1) & one.gather(1, mask.key_spans[..., 0].long().clamp(max=s - 1))
        assert (dk[only] == 0).all() and (dv != 0).any()
    _done()


@pytest.mark.parametrize("turned", [False, True])
def test_attention_of_scores_that_grow_along_the_row(turned):
    """Keys ten times as long at the end of a row as at its start, or the other way round: references that have to move by more than 2^40, or that
    stay far above what comes later."""
    from yafsdp_b200.ops import functional as Fn

    b, s, hq, hkv = 2, 300, 4, 2
    q, k, v = (t.detach() for t in _qkv(b, s, hq, hkv))
    growth = 1 + torch.arange(s, device=DEV) / 32
    k = (k.float() * (growth.flip(0) if turned else growth)[:, None, None]).bfloat16()
    q, k, v = (t.requires_grad_() for t in (q, k, v))
    out = Fn.attention(q, k, v)
    dout = torch.randn(out.shape, device=DEV, generator=torch.Generator(device=DEV).manual_seed(1)).bfloat16()
    grads = torch.autograd.grad(out, (q, k, v), dout)
    _done()
    want = oracle.attention(q.detach(), k.detach(), v.detach(), _seen(None, b, s), 128**-0.5, 0.0, None, dout)
    scores = torch.einsum("bihd,bjhd->bhij", q.detach().float(), k.detach().float().repeat_interleave(2, 2)) * 128**-0.5 * 1.4427
    scores = scores.masked_fill(~_seen(None, b, s)[:, None], -math.inf)
    moved = scores.amax(-1) - scores[..., :64].amax(-1)
    assert turned or (moved > 40).any()
    for name, got, w in zip(("out", "dq", "dk", "dv"), (out, *grads), want):
        oracle.close(got.detach(), w, name)


@pytest.mark.parametrize("gate", ["none", "channel", "sample", "token"])
@pytest.mark.parametrize("post", [False, True])
def test_residual_norm_gradients_of_one_result_or_none(gate, post):
    """One of the two gradients missing is a gradient of zeros, whatever the gate; both missing: no input gets one, and the C entry refuses."""
    from yafsdp_b200.ops import functional as Fn
    from yafsdp_b200.ops import kernels

    x, y, w, p, g, dh, dn = _norm_case((3, 37, 512), gate, post, torch.bfloat16)
    leaves = [t.requires_grad_() for t in (x, y, w, p, g) if t is not None]
    for which, given in ((0, dh), (1, dn)):
        one = torch.autograd.grad(Fn.residual_norm(x, y, w, post_weight=p, gate=g)[which], leaves, given, allow_unused=True)
        both = torch.autograd.grad(Fn.residual_norm(x, y, w, post_weight=p, gate=g), leaves, (dh, dn * 0) if which == 0 else (dh * 0, dn))
        assert all(torch.equal(a, z) for a, z in zip(one, both))

    class NoGradient(torch.autograd.Function):
        @staticmethod
        def forward(ctx, h, n):
            return h.sum() * 0

        @staticmethod
        def backward(ctx, grad):
            return None, None

    NoGradient.apply(*Fn.residual_norm(x, y, w, post_weight=p, gate=g)).backward()
    assert all(t.grad is None for t in leaves)
    rows = {"none": 0, "channel": 1, "sample": 3, "token": 111}[gate]
    plain = [None if t is None else t.detach() for t in (x, y, w, p, g)]
    rstd = kernels.residual_norm_fwd(*plain, rows, 1.0, 1e-5)[2]
    with pytest.raises(RuntimeError):
        kernels.residual_norm_bwd(*plain, rows, rstd, None, None, 1.0, torch.empty_like(w), torch.empty_like(w) if post else None)
    _done()


@pytest.mark.parametrize("beyond", [1, 100, 2**31 - 1])
@pytest.mark.parametrize("window", [0, 40])
def test_attention_under_ranges_beyond_the_row(beyond, window):
    """A mask put together by hand whose ranges start before their row or end behind it: the same as cut to the row, to the bit (but dQ)."""
    from yafsdp_b200.ops import functional as Fn

    b, s, hq, hkv = 2, 300, 4, 2
    ids = _ids(b, s, 60, True).to(DEV)
    ids[0, -1] = 77  # a document of the row's last token: it sees itself alone
    flags = torch.zeros(b, s, device=DEV, dtype=torch.bool)
    flags[1, -30:] = True
    ids[1, -30:] = 99  # a prefix up to the row's end
    mask = Fn.document_mask(ids, flags, window)
    far = min(s + beyond, 2**31 - 1)
    wide = Fn.DocumentMask(*(torch.where(t == s, far, torch.where(t == 0, -beyond, t)) for t in (mask.spans, mask.key_spans)), mask.positions, mask.padding)
    assert (wide.spans != mask.spans).any() and (wide.key_spans != mask.key_spans).any()
    results = []
    for m in (mask, wide):
        q, k, v = _qkv(b, s, hq, hkv)
        out = Fn.attention(q, k, v, m)
        dout = torch.randn(out.shape, device=DEV, generator=torch.Generator(device=DEV).manual_seed(1)).bfloat16()
        results.append((out.detach(), *torch.autograd.grad(out, (q, k, v), dout)))
    _done()
    for i, (a, z) in enumerate(zip(*results)):
        assert torch.allclose(a.float(), z.float(), rtol=2.0**-7, atol=1e-4) if i == 1 else torch.equal(a, z), i
    assert (results[1][1][0, -1] == 0).all() and (results[1][2][0, -1] == 0).all()


def test_residual_norm_refuses_rows_beyond_32_bits():
    from yafsdp_b200.ops import functional as Fn
    from yafsdp_b200.ops import kernels

    w = torch.ones(8, device=DEV, dtype=torch.bfloat16)
    for rows in (kernels.MAX_NORM_ROWS + 1, 2**31 + 1, 2**32 + 1):  # one row, many times
        x = w.expand(rows, 8)
        with pytest.raises(ValueError):
            Fn.residual_norm(x, x, w)


def _three_calls(dtype=torch.bfloat16):
    """The operators with gradients, each as a function of all its inputs that may have one."""
    from yafsdp_b200.ops import functional as Fn

    mask = Fn.document_mask(_ids(2, 40, 9, True).to(DEV))
    q, k, v = (t.detach() for t in _qkv(2, 40, 4, 2))
    x, y, w, post, gate, _, _ = _norm_case((2, 40, 512), "sample", True, dtype)
    axes = Fn.RotaryAxes(128, 1e4)
    return {"rotary": (lambda *a: Fn.rotary(*a, mask.positions, axes), (q, k)), "attention": (lambda *a: Fn.attention(*a, mask, softcap=9.0), (q, k, v)),
            "residual_norm": (lambda *a: Fn.residual_norm(a[0], a[1], a[2], post_weight=a[3], gate=a[4]), (x, y, w, post, gate))}


@pytest.mark.parametrize("name", ["rotary", "attention", "residual_norm"])
@pytest.mark.parametrize("grad", [False, True])
def test_forward_mode_tangents_are_refused(name, grad):
    """The kernels have no forward-mode derivative: a tangent is refused, whichever input has it, and not dropped."""
    from torch.autograd import forward_ad

    call, tensors = _three_calls()[name]
    first = lambda out: out if torch.is_tensor(out) else out[0]  # noqa: E731
    with torch.set_grad_enabled(grad), forward_ad.dual_level():
        for i, t in enumerate(tensors):
            duals = [forward_ad.make_dual(t, torch.ones_like(t)) if j == i else z for j, z in enumerate(tensors)]
            with pytest.raises(RuntimeError, match="jvp"):
                call(*duals)
        assert torch.equal(first(call(*tensors)), first(call(*tensors)))  # no tangent anywhere
    _done()


@pytest.mark.parametrize("name,power", [("rotary", 2), ("attention", 1), ("attention", 2), ("residual_norm", 1), ("residual_norm", 2)])
def test_second_derivatives_are_refused(name, power):
    """A gradient taken with ``create_graph`` is right, and a derivative of it is refused, not zero, also where the loss reaches the inputs on another
    way.  (The derivative of the gradient of a sum of what ``rotary`` gives is zero.)"""
    call, tensors = _three_calls()[name]
    leaves = [t.clone().requires_grad_() for t in tensors]

    def total():
        out = call(*leaves)
        return sum(t.float().pow(power).sum() for t in (out if isinstance(out, tuple) else (out,)))

    once = torch.autograd.grad(total(), leaves)
    loss = total()
    grads = torch.autograd.grad(loss, leaves, create_graph=True)
    for i, (a, z) in enumerate(zip(grads, once)):
        assert torch.allclose(a.float(), z.float(), rtol=2.0**-7, atol=1e-4) if name == "attention" and i == 0 else torch.equal(a, z)
    for take in (lambda t: torch.autograd.grad(t, leaves, retain_graph=True), lambda t: torch.autograd.grad(t, leaves[:1], retain_graph=True), lambda t: t.backward(retain_graph=True)):
        with pytest.raises(RuntimeError, match="differentiated once"):
            take(loss + sum(g.float().pow(2).sum() for g in grads))
    _done()


def test_rotary_trains_after_inference_mode():
    """The table of frequencies that an evaluation under ``inference_mode`` made serves the training behind it."""
    from yafsdp_b200.ops import functional as Fn

    axes = Fn.RotaryAxes(64, 1e4)
    q, k = torch.randn(2, 33, 4, 64, device=DEV).bfloat16(), torch.randn(2, 33, 2, 64, device=DEV).bfloat16()
    positions = torch.randint(0, 1000, (2, 33), device=DEV)
    with torch.inference_mode():
        want = [t.clone() for t in Fn.rotary(q, k, positions, axes)]
    q.requires_grad_()
    out = Fn.rotary(q, k, positions, axes)
    assert all(torch.equal(a, z) for a, z in zip(out, want))
    assert torch.autograd.grad(out[0].sum(), q)[0].shape == q.shape


def test_rotary_table_of_the_current_device():
    from yafsdp_b200.ops import functional as Fn

    axes = Fn.RotaryAxes(64, 1e4)
    table = axes.table(torch.device("cuda"))
    assert axes.table(torch.device("cuda", torch.cuda.current_device())) is table and axes.table("cuda") is table


@pytest.mark.parametrize("theta", [1e4, 5e5])
@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_rotary_at_far_positions(theta, dtype):
    """Angles to 2^-32 of a turn up to positions of 2^32, in all quarters of a turn, and to what the frequency's last bit leaves over beyond."""
    from test_packed import FAR, far_positions

    near = list(range(0, 4000, 7)) + [p for p in FAR if dtype == torch.int64 or abs(p) < 2**31]
    got, want, off = far_positions(theta, DEV, torch.tensor(near, dtype=dtype))
    _done()
    # cosines and sines of at most an eighth of a turn to two units (2^-23 each), the turn by what the float leaves over to half of one
    assert ((got - want).abs() <= 5 * 2.0**-24 * want.abs() + off).all()


def _long_rows(s):
    """Documents that start or end beside the places up to which a tile of 1024 tokens reads at once: its neighbours and then 4096 tokens at a time."""
    ids = torch.zeros(8, s, dtype=torch.int64)  # 0: one document
    for row, at in ((1, 1024), (2, 1023), (3, 4096 + 1024), (4, 4096 + 1025)):
        ids[row, at:] = 5  # two
    ids[5, s - 1 :] = 6  # the last token alone
    ids[6, :1500] = ids[6, -2500:] = -1  # padding at either end
    ids[7, 9000:9010] = -3  # and in the middle
    return ids


@pytest.mark.parametrize("s", [20000, 13312, 9217])
@pytest.mark.parametrize("window", [0, 6000])
@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_document_mask_of_long_documents(s, window, dtype):
    """Starts, ends and unflagged tokens many tiles away, with and without prefixes."""
    from yafsdp_b200.ops import functional as Fn

    ids = _long_rows(s).to(dtype)
    at = torch.arange(s)
    # nothing flagged; all; all but one token far from the row's ends; the first tokens of a document; the last ones
    flags = [torch.zeros_like(ids, dtype=torch.bool), torch.ones_like(ids, dtype=torch.bool), *((at != p).expand_as(ids) for p in (0, 1030, 7000, s - 2)),
             (at < 5500).expand_as(ids), (at > 3000).expand_as(ids)]
    for prefix in (None, *flags):
        want = Fn._document_mask_ref(ids, prefix, window)
        got = Fn.document_mask(ids.to(DEV), None if prefix is None else prefix.contiguous().to(DEV), window)
        for name in ("spans", "key_spans", "positions", "padding"):
            assert torch.equal(getattr(got, name).cpu(), getattr(want, name)), name
    _done()


@pytest.mark.parametrize("packed", [False, True])
def test_attention_of_scores_up_to_a_billion(packed):
    """Scores so large that fp32 has no fractions of them: the largest take all, shared evenly, and nothing overflows."""
    from yafsdp_b200.ops import functional as Fn

    b, s, hq, hkv = 2, 300, 4, 2
    mask = Fn.document_mask(_ids(b, s, 70, True).to(DEV)) if packed else None
    _, _, v = (t.detach() for t in _qkv(b, s, hq, hkv))
    # powers of two, whose products and sums are exact: 128 * 2^10 * 2^0 to 2^15, by 0.2 up to 0.86e9
    q = torch.full((b, s, hq, 128), 2.0**10, device=DEV, dtype=torch.bfloat16)
    k = (2.0 ** (torch.arange(s, device=DEV) * 7 % 16)).bfloat16()[None, :, None, None].expand(b, s, hkv, 128)
    out = Fn.attention(q, k, v, mask, scale=0.2)
    _done()
    oracle.close(out, oracle.attention(q, k, v, _seen(mask, b, s), 0.2, 0.0, None))
