"""Packed documents on the CPU: plain forms of the mask, rotary positions, attention and the residual norm step, and what is refused."""

import math

import packed_oracle as oracle
import pytest
import torch

from yafsdp_b200.ops import functional as Fn

CASES = [
    [[0]], [[-1]], [[5, 5, 5, 5]], [[-1, -3, 2, 2, -1, 4, 4, 4, -1]], [[1, 1, 2, 2, 1, 1, 0], [7, 7, 7, 7, 7, 7, -2]], [[3, 2, 1, 0, -1, -1, -1]],
]


@pytest.mark.parametrize("ids", CASES)
@pytest.mark.parametrize("window", [0, 1, 2, 100])
@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_document_mask(ids, window, dtype):
    ids = torch.tensor(ids, dtype=dtype)
    gen = torch.Generator().manual_seed(0)
    for prefix in (None, torch.ones_like(ids, dtype=torch.bool), torch.rand(ids.shape, generator=gen) < 0.6):
        m = Fn.document_mask(ids, prefix, window)
        for got, want in zip((m.spans, m.key_spans, m.positions), oracle.spans_of(ids, prefix, window)):
            assert torch.equal(got, want) and got.dtype == torch.int32
        # both views of the mask say the same
        at = torch.arange(ids.shape[1])
        by_query = (at >= m.spans[..., :1]) & (at < m.spans[..., 1:])
        by_key = (at >= m.key_spans[..., :1]) & (at < m.key_spans[..., 1:])
        assert torch.equal(by_query, by_key.transpose(1, 2))
        assert m.padding.tolist() == [[int((row < 0).sum())] for row in ids]


def test_document_mask_of_nothing():
    for shape in ((0, 5), (3, 0)):
        m = Fn.document_mask(torch.zeros(shape, dtype=torch.int64))
        assert m.spans.shape == (*shape, 2) and m.positions.shape == shape


@pytest.mark.parametrize("softcap,biased", [(0.0, False), (5.0, False), (0.0, True), (3.0, True)])
@pytest.mark.parametrize("masked", [False, True])
def test_attention_reference_and_differences(softcap, biased, masked):
    torch.manual_seed(0)
    b, s, hq, hkv, d = 2, 9, 4, 2, 16
    ids = torch.tensor([[0, 0, 0, 1, 1, 1, 1, -1, -1], [-1, 4, 4, 4, 4, 4, 4, 4, 5]])
    mask = Fn.document_mask(ids, ids % 4 == 0, 4) if masked else None
    q, k, v = (torch.randn(b, s, h, d, requires_grad=True) for h in (hq, hkv, hkv))
    slopes = torch.tensor([0.5, 0.25, 0.125, 0.0625]) if biased else None
    out = Fn.attention(q, k, v, mask, softcap=softcap, slopes=slopes)
    dout = torch.randn_like(out)
    grads = torch.autograd.grad(out, (q, k, v), dout)
    at = torch.arange(s)
    seen = (at >= mask.spans[..., :1]) & (at < mask.spans[..., 1:]) if masked else (at <= at[:, None]).expand(b, s, s)
    want = oracle.attention(q.detach(), k.detach(), v.detach(), seen, d**-0.5, softcap, slopes, dout)
    for got, w in zip((out, *grads), want):
        oracle.close(got.detach(), w)
    assert not masked or (out[0, 7:] == 0).all()
    # the formulas of the gradients against differences of the definition
    step = 1e-5
    for i, (x, g) in enumerate(zip((q, k, v), (w[0] for w in want[1:]))):
        way = torch.randn(x.shape, dtype=torch.float64)
        ends = []
        for sign in (1, -1):
            args = [t.detach().double() for t in (q, k, v)]
            args[i] = args[i] + sign * step * way
            ends.append((oracle.attention(*args, seen, d**-0.5, softcap, slopes)[0] * dout.double()).sum())
        assert (ends[0] - ends[1]).item() / (2 * step) == pytest.approx((g * way).sum().item(), rel=1e-6, abs=1e-7)


@pytest.mark.parametrize("gate", [None, "channel", "sample", "token"])
@pytest.mark.parametrize("post", [False, True])
def test_residual_norm_reference_and_differences(gate, post):
    torch.manual_seed(0)
    b, s, d = 2, 3, 8
    x, y, dh, dn = (torch.randn(b, s, d) for _ in range(4))
    w, p = 1 + 0.1 * torch.randn(d), 1 + 0.1 * torch.randn(d) if post else None
    g = None if gate is None else torch.randn({"channel": (d,), "sample": (b, 1, d), "token": (b, s, d)}[gate])
    leaves = {n: t.requires_grad_() for n, t in (("dx", x), ("dy", y), ("dw", w), ("dpost", p), ("dgate", g)) if t is not None}
    h, n = Fn.residual_norm(x, y, w, post_weight=p, gate=g, scale=0.7)
    grads = dict(zip(leaves, torch.autograd.grad((h, n), list(leaves.values()), (dh, dn))))
    plain = [None if t is None else t.detach() for t in (x, y, w, p, g)]
    want = oracle.residual_norm(*plain, 0.7, 1e-5, dh, dn)
    for name, got in {"h": h.detach(), "n": n.detach(), **grads}.items():
        oracle.close(got, want[name], name)
    step = 1e-5
    for i, name in enumerate(("dx", "dy", "dw", "dpost", "dgate")):
        if name not in want:
            continue
        way = torch.randn(plain[i].shape, dtype=torch.float64)
        ends = []
        for sign in (1, -1):
            args = [None if t is None else t.double() for t in plain]
            args[i] = args[i] + sign * step * way
            # bounds are not asked for here, so any type will do for them
            o = _in_64_bits(args)
            ends.append((o[0] * dh.double() + o[1] * dn.double()).sum())
        assert (ends[0] - ends[1]).item() / (2 * step) == pytest.approx((want[name][0] * way).sum().item(), rel=1e-6, abs=1e-7)


def _in_64_bits(args):
    x, y, w, p, g = args
    u = y if p is None else y / (y.pow(2).mean(-1, keepdim=True) + 1e-5).sqrt() * p
    h = x + 0.7 * (u if g is None else g * u)
    return h, h / (h.pow(2).mean(-1, keepdim=True) + 1e-5).sqrt() * w


def test_rotary_of_one_axis_is_the_table_form():
    torch.manual_seed(0)
    q, k = torch.randn(2, 7, 4, 32), torch.randn(2, 7, 2, 32)
    axes = Fn.RotaryAxes(32, 10000.0)
    got_q, got_k = Fn.rotary(q, k, torch.arange(7).expand(2, 7), axes)
    table = Fn.rope_table(7, 32, 10000.0, "cpu")
    assert torch.equal(got_q, Fn.rope_ref(q, table)) and torch.equal(got_k, Fn.rope_ref(k, table))


def test_rotary_axes_layouts():
    assert Fn.RotaryAxes(16, 1e4, (3, 3, 2)).axis == [0, 0, 0, 1, 1, 1, 2, 2]
    assert Fn.RotaryAxes(16, 1e4, (4, 3, 1), interleaved=True).axis == [0, 1, 2, 0, 1, 0, 1, 0]
    # the fixed-point table against a turn's fraction
    axes = Fn.RotaryAxes(128, 5e5, (16, 24, 24))
    table = axes.table(torch.device("cpu"))
    for j in (0, 1, 17, 63):
        assert (int(table[j, 0]) % 2**64) / 2.0**64 == pytest.approx(5e5 ** (-j / 64) / (2 * math.pi), rel=1e-15)
    assert table[:, 1].tolist() == axes.axis


@pytest.mark.parametrize("call,error", [
    (lambda: Fn.document_mask(torch.zeros(4, dtype=torch.int64)), ValueError),
    (lambda: Fn.document_mask(torch.zeros(1, 4)), ValueError),
    (lambda: Fn.document_mask(torch.zeros(1, 4, dtype=torch.int64), torch.zeros(1, 4)), ValueError),
    (lambda: Fn.document_mask(torch.zeros(1, 4, dtype=torch.int64), torch.zeros(1, 3, dtype=torch.bool)), ValueError),
    (lambda: Fn.document_mask(torch.zeros(1, 4, dtype=torch.int64), window=-1), ValueError),
    (lambda: Fn.RotaryAxes(24, 1e4), ValueError),
    (lambda: Fn.RotaryAxes(32, -1.0), ValueError),
    (lambda: Fn.RotaryAxes(32, 1e4, (8, 4)), ValueError),
    (lambda: Fn.rotary(torch.zeros(1, 2, 1, 32), torch.zeros(1, 2, 1, 16), torch.zeros(1, 2, dtype=torch.int64), Fn.RotaryAxes(32, 1e4)), ValueError),
    (lambda: Fn.rotary(torch.zeros(1, 2, 1, 32), torch.zeros(1, 2, 1, 32), torch.zeros(1, 2), Fn.RotaryAxes(32, 1e4)), ValueError),
    (lambda: Fn.rotary(torch.zeros(1, 2, 1, 32), torch.zeros(1, 2, 1, 32), torch.zeros(1, 2, dtype=torch.int64), Fn.RotaryAxes(32, 1e4, (8, 8))), ValueError),
    (lambda: Fn.rotary(torch.zeros(1, 2, 1, 32), torch.zeros(1, 2, 1, 32).half(), torch.zeros(1, 2, dtype=torch.int64), Fn.RotaryAxes(32, 1e4)), TypeError),
    (lambda: Fn.attention(torch.zeros(1, 2, 3, 16), *[torch.zeros(1, 2, 2, 16)] * 2), ValueError),
    (lambda: Fn.attention(torch.zeros(1, 2, 2, 16), torch.zeros(1, 3, 2, 16), torch.zeros(1, 3, 2, 16)), ValueError),
    (lambda: Fn.attention(torch.zeros(1, 2, 2, 16), *[torch.zeros(1, 2, 2, 16).half()] * 2), TypeError),
    (lambda: Fn.attention(*[torch.zeros(1, 2, 2, 16)] * 3, softcap=-1.0), ValueError),
    (lambda: Fn.attention(*[torch.zeros(1, 2, 2, 16)] * 3, softcap=math.inf), ValueError),
    (lambda: Fn.attention(*[torch.zeros(1, 2, 2, 16)] * 3, scale=0.0), ValueError),
    (lambda: Fn.attention(*[torch.zeros(1, 2, 2, 16)] * 3, scale=math.nan), ValueError),
    (lambda: Fn.attention(*[torch.zeros(1, 2, 2, 16)] * 3, Fn.document_mask(torch.zeros(1, 3, dtype=torch.int64))), ValueError),
    (lambda: Fn.attention(*[torch.zeros(1, 2, 2, 16)] * 3, slopes=torch.zeros(3)), ValueError),
    (lambda: Fn.attention(*[torch.zeros(1, 2, 2, 16)] * 3, slopes=torch.zeros(2, requires_grad=True)), ValueError),
    (lambda: Fn.residual_norm(torch.zeros(2, 8), torch.zeros(3, 8), torch.ones(8)), ValueError),
    (lambda: Fn.residual_norm(torch.zeros(2, 8), torch.zeros(2, 8), torch.ones(7)), ValueError),
    (lambda: Fn.residual_norm(torch.zeros(2, 8), torch.zeros(2, 8), torch.ones(8), post_weight=torch.ones(1, 8)), ValueError),
    (lambda: Fn.residual_norm(torch.zeros(2, 8), torch.zeros(2, 8).half(), torch.ones(8)), TypeError),
    (lambda: Fn.residual_norm(torch.zeros(2, 8), torch.zeros(2, 8), torch.ones(8), gate=torch.ones(3, 8)), ValueError),
    (lambda: Fn.residual_norm(torch.zeros(2, 3, 8), torch.zeros(2, 3, 8), torch.ones(8), gate=torch.ones(1, 3, 8)), ValueError),
    (lambda: Fn.residual_norm(torch.zeros(2, 8), torch.zeros(2, 8), torch.ones(8), scale=math.inf), ValueError),
    (lambda: Fn.residual_norm(torch.zeros(2, 8), torch.zeros(2, 8), torch.ones(8), eps=0.0), ValueError),
])
def test_refusals(call, error):
    with pytest.raises(error):
        call()


def test_hand_made_masks():
    m = Fn.document_mask(torch.zeros(2, 130, dtype=torch.int64))
    parts = {n: getattr(m, n) for n in ("spans", "key_spans", "positions", "padding")}
    assert Fn.DocumentMask(**{n: t[:1] for n, t in parts.items()}).spans.shape == (1, 130, 2)
    for name, wrong in (("spans", m.spans[..., :1]), ("key_spans", m.key_spans[:, :129]), ("positions", m.positions[0]), ("padding", m.padding[:, :1]),
                        ("spans", m.spans.long()), ("padding", m.padding.float()), ("key_spans", m.key_spans.transpose(0, 1).contiguous().transpose(0, 1)),
                        ("positions", m.positions.to("meta"))):
        with pytest.raises(ValueError):
            Fn.DocumentMask(**{**parts, name: wrong})


@pytest.mark.parametrize("call", [
    lambda t, w: Fn.attention(t, t, t, softcap=1e-13), lambda t, w: Fn.attention(t, t, t, softcap=1e13), lambda t, w: Fn.attention(t, t, t, scale=1e-13),
    lambda t, w: Fn.attention(t, t, t, scale=1e13), lambda t, w: Fn.residual_norm(t, t, w, post_weight=w),
])
def test_refused_values(call):
    with pytest.raises(ValueError):
        call(torch.zeros(1, 2, 2, 16), torch.ones(16))


class _NoGradient(torch.autograd.Function):
    """Something behind an operator that has no gradient for what it was given."""

    @staticmethod
    def forward(ctx, *tensors):
        return tensors[0].sum() * 0.0

    @staticmethod
    def backward(ctx, grad):
        return None, None


def test_residual_norm_without_any_gradient(monkeypatch):
    """Neither result has a gradient: neither has any input, and no kernel is asked for one."""
    from yafsdp_b200.ops import kernels

    def forward(x, y, weight, post, gate, gate_rows, scale, eps):
        return *Fn._residual_norm_ref(x, y, weight, post, gate, scale, eps), torch.ones(x.numel() // x.shape[-1], 2)

    def backward(*args, **kwargs):
        raise AssertionError("a kernel without a gradient to read")

    monkeypatch.setattr(kernels, "residual_norm_fwd", forward)
    monkeypatch.setattr(kernels, "residual_norm_bwd", backward)
    x, y, gate = (torch.randn(3, 8, requires_grad=True) for _ in range(3))
    w, post = (torch.ones(8, requires_grad=True) for _ in range(2))
    results = Fn.ResidualNormFn.apply(x, y, w, post, gate, 3, 1.0, 1e-5)
    _NoGradient.apply(*results).backward()
    assert all(t.grad is None for t in (x, y, w, post, gate))


def test_attention_under_ranges_beyond_the_row():
    torch.manual_seed(0)
    ids = torch.tensor([[3, 3, 3, 4, 5, 5, 5], [-1, 4, 4, 6, 6, 6, 6]])
    m = Fn.document_mask(ids, ids == 6)
    wide = Fn.DocumentMask(*(torch.where(t == 7, 2**31 - 1, torch.where(t == 0, -9, t)) for t in (m.spans, m.key_spans)), m.positions, m.padding)
    q, k, v = (torch.randn(2, 7, 2, 16) for _ in range(3))
    assert torch.equal(Fn.attention(q, k, v, wide), Fn.attention(q, k, v, m))


def test_residual_norm_rows_that_are_counted():
    """The C entry refuses more rows than 32 bits can walk over (their number plus a step's would overflow)."""
    from yafsdp_b200 import _native
    from yafsdp_b200.ops import kernels

    parts = _native.lib().yf_residual_norm_parts
    for rows in (kernels.MAX_NORM_ROWS + 1, 2**31 - 1):
        assert parts(rows, 8, 0) == -1
    # rows that fill every block
    assert parts(kernels.MAX_NORM_ROWS, 8, 0) == parts(1 << 24, 8, 0) > 1


def test_rotary_table_outlives_inference_mode():
    axes = Fn.RotaryAxes(32, 1e4)
    with torch.inference_mode():
        first = axes.table(torch.device("cpu"))
    assert axes.table(torch.device("cpu")) is first and not first.is_inference()


def test_rotary_table_by_name():
    axes = Fn.RotaryAxes(32, 1e4)
    assert axes.table("cpu") is axes.table(torch.device("cpu"))


def test_cpu_tensors_under_another_default_device():
    """What the forms for CPU tensors make on the way is on the CPU whatever the default device is."""
    torch.manual_seed(0)
    ids, q, k = torch.tensor([[4, 4, 4, -1], [0, 1, 1, 1]]), torch.randn(2, 4, 2, 16), torch.randn(2, 4, 1, 16)

    def call():
        m, axes = Fn.document_mask(ids, ids == 1, 2), Fn.RotaryAxes(16, 1e4)
        empty = Fn.document_mask(ids[:, :0])
        out = [Fn.attention(q, k, k, mask, softcap=3.0) for mask in (m, None)]
        return [m.spans, m.key_spans, m.positions, m.padding, empty.spans, empty.positions, *Fn.rotary(q, k, m.positions, axes), *out, axes.table("cpu")]

    want = call()
    with torch.device("meta"):
        got = call()
    assert all(torch.equal(a, z) for a, z in zip(got, want))


FAR = [0, 1, -1, 3999, 100000, 2**20 + 3, 2**30 + 1, 2**31 - 1, 5 - 2**31, 2**32, 2**33 + 7, 2**40 + 11, 3 - 2**45, 2**53 + 1, 2**62 + 9]


def far_positions(theta, device, positions):
    """(cosines and sines that ``rotary`` turns by, those of the definition, how far the angle may be off) at the positions."""
    ones = torch.zeros(1, len(positions), 1, 64, device=device)
    ones[..., :32] = 1.0
    got = Fn.rotary(ones, ones, positions[None].to(device), Fn.RotaryAxes(64, theta))[0][0, :, 0].double().cpu()
    want = torch.tensor(oracle.turned(positions.tolist(), theta, 64), dtype=torch.float64).transpose(0, 1).reshape(len(positions), 64)
    # half a unit of a frequency of 2^-64 turns for each position, and of the fraction's 32 bits
    return got, want, 2.0 * math.pi * (2.0**-33 + positions.double().abs() * 2.0**-65)[:, None]


@pytest.mark.parametrize("theta", [1e4, 5e5])
def test_rotary_at_far_positions(theta):
    got, want, off = far_positions(theta, "cpu", torch.tensor(FAR))
    assert ((got - want).abs() <= 2.0**-24 * want.abs() + off).all()
    near = torch.tensor([p for p in FAR if abs(p) < 2**31], dtype=torch.int32)
    got, want, off = far_positions(theta, "cpu", near)
    assert ((got - want).abs() <= 2.0**-24 * want.abs() + off).all()


def test_document_mask_of_long_documents():
    ids = torch.zeros(3, 9217, dtype=torch.int64)
    ids[1, 5120:] = 5
    ids[2, :1500] = ids[2, -2500:] = -1
    at = torch.arange(9217)
    for prefix in (None, (at != 7000).expand_as(ids), (at < 5500).expand_as(ids)):
        for window in (0, 6000):
            m = Fn.document_mask(ids, prefix, window)
            for got, want in zip((m.spans, m.key_spans, m.positions), oracle.spans_of(ids, prefix, window)):
                assert torch.equal(got, want)
