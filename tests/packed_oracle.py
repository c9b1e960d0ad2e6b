"""The operators around packed documents in 64 bits, with bounds on what roundings may move (shared by the CPU and GPU tests)."""

import decimal
import math

import torch

HALF_STEP = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: 2.0**-24}


def spans_of(ids, prefix, window):
    """(spans, key_spans, positions) of rows of document ids, by walking over the documents."""
    b, s = ids.shape
    spans, key_spans = torch.zeros(b, s, 2, dtype=torch.int32), torch.zeros(b, s, 2, dtype=torch.int32)
    positions = torch.zeros(b, s, dtype=torch.int32)
    for r in range(b):
        row, i = ids[r].tolist(), 0
        flags = [False] * s if prefix is None else prefix[r].tolist()
        while i < s:
            if row[i] < 0:
                spans[r, i] = key_spans[r, i] = torch.tensor([i, i])
                i += 1
                continue
            end = i
            while end < s and row[end] == row[i]:
                end += 1
            lead = i
            while lead < end and flags[lead]:
                lead += 1
            for t in range(i, end):
                spans[r, t, 0] = max(i, t - window + 1) if window else i
                spans[r, t, 1] = lead if t < lead else t + 1
                key_spans[r, t, 0] = i if t < lead else t
                key_spans[r, t, 1] = min(end, t + window) if window else end
                positions[r, t] = t - i
            i = end
    return spans, key_spans, positions


def turned(positions, theta, head_dim):
    """(cosines, sines), float64 lists of rows of head_dim / 2, of positions (whole numbers) times theta^(-2 j / head_dim), the angles in 80 digits."""
    with decimal.localcontext() as c:
        c.prec = 80
        # pi by Machin's formula: 16 atan(1/5) - 4 atan(1/239)
        unit = 10**90
        atan = lambda n: sum((-1) ** i * (unit // n ** (2 * i + 1)) // (2 * i + 1) for i in range(70))  # noqa: E731
        two_pi = decimal.Decimal(2 * (16 * atan(5) - 4 * atan(239))) / unit
        step = [(decimal.Decimal(theta).ln() * -2 * j / head_dim).exp() / two_pi for j in range(head_dim // 2)]
        angles = [[float((f * p) % 1 * two_pi) for f in step] for p in positions]
    return [[math.cos(a) for a in row] for row in angles], [[math.sin(a) for a in row] for row in angles]


def attention(q, k, v, seen, scale, softcap, slopes, dout=None):
    """Output, gradients and, for each, how far bf16 kernels may be off: probabilities, score gradients and results are rounded to bf16
    (half a step each, relative), the row sums D = dO . O read the rounded output; everything else is fp32, 2^-14 of the terms in all
    (exponents up to 2^6 and their exponentials to 2^-20, sums of some hundred terms).  ``seen``: [B, S, S].

    With weights w_j = p_j / l, roundings d_j <= u of them, and those of some keys T (the largest ones) taken into the sum that is divided by, the
    output before its own rounding is sum (1 + d_j) w_j v_j / (1 + sum_T d_j w_j), off to first order by sum_T d_j w_j (v_j - o) + sum_rest d_j w_j v_j
    <= u (mass + |o| sum_T w_j) <= u (mass + |o|), where mass = sum w_j |v_j|."""
    u, f = 2.0**-8, 2.0**-14
    q, k, v = (t.double() for t in (q, k, v))
    b, s, hq, d = q.shape
    group = hq // k.shape[2]
    ke, ve = k.repeat_interleave(group, 2), v.repeat_interleave(group, 2)
    x = torch.einsum("bihd,bjhd->bhij", q, ke) * scale
    t = torch.tanh(x / softcap) if softcap else torch.zeros_like(x)
    if softcap:
        x = softcap * t
    at = torch.arange(s, device=q.device)
    if slopes is not None:
        x = x - slopes.double()[:, None, None] * (at[:, None] - at[None, :]).abs()
    some = seen.any(2)[:, None, :, None]
    p = x.masked_fill(~seen[:, None] & some, -math.inf).softmax(-1) * some
    o = torch.einsum("bhij,bjhd->bihd", p, ve)
    mass = torch.einsum("bhij,bjhd->bihd", p, ve.abs())
    o_off = u * (mass + 2 * o.abs()) + f * mass  # roundings of P, taken into its sum or not, and of the output
    if dout is None:
        return o, o_off
    g = dout.double()
    dp = torch.einsum("bihd,bjhd->bhij", g, ve)
    rows = (g * o).sum(-1).transpose(1, 2)[..., None]
    rows_off = (g.abs() * o_off).sum(-1).transpose(1, 2)[..., None]
    slope = 1 - t * t
    ds = p * (dp - rows) * slope
    dp_mass = torch.einsum("bihd,bjhd->bhij", g.abs(), ve.abs())
    ds_off = u * ds.abs() + p * slope * rows_off + f * p * (dp_mass + rows.abs())
    fold = lambda z: z.unflatten(2, (hq // group, group)).sum(3)  # noqa: E731  shared key heads
    dq = torch.einsum("bhij,bjhd->bihd", ds, ke) * scale
    dk = fold(torch.einsum("bhij,bihd->bjhd", ds, q) * scale)
    dv = fold(torch.einsum("bhij,bihd->bjhd", p, g))
    dq_off = torch.einsum("bhij,bjhd->bihd", ds_off, ke.abs()) * scale + u * dq.abs()
    dk_off = fold(torch.einsum("bhij,bihd->bjhd", ds_off, q.abs()) * scale) + u * dk.abs()
    dv_off = fold(torch.einsum("bhij,bihd->bjhd", p, g.abs())) * (u + f) + u * dv.abs()
    return (o, o_off), (dq, dq_off), (dk, dk_off), (dv, dv_off)


def residual_norm(x, y, w, post, gate, scale, eps, dh=None, dn=None):
    """Outputs, gradients and bounds: a half step of the type for each result, and for fp32 sums ``f`` of the terms' magnitudes (a sum of 2^14
    terms in threads, warps and blocks is a chain of fewer than 128 additions; the sums over tokens are a chain of fewer than 1024)."""
    step, f, chain = HALF_STEP[x.dtype], 2.0**-17, 2.0**-14
    x, y, w = (t.double() for t in (x, y, w))
    post, gate = (None if t is None else t.double() for t in (post, gate))
    ry = None if post is None else torch.rsqrt(y.pow(2).mean(-1, keepdim=True) + eps)
    yhat = y if post is None else y * ry
    p = torch.ones_like(w) if post is None else post
    s = scale * (torch.ones_like(x) if gate is None else gate.expand_as(x))
    u = yhat * p
    h = x + s * u
    rh = torch.rsqrt(h.pow(2).mean(-1, keepdim=True) + eps)
    hhat = h * rh
    h_off = f * (x.abs() + (s * u).abs())
    hhat_off = rh * h_off + f * hhat.abs()
    n = hhat * w
    out = {"h": (h, h_off + step * h.abs()), "n": (n, hhat_off * w.abs() + step * n.abs())}
    if dh is None:
        return out
    dh, dn = dh.double(), dn.double()
    c = dn * w
    dot = (c * hhat).mean(-1, keepdim=True)
    dot_off = (c.abs() * (hhat_off + f * hhat.abs())).mean(-1, keepdim=True)
    g = dh + rh * (c - hhat * dot)
    g_off = f * (dh.abs() + rh * (c.abs() + (hhat * dot).abs())) + rh * (hhat_off * dot.abs() + hhat.abs() * dot_off)
    e = s * g
    e_off = s.abs() * g_off + f * e.abs()
    out["dx"] = (g, g_off + step * g.abs())
    lead = tuple(range(x.dim() - 1))
    dw = (dn * hhat).sum(lead)
    out["dw"] = (dw, (dn.abs() * (hhat_off + chain * hhat.abs())).sum(lead) + step * dw.abs())
    if post is None:
        out["dy"] = (e, e_off + step * e.abs())
    else:
        ep = e * p
        dot2 = (ep * yhat).mean(-1, keepdim=True)
        dot2_off = (p.abs() * yhat.abs() * (e_off + f * e.abs())).mean(-1, keepdim=True)
        dy = ry * (ep - yhat * dot2)
        dy_off = ry * (e_off * p.abs() + f * (ep.abs() + (yhat * dot2).abs()) + yhat.abs() * dot2_off)
        out["dy"] = (dy, dy_off + step * dy.abs())
        dpost = (e * yhat).sum(lead)
        out["dpost"] = (dpost, (yhat.abs() * (e_off + chain * e.abs())).sum(lead) + step * dpost.abs())
    if gate is not None:
        d, off = scale * g * u, abs(scale) * u.abs() * (g_off + chain * g.abs())
        fold = lambda z: z.sum_to_size(gate.shape)  # noqa: E731
        out["dgate"] = (fold(d), fold(off) + step * fold(d).abs())
    return out


# Half a step where a type's numbers are evenly spaced (below its smallest normal number, 2^-14 of fp16): 2^-24 / 2 of fp16; for bf16 and
# fp32, 2^-126 and what the exponentials flush there.
FLOOR = {torch.bfloat16: 1e-35, torch.float16: 2.0**-25, torch.float32: 1e-35}


def close(got, want_and_off, name=""):
    want, off = want_and_off
    bad = (got.double() - want).abs() - off
    assert got.shape == want.shape and not torch.isnan(got).any(), f"{name}: shape or NaN"
    worst, floor = bad.max().item() if bad.numel() else 0.0, FLOOR[got.dtype]
    assert worst <= floor, f"{name}: {(bad > floor).sum().item()} of {bad.numel()} out of bounds, by up to {worst}, of {want.abs().max().item()}"
