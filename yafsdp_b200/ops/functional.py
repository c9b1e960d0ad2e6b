"""Autograd-level ops of the Llama training step.

CUDA tensors run the hand-written sm_100a kernels (:mod:`yafsdp_b200.ops.kernels`) through three
coarse autograd Functions with hand-derived backward passes: the embedding, a whole decoder layer,
and final-norm + LM head + cross-entropy.  Coarse Functions keep the gradient adds of the residual
stream fused into the RMSNorm backward kernel and let every weight gradient go straight from the
tcgen05 GEMM epilogue (fp32, accumulating) into the parameter's *gradient sink* (see
``yafsdp_b200.group.GradSink``) when the parameter is managed by ``fully_shard``.

CPU tensors (gloo plumbing tests) run the same math in plain PyTorch and rely on autograd.  On a CUDA
device the native path is the only one: there is no fallback to library kernels.
"""

from __future__ import annotations

import decimal
import functools
import math
from dataclasses import dataclass
from typing import Any

import torch
import torch.nn.functional as F
from torch.autograd import forward_ad

from . import kernels


def rope_table(seq_len: int, head_dim: int, theta: float, device: torch.device | str) -> torch.Tensor:
    """``[seq_len, head_dim/2, 2]`` fp32 table of (cos, sin) for the rotate-half RoPE convention."""
    half = head_dim // 2
    inv_freq = 1.0 / (theta ** (torch.arange(0, half, dtype=torch.float64) * 2.0 / head_dim))
    ang = torch.arange(seq_len, dtype=torch.float64)[:, None] * inv_freq[None, :]
    return torch.stack([ang.cos(), ang.sin()], dim=-1).to(torch.float32).to(device).contiguous()


@dataclass(frozen=True)
class LayerDims:
    batch: int
    seq: int
    n_heads: int
    n_kv_heads: int
    head_dim: int
    eps: float


# ------------------------------------------------------------------------------------- helpers
def _sink(p: torch.Tensor) -> Any:
    return getattr(p, "_yf_grad_sink", None)


def fuse_adjacent(ts: list[torch.Tensor]) -> torch.Tensor:
    """One ``[sum(rows), cols]`` view over 2-D tensors that sit back to back in memory (consecutive
    parameters of a flat group buffer); a concatenated copy otherwise."""
    fused = _adjacent_view(ts)
    return torch.cat([t.detach() for t in ts], dim=0) if fused is None else fused


def fuse_rows(ts: list[torch.Tensor]) -> "torch.Tensor | list[torch.Tensor]":
    """The same matrix for :func:`_gemm_fused`, which takes weights that do not sit back to back as they are (parameters
    of a module that ``fully_shard`` does not manage)."""
    fused = _adjacent_view(ts)
    if fused is not None:
        return fused
    parts = [t.detach() for t in ts]
    return parts if kernels.can_be_parts(parts) else torch.cat(parts, dim=0)


def _adjacent_view(ts: list[torch.Tensor]) -> torch.Tensor | None:
    first = ts[0]
    cols = first.shape[1]
    adjacent = all(t.is_contiguous() and t.shape[1] == cols and t.dtype == first.dtype for t in ts)
    if adjacent:
        base = first.untyped_storage().data_ptr()
        end = first.data_ptr() + first.numel() * first.element_size()
        for t in ts[1:]:
            # back to back AND inside one allocation (two allocator blocks can touch by accident)
            if t.data_ptr() != end or t.untyped_storage().data_ptr() != base:
                adjacent = False
                break
            end += t.numel() * t.element_size()
    if not adjacent:
        return None
    rows = sum(t.shape[0] for t in ts)
    return torch.as_strided(first.detach(), (rows, cols), (cols, 1))


def _gemm_fused(a: torch.Tensor, w: "torch.Tensor | list[torch.Tensor]", b_mn_major: bool = False) -> torch.Tensor:
    if isinstance(w, list):
        return kernels.gemm_parts(a, w, b_mn_major=b_mn_major)
    return kernels.gemm(a, w, b_mn_major=b_mn_major)


class _WeightGrad:
    """Where the gradient of one (possibly fused) weight goes: the fp32 sinks of the parameters when all
    of them have one and they are adjacent, else a fresh bf16 tensor split per parameter."""

    def __init__(self, params: list[torch.Tensor]):
        self.params = params
        self.sinks = [_sink(p) for p in params]
        self.use_sinks = all(s is not None for s in self.sinks)

    def run(self, dy: torch.Tensor, x: torch.Tensor, deferred: "list[tuple[Any, ...]] | None" = None,
            scale: torch.Tensor | None = None) -> list[torch.Tensor | None]:
        """dW = dy^T x (times ``scale``, one fp32 value on the device) for the fused weight; returns per-parameter gradients
        (None when sunk).  ``deferred``: in push mode the GEMM is not launched but recorded there, for one grouped launch at
        the end of the layer's backward (:func:`flush_pushed`)."""
        if self.use_sinks and all(s.pushes() for s in self.sinks):
            if scale is not None:
                x = x * scale.to(x.dtype)
            # fused GEMM -> reduce-scatter: parameters that follow each other in the flat gradient are one GEMM
            i, r0 = 0, 0
            while i < len(self.sinks):
                ptrs, off, shard, rank, world, bf16 = self.sinks[i].begin_push()
                rows, nxt, j = self.params[i].shape[0], off + self.params[i].numel(), i + 1
                while j < len(self.sinks) and self.sinks[j].group is self.sinks[i].group:
                    _, off_j, *_ = self.sinks[j].begin_push()
                    assert off_j == nxt, "fused weights must be adjacent in the flat layout"
                    rows, nxt, j = rows + self.params[j].shape[0], nxt + self.params[j].numel(), j + 1
                if deferred is not None:
                    deferred.append((dy[:, r0 : r0 + rows], x, off, ptrs, shard, rank, world, bf16))
                else:
                    kernels.gemm_scatter(dy[:, r0 : r0 + rows], x, a_mn_major=True, b_mn_major=True, peer_grad=ptrs, c_flat_off=off,
                                         shard_numel=shard, rank=rank, world=world, wire_bf16=bf16)
                i, r0 = j, r0 + rows
            return [None] * len(self.params)
        if self.use_sinks and all(s.local_ok for s in self.sinks):
            views, accs = zip(*[s.begin() for s in self.sinks])
            fused = fuse_adjacent(list(views)) if len(views) > 1 else views[0]
            targets = [s.norm_target(acc) for s, acc in zip(self.sinks, accs)]
            if len(views) == 1 or (fused.data_ptr() == views[0].data_ptr() and len(set(accs)) == 1):
                kernels.gemm(dy, x, a_mn_major=True, b_mn_major=True, out=fused, accumulate=accs[0], sumsq=targets[0], alpha_tensor=scale)
            else:
                r0 = 0
                for v, acc, tgt in zip(views, accs, targets):
                    kernels.gemm(dy[:, r0 : r0 + v.shape[0]], x, a_mn_major=True, b_mn_major=True, out=v, accumulate=acc, sumsq=tgt,
                                 alpha_tensor=scale)
                    r0 += v.shape[0]
            return [None] * len(self.params)
        dw = kernels.gemm(dy, x, a_mn_major=True, b_mn_major=True, alpha_tensor=scale)
        out: list[torch.Tensor | None] = []
        r0 = 0
        for p in self.params:
            out.append(dw[r0 : r0 + p.shape[0]])
            r0 += p.shape[0]
        return out


def flush_pushed(deferred: "list[tuple[Any, ...]]") -> None:
    """Launch the recorded weight-gradient GEMMs of a layer: one grouped launch (owners' tiles dealt round-robin) when they share the token
    dimension and the destination (the usual case), one launch each otherwise."""
    if not deferred:
        return
    deferred.sort(key=lambda d: d[2])
    _, _, _, ptrs, shard, rank, world, bf16 = deferred[0]
    same = all(d[3] is ptrs and d[0].shape[0] == deferred[0][0].shape[0] for d in deferred)
    if same and len(deferred) <= 4:
        kernels.gemm_scatter_grouped([(dy, x, off) for dy, x, off, *_ in deferred], peer_grad=ptrs, shard_numel=shard, rank=rank, world=world,
                                     wire_bf16=bf16)
    else:
        for dy, x, off, p, sh, r, w, b16 in deferred:
            kernels.gemm_scatter(dy, x, a_mn_major=True, b_mn_major=True, peer_grad=p, c_flat_off=off, shard_numel=sh, rank=r, world=w,
                                 wire_bf16=b16)
    deferred.clear()


def _norm_weight_grad(w: torch.Tensor, fn: Any, self_zeroing: bool = True) -> torch.Tensor | None:
    """Run ``fn(dw_fp32, zero, target)``, a kernel that accumulates into ``dw_fp32``; returns the gradient unless sunk.  ``zero``: the
    kernel is to clear ``dw_fp32`` first (with ``self_zeroing`` only; else it starts from zeros already).  ``target``: where the
    kernel adds the squares of the gradient, or ``None``; given only where the gradient starts from zeros and is final."""
    s = _sink(w)
    if s is not None and not s.pushes() and s.local_ok:
        zeroed_now = not s.would_accumulate()
        view, _ = s.begin(zero=not self_zeroing)
        fn(view, zeroed_now and self_zeroing, s.norm_target(not zeroed_now))
        return None
    dw = (torch.empty if self_zeroing else torch.zeros)(w.shape, device=w.device, dtype=torch.float32)
    fn(dw, self_zeroing, None)
    if s is not None and s.pushes():
        s.push_from(dw)
        return None
    return dw.to(w.dtype)


def _c(t: torch.Tensor) -> torch.Tensor:
    return t if t.is_contiguous() else t.contiguous()


# ------------------------------------------------------------------------------------- embedding
class EmbeddingFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx: Any, ids: torch.Tensor, table: torch.Tensor) -> torch.Tensor:  # type: ignore[override]
        ctx.save_for_backward(ids)
        ctx.table = table
        return kernels.embedding_fwd(table.detach(), ids.reshape(-1)).view(*ids.shape, table.shape[1])

    @staticmethod
    def backward(ctx: Any, dout: torch.Tensor) -> Any:  # type: ignore[override]
        (ids,) = ctx.saved_tensors
        table = ctx.table
        dout2 = _c(dout).view(-1, table.shape[1])
        grad = _norm_weight_grad(table, lambda dw, _, sq: kernels.embedding_bwd_(dout2, ids.reshape(-1), dw, sq), self_zeroing=False)
        return None, grad


def embedding(ids: torch.Tensor, table: torch.Tensor) -> torch.Tensor:
    if table.is_cuda:
        return EmbeddingFn.apply(ids, table)
    return F.embedding(ids, table)


# ------------------------------------------------------------------------------------- decoder layer
class DecoderLayerFn(torch.autograd.Function):
    """x -> x + Attn(RMSNorm(x)) -> h + MLP(RMSNorm(h)); tokens flattened to ``[B*S, d]``."""

    @staticmethod
    def forward(ctx: Any, x: torch.Tensor, w_n1: torch.Tensor, wq: torch.Tensor, wk: torch.Tensor, wv: torch.Tensor,  # type: ignore[override]
                wo: torch.Tensor, w_n2: torch.Tensor, wg: torch.Tensor, wu: torch.Tensor, wd: torch.Tensor,
                cos_sin: torch.Tensor, dims: LayerDims, keep: bool = True) -> torch.Tensor:
        """``keep``: the values that the backward pass reads are wanted."""
        x = _c(x)
        hd, hq, hkv = dims.head_dim, dims.n_heads, dims.n_kv_heads
        w_qkv = fuse_rows([wq, wk, wv])
        n1, rstd1 = kernels.rmsnorm_fwd(x, w_n1.detach(), dims.eps)
        owner = getattr(wq, "_yf_group_index", None)
        ticket = owner[0].take_in_kernel_gather(owner[1], wq.shape[0] + wk.shape[0] + wv.shape[0]) if owner is not None else None
        if ticket is not None:
            assert isinstance(w_qkv, torch.Tensor)  # views of one gather buffer
            # this forward pass has not gathered the layer: the QKV GEMM pulls it from the peers while it computes
            qkv = kernels.gemm_gathered(n1, w_qkv.shape[0], w_qkv.shape[1], peer_in=ticket["peer_in"], layer_buf=ticket["layer_buf"],
                                        shard_bytes=ticket["shard_bytes"], b_byte_off=ticket["b_byte_off"], rank=ticket["rank"],
                                        world=ticket["world"], counters=ticket["counters"], epoch=ticket["epoch"])
        else:
            qkv = _gemm_fused(n1, w_qkv)
        kernels.rope_(qkv, cos_sin, dims.seq, 0, hq + hkv, hd)
        q, k, v = qkv[:, : hq * hd], qkv[:, hq * hd : (hq + hkv) * hd], qkv[:, (hq + hkv) * hd :]
        att, lse = kernels.attn_fwd(q, k, v, dims.batch, dims.seq, hq, hkv, 1.0 / math.sqrt(hd), True)
        h = kernels.gemm(att, wo.detach(), residual=x)  # x + attention block: the residual is added in the GEMM's epilogue
        n2, rstd2 = kernels.rmsnorm_fwd(h, w_n2.detach(), dims.eps)
        t, d, f = n2.shape[0], n2.shape[1], wg.shape[0]
        if kernels.swiglu_pays(t, f, d, n2.device.index) and kernels.can_fuse_swiglu(wg, wu):
            gu, a = kernels.gemm_swiglu(n2, wg.detach(), wu.detach(), keep_gu=keep)
        else:
            gu = _gemm_fused(n2, fuse_rows([wg, wu]))
            a = kernels.swiglu_fwd(gu)
        out = kernels.gemm(a, wd.detach(), residual=h)
        if keep:
            ctx.save_for_backward(x, rstd1, n1, qkv, att, lse, h, rstd2, n2, gu, a, cos_sin)
        ctx.weights = (w_n1, wq, wk, wv, wo, w_n2, wg, wu, wd)
        ctx.dims = dims
        return out

    @staticmethod
    def backward(ctx: Any, dout: torch.Tensor) -> Any:  # type: ignore[override]
        x, rstd1, n1, qkv, att, lse, h, rstd2, n2, gu, a, cos_sin = ctx.saved_tensors
        w_n1, wq, wk, wv, wo, w_n2, wg, wu, wd = ctx.weights
        dims: LayerDims = ctx.dims
        hd, hq, hkv = dims.head_dim, dims.n_heads, dims.n_kv_heads
        dout = _c(dout)
        # the weights are views of a rotating gather buffer: read them now, as gathered for this backward
        w_qkv = fuse_rows([wq, wk, wv])
        w_gu = fuse_rows([wg, wu])
        # ---- MLP
        pushed: list[tuple[Any, ...]] = []  # push mode: the four weight-gradient GEMMs run as one grouped launch at the end
        da = kernels.gemm(dout, wd.detach(), b_mn_major=True)
        (g_wd,) = _WeightGrad([wd]).run(dout, a, pushed)
        dgu = kernels.swiglu_bwd(gu, da)
        del da
        dn2 = _gemm_fused(dgu, w_gu, b_mn_major=True)
        g_wg, g_wu = _WeightGrad([wg, wu]).run(dgu, n2, pushed)
        del dgu
        box: list[torch.Tensor] = []
        g_n2 = _norm_weight_grad(w_n2, lambda dw, z, sq: box.append(kernels.rmsnorm_bwd(h, w_n2.detach(), dn2, rstd2, dw, dres=dout, zero_dw=z, sumsq=sq)))
        dh = box.pop()
        # ---- attention
        datt = kernels.gemm(dh, wo.detach(), b_mn_major=True)
        (g_wo,) = _WeightGrad([wo]).run(dh, att, pushed)
        dqkv = torch.empty_like(qkv)
        # the attention kernels turn dq and dk back themselves, given a table that 16-byte loads can read
        rotates = cos_sin.is_contiguous() and cos_sin.numel() >= dims.seq * hd and cos_sin.data_ptr() % 16 == 0
        q, k, v = qkv[:, : hq * hd], qkv[:, hq * hd : (hq + hkv) * hd], qkv[:, (hq + hkv) * hd :]
        kernels.attn_bwd(q, k, v, att, datt, lse, dqkv[:, : hq * hd], dqkv[:, hq * hd : (hq + hkv) * hd],
                         dqkv[:, (hq + hkv) * hd :], dims.batch, dims.seq, hq, hkv, 1.0 / math.sqrt(hd), True,
                         rope=cos_sin if rotates else None)
        if not rotates:
            kernels.rope_(dqkv, cos_sin, dims.seq, 0, hq + hkv, hd, backward=True)
        dn1 = _gemm_fused(dqkv, w_qkv, b_mn_major=True)
        g_wq, g_wk, g_wv = _WeightGrad([wq, wk, wv]).run(dqkv, n1, pushed)
        g_n1 = _norm_weight_grad(w_n1, lambda dw, z, sq: box.append(kernels.rmsnorm_bwd(x, w_n1.detach(), dn1, rstd1, dw, dres=dh, zero_dw=z, sumsq=sq)))
        dx = box.pop()
        flush_pushed(pushed)
        return dx, g_n1, g_wq, g_wk, g_wv, g_wo, g_n2, g_wg, g_wu, g_wd, None, None, None


# ------------------------------------------------------------------------------------- final norm + head + loss
class HeadLossFn(torch.autograd.Function):
    """mean cross-entropy of ``lm_head(RMSNorm(h))`` against ``labels`` (``-100`` rows ignored).  The logits are
    overwritten by their own gradient in the forward pass, so the ``[T, vocab]`` tensor exists once."""

    @staticmethod
    def forward(ctx: Any, h: torch.Tensor, w_norm: torch.Tensor, w_head: torch.Tensor, labels: torch.Tensor, eps: float) -> torch.Tensor:  # type: ignore[override]
        h = _c(h)
        n, rstd = kernels.rmsnorm_fwd(h, w_norm.detach(), eps)
        logits = kernels.gemm(n, w_head.detach())
        # the mean's 1 / (number of valid labels) goes into the gradient that the loss kernel leaves in place of the logits
        labels = _c(labels)
        inv_valid = kernels.inv_valid_labels(labels)
        loss_rows = kernels.cross_entropy_(logits, labels, 1.0, write_grad=True, scale=inv_valid)
        ctx.save_for_backward(h, rstd, n, logits)
        ctx.weights = (w_norm, w_head)
        return kernels.scaled_sum(loss_rows, inv_valid)

    @staticmethod
    def backward(ctx: Any, dloss: torch.Tensor) -> Any:  # type: ignore[override]
        h, rstd, n, dlogits = ctx.saved_tensors
        w_norm, w_head = ctx.weights
        # the incoming gradient of the loss (a device scalar) is a factor of the two products: the GEMMs read it themselves
        scale = dloss.float()
        dn = kernels.gemm(dlogits, w_head.detach(), b_mn_major=True, alpha_tensor=scale)
        (g_head,) = _WeightGrad([w_head]).run(dlogits, n, scale=scale)
        box: list[torch.Tensor] = []
        g_norm = _norm_weight_grad(w_norm, lambda dw, z, sq: box.append(kernels.rmsnorm_bwd(h, w_norm.detach(), dn, rstd, dw, zero_dw=z, sumsq=sq)))
        return box.pop(), g_norm, g_head, None, None


class HeadLogitsFn(torch.autograd.Function):
    """logits = lm_head(RMSNorm(h)) (inference / evaluation path)."""

    @staticmethod
    def forward(ctx: Any, h: torch.Tensor, w_norm: torch.Tensor, w_head: torch.Tensor, eps: float) -> torch.Tensor:  # type: ignore[override]
        h = _c(h)
        n, rstd = kernels.rmsnorm_fwd(h, w_norm.detach(), eps)
        ctx.save_for_backward(h, rstd, n)
        ctx.weights = (w_norm, w_head)
        return kernels.gemm(n, w_head.detach())

    @staticmethod
    def backward(ctx: Any, dlogits: torch.Tensor) -> Any:  # type: ignore[override]
        h, rstd, n = ctx.saved_tensors
        w_norm, w_head = ctx.weights
        dlogits = _c(dlogits)
        dn = kernels.gemm(dlogits, w_head.detach(), b_mn_major=True)
        (g_head,) = _WeightGrad([w_head]).run(dlogits, n)
        box: list[torch.Tensor] = []
        g_norm = _norm_weight_grad(w_norm, lambda dw, z, sq: box.append(kernels.rmsnorm_bwd(h, w_norm.detach(), dn, rstd, dw, zero_dw=z, sumsq=sq)))
        return box.pop(), g_norm, g_head, None


# ------------------------------------------------------------------------------------- CPU restatements
def rmsnorm_ref(x: torch.Tensor, w: torch.Tensor, eps: float) -> torch.Tensor:
    xf = x.float()
    return (xf * torch.rsqrt(xf.pow(2).mean(-1, keepdim=True) + eps)).to(x.dtype) * w


def rope_ref(t: torch.Tensor, cos_sin: torch.Tensor) -> torch.Tensor:
    """t: [B, S, H, D]; rotate-half convention."""
    half = t.shape[-1] // 2
    cos = cos_sin[: t.shape[1], :, 0].view(1, t.shape[1], 1, half).to(torch.float32)
    sin = cos_sin[: t.shape[1], :, 1].view(1, t.shape[1], 1, half).to(torch.float32)
    t1, t2 = t[..., :half].float(), t[..., half:].float()
    return torch.cat([t1 * cos - t2 * sin, t2 * cos + t1 * sin], dim=-1).to(t.dtype)


def decoder_layer_ref(x: torch.Tensor, w_n1: torch.Tensor, wq: torch.Tensor, wk: torch.Tensor, wv: torch.Tensor, wo: torch.Tensor,
                      w_n2: torch.Tensor, wg: torch.Tensor, wu: torch.Tensor, wd: torch.Tensor, cos_sin: torch.Tensor,
                      dims: LayerDims) -> torch.Tensor:
    b, s, hq, hkv, hd = dims.batch, dims.seq, dims.n_heads, dims.n_kv_heads, dims.head_dim
    n1 = rmsnorm_ref(x, w_n1, dims.eps)
    q = F.linear(n1, wq).view(b, s, hq, hd)
    k = F.linear(n1, wk).view(b, s, hkv, hd)
    v = F.linear(n1, wv).view(b, s, hkv, hd)
    q, k = rope_ref(q, cos_sin), rope_ref(k, cos_sin)
    att = F.scaled_dot_product_attention(q.transpose(1, 2), k.transpose(1, 2), v.transpose(1, 2), is_causal=True,
                                         enable_gqa=hq != hkv)
    att = att.transpose(1, 2).reshape(b * s, hq * hd)
    h = x + F.linear(att, wo)
    n2 = rmsnorm_ref(h, w_n2, dims.eps)
    return h + F.linear(F.silu(F.linear(n2, wg)) * F.linear(n2, wu), wd)


def decoder_layer(x: torch.Tensor, *weights_and_table: Any) -> torch.Tensor:
    """``x [B*S, d]`` through one decoder layer (arguments as ``DecoderLayerFn.forward``)."""
    if x.is_cuda:
        return DecoderLayerFn.apply(x, *weights_and_table, torch.is_grad_enabled())
    return decoder_layer_ref(x, *weights_and_table)


def shift_labels(labels: torch.Tensor) -> torch.Tensor:
    """``labels [B, S]`` moved one to the left, -100 (ignored) at the end of every row."""
    if labels.is_cuda and labels.dtype == torch.int64 and labels.stride(1) == 1:
        return kernels.shift_labels(labels)
    return torch.cat([labels[:, 1:], labels.new_full((labels.shape[0], 1), -100)], dim=1)


def head_loss(h: torch.Tensor, w_norm: torch.Tensor, w_head: torch.Tensor, labels: torch.Tensor, eps: float) -> torch.Tensor:
    if h.is_cuda:
        return HeadLossFn.apply(h, w_norm, w_head, labels, eps)
    logits = F.linear(rmsnorm_ref(h, w_norm, eps), w_head)
    return F.cross_entropy(logits.float(), labels, ignore_index=-100)


def head_logits(h: torch.Tensor, w_norm: torch.Tensor, w_head: torch.Tensor, eps: float) -> torch.Tensor:
    if h.is_cuda:
        return HeadLogitsFn.apply(h, w_norm, w_head, eps)
    return F.linear(rmsnorm_ref(h, w_norm, eps), w_head)


# ------------------------------------------------------------------------------------- packed documents
def _device_of(what: str, first: torch.Tensor, *others: torch.Tensor | None) -> bool:
    """Whether the tensors, which must share a device, are on the current CUDA device (then kernels can be launched) or on the CPU."""
    dev = first.device
    for t in others:
        if t is not None and t.device != dev:
            raise ValueError(f"{what}: tensors on {dev} and on {t.device}")
    return dev.type != "cuda" or dev.index == torch._C._cuda_getDevice()


def _tangents() -> bool:
    """Whether tensors may carry forward-mode tangents, which only an autograd function refuses: a kernel reads their values alone."""
    return forward_ad._current_level >= 0


class _RefuseDerivative(torch.autograd.Function):
    """Passes on ``n`` tensors; a derivative of them with respect to the others is refused."""

    @staticmethod
    def forward(ctx: Any, n: int, *tensors: torch.Tensor | None) -> Any:  # type: ignore[override]
        return tuple(None if t is None else t.view_as(t) for t in tensors[:n])

    @staticmethod
    def backward(ctx: Any, *grads: torch.Tensor | None) -> Any:  # type: ignore[override]
        raise RuntimeError("the gradients of these kernels have no derivative: they can be differentiated once only")


def _once(backward: Any) -> Any:
    """A ``backward(ctx, saved, *grads)`` whose results cannot be differentiated, neither through the incoming gradients nor through what was
    saved.  (``once_differentiable`` sees incoming gradients with a history only, and its error is left out where ``torch.autograd.grad``
    is asked for tensors that the loss reaches on another way too: the derivative would be lost.)"""

    @functools.wraps(backward)
    def once(ctx: Any, *grads: torch.Tensor | None) -> Any:
        saved = ctx.saved_tensors
        if not torch.is_grad_enabled():
            return backward(ctx, saved, *grads)
        with torch.no_grad():
            out = backward(ctx, saved, *grads)
        return _RefuseDerivative.apply(len(out), *out, *saved, *grads)

    return once


@dataclass(frozen=True)
class DocumentMask:
    """Which tokens of a packed batch see each other (:func:`document_mask`): query ``i`` of a row sees the keys ``spans[i, 0] <= j <
    spans[i, 1]``, key ``j`` is seen by the queries ``key_spans[j, 0] <= i < key_spans[j, 1]``.  ``positions``: index of a token in its
    document.  ``padding``: padded tokens in every 128 of a row.  Neither end of
    a span moves back along a row, and both views say the same: the kernels rely on it.  What a span has beyond the row counts for nothing."""

    spans: torch.Tensor  # [B, S, 2] int32
    key_spans: torch.Tensor  # [B, S, 2] int32
    positions: torch.Tensor  # [B, S] int32
    padding: torch.Tensor  # [B, ceil(S / 128)] int32

    def __post_init__(self) -> None:
        parts = (self.positions, self.padding, self.spans, self.key_spans)
        pos = self.positions
        b, s = pos.shape if pos.dim() == 2 else (-1, -1)
        if self.spans.shape != (b, s, 2) or self.key_spans.shape != (b, s, 2) or self.padding.shape != (b, (s + 127) // 128):
            raise ValueError(f"DocumentMask: spans and key_spans [B, S, 2], positions [B, S], padding [B, ceil(S / 128)] expected, got {[list(t.shape) for t in parts[2:] + parts[:2]]}")
        for t in parts:
            if t.dtype != torch.int32 or t.device != pos.device or not t.is_contiguous():
                raise ValueError("DocumentMask: int32 tensors without gaps on one device expected")


def document_mask(document_ids: torch.Tensor, prefix: torch.Tensor | None = None, window: int = 0) -> DocumentMask:
    """The mask of packed rows ``document_ids [B, S]`` (int32 or int64).  Tokens see each other inside a document, which is a run of equal ids
    >= 0, and causally; negative ids are padding, which sees and is seen by nothing.  ``prefix [B, S]`` (bool): the flagged tokens
    that a document starts with also see each other backwards.  ``window``: keys ``window`` or more tokens back are hidden (0: none are)."""
    if document_ids.dim() != 2 or document_ids.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"document_mask: document_ids must be [B, S] int32 or int64, got {list(document_ids.shape)} {document_ids.dtype}")
    if prefix is not None and (prefix.shape != document_ids.shape or prefix.dtype != torch.bool):
        raise ValueError(f"document_mask: prefix must be bool {list(document_ids.shape)}, got {list(prefix.shape)} {prefix.dtype}")
    if not 0 <= window < 1 << 31:
        raise ValueError(f"document_mask: window must be at least 0 and below 2^31, got {window}")
    if document_ids.shape[0] > 65535 or document_ids.shape[1] > 1 << 30:
        raise ValueError(f"document_mask: at most 65535 rows of at most 2^30 tokens, got {list(document_ids.shape)}")
    here = _device_of("document_mask", document_ids, prefix)
    if not document_ids.is_cuda:
        return _document_mask_ref(document_ids, prefix, window)
    if not here:
        with torch.cuda.device(document_ids.device):
            return document_mask(document_ids, prefix, window)
    if document_ids.shape[1] > 1:
        if document_ids.stride(1) != 1:
            document_ids = document_ids.contiguous()
        if prefix is not None and prefix.stride(1) != 1:
            prefix = prefix.contiguous()
    return DocumentMask(*kernels.document_mask(document_ids, prefix, window))


def _document_mask_ref(ids: torch.Tensor, prefix: torch.Tensor | None, window: int) -> DocumentMask:
    b, s = ids.shape
    at = torch.arange(s, device=ids.device).expand(b, s)
    if b * s == 0:
        empty = ids.new_zeros((b, s, 2), dtype=torch.int32)
        return DocumentMask(empty, empty.clone(), ids.new_zeros((b, s), dtype=torch.int32), ids.new_zeros((b, (s + 127) // 128), dtype=torch.int32))
    starts = torch.cat([ids.new_ones((b, 1), dtype=torch.bool), ids[:, 1:] != ids[:, :-1]], 1)
    start = torch.where(starts, at, 0).cummax(1).values
    end = torch.where(starts.roll(-1, 1), at + 1, s).flip(1).cummin(1).values.flip(1)
    lead, run_end = torch.zeros_like(starts), end
    if prefix is not None:
        lead = torch.where(prefix, -1, at).cummax(1).values < start
        run_end = torch.minimum(end, torch.where(prefix, s, at).flip(1).cummin(1).values.flip(1))
    lo, hi = start, torch.where(lead, run_end, at + 1)
    first, stop = torch.where(lead, start, at), end
    if window:
        lo, stop = torch.maximum(lo, at - window + 1), torch.minimum(stop, at + window)
    pad = ids < 0
    lo, hi, first, stop = (torch.where(pad, at, t) for t in (lo, hi, first, stop))
    padding = F.pad(pad, (0, -s % 128)).view(b, -1, 128).sum(2)
    return DocumentMask(torch.stack([lo, hi], -1).int(), torch.stack([first, stop], -1).int(), torch.where(pad, 0, at - start).int(), padding.int())


_PI = decimal.Decimal("3.14159265358979323846264338327950288419716939937510582097494459230781640628620899862803")


class RotaryAxes:
    """Frequencies of rotary positions with one or several axes.  Pair ``j`` of a head (dims ``j`` and ``j + head_dim / 2``) turns by
    ``positions[axis of j] * theta ** (-2 j / head_dim)``.  ``sections``: how many pairs follow each axis (their sum is ``head_dim / 2``; one
    axis by default).  The pairs of an axis lie side by side, or, with ``interleaved``, are dealt to the axes in turn as long as an
    axis has pairs left."""

    def __init__(self, head_dim: int, theta: float, sections: "tuple[int, ...] | None" = None, interleaved: bool = False):
        if head_dim <= 0 or head_dim % 16 or head_dim > 512:
            raise ValueError(f"RotaryAxes: head_dim must be a multiple of 16 up to 512, got {head_dim}")
        if not theta > 0:
            raise ValueError(f"RotaryAxes: theta must be positive, got {theta}")
        half = head_dim // 2
        self.sections = (half,) if sections is None else tuple(sections)
        if any(n < 0 for n in self.sections) or sum(self.sections) != half:
            raise ValueError(f"RotaryAxes: sections must add up to head_dim / 2 = {half}, got {self.sections}")
        self.head_dim, self.theta = head_dim, theta
        self.axis = [a for a, n in enumerate(self.sections) for _ in range(n)]
        if interleaved:
            left, self.axis = list(self.sections), []
            while any(left):
                for a in range(len(left)):
                    if left[a]:
                        left[a] -= 1
                        self.axis.append(a)
        self.frequency = [theta ** (-2.0 * j / head_dim) for j in range(half)]
        base = decimal.Decimal(float(theta))
        # in turns of 2^-64, from more than the 53 bits of a float: far positions multiply what is missing
        with decimal.localcontext(decimal.Context(prec=60 + max(0, -base.adjusted()))):
            turn, ratio = decimal.Decimal(2) ** 64 / (2 * _PI), base ** (decimal.Decimal(-2) / head_dim)
            self._turns: list[int] = []
            for _ in range(half):
                self._turns.append(int(turn.to_integral_value()) % 2**64)
                turn *= ratio
        self._tables: dict[torch.device, torch.Tensor] = {}

    def table(self, device: torch.device | str) -> torch.Tensor:
        """``[head_dim / 2, 2]`` int64: the fraction of a turn per position in 2^-64, and the axis.  Made once per device, outside of graph
        captures."""
        device = torch.device(device)
        if device.type == "cuda" and device.index is None:  # what a tensor's device says
            device = torch.device("cuda", torch.cuda.current_device())
        t = self._tables.get(device)
        if t is None:
            if device.type == "cuda" and torch.cuda.is_current_stream_capturing():
                raise RuntimeError("RotaryAxes: call rotary() or table() on this device once before capturing a graph")
            with torch.inference_mode(False):  # a later call may save it for its backward pass
                t = torch.tensor([[f - 2**64 if f >= 2**63 else f, a] for f, a in zip(self._turns, self.axis)], dtype=torch.int64, device="cpu").to(device)
            self._tables[device] = t
        return t


class RotaryFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx: Any, q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor, table: torch.Tensor) -> Any:  # type: ignore[override]
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(positions, table)
        return kernels.rotary(q, k, positions, table)

    @staticmethod
    @_once
    def backward(ctx: Any, saved: Any, dq: torch.Tensor | None, dk: torch.Tensor | None) -> Any:  # type: ignore[override]
        if dq is None and dk is None:
            return None, None, None, None
        return *kernels.rotary(dq, dk, *saved, backward=True), None, None


def rotary(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor, axes: RotaryAxes) -> tuple[torch.Tensor, torch.Tensor]:
    """``q [B, S, Hq, D]`` and ``k [B, S, Hk, D]`` (bf16, fp16 or fp32) turned by ``positions`` (int32 or int64): ``[B, S]`` for one axis, else
    ``[axes, B, S]``.  Angles are exact to 2^-32 of a turn at positions of up to 2^32 in size,
    beyond that to 2^-65 of a turn for each position; cosines and sines are fp32."""
    if q.dim() != 4 or k.dim() != 4 or q.shape[:2] != k.shape[:2] or q.shape[3] != axes.head_dim or k.shape[3] != axes.head_dim:
        raise ValueError(f"rotary: q and k must be [B, S, heads, {axes.head_dim}] of the same batch, got {list(q.shape)} and {list(k.shape)}")
    if q.dtype != k.dtype or q.dtype not in kernels._DTYPES:
        raise TypeError(f"rotary: q and k must both be bf16, fp16 or fp32, got {q.dtype} and {k.dtype}")
    n, tokens = len(axes.sections), q.shape[:2]
    if positions.dtype not in (torch.int32, torch.int64) or (positions.shape != (n, *tokens) and not (n == 1 and positions.shape == tokens)):
        raise ValueError(f"rotary: positions must be int32 or int64 {[n, *tokens]}, got {list(positions.shape)} {positions.dtype}")
    here = _device_of("rotary", q, k, positions)
    if not q.is_cuda:
        return _rotary_ref(q, positions, axes), _rotary_ref(k, positions, axes)
    if not here:
        with torch.cuda.device(q.device):
            return rotary(q, k, positions, axes)
    positions, table = positions.contiguous(), axes.table(q.device)
    if (torch.is_grad_enabled() and (q.requires_grad or k.requires_grad)) or _tangents():
        return RotaryFn.apply(q, k, positions, table)  # type: ignore[no-any-return]
    return kernels.rotary(q, k, positions, table)  # type: ignore[return-value]


def _rotary_ref(t: torch.Tensor, positions: torch.Tensor, axes: RotaryAxes) -> torch.Tensor:
    pos = positions.reshape(-1, *t.shape[:2])[axes.axis].permute(1, 2, 0).long()
    ang = (pos * axes.table(t.device)[:, 0]).double() * (2.0 * math.pi / 2.0**64)  # modulo a whole turn
    cos, sin = ang.cos().float().unsqueeze(2), ang.sin().float().unsqueeze(2)
    a, b = t.float().chunk(2, dim=-1)
    return torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1).to(t.dtype)


# ------------------------------------------------------------------------------------- attention with masks, capped scores and a distance bias
class AttentionFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx: Any, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, mask: DocumentMask | None, scale: float, softcap: float,  # type: ignore[override]
                slopes: torch.Tensor | None) -> torch.Tensor:
        spans, key_spans, padding = (None, None, None) if mask is None else (mask.spans, mask.key_spans, mask.padding)
        out, out_lo, lse = kernels.attn_fwd_mods(q, k, v, scale, softcap, slopes, spans, padding)
        ctx.save_for_backward(q, k, v, out, out_lo, lse, slopes, spans, key_spans, padding)
        ctx.args = (scale, softcap)
        return out

    @staticmethod
    @_once
    def backward(ctx: Any, saved: Any, dout: torch.Tensor) -> Any:  # type: ignore[override]
        q, k, v, out, out_lo, lse, slopes, spans, key_spans, padding = saved
        return *kernels.attn_bwd_mods(q, k, v, out, out_lo, dout, lse, *ctx.args, slopes, spans, key_spans, padding), None, None, None, None


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, mask: DocumentMask | None = None, *, scale: float | None = None, softcap: float = 0.0,
              slopes: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of ``q [B, S, Hq, D]`` over ``k``, ``v [B, S, Hkv, D]`` (query head ``h`` reads key head ``h // (Hq // Hkv)``), causal or under
    ``mask``; the result has the shape of ``q``, zeros where a token sees nothing.  The score of query ``i`` and key ``j`` is ``t = scale *
    q.k`` (``scale``: ``D ** -0.5``), ``softcap * tanh(t / softcap)`` with a ``softcap``, less ``slopes[h] * |i - j|`` with ``slopes [Hq]``
    (constants: they get no gradient).  On CUDA: bf16, ``D`` = 128; for the backward pass the output is kept in twice its bits.  Tensors whose heads lie side by side in rows at a pitch of
    16 bytes are read in place (parts of a fused projection), others are copied first.  What padding holds does not matter; any other
    value is taken to be finite: an infinity or NaN of one document may reach the documents that share a tile of 128 tokens with it."""
    if q.dim() != 4 or k.dim() != 4 or k.shape != v.shape or q.shape[:2] != k.shape[:2] or q.shape[3] != k.shape[3]:
        raise ValueError(f"attention: q [B, S, Hq, D], k and v [B, S, Hkv, D] expected, got {list(q.shape)}, {list(k.shape)}, {list(v.shape)}")
    if k.shape[2] == 0 or q.shape[2] == 0 or q.shape[2] % k.shape[2]:
        raise ValueError(f"attention: {q.shape[2]} query heads are no multiple of {k.shape[2]} key heads")
    if not q.dtype == k.dtype == v.dtype:
        raise TypeError(f"attention: q, k and v must have one type, got {q.dtype}, {k.dtype}, {v.dtype}")
    scale = q.shape[3] ** -0.5 if scale is None else float(scale)
    softcap = float(softcap)
    if not 1e-12 <= scale <= 1e12 or not (softcap == 0.0 or 1e-12 <= softcap <= 1e12):  # beyond, their squares and ratios leave fp32
        raise ValueError(f"attention: scale must be from 1e-12 to 1e12 and softcap zero or from 1e-12 to 1e12, got {scale} and {softcap}")
    if mask is not None and mask.positions.shape != q.shape[:2]:
        raise ValueError(f"attention: the mask is for {list(mask.positions.shape)} tokens, q has {list(q.shape[:2])}")
    if slopes is not None and slopes.shape != (q.shape[2],):
        raise ValueError(f"attention: slopes must have one value for each of {q.shape[2]} query heads, got {list(slopes.shape)}")
    if slopes is not None and slopes.requires_grad:
        raise ValueError("attention: slopes get no gradient; pass slopes.detach()")
    here = _device_of("attention", q, k, v, slopes, None if mask is None else mask.spans)
    if not q.is_cuda:
        return _attention_ref(q, k, v, mask, scale, softcap, slopes)
    if q.dtype != torch.bfloat16 or q.shape[3] != 128:
        raise TypeError(f"attention: the CUDA kernels take bf16 heads of 128, got {q.dtype} heads of {q.shape[3]}")
    if q.shape[0] > 65535 or q.shape[1] > 1 << 23:
        raise ValueError(f"attention: the CUDA kernels take at most 65535 rows of at most 2^23 tokens, got {list(q.shape[:2])}")
    if not here:
        with torch.cuda.device(q.device):
            return attention(q, k, v, mask, scale=scale, softcap=softcap, slopes=slopes)
    if slopes is not None:
        slopes = _c(slopes.float())
    if (torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad)) or _tangents():
        return AttentionFn.apply(q, k, v, mask, scale, softcap, slopes)  # type: ignore[no-any-return]
    spans, padding = (None, None) if mask is None else (mask.spans, mask.padding)
    return kernels.attn_fwd_mods(q, k, v, scale, softcap, slopes, spans, padding, keep=False)[0]


def _attention_ref(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, mask: DocumentMask | None, scale: float, softcap: float,
                   slopes: torch.Tensor | None) -> torch.Tensor:
    s, group = q.shape[1], q.shape[2] // k.shape[2]
    at = torch.arange(s, device=q.device)
    if mask is None:
        seen = (at[None, :] <= at[:, None])[None]
    else:
        seen = (at >= mask.spans[..., :1]) & (at < mask.spans[..., 1:])
    score = torch.einsum("bihd,bjhd->bhij", q.float(), k.float().repeat_interleave(group, 2)) * scale
    if softcap:
        score = softcap * torch.tanh(score / softcap)
    if slopes is not None:
        score = score - slopes.float()[:, None, None] * (at[:, None] - at[None, :]).abs()
    # a row without keys is given all of them, and zeros afterwards
    some = seen.any(2)[:, None, :, None]
    p = score.masked_fill(~seen[:, None] & some, -math.inf).softmax(-1) * some
    return torch.einsum("bhij,bjhd->bihd", p, v.float().repeat_interleave(group, 2)).to(q.dtype)


# ------------------------------------------------------------------------------------- the residual step between two blocks
class ResidualNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx: Any, x: torch.Tensor, y: torch.Tensor, weight: torch.Tensor, post: torch.Tensor | None, gate: torch.Tensor | None,  # type: ignore[override]
                gate_rows: int, scale: float, eps: float) -> Any:
        ctx.set_materialize_grads(False)
        h, n, rstd = kernels.residual_norm_fwd(x, y, weight, post, gate, gate_rows, scale, eps)
        # the inputs themselves, as torch's own layers do: the values of a sharded parameter are gathered anew for the backward pass
        ctx.save_for_backward(x, y, weight, post, gate, rstd)
        ctx.params = (weight, post)  # as parameters of a group they know where their gradients go
        ctx.args = (gate_rows, scale)
        return h, n

    @staticmethod
    @_once
    def backward(ctx: Any, saved: Any, dh: torch.Tensor | None, dn: torch.Tensor | None) -> Any:  # type: ignore[override]
        if dh is None and dn is None:  # nothing behind this step has a gradient: there is none for its inputs, and no sink is begun
            return (None,) * 8
        x, y, w, p, g, rstd = saved
        gate_rows, scale = ctx.args
        if x.numel() == 0:
            return *(None if t is None else torch.zeros_like(t) for t in (x, y, w, p, g)), None, None, None
        weight, post = ctx.params
        if _sink(weight) is None and (post is None or _sink(post) is None):
            dw, dpost = torch.empty_like(w), None if p is None else torch.empty_like(p)
            dx, dy, dgate = kernels.residual_norm_bwd(x, y, w, p, g, gate_rows, rstd, dh, dn, scale, dw, dpost)
            return dx, dy, dw, dpost, dgate, None, None, None
        a, b = _ParamGrad(weight), None if post is None else _ParamGrad(post)
        if b is None:
            dx, dy, dgate = kernels.residual_norm_bwd(x, y, w, None, g, gate_rows, rstd, dh, dn, scale, a.out, None, add_dw=a.add, dw_sumsq=a.sumsq)
        else:
            dx, dy, dgate = kernels.residual_norm_bwd(x, y, w, p, g, gate_rows, rstd, dh, dn, scale, a.out, b.out, add_dw=a.add, add_dpost=b.add,
                                                      dw_sumsq=a.sumsq, dpost_sumsq=b.sumsq)
        return dx, dy, a.result(), None if b is None else b.result(), dgate, None, None, None


class _ParamGrad:
    """Where a kernel that finishes a whole norm weight gradient in one go writes it: the parameter's fp32 sink when it has one, else a tensor of
    the parameter's type."""

    def __init__(self, p: torch.Tensor):
        self.sink, self.add, self.sumsq = _sink(p), False, None
        self.pushed = self.sink is not None and self.sink.pushes()
        self.sunk = self.sink is not None and not self.pushed and self.sink.local_ok
        if self.sunk:
            self.out, self.add = self.sink.begin()
            self.sumsq = self.sink.norm_target(self.add)
        else:
            self.out = torch.empty(p.shape, device=p.device, dtype=torch.float32 if self.pushed else p.dtype)

    def result(self) -> torch.Tensor | None:
        if self.pushed:
            self.sink.push_from(self.out)
        return None if self.pushed or self.sunk else self.out


def _gate_rows(gate: torch.Tensor, x: torch.Tensor) -> int:
    """How many rows of ``x.shape[-1]`` the gate has, each for as many consecutive tokens."""
    lead = (1,) * (x.dim() - gate.dim()) + tuple(gate.shape[:-1])
    same = 0
    while same < len(lead) and lead[same] == x.shape[same]:
        same += 1
    if gate.dim() == 0 or gate.dim() > x.dim() or gate.shape[-1] != x.shape[-1] or any(n != 1 for n in lead[same:]):
        raise ValueError(f"residual_norm: gate must have the shape of x, {list(x.shape)}, with trailing axes before the last left out or of size one, got {list(gate.shape)}")
    return math.prod(lead)


def residual_norm(x: torch.Tensor, y: torch.Tensor, weight: torch.Tensor, *, post_weight: torch.Tensor | None = None, gate: torch.Tensor | None = None,
                  scale: float = 1.0, eps: float = 1e-5) -> tuple[torch.Tensor, torch.Tensor]:
    """The residual step between two blocks, in one kernel: ``h = x + scale * gate * u``, where ``u`` is the block's output ``y``, normalised
    with ``post_weight`` if that is given, and ``n = rmsnorm(h) * weight``, the input of the next block.  Returns ``(h, n)``.  ``x``, ``y``: ``[...,
    D]``; weights ``[D]``; ``gate``: ``[D]`` for every channel, ``[B, 1, D]`` for every sample of ``[B, S, D]``, or the shape of ``x``.  All of
    one type (bf16, fp16 or fp32); sums are fp32 and each result is rounded once.  ``D``: a multiple of 8 up to 8192, and
    at most 2^31 - 2^20 - 1 rows, on CUDA."""
    if x.dim() < 1 or x.shape != y.shape:
        raise ValueError(f"residual_norm: x and y must have one shape [..., D], got {list(x.shape)} and {list(y.shape)}")
    dtype, others = x.dtype, (y, weight) if post_weight is None else (y, weight, post_weight)
    for t in others[1:]:
        if t.shape != x.shape[-1:]:
            raise ValueError(f"residual_norm: weights must be [{x.shape[-1]}], got {list(t.shape)}")
    if post_weight is weight:  # one launch finishes both gradients, which then have one place to go
        raise ValueError("residual_norm: weight and post_weight must be two tensors")
    if gate is not None:
        others = (*others, gate)
    if dtype not in kernels._DTYPES:
        raise TypeError(f"residual_norm: the type must be bf16, fp16 or fp32, got {dtype}")
    grad = torch.is_grad_enabled()
    wanted = grad and x.requires_grad
    for t in others:
        if t.dtype != dtype:
            raise TypeError(f"residual_norm: all tensors must have one type, got {dtype} and {t.dtype}")
        wanted = wanted or (grad and t.requires_grad)
    scale, eps = float(scale), float(eps)
    if not math.isfinite(scale) or not 0.0 < eps < math.inf:
        raise ValueError(f"residual_norm: scale must be finite and eps positive, got {scale} and {eps}")
    rows = 0 if gate is None else _gate_rows(gate, x)
    here = _device_of("residual_norm", x, *others)
    if not x.is_cuda:
        return _residual_norm_ref(x, y, weight, post_weight, gate, scale, eps)
    if x.shape[-1] % 8 or not 0 < x.shape[-1] <= 8192:
        raise ValueError(f"residual_norm: the CUDA kernels take widths that are multiples of 8 up to 8192, got {x.shape[-1]}")
    if x.numel() // x.shape[-1] > kernels.MAX_NORM_ROWS:
        raise ValueError(f"residual_norm: the CUDA kernels take at most {kernels.MAX_NORM_ROWS} rows, got {x.numel() // x.shape[-1]}")
    if not here:
        with torch.cuda.device(x.device):
            return residual_norm(x, y, weight, post_weight=post_weight, gate=gate, scale=scale, eps=eps)
    if wanted or _tangents():
        return ResidualNormFn.apply(x, y, weight, post_weight, gate, rows, scale, eps)  # type: ignore[no-any-return]
    return kernels.residual_norm_fwd(x, y, weight, post_weight, gate, rows, scale, eps, keep=False)[:2]


def _residual_norm_ref(x: torch.Tensor, y: torch.Tensor, weight: torch.Tensor, post: torch.Tensor | None, gate: torch.Tensor | None, scale: float,
                       eps: float) -> tuple[torch.Tensor, torch.Tensor]:
    u = y.float()
    if post is not None:
        u = u * torch.rsqrt(u.pow(2).mean(-1, keepdim=True) + eps) * post.float()
    if gate is not None:
        u = u * gate.float()
    h = x.float() + scale * u
    n = h * torch.rsqrt(h.pow(2).mean(-1, keepdim=True) + eps) * weight.float()
    return h.to(x.dtype), n.to(x.dtype)
