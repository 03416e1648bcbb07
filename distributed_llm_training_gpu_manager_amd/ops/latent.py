"""Latent attention (kernels: csrc/kernels/shared_attn.hip, csrc/kernels/shared_decode.hip): the keys and values of all
heads come from ONE latent vector ``c`` [r] a token, plus one rope key ``k_rope`` [rope] shared by the heads:

    [k_nope[h] | v[h]] = w_kv[h] c,    k[h] = [k_nope[h] | k_rope],    out[h] = softmax(scale q[h] . k[h]) v[h]

* training (expanded): ``w_kv`` is applied to every token by one dense GEMM and the kernels read its packed rows
  ``kv`` [B, S, H, nope + value]; the rope key is never copied per head. :func:`latent_attention` is the differentiable
  whole, :func:`latent_attn_fwd` / :func:`latent_attn_bwd` the pair that explicit-backward units call.
* one token per sequence (absorbed): :func:`latent_attention_decode` moves ``w_kv`` to the query and the output, so the
  cache holds r + rope values a token whatever the number of heads and is read once.

On the GPU: bf16 or fp16; head dims (nope, rope, value) (128, 64, 128) or (64, 32, 64); r any multiple of 8 in training, 256
or 512 in the single-token form; strided views with 16-byte rows. ``lens`` (int32 [B], values beyond the tensor's length
count as its length): only the first ``lens[b]`` tokens of sequence b exist. What lies behind them may hold anything; their
outputs and gradients are zeros, their log-sum-exp is -inf (:func:`latent_attention` alone reads every row of ``c`` in its
GEMMs, so there they must be finite). A NaN in a live row may reach every other live row of its sequence. CPU tensors take the
fp32 reference below, which refuses what the kernels refuse but for types, head dims and strides.
"""
from __future__ import annotations

import math
from typing import Optional, Tuple

import torch

from .._native import hip_ops, use_native
from .gemm import grad_mm, mm

Lens = Optional[torch.Tensor]


def live_rows(lens: Lens, B: int, S: int, device) -> torch.Tensor:
    """[B, S]: whether token i of sequence b exists."""
    i = torch.arange(S, device=device)
    return (i < (lens.clamp(0, S).unsqueeze(1) if lens is not None else S)).expand(B, S)


def softmax_lse(s: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """Softmax and log-sum-exp over the last axis; a row of nothing but -inf gives zeros and -inf."""
    m = s.amax(-1, keepdim=True) if s.shape[-1] else s.new_full((*s.shape[:-1], 1), float("-inf"))
    m = torch.where(m == float("-inf"), torch.zeros_like(m), m)
    e = torch.exp(s - m)
    t = e.sum(-1, keepdim=True)
    return e / torch.where(t == 0, torch.ones_like(t), t), (m + t.log()).squeeze(-1)


def _dims(q: torch.Tensor, kv: torch.Tensor, k_rope: torch.Tensor) -> Tuple[int, int, int]:
    dr = k_rope.shape[-1]
    dn = q.shape[-1] - dr
    return dn, dr, kv.shape[-1] - dn


def scale_of(q: torch.Tensor, softmax_scale: Optional[float]) -> float:
    scale = softmax_scale if softmax_scale is not None else 1.0 / math.sqrt(q.shape[-1])
    if not 1e-20 <= scale <= 1e20:
        raise ValueError(f"softmax_scale must lie between 1e-20 and 1e20, got {scale}")
    return scale


def check_reference(op: str, fits: bool, tensors: Tuple[torch.Tensor, ...], *lengths: Tuple[Lens, int]) -> None:
    """What the kernels refuse is refused by the reference, too: shapes that would broadcast, mixed types, lengths of another
    type or number."""
    q = tensors[0]
    if not fits:
        raise ValueError(f"{op}: shapes {', '.join(str(tuple(t.shape)) for t in tensors)} do not fit together")
    if any(t.dtype != q.dtype or t.device != q.device for t in tensors):
        raise ValueError(f"{op}: all tensors must share q's device and type")
    for lens, n in lengths:
        if lens is not None and not (lens.dtype == torch.int32 and lens.shape == (n,) and lens.device == q.device):
            raise ValueError(f"{op}: lengths must be an int32 tensor [{n}] on q's device, got {lens.dtype} {tuple(lens.shape)}")


def _check_latent(op, q, kv, k_rope, lens, *outs):
    fits = q.dim() == kv.dim() == 4 and k_rope.dim() == 3 and kv.shape[:3] == q.shape[:3] and k_rope.shape[:2] == q.shape[:2] \
        and 0 <= q.shape[3] - k_rope.shape[2] < kv.shape[3]
    fits = fits and all(t.shape == (*q.shape[:3], _dims(q, kv, k_rope)[2]) for t in outs)
    check_reference(op, fits, (q, kv, k_rope, *outs), (lens, q.shape[0]))


def _ref_parts(q, kv, k_rope, scale, causal, lens):
    """fp32 (or wider) q, k, v, weights and log-sum-exp, head-major; rows past a length are zeros in all of them. Also the
    ways there and back ([B, S, H, ...] -> head-major -> [B, S, H, ...] in q's type), both with zeros past a length."""
    B, S, H, _ = q.shape
    dn, dr, _ = _dims(q, kv, k_rope)
    live = live_rows(lens, B, S, q.device)
    wide = torch.promote_types(q.dtype, torch.float32)
    rows = lambda t: torch.where(live[:, :, None, None], t.to(wide), 0.0).permute(0, 2, 1, 3)  # noqa: E731
    back = lambda t: torch.where(live[:, :, None, None], t.permute(0, 2, 1, 3), 0.0).to(q.dtype).contiguous()  # noqa: E731
    qf, kvf = rows(q), rows(kv)
    kf = torch.cat([kvf[..., :dn], rows(k_rope.unsqueeze(2)).expand(B, H, S, dr)], -1)
    ok = live[:, None, :] & live[:, :, None]
    if causal:
        ok = ok & torch.ones(S, S, dtype=torch.bool, device=q.device).tril()
    p, lse = softmax_lse((torch.matmul(qf, kf.transpose(-1, -2)) * scale).masked_fill(~ok.unsqueeze(1), float("-inf")))
    return qf, kf, kvf[..., dn:], p, lse, rows, back


def latent_attn_fwd(q: torch.Tensor, kv: torch.Tensor, k_rope: torch.Tensor, softmax_scale: Optional[float] = None,
                    causal: bool = True, lens: Lens = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """q [B, S, H, nope + rope], kv [B, S, H, nope + value], k_rope [B, S, rope] -> (out [B, S, H, value] contiguous,
    log-sum-exp fp32 [B, H, S])."""
    scale = scale_of(q, softmax_scale)
    if use_native(q):
        return hip_ops().latent_attn_fwd(q, kv, k_rope, scale, causal, lens)
    _check_latent("latent_attn_fwd", q, kv, k_rope, lens)
    _, _, v, p, lse, _, back = _ref_parts(q, kv, k_rope, scale, causal, lens)
    return back(torch.matmul(p, v)), lse


def latent_attn_bwd(dout: torch.Tensor, q: torch.Tensor, kv: torch.Tensor, k_rope: torch.Tensor, out: torch.Tensor,
                    lse: torch.Tensor, softmax_scale: Optional[float] = None, causal: bool = True,
                    lens: Lens = None) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(dq, dkv, dk_rope), contiguous; dk_rope is summed over the heads in fp32. ``out`` and ``lse`` are the forward's."""
    scale = scale_of(q, softmax_scale)
    if use_native(q):
        return hip_ops().latent_attn_bwd(dout, q, kv, k_rope, out, lse, scale, causal, lens)
    _check_latent("latent_attn_bwd", q, kv, k_rope, lens, dout, out)
    dn = _dims(q, kv, k_rope)[0]
    qf, kf, v, p, _, rows, back = _ref_parts(q, kv, k_rope, scale, causal, lens)
    do, o = rows(dout), rows(out)
    ds = p * (torch.matmul(do, v.transpose(-1, -2)) - (do * o).sum(-1, keepdim=True)) * scale
    dk = torch.matmul(ds.transpose(-1, -2), qf)
    dkv = torch.cat([dk[..., :dn], torch.matmul(p.transpose(-1, -2), do)], -1)
    return back(torch.matmul(ds, kf)), back(dkv), back(dk[..., dn:].sum(1, keepdim=True)).squeeze(2)


def once(grads: Tuple[torch.Tensor, ...], inputs: Tuple[torch.Tensor, ...]) -> Tuple[torch.Tensor, ...]:
    """Gradients recorded for a second differentiation (create_graph) with regard to ``inputs`` raise an error there: no
    kernel has one."""
    if not torch.is_grad_enabled():
        return grads
    args = [g.detach() for g in grads] + list(inputs)
    msg = "a gradient of latent_attention or prefix_attention cannot be differentiated again"
    return tuple(torch._C._functions.DelayedError(msg, len(args))(*args)[:len(grads)])


class LatentAttentionFunction(torch.autograd.Function):
    """Expanded form: kv = c w_kv^T, attention, and in the backward dc = dkv w_kv, dw_kv = dkv^T c. The latent vectors and
    the packed kv rows are saved (kv again costs a GEMM, its rows H (nope + value) values a token)."""

    @staticmethod
    def forward(ctx, q, c, k_rope, w_kv, softmax_scale, causal, lens):
        B, S, H, _ = q.shape
        kv = mm(c.reshape(B * S, c.shape[-1]), w_kv.t()).view(B, S, H, -1)
        out, lse = latent_attn_fwd(q, kv, k_rope, softmax_scale, causal, lens)
        ctx.save_for_backward(q, c, k_rope, w_kv, kv, out, lse, lens)
        ctx.scale, ctx.causal = softmax_scale, causal
        return out

    @staticmethod
    def backward(ctx, dout):
        q, c, k_rope, w_kv, kv, out, lse, lens = ctx.saved_tensors
        dq, dkv, dkr = latent_attn_bwd(dout.contiguous(), q, kv, k_rope, out, lse, ctx.scale, ctx.causal, lens)
        dkv2, c2 = dkv.view(-1, w_kv.shape[0]), c.reshape(-1, c.shape[-1])
        with torch.no_grad():
            dc, dw = mm(dkv2, w_kv).view(c.shape), grad_mm(torch.empty_like(w_kv), dkv2.t(), c2, False)
        return (*once((dq, dc, dkr, dw), (dout, q, c, k_rope, w_kv)), None, None, None)


def latent_attention(q: torch.Tensor, c: torch.Tensor, k_rope: torch.Tensor, w_kv: torch.Tensor,
                     softmax_scale: Optional[float] = None, causal: bool = True, lens: Lens = None) -> torch.Tensor:
    """out [B, S, H, value] of queries q [B, S, H, nope + rope] over latent vectors c [B, S, r], rope keys k_rope [B, S,
    rope] and the up-projection w_kv [H (nope + value), r] (per head: its nope rows, then its value rows). Differentiable in
    q, c, k_rope and w_kv. The GEMMs of w_kv run over every row of c, so rows behind a length must be finite here."""
    B, S, H, d = q.shape
    if c.shape[:2] != (B, S) or k_rope.shape[:2] != (B, S) or w_kv.dim() != 2 or w_kv.shape[1] != c.shape[-1] \
            or w_kv.shape[0] % max(H, 1) or w_kv.shape[0] <= H * (d - k_rope.shape[-1]):
        raise ValueError(f"latent_attention: q {tuple(q.shape)}, c {tuple(c.shape)}, k_rope {tuple(k_rope.shape)} and "
                         f"w_kv {tuple(w_kv.shape)} do not fit together")
    if use_native(q):  # the same composition as one operator each way (csrc/autograd.cpp)
        return hip_ops().latent_attention(q, c, k_rope, w_kv, scale_of(q, softmax_scale), causal, lens)
    return LatentAttentionFunction.apply(q, c, k_rope, w_kv, softmax_scale, causal, lens)


def latent_attention_decode(q: torch.Tensor, cache: torch.Tensor, lens: torch.Tensor, w_kv: torch.Tensor,
                            softmax_scale: Optional[float] = None) -> torch.Tensor:
    """One token per sequence: q [B, H, nope + rope] over cache [B, L, r + rope] (per token the latent vector, then the
    rope key; the token's own row already stored), lens int32 [B] -> out [B, H, value]. A sequence of length 0 gives zeros."""
    scale = scale_of(q, softmax_scale)
    if use_native(q):
        return hip_ops().latent_attn_decode(q, cache, lens, w_kv, scale)
    fits = q.dim() == cache.dim() == 3 and w_kv.dim() == 2 and cache.shape[0] == q.shape[0] and q.shape[1] > 0 \
        and w_kv.shape[0] % q.shape[1] == 0 and 0 <= cache.shape[2] - w_kv.shape[1] <= q.shape[2]
    check_reference("latent_attention_decode", fits, (q, cache, w_kv), (lens, q.shape[0]))
    B, H, d = q.shape
    r, L = w_kv.shape[1], cache.shape[1]
    dn = d - (cache.shape[-1] - r)
    wide = torch.promote_types(q.dtype, torch.float32)
    live = live_rows(lens, B, L, q.device)
    cf, qf, w = torch.where(live.unsqueeze(-1), cache.to(wide), 0.0), q.to(wide), w_kv.to(wide).view(H, -1, r)
    qa = torch.matmul(qf[..., :dn].transpose(0, 1), w[:, :dn]).transpose(0, 1)
    s = torch.matmul(torch.cat([qa, qf[..., dn:]], -1), cf.transpose(1, 2)) * scale
    p, _ = softmax_lse(s.masked_fill(~live.unsqueeze(1), float("-inf")))
    o = torch.matmul(p, cf[..., :r]).transpose(0, 1)
    return torch.matmul(o, w[:, dn:].transpose(1, 2)).transpose(0, 1).to(q.dtype).contiguous()
