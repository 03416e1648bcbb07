"""Attention of a batch whose sequences share a long prefix (kernels: csrc/kernels/shared_attn.hip,
csrc/kernels/shared_decode.hip) -- several answers to one prompt, sampled or trained on as a group. The prefix's keys and
values are stored once per group, [G, P, Hkv, D]; the batch holds B = G n sequences, sequence b belonging to group
b // n. Every query attends to its group's prefix and then (causally) to its own sequence's keys, one softmax over both.

* training: :func:`prefix_attention` (differentiable), :func:`prefix_attn_fwd` / :func:`prefix_attn_bwd` (the pair for
  explicit-backward units). The prefix's gradient is the sum over its group, accumulated in fp32, no atomics.
* one token per sequence: :func:`prefix_attention_decode` stacks a group's queries against the prefix, so it is read once
  for all of them, beside each sequence's own cache.

On the GPU: bf16 or fp16; head dim 64 or 128; Hq a multiple of Hkv; strided views with 16-byte rows. ``lens`` (int32 [B])
and ``prefix_lens`` (int32 [G]) say how many tokens exist (values beyond the tensors' lengths count as those); what lies
behind may hold anything; outputs and gradients there are zeros, the log-sum-exp is -inf. CPU tensors take the fp32 reference.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from .._native import hip_ops, use_native
from .latent import Lens, check_reference, live_rows, once, scale_of, softmax_lse


def _check(q, k, prefix_k):
    B, Hq, Hkv, G = q.shape[0], q.shape[-2], k.shape[2], prefix_k.shape[0]
    if not G or B % G:
        raise ValueError(f"prefix attention: a batch of {B} does not hold equally many sequences of {G} prefixes")
    if not Hkv or Hq % Hkv or prefix_k.shape[2] != Hkv:
        raise ValueError(f"prefix attention: {Hq} q heads, {Hkv} kv heads, {prefix_k.shape[2]} prefix kv heads")


def _check_reference(op, q, k, v, pk, pv, lens, plens, *outs):
    fits = k.dim() == v.dim() == pk.dim() == pv.dim() == 4 and k.shape[0] == q.shape[0] and k.shape[3] == q.shape[-1] \
        and v.shape == k.shape and pk.shape[2:] == k.shape[2:] and pv.shape == pk.shape
    fits = fits and (q.dim() == 3 or q.dim() == 4 and k.shape[1] == q.shape[1]) and all(t.shape == q.shape for t in outs)
    check_reference(op, fits, (q, k, v, pk, pv, *outs), (lens, q.shape[0]), (plens, pk.shape[0]))


def _ref_keys(x, px, lens, plens, rep):
    """[prefix | own] keys (or values) of every sequence and q head, fp32 (or wider): [B, Hq, P + S, D]; zeros past the
    lengths. Also which of them exist, [B, P + S]."""
    B, S = x.shape[:2]
    G, P = px.shape[:2]
    pl = live_rows(plens, G, P, x.device).repeat_interleave(B // G, 0)
    live = torch.cat([pl, live_rows(lens, B, S, x.device)], 1)
    both = torch.cat([px.repeat_interleave(B // G, 0), x], 1).to(torch.promote_types(x.dtype, torch.float32))
    both = torch.where(live[:, :, None, None], both, 0.0)
    return both.permute(0, 2, 1, 3).repeat_interleave(rep, 1), live


def _ref_parts(q, k, v, pk, pv, scale, causal, lens, plens):
    B, S, Hq, _ = q.shape
    P, rep = pk.shape[1], Hq // k.shape[2]
    kf, live = _ref_keys(k, pk, lens, plens, rep)
    vf, _ = _ref_keys(v, pv, lens, plens, rep)
    row = live_rows(lens, B, S, q.device)
    rows = lambda t: torch.where(row[:, :, None, None], t.to(kf.dtype), 0.0).permute(0, 2, 1, 3)  # noqa: E731
    back = lambda t: torch.where(row[:, :, None, None], t.permute(0, 2, 1, 3), 0.0).to(q.dtype).contiguous()  # noqa: E731
    qf = rows(q)
    ok = live[:, None, :] & row[:, :, None]
    if causal:
        own = torch.ones(S, S, dtype=torch.bool, device=q.device).tril()
        ok = ok & torch.cat([own.new_ones(S, P), own], 1)
    p, lse = softmax_lse((torch.matmul(qf, kf.transpose(-1, -2)) * scale).masked_fill(~ok.unsqueeze(1), float("-inf")))
    return qf, kf, vf, p, lse, rows, back


def prefix_attn_fwd(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, prefix_k: torch.Tensor, prefix_v: torch.Tensor,
                    softmax_scale: Optional[float] = None, causal: bool = True, lens: Lens = None,
                    prefix_lens: Lens = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """q [B, S, Hq, D], k / v [B, S, Hkv, D], prefix_k / prefix_v [G, P, Hkv, D] -> (out [B, S, Hq, D] contiguous,
    log-sum-exp fp32 [B, Hq, S]). ``causal`` concerns a sequence's own keys; its prefix is always seen whole."""
    _check(q, k, prefix_k)
    scale = scale_of(q, softmax_scale)
    if use_native(q):
        return hip_ops().prefix_attn_fwd(q, k, v, prefix_k, prefix_v, scale, causal, lens, prefix_lens)
    _check_reference("prefix_attn_fwd", q, k, v, prefix_k, prefix_v, lens, prefix_lens)
    _, _, vf, p, lse, _, back = _ref_parts(q, k, v, prefix_k, prefix_v, scale, causal, lens, prefix_lens)
    return back(torch.matmul(p, vf)), lse


def prefix_attn_bwd(dout: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, prefix_k: torch.Tensor,
                    prefix_v: torch.Tensor, out: torch.Tensor, lse: torch.Tensor, softmax_scale: Optional[float] = None,
                    causal: bool = True, lens: Lens = None, prefix_lens: Lens = None):
    """(dq, dk, dv, dprefix_k, dprefix_v), contiguous. ``out`` and ``lse`` are the forward's."""
    _check(q, k, prefix_k)
    scale = scale_of(q, softmax_scale)
    if use_native(q):
        return hip_ops().prefix_attn_bwd(dout, q, k, v, prefix_k, prefix_v, out, lse, scale, causal, lens, prefix_lens)
    _check_reference("prefix_attn_bwd", q, k, v, prefix_k, prefix_v, lens, prefix_lens, dout, out)
    B, S, Hq, D = q.shape
    G, P, Hkv = prefix_k.shape[:3]
    qf, kf, vf, p, _, rows, back = _ref_parts(q, k, v, prefix_k, prefix_v, scale, causal, lens, prefix_lens)
    do, o = rows(dout), rows(out)
    ds = p * (torch.matmul(do, vf.transpose(-1, -2)) - (do * o).sum(-1, keepdim=True)) * scale

    some = live_rows(prefix_lens, G, P, q.device)[:, :, None, None]

    def split(t):  # [B, Hq, P + S, D] -> (own [B, S, Hkv, D], prefix [G, P, Hkv, D])
        t = t.view(B, Hkv, Hq // Hkv, P + S, D).sum(2)
        of_prefix = t[:, :, :P].permute(0, 2, 1, 3).reshape(G, B // G, P, Hkv, D).sum(1)
        return back(t[:, :, P:]), torch.where(some, of_prefix, 0.0).to(q.dtype)

    dk, dpk = split(torch.matmul(ds.transpose(-1, -2), qf))
    dv, dpv = split(torch.matmul(p.transpose(-1, -2), do))
    return back(torch.matmul(ds, kf)), dk, dv, dpk, dpv


class PrefixAttentionFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, prefix_k, prefix_v, softmax_scale, causal, lens, prefix_lens):
        out, lse = prefix_attn_fwd(q, k, v, prefix_k, prefix_v, softmax_scale, causal, lens, prefix_lens)
        ctx.save_for_backward(q, k, v, prefix_k, prefix_v, out, lse, lens, prefix_lens)
        ctx.scale, ctx.causal = softmax_scale, causal
        return out

    @staticmethod
    def backward(ctx, dout):
        q, k, v, pk, pv, out, lse, lens, plens = ctx.saved_tensors
        g = prefix_attn_bwd(dout.contiguous(), q, k, v, pk, pv, out, lse, ctx.scale, ctx.causal, lens, plens)
        return (*once(g, (dout, q, k, v, pk, pv)), None, None, None, None)


def prefix_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, prefix_k: torch.Tensor, prefix_v: torch.Tensor,
                     softmax_scale: Optional[float] = None, causal: bool = True, lens: Lens = None,
                     prefix_lens: Lens = None) -> torch.Tensor:
    """out [B, S, Hq, D] as :func:`prefix_attn_fwd`, differentiable in q, k, v, prefix_k and prefix_v."""
    _check(q, k, prefix_k)
    if use_native(q):  # one operator each way (csrc/autograd.cpp)
        return hip_ops().prefix_attention(q, k, v, prefix_k, prefix_v, scale_of(q, softmax_scale), causal, lens, prefix_lens)
    return PrefixAttentionFunction.apply(q, k, v, prefix_k, prefix_v, softmax_scale, causal, lens, prefix_lens)


def prefix_attention_decode(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, lens: torch.Tensor,
                            prefix_k: torch.Tensor, prefix_v: torch.Tensor, prefix_lens: Lens = None,
                            softmax_scale: Optional[float] = None) -> torch.Tensor:
    """One token per sequence: q [B, Hq, D] over the group's prefix and the sequence's own cache k / v [B, L, Hkv, D] of
    lens int32 [B] tokens (the token's own row already stored) -> out [B, Hq, D]. No keys at all give zeros. The kernel's work is
    cut by L and P, not by the lengths: pass views of a cache that is allocated well beyond its longest sequence."""
    _check(q, k, prefix_k)
    scale = scale_of(q, softmax_scale)
    if use_native(q):
        return hip_ops().prefix_attn_decode(q, k, v, lens, prefix_k, prefix_v, scale, prefix_lens)
    _check_reference("prefix_attention_decode", q, k, v, prefix_k, prefix_v, lens, prefix_lens)
    rep = q.shape[1] // k.shape[2]
    kf, live = _ref_keys(k, prefix_k, lens, prefix_lens, rep)
    vf, _ = _ref_keys(v, prefix_v, lens, prefix_lens, rep)
    s = torch.matmul(q.to(kf.dtype).unsqueeze(2), kf.transpose(-1, -2)) * scale
    p, _ = softmax_lse(s.masked_fill(~live[:, None, None, :], float("-inf")))
    return torch.matmul(p, vf).squeeze(2).to(q.dtype)
