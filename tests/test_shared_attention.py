"""Latent attention and attention over a shared prefix, training and single-token forms, against the definition in 64 bits.

Tolerances are elementwise bounds computed beside each expected value (:func:`attend64`). With u = eps / 2 of the type:
the weights P (and dS) are rounded to the type before their products, so a product with them is off by at most
u sum |P| |x|; sums run in fp32, an n-term one off by at most n 2^-24 sum |terms|; the result is rounded once more. A score
that is off by d changes its weight by a factor exp(d). Gradients use delta = rowsum(dO * O) of the ROUNDED output. fp16
values under 2^-14 have a fixed step: half of it, 2^-25, is added per weight.
"""
import math

import pytest
import torch

from distributed_llm_training_gpu_manager_amd import _native, ops

F32 = 2.0 ** -24
CPU, GPU = "cpu", "cuda"
WIDE, HALF = (128, 64, 128), (64, 32, 64)


def attend64(q, k, v, ok, scale, dt, do=None):
    """Attention of q [..., i, d] over k, v [..., j, d] where ok [..., i, j], in 64 bits, and how far a 16-bit
    implementation may be off BEFORE its last rounding: {name: (value, bound)}."""
    u = torch.finfo(dt).eps / 2 if dt in (torch.bfloat16, torch.float16) else 0.0
    sub = 2.0 ** -25 if dt == torch.float16 else 0.0
    q, k, v = q.double(), k.double(), v.double()
    d, e, n = q.shape[-1], v.shape[-1], max(q.shape[-2], k.shape[-2])
    kt, vt = k.transpose(-1, -2), v.transpose(-1, -2)
    s = (q @ kt) * scale
    off = (d + 8) * F32 * (q.abs() @ kt.abs()) * scale + 4 * F32 * s.abs()  # of a score
    off = torch.where(ok, off, 0.0)
    s = s.masked_fill(~ok, float("-inf"))
    none = ~ok.any(-1, keepdim=True)
    m = s.amax(-1, keepdim=True).masked_fill(none, 0.0) if s.shape[-1] else none.double() * 0
    x = torch.exp(s - m)
    l = x.sum(-1, keepdim=True)
    p = x / l.masked_fill(none, 1.0)
    lse = (m + l.log()).squeeze(-1)
    top = off.amax(-1, keepdim=True) if s.shape[-1] else none.double() * 0
    rel = off + top + 2.0 ** -20 + 8 * F32 * lse.abs().masked_fill(none.squeeze(-1), 0.0).unsqueeze(-1)  # of a weight
    vis = ok.double()
    out = p @ v
    res = {"out": (out, (p * (u + rel)) @ v.abs() + (n * F32) * (p @ v.abs()) + sub * (vis @ v.abs())),
           "lse": (lse, top.squeeze(-1) + 2.0 ** -20 + 8 * F32 * lse.abs().masked_fill(none.squeeze(-1), 0.0))}
    if do is not None:
        do = do.double()
        pt, dot = p.transpose(-1, -2), do.abs()
        res["dv"] = (pt @ do, (p * (u + rel)).transpose(-1, -2) @ dot + (n * F32) * (pt @ dot) + sub * (vis.transpose(-1, -2) @ dot))
        dp, delta = do @ vt, (do * out).sum(-1, keepdim=True)
        dp_off = (e + 8) * F32 * (dot @ vt.abs())
        delta_off = (dot * (res["out"][1] + u * out.abs() + (e + 8) * F32 * out.abs())).sum(-1, keepdim=True)
        ds = p * (dp - delta)
        ds_off = p * (dp_off + delta_off) + ds.abs() * (u + rel + 4 * F32) + sub * vis
        res["dq"] = ((ds @ k) * scale, scale * (ds_off @ k.abs() + n * F32 * (ds.abs() @ k.abs())))
        res["dk"] = ((ds.transpose(-1, -2) @ q) * scale,
                     scale * (ds_off.transpose(-1, -2) @ q.abs() + n * F32 * (ds.abs().transpose(-1, -2) @ q.abs())))
    return res


def close(got, pair, dt, what):
    """got is within the bound and one rounding of the type."""
    want, bound = pair
    u = torch.finfo(dt).eps / 2 if dt in (torch.bfloat16, torch.float16) else 2.0 ** -22
    tiny = torch.finfo(dt).smallest_normal * u * 2 if dt in (torch.bfloat16, torch.float16) else 0.0
    got = got.double()
    assert got.shape == want.shape, what
    allow = bound * (1 + u) + u * want.abs() + tiny
    bad = ~((got - want).abs() <= allow) & ~((got == want))
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float(((got - want).abs() - allow)[bad].max()):.3g}"


def heads(t):  # [B, S, H, D] -> [B, H, S, D]
    return t.transpose(1, 2)


def group_sum(pair, rep):  # [B, H, S, D] -> [B, H / rep, S, D]
    return tuple(t.view(t.shape[0], -1, rep, *t.shape[2:]).sum(2) for t in pair)


def live(lens, B, S, dev):
    if lens is None:
        return torch.ones(B, S, dtype=torch.bool, device=dev)
    return torch.arange(S, device=dev)[None] < torch.tensor(lens, device=dev)[:, None].clamp(0, S)


def rnd(g, *shape, dt, dev, std=1.0):
    return (torch.randn(*shape, generator=g) * std).to(dt).to(dev)


def spoil(t, alive, value=float("nan")):
    """What lies behind the lengths may hold anything."""
    t[~alive] = value
    return t


def ramp(t, dim, lo, hi):
    """Keys that grow along the sequence, so that a running maximum is raised again and again."""
    f = torch.linspace(lo, hi, t.shape[dim], device=t.device).view([-1 if i == dim else 1 for i in range(t.dim())])
    return t.copy_((t.float() * f).to(t.dtype))


def check_latent(dev, dt, layout, B, S, H, causal=True, lens=None, strided=False, scale=None, grow=False):
    dn, dr, dv = layout
    g = torch.Generator().manual_seed(B * 1000 + S)
    if strided:  # views of wider rows, the rope key inside the latent projection's row
        q = rnd(g, B, S, H * (dn + dr) + 16, dt=dt, dev=dev)[..., 16:].unflatten(2, (H, dn + dr))
        kv = rnd(g, S, B, H + 1, dn + dv, dt=dt, dev=dev).transpose(0, 1)[:, :, 1:]
        kr = rnd(g, B, S, 64 + dr, dt=dt, dev=dev)[..., 64:]
        do = rnd(g, B, H, S, dv, dt=dt, dev=dev).transpose(1, 2)
    else:
        q, kv = rnd(g, B, S, H, dn + dr, dt=dt, dev=dev), rnd(g, B, S, H, dn + dv, dt=dt, dev=dev)
        kr, do = rnd(g, B, S, dr, dt=dt, dev=dev), rnd(g, B, S, H, dv, dt=dt, dev=dev)
    if grow:
        ramp(kv[..., :dn], 1, 0.1, 8), ramp(kr, 1, 0.1, 8)
    alive = live(lens, B, S, dev)
    for t in (q, kv, kr, do):
        spoil(t, alive)
    lt = None if lens is None else torch.tensor(lens, dtype=torch.int32, device=dev)
    out, lse = ops.latent_attn_fwd(q, kv, kr, scale, causal, lt)
    dq, dkv, dkr = ops.latent_attn_bwd(do, q, kv, kr, out, lse, scale, causal, lt)
    z = lambda t: torch.where(alive.view(B, S, *[1] * (t.dim() - 2)), t.double(), 0.0)  # noqa: E731
    k = torch.cat([z(kv)[..., :dn], z(kr).unsqueeze(2).expand(B, S, H, dr)], -1)
    ok = alive[:, None, :] & alive[:, :, None]
    if causal:
        ok = ok & torch.ones(S, S, dtype=torch.bool, device=dev).tril()
    e = attend64(heads(z(q)), heads(k), heads(z(kv)[..., dn:]), ok[:, None].expand(B, H, S, S),
                 scale or (dn + dr) ** -0.5, dt, heads(z(do)))
    close(heads(out), e["out"], dt, "out")
    close(lse, e["lse"], torch.float32, "lse")
    close(heads(dq), e["dq"], dt, "dq")
    close(heads(dkv)[..., :dn], tuple(t[..., :dn] for t in e["dk"]), dt, "dk_nope")
    close(heads(dkv)[..., dn:], e["dv"], dt, "dv")
    close(dkr, tuple(t[..., dn:].sum(1) for t in e["dk"]), dt, "dk_rope")
    for t in (out, dq, dkv, dkr):
        assert not t[~alive].any(), "rows behind a length are zeros"


def check_prefix(dev, dt, D, G, n, P, S, Hq, Hkv, causal=True, lens=None, plens=None, strided=False, grow=False):
    B, rep = G * n, Hq // Hkv
    g = torch.Generator().manual_seed(P * 1000 + S)
    if strided:  # q, k, v as parts of one packed row; the prefix cut from a longer one
        row = rnd(g, B, S, (Hq + 2 * Hkv) * D, dt=dt, dev=dev)
        q, k, v = (row[..., a * D:b * D].unflatten(2, (b - a, D)) for a, b in ((0, Hq), (Hq, Hq + Hkv), (Hq + Hkv, Hq + 2 * Hkv)))
        pk, pv = (rnd(g, G, Hkv, P + 5, D, dt=dt, dev=dev).transpose(1, 2)[:, 5:] for _ in range(2))
    else:
        q, k, v = (rnd(g, B, S, h, D, dt=dt, dev=dev) for h in (Hq, Hkv, Hkv))
        pk, pv = (rnd(g, G, P, Hkv, D, dt=dt, dev=dev) for _ in range(2))
    do = rnd(g, B, S, Hq, D, dt=dt, dev=dev)
    if grow:
        ramp(pk, 1, 0.1, 4), ramp(k, 1, 4, 8)
    alive, palive = live(lens, B, S, dev), live(plens, G, P, dev)
    for t in (q, k, v, do):
        spoil(t, alive)
    for t in (pk, pv):
        spoil(t, palive, float("inf"))
    i32 = lambda x: None if x is None else torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    out, lse = ops.prefix_attn_fwd(q, k, v, pk, pv, None, causal, i32(lens), i32(plens))
    dq, dk, dv, dpk, dpv = ops.prefix_attn_bwd(do, q, k, v, pk, pv, out, lse, None, causal, i32(lens), i32(plens))
    z = lambda t: torch.where(alive[:, :, None, None], t.double(), 0.0)  # noqa: E731
    zp = lambda t: torch.where(palive[:, :, None, None], t.double(), 0.0)  # noqa: E731
    both = lambda a, p: heads(torch.cat([zp(p).repeat_interleave(n, 0), z(a)], 1)).repeat_interleave(rep, 1)  # noqa: E731
    own = alive[:, None, :] & alive[:, :, None]
    if causal:
        own = own & torch.ones(S, S, dtype=torch.bool, device=dev).tril()
    ok = torch.cat([palive.repeat_interleave(n, 0)[:, None, :] & alive[:, :, None], own], 2)
    e = attend64(heads(z(q)), both(k, pk), both(v, pv), ok[:, None].expand(B, Hq, S, P + S), D ** -0.5, dt, heads(z(do)))
    close(heads(out), e["out"], dt, "out")
    close(lse, e["lse"], torch.float32, "lse")
    close(heads(dq), e["dq"], dt, "dq")
    for name, own_g, pre_g in (("dk", dk, dpk), ("dv", dv, dpv)):
        pair = group_sum(e[name], rep)
        close(heads(own_g), tuple(t[:, :, P:] for t in pair), dt, name)
        close(heads(pre_g), tuple(t[:, :, :P].reshape(G, n, Hkv, P, D).sum(1) for t in pair), dt, name + " of the prefix")
    for t, a in ((out, alive), (dq, alive), (dk, alive), (dv, alive), (dpk, palive), (dpv, palive)):
        assert not t[~a].any(), "rows behind a length are zeros"


def check_latent_decode(dev, dt, layout, r, B, H, L, lens, strided=False, grow=False):
    """Four roundings (absorbed query, weights, latent output, result), each off by at most u of what it rounds: 4 u in
    the 2-norm of a head's output. `grow`: queries of 3 times the size; the absorbed query's rounding, r independent ones of at
    most u, moves a score by u / sqrt(3) times its own size, some 3 in the mean, and a weight and its sum by that factor each:
    3.5 u more, 8 u in all."""
    dn, dr, dv = layout
    g = torch.Generator().manual_seed(B * 1000 + L)
    w = rnd(g, H * (dn + dv), r, dt=dt, dev=dev, std=r ** -0.5)
    if strided:
        q = rnd(g, H, B, dn + dr + 8, dt=dt, dev=dev).transpose(0, 1)[..., 8:]
        cache = rnd(g, L, B, r + dr + 32, dt=dt, dev=dev).transpose(0, 1)[..., :r + dr]
    else:
        q, cache = rnd(g, B, H, dn + dr, dt=dt, dev=dev), rnd(g, B, L, r + dr, dt=dt, dev=dev)
    if grow:
        q.mul_(3), ramp(cache, 1, 0.05, 1)
    alive = live(lens, B, L, dev)
    spoil(cache, alive)
    out = ops.latent_attention_decode(q, cache, torch.tensor(lens, dtype=torch.int32, device=dev), w)
    w3, c = w.double().view(H, dn + dv, r), torch.where(alive[..., None], cache.double(), 0.0)
    kv = torch.einsum("blr,hxr->bhlx", c[..., :r].cpu(), w3.cpu()).to(dev)
    k = torch.cat([kv[..., :dn], c[:, None, :, r:].expand(B, H, L, dr)], -1)
    want = attend64(q.double().unsqueeze(2), k, kv[..., dn:], alive[:, None, None, :].expand(B, H, 1, L),
                    (dn + dr) ** -0.5, dt)["out"][0].squeeze(2)
    u = torch.finfo(dt).eps / 2 if dt != torch.float32 else 2.0 ** -20
    err = (out.double() - want).norm(dim=-1)
    assert (err <= (8 if grow else 4) * u * want.norm(dim=-1)).all(), float((err / want.norm(dim=-1).clamp_min(1e-30)).max())
    assert not out[~alive[:, 0]].any()


def check_prefix_decode(dev, dt, D, G, n, P, L, Hq, Hkv, lens, plens=None, strided=False, grow=False):
    B, rep = G * n, Hq // Hkv
    g = torch.Generator().manual_seed(P * 1000 + L)
    q = rnd(g, Hq, B, D, dt=dt, dev=dev).transpose(0, 1) if strided else rnd(g, B, Hq, D, dt=dt, dev=dev)
    if strided:
        k, v = (rnd(g, B, Hkv, L, D, dt=dt, dev=dev).transpose(1, 2) for _ in range(2))
        pk, pv = (rnd(g, P, G, Hkv, D + 8, dt=dt, dev=dev).transpose(0, 1)[..., :D] for _ in range(2))
    else:
        k, v = (rnd(g, B, L, Hkv, D, dt=dt, dev=dev) for _ in range(2))
        pk, pv = (rnd(g, G, P, Hkv, D, dt=dt, dev=dev) for _ in range(2))
    if grow:
        ramp(pk, 1, 0.1, 4), ramp(k, 1, 4, 8)
    alive, palive = live(lens, B, L, dev), live(plens, G, P, dev)
    for t in (k, v):
        spoil(t, alive)
    for t in (pk, pv):
        spoil(t, palive)
    i32 = lambda x: None if x is None else torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    out = ops.prefix_attention_decode(q, k, v, i32(lens), pk, pv, i32(plens))
    z = lambda t, a: torch.where(a[:, :, None, None], t.double(), 0.0)  # noqa: E731
    both = lambda a, p: heads(torch.cat([z(p, palive).repeat_interleave(n, 0), z(a, alive)], 1)).repeat_interleave(rep, 1)  # noqa: E731
    ok = torch.cat([palive.repeat_interleave(n, 0), alive], 1)
    e = attend64(q.double().unsqueeze(2), both(k, pk), both(v, pv), ok[:, None, None, :].expand(B, Hq, 1, P + L), D ** -0.5, dt)
    close(out, tuple(t.squeeze(2) for t in e["out"]), dt, "out")
    assert not out[~ok.any(1)].any()


# ---- the reference path (CPU) ------------------------------------------------------------------

def test_reference_latent():
    for causal in (True, False):
        check_latent(CPU, torch.float32, HALF, 3, 17, 3, causal, [17, 0, 5])
    check_latent(CPU, torch.float32, (16, 8, 24), 1, 9, 2, strided=True)


def test_reference_prefix():
    check_prefix(CPU, torch.float32, 16, 2, 2, 7, 9, 4, 2, True, [9, 0, 1, 4], [7, 3])
    check_prefix(CPU, torch.float32, 16, 1, 3, 0, 5, 3, 3, False, [5, 0, 2], strided=True)


def test_reference_decode():
    check_latent_decode(CPU, torch.float32, (16, 8, 24), 32, 3, 5, 11, [11, 0, 1])
    check_prefix_decode(CPU, torch.float32, 16, 2, 2, 7, 9, 4, 2, [9, 0, 0, 4], [7, 0])


@pytest.mark.parametrize("lens", [None, [4, 2]])
def test_gradients_match_differences(lens):
    """The differentiable entry points against finite differences in 64 bits."""
    g = torch.Generator().manual_seed(0)
    x = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64, requires_grad=True)  # noqa: E731
    lt = None if lens is None else torch.tensor(lens, dtype=torch.int32)
    assert torch.autograd.gradcheck(lambda *a: ops.latent_attention(*a, lens=lt), (x(2, 4, 2, 5), x(2, 4, 6), x(2, 4, 2), x(2 * 7, 6)))
    assert torch.autograd.gradcheck(lambda *a: ops.prefix_attention(*a, lens=lt),
                                    (x(2, 4, 4, 3), x(2, 4, 2, 3), x(2, 4, 2, 3), x(1, 3, 2, 3), x(1, 3, 2, 3)))


@pytest.mark.parametrize("dev", [CPU, pytest.param(GPU, marks=pytest.mark.gpu)])
def test_a_second_differentiation_is_refused(dev):
    """Gradients may be recorded (create_graph), for losses that use others of them; differentiating these raises."""
    q, kv, kr = (t.requires_grad_(True) for t in _latent_args(dev))
    g = torch.Generator().manual_seed(4)
    c, w = (rnd(g, *s, dt=q.dtype, dev=dev).requires_grad_(True) for s in ((2, 8, 16), (2 * 128, 16)))
    k, pk = (rnd(g, *s, dt=q.dtype, dev=dev).requires_grad_(True) for s in ((2, 8, 2, 64), (1, 5, 2, 64)))
    for out, x in ((ops.latent_attention(q, c, kr, w), (q, c, kr, w)), (ops.prefix_attention(q[..., :64], k, k, pk, pk), (k, pk))):
        plain = torch.autograd.grad(out.sum(), x, retain_graph=True)
        recorded = torch.autograd.grad(out.sum(), x, create_graph=True)
        assert all(torch.equal(a, b.detach()) for a, b in zip(plain, recorded))
        for r in recorded:
            with pytest.raises(RuntimeError, match="differentiated again"):
                torch.autograd.grad(r.sum(), x, allow_unused=True, retain_graph=True)


def test_absorbed_and_expanded_agree():
    """The last token of the expanded form is the absorbed form over the cache of all tokens."""
    g = torch.Generator().manual_seed(1)
    B, S, H, dn, dr, dv, r = 2, 6, 3, 8, 4, 5, 16
    q, c, kr = (torch.randn(*s, generator=g, dtype=torch.float64) for s in ((B, S, H, dn + dr), (B, S, r), (B, S, dr)))
    w = torch.randn(H * (dn + dv), r, generator=g, dtype=torch.float64)
    a = ops.latent_attention(q, c, kr, w)[:, -1]
    b = ops.latent_attention_decode(q[:, -1], torch.cat([c, kr], -1), torch.full((B,), S, dtype=torch.int32), w)
    assert torch.allclose(a, b, rtol=1e-12, atol=1e-12)


def _latent_args(dev, dt=torch.bfloat16, B=2, S=8, H=2, layout=HALF):
    dn, dr, dv = layout
    g = torch.Generator().manual_seed(0)
    return [rnd(g, *s, dt=dt, dev=dev) for s in ((B, S, H, dn + dr), (B, S, H, dn + dv), (B, S, dr))]


@pytest.mark.parametrize("dev", [CPU, pytest.param(GPU, marks=pytest.mark.gpu)])
@pytest.mark.parametrize("S,causal", [(70, True), (150, False)])
def test_rows_behind_a_length_are_zeros_beside_a_nan(dev, S, causal):
    """NaN and infinity in live rows stay out of the rows that do not exist."""
    g = torch.Generator().manual_seed(19)
    lens, plens = [S - 9, 0, 5], [70]
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    alive, palive = live(lens, 3, S, dev), live(plens, 1, 90, dev)

    def behind(*tensors):
        for t, a in tensors:
            assert not t[~a].any()

    q, kv, kr = _latent_args(dev, B=3, S=S)
    do = rnd(g, 3, S, 2, 64, dt=torch.bfloat16, dev=dev)
    for t, bad in ((q, float("nan")), (kv, float("inf")), (kr, float("nan")), (do, float("nan"))):
        t[0, 2, ..., 3] = bad
        out, lse = ops.latent_attn_fwd(q, kv, kr, causal=causal, lens=i32(lens))
        assert (lse.transpose(1, 2)[~alive] == float("-inf")).all()
        dq, dkv, dkr = ops.latent_attn_bwd(do, q, kv, kr, out, lse, causal=causal, lens=i32(lens))
        behind(*((x, alive) for x in (out, dq, dkv, dkr)))
        t[0, 2] = 1
    q, k, v, do = (rnd(g, 3, S, h, 64, dt=torch.bfloat16, dev=dev) for h in (4, 2, 2, 4))
    pk, pv = (rnd(g, 1, 90, 2, 64, dt=torch.bfloat16, dev=dev) for _ in range(2))
    for t, bad in ((q, float("nan")), (k, float("inf")), (v, float("nan")), (pk, float("nan")), (pv, float("inf")), (do, float("nan"))):
        t[0, 2, 0, 3] = bad
        out, lse = ops.prefix_attn_fwd(q, k, v, pk, pv, None, causal, i32(lens), i32(plens))
        assert (lse.transpose(1, 2)[~alive] == float("-inf")).all()
        dq, dk, dv, dpk, dpv = ops.prefix_attn_bwd(do, q, k, v, pk, pv, out, lse, None, causal, i32(lens), i32(plens))
        behind((out, alive), (dq, alive), (dk, alive), (dv, alive), (dpk, palive), (dpv, palive))
        t[0, 2] = 1


@pytest.mark.parametrize("dev", [CPU, pytest.param(GPU, marks=pytest.mark.gpu)])
def test_shapes_that_do_not_fit_are_refused(dev):
    q, kv, kr = _latent_args(dev)
    c, w = torch.zeros(2, 8, 16, dtype=q.dtype, device=dev), torch.zeros(2 * 128, 16, dtype=q.dtype, device=dev)
    for bad in ((q, c[:, :4], kr, w), (q, c, kr[:1], w), (q, c, kr, w[:, :8]), (q, c, kr, w[:-1]), (q, c, kr, w[:64])):
        with pytest.raises(ValueError):
            ops.latent_attention(*bad)
    k = torch.zeros(6, 8, 2, 64, dtype=q.dtype, device=dev)
    qq, pk = torch.zeros(6, 8, 4, 64, dtype=q.dtype, device=dev), torch.zeros(4, 3, 2, 64, dtype=q.dtype, device=dev)
    for args in ((qq, k, k, pk, pk), (qq, k, k, pk[:2, :, :1], pk[:2, :, :1]), (qq[:, :, :3], k, k, pk[:2], pk[:2]), (qq, k, k, pk[:0], pk[:0])):
        with pytest.raises(ValueError):
            ops.prefix_attention(*args)
        with pytest.raises(ValueError):
            ops.prefix_attention_decode(args[0][:, 0], *args[1:3], torch.zeros(6, dtype=torch.int32, device=dev), *args[3:])


@pytest.mark.parametrize("dev", [CPU, pytest.param(GPU, marks=pytest.mark.gpu)])
def test_reference_and_kernels_refuse_the_same(dev):
    """Shapes that would broadcast, mixed types, lengths of another type or number, scales without a softmax."""
    q, kv, kr = _latent_args(dev)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    out, lse = ops.latent_attn_fwd(q, kv, kr, lens=i32(8, 3))
    cache, w = torch.zeros(2, 9, 256 + 32, dtype=q.dtype, device=dev), torch.zeros(2 * 128, 256, dtype=q.dtype, device=dev)
    pq, k, pk = (torch.zeros(*s, dtype=q.dtype, device=dev) for s in ((4, 8, 4, 64), (4, 8, 2, 64), (2, 5, 2, 64)))
    po, plse = ops.prefix_attn_fwd(pq, k, k, pk, pk, lens=i32(1, 2, 3, 4), prefix_lens=i32(5, 0))
    ops.latent_attn_bwd(out, q, kv, kr, out, lse, lens=i32(8, 3)), ops.prefix_attn_bwd(po, pq, k, k, pk, pk, po, plse)
    ops.latent_attention_decode(q[:, 0], cache, i32(1, 2), w), ops.prefix_attention_decode(pq[:, 0], k, k, i32(1, 2, 3, 4), pk, pk)
    bad = [
        lambda: ops.latent_attn_fwd(q, kv[:1], kr),
        lambda: ops.latent_attn_fwd(q, kv, kr[:, :1]),
        lambda: ops.latent_attn_fwd(q, kv[:, :, :1], kr),
        lambda: ops.latent_attn_fwd(q.half(), kv, kr),
        lambda: ops.latent_attn_fwd(q, kv, kr, lens=i32(8, 8).long()),
        lambda: ops.latent_attn_fwd(q, kv, kr, lens=i32(8)),
        lambda: ops.latent_attn_fwd(q, kv, kr, lens=i32(8, 8).view(2, 1)),
        lambda: ops.latent_attn_bwd(out[:1], q, kv, kr, out, lse),
        lambda: ops.latent_attn_bwd(out, q, kv, kr, out[:, :1], lse),
        lambda: ops.latent_attention_decode(q[:, 0], cache[:1], i32(1, 2), w),
        lambda: ops.latent_attention_decode(q[:, 0], cache, i32(1, 2).long(), w),
        lambda: ops.latent_attention_decode(q[:, 0], cache, i32(1), w),
        lambda: ops.latent_attention_decode(q[:, 0], cache, i32(1, 2), w[:-1]),
        lambda: ops.prefix_attn_fwd(pq, k, k[:, :4], pk, pk),
        lambda: ops.prefix_attn_fwd(pq, k[:1], k[:1], pk, pk),
        lambda: ops.prefix_attn_fwd(pq, k[:, :1], k[:, :1], pk, pk),
        lambda: ops.prefix_attn_fwd(pq, k, k, pk, pk[:1]),
        lambda: ops.prefix_attn_fwd(pq, k, k.half(), pk, pk),
        lambda: ops.prefix_attn_fwd(pq, k, k, pk, pk, lens=i32(1, 2, 3)),
        lambda: ops.prefix_attn_fwd(pq, k, k, pk, pk, prefix_lens=i32(1)),
        lambda: ops.prefix_attn_bwd(po[:1], pq, k, k, pk, pk, po, plse),
        lambda: ops.prefix_attention_decode(pq[:, 0], k, k, i32(1, 2, 3, 4).long(), pk, pk),
        lambda: ops.prefix_attention_decode(pq[:, 0], k, k[:1], i32(1, 2, 3, 4), pk, pk),
    ]
    for scale in (0.0, -1.0, 1e-30, 1e30, float("nan"), float("inf")):
        bad += [lambda x=scale: ops.latent_attn_fwd(q, kv, kr, x), lambda x=scale: ops.latent_attn_bwd(out, q, kv, kr, out, lse, x),
                lambda x=scale: ops.latent_attention_decode(q[:, 0], cache, i32(1, 2), w, x),
                lambda x=scale: ops.prefix_attn_fwd(pq, k, k, pk, pk, x), lambda x=scale: ops.prefix_attn_bwd(po, pq, k, k, pk, pk, po, plse, x),
                lambda x=scale: ops.prefix_attention_decode(pq[:, 0], k, k, i32(1, 2, 3, 4), pk, pk, None, x)]
    for i, call in enumerate(bad):
        with pytest.raises((RuntimeError, ValueError)):
            call()
            pytest.fail(f"call {i} was not refused")


# ---- the kernels (GPU) -------------------------------------------------------------------------

BF, FP = torch.bfloat16, torch.float16


@pytest.mark.gpu
@pytest.mark.parametrize("dt,layout,B,S,H,causal,lens,strided", [
    (BF, WIDE, 1, 1, 1, True, None, False),
    (BF, WIDE, 2, 128, 2, True, None, False),
    (FP, WIDE, 3, 129, 3, True, [129, 0, 64], False),
    (BF, WIDE, 2, 333, 2, False, [333, 1], True),
    (FP, WIDE, 1, 511, 5, False, None, False),
    (BF, HALF, 2, 63, 3, True, None, True),
    (FP, HALF, 4, 200, 2, True, [1, 200, 31, 97], False),
    (BF, HALF, 2, 65, 1, False, [65, 33], True),
    (FP, HALF, 1, 640, 9, True, None, False),
    (BF, WIDE, 3, 257, 30, True, [257, 100, 0], False),  # more workgroups than CUs: one wave to 32 queries
    (FP, HALF, 2, 130, 70, False, None, True),
])
def test_latent_kernels(dt, layout, B, S, H, causal, lens, strided):
    check_latent(GPU, dt, layout, B, S, H, causal, lens, strided)


@pytest.mark.gpu
@pytest.mark.parametrize("dt,D,G,n,P,S,Hq,Hkv,causal,lens,plens,strided", [
    (BF, 128, 1, 1, 1, 1, 1, 1, True, None, None, False),
    (BF, 128, 1, 4, 256, 128, 8, 2, True, None, None, False),
    (FP, 128, 2, 2, 130, 65, 4, 4, True, [65, 0, 7, 64], [130, 63], True),
    (BF, 128, 1, 3, 0, 200, 6, 2, True, [200, 1, 128], None, False),
    (FP, 128, 3, 1, 77, 33, 3, 1, False, [33, 0, 5], [0, 77, 1], False),
    (BF, 64, 2, 3, 300, 40, 4, 2, True, None, [300, 129], True),
    (FP, 64, 1, 5, 64, 129, 12, 12, True, [129, 64, 0, 1, 100], None, False),
    (BF, 64, 1, 2, 513, 17, 6, 1, False, None, [0], False),
    (FP, 64, 1, 8, 1000, 3, 2, 2, True, None, None, False),
    (BF, 128, 2, 4, 200, 140, 24, 4, True, [140, 1, 139, 0, 64, 65, 128, 140], [200, 7], False),  # more workgroups than CUs
    (FP, 64, 1, 9, 70, 60, 30, 10, False, None, None, False),
])
def test_prefix_kernels(dt, D, G, n, P, S, Hq, Hkv, causal, lens, plens, strided):
    check_prefix(GPU, dt, D, G, n, P, S, Hq, Hkv, causal, lens, plens, strided)


@pytest.mark.gpu
@pytest.mark.parametrize("dt,layout,r,B,H,L,lens,strided", [
    (BF, WIDE, 512, 1, 1, 1, [1], False),
    (BF, WIDE, 512, 3, 32, 300, [300, 0, 64], False),
    (FP, WIDE, 512, 2, 65, 129, [129, 65], True),
    (FP, WIDE, 256, 5, 8, 1000, [1000, 999, 63, 1, 0], False),
    (BF, WIDE, 256, 33, 2, 70, [70 - 2 * i for i in range(33)], True),
    (BF, HALF, 512, 2, 20, 513, [500, 513], False),
    (FP, HALF, 256, 1, 130, 4100, [4100], False),
    (BF, HALF, 256, 40, 3, 5, [i % 6 for i in range(40)], False),
    (BF, WIDE, 512, 40, 70, 1000, [1000 - 25 * i for i in range(40)], False),  # several tiles to a workgroup
    (BF, HALF, 512, 150, 4, 700, [0 if 20 <= i < 100 else 7 * i % 701 for i in range(150)], False),  # idle slots in between
    (FP, WIDE, 256, 200, 130, 130, [(37 * i) % 131 for i in range(200)], False),  # several sequences to a workgroup
    (BF, WIDE, 512, 70, 2, 9000, [9000 if i == 66 else 0 for i in range(70)], False),  # one of many
    (BF, WIDE, 512, 3, 8, 100, [0, 0, 0], False),
])
def test_latent_decode_kernel(dt, layout, r, B, H, L, lens, strided):
    check_latent_decode(GPU, dt, layout, r, B, H, L, lens, strided)


@pytest.mark.gpu
@pytest.mark.parametrize("dt,D,G,n,P,L,Hq,Hkv,lens,plens,strided", [
    (BF, 128, 1, 1, 1, 1, 1, 1, [0], None, False),
    (BF, 128, 1, 4, 500, 60, 8, 8, [60, 1, 0, 33], None, False),
    (FP, 128, 2, 17, 300, 129, 8, 2, [129 - 4 * i % 130 for i in range(34)], [300, 0], False),
    (BF, 128, 1, 40, 1500, 20, 8, 2, [i % 21 for i in range(40)], [1401], True),
    (FP, 128, 1, 3, 0, 260, 40, 1, [260, 0, 128], None, False),
    (BF, 64, 3, 2, 127, 0, 6, 2, [0] * 6, [127, 0, 128], False),
    (FP, 64, 1, 6, 9000, 300, 12, 12, [300, 299, 0, 1, 128, 127], None, True),
    (BF, 64, 2, 2, 64, 1000, 70, 1, [1000, 5, 0, 640], [0, 64], False),
])
def test_prefix_decode_kernel(dt, D, G, n, P, L, Hq, Hkv, lens, plens, strided):
    check_prefix_decode(GPU, dt, D, G, n, P, L, Hq, Hkv, lens, plens, strided)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [BF, FP])
def test_growing_scores(dt):
    """Running maxima that are raised all along the keys (the rescaling branches of every kernel)."""
    check_latent(GPU, dt, WIDE, 1, 400, 2, False, grow=True)
    check_latent(GPU, dt, HALF, 1, 400, 2, True, grow=True)
    check_prefix(GPU, dt, 128, 1, 2, 300, 100, 4, 2, grow=True)
    check_prefix(GPU, dt, 64, 1, 2, 300, 100, 2, 2, False, grow=True)
    check_latent_decode(GPU, dt, WIDE, 512, 40, 66, 900, [900] * 40, grow=True)
    check_latent_decode(GPU, dt, HALF, 256, 40, 3, 900, [900] * 40, grow=True)
    check_prefix_decode(GPU, dt, 128, 1, 40, 3000, 100, 4, 1, [100] * 40, grow=True)
    check_prefix_decode(GPU, dt, 64, 2, 3, 3000, 100, 4, 2, [100] * 6, grow=True)


def _train_inputs(seed, dev=GPU, dt=BF):
    g = torch.Generator().manual_seed(seed)
    B, S, H, (dn, dr, dv), r = 2, 150, 4, WIDE, 256
    q, c, kr = (rnd(g, *s, dt=dt, dev=dev) for s in ((B, S, H, dn + dr), (B, S, r), (B, S, dr)))
    w, do = rnd(g, H * (dn + dv), r, dt=dt, dev=dev, std=r ** -0.5), rnd(g, B, S, H, dv, dt=dt, dev=dev)
    return q, c, kr, w, do


@pytest.mark.gpu
def test_latent_attention_is_its_parts():
    """The differentiable entry point is the GEMM, the kernel pair and the GEMMs of the backward, bit for bit; its values and
    gradients are those of the CPU reference up to the roundings on the way (up-projection, weights, output, and in a
    gradient two more: at most 6 u in the 2-norm)."""
    q, c, kr, w, do = _train_inputs(0)
    lens = torch.tensor([150, 77], dtype=torch.int32, device=GPU)
    leaves = [t.clone().requires_grad_(True) for t in (q, c, kr, w)]
    out = ops.latent_attention(*leaves, lens=lens)
    grads = torch.autograd.grad(out, leaves, do)
    kv = torch.empty(2, 150, 4, 256, dtype=BF, device=GPU)
    torch.ops.dlgm.gemm_lt(kv.view(300, -1), c.view(300, -1), w.t(), 0.0, -1)
    o, lse = ops.latent_attn_fwd(q, kv, kr, lens=lens)
    dq, dkv, dkr = ops.latent_attn_bwd(do, q, kv, kr, o, lse, lens=lens)
    assert torch.equal(out, o) and torch.equal(grads[0], dq) and torch.equal(grads[2], dkr)
    ref = [t.cpu().double().requires_grad_(True) for t in (q, c, kr, w)]
    ro = ops.latent_attention(*ref, lens=lens.cpu())
    rg = torch.autograd.grad(ro, ref, do.cpu().double())
    u = torch.finfo(BF).eps / 2
    for a, b in zip((out, *grads), (ro, *rg)):
        assert float((a.detach().cpu().double() - b.detach()).norm()) <= 6 * u * float(b.detach().norm())


@pytest.mark.gpu
@pytest.mark.parametrize("causal,scale,lens,plens", [
    (True, None, None, None), (False, 0.3, [40, 7, 0, 33], [90, 31]), (True, 0.05, [40, 40, 1, 12], None), (False, None, None, [0, 90])])
def test_prefix_attention_is_its_parts(causal, scale, lens, plens):
    """The differentiable entry point is the kernel pair, bit for bit, each argument in its place."""
    g = torch.Generator().manual_seed(22)
    x = [rnd(g, *s, dt=BF, dev=GPU) for s in ((4, 40, 4, 64), (4, 40, 2, 64), (4, 40, 2, 64), (2, 90, 2, 64), (2, 90, 2, 64))]
    do = rnd(g, 4, 40, 4, 64, dt=BF, dev=GPU)
    lt, pt = (None if n is None else torch.tensor(n, dtype=torch.int32, device=GPU) for n in (lens, plens))
    leaves = [t.clone().requires_grad_(True) for t in x]
    out = ops.prefix_attention(*leaves, scale, causal, lt, pt)
    o, lse = ops.prefix_attn_fwd(*x, scale, causal, lt, pt)
    assert torch.equal(out, o)
    want = ops.prefix_attn_bwd(do, *x, o, lse, scale, causal, lt, pt)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(out, leaves, do), want))


@pytest.mark.gpu
@pytest.mark.parametrize("dt,layout,r,causal,scale,lens", [
    (FP, HALF, 512, False, 0.2, [100, 41]), (BF, WIDE, 512, True, 0.02, None), (FP, WIDE, 256, False, None, [99, 0]),
    (BF, HALF, 256, True, 0.3, [1, 100])])
def test_latent_attention_against_the_reference(dt, layout, r, causal, scale, lens):
    """Both types and layouts, with and without a mask, a scale and lengths. Roundings on the way as above (6 u); scores s
    from the rounded up-projection are off by u |s| each, a weight and its sum by that factor: 2 u max |s| more."""
    dn, dr, dv = layout
    B, S, H = 2, 100, 3
    g = torch.Generator().manual_seed(23)
    x = [rnd(g, *s, dt=dt, dev=GPU) for s in ((B, S, H, dn + dr), (B, S, r), (B, S, dr))]
    x.append(rnd(g, H * (dn + dv), r, dt=dt, dev=GPU, std=r ** -0.5))
    do = rnd(g, B, S, H, dv, dt=dt, dev=GPU)
    lt = None if lens is None else torch.tensor(lens, dtype=torch.int32)
    leaves = [t.clone().requires_grad_(True) for t in x]
    out = ops.latent_attention(*leaves, scale, causal, None if lt is None else lt.to(GPU))
    got = (out, *torch.autograd.grad(out, leaves, do))
    ref = [t.cpu().double().requires_grad_(True) for t in x]
    ro = ops.latent_attention(*ref, scale, causal, lt)
    want = (ro, *torch.autograd.grad(ro, ref, do.cpu().double()))
    kv = (ref[1].detach() @ ref[3].detach().t()).view(B, S, H, -1)
    s = torch.einsum("bihd,bjhd->bhij", ref[0].detach(), torch.cat([kv[..., :dn], ref[2].detach().unsqueeze(2).expand(B, S, H, dr)], -1))
    u = torch.finfo(dt).eps / 2
    allow = (6 + 2 * float(s.abs().max()) * (scale or (dn + dr) ** -0.5)) * u
    for a, b in zip(got, want):
        assert float((a.detach().cpu().double() - b.detach()).norm()) <= allow * float(b.detach().norm())


@pytest.mark.gpu
def test_large_weight_gradient():
    """8192 tokens and weights of 32 x 256 rows: dw_kv is a product with c transposed first. dc and dw_kv against dkv w_kv and
    dkv^T c in 64 bits: an fp32 chain of 8192 terms and one rounding."""
    B, S, H, (dn, dr, dv), r = 16, 512, 32, WIDE, 512
    g = torch.Generator(device=GPU).manual_seed(24)
    q, c, kr, w, do = (torch.randn(*s, generator=g, device=GPU) for s in ((B, S, H, dn + dr), (B, S, r), (B, S, dr), (H * (dn + dv), r), (B, S, H, dv)))
    q, c, kr, w, do = (t.to(BF) for t in (q, c, kr, w * r ** -0.5, do))
    leaves = [t.requires_grad_(True) for t in (q, c, kr, w)]
    out = ops.latent_attention(*leaves)
    dq, dc, dkr, dw = torch.autograd.grad(out, leaves, do)
    q, c, kr, w = (t.detach() for t in leaves)
    kv = torch.empty(B, S, H, dn + dv, dtype=BF, device=GPU)
    torch.ops.dlgm.gemm_lt(kv.view(B * S, -1), c.view(B * S, r), w.t(), 0.0, -1)
    o, lse = ops.latent_attn_fwd(q, kv, kr)
    want = ops.latent_attn_bwd(do, q, kv, kr, o, lse)
    assert torch.equal(out.detach(), o) and torch.equal(dq, want[0]) and torch.equal(dkr, want[2])
    d2, c2, u = want[1].view(B * S, -1).double(), c.view(B * S, r).double(), torch.finfo(BF).eps / 2
    for got, a, b in ((dw, d2.t().contiguous(), c2), (dc.view(B * S, r), d2, w.double())):
        exact = a @ b
        assert ((got.double() - exact).abs() <= u * exact.abs() + (1 + u) * 8192 * F32 * (a.abs() @ b.abs())).all()


@pytest.mark.gpu
def test_training_and_sampling_of_a_group():
    """As used together: answers sampled token by token over a shared prefix get the outputs that the training form gives
    the whole answers, and the same for a latent cache."""
    g = torch.Generator().manual_seed(3)
    G, n, P, S, Hq, Hkv, D, dt = 1, 3, 200, 20, 4, 2, 128, BF
    q, k, v = (rnd(g, G * n, S, h, D, dt=dt, dev=GPU) for h in (Hq, Hkv, Hkv))
    pk, pv = (rnd(g, G, P, Hkv, D, dt=dt, dev=GPU) for _ in range(2))
    whole = ops.prefix_attention(q, k, v, pk, pv)
    u = torch.finfo(dt).eps / 2
    for t in (0, 7, S - 1):
        one = ops.prefix_attention_decode(q[:, t], k, v, torch.full((n,), t + 1, dtype=torch.int32, device=GPU), pk, pv)
        # both are within their own bound of the exact value: two roundings of each side, at most 4 u of sum p |v|
        assert float((one - whole[:, t]).abs().max()) <= 4 * u * float(v.abs().max())
    q, c, kr, w, _ = _train_inputs(4)
    whole = ops.latent_attention(q, c, kr, w)
    cache = torch.cat([c, kr], -1)
    for t in (0, 63, 149):
        one = ops.latent_attention_decode(q[:, t], cache, torch.full((2,), t + 1, dtype=torch.int32, device=GPU), w)
        # seven roundings between the two (kv, weights, output; absorbed query, weights, latent output, output)
        err = (one.double() - whole[:, t].double()).norm()
        assert float(err) <= 7 * u * float(whole[:, t].double().norm())


@pytest.mark.gpu
def test_same_inputs_same_bits():
    g = torch.Generator().manual_seed(5)
    q, k, v, do = (rnd(g, 6, 70, h, 64, dt=BF, dev=GPU) for h in (8, 2, 2, 8))
    pk, pv = (rnd(g, 2, 300, 2, 64, dt=BF, dev=GPU) for _ in range(2))

    def once():
        out, lse = ops.prefix_attn_fwd(q, k, v, pk, pv)
        lens = torch.full((6,), 70, dtype=torch.int32, device=GPU)
        return (out, lse, *ops.prefix_attn_bwd(do, q, k, v, pk, pv, out, lse),
                ops.prefix_attention_decode(q[:, 0], k, v, lens, pk, pv))

    a, b = once(), once()
    assert all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.gpu
def test_captured_graphs_replay():
    """Both training pairs and both single-token forms captured into two graphs, replayed on new inputs with eager work
    between the replays; every replay equals the eager result."""
    q, c, kr, w, do = _train_inputs(6)
    kv = (c.view(300, -1) @ w.t()).view(2, 150, 4, -1)
    cache = torch.cat([c, kr], -1)
    lens = torch.tensor([150, 33], dtype=torch.int32, device=GPU)
    g = torch.Generator().manual_seed(7)
    pq, pk_, pv_, pdo = (rnd(g, 4, 50, h, 64, dt=BF, dev=GPU) for h in (4, 2, 2, 4))
    xk, xv = (rnd(g, 1, 190, 2, 64, dt=BF, dev=GPU) for _ in range(2))
    plens = torch.tensor([50, 3, 0, 20], dtype=torch.int32, device=GPU)

    def latent():
        out, lse = ops.latent_attn_fwd(q, kv, kr, lens=lens)
        return (out, *ops.latent_attn_bwd(do, q, kv, kr, out, lse, lens=lens), ops.latent_attention_decode(q[:, 0], cache, lens, w))

    def prefix():
        out, lse = ops.prefix_attn_fwd(pq, pk_, pv_, xk, xv, lens=plens)
        return (out, *ops.prefix_attn_bwd(pdo, pq, pk_, pv_, xk, xv, out, lse, lens=plens),
                ops.prefix_attention_decode(pq[:, 0], pk_, pv_, plens, xk, xv))

    graphs = []
    for fn in (latent, prefix):
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            fn()
        torch.cuda.current_stream().wait_stream(s)
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs = fn()
        graphs.append((gr, outs, fn))
    for i in range(4):
        for t in (q, kv, kr, do, cache, pq, pk_, pv_, pdo, xk, xv):
            t.mul_(0.9 + 0.1 * i)
        lens[1] = 33 + i
        plens[2] = i
        for gr, _, _ in graphs:
            gr.replay()
        want = [fn() for _, _, fn in graphs]
        torch.cuda.synchronize()
        for (_, outs, _), ws in zip(graphs, want):
            assert all(torch.equal(a, b) for a, b in zip(outs, ws)), f"replay {i}"


@pytest.mark.gpu
def test_runs_on_the_current_stream():
    """Inputs made on a side stream and used there, without any synchronisation with the default stream."""
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        q, kv, kr = _latent_args(GPU, S=300)
        out, lse = ops.latent_attn_fwd(q, kv, kr)
        grads = ops.latent_attn_bwd(torch.ones_like(out), q, kv, kr, out, lse)
    s.synchronize()
    out2, lse2 = ops.latent_attn_fwd(q, kv, kr)
    grads2 = ops.latent_attn_bwd(torch.ones_like(out), q, kv, kr, out2, lse2)
    assert torch.equal(out, out2) and all(torch.equal(a, b) for a, b in zip(grads, grads2))


@pytest.mark.gpu
def test_two_calls_at_once():
    """Calls on two streams do not share a workspace: each gives what it gives alone."""
    args = [_train_inputs(i) for i in (10, 11)]
    lens = torch.tensor([150, 99], dtype=torch.int32, device=GPU)

    def whole(q, c, kr, w, do):
        leaves = [t.clone().requires_grad_(True) for t in (q, c, kr, w)]
        out = ops.latent_attention(*leaves, lens=lens)
        return (out.detach(), *torch.autograd.grad(out, leaves, do), ops.latent_attention_decode(q[:, 3], torch.cat([c, kr], -1), lens, w))

    alone = [whole(*a) for a in args]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(3):
        got = []
        for s, a in zip(streams, args):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                got.append(whole(*a))
        torch.cuda.synchronize()
        for x, y in zip(got, alone):
            assert all(torch.equal(i, j) for i, j in zip(x, y))


@pytest.mark.gpu
def test_differentiable_calls_are_captured():
    """Forward and gradients of both differentiable entry points in one graph, replayed on new values."""
    q, c, kr, w, do = (t.requires_grad_(i < 4) for i, t in enumerate(_train_inputs(12)))
    g = torch.Generator().manual_seed(13)
    x = [rnd(g, *s, dt=BF, dev=GPU).requires_grad_(True) for s in ((2, 40, 4, 64), (2, 40, 2, 64), (2, 40, 2, 64), (1, 90, 2, 64), (1, 90, 2, 64))]
    xdo = rnd(g, 2, 40, 4, 64, dt=BF, dev=GPU)

    def both():
        a, b = ops.latent_attention(q, c, kr, w), ops.prefix_attention(*x)
        return (a.detach(), b.detach(), *torch.autograd.grad(a, (q, c, kr, w), do), *torch.autograd.grad(b, x, xdo))

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        both()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, stream=s):
            outs = both()
    torch.cuda.current_stream().wait_stream(s)
    for i in range(3):
        with torch.no_grad():
            for t in (q, c, w, x[0], x[3]):
                t.mul_(0.8 + 0.2 * i)
        gr.replay()
        torch.cuda.synchronize()
        with torch.cuda.stream(s):  # the same library workspace as the captured calls
            want = both()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want)), i


@pytest.mark.gpu
def test_capture_of_a_backward_beside_an_eager_graph_is_refused():
    """The engine would make the default stream, on which the eager graph recorded the leaves' accumulation, wait for a
    captured kernel. The call raises, the capture goes on, and the backward is captured once the eager graph is gone."""
    q, c, kr, w, do = (t.requires_grad_(i < 4) for i, t in enumerate(_train_inputs(20)))
    g = torch.Generator().manual_seed(21)
    x = [rnd(g, *s, dt=BF, dev=GPU).requires_grad_(True) for s in ((2, 40, 4, 64), (2, 40, 2, 64), (2, 40, 2, 64), (1, 90, 2, 64), (1, 90, 2, 64))]
    xdo = rnd(g, 2, 40, 4, 64, dt=BF, dev=GPU)
    for fn, leaves, grad, name in ((ops.latent_attention, (q, c, kr, w), do, "latent_attention"), (ops.prefix_attention, x, xdo, "prefix_attention")):
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            torch.autograd.grad(fn(*leaves), leaves, grad)
        torch.cuda.current_stream().wait_stream(s)
        eager = fn(*leaves)
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, stream=s):
            out = fn(*leaves)
            with pytest.raises(RuntimeError, match=name + ": this backward is captured"):
                torch.autograd.grad(out, leaves, grad)
        gr.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager)
        want = torch.autograd.grad(eager, leaves, grad)
        del eager, out, gr
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, stream=s):
            got = torch.autograd.grad(fn(*leaves), leaves, grad)
        for _ in range(2):
            gr.replay()
            torch.cuda.synchronize()
            u = torch.finfo(BF).eps / 2  # a GEMM may be another one on the stream's own workspace
            assert all(float((a.double() - b.double()).norm()) <= 2 * u * float(b.double().norm()) for a, b in zip(got, want))


@pytest.mark.gpu
def test_odd_arguments():
    """Lengths outside the tensors' count as their ends; views that a GEMM cannot read in place; no gradient to record."""
    q, c, kr, w, do = _train_inputs(14)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=GPU)  # noqa: E731
    full = ops.latent_attention(q, c, kr, w, lens=i32(150, 0))
    assert torch.equal(full, ops.latent_attention(q, c, kr, w, lens=i32(1 << 30, -5)))
    cache = torch.cat([c, kr], -1)
    assert torch.equal(ops.latent_attention_decode(q[:, 0], cache, i32(1 << 30, -5), w), ops.latent_attention_decode(q[:, 0], cache, i32(150, 0), w))
    pk = rnd(torch.Generator().manual_seed(15), 1, 30, 2, 64, dt=BF, dev=GPU)
    k, pq = pk[:, :9].repeat(2, 1, 1, 1), torch.ones(2, 4, 64, dtype=BF, device=GPU)
    a = ops.prefix_attention_decode(pq, k, k, i32(99, -1), pk, pk, i32(77))
    assert torch.equal(a, ops.prefix_attention_decode(pq, k, k, i32(9, 0), pk, pk))
    # rows of a wider tensor, and contiguous weights at an odd address
    wide = torch.zeros(2, 150, c.shape[-1] + 8, dtype=BF, device=GPU)
    wide[..., :c.shape[-1]] = c
    odd = torch.zeros(w.numel() + 1, dtype=BF, device=GPU)[1:].view_as(w).copy_(w)
    leaves = [t.clone().requires_grad_(True) for t in (q, c, kr, w)]
    views = [leaves[0].detach(), wide[..., :c.shape[-1]], kr, odd]
    views = [v.detach().requires_grad_(True) for v in views]
    res = []
    for x in (leaves, views):
        out = ops.latent_attention(*x)
        res.append((out.detach(), *torch.autograd.grad(out.sum(), x)))  # an expanded dO
    u = torch.finfo(BF).eps / 2
    for x, y in zip(*res):  # another GEMM may be picked for other strides: each result within its 6 u of the exact one
        assert float((x.double() - y.double()).norm()) <= 12 * u * float(x.double().norm())
    with torch.no_grad():
        a = ops.latent_attention(q, c, kr, w)
    with torch.inference_mode():
        b = ops.latent_attention(q, c, kr, w)
        ops.prefix_attention(pq.unsqueeze(1), k[:, :1], k[:, :1], pk, pk)
    assert torch.equal(a, b) and not a.requires_grad
    assert torch.equal(a, ops.latent_attention(*leaves))


@pytest.mark.gpu
def test_gradients_that_start_anywhere():
    """The output behind a single element in a concatenation: its gradient is contiguous from an odd address on."""
    q, c, kr, w, do = _train_inputs(17)
    g = torch.Generator().manual_seed(18)
    x = [rnd(g, *s, dt=BF, dev=GPU) for s in ((2, 40, 4, 64), (2, 40, 2, 64), (2, 40, 2, 64), (1, 90, 2, 64), (1, 90, 2, 64))]
    for fn, args, grad in ((ops.latent_attention, (q, c, kr, w), do), (ops.prefix_attention, x, rnd(g, 2, 40, 4, 64, dt=BF, dev=GPU))):
        leaves = [t.clone().requires_grad_(True) for t in args]
        want = torch.autograd.grad(fn(*leaves), leaves, grad)
        one = torch.zeros(1, dtype=BF, device=GPU, requires_grad=True)
        whole = torch.cat([one, fn(*leaves).flatten()])
        got = torch.autograd.grad(whole, leaves, torch.cat([one.detach(), grad.flatten()]))
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.gpu
def test_strides_of_dimensions_of_one():
    """A dimension of one may carry any stride: 1 here, as a permutation of a trailing one gives it."""
    g = torch.Generator().manual_seed(25)
    one = lambda t: t.unsqueeze(-1).movedim(-1, 1)  # noqa: E731  [B, H, D] -> [B, 1, H, D] with a row stride of 1
    x = [rnd(g, 3, h, d, dt=BF, dev=GPU) for h, d in ((2, 96), (2, 128), (2, 64))]
    kr = rnd(g, 3, 32, dt=BF, dev=GPU)
    res = []
    for f in (one, lambda t: t.unsqueeze(1).contiguous()):
        q, kv, do = (f(t) for t in x)
        assert f is not one or q.stride(1) == kv.stride(1) == do.stride(1) == f(kr).stride(1) == 1
        out, lse = ops.latent_attn_fwd(q, kv, f(kr))
        p = [f(t[..., :64].contiguous()) for t in x]
        pk = f(x[0][:1, :, :64].contiguous())
        po, plse = ops.prefix_attn_fwd(*p, pk, pk)
        lens = torch.tensor([1, 0, 1], dtype=torch.int32, device=GPU)
        cache, w = f(torch.cat([x[1], x[1], kr.unsqueeze(1).expand(3, 2, 32)], -1)[:, 0].contiguous()), torch.ones(256, 256, dtype=BF, device=GPU) / 16
        res.append((out, lse, *ops.latent_attn_bwd(do, q, kv, f(kr), out, lse), po, plse, *ops.prefix_attn_bwd(p[2], *p, pk, pk, po, plse),
                    ops.latent_attention_decode(x[0], cache, lens, w), ops.prefix_attention_decode(p[0][:, 0], p[1], p[2], lens, pk, pk)))
    assert all(torch.equal(a, b) for a, b in zip(*res))


@pytest.mark.gpu
def test_rows_beyond_32_bit_offsets():
    """Row strides and cache lengths whose byte offsets pass 32 bits."""
    dn, dr, dv = HALF
    g = torch.Generator().manual_seed(8)
    S, H = 520, 2
    buf = torch.empty(S, 1 << 22, dtype=BF, device=GPU)  # 4.4 GB
    kv = buf[:, -H * (dn + dv):].view(1, S, H, dn + dv)
    kv.copy_(rnd(g, 1, S, H, dn + dv, dt=BF, dev=GPU))
    q, kr, do = (rnd(g, *s, dt=BF, dev=GPU) for s in ((1, S, H, dn + dr), (1, S, dr), (1, S, H, dv)))
    out, lse = ops.latent_attn_fwd(q, kv, kr)
    a = (out, *ops.latent_attn_bwd(do, q, kv, kr, out, lse))
    out2, lse2 = ops.latent_attn_fwd(q, kv.contiguous(), kr)
    b = (out2, *ops.latent_attn_bwd(do, q, kv.contiguous(), kr, out2, lse2))
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    del buf, kv
    # a cache of 3.9 million tokens, 4.5 GB: zeros but for the last 40, which a scaled query picks out
    r, L, n = 512, 3_900_000, 40
    w = rnd(g, H * (dn + dv), r, dt=BF, dev=GPU, std=r ** -0.5)
    cache = torch.zeros(1, L, r + dr, dtype=BF, device=GPU)
    cache[:, -n:] = rnd(g, 1, n, r + dr, dt=BF, dev=GPU)
    q = rnd(g, 1, H, dn + dr, dt=BF, dev=GPU) * 8
    got = ops.latent_attention_decode(q, cache, torch.tensor([L], dtype=torch.int32, device=GPU), w).double()
    w3, c = w.double().view(H, dn + dv, r), cache[0, -n:].double()
    for h in range(H):
        s = (c[:, :r] @ (w3[h, :dn].t() @ q[0, h, :dn].double()) + c[:, r:] @ q[0, h, dn:].double()) * (dn + dr) ** -0.5
        e = torch.exp(s)
        want = w3[h, dn:] @ ((e / (e.sum() + (L - n))) @ c[:, :r])
        # the absorbed query's rounding moves a score by at most u sum |qa| |c| scale
        qa = (w3[h, :dn].t() @ q[0, h, :dn].double()).abs()
        u = torch.finfo(BF).eps / 2
        off = float((c[:, :r].abs() @ qa).max()) * u * (dn + dr) ** -0.5
        assert float((got[0, h] - want).norm()) <= (3 * u + math.expm1(2 * off)) * float(want.norm())


@pytest.mark.gpu
def test_group_of_millions():
    """A group whose sequences times the parts they are cut into (1024 for so short a prefix) pass 31 bits. The prefix's
    value gradient sums over all of them, positive terms: the weights are off by at most u each, the result once more, and
    an fp32 chain runs over a part's sequences and then over the parts. Scores of sum |q| |k| < 96 are off by at most (D + 8)
    2^-24 96 / 8, a weight by twice that: 2^-13."""
    n, D, P, parts = 2_200_000, 64, 3, 1024
    g = torch.Generator(device=GPU).manual_seed(16)
    q, k, v, do = (torch.randn(n, 1, 1, D, generator=g, device=GPU).to(BF) for _ in range(4))
    do = do.abs()
    pk, pv = (torch.randn(1, P, 1, D, generator=g, device=GPU).to(BF) for _ in range(2))
    assert n * (parts - 1) > 2 ** 31
    out, lse = ops.prefix_attn_fwd(q, k, v, pk, pv)
    dv, dpv = ops.prefix_attn_bwd(do, q, k, v, pk, pv, out, lse)[2::2]
    q, k, do = (t.view(n, D).double() for t in (q, k, do))
    p = torch.softmax(torch.cat([q @ pk.view(P, D).double().t(), (q * k).sum(-1, keepdim=True)], 1) * D ** -0.5, -1)
    assert float((q * k).abs().sum(-1).max()) < 96 and float((q.abs() @ pk.view(P, D).double().abs().t()).max()) < 96
    u = torch.finfo(BF).eps / 2
    want = p[:, :P].t() @ do
    chain = (n / parts + parts) * F32
    assert ((dpv.view(P, D).double() - want).abs() <= (2 * u + u * u + 2 ** -13 + chain) * want).all()
    own = p[:, P:] * do
    assert ((dv.view(n, D).double() - own).abs() <= (2 * u + u * u + 2 ** -13) * own).all()


@pytest.mark.gpu
def test_kernels_refuse_what_they_cannot_do():
    q, kv, kr = _latent_args(GPU)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=GPU)  # noqa: E731
    out, lse = ops.latent_attn_fwd(q, kv, kr)
    bad = [
        lambda: ops.latent_attn_fwd(q.float(), kv.float(), kr.float()),
        lambda: ops.latent_attn_fwd(q.half(), kv, kr),
        lambda: ops.latent_attn_fwd(q, kv[:1], kr),
        lambda: ops.latent_attn_fwd(q, kv[..., :96], kr),
        lambda: ops.latent_attn_fwd(q, kv, kr[..., :16]),
        lambda: ops.latent_attn_fwd(q, kv.cpu(), kr),
        lambda: ops.latent_attn_fwd(q, kv, kr, lens=i32(8, 8).long()),
        lambda: ops.latent_attn_fwd(q, kv, kr, lens=i32(8)),
        lambda: ops.latent_attn_fwd(q, kv, kr, lens=i32(8, 8).cpu()),
        lambda: ops.latent_attn_fwd(q, kv, kr, softmax_scale=0.0),
        lambda: ops.latent_attn_fwd(q, kv, kr, softmax_scale=1e-30),
        lambda: ops.latent_attn_fwd(q, kv, kr, softmax_scale=1e30),
        lambda: ops.latent_attention(q, kr[..., :0], kr, kr.new_zeros(256, 0)),
        lambda: ops.latent_attention(q, kr[..., :12], kr, kr.new_zeros(256, 12)),
        lambda: ops.latent_attn_fwd(q, kv, kr, softmax_scale=float("nan")),
        lambda: ops.latent_attn_fwd(q.transpose(2, 3), kv, kr),
        lambda: ops.latent_attn_fwd(torch.zeros(2, 8, 2, 97, dtype=BF, device=GPU)[..., 1:], kv, kr),
        lambda: ops.latent_attn_bwd(out[:1], q, kv, kr, out, lse),
        lambda: ops.latent_attn_bwd(out, q, kv, kr, out, lse.double()),
        lambda: ops.latent_attn_bwd(out, q, kv, kr, out.transpose(1, 2).contiguous().transpose(1, 2), lse),
    ]
    cache, w = torch.zeros(2, 9, 256 + 32, dtype=BF, device=GPU), torch.zeros(2 * 128, 256, dtype=BF, device=GPU)
    one = q[:, 0]
    bad += [
        lambda: ops.latent_attention_decode(one, cache, i32(1, 2), w[:, :248]),
        lambda: ops.latent_attention_decode(one, cache, i32(1, 2), w[:-1]),
        lambda: ops.latent_attention_decode(one, cache[:1], i32(1, 2), w),
        lambda: ops.latent_attention_decode(one, cache, i32(1), w),
        lambda: ops.latent_attention_decode(one, cache.half(), i32(1, 2), w),
        lambda: ops.latent_attention_decode(one, cache[..., :-1], i32(1, 2), w),
    ]
    pq, k, pk = (torch.zeros(*s, dtype=BF, device=GPU) for s in ((4, 8, 4, 64), (4, 8, 2, 64), (2, 5, 2, 64)))
    bad += [
        lambda: ops.prefix_attn_fwd(pq[..., :32], k[..., :32], k[..., :32], pk[..., :32], pk[..., :32]),
        lambda: ops.prefix_attn_fwd(pq, k, k[:, :4], pk, pk),
        lambda: ops.prefix_attn_fwd(pq, k, k, pk, pk[:, :4]),
        lambda: ops.prefix_attn_fwd(pq, k, k, pk, pk, prefix_lens=i32(1, 2, 3)),
        lambda: ops.prefix_attn_fwd(pq, k.half(), k.half(), pk, pk),
        lambda: ops.prefix_attention_decode(pq[:, 0], k, k, i32(1, 2, 3), pk, pk),
        lambda: ops.prefix_attention_decode(pq[:, 0], k, k[:3], i32(1, 2, 3, 4), pk, pk),
    ]
    for i, call in enumerate(bad):
        with pytest.raises((RuntimeError, ValueError, NotImplementedError)):
            call()
            pytest.fail(f"call {i} was not refused")


@pytest.mark.gpu
def test_empty_tensors():
    q, kv, kr = _latent_args(GPU)
    out, lse = ops.latent_attn_fwd(q[:0], kv[:0], kr[:0])
    assert out.shape == (0, 8, 2, 64) and all(t.numel() == 0 for t in ops.latent_attn_bwd(out, q[:0], kv[:0], kr[:0], out, lse))
    out, lse = ops.latent_attn_fwd(q[:, :0], kv[:, :0], kr[:, :0])
    assert out.shape == (2, 0, 2, 64)
    cache, w = torch.zeros(2, 0, 288, dtype=BF, device=GPU), torch.zeros(256, 256, dtype=BF, device=GPU)
    assert not ops.latent_attention_decode(q[:, 0], cache, torch.zeros(2, dtype=torch.int32, device=GPU), w).any()
    pq, k, pk = (torch.zeros(*s, dtype=BF, device=GPU) for s in ((2, 0, 4, 64), (2, 0, 2, 64), (1, 5, 2, 64)))
    out, lse = ops.prefix_attn_fwd(pq, k, k, pk, pk)
    g = ops.prefix_attn_bwd(out, pq, k, k, pk, pk, out, lse)
    assert g[3].shape == pk.shape and not g[3].any() and not g[4].any()
    none = ops.prefix_attention_decode(torch.ones(2, 4, 64, dtype=BF, device=GPU), k, k, torch.zeros(2, dtype=torch.int32, device=GPU), pk[:, :0], pk[:, :0])
    assert none.shape == (2, 4, 64) and not none.any()


@pytest.mark.gpu
def test_nan_reaches_the_output():
    """A NaN in a live row is a NaN in what depends on it (the NaN trap sees it), never a zero."""
    q, kv, kr = _latent_args(GPU, S=70)
    kv[0, 3, 0, 0] = float("nan")
    out, _ = ops.latent_attn_fwd(q, kv, kr)
    assert out[0, 3:, 0].isnan().all() and not out[0, :, 1].isnan().any() and not out[1].isnan().any()
    cache, w = torch.ones(2, 70, 288, dtype=BF, device=GPU), torch.ones(256, 256, dtype=BF, device=GPU)
    cache[0, 5, 7] = float("nan")
    o = ops.latent_attention_decode(q[:, 0] * 0.01, cache, torch.tensor([70, 70], dtype=torch.int32, device=GPU), w * 0.01)
    assert o[0].isnan().all() and not o[1].isnan().any()
    k = torch.ones(2, 9, 2, 64, dtype=BF, device=GPU)
    pk = k[:1].clone()
    k[1, 2, 1, 5] = float("nan")
    qq = torch.ones(2, 4, 64, dtype=BF, device=GPU)
    o = ops.prefix_attention_decode(qq, k, k.nan_to_num(), torch.tensor([9, 9], dtype=torch.int32, device=GPU), pk, pk)
    assert o[1, 2:].isnan().all() and not o[1, :2].isnan().any() and not o[0].isnan().any()


@pytest.mark.gpu
def test_native_kernels_are_registered():
    assert _native.hip_available() and hasattr(torch.ops.dlgm, "latent_attn_decode") and hasattr(torch.ops.dlgm, "prefix_attn_bwd")
