"""What the shared-key attention operators are measured on: latent attention (keys and values from one latent vector a
token) and attention of a batch over a shared prefix, each in its training form (forward and backward) and in its
single-token form over a cache.

``run`` computes either the plain form (elementary torch operations in 32 bits) or, where ``own`` is true, makes the
calls of the framework. ``exact`` gives the same outputs in 64 bits, one sequence and head at a time."""
from __future__ import annotations

import math

import torch

own = False

# (heads' nope dim, rope dim, value dim) of latent attention
LAYOUTS = {"wide": (128, 64, 128), "half": (64, 32, 64)}
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def listed():
    return [
        # a unit test's or a smoke run's layer
        dict(name="latent-train-small", op="latent_train", B=2, S=128, H=4, layout="half", r=256, ragged=False,
             dtype="bf16"),
        # a padded fine-tuning batch of odd length
        dict(name="latent-train-odd", op="latent_train", B=3, S=777, H=8, layout="wide", r=512, ragged=True,
             dtype="fp16"),
        # one layer of a pre-training micro-batch at the sequence lengths of the benchmark models
        dict(name="latent-train-4k", op="latent_train", B=2, S=4096, H=32, layout="wide", r=512, ragged=False,
             dtype="bf16"),
        dict(name="latent-train-8k", op="latent_train", B=1, S=8192, H=32, layout="wide", r=512, ragged=False,
             dtype="bf16"),
        # one request being answered, where latency counts
        dict(name="latent-decode-one", op="latent_decode", B=1, L=1000, H=8, layout="half", r=256, ragged=False,
             dtype="bf16"),
        # a served batch of unequal lengths, idle slots among it
        dict(name="latent-decode-batch", op="latent_decode", B=32, L=4000, H=32, layout="wide", r=512, ragged=True,
             dtype="bf16"),
        # many heads over long caches
        dict(name="latent-decode-long", op="latent_decode", B=32, L=16384, H=128, layout="wide", r=512, ragged=False,
             dtype="bf16"),
        # four short answers to one prompt
        dict(name="prefix-train-odd", op="prefix_train", G=2, n=4, P=333, S=200, Hq=4, Hkv=2, D=64, ragged=True,
             dtype="fp16"),
        # a group of sampled answers being trained on
        dict(name="prefix-train-group", op="prefix_train", G=1, n=8, P=4096, S=1024, Hq=32, Hkv=8, D=128, ragged=False,
             dtype="bf16"),
        # the first tokens of a few answers
        dict(name="prefix-decode-small", op="prefix_decode", G=1, n=4, P=500, L=60, Hq=8, Hkv=8, D=128, ragged=False,
             dtype="bf16"),
        # a group of answers being sampled
        dict(name="prefix-decode-group", op="prefix_decode", G=1, n=16, P=8000, L=700, Hq=32, Hkv=8, D=128,
             ragged=True, dtype="bf16"),
        # several large groups behind long prompts
        dict(name="prefix-decode-large", op="prefix_decode", G=2, n=64, P=16384, L=1024, Hq=32, Hkv=8, D=128,
             ragged=True, dtype="bf16"),
    ]


def _spread(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def _cost(case):
    w = work(case)
    return max(w["bytes"] / 8e12, w["flops"] / 2.5e15)


def draw(rng):
    op = rng.choice(["latent_train", "latent_decode", "prefix_train", "prefix_decode"])
    case = dict(op=op, dtype=rng.choice(["bf16", "bf16", "fp16"]), ragged=rng.random() < 0.5)
    if op == "latent_train":
        case.update(B=rng.randint(1, 4), S=_spread(rng, 16, 8192), H=rng.choice([2, 4, 8, 32]),
                    layout=rng.choice(["wide", "wide", "half"]), r=rng.choice([128, 256, 512]))
    elif op == "latent_decode":
        case.update(B=_spread(rng, 1, 128), L=_spread(rng, 1, 16384), H=rng.choice([2, 8, 20, 32, 64, 128]),
                    layout=rng.choice(["wide", "wide", "half"]), r=rng.choice([256, 512]))
    else:
        hq, hkv, d = rng.choice([(32, 8, 128), (8, 8, 128), (4, 2, 64), (12, 12, 64)])
        case.update(G=rng.randint(1, 3), n=_spread(rng, 2, 8 if op == "prefix_train" else 64), Hq=hq, Hkv=hkv, D=d)
        if op == "prefix_train":
            case.update(P=_spread(rng, 1, 4096), S=_spread(rng, 16, 1024))
        else:
            case.update(P=_spread(rng, 1, 16384), L=_spread(rng, 1, 2048))
    most = max(_cost(c) for c in listed() if c["op"] == op)
    key = "S" if "S" in case else "L"
    while _cost(case) > most:  # a drawn case costs no more than the largest listed one
        case[key if case[key] > 1 else "P"] //= 2
    return case


def _lens(case, count, most):
    """Lengths of a padded batch: between 1/16 of the whole and the whole; in a served batch a slot may be idle."""
    if not case["ragged"]:
        return [most] * count
    idle = case["op"].endswith("decode")
    return [0 if idle and b % 16 == 9 else max(1, most * (16 - 7 * b % 16) // 16) for b in range(count)]


def _sizes(case):
    dn, dr, dv = LAYOUTS[case["layout"]]
    return dn, dr, dv, case["r"], case["H"]


def prepare(case, seed):
    dev, dt = torch.device("cuda"), DTYPES[case["dtype"]]
    g = torch.Generator(device=dev)
    g.manual_seed(seed)

    def rnd(*shape, std=1.0):
        return (torch.randn(*shape, generator=g, device=dev) * std).to(dt)

    st = {"op": case["op"]}
    if case["op"].startswith("latent"):
        dn, dr, dv, r, H = _sizes(case)
        B = case["B"]
        st["w"] = rnd(H * (dn + dv), r, std=r ** -0.5)
        if case["op"] == "latent_train":
            S = case["S"]
            st["q"], st["c"], st["kr"] = rnd(B, S, H, dn + dr), rnd(B, S, r), rnd(B, S, dr)
            st["dout"] = rnd(B, S, H, dv)
            for k in ("q", "c", "kr", "w"):
                st[k].requires_grad_(True)
            most = S
        else:
            most = case["L"]
            st["q"], st["cache"] = rnd(B, H, dn + dr), rnd(B, most, r + dr)
    else:
        G, n, P, Hq, Hkv, D = (case[k] for k in ("G", "n", "P", "Hq", "Hkv", "D"))
        B = G * n
        st["pk"], st["pv"] = rnd(G, P, Hkv, D), rnd(G, P, Hkv, D)
        if case["op"] == "prefix_train":
            S = case["S"]
            st["q"], st["k"], st["v"] = rnd(B, S, Hq, D), rnd(B, S, Hkv, D), rnd(B, S, Hkv, D)
            st["dout"] = rnd(B, S, Hq, D)
            for k in ("q", "k", "v", "pk", "pv"):
                st[k].requires_grad_(True)
            most = S
        else:
            most = case["L"]
            st["q"], st["k"], st["v"] = rnd(B, Hq, D), rnd(B, most, Hkv, D), rnd(B, most, Hkv, D)
    # a training batch without padding has no lengths to pass; a cache always has them
    whole = case["op"].endswith("train") and not case["ragged"]
    st["lens"] = None if whole else torch.tensor(_lens(case, B, most), dtype=torch.int32, device=dev)
    return st


def run(st):
    return {"latent_train": _latent_train, "latent_decode": _latent_decode, "prefix_train": _prefix_train,
            "prefix_decode": _prefix_decode}[st["op"]](st)


def _softmax(s):
    """Softmax over the last axis; a row with nothing but -inf gives zeros."""
    e = torch.exp(s - s.amax(-1, keepdim=True).clamp_min(-1e30))
    return e / e.sum(-1, keepdim=True).clamp_min(1e-30)


def _seen(S, lens, B, device):
    """[B, S, S]: whether query row i of sequence b sees key j."""
    i = torch.arange(S, device=device)
    ok = (i[None, :] <= i[:, None]).expand(B, S, S)
    if lens is not None:
        inside = i[None, :] < lens[:, None]
        ok = ok & inside[:, None, :] & inside[:, :, None]
    return ok


def _latent_train(st):
    q, c, kr, w, do, lens = (st[k] for k in ("q", "c", "kr", "w", "dout", "lens"))
    if own:
        from distributed_llm_training_gpu_manager_amd import ops

        out = ops.latent_attention(q, c, kr, w, lens=lens)
        dq, dc, dkr, dw = torch.autograd.grad(out, (q, c, kr, w), do)
        return {"out": out.detach(), "dq": dq, "dc": dc, "dkr": dkr, "dw": dw}
    dt = q.dtype
    q, c, kr, w, do = (t.detach().float() for t in (q, c, kr, w, do))
    B, S, H, dqk = q.shape
    dr, r, dv = kr.shape[-1], c.shape[-1], do.shape[-1]
    dn, scale = dqk - dr, dqk ** -0.5
    kv = (c.reshape(B * S, r) @ w.t()).view(B, S, H, dn + dv)
    k = torch.cat([kv[..., :dn], kr[:, :, None].expand(B, S, H, dr)], -1).transpose(1, 2).contiguous()
    v = kv[..., dn:].transpose(1, 2).contiguous()
    q, do = q.transpose(1, 2).contiguous(), do.transpose(1, 2).contiguous()
    s = (q @ k.transpose(-1, -2)) * scale
    p = _softmax(s.masked_fill_(~_seen(S, lens, B, q.device)[:, None], float("-inf")))
    del s
    out = p @ v
    dp = do @ v.transpose(-1, -2)
    ds = p * (dp - (p * dp).sum(-1, keepdim=True)) * scale
    dq, dk, dvv = ds @ k, ds.transpose(-1, -2) @ q, p.transpose(-1, -2) @ do
    dkv = torch.cat([dk[..., :dn], dvv], -1).transpose(1, 2).reshape(B * S, H * (dn + dv))
    return {"out": out.transpose(1, 2).to(dt).contiguous(), "dq": dq.transpose(1, 2).to(dt).contiguous(),
            "dc": (dkv @ w).view(B, S, r).to(dt), "dkr": dk[..., dn:].sum(1).to(dt), "dw": (dkv.t() @ c.reshape(B * S, r)).to(dt)}


def _latent_decode(st):
    q, cache, w, lens = (st[k] for k in ("q", "cache", "w", "lens"))
    if own:
        from distributed_llm_training_gpu_manager_amd import ops

        return ops.latent_attention_decode(q, cache, lens, w)
    dt = q.dtype
    q, cache, w = q.float(), cache.float(), w.float()
    B, H, dqk = q.shape
    r, L = w.shape[1], cache.shape[1]
    dn = dqk - (cache.shape[-1] - r)
    w = w.view(H, -1, r)
    c = cache[..., :r]
    qa = (q[..., :dn].transpose(0, 1) @ w[:, :dn]).transpose(0, 1)
    s = (torch.cat([qa, q[..., dn:]], -1) @ cache.transpose(1, 2)) * dqk ** -0.5
    gone = torch.arange(L, device=q.device)[None, :] >= lens[:, None]
    ol = _softmax(s.masked_fill(gone[:, None], float("-inf"))) @ c
    return (ol.transpose(0, 1) @ w[:, dn:].transpose(1, 2)).transpose(0, 1).to(dt).contiguous()


def _prefix_train(st):
    q, k, v, pk, pv, do, lens = (st[x] for x in ("q", "k", "v", "pk", "pv", "dout", "lens"))
    if own:
        from distributed_llm_training_gpu_manager_amd import ops

        out = ops.prefix_attention(q, k, v, pk, pv, lens=lens)
        dq, dk, dv, dpk, dpv = torch.autograd.grad(out, (q, k, v, pk, pv), do)
        return {"out": out.detach(), "dq": dq, "dk": dk, "dv": dv, "dpk": dpk, "dpv": dpv}
    dt = q.dtype
    q, k, v, pk, pv, do = (t.detach().float() for t in (q, k, v, pk, pv, do))
    B, S, Hq, D = q.shape
    G, P, Hkv = pk.shape[:3]
    n, rep, scale = B // G, Hq // Hkv, D ** -0.5

    def rows(t):  # [B, S, Hq, D] -> [G, Hkv, n, rep * S, D]
        return t.view(G, n, S, Hkv, rep, D).permute(0, 3, 1, 4, 2, 5).reshape(G, Hkv, n, rep * S, D)

    def back(t):  # the other way
        return t.view(G, Hkv, n, rep, S, D).permute(0, 2, 4, 1, 3, 5).reshape(B, S, Hq, D)

    def keys(t):  # [B, S, Hkv, D] -> [G, Hkv, n, S, D]
        return t.view(G, n, S, Hkv, D).permute(0, 3, 1, 2, 4).contiguous()

    qr, dor, ko, vo = rows(q), rows(do), keys(k), keys(v)
    pkh, pvh = pk.transpose(1, 2).contiguous(), pv.transpose(1, 2).contiguous()

    def both(a, kp, kw):  # products of the rows with the prefix and with their own keys, side by side
        ap = (a.view(G, Hkv, -1, D) @ kp.transpose(-1, -2)).view(G, Hkv, n, rep * S, P)
        return torch.cat([ap, a @ kw.transpose(-1, -2)], -1)

    ok = _seen(S, lens, B, q.device)
    seen = torch.cat([ok.any(-1, keepdim=True).expand(B, S, P), ok], -1)  # a padded row sees nothing at all
    seen = seen.view(G, 1, n, 1, S, P + S).expand(G, 1, n, rep, S, P + S).reshape(G, 1, n, rep * S, P + S)
    p = _softmax((both(qr, pkh, ko) * scale).masked_fill_(~seen, float("-inf")))

    def onto(a, kp, kw):  # the weights' product with the prefix's rows and with the sequence's own
        return (a[..., :P].reshape(G, Hkv, -1, P) @ kp).view(G, Hkv, n, rep * S, D) + a[..., P:] @ kw

    out = onto(p, pvh, vo)
    dp = both(dor, pvh, vo)
    ds = p * (dp - (p * dp).sum(-1, keepdim=True)) * scale
    del dp

    def down(a, x):  # a^T x: [prefix, own]
        ap = a[..., :P].reshape(G, Hkv, -1, P).transpose(-1, -2) @ x.view(G, Hkv, -1, D)
        return ap.transpose(1, 2).to(dt).contiguous(), (a[..., P:].transpose(-1, -2) @ x).permute(0, 2, 3, 1, 4).reshape(B, S, Hkv, D).to(dt)

    dq = onto(ds, pkh, ko)
    dpk, dk = down(ds, qr)
    dpv, dv = down(p, dor)
    return {"out": back(out).to(dt), "dq": back(dq).to(dt), "dk": dk, "dv": dv, "dpk": dpk, "dpv": dpv}


def _prefix_decode(st):
    q, k, v, pk, pv, lens = (st[x] for x in ("q", "k", "v", "pk", "pv", "lens"))
    if own:
        from distributed_llm_training_gpu_manager_amd import ops

        return ops.prefix_attention_decode(q, k, v, lens, pk, pv)
    dt = q.dtype
    q, k, v, pk, pv = (t.float() for t in (q, k, v, pk, pv))
    B, Hq, D = q.shape
    G, P, Hkv = pk.shape[:3]
    L, n, rep = k.shape[1], B // G, Hq // Hkv
    qr = q.view(B, Hkv, rep, D)
    qp = q.view(G, n, Hkv, rep, D).transpose(1, 2).reshape(G, Hkv, n * rep, D)
    sp = qp @ pk.permute(0, 2, 3, 1)
    sp = sp.view(G, Hkv, n, rep, P).transpose(1, 2).reshape(B, Hkv, rep, P)
    gone = torch.arange(L, device=q.device)[None, :] >= lens[:, None]
    so = (qr @ k.permute(0, 2, 3, 1)).masked_fill(gone[:, None, None], float("-inf"))
    p = _softmax(torch.cat([sp, so], -1) * D ** -0.5)
    pp = p[..., :P].reshape(G, n, Hkv, rep, P).transpose(1, 2).reshape(G, Hkv, n * rep, P)
    op = (pp @ pv.transpose(1, 2)).view(G, Hkv, n, rep, D).transpose(1, 2).reshape(B, Hkv, rep, D)
    return (op + p[..., P:] @ v.transpose(1, 2)).reshape(B, Hq, D).to(dt)


def work(case):
    op = case["op"]
    if op.startswith("latent"):
        dn, dr, dv, r, H = _sizes(case)
        B = case["B"]
        wn = H * (dn + dv) * r
        if op == "latent_train":
            T = B * case["S"]
            pairs = sum(n * (n + 1) // 2 for n in _lens(case, B, case["S"]))
            per = T * (H * (dn + dr) + r + dr)
            return {"bytes": 2.0 * (2 * per + 2 * T * H * dv + 2 * wn),
                    "flops": 2.0 * pairs * H * (4 * (dn + dr) + 3 * dv) + 6.0 * T * wn}
        lens = _lens(case, B, case["L"])
        rows = sum(lens)
        return {"bytes": 2.0 * (rows * (r + dr) + wn + B * H * (dn + dr + dv)) + 4 * B,
                "flops": 2.0 * H * rows * (2 * r + dr) + 2.0 * B * wn}
    G, n, P, Hq, Hkv, D = (case[k] for k in ("G", "n", "P", "Hq", "Hkv", "D"))
    B = G * n
    if op == "prefix_train":
        lens = _lens(case, B, case["S"])
        T = B * case["S"]
        pairs = sum(m * (m + 1) // 2 + m * P for m in lens)
        return {"bytes": 2.0 * D * (4 * T * Hq + 4 * T * Hkv + 4 * G * P * Hkv), "flops": 14.0 * pairs * Hq * D}
    lens = _lens(case, B, case["L"])
    return {"bytes": 2.0 * D * (2 * Hkv * (G * P + sum(lens)) + 2 * B * Hq) + 4 * B,
            "flops": 4.0 * D * Hq * (B * P + sum(lens))}


def exact(case, seed):
    """The definition in 64 bits, one sequence and one (shared) head at a time; gradients by differentiation."""
    st = prepare(case, seed)
    f = {k: v.detach().double() for k, v in st.items() if torch.is_tensor(v) and v.is_floating_point()}
    q = f["q"]
    B = q.shape[0]
    most = case["S"] if "S" in case else case["L"]
    lens = _lens(case, B, most)
    if case["op"].startswith("latent"):
        dn, dr, dv, r, H = _sizes(case)
        w = f["w"].view(H, dn + dv, r)
        scale = 1.0 / math.sqrt(dn + dr)
        if case["op"] == "latent_decode":
            out = q.new_zeros(B, H, dv)
            for b, m in enumerate(lens):
                if m:
                    c, kr = f["cache"][b, :m, :r], f["cache"][b, :m, r:]
                    for h in range(H):
                        # keys and values are expanded here; expanding W instead of the cache gives the same numbers
                        a = torch.softmax((c @ (w[h, :dn].t() @ q[b, h, :dn]) + kr @ q[b, h, dn:]) * scale, 0)
                        out[b, h] = w[h, dn:] @ (a @ c)
            return out
        res = {"out": q.new_zeros(f["dout"].shape), "dq": torch.zeros_like(q), "dc": torch.zeros_like(f["c"]),
               "dkr": torch.zeros_like(f["kr"]), "dw": torch.zeros_like(w)}
        for b, m in enumerate(lens):
            above = torch.ones(m, m, dtype=torch.bool, device=q.device).triu(1)
            for h in range(H):
                x = [t.clone().requires_grad_(True) for t in (q[b, :m, h], f["c"][b, :m], f["kr"][b, :m], w[h])]
                kv = x[1] @ x[3].t()
                s = (x[0] @ torch.cat([kv[:, :dn], x[2]], 1).t() * scale).masked_fill(above, float("-inf"))
                o = torch.softmax(s, -1) @ kv[:, dn:]
                g = torch.autograd.grad(o, x, f["dout"][b, :m, h])
                res["out"][b, :m, h], res["dq"][b, :m, h] = o.detach(), g[0]
                res["dc"][b, :m] += g[1]
                res["dkr"][b, :m] += g[2]
                res["dw"][h] += g[3]
        res["dw"] = res["dw"].view(-1, r)
        return res
    G, n, P, Hq, Hkv, D = (case[k] for k in ("G", "n", "P", "Hq", "Hkv", "D"))
    rep, scale = Hq // Hkv, 1.0 / math.sqrt(D)
    if case["op"] == "prefix_decode":
        out = torch.zeros_like(q)
        for b, m in enumerate(lens):
            for h in range(Hkv):
                kk = torch.cat([f["pk"][b // n, :, h], f["k"][b, :m, h]])
                vv = torch.cat([f["pv"][b // n, :, h], f["v"][b, :m, h]])
                hs = slice(h * rep, (h + 1) * rep)
                out[b, hs] = torch.softmax(q[b, hs] @ kk.t() * scale, -1) @ vv
        return out
    res = {"out": torch.zeros_like(q), "dq": torch.zeros_like(q), "dk": torch.zeros_like(f["k"]),
           "dv": torch.zeros_like(f["v"]), "dpk": torch.zeros_like(f["pk"]), "dpv": torch.zeros_like(f["pv"])}
    for b, m in enumerate(lens):
        above = torch.ones(m, m, dtype=torch.bool, device=q.device).triu(1)
        above = torch.cat([above.new_zeros(m, P), above], 1)
        for h in range(Hkv):
            hs, g = slice(h * rep, (h + 1) * rep), b // n
            x = [t.clone().requires_grad_(True) for t in (q[b, :m, hs].transpose(0, 1), f["k"][b, :m, h], f["v"][b, :m, h],
                                                          f["pk"][g, :, h], f["pv"][g, :, h])]
            s = (x[0] @ torch.cat([x[3], x[1]]).t() * scale).masked_fill(above, float("-inf"))
            o = torch.softmax(s, -1) @ torch.cat([x[4], x[2]])
            d = torch.autograd.grad(o, x, f["dout"][b, :m, hs].transpose(0, 1))
            res["out"][b, :m, hs], res["dq"][b, :m, hs] = o.detach().transpose(0, 1), d[0].transpose(0, 1)
            res["dk"][b, :m, h], res["dv"][b, :m, h] = d[1], d[2]
            res["dpk"][g, :, h] += d[3]
            res["dpv"][g, :, h] += d[4]
    return res
