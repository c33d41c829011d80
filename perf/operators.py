"""Measured cases of the training operators around the Lighthouse layers: the
root-mean-square norm with the residual's addition, the linear cross entropy and
the linear distillation loss.

Each case is one pass through one operator, in its plain form (elementary torch
operations in 32 bits) or, with ``own`` set, through the framework's kernels.

Shapes: N tokens, D model width, V vocabulary, K teacher entries per token.
"""
from __future__ import annotations

import math
import random

import torch

own = False

E4M3_MAX = 448.0
AMAX_MIN = 2.0 ** -100        # floor of a group's largest magnitude, so that an all-zero group keeps a scale above zero


# --------------------------------------------------------------------------- cases
def listed() -> list[dict]:
    return [
        # One norm of the 270M byte model at its own sequence length: a bf16 branch is added to the
        # fp32 residual stream, the norm's output feeds bf16 projections.
        dict(name="norm_train_stream", op="norm", N=65536, D=1024, x="bf16", res="f32", w="f32", grad=True, out="bf16",
             group=0),
        # A bf16 residual stream of a wider model, with a ragged number of tokens.
        dict(name="norm_train_wide", op="norm", N=8191, D=4096, x="bf16", res="bf16", w="bf16", grad=True, out="bf16",
             group=0),
        # Serving: four sequences decode one token each, the projections take 8-bit rows.
        dict(name="norm_fp8_tokens", op="norm", N=4, D=4096, x="bf16", res="bf16", w="bf16", grad=False, out="e4m3",
             group=0),
        # Serving: a long prompt, 8-bit output with one scale per 128 columns.
        dict(name="norm_fp8_prompt", op="norm", N=32768, D=5120, x="bf16", res="bf16", w="bf16", grad=False,
             out="e4m3", group=128),
        # The loss of the 270M byte model's training step: 65536 positions, 256 classes.
        dict(name="xent_bytes", op="xent", N=65536, V=256, D=1024, ignore=0.0, grad=True, reduction="mean"),
        # A training step over a large vocabulary.
        dict(name="xent_large", op="xent", N=8192, V=128000, D=2048, ignore=0.0, grad=True, reduction="mean"),
        # Fine-tuning: odd sizes, the prompt's positions are ignored.
        dict(name="xent_odd", op="xent", N=1999, V=50261, D=768, ignore=0.3, grad=True, reduction="mean"),
        # Scoring of a document: the loss of every position, no gradient.
        dict(name="xent_score", op="xent", N=4096, V=32000, D=4096, ignore=0.0, grad=False, reduction="none"),
        # Scoring of a few candidate tokens: bound by one read of the output weights.
        dict(name="xent_few", op="xent", N=16, V=128000, D=4096, ignore=0.0, grad=False, reduction="none"),
        # Distillation of a byte model.
        dict(name="distill_bytes", op="distill", N=16384, V=256, D=1024, K=16, T=1.0, empty=0.0, grad=True),
        # Distillation over a large vocabulary from a teacher's 64 top logits.
        dict(name="distill_large", op="distill", N=4096, V=128000, D=2048, K=64, T=2.0, empty=0.0, grad=True),
        # Odd sizes; some positions have no teacher.
        dict(name="distill_odd", op="distill", N=777, V=50261, D=896, K=13, T=1.5, empty=0.2, grad=True),
    ]


def _log_int(rng: random.Random, lo: int, hi: int) -> int:
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng: random.Random) -> dict:
    op = rng.choice(["norm", "xent", "distill"])
    if op == "norm":
        D = 8 * _log_int(rng, 32, 1024)
        N = _log_int(rng, 1, min(65536, 32768 * 5120 // D))
        out = rng.choice(["bf16", "f32", "e4m3"])
        x = rng.choice(["bf16", "f32"])
        if out == "f32":
            x = "f32"
        return dict(op=op, N=N, D=D, x=x, res=rng.choice(["none", "bf16", "f32"]), w=rng.choice(["bf16", "f32"]),
                    grad=out != "e4m3" and rng.random() < 0.7, out=out, group=rng.choice([0, 128]))
    D = 8 * _log_int(rng, 32, 512)
    V = _log_int(rng, 256, 131072)
    N = _log_int(rng, 1, max(1, min(65536, 8192 * 128000 * 2048 // (2 * V * D))))
    if op == "xent":
        return dict(op=op, N=N, V=V, D=D, ignore=rng.choice([0.0, 0.1, 0.5]), grad=rng.random() < 0.7,
                    reduction=rng.choice(["mean", "sum", "none"]))
    return dict(op=op, N=N, V=V, D=D, K=_log_int(rng, 1, 128), T=rng.choice([1.0, 1.5, 2.0, 4.0]),
                empty=rng.choice([0.0, 0.1, 0.5]), grad=rng.random() < 0.8)


# --------------------------------------------------------------------------- inputs
_DT = {"bf16": torch.bfloat16, "f32": torch.float32}


def _gen(seed: int) -> torch.Generator:
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def _teacher(g, N, V, K):
    """Top-K logits of a teacher: a frequency prior that falls with the token's number plus noise."""
    prior = -torch.log(torch.arange(V, device="cuda", dtype=torch.float32) + 10.0)
    vals, idxs = [], []
    for lo in range(0, N, 1024):
        n = min(1024, N - lo)
        s = torch.randn(n, V, generator=g, device="cuda") * 2.0 + prior + 8.0
        v, i = torch.topk(s, K, dim=1)
        vals.append(v)
        idxs.append(i)
    return torch.cat(vals), torch.cat(idxs)


def prepare(case: dict, seed: int) -> dict:
    g = _gen(seed)
    N, D = case["N"], case["D"]
    st = {"case": case}
    if case["op"] == "norm":
        xd, wd = _DT[case["x"]], _DT[case["w"]]
        st["x"] = _randn(g, N, D, dtype=xd)
        # a residual stream grows through the layers and has a few large channels
        chan = torch.ones(D, device="cuda")
        chan[torch.randint(0, D, (max(1, D // 256),), generator=g, device="cuda")] = 8.0
        st["res"] = None if case["res"] == "none" else (_randn(g, N, D, scale=2.0) * chan).to(_DT[case["res"]])
        st["w"] = (1.0 + 0.1 * torch.randn(D, generator=g, device="cuda")).to(wd)
        if case["grad"]:
            for k in ("x", "res", "w"):
                if st[k] is not None:
                    st[k].requires_grad_(True)
            st["dy"] = _randn(g, N, D, dtype=_DT[case["out"]])
            st["dh"] = None if st["res"] is None else _randn(g, N, D, dtype=_DT[case["res"]])
        return st
    V = case["V"]
    st["weight"] = _randn(g, V, D, dtype=torch.bfloat16, scale=0.02)
    hidden = torch.randn(N, D, generator=g, device="cuda")
    if case["op"] == "xent":
        target = torch.randint(0, V, (N,), generator=g, device="cuda")
        guess = target
        if case["ignore"]:
            # a prompt in front, its positions carry no target
            target = target.clone()
            target[:int(N * case["ignore"])] = -100
        st["target"] = target
    else:
        st["tv"], st["ti"] = _teacher(g, N, V, min(case["K"], V))
        guess = st["ti"][:, 0].clone()
        if case["empty"]:
            st["ti"][:int(N * case["empty"])] = -1
    # a student that gives the right token a logit a few units above the rest
    st["hidden"] = (hidden + st["weight"][guess].float() * (5.0 / (0.0004 * D))).to(torch.bfloat16)
    if case["grad"]:
        st["hidden"].requires_grad_(True)
        st["weight"].requires_grad_(True)
        if case.get("reduction") == "none":
            st["dloss"] = torch.rand(N, generator=g, device="cuda")
    return st


# --------------------------------------------------------------------------- one pass
def run(st: dict):
    op = st["case"]["op"]
    if own:
        return {"norm": _own_norm, "xent": _own_xent, "distill": _own_distill}[op](st)
    with torch.no_grad():
        return {"norm": _plain_norm, "xent": _plain_xent, "distill": _plain_distill}[op](st)


def _lib():
    from __graft_entry__ import load_package
    return load_package()


def _own_norm(st):
    lh, c = _lib(), st["case"]
    if c["out"] == "e4m3":
        if st["res"] is None:
            q, s = lh.rms_norm_fp8(st["x"], st["w"], group=c["group"])
            return {"q": q.to(torch.bfloat16), "scale": s}
        q, s, h = lh.add_rms_norm_fp8(st["x"], st["res"], st["w"], group=c["group"])
        return {"q": q.to(torch.bfloat16), "scale": s, "h": h}
    out = _DT[c["out"]]
    if st["res"] is None:
        y = lh.rms_norm(st["x"], st["w"], out_dtype=out)
        res = {"y": y}
        if c["grad"]:
            res["dx"], res["dw"] = torch.autograd.grad(y, (st["x"], st["w"]), st["dy"])
        return _detach(res)
    y, h = lh.add_rms_norm(st["x"], st["res"], st["w"], out_dtype=out)
    res = {"y": y, "h": h}
    if c["grad"]:
        res["dx"], res["dres"], res["dw"] = torch.autograd.grad((y, h), (st["x"], st["res"], st["w"]),
                                                                (st["dy"], st["dh"]))
    return _detach(res)


def _own_xent(st):
    lh, c = _lib(), st["case"]
    if not c["grad"]:
        return {"loss": lh.linear_cross_entropy(st["hidden"], st["weight"], st["target"], reduction=c["reduction"])}
    loss = lh.linear_cross_entropy(st["hidden"], st["weight"], st["target"], reduction=c["reduction"])
    dh, dw = torch.autograd.grad(loss, (st["hidden"], st["weight"]), st.get("dloss"))
    return _detach({"loss": loss, "dhidden": dh, "dweight": dw})


def _own_distill(st):
    lh, c = _lib(), st["case"]
    loss = lh.linear_distillation(st["hidden"], st["weight"], st["tv"], st["ti"], temperature=c["T"])
    if not c["grad"]:
        return {"loss": loss}
    dh, dw = torch.autograd.grad(loss, (st["hidden"], st["weight"]))
    return _detach({"loss": loss, "dhidden": dh, "dweight": dw})


def _detach(d):
    return {k: v.detach() for k, v in d.items()}


# --------------------------------------------------------------------------- plain forms
def _group_amax(t, group):
    if not group:
        return t.abs().amax(-1, keepdim=True)
    D = t.shape[-1]
    G = (D + group - 1) // group
    pad = torch.zeros(*t.shape[:-1], G * group, dtype=t.dtype, device=t.device)
    pad[..., :D] = t.abs()
    return pad.view(*t.shape[:-1], G, group).amax(-1)


def _plain_norm(st, eps=1e-5):
    c = st["case"]
    x, w = st["x"].float(), st["w"].float()
    h_store = None
    if st["res"] is not None:
        h_store = (x + st["res"].float()).to(st["res"].dtype)      # the norm reads the stream as it is stored
    h = x if h_store is None else h_store.float()
    rstd = torch.rsqrt((h * h).mean(-1, keepdim=True) + eps)
    if c["out"] == "e4m3":
        t = h * w
        a = _group_amax(t, c["group"]).clamp(min=AMAX_MIN)
        a_e = a if not c["group"] else a.repeat_interleave(c["group"], dim=-1)[..., :t.shape[-1]]
        # the codes' values (4 significant bits: bf16 holds them exactly) and the scales beside them
        res = {"q": (t * E4M3_MAX / a_e).to(torch.float8_e4m3fn).to(torch.bfloat16), "scale": a * rstd / E4M3_MAX}
        return res if h_store is None else {**res, "h": h_store}
    xhat = h * rstd
    res = {"y": (xhat * w).to(_DT[c["out"]])}
    if h_store is not None:
        res["h"] = h_store
    if c["grad"]:
        dy = st["dy"].float()
        g = dy * w
        d = rstd * (g - xhat * (g * xhat).mean(-1, keepdim=True))
        if h_store is not None:
            d = d + st["dh"].float()
        res["dx"] = d.to(st["x"].dtype)
        if h_store is not None:
            res["dres"] = d.to(st["res"].dtype)
        res["dw"] = (dy * xhat).sum(0).to(st["w"].dtype)
    return res


def _plain_xent(st):
    c = st["case"]
    h, w, t = st["hidden"].float(), st["weight"].float(), st["target"]
    s = h @ w.T
    valid = t != -100
    tt = t.clamp(min=0)
    m = s.amax(-1, keepdim=True)
    lse = (m + (s - m).exp().sum(-1, keepdim=True).log())
    loss = torch.where(valid, (lse - s.gather(1, tt[:, None])).squeeze(1), torch.zeros_like(lse[:, 0]))
    red = c["reduction"]
    count = valid.sum().clamp(min=1).float()
    total = loss if red == "none" else loss.sum() / count if red == "mean" else loss.sum()
    if not c["grad"]:
        return {"loss": total}
    coef = valid.float() * (st["dloss"] if red == "none" else 1.0)
    if red == "mean":
        coef = coef / count
    p = (s - lse).exp()
    p.scatter_add_(1, tt[:, None], torch.full_like(lse, -1.0))
    p *= coef[:, None]
    return {"loss": total, "dhidden": (p @ w).to(torch.bfloat16), "dweight": (p.T @ h).to(torch.bfloat16)}


def _plain_distill(st):
    c = st["case"]
    T = c["T"]
    h, w = st["hidden"].float(), st["weight"].float()
    here = st["ti"] >= 0
    ti = st["ti"].clamp(min=0)
    valid = here.any(-1)
    tv = (st["tv"].float() / T).masked_fill(~here, float("-inf"))
    tv = torch.where(valid[:, None], tv, torch.zeros_like(tv))
    tm = tv.amax(-1, keepdim=True)
    logp = tv - (tm + (tv - tm).exp().sum(-1, keepdim=True).log())
    p = torch.where(valid[:, None], logp.exp(), torch.zeros_like(logp))
    s = (h @ w.T) / T
    m = s.amax(-1, keepdim=True)
    lse = m + (s - m).exp().sum(-1, keepdim=True).log()
    logq = s.gather(1, ti) - lse
    terms = torch.where(p > 0, p * (logp - logq), torch.zeros_like(p))
    count = valid.sum().clamp(min=1).float()
    loss = terms.sum(-1).sum() * (T * T) / count
    if not c["grad"]:
        return {"loss": loss}
    d = (s - lse).exp()
    d.scatter_add_(1, ti, -p)
    d *= (valid.float() * T / count)[:, None]
    return {"loss": loss, "dhidden": (d @ w).to(torch.bfloat16), "dweight": (d.T @ h).to(torch.bfloat16)}


# --------------------------------------------------------------------------- work
def work(case: dict) -> dict:
    N, D = case["N"], case["D"]
    if case["op"] == "norm":
        sz = {"bf16": 2, "f32": 4, "e4m3": 1, "none": 0}
        e = N * D
        b = e * (sz[case["x"]] + 2 * sz[case["res"]] + sz[case["out"]]) + D * sz[case["w"]]
        flops = 5 * e
        if case["out"] == "e4m3":
            b += N * 4 * (1 if not case["group"] else (D + case["group"] - 1) // case["group"])
        if case["grad"]:
            # dy, dh and the stored stream (the input itself where there is no residual) in; dx, dres, dw out
            b += e * (sz[case["out"]] + sz[case["res"]] + (sz[case["res"]] or sz[case["x"]]))
            b += e * (sz[case["x"]] + sz[case["res"]]) + 2 * D * sz[case["w"]]
            flops += 10 * e
        return {"bytes": b, "flops": flops}
    V = case["V"]
    rows = N - int(N * (case["ignore"] if case["op"] == "xent" else case["empty"]))
    per = 8 if case["op"] == "xent" else 12 * min(case["K"], V)
    # hidden and weight in; with gradients both once more and their gradients out
    b = (N * D + V * D) * 2 + N * per
    flops = 2 * rows * V * D
    if case["grad"]:
        b += (N * D + V * D) * 2
        flops *= 3
    return {"bytes": b, "flops": flops}


# --------------------------------------------------------------------------- 64-bit results
def exact(case: dict, seed: int):
    st = prepare(case, seed)
    with torch.no_grad():
        return _exact_norm(st) if case["op"] == "norm" else _exact_loss(st)


def _exact_norm(st, eps=1e-5):
    c = st["case"]
    w = st["w"].double()
    out = {k: [] for k in ("y", "q", "scale", "h", "dx", "dres")}
    dw = torch.zeros_like(w)
    D = w.numel()
    for lo in range(0, c["N"], 4096):
        sl = slice(lo, lo + 4096)
        h = st["x"][sl].double()
        if st["res"] is not None:
            # the stream's new value is rounded to its own type, the norm is that of the rounded value
            h = (h + st["res"][sl].double()).to(st["res"].dtype)
            out["h"].append(h)
            h = h.double()
        ms = h.square().sum(-1, keepdim=True) / D + eps
        n = h / ms.sqrt()
        if c["out"] == "e4m3":
            q, scales = torch.empty_like(n), []
            step = c["group"] or D
            for g0 in range(0, D, step):
                t = h[:, g0:g0 + step] * w[g0:g0 + step]
                a = t.abs().amax(-1, keepdim=True).clamp(min=AMAX_MIN)
                q[:, g0:g0 + step] = _e4m3(t * E4M3_MAX / a)
                scales.append(a / E4M3_MAX / ms.sqrt())
            out["q"].append(q)
            out["scale"].append(torch.cat(scales, -1))
            continue
        out["y"].append(n * w)
        if c["grad"]:
            dy = st["dy"][sl].double()
            g = dy * w
            d = (g - n * ((g * n).sum(-1, keepdim=True) / D)) / ms.sqrt()
            if st["res"] is not None:
                d = d + st["dh"][sl].double()
                out["dres"].append(d)
            out["dx"].append(d)
            dw += (dy * n).sum(0)
    res = {k: torch.cat(v) for k, v in out.items() if v}
    if c["grad"]:
        res["dw"] = dw
    return res


def _e4m3(v):
    """Nearest value of 4 exponent and 3 mantissa bits, ties to even, for |v| <= 448."""
    e = torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6)))
    e = torch.where(v.abs() < torch.exp2(e), e - 1, e)
    step = torch.exp2(e.clamp(min=-6.0) - 3)
    return torch.round(v / step) * step


def _exact_loss(st):
    c = st["case"]
    N, V, D = c["N"], c["V"], c["D"]
    if 8 * N * V * D > 4e13:
        return None
    w = st["weight"].double()
    xent = c["op"] == "xent"
    T = 1.0 if xent else c["T"]
    if xent:
        idx = st["target"].clamp(min=0)[:, None]
        ok = (st["target"] != -100)
        prob = ok.double()[:, None]
    else:
        idx = st["ti"].clamp(min=0)
        here = st["ti"] >= 0
        ok = here.any(-1)
        prob = torch.zeros(idx.shape, dtype=torch.float64, device="cuda")
        prob[ok] = torch.softmax((st["tv"].double() / T).masked_fill(~here, float("-inf"))[ok], -1)
    red = c.get("reduction", "mean")
    n_ok = max(1, int(ok.sum()))
    coef = ok.double() * T
    if red == "mean":
        coef = coef / n_ok
    elif red == "none" and c["grad"]:
        coef = coef * st["dloss"].double()
    losses, dh, dw = [], [], torch.zeros_like(w) if c["grad"] else None
    rows = max(1, min(N, 2 ** 28 // V))
    for lo in range(0, N, rows):
        sl = slice(lo, lo + rows)
        h = st["hidden"][sl].double()
        s = h @ w.T / T
        logq = s - torch.logsumexp(s, -1, keepdim=True)
        del s
        lq = logq.gather(1, idx[sl])
        pr = prob[sl]
        ent = torch.where(pr > 0, pr * pr.clamp(min=1e-300).log(), torch.zeros_like(pr))
        losses.append((ent - torch.where(pr > 0, pr * lq, torch.zeros_like(pr))).sum(-1) * T * T)
        if c["grad"]:
            d = logq.exp_()
            d.scatter_add_(1, idx[sl], -pr)
            d *= coef[sl, None]
            dh.append(d @ w)
            dw += d.T @ h
    loss = torch.cat(losses)
    loss = loss if red == "none" else loss.sum() / (n_ok if red == "mean" else 1)
    return {"loss": loss, "dhidden": torch.cat(dh), "dweight": dw} if c["grad"] else {"loss": loss}
