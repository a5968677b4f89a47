"""The operators of a language-model step that stand beside this library's memory rules, glue and loss:
what is timed, in their plain form and through the framework's entry points.

A case is a dict of plain values; ``op`` names the operator:

  gd_train    gated delta rule: forward and backward of a training step
  gd_prefill  gated delta rule: forward over a packed batch of prompts, final states kept
  gd_step     gated delta rule: one token (or a few) for every sequence on its stored state
  embed       scaled embedding lookup and its gradient, added into the gradient arena
  distill     distillation from a teacher's top logits with a hard-target term: loss and gradient

The plain forms are torch products, sums, exponentials, comparisons and indexing in fp32; sums of
log-decays are taken in fp64, where fp32 would lose the small ones behind large ones. The stored states
of gd_step and the gradient arena of embed are updated in place, as in a program that serves or trains.
"""
from __future__ import annotations

import math

import torch

own = False

DT = {"bf16": torch.bfloat16, "f32": torch.float32}


def listed():
    return [
        # level 0 of the stacked model at its full batch: 64 sequences x 8 heads of 64, fp32 streams
        {"name": "gd_train_model", "op": "gd_train", "batch": 64, "seq": 512, "hk": 8, "hv": 8, "dk": 64, "dv": 64,
         "dtype": "f32", "carry": True},
        # bf16 streams at long context
        {"name": "gd_train_long_bf16", "op": "gd_train", "batch": 4, "seq": 4096, "hk": 16, "hv": 16, "dk": 64,
         "dv": 64, "dtype": "bf16", "carry": False},
        # heads of 128, two value heads share a key head, a length that is no multiple of a chunk
        {"name": "gd_train_shared_d128", "op": "gd_train", "batch": 2, "seq": 1000, "hk": 4, "hv": 8, "dk": 128,
         "dv": 128, "dtype": "bf16", "carry": True},
        # prompts of very different lengths packed into one call
        {"name": "gd_prefill_ragged", "op": "gd_prefill", "batch": 13, "seq": 9001, "hk": 8, "hv": 8, "dk": 64,
         "dv": 64, "dtype": "bf16", "carry": False},
        # one sequence writes one token: latency
        {"name": "gd_step_one", "op": "gd_step", "batch": 1, "seq": 1, "hk": 8, "hv": 8, "dk": 64, "dv": 64,
         "dtype": "bf16", "carry": True},
        # a full serving batch, states of 128 x 128 in a pool addressed by slots
        {"name": "gd_step_batch", "op": "gd_step", "batch": 256, "seq": 1, "hk": 8, "hv": 16, "dk": 128, "dv": 128,
         "dtype": "bf16", "carry": True},
        # the smallest model's lookup: two sequences of 256 bytes
        {"name": "embed_small", "op": "embed", "tokens": 512, "vocab": 256, "d": 64, "dtype": "f32"},
        # the stacked model's lookup at its full batch
        {"name": "embed_model", "op": "embed", "tokens": 32768, "vocab": 8192, "d": 512, "dtype": "f32"},
        # a larger vocabulary and wider rows, bf16 activations, an odd number of tokens
        {"name": "embed_wide_bf16", "op": "embed", "tokens": 65521, "vocab": 50001, "d": 1024, "dtype": "bf16"},
        # distillation of the smallest model
        {"name": "distill_small", "op": "distill", "rows": 512, "vocab": 256, "k": 8, "tau": 2.0, "hard": 0.5,
         "dtype": "f32"},
        # distillation of the stacked model at its full batch
        {"name": "distill_model", "op": "distill", "rows": 32768, "vocab": 8192, "k": 64, "tau": 2.0, "hard": 0.5,
         "dtype": "bf16"},
        # a wide vocabulary of odd size, soft targets alone at temperature 1
        {"name": "distill_wide", "op": "distill", "rows": 2047, "vocab": 100003, "k": 32, "tau": 1.0, "hard": 0.0,
         "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("gd_train", "gd_train", "gd_prefill", "gd_step", "embed", "distill"))
    if op in ("gd_train", "gd_prefill"):
        dk, dv = rng.choice(((64, 64), (64, 64), (128, 128), (64, 128), (32, 32), (48, 80)))
        hk, share = rng.choice(((1, 1), (4, 1), (8, 1), (8, 2), (2, 4)))
        hv = hk * share
        top = 262144 * 4096 // (hv * max(dk * dv, 4096))
        seq = _log(rng, 1, 4096)
        batch = _log(rng, 1, max(1, min(64, top // seq)))
        if op == "gd_prefill":
            seq = max(batch, min(16384, seq * batch))
        return {"op": op, "batch": batch, "seq": seq, "hk": hk, "hv": hv, "dk": dk, "dv": dv,
                "dtype": rng.choice(("f32", "bf16")), "carry": rng.random() < 0.5}
    if op == "gd_step":
        dk, dv = rng.choice(((64, 64), (128, 128), (32, 64), (48, 80)))
        hk, share = rng.choice(((1, 1), (8, 1), (8, 2), (4, 4)))
        return {"op": op, "batch": _log(rng, 1, 256), "seq": rng.choice((1, 1, 1, 2, 5)), "hk": hk, "hv": hk * share,
                "dk": dk, "dv": dv, "dtype": rng.choice(("f32", "bf16")), "carry": True}
    if op == "embed":
        return {"op": op, "tokens": _log(rng, 1, 65536), "vocab": _log(rng, 64, 60000), "d": 8 * _log(rng, 4, 128),
                "dtype": rng.choice(("f32", "bf16"))}
    vocab = _log(rng, 100, 130000)
    return {"op": op, "rows": _log(rng, 1, max(1, 200_000_000 // vocab)) if vocab > 6000 else _log(rng, 1, 32768),
            "vocab": vocab, "k": rng.choice((1, 5, 8, 20, 32, 64, 100)),
            "tau": rng.choice((1.0, 1.5, 2.0, 4.0)), "hard": rng.choice((0.0, 0.25, 0.5)),
            "dtype": rng.choice(("f32", "bf16"))}


# ── inputs ─────────────────────────────────────────────────────────────────
def _zipf(g, vocab, n):
    """Zipf(1.1) token ids, the usual stand-in for text, spread over the vocabulary."""
    w = torch.arange(1, vocab + 1, device="cuda", dtype=torch.float64).pow(-1.1)
    c = torch.cumsum(w, 0)
    u = torch.rand(n, generator=g, device="cuda", dtype=torch.float64) * c[-1]
    rank = torch.searchsorted(c, u).clamp_max(vocab - 1)
    return torch.randperm(vocab, generator=g, device="cuda")[rank]


def _starts(g, batch, total):
    """Ascending starts of `batch` sequences of very different lengths that fill `total` tokens."""
    w = torch.rand(batch, generator=g, device="cuda", dtype=torch.float64).pow(3) + 1e-3
    cut = torch.round(torch.cumsum(w, 0) / w.sum() * total).to(torch.int32)
    return torch.cat([torch.zeros(1, dtype=torch.int32, device="cuda"), cut])


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    normal = lambda *s: torch.randn(*s, generator=g, device="cuda")
    uniform = lambda *s: torch.rand(*s, generator=g, device="cuda")
    op, dt = case["op"], DT[case["dtype"]]
    s = {"case": dict(case)}
    if op.startswith("gd_"):
        hk, hv, dk, dv = case["hk"], case["hv"], case["dk"], case["dv"]
        b, n = (1, case["seq"]) if op == "gd_prefill" else (case["batch"], case["seq"])
        unit = lambda *sh: torch.nn.functional.normalize(normal(*sh), dim=-1)
        s["k"], s["q"] = unit(b, n, hk, dk).to(dt), unit(b, n, hk, dk).to(dt)
        s["v"] = normal(b, n, hv, dv).to(dt)
        # heads that forget at rates from a few tokens to thousands, modulated by the token
        rate = torch.exp(torch.linspace(math.log(0.5), math.log(5e-4), hv, device="cuda"))
        s["log_retain"] = -rate * torch.nn.functional.softplus(normal(b, n, hv) + 0.5)
        s["theta"] = torch.sigmoid(normal(b, n, hv))
        s["scale"] = dk ** -0.5
        s["m0"] = None
        if case["carry"]:
            s["m0"] = 0.1 * normal(case["batch"], hv, dv, dk)
        if op == "gd_train":
            s["d_y"] = normal(b, n, hv, dv).to(dt)
            s["d_m"] = 0.1 * normal(b, hv, dv, dk) if case["carry"] else None
        if op == "gd_prefill":
            s["starts"] = _starts(g, case["batch"], n)
        if op == "gd_step":
            # the pool has more slots than the batch, in no order
            s["pool"] = 0.1 * normal(case["batch"] + 3, hv, dv, dk)
            s["slots"] = torch.randperm(case["batch"] + 3, generator=g, device="cuda")[:case["batch"]].to(torch.int32)
        return s
    if op == "embed":
        n, vocab, d = case["tokens"], case["vocab"], case["d"]
        s["w"] = (normal(vocab, d) * d ** -0.5).to(dt)
        s["ids"] = _zipf(g, vocab, n).to(torch.int32)
        s["d_y"] = normal(n, d).to(dt)
        s["grad"] = normal(vocab, d)          # what the unembedding has added to the tied gradient already
        s["scale"] = float(d) ** 0.5
        return s
    n, vocab, k = case["rows"], case["vocab"], min(case["k"], case["vocab"])
    z = 2.0 * normal(n, vocab)
    # a teacher that agrees with the student in part: its top entries are the top of noisy copies of the logits
    z[:, : max(1, vocab // 50)] += 1.5
    s["logits"] = z.to(dt)
    step = max(1, (1 << 28) // vocab)
    ids, val = [], []
    for i in range(0, n, step):
        t = s["logits"][i:i + step].float() + normal(min(step, n - i), vocab)
        v, j = torch.topk(t, k, dim=1)
        ids.append(j.to(torch.int32))
        val.append(v)
    s["teacher_ids"], s["teacher_logits"] = torch.cat(ids), torch.cat(val).to(dt)
    s["targets"] = s["teacher_ids"][:, 0].clone()
    s["targets"][uniform(n) < 0.1] = -1        # padded positions carry no target ...
    s["teacher_ids"][uniform(n) < 0.1] = -1    # ... and some positions no teacher
    return s


# ── the plain forms ────────────────────────────────────────────────────────
def _chunk(S, k, v, q, g, theta, scale):
    """One chunk of the gated delta rule in matrix form: heads [..., L, d], S = M^T [..., dk, dv]."""
    L = k.shape[-2]
    G = torch.cumsum(g.double(), -1)
    diff = G.unsqueeze(-1) - G.unsqueeze(-2)
    low = torch.ones(L, L, dtype=torch.bool, device=k.device).tril()
    decay = torch.exp(torch.where(low, diff, torch.full_like(diff, -math.inf))).to(k.dtype)
    eG, eR = torch.exp(G).to(k.dtype).unsqueeze(-1), torch.exp(G[..., -1:] - G).to(k.dtype).unsqueeze(-1)
    A = ((k @ k.transpose(-1, -2)) * decay).tril(-1) * theta.unsqueeze(-2)
    T = torch.eye(L, dtype=k.dtype, device=k.device) - A       # (I + A)^-1 = (I - A)(I + A^2)(I + A^4)...
    P = A @ A
    for _ in range(max(0, math.ceil(math.log2(max(L, 2))) - 1)):
        T = T + T @ P
        P = P @ P
    u = theta.unsqueeze(-1) * (T @ (v - eG * (k @ S)))
    y = scale * (eG * (q @ S) + ((q @ k.transpose(-1, -2)) * decay) @ u)
    return y, eG[..., -1:, :] * S + (eR * k).transpose(-1, -2) @ u


def _rule(k, v, q, g, theta, S, scale):
    """[B, H, S, d] through all chunks of 64."""
    ys = []
    for c in range(0, k.shape[2], 64):
        e = slice(c, c + 64)
        y, S = _chunk(S, k[:, :, e], v[:, :, e], q[:, :, e], g[:, :, e], theta[:, :, e], scale)
        ys.append(y)
    return torch.cat(ys, 2), S


def _heads(t, share):
    return t.repeat_interleave(share, dim=2).transpose(1, 2)


def _plain_gd(s):
    c = s["case"]
    share, b, dk, dv, hv = c["hv"] // c["hk"], c["batch"], c["dk"], c["dv"], c["hv"]
    if c["op"] == "gd_step":
        at = s["slots"].long()
        M = s["pool"][at]
        ys = []
        k, q = (s[x].float().repeat_interleave(share, dim=2) for x in ("k", "q"))
        v = s["v"].float()
        for t in range(c["seq"]):
            M = M * torch.exp(s["log_retain"][:, t])[..., None, None]
            e = s["theta"][:, t].unsqueeze(-1) * (v[:, t] - (M * k[:, t].unsqueeze(-2)).sum(-1))
            M = M + e.unsqueeze(-1) * k[:, t].unsqueeze(-2)
            ys.append(s["scale"] * (M * q[:, t].unsqueeze(-2)).sum(-1))
        s["pool"][at] = M
        return {"y": torch.stack(ys, 1).to(s["v"].dtype), "pool": s["pool"]}
    leaves = {x: s[x].float() for x in ("k", "v", "q", "log_retain", "theta")}
    S0 = s["m0"].transpose(-1, -2) if s["m0"] is not None else torch.zeros(b, hv, dk, dv, device="cuda")
    if c["op"] == "gd_train":
        leaves = {x: t.detach().requires_grad_(True) for x, t in leaves.items()}
        S0 = S0.detach().requires_grad_(True)
        y, S = _rule(_heads(leaves["k"], share), leaves["v"].transpose(1, 2), _heads(leaves["q"], share),
                     leaves["log_retain"].transpose(1, 2), leaves["theta"].transpose(1, 2), S0, s["scale"])
        y = y.transpose(1, 2)
        out, gout = [y], [s["d_y"].float()]
        if s["d_m"] is not None:
            out.append(S)
            gout.append(s["d_m"].transpose(-1, -2))
        grads = torch.autograd.grad(out, [*leaves.values(), S0], gout)
        dt = s["k"].dtype
        r = {"y": y.detach().to(dt), "m_final": S.detach().transpose(-1, -2).contiguous()}
        r |= {"d_" + x: gr.to(dt if x in ("k", "v", "q") else torch.float32) for x, gr in zip(leaves, grads)}
        if s["m0"] is not None:
            r["d_m_initial"] = grads[-1].transpose(-1, -2).contiguous()
        return r
    ends = s["starts"].tolist()
    y, M = torch.empty_like(s["v"]), []
    for i in range(b):
        e = slice(ends[i], ends[i + 1])
        if ends[i + 1] == ends[i]:
            M.append(S0[i:i + 1])
            continue
        yi, Si = _rule(_heads(leaves["k"][:, e], share), leaves["v"][:, e].transpose(1, 2), _heads(leaves["q"][:, e], share),
                       leaves["log_retain"][:, e].transpose(1, 2), leaves["theta"][:, e].transpose(1, 2), S0[i:i + 1], s["scale"])
        y[:, e] = yi.transpose(1, 2).to(y.dtype)
        M.append(Si)
    return {"y": y, "m_final": torch.cat(M).transpose(-1, -2).contiguous()}


def _plain_embed(s):
    ids = s["ids"].long()
    out = (s["w"][ids].float() * s["scale"]).to(s["w"].dtype)
    s["grad"].index_add_(0, ids, s["d_y"].float() * s["scale"])
    return {"out": out, "grad": s["grad"]}


def _plain_distill(s):
    c = s["case"]
    z, tau = s["logits"].float(), c["tau"]
    hard_w, soft_w = c["hard"], 1.0 - c["hard"]
    ids, t = s["teacher_ids"], s["teacher_logits"].float() / tau
    there = ids >= 0
    at = ids.clamp_min(0).long()
    any_t = there.any(1, keepdim=True)
    t = torch.where(there, t, torch.full_like(t, -math.inf))
    t = torch.where(any_t, t, torch.zeros_like(t))
    p = torch.exp(t - t.max(1, keepdim=True).values)
    logp = t - t.max(1, keepdim=True).values - torch.log(p.sum(1, keepdim=True))
    p = torch.where(there, p / p.sum(1, keepdim=True), torch.zeros_like(p))
    m = z.max(1, keepdim=True).values
    eh, es = torch.exp(z - m), torch.exp((z - m) / tau)
    sh, ss = eh.sum(1, keepdim=True), es.sum(1, keepdim=True)
    valid = s["targets"] >= 0
    tgt = s["targets"].clamp_min(0).long().unsqueeze(1)
    ce = torch.where(valid, (m + torch.log(sh) - z.gather(1, tgt)).squeeze(1), torch.zeros_like(m.squeeze(1)))
    kl = torch.where(there, p * (logp - ((z.gather(1, at) - m) / tau - torch.log(ss))), torch.zeros_like(p)).sum(1)
    n_hard, n_soft = valid.sum().clamp_min(1).float(), any_t.sum().clamp_min(1).float()
    loss = hard_w * ce.double().sum().float() / n_hard + soft_w * tau * tau * kl.double().sum().float() / n_soft
    gh = (hard_w / n_hard) * valid.unsqueeze(1).float()
    gs = (soft_w * tau / n_soft) * any_t.float()
    d = gh * (eh / sh) + gs * (es / ss)
    d.scatter_add_(1, tgt, -gh)
    d.scatter_add_(1, at, -gs * p)
    return {"loss": loss, "d_logits": d.to(s["logits"].dtype)}


# ── the framework's calls ──────────────────────────────────────────────────
def _own(s):
    from nl_hecate_b200 import dispatch as D
    c = s["case"]
    op = c["op"]
    if op == "gd_step":
        y = D.gated_delta_step(s["k"], s["v"], s["q"], s["log_retain"], s["theta"], s["pool"], slots=s["slots"],
                               scale=s["scale"])
        return {"y": y, "pool": s["pool"]}
    if op == "gd_prefill":
        y, m, _ = D.gated_delta_forward(s["k"], s["v"], s["q"], s["log_retain"], s["theta"], m0=s["m0"],
                                        seq_starts=s["starts"], scale=s["scale"], want_saved=False)
        return {"y": y, "m_final": m}
    if op == "gd_train":
        y, m, saved = D.gated_delta_forward(s["k"], s["v"], s["q"], s["log_retain"], s["theta"], m0=s["m0"], scale=s["scale"])
        g = D.gated_delta_backward(s["k"], s["v"], s["q"], s["log_retain"], s["theta"], saved, s["d_y"],
                                   d_m_final=s["d_m"], want_initial=s["m0"] is not None, scale=s["scale"])
        r = {"y": y, "m_final": m}
        r |= {x: g[x] for x in ("d_k", "d_v", "d_q", "d_log_retain", "d_theta")}
        if s["m0"] is not None:
            r["d_m_initial"] = g["d_m_initial"]
        return r
    if op == "embed":
        out = D.embedding_forward(s["w"], s["ids"], scale=s["scale"])
        D.embedding_backward(s["d_y"], s["ids"], s["grad"], scale=s["scale"], accumulate=True)
        return {"out": out, "grad": s["grad"]}
    loss, saved = D.distill_forward(s["logits"], s["teacher_ids"], s["teacher_logits"], targets=s["targets"],
                                    temperature=c["tau"], soft_weight=1.0 - c["hard"], hard_weight=c["hard"])
    return {"loss": loss, "d_logits": D.distill_backward(s["logits"], saved)}


def run(s):
    if own:
        return _own(s)
    op = s["case"]["op"]
    return _plain_gd(s) if op.startswith("gd_") else _plain_embed(s) if op == "embed" else _plain_distill(s)


# ── what a pass cannot do without ──────────────────────────────────────────
def work(case):
    op, e = case["op"], 2 if case["dtype"] == "bf16" else 4
    if op.startswith("gd_"):
        b, hk, hv, dk, dv = case["batch"], case["hk"], case["hv"], case["dk"], case["dv"]
        n = case["seq"] * (1 if op == "gd_prefill" else b)
        state = 4 * b * hv * dk * dv
        stream = e * n * (2 * hk * dk + hv * dv) + 8 * n * hv      # k, q, v, gates
        y = e * n * hv * dv
        # the rule itself, token by token: M k, the update, M q
        fwd = 6.0 * n * hv * dk * dv
        if op == "gd_train":
            both = (3 if case["carry"] else 1) * state + (state if case["carry"] else 0)   # m0, m_final, d_m, d_m0
            return {"bytes": 2 * stream + 2 * y + both, "flops": 3 * fwd}
        if op == "gd_step":
            return {"bytes": stream + y + 2 * state, "flops": fwd}
        return {"bytes": stream + y + state * (2 if case["carry"] else 1), "flops": fwd}
    if op == "embed":
        n, vocab, d = case["tokens"], case["vocab"], case["d"]
        p = torch.arange(1, vocab + 1, dtype=torch.float64).pow(-1.1)
        rows = float((1 - (1 - p / p.sum()).pow(n)).sum())     # distinct ids to be expected
        # lookup: touched rows in, n rows out; gradient: n rows in, the arena's touched rows read and written
        return {"bytes": e * d * (rows + 2 * n) + 8 * rows * d + 8 * n, "flops": 2.0 * n * d}
    n, vocab, k = case["rows"], case["vocab"], case["k"]
    return {"bytes": 3 * e * n * vocab + n * (k * (4 + e) + 4), "flops": 10.0 * n * vocab}


# ── the definitions in 64 bits, token by token ─────────────────────────────
def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op.startswith("gd_"):
        return _exact_gd(case, s)
    f = lambda t: t.double()
    if op == "embed":
        ids = s["ids"].long()
        order = torch.argsort(ids, stable=True)
        rows = f(s["d_y"])[order]
        total = torch.cat([torch.zeros(1, rows.shape[1], dtype=torch.float64, device="cuda"), torch.cumsum(rows, 0)])
        first = torch.searchsorted(ids[order], torch.arange(case["vocab"] + 1, device="cuda"))
        return {"out": f(s["w"])[ids] * s["scale"], "grad": f(s["grad"]) + s["scale"] * (total[first[1:]] - total[first[:-1]])}
    n, tau, hw = case["rows"], case["tau"], case["hard"]
    nh = max(1, int((s["targets"] >= 0).sum()))
    ns = max(1, int((s["teacher_ids"] >= 0).any(1).sum()))
    loss, grad = 0.0, torch.empty(n, case["vocab"], dtype=torch.float64, device="cuda")
    step = max(1, (1 << 27) // case["vocab"])
    for i in range(0, n, step):
        e = slice(i, i + step)
        z, ids, t, y = f(s["logits"][e]), s["teacher_ids"][e].long(), f(s["teacher_logits"][e]) / tau, s["targets"][e].long()
        d = torch.zeros_like(z)
        ok = y >= 0
        rows = torch.arange(z.shape[0], device="cuda")
        lp = torch.log_softmax(z, 1)
        loss = loss - hw / nh * lp[rows[ok], y[ok]].sum()
        d[ok] += hw / nh * torch.exp(lp[ok])
        d[rows[ok], y[ok]] -= hw / nh
        has = (ids >= 0).any(1)
        lq = torch.log_softmax(z / tau, 1)
        dense = torch.zeros_like(z)
        w = torch.softmax(torch.where(ids >= 0, t, torch.full_like(t, -math.inf))[has], 1)
        dense[has] = dense[has].scatter_add(1, ids[has].clamp_min(0), w)
        loss = loss + (1 - hw) * tau * tau / ns * (torch.special.xlogy(w, w).sum() - (dense[has] * lq[has]).sum())
        d[has] += (1 - hw) * tau / ns * (torch.exp(lq[has]) - dense[has])
        grad[e] = d
    return {"loss": loss.reshape(()), "d_logits": grad}


def _exact_gd(case, s):
    """The recurrence and its adjoint, one token after the other, in 64 bits."""
    op, hv, dk, dv, b = case["op"], case["hv"], case["dk"], case["dv"], case["batch"]
    share = hv // case["hk"]
    k, q = (s[x].double().repeat_interleave(share, dim=2) for x in ("k", "q"))
    v, r, th, sc = s["v"].double(), torch.exp(s["log_retain"].double()), s["theta"].double(), s["scale"]
    if op == "gd_prefill":
        # all sequences side by side: token t of each, where it has one
        st = s["starts"].long()
        length = st[1:] - st[:-1]
        M = s["m0"].double() if s["m0"] is not None else torch.zeros(b, hv, dv, dk, dtype=torch.float64, device="cuda")
        y = torch.zeros(1, case["seq"], hv, dv, dtype=torch.float64, device="cuda")
        if int(length.max()) > 20000:
            return None
        M = M.clone()
        for t in range(int(length.max())):
            on = torch.nonzero(length > t).squeeze(1)
            at = st[on] + t
            kt, Mt = k[0, at], M[on] * r[0, at][..., None, None]
            u = th[0, at].unsqueeze(-1) * (v[0, at] - torch.einsum("bhvk,bhk->bhv", Mt, kt))
            Mt = Mt + u.unsqueeze(-1) * kt.unsqueeze(-2)
            M[on] = Mt
            y[0, at] = sc * torch.einsum("bhvk,bhk->bhv", Mt, q[0, at])
        return {"y": y, "m_final": M}
    n = case["seq"]
    if op == "gd_step":
        M = s["pool"].double()[s["slots"].long()]
    else:
        M = s["m0"].double() if s["m0"] is not None else torch.zeros(b, hv, dv, dk, dtype=torch.float64, device="cuda")
    if 8.0 * n * b * hv * dk * dv > 60e9:
        return None
    hist, es, y = [], [], torch.empty(b, n, hv, dv, dtype=torch.float64, device="cuda")
    for t in range(n):
        hist.append(M)
        R = M * r[:, t][..., None, None]
        e = v[:, t] - torch.einsum("bhvk,bhk->bhv", R, k[:, t])
        M = R + (th[:, t].unsqueeze(-1) * e).unsqueeze(-1) * k[:, t].unsqueeze(-2)
        es.append(e)
        y[:, t] = sc * torch.einsum("bhvk,bhk->bhv", M, q[:, t])
    if op == "gd_step":
        pool = s["pool"].double()
        pool[s["slots"].long()] = M
        return {"y": y, "pool": pool}
    dy = s["d_y"].double()
    lam = s["d_m"].double() if s["d_m"] is not None else torch.zeros_like(M)
    out = {"y": y, "m_final": M}
    dk_, dq_, dv_ = torch.zeros_like(k), torch.zeros_like(q), torch.zeros_like(v)
    dg, dth = torch.zeros_like(r), torch.zeros_like(th)
    Mt = M
    for t in reversed(range(n)):
        kt, e, u = k[:, t], es[t], th[:, t].unsqueeze(-1) * es[t]
        dq_[:, t] = sc * torch.einsum("bhvk,bhv->bhk", Mt, dy[:, t])
        lam = lam + sc * dy[:, t].unsqueeze(-1) * q[:, t].unsqueeze(-2)
        du = torch.einsum("bhvk,bhk->bhv", lam, kt)
        x = th[:, t].unsqueeze(-1) * du
        dv_[:, t], dth[:, t] = x, (du * e).sum(-1)
        R = hist[t] * r[:, t][..., None, None]
        dk_[:, t] = torch.einsum("bhvk,bhv->bhk", lam, u) - torch.einsum("bhvk,bhv->bhk", R, x)
        lam = lam - x.unsqueeze(-1) * kt.unsqueeze(-2)         # the gradient of r M_{t-1}
        dg[:, t] = (lam * R).sum((-1, -2))
        lam = lam * r[:, t][..., None, None]
        Mt = hist[t]
    fold = lambda t: t.view(b, n, case["hk"], share, dk).sum(3)
    out |= {"d_k": fold(dk_), "d_v": dv_, "d_q": fold(dq_), "d_log_retain": dg, "d_theta": dth}
    if s["m0"] is not None:
        out["d_m_initial"] = lam
    return out
