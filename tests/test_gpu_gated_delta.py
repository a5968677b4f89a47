"""Gated delta rule (chunked forward and backward, recurrent step) against the token-by-token recurrence and its
adjoint in 64 bits.

Tolerances, relative to the largest value of a tensor. fp32: operands of the products carry 24 bits (three bf16
parts; the parts of the product that are left out and the operand's own rounding stay below 2^-23 = 1.2e-7 a factor), about
eight products follow one another, sums of up to 128 terms in fp32 between them: 8 x 2 x 1.2e-7 = 2e-6;
gradients pass twice as many: 4e-6; gate gradients are sums of up to 64 of those with both signs: 2e-5. Results in bf16:
half a step, 2^-9 of the value's binade = 2^-8 relative at most, and the same again in y for its products of
operands in two bf16 parts (2^-17 an operand, far less)."""
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

pytestmark = pytest.mark.gpu

TOL = {"y": 2e-6, "m_final": 2e-6, "d_k": 4e-6, "d_v": 4e-6, "d_q": 4e-6, "d_m_initial": 4e-6, "d_theta": 2e-5,
       "d_log_retain": 2e-5}
BF16 = 2.0 ** -8


def inputs(b, s, hk, hv, dk, dv, dtype, seed=0, carry=True, retain=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    n = lambda *sh: torch.randn(*sh, generator=g, device="cuda")
    unit = lambda *sh: torch.nn.functional.normalize(n(*sh), dim=-1)
    p = dict(k=unit(b, s, hk, dk).to(dtype), v=n(b, s, hv, dv).to(dtype), q=unit(b, s, hk, dk).to(dtype),
             log_retain=-retain * torch.exp(n(b, s, hv) - 2), theta=torch.sigmoid(n(b, s, hv)))
    p["m0"] = 0.3 * n(b, hv, dv, dk) if carry else None
    p["d_y"] = n(b, s, hv, dv).to(dtype)
    p["d_m"] = 0.3 * n(b, hv, dv, dk) if carry else None
    return p


def reference(p, scale, d_y=None, d_m=None):
    """y, m_final and, with d_y, all gradients: 64 bits, one token after the other."""
    hv = p["v"].shape[2]
    share = hv // p["k"].shape[2]
    leaves = {x: p[x].double().detach().requires_grad_(True) for x in ("k", "v", "q", "log_retain", "theta")}
    b, s, _, dv = p["v"].shape
    dk = p["k"].shape[3]
    M0 = (p["m0"].double() if p["m0"] is not None else torch.zeros(b, hv, dv, dk, dtype=torch.float64, device="cuda"))
    M = M0 = M0.detach().requires_grad_(True)
    k, q = (leaves[x].repeat_interleave(share, dim=2) for x in ("k", "q"))
    ys = []
    for t in range(s):
        R = M * torch.exp(leaves["log_retain"][:, t])[..., None, None]
        u = leaves["theta"][:, t, :, None] * (leaves["v"][:, t] - (R * k[:, t, :, None]).sum(-1))
        M = R + u[..., None] * k[:, t, :, None]
        ys.append(scale * (M * q[:, t, :, None]).sum(-1))
    y = torch.stack(ys, 1) if ys else torch.zeros(b, 0, hv, dv, dtype=torch.float64, device="cuda")
    out = {"y": y.detach(), "m_final": M.detach()}
    if d_y is not None:
        outs, grads = [y], [d_y.double()]
        if d_m is not None:
            outs.append(M)
            grads.append(d_m.double())
        gr = torch.autograd.grad(outs, [*leaves.values(), M0], grads, allow_unused=True)
        for x, t in zip([*leaves, "m_initial"], gr):
            out["d_" + x] = t if t is not None else torch.zeros_like(M0)
    return out


def check(got, want, dtype, where=""):
    for name, w in want.items():
        t = got[name]
        assert t.shape == w.shape, (where, name)
        if not w.numel():
            continue
        d = (t.double() - w).abs()
        top = float(w.abs().max())
        tol = TOL[name] * max(top, 1e-30)
        if t.dtype == torch.bfloat16:
            assert bool((d <= BF16 * w.abs() + 4 * tol + 2.0 ** -11 * top).all()), (where, name, float(d.max() / top))
        else:
            assert float(d.max()) <= tol, (where, name, float(d.max()) / max(top, 1e-30))


def run(p, scale=1.0, backward=True, starts=None):
    from nl_hecate_b200 import dispatch as D
    a = [p[x] for x in ("k", "v", "q", "log_retain", "theta")]
    y, m, saved = D.gated_delta_forward(*a, m0=p["m0"], scale=scale, seq_starts=starts)
    out = {"y": y, "m_final": m}
    if backward:
        out |= D.gated_delta_backward(*a, saved, p["d_y"], d_m_final=p["d_m"], scale=scale, seq_starts=starts)
    return out


DTYPES = [torch.float32, torch.bfloat16]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("b,s,hk,hv,dk,dv", [
    (1, 1, 1, 1, 64, 64), (2, 63, 2, 2, 64, 64), (1, 64, 1, 1, 64, 64), (2, 65, 1, 2, 64, 64), (3, 130, 2, 2, 32, 32),
    (1, 200, 1, 1, 128, 128), (2, 97, 2, 4, 64, 128), (1, 129, 1, 3, 128, 64), (2, 70, 1, 1, 48, 80), (1, 66, 2, 2, 7, 5),
    (2, 33, 1, 1, 1, 1), (1, 321, 1, 1, 100, 33)])
def test_pair_against_the_recurrence(dtype, b, s, hk, hv, dk, dv):
    p = inputs(b, s, hk, hv, dk, dv, dtype, seed=s)
    check(run(p, 0.5), reference(p, 0.5, p["d_y"], p["d_m"]), dtype)


@pytest.mark.parametrize("dtype", DTYPES)
def test_without_initial_state(dtype):
    p = inputs(2, 100, 2, 2, 64, 64, dtype, carry=False)
    want = reference(p, 1.0, p["d_y"])
    check(run(p), want, dtype)


def test_zero_tokens_and_zero_sequences():
    p = inputs(2, 0, 2, 2, 64, 64, torch.float32)
    out = run(p)
    assert torch.equal(out["m_final"], p["m0"]) and torch.equal(out["d_m_initial"], p["d_m"])
    p = inputs(0, 5, 2, 2, 64, 64, torch.float32)
    assert run(p)["y"].shape == (0, 5, 2, 64)


@pytest.mark.parametrize("dtype", DTYPES)
def test_strong_decay_and_gates_of_zero(dtype):
    """Retentions down to 0 (log -infinity) between tokens that keep nearly all, learning rates of exactly 0 and of 1."""
    p = inputs(2, 150, 2, 2, 64, 64, dtype, seed=5)
    p["log_retain"][:, ::7] = -60.0
    p["log_retain"][:, 3::11] = -float("inf")
    p["theta"][:, ::5] = 0.0
    p["theta"][:, 1::5] = 1.0
    want = reference({**p, "log_retain": p["log_retain"].clamp_min(-200.0)}, 1.0, p["d_y"], p["d_m"])
    out = run(p)
    check(out, want, dtype)
    assert not out["d_v"][:, ::5].any()


def test_gradients_against_differences():
    """Central differences of <d_y, y> + <d_m, m_final> (fp32 outputs, summed in 64 bits) along random directions of every input:
    with a step of 2^-6 the cubic term is below 1e-3 of the directional derivative here, the rounding of y far below that."""
    from nl_hecate_b200 import dispatch as D
    p = inputs(1, 90, 1, 2, 32, 32, torch.float32, seed=9)
    names = ("k", "v", "q", "log_retain", "theta", "m0")
    g = run(p)
    grads = dict(zip(names, (g["d_k"], g["d_v"], g["d_q"], g["d_log_retain"], g["d_theta"], g["d_m_initial"])))

    def f(q):
        y, m, _ = D.gated_delta_forward(*[q[x] for x in names[:5]], m0=q["m0"])
        return float((y.double() * p["d_y"].double()).sum() + (m.double() * p["d_m"].double()).sum())

    for i, name in enumerate(names):
        u = torch.randn(p[name].shape, generator=torch.Generator(device="cuda").manual_seed(i), device="cuda")
        u = u * (0.05 if name in ("log_retain", "theta") else 1.0) / u.norm() * 4
        h = 2.0 ** -6
        num = (f({**p, name: p[name] + h * u}) - f({**p, name: p[name] - h * u})) / (2 * h)
        want = float((grads[name].double() * u.double()).sum())
        size = float(grads[name].double().norm() * u.double().norm()) / u.numel() ** 0.5
        assert abs(num - want) <= 2e-3 * max(abs(want), size), (name, num, want)


def packed(lengths, hk, hv, dk, dv, dtype, seed=0, before=0, behind=0):
    total = sum(lengths) + before + behind
    p = inputs(1, total, hk, hv, dk, dv, dtype, seed=seed)
    n = len(lengths)
    g = torch.Generator(device="cuda").manual_seed(seed + 1)
    p["m0"] = 0.3 * torch.randn(n, hv, dv, dk, generator=g, device="cuda")
    p["d_m"] = 0.3 * torch.randn(n, hv, dv, dk, generator=g, device="cuda")
    at = [before]
    for x in lengths:
        at.append(at[-1] + x)
    return p, torch.tensor(at, dtype=torch.int32, device="cuda"), at


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lengths,before,behind,share", [
    ((5,), 0, 0, 1), ((64, 64), 0, 0, 1), ((1, 0, 130, 63, 0, 65), 0, 0, 1), ((0, 0, 3), 7, 11, 2), ((200, 1, 1, 1, 77), 3, 70, 2)])
def test_packed_batch(lengths, before, behind, share, dtype):
    """Sequences of any lengths, empty ones among them, in one call; nothing outside them is read or changed."""
    p, starts, at = packed(lengths, 2, 2 * share, 64, 48, dtype, seed=len(lengths), before=before, behind=behind)
    for x in ("k", "v", "q", "log_retain", "theta", "d_y"):
        p[x][:, :before] = float("nan")
        p[x][:, at[-1]:] = float("nan")
    out = run(p, 0.5, starts=starts)
    for x in ("y", "d_k", "d_v", "d_q", "d_log_retain", "d_theta"):
        assert not out[x][:, :before].any() and not out[x][:, at[-1]:].any(), x
    for i, n in enumerate(lengths):
        e = slice(at[i], at[i + 1])
        q = {x: p[x][:, e] for x in ("k", "v", "q", "log_retain", "theta")} | {"m0": p["m0"][i:i + 1]}
        got = {x: out[x][:, e] for x in ("y", "d_k", "d_v", "d_q", "d_log_retain", "d_theta")}
        got |= {"m_final": out["m_final"][i:i + 1], "d_m_initial": out["d_m_initial"][i:i + 1]}
        if n == 0:
            assert torch.equal(got["m_final"], q["m0"]) and torch.equal(got["d_m_initial"], p["d_m"][i:i + 1])
            continue
        check(got, reference(q, 0.5, p["d_y"][:, e], p["d_m"][i:i + 1]), dtype, f"sequence {i}")


@pytest.mark.parametrize("bad", [[9, 3, 200, 50], [-5, 1000, 20, 2 ** 31 - 1], [0, 0, 0, 0], [100, 0, 0, 100], [-(2 ** 31), -1, 99, 100]])
def test_starts_that_are_out_of_order_or_range_stay_inside(bad):
    """Starts count at their running maximum inside the batch: what they leave as sequences is computed, nothing else touched."""
    p, _, _ = packed((40, 30, 30), 1, 1, 64, 64, torch.float32)
    at, top = [], 0
    for x in bad:
        top = max(top, min(max(x, 0), 100))
        at.append(top)
    out = run(p, starts=torch.tensor(bad, dtype=torch.int32, device="cuda"))
    ref = run(p, starts=torch.tensor(at, dtype=torch.int32, device="cuda"))
    for x in out:
        assert torch.equal(out[x], ref[x]), x
    assert not out["y"][:, :at[0]].any() and not out["y"][:, at[-1]:].any()


def test_rows_outside_the_sequences_are_left_as_they_were():
    """The C entries themselves, which the wrapper hands zeroed buffers: shared heads, so that the sums over them are reached too."""
    import ctypes as C
    from nl_hecate_b200 import dispatch as D
    from nl_hecate_b200 import ffi
    p, starts, at = packed((70, 0, 5), 2, 4, 64, 48, torch.float32, before=3, behind=9)
    total = p["k"].shape[1]
    names = ("k", "v", "q", "log_retain", "theta")
    want = run(p, starts=starts)
    out = {x: torch.full_like(p[x], 7.0) for x in names} | {"y": torch.full_like(p["v"], 7.0)}
    st = lambda t: t.stride()[:3]
    d = ffi.GatedDeltaDesc(1, total, 2, 4, 64, 48, 3, 0, *st(p["k"]), *st(p["v"]), *st(p["q"]), *st(p["theta"]), *st(p["d_y"]), 1.0)
    ref = C.byref(d)
    saved = torch.empty(ffi.lib().nlh_gated_delta_saved_bytes(ref), dtype=torch.uint8, device="cuda")
    work = torch.full((ffi.lib().nlh_gated_delta_backward_bytes(ref),), 255, dtype=torch.uint8, device="cuda")
    m, dm = torch.empty_like(p["m0"]), torch.empty_like(p["m0"])
    ins = {x: p[x] for x in names}
    D.call("nlh_gated_delta_forward", desc=ref, **ins, m_initial=p["m0"], seq_starts=starts, y=out["y"], m_final=m, saved=saved,
           saved_bytes=saved.numel())
    D.call("nlh_gated_delta_backward", desc=ref, **ins, seq_starts=starts, saved=saved, saved_bytes=saved.numel(), d_y=p["d_y"],
           d_m_final=p["d_m"], **{"d_" + x: out[x] for x in names}, d_m_initial=dm, workspace=work, workspace_bytes=work.numel())
    assert torch.equal(m, want["m_final"]) and torch.equal(dm, want["d_m_initial"])
    for x in out:
        w = want["y" if x == "y" else "d_" + x]
        assert torch.equal(out[x][:, at[0]:at[-1]], w[:, at[0]:at[-1]]), x
        assert bool((out[x][:, :at[0]] == 7).all()) and bool((out[x][:, at[-1]:] == 7).all()), x


def test_many_sequences():
    """More sequences than the threads that number them."""
    lengths = [(i * 7) % 5 for i in range(2500)]
    p, starts, at = packed(lengths, 1, 1, 8, 8, torch.float32)
    out = run(p, starts=starts)
    for i in (0, 1, 3, 1023, 1024, 1025, 2047, 2048, 2499):
        e = slice(at[i], at[i + 1])
        if lengths[i]:
            q = {x: p[x][:, e] for x in ("k", "v", "q", "log_retain", "theta")} | {"m0": p["m0"][i:i + 1]}
            check({"y": out["y"][:, e], "m_final": out["m_final"][i:i + 1]}, reference(q, 1.0), torch.float32)


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides_alignment_and_order(dtype):
    """[batch, head, token, d] views, tensors cut out of wider rows, starts that no vector load takes, a gradient expanded over
    the batch: the same bits as their contiguous copies."""
    from nl_hecate_b200 import dispatch as D
    p = inputs(2, 75, 2, 2, 40, 40, dtype, seed=3)
    names = ("k", "v", "q", "log_retain", "theta")
    base = [p[x] for x in names]
    y, m, saved = D.gated_delta_forward(*base, m0=p["m0"])
    d_y = p["d_y"][:1].expand(2, -1, -1, -1)
    g = D.gated_delta_backward(*base, saved, d_y.contiguous(), d_m_final=p["d_m"])

    def heads_first(t):
        return t.transpose(1, 2).contiguous().transpose(1, 2)

    def cut(t, off):
        wide = torch.full((*t.shape[:-1], t.shape[-1] + 9), 5.0, dtype=t.dtype, device="cuda")
        wide[..., off:off + t.shape[-1]] = t
        return wide[..., off:off + t.shape[-1]]

    for f in (heads_first, lambda t: cut(t, 4), lambda t: cut(t, 1)):
        a = [f(t) if t.dim() == 4 else heads_first(t) for t in base]
        a[4] = a[4].contiguous()             # gates of different strides
        y2, m2, saved2 = D.gated_delta_forward(*a, m0=p["m0"])
        assert torch.equal(y, y2) and torch.equal(m, m2)
        g2 = D.gated_delta_backward(*a, saved2, d_y, d_m_final=p["d_m"])
        for x in g:
            assert torch.equal(g[x], g2[x]), x


def test_same_bits_every_time_and_on_another_stream():
    p = inputs(3, 200, 2, 4, 64, 64, torch.bfloat16, seed=2)
    a, b = run(p), run(p)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        c = run(p)
    torch.cuda.current_stream().wait_stream(st)
    torch.cuda.synchronize()
    for x in a:
        assert torch.equal(a[x], b[x]) and torch.equal(a[x], c[x]), x


def test_captured_pair_replays_on_new_inputs():
    """Two graphs, whose buffers are their own, replayed in turn."""
    sets = [inputs(2, 100, 1, 2, 64, 64, torch.float32, seed=s) for s in (1, 2)]
    run(sets[0])
    graphs, outs = [], []
    for p in sets:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(run(p))
        graphs.append(g)
    for seed in (11, 12):
        fresh = [inputs(2, 100, 1, 2, 64, 64, torch.float32, seed=seed + 10 * i) for i in range(2)]
        for p, f in zip(sets, fresh):
            for x in p:
                p[x].copy_(f[x])
        for g in graphs:
            g.replay()
        for o, f in zip(outs, fresh):
            want = run(f)
            for x in want:
                assert torch.equal(o[x], want[x]), x


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("at", [0, 17, 63, 64, 100, 129])
def test_values_that_are_not_finite_stay_behind_their_token(dtype, at):
    """A NaN or an infinity at one token (what padding may hold) leaves the tokens before it and the other sequences as they were;
    one in V stays in its column of y and its row of M."""
    p = inputs(3, 130, 2, 2, 64, 64, dtype, seed=4)
    clean = run(p)
    want = reference(p, 1.0)
    for x, bad in (("k", float("nan")), ("v", float("inf")), ("v", float("nan")), ("q", float("nan")), ("log_retain", float("nan")),
                   ("theta", float("nan"))):
        q = {**p, x: p[x].clone()}
        if x in ("k", "v", "q"):
            q[x][1, at, :, 5] = bad
        else:
            q[x][1, at] = bad
        out = run(q)
        for name in clean:
            assert torch.equal(out[name][[0, 2]], clean[name][[0, 2]]), (x, name)
        check({"y": out["y"][1:2, :at]}, {"y": want["y"][1:2, :at]}, dtype, x)
        assert not bool(torch.isfinite(out["y"][1, at, :, 5]).any()), x
        if x == "v":
            other = [c for c in range(64) if c != 5]
            check({"y": out["y"][1:2][..., other], "m_final": out["m_final"][1:2][:, :, other]},
                  {"y": want["y"][1:2][..., other], "m_final": want["m_final"][1:2][:, :, other]}, dtype, x)
        if x == "q":
            check({"y": out["y"][1:2, at + 1:], "m_final": out["m_final"][1:2]},
                  {"y": want["y"][1:2, at + 1:], "m_final": want["m_final"][1:2]}, dtype, x)


# ── recurrent step ──
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("b,s,hk,hv,dk,dv", [(1, 1, 1, 1, 64, 64), (5, 1, 2, 4, 128, 128), (3, 4, 1, 2, 48, 80), (2, 2, 1, 1, 7, 5),
                                             (300, 1, 2, 2, 64, 128), (4, 1, 1, 1, 1, 1), (7, 3, 2, 2, 128, 33)])
def test_step_against_the_recurrence(dtype, b, s, hk, hv, dk, dv):
    from nl_hecate_b200 import dispatch as D
    p = inputs(b, s, hk, hv, dk, dv, dtype, seed=b)
    want = reference(p, 0.5)
    m = p["m0"].clone()
    y = D.gated_delta_step(*[p[x] for x in ("k", "v", "q", "log_retain", "theta")], m, scale=0.5)
    check({"y": y, "m_final": m}, want, dtype)


def test_step_slots():
    """Slots in any order, unused places of the batch, states that no one names, and a slot that is named three times."""
    from nl_hecate_b200 import dispatch as D
    p = inputs(8, 2, 2, 2, 64, 64, torch.float32, seed=1)
    names = ("k", "v", "q", "log_retain", "theta")
    pool = torch.randn(10, 2, 64, 64, device="cuda")
    slots = torch.tensor([7, -1, 3, 7, 10, 0, 7, 2 ** 31 - 1], dtype=torch.int32, device="cuda")
    old = pool.clone()
    y = D.gated_delta_step(*[p[x] for x in names], pool, slots=slots)
    assert not y[1].any() and not y[4].any() and not y[7].any()
    for i in (1, 2, 4, 5, 6, 8, 9):
        assert torch.equal(pool[i], old[i])
    for slot, who in ((7, (0, 3, 6)), (3, (2,)), (0, (5,))):
        q = {x: torch.cat([p[x][i:i + 1] for i in who], 1) for x in names} | {"m0": old[slot:slot + 1]}
        want = reference(q, 1.0)
        got = torch.cat([y[i:i + 1] for i in who], 1)
        check({"y": got, "m_final": pool[slot:slot + 1]}, want, torch.float32, f"slot {slot}")


def test_captured_step_and_inference_mode():
    """A captured step advances the stored states at every replay, on the inputs of that replay; the same calls in inference mode."""
    from nl_hecate_b200 import dispatch as D
    names = ("k", "v", "q", "log_retain", "theta")
    toks = [inputs(4, 1, 2, 2, 64, 64, torch.bfloat16, seed=s) for s in range(3)]
    slots = torch.tensor([2, 0, 5, 1], dtype=torch.int32, device="cuda")
    start = torch.randn(6, 2, 64, 64, device="cuda")
    with torch.inference_mode():
        want_m, want = start.clone(), []
        for p in toks:
            want.append(D.gated_delta_step(*[p[x] for x in names], want_m, slots=slots))
    pool, cur = start.clone(), {x: toks[0][x].clone() for x in names}
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = D.gated_delta_step(*[cur[x] for x in names], pool, slots=slots)
    for p, w in zip(toks, want):
        for x in names:
            cur[x].copy_(p[x])
        g.replay()
        assert torch.equal(y, w)
    assert torch.equal(pool, want_m)


def test_two_threads_with_streams_of_their_own():
    import threading
    sets = [inputs(2, 150, 2, 2, 64, 64, torch.float32, seed=s) for s in (1, 2)]
    want, got, failed = [run(p) for p in sets], [[], []], []

    def work(i):
        try:
            st = torch.cuda.Stream()
            with torch.cuda.stream(st):
                for _ in range(20):
                    got[i].append(run(sets[i]))
            st.synchronize()
        except Exception as e:           # noqa: BLE001 - shown by the assertion below
            failed.append(e)

    torch.cuda.synchronize()
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed
    for w, outs in zip(want, got):
        for o in outs:
            for x in w:
                assert torch.equal(o[x], w[x]), x


def test_prompt_then_tokens():
    """A packed prompt's final states, stepped token by token from a pool, against the whole sequences at once."""
    from nl_hecate_b200 import dispatch as D
    lengths, extra = (70, 0, 9), 5
    whole = [inputs(1, n + extra, 2, 4, 64, 64, torch.float32, seed=i, carry=False) for i, n in enumerate(lengths)]
    names = ("k", "v", "q", "log_retain", "theta")
    prompt = [torch.cat([w[x][:, :n] for w, n in zip(whole, lengths)], 1) for x in names]
    starts = torch.tensor([0, 70, 70, 79], dtype=torch.int32, device="cuda")
    y0, m, saved = D.gated_delta_forward(*prompt, seq_starts=starts, want_saved=False)
    assert saved is None
    pool = torch.zeros(5, 4, 64, 64, device="cuda")
    slots = torch.tensor([4, 1, 0], dtype=torch.int32, device="cuda")
    pool[slots.long()] = m
    ys = []
    for t in range(extra):
        tok = [torch.cat([w[x][:, n + t:n + t + 1] for w, n in zip(whole, lengths)]) for x in names]
        ys.append(D.gated_delta_step(*tok, pool, slots=slots))
    for i, (w, n) in enumerate(zip(whole, lengths)):
        want = reference(w, 1.0)
        got = torch.cat([y0[:, int(starts[i]):int(starts[i + 1])], torch.cat([y[i:i + 1] for y in ys], 1)], 1)
        check({"y": got, "m_final": pool[slots[i]][None]}, want, torch.float32)


def test_refusals():
    from nl_hecate_b200 import dispatch as D
    p = inputs(2, 6, 2, 4, 16, 16, torch.float32)
    a = [p[x] for x in ("k", "v", "q", "log_retain", "theta")]
    bad = [
        [a[0].cpu(), *a[1:]], [a[0].half(), *a[1:]], [a[0].bfloat16(), *a[1:]], [a[0][:, :5], *a[1:]], [a[0][0], *a[1:]],
        [a[0], a[1][..., :3, :], a[2], a[3][..., :3], a[4][..., :3]], [*a[:3], a[3].double(), a[4]], [*a[:3], a[3][..., :1], a[4]],
        [a[0].transpose(2, 3).contiguous().transpose(2, 3), *a[1:]]]
    for q in bad:
        with pytest.raises((ValueError, RuntimeError)):
            D.gated_delta_forward(*q)
    wide = inputs(1, 3, 1, 1, 129, 16, torch.float32)
    with pytest.raises(RuntimeError, match="1..128"):
        D.gated_delta_forward(*[wide[x] for x in ("k", "v", "q", "log_retain", "theta")])
    with pytest.raises(ValueError):
        D.gated_delta_forward(*a, m0=p["m0"][:1])
    with pytest.raises(ValueError):
        D.gated_delta_forward(*a, seq_starts=torch.zeros(3, dtype=torch.int32, device="cuda"))     # batch 2
    y, m, saved = D.gated_delta_forward(*a)
    with pytest.raises(ValueError, match="other shapes"):
        D.gated_delta_backward(*[t[:1] for t in a], saved, p["d_y"][:1])
    cut = D.GatedDeltaSaved()
    cut.buffer, cut.desc = saved.buffer[:-256], saved.desc
    with pytest.raises(RuntimeError, match="too small"):
        D.gated_delta_backward(*a, cut, p["d_y"])
    with pytest.raises(ValueError):
        D.gated_delta_backward(*a, saved, p["d_y"].bfloat16())
    with pytest.raises(ValueError):
        D.gated_delta_step(*a, m.transpose(2, 3))
    with pytest.raises(ValueError):
        D.gated_delta_step(*a, m, slots=torch.zeros(3, dtype=torch.int32, device="cuda"))
    with pytest.raises(RuntimeError, match="fewer states"):
        D.gated_delta_step(*a, m[:1])
    D.gated_delta_step(*a, m)          # and the library goes on working


def test_sequences_of_many_lengths_in_any_order_and_no_wait_ran_out():
    """The order in which sequences are begun (longest first up to 256 of them, else as they come) does not show: the same bits as
    each sequence by itself."""
    from nl_hecate_b200 import dispatch as D, ffi
    for n in (5, 256, 257):
        lengths = tuple((37 * i) % 200 for i in range(n))
        p, starts, at = packed(lengths, 1, 1, 64, 64, torch.bfloat16)
        y, m, _ = D.gated_delta_forward(p["k"], p["v"], p["q"], p["log_retain"], p["theta"], m0=p["m0"], seq_starts=starts)
        begin = starts.tolist()
        for i in {0, 1, n // 2, n - 1}:
            cut = lambda x: p[x][:, begin[i]:begin[i + 1]].contiguous()
            y1, m1, _ = D.gated_delta_forward(cut("k"), cut("v"), cut("q"), cut("log_retain"), cut("theta"), m0=p["m0"][i:i + 1].contiguous())
            assert torch.equal(y[:, begin[i]:begin[i + 1]], y1) and torch.equal(m[i:i + 1], m1)
    assert ffi.lib().nlh_gated_delta_timeout_flag() == 0
