"""Gated delta rule (chunked forward and backward, recurrent step) against the token-by-token recurrence and its
adjoint in 64 bits.

Tolerances, relative to the largest value of a tensor. fp32: operands of the products carry 22 bits (2^-23 = 1.2e-7 a
factor), about eight products follow one another, sums of up to 128 terms in fp32 between them: 8 x 2 x 1.2e-7 = 2e-6;
gradients pass twice as many: 4e-6; gate gradients are sums of up to 64 of those with both signs: 2e-5. Results in bf16:
half a step, 2^-9 of the value's binade = 2^-8 relative at most, and the same again in y for its one-pass products
(2^-12 an operand, far less)."""
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
