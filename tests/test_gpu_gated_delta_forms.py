"""Gated delta rule: the kernels' variants at the sizes that choose them, against the recurrence in 64 bits with the tolerances of
test_gpu_gated_delta.py, and what the variants have in common bit by bit."""
import math
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
from test_gpu_gated_delta import TOL, check, inputs, packed, reference, run  # noqa: E402
from test_gpu_language_step import gated_delta_ref  # noqa: E402

pytestmark = pytest.mark.gpu

STREAMS = ("k", "v", "q", "d_y")


@pytest.mark.parametrize("b,s,hk,hv,dk,dv", [(2, 150, 1, 2, 64, 64), (1, 70, 2, 2, 128, 128), (10, 130, 4, 4, 64, 64), (3, 67, 1, 1, 40, 24)])
def test_bf16_is_the_fp32_form_rounded_once(b, s, hk, hv, dk, dv):
    """A bf16 stream is exact in its one part, every other operand has the fp32 form's three: the same fp32 sums, so results
    in bf16 are those of the fp32 form rounded to nearest, and fp32 results (states, gate gradients) have the same bits."""
    p = inputs(b, s, hk, hv, dk, dv, torch.bfloat16, seed=s)
    wide = {x: (t.float() if x in STREAMS else t) for x, t in p.items()}
    got, want = run(p, 0.5), run(wide, 0.5)
    for x in want:
        assert torch.equal(got[x], want[x].to(got[x].dtype)), (x, float((got[x].double() - want[x].double()).abs().max()))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("hk,hv", [(2, 2), (2, 4)])
def test_packed_batch_without_a_token(hk, hv, dtype):
    """Sequences that are all empty, in a batch of no tokens: the states and their gradients pass through."""
    p = inputs(1, 0, hk, hv, 64, 48, dtype)
    p["m0"], p["d_m"] = torch.randn(2, hv, 48, 64, device="cuda"), torch.randn(2, hv, 48, 64, device="cuda")
    out = run(p, starts=torch.zeros(3, dtype=torch.int32, device="cuda"))
    assert torch.equal(out["m_final"], p["m0"]) and torch.equal(out["d_m_initial"], p["d_m"])
    for x in ("y", "d_k", "d_v", "d_q", "d_log_retain", "d_theta"):
        assert out[x].numel() == 0, x


WAIT = 6      # NLH_OPT_GATED_DELTA_WAIT


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_wait_that_runs_out_shows(dtype):
    """With no time for the waits of the state kernels every copy counts as lost: NaN in the states, outputs and gradients that
    depend on it, the flag set until it is cleared, and the next call right again."""
    from nl_hecate_b200 import dispatch as D
    from nl_hecate_b200 import ffi
    lib = ffi.lib()
    nan = lambda t: bool(torch.isnan(t).all())
    cases = [(inputs(2, 150, 2, 2, 64, 48, dtype, seed=1), None), (inputs(2, 70, 1, 1, 128, 128, dtype, seed=2), None),
             packed((130, 0, 7), 1, 2, 64, 64, dtype)[:2]]
    D.gated_delta_check()
    for p, starts in cases:
        a = [p[x] for x in ("k", "v", "q", "log_retain", "theta")]
        want = run(p, starts=starts)
        y, m, saved = D.gated_delta_forward(*a, m0=p["m0"], seq_starts=starts)
        try:
            assert lib.nlh_set_option(WAIT, 0) == 0
            ynan, mnan, _ = D.gated_delta_forward(*a, m0=p["m0"], seq_starts=starts)
            with pytest.raises(RuntimeError, match="did not arrive"):
                D.gated_delta_check()
            D.gated_delta_check()                     # raised once
            g = D.gated_delta_backward(*a, saved, p["d_y"], d_m_final=p["d_m"], seq_starts=starts)
            assert lib.nlh_gated_delta_timeout_flag() == 1 and lib.nlh_gated_delta_timeout_flag() == 1
        finally:
            lib.nlh_set_option(WAIT, 1)
        assert lib.nlh_gated_delta_timeout_clear() == 0 and lib.nlh_gated_delta_timeout_flag() == 0
        here = [0, 2] if starts is not None else slice(None)      # the empty sequence has no copy to wait for
        assert nan(ynan) and nan(mnan[here])
        if starts is not None:
            assert torch.equal(mnan[1], p["m0"][1]) and torch.equal(g["d_m_initial"][1], p["d_m"][1])
        for x in ("d_k", "d_v", "d_log_retain", "d_theta"):
            assert nan(g[x]), x
        assert nan(g["d_m_initial"][here])
        assert torch.equal(g["d_q"], want["d_q"])     # needs the forward's states alone
        again = run(p, starts=starts)
        for x in want:
            assert torch.equal(again[x], want[x]), x
    D.gated_delta_check()


RETAIN = (0.01, 1e-4, 1e-6, 6e-8, 1e-12)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("b,s,hk,hv,dk,dv", [(2, 150, 2, 2, 64, 64), (1, 130, 1, 2, 128, 40), (1, 64, 1, 1, 24, 128)])
def test_gate_gradient_keeps_its_factor(b, s, hk, hv, dk, dv, dtype):
    """The gradient of log_retain divided by the retention, which it carries as a factor, is the gradient of the retention: as
    accurate, at retentions of any size, as the gate gradients' tolerance says of the largest one."""
    p = inputs(b, s, hk, hv, dk, dv, dtype, seed=8)
    for i, t in enumerate((0, 5, 6, 20, 40, 62, 63, 64, 100, 101, 127, 128)):
        if t < s:
            p["log_retain"][:, t] = math.log(RETAIN[i % 5])
    r = torch.exp(p["log_retain"].double())
    want = reference(p, 0.5, p["d_y"], p["d_m"])["d_log_retain"] / r
    got = run(p, 0.5)["d_log_retain"].double() / r
    assert float((got - want).abs().max()) <= TOL["d_log_retain"] * float(want.abs().max())


@pytest.mark.parametrize("retain", [0.5, *RETAIN[:4], 0.0])
def test_memory_gradient_at_saturated_gates(retain):
    """gated_delta_memory for alpha near and at 1: the gradient of alpha against 64 bits, and small alphas that 1 - alpha would lose."""
    from nl_hecate_b200.stacked_mag import gated_delta_memory
    g = torch.Generator(device="cuda").manual_seed(3)
    n = lambda *sh: torch.randn(*sh, generator=g, device="cuda")
    unit = lambda t: torch.nn.functional.normalize(t, dim=-1)
    a = dict(k=unit(n(4, 150, 32)), v=n(4, 150, 32), q=unit(n(4, 150, 32)), alpha=0.3 * torch.sigmoid(n(4, 150)), theta=torch.sigmoid(n(4, 150)))
    a["alpha"][:, [0, 9, 10, 50, 63, 64, 130]] = 1.0 - retain
    a["alpha"][:, 70:110] = 1e-9
    m0, d_y = 0.3 * n(4, 32 * 32), n(4, 150, 32)
    leaves = {x: t.clone().requires_grad_(True) for x, t in a.items()}
    exact = {x: t.double().requires_grad_(True) for x, t in a.items()}
    y, _ = gated_delta_memory(*leaves.values(), None, m0, 64)
    w, _ = gated_delta_ref(*exact.values(), None, m0.double(), 64)
    got, want = torch.autograd.grad(y, list(leaves.values()), d_y), torch.autograd.grad(w, list(exact.values()), d_y.double())
    for x, u, v in zip(a, got, want):
        tol = TOL["d_log_retain"] if x == "alpha" else TOL["d_" + x]
        assert float((u.double() - v).abs().max()) <= tol * float(v.abs().max()), x
    assert float((y.detach().double() - w.detach()).abs().max()) <= TOL["y"] * float(w.detach().abs().max())


DTYPES = [torch.float32, torch.bfloat16]
STREAM_NAMES = ("k", "v", "q", "log_retain", "theta")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("b,s,hk,hv,dk,dv", [(10, 150, 4, 4, 64, 64), (5, 130, 2, 4, 128, 128), (38, 70, 1, 1, 128, 64), (38, 66, 1, 1, 64, 128),
                                             (38, 200, 1, 1, 7, 5), (13, 65, 1, 3, 100, 33)])
def test_pair_with_many_heads(b, s, hk, hv, dk, dv, dtype):
    """More than 148 CTAs of 16 columns: the state kernels of 32 columns, over several chunks, in both directions."""
    p = inputs(b, s, hk, hv, dk, dv, dtype, seed=s)
    check(run(p, 0.5), reference(p, 0.5, p["d_y"], p["d_m"]), dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,hk,hv,dk,dv", [(230, 1, 2, 64, 64), (300, 1, 1, 64, 40), (80, 1, 2, 128, 64), (75, 2, 2, 96, 128)])
def test_packed_batch_of_many_sequences(n, hk, hv, dk, dv, dtype):
    """The same kernels for packed batches, up to 256 sequences and more, some empty, some of three chunks."""
    lengths = tuple((53 * i) % 140 if i % 9 else 0 for i in range(n))
    p, starts, at = packed(lengths, hk, hv, dk, dv, dtype, before=2, behind=3)
    out = run(p, 0.5, starts=starts)
    for x in ("y", "d_k", "d_v", "d_q", "d_log_retain", "d_theta"):
        assert not out[x][:, :2].any() and not out[x][:, at[-1]:].any(), x
    for i in {1, 2, n // 2 + 1, n - 1, lengths.index(max(lengths)), lengths.index(0)}:
        e = slice(at[i], at[i + 1])
        if lengths[i] == 0:
            assert torch.equal(out["m_final"][i], p["m0"][i]) and torch.equal(out["d_m_initial"][i], p["d_m"][i])
            continue
        q = {x: p[x][:, e] for x in STREAM_NAMES} | {"m0": p["m0"][i:i + 1]}
        got = {x: out[x][:, e] for x in ("y", "d_k", "d_v", "d_q", "d_log_retain", "d_theta")}
        got |= {"m_final": out["m_final"][i:i + 1], "d_m_initial": out["d_m_initial"][i:i + 1]}
        check(got, reference(q, 0.5, p["d_y"][:, e], p["d_m"][i:i + 1]), dtype, f"sequence {i}")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("b,s,hk,hv,dk,dv", [(75, 1, 2, 4, 128, 128), (150, 2, 1, 2, 72, 100), (300, 1, 1, 1, 97, 64)])
def test_step_of_a_full_batch(b, s, hk, hv, dk, dv, dtype):
    """64 rows of a state a CTA where that gives every SM two."""
    from nl_hecate_b200 import dispatch as D
    p = inputs(b, s, hk, hv, dk, dv, dtype, seed=b)
    want = reference(p, 0.5)
    slots = torch.randperm(b + 3, device="cuda")[:b].to(torch.int32)
    pool = torch.full((b + 3, hv, dv, dk), 3.0, device="cuda")
    pool[slots.long()] = p["m0"]
    y = D.gated_delta_step(*[p[x] for x in STREAM_NAMES], pool, slots=slots, scale=0.5)
    check({"y": y, "m_final": pool[slots.long()]}, want, dtype)
    free = torch.ones(b + 3, dtype=torch.bool, device="cuda")
    free[slots.long()] = False
    assert bool((pool[free] == 3.0).all())
