"""Gated delta rule: the kernels' variants at the sizes that choose them, against the recurrence in 64 bits with the tolerances of
test_gpu_gated_delta.py, and what the variants have in common bit by bit."""
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
from test_gpu_gated_delta import inputs, run  # noqa: E402

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
