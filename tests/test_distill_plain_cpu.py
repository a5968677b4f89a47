"""The distillation loss in PyTorch operators (fused_glue = False) on the CPU, against the definition row by row in 64 bits. fp32 sums
of some hundred terms of one size: 2^-24 x 100 = 6e-6, held to 1e-5 of the loss and of the largest gradient."""
import math
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))


def rows(z, ids, t, y, tau, sw, hw):
    soft, hard = [], []
    for i in range(z.shape[0]):
        use = [j for j in range(ids.shape[1]) if 0 <= int(ids[i, j]) < z.shape[1] and float(t[i, j]) != -math.inf]
        lq = torch.log_softmax(z[i] / tau, 0)
        if use:
            p = torch.softmax(t[i, use].double() / tau, 0)
            soft.append(sum(p[n] * (torch.log(p[n]) - lq[int(ids[i, j])]) for n, j in enumerate(use) if p[n] > 0))
        if 0 <= int(y[i]) < z.shape[1]:
            hard.append(-torch.log_softmax(z[i], 0)[int(y[i])])
    return sw * tau ** 2 * sum(soft) / max(len(soft), 1) + hw * sum(hard) / max(len(hard), 1)


@pytest.mark.parametrize("tau", [1.0, 2.0])
def test_entries_and_rows_that_do_not_count(tau):
    """Teacher logits of -infinity, alone and as a whole row; ids outside the vocabulary; no target; a student's -infinity where the
    teacher has no mass."""
    from nl_hecate_b200.stacked_mag import _distill_plain
    g = torch.Generator().manual_seed(1)
    z = torch.randn(12, 30, generator=g)
    ids = torch.randint(0, 30, (12, 5), generator=g, dtype=torch.int32)
    ids[:] = torch.stack([torch.randperm(29, generator=g)[:5] for _ in range(12)]).int()
    t = torch.randn(12, 5, generator=g)
    y = torch.randint(-1, 29, (12,), generator=g)
    t[0:2] = -math.inf
    t[2:5, ::2] = -math.inf
    ids[5, :3], ids[6] = -1, 30
    z[7:9, 29] = -math.inf
    ids[7, 1], t[7, 1] = 29, -math.inf
    ids[8, 1], t[8, 1] = 29, -1e4          # no mass left of it in fp32
    a, b = z.clone().requires_grad_(True), z.double().requires_grad_(True)
    got, want = _distill_plain(a, ids, t, y, tau, 0.7, 0.3), rows(b, ids, t, y, tau, 0.7, 0.3)
    assert math.isfinite(float(want.detach())) and abs(float(got.detach()) - float(want.detach())) <= 1e-5 * abs(float(want.detach()))
    got.backward()
    want.backward()
    assert float((a.grad.double() - b.grad).abs().max()) <= 1e-5 * float(b.grad.abs().max())
