"""Distillation loss and gradient against the definition in 64 bits.

Tolerances. The exponentials (ex2.approx 2^-22, its argument one fused multiply-add: |z| log2 e / tau 2^-24, up to 2^-19 for the
logits here) give each softmax value a relative error below 2^-18; a log-sum-exp is off by that much absolutely, and by
half a step of its own size (2^-24 x 32). Loss: 2^-17 of the sum of the two terms' sizes. Gradient: 2^-17 of the row's
weights on the values before rounding, plus half a step of the type (bf16 2^-8, fp32 2^-24 relative)."""
import math
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

pytestmark = pytest.mark.gpu


def make(n, vocab, k, dtype, seed=0, hard=True):
    g = torch.Generator(device="cuda").manual_seed(seed)
    z = (3 * torch.randn(n, vocab, generator=g, device="cuda")).to(dtype)
    ids = torch.randint(0, vocab, (n, k), generator=g, device="cuda", dtype=torch.int32)
    t = (2 * torch.randn(n, k, generator=g, device="cuda")).to(dtype)
    y = torch.randint(-1, vocab + 1, (n,), generator=g, device="cuda", dtype=torch.int32) if hard else None
    return z, ids, t, y


def definition(z, ids, t, y, tau, sw, hw):
    """(loss, gradient, sizes of the terms) in 64 bits; every entry on its own, ids may repeat."""
    z = z.double().detach().requires_grad_(True)
    n, vocab = z.shape
    loss = torch.zeros((), dtype=torch.float64, device="cuda")
    size = 0.0
    if y is not None and hw:
        ok = (y >= 0) & (y < vocab)
        if bool(ok.any()):
            ce = -torch.log_softmax(z[ok], 1).gather(1, y[ok].long().unsqueeze(1))
            loss = loss + hw * ce.sum() / ok.sum()
            size += float(hw * ce.detach().abs().mean())
    if sw:
        t = t.double() / tau
        ok = (ids >= 0) & (ids < vocab) & (t != -math.inf)
        rows = ok.any(1)
        if bool(rows.any()):
            t = torch.where(ok, t, torch.full_like(t, -math.inf))[rows]
            p = torch.softmax(t, 1)
            logq = torch.log_softmax(z[rows] / tau, 1).gather(1, ids[rows].clamp(0, vocab - 1).long())
            kl = (torch.special.xlogy(p, p) - torch.where(p > 0, p * logq, torch.zeros_like(p))).sum(1)
            loss = loss + sw * tau * tau * kl.sum() / rows.sum()
            size += float(sw * tau * tau * (p * torch.where(p > 0, logq, torch.zeros_like(p)).abs()).sum(1).mean().detach())
    grad = torch.autograd.grad(loss, z)[0] if loss.requires_grad else torch.zeros_like(z)
    return loss.detach(), grad, size


def check(z, ids, t, y, tau, sw, hw, out=None, grad=None):
    from nl_hecate_b200 import dispatch as D
    want, wg, size = definition(z, ids, t, y, tau, sw, hw)
    loss, saved = D.distill_forward(z, ids, t, targets=y, temperature=tau, soft_weight=sw, hard_weight=hw)
    assert abs(float(loss) - float(want)) <= 2.0 ** -17 * size + 1e-30, (float(loss), float(want))
    d = D.distill_backward(z, saved, grad=grad, out=out)
    g = 1.0 if grad is None else float(grad)
    n = z.shape[0]
    half = 2.0 ** -8 if d.dtype == torch.bfloat16 else 2.0 ** -24
    # each softmax value is off by 2^-18 of itself; the sum of both may cancel against p, whose weight bounds it
    weight = g * (abs(hw) + abs(sw) * tau) / 1.0
    rows_h = int(((y >= 0) & (y < z.shape[1])).sum()) if y is not None else 0
    unit = abs(hw) / max(rows_h, 1) + abs(sw) * tau / max(int(((ids >= 0) & (ids < z.shape[1])).any(1).sum()), 1)
    tol = half * (g * wg).abs() * 1.01 + 2.0 ** -17 * abs(g) * unit
    assert d.shape == z.shape and bool(((d.double() - g * wg).abs() <= tol).all()), float((d.double() - g * wg).abs().max() / unit)
    return loss, d


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("tau,sw,hw", [(1.0, 1.0, 0.0), (1.0, 0.5, 0.5), (2.0, 0.5, 0.5), (2.0, 1.0, 0.0), (3.5, 0.7, 0.3), (0.5, 0.3, 2.0),
                                       (2.0, 0.0, 1.0)])
@pytest.mark.parametrize("n,vocab,k", [(1, 1, 1), (3, 17, 5), (40, 256, 8), (7, 5003, 64), (200, 1000, 33), (2, 70001, 20)])
def test_pair_against_the_definition(n, vocab, k, tau, sw, hw, dtype):
    z, ids, t, y = make(n, vocab, k, dtype, seed=vocab)
    check(z, ids, t, y, tau, sw, hw)


@pytest.mark.parametrize("tau", [1.0, 2.0, 3.0])
def test_rows_that_masks_leave_empty(tau):
    z, ids, t, y = make(32, 300, 9, torch.float32)
    ids[:8] = -1                          # no teacher at all
    ids[8:12, 1:] = 300                   # one entry left
    t[12:16] = -math.inf                  # no teacher mass
    t[16:20, ::2] = -math.inf
    y[4:20] = -1
    y[:4] = 5
    _, d = check(z, ids, t, y, tau, 0.5, 0.5)
    assert not d[4:8].any() and not d[12:16].any()
    check(z, torch.full_like(ids, -1), t, torch.full_like(y, -1), tau, 0.5, 0.5)
    check(z, ids[:, :0].contiguous(), t[:, :0].contiguous(), y, tau, 0.5, 0.5)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_an_id_named_more_than_once(dtype):
    z, ids, t, y = make(20, 64, 12, dtype)
    ids[:, 3:9] = ids[:, :1]
    y[:10] = ids[:10, 0]
    check(z, ids, t, y, 2.0, 0.5, 0.5)


def test_masked_logits():
    """Logits of -infinity have probability 0 and gradient 0 - p; a teacher entry with mass on one makes the loss infinite."""
    from nl_hecate_b200 import dispatch as D
    z, ids, t, y = make(16, 500, 6, torch.float32)
    ids.copy_(torch.arange(6, dtype=torch.int32, device="cuda"))
    y.fill_(3)
    z[:, 100:] = -math.inf
    check(z, ids, t, y, 2.0, 0.5, 0.5)
    ids[0, 0] = 200
    loss, saved = D.distill_forward(z, ids, t, targets=y, temperature=2.0, soft_weight=0.5, hard_weight=0.5)
    assert float(loss) == math.inf
    assert bool(torch.isfinite(D.distill_backward(z, saved)).all())
    z[5, 7] = math.nan
    loss, saved = D.distill_forward(z, ids, t, targets=y, temperature=2.0, soft_weight=0.5, hard_weight=0.5)
    d = D.distill_backward(z, saved)
    assert math.isnan(float(loss)) and bool(torch.isnan(d[5]).all()) and bool(torch.isfinite(d[6:]).all())
    z.fill_(-math.inf)
    assert math.isnan(float(D.distill_forward(z, ids, t, targets=y, hard_weight=1.0)[0]))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,vocab", [(50, 777), (3, 20001)])
def test_in_place_strided_and_scaled(n, vocab, dtype):
    """Rows of a padded vocabulary; the gradient over the logits, and in rows of another alignment; columns behind stay."""
    from nl_hecate_b200 import dispatch as D
    z, ids, t, y = make(n, vocab, 16, dtype)
    wide = torch.full((n, vocab + 9), 7.0, dtype=dtype, device="cuda")
    wide[:, :vocab] = z
    grad = torch.tensor(0.37, device="cuda")
    _, d = check(z, ids, t, y, 2.0, 0.5, 0.5, grad=grad)
    _, d2 = check(wide[:, :vocab], ids, t, y, 2.0, 0.5, 0.5, grad=grad)
    # d and d2 are each held to the definition; not to the same bits, since where a row starts decides which thread adds which
    # of its elements, and fp32 sums of another grouping differ in their last bits
    odd = torch.full((n, vocab + 1), 7.0, dtype=dtype, device="cuda")
    _, d3 = check(z, ids, t, y, 2.0, 0.5, 0.5, grad=grad, out=odd[:, 1:])
    assert torch.equal(d, d3.contiguous()) and bool((odd[:, 0] == 7).all())
    loss, saved = D.distill_forward(wide[:, :vocab], ids, t, targets=y, temperature=2.0, soft_weight=0.5, hard_weight=0.5)
    D.distill_backward(wide[:, :vocab], saved, grad=grad, out=wide[:, :vocab])
    assert torch.equal(wide[:, :vocab], d2) and bool((wide[:, vocab:] == 7).all())


def test_captured_pair_replays_on_new_inputs():
    from nl_hecate_b200 import dispatch as D
    z, ids, t, y = make(300, 400, 7, torch.bfloat16)
    call = lambda a: D.distill_forward(a[0], a[1], a[2], targets=a[3], temperature=2.0, soft_weight=0.5, hard_weight=0.5)
    D.distill_backward(z, call((z, ids, t, y))[1])
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        loss, saved = call((z, ids, t, y))
        d = D.distill_backward(z, saved)
    for seed in (1, 2):
        fresh = make(300, 400, 7, torch.bfloat16, seed=seed)
        for dst, src in zip((z, ids, t, y), fresh):
            dst.copy_(src)
        g.replay()
        w, s = call(fresh)
        assert torch.equal(loss, w) and torch.equal(d, D.distill_backward(fresh[0], s))


def test_refusals():
    from nl_hecate_b200 import dispatch as D
    z, ids, t, y = make(6, 50, 4, torch.float32)
    for bad in ((z.half(), ids, t), (z[0], ids, t), (z, ids.long(), t), (z, ids[:5], t[:5]), (z, ids, t[:, :3]), (z, ids, t.half()),
                (z.t().contiguous().t(), ids, t), (z, ids.cpu(), t)):
        with pytest.raises(ValueError):
            D.distill_forward(*bad)
    with pytest.raises(ValueError):
        D.distill_forward(z, ids, t, targets=y[:5])
    with pytest.raises(RuntimeError, match="temperature"):
        D.distill_forward(z, ids, t, temperature=0.0)
    wide = torch.randn(6, 100, device="cuda")
    loss, saved = D.distill_forward(wide[:, :50], ids, t)
    with pytest.raises(ValueError, match="overlaps"):
        D.distill_backward(wide[:, :50], saved, out=wide[:, 8:58])
    with pytest.raises(ValueError):
        D.distill_backward(z[:, :49], saved)
    with pytest.raises(ValueError):
        D.distill_backward(z, saved, grad=torch.ones(2, device="cuda"))


def test_no_rows_and_repeatable_bits():
    from nl_hecate_b200 import dispatch as D
    z, ids, t, y = make(0, 100, 4, torch.float32)
    loss, saved = D.distill_forward(z, ids, t, targets=y, hard_weight=1.0)
    assert float(loss) == 0.0 and D.distill_backward(z, saved).shape == (0, 100)
    z, ids, t, y = make(3000, 513, 8, torch.float32)
    a = [D.distill_forward(z, ids, t, targets=y, temperature=1.5, hard_weight=1.0)[0] for _ in range(3)]
    assert torch.equal(a[0], a[1]) and torch.equal(a[0], a[2])


def test_gradient_against_differences():
    """Central differences of the fp32 loss along random directions: step h, error h^2 and 2^-22 / h of the loss."""
    from nl_hecate_b200 import dispatch as D
    z, ids, t, y = make(6, 40, 5, torch.float32)
    f = lambda x: float(D.distill_forward(x.contiguous(), ids, t, targets=y, temperature=2.0, soft_weight=0.5, hard_weight=0.5)[0])
    _, saved = D.distill_forward(z, ids, t, targets=y, temperature=2.0, soft_weight=0.5, hard_weight=0.5)
    d = D.distill_backward(z, saved)
    for i in range(4):
        u = torch.randn(z.shape, generator=torch.Generator(device="cuda").manual_seed(i), device="cuda")
        h = 2.0 ** -7
        num = (f(z + h * u) - f(z - h * u)) / (2 * h)
        assert abs(num - float((d * u).sum())) <= 2e-3
