"""Distillation: logits of any size, and the kernels' variants at the sizes that choose them, against the definition in 64 bits.

Tolerances of `close`. A softmax value p is e^-d over a sum, d = (max - z) / tau: the subtraction, log2 e / tau and their product
are rounded, 2^-24 of d log2 e each, and ex2.approx is within 2^-22, so that p is off by p (3 d 2^-24 + 2^-22) before the sum, and p d
is 0.37 at most; the sum's error is a mean of the same and its own rounding: below 2^-20 of the row's weights in all, whatever the
logits' size. A row's loss is a sum of five numbers that are each rounded at 2^-24 of some 30: 2^-18 of the terms' mean
size, and half a step of fp32. bf16 gradients: half a step (2^-8) on top."""
import math
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
from test_gpu_distill import definition, make  # noqa: E402

pytestmark = pytest.mark.gpu


def close(z, ids, t, y, tau, sw, hw):
    from nl_hecate_b200 import dispatch as D
    want, wg, size = definition(z, ids, t, y, tau, sw, hw)
    loss, saved = D.distill_forward(z, ids, t, targets=y, temperature=tau, soft_weight=sw, hard_weight=hw)
    d = D.distill_backward(z, saved)
    assert abs(float(loss) - float(want)) <= 2.0 ** -18 * size + 2.0 ** -24 * abs(float(want)), (float(loss), float(want), size)
    rows_h = int(((y >= 0) & (y < z.shape[1])).sum()) if y is not None else 0
    rows_s = int(((ids >= 0) & (ids < z.shape[1])).any(1).sum())
    unit = hw / max(rows_h, 1) + sw * tau / max(rows_s, 1)
    half = 2.0 ** -8 if d.dtype == torch.bfloat16 else 2.0 ** -24
    err = (d.double() - wg).abs()
    assert bool((err <= half * wg.abs() + 2.0 ** -20 * unit).all()), float(err.max() / unit)


MODES = [(1.0, 1.0, 0.0), (2.0, 0.5, 0.5), (1.5, 0.7, 0.3), (2.0, 0.0, 1.0)]


@pytest.mark.parametrize("tau,sw,hw", MODES)
@pytest.mark.parametrize("offset", [0.0, 30.0, -300.0, 1000.0, 1e5])
@pytest.mark.parametrize("n,vocab", [(60, 50), (4100, 40), (3, 20001)])
def test_logits_far_from_zero(n, vocab, offset, tau, sw, hw):
    """An offset of all logits changes nothing but their own rounding, which the definition sees too."""
    z, ids, t, y = make(n, vocab, 9, torch.float32, seed=n)
    close(z + offset, ids, t, y, tau, sw, hw)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("tau,sw,hw", [*MODES, (0.5, 0.5, 0.5), (1e-3, 0.5, 0.5)])
def test_lowest_values_as_masks(tau, sw, hw, dtype):
    """The type's lowest value in masked places: no mass beside any other value, equal shares where a row holds nothing else; the
    same for the teacher's logits."""
    low = torch.finfo(dtype).min
    z, ids, t, y = make(24, 300, 6, dtype, seed=3)
    z[:8, 100:] = low
    z[8:12] = low
    ids[:8] %= 100
    y[:8].clamp_(0, 99)
    t[4:14, 2:] = low
    t[16:20] = low
    if tau < 0.1:
        z /= 64
        z[:8, 100:], z[8:12] = low, low
    close(z, ids, t, y, tau, sw, hw)


@pytest.mark.parametrize("n,vocab", [(6, 90), (5000, 90), (3, 20001)])
@pytest.mark.parametrize("tau", [1.0, 2.0, 3.0])
def test_an_infinite_logit_at_an_entry_is_not_left_out(tau, n, vocab):
    """The row's loss is no number, and neither is the mean; the other rows keep their gradients."""
    from nl_hecate_b200 import dispatch as D
    z, ids, t, y = make(n, vocab, 4, torch.float32, seed=1)
    y.fill_(1)
    ids.clamp_(0, vocab - 1)
    _, saved = D.distill_forward(z, ids, t, targets=y, temperature=tau, soft_weight=0.5, hard_weight=0.5)
    want = D.distill_backward(z, saved)
    bad = z.clone()
    bad[1, int(ids[1, 2])] = math.inf
    for sw, hw in ((0.5, 0.5), (1.0, 0.0)):
        loss, saved = D.distill_forward(bad, ids, t, targets=y, temperature=tau, soft_weight=sw, hard_weight=hw)
        d = D.distill_backward(bad, saved)
        assert math.isnan(float(loss)) and bool(torch.isnan(d[1]).all())
        if hw:
            assert torch.equal(d[2:], want[2:]) and torch.equal(d[:1], want[:1])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_gradient_between_the_rows_of_its_logits(dtype):
    """Logits and gradient as the two halves of one buffer's rows: no element in common, so no refusal, and neither touches the other."""
    from nl_hecate_b200 import dispatch as D
    z, ids, t, y = make(40, 300, 5, dtype)
    both = torch.full((40, 600), 7.0, dtype=dtype, device="cuda")
    both[:, :300] = z
    _, saved = D.distill_forward(both[:, :300], ids, t, targets=y, temperature=2.0, hard_weight=0.5)
    want = D.distill_backward(both[:, :300], saved)
    got = D.distill_backward(both[:, :300], saved, out=both[:, 300:])
    assert torch.equal(got, want) and torch.equal(both[:, :300], z)
    with pytest.raises(ValueError, match="overlaps"):
        D.distill_backward(both[:, :300], saved, out=both[:, 299:599])
    with pytest.raises(ValueError, match="overlaps"):
        D.distill_backward(both[:20, :300], saved_of(both[:20, :300], ids, t, y), out=both[1:21, :300])


def saved_of(z, ids, t, y):
    from nl_hecate_b200 import dispatch as D
    n = z.shape[0]
    return D.distill_forward(z, ids[:n].contiguous(), t[:n].contiguous(), targets=y[:n].contiguous(), temperature=2.0, hard_weight=0.5)[1]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("tau,sw,hw", MODES)
@pytest.mark.parametrize("n,vocab,k", [(4096, 12288, 7), (4097, 12289, 7), (5001, 513, 40), (150, 16400, 33), (149, 40003, 5), (150, 16384, 3)])
def test_the_sizes_that_choose_a_kernel(n, vocab, k, tau, sw, hw, dtype):
    """A warp per row (4096 rows and more, up to 12288 columns), a CTA of 128 or (above 16384 columns) 256 threads per row, none of them
    divided."""
    z, ids, t, y = make(n, vocab, k, dtype, seed=vocab)
    close(z, ids, t, y, tau, sw, hw)


@pytest.mark.parametrize("tau", [1e-6, 1e-4, 1e-2, 1e4, 1e6])
def test_temperatures_at_their_limits(tau):
    """At the lowest the softmax is its maximum's alone, at the highest uniform; exponents are rounded relative to themselves."""
    z, ids, t, y = make(70, 200, 6, torch.float32, seed=5)
    close(10 * z, ids, t, y, tau, 0.5, 0.5)
