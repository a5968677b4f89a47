"""Scaled embedding lookup and its gradient by sorted tokens against 64-bit sums.

Tolerances. Lookup: one product, half a step of the result's type (fp32 2^-24, bf16 2^-8 relative). Gradient: a sum of m rows in
fp32, taken one after the other in the worst case, is off by at most (m + 2) 2^-24 times the sum of the magnitudes, the product
with the scale and the sum with the old value included."""
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

pytestmark = pytest.mark.gpu


def make(n, vocab, d, dtype, kind, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    if kind == "same":
        ids = torch.full((n,), vocab // 2, dtype=torch.int32, device="cuda")
    elif kind == "hot":            # half of the tokens are one id, the rest spread, some outside the vocabulary
        ids = torch.randint(-1, vocab + 1, (n,), generator=g, device="cuda", dtype=torch.int32)
        ids[torch.rand(n, generator=g, device="cuda") < 0.5] = vocab - 1
    elif kind == "none":
        ids = torch.full((n,), -1, dtype=torch.int32, device="cuda")
        ids[::2] = vocab
    else:
        ids = torch.randint(0, vocab, (n,), generator=g, device="cuda", dtype=torch.int32)
    dy = torch.randn(n, d, generator=g, device="cuda").to(dtype)
    dw = torch.randn(vocab, d, generator=g, device="cuda")
    return ids, dy, dw


def sums(ids, dy, vocab):
    ok = (ids >= 0) & (ids < vocab)
    at, rows = ids[ok].long(), dy[ok].double()
    z = lambda: torch.zeros(vocab, dy.shape[1], dtype=torch.float64, device="cuda")
    count = torch.zeros(vocab, dtype=torch.float64, device="cuda").index_add_(0, at, torch.ones_like(at, dtype=torch.float64))
    return z().index_add_(0, at, rows), z().index_add_(0, at, rows.abs()), count.unsqueeze(1)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,vocab,d", [(0, 5, 8), (1, 1, 1), (7, 3, 5), (33, 100, 64), (100, 7, 12), (257, 50, 136), (3000, 911, 24)])
def test_lookup(dtype, n, vocab, d):
    from nl_hecate_b200 import dispatch as D
    g = torch.Generator(device="cuda").manual_seed(1)
    w = torch.randn(vocab, d, generator=g, device="cuda").to(dtype)
    ids = torch.randint(-2, vocab + 2, (n,), generator=g, device="cuda", dtype=torch.int32)
    out = D.embedding_forward(w, ids, scale=1.7)
    ok = (ids >= 0) & (ids < vocab)
    want = torch.where(ok.unsqueeze(1), w.double()[ids.clamp(0, vocab - 1).long()] * float(torch.tensor(1.7, dtype=torch.float32)),
                       torch.zeros((), dtype=torch.float64, device="cuda"))
    half = torch.finfo(dtype).eps / 2 if dtype == torch.float32 else 2.0 ** -8
    assert out.dtype == dtype and bool(((out.double() - want).abs() <= half * want.abs() * (1 + 1e-6)).all())
    assert D.embedding_forward(w, ids.view(1, -1)).shape == (1, n, d)


@pytest.mark.parametrize("accumulate", [True, False])
@pytest.mark.parametrize("kind", ["spread", "hot", "same", "none"])
@pytest.mark.parametrize("n,vocab,d,dtype", [
    (1, 1, 1, torch.float32), (5, 9, 3, torch.bfloat16), (64, 256, 64, torch.float32), (2048, 300, 40, torch.bfloat16),
    (2049, 300, 40, torch.bfloat16), (2049, 70000, 9, torch.float32), (5000, 513, 512, torch.float32), (4096, 31, 1032, torch.bfloat16),
    (140000, 1000, 8, torch.float32), (270000, 300000, 4, torch.float32), (6007, 511, 1, torch.float32), (6007, 512, 2, torch.float32),
    (4096, 300, 40, torch.bfloat16), (4097, 300, 40, torch.float32), (1024, 90, 1024, torch.float32), (1025, 90, 1024, torch.bfloat16),
    (30, 11, 35003, torch.float32), (1, 2, 1 << 20, torch.bfloat16), (2, 2, 1 << 20, torch.float32)])
def test_gradient(n, vocab, d, dtype, kind, accumulate):
    from nl_hecate_b200 import dispatch as D
    ids, dy, dw = make(n, vocab, d, dtype, kind, seed=n)
    old = dw.clone()
    D.embedding_backward(dy, ids, dw, scale=0.75, accumulate=accumulate)
    s, mag, count = sums(ids, dy, vocab)
    want = 0.75 * s + (old.double() if accumulate else 0.0)
    tol = 2.0 ** -24 * ((count + 2) * 0.75 * mag + (old.double().abs() if accumulate else 0.0) + want.abs())
    assert bool(((dw.double() - want).abs() <= tol).all())
    if accumulate:
        untouched = (count == 0).squeeze(1)
        assert torch.equal(dw[untouched], old[untouched])
    again = old.clone()
    D.embedding_backward(dy, ids, again, scale=0.75, accumulate=accumulate)
    assert torch.equal(again, dw), "the same call, other bits"


def test_gradient_is_the_adjoint_of_the_lookup():
    """<d_out, lookup(w + h) - lookup(w)> = <gradient, h>: the lookup is linear, so differences are exact up to rounding
    (4096 x 32 products of normal numbers: 2^-24 times the square root of their count, a hundredfold allowed)."""
    from nl_hecate_b200 import dispatch as D
    ids, dy, dw = make(4096, 97, 32, torch.float32, "hot")
    h = torch.randn_like(dw)
    D.embedding_backward(dy, ids, dw, scale=2.0, accumulate=False)
    left = (D.embedding_forward(h, ids, scale=2.0).double() * dy.double()).sum()
    right = (dw.double() * h.double()).sum()
    assert abs(float(left - right)) <= 100 * 2.0 ** -24 * 362 * 2


def test_unaligned_buffers():
    from nl_hecate_b200 import dispatch as D
    ids, dy, dw = make(3000, 50, 16, torch.float32, "spread")
    buf, gbuf = torch.empty(3000 * 16 + 1, device="cuda"), torch.zeros(50 * 16 + 1, device="cuda")
    dy1, dw1 = buf[1:].view(3000, 16), gbuf[1:].view(50, 16)
    dy1.copy_(dy)
    dw1.copy_(dw)
    assert torch.equal(D.embedding_backward(dy1, ids, dw1), D.embedding_backward(dy, ids, dw))


def test_captured_gradient_replays():
    from nl_hecate_b200 import dispatch as D
    ids, dy, dw = make(5000, 513, 64, torch.float32, "hot")
    dw.zero_()
    D.embedding_backward(dy, ids, dw)              # sizes and attributes
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        D.embedding_backward(dy, ids, dw, accumulate=False)
    for seed in (3, 4):
        i2, d2, _ = make(5000, 513, 64, torch.float32, "hot", seed)
        ids.copy_(i2)
        dy.copy_(d2)
        g.replay()
        want = D.embedding_backward(d2, i2, torch.zeros_like(dw))
        assert torch.equal(dw, want)


@pytest.mark.parametrize("n,vocab", [(2500, 1), (3000, 7), (40000, 2), (70000, 300), (131072, 40), (131073, 40)])
def test_tiny_vocabularies_and_borders_of_the_sorts(n, vocab):
    """Fewer ids than a warp has lanes; the largest list that one launch sorts, and the first that it does not."""
    from nl_hecate_b200 import dispatch as D
    ids, dy, dw = make(n, vocab, 4, torch.float32, "hot", seed=vocab)
    old = dw.clone()
    D.embedding_backward(dy, ids, dw)
    s, mag, count = sums(ids, dy, vocab)
    tol = 2.0 ** -24 * ((count + 2) * mag + old.double().abs() + (old.double() + s).abs())
    assert bool(((dw.double() - old.double() - s).abs() <= tol).all())


def test_refusals():
    from nl_hecate_b200 import dispatch as D
    ids, dy, dw = make(30, 50, 8, torch.float32, "spread")
    w = dw.clone()
    for bad in ((w.half(), ids), (w.t(), ids), (w[0], ids), (w, ids.long()), (w, ids.cpu()), (w, ids[::2])):
        with pytest.raises(ValueError):
            D.embedding_forward(*bad)
    for bad in ((dy.half(), ids, dw), (dy[:29], ids, dw), (dy[:, :4], ids, dw), (dy, ids.long(), dw), (dy, ids, dw.bfloat16()),
                (dy, ids, dw.t()), (dy.t().contiguous().t(), ids, dw), (dy.cpu(), ids, dw)):
        with pytest.raises(ValueError):
            D.embedding_backward(*bad)
