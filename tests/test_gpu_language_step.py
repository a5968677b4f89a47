"""The operators together, as the stacked model uses them: scaled embedding with its gradient by sorted tokens, gated delta memory on
every level, distillation loss; against the same model in plain PyTorch operators."""
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
from torch_ref import swa_ref  # noqa: E402

pytestmark = pytest.mark.gpu


def gated_delta_ref(k, v, q, alpha, theta, eta, m0, chunk):
    n, s, d = k.shape
    M, ys = m0.clone().view(n, d, d), []        # the model updates its memories in place
    for t in range(s):
        M = M * (1 - alpha[:, t])[:, None, None]
        u = theta[:, t, None] * (v[:, t] - (M * k[:, t, None]).sum(-1))
        M = M + u[..., None] * k[:, t, None]
        ys.append((M * q[:, t, None]).sum(-1))
    return torch.stack(ys, 1), M.reshape(n, d * d).detach()


def config(bf16=False, fused=True, **kw):
    from nl_hecate_b200.stacked_mag import StackedMAGConfig
    return StackedMAGConfig(d_model=128, num_heads=2, n_blocks=2, k=3, chunk_sizes=(1, 4, 16), seq_len=96, window=32, vocab=97, bf16=bf16,
                            fused_glue=fused, memory_rule="gated_delta", embed_scale=11.3, embed_sorted_grad=True, **kw)


def data(batch, seed=0):
    g = torch.Generator().manual_seed(seed)
    tok = torch.randint(0, 97, (batch, 97), generator=g)
    ids = torch.randint(-1, 97, (batch, 96, 6), generator=g).to(torch.int32)
    top = torch.randn(batch, 96, 6, generator=g)
    return tok[:, :-1].contiguous().cuda(), tok[:, 1:].contiguous().cuda(), (ids.cuda(), top.cuda())


def test_model_step_matches_plain_operators():
    """fp32: loss within 1e-5, every gradient within 2e-3 of its tensor's largest entry, as the model's other parity tests."""
    from nl_hecate_b200.stacked_mag import StackedMAG
    ours = StackedMAG(config(), 3, seed=7)
    ref = StackedMAG(config(fused=False), 3, seed=7, memory_fn=gated_delta_ref, swa_fn=swa_ref)
    tok, tgt, teacher = data(3)
    for _ in range(2):                       # the second pass runs on carried memories
        ours.opt.g.zero_()
        ref.opt.g.zero_()
        a, b = ours.forward_backward(tok, tgt, teacher=teacher), ref.forward_backward(tok, tgt, teacher=teacher)
        assert abs(float(a) - float(b)) <= 1e-5 * abs(float(b))
    for i, n in enumerate(ours.names):
        x, y = ours.opt.view(ours.opt.g, i), ref.opt.view(ref.opt.g, i)
        top = float(y.abs().max())
        if top < 1e-7:
            assert float(x.abs().max()) < 1e-5, n
            continue
        assert float((x - y).abs().max()) <= 2e-3 * top, n
    for b in range(2):
        for l in range(3):
            x, y = ours.context[b][l], ref.context[b][l]
            assert float((x - y).abs().max()) <= 1e-3 * max(float(y.abs().max()), 1e-6)


def test_teacher_entries_without_mass():
    """Teacher logits of -infinity, a whole position of them among others: unused for the kernels and for the plain operators alike."""
    from nl_hecate_b200.stacked_mag import StackedMAG
    ours = StackedMAG(config(), 3, seed=7)
    ref = StackedMAG(config(fused=False), 3, seed=7, memory_fn=gated_delta_ref, swa_fn=swa_ref)
    tok, tgt, (ids, top) = data(3)
    top[:, ::5] = -float("inf")
    top[:, 1::5, ::2] = -float("inf")
    with torch.no_grad():
        a, b = ours.forward(tok, tgt, (ids, top)), ref.forward(tok, tgt, (ids, top))
    assert abs(float(a) - float(b)) <= 1e-5 * abs(float(b))


@pytest.mark.parametrize("with_teacher", [True, False])
def test_graphed_step_equals_eager(with_teacher):
    from nl_hecate_b200.stacked_mag import StackedMAG
    a, b = StackedMAG(config(bf16=True), 2, seed=1), StackedMAG(config(bf16=True), 2, seed=1)
    kw = lambda t: {"teacher": t} if with_teacher else {}
    tok, tgt, teacher = data(2)
    for _ in range(3):
        la = a.step(tok, tgt, **kw(teacher))
    lb = b.step_graphed(tok, tgt, **kw(teacher))        # two eager steps and the captured one
    for seed in (5, 6):
        tok, tgt, teacher = data(2, seed)
        la, lb = a.step(tok, tgt, **kw(teacher)), b.step_graphed(tok, tgt, **kw(teacher))
        assert abs(float(la) - float(lb)) <= 1e-3 * abs(float(la))
    with pytest.raises(ValueError, match="teacher"):
        b.step_graphed(tok, tgt, **({} if with_teacher else {"teacher": teacher}))
    if with_teacher:      # one entry would be broadcast to all of the captured step's
        with pytest.raises(ValueError, match="shapes"):
            b.step_graphed(tok, tgt, teacher=tuple(t[..., :1] for t in teacher))


def test_unknown_rule_is_refused():
    from nl_hecate_b200.stacked_mag import StackedMAG, StackedMAGConfig
    with pytest.raises(ValueError, match="memory_rule"):
        StackedMAG(StackedMAGConfig(d_model=64, num_heads=1, n_blocks=1, k=1, chunk_sizes=(1,), memory_rule="delta2"), 1)


def test_sizes_of_more_than_32_bits_are_refused():
    """Sizes go to the C entries in 32 bits: 2^32 + 2 rows would count as two. The buffers are allocated, not touched."""
    from nl_hecate_b200 import dispatch as D
    n = 2 ** 32 + 2
    few = torch.zeros(3, dtype=torch.int32, device="cuda")
    row = torch.empty(n, 1, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ValueError, match="2\\^31"):
        D.embedding_forward(row, few)
    with pytest.raises(ValueError, match="2\\^31"):
        D.distill_forward(row, few.new_zeros(n, 0), row[:, :0].contiguous())
    ids = torch.empty(n, dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError, match="2\\^31"):
        D.embedding_forward(row[:4], ids)
    with pytest.raises(ValueError, match="2\\^31"):
        D.embedding_backward(row, ids, torch.zeros(4, 1, device="cuda"))
    one = torch.zeros(1, 1, 1, 1, device="cuda")
    pool = torch.empty(n, 1, 1, 1, device="cuda")
    with pytest.raises(ValueError, match="2\\^31"):
        D.gated_delta_step(one, one, one, one[0], one[0], pool)
