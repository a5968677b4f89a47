"""What the C entries of the gated delta rule, the sorted embedding gradient and the distillation refuse before they touch a
device, and the sizes they ask for. Nothing is launched here."""
import ctypes as C
import os
import sys

import pytest

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

OK, BAD = 0, 1


@pytest.fixture(scope="module")
def lib():
    from nl_hecate_b200 import build, ffi
    build.build()
    return ffi.lib()


@pytest.fixture(autouse=True)
def clear(lib):
    yield
    lib.nlh_clear_status()


def desc(**kw):
    from nl_hecate_b200 import ffi
    d = dict(batch=2, seq=70, heads_k=2, heads_v=4, dk=64, dv=64, n_seqs=0, is_bf16=0, scale=1.0)
    d.update(kw)
    return ffi.GatedDeltaDesc(**d)


def test_desc_layout_matches_header_and_packing():
    import re
    from nl_hecate_b200 import dispatch, ffi
    text = open(ffi.HEADER).read()
    body = re.search(r"typedef struct nlh_gated_delta_desc \{(.*?)\}", text, re.S).group(1)
    body = re.sub(r"/\*.*?\*/", "", body, flags=re.S)
    names = [n.strip() for decl in re.findall(r"(?:int32_t|int64_t|float)\s+([^;]+);", body) for n in decl.split(",")]
    assert names == [f[0] for f in ffi.GatedDeltaDesc._fields_]
    vals = list(range(1, 24)) + [0.5]
    assert bytes(ffi.GatedDeltaDesc(*vals))[:dispatch._DESC.size] == dispatch._DESC.pack(*vals)


def test_sizes(lib):
    d = desc()
    saved, back = lib.nlh_gated_delta_saved_bytes(C.byref(d)), lib.nlh_gated_delta_backward_bytes(C.byref(d))
    tiles = 2 * 2 * 4                      # two chunks of 64 a sequence, four heads
    assert saved >= tiles * (64 * 64 * 4 * 3) and back >= tiles * 64 * 64 * 4 * 3
    assert lib.nlh_gated_delta_saved_bytes(C.byref(desc(seq=0))) == 0
    assert lib.nlh_gated_delta_saved_bytes(C.byref(desc(batch=1, seq=100, n_seqs=7))) > 0
    assert lib.nlh_embedding_backward_bytes(100, 1000, 64) == 0 and lib.nlh_embedding_backward_bytes(5000, 1000, 64) >= 5000 * 16
    assert lib.nlh_embedding_backward_bytes((1 << 30) + 1, 10, 4) == -1
    assert lib.nlh_embedding_backward_bytes(1, 10, (1 << 20) + 1) == -1 and lib.nlh_embedding_backward_bytes(0, 10, 1 << 20) == 0
    assert lib.nlh_embedding_backward_bytes(-1, 10, 4) == -1 and lib.nlh_embedding_backward_bytes(1, 0, 4) == -1
    assert lib.nlh_distill_saved_bytes(0, 10) >= 0 and lib.nlh_distill_saved_bytes(-1, 10) == -1
    assert lib.nlh_distill_saved_bytes((1 << 30) + 1, 1) == -1 and lib.nlh_distill_saved_bytes(1, (1 << 30) + 1) == -1
    # bytes that pass 32 bits
    assert lib.nlh_gated_delta_saved_bytes(C.byref(desc(batch=64, seq=65536, heads_k=16, heads_v=16, dk=128, dv=128))) > 1 << 36


@pytest.mark.parametrize("bad", [dict(batch=-1), dict(seq=-1), dict(heads_k=0), dict(heads_v=3), dict(dk=0), dict(dk=129), dict(dv=200),
                                 dict(n_seqs=-1), dict(n_seqs=3), dict(batch=1 << 20, seq=1 << 12),
                                 dict(batch=1 << 15, seq=(1 << 15) + 1), dict(batch=1, seq=10, n_seqs=(1 << 30) + 1), dict(batch=1 << 29, seq=1)])
def test_gated_delta_refuses(lib, bad):
    d = desc(**bad)
    p = C.c_void_p(4096)                   # never followed: the descriptor is refused first
    assert lib.nlh_gated_delta_saved_bytes(C.byref(d)) == -1
    assert lib.nlh_gated_delta_forward(C.byref(d), p, p, p, p, p, None, None, p, p, p, 1 << 40) == BAD
    assert lib.nlh_gated_delta_backward(C.byref(d), p, p, p, p, p, None, p, 1 << 40, p, None, p, p, p, p, p, None, p, 1 << 40) == BAD
    assert lib.nlh_gated_delta_step(C.byref(d), p, p, p, p, p, p, None, 1 << 20, p) == BAD
    assert lib.nlh_last_status() == BAD and lib.nlh_last_error()


def test_gated_delta_refuses_buffers(lib):
    d, p = desc(), C.c_void_p(4096)
    n = lib.nlh_gated_delta_saved_bytes(C.byref(d))
    f = lib.nlh_gated_delta_forward
    assert f(None, p, p, p, p, p, None, None, p, p, p, n) == BAD
    assert f(C.byref(d), None, p, p, p, p, None, None, p, p, p, n) == BAD
    assert f(C.byref(d), p, p, p, p, p, None, None, None, p, p, n) == BAD
    assert f(C.byref(d), p, p, p, p, p, None, None, p, None, p, n) == BAD
    assert f(C.byref(d), p, p, p, p, p, None, None, p, p, None, n) == BAD
    assert f(C.byref(d), p, p, p, p, p, None, None, p, p, p, n - 1) == BAD
    assert f(C.byref(d), p, p, p, p, p, None, None, p, p, C.c_void_p(4100), n) == BAD
    assert f(C.byref(d), p, p, p, p, p, None, p, p, p, p, n) == BAD             # starts without n_seqs
    assert f(C.byref(desc(batch=1, n_seqs=2)), p, p, p, p, p, None, None, p, p, p, 1 << 40) == BAD
    w = lib.nlh_gated_delta_backward_bytes(C.byref(d))
    b = lib.nlh_gated_delta_backward
    assert b(C.byref(d), p, p, p, p, p, None, p, n, p, None, p, p, p, p, p, None, p, w - 1) == BAD
    assert b(C.byref(d), p, p, p, p, p, None, p, n - 1, p, None, p, p, p, p, p, None, p, w) == BAD
    assert b(C.byref(d), p, p, p, p, p, None, p, n, None, None, p, p, p, p, p, None, p, w) == BAD
    s = lib.nlh_gated_delta_step
    assert s(C.byref(d), p, p, p, p, p, None, None, 2, p) == BAD and s(C.byref(d), p, p, p, p, p, p, None, 1, p) == BAD
    assert s(C.byref(d), p, p, p, p, p, p, p, -1, p) == BAD


def test_packed_batch_without_a_token_needs_its_buffers(lib):
    """It has chunk slots to number although it has no rows: a NULL buffer of the right size is refused."""
    d, p = desc(batch=1, seq=0, n_seqs=2), C.c_void_p(4096)
    n, w = lib.nlh_gated_delta_saved_bytes(C.byref(d)), lib.nlh_gated_delta_backward_bytes(C.byref(d))
    assert n > 0 and w > 0
    none = (None,) * 5
    assert lib.nlh_gated_delta_forward(C.byref(d), *none, p, p, None, p, None, n) == BAD
    b = lib.nlh_gated_delta_backward
    assert b(C.byref(d), *none, p, None, n, None, None, *none, p, p, w) == BAD
    assert b(C.byref(d), *none, p, p, n, None, None, *none, p, None, w) == BAD


def test_embedding_refuses(lib):
    p = C.c_void_p(4096)
    assert lib.nlh_embedding_forward(p, 0, p, p, -1, 10, 4, 1.0) == BAD and lib.nlh_embedding_forward(None, 0, p, p, 3, 10, 4, 1.0) == BAD
    assert lib.nlh_embedding_forward(p, 0, p, p, 3, 0, 4, 1.0) == BAD and lib.nlh_embedding_forward(p, 0, p, p, 3, 10, (1 << 20) + 1, 1.0) == BAD
    assert lib.nlh_embedding_forward(None, 0, None, None, 0, 10, 4, 1.0) == OK
    f = lib.nlh_embedding_backward
    need = lib.nlh_embedding_backward_bytes(5000, 10, 4)
    assert f(p, 0, p, None, 3, 10, 4, 1.0, 1, None, 0) == BAD and f(None, 0, p, p, 3, 10, 4, 1.0, 1, None, 0) == BAD
    assert f(p, 0, p, p, 5000, 10, 4, 1.0, 1, None, need) == BAD and f(p, 0, p, p, 5000, 10, 4, 1.0, 1, p, need - 1) == BAD
    assert f(p, 0, p, p, 5000, 10, 4, 1.0, 1, C.c_void_p(4104), need) == BAD
    assert f(None, 0, None, p, 0, 10, 4, 1.0, 1, None, 0) == OK


def test_distill_refuses(lib):
    p = C.c_void_p(4096)
    n = lib.nlh_distill_saved_bytes(3, 50)

    def fwd(logits=p, stride=50, targets=p, ids=p, top=p, loss=p, saved=p, nbytes=n, rows=3, vocab=50, k=4, tau=2.0, hard=0.5, soft=0.5):
        return lib.nlh_distill_forward(logits, 0, stride, targets, ids, top, 0, loss, saved, nbytes, rows, vocab, k, tau, hard, soft)

    for kw in (dict(logits=None), dict(stride=49), dict(top=None), dict(loss=None), dict(saved=None), dict(nbytes=n - 1), dict(rows=-1),
               dict(vocab=0), dict(vocab=(1 << 30) + 1, stride=1 << 31), dict(k=-1), dict(k=1025), dict(tau=0.0), dict(tau=-1.0), dict(tau=float("nan")), dict(tau=float("inf")),
               dict(saved=C.c_void_p(4104))):
        assert fwd(**kw) == BAD, kw
    b = lib.nlh_distill_backward
    assert b(p, 0, 50, p, p, p, 0, p, n, None, None, 50, 3, 50, 4, 2.0, 0.5, 0.5) == BAD
    assert b(p, 0, 50, p, p, p, 0, p, n, None, p, 49, 3, 50, 4, 2.0, 0.5, 0.5) == BAD
    assert b(p, 0, 50, p, p, p, 0, p, n - 1, None, p, 50, 3, 50, 4, 2.0, 0.5, 0.5) == BAD


def test_host_tensors_are_refused():
    import torch
    from nl_hecate_b200 import dispatch as D
    z = torch.zeros
    with pytest.raises(ValueError, match="CUDA"):
        D.embedding_forward(z(4, 8), z(3, dtype=torch.int32))
    with pytest.raises(ValueError, match="CUDA"):
        D.embedding_backward(z(3, 8), z(3, dtype=torch.int32), z(4, 8))
    with pytest.raises(ValueError, match="CUDA"):
        D.distill_forward(z(3, 9), z(3, 2, dtype=torch.int32), z(3, 2))
    with pytest.raises(ValueError, match="CUDA"):
        D.gated_delta_step(z(1, 1, 1, 8), z(1, 1, 1, 8), z(1, 1, 1, 8), z(1, 1, 1), z(1, 1, 1), z(1, 1, 8, 8))


def test_package_imports_and_refuses_without_cuda_bindings():
    """A PyTorch built without CUDA has no device and stream queries: importing works, and the operators refuse its tensors."""
    import subprocess
    code = """
import torch
for x in ("_cuda_getDevice", "_cuda_getCurrentRawStream"):
    delattr(torch._C, x)
import nl_hecate_b200.stacked_mag
from nl_hecate_b200 import dispatch as D
z = torch.zeros
try:
    D.embedding_forward(z(4, 8), z(3, dtype=torch.int32))
except ValueError as e:
    assert "CUDA" in str(e)
else:
    raise SystemExit("not refused")
"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-800:]


def test_gradients_that_overlap_their_logits(lib):
    """Rows of both as sets of elements, against the wrapper's and the C entry's answers: the same elements in the same places are
    allowed, rows that lie between each other's, and nothing that shares an element otherwise."""
    import torch
    from nl_hecate_b200 import dispatch as D
    store = torch.zeros(400)
    base = store.data_ptr()
    n, need = 0, lib.nlh_distill_saved_bytes(4, 7)
    p = C.c_void_p(4096)
    for rows in (1, 2, 4):
        for width, za, zr, dr in ((7, 40, 20, 20), (7, 40, 14, 14), (7, 40, 7, 7), (5, 100, 9, 9), (7, 60, 20, 10), (7, 60, 7, 20)):
            for da in range(0, 200):
                if da + (rows - 1) * dr + width > 400:
                    continue
                z = store.as_strided((rows, width), (zr, 1), za)
                d = store.as_strided((rows, width), (dr, 1), da)
                at = lambda a, r: [a + i * r + j for i in range(rows) for j in range(width)]
                same = at(za, zr) == at(da, dr)
                shares = not same and bool(set(at(za, zr)) & set(at(da, dr)))
                got = D._overlap(z, d)
                assert got == shares or (got and rows > 1 and zr != dr), (rows, width, za, zr, da, dr)
                if shares:
                    rc = lib.nlh_distill_backward(C.c_void_p(base + 4 * za), 0, zr, p, p, p, 0, p, need, None, C.c_void_p(base + 4 * da), dr,
                                                  rows, width, 2, 2.0, 0.5, 0.5)
                    assert rc == BAD, (rows, width, za, zr, da, dr)
                    n += 1
    assert n > 500
