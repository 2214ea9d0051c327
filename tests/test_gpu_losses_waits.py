"""Failure detection of the losses without a fault: the wait for a row's copy is bounded. A test hook announces bytes that
never arrive for one row; the wait has to run out, the kernel to return, b200amp_device_error to report it once, the
row and those that the same blocks take after it to be marked, every other row to be right, and the context and the workspace to stay usable."""
import ctypes as C
import math
import time

import pytest
import torch

import test_gpu_losses as L

pytestmark = pytest.mark.gpu


class starved:
    def __init__(self, row):
        self.row = row

    def __enter__(self):
        from cuda_transformer_b200 import _lib, amp
        amp.device_error()                                      # clear anything older
        _lib.check(_lib.load().b200amp_tune_set(b"loss_test_starve", self.row + 1))
        self.t0 = time.perf_counter()

    def __exit__(self, *exc):
        from cuda_transformer_b200 import _lib, amp
        torch.cuda.synchronize()
        waited = time.perf_counter() - self.t0
        _lib.check(_lib.load().b200amp_tune_set(b"loss_test_starve", 0))
        if exc[0] is None:
            assert waited < 10.0, f"the bounded waits took {waited:.1f} s"
            assert amp.device_error() == 4 and amp.device_error() == 0


def _marked(bad, row, rows):
    """The rows that are marked: the starved one and every n-th behind it, n the number of clusters."""
    at = bad.nonzero()[:, 0].tolist()
    assert at and at[0] == row
    step = at[1] - at[0] if len(at) > 1 else rows
    assert at == list(range(row, rows, step))
    return bad


@pytest.mark.parametrize("rows,vocab,dtype,k,row,ignored", [
    (1500, 4098, "f16", 8, 700, 0.0), (1500, 4098, "f16", 0, 3, 0.0), (400, 50257, "bf16", 16, 310, 0.0), (200, 131072, "f32", 0, 45, 0.0),
    (200, 131072, "f32", 8, 45, 0.0), (900, 4098, "f32", 3, 1, 0.4)])
def test_distill_gives_up_a_copy_that_never_completes(rows, vocab, dtype, k, row, ignored):
    from cuda_transformer_b200 import losses
    p = L._problem(20, vocab, vocab, L.TYPES[dtype], k, 1.0, True, 0.5)
    pick = torch.arange(rows) % 20
    z = p["logits"].cuda()[pick.cuda()]
    targets = p["targets"][pick].clone()
    targets[torch.rand(rows, generator=torch.Generator().manual_seed(1)) < ignored] = -1
    targets[row] = 1
    targets, ws = targets.cuda(), losses.loss_workspace()
    rec = [None if p[n] is None else p[n][pick].contiguous().cuda() for n in ("values", "indices", "lse")]

    def call():
        state, d, out = L._state(1024.0), torch.full_like(z, 7.0), torch.full((rows,), 7.0, device="cuda")
        losses.distill_loss(z, d, targets, *rec, state, out, ws, vocab=vocab, soft_weight=p["soft"], hard_weight=0.5)
        torch.cuda.synchronize()
        return d, out, L._fields(state)

    good = call()
    with starved(row):
        d, out, st = call()
    bad = torch.isnan(out)
    if not ignored:
        _marked(bad, row, rows)
    assert bool(bad[row]) and not bool(bad[:row].any()) and not bool((bad & (targets < 0)).any())
    assert bool(torch.isnan(d[bad].float()).all()) and math.isnan(st.loss)
    assert torch.equal(d[~bad], good[0][~bad]) and torch.equal(out[~bad], good[1][~bad])
    again = call()
    assert torch.equal(again[0], good[0]) and torch.equal(again[1], good[1]) and again[2].loss == good[2].loss


@pytest.mark.parametrize("rows,vocab,dtype,k,row,lse", [
    (1500, 4098, "f16", 8, 700, True), (1500, 4098, "f32", 40, 2, False), (400, 50257, "bf16", 16, 310, True),
    (200, 131072, "f32", 300, 45, True), (200, 131072, "f32", 5000 // 5, 45, False)])
def test_top_logits_gives_up_a_copy_that_never_completes(rows, vocab, dtype, k, row, lse):
    from cuda_transformer_b200 import losses
    gen = torch.Generator(device="cuda").manual_seed(k)
    z = torch.randn(rows, vocab, generator=gen, device="cuda").to(L.TYPES[dtype])

    def call():
        v, i = torch.empty(rows, k, dtype=z.dtype, device="cuda"), torch.empty(rows, k, dtype=torch.int32, device="cuda")
        s = torch.zeros(rows, device="cuda")
        losses.top_logits(z, k, v, i, s if lse else None)
        torch.cuda.synchronize()
        return v, i, s

    good = call()
    with starved(row):
        v, i, s = call()
    bad = _marked(torch.isnan(v.float()).any(1), row, rows)
    assert bool(torch.isnan(v[bad].float()).all()) and bool(torch.isnan(s[bad]).all()) == lse
    assert bool(((i >= 0) & (i < vocab)).all())
    for a, b in zip((v, i, s), good):
        assert torch.equal(a[~bad], b[~bad])
    for a, b in zip(call(), good):
        assert torch.equal(a, b)


def test_the_hook_has_a_range():
    from cuda_transformer_b200 import _lib
    v = C.c_int(-1)
    _lib.check(_lib.load().b200amp_tune_get(b"loss_test_starve", C.byref(v)))
    assert v.value == 0 and _lib.load().b200amp_tune_set(b"loss_test_starve", -1) == _lib.ERR_ARG
