"""The losses' host side on the CPU: refusals of the C entry points before any CUDA call, of the Python calls before
they reach the library, and the 64-bit oracle against autograd. No kernel is launched here."""
import ctypes as C
import math

import pytest
import torch

import loss_ref as R
from cuda_transformer_b200 import _lib, build, losses


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _lib.load()


A = 1 << 20         # stands for an aligned device pointer: never read, the calls below end on the host


def test_workspace_size_is_the_headers(lib, tmp_path):
    import os
    import subprocess
    repo = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    src = tmp_path / "sizes.c"
    src.write_text('#include <stdio.h>\n#include "b200amp.h"\nint main(void) { printf("%d %d %d %d %d %d\\n", '
                   'B200AMP_LOSS_WORKSPACE_BYTES, B200AMP_MAX_LISTED, B200AMP_MAX_EXPERTS, B200AMP_F16, B200AMP_BF16, '
                   'B200AMP_F32); return 0; }\n')
    exe = tmp_path / "sizes"
    subprocess.run(["gcc", "-I", os.path.join(repo, "include"), str(src), "-o", str(exe)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    assert got == [_lib.LOSS_WORKSPACE_BYTES, _lib.MAX_LISTED, _lib.MAX_EXPERTS, _lib.F16, _lib.BF16, _lib.F32]


DISTILL = dict(logits=A, ld=64, dlogits=A + 4096, dld=64, dtype=_lib.F16, rows=4, vocab=60, cols=64, targets=A, values=A,
               value_dtype=_lib.F16, indices=A, lse=A, k=3, temperature=1.0, soft=1.0, hard=1.0, st=A, row_loss=A, ws=A,
               stream=None)


@pytest.mark.parametrize("change,text", [
    (dict(dtype=3), b"dtype"), (dict(dtype=-1), b"dtype"), (dict(rows=-1), b"rows"), (dict(rows=1 << 31), b"rows"),
    (dict(vocab=0), b"vocab"), (dict(vocab=65), b"vocab"), (dict(cols=65), b"ld"), (dict(dld=63), b"dld"),
    (dict(ld=0), b"ld"), (dict(k=-1), b"k = -1"), (dict(k=1025), b"k = 1025"), (dict(temperature=0.0), b"temperature"),
    (dict(temperature=-1.0), b"temperature"), (dict(temperature=math.inf), b"temperature"),
    (dict(temperature=math.nan), b"temperature"), (dict(temperature=1e-45), b"temperature"),
    (dict(soft=math.nan), b"weights"), (dict(hard=math.inf), b"weights"), (dict(logits=None), b"logits is null"),
    (dict(logits=A + 1), b"aligned"), (dict(dlogits=A + 1), b"aligned"), (dict(dlogits=A, dld=65), b"in place"),
    (dict(targets=None), b"needs targets"), (dict(targets=A + 2), b"targets"), (dict(values=None), b"needs values"),
    (dict(indices=None), b"needs values"), (dict(value_dtype=7), b"value dtype"), (dict(indices=A + 2), b"misaligned"),
    (dict(lse=A + 1), b"misaligned"), (dict(values=A + 1), b"misaligned"), (dict(st=None), b"null"),
    (dict(row_loss=None), b"null"), (dict(ws=None), b"null"), (dict(ws=A + 8), b"misaligned"),
    (dict(row_loss=A + 2), b"misaligned"),
])
def test_distill_refusals(lib, change, text):
    args = {**DISTILL, **change}
    assert lib.b200amp_distill_loss(*args.values()) == _lib.ERR_ARG
    assert lib.b200amp_last_error().startswith(b"distill_loss") and text in lib.b200amp_last_error()


TOP = dict(logits=A, dtype=_lib.F16, rows=4, vocab=60, ld=64, k=3, temperature=1.0, values=A, indices=A, lse=A, stream=None)


@pytest.mark.parametrize("change,text", [
    (dict(dtype=9), b"dtype"), (dict(rows=-1), b"rows"), (dict(vocab=0), b"vocab"), (dict(ld=59), b"vocab"),
    (dict(k=0), b"k = 0"), (dict(k=1025), b"k = 1025"), (dict(temperature=0.0), b"temperature"),
    (dict(logits=None), b"null"), (dict(values=None), b"null"), (dict(indices=None), b"null"),
    (dict(values=A + 1), b"aligned"), (dict(indices=A + 2), b"aligned"), (dict(lse=A + 2), b"aligned"),
])
def test_top_logits_refusals(lib, change, text):
    args = {**TOP, **change}
    assert lib.b200amp_top_logits(*args.values()) == _lib.ERR_ARG
    assert lib.b200amp_last_error().startswith(b"top_logits") and text in lib.b200amp_last_error()


BALANCE = dict(logits=A, ld=64, dlogits=A + 4096, dld=64, dtype=_lib.F32, rows=4, experts=60, chosen=A, k=2, targets=A,
               weight=0.01, accumulate=0, add=0, st=A, counts=A, loss=A, ws=A, stream=None)


@pytest.mark.parametrize("change,text", [
    (dict(dtype=9), b"dtype"), (dict(rows=-1), b"rows"), (dict(rows=1 << 30, k=2), b"rows"), (dict(experts=0), b"experts"),
    (dict(experts=1025, ld=2048, dld=2048), b"experts"), (dict(experts=65), b"experts"), (dict(k=0), b"k = 0"),
    (dict(k=1025), b"k = 1025"), (dict(weight=math.nan), b"weight"), (dict(logits=None), b"null"),
    (dict(chosen=None), b"null"), (dict(chosen=A + 2), b"aligned"), (dict(dld=59), b"dld"),
    (dict(dlogits=A, accumulate=1), b"in place"), (dict(dlogits=A, dld=70), b"in place"), (dict(st=None), b"null"),
    (dict(counts=None), b"null"), (dict(loss=None), b"null"), (dict(ws=None), b"null"), (dict(ws=A + 4), b"misaligned"),
])
def test_balance_refusals(lib, change, text):
    args = {**BALANCE, **change}
    assert lib.b200amp_balance_loss(*args.values()) == _lib.ERR_ARG
    assert lib.b200amp_last_error().startswith(b"balance_loss") and text in lib.b200amp_last_error()


def test_workspace_init_refusals(lib):
    assert lib.b200amp_loss_workspace_init(None, None) == _lib.ERR_ARG
    assert lib.b200amp_loss_workspace_init(A + 8, None) == _lib.ERR_ARG


def test_python_calls_refuse_tensors_that_are_not_on_a_gpu():
    z = torch.zeros(4, 8)
    st, ws, row = torch.zeros(60, dtype=torch.uint8), torch.zeros(_lib.LOSS_WORKSPACE_BYTES, dtype=torch.uint8), torch.zeros(4)
    with pytest.raises(ValueError, match="logits"):
        losses.distill_loss(z, None, None, None, None, None, st, row, ws)
    with pytest.raises(ValueError, match="logits"):
        losses.top_logits(z, 2, torch.zeros(4, 2), torch.zeros(4, 2, dtype=torch.int32))
    with pytest.raises(ValueError, match="logits"):
        losses.balance_loss(z, None, torch.zeros(4, 2, dtype=torch.int32), None, st, torch.zeros(8, dtype=torch.int32),
                            torch.zeros(1), ws)


@pytest.mark.parametrize("rest", [False, True])
def test_the_oracle_agrees_with_autograd(rest):
    """The 64-bit oracle's gradient is the derivative of its own loss written with torch's functions."""
    gen = torch.Generator().manual_seed(3)
    T, soft, hard, vocab = 1.7, 2.0, 0.3, 23
    z = torch.randn(vocab, generator=gen, dtype=torch.float64, requires_grad=True)
    t = torch.randn(vocab, generator=gen, dtype=torch.float64)
    best = torch.topk(t, 5)
    lse = float(torch.logsumexp(t / T, 0))
    logp = best.values / T - (lse if rest else torch.logsumexp(best.values / T, 0))
    p, logq = logp.exp(), torch.log_softmax(z / T, 0)
    kl = (p * (logp - logq[best.indices])).sum()
    if rest:
        r = 1 - p.sum()
        others = torch.ones(vocab, dtype=torch.bool)
        others[best.indices] = False
        kl = kl + r * (r.log() - torch.logsumexp(logq[others], 0))
    want = soft * kl - hard * torch.log_softmax(z, 0)[7]
    want.backward()
    loss, grad, _ = R.distill_row(z.detach(), 7, best.values.tolist(), best.indices.tolist(), lse if rest else None, vocab,
                                  T, soft, hard)
    assert abs(loss - float(want)) < 1e-12 and float((grad - z.grad).abs().max()) < 1e-12


def test_the_balance_oracle_agrees_with_autograd():
    gen = torch.Generator().manual_seed(4)
    z = torch.randn(11, 6, generator=gen, dtype=torch.float64, requires_grad=True)
    chosen = torch.topk(z.detach(), 2, dim=1).indices.to(torch.int32)
    targets = torch.arange(11, dtype=torch.int32) - 3
    valid = targets >= 0
    share = torch.nn.functional.one_hot(chosen[valid].long(), 6).sum((0, 1)).double() / (8 * 2)
    want = 0.05 * 6 * (share * torch.softmax(z, 1)[valid].mean(0)).sum()
    (want * 8.0).backward()
    got = R.balance(z.detach(), chosen, targets, 0.05, 8.0)
    assert abs(got["loss"] - float(want)) < 1e-12 and float((got["dlogits"] - z.grad).abs().max()) < 1e-12
