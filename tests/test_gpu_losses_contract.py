"""What include/b200amp.h says of the losses where a row has no answer, and where a call has more than one user."""
import math

import pytest
import torch

import test_gpu_losses as L

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", list(L.TYPES))
@pytest.mark.parametrize("hard,T", [(0.0, 1.0), (0.5, 1.0), (0.5, 2.0)])
@pytest.mark.parametrize("vocab,cols,ld,dld", [(9, 13, 13, 13), (13, 16, 16, 16), (4098, 4160, 4160, 4160), (4097, 4103, 4103, 4104),
                                               (50257, 50304, 50304, 50304), (131072, 131100, 131100, 131100)])
def test_a_bad_row_is_nan_in_all_its_columns_and_0_in_its_padding(vocab, cols, ld, dld, hard, T, dtype):
    rows = 12
    p = L._problem(rows, vocab, cols, L.TYPES[dtype], 3, T, True, hard)
    p["logits"][0, vocab - 1] = math.nan
    p["logits"][1, int(p["indices"][1, 0])] = math.nan
    p["logits"][2, 1] = math.inf
    p["logits"][3, :] = -math.inf
    p["indices"][4, 2] = vocab
    p["indices"][5, 0] = 2 ** 31 - 1
    p["values"][6, 1] = math.nan
    p["targets"][7] = vocab if hard else int(p["targets"][7])   # without a hard weight the label is not looked at
    p["logits"][8, vocab:] = math.nan                           # the padding is not read
    p["logits"][9, vocab:] = math.inf
    bad = torch.tensor([True] * 7 + [bool(hard)] + [False] * 4)
    got = L._run(p, ld=ld, dld=dld)
    assert torch.equal(torch.isnan(got["row_loss"]), bad)
    nan = torch.isnan(got["dlogits"].float())
    assert bool(nan[bad, :vocab].all()) and not bool(nan[~bad].any()) and not bool(got["dlogits"][:, vocab:].any())
    assert math.isnan(got["loss"])
    good = {**p, **{n: p[n][~bad] for n in ("logits", "targets", "values", "indices", "lse")}}
    want = L._want(good)["row_loss"]
    assert bool(((got["row_loss"][~bad].double() - want).abs() <= L._rel(vocab, 90.0) * (T * T + hard) + 2 * L.U * want.abs()).all())


def test_a_loss_scale_beyond_fp32_leaves_the_padding_0():
    p = L._problem(3, 500, 520, torch.float32, 4, 1.0, True, 2.0)
    p["soft"] = 100.0
    got = L._run(p, scale=2.0 ** 127)
    assert not bool(got["dlogits"][:, 500:].any()) and not bool(torch.isfinite(got["dlogits"][:, :500]).all())


@pytest.mark.parametrize("vocab", [2, 7, 100, 999])
@pytest.mark.parametrize("T,hard", [(1.0, 0.0), (1.0, 0.5), (2.0, 0.5), (0.7, 0.0)])
@pytest.mark.parametrize("rest", [False, True])
def test_fp32_gradients_of_listed_columns_are_rounded_once(rest, T, hard, vocab):
    """Student and teacher agree but for a hundredth, so each gradient is a small difference of two terms. All columns are
    listed, or all but the label's: no fp32 sum enters. Each term is off by at most 2^-40 of itself (sums of up to 999 terms
    in 64 bits: 2^-43; powers of up to 20: 2^-47), the gradient then by half a step of fp32."""
    p = L._problem(9, vocab, vocab, torch.float32, vocab, T, rest, hard, seed=vocab)
    gen = torch.Generator().manual_seed(vocab)
    teacher = torch.zeros(9, vocab).scatter_(1, p["indices"].long(), p["values"])
    p["logits"] = teacher + 0.01 * torch.randn(9, vocab, generator=gen)
    if hard and rest:
        for i in range(9):                                      # the label's column is not listed
            p["indices"][i][p["indices"][i] == p["targets"][i]] = -1
    got, want = L._run(p), L._want(p)
    limit = want["dlogits"].abs() * L.U + want["size"] * 2.0 ** -40 + L.TINY[torch.float32]
    err = (got["dlogits"].double() - want["dlogits"]).abs()
    assert bool((err <= limit).all()), float((err / limit).max())


def test_an_optimizers_calls_on_two_streams_with_a_workspace_each():
    """Two layers' routers at once, each on its stream, on one optimizer's state (read only: nothing is added to its loss)."""
    from cuda_transformer_b200 import losses
    opt, _, _ = L._step_case()
    layers = []
    for seed in (1, 2):
        z, chosen, targets = L._balance_problem(20011, 60, torch.float32, 4, 0.2, 0.1, seed=seed)
        layers.append(dict(z=z.cuda(), c=chosen.cuda(), y=targets.cuda(), d=torch.empty(20011, 60, device="cuda"),
                           counts=torch.empty(60, dtype=torch.int32, device="cuda"), loss=torch.empty(1, device="cuda"),
                           ws=losses.loss_workspace(), s=torch.cuda.Stream()))
    alone = []
    for q in layers:
        opt.balance_loss(q["z"], q["d"], q["c"], q["y"], q["counts"], q["loss"], add_to_state=False)
        alone.append([q[n].clone() for n in ("d", "counts", "loss")])
    torch.cuda.synchronize()
    for _ in range(20):
        for q in layers:
            opt.balance_loss(q["z"], q["d"], q["c"], q["y"], q["counts"], q["loss"], add_to_state=False, stream=q["s"], workspace=q["ws"])
    torch.cuda.synchronize()
    for q, want in zip(layers, alone):
        assert all(torch.equal(q[n], w) for n, w in zip(("d", "counts", "loss"), want)) and not bool(q["ws"][:L.COUNTERS].any())


@pytest.mark.parametrize("dtype,vocab,k", [("f16", 1_200_000, 1024), ("f32", 600_000, 1024), ("bf16", 1_660_000, 3), ("f32", 850_000, 3)])
def test_the_longest_rows(dtype, vocab, k):
    p = L._problem(2, vocab, vocab, L.TYPES[dtype], k, 1.0, True, 0.5)
    L._check(p, L._run(p))
    z = p["logits"]
    values, indices, lse = L._top(z, k)
    want = torch.sort(z.float(), dim=1, descending=True, stable=True)
    assert torch.equal(indices.long(), want.indices[:, :k]) and torch.equal(values.float(), want.values[:, :k])
    exact = torch.logsumexp(z.double(), dim=1)
    assert bool(((lse.double() - exact).abs() <= L._rel(vocab, 30.0) + 2 * L.U * exact.abs()).all())
