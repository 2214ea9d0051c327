"""Many rows one behind the other through every size of cluster, with rows between them that do not count: what a block
keeps of a row, and what the blocks of a cluster write to each other, must not meet the next row's.

The batches repeat a few different rows in a random order, so that the 64-bit oracle works out few of them and a row
that took anything from a neighbour shows. Tolerances are those of test_gpu_losses.py."""
import pytest
import torch

import loss_ref as R
import test_gpu_losses as L

pytestmark = pytest.mark.gpu


def _batch(p, rows, ignored, seed):
    """(row of p for each row of the batch, targets of the batch): every row counts with probability 1 - ignored, so runs of
    one, two, three and more rows that do not lie between those that do, whatever the number of clusters."""
    gen = torch.Generator().manual_seed(seed)
    pick = torch.randint(0, p["logits"].shape[0], (rows,), generator=gen)
    targets = p["targets"][pick].clone()
    targets[torch.rand(rows, generator=gen) < ignored] = -1
    return pick, targets


def _call(p, pick, targets, gradient, scale):
    from cuda_transformer_b200 import losses
    z = p["logits"].cuda()[pick.cuda()]
    d = torch.full_like(z, 7.0) if gradient else None
    state, row = L._state(scale), torch.full((len(pick),), 7.0, device="cuda")
    rec = [None if p[n] is None else p[n][pick].contiguous().cuda() for n in ("values", "indices", "lse")]
    losses.distill_loss(z, d, targets.cuda(), *rec, state, row, losses.loss_workspace(), vocab=p["vocab"], temperature=p["T"],
                        soft_weight=p["soft"], hard_weight=p["hard"])
    st = L._fields(state)
    return d, row, st.loss, st.n_valid


def _check(p, pick, targets, got, scale):
    d, row, loss, n_valid = got
    vocab, dtype, counts = p["vocab"], p["logits"].dtype, targets >= 0
    n = int(counts.sum())
    assert n_valid == n
    rel = L._rel(vocab, 90.0)
    few = [R.distill_row(p["logits"][i].double(), int(p["targets"][i]), p["values"][i].double().tolist(), p["indices"][i].tolist(),
                         None if p["lse"] is None else float(p["lse"][i]), vocab, p["T"], p["soft"], p["hard"])
           for i in range(p["logits"].shape[0])]
    want = torch.where(counts, torch.tensor([float(f[0]) for f in few], dtype=torch.float64)[pick], torch.zeros(1, dtype=torch.float64))
    limit = rel * (abs(p["soft"]) + abs(p["hard"])) + 2 * L.U * want.abs()
    err = (row.cpu().double() - want).abs()
    assert bool((err <= limit).all()), (err / limit).max()
    assert not bool(row.cpu()[~counts].any())
    assert abs(loss - float(want.sum()) / n) <= float(limit.max()) + 2 * L.U * abs(float(want.sum()) / n)
    if d is None:
        return
    grad = torch.stack([f[1] for f in few]).cuda() * (scale / n)
    size = torch.stack([f[2] for f in few]).cuda() * (scale / n)
    cut = 2.0 ** -120 * scale * (abs(p["soft"]) / p["T"] + abs(p["hard"]))
    limits = rel * size + torch.finfo(dtype).eps / 2 * (grad.abs() + rel * size) + L.TINY[dtype] + cut
    for i, (r, c) in enumerate(zip(pick.tolist(), counts.tolist())):
        if not c:
            assert not bool(d[i].any()), f"row {i} does not count and has a gradient"
            continue
        ok = bool(((d[i, :vocab].double() - grad[r]).abs() <= limits[r]).all()) and not bool(d[i, vocab:].any())
        assert ok, f"row {i}: {float(((d[i, :vocab].double() - grad[r]).abs() / limits[r]).max())} of what is allowed"


CLUSTERS = [
    # rows, different rows, vocab, cols, dtype, k, T, rest, hard (blocks a row)
    (700, 16, 128256, 128256, "f16", 64, 1.0, True, 0.5),       # 2
    (600, 16, 128001, 128001, "bf16", 300, 2.0, False, 0.0),    # 2, rows at every alignment
    (300, 12, 131072, 131072, "f32", 64, 1.0, True, 0.5),       # 4
    (150, 8, 262144, 262144, "f32", 16, 2.0, True, 0.3),        # 8
    (60, 5, 1000003, 1000003, "f16", 40, 1.0, False, 0.5),      # 16
]


@pytest.mark.parametrize("ignored", [0.0, 0.3, 0.6])
@pytest.mark.parametrize("case", CLUSTERS, ids=lambda c: f"{c[2]}-{c[4]}")
def test_distill_several_rows_a_cluster_some_of_which_do_not_count(case, ignored):
    rows, different, vocab, cols, dtype, k, T, rest, hard = case
    p = L._problem(different, vocab, cols, L.TYPES[dtype], k, T, rest, hard)
    pick, targets = _batch(p, rows, ignored, seed=rows + int(10 * ignored))
    first = _call(p, pick, targets, True, 1024.0)
    _check(p, pick, targets, first, 1024.0)
    for gradient in (True, False):
        again = _call(p, pick, targets, gradient, 1024.0)
        assert torch.equal(first[1], again[1]) and first[2:] == again[2:] and (not gradient or torch.equal(first[0], again[0]))


@pytest.mark.parametrize("ignored", [0.3, 0.6])
@pytest.mark.parametrize("dtype,vocab,k", [("f32", 1100, 1024), ("f16", 1030, 1024), ("bf16", 300, 290), ("f16", 9000, 1024), ("f32", 12000, 700),
                                           ("f16", 40, 3)])
def test_distill_long_records_of_short_rows_some_of_which_do_not_count(dtype, vocab, k, ignored):
    """One block a row, with most of a row's work in its record: the rows behind a counted one read theirs meanwhile."""
    p = L._problem(24, vocab, vocab + 5, L.TYPES[dtype], k, 1.0, True, 0.5)
    pick, targets = _batch(p, 12000, ignored, seed=vocab + k)
    first = _call(p, pick, targets, True, 1024.0)
    _check(p, pick, targets, first, 1024.0)
    for gradient in (True, False):
        again = _call(p, pick, targets, gradient, 1024.0)
        assert torch.equal(first[1], again[1]) and first[2:] == again[2:] and (not gradient or torch.equal(first[0], again[0]))


@pytest.mark.parametrize("rows,vocab,dtype,k", [(700, 128256, "f16", 64), (300, 131072, "f32", 1024), (150, 262144, "f32", 16),
                                                (60, 1000003, "f16", 300), (60, 1000003, "bf16", 3)])
def test_top_logits_several_rows_a_cluster(rows, vocab, dtype, k):
    from cuda_transformer_b200 import losses
    gen = torch.Generator(device="cuda").manual_seed(rows + k)
    z = (torch.randn(rows, vocab, generator=gen, device="cuda") * 2).to(L.TYPES[dtype])
    z[::5, ::7] = 1.0                                           # many ties
    values, indices = torch.empty(rows, k, dtype=z.dtype, device="cuda"), torch.empty(rows, k, dtype=torch.int32, device="cuda")
    lse = torch.empty(rows, device="cuda")
    losses.top_logits(z, k, values, indices, lse)
    for i in range(rows):
        want = torch.sort(z[i].float(), descending=True, stable=True)
        assert torch.equal(indices[i].long(), want.indices[:k]) and torch.equal(values[i].float(), want.values[:k])
        exact = float(torch.logsumexp(z[i].double(), dim=0))
        assert abs(float(lse[i]) - exact) <= L._rel(vocab, 30.0) + 2 * L.U * abs(exact)
