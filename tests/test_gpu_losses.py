"""top_logits, distill_loss and balance_loss on the GPU against the 64-bit oracle of loss_ref.py, at the sizes, masks,
strides and records where they can go wrong.

Tolerances. With u = 2^-24 (half a step of fp32) and x the distance of a logit below the maximum its sum is taken
from, over the temperature, capped at 90 (2^x is 0 beyond): the distance is one rounding, its product with
log2(e) / T two more, which moves e^x by 3 u x; the exponential itself is 2 ulp, 4 u; a sum adds at most V / 128 + 64
roundings in a row; the factors and the last product 8 more. So a gradient is off by at most
    (6 x + V / 128 + 128) u * (sum of the magnitudes of its terms)
and then half a step of its type (eps / 2 relative; half the smallest subnormal absolute), and what the ends of the
range of 2^x cut off, 2^-120 of the scale. The loss of a row moves by the same relative amount of what its sums
carry, which is at most soft + hard, and is rounded to fp32 once."""
import ctypes as C
import math

import pytest
import torch

import loss_ref as R

pytestmark = pytest.mark.gpu

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -126}
U = 2.0 ** -24
PATTERN = 0x5A
COUNTERS = 64 + 4 * 1024    # bytes of the workspace that a call has to leave at zero (tickets and counts; what follows is scratch)


def _state(scale):
    from cuda_transformer_b200 import amp
    return torch.frombuffer(bytearray(bytes(amp.initial_state(scale))), dtype=torch.uint8).cuda()


def _fields(state):
    from cuda_transformer_b200._lib import StepState
    return StepState.from_buffer_copy(state.cpu().numpy().tobytes())


def _rel(vocab, x):
    return (6.0 * x + vocab / 128 + 128) * U


class Guarded:
    """rows x cols of a type inside a larger buffer: `ld` elements a row, `shift` elements into a 64-byte line, with
    pattern bytes before, between and behind the rows."""

    def __init__(self, rows, cols, dtype, ld=None, shift=0):
        self.ld = cols if ld is None else ld
        self.size = torch.empty((), dtype=dtype).element_size()
        self.start = 128 + shift * self.size
        self.raw = torch.full((self.start + rows * self.ld * self.size + 256,), PATTERN, dtype=torch.uint8, device="cuda")
        flat = self.raw.view(dtype) if self.raw.numel() % self.size == 0 else self.raw[:self.raw.numel() // self.size * self.size].view(dtype)
        self.t = flat.as_strided((rows, cols), (self.ld, 1), 128 // self.size + shift)
        self.rows, self.cols = rows, cols

    def intact(self):
        raw = self.raw.clone()
        body = raw[self.start:self.start + self.rows * self.ld * self.size].view(self.rows, self.ld * self.size)
        body[:, :self.cols * self.size] = PATTERN
        return bool((raw == PATTERN).all())


def _record(t, k, gen, empty=0.0):
    """The k best of each row as a record, padded with empty slots behind the last column, some slots empty."""
    rows, vocab = t.shape
    best = torch.topk(t.float(), min(k, vocab), dim=1)
    values = torch.full((rows, k), -math.inf, dtype=t.dtype)
    indices = torch.full((rows, k), -1, dtype=torch.int32)
    values[:, :min(k, vocab)], indices[:, :min(k, vocab)] = best.values.to(t.dtype), best.indices.to(torch.int32)
    if empty:
        indices[torch.rand(rows, k, generator=gen) < empty] = -1
    return values, indices


def _problem(rows, vocab, cols, dtype, k, T, rest, hard, seed=0, ignored=0.0, empty=0.0, spread=3.0):
    gen = torch.Generator().manual_seed(1000 * seed + rows + vocab)
    z = torch.randn(rows, cols, generator=gen) * spread
    t = (0.8 * z[:, :vocab] + torch.randn(rows, vocab, generator=gen)).to(dtype)
    values, indices = _record(t, k, gen, empty) if k else (None, None)
    lse = torch.logsumexp(t.double() / T, dim=1).float() if k and rest else None
    targets = torch.randint(0, vocab, (rows,), generator=gen, dtype=torch.int32)
    targets[torch.rand(rows, generator=gen) < ignored] = -1
    return dict(logits=z.to(dtype), targets=targets, values=values, indices=indices, lse=lse, vocab=vocab, T=T,
                soft=T * T if k else 0.0, hard=hard)


def _gpu(t):
    return None if t is None else t.cuda()


def _run(p, scale=1024.0, ld=None, shift=0, dld=None, dshift=0, in_place=False, gradient=True, workspace=None, stream=None):
    """One call between guards; returns dict(dlogits, row_loss, loss, n_valid) on the CPU."""
    from cuda_transformer_b200 import losses
    rows, cols = p["logits"].shape
    dtype = p["logits"].dtype
    z = Guarded(rows, cols, dtype, ld, shift)
    z.t.copy_(p["logits"])
    d = z if in_place else Guarded(rows, cols, dtype, dld, dshift)
    row_loss = Guarded(1, max(1, rows), torch.float32)
    state, ws = _state(scale), losses.loss_workspace() if workspace is None else workspace
    losses.distill_loss(z.t, d.t if gradient else None, _gpu(p["targets"]), _gpu(p["values"]), _gpu(p["indices"]),
                        _gpu(p["lse"]), state, row_loss.t[0, :rows], ws, vocab=p["vocab"], temperature=p["T"],
                        soft_weight=p["soft"], hard_weight=p["hard"], stream=stream)
    torch.cuda.synchronize()
    assert z.intact() and d.intact() and row_loss.intact(), "wrote outside its arrays"
    if not in_place:
        got, want = z.t.cpu(), p["logits"]
        assert torch.equal(got.view(torch.uint8 if False else got.dtype).nan_to_num(7.0), want.nan_to_num(7.0)), "the logits changed"
    assert not bool(ws[:COUNTERS].any()), "the workspace's counters are not as they were found"
    st = _fields(state)
    assert st.loss_scale == scale and st.inv_scale == 1.0 / scale and st.found_inf == 0 and st.step == 0
    return dict(dlogits=d.t.cpu() if gradient else None, row_loss=row_loss.t[0, :rows].cpu(), loss=st.loss, n_valid=st.n_valid)


def _want(p, scale=1024.0):
    return R.distill(p["logits"], p["targets"], p["values"], p["indices"], p["lse"], p["vocab"], p["T"], p["soft"], p["hard"], scale)


def _check(p, got, scale=1024.0, spread=90.0):
    want = _want(p, scale)
    rows, cols = p["logits"].shape
    vocab, dtype = p["vocab"], p["logits"].dtype
    assert got["n_valid"] == want["n_valid"]
    rel = _rel(vocab, min(90.0, spread))
    r, w = got["row_loss"].double(), want["row_loss"]
    assert torch.equal(torch.isnan(r), torch.isnan(w)), (r, w)
    same = torch.isnan(w) | (r == w)
    err = torch.where(same, torch.zeros_like(w), (r - w).abs())
    limit = rel * (abs(p["soft"]) + abs(p["hard"])) + 2 * U * torch.where(torch.isfinite(w), w.abs(), torch.zeros_like(w))
    assert bool((err <= limit).all()), (float((err - limit).max()), r, w)
    if not bool(torch.isnan(w).any()) and math.isfinite(want["loss"]):
        assert abs(got["loss"] - want["loss"]) <= float(limit.max()) + 2 * U * abs(want["loss"])
    if got["dlogits"] is None:
        return
    g, d = got["dlogits"].double(), want["dlogits"]
    assert torch.equal(torch.isnan(g[:, :vocab]), torch.isnan(d[:, :vocab]))
    alive = ~torch.isnan(d[:, 0])
    assert not bool(g[alive][:, vocab:].any()), "the padding's gradient is not 0"
    g, d, size = g[alive], d[alive], want["size"][alive]
    cut = 2.0 ** -120 * scale * (abs(p["soft"]) / p["T"] + abs(p["hard"]))
    limit = rel * size + torch.finfo(dtype).eps / 2 * (d.abs() + rel * size) + TINY[dtype] + cut
    err = (g - d).abs()
    assert bool((err <= limit).all()), f"off by {float((err / limit).max())} of what is allowed"


SIZES = [
    # rows, vocab, cols, k, T, rest, hard
    (1, 1, 1, 1, 1.0, False, 1.0), (2, 1, 8, 3, 1.0, True, 0.5), (3, 2, 2, 1, 2.0, True, 0.0), (5, 7, 8, 7, 0.7, True, 0.3),
    (4, 8, 8, 2, 1.0, True, 0.0), (7, 31, 40, 31, 1.0, False, 0.0), (6, 33, 33, 5, 3.3, True, 1.0),
    (9, 255, 256, 16, 1.0, True, 0.5), (3, 1000, 1001, 1024, 2.0, True, 0.2), (17, 4098, 4160, 32, 2.0, False, 0.5),
    (5, 4098, 4160, 8, 1.0, True, 0.0), (4, 12289, 12289, 64, 1.0, True, 0.7), (3, 50257, 50304, 64, 1.0, True, 0.5),
    (2, 50257, 50257, 300, 1.5, True, 0.25), (2, 131073, 131080, 128, 1.0, False, 0.0), (2, 262144, 262144, 16, 2.0, True, 0.5),
]


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("size", SIZES, ids=lambda s: "x".join(str(v) for v in s))
def test_distill_matches_the_formula(size, dtype):
    rows, vocab, cols, k, T, rest, hard = size
    p = _problem(rows, vocab, cols, TYPES[dtype], k, T, rest, hard, ignored=0.2 if rows > 3 else 0.0)
    _check(p, _run(p), spread=30.0 / T if not hard else 90.0)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("vocab", [1, 5, 4098, 50257])
def test_distill_without_a_teacher_is_the_cross_entropy(vocab, dtype):
    p = _problem(6, vocab, vocab + 3, TYPES[dtype], 0, 1.0, False, 1.3, ignored=0.3)
    _check(p, _run(p))
    teacher = _problem(6, vocab, vocab + 3, TYPES[dtype], min(4, vocab), 2.0, True, 1.3)
    off = dict(p, values=teacher["values"], indices=teacher["indices"], lse=teacher["lse"], soft=0.0)
    a, b = _run(p), _run(off)
    assert torch.equal(a["dlogits"], b["dlogits"]) and torch.equal(a["row_loss"], b["row_loss"])


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("ld,shift,dld,dshift", [(4104, 0, 4104, 0), (4099, 0, 4099, 0), (4099, 3, 4099, 3), (4099, 1, 4104, 0),
                                                 (4104, 0, 4101, 5), (4103, 7, 4098, 2), (8192, 1, 4098, 1)])
def test_distill_strides_and_alignment(ld, shift, dld, dshift, dtype):
    p = _problem(9, 4097, 4098, TYPES[dtype], 20, 1.0, True, 0.5)
    got = _run(p, ld=ld, shift=shift, dld=dld, dshift=dshift)
    _check(p, got)
    plain = _run(p)
    assert torch.equal(got["n_valid"] if torch.is_tensor(got["n_valid"]) else torch.tensor(got["n_valid"]), torch.tensor(plain["n_valid"]))


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("vocab,cols,ld,shift", [(4098, 4160, 4160, 0), (4098, 4100, 4101, 1), (50257, 50257, 50257, 0), (9, 9, 9, 1)])
def test_distill_in_place_and_without_a_gradient(vocab, cols, ld, shift, dtype):
    p = _problem(7, vocab, cols, TYPES[dtype], min(11, vocab), 2.0, True, 0.5, ignored=0.2)
    apart = _run(p, ld=ld, shift=shift, dld=ld, dshift=shift)
    inside = _run(p, ld=ld, shift=shift, in_place=True)
    assert torch.equal(apart["dlogits"], inside["dlogits"]) and torch.equal(apart["row_loss"], inside["row_loss"])
    alone = _run(p, ld=ld, shift=shift, gradient=False)
    assert torch.equal(alone["row_loss"], inside["row_loss"]) and alone["loss"] == inside["loss"]


@pytest.mark.parametrize("vocab", [19, 4098, 50257])
@pytest.mark.parametrize("rest", [False, True])
def test_distill_records_with_gaps_and_columns_listed_twice(vocab, rest):
    p = _problem(8, vocab, vocab, torch.float16, 12, 1.0, rest, 0.5, empty=0.3)
    p["indices"][1] = -1                                        # nothing listed
    p["indices"][2, 1:] = -1                                    # one listed
    p["indices"][3, :] = 4                                      # one column, listed twelve times
    p["indices"][4, 6:] = p["indices"][4, :6]                   # six columns, twice each
    p["indices"][5, 0], p["targets"][5] = 3, 3                  # the label is listed
    p["indices"][6] = torch.arange(12, dtype=torch.int32)
    p["indices"][6, 5], p["indices"][6, 9], p["targets"][6] = 7, 7, 7     # and listed three times
    p["values"][7, :6] = -math.inf                              # listed without mass
    _check(p, _run(p))
    p["values"][:] = -math.inf                                  # a teacher without any mass
    if not rest:
        _check(p, _run(p))


@pytest.mark.parametrize("vdtype", list(TYPES))
@pytest.mark.parametrize("dtype", list(TYPES))
def test_distill_record_of_another_type(dtype, vdtype):
    p = _problem(4, 999, 1000, TYPES[dtype], 9, 1.0, False, 0.0)
    p["values"] = p["values"].to(TYPES[vdtype])
    _check(p, _run(p))


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("vocab", [11, 4098, 50257])
@pytest.mark.parametrize("low", ["inf", "lowest"])
def test_distill_masked_logits(low, vocab, dtype):
    """Columns masked with -inf or the type's lowest value: single ones, listed ones, the label, all but the listed."""
    t = TYPES[dtype]
    mask = -math.inf if low == "inf" else torch.finfo(t).min
    p = _problem(7, vocab, vocab, t, 4, 1.0, True, 0.5)
    z, idx, y = p["logits"], p["indices"], p["targets"]
    z[0, ::2] = mask
    z[1, idx[1, 0]] = mask                                      # has teacher mass: an infinite loss, or a huge one
    z[2, y[2]] = mask
    keep = torch.zeros(vocab, dtype=torch.bool)
    keep[idx[3].long()] = True
    z[3, ~keep] = mask                                          # the student gives the rest nothing
    z[4, :] = mask                                              # no logit left: NaN, or all equal
    z[5, keep.nonzero()[0]] = mask
    z[6, :] = mask
    z[6, y[6]] = 1.0                                            # the label alone
    got, want = _run(p), _want(p)
    if low == "lowest":
        # a distance of the type's whole range: the loss is that far too, and fp32 holds it to half a step
        # (beyond fp32's largest number, as the lowest bf16 or fp32 logit times two weights is, the nearest is inf)
        w = want["row_loss"]
        lim = _rel(vocab, 90.0) * 1.5 + 4 * U * w.abs()
        over = torch.isinf(w.float()) & (got["row_loss"] == w.float())
        assert bool((over | ((got["row_loss"].double() - w).abs() <= lim)).all()), (got["row_loss"], w)
        p2 = dict(p)
        g, d, size = got["dlogits"].double(), want["dlogits"], want["size"]
        assert not bool(torch.isnan(g).any())
        lim = _rel(vocab, 90.0) * size * 2 + torch.finfo(t).eps / 2 * d.abs() + TINY[t] + 2.0 ** -110 * 1024
        assert bool(((g - d).abs() <= lim).all())
    else:
        assert math.isnan(float(got["row_loss"][4])) and math.isinf(float(got["row_loss"][1]))
        _check(p, got)


@pytest.mark.parametrize("vocab", [13, 4098, 50257])
def test_distill_bad_values_make_their_own_row_nan(vocab):
    """NaN and +inf logits, an index or a label beyond the vocabulary, NaN in the record: that row is NaN, the others are not."""
    p = _problem(10, vocab, vocab + 1, torch.float16, 3, 1.0, True, 0.5)
    p["logits"][0, vocab - 1] = math.nan
    p["logits"][1, int(p["indices"][1, 0])] = math.nan
    p["logits"][2, 1] = math.inf
    p["indices"][3, 2] = vocab
    p["targets"][4] = vocab
    p["values"][5, 1] = math.nan
    p["indices"][6, 0] = 2 ** 31 - 1
    p["logits"][7, vocab] = math.nan                            # padding is not read
    got = _run(p)
    assert torch.isnan(got["row_loss"]).tolist() == [True] * 7 + [False] * 3
    nan_rows = torch.isnan(got["dlogits"][:, :vocab].float()).any(1).tolist()
    assert nan_rows == [True] * 7 + [False] * 3
    assert torch.isnan(got["dlogits"][:7, :vocab].float()).all(1).tolist() == [True] * 7 or vocab > 0
    assert math.isnan(got["loss"])
    good = {**p, "logits": p["logits"][7:], "targets": p["targets"][7:], "values": p["values"][7:], "indices": p["indices"][7:],
            "lse": p["lse"][7:]}
    want = _want(good)
    assert float((got["row_loss"][7:].double() - want["row_loss"]).abs().max()) <= _rel(vocab, 90.0) * 2


def test_distill_no_row_counts_and_no_rows():
    p = _problem(5, 300, 320, torch.float16, 4, 1.0, True, 1.0)
    p["targets"][:] = -1
    got = _run(p)
    assert got["n_valid"] == 0 and got["loss"] == 0.0 and not bool(got["dlogits"].any()) and not bool(got["row_loss"].any())
    from cuda_transformer_b200 import losses
    state, ws = _state(4.0), losses.loss_workspace()
    state.view(torch.float32)[13] = 5.0
    losses.distill_loss(torch.empty(0, 8, device="cuda"), torch.empty(0, 8, device="cuda"),
                        torch.empty(0, dtype=torch.int32, device="cuda"), torch.empty(0, 2, device="cuda"),
                        torch.empty(0, 2, dtype=torch.int32, device="cuda"), None, state, torch.empty(0, device="cuda"), ws)
    st = _fields(state)
    assert st.loss == 0.0 and st.n_valid == 0


def test_distill_targets_may_be_left_out():
    p = _problem(5, 300, 300, torch.bfloat16, 4, 1.0, True, 0.0)
    with_targets = _run(p)
    p["targets"] = None
    got = _run(p)
    _check(p, got)
    assert got["n_valid"] == 5 and torch.equal(got["dlogits"], with_targets["dlogits"])
    p = _problem(5, 300, 300, torch.bfloat16, 4, 1.0, True, 0.0)
    p["targets"][:] = 2 ** 31 - 1               # without a hard weight the label is only a sign
    assert torch.equal(_run(p)["dlogits"], got["dlogits"])


@pytest.mark.parametrize("gap", [50.0, 88.0, 100.0, 700.0, 3000.0])
def test_distill_a_student_far_surer_than_its_teacher(gap):
    """The listed columns stand so far above the others that their probability is 0 in fp32: the rest's loss and gradient
    are relative to the others alone and stay exact."""
    p = _problem(6, 2000, 2000, torch.float32, 4, 1.0, True, 0.5, spread=1.0)
    p["logits"].scatter_add_(1, p["indices"].long(), torch.full((6, 4), gap))
    p["targets"][:3] = p["indices"][:3, 0]
    got, want = _run(p), _want(p)
    lim = _rel(2000, 20.0) * 1.5 + 4 * U * want["row_loss"].abs()
    assert bool(((got["row_loss"].double() - want["row_loss"]).abs() <= lim).all())
    d = want["dlogits"]
    lim = _rel(2000, 20.0) * want["size"] + U * d.abs() + 2.0 ** -110 * 1024
    assert bool(((got["dlogits"].double() - d).abs() <= lim).all())


@pytest.mark.parametrize("T", [0.01, 0.5, 1.0, 8.0, 1000.0])
def test_distill_temperatures(T):
    p = _problem(5, 1500, 1500, torch.float32, 10, T, True, 0.4)
    p["soft"] = 1.0
    _check(p, _run(p))


def test_distill_gradient_is_the_difference_of_losses():
    """Central differences of the kernel's own losses. The third derivative of each term is at most 1 / T^3, so a
    step h misses by h^2 / 6; the losses are off by 1e-6, which the quotient divides by h."""
    from cuda_transformer_b200 import losses
    p = _problem(1, 50, 50, torch.float32, 6, 1.0, True, 0.5)
    grad = _run(p, scale=1.0)["dlogits"][0]
    h = 0.02
    big = p["logits"].repeat(100, 1)
    for v in range(50):
        big[2 * v, v] += h
        big[2 * v + 1, v] -= h
    up = big.double()
    many = {**p, "logits": big, **{n: p[n].repeat(100, *([1] * (p[n].dim() - 1))) for n in ("targets", "values", "indices", "lse")}}
    loss = _run(many, scale=1.0, gradient=False)["row_loss"].double()
    step = torch.stack([up[2 * v, v] - up[2 * v + 1, v] for v in range(50)])
    diff = (loss[0::2] - loss[1::2]) / step
    assert float((diff - grad.double()).abs().max()) <= h * h / 6 * 1.5 + 2 * 1e-6 / (2 * h)


def test_distill_offsets_past_32_bits():
    """Rows so far apart that the last one starts 2^31 elements and more behind the first."""
    from cuda_transformer_b200 import losses
    ld, vocab = (1 << 30) + 24, 4098
    buf = torch.empty(2 * ld + 4160, dtype=torch.float16, device="cuda")
    z = buf.as_strided((3, 4160), (ld, 1))
    p = _problem(3, vocab, 4160, torch.float16, 8, 1.0, True, 0.5)
    z.copy_(p["logits"])
    state, ws, row = _state(1024.0), losses.loss_workspace(), torch.empty(3, device="cuda")
    losses.distill_loss(z, z, _gpu(p["targets"]), _gpu(p["values"]), _gpu(p["indices"]), _gpu(p["lse"]), state, row, ws,
                        vocab=vocab, hard_weight=0.5)
    st = _fields(state)
    _check(p, dict(dlogits=z.cpu(), row_loss=row.cpu(), loss=st.loss, n_valid=st.n_valid))
    z.copy_(p["logits"])
    values, indices = torch.empty(3, 5, dtype=torch.float16, device="cuda"), torch.empty(3, 5, dtype=torch.int32, device="cuda")
    losses.top_logits(z, 5, values, indices, vocab=vocab)
    want = R.top(p["logits"], 5, vocab, 1.0)
    assert torch.equal(indices.cpu(), want[1]) and torch.equal(values.cpu().double(), want[0])


def test_distill_many_rows_same_bits_every_time_and_any_loss_scale():
    """More rows than blocks; the sums do not depend on which block is last; a power of two in the scale moves exponents only."""
    p = _problem(3001, 517, 520, torch.float32, 6, 2.0, True, 0.5, ignored=0.3)
    a = _run(p)
    for _ in range(3):
        b = _run(p)
        assert torch.equal(a["dlogits"], b["dlogits"]) and a["loss"] == b["loss"] and torch.equal(a["row_loss"], b["row_loss"])
    _check(p, a)
    c = _run(p, scale=4096.0)
    assert torch.equal(a["dlogits"] * 4, c["dlogits"]) and a["loss"] == c["loss"]


@pytest.mark.parametrize("rows,vocab,dtype,k,T,rest,hard", [
    (331, 4098, "f16", 16, 1.0, True, 0.5), (331, 12000, "f32", 8, 2.0, False, 0.3), (305, 12001, "f32", 8, 1.0, True, 0.0),
    (301, 30011, "bf16", 70, 1.0, True, 0.5), (299, 50257, "f16", 33, 1.0, False, 0.0), (640, 9, "f16", 3, 1.0, True, 0.5),
    (700, 130, "bf16", 130, 0.8, True, 0.2)])
def test_distill_more_rows_than_blocks(rows, vocab, dtype, k, T, rest, hard):
    """Every size of block, each with several rows one behind the other, some of which do not count."""
    p = _problem(rows, vocab, vocab + 2, TYPES[dtype], k, T, rest, hard, ignored=0.3)
    p["targets"][:40] = -1                                      # whole blocks begin with rows that do not count
    p["indices"][rows - 1, 1:] = p["indices"][rows - 1, 0]
    _check(p, _run(p))


@pytest.mark.parametrize("rows,vocab,dtype,k", [(331, 4098, "f16", 16), (303, 20011, "bf16", 100), (299, 50257, "f16", 64),
                                                (160, 100003, "f16", 300), (900, 33, "f32", 33), (40, 131072, "f32", 1024)])
def test_top_logits_more_rows_than_blocks(rows, vocab, dtype, k):
    z = (torch.randn(rows, vocab, generator=torch.Generator().manual_seed(rows + k)) * 2).to(TYPES[dtype])
    z[::5, ::7] = 1.0                                           # many ties
    z[3] = -math.inf
    values, indices, lse = _top(z, k, vocab)
    want = torch.sort(z.float(), dim=1, descending=True, stable=True)
    assert torch.equal(indices.long(), want.indices[:, :k]) and torch.equal(values.float(), want.values[:, :k])
    exact = torch.logsumexp(z.double(), dim=1)
    same = lse.double() == exact
    assert bool((same | ((lse.double() - exact).abs() <= _rel(vocab, 30.0) + 2 * U * exact.abs())).all())


def test_distill_overflow_becomes_inf():
    """A loss scale that takes the gradient out of fp16's range: inf in the gradient, so that the step is skipped."""
    p = _problem(1, 64, 64, torch.float16, 2, 1.0, False, 1.0)
    got = _run(p, scale=float(1 << 24))
    assert torch.isinf(got["dlogits"]).any() and math.isfinite(got["loss"])


# ---------------------------------------------------------------- top_logits

def _top(logits, k, vocab=None, T=1.0, ld=None, shift=0, lse=True):
    from cuda_transformer_b200 import losses
    rows, cols = logits.shape
    z = Guarded(rows, cols, logits.dtype, ld, shift)
    z.t.copy_(logits)
    values, indices, out = Guarded(rows, k, logits.dtype), Guarded(rows, k, torch.int32), Guarded(1, rows, torch.float32)
    losses.top_logits(z.t, k, values.t, indices.t, out.t[0] if lse else None, vocab=vocab, temperature=T)
    torch.cuda.synchronize()
    assert z.intact() and values.intact() and indices.intact() and out.intact()
    return values.t.cpu(), indices.t.cpu(), out.t[0].cpu()


def _check_top(logits, k, vocab, T, got, x=90.0):
    want = R.top(logits, k, vocab, T)
    assert torch.equal(got[1], want[1]), (got[1], want[1])
    v, w = got[0].double(), want[0]
    assert torch.equal(torch.isnan(v), torch.isnan(w)) and torch.equal(v.nan_to_num(7.0), w.nan_to_num(7.0))
    lse, w = got[2].double(), want[2]
    assert torch.equal(torch.isnan(lse), torch.isnan(w))
    bad = torch.isnan(w) | (lse == w)
    assert bool((bad | ((lse - w).abs() <= _rel(vocab, x) + 2 * U * w.abs())).all()), (lse, w)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows,vocab,cols,k,T", [
    (1, 1, 1, 1, 1.0), (2, 1, 4, 3, 2.0), (3, 2, 2, 2, 1.0), (5, 7, 9, 7, 0.5), (4, 8, 8, 1, 1.0), (3, 33, 40, 32, 1.0),
    (6, 255, 256, 16, 3.0), (2, 1000, 1001, 1024, 1.0), (3, 1024, 1024, 1024, 1.0), (9, 4098, 4160, 32, 1.0),
    (1, 4098, 4160, 1000, 1.0), (2, 12289, 12289, 64, 2.0), (1, 50257, 50304, 64, 1.0), (3, 50257, 50257, 500, 1.0),
    (2, 131073, 131073, 256, 1.0), (1, 262144, 262144, 1024, 1.0)])
def test_top_logits(rows, vocab, cols, k, T, dtype):
    gen = torch.Generator().manual_seed(vocab + k)
    z = (torch.randn(rows, cols, generator=gen) * 3).to(TYPES[dtype])
    _check_top(z, k, vocab, T, _top(z, k, vocab, T))


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("ld,shift", [(4099, 0), (4099, 1), (4104, 0), (4101, 7)])
def test_top_logits_strides(ld, shift, dtype):
    gen = torch.Generator().manual_seed(ld + shift)
    z = torch.randn(6, 4098, generator=gen).to(TYPES[dtype])
    _check_top(z, 20, 4097, 1.0, _top(z, 20, 4097, 1.0, ld, shift))


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("vocab", [40, 4098, 50257])
def test_top_logits_ties_masks_and_special_values(vocab, dtype):
    """Ties go to the lowest column, also where the whole row is one value; -0 is +0; NaN comes first; masks of -inf and of
    the type's lowest value leave fewer numbers than k; equal values everywhere but a few; values in order."""
    t = TYPES[dtype]
    gen = torch.Generator().manual_seed(vocab)
    z = torch.randn(14, vocab, generator=gen).to(t)
    z[0] = 1.5
    z[1] = -math.inf
    z[2] = torch.finfo(t).min
    z[3] = -math.inf
    z[3, [5, vocab - 1, 17]] = torch.tensor([2.0, 2.0, -3.0]).to(t)
    z[4] = 0.0
    z[4, ::3] = -0.0
    z[5, [3, vocab - 2]] = math.nan
    z[6, 7] = math.inf
    z[7] = torch.arange(vocab).remainder(3).to(t)
    z[8] = -1.0
    z[8, vocab // 2:] = 1.0
    z[9] = torch.linspace(-3, 3, vocab).to(t)
    z[10] = torch.linspace(3, -3, vocab).to(t)
    z[11] = (torch.randn(vocab, generator=gen) * 1e-3).to(t)
    z[12] = torch.randint(-2, 3, (vocab,), generator=gen).to(t)
    z[13] = torch.finfo(t).tiny
    z[13, 9] = -torch.finfo(t).tiny
    for k in (1, 16, 33):
        _check_top(z, k, vocab, 1.0, _top(z, k, vocab))


def test_top_logits_without_lse_and_without_rows():
    z = torch.randn(3, 100, generator=torch.Generator().manual_seed(1))
    assert torch.equal(_top(z, 5, lse=False)[1], R.top(z, 5, 100, 1.0)[1])
    from cuda_transformer_b200 import losses
    losses.top_logits(torch.empty(0, 8, device="cuda"), 2, torch.empty(0, 2, device="cuda"),
                      torch.empty(0, 2, dtype=torch.int32, device="cuda"), torch.empty(0, device="cuda"))
    torch.cuda.synchronize()


# ---------------------------------------------------------------- balance_loss

def _balance_problem(rows, experts, dtype, k, ignored=0.0, dropped=0.0, seed=0):
    gen = torch.Generator().manual_seed(31 * seed + rows + experts)
    z = torch.randn(rows, experts, generator=gen) * 2 + torch.randn(experts, generator=gen)
    chosen = torch.topk(z, min(k, experts), dim=1).indices.to(torch.int32) if rows else torch.empty(0, min(k, experts), dtype=torch.int32)
    chosen = chosen.repeat(1, -(-k // chosen.shape[1]))[:, :k].contiguous()
    chosen[torch.rand(rows, k, generator=gen) < dropped] = -1
    targets = torch.zeros(rows, dtype=torch.int32)
    targets[torch.rand(rows, generator=gen) < ignored] = -1
    return z.to(dtype), chosen, targets


def _balance(z, chosen, targets, weight=0.01, scale=65536.0, ld=None, shift=0, accumulate=None, add=False, gradient=True,
             in_place=False, start_loss=0.0):
    from cuda_transformer_b200 import losses
    rows, experts = z.shape
    a = Guarded(rows, experts, z.dtype, ld, shift)
    a.t.copy_(z)
    d = a if in_place else Guarded(rows, experts, z.dtype, ld, shift)
    if accumulate is not None:
        d.t.copy_(accumulate)
    counts, loss = Guarded(1, experts, torch.int32), Guarded(1, 1, torch.float32)
    state, ws = _state(scale), losses.loss_workspace()
    state.view(torch.float32)[13] = start_loss
    losses.balance_loss(a.t, d.t if gradient else None, chosen.cuda(), _gpu(targets), state, counts.t[0], loss.t[0], ws,
                        weight=weight, accumulate=accumulate is not None, add_to_state=add)
    torch.cuda.synchronize()
    assert a.intact() and d.intact() and counts.intact() and loss.intact() and not bool(ws[:COUNTERS].any())
    st = _fields(state)
    assert st.loss_scale == scale and st.n_valid == 0
    return dict(dlogits=d.t.cpu(), counts=counts.t[0].cpu(), loss=float(loss.t[0, 0]), state_loss=st.loss)


def _check_balance(z, chosen, targets, got, weight=0.01, scale=65536.0, base=None):
    want = R.balance(z, chosen, targets, weight, scale)
    assert torch.equal(got["counts"], want["counts"])
    rel = _rel(z.shape[1], 40.0)
    assert abs(got["loss"] - want["loss"]) <= (rel + 4 * U) * abs(want["loss"])
    d = want["dlogits"] + (0.0 if base is None else base.double())
    lim = rel * want["size"] + torch.finfo(z.dtype).eps / 2 * (d.abs() + rel * want["size"]) + TINY[z.dtype] + U * d.abs() + 2.0 ** -120
    assert bool(((got["dlogits"].double() - d).abs() <= lim).all())


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows,experts,k", [(1, 1, 1), (1, 8, 2), (3, 5, 5), (64, 8, 2), (33, 7, 3), (100, 64, 8), (65, 96, 1),
                                            (257, 128, 6), (40, 333, 9), (19, 512, 4), (12, 1000, 2), (9, 1024, 1024),
                                            (3000, 16, 2), (20011, 60, 4)])
def test_balance(rows, experts, k, dtype):
    z, chosen, targets = _balance_problem(rows, experts, TYPES[dtype], k, 0.2 if rows > 4 else 0.0, 0.1)
    _check_balance(z, chosen, targets, _balance(z, chosen, targets))


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("ld,shift", [(64, 0), (67, 0), (71, 3), (72, 0)])
def test_balance_strides_accumulation_and_the_state(ld, shift, dtype):
    z, chosen, targets = _balance_problem(50, 64, TYPES[dtype], 4, 0.3, 0.0)
    _check_balance(z, chosen, targets, _balance(z, chosen, targets, ld=ld, shift=shift))
    base = torch.randn(50, 64, generator=torch.Generator().manual_seed(9)).to(z.dtype)
    got = _balance(z, chosen, targets, ld=ld, shift=shift, accumulate=base, add=True, start_loss=2.5)
    _check_balance(z, chosen, targets, got, base=base)
    assert torch.equal(got["dlogits"][targets < 0], base[targets < 0])
    assert abs(got["state_loss"] - (2.5 + got["loss"])) <= U * 4
    # the same layout gives the same bits (another one is summed in another order)
    inside = _balance(z, chosen, targets, ld=ld, shift=shift, in_place=True)
    assert torch.equal(inside["dlogits"], _balance(z, chosen, targets, ld=ld, shift=shift)["dlogits"])
    alone = _balance(z, chosen, targets, ld=ld, shift=shift, gradient=False)
    assert alone["loss"] == inside["loss"] and alone["state_loss"] == 0.0
    assert torch.equal(alone["counts"], inside["counts"])


def test_balance_all_rows_count_without_targets():
    z, chosen, targets = _balance_problem(70, 16, torch.float32, 2)
    a, b = _balance(z, chosen, None), _balance(z, chosen, targets)
    assert torch.equal(a["dlogits"], b["dlogits"]) and a["loss"] == b["loss"] and torch.equal(a["counts"], b["counts"])


def test_balance_nothing_counts():
    z, chosen, targets = _balance_problem(20, 8, torch.float16, 2)
    targets[:] = -1
    got = _balance(z, chosen, targets)
    assert got["loss"] == 0.0 and not bool(got["counts"].any()) and not bool(got["dlogits"].any())
    chosen[:] = -1                                              # rows that count, without a choice
    got = _balance(z, chosen, None)
    assert got["loss"] == 0.0 and not bool(got["counts"].any()) and not bool(got["dlogits"].any())
    empty = _balance(z[:0], chosen[:0], None)
    assert empty["loss"] == 0.0 and not bool(empty["counts"].any())


def test_balance_an_expert_beyond_the_last_and_masked_logits():
    z, chosen, targets = _balance_problem(30, 8, torch.float32, 2)
    chosen[7, 1] = 8
    got = _balance(z, chosen, targets)
    assert math.isnan(got["loss"]) and bool(torch.isnan(got["dlogits"]).all())
    assert torch.equal(got["counts"], R.balance(z, chosen, targets, 0.01, 1.0)["counts"])
    chosen[7, 1] = -1
    z[:, 3] = -math.inf                                         # an expert that is switched off
    z[2, [0, 1]] = torch.finfo(torch.float32).min
    _check_balance(z, chosen, targets, _balance(z, chosen, targets))
    targets[7], chosen[7, 0] = -1, 900                          # a row that does not count may say anything
    z[7] = math.nan
    got = _balance(z, chosen, targets)
    assert math.isfinite(got["loss"]) and bool(torch.isfinite(got["dlogits"]).all())


@pytest.mark.parametrize("rows,experts", [(40, 8), (700, 64), (300, 67)])
def test_balance_a_row_without_a_softmax_is_nan_alone(rows, experts):
    z, chosen, targets = _balance_problem(rows, experts, torch.float16, 8)
    bad = {3: -math.inf, 11: math.nan, 20: math.inf}
    for row, value in bad.items():
        z[row, :] = value if value == -math.inf else z[row]
        z[row, experts - 1] = value
    got = _balance(z, chosen, None)
    assert math.isnan(got["loss"]) and torch.equal(got["counts"], R.balance(z, chosen, None, 0.01, 1.0)["counts"])
    assert torch.isnan(got["dlogits"].float()).any(1).nonzero()[:, 0].tolist() == list(bad)
    targets[list(bad)] = -1                                     # the same rows, left out
    _check_balance(z.nan_to_num(0.0, 0.0, 0.0), chosen, targets, _balance(z, chosen, targets))


# ---------------------------------------------------------------- streams, graphs, the step

def test_calls_on_two_streams_with_a_workspace_each():
    from cuda_transformer_b200 import losses
    problems = [_problem(700, 4098, 4160, torch.float16, 8, 1.0, True, 0.5, seed=s) for s in (1, 2)]
    alone = [_run(p) for p in problems]
    streams = [torch.cuda.Stream() for _ in problems]
    devs = []
    for p in problems:
        devs.append(dict(z=p["logits"].cuda(), d=torch.empty(700, 4160, dtype=torch.float16, device="cuda"), y=_gpu(p["targets"]),
                         v=_gpu(p["values"]), i=_gpu(p["indices"]), l=_gpu(p["lse"]), st=_state(1024.0),
                         row=torch.empty(700, device="cuda"), ws=losses.loss_workspace()))
    torch.cuda.synchronize()
    for _ in range(5):
        for q, s in zip(devs, streams):
            losses.distill_loss(q["z"], q["d"], q["y"], q["v"], q["i"], q["l"], q["st"], q["row"], q["ws"], vocab=4098,
                                hard_weight=0.5, stream=s)
    torch.cuda.synchronize()
    for q, want in zip(devs, alone):
        assert torch.equal(q["d"].cpu(), want["dlogits"]) and _fields(q["st"]).loss == want["loss"]


def _step_case():
    """A linear head on hidden states, a teacher, a router: what one step calls, on an optimizer's own state."""
    from cuda_transformer_b200 import amp
    from cuda_transformer_b200.layout import ParamSlot
    gen = torch.Generator().manual_seed(11)
    rows, width, vocab, cols, experts = 96, 64, 500, 512, 8
    slots = [ParamSlot("head", 0, cols * width, 2, (cols, width)), ParamSlot("router", cols * width, experts * width, 2, (experts, width))]
    opt = amp.AmpOptimizer(slots, amp.make_schedule(grad_clip=1.0), loss_scale=256.0, history_len=8)
    opt.set_params(torch.randn(cols * width + experts * width, generator=gen) * 0.05)
    d = dict(h=(torch.randn(rows, width, generator=gen)).half().cuda(), teacher=(torch.randn(rows, cols, generator=gen) * 3).half().cuda(),
             y=torch.randint(0, vocab, (rows,), generator=gen, dtype=torch.int32).cuda(),
             values=torch.empty(rows, 16, dtype=torch.float16, device="cuda"), indices=torch.empty(rows, 16, dtype=torch.int32, device="cuda"),
             lse=torch.empty(rows, device="cuda"), row=torch.empty(rows, device="cuda"),
             z=torch.empty(rows, cols, dtype=torch.float16, device="cuda"), r=torch.empty(rows, experts, dtype=torch.float16, device="cuda"),
             counts=torch.empty(experts, dtype=torch.int32, device="cuda"), aux=torch.empty(1, device="cuda"))
    d["y"][::7] = -1
    return opt, d, (rows, width, vocab, cols, experts)


def _step(opt, d, sizes):
    from cuda_transformer_b200 import amp, losses
    rows, width, vocab, cols, experts = sizes
    head = opt.weights16[:cols * width].view(cols, width)
    router = opt.weights16[cols * width:cols * width + experts * width].view(experts, width)
    amp.begin_step(opt.state)
    losses.top_logits(d["teacher"], 16, d["values"], d["indices"], d["lse"], vocab=vocab, temperature=2.0)
    torch.mm(d["h"], head.t(), out=d["z"])
    torch.mm(d["h"], router.t(), out=d["r"])
    chosen = torch.topk(d["r"].float(), 2, dim=1).indices.to(torch.int32)
    opt.distill_loss(d["z"], d["z"], d["y"], d["values"], d["indices"], d["lse"], d["row"], vocab=vocab, temperature=2.0,
                     soft_weight=4.0, hard_weight=0.5)
    opt.balance_loss(d["r"], d["r"], chosen, d["y"], d["counts"], d["aux"], weight=0.02)
    torch.mm(d["z"].t(), d["h"], out=opt.grads16[:cols * width].view(cols, width))
    torch.mm(d["r"].t(), d["h"], out=opt.grads16[cols * width:cols * width + experts * width].view(experts, width))
    opt.optimizer_step()


def test_a_step_of_all_three_lands_in_the_state_the_history_and_the_weights():
    opt, d, sizes = _step_case()
    rows, width, vocab, cols, experts = sizes
    w = opt.weights16.clone().double().cpu()
    h = d["h"].double().cpu()
    head = w[:cols * width].view(cols, width).requires_grad_()
    _step(opt, d, sizes)
    torch.cuda.synchronize()
    z16 = (d["h"] @ opt.weights16.new_tensor(head.detach().numpy()).view(cols, width).t()).cpu()
    want = R.distill(z16, d["y"].cpu(), d["values"].cpu(), d["indices"].cpu(), d["lse"].cpu(), vocab, 2.0, 4.0, 0.5, 256.0)
    top = R.top(d["teacher"].cpu(), 16, vocab, 2.0)
    assert torch.equal(d["indices"].cpu(), top[1])
    grads = opt.grads16[:cols * width].view(cols, width).double().cpu()
    exact = want["dlogits"].t() @ h
    # each dlogit is half a fp16 step off (and half a subnormal step), the product is rounded to fp16 once more
    slack = (want["dlogits"].abs() * 2.0 ** -10 + 2.0 ** -24).t() @ h.abs() + exact.abs() * 2.0 ** -10 + 2.0 ** -24
    assert bool(((grads - exact).abs() <= slack).all())
    st = opt.read_state()
    assert st.n_valid == want["n_valid"] and st.found_inf == 0 and st.step == 1 and st.adam_t == 1
    aux = float(d["aux"])
    assert abs(st.loss - (want["loss"] + aux)) <= 1e-5 * abs(want["loss"]) and aux > 0.0
    assert int(d["counts"].sum()) == 2 * want["n_valid"]
    first = opt.read_history()[0]
    assert first.loss == st.loss and first.n_valid == st.n_valid


def test_captured_steps_replay_to_the_same_bits():
    eager, d, sizes = _step_case()
    for _ in range(4):
        _step(eager, d, sizes)
    torch.cuda.synchronize()
    captured, d2, _ = _step_case()
    warm, d3, _ = _step_case()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _step(warm, d3, sizes)                                  # the matrix library's first calls are not capturable
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        _step(captured, d2, sizes)
    assert captured.read_state().step == 0                      # a capture runs nothing
    for _ in range(4):
        graph.replay()
    torch.cuda.synchronize()
    a, b = eager.read_state(), captured.read_state()
    assert (a.step, a.loss, a.n_valid, a.grad_norm) == (b.step, b.loss, b.n_valid, b.grad_norm)
    assert torch.equal(eager.master, captured.master) and torch.equal(eager.weights16, captured.weights16)
    assert torch.equal(d["row"], d2["row"]) and torch.equal(d["counts"], d2["counts"])


FIRST_CALLS_IN_A_CAPTURE = """
import torch
from cuda_transformer_b200 import amp, losses
gen = torch.Generator().manual_seed(5)
rows, vocab, experts = 300, 12000, 64
z = torch.randn(rows, vocab, generator=gen).bfloat16().cuda()
t = torch.randn(rows, vocab, generator=gen).bfloat16().cuda()
r = torch.randn(4096, experts, generator=gen).cuda()
c = torch.randint(-1, experts, (4096, 4), generator=gen, dtype=torch.int32).cuda()
y = torch.randint(-1, vocab, (rows,), generator=gen, dtype=torch.int32).cuda()
v = torch.empty(rows, 9, dtype=torch.bfloat16, device="cuda")
i = torch.empty(rows, 9, dtype=torch.int32, device="cuda")
l, row, loss, ws = torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda"), torch.empty(1, device="cuda"), losses.loss_workspace()
counts = torch.empty(experts, dtype=torch.int32, device="cuda")
st = torch.frombuffer(bytearray(bytes(amp.initial_state(64.0))), dtype=torch.uint8).cuda()
dz, dr = torch.empty_like(z), torch.empty_like(r)
def calls():
    losses.top_logits(t, 9, v, i, l)
    losses.distill_loss(z, dz, y, v, i, l, st, row, ws, hard_weight=0.5)
    losses.balance_loss(r, dr, c, None, st, counts, loss, ws, add_to_state=True)
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    calls()
outs = []
for _ in range(3):
    graph.replay()
    torch.cuda.synchronize()
    outs.append([x.clone() for x in (v, i, l, dz, row, dr, counts, loss, st)])
calls()
torch.cuda.synchronize()
outs.append([x.clone() for x in (v, i, l, dz, row, dr, counts, loss, st)])
assert all(torch.equal(a, b) for o in outs[1:] for a, b in zip(outs[0], o))
assert int(counts.sum()) == int((c >= 0).sum()) and bool(torch.isfinite(loss).all())
for _ in range(20):                 # nothing waits between the calls
    calls()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(outs[0], (v, i, l, dz, row, dr, counts, loss, st)))
print("same bits")
"""


def test_the_first_calls_of_a_process_may_be_captured():
    """Nothing is set up on a first call that a capture forbids, the counting launch and the one that starts behind it
    early among them; replays, eager calls and calls without a wait in between give the same bits."""
    import os
    import subprocess
    import sys
    repo = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    out = subprocess.run([sys.executable, "-c", FIRST_CALLS_IN_A_CAPTURE], cwd=repo, capture_output=True, text=True, timeout=300)
    assert out.returncode == 0 and "same bits" in out.stdout, out.stderr[-2000:]


def test_a_row_gone_wrong_skips_the_step():
    opt, d, sizes = _step_case()
    before = opt.master.clone()
    d["y"][3] = sizes[2]                                        # a label beyond the vocabulary
    _step(opt, d, sizes)
    st = opt.read_state()
    assert st.found_inf == 1 and st.skipped == 1 and st.loss_scale == 128.0 and torch.equal(opt.master, before)


def test_python_refusals():
    from cuda_transformer_b200 import _lib, losses
    dev = "cuda"
    z, st, ws = torch.zeros(4, 32, dtype=torch.float16, device=dev), _state(1.0), losses.loss_workspace()
    row, y = torch.zeros(4, device=dev), torch.zeros(4, dtype=torch.int32, device=dev)
    v, i = torch.zeros(4, 3, device=dev), torch.zeros(4, 3, dtype=torch.int32, device=dev)
    good = dict(logits=z, dlogits=z, targets=y, values=v, indices=i, lse=None, state=st, row_loss=row, workspace=ws)
    losses.distill_loss(**good)
    for change in (dict(logits=z.double()), dict(logits=z[0]), dict(logits=z.t()), dict(dlogits=z[:3]), dict(dlogits=z.float()),
                   dict(targets=y.long()), dict(targets=y[:3]), dict(targets=y.cpu()), dict(values=v[:, :2]), dict(values=None),
                   dict(indices=None), dict(indices=i.long()), dict(lse=row.double()), dict(row_loss=row[:3]),
                   dict(row_loss=row.double()), dict(state=st[:56]), dict(workspace=ws[:-1]), dict(values=v.double())):
        with pytest.raises(ValueError):
            losses.distill_loss(**{**good, **change})
    for change in (dict(vocab=0), dict(vocab=33), dict(temperature=0.0), dict(soft_weight=math.nan), dict(targets=None, hard_weight=1.0),
                   dict(logits=z[:1].expand(4, 32)), dict(workspace=torch.zeros(40000, dtype=torch.uint8, device=dev)[1:])):
        with pytest.raises(_lib.B200AmpError) as err:
            losses.distill_loss(**{**good, **change})
        assert err.value.status == _lib.ERR_ARG
    with pytest.raises(_lib.B200AmpError) as err:
        losses.distill_loss(**{**good, "values": torch.zeros(4, 1025, device=dev), "indices": torch.zeros(4, 1025, dtype=torch.int32, device=dev)})
    assert err.value.status == _lib.ERR_ARG
    for k, bad in ((3, dict(values=v)), (3, dict(indices=i.long())), (2, {}), (3, dict(lse=row[:2])), (3, dict(vocab=40))):
        with pytest.raises(ValueError):
            losses.top_logits(**{**dict(logits=z, k=k, values=v.half(), indices=i, lse=row), **bad})
    counts, loss = torch.zeros(32, dtype=torch.int32, device=dev), torch.zeros(1, device=dev)
    good = dict(logits=z, dlogits=z, chosen=i, targets=y, state=st, counts=counts, loss=loss, workspace=ws)
    losses.balance_loss(**good)
    for change in (dict(chosen=i[0]), dict(chosen=i.long()), dict(counts=counts[:3]), dict(loss=row), dict(dlogits=z.float()),
                   dict(state=st[:1]), dict(workspace=ws[:100]), dict(targets=y[:1])):
        with pytest.raises(ValueError):
            losses.balance_loss(**{**good, **change})
    with pytest.raises(_lib.B200AmpError):
        losses.balance_loss(**{**good, "accumulate": True})     # in place and accumulated
    torch.cuda.synchronize()


def test_tensors_on_another_device_than_the_current_one():
    if torch.cuda.device_count() < 2:
        pytest.skip("needs two GPUs")
    from cuda_transformer_b200 import losses
    p = _problem(5, 300, 320, torch.float16, 4, 1.0, True, 0.5)
    want = _run(p)
    dev = torch.device("cuda:1")
    g = {n: (t.to(dev) if torch.is_tensor(t) else t) for n, t in p.items()}
    d, st = torch.empty(5, 320, dtype=torch.float16, device=dev), _state(1024.0).to(dev)
    row, ws = torch.empty(5, device=dev), losses.loss_workspace(dev)
    losses.distill_loss(g["logits"], d, g["targets"], g["values"], g["indices"], g["lse"], st, row, ws, vocab=300, hard_weight=0.5)
    torch.cuda.synchronize(dev)
    assert torch.equal(d.cpu(), want["dlogits"]) and torch.equal(row.cpu(), want["row_loss"])
