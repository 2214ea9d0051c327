"""The operators that open a training step's backward pass, and the cases they are measured on.

Three operators belong together: a teacher's full logits are cut down to its k largest (`top_logits`), a student
is trained on that record (`distill_loss`: loss and loss-scaled gradient of the logits, mixed with the usual
cross-entropy), and a mixture-of-experts router is kept balanced (`balance_loss`: per-expert counts, loss and
loss-scaled gradient). Each is given here in its plain form, in elementary torch operations, and as the calls of
cuda_transformer_b200.losses (where `own` is true). `exact` restates the definitions in 64 bits.
"""
import math

import torch

own = False

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
WORKSPACE_BYTES = 32768     # B200AMP_LOSS_WORKSPACE_BYTES of include/b200amp.h, zeroed once


# ---------------------------------------------------------------- the cases

def listed():
    return [
        # one small sequence of the debug model (vocabulary 4098 in 4160 columns): latency counts
        dict(name="distill_debug", op="distill", rows=64, vocab=4098, cols=4160, dtype="f16", k=8, temperature=1.0,
             rest=True, hard=0.0, ignored=0.0),
        # a step of the 6-layer model: 16 x 256 tokens, temperature 2, a tenth of the tokens is padding
        dict(name="distill_readme", op="distill", rows=4096, vocab=4098, cols=4160, dtype="f16", k=32, temperature=2.0,
             rest=False, hard=0.5, ignored=0.1),
        # a step at the 50304-column vocabulary, 8 x 1024 tokens: the ordinary large call
        dict(name="distill_50304", op="distill", rows=8192, vocab=50257, cols=50304, dtype="f16", k=64, temperature=1.0,
             rest=True, hard=0.5, ignored=0.05),
        # an unpadded odd vocabulary: every row starts at another alignment; bf16; two softmaxes in one call
        dict(name="distill_odd_bf16", op="distill", rows=1023, vocab=50257, cols=50257, dtype="bf16", k=100,
             temperature=2.0, rest=True, hard=0.3, ignored=0.0),
        # fp32 logits of a long vocabulary: the largest call
        dict(name="distill_long_f32", op="distill", rows=2048, vocab=131072, cols=131072, dtype="f32", k=256,
             temperature=1.0, rest=False, hard=0.0, ignored=0.0),
        # a teacher answering one token at a time: a single row
        dict(name="top_one_row", op="top", rows=1, vocab=50257, cols=50304, dtype="f16", k=64, temperature=1.0),
        # a teacher scoring a batch for the 50304-column student
        dict(name="top_50304", op="top", rows=8192, vocab=50257, cols=50304, dtype="f16", k=64, temperature=1.0),
        # fewer rows of a long odd vocabulary, many entries kept
        dict(name="top_wide_bf16", op="top", rows=510, vocab=128001, cols=128001, dtype="bf16", k=256, temperature=2.0),
        # fp32 logits of the 4160-column vocabulary
        dict(name="top_readme_f32", op="top", rows=4096, vocab=4098, cols=4160, dtype="f32", k=32, temperature=1.0),
        # a router of few experts on one short sequence
        dict(name="balance_small", op="balance", rows=64, experts=8, dtype="f32", k=2, ignored=0.0, dropped=0.0),
        # a layer of a training step: 8 x 2048 tokens, 64 experts, padding and dropped choices
        dict(name="balance_64", op="balance", rows=16384, experts=64, dtype="f16", k=8, ignored=0.1, dropped=0.05),
        # many tokens, many experts, fp32 router
        dict(name="balance_256", op="balance", rows=65536, experts=256, dtype="f32", k=8, ignored=0.0, dropped=0.02),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["distill", "top", "balance"])
    dtype = rng.choice(["f16", "bf16", "f32"])
    size = 4 if dtype == "f32" else 2
    if op == "balance":
        experts = _log_int(rng, 4, 512)
        rows = min(_log_int(rng, 1, 65536), 65536 * 256 * 4 // (experts * size))
        return dict(op=op, rows=rows, experts=experts, dtype=dtype, k=rng.randint(1, min(8, experts)),
                    ignored=rng.choice([0.0, rng.uniform(0.0, 0.5)]), dropped=rng.choice([0.0, rng.uniform(0.0, 0.2)]))
    vocab = _log_int(rng, 256, 131072)
    cols = rng.choice([vocab, -(-vocab // 64) * 64, vocab + rng.randint(0, 37)])
    rows = min(_log_int(rng, 1, 8192), 8192 * 50304 * 2 // (cols * size))
    case = dict(op=op, rows=rows, vocab=vocab, cols=cols, dtype=dtype, k=min(_log_int(rng, 1, 256), vocab // 4),
                temperature=rng.choice([1.0, 2.0, round(rng.uniform(0.5, 4.0), 3)]))
    if op == "distill":
        case.update(rest=rng.random() < 0.5, hard=rng.choice([0.0, round(rng.uniform(0.1, 1.0), 3)]),
                    ignored=rng.choice([0.0, rng.uniform(0.0, 0.5)]))
    return case


# ---------------------------------------------------------------- inputs

def _loss_scale(case):
    """What a run starts with, or what it has come down to where the mean is over few rows (fp16 ends at 65504)."""
    return 65536.0 if case["rows"] >= 64 else 256.0


def _state(case, dev):
    """The step state of 15 four-byte fields: loss_scale, inv_scale, ..., loss (13), n_valid (14)."""
    state = torch.zeros(15, dtype=torch.float32, device=dev)
    state[0], state[1] = _loss_scale(case), 1.0 / _loss_scale(case)
    return state


def _targets(rows, classes, ignored, gen, dev):
    """Labels, and -1 for the rows that do not count (padding)."""
    targets = torch.randint(0, classes, (rows,), generator=gen, device=dev, dtype=torch.int32)
    if ignored:
        out = torch.rand(rows, generator=gen, device=dev) < ignored
        out[0] = False
        targets[out] = -1
    return targets


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(int(seed) * 7919 + 17)
    rows, dtype = case["rows"], TYPES[case["dtype"]]
    s = {"case": case, "workspace": torch.zeros(WORKSPACE_BYTES, dtype=torch.uint8, device=dev), "state": _state(case, dev)}
    if case["op"] == "balance":
        experts, k = case["experts"], case["k"]
        # a router with favourites, and its k best choices of each token
        bias = torch.randn(experts, generator=gen, device=dev)
        logits = torch.randn(rows, experts, generator=gen, device=dev) + bias
        choice = torch.topk(logits, k, dim=1).indices.to(torch.int32)
        if case["dropped"]:
            choice[torch.rand(rows, k, generator=gen, device=dev) < case["dropped"]] = -1
        s.update(logits=logits.to(dtype), experts=choice, targets=_targets(rows, 1000, case["ignored"], gen, dev),
                 dlogits=torch.empty(rows, experts, dtype=dtype, device=dev),
                 counts=torch.empty(experts, dtype=torch.int32, device=dev), loss=torch.empty(1, device=dev))
        return s
    vocab, cols, k = case["vocab"], case["cols"], case["k"]
    # logits as a language model leaves them: token frequencies, noise, and a few tokens that stand out
    freq = -1.0 * torch.log1p(torch.arange(vocab, device=dev, dtype=torch.float32))[torch.randperm(vocab, generator=gen, device=dev)]
    logits = torch.empty(rows, cols, dtype=dtype, device=dev)
    logits[:, vocab:] = 0
    values = torch.empty(rows, k, dtype=dtype, device=dev)
    indices = torch.empty(rows, k, dtype=torch.int32, device=dev)
    lse = torch.empty(rows, dtype=torch.float32, device=dev)
    s.update(logits=logits, values=values, indices=indices, lse=lse)
    for at in range(0, rows, 1024):
        n = min(1024, rows - at)
        z = torch.randn(n, vocab, generator=gen, device=dev).mul_(1.5).add_(freq)
        z.scatter_add_(1, torch.randint(0, vocab, (n, 8), generator=gen, device=dev),
                       torch.rand(n, 8, generator=gen, device=dev).mul_(10.0))
        logits[at:at + n, :vocab] = z
        if case["op"] == "distill":
            # the teacher: near the student, and surer
            t = z.mul_(0.9).add_(torch.randn(n, vocab, generator=gen, device=dev), alpha=0.5).to(dtype)
            best = torch.topk(t, k, dim=1)
            values[at:at + n], indices[at:at + n] = best.values, best.indices
            lse[at:at + n] = torch.logsumexp(t.float() / case["temperature"], dim=1)
    if case["op"] == "distill":
        s.update(targets=_targets(rows, vocab, case["ignored"], gen, dev), dlogits=torch.empty_like(logits),
                 row_loss=torch.empty(rows, device=dev))
    return s


# ---------------------------------------------------------------- one pass

def run(s):
    return {"distill": _distill, "top": _top, "balance": _balance}[s["case"]["op"]](s)


def _distill(s):
    c = s["case"]
    if own:
        from cuda_transformer_b200 import losses
        losses.distill_loss(s["logits"], s["dlogits"], s["targets"], s["values"], s["indices"],
                            s["lse"] if c["rest"] else None, s["state"], s["row_loss"], s["workspace"],
                            vocab=c["vocab"], temperature=c["temperature"], soft_weight=c["temperature"] ** 2,
                            hard_weight=c["hard"])
        return {"dlogits": s["dlogits"], "row_loss": s["row_loss"], "loss": s["state"][13:14],
                "n_valid": s["state"].view(torch.int32)[14:15]}
    T, soft, hard = c["temperature"], c["temperature"] ** 2, c["hard"]
    valid = s["targets"] >= 0
    n_valid = valid.sum()
    z = s["logits"][:, :c["vocab"]].float()
    top_z = z.max(1, keepdim=True).values
    index = s["indices"].long()

    # a row has few listed tokens: they are held in 64 bits, and the others' sum is taken without them, since the loss
    # (and the mass that the teacher leaves to the others) is a difference between the two
    t = s["values"].double() / T
    if not c["rest"]:
        t = t - t.amax(1, keepdim=True)
    log_p = t - (s["lse"].double()[:, None] if c["rest"] else t.exp().sum(1, keepdim=True).log())
    p = log_p.exp()
    x = (z.gather(1, index).double() - top_z.double()) / T
    grad = ((z - top_z) / T).exp().scatter_(1, index, 0.0)
    others = grad.sum(1).double()
    total = others + x.exp().sum(1)
    loss = (p * (log_p - x)).sum(1)
    mass = p.sum(1)
    factor = mass / total
    if c["rest"]:
        rest = (1.0 - mass).clamp(min=0.0)
        loss += torch.where(rest > 0, rest * (rest / others).log(), torch.zeros_like(rest))
        mass = mass + rest
        factor = mass / total - rest / others
    loss = soft * (loss + mass * total.log())
    grad *= (soft / T * factor).float()[:, None]
    grad.scatter_(1, index, (soft / T * ((mass / total)[:, None] * x.exp() - p)).float())
    if hard:
        label = s["targets"].long().clamp(min=0)[:, None]
        x = z.gather(1, label).double() - top_z.double()
        e = (z - top_z).exp().scatter_(1, label, 0.0)
        others = e.sum(1, keepdim=True).double()
        total = others + x.exp()
        loss += hard * (total.log() - x)[:, 0]
        e.scatter_(1, label, -others.float())
        grad += e.mul_((hard / total).float())
        del e
    loss = torch.where(valid, loss, torch.zeros_like(loss))
    count = n_valid.clamp(min=1)
    grad *= torch.where(valid, s["state"][0] / count, torch.zeros_like(s["state"][0]))[:, None]
    dlogits = torch.zeros_like(s["logits"])
    dlogits[:, :c["vocab"]] = grad
    return {"dlogits": dlogits, "row_loss": loss.float(), "loss": (loss.sum() / count).float().reshape(1),
            "n_valid": n_valid.to(torch.int32).reshape(1)}


def _top(s):
    c = s["case"]
    if own:
        from cuda_transformer_b200 import losses
        losses.top_logits(s["logits"], c["k"], s["values"], s["indices"], s["lse"], vocab=c["vocab"],
                          temperature=c["temperature"])
        return {"values": s["values"], "indices": s["indices"], "lse": s["lse"]}
    z = s["logits"][:, :c["vocab"]]
    values, indices = torch.sort(z, dim=1, descending=True, stable=True)    # stable: ties to the lowest index
    x = z.float() / c["temperature"]
    m = x.amax(1, keepdim=True)
    lse = m[:, 0] + (x - m).exp().sum(1).log()
    return {"values": values[:, :c["k"]].contiguous(), "indices": indices[:, :c["k"]].to(torch.int32), "lse": lse}


def _balance(s):
    c = s["case"]
    if own:
        from cuda_transformer_b200 import losses
        losses.balance_loss(s["logits"], s["dlogits"], s["experts"], s["targets"], s["state"], s["counts"], s["loss"],
                            s["workspace"], weight=0.01)
        return {"dlogits": s["dlogits"], "counts": s["counts"], "loss": s["loss"]}
    experts, k = c["experts"], c["k"]
    valid = s["targets"] >= 0
    n_valid = valid.sum().clamp(min=1)
    taken = (s["experts"] >= 0) & valid[:, None]
    counts = torch.zeros(experts + 1, dtype=torch.int32, device=taken.device)
    where = torch.where(taken, s["experts"], torch.full_like(s["experts"], experts)).reshape(-1).long()
    counts.scatter_add_(0, where, torch.ones_like(where, dtype=torch.int32))
    counts = counts[:experts]
    share = counts / (n_valid * k).float()
    z = s["logits"].float()
    p = (z - z.amax(1, keepdim=True)).exp()
    p = p / p.sum(1, keepdim=True)
    dot = (p * share).sum(1, keepdim=True)
    factor = 0.01 * experts / n_valid.float()
    loss = factor * torch.where(valid, dot[:, 0], torch.zeros_like(dot[:, 0])).double().sum()
    grad = factor * s["state"][0] * p * (share - dot)
    grad = torch.where(valid[:, None], grad, torch.zeros_like(grad))
    return {"dlogits": grad.to(s["logits"].dtype), "counts": counts, "loss": loss.float().reshape(1)}


# ---------------------------------------------------------------- what a pass cannot do without

def work(case):
    size = TYPES[case["dtype"]].itemsize
    rows, k = case["rows"], case["k"]
    if case["op"] == "balance":
        cells = rows * case["experts"]
        return {"bytes": 2 * cells * size + rows * k * 4 + rows * 4 + case["experts"] * 4 + 4, "flops": 8 * cells}
    record = rows * k * (size + 4)
    if case["op"] == "top":
        return {"bytes": rows * case["vocab"] * size + record + rows * 4, "flops": 4 * rows * case["vocab"]}
    # rows that do not count are not read, only their zero gradient is written
    read = int(rows * (1.0 - case["ignored"])) * case["vocab"] * size
    return {"bytes": read + rows * case["cols"] * size + record + rows * (12 if case["rest"] else 8),
            "flops": (10 if case["hard"] and case["temperature"] != 1.0 else 6) * rows * case["vocab"]}


# ---------------------------------------------------------------- the definitions in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    return {"distill": _exact_distill, "top": _exact_top, "balance": _exact_balance}[case["op"]](s, case)


def _exact_distill(s, c):
    T, rows, vocab = c["temperature"], c["rows"], c["vocab"]
    valid = s["targets"] >= 0
    count = int(valid.sum())
    dlogits = torch.zeros(rows, c["cols"], dtype=torch.float64, device=valid.device)
    losses = torch.zeros(rows, dtype=torch.float64, device=valid.device)
    for at in range(0, rows, 512):
        part = slice(at, min(rows, at + 512))
        z = s["logits"][part, :vocab].double()
        index = s["indices"][part].long()
        # the teacher's distribution over its listed tokens and one more outcome: all the others
        t = s["values"][part].double() / T
        norm = s["lse"][part].double() if c["rest"] else torch.logsumexp(t, dim=1)
        p = torch.exp(t - norm[:, None])
        log_z = torch.logsumexp(z / T, dim=1, keepdim=True)
        q = torch.exp(z / T - log_z)
        listed_ = torch.zeros_like(z, dtype=torch.bool).scatter_(1, index, True)
        target = torch.zeros_like(z).scatter_(1, index, p)      # d loss / d(z/T) = q - (target mass seen by each token)
        loss = (torch.xlogy(p, p) - p * (z.gather(1, index) / T - log_z)).sum(1)
        if c["rest"]:
            rest = (1.0 - p.sum(1)).clamp(min=0.0)
            others = torch.where(listed_, torch.full_like(z, -math.inf), z / T)
            log_others = torch.logsumexp(others, dim=1)
            loss = loss + torch.xlogy(rest, rest) - rest * (log_others - log_z[:, 0])
            target = target + rest[:, None] * torch.exp(others - log_others[:, None])
        else:
            rest = 0.0
        mass = p.sum(1, keepdim=True) + (rest[:, None] if c["rest"] else 0.0)
        grad = T * T * (mass * q - target) / T
        loss = T * T * loss
        if c["hard"]:
            label = s["targets"][part].long().clamp(min=0)[:, None]
            log_1 = torch.logsumexp(z, dim=1, keepdim=True)
            loss = loss + c["hard"] * (log_1 - z.gather(1, label))[:, 0]
            grad = grad + c["hard"] * (torch.exp(z - log_1) - torch.zeros_like(z).scatter_(1, label, 1.0))
        ok = valid[part]
        dlogits[part, :vocab] = torch.where(ok[:, None], grad * (_loss_scale(c) / max(1, count)), torch.zeros_like(grad))
        losses[part] = torch.where(ok, loss, torch.zeros_like(loss))
    return {"dlogits": dlogits, "row_loss": losses, "loss": (losses.sum() / max(1, count)).reshape(1),
            "n_valid": valid.sum().to(torch.int32).reshape(1)}


def _exact_top(s, c):
    lse = torch.empty(c["rows"], dtype=torch.float64, device=s["logits"].device)
    for at in range(0, c["rows"], 512):
        lse[at:at + 512] = torch.logsumexp(s["logits"][at:at + 512, :c["vocab"]].double() / c["temperature"], dim=1)
    return {"values": None, "indices": None, "lse": lse}


def _exact_balance(s, c):
    z = s["logits"].double()
    valid = s["targets"] >= 0
    n = max(1, int(valid.sum()))
    chosen = s["experts"][valid]
    counts = torch.bincount(chosen[chosen >= 0].long(), minlength=c["experts"])
    share = counts.double() / (n * c["k"])
    p = torch.exp(z - torch.logsumexp(z, dim=1, keepdim=True)) * valid[:, None]
    mean = p.sum(0) / n
    loss = 0.01 * c["experts"] * torch.dot(share, mean)
    grad = 0.01 * c["experts"] / n * _loss_scale(c) * p * (share[None, :] - torch.mv(p, share)[:, None])
    return {"dlogits": grad, "counts": counts.to(torch.int32), "loss": loss.reshape(1)}
