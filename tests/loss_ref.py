"""The losses in 64 bits on the CPU, row by row from their definitions: what the tests of
cuda_transformer_b200.losses compare with. Nothing here comes from the kernels."""
from __future__ import annotations

import math

import torch

INF = math.inf


def _xlogy(a: float, b: float) -> float:
    return 0.0 if a == 0.0 else (a * math.log(b) if b > 0.0 else -INF * a)


def distill_row(z, label, values, indices, lse, vocab, T, soft, hard):
    """(loss, gradient[vocab], size[vocab]) of one row; z double[>= vocab]; label is None where it does not count for
    the loss; values / indices python lists (empty: no teacher). size is the sum of the magnitudes of the terms
    that each gradient is made of, which rounding errors are relative to."""
    z = z[:vocab]
    nan = torch.full((vocab,), math.nan, dtype=torch.float64)
    listed = {}
    for t, v in zip(values, indices):
        if v >= vocab:
            return math.nan, nan, nan
        if v >= 0:
            listed.setdefault(v, []).append(t / T)
    if hard and label >= vocab:
        return math.nan, nan, nan
    if bool(torch.isnan(z).any()) or float(z.max()) in (INF, -INF):
        return math.nan, nan, nan
    z = z - z.max()     # the distances are what counts: next to the lowest bf16 or fp32 value a logarithm is lost even in 64 bits
    loss, grad, size = 0.0, torch.zeros(vocab, dtype=torch.float64), torch.zeros(vocab, dtype=torch.float64)
    if values and soft:
        x = z / T
        log_z = torch.logsumexp(x, 0)
        q = torch.exp(x - log_z)
        every = [t for ts in listed.values() for t in ts]
        if lse is None:
            norm = float(torch.logsumexp(torch.tensor(every, dtype=torch.float64), 0)) if every else 0.0
            norm = 0.0 if norm == -INF else norm
        else:
            norm = lse
        p = {v: sum(math.exp(t - norm) for t in ts) for v, ts in listed.items()}
        mass = sum(p.values())
        others = torch.ones(vocab, dtype=torch.bool)
        others[list(p)] = False
        has_others = bool(others.any()) and float(x[others].max()) > -INF
        rest = max(0.0, 1.0 - mass) if lse is not None and has_others else 0.0
        kl = sum(_xlogy(m, m) - (m * float(x[v] - log_z) if m > 0.0 else 0.0) for v, m in p.items())
        target = torch.zeros(vocab, dtype=torch.float64)
        for v, m in p.items():
            target[v] = m
        if rest > 0.0:
            kl += rest * (math.log(rest) - float(torch.logsumexp(x[others], 0) - log_z))
            near = x[others] - x[others].max()
            target[others] = rest * torch.exp(near - torch.logsumexp(near, 0))
        loss += soft * kl
        grad += soft / T * ((mass + rest) * q - target)
        size += abs(soft) / T * ((mass + rest) * q + target)
    if hard:
        log_1 = torch.logsumexp(z, 0)
        one = torch.zeros(vocab, dtype=torch.float64)
        one[label] = 1.0
        loss += hard * float(log_1 - z[label])
        grad += hard * (torch.exp(z - log_1) - one)
        size += abs(hard) * (torch.exp(z - log_1) + one)
    return loss, grad, size


def distill(logits, targets, values, indices, lse, vocab, T, soft, hard, loss_scale):
    """All rows: dict of row_loss[rows], loss, n_valid, dlogits[rows, cols], size[rows, cols] (doubles)."""
    rows, cols = logits.shape
    counts = [True] * rows if targets is None else [int(t) >= 0 for t in targets]
    n = sum(counts)
    scale = loss_scale / max(1, n)
    out = {"n_valid": n, "row_loss": torch.zeros(rows, dtype=torch.float64),
           "dlogits": torch.zeros(rows, cols, dtype=torch.float64), "size": torch.zeros(rows, cols, dtype=torch.float64)}
    for i in range(rows):
        if not counts[i]:
            continue
        rec = ([], []) if values is None else ([float(t) for t in values[i]], [int(v) for v in indices[i]])
        loss, grad, size = distill_row(logits[i].double(), None if targets is None else int(targets[i]), *rec,
                                       None if lse is None else float(lse[i]), vocab, T, soft, hard)
        out["row_loss"][i] = loss
        out["dlogits"][i, :vocab] = grad * scale
        out["size"][i, :vocab] = size * scale
    out["loss"] = float(out["row_loss"].sum()) / max(1, n)
    return out


def top(logits, k, vocab, T):
    """(values, indices, lse): python's sort by (NaN first, larger value, lower column)."""
    rows = logits.shape[0]
    values = torch.full((rows, k), -INF, dtype=torch.float64)
    indices = torch.full((rows, k), -1, dtype=torch.int32)
    lse = torch.empty(rows, dtype=torch.float64)
    for i in range(rows):
        z = logits[i, :vocab].double()
        row = z.tolist()
        order = sorted(range(vocab), key=lambda v: (not math.isnan(row[v]), -row[v] if not math.isnan(row[v]) else 0.0, v))
        for j, v in enumerate(order[:k]):
            values[i, j], indices[i, j] = row[v], v
        lse[i] = torch.logsumexp(z / T, 0)
    return values, indices, lse


def balance(logits, chosen, targets, weight, loss_scale):
    rows, experts = logits.shape
    k = chosen.shape[1]
    valid = torch.ones(rows, dtype=torch.bool) if targets is None else targets >= 0
    n = max(1, int(valid.sum()))
    counts = torch.zeros(experts, dtype=torch.int64)
    beyond = False
    for i in range(rows):
        for e in chosen[i].tolist():
            if bool(valid[i]) and e >= 0:
                beyond = beyond or e >= experts
                if e < experts:
                    counts[e] += 1
    share = counts.double() / (n * k)
    if beyond:
        share = share * math.nan
    p = torch.softmax(logits.double(), dim=1) if rows else logits.double()
    p = torch.where(valid[:, None], p, torch.zeros_like(p))
    dot = p @ share
    factor = weight * experts / n
    grad = factor * loss_scale * p * (share[None, :] - dot[:, None])
    size = abs(factor) * loss_scale * p * (share[None, :] + dot[:, None])
    zero = torch.zeros_like(grad)
    return {"counts": counts.to(torch.int32), "loss": factor * float(dot[valid].sum()) if rows else 0.0,
            "dlogits": torch.where(valid[:, None], grad, zero), "size": torch.where(valid[:, None], size, zero)}
