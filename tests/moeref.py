"""Plain implementations of the mixture-of-experts operators for their tests: numpy and torch on the CPU, 64 bits, or the
32-bit arithmetic that a result has to equal bit for bit."""
import math

import numpy as np
import torch

HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}  # a rounding's most, relative


def route(logits, top_k, score="softmax", renormalize=True, scale=1.0, mask=None):
    """(weights f64, experts) of [tokens, n_experts] logits, an expert at a time."""
    x = logits.double().cpu().numpy()
    tokens, n = x.shape
    weights, experts = np.zeros((tokens, top_k)), np.full((tokens, top_k), -1)
    for t in range(tokens):
        if mask is not None and not bool(mask[t]):
            continue
        row = np.where(np.isnan(x[t]), -np.inf, x[t])
        order = sorted(range(n), key=lambda e: (-row[e], e))[:top_k]
        order = [e for e in order if row[e] > -np.inf]
        if not order:
            continue
        top = row[order[0]]
        if score == "softmax":
            part = np.array([1.0 if v == top else math.exp(v - top) for v in row])
            total = part[order].sum() if renormalize else part.sum()
            w = part[order] / total
        else:
            # log sigma(v) = min(v, 0) - log(1 + exp(-|v|)): sums of far negative ones stay sums
            logs = np.array([min(row[e], 0.0) - math.log1p(math.exp(-abs(row[e]))) for e in order])
            w = np.exp(logs - logs.max()) / np.exp(logs - logs.max()).sum() if renormalize else np.exp(logs)
        weights[t, :len(order)], experts[t, :len(order)] = w * scale, order
    return weights, experts


def plan(experts, n_experts, first=0):
    """(offsets, rows, slots) of [tokens, top_k] experts."""
    experts = np.asarray(experts)
    top_k = experts.shape[1]
    flat = experts.reshape(-1).astype(np.int64) - first
    lists = [[i for i in range(flat.size) if flat[i] == e] for e in range(n_experts)] if flat.size * n_experts < 200000 else \
        [np.nonzero(flat == e)[0].tolist() for e in range(n_experts)]
    offsets = np.concatenate([[0], np.cumsum([len(a) for a in lists])])
    places = [i for a in lists for i in a]
    slots = np.full(flat.size, -1)
    slots[places] = np.arange(len(places))
    return offsets, np.array([i // top_k for i in places], dtype=np.int64), slots.reshape(experts.shape)


def sums(xq, wq, offsets, rows, places):
    """Exact sums [places, n] as f64 integers, 0 where a place's row is outside xq; which places are in a group, and which have a
    row."""
    x, w = xq.cpu().view(torch.int8).double(), wq.cpu().view(torch.int8).double()
    acc = torch.zeros(places, w.shape[1], dtype=torch.float64)
    used, there = torch.zeros(places, dtype=torch.bool), torch.zeros(places, dtype=torch.bool)
    row = torch.arange(places) if rows is None else rows.cpu().long()
    group = torch.zeros(places, dtype=torch.long)
    for e in range(w.shape[0]):
        a, b = (min(int(offsets[e + i]), places) for i in (0, 1))
        if a >= b:
            continue
        ok = (row[a:b] >= 0) & (row[a:b] < x.shape[0])
        used[a:b], there[a:b], group[a:b] = True, ok, e
        acc[a:b][ok] = x[row[a:b][ok]] @ w[e].t()
    return acc, used, there, group, torch.where(there, row, 0)


def product(xq, wq, sx, sw, offsets, rows=None, bias=None):
    """The f32 values that a product has to equal bit for bit (its order of roundings), [places, n], and which are in a group."""
    places = xq.shape[0] if rows is None else rows.numel()
    acc, used, there, group, row = sums(xq, wq, offsets, rows, places)
    v = acc.to(torch.int32).float() * sx.cpu()[row][:, None] * sw.cpu()[group]
    if bias is not None:
        v = v + bias.cpu()[group]
    return torch.where(there[:, None], v, torch.zeros(())), used


def glu(v, dtype=torch.float32):
    """silu(gate) * up in 64 bits of f32 products [places, 2 f], and how far an output of `dtype` may be from it: exp's 2 ulp (4 half steps),
    the sum, the quotient and the product a half step each; below exp's range (|gate| > 87) less than |gate * up| 2^-126 is left.
    For bf16, exp(-gate) may be 2^p of a p = -gate log2(e) of 32 bits, log2(e) too: p is then off by a half step for each of the two,
    |p| 2^-24 (1 + 1 / 4) (log2(e) in 32 bits is off by 1.93e-8, under a quarter of 2^-24 of it), which moves 2^p by ln(2) times as
    much, relatively: |gate| 2^-24 (5 / 4). And the result is rounded to bf16."""
    gate, up = v.double().split(v.shape[1] // 2, 1)
    h = gate / (1.0 + torch.exp(-gate)) * up
    tol = 7 * 2.0 ** -24 * h.abs() + (gate * up).abs() * 2.0 ** -126
    if dtype == torch.bfloat16:
        tol = tol + 1.25 * 2.0 ** -24 * gate.abs() * h.abs()
        tol = tol + HALF[dtype] * (h.abs() + tol)
    return h, tol


def combine(y, weights, slots, add=None):
    """The weighted sum in 64 bits, and the sum of magnitudes that its roundings are relative to."""
    y, weights, slots = y.double().cpu(), weights.double().cpu(), slots.cpu().long()
    ok = (slots >= 0) & (slots < y.shape[0])
    part = torch.where(ok[..., None], y[torch.where(ok, slots, 0)] if y.shape[0] else torch.zeros(1), 0.0) * weights[..., None]
    out, size = part.sum(1), part.abs().sum(1)
    if add is not None:
        out, size = out + add.double().cpu(), size + add.double().cpu().abs()
    return out, size
