"""Plain 64-bit forms of the int8 paged cache's operators, and caches to try them on (CPU torch).

EPS is half a step of f32: a rounding moves a value by at most that much of itself. The bounds returned beside the values count
roundings along the longest chain of a plain summation, so they hold for any order of it."""
import math

import torch

EPS = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}


class Cache:
    """Codes and scales of `slots` slots, tables in a shuffled order; `spare` blocks more than the sequences need."""

    def __init__(self, g, batch, max_blocks, bs, nkv, hd, spare=1):
        nblk = batch * max_blocks + spare
        self.bs, self.nkv, self.hd, self.slots = bs, nkv, hd, nblk * bs
        self.codes = [torch.randint(-127, 128, (self.slots, nkv, hd), generator=g, dtype=torch.int8) for _ in "kv"]
        self.scales = [(torch.rand(self.slots, nkv, generator=g) + 0.2) / 60 for _ in "kv"]
        order = torch.randperm(nblk, generator=g)
        self.table = order[: batch * max_blocks].view(batch, max_blocks).to(torch.int32).contiguous()
        self.free = order[batch * max_blocks:].to(torch.int32)

    def slot(self, b, j, table=None):
        """Slot of position j, or -1."""
        t = self.table if table is None else table
        if j // self.bs >= t.shape[1]:
            return -1
        s = (int(t[b, j // self.bs]) & 0xFFFFFFFF) * self.bs + j % self.bs
        return s if s < self.slots else -1

    def words(self, which):
        return self.codes[which].contiguous().view(torch.int32).view(self.slots, -1)

    def kv(self, ops, dev):
        """The cache on the GPU."""
        return ops.PagedKV8(self.words(0).to(dev), self.words(1).to(dev), self.scales[0].to(dev), self.scales[1].to(dev),
                            self.table.to(dev), self.bs, self.hd)


def turn(x, w, eps, pos, freq):
    """RMSNorm and rotation of [rows, heads, hd] in 64 bits, and a bound on the error of 32-bit arithmetic."""
    x = x.double()
    hd, half = x.shape[-1], freq.numel()
    n = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * w.double() if w is not None else x
    a = pos.double()[:, None, None] * freq.double()
    c, s = a.cos(), a.sin()
    lo, hi, rest = n[..., :half], n[..., half:2 * half], n[..., 2 * half:]
    # The norm: hd + 1 products and sums at half weight (a root), the root, a division, two products. The rotation: cos and
    # sin to 8 half steps of 1 (the angle in turns is f32: 2 pi 2^-25, and their own error), two products, a sum.
    rel = (hd / 2 + 8) * EPS if w is not None else 0.0
    size = lo.abs() + hi.abs()
    bound = torch.cat([size * (rel + 12 * EPS), size * (rel + 12 * EPS), rest.abs() * rel], -1)
    return torch.cat([lo * c - hi * s, hi * c + lo * s, rest], -1), bound


def chunk_rows(start, lens, b):
    """[(row, the number of keys that it sees)] of sequence b."""
    r0, r1 = int(start[b]), int(start[b + 1])
    return [(r, max(0, int(lens[b]) - (r1 - r))) if int(lens[b]) < r1 - r else (r, int(lens[b]) - (r1 - r) + 1)
            for r in range(r0, r1)]


def scores(c, q, start, lens, b, h, scale):
    """(rows, [rows, keys] scores with -inf where unseen, their error bound, the keys' slots) of a sequence and query head."""
    group = q.shape[1] // c.nkv
    rows = chunk_rows(start, lens, b)
    slots = [c.slot(b, j) for j in range(int(lens[b]))]
    at = torch.tensor([max(s, 0) for s in slots], dtype=torch.long)
    k = c.codes[0][at, h // group].double() * c.scales[0][at, h // group].double()[:, None]
    qd = q[[r for r, _ in rows], h].double() if rows else torch.zeros(0, c.hd, dtype=torch.float64)
    s = qd @ k.t() * scale
    bound = (c.hd + 6) * EPS * (qd.abs() @ k.abs().t() * abs(scale))
    seen = torch.arange(len(slots))[None] < torch.tensor([n for _, n in rows], dtype=torch.long)[:, None]
    seen = seen & torch.tensor([x >= 0 for x in slots], dtype=torch.bool)[None]
    return [r for r, _ in rows], s.masked_fill(~seen, -math.inf), bound.masked_fill(~seen, 0.0), torch.tensor(slots, dtype=torch.long)


def attention(c, q, start, lens, scale):
    """(out, lse, their bounds) of all rows, 64 bits; rows of no sequence are NaN."""
    rows, nh, hd = q.shape
    out = torch.full((rows, nh, hd), math.nan, dtype=torch.float64)
    lse = torch.full((rows, nh), math.nan, dtype=torch.float64)
    ob, lb = torch.zeros_like(out), torch.zeros_like(lse)
    w_half = 0.0 if q.dtype == torch.float32 else HALF[q.dtype]  # the weights' own rounding
    for b in range(len(lens)):
        for h in range(nh):
            at_rows, s, e, at = scores(c, q, start, lens, b, h, scale)
            if not at_rows:
                continue
            top = s.amax(1) if s.shape[1] else torch.full((len(at_rows),), -math.inf, dtype=torch.float64)
            none = top == -math.inf
            p = (s - torch.where(none, 0.0, top)[:, None]).exp()
            total = p.sum(1)
            p = p / torch.where(none, 1.0, total)[:, None]
            v = c.codes[1][at, h * c.nkv // nh].double() * c.scales[1][at, h * c.nkv // nh].double()[:, None]
            v[at < 0] = 0.0  # a key without a slot has no value
            n = s.shape[1]
            # A weight: the score's error, the exponential's (2 steps, and a step of its argument, at most 150).
            far = torch.where(s == -math.inf, 0.0, (top[:, None] - s)).clamp_max(150.0)
            err = (e + e.amax(1, keepdim=True) if n else e) + (8 + 2 * far) * EPS
            rel = ((p * err).sum(1) + (n + 16) * EPS)[:, None]  # of the sums, top and bottom
            out[at_rows, h] = p @ v
            ob[at_rows, h] = (p * (err + w_half)) @ v.abs() + (rel + (n + 16) * EPS) * (p @ v.abs()) + HALF[q.dtype] * (p @ v).abs()
            lse[at_rows, h] = torch.where(none, -math.inf, top + total.log())
            lb[at_rows, h] = rel[:, 0] + 4 * EPS * torch.where(none, 0.0, lse[at_rows, h].abs() + top.abs())
    return out, lse, ob, lb


def weight_sums(c, q, lse, start, lens, scale, acc):
    """(acc after the call, its bound)."""
    new, bound = acc.double().clone(), torch.zeros_like(acc, dtype=torch.float64)
    group = q.shape[1] // c.nkv
    for b in range(len(lens)):
        n = int(start[b + 1] - start[b])
        t = min(int(lens[b]), acc.shape[2])
        for kvh in range(c.nkv):
            new[b, kvh, max(0, int(lens[b]) - n):t] = 0.0
            before = new[b, kvh, :t].clone()
            for h in range(kvh * group, (kvh + 1) * group):
                rows, s, e, _ = scores(c, q, start, lens, b, h, scale)
                if rows and t:
                    given = lse[rows, h].double()[:, None]
                    p = torch.where(s == -math.inf, 0.0, (s - given).exp())
                    size = torch.where(s == -math.inf, 0.0, s.abs() + given.abs()).clamp_max(1e6)
                    new[b, kvh, :t] += p.sum(0)[:t]
                    bound[b, kvh, :t] += (p * (e + (8 + 3 * size) * EPS)).sum(0)[:t]
            # the sums of rows and heads, and the last one onto acc
            bound[b, kvh, :t] += (n * group + 2) * EPS * (new[b, kvh, :t] - before).abs() + EPS * new[b, kvh, :t].abs()
    return new, bound


def evict(lens, acc, budget, sink, recent):
    """(keep, new_lens) as the operator gives them."""
    batch, nkv = acc.shape[:2]
    keep = torch.full((batch, nkv, budget), -1, dtype=torch.int32)
    new = []
    for b in range(batch):
        t = min(int(lens[b]), acc.shape[2])
        new.append(min(t, budget))
        for h in range(nkv):
            at = list(range(t))
            if t > budget:
                w = [-math.inf if math.isnan(v) else v for v in acc[b, h, :t].tolist()]
                middle = sorted(range(sink, t - recent), key=lambda j: (-w[j], j))
                at = sorted(list(range(sink)) + middle[: budget - sink - recent] + list(range(t - recent, t)))
            keep[b, h, : len(at)] = torch.tensor(at, dtype=torch.int32)
    return keep, torch.tensor(new, dtype=torch.int32)


def starts(rows):
    s = [0]
    for n in rows:
        s.append(s[-1] + n)
    return torch.tensor(s, dtype=torch.int32)
