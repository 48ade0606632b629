"""The operators of a token's life in the int8 paged KV cache, as cases that can be timed and checked.

A case is a dict of plain values; `prepare` makes what a serving program holds before the call, `run` is one pass through an
operator (the plain form in 32-bit torch, or with `own` the library's), `exact` the same outputs in 64 bits.

Kinds
  rope    per-head RMSNorm of queries and keys and their rotation (ops.qk_norm_rope)
  append  the same, and the rotated keys and the values into the int8 paged cache (ops.qk_norm_rope_append_i8)
  attend  attention of every sequence's new tokens over its cached keys (ops.paged_attention_i8)
  sums    the attention weight that each cached key has received, accumulated (ops.paged_weight_sums_i8)
  evict   the lightest entries of too long sequences leave the cache (ops.paged_kv_evict_i8)

A batch is ragged: sequence b has the rows row_start[b] .. row_start[b + 1] of the activations, the last ones of its
seq_lens[b] cached positions. How long each sequence and its chunk are follows from the case alone; the seed makes the values.
"""
import math
import random

import torch

own = False

EPS = 1e-6
THETA = 1.0e6


def listed():
    return [
        # One layer's queries and keys of one decoding sequence: launch and latency.
        dict(name="rope_step", kind="rope", rows=1, heads=16, kv_heads=8, head_dim=128, dtype="f32"),
        # The same of a long prompt, bf16 activations: memory traffic.
        dict(name="rope_prompt", kind="rope", rows=8192, heads=32, kv_heads=8, head_dim=128, dtype="bf16"),
        # A decode step of 33 sequences, heads of 64: each appends one token.
        dict(name="append_steps", kind="append", batch=33, chunk=1, ctx=700, heads=8, kv_heads=8, head_dim=64, block=16,
             dtype="f32"),
        # The next prompt pieces of four sequences, up to 2048 tokens each.
        dict(name="append_chunks", kind="append", batch=4, chunk=2048, ctx=4096, heads=16, kv_heads=8, head_dim=128,
             block=32, dtype="bf16"),
        # A single decoding sequence of 2000 tokens: few heads for many compute units.
        dict(name="attend_step", kind="attend", batch=1, chunk=1, ctx=2000, heads=16, kv_heads=8, head_dim=128, block=32,
             dtype="f32"),
        # A full server's decode step: 64 sequences of up to 8192 tokens, a stream of the cache.
        dict(name="attend_steps_64", kind="attend", batch=64, chunk=1, ctx=8192, heads=32, kv_heads=8, head_dim=128,
             block=32, dtype="bf16"),
        # Prompt pieces, drafts and single tokens of 12 sequences in one batch; seven query heads per kv head.
        dict(name="attend_mixed", kind="attend", batch=12, chunk=511, ctx=4000, heads=28, kv_heads=4, head_dim=128,
             block=16, dtype="f32"),
        # The last piece of a 32768-token prompt: matrix products.
        dict(name="attend_chunk", kind="attend", batch=1, chunk=2048, ctx=32768, heads=32, kv_heads=8, head_dim=128,
             block=32, dtype="bf16"),
        # The weights of one decode step of 32 sequences.
        dict(name="sums_steps", kind="sums", batch=32, chunk=1, ctx=4096, heads=16, kv_heads=8, head_dim=128, block=32,
             dtype="f32"),
        # The weights of a prompt piece over 16384 cached tokens.
        dict(name="sums_chunk", kind="sums", batch=1, chunk=1024, ctx=16384, heads=32, kv_heads=8, head_dim=128, block=32,
             dtype="bf16"),
        # One sequence a little over its budget.
        dict(name="evict_one", kind="evict", batch=1, ctx=1111, budget=700, sink=4, recent=100, kv_heads=8, head_dim=64,
             block=16),
        # Sixteen sequences of up to 8192 tokens cut to 2048.
        dict(name="evict_batch", kind="evict", batch=16, ctx=8192, budget=2048, sink=4, recent=512, kv_heads=8,
             head_dim=128, block=32),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["rope", "append", "attend", "attend", "attend", "sums", "sums", "evict"])
    heads, kv_heads, head_dim = rng.choice([(16, 8, 128), (16, 8, 128), (32, 8, 128), (8, 8, 64), (28, 4, 128), (9, 3, 64)])
    c = dict(kind=kind, heads=heads, kv_heads=kv_heads, head_dim=head_dim, dtype=rng.choice(["f32", "bf16"]))
    if kind == "rope":
        return dict(c, rows=_log(rng, 1, 8192))
    c.update(batch=_log(rng, 1, 64), block=rng.choice([1, 16, 16, 24, 32, 32, 64, 256]))
    if kind == "evict":
        del c["heads"], c["dtype"]
        c["batch"] = _log(rng, 1, 16)
        ctx = _log(rng, 64, 8192)
        budget = rng.randint(16, ctx)
        return dict(c, ctx=ctx, budget=budget, sink=rng.choice([0, 1, 4]), recent=rng.randint(0, budget // 2))
    # A step of one token, a draft, or a piece of a prompt: all the batch's rows are at most 8192.
    chunk = rng.choice([1, 1, _log(rng, 2, 16), _log(rng, 16, 2048)])
    if chunk > 16:
        c["batch"] = min(c["batch"], 8192 // chunk, 16)
    # As many keys as the longest listed batch has, and as many products as the largest listed case.
    most = min(32768, 64 * 8192 // c["batch"], 2 ** 27 // (c["batch"] * heads * chunk // 16 + 1))
    return dict(c, chunk=chunk, ctx=_log(rng, max(chunk, 16), max(chunk, 16, most)))


# ------------------------------------------------------------------ inputs


def _gen(seed, salt=0):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 1000003 + salt)
    return g


def _randn(g, *shape):
    return torch.randn(*shape, device="cuda", generator=g)


def _dtype(c):
    return torch.bfloat16 if c["dtype"] == "bf16" else torch.float32


def _lengths(c):
    """Each sequence's cached length and the rows of its chunk; the first sequence has the longest of both."""
    rng = random.Random("%d %d %d" % (c["batch"], c["ctx"], c.get("chunk", 1)))
    lens = [c["ctx"]] + [rng.randint(max(1, c["ctx"] // 2), c["ctx"]) for _ in range(c["batch"] - 1)]
    chunk = c.get("chunk", 1)
    rows = [chunk] + [min(n, _log(rng, 1, chunk)) for n in lens[1:]]
    return lens, rows


def _tables(c, g, nblk, at, count):
    """`count` blocks for each sequence from `at` on, in an order of their own."""
    order = torch.randperm(c["batch"] * count, device="cuda", generator=g).to(torch.int32) + at
    return order.view(c["batch"], count).contiguous()


def _ints(v):
    return torch.tensor(v, device="cuda", dtype=torch.int32)


def _cache(c, g, more=0):
    """Keys and values as a decoder leaves them: int8 codes with one scale for each token and head, `more` spare blocks for
    each sequence behind them."""
    bs, nkv, hd = c["block"], c["kv_heads"], c["head_dim"]
    per = -(-c["ctx"] // bs)
    slots = c["batch"] * (per + more) * bs
    pool = torch.empty(2, slots, nkv * hd // 4, device="cuda", dtype=torch.int32)
    scales = torch.empty(2, slots, nkv, device="cuda")
    for i in range(2):
        x = _randn(g, slots, nkv, hd) * (1.0 if i == 0 else 0.5)
        scales[i] = x.abs().amax(-1) / 127
        pool[i] = (x / scales[i][..., None]).round().clamp(-127, 127).to(torch.int8).view(torch.int32).view(slots, -1)
    lens, rows = _lengths(c)
    start = [0]
    for n in rows:
        start.append(start[-1] + n)
    return dict(c=c, pool=pool, scales=scales, table=_tables(c, g, per, 0, per), lens=_ints(lens), start=_ints(start),
                rows=start[-1], most=max(rows), longest=max(lens))


def _qkv(c, g, rows):
    """Rows of the joined projection, as one linear writes them: queries, keys and values of a row side by side."""
    nh, nkv, hd = c["heads"], c["kv_heads"], c["head_dim"]
    x = _randn(g, rows, (nh + 2 * nkv) * hd).to(_dtype(c))
    q, k, v = x[:, : nh * hd], x[:, nh * hd: (nh + nkv) * hd], x[:, (nh + nkv) * hd:]
    return dict(q=q.unflatten(1, (nh, hd)), k=k.unflatten(1, (nkv, hd)), v=v.unflatten(1, (nkv, hd)),
                qw=1.0 + 0.2 * _randn(g, hd), kw=1.0 + 0.2 * _randn(g, hd),
                freq=THETA ** (-torch.arange(0, hd, 2, device="cuda", dtype=torch.float64) / hd))


def _slots(s):
    """The cache slot of each row, and its sequence."""
    c, start = s["c"], s["start"].long()
    r = torch.arange(s["rows"], device="cuda")
    b = torch.searchsorted(start, r, right=True) - 1
    at = s["lens"].long()[b] - (start[b + 1] - r)
    return s["table"].long()[b, at // c["block"]] * c["block"] + at % c["block"], at


def _heavy(g, *shape):
    """Accumulated weights: a few keys have most of it."""
    return torch.exp(2.0 * _randn(g, *shape))


def prepare(case, seed):
    c, g = dict(case), _gen(seed)
    if c["kind"] == "rope":
        s = dict(_qkv(c, g, c["rows"]), c=c)
        s["pos"] = torch.randint(0, 131072, (c["rows"],), device="cuda", generator=g).to(torch.int32)
        return s
    if c["kind"] == "evict":
        more = -(-c["budget"] // c["block"])
        s = _cache(c, g, more)
        s["to"] = _tables(c, g, more, s["table"].numel(), more)
        s["acc"] = _heavy(g, c["batch"], c["kv_heads"], c["ctx"])
        s["kept"] = torch.zeros(c["batch"], c["kv_heads"], c["budget"], device="cuda")
        return s
    s = _cache(c, g)
    if c["kind"] == "append":
        s.update(_qkv(c, g, s["rows"]))
        s["slot"], at = _slots(s)
        s["pos"] = at.to(torch.int32)
        s["clip"] = 4.0 + torch.rand(2, c["kv_heads"], device="cuda", generator=g)
        return s
    s["q"] = (1.5 * _randn(g, s["rows"], c["heads"], c["head_dim"])).to(_dtype(c))
    if c["kind"] == "sums":
        s["lse"] = _plain_attend(s)[1]
        # A few earlier chunks' weights.
        s["acc"] = _heavy(g, c["batch"], c["kv_heads"], c["ctx"]) * (c["heads"] // c["kv_heads"] * c["chunk"] / c["ctx"])
    return s


# ------------------------------------------------------------------ the plain forms


def _norm_rope(x, w, pos, freq):
    """[rows, heads, hd]: the head's RMSNorm, then the rotation of the pairs (i, i + hd / 2)."""
    x = x.float()
    x = x * (x.square().mean(-1, keepdim=True) + EPS).rsqrt() * w
    angle = pos.double()[:, None] * freq
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    a, b = x[..., : freq.numel()], x[..., freq.numel():]
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)


def _plain_rope(s):
    return [_norm_rope(s[n], s[n + "w"], s["pos"], s["freq"]).to(_dtype(s["c"])) for n in "qk"]


def _read_back(s):
    """What the cache now holds at the appended slots: the values that the codes stand for, and the scales. (A code has
    seven bits and a sign, which bf16 holds.)"""
    codes = s["pool"].view(torch.int8).unflatten(2, (s["c"]["kv_heads"], -1))[:, s["slot"]]
    scales = s["scales"][:, s["slot"]]
    return (codes * scales[..., None]).to(torch.bfloat16), scales


def _plain_append(s):
    c = s["c"]
    q, k = _norm_rope(s["q"], s["qw"], s["pos"], s["freq"]), _norm_rope(s["k"], s["kw"], s["pos"], s["freq"])
    x = torch.stack([k, s["v"].float()])
    scale = torch.minimum(x.abs().amax(-1), s["clip"][:, None]) / 127.0
    scale = torch.where(scale == 0, torch.ones_like(scale), scale)
    codes = (x / scale[..., None]).round().clamp(-127, 127).to(torch.int8)
    slot = _slots(s)[0]
    s["pool"][:, slot] = codes.view(torch.int32).flatten(2)
    s["scales"][:, slot] = scale
    return [q.to(_dtype(c)), *_read_back(s)]


def _cached(s, which):
    """[batch, kv_heads, ctx, hd] f32 keys (0) or values (1) of every sequence."""
    c = s["c"]
    at = torch.arange(c["ctx"], device="cuda")
    slot = s["table"].long()[:, at // c["block"]] * c["block"] + at % c["block"]
    x = s["pool"][which].view(torch.int8).unflatten(1, (c["kv_heads"], -1))[slot].float()
    return (x * s["scales"][which][slot][..., None]).transpose(1, 2).contiguous()


def _scores(s):
    """[batch, kv_heads, chunk, group, ctx] scores, -inf where a row does not see a key or there is no row; where each row of
    the batch is."""
    c = s["c"]
    nkv, group, hd, n, t = c["kv_heads"], c["heads"] // c["kv_heads"], c["head_dim"], s["most"], c["ctx"]
    start = s["start"].long()
    count, i = start[1:] - start[:-1], torch.arange(n, device="cuda")
    q = s["q"].float()[(start[:-1, None] + i).clamp_max(s["rows"] - 1)]
    q = q.view(-1, n, nkv, group, hd).permute(0, 2, 1, 3, 4).reshape(-1, nkv, n * group, hd)
    sc = torch.matmul(q, _cached(s, 0).transpose(2, 3)).mul_(hd ** -0.5).view(-1, nkv, n, group, t)
    last = torch.where(i < count[:, None], s["lens"].long()[:, None] - count[:, None] + i, -1)
    sc.masked_fill_((torch.arange(t, device="cuda") > last[..., None])[:, None, :, None], -math.inf)
    r = torch.arange(s["rows"], device="cuda")
    b = torch.searchsorted(start, r, right=True) - 1
    return sc, b, r - start[b]


def _plain_attend(s):
    c = s["c"]
    sc, b, i = _scores(s)
    top = sc.amax(-1, keepdim=True)
    top = torch.where(top > -math.inf, top, torch.zeros_like(top))
    p = sc.sub_(top).exp_()
    total = p.sum(-1)
    out = torch.matmul(p.flatten(2, 3), _cached(s, 1)).view(*p.shape[:4], -1)
    out = out / torch.where(total > 0, total, torch.ones_like(total))[..., None]
    lse = top[..., 0] + total.log()
    out, lse = out.transpose(1, 2)[b, i], lse.transpose(1, 2)[b, i]
    return [out.flatten(1, 2).to(_dtype(c)), lse.flatten(1)]


def _plain_sums(s):
    sc, b, i = _scores(s)
    lse = torch.zeros(*sc.shape[:4], device="cuda").transpose(1, 2)
    lse[b, i] = s["lse"].unflatten(1, lse.shape[2:])
    p = sc.sub_(lse.transpose(1, 2)[..., None]).exp_().sum((2, 3))
    count = (s["start"][1:] - s["start"][:-1])[:, None, None]
    at, lens = torch.arange(s["c"]["ctx"], device="cuda"), s["lens"][:, None, None]
    s["acc"].copy_(torch.where(at < lens - count, s["acc"] + p, torch.where(at < lens, p, s["acc"])))
    return [s["acc"]]


def _plain_evict(s):
    c = s["c"]
    nkv, bs, budget, t = c["kv_heads"], c["block"], c["budget"], c["ctx"]
    at, lens = torch.arange(t, device="cuda"), s["lens"].long()[:, None, None]
    rank = torch.where((at < c["sink"]) | (at >= lens - c["recent"]), math.inf, s["acc"])
    rank = torch.where(at < lens, rank, -math.inf)
    # Where all are kept, the places behind the sequence come last.
    keep = rank.sort(dim=-1, descending=True, stable=True).indices[..., :budget]
    keep = torch.where(keep < lens, keep, t).sort(-1).values
    live = keep < t
    b = torch.arange(c["batch"], device="cuda")[:, None, None]
    src = keep.clamp_max(t - 1)
    to = torch.arange(budget, device="cuda")
    src = s["table"].long()[b, src // bs] * bs + src % bs
    dst = (s["to"].long()[:, to // bs] * bs + to % bs)[:, None]
    h = torch.arange(nkv, device="cuda")[:, None]
    codes = s["pool"].unflatten(2, (nkv, -1))
    codes[:, dst, h] = torch.where(live[..., None], codes[:, src, h], codes[:, dst, h])
    s["scales"][:, dst, h] = torch.where(live, s["scales"][:, src, h], s["scales"][:, dst, h])
    s["kept"].copy_(torch.where(live, s["acc"].gather(2, keep.clamp_max(t - 1)), s["kept"]))
    new = s["lens"].clamp_max(budget)
    return [torch.where(live, keep, -1).to(torch.int32), new, s["kept"], s["pool"], s["scales"]]


# ------------------------------------------------------------------ the library's


def _kv(s):
    """The cache as the library takes it; a program makes it once."""
    from brain_amd import ops

    if "kv" not in s:
        c = s["c"]
        s["kv"] = ops.PagedKV8(s["pool"][0], s["pool"][1], s["scales"][0], s["scales"][1], s["table"], c["block"],
                               c["head_dim"])
    return s["kv"]


def _own_rope(s):
    from brain_amd import ops

    return ops.qk_norm_rope(s["q"], s["k"], s["pos"], s["freq"], s["qw"], s["kw"], eps=EPS)


def _own_append(s):
    from brain_amd import ops

    q = ops.qk_norm_rope_append_i8(s["q"], s["k"], s["v"], s["pos"], s["freq"], _kv(s), s["lens"], s["start"],
                                   s["qw"], s["kw"], eps=EPS, k_clip=s["clip"][0], v_clip=s["clip"][1])
    return [q, *_read_back(s)]


def _own_attend(s):
    from brain_amd import ops

    return ops.paged_attention_i8(s["q"], _kv(s), s["lens"], s["start"], max_rows=s["most"], max_len=s["longest"])


def _own_sums(s):
    from brain_amd import ops

    return [ops.paged_weight_sums_i8(s["q"], s["lse"], _kv(s), s["lens"], s["acc"], s["start"], max_rows=s["most"],
                                     max_len=s["longest"])]


def _own_evict(s):
    from brain_amd import ops

    c = s["c"]
    keep, new = ops.paged_kv_evict_i8(_kv(s), s["lens"], s["acc"], c["budget"], sink=c["sink"], recent=c["recent"],
                                      out_tables=s["to"], acc_out=s["kept"])
    return [keep, new, s["kept"], s["pool"], s["scales"]]


def run(state):
    kind = state["c"]["kind"]
    if own:
        return dict(rope=_own_rope, append=_own_append, attend=_own_attend, sums=_own_sums, evict=_own_evict)[kind](state)
    return dict(rope=_plain_rope, append=_plain_append, attend=_plain_attend, sums=_plain_sums,
                evict=_plain_evict)[kind](state)


# ------------------------------------------------------------------ 64 bits


def _turned(x, w, pos, freq):
    """The norm and the rotation as complex numbers, 64 bits."""
    x = x.double()
    x = x / (x.pow(2).sum(-1, keepdim=True) / x.shape[-1] + EPS).sqrt() * w.double()
    half = freq.numel()
    z = torch.complex(x[..., :half], x[..., half:])
    angle = pos.double()[:, None, None] * freq
    z = z * torch.polar(torch.ones_like(angle), angle)
    return torch.cat([z.real, z.imag], -1)


def _sequence(s, b):
    """Positions' slots, and rows, of one sequence."""
    bs, lens = s["c"]["block"], int(s["lens"][b])
    at = torch.arange(lens, device="cuda")
    return s["table"][b].long()[at // bs] * bs + at % bs, range(int(s["start"][b]), int(s["start"][b + 1]))


def _values(s, which, slot, h):
    c = s["c"]
    codes = s["pool"][which].view(torch.int8).view(-1, c["kv_heads"], c["head_dim"])[slot, h]
    return codes.double() * s["scales"][which][slot, h].double()[:, None]


def _weights(s, b, h, slot, rows):
    """Scores [group, rows, keys] of one sequence and kv head."""
    c = s["c"]
    group, n, t = c["heads"] // c["kv_heads"], len(rows), slot.numel()
    q = s["q"][rows.start:rows.stop, h * group:(h + 1) * group].double().transpose(0, 1)
    sc = (q.reshape(group * n, -1) @ _values(s, 0, slot, h).t()).view(group, n, t) / math.sqrt(c["head_dim"])
    seen = torch.arange(t, device="cuda")[None] <= torch.arange(t - n, t, device="cuda")[:, None]
    return sc.masked_fill_(~seen, -math.inf)


def exact(case, seed):
    s = prepare(case, seed)
    c = s["c"]
    kind, nkv = c["kind"], c["kv_heads"]
    if kind == "rope":
        return [_turned(s[n], s[n + "w"], s["pos"], s["freq"]) for n in "qk"]
    if kind == "append":
        q, k = (_turned(s[n], s[n + "w"], s["pos"], s["freq"]) for n in "qk")
        held, scales = [], []
        for x, clip in ((k, s["clip"][0]), (s["v"].double(), s["clip"][1])):
            sc = torch.minimum(x.abs().amax(-1), clip.double()) / 127
            held.append((x / sc[..., None]).round().clamp(-127, 127) * sc[..., None])
            scales.append(sc)
        return [q, torch.stack(held), torch.stack(scales)]
    if kind == "evict":
        kept = torch.zeros_like(s["kept"], dtype=torch.float64)
        for b, t in enumerate(s["lens"].tolist()):
            for h in range(nkv):
                w = s["acc"][b, h, :t].double().tolist()
                middle = sorted(range(c["sink"], max(c["sink"], t - c["recent"])), key=lambda j: (-w[j], j))
                gone = set(middle[len(middle) - max(0, t - c["budget"]):]) if t > c["budget"] else set()
                left = [w[j] for j in range(t) if j not in gone]
                kept[b, h, :len(left)] = torch.tensor(left, dtype=torch.float64)
        return [None, None, kept, None, None]
    group = c["heads"] // nkv
    out = torch.zeros(s["rows"], nkv, group, c["head_dim"], device="cuda", dtype=torch.float64)
    lse = torch.zeros(s["rows"], nkv, group, device="cuda", dtype=torch.float64)
    acc = s["acc"].double() if kind == "sums" else None
    for b in range(c["batch"]):
        slot, rows = _sequence(s, b)
        for h in range(nkv):
            sc = _weights(s, b, h, slot, rows)
            if kind == "sums":
                given = s["lse"][rows.start:rows.stop, h * group:(h + 1) * group].double().t()
                t, n = slot.numel(), len(rows)
                acc[b, h, t - n:t] = 0
                acc[b, h, :t] += (sc - given[..., None]).exp_().sum((0, 1))
                continue
            lse[rows.start:rows.stop, h] = sc.logsumexp(-1).t()
            p = sc.sub_(lse[rows.start:rows.stop, h].t()[..., None]).exp_()
            o = p.flatten(0, 1) @ _values(s, 1, slot, h)
            out[rows.start:rows.stop, h] = o.view(group, len(rows), -1).transpose(0, 1)
    return [acc] if kind == "sums" else [out.flatten(1, 2), lse.flatten(1)]


# ------------------------------------------------------------------ what a pass cannot do without


def work(case):
    c, kind, nkv, hd = case, case["kind"], case["kv_heads"], case["head_dim"]
    e = 2 if c.get("dtype") == "bf16" else 4
    if kind == "rope":
        elems = c["rows"] * (c["heads"] + nkv) * hd
        return dict(bytes=2 * e * elems + 4 * c["rows"] + 12 * hd, flops=10 * elems)
    lens, rows = _lengths(c)
    entry = nkv * (hd + 4)  # one token's codes and scales, keys or values
    if kind == "append":
        n = sum(rows)
        return dict(bytes=n * (e * (2 * c["heads"] + 2 * nkv) * hd + 2 * entry + 8), flops=12 * n * (c["heads"] + 2 * nkv) * hd)
    if kind == "evict":
        kept = sum(min(t, c["budget"]) for t in lens)
        return dict(bytes=4 * nkv * sum(lens) + kept * (4 * entry + 8 * nkv), flops=0)
    pairs = sum(n * (t - n) + n * (n + 1) // 2 for t, n in zip(lens, rows)) * c["heads"]
    each = sum(rows) * c["heads"]
    table = 4 * sum(-(-t // c["block"]) for t in lens)
    if kind == "sums":
        return dict(bytes=sum(lens) * (entry + 8 * nkv) + each * (e * hd + 4) + table, flops=2 * hd * pairs)
    return dict(bytes=sum(lens) * 2 * entry + each * (2 * e * hd + 4) + table, flops=4 * hd * pairs)
