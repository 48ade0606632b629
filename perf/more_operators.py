"""The operators of a sparse mixture of experts on int8 weights, as cases that can be timed and checked.

A case is a dict of plain values; `prepare` makes what a serving program holds before the call, `run` is one pass through an
operator (the plain form in 32-bit torch, or with `own` the library's), `exact` the same outputs in 64 bits.

Kinds
  route    every token's top_k experts, their weights, and the plan: the tokens in the order of their experts (ops.moe_route)
  glu      the gate and up products of every token with its experts and silu(gate) * up, one call for all experts
           (ops.matmul_i8_grouped_glu)
  product  one product of the rows of a plan, each group of rows with its expert's weights (ops.matmul_i8_grouped)
  combine  the weighted sum of each token's expert rows (ops.moe_combine)

A plan has a place for each routed (token, choice): the places of expert e are offsets[e] .. offsets[e + 1], in the order of
the tokens, rows[place] is the token and slots[token, choice] the place (-1: none).

How many rows each expert has follows from the case alone, as uneven as routers leave it; the seed makes the values and says
which expert has which.
"""
import math

import numpy as np
import torch

own = False


def listed():
    return [
        # One decoded token's router: launch and latency.
        dict(name="route_step", kind="route", tokens=1, experts=128, top=8, dtype="f32", score="softmax", masked=False),
        # A padded batch whose last tokens are none, sigmoid scores from a bf16 router.
        dict(name="route_padded", kind="route", tokens=777, experts=60, top=4, dtype="bf16", score="sigmoid", masked=True),
        # The router of a long prompt.
        dict(name="route_prompt", kind="route", tokens=16384, experts=128, top=8, dtype="f32", score="softmax", masked=False),
        # One decoded token through eight small experts of 128: latency, few bytes.
        dict(name="glu_step", kind="glu", tokens=1, experts=128, top=8, k=2048, n=768, dtype="f32", bias=False, masked=False),
        # A decode step of 48 sequences: nearly every expert has a row or a few, a stream of all weights.
        dict(name="glu_steps", kind="glu", tokens=48, experts=128, top=8, k=2048, n=768, dtype="f32", bias=False,
             masked=False),
        # A prompt over many small experts: some 256 rows each.
        dict(name="glu_prompt", kind="glu", tokens=4096, experts=128, top=8, k=2048, n=768, dtype="bf16", bias=False,
             masked=False),
        # A long prompt over few large experts: matrix products.
        dict(name="glu_wide", kind="glu", tokens=8192, experts=8, top=2, k=2048, n=4096, dtype="bf16", bias=False,
             masked=False),
        # The down projection of a decode step.
        dict(name="product_steps", kind="product", tokens=33, experts=128, top=8, k=768, n=2048, dtype="f32", bias=False,
             masked=False),
        # Sizes that no tile divides, with a bias, tokens that are padding.
        dict(name="product_odd", kind="product", tokens=900, experts=7, top=2, k=500, n=333, dtype="f32", bias=True,
             masked=True),
        # The down projection of a prompt.
        dict(name="product_prompt", kind="product", tokens=4096, experts=128, top=8, k=768, n=2048, dtype="bf16", bias=False,
             masked=False),
        # One token's eight expert rows.
        dict(name="combine_step", kind="combine", tokens=1, experts=128, top=8, n=2048, dtype="f32", masked=False, add=True),
        # A prompt's expert rows: memory traffic.
        dict(name="combine_prompt", kind="combine", tokens=8192, experts=128, top=8, n=2048, dtype="bf16", masked=False,
             add=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["route", "glu", "glu", "product", "product", "combine"])
    experts, top, model, ff = rng.choice([(128, 8, 2048, 768), (128, 8, 2048, 768), (64, 6, 2048, 1408), (8, 2, 2048, 4096),
                                          (60, 4, 1024, 1408), (16, 1, 1024, 2048), (7, 2, 500, 332), (256, 8, 1024, 512)])
    c = dict(kind=kind, experts=experts, top=top, dtype=rng.choice(["f32", "bf16"]), masked=rng.random() < 0.25)
    if kind == "route":
        return dict(c, tokens=_log(rng, 1, 16384), score=rng.choice(["softmax", "softmax", "sigmoid"]))
    if kind == "combine":
        return dict(c, tokens=_log(rng, 1, 8192), n=model, add=rng.random() < 0.5)
    # As many products as the largest listed case has, at most.
    c.update(k=model, n=ff) if kind == "glu" else c.update(k=ff, n=model + rng.choice([0, 0, 0, 1]))
    each = top * c["k"] * c["n"] * (2 if kind == "glu" else 1)
    return dict(c, tokens=_log(rng, 1, min(8192, 8192 * 2 * 2048 * 8192 // each)), bias=rng.random() < 0.25)


# ------------------------------------------------------------------ inputs


def _gen(seed, salt=0):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 1000003 + salt)
    return g


def _randn(g, *shape):
    return torch.randn(*shape, device="cuda", generator=g)


def _dtype(c):
    return torch.bfloat16 if c["dtype"] == "bf16" else torch.float32


def _live_tokens(c):
    """How many tokens are real; the others are padding."""
    return c["tokens"] - c["tokens"] // 8 if c["masked"] else c["tokens"]


def _choices(c):
    """[tokens, top] experts as a router leaves them: some are chosen more often. Padding has none (-1)."""
    rng = np.random.default_rng([c["tokens"], c["experts"], c["top"]])
    liked = 0.5 * rng.standard_normal(c["experts"])
    score = (liked + rng.gumbel(size=(c["tokens"], c["experts"]))).astype(np.float32)
    chosen = np.argsort(-score, axis=1, kind="stable")[:, : c["top"]]
    chosen[_live_tokens(c):] = -1
    return chosen


def _padding(c):
    """The mask of a padded batch: true for the tokens that are real."""
    return torch.arange(c["tokens"], device="cuda") < _live_tokens(c)


def _plan(chosen, experts):
    """offsets, rows and slots of [tokens, top] experts, int32; rows behind the last place are -1."""
    flat = chosen.flatten().long()
    key = torch.where(flat >= 0, flat, experts)
    order = key.sort(stable=True).indices
    count = (key[:, None] == torch.arange(experts, device="cuda")).sum(0)
    offsets = torch.cat([count.new_zeros(1), count.cumsum(0)])
    place = torch.empty_like(order)
    place[order] = torch.arange(order.numel(), device="cuda")
    rows = torch.where(torch.arange(order.numel(), device="cuda") < offsets[-1], order // chosen.shape[1], -1)
    slots = torch.where(flat >= 0, place, -1).view_as(chosen)
    return [x.to(torch.int32) for x in (offsets, rows, slots)]


def _codes(g, *shape):
    """int8 codes as a quantizer leaves them: bell-shaped, a row's largest near 127."""
    return (38.0 * _randn(g, *shape)).round_().clamp_(-127, 127).to(torch.int8)


def _words(codes):
    return codes.view(torch.int32)


def prepare(case, seed):
    c, g = dict(case), _gen(seed)
    s = dict(c=c)
    t, top, experts = c["tokens"], c["top"], c["experts"]
    if c["kind"] == "route":
        s["logits"] = (1.5 * _randn(g, t, experts) + 0.5 * _randn(g, experts)).to(_dtype(c))
        s["mask"] = _padding(c) if c["masked"] else None
        # The plan's buffers, which a serving program keeps (a captured step writes them again and again).
        s["plan"] = [torch.full((n,), -1, device="cuda", dtype=torch.int32) for n in (experts + 1, t * top, t * top)]
        s["plan"][2] = s["plan"][2].view(t, top)
        return s
    who = torch.randperm(experts, device="cuda", generator=g)
    chosen = torch.from_numpy(_choices(c)).to("cuda")
    chosen = torch.where(chosen >= 0, who[chosen.clamp_min(0)], -1)
    s["offsets"], s["rows"], s["slots"] = _plan(chosen, experts)
    places = t * top
    if c["kind"] == "combine":
        s["y"] = _randn(g, places, c["n"]).to(_dtype(c))
        s["weights"] = torch.rand(t, top, device="cuda", generator=g)
        s["weights"] /= s["weights"].sum(1, keepdim=True)
        s["add"] = _randn(g, t, c["n"]).to(_dtype(c)) if c["add"] else None
        return s
    wide = 2 * c["n"] if c["kind"] == "glu" else c["n"]
    # The tokens' quantised activations, which several experts read (glu), or those of the places (product).
    x_rows = t if c["kind"] == "glu" else places
    s["xq"] = _words(_codes(g, x_rows, c["k"]))
    s["sx"] = 0.02 + 0.02 * torch.rand(x_rows, device="cuda", generator=g)
    s["wq"] = torch.empty(experts, wide, c["k"] // 4, device="cuda", dtype=torch.int32)
    for e in range(experts):
        s["wq"][e] = _words(_codes(g, wide, c["k"]))
    s["sw"] = (0.5 + torch.rand(experts, wide, device="cuda", generator=g)) * (0.8 / math.sqrt(c["k"]))
    s["bias"] = 0.5 * _randn(g, experts, wide) if c["bias"] else None
    s["out"] = torch.zeros(places, c["n"], device="cuda", dtype=_dtype(c))
    # What the plain form needs beside the plan: the experts that have rows, and the most rows of one.
    count = s["offsets"].diff()
    s["busy"] = count.nonzero()[:, 0]
    s["most"] = int(count.max())
    return s


# ------------------------------------------------------------------ the plain forms


def _plain_route(s):
    c, x = s["c"], s["logits"].float()
    top = x.sort(dim=1, descending=True, stable=True).indices[:, : c["top"]]
    if c["score"] == "softmax":
        p = (x - x.amax(1, keepdim=True)).exp()
    else:
        p = 1.0 / (1.0 + (-x).exp())
    w = p.gather(1, top)
    w = w / w.sum(1, keepdim=True)
    if s["mask"] is not None:
        top = torch.where(s["mask"][:, None], top, -1)
        w = torch.where(s["mask"][:, None], w, torch.zeros_like(w))
    for mine, made in zip(s["plan"], _plan(top, c["experts"])):
        mine.copy_(made)
    return [w, top.to(torch.int32), *s["plan"]]


def _grouped(s, rows):
    """f32 [places, wide] products of the rows with their experts' weights; where a place is routed. The rows of each busy
    expert are laid side by side, as many as the busiest one has."""
    c, experts, busy = s["c"], s["c"]["experts"], s["busy"]
    offsets = s["offsets"].long()
    place = torch.arange(s["rows"].numel(), device="cuda")
    e = (torch.searchsorted(offsets, place, right=True) - 1).clamp_max(experts - 1)
    side = offsets[busy, None] + torch.arange(s["most"], device="cuda")
    side = side.clamp_max(place.numel() - 1)
    x = s["xq"].view(torch.int8)[rows[side].clamp_min(0)].float()
    w = s["wq"].view(torch.int8)[busy].float()
    acc = torch.bmm(w, x.transpose(1, 2).contiguous())
    at = torch.zeros(experts, device="cuda", dtype=torch.long)
    at[busy] = torch.arange(busy.numel(), device="cuda")
    acc = acc[at[e], :, (place - offsets[e]).clamp_max(s["most"] - 1)]
    y = acc * s["sx"][rows.clamp_min(0)][:, None] * s["sw"][e]
    if s["bias"] is not None:
        y = y + s["bias"][e]
    return y, (place < offsets[-1])[:, None]


def _plain_glu(s):
    y, routed = _grouped(s, s["rows"].long())
    gate, up = y[:, : s["c"]["n"]], y[:, s["c"]["n"]:]
    h = gate / (1.0 + (-gate).exp()) * up
    return [torch.where(routed, h.to(_dtype(s["c"])), s["out"])]


def _plain_product(s):
    y, routed = _grouped(s, torch.arange(s["rows"].numel(), device="cuda"))
    return [torch.where(routed, y.to(_dtype(s["c"])), s["out"])]


def _plain_combine(s):
    slots = s["slots"].long()
    y = torch.where((slots >= 0)[..., None], s["y"][slots.clamp_min(0)].float(), 0.0)
    y = (y * s["weights"][..., None]).sum(1)
    if s["add"] is not None:
        y = y + s["add"].float()
    return [y.to(_dtype(s["c"]))]


# ------------------------------------------------------------------ the library's


def _own_route(s):
    from brain_amd import ops

    c = s["c"]
    weights, experts, plan = ops.moe_route(s["logits"], c["top"], score=c["score"], mask=s["mask"],
                                           plan=ops.MoePlan(*s["plan"]))
    return [weights, experts, *plan]


def _own_glu(s):
    from brain_amd import ops

    return [ops.matmul_i8_grouped_glu(s["xq"], s["wq"], s["sx"], s["sw"], s["offsets"], rows=s["rows"], bias=s["bias"],
                                      out=s["out"])]


def _own_product(s):
    from brain_amd import ops

    return [ops.matmul_i8_grouped(s["xq"], s["wq"], s["sx"], s["sw"], s["offsets"], bias=s["bias"], out=s["out"])]


def _own_combine(s):
    from brain_amd import ops

    return [ops.moe_combine(s["y"], s["weights"], s["slots"], add=s["add"])]


def run(state):
    kind = state["c"]["kind"]
    if own:
        return dict(route=_own_route, glu=_own_glu, product=_own_product, combine=_own_combine)[kind](state)
    return dict(route=_plain_route, glu=_plain_glu, product=_plain_product, combine=_plain_combine)[kind](state)


# ------------------------------------------------------------------ 64 bits


def _exact_weights(s):
    c, x = s["c"], s["logits"].double()
    # The scores rise with the logits, so the largest scores are the chosen experts' (equal ones count alike).
    most = x.topk(c["top"], dim=1).values
    best = torch.sigmoid(most) if c["score"] == "sigmoid" else (most - torch.logsumexp(x, 1, keepdim=True)).exp()
    best = best / best.sum(1, keepdim=True)
    return best if s["mask"] is None else best * s["mask"].double()[:, None]


def exact(case, seed):
    s = prepare(case, seed)
    c = s["c"]
    if c["kind"] == "route":
        return [_exact_weights(s), None, None, None, None]
    if c["kind"] == "combine":
        out = torch.zeros(c["tokens"], c["n"], device="cuda", dtype=torch.float64)
        for j in range(c["top"]):
            slot = s["slots"][:, j].long()
            here = (slot >= 0).nonzero()[:, 0]
            out[here] += s["weights"][here, j].double()[:, None] * s["y"][slot[here]].double()
        return [out if s["add"] is None else out + s["add"].double()]
    out = torch.zeros(s["out"].shape, device="cuda", dtype=torch.float64)
    x8, w8, ends = s["xq"].view(torch.int8), s["wq"].view(torch.int8), s["offsets"].tolist()
    for e in range(c["experts"]):
        a, b = ends[e], ends[e + 1]
        if a == b:
            continue
        rows = s["rows"][a:b].long() if c["kind"] == "glu" else torch.arange(a, b, device="cuda")
        x = x8[rows].double() * s["sx"][rows].double()[:, None]
        y = x @ (w8[e].double() * s["sw"][e].double()[:, None]).t()
        if s["bias"] is not None:
            y += s["bias"][e].double()
        if c["kind"] == "glu":
            gate, up = y.split(c["n"], 1)
            y = gate * torch.sigmoid(gate) * up
        out[a:b] = y
    return [out]


# ------------------------------------------------------------------ what a pass cannot do without


def work(case):
    c = case
    t, top, experts = c["tokens"], c["top"], c["experts"]
    e = 2 if c["dtype"] == "bf16" else 4
    entries, live = t * top, _live_tokens(c) * top
    if c["kind"] == "route":
        return dict(bytes=e * t * experts + 16 * entries + 4 * experts + (t if c["masked"] else 0), flops=4 * t * experts)
    if c["kind"] == "combine":
        return dict(bytes=e * c["n"] * (live + t + (t if c["add"] else 0)) + 8 * entries, flops=2 * live * c["n"])
    chosen = _choices(c)
    busy = np.unique(chosen[chosen >= 0]).size
    wide = 2 * c["n"] if c["kind"] == "glu" else c["n"]
    x_rows = _live_tokens(c) if c["kind"] == "glu" else live
    weights = busy * wide * (c["k"] + 4 + (4 if c["bias"] else 0))
    plan = 4 * experts + (4 * live if c["kind"] == "glu" else 0)
    return dict(bytes=weights + x_rows * (c["k"] + 4) + plan + live * c["n"] * e, flops=2 * live * wide * c["k"])
