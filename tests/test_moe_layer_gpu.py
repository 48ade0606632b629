"""The mixture-of-experts operators one after another, as a decoder layer calls them: against 64 bits, captured and replayed, on another
stream than the default one, and as expert-parallel ranks."""
import pytest
import torch

import moeref
from brain_amd import moe, ops
from moeref import HALF

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


def gen(seed):
    return torch.Generator().manual_seed(seed)


def make(gpu, experts, model, ff, top_k, seed=0, **router):
    g = gen(seed)
    gate_up = torch.randn(experts, 2 * ff, model, generator=g) / model ** 0.5
    down = torch.randn(experts, model, ff, generator=g) / ff ** 0.5
    return moe.MoeInt8.quantize(gate_up.to(gpu), down.to(gpu), top_k, **router)


def inputs(gpu, layer, tokens, dtype, seed):
    g = gen(seed)
    return (torch.randn(tokens, layer.d_model, generator=g).to(dtype).to(gpu),
            (1.5 * torch.randn(tokens, layer.n_experts, generator=g)).to(gpu))


def values(words, scale):
    """64-bit values of codes [..., k / 4] with their scales."""
    return words.cpu().view(torch.int8).double() * scale.cpu().double()[..., None]


def reference(layer, x, logits, mask=None, add=None):
    """The layer in 64 bits on the same codes of x and weights, without the quantisation of h; and how far the layer may be from it."""
    quantize = ops.quantize_rows_bf16 if x.dtype == BF16 else ops.quantize_rows
    sx, xq = quantize(x)
    xv, gu, dn = values(xq, sx), values(layer.gate_up, layer.gate_up_scale), values(layer.down, layer.down_scale)
    w, experts = moeref.route(logits, layer.top_k, layer.score, layer.renormalize, layer.scale, mask)
    out, tol = torch.zeros(x.shape, dtype=torch.float64), torch.zeros(x.shape, dtype=torch.float64)
    half = HALF[x.dtype]
    for t in range(x.shape[0]):
        for j, e in enumerate(experts[t]):
            if e < 0:
                continue
            v = gu[e] @ xv[t]
            gate, up = v.split(layer.d_ff)
            h = gate / (1 + torch.exp(-gate)) * up
            # h: the two products' four roundings each move it by less than 5 (1 + |gate|) half steps of f32, silu's own 7, and it is
            # rounded to x's type (twice that where f32 moves it first); then its code is half a step of its scale off, a
            # little more where h itself was off.
            dh = (5 * 2 * (1 + gate.abs()) + 7) * HALF[F32] * h.abs() + (half if half > HALF[F32] else 0) * h.abs() * 1.001
            step = (h.abs() + dh).max().clamp_min(1e-8) / 127
            dh = dh + 0.5 * step * (1 + 2.0 ** -18) + 128 * 4 * HALF[F32] * step
            y, dy = dn[e] @ h, dn[e].abs() @ dh
            # y: four roundings of f32, one to x's type; its weight and place in the sum.
            dy = dy + (4 * HALF[F32] + half * 1.001) * (y.abs() + dy)
            wt = float(w[t, j])
            out[t] += wt * y
            tol[t] += wt * (dy + (2 ** 8 + layer.top_k + 2) * HALF[F32] * (y.abs() + dy))
        if add is not None:
            out[t] += add[t].double().cpu()
    return out, tol + 1.001 * half * (out.abs() + tol) + HALF[F32] * out.abs()


@pytest.mark.parametrize("tokens", [1, 3, 40, 200])
@pytest.mark.parametrize("shape", [(8, 128, 256, 2), (60, 64, 96, 4), (5, 36, 20, 3), (16, 256, 128, 1)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_layer(gpu, tokens, shape, dtype):
    score = "sigmoid" if shape[3] == 3 else "softmax"
    layer = make(gpu, *shape, score=score, scale=1.5)
    x, logits = inputs(gpu, layer, tokens, dtype, tokens)
    mask = torch.arange(tokens, device=gpu) % 4 != 2 if tokens > 1 else None
    add = x.flip(0).contiguous() if tokens == 40 else None
    want, tol = reference(layer, x, logits, None if mask is None else mask.cpu(), add)
    out = layer(x, logits, mask=mask, add=add)
    assert out.dtype == dtype
    assert bool(((out.cpu().double() - want).abs() <= tol).all())
    if mask is not None and add is None:
        assert bool((out[~mask] == 0).all())


def test_layer_shares_experts_between_ranks(gpu):
    """Two expert-parallel ranks, half of the experts each, add up to the layer."""
    layer = make(gpu, 12, 128, 64, 3)
    x, logits = inputs(gpu, layer, 90, F32, 1)
    want = layer(x, logits)
    sx, xq = ops.quantize_rows(x)
    weights, experts, whole = ops.moe_route(logits, 3)
    out, parts = None, []
    for first in (0, 6):
        mine = slice(first, first + 6)
        plan = ops.moe_plan(experts, 6, first=first)
        parts.append(int(plan.offsets[-1]))
        h = ops.matmul_i8_grouped_glu(xq, layer.gate_up[mine], sx, layer.gate_up_scale[mine], plan.offsets, plan.rows)
        hx, hq = ops.quantize_rows(h)
        y = ops.matmul_i8_grouped(hq, layer.down[mine], hx, layer.down_scale[mine], plan.offsets)
        out = ops.moe_combine(y, weights, plan.slots, add=out)
    assert sum(parts) == 270 == int(whole.offsets[-1])
    # The same products in another order of sums: three terms, a half step each sum.
    assert bool(((out - want).abs() <= 8 * HALF[F32] * (want.abs() + 4 * want.abs().max())).all())


@pytest.mark.parametrize("tokens", [1, 7, 300])
def test_layer_in_a_graph(gpu, tokens):
    """Captured once, replayed on other inputs in the same buffers, eager work and synchronisations between: the eager bits. Two graphs of the
    layer alternate (each has its own buffers)."""
    layer = make(gpu, 24, 128, 96, 4)
    sets = []
    side = torch.cuda.Stream()
    for s in range(2):
        x, logits = inputs(gpu, layer, tokens, BF16, s)
        mask = torch.ones(tokens, dtype=torch.bool, device=gpu)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            layer(x, logits, mask=mask)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = layer(x, logits, mask=mask)
        sets.append((graph, x, logits, mask, out))
    for rep in range(4):
        for s, (graph, x, logits, mask, out) in enumerate(sets):
            new = inputs(gpu, layer, tokens, BF16, 10 * rep + s)
            x.copy_(new[0])
            logits.copy_(new[1])
            mask.copy_(torch.arange(tokens, device=gpu) < tokens - rep // 2)
            want = layer(x, logits, mask=mask)
            out.fill_(7)
            graph.replay()
            torch.randn(1000, device=gpu).sum()
            torch.cuda.synchronize()
            assert torch.equal(out.view(torch.int16), want.view(torch.int16)), (rep, s)
    torch.cuda.synchronize()


def test_layer_on_streams(gpu):
    """Two streams at once, each with its own calls: the bits of the calls one after another."""
    layer = make(gpu, 16, 256, 128, 2)
    data = [inputs(gpu, layer, t, F32, t) for t in (5, 700)]
    want = [layer(*d) for d in data]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in data]
    for _ in range(5):
        got = []
        for s, d in zip(streams, data):
            with torch.cuda.stream(s):
                got.append(layer(*d))
        torch.cuda.synchronize()
        for g, w in zip(got, want):
            assert torch.equal(g, w)


def test_runs_repeat(gpu):
    """The same call gives the same bits, plan included."""
    layer = make(gpu, 60, 128, 64, 4)
    x, logits = inputs(gpu, layer, 1500, BF16, 3)
    first = layer(x, logits)
    plan = ops.moe_route(logits, 4)[2]
    for _ in range(5):
        assert torch.equal(layer(x, logits).view(torch.int16), first.view(torch.int16))
        assert all(torch.equal(a, b) for a, b in zip(ops.moe_route(logits, 4)[2], plan))


def test_layer_without_tokens(gpu):
    layer = make(gpu, 4, 64, 32, 2)
    assert layer(torch.empty(0, 64, device=gpu), torch.empty(0, 4, device=gpu)).shape == (0, 64)
    x, logits = inputs(gpu, layer, 9, F32, 1)
    none = layer(x, logits, mask=torch.zeros(9, dtype=torch.bool, device=gpu), add=x)
    assert torch.equal(none, x)
