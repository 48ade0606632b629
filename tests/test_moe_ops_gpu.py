"""The mixture-of-experts operators (ops.moe_route, moe_plan, matmul_i8_grouped[_glu], moe_combine) against plain ones in 64 bits."""
import numpy as np
import pytest
import torch

import moeref
from brain_amd import ops
from moeref import HALF

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
INF = float("inf")


def gen(seed):
    return torch.Generator().manual_seed(seed)


def same_ints(got, want):
    assert np.array_equal(got.cpu().numpy(), np.asarray(want)), (got, want)


def check_plan(plan, experts, n_experts, first=0):
    offsets, rows, slots = moeref.plan(experts, n_experts, first)
    same_ints(plan.offsets, offsets)
    same_ints(plan.rows[: len(rows)], rows)
    same_ints(plan.slots, slots)
    return len(rows)


# ---------------------------------------------------------------- routing

SIZES = [(1, 1, 1), (1, 8, 2), (1, 128, 8), (3, 7, 7), (5, 60, 4), (64, 64, 8), (65, 65, 6), (128, 128, 8), (129, 128, 8),
         (130, 256, 8), (128, 1024, 64), (2, 17, 17), (6, 33, 20), (300, 512, 16), (200, 1024, 64), (1000, 3, 2), (777, 16, 1), (2049, 130, 5)]


def logits_of(tokens, n, dtype, seed):
    """Bell-shaped logits within +-12; every third token's are halves (many equal ones)."""
    x = (1.5 * torch.randn(tokens, n, generator=gen(seed))).clamp(-12, 12)
    x[::3] = (2 * x[::3]).round() / 2
    return x.to(dtype)


def check_weights(got, want, top_k, spread=24.0):
    # The difference to the largest logit is rounded by half a step of up to `spread`, exp by 2 ulp, twice (a chosen score and the sum's
    # terms), the sum by a half step each term, and the quotient, 1 + exp and the scale by one each.
    tol = (2 * (spread + 4) + top_k + 64 + 6) * HALF[F32]
    assert np.all(np.abs(got.double().cpu().numpy() - want) <= tol * np.abs(want) + 1e-38)


@pytest.mark.parametrize("tokens,n,top_k", SIZES)
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("score,renormalize,scale", [("softmax", True, 1.0), ("softmax", False, 2.5), ("sigmoid", True, 1.0),
                                                     ("sigmoid", False, 0.5)])
def test_route(gpu, tokens, n, top_k, dtype, score, renormalize, scale):
    x = logits_of(tokens, n, dtype, tokens + n)
    mask = torch.arange(tokens) % 5 != 3 if renormalize else None
    want, experts = moeref.route(x, top_k, score, renormalize, scale, mask)
    w, e, plan = ops.moe_route(x.to(gpu), top_k, score, renormalize, scale, None if mask is None else mask.to(gpu))
    same_ints(e, experts)
    check_weights(w, want, top_k)
    check_plan(plan, experts, n)
    w2, e2, none = ops.moe_route(x.to(gpu), top_k, score, renormalize, scale, None if mask is None else mask.to(gpu), plan=False)
    assert none is None and torch.equal(e2, e) and torch.equal(w2, w)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalize", [True, False])
def test_route_values_without_order(gpu, dtype, score, renormalize):
    """NaN, infinities, lowest values, zeros of both signs, all masked: what is chosen and what is not."""
    low = torch.finfo(dtype).min
    nan = float("nan")
    rows = [[nan] * 6, [-INF] * 6, [-INF, 1.0, nan, -INF, -INF, 0.5], [low] * 6, [low, low, 0.0, low, low, low],
            [INF, 0.0, INF, 1.0, -1.0, INF], [INF, -INF, nan, low, 0.0, 1.0], [0.0, -0.0, 0.0, -0.0, 0.0, -0.0],
            [-150.0, -160.0, -150.0, -200.0, -300.0, -150.5], [nan, nan, nan, nan, nan, -1.0], [80.0, 90.0, -80.0, 85.0, 0.0, 89.0]]
    x = torch.tensor(rows).to(dtype)
    want, experts = moeref.route(x, 4, score, renormalize)
    w, e, plan = ops.moe_route(x.to(gpu), 4, score, renormalize)
    same_ints(e, experts)
    assert bool(torch.isfinite(w).all())
    # Differences of up to 350 here; scores below f32's range are 0 (or what is left of them).
    check_weights(w, want, 4, spread=350.0)
    n = check_plan(plan, experts, 6)
    assert n == (experts >= 0).sum()


def test_route_many_tokens(gpu):
    """Enough workgroups that their counts are summed in a launch of its own; every entry checked."""
    tokens, n, top_k = 600000, 16, 4
    x = torch.randn(tokens, n, generator=gen(1)).to(gpu)
    mask = (torch.arange(tokens) % 7 != 0).to(gpu)
    w, e, plan = ops.moe_route(x, top_k, mask=mask)
    want = x.double().sort(dim=1, descending=True, stable=True)
    assert torch.equal(e, torch.where(mask[:, None], want.indices[:, :top_k], -1).int())
    same_ints(plan.offsets, moeref.plan(e.cpu().numpy(), n)[0])
    flat = e.flatten().long()
    order = torch.where(flat >= 0, flat, n).sort(stable=True).indices
    live = int(plan.offsets[-1])
    assert torch.equal(plan.rows[:live], (order[:live] // top_k).int())
    place = torch.full_like(flat, -1)
    place[order[:live]] = torch.arange(live, device=gpu)
    assert torch.equal(plan.slots.flatten().long(), place)


def test_route_rows_of_a_wider_matrix(gpu):
    """A stride, and rows that do not begin at aligned addresses."""
    wide = logits_of(50, 77, F32, 1).to(gpu)
    x = wide[:, 3:63]
    want, experts = moeref.route(x.cpu(), 4)
    w, e, plan = ops.moe_route(x, 4)
    same_ints(e, experts)
    check_weights(w, want, 4)
    check_plan(plan, experts, 60)


def test_route_leaves_the_rest(gpu):
    """rows behind the last place, and buffers longer than the call's, stay as they were."""
    x = logits_of(40, 8, F32, 2).to(gpu)
    mask = (torch.arange(40) < 33).to(gpu)
    plan = ops.MoePlan(*(torch.full((n,), 77, device=gpu, dtype=torch.int32) for n in (12, 100, 90)))
    w = torch.full((90,), 5.0, device=gpu)
    ops.moe_route(x, 2, mask=mask, plan=plan, weights=w)
    assert int(plan.offsets[8]) == 66
    assert bool((plan.offsets[9:] == 77).all()) and bool((plan.rows[66:] == 77).all()) and bool((plan.slots[80:] == 77).all())
    assert bool((plan.slots[66:80] == -1).all()) and bool((w[66:80] == 0).all()) and bool((w[80:] == 5).all())


def test_no_tokens(gpu):
    plan = ops.moe_route(torch.empty(0, 9, device=gpu), 3)[2]
    same_ints(plan.offsets, [0] * 10)
    plan = ops.moe_plan(torch.empty(0, 3, device=gpu, dtype=torch.int32), 5)
    same_ints(plan.offsets, [0] * 6)
    plan = ops.moe_plan(torch.empty(4, 0, device=gpu, dtype=torch.int32), 5)
    same_ints(plan.offsets, [0] * 6)


@pytest.mark.parametrize("tokens,top_k,n,first", [(1, 1, 1, 0), (1, 70, 3, 0), (7, 3, 4, 2), (100, 8, 1024, 0), (1000, 5, 11, 4),
                                                  (5000, 3, 64, 0), (4097, 1, 300, 10), (20000, 8, 128, 0), (1, 30000, 2, 0),
                                                  (1000000, 3, 5, 0)])
def test_plan(gpu, tokens, top_k, n, first):
    """Experts from elsewhere: the same one twice in a token, and ones outside the range."""
    e = torch.randint(-2, n + first + 3, (tokens, top_k), generator=gen(tokens), dtype=torch.int32)
    e.view(-1)[0] = -2 ** 31
    e.view(-1)[-1] = 2 ** 31 - 1
    check_plan(ops.moe_plan(e.to(gpu), n, first), e.numpy(), n, first)


@pytest.mark.parametrize("tokens", [100, 3000])
def test_plan_of_one_expert(gpu, tokens):
    e = torch.full((tokens, 4), 3, dtype=torch.int32)
    check_plan(ops.moe_plan(e.to(gpu), 7), e.numpy(), 7)


# ---------------------------------------------------------------- products

def operands(x_rows, experts, n, k, seed, gpu, word=0):
    """Codes over the whole range, scales and bias; `word`: the operands begin that many words into their memory."""
    g = gen(seed)

    def at(t):
        t = t.contiguous()
        if not word:
            return t.to(gpu)
        room = torch.zeros(t.numel() + word, dtype=t.dtype, device=gpu)
        room[word:] = t.flatten().to(gpu)
        return room[word:].view(t.shape)

    codes = lambda *s: torch.randint(-128, 128, s, generator=g, dtype=torch.int8).view(torch.int32)  # noqa: E731
    xq, wq = (torch.zeros(x_rows, 0, dtype=torch.int32), torch.zeros(experts, n, 0, dtype=torch.int32)) if k == 0 else \
        (codes(x_rows, k), codes(experts, n, k))
    sx = 0.001 + 0.01 * torch.rand(x_rows, generator=g)
    sw = 0.001 + 0.002 * torch.rand(experts, n, generator=g)
    bias = torch.randn(experts, n, generator=g)
    return [at(t) for t in (xq, wq, sx, sw, bias)]


def offsets_of(counts, gpu):
    return torch.tensor(np.concatenate([[0], np.cumsum(counts)]), dtype=torch.int32, device=gpu)


def same_bits(got, want):
    view = torch.int16 if got.dtype == BF16 else torch.int32
    got = got.cpu()
    bad = (got.view(view) != want.to(got.dtype).view(view)).nonzero()
    assert not len(bad), (len(bad), bad[:5], got[tuple(bad[0])], want[tuple(bad[0])])


def check_products(gpu, xq, wq, sx, sw, bias, offsets, rows, glu_too=True, word=0):
    places = xq.shape[0] if rows is None else rows.numel()
    n = wq.shape[1]
    host = offsets.tolist()
    want, used = moeref.product(xq, wq, sx, sw, host, rows, None)
    biased, _ = moeref.product(xq, wq, sx, sw, host, rows, bias)
    acc = moeref.sums(xq, wq, host, rows, places)[0]

    def empty(dtype, cols):
        room = torch.full((places * cols + word,), 99, dtype=dtype, device=gpu)
        return room[word:].view(places, cols)

    for dtype in (torch.int32, F32, BF16):
        out = ops.matmul_i8_grouped(xq, wq, sx, sw, offsets, rows, out=empty(dtype, n))
        assert bool((out[~used] == 99).all())
        if dtype == torch.int32:
            assert torch.equal(out.cpu()[used].double(), acc[used])
            continue
        same_bits(out[used], want[used])
        out = ops.matmul_i8_grouped(xq, wq, sx, sw, offsets, rows, bias=bias, out=empty(dtype, n))
        assert bool((out[~used] == 99).all())
        same_bits(out[used], biased[used])
        if n % 2 or not glu_too:
            continue
        for b, v in ((None, want), (bias, biased)):
            h, tol = moeref.glu(v, dtype)
            out = ops.matmul_i8_grouped_glu(xq, wq, sx, sw, offsets, rows, bias=b, out=empty(dtype, n // 2))
            assert bool((out[~used] == 99).all())
            off = (out.cpu().double() - h).abs() - tol
            assert bool((off[used] <= 0).all()), off[used].max()


COUNTS = {"none": [0, 0, 0], "one": [1], "single": [0, 1, 0, 1, 0], "ends": [15, 16, 17, 0, 31, 32, 33], "tiles": [63, 64, 65, 0, 1, 127, 128, 129],
          "skewed": [0, 300, 0, 2], "many": [i % 3 for i in range(300)], "large": [257, 5, 511, 1]}


@pytest.mark.parametrize("counts", list(COUNTS))
@pytest.mark.parametrize("k,n", [(64, 64), (128, 128), (256, 96), (500, 333), (60, 30), (4, 2), (768, 256), (2048, 34)])
def test_grouped(gpu, counts, k, n):
    counts = COUNTS[counts]
    real = sum(counts)
    places = real + 7  # some of no group
    x_rows = max(1, real // 3)
    xq, wq, sx, sw, bias = operands(x_rows, len(counts), n, k, k + n + real, gpu)
    rows = torch.randint(0, x_rows, (places,), generator=gen(real), dtype=torch.int32).to(gpu)
    check_products(gpu, xq, wq, sx, sw, bias, offsets_of(counts, gpu), rows)


@pytest.mark.parametrize("counts,n", [([20] * 40, 1100), ([100, 3, 200] * 4, 1500), ([100] * 28 + [0, 199], 1500), ([300, 0, 500, 1], 700),
                                      ([1, 0, 2], 400), ([9, 30, 0, 11], 300), ([3, 5, 0, 40, 1, 2] * 10, 800), ([1, 0, 33, 2] * 8, 1700)])
@pytest.mark.parametrize("k", [128, 384, 1152, 1156])
def test_grouped_tiles(gpu, counts, n, k):
    """Few and many tiles of every height, and K of one stage, of a few and of many, and one that is not whole."""
    places = sum(counts) + 2
    xq, wq, sx, sw, bias = operands(90, len(counts), n, k, k + n, gpu)
    rows = torch.randint(0, 90, (places,), generator=gen(n), dtype=torch.int32).to(gpu)
    check_products(gpu, xq, wq, sx, sw, bias, offsets_of(counts, gpu), rows)


@pytest.mark.parametrize("k,n", [(128, 130), (500, 34), (1024, 256)])
def test_grouped_without_rows(gpu, k, n):
    counts = [3, 70, 0, 200]
    xq, wq, sx, sw, bias = operands(280, 4, n, k, 3, gpu)
    check_products(gpu, xq, wq, sx, sw, bias, offsets_of(counts, gpu), None)


@pytest.mark.parametrize("counts", [[3, 20], [300, 500]])
@pytest.mark.parametrize("size", [0.1, 10.0, 1e3, 1e8, 1e30])
def test_glu_far_gates(gpu, counts, size):
    """Gates far outside exp's range, of both signs: no NaN, nothing where the up product is not."""
    xq, wq, sx, sw, bias = operands(80, 2, 64, 128, 11, gpu)
    sx = sx * (size / 0.005 / 0.002 / 5e4)
    rows = torch.randint(0, 80, (sum(counts),), generator=gen(11), dtype=torch.int32).to(gpu)
    sw[:, 32:] = 1e-3 / size  # up products of about 1
    check_products(gpu, xq, wq, sx, sw, bias, offsets_of(counts, gpu), rows)


@pytest.mark.parametrize("word", [1, 2, 3])
@pytest.mark.parametrize("counts", [[3, 20], [70, 300]])
def test_grouped_unaligned(gpu, word, counts):
    """Operands and outputs that begin a few elements into their memory."""
    xq, wq, sx, sw, bias = operands(50, 2, 128, 256, 4, gpu, word)
    rows = torch.randint(0, 50, (sum(counts) + 3,), generator=gen(4), dtype=torch.int32).to(gpu)
    check_products(gpu, xq, wq, sx, sw, bias, offsets_of(counts, gpu), rows, word=word)


def test_grouped_without_depth(gpu):
    """K = 0: zeros, or the bias."""
    xq, wq, sx, sw, bias = operands(5, 2, 6, 0, 5, gpu)
    rows = torch.tensor([0, 1, 2, 3, 4, 0], dtype=torch.int32, device=gpu)
    check_products(gpu, xq, wq, sx, sw, bias, offsets_of([2, 3], gpu), rows)


@pytest.mark.parametrize("counts", [[20, 0, 30], [100, 150, 90], [300, 500]])
def test_grouped_without_depth_many_rows(gpu, counts):
    xq, wq, sx, sw, bias = operands(7, len(counts), 900, 0, 5, gpu)
    rows = torch.randint(0, 7, (sum(counts) + 1,), generator=gen(5), dtype=torch.int32).to(gpu)
    check_products(gpu, xq, wq, sx, sw, bias, offsets_of(counts, gpu), rows)


@pytest.mark.parametrize("counts", [[3, 2], [90, 30], [400, 300]])
def test_grouped_far_rows_of_x(gpu, counts):
    """Rows whose bytes pass 32 bits: 4.3 GB of activations, the first and the last ones read."""
    k, x_rows, n = 1024, (1 << 22) + 37, 300
    xq = torch.zeros(x_rows, k // 4, dtype=torch.int32, device=gpu)
    near, far = torch.arange(40), torch.arange(x_rows - 40, x_rows)
    pick = torch.cat([near, far])
    small, wq, _, sw, _ = operands(80, 2, n, k, 12, gpu)
    xq[pick.to(gpu)] = small
    sx = torch.rand(x_rows, device=gpu)
    at = torch.randint(0, 80, (sum(counts),), generator=gen(12))
    out = ops.matmul_i8_grouped(xq, wq, sx, sw, offsets_of(counts, gpu), pick[at].int().to(gpu))
    want, _ = moeref.product(small, wq, sx[pick.to(gpu)], sw, [0, counts[0], sum(counts)], at.int())
    same_bits(out, want)


@pytest.mark.parametrize("experts", [1, 1000])
def test_grouped_far_outputs(gpu, experts):
    """More than 2^31 results: the rows at both ends and around every 2^30th of them."""
    places, n, k = 140000, 16384, 128
    g = gen(13)
    wq = torch.randint(-128, 128, (experts, n, k), device=gpu, dtype=torch.int8).view(torch.int32)
    xq = torch.randint(-128, 128, (places, k), generator=g, dtype=torch.int8).view(torch.int32).to(gpu)
    sx, sw = torch.rand(places, device=gpu), torch.rand(experts, n, device=gpu)
    out = ops.matmul_i8_grouped(xq, wq, sx, sw, offsets_of([places // experts] * experts, gpu), out_dtype=BF16)
    for r in sorted({r for c in (0, 65535, 131071, places - 1) for r in range(max(0, c - 2), min(places, c + 3))}):
        e = r // (places // experts)
        want, _ = moeref.product(xq[r:r + 1], wq[e:e + 1], sx[r:r + 1], sw[e:e + 1], [0, 1])
        same_bits(out[r:r + 1], want)


@pytest.mark.parametrize("k,n", [(64, 32), (256, 256)])
def test_grouped_rows_outside(gpu, k, n):
    """Rows that x does not have give zeros; offsets past the places, descending ones and repeated ones stay inside."""
    xq, wq, sx, sw, bias = operands(40, 6, n, k, 6, gpu)
    rows = torch.randint(0, 40, (150,), generator=gen(6), dtype=torch.int32)
    rows[[0, 7, 60, 100]] = torch.tensor([40, -1, 2 ** 31 - 1, -2 ** 31], dtype=torch.int32)
    offsets = torch.tensor([0, 30, 30, 20, 20, 130, 2 ** 31 - 1], dtype=torch.int32, device=gpu)
    # (group 3, [20, 20), and the descending group 2 are empty; group 4 [20, 130) would share places with group 0.)
    offsets[3] = offsets[4] = 30
    check_products(gpu, xq, wq, sx, sw, bias, offsets, rows.to(gpu))
    offsets = torch.tensor([5, 90, 90, 80, 100, 110, 120], dtype=torch.int32, device=gpu)
    offsets[3] = 90
    check_products(gpu, xq, wq, sx, sw, bias, offsets, rows.to(gpu))


def test_grouped_descending_offsets(gpu):
    """A group that ends before it begins is empty."""
    xq, wq, sx, sw, bias = operands(64, 3, 64, 128, 7, gpu)
    check_products(gpu, xq, wq, sx, sw, bias, torch.tensor([50, 60, 20, 40], dtype=torch.int32, device=gpu), None)


def test_grouped_no_rows_of_x(gpu):
    xq, wq, sx, sw, bias = operands(0, 2, 8, 64, 8, gpu)
    rows = torch.zeros(5, dtype=torch.int32, device=gpu)
    out = torch.full((5, 8), 9.0, device=gpu)
    ops.matmul_i8_grouped(xq, wq, sx, sw, offsets_of([1, 2], gpu), rows, out=out)
    assert bool((out[:3] == 0).all()) and bool((out[3:] == 9).all())


def test_grouped_far_weights(gpu):
    """Weights whose bytes pass 32 bits: 4.3 GB of experts, the last ones with rows."""
    experts, n, k = 1030, 2048, 2048
    w = torch.zeros(experts, n, k // 4, device=gpu, dtype=torch.int32)
    for e in (0, experts - 2, experts - 1):
        w[e] = torch.randint(-128, 128, (n, k), generator=gen(e), dtype=torch.int8).view(torch.int32).to(gpu)
    counts = [0] * experts
    counts[0], counts[-2], counts[-1] = 2, 70, 3
    xq, _, sx, _, _ = operands(75, 1, 8, k, 9, gpu)
    sw = 0.001 + torch.rand(experts, n, device=gpu)
    out = ops.matmul_i8_grouped(xq, w, sx, sw, offsets_of(counts, gpu))
    host = [0, 2, 72, 75]
    pick = [0, experts - 2, experts - 1]
    want, _ = moeref.product(xq, w[pick], sx, sw[pick], host)
    same_bits(out, want)


# ---------------------------------------------------------------- the weighted sum

@pytest.mark.parametrize("tokens,top_k,n", [(1, 1, 1), (1, 8, 2048), (3, 2, 7), (33, 4, 500), (100, 8, 64), (17, 64, 36), (5, 0, 12),
                                            (1000, 6, 333)])
@pytest.mark.parametrize("dtype,out_dtype", [(F32, F32), (BF16, BF16), (F32, BF16), (BF16, F32)])
@pytest.mark.parametrize("word", [0, 1])
def test_combine(gpu, tokens, top_k, n, dtype, out_dtype, word):
    g = gen(tokens + n)
    places = max(1, tokens * top_k - 2)
    room = torch.randn(places * n + word, generator=g).to(dtype).to(gpu)
    y = room[word:].view(places, n)
    w = torch.rand(tokens, top_k, generator=g)
    slots = torch.randint(-2, places + 2, (tokens, top_k), generator=g, dtype=torch.int32)
    add = torch.randn(tokens * n + word, generator=g).to(out_dtype).to(gpu)[word:].view(tokens, n)
    for extra in (None, add):
        want, size = moeref.combine(y, w, slots, extra)
        # A half step of a product and of a sum, each choice; one of the sum with `add`; the output's.
        tol = (top_k + 2) * HALF[F32] * size
        if out_dtype == BF16:
            tol = tol + HALF[BF16] * (want.abs() + tol)
        out = ops.moe_combine(y, w.to(gpu), slots.to(gpu), add=extra, out_dtype=out_dtype)
        assert bool(((out.cpu().double() - want).abs() <= tol).all())
    ops.moe_combine(y, w.to(gpu), slots.to(gpu), add=add, out=add)  # in place
    assert torch.equal(add, out)


def test_combine_skips_what_is_not_there(gpu):
    """NaN rows that no slot names, and no rows at all."""
    y = torch.full((4, 8), float("nan"), device=gpu)
    y[2] = 3.0
    slots = torch.tensor([[2, -1], [-1, 9]], dtype=torch.int32, device=gpu)
    w = torch.ones(2, 2, device=gpu)
    out = ops.moe_combine(y, w, slots)
    assert bool((out[0] == 3).all()) and bool((out[1] == 0).all())
    out = ops.moe_combine(y[:0], w, slots)
    assert bool((out == 0).all())


def test_combine_far_rows(gpu):
    """Rows whose bytes pass 32 bits: 4.3 GB of bf16, the first and the last."""
    places, n = (1 << 20) + 5, 2056
    y = torch.zeros(places, n, dtype=BF16, device=gpu)
    pick = torch.tensor([0, 1, places - 2, places - 1])
    y[pick.to(gpu)] = torch.randn(4, n, generator=gen(20)).to(BF16).to(gpu)
    slots = torch.tensor([[places - 1, 0], [1, places - 2], [places, places - 1]], dtype=torch.int32)
    w = torch.rand(3, 2, generator=gen(21))
    small = torch.tensor([[3, 0], [1, 2], [4, 3]], dtype=torch.int32)
    want, size = moeref.combine(y[pick.to(gpu)], w, small)
    out = ops.moe_combine(y, w.to(gpu), slots.to(gpu), out_dtype=F32)
    assert bool(((out.cpu().double() - want).abs() <= 4 * HALF[F32] * size).all())


def test_route_far_rows(gpu):
    """Rows of logits 2^31 elements apart."""
    base = torch.empty(2 * 2 ** 31 + 64, dtype=BF16, device=gpu)
    x = base.as_strided((3, 60), (2 ** 31, 1))
    logits = logits_of(3, 60, BF16, 22)
    x.copy_(logits)
    want, experts = moeref.route(logits, 5)
    w, e, plan = ops.moe_route(x, 5)
    same_ints(e, experts)
    check_weights(w, want, 5)
    check_plan(plan, experts, 60)


def test_grouped_sums_need_no_scales(gpu):
    """The C entry's raw sums, without scales."""
    import ctypes as C

    from brain_amd import _lib

    for counts in ([2, 3], [90, 200]):
        xq, wq, sx, sw, _ = operands(50, 2, 130, 128, 23, gpu)
        rows = torch.randint(0, 50, (sum(counts),), generator=gen(23), dtype=torch.int32).to(gpu)
        offsets = offsets_of(counts, gpu)
        out = torch.zeros(sum(counts), 130, dtype=torch.int32, device=gpu)
        g = _lib.GroupedI8T(xq.data_ptr(), None, 50, rows.data_ptr(), offsets.data_ptr(), sum(counts), 2, wq.data_ptr(), None, None, 32, 130)
        _lib.check(_lib.load().bh_matmul_i8_grouped(torch.cuda.current_stream().cuda_stream, C.byref(g), out.data_ptr(), _lib.BH_OUT_I32))
        acc = moeref.sums(xq, wq, offsets.tolist(), rows, sum(counts))[0]
        assert torch.equal(out.cpu().double(), acc)


@pytest.mark.parametrize("tokens", [3, 3000])
def test_route_on_two_streams(gpu, tokens):
    """Calls at once, each with its own buffers: the bits of the calls one after another."""
    data = [logits_of(tokens, 128, F32, s).to(gpu) for s in range(4)]
    want = [ops.moe_route(x, 8) for x in data]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in data]
    for _ in range(5):
        got = []
        for s, x in zip(streams, data):
            with torch.cuda.stream(s):
                got.append(ops.moe_route(x, 8))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1]) and all(torch.equal(p, q) for p, q in zip(a[2], b[2]))


def test_route_many_tokens_in_a_graph(gpu):
    """Many tokens (three launches and a workspace), captured; replays on other logits equal eager calls."""
    tokens, n, top_k = 9000, 64, 4
    x = logits_of(tokens, n, F32, 30).to(gpu)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.moe_route(x, top_k)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        w, e, plan = ops.moe_route(x, top_k)
    for rep in range(4):
        x.copy_(logits_of(tokens, n, F32, 31 + rep))
        want = ops.moe_route(x, top_k)
        for t in (w, e, *plan):
            t.fill_(-7)
        torch.randn(1000, device=gpu).sum()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(w, want[0]) and torch.equal(e, want[1]) and all(torch.equal(p, q) for p, q in zip(plan, want[2]))
