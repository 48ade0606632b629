"""The int8 paged cache's operators where their arguments end: lengths, sizes and values that programs do have, and that the
parametrised cases of tests/test_kvops_gpu.py do not."""
import ctypes as C
import math

import pytest
import torch

import kvref as ref
from brain_amd import load, ops
from brain_amd._lib import Kv8BatchT, check
from test_kvops_gpu import BF16, F32, gen, joined, near

pytestmark = pytest.mark.gpu

# rows, heads, kv heads, head_dim, block size: each kernel of attention and of the weight sums.
KERNELS = [(1, 4, 2, 36, 8), (3, 4, 2, 64, 16), (60, 4, 2, 128, 16), (300, 4, 2, 64, 24), (3, 2, 1, 96, 5)]


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("n,nh,nkv,hd,bs", KERNELS)
def test_lengths_below_zero_and_past_the_table(gpu, n, nh, nkv, hd, bs, dtype):
    """Sequences that are off (-1 and other lengths below zero) see, store and keep nothing; one that is longer than its table
    sees what the table has."""
    g = gen(n, hd, bs, 31)
    lens = [-1, 50, -5, 0x7FFFFFFF, -(1 << 31), 64]
    c = ref.Cache(g, len(lens), -(-64 // bs), bs, nkv, hd, spare=6)
    room = c.table.shape[1] * bs
    start = ref.starts([1, n, n, n, 2, 1])
    total = int(start[-1])
    q = torch.randn(total, nh, hd, generator=g).to(dtype)
    # The same for the plain forms: no length is 0, and the long one's rows all lie behind the table.
    plain = [max(0, min(t, room + n)) for t in lens]
    want, lse, ob, lb = ref.attention(c, q, start, plain, 0.1)
    dl, ds = torch.tensor(lens, dtype=torch.int32, device=gpu), start.to(gpu)
    acc = torch.rand(len(lens), nkv, room, generator=g)
    new, bound = ref.weight_sums(c, q, lse.float(), start, plain, 0.1, acc)
    for hints in ({}, dict(max_rows=n, max_len=room)):
        kv = c.kv(ops, gpu)
        out, got = ops.paged_attention_i8(q.to(gpu), kv, dl, ds, 0.1, **hints)
        near(out, want, ob, f"out {hints}")
        near(got, lse, lb, f"lse {hints}")
        near(ops.paged_weight_sums_i8(q.to(gpu), lse.float().to(gpu), kv, dl, acc.to(gpu), ds, 0.1, **hints), new, bound, f"acc {hints}")
    x, cut = joined(g, total, nh, nkv, hd, dtype)
    dq, dk, dv = cut(x.to(gpu))
    kv = c.kv(ops, gpu)
    ops.qk_norm_rope_append_i8(dq, dk, dv, torch.zeros(total, dtype=torch.int32, device=gpu), ops.rope_frequencies(hd, 1e4), kv, dl, ds)
    stored = sorted(s for b in (1, 5) for _, k in ref.chunk_rows(start, lens, b) if k > 0 and (s := c.slot(b, k - 1)) >= 0)
    assert (kv.v_scales.cpu() != c.scales[1]).any(1).nonzero().view(-1).tolist() == stored
    kv = c.kv(ops, gpu)
    keep, new_lens = ops.paged_kv_evict_i8(kv, dl, acc.to(gpu), 20)
    want_keep, want_lens = ref.evict(plain, acc, 20, 0, 0)
    assert torch.equal(keep.cpu(), want_keep) and torch.equal(new_lens.cpu(), want_lens)
    off = torch.tensor([c.slot(b, j) for b in (0, 2, 4) for j in range(room)])
    assert torch.equal(kv.k_scales.cpu()[off], c.scales[0][off])


@pytest.mark.parametrize("n,nh,nkv,hd,dtype", [(60, 4, 2, 128, F32), (90, 4, 2, 64, F32), (100, 4, 2, 128, BF16), (300, 4, 2, 64, BF16)])
def test_tiny_queries_over_large_key_scales(gpu, n, nh, nkv, hd, dtype):
    """Queries whose squares are below f32's range, key scales that make up for it: scores of some hundred binades behind a
    first part of small ones, over several tiles."""
    g = gen(n, hd, 32)
    bs, t = 16, 700
    c = ref.Cache(g, 1, -(-t // bs), bs, nkv, hd)
    # A score's deviation: 1e-25 * 73 * sqrt(hd) * scale.
    for j in range(t):
        c.scales[0][c.slot(0, j)] = (3.0 if j < 150 else 50.0) / (73 * hd ** 0.5) * 1e25
    start, lens = ref.starts([n]), [t]
    q = (torch.randn(n, nh, hd, generator=g) * 1e-25).to(dtype)
    want, lse, ob, lb = ref.attention(c, q, start, lens, 1.0)
    assert float(lse.min()) > 80 and float(ob.max()) < 0.1 * float(want.abs().max())
    out, got = ops.paged_attention_i8(q.to(gpu), c.kv(ops, gpu), torch.tensor(lens, dtype=torch.int32, device=gpu), start.to(gpu), 1.0)
    near(got, lse, lb, "lse")
    # A weight of less than 2^-126 of its row's largest lies below f32's range and may be lost (the bounds count roundings
    # only): at most that for each of the t keys, whose values are at most 127 * 1.2 / 60 (kvref.Cache's scales).
    near(out, want, ob + t * 2.0 ** -126 * 127 * 1.2 / 60, "out")


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("many,n,hd", [(20, 70, 128), (70, 150, 64), (33, 300, 128)])
def test_single_tokens_beside_a_chunk(gpu, many, n, hd, dtype):
    """Dozens of single tokens and one prompt piece in a batch, keys split; with a workspace of exactly the size asked for."""
    g = gen(many, n, hd)
    nh, nkv, bs = 8, 4, 16
    rows = [1] * many
    rows.insert(many // 3, n)
    rows.insert(2, 0)
    lens = [max(r, int(torch.randint(1, 1400, (1,), generator=g))) for r in rows]
    lens[many // 2] = 1400
    c = ref.Cache(g, len(rows), -(-1400 // bs), bs, nkv, hd)
    start = ref.starts(rows)
    total = int(start[-1])
    q = torch.randn(total, nh, hd, generator=g).to(dtype)
    want, lse, ob, lb = ref.attention(c, q, start, lens, 0.1)
    kv, dq, dl, ds = c.kv(ops, gpu), q.to(gpu), torch.tensor(lens, dtype=torch.int32, device=gpu), start.to(gpu)
    for max_rows in (0, n, 1):
        b, need = Kv8BatchT(ds.data_ptr(), dl.data_ptr(), len(rows), total, max_rows, 1400), C.c_uint64()
        check(load().bh_paged_attention_i8_workspace(kv.ref, C.byref(b), nh, C.byref(need)))
        assert need.value > 0
        ws = torch.full((need.value // 4 + 64,), math.nan, device=gpu)
        out, got = torch.full_like(dq, math.nan), torch.full((total, nh), math.nan, device=gpu)
        check(load().bh_paged_attention_i8(torch.cuda.current_stream().cuda_stream, dq.data_ptr(), nh * hd, ops._ACT[dtype], nh,
                                           kv.ref, C.byref(b), 0.1, out.data_ptr(), got.data_ptr(), ws.data_ptr(), need.value))
        near(out, want, ob, f"out {max_rows}")
        near(got, lse, lb, f"lse {max_rows}")
        assert bool(torch.isnan(ws[need.value // 4:]).all()), "behind the workspace"


@pytest.mark.parametrize("batch,nkv,hd,bs,cap,budget,in_place", [
    (4, 8, 64, 16, 900, 704, False), (4, 8, 64, 16, 900, 705, False), (5, 7, 64, 8, 300, 100, False), (2, 3, 36, 7, 700, 312, False),
    (2, 3, 36, 7, 700, 313, False), (1, 2, 128, 32, 4096, 3000, True), (1, 2, 128, 32, 4097, 3000, True), (32, 8, 16, 4, 90, 50, True),
    (33, 8, 16, 4, 90, 50, True), (9, 2, 36, 5, 1100, 1000, True)])
def test_evict_in_one_launch_or_two(gpu, batch, nkv, hd, bs, cap, budget, in_place):
    """Either side of each limit that chooses how the eviction is launched; lengths around the budget among the long ones."""
    g = gen(batch, nkv, hd, cap, budget)
    c = ref.Cache(g, batch, -(-cap // bs), bs, nkv, hd, spare=batch * -(-budget // bs))
    lens = torch.randint(budget, cap + 1, (batch,), generator=g).tolist()
    lens[0] = cap
    lens[-1] = [budget, budget - 1, cap][batch % 3]
    acc = torch.randn(batch, nkv, cap, generator=g)
    to = c.table if in_place else c.free.view(batch, -1).contiguous()
    kv, dl = c.kv(ops, gpu), torch.tensor(lens, dtype=torch.int32, device=gpu)
    out = torch.zeros(batch, nkv, budget, device=gpu)
    keep, new = ops.paged_kv_evict_i8(kv, dl, acc.to(gpu), budget, 3, 20, None if in_place else to.to(gpu), out)
    want, want_lens = ref.evict(lens, acc, budget, 3, 20)
    assert torch.equal(keep.cpu(), want) and torch.equal(new.cpu(), want_lens)
    assert torch.equal(dl.cpu(), torch.tensor(lens, dtype=torch.int32))
    live, at = want >= 0, want.long().clamp_min(0)
    assert torch.equal(out.cpu(), torch.where(live, acc.gather(2, at), torch.zeros(())))
    slots = lambda t, j: t.long().gather(1, j.flatten(1) // bs).view(j.shape) * bs + j % bs  # noqa: E731
    src, dst = slots(c.table, at), slots(to, torch.arange(budget).expand_as(at))
    head = torch.arange(nkv)[None, :, None].expand_as(at)
    for w, (pool, sc) in enumerate(((kv.k_pool, kv.k_scales), (kv.v_pool, kv.v_scales))):
        codes, scales = c.codes[w].clone(), c.scales[w].clone()
        codes[dst[live], head[live]], scales[dst[live], head[live]] = c.codes[w][src[live], head[live]], c.scales[w][src[live], head[live]]
        assert torch.equal(pool.cpu().view(torch.int8).view(codes.shape), codes) and torch.equal(sc.cpu(), scales)


@pytest.mark.parametrize("batch", [63, 64, 65])
@pytest.mark.parametrize("hd,dtype", [(64, F32), (128, BF16), (36, F32)])
def test_as_many_sequences_as_lanes(gpu, batch, hd, dtype):
    """Batches at the wave's width, where the look-up of a row's sequence changes; empty sequences first, last and between."""
    g = gen(batch, hd, 41)
    nh, nkv, bs = 4, 2, 16
    rows = torch.randint(0, 4, (batch,), generator=g).tolist()
    rows[0] = rows[-1] = rows[-2] = 0
    rows[batch // 2] = 9
    lens = [max(r, int(torch.randint(0, 90, (1,), generator=g))) for r in rows]
    c = ref.Cache(g, batch, 6, bs, nkv, hd)
    start = ref.starts(rows)
    total, pad = int(start[-1]), 3
    dl, ds = torch.tensor(lens, dtype=torch.int32, device=gpu), start.to(gpu)
    q = torch.randn(total + pad, nh, hd, generator=g).to(dtype)
    want, lse, ob, lb = ref.attention(c, q, start, lens, 0.1)
    acc = torch.rand(batch, nkv, 96, generator=g)
    given = lse.float()
    new, bound = ref.weight_sums(c, q, given, start, lens, 0.1, acc)
    for hints in ({}, dict(max_rows=9, max_len=90)):
        out = torch.full((total + pad, nh, hd), math.nan, dtype=dtype, device=gpu)
        got = torch.full((total + pad, nh), math.nan, device=gpu)
        kv = c.kv(ops, gpu)
        ops.paged_attention_i8(q.to(gpu), kv, dl, ds, 0.1, out=out, lse=got, **hints)
        near(out, want, ob, f"out {hints}")
        near(got, lse, lb, f"lse {hints}")
        near(ops.paged_weight_sums_i8(q.to(gpu), given.to(gpu), kv, dl, acc.to(gpu), ds, 0.1, **hints), new, bound, f"acc {hints}")
    x, cut = joined(g, total + pad, nh, nkv, hd, dtype)
    dq, dk, dv = cut(x.to(gpu))
    kv = c.kv(ops, gpu)
    q_out = torch.full((total + pad, nh, hd), 7.0, dtype=dtype, device=gpu)
    ops.qk_norm_rope_append_i8(dq, dk, dv, torch.zeros(total + pad, dtype=torch.int32, device=gpu), ops.rope_frequencies(hd, 1e4), kv,
                               dl, ds, q_out=q_out)
    assert torch.equal(q_out[:total], dq[:total]) and bool((q_out[total:] == 7.0).all())  # no norm, no turn at position 0
    where = [(r, c.slot(b, n - 1)) for b in range(batch) for r, n in ref.chunk_rows(start, lens, b)]
    r, slots = torch.tensor([a for a, _ in where]), torch.tensor([s for _, s in where])
    v = cut(x)[2][r].float()
    # A code is within half a step of its scale, which is the largest element's 127th part.
    scale = v.abs().amax(-1) / 127
    got_scale = kv.v_scales.cpu()[slots]
    assert bool(((got_scale - scale).abs() <= 2 * ref.EPS * scale).all())
    codes = kv.v_pool.cpu().view(torch.int8).view(-1, nkv, hd)[slots].double()
    assert bool(((codes - v.double() / got_scale.double()[..., None]).abs() <= 0.5 + 127 * 2 * ref.EPS).all())
    rest = torch.ones(c.slots, dtype=torch.bool)
    rest[slots] = False
    assert torch.equal(kv.v_scales.cpu()[rest], c.scales[1][rest]) and torch.equal(kv.k_scales.cpu()[rest], c.scales[0][rest])


@pytest.mark.parametrize("hd", [64, 128, 100])
def test_norm_of_extremes_in_keys(gpu, hd):
    """Zero, huge and non-finite heads among the keys: as the same values among the queries, each head for itself."""
    q = torch.ones(4, 2, hd)
    q[0, 0] = 0.0
    q[1, 0] = 1e15
    q[2, 0, 3] = math.inf
    q[3, 1, 5] = math.nan
    freq, pos, w = ops.rope_frequencies(hd, 1e4), torch.arange(4, dtype=torch.int32, device=gpu), torch.full((hd,), 0.5, device=gpu)
    oq, ok = (t.cpu() for t in ops.qk_norm_rope(q.to(gpu), q.to(gpu), pos, freq, w, w))
    assert torch.equal(torch.isnan(oq), torch.isnan(ok)) and torch.equal(oq.nan_to_num(9.0), ok.nan_to_num(9.0))
    finite = torch.ones(4, 2, dtype=torch.bool)
    finite[2, 0] = finite[3, 1] = False
    want, bound = ref.turn(q, w.cpu(), 1e-6, pos.cpu(), freq.cpu())
    for name, t in (("q", oq), ("k", ok)):
        near(t[finite], want[finite], bound[finite] + ref.EPS * want[finite].abs(), name)
        assert bool(torch.isnan(t[3, 1]).all()) and bool(torch.isnan(t[2, 0]).any())
