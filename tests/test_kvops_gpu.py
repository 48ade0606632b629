"""The operators of the int8 paged KV cache (qk_norm_rope[_append_i8], paged_attention_i8, paged_weight_sums_i8,
paged_kv_evict_i8) against plain 64-bit forms (tests/kvref.py), whose bounds count the roundings of 32-bit arithmetic and of
the outputs' type."""
import ctypes as C
import math

import pytest
import torch

import kvref as ref
from brain_amd import load, ops
from brain_amd._lib import check

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


def gen(*seed):
    g = torch.Generator()
    g.manual_seed(hash(seed) % (1 << 31))
    return g


def near(got, want, bound, what):
    got, want = got.detach().cpu().double(), want
    assert got.shape == want.shape, what
    same_nan = torch.isnan(got) == torch.isnan(want)
    assert bool(same_nan.all()), f"{what}: NaN at other places"
    fine = torch.isfinite(want)
    odd = ~fine & ~torch.isnan(want)
    assert bool((got[odd] == want[odd]).all()), f"{what}: infinities at other places"
    off = (got - want).abs()[fine]
    bad = off > bound[fine]
    if bool(bad.any()):
        i = int((off / bound[fine].clamp_min(1e-300)).argmax())
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {off[i]:.3g} where {bound[fine][i]:.3g} is "
                             f"allowed (value {want[fine][i]:.6g})")


def joined(g, rows, nh, nkv, hd, dtype, more=0):
    """q, k, v as views of one projection's rows, `more` unused elements behind each."""
    x = torch.randn(rows, (nh + 2 * nkv) * hd + more, generator=g).to(dtype)
    cut = lambda t: (t[:, : nh * hd].unflatten(1, (nh, hd)), t[:, nh * hd: (nh + nkv) * hd].unflatten(1, (nkv, hd)),  # noqa: E731
                     t[:, (nh + nkv) * hd: (nh + 2 * nkv) * hd].unflatten(1, (nkv, hd)))
    return x, cut


# ------------------------------------------------------------------ norm and rotation

ROPE = [(1, 16, 8, 128, 128, 0), (7, 8, 8, 64, 64, 0), (300, 32, 8, 128, 128, 8), (33, 9, 3, 64, 64, 2), (5, 28, 4, 128, 128, 0),
        (65, 4, 2, 128, 64, 0), (3, 3, 1, 36, 36, 1), (4, 2, 2, 256, 256, 0), (2, 5, 5, 96, 32, 0), (9, 1, 1, 4, 2, 0), (6, 2, 1, 80, 0, 0)]


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("norm", [True, False], ids=["norm", "plain"])
@pytest.mark.parametrize("rows,nh,nkv,hd,rot,more", ROPE)
def test_qk_norm_rope(gpu, rows, nh, nkv, hd, rot, more, norm, dtype):
    g = gen(rows, hd, rot)
    x, cut = joined(g, rows, nh, nkv, hd, dtype, more)
    q, k, _ = cut(x)
    w = [torch.randn(hd, generator=g) if norm else None for _ in "qk"]
    pos = torch.randint(0, 1 << 20, (rows,), generator=g, dtype=torch.int32)
    pos[0] = 0
    freq = 1e4 ** (-torch.arange(rot // 2, dtype=torch.float64) * 2 / max(rot, 1))
    dq, dk, _ = cut(x.to(gpu))
    dw = [None if t is None else t.to(gpu) for t in w]
    got = ops.qk_norm_rope(dq, dk, pos.to(gpu), freq.to(gpu), *dw, eps=1e-5)
    for name, o, t, wt in (("q", got[0], q, w[0]), ("k", got[1], k, w[1])):
        want, bound = ref.turn(t, wt, 1e-5, pos, freq)
        near(o, want, bound + ref.HALF[dtype] * (want.abs() + bound), name)
    # in place, through the views
    ops.qk_norm_rope(dq, dk, pos.to(gpu), freq.to(gpu), *dw, eps=1e-5, q_out=dq, k_out=dk)
    assert torch.equal(dq, got[0]) and torch.equal(dk, got[1])


def test_norm_of_extremes(gpu):
    """Zero heads, huge and non-finite elements: each head for itself."""
    hd = 128
    q = torch.ones(4, 2, hd)
    q[0, 0] = 0.0
    q[1, 0] = 1e15
    q[2, 0, 3] = math.inf
    q[3, 1, 5] = math.nan
    k = q[:, :1].contiguous()
    freq = ops.rope_frequencies(hd, 1e4, "cpu")
    pos = torch.zeros(4, dtype=torch.int32)
    w = torch.ones(hd)
    oq, ok = (t.cpu() for t in ops.qk_norm_rope(q.to(gpu), k.to(gpu), pos.to(gpu), freq.to(gpu), w.to(gpu), w.to(gpu)))
    assert bool((oq[0, 0] == 0).all())
    assert bool(((oq[1, 0] - 1).abs() < 1e-5).all())
    assert bool(torch.isnan(oq[2, 0, 3])) and bool(torch.isfinite(oq[2, 1]).all())
    assert bool(torch.isnan(oq[3, 1]).all()) and bool(torch.isfinite(oq[3, 0]).all())
    assert torch.equal(ok, oq[:, :1]) or bool((torch.isnan(ok) == torch.isnan(oq[:, :1])).all())


# ------------------------------------------------------------------ append


def append_plain(dev, src, slots, clip, cache_kv, which, bs, hd):
    """The one-token kernel on the same rows."""
    rows, nkv = src.shape[:2]
    pool, sc = (cache_kv.k_pool, cache_kv.k_scales) if which == 0 else (cache_kv.v_pool, cache_kv.v_scales)
    blk, off = (slots // bs).to(torch.int32).to(dev), (slots % bs).to(torch.int32).to(dev)
    check(load().bh_paged_kv_append_i8(torch.cuda.current_stream().cuda_stream, src.data_ptr(), blk.data_ptr(), off.data_ptr(),
                                       clip.data_ptr(), pool.data_ptr(), pool.numel(), sc.data_ptr(), sc.numel(), rows,
                                       nkv * hd, bs, hd))


APPEND = [([1] * 5, [3, 17, 1, 40, 9], 8, 8, 64, 16), ([4, 0, 33, 1], [4, 7, 61, 64], 16, 8, 128, 32), ([70], [70], 6, 2, 128, 5),
          ([3, 2], [2, 9], 3, 3, 36, 4), ([2], [300], 2, 1, 256, 1), ([9] * 70, [9] * 70, 4, 2, 64, 3)]


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("rows,lens,nh,nkv,hd,bs", APPEND)
def test_append(gpu, rows, lens, nh, nkv, hd, bs, dtype):
    g = gen(len(rows), hd, bs)
    batch, pad = len(rows), 3
    c = ref.Cache(g, batch, (max(lens) + bs - 1) // bs, bs, nkv, hd)
    start = ref.starts(rows)
    total = int(start[-1])
    x, cut = joined(g, total + pad, nh, nkv, hd, dtype)
    x[0, nh * hd:] = 0.0  # zero heads: scale 1
    pos = torch.randint(0, 5000, (total + pad,), generator=g, dtype=torch.int32)
    w = [torch.rand(hd, generator=g) + 0.5 for _ in "qk"]
    clip = [torch.rand(nkv, generator=g) * 3 + 1 for _ in "kv"]
    freq = ops.rope_frequencies(hd, 1e5, "cpu")
    kv = c.kv(ops, gpu)
    q_out = torch.full((total + pad, nh, hd), 7.0, dtype=dtype, device=gpu)
    dq, dk, dv = cut(x.to(gpu))
    ops.qk_norm_rope_append_i8(dq, dk, dv, pos.to(gpu), freq.to(gpu), kv, torch.tensor(lens, dtype=torch.int32, device=gpu),
                               start.to(gpu), w[0].to(gpu), w[1].to(gpu), k_clip=clip[0].to(gpu), v_clip=clip[1].to(gpu),
                               q_out=q_out)
    plain_q, plain_k = ops.qk_norm_rope(dq, dk, pos.to(gpu), freq.to(gpu), w[0].to(gpu), w[1].to(gpu))
    assert torch.equal(q_out[:total], plain_q[:total])
    assert bool((q_out[total:] == 7.0).all()), "rows behind the last sequence"
    where = [(r, c.slot(b, n - 1)) for b in range(batch) for r, n in ref.chunk_rows(start, lens, b) if n > 0]
    r, slots = torch.tensor([a for a, _ in where]), torch.tensor([s for _, s in where])
    # Values: the codes of the one-token kernel, bit for bit; nothing else touched.
    other = c.kv(ops, gpu)
    append_plain(gpu, dv[r.to(gpu)].float().contiguous(), slots, clip[1].to(gpu), other, 1, bs, hd)
    assert torch.equal(kv.v_pool, other.v_pool) and torch.equal(kv.v_scales, other.v_scales)
    # Keys: the scale within the turned values' bound, a code within half a step and that bound.
    _, k, _ = cut(x)
    want, bound = ref.turn(k, w[1], 1e-6, pos, freq)
    want, bound = want[r], bound[r]
    mx = torch.minimum(want.abs().amax(-1), clip[0].double())
    sc = torch.where(mx == 0, 1.0, mx / 127)
    got_sc = kv.k_scales.cpu()[slots].double()
    assert bool(((got_sc - sc).abs() <= bound.amax(-1) / 127 + 2 * ref.EPS * sc).all())
    codes = kv.k_pool.cpu().view(torch.int8).view(-1, nkv, hd)
    ideal = (want / sc[..., None])
    slack = bound / sc[..., None] + ideal.abs() * (bound.amax(-1) / mx.clamp_min(1e-30))[..., None] + 1e-4
    off = (codes[slots].double() - ideal.clamp(-127, 127)).abs()
    assert bool((off <= 0.5 + slack).all())
    if dtype == F32:  # and those of the one-token kernel on the turned keys
        append_plain(gpu, plain_k[r.to(gpu)].contiguous(), slots, clip[0].to(gpu), other, 0, bs, hd)
        assert torch.equal(kv.k_pool, other.k_pool) and torch.equal(kv.k_scales, other.k_scales)
    mask = torch.ones(c.slots, dtype=torch.bool)
    mask[slots] = False
    assert torch.equal(codes[mask], c.codes[0][mask]) and torch.equal(kv.k_scales.cpu()[mask], c.scales[0][mask])


def test_append_bad_slots(gpu):
    """Table entries outside the pool, and positions behind the tables, store nothing."""
    g = gen(1)
    c = ref.Cache(g, 3, 2, 8, 2, 64)
    c.table[0, 0] = c.slots // 8 + 5
    c.table[1, 1] = -1
    lens, start = torch.tensor([4, 16, 20], dtype=torch.int32), ref.starts([4, 10, 5])
    x, cut = joined(g, 19, 4, 2, 64, F32)
    kv = c.kv(ops, gpu)
    dq, dk, dv = cut(x.to(gpu))
    ops.qk_norm_rope_append_i8(dq, dk, dv, torch.zeros(19, dtype=torch.int32, device=gpu), ops.rope_frequencies(64, 1e4), kv,
                               lens.to(gpu), start.to(gpu))
    good = sorted(s for b in range(3) for _, n in ref.chunk_rows(start, lens, b) if (s := c.slot(b, n - 1)) >= 0)
    assert len(good) == 2 + 1
    changed = (kv.v_scales.cpu() != c.scales[1]).any(1).nonzero().view(-1).tolist()
    assert changed == good


# ------------------------------------------------------------------ attention

# rows, lens, heads, kv heads, head_dim, block size
ATTN = [([1], [1], 16, 8, 128, 16), ([1, 1, 1], [5, 64, 300], 16, 8, 128, 32), ([1] * 3, [33, 1, 500], 28, 4, 128, 16),
        ([3, 0, 20, 1], [3, 9, 77, 0], 9, 3, 64, 5), ([130], [130], 8, 8, 64, 16), ([65, 7, 1], [200, 7, 129], 16, 8, 128, 24),
        ([17], [400], 6, 2, 36, 7), ([5, 2], [260, 1], 4, 1, 256, 64), ([1, 2], [70, 33], 40, 1, 64, 1), ([40], [33], 4, 2, 128, 8),
        ([2] * 70, [40] * 70, 4, 2, 64, 16), ([300], [700], 32, 8, 128, 256), ([33], [97], 2, 2, 96, 32)]


def run_attention(gpu, c, q, start, lens, scale, **more):
    return ops.paged_attention_i8(q, c.kv(ops, gpu), torch.as_tensor(lens, dtype=torch.int32).to(gpu),
                                  None if start is None else start.to(gpu), scale, **more)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("rows,lens,nh,nkv,hd,bs", ATTN)
def test_attention(gpu, rows, lens, nh, nkv, hd, bs, dtype):
    g = gen(sum(lens), nh, hd, bs)
    c = ref.Cache(g, len(rows), max(1, (max(lens) + bs - 1) // bs), bs, nkv, hd)
    start = ref.starts(rows)
    total, pad = int(start[-1]), 2
    q = torch.randn(total + pad, nh, hd, generator=g).to(dtype)
    scale = 1.3 * hd ** -0.5
    want, lse, ob, lb = ref.attention(c, q, start, lens, scale)
    wide = torch.zeros(total + pad, nh * hd + 8, dtype=dtype, device=gpu)  # rows further apart than they are long
    wide[:, : nh * hd] = q.flatten(1).to(gpu)
    view = wide[:, : nh * hd].unflatten(1, (nh, hd))
    first = None
    for hints in ({}, dict(max_rows=max(rows), max_len=max(lens))):
        out = torch.full((total + pad, nh, hd), math.nan, dtype=dtype, device=gpu)
        got_lse = torch.full((total + pad, nh), math.nan, device=gpu)
        run_attention(gpu, c, view, start, lens, scale, out=out, lse=got_lse, **hints)
        near(out, want, ob, f"out {hints}")
        near(got_lse, lse, lb, f"lse {hints}")
        first = out if first is None else first
    again = torch.full_like(out, math.nan)
    run_attention(gpu, c, q.to(gpu), start, lens, scale, out=again, max_rows=max(rows), max_len=max(lens))
    assert torch.equal(again[:total], out[:total]), "the same call twice"
    if rows == [1] * len(rows):
        alone, _ = run_attention(gpu, c, q[:total].to(gpu), None, lens, scale)
        near(alone, want[:total], ob[:total], "without row_start")


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("rows", [1, 40])
def test_attention_odd_values(gpu, rows, dtype):
    """Scales that are infinite or NaN where no row sees them, blocks outside the pool, zero and negative scales, a query that
    is not finite: only what sees them changes."""
    g = gen(7, rows)
    nh, nkv, hd, bs = 4, 2, 128, 16
    c = ref.Cache(g, 2, 8, bs, nkv, hd)
    start, lens = ref.starts([rows, rows]), [70, 90]
    for b, n in enumerate(lens):  # behind the sequences, inside their last blocks and behind them
        for j in range(n, 8 * bs):
            c.scales[0][c.slot(b, j)] = math.nan if j % 2 else math.inf
            c.scales[1][c.slot(b, j)] = math.inf if j % 2 else math.nan
    c.table[0, 1] = 1 << 20
    q = torch.randn(2 * rows, nh, hd, generator=g).to(dtype)
    for scale in (0.1, 0.0, -0.2):
        want, lse, ob, lb = ref.attention(c, q, start, lens, scale)
        out, got = run_attention(gpu, c, q.to(gpu), start, lens, scale)
        near(out, want, ob, f"out at scale {scale}")
        near(got, lse, lb, f"lse at scale {scale}")
    clean = run_attention(gpu, c, q.to(gpu), start, lens, 0.1)[0]
    q[0, 1, 5] = math.nan
    q[rows, 2, 0] = math.inf
    out = run_attention(gpu, c, q.to(gpu), start, lens, 0.1)[0]
    assert bool(torch.isnan(out[0, 1]).all()) and bool(torch.isnan(out[rows, 2]).all())
    out[0, 1], out[rows, 2] = clean[0, 1], clean[rows, 2]
    assert torch.equal(out, clean), "other rows and heads"
    # Visible, an infinite value scale reaches every row that sees the key.
    c.scales[1][c.slot(1, 30), 0] = math.inf
    out = run_attention(gpu, c, q.to(gpu), start, lens, 0.1)[0]
    assert not bool(torch.isfinite(out[rows:, :2]).any()) and bool(torch.isfinite(out[rows:, 3]).all())


def test_attention_wide_range(gpu):
    """Queries whose elements span 60 binades, f32: the bound is that of each row's own products."""
    g = gen(8)
    c = ref.Cache(g, 1, 4, 32, 2, 128)
    q = torch.randn(20, 4, 128, generator=g) * 2.0 ** torch.randint(-60, 1, (20, 4, 128), generator=g).float()
    q[3] *= 1e-30
    q[4, 0, 0] = 3.3e38
    c.codes[0][:, 0, 0] = 0
    start, lens = ref.starts([20]), [128]
    for scale in (0.3, 1e-3):
        want, lse, ob, lb = ref.attention(c, q, start, lens, scale)
        out, got = run_attention(gpu, c, q.to(gpu), start, lens, scale)
        near(out, want, ob, "out")
        near(got, lse, lb, "lse")


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("rows,t,nh,nkv", [(1, 20000, 16, 8), (1, 9001, 8, 1), (3, 12345, 32, 8), (200, 6000, 4, 2)])
def test_attention_finds_each_key(gpu, rows, t, nh, nkv, dtype):
    """A long sequence whose every key in turn (a sample of them) outweighs the rest for one query: the output is its value."""
    hd, bs = 128, 16
    g = gen(rows, t)
    nblk = (t + bs - 1) // bs
    codes = torch.randint(-6, 7, (nblk * bs, nkv, hd), generator=g, dtype=torch.int8)
    v = torch.randint(-127, 128, (nblk * bs, nkv, hd), generator=g, dtype=torch.int8)
    scales = torch.full((nblk * bs, nkv), 1 / 64)
    table = torch.randperm(nblk, generator=g).to(torch.int32).view(1, -1)
    words = lambda x: x.view(torch.int32).view(nblk * bs, -1).to(gpu)  # noqa: E731
    kv = ops.PagedKV8(words(codes), words(v), scales.to(gpu), scales.to(gpu), table.to(gpu), bs, hd)
    # For row i and head h, the key at `pick` is 80 * a pattern of signs that only this query has.
    near_end = [0, 1, 15, 16, 31, 32, 63, 64, 127, 128, t - rows - 1, t - rows, t - rows - 33, t // 2, t // 3]
    picks = [(near_end[i] if i < len(near_end) else int(torch.randint(0, t - rows, (1,), generator=g)))
             for i in range(rows * nh)]
    picks = torch.tensor(picks[: rows * nh]).view(rows, nh)
    q = torch.randint(0, 2, (rows, nh, hd), generator=g).float() * 2 - 1
    at = table[0].long()[picks // bs] * bs + picks % bs
    kvh = (torch.arange(nh) * nkv // nh).expand(rows, nh)
    dense = codes.clone()
    dense[at.view(-1), kvh.reshape(-1)] = (80 * q).to(torch.int8).view(-1, hd)  # a key picked twice: the last one holds
    kv.k_pool.copy_(words(dense))
    held = (dense[at, kvh].float() == 80 * q).all(-1)
    assert int(held.sum()) >= held.numel() // 2
    out, lse = ops.paged_attention_i8(q.to(dtype).to(gpu), kv, torch.tensor([t], dtype=torch.int32, device=gpu),
                                      ref.starts([rows]).to(gpu), 1.0, max_rows=rows, max_len=t)
    want = v[at, kvh].float() / 64
    # The picked key's score is 128 * 80 / 64 = 160; another key's, sums of random signs, stays below 80 (checked), so the
    # others weigh less than t e^-80 together.
    rival = (q.view(rows, nkv, nh // nkv, hd) @ dense.float().permute(1, 2, 0)[None] / 64).view(rows, nh, -1)
    rival.scatter_(2, at[..., None], 0.0)
    held &= rival.amax(-1) < 80
    assert int(held.sum()) >= held.numel() // 2
    assert bool((out.cpu().float()[held] - want[held]).abs().max() <= 2 * ref.HALF[dtype] * 2)
    assert bool(((lse.cpu() - 160).abs()[held] <= 160 * 4 * 2.0 ** -23).all())


def test_attention_past_32_bits(gpu):
    """Blocks whose bytes lie past 2^32 in each pool."""
    nkv, hd, bs = 8, 128, 32
    nblk = (1 << 32) // (nkv * hd * bs) + 64
    g = gen(9)
    c = ref.Cache(g, 2, 4, bs, nkv, hd)
    pools = [torch.zeros(nblk * bs, nkv * hd // 4, dtype=torch.int32, device=gpu) for _ in "kv"]
    scales = [torch.zeros(nblk * bs, nkv, device=gpu) for _ in "kv"]
    far = nblk - 1 - torch.arange(c.slots // bs)  # where block i of the small cache is
    for i in range(2):
        pools[i].view(nblk, bs, -1)[far.to(gpu)] = c.words(i).view(-1, bs, nkv * hd // 4).to(gpu)
        scales[i].view(nblk, bs, -1)[far.to(gpu)] = c.scales[i].view(-1, bs, nkv).to(gpu)
    kv = ops.PagedKV8(*pools, *scales, far[c.table.long()].to(torch.int32).to(gpu), bs, hd)
    for rows in ([1, 1], [40, 3]):
        start, lens = ref.starts(rows), [128, 77]
        dl = torch.tensor(lens, dtype=torch.int32, device=gpu)
        q = torch.randn(sum(rows), 16, hd, generator=g)
        want, lse, ob, lb = ref.attention(c, q, start, lens, 0.1)
        out, got = ops.paged_attention_i8(q.to(gpu), kv, dl, start.to(gpu), 0.1)
        near(out, want, ob, "out")
        near(got, lse, lb, "lse")
        acc = torch.zeros(2, nkv, 128)
        new, bound = ref.weight_sums(c, q, got.cpu(), start, lens, 0.1, acc)
        near(ops.paged_weight_sums_i8(q.to(gpu), got, kv, dl, acc.to(gpu), start.to(gpu), 0.1), new, bound, "acc")
    # A row stored there, and entries moved there.
    x = torch.randn(2, 24, hd, generator=g).to(gpu)
    qo = ops.qk_norm_rope_append_i8(x[:, :8], x[:, 8:16], x[:, 16:], torch.zeros(2, dtype=torch.int32, device=gpu),
                                    ops.rope_frequencies(hd, 1e4), kv, dl)
    assert torch.equal(qo, x[:, :8])  # no norm, no turn at position 0
    for b, n in enumerate([128, 77]):
        s = int(kv.block_tables[b, (n - 1) // bs]) * bs + (n - 1) % bs
        back = kv.v_pool.view(torch.int8).view(-1, nkv, hd)[s].float() * kv.v_scales[s][:, None]
        assert bool(((back - x[b, 16:]).abs() <= kv.v_scales[s][:, None] * 0.5001).all())
    keep, new_lens = ops.paged_kv_evict_i8(kv, dl, acc.to(gpu), 20)
    want_keep, want_lens = ref.evict([128, 77], acc, 20, 0, 0)
    assert torch.equal(keep.cpu(), want_keep) and torch.equal(new_lens.cpu(), want_lens)


# ------------------------------------------------------------------ weight sums


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("rows,lens,nh,nkv,hd,bs", ATTN)
def test_weight_sums(gpu, rows, lens, nh, nkv, hd, bs, dtype):
    g = gen(sum(lens), nh, hd, bs, 1)
    c = ref.Cache(g, len(rows), max(1, (max(lens) + bs - 1) // bs), bs, nkv, hd)
    start = ref.starts(rows)
    total = int(start[-1])
    q = torch.randn(total + 2, nh, hd, generator=g).to(dtype)
    scale = hd ** -0.5
    lse = ref.attention(c, q, start, lens, scale)[1].float()
    for cap in (max(lens) + 9, max(1, max(lens) - 3)):
        acc = torch.randn(len(rows), nkv, cap, generator=g)
        want, bound = ref.weight_sums(c, q, lse, start, lens, scale, acc)
        for hints in ({}, dict(max_rows=max(rows), max_len=max(lens))):
            got = ops.paged_weight_sums_i8(q.to(gpu), lse.to(gpu), c.kv(ops, gpu), torch.tensor(lens, dtype=torch.int32, device=gpu),
                                           acc.to(gpu), start.to(gpu), scale, **hints)
            near(got, want, bound, f"acc, cap {cap}, {hints}")


def test_weight_sums_add_up(gpu):
    """Every row gives away 1 for each query head."""
    g = gen(11)
    nh, nkv, hd = 16, 8, 128
    c = ref.Cache(g, 2, 70, 32, nkv, hd)
    start, lens = ref.starts([300, 1]).to(gpu), torch.tensor([2000, 2240], dtype=torch.int32, device=gpu)
    q = torch.randn(301, nh, hd, generator=g).to(gpu)
    kv = c.kv(ops, gpu)
    _, lse = ops.paged_attention_i8(q, kv, lens, start)
    acc = torch.zeros(2, nkv, 2240, device=gpu)
    ops.paged_weight_sums_i8(q, lse, kv, lens, acc, start)
    want = torch.tensor([300.0, 1.0], device=gpu)[:, None].expand(2, nkv) * (nh // nkv)
    # A weight is off by some hundred half steps (its score is), a sum of n by n more at most.
    assert bool(((acc.double().sum(2) - want).abs() <= want * 3000 * ref.EPS).all())
    assert bool((acc[0, :, 2000:] == 0).all())


def test_weight_sums_unseen_blocks(gpu):
    """A key in a block outside the pool gets nothing; one behind every row's position neither."""
    g = gen(12)
    c = ref.Cache(g, 2, 6, 16, 2, 64)
    c.table[0, 2] = -1
    for j in range(50, 96):
        c.scales[0][c.slot(1, j)] = math.nan
    start, lens = ref.starts([5, 40]), [90, 50]
    q = torch.randn(45, 4, 64, generator=g)
    lse = ref.attention(c, q, start, lens, 0.2)[1].float()
    acc = torch.rand(2, 2, 96, generator=g)
    want, bound = ref.weight_sums(c, q, lse, start, lens, 0.2, acc)
    got = ops.paged_weight_sums_i8(q.to(gpu), lse.to(gpu), c.kv(ops, gpu), torch.tensor(lens, dtype=torch.int32, device=gpu),
                                   acc.to(gpu), start.to(gpu), 0.2)
    near(got, want, bound, "acc")
    assert torch.equal(got.cpu()[0, :, 32:48], acc[0, :, 32:48]) and torch.equal(got.cpu()[1, :, 50:], acc[1, :, 50:])


# ------------------------------------------------------------------ eviction

EVICT = [([50, 7, 0, 31], 20, 2, 5, 8, 64, 16), ([300], 299, 0, 0, 1, 128, 32), ([300, 100], 1, 0, 0, 3, 36, 7), ([64, 65], 64, 64, 0, 2, 64, 8),
         ([2000, 3000], 700, 4, 100, 2, 128, 16), ([5000], 4999, 4000, 999, 1, 4, 64), ([40, 41], 40, 0, 40, 2, 256, 1),
         ([9000], 3000, 0, 1, 1, 64, 24), ([17000, 20], 5000, 3, 50, 1, 64, 16)]


@pytest.mark.parametrize("in_place", [True, False], ids=["in_place", "copied"])
@pytest.mark.parametrize("values", ["spread", "ties", "odd"])
@pytest.mark.parametrize("lens,budget,sink,recent,nkv,hd,bs", EVICT)
def test_evict(gpu, lens, budget, sink, recent, nkv, hd, bs, values, in_place):
    g = gen(sum(lens), budget, hd)
    batch, blocks = len(lens), (budget + bs - 1) // bs
    c = ref.Cache(g, batch, (max(lens) + bs - 1) // bs, bs, nkv, hd, spare=batch * blocks)
    acc = torch.randn(batch, nkv, max(lens) + 3, generator=g)
    if values == "ties":
        acc = (acc * 2).round() / 2
    elif values == "odd":
        pick = torch.randint(0, 8, acc.shape, generator=g)
        for i, v in enumerate((math.nan, math.inf, -math.inf, 0.0, -0.0, 1e-42)):
            acc[pick == i] = v
    to = None if in_place else c.free[: batch * blocks].view(batch, blocks).contiguous()
    want_keep, want_lens = ref.evict(lens, acc, budget, sink, recent)
    codes, scales = [x.clone() for x in c.codes], [x.clone() for x in c.scales]
    want_acc = acc.clone() if in_place else torch.full((batch, nkv, budget + 2), 5.0)
    for b in range(batch):
        for h in range(nkv):
            for i, j in enumerate(want_keep[b, h].tolist()):
                if j >= 0:
                    s, d = c.slot(b, j), c.slot(b, i, to)
                    for w in range(2):
                        codes[w][d, h], scales[w][d, h] = c.codes[w][s, h], c.scales[w][s, h]
                    want_acc[b, h, i] = acc[b, h, j]
    kv, dacc = c.kv(ops, gpu), acc.to(gpu)
    dlens = torch.tensor(lens, dtype=torch.int32, device=gpu)
    out = dacc if in_place else torch.full((batch, nkv, budget + 2), 5.0, device=gpu)
    keep, new = ops.paged_kv_evict_i8(kv, dlens, dacc, budget, sink, recent, None if to is None else to.to(gpu), out,
                                      new_lens=dlens if in_place else None)
    assert torch.equal(keep.cpu(), want_keep)
    assert torch.equal(new.cpu(), want_lens) and (new.data_ptr() == dlens.data_ptr()) == in_place
    for w, (pool, sc) in enumerate(((kv.k_pool, kv.k_scales), (kv.v_pool, kv.v_scales))):
        assert torch.equal(pool.cpu().view(torch.int8).view(codes[w].shape), codes[w]), "codes"
        assert torch.equal(sc.cpu(), scales[w]), "scales"
    assert torch.equal(out.cpu().view(torch.int32), want_acc.view(torch.int32)), "acc"


def test_evict_bad_blocks(gpu):
    """An entry whose block, old or new, lies outside the pool is not moved."""
    g = gen(13)
    c = ref.Cache(g, 1, 4, 8, 2, 64, spare=2)
    c.table[0, 3] = 1 << 24
    to = torch.tensor([[int(c.free[0]), -1]], dtype=torch.int32)
    acc = torch.rand(1, 2, 32, generator=g)
    kv = c.kv(ops, gpu)
    keep, _ = ops.paged_kv_evict_i8(kv, torch.tensor([32], dtype=torch.int32, device=gpu), acc.to(gpu), 16, 0, 12, to.to(gpu))
    want = [x.clone() for x in c.scales]
    for h in range(2):
        for i, j in enumerate(keep[0, h].tolist()):
            s, d = c.slot(0, j), c.slot(0, i, to)
            if s >= 0 and d >= 0:
                for w in range(2):
                    want[w][d, h] = c.scales[w][s, h]
    assert torch.equal(kv.k_scales.cpu(), want[0]) and torch.equal(kv.v_scales.cpu(), want[1])


# ------------------------------------------------------------------ together


class Life:
    """Two sequences through a layer's attention: prompt pieces, weights, eviction, single tokens, on one cache."""

    def __init__(self, dev, dtype, nh=8, nkv=2, hd=128, bs=16, blocks=12):
        self.nh, self.nkv, self.hd, self.dtype = nh, nkv, hd, dtype
        g = torch.Generator(device=dev)
        g.manual_seed(3)
        self.g, self.dev = g, dev
        slots = 2 * blocks * bs
        z = lambda *s, t=torch.int32: torch.zeros(*s, dtype=t, device=dev)  # noqa: E731
        table = torch.randperm(2 * blocks, generator=g, device=dev).to(torch.int32).view(2, blocks)
        self.kv = ops.PagedKV8(z(slots, nkv * hd // 4), z(slots, nkv * hd // 4), z(slots, nkv, t=F32), z(slots, nkv, t=F32), table,
                               bs, hd)
        self.lens, self.acc = z(2), z(2, nkv, blocks * bs, t=F32)
        self.freq = ops.rope_frequencies(hd, 1e4, dev)
        self.seen = [0, 0]

    def chunk(self, rows):
        x = torch.randn(sum(rows), self.nh + 2 * self.nkv, self.hd, generator=self.g, device=self.dev).to(self.dtype)
        pos = torch.cat([torch.arange(s, s + n, dtype=torch.int32, device=self.dev) for s, n in zip(self.seen, rows)])
        self.seen = [s + n for s, n in zip(self.seen, rows)]
        return x, pos, ref.starts(rows).to(self.dev), torch.tensor(rows, dtype=torch.int32, device=self.dev)

    def layer(self, x, pos, start, rows):
        self.lens += rows
        q, k, v = x.split((self.nh, self.nkv, self.nkv), 1)
        q = ops.qk_norm_rope_append_i8(q, k, v, pos, self.freq, self.kv, self.lens, start)
        out, lse = ops.paged_attention_i8(q, self.kv, self.lens, start)
        ops.paged_weight_sums_i8(q, lse, self.kv, self.lens, self.acc, start)
        return q, out, lse

    def twin(self):
        """The cache as it is now, for the 64-bit forms."""
        c = ref.Cache.__new__(ref.Cache)
        c.bs, c.nkv, c.hd, c.slots = self.kv.block_size, self.nkv, self.hd, self.kv.k_scales.shape[0]
        c.codes = [p.cpu().view(torch.int8).view(c.slots, c.nkv, c.hd) for p in (self.kv.k_pool, self.kv.v_pool)]
        c.scales = [self.kv.k_scales.cpu(), self.kv.v_scales.cpu()]
        c.table = self.kv.block_tables.cpu()
        return c


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_life_of_a_cache(gpu, dtype):
    s = Life(gpu, dtype)
    for rows in ([50, 30], [40, 1], [1, 1]):
        before = s.acc.cpu()
        args = s.chunk(rows)
        q, out, lse = s.layer(*args)
        c, start, lens = s.twin(), args[2].cpu(), s.lens.tolist()
        want, wl, ob, lb = ref.attention(c, q.cpu(), start, lens, s.hd ** -0.5)
        near(out, want, ob, f"out {rows}")
        near(lse, wl, lb, f"lse {rows}")
        new, bound = ref.weight_sums(c, q.cpu(), lse.cpu(), start, lens, s.hd ** -0.5, before)
        near(s.acc, new, bound, f"acc {rows}")
    acc = s.acc.cpu()
    keep, _ = ops.paged_kv_evict_i8(s.kv, s.lens, s.acc, 48, sink=2, recent=8, acc_out=s.acc, new_lens=s.lens)
    want_keep, want_lens = ref.evict(lens, acc, 48, 2, 8)
    assert torch.equal(keep.cpu(), want_keep) and torch.equal(s.lens.cpu(), want_lens)
    after = s.twin()
    for b in range(2):
        for h in range(s.nkv):
            old = torch.tensor([c.slot(b, j) for j in want_keep[b, h].tolist() if j >= 0])
            at = torch.tensor([c.slot(b, i) for i in range(len(old))])
            for w in range(2):
                assert torch.equal(after.codes[w][at, h], c.codes[w][old, h])
    args = s.chunk([1, 20])  # and on: positions go on counting, the cache is shorter
    q, out, lse = s.layer(*args)
    want, wl, ob, lb = ref.attention(s.twin(), q.cpu(), args[2].cpu(), s.lens.tolist(), s.hd ** -0.5)
    near(out, want, ob, "out after")
    near(lse, wl, lb, "lse after")


def test_captured(gpu):
    """The whole layer and an eviction in one graph, replayed with other work between: every replay equals the eager run."""
    def step(s, args):
        r = s.layer(*args)
        keep, _ = ops.paged_kv_evict_i8(s.kv, s.lens, s.acc, 40, 2, 8, acc_out=s.acc, new_lens=s.lens)
        return (*r, keep)

    eager, s = Life(gpu, BF16), Life(gpu, BF16)
    for t in (eager, s):
        t.layer(*t.chunk([60, 45]))
    args = eager.chunk([1, 3])
    held = [a.clone() for a in args]
    state = [s.kv.k_pool, s.kv.v_pool, s.kv.k_scales, s.kv.v_scales, s.lens, s.acc]
    warm = [t.clone() for t in state]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(s, held)
    torch.cuda.current_stream().wait_stream(side)
    for t, w in zip(state, warm):
        t.copy_(w)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(s, held)
    for _ in range(4):
        want = step(eager, args)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(want, got):
            assert torch.equal(a, b)
        for a, b in zip((eager.kv.k_pool, eager.kv.v_pool, eager.kv.k_scales, eager.kv.v_scales, eager.lens, eager.acc), state):
            assert torch.equal(a, b)
        args = eager.chunk([1, 3])
        for h, a in zip(held, args):
            h.copy_(a)
        torch.randn(1000, 1000, device=gpu).sum().item()


def test_two_streams(gpu):
    """Two programs' calls at once on streams of their own."""
    g = gen(14)
    caches = [ref.Cache(g, 3, 40, 32, 2, 128) for _ in "ab"]
    lens = [1200, 700, 1]
    qs = [torch.randn(3, 8, 128, generator=g).to(gpu) for _ in "ab"]
    kvs = [c.kv(ops, gpu) for c in caches]
    dl = torch.tensor(lens, dtype=torch.int32, device=gpu)
    alone = [ops.paged_attention_i8(q, kv, dl) for q, kv in zip(qs, kvs)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in "ab"]
    got = [[], []]
    for _ in range(10):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(ops.paged_attention_i8(qs[i], kvs[i], dl))
    torch.cuda.synchronize()
    for i in range(2):
        for out, lse in got[i]:
            assert torch.equal(out, alone[i][0]) and torch.equal(lse, alone[i][1])


# ------------------------------------------------------------------ hints, and batches without rows


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("rows,lens,nh,nkv,hd,bs", [ATTN[3], ATTN[5], ATTN[6], ATTN[11], ([1, 1], [5000, 129], 8, 2, 128, 16)])
def test_wrong_hints(gpu, rows, lens, nh, nkv, hd, bs, dtype):
    """max_rows and max_len only choose how the work is split: too small or too large ones give the same values."""
    g = gen(sum(lens), nh, hd, bs, 2)
    c = ref.Cache(g, len(rows), max(1, (max(lens) + bs - 1) // bs), bs, nkv, hd)
    start = ref.starts(rows)
    q = torch.randn(int(start[-1]), nh, hd, generator=g).to(dtype)
    want, lse, ob, lb = ref.attention(c, q, start, lens, 0.1)
    acc = torch.randn(len(rows), nkv, max(lens), generator=g)
    given = lse.float()
    want_acc, bound = ref.weight_sums(c, q, given, start, lens, 0.1, acc)
    dl = torch.tensor(lens, dtype=torch.int32, device=gpu)
    for max_rows in (1, 9, 1 << 30):
        for max_len in (1, 200, 1 << 30):
            hints = dict(max_rows=max_rows, max_len=max_len)
            out, got = run_attention(gpu, c, q.to(gpu), start, lens, 0.1, **hints)
            near(out, want, ob, f"out {hints}")
            near(got, lse, lb, f"lse {hints}")
            sums = ops.paged_weight_sums_i8(q.to(gpu), given.to(gpu), c.kv(ops, gpu), dl, acc.to(gpu), start.to(gpu), 0.1, **hints)
            near(sums, want_acc, bound, f"acc {hints}")


def test_no_rows(gpu):
    """Batches without sequences or without rows: nothing is done, acc keeps what it has."""
    g = gen(21)
    c = ref.Cache(g, 2, 3, 16, 2, 64)
    kv, none = c.kv(ops, gpu), torch.zeros(0, dtype=torch.int32, device=gpu)
    lens, start = torch.tensor([40, 3], dtype=torch.int32, device=gpu), torch.zeros(3, dtype=torch.int32, device=gpu)
    q, k, pos = torch.zeros(0, 4, 64, device=gpu), torch.zeros(0, 2, 64, device=gpu), none
    freq = ops.rope_frequencies(64, 1e4)
    acc = torch.rand(2, 2, 48, generator=g).to(gpu)
    old = acc.clone()
    for at, st in ((none, None), (lens, start)):
        assert ops.qk_norm_rope(q, k, pos, freq)[0].shape == q.shape
        ops.qk_norm_rope_append_i8(q, k, k, pos, freq, kv, at, st)
        out, lse = ops.paged_attention_i8(q, kv, at, st)
        assert out.shape == q.shape and lse.shape == (0, 4)
        ops.paged_weight_sums_i8(q, lse, kv, at, acc, st)
    assert ops.paged_kv_evict_i8(kv, none, acc, 5)[0].shape == (0, 2, 5)
    assert torch.equal(acc, old) and torch.equal(kv.k_scales.cpu(), c.scales[0]) and torch.equal(kv.k_pool.cpu(), c.words(0))


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_attention_large_value_scales(gpu, sign, dtype):
    """Value scales of 2^60 at a key whose score is far above those before it: the weighted values stay finite."""
    g = gen(22)
    rows, t, nh, nkv, hd, bs = 40, 470, 4, 2, 128, 16
    c = ref.Cache(g, 1, (t + bs - 1) // bs, bs, nkv, hd)
    c.codes[0].zero_()
    for j in (200, 210):
        c.codes[0][c.slot(0, j)] = 127
        c.scales[0][c.slot(0, j)] = 45.0 / 127 / 128
        c.scales[1][c.slot(0, j)] = sign * 2.0 ** 60
    start, lens = ref.starts([rows]), [t]
    q = torch.ones(rows, nh, hd).to(dtype)
    want, lse, ob, lb = ref.attention(c, q, start, lens, 1.0)  # scores 45 = 65 binades, and 0
    out, got = run_attention(gpu, c, q.to(gpu), start, lens, 1.0)
    near(out, want, ob, "out")
    near(got, lse, lb, "lse")


# ------------------------------------------------------------------ many rows and long sequences together

# Drafts of a few blocks of query vectors over split keys; prompts' pieces with heads of 64 and 128.
LONG = [([20, 1, 11], [3000, 2500, 700], 16, 4, 128, 16), ([9, 20], [1111, 2049], 16, 4, 128, 24), ([70, 5], [1500, 64], 8, 2, 64, 16),
        ([400, 7], [900, 1300], 8, 2, 64, 16), ([150, 90], [1000, 90], 8, 2, 128, 5)]


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("rows,lens,nh,nkv,hd,bs", LONG)
def test_attention_long(gpu, rows, lens, nh, nkv, hd, bs, dtype):
    """With a block outside the pool, and an output that is not aligned."""
    g = gen(sum(lens), nh, hd, bs, 3)
    c = ref.Cache(g, len(rows), (max(lens) + bs - 1) // bs, bs, nkv, hd)
    c.table[0, 300 // bs] = -1
    start = ref.starts(rows)
    total = int(start[-1])
    q = torch.randn(total, nh, hd, generator=g).to(dtype)
    want, lse, ob, lb = ref.attention(c, q, start, lens, 0.1)
    for hints in ({}, dict(max_rows=max(rows), max_len=max(lens))):
        room = torch.full((total * nh * hd + 1,), math.nan, dtype=dtype, device=gpu)
        out, got = run_attention(gpu, c, q.to(gpu), start, lens, 0.1, out=room[1:].view(total, nh, hd), **hints)
        near(out, want, ob, f"out {hints}")
        near(got, lse, lb, f"lse {hints}")
        assert bool(torch.isnan(room[0]))


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("rows", [[20, 3, 0], [1, 1, 1]])
def test_weight_sums_long(gpu, rows, hd, dtype):
    """More keys than there are workgroups at once, with a block outside the pool."""
    g = gen(sum(rows), hd, 4)
    nh, nkv, bs, lens = 32, 8, 16, [3500, 3111, 3300]
    c = ref.Cache(g, 3, (max(lens) + bs - 1) // bs, bs, nkv, hd)
    c.table[1, 100] = -1
    start = ref.starts(rows)
    q = torch.randn(int(start[-1]), nh, hd, generator=g).to(dtype)
    lse = ref.attention(c, q, start, lens, 0.1)[1].float()
    acc = torch.rand(3, nkv, 3600, generator=g)
    want, bound = ref.weight_sums(c, q, lse, start, lens, 0.1, acc)
    dl = torch.tensor(lens, dtype=torch.int32, device=gpu)
    for hints in ({}, dict(max_rows=max(rows), max_len=max(lens))):
        got = ops.paged_weight_sums_i8(q.to(gpu), lse.to(gpu), c.kv(ops, gpu), dl, acc.to(gpu), start.to(gpu), 0.1, **hints)
        near(got, want, bound, f"acc {hints}")


@pytest.mark.parametrize("lens,budget,sink,recent,nkv,hd,bs", EVICT + [([900, 3, 1024, 700], 512, 4, 100, 3, 128, 16),
                                                                       ([900, 3, 1024, 700], 513, 4, 100, 3, 128, 16)])
def test_evict_lens_of_their_own(gpu, lens, budget, sink, recent, nkv, hd, bs):
    """In place, the new lengths beside the old ones or in their place: the same cache, and the old lengths kept in the first case."""
    g = gen(sum(lens), budget, hd, 5)
    c = ref.Cache(g, len(lens), (max(lens) + bs - 1) // bs, bs, nkv, hd)
    acc = torch.randn(len(lens), nkv, max(lens), generator=g).to(gpu)
    dl = torch.tensor(lens, dtype=torch.int32, device=gpu)
    over, apart = c.kv(ops, gpu), c.kv(ops, gpu)
    keep, new = ops.paged_kv_evict_i8(over, dl.clone(), acc, budget, sink, recent, new_lens=(same := dl.clone()))
    ops.paged_kv_evict_i8(apart_ := c.kv(ops, gpu), same2 := dl.clone(), acc, budget, sink, recent, new_lens=same2)
    keep2, new2 = ops.paged_kv_evict_i8(apart, dl, acc, budget, sink, recent)
    want_keep, want_lens = ref.evict(lens, acc.cpu(), budget, sink, recent)
    assert new is same and torch.equal(dl.cpu(), torch.tensor(lens, dtype=torch.int32))
    for k, n in ((keep, new), (keep2, new2), (keep, same2)):
        assert torch.equal(k.cpu(), want_keep) and torch.equal(n.cpu(), want_lens)
    for t in ("k_pool", "v_pool", "k_scales", "v_scales"):
        assert torch.equal(getattr(over, t), getattr(apart_, t)) and torch.equal(getattr(apart, t), getattr(apart_, t)), t
