"""What the int8 paged cache's operators refuse, by the C entry and by brain_amd.ops, before anything reaches the GPU (no GPU
needed: the checks come first)."""
import ctypes as C

import pytest
import torch

from brain_amd import load, ops
from brain_amd._lib import BH_ERR_INVALID, BH_OK, BH_OUT_BF16, BH_OUT_F32, BH_OUT_I32, Kv8BatchT, Kv8T, QkRowsT

P = 4096  # a pointer that nothing may follow


def kv(**change):
    d = dict(k_pool=P, v_pool=P, k_scales=P, v_scales=P, pool_words=8 * 16 * 32, n_scales=8 * 16, block_tables=P, max_blocks=4,
             block_size=16, n_kv_heads=2, head_dim=64)
    d.update(change)
    return C.byref(Kv8T(**d))


def batch(**change):
    d = dict(row_start=P, seq_lens=P, batch=2, rows=5, max_rows=3, max_len=20)
    d.update(change)
    return C.byref(Kv8BatchT(**d))


def rows(**change):
    d = dict(q=P, k=P, v=P, q_stride=512, k_stride=512, v_stride=512, dtype=BH_OUT_F32, rows=5, n_heads=4, n_kv_heads=2,
             head_dim=64, positions=P, inv_freq=P, rotary_dim=64, q_weight=P, k_weight=P, eps=1e-6)
    d.update(change)
    return C.byref(QkRowsT(**d))


def refused(rc, *words):
    text = load().bh_last_error().decode()
    assert rc == BH_ERR_INVALID, rc
    assert all(w in text for w in words), text


BAD_KV = [(dict(head_dim=0), "head_dim 0"), (dict(head_dim=66), "head_dim 66"), (dict(head_dim=260), "head_dim 260"),
          (dict(n_kv_heads=0), "0 kv heads"), (dict(block_size=0), "block_size 0"), (dict(k_pool=None), "null"),
          (dict(v_scales=None), "null"), (dict(block_tables=None), "null"), (dict(max_blocks=0), "max_blocks 0"), (dict(n_kv_heads=1 << 26), "fit")]


@pytest.mark.parametrize("change,word", BAD_KV)
def test_cache(change, word):
    lib, n = load(), C.c_uint64()
    refused(lib.bh_paged_attention_i8(None, P, 256, BH_OUT_F32, 4, kv(**change), batch(), 0.1, P, P, None, 0), word)
    refused(lib.bh_paged_attention_i8_workspace(kv(**change), batch(), 4, C.byref(n)), word)
    refused(lib.bh_paged_weight_sums_i8(None, P, 256, BH_OUT_F32, 4, P, kv(**change), batch(), 0.1, P, 64), word)
    refused(lib.bh_paged_kv_evict_i8(None, kv(**change), P, 2, P, 64, 8, 1, 1, None, 0, None, 0, P, P), word)
    refused(lib.bh_qk_norm_rope_append_i8(None, rows(), kv(**change), batch(), None, None, P, 256), word)


@pytest.mark.parametrize("change,word", [(dict(seq_lens=None), "lengths"), (dict(row_start=None), "row_start")])
def test_batch(change, word):
    lib = load()
    refused(lib.bh_paged_attention_i8(None, P, 256, BH_OUT_F32, 4, kv(), batch(**change), 0.1, P, P, None, 0), word)
    refused(lib.bh_paged_weight_sums_i8(None, P, 256, BH_OUT_F32, 4, P, kv(), batch(**change), 0.1, P, 64), word)
    refused(lib.bh_qk_norm_rope_append_i8(None, rows(), kv(), batch(**change), None, None, P, 256), word)


def test_attention_and_sums():
    lib = load()

    def attend(q=P, stride=256, dtype=BH_OUT_BF16, heads=4, out=P):
        return lib.bh_paged_attention_i8(None, q, stride, dtype, heads, kv(), batch(), 0.1, out, None, None, 0)

    def sums(q=P, stride=256, dtype=BH_OUT_BF16, heads=4, lse=P, acc=P):
        return lib.bh_paged_weight_sums_i8(None, q, stride, dtype, heads, lse, kv(), batch(), 0.1, acc, 64)

    for call in (attend, sums):
        refused(call(dtype=BH_OUT_I32), "dtype")
        refused(call(heads=0), "heads")
        refused(call(heads=3), "3 query heads over 2 kv heads")
        refused(call(heads=1 << 30), "heads")
        refused(call(stride=255), "row stride 255")
        refused(call(q=None), "null")
    refused(attend(out=None), "null")
    refused(sums(lse=None), "null")
    refused(sums(acc=None), "null")
    refused(lib.bh_paged_attention_i8_workspace(kv(), batch(), 4, None), "null")
    refused(lib.bh_paged_attention_i8(None, P, 256, 0, 4, None, batch(), 0.1, P, P, None, 0), "no cache")
    refused(lib.bh_paged_attention_i8(None, P, 256, 0, 4, kv(), None, 0.1, P, P, None, 0), "no batch")
    # Nothing to do is no error.
    none = batch(batch=0, rows=0, row_start=None, seq_lens=None)
    assert lib.bh_paged_attention_i8(None, None, 0, 0, 4, kv(), none, 0.1, None, None, None, 0) == BH_OK
    assert lib.bh_paged_weight_sums_i8(None, None, 0, 0, 4, None, kv(), none, 0.1, None, 64) == BH_OK


def test_norm_rope():
    lib = load()
    call = lambda r, q=P, qs=256, k=P, ks=128: lib.bh_qk_norm_rope(None, r, q, qs, k, ks)  # noqa: E731
    refused(call(rows(dtype=BH_OUT_I32)), "dtype")
    refused(call(rows(head_dim=30)), "head_dim 30")
    refused(call(rows(head_dim=512)), "head_dim 512")
    refused(call(rows(rotary_dim=7)), "rotary_dim 7")
    refused(call(rows(rotary_dim=66)), "rotary_dim 66")
    refused(call(rows(n_heads=0)), "0 query heads")
    refused(call(rows(n_kv_heads=0)), "0 kv heads")
    refused(call(rows(rows=1 << 30)), "rows")
    refused(call(rows(q_stride=255)), "row strides")
    refused(call(rows(k_stride=127)), "row strides")
    for name in ("q", "k", "positions", "inv_freq"):
        refused(call(rows(**{name: None})), "null")
    refused(call(rows(), q=None), "null")
    refused(call(rows(), k=None), "null")
    refused(call(rows(), qs=255), "output row strides")
    refused(call(rows(), ks=1), "output row strides")
    refused(lib.bh_qk_norm_rope(None, None, P, 256, P, 128), "no rows")
    assert call(rows(rows=0, q=None, k=None, positions=None), q=None, k=None) == BH_OK
    app = lambda r, b=batch(), q=P, qs=256: lib.bh_qk_norm_rope_append_i8(None, r, kv(), b, None, None, q, qs)  # noqa: E731
    refused(app(rows(v=None)), "null")
    refused(app(rows(v_stride=127)), "row strides")
    refused(app(rows(rows=4)), "batch of 5")
    refused(app(rows(head_dim=32, rotary_dim=32)), "cache of 2 of 64")
    refused(app(rows(n_kv_heads=1)), "cache of 2 of 64")
    refused(app(rows(), q=None), "null")
    refused(app(rows(), qs=255), "output row stride")


def test_evict():
    lib = load()

    def call(lens=P, n=2, acc=P, cap=64, budget=8, sink=2, recent=2, to=None, cols=0, acc_out=None, cap_out=0, keep=P, new=P):
        return lib.bh_paged_kv_evict_i8(None, kv(), lens, n, acc, cap, budget, sink, recent, to, cols, acc_out, cap_out, keep, new)

    refused(call(budget=0), "budget of 0")
    refused(call(sink=5, recent=4), "5 first and 4 last")
    refused(call(sink=0xFFFFFFFF, recent=2), "first")
    refused(call(budget=1 << 31, sink=0), "budget")
    refused(call(cap=1 << 31), "acc_stride")
    for name in ("lens", "acc", "keep", "new"):
        refused(call(**{name: None}), "null")
    refused(call(acc_out=P + 4096, cap_out=7), "acc_out")
    refused(call(acc_out=P, cap_out=32), "acc_out")
    refused(call(n=1 << 30), "grid")
    refused(call(to=P, cols=0), "out_max_blocks")
    assert call(n=0, lens=None, acc=None, keep=None, new=None) == BH_OK


class Fake:
    """A CPU tensor that says it is on GPU 0; whoever asks for its memory launches."""

    def __init__(self, t, ptr=None):
        self.t, self.ptr = t, ptr

    def get_device(self):
        return 0

    def __getattr__(self, name):
        return getattr(self.t, name)

    def data_ptr(self):
        assert self.ptr, "reached a launch"
        return self.ptr


def f(*shape, dtype=torch.float32, ptr=None):
    return Fake(torch.zeros(*shape, dtype=dtype), ptr)


def i(*shape, ptr=None):
    return f(*shape, dtype=torch.int32, ptr=ptr)


def cache(**change):
    d = dict(k_pool=i(32, 32, ptr=P), v_pool=i(32, 32, ptr=P), k_scales=f(32, 2, ptr=P), v_scales=f(32, 2, ptr=P),
             block_tables=i(2, 4, ptr=P), block_size=4, head_dim=64)
    d.update(change)
    return ops.PagedKV8(**d)


@pytest.mark.parametrize("change,word", [
    (dict(head_dim=62), "head_dim"), (dict(head_dim=0), "head_dim"), (dict(block_size=0), "block_size"), (dict(k_pool=f(32, 32)), "k_pool"),
    (dict(v_pool=i(31, 32)), "v_pool"), (dict(k_scales=f(64)), "scales"), (dict(v_scales=f(31, 2)), "v_scales"),
    (dict(block_tables=f(2, 4)), "block_tables"), (dict(block_tables=i(8)), "block_tables")])
def test_ops_cache(change, word):
    with pytest.raises(ValueError, match=word):
        cache(**change)


def test_ops_attention():
    c = cache()
    ok = dict(q=f(3, 4, 64), cache=c, seq_lens=i(2, ptr=P), row_start=i(3, ptr=P), out=f(3, 4, 64), lse=f(3, 4))

    def no(word, **change):
        with pytest.raises(ValueError, match=word):
            ops.paged_attention_i8(**dict(ok, **change))

    no("q: dtype", q=f(3, 4, 64, dtype=torch.float16))
    no("q: shape", q=f(3, 4, 32))
    no("q: 3 heads", q=f(3, 3, 64))
    no("strides", q=Fake(torch.zeros(3, 64, 4).transpose(1, 2)))
    no("seq_lens: dtype", seq_lens=f(2))
    no("sequences", seq_lens=i(3), row_start=i(4))
    no("row_start", row_start=None)
    no("row_start", row_start=i(2))
    no("row_start", row_start=i(4))
    no("out: dtype", out=f(3, 4, 64, dtype=torch.bfloat16), lse=f(3, 4))
    no("out: 700", out=f(700), lse=f(3, 4))
    no("lse: 11", out=f(3, 4, 64), lse=f(11))
    no("one GPU", lse=torch.zeros(3, 4))
    no("one GPU", row_start=Fake(torch.zeros(6, dtype=torch.int32)[::2], ptr=P))
    no("q is on -1", q=torch.zeros(3, 4, 64))
    with pytest.raises(ValueError, match="acc"):
        ops.paged_weight_sums_i8(ok["q"], f(3, 4), c, ok["seq_lens"], f(2, 3, 9), ok["row_start"])
    with pytest.raises(ValueError, match="acc"):
        ops.paged_weight_sums_i8(ok["q"], f(3, 4), c, ok["seq_lens"], f(1, 2, 9), ok["row_start"])
    with pytest.raises(ValueError, match="lse"):
        ops.paged_weight_sums_i8(ok["q"], f(3, 3), c, ok["seq_lens"], f(2, 2, 9), ok["row_start"])


def test_ops_norm_rope():
    q, k, v, pos, freq = f(3, 4, 64), f(3, 2, 64), f(3, 2, 64), i(3), f(32, dtype=torch.float64)

    def no(word, *args, **more):
        with pytest.raises(ValueError, match=word):
            ops.qk_norm_rope(*args, **more)

    no("q: dtype", f(3, 4, 64, dtype=torch.float64), k, pos, freq)
    no("k: dtype", q, f(3, 2, 64, dtype=torch.bfloat16), pos, freq)
    no("k: shape", q, f(3, 2, 32), pos, freq)
    no("k: 2 rows", q, f(2, 2, 64), pos, freq)
    no("positions", q, k, f(3), freq)
    no("positions", q, k, i(2), freq)
    no("inv_freq: dtype", q, k, pos, f(32))
    no("inv_freq: 33", q, k, pos, f(33, dtype=torch.float64))
    no("q_weight", q, k, pos, freq, f(32))
    no("k_weight", q, k, pos, freq, None, f(64, dtype=torch.bfloat16))
    ptr = dict(ptr=P)
    args = (f(3, 4, 64, **ptr), f(3, 2, 64, **ptr), f(3, 2, 64, **ptr), i(3, **ptr), f(32, dtype=torch.float64, **ptr))
    no("q_out", args[0], args[1], args[3], args[4], q_out=f(3, 4, 60))
    no("k_out", args[0], args[1], args[3], args[4], q_out=f(3, 4, 64), k_out=f(3, 4, 64))

    def not_appended(word, *a, **more):
        with pytest.raises(ValueError, match=word):
            ops.qk_norm_rope_append_i8(*a, **more)

    lens, start = i(2, ptr=P), i(3, ptr=P)
    not_appended("v: shape", args[0], args[1], f(3, 1, 64), args[3], args[4], cache(), lens, start)
    not_appended("cache has", args[0], f(3, 1, 64, **ptr), f(3, 1, 64, **ptr), args[3], args[4], cache(), lens, start)
    not_appended("row_start", *args, cache(), lens)
    not_appended("k_clip", *args, cache(), lens, start, k_clip=f(1))
    not_appended("v_clip", *args, cache(), lens, start, v_clip=i(2))


def test_ops_evict():
    c, lens, acc = cache(), i(2), f(2, 2, 16)

    def no(word, *args, **more):
        with pytest.raises(ValueError, match=word):
            ops.paged_kv_evict_i8(*args, **more)

    no("budget", c, lens, acc, 0)
    no("budget", c, lens, acc, 4, 3, 2)
    no("budget", c, lens, acc, 4, -1, 2)
    no("acc", c, lens, f(2, 1, 16), 4)
    no("acc", c, lens, f(1, 2, 16), 4)
    no("seq_lens", c, f(2), acc, 4)
    no("sequences", c, i(3), f(3, 2, 16), 4)
    no("out_tables", c, lens, acc, 4, out_tables=f(2, 2))
    no("out_tables", c, lens, acc, 4, out_tables=i(1, 2))
    no("acc_out", c, lens, acc, 4, acc_out=f(2, 1, 4))
    no("keep", c, lens, acc, 4, keep=i(2, 2, 3), new_lens=i(2))
    no("new_lens", c, lens, acc, 4, keep=i(2, 2, 4), new_lens=i(1))


def test_sizes_at_the_ends():
    lib = load()
    for some in (dict(batch=0, rows=0, row_start=None, seq_lens=None), dict(batch=0, rows=0), dict(rows=0)):
        n = C.c_uint64(1)
        assert lib.bh_paged_attention_i8_workspace(kv(), batch(**some), 4, C.byref(n)) == BH_OK and n.value == 0
    refused(lib.bh_paged_attention_i8_workspace(kv(), batch(batch=1 << 30), 4, C.byref(C.c_uint64())), "sequences")
    refused(lib.bh_paged_weight_sums_i8(None, P, 256, 0, 4, P, kv(), batch(), 0.1, P, 0x7FFFFFFF), "acc_stride")
    # max_blocks * block_size past 32 bits: no more than the positions there can be.
    n = C.c_uint64()
    assert lib.bh_paged_attention_i8_workspace(kv(max_blocks=0xFFFFFFFF, block_size=1 << 20), batch(max_len=0), 4, C.byref(n)) == BH_OK
    assert 0 < n.value < 1 << 22  # 2 blocks of 16 vectors, 2 heads, 64 splits at most
    # Tables without room for what is kept.
    evict = lambda budget, cap, cols: lib.bh_paged_kv_evict_i8(None, kv(), P, 2, P, cap, budget, 0, 0, P + 64, cols, None, 0,  # noqa: E731
                                                               P, P)
    refused(evict(9, 64, 8 // kv()._obj.block_size), "for 9 positions")
    refused(evict(64, 9, 8 // kv()._obj.block_size), "for 9 positions")
