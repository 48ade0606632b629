"""More of what brain_amd.ops refuses around the int8 paged cache (no GPU needed; tests/test_kvops_validation.py has the rest)."""
import pytest
import torch

from brain_amd import ops
from test_kvops_validation import P, Fake, cache, f, i

PAST = (1 << 32) + 4  # cut to 32 bits: 4


def test_a_cache_is_fixed():
    """A cache holds addresses: a tensor assigned to it would change what it shows and not what the calls read."""
    c, was = cache(), cache().desc.max_blocks
    for name, value in (("block_tables", i(2, 9, ptr=P)), ("k_pool", i(32, 32, ptr=P)), ("v_scales", i(32, 2, ptr=P)), ("block_size", 8),
                        ("sequences", 5)):
        before = getattr(c, name)
        with pytest.raises(AttributeError, match=f"{name} is fixed; make another"):
            setattr(c, name, value)
        assert getattr(c, name) is before
    assert c.desc.max_blocks == was
    assert cache(block_tables=i(2, 9, ptr=P)).desc.max_blocks == 9


def big(*shape, dtype=torch.float32):
    """A tensor of that shape without memory."""
    return Fake(torch.empty(*shape, dtype=dtype, device="meta"), P)


def test_sizes_past_32_bits():
    """What a C entry would see cut to 32 bits is refused, not computed for the rest."""
    c, lens, start = cache(), i(2, ptr=P), i(3, ptr=P)
    freq, pos = f(32, dtype=torch.float64, ptr=P), big(PAST, dtype=torch.int32)

    def no(word, call, *args, **more):
        with pytest.raises(ValueError, match=word):
            call(*args, **more)

    no("block_size", cache, block_size=PAST)
    no("block_tables", cache, block_tables=big(2, PAST, dtype=torch.int32))
    no("block_tables", cache, block_tables=big(PAST, 2, dtype=torch.int32))
    no("kv heads", cache, k_scales=big(1, PAST), v_scales=big(1, PAST), k_pool=big(PAST * 16, dtype=torch.int32), v_pool=big(PAST * 16, dtype=torch.int32))
    no("q: 4294967300 rows", ops.qk_norm_rope, big(PAST, 1, 64), big(PAST, 1, 64), pos, freq)
    no("k: 2 rows of 4294967300 heads", ops.qk_norm_rope, big(2, 1, 64), big(2, PAST, 64), i(2, ptr=P), freq)
    no("head_dim", ops.qk_norm_rope, big(2, 1, PAST), big(2, 1, PAST), i(2, ptr=P), freq)
    no("q: 4294967300 rows", ops.paged_attention_i8, big(PAST, 2, 64), c, lens, start)
    no("q: 2147483648 rows", ops.paged_attention_i8, big(1 << 31, 2, 64), c, lens, start)
    no("acc", ops.paged_weight_sums_i8, big(3, 2, 64), big(3, 2), c, lens, big(2, 2, PAST), start)
    no("acc", ops.paged_kv_evict_i8, c, lens, big(2, 2, PAST), 4)
    no("budget", ops.paged_kv_evict_i8, c, lens, big(2, 2, 16), PAST)
    no("out_tables", ops.paged_kv_evict_i8, c, lens, big(2, 2, 16), 4, out_tables=big(2, PAST, dtype=torch.int32))
    no("acc_out", ops.paged_kv_evict_i8, c, lens, big(2, 2, 16), 4, acc_out=big(2, 2, PAST))


def test_the_largest_sizes_are_taken():
    """What fits in 32 bits is no error of the wrapper's: a block of up to 2^32 - 1 positions, tables as wide."""
    assert cache(block_size=0xFFFFFFFF).desc.block_size == 0xFFFFFFFF
    assert cache(block_tables=big(2, 0xFFFFFFFF, dtype=torch.int32)).desc.max_blocks == 0xFFFFFFFF
