"""More of what brain_amd.ops refuses around the int8 paged cache (no GPU needed; tests/test_kvops_validation.py has the rest)."""
import pytest

from test_kvops_validation import P, cache, i


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
