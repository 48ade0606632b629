"""The workspace of paged_attention_i8 for batches that mix single tokens with longer chunks: it goes with the rows of the call,
not with the blocks that each sequence begins (bh_paged_attention_i8_workspace, no GPU needed)."""
import ctypes as C

import pytest

from brain_amd import load
from brain_amd._lib import BH_OK, Kv8BatchT, Kv8T

P = 4096  # a pointer that nothing may follow


def workspace(batch, rows, max_rows, max_len, heads=32, kv_heads=8, hd=128, bs=32, ragged=True):
    kv = Kv8T(P, P, P, P, 1 << 34, 1 << 28, P, -(-max_len // bs), bs, kv_heads, hd)
    b, n = Kv8BatchT(P if ragged else None, P, batch, rows, max_rows, max_len), C.c_uint64()
    assert load().bh_paged_attention_i8_workspace(C.byref(kv), C.byref(b), heads, C.byref(n)) == BH_OK
    return n.value


@pytest.mark.parametrize("batch,rows,max_rows,max_len", [
    (64, 63 + 256, 256, 8192), (64, 63 + 41, 41, 8192), (256, 255 + 256, 256, 32768), (256, 255 + 41, 41, 32768),
    (512, 511 + 64, 64, 8192), (64, 64, 0, 8192), (256, 256, 0, 32768)])
def test_single_tokens_beside_a_chunk(batch, rows, max_rows, max_len):
    """At most 32 splits of the rows' own sums, and less than 150 MiB."""
    assert workspace(batch, rows, max_rows, max_len) <= min(150 << 20, 32 * rows * 32 * (128 + 2) * 4)


def test_steps():
    """A step's 64 splits at most, however the call says that each sequence has one row."""
    for hint, ragged in ((0, True), (1, True), (0, False)):
        assert workspace(64, 64, hint, 8192, ragged=ragged) <= 64 * 64 * 32 * 130 * 4
