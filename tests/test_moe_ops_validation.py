"""What the mixture-of-experts operators refuse, by the C entry and by brain_amd.ops, before anything reaches the GPU (no GPU needed)."""
import ctypes as C

import numpy as np
import pytest
import torch

import moeref
from brain_amd import load, moe, ops
from brain_amd._lib import BH_ERR_INVALID, BH_OK, BH_OUT_BF16, BH_OUT_F32, BH_OUT_I32, GroupedI8T, MoePlanT, MoeRouterT
from test_kvops_validation import Fake, P, f, i, refused

PAST = (1 << 32) + 4  # cut to 32 bits: 4


def big(*shape, dtype=torch.float32):
    return Fake(torch.empty(*shape, dtype=dtype, device="meta"), P)


def router(**change):
    d = dict(logits=P, stride=60, dtype=BH_OUT_F32, tokens=5, n_experts=60, top_k=4, mask=None, score=0, renormalize=1, scale=1.0)
    d.update(change)
    return C.byref(MoeRouterT(**d))


def plan(**change):
    d = dict(offsets=P, rows=P, slots=P)
    d.update(change)
    return C.byref(MoePlanT(**d))


def group(**change):
    d = dict(xq=P, sx=P, x_rows=20, rows=P, offsets=P, places=30, n_experts=4, wq=P, sw=P, bias=None, kg=16, n=32)
    d.update(change)
    return C.byref(GroupedI8T(**d))


@pytest.mark.parametrize("change,word", [
    (dict(n_experts=0), "0 experts"), (dict(n_experts=1025, stride=1025), "1025 experts"), (dict(top_k=0), "top 0"), (dict(top_k=61), "top 61"),
    (dict(n_experts=100, stride=100, top_k=65), "top 65"), (dict(dtype=BH_OUT_I32), "dtype"), (dict(score=2), "score 2"), (dict(stride=59), "stride 59"),
    (dict(logits=None), "null"), (dict(tokens=1 << 30), "tokens")])
def test_route(change, word):
    refused(load().bh_moe_route(None, router(**change), P, P, None, None, 0), word)


def test_route_buffers():
    lib, n = load(), C.c_uint64()
    refused(lib.bh_moe_route(None, None, P, P, None, None, 0), "null router")
    refused(lib.bh_moe_route(None, router(), None, P, None, None, 0), "null")
    refused(lib.bh_moe_route(None, router(), P, None, None, None, 0), "null")
    for part in ("offsets", "rows", "slots"):
        refused(lib.bh_moe_route(None, router(), P, P, plan(**{part: None}), None, 0), "plan")
        refused(lib.bh_moe_plan_rows(None, P, 5, 4, 0, 60, plan(**{part: None}), None, 0), "plan")
    assert lib.bh_moe_route(None, router(tokens=0, logits=None), None, None, None, None, 0) == BH_OK  # nothing to do
    # A batch of several workgroups: its workspace.
    assert lib.bh_moe_workspace(20000, 4, 60, C.byref(n)) == BH_OK and n.value > 0
    refused(lib.bh_moe_route(None, router(tokens=20000), P, P, plan(), P, n.value - 1), "workspace", str(n.value))
    refused(lib.bh_moe_route(None, router(tokens=20000), P, P, plan(), None, n.value), "workspace")
    refused(lib.bh_moe_route(None, router(tokens=20000), P, P, plan(), P + 2, n.value), "workspace")
    refused(lib.bh_moe_plan_rows(None, P, 20000, 4, 0, 60, plan(), P, n.value - 1), "workspace")
    refused(lib.bh_moe_workspace(5, 4, 60, None), "null")
    refused(lib.bh_moe_workspace(5, 4, 0, C.byref(n)), "0 experts")
    refused(lib.bh_moe_workspace(5, 4, 1025, C.byref(n)), "1025 experts")
    refused(lib.bh_moe_workspace(1 << 31, 1, 8, C.byref(n)), "tokens")
    refused(lib.bh_moe_plan_rows(None, None, 5, 4, 0, 60, plan(), None, 0), "null")
    refused(lib.bh_moe_plan_rows(None, P, 5, 4, 0, 60, None, None, 0), "null")
    refused(lib.bh_moe_plan_rows(None, P, 5, 4, 0, 1025, plan(), None, 0), "experts")
    refused(lib.bh_moe_plan_rows(None, P, 1 << 16, 1 << 15, 0, 8, plan(), None, 0), "choices")


BAD_GROUP = [(dict(places=1 << 31), "range"), (dict(x_rows=1 << 31), "range"), (dict(n_experts=1 << 31), "range"), (dict(n=1 << 31), "range"),
             (dict(kg=1 << 29), "range"), (dict(rows=None), "rows"), (dict(offsets=None), "null"), (dict(xq=None), "null"), (dict(wq=None), "null"),
             (dict(sx=None), "null"), (dict(sw=None), "null"), (dict(places=0x7fffffff, n=0x7ffffffe), "grid")]


@pytest.mark.parametrize("change,word", BAD_GROUP)
def test_grouped(change, word):
    lib = load()
    for fn in (lib.bh_matmul_i8_grouped, lib.bh_matmul_i8_grouped_glu):
        for dtype in (BH_OUT_F32, BH_OUT_BF16):
            refused(fn(None, group(**change), P, dtype), word)


def test_grouped_outputs():
    lib = load()
    refused(lib.bh_matmul_i8_grouped(None, group(), P, 3), "out_dtype 3")
    refused(lib.bh_matmul_i8_grouped_glu(None, group(), P, BH_OUT_I32), "out_dtype")
    refused(lib.bh_matmul_i8_grouped_glu(None, group(n=33), P, BH_OUT_F32), "n=33")
    for fn in (lib.bh_matmul_i8_grouped, lib.bh_matmul_i8_grouped_glu):
        refused(fn(None, None, P, BH_OUT_F32), "null")
        refused(fn(None, group(), None, BH_OUT_F32), "null")
        for nothing in (dict(places=0), dict(n_experts=0), dict(n=0)):  # nothing to do
            assert fn(None, group(xq=None, wq=None, offsets=None, **nothing), None, BH_OUT_F32) == BH_OK


def test_combine():
    lib = load()

    def call(y=P, y_dtype=BH_OUT_F32, places=8, w=P, slots=P, tokens=4, top_k=2, n=16, add=None, out=P, out_dtype=BH_OUT_F32):
        return lib.bh_moe_combine(None, y, y_dtype, places, w, slots, tokens, top_k, n, add, out, out_dtype)

    refused(call(y_dtype=BH_OUT_I32), "dtype")
    refused(call(out_dtype=5), "dtype")
    refused(call(y=None), "null")
    refused(call(w=None), "null")
    refused(call(slots=None), "null")
    refused(call(out=None), "null")
    refused(call(places=1 << 31), "places")
    refused(call(tokens=1 << 31), "tokens")
    refused(call(n=1 << 31), "rows of")
    refused(call(tokens=1 << 20, top_k=1 << 12), "choices")
    assert call(tokens=0, out=None) == BH_OK
    assert call(n=0, out=None) == BH_OK


# ---------------------------------------------------------------- brain_amd.ops

def no(word, call, *args, **more):
    with pytest.raises(ValueError, match=word):
        call(*args, **more)


def test_ops_route():
    x = f(5, 60)
    no("n_experts", ops.moe_route, f(5), 1)
    no("float32 or bfloat16", ops.moe_route, f(5, 60, dtype=torch.float16), 1)
    no("1025 experts", ops.moe_route, f(5, 1025), 1)
    no("0 experts", ops.moe_route, f(5, 0), 1)
    no("top 0", ops.moe_route, x, 0)
    no("top -1", ops.moe_route, x, -1)
    no("top 61", ops.moe_route, x, 61)
    no("top 65", ops.moe_route, f(5, 100), 65)
    no("score", ops.moe_route, x, 4, score="tanh")
    no("side by side", ops.moe_route, Fake(torch.zeros(60, 5).t()), 4)
    no("side by side", ops.moe_route, Fake(torch.zeros(60).expand(5, 60)), 4)
    no("mask", ops.moe_route, x, 4, mask=f(5))
    no("mask", ops.moe_route, x, 4, mask=f(4, dtype=torch.bool))
    no("weights", ops.moe_route, x, 4, weights=f(5, 3))
    no("weights", ops.moe_route, x, 4, weights=i(5, 4))
    no("experts", ops.moe_route, x, 4, experts=f(5, 4))
    no("one GPU", ops.moe_route, x, 4, experts=Fake(torch.zeros(4, 5, dtype=torch.int32).t()))
    no("tokens", ops.moe_route, big(1 << 31, 60), 1)
    no("tokens", ops.moe_route, big(PAST, 60), 1)
    no("must live on the GPU", ops.moe_route, torch.zeros(5, 60), 4)


def test_ops_plan():
    e = i(5, 4)
    no("top_k", ops.moe_plan, i(5), 8)
    no("experts: dtype", ops.moe_plan, f(5, 4), 8)
    no("0 experts", ops.moe_plan, e, 0)
    no("experts, 1 to", ops.moe_plan, e, PAST)
    no("first", ops.moe_plan, e, 8, first=-1)
    no("first", ops.moe_plan, e, 8, first=PAST)
    no("choices", ops.moe_plan, big(1 << 20, 1 << 12, dtype=torch.int32), 8)
    no("choices", ops.moe_plan, big(0, PAST, dtype=torch.int32), 8)
    no("must live on the GPU", ops.moe_plan, torch.zeros(5, 4, dtype=torch.int32), 8)


@pytest.mark.parametrize("change,word", [
    (dict(offsets=i(8)), "plan.offsets"), (dict(offsets=f(9)), "plan.offsets"), (dict(rows=i(19)), "plan.rows"), (dict(slots=i(5, 3)), "plan.slots"),
    (dict(rows=Fake(torch.zeros(40, dtype=torch.int32)[::2])), "one GPU")])
def test_ops_plan_buffers(change, word, monkeypatch):
    monkeypatch.setattr(ops, "_stream_of", lambda dev: 0)
    d = dict(offsets=i(9), rows=i(20), slots=i(5, 4))
    d.update(change)
    no(word, ops.moe_plan, i(5, 4), 8, plan=ops.MoePlan(**d))
    no(word, ops.moe_route, f(5, 8), 4, plan=ops.MoePlan(**d), weights=f(5, 4), experts=i(5, 4))


@pytest.mark.parametrize("call", [ops.matmul_i8_grouped, ops.matmul_i8_grouped_glu])
def test_ops_grouped(call):
    ok = dict(xq=i(20, 16), wq=i(4, 32, 16), sx=f(20), sw=f(4, 32), offsets=i(5), rows=i(30), out=f(30, 32))

    def bad(word, **change):
        no(word, call, **{**ok, **change})

    bad("expected", xq=i(20, 1, 16))
    bad("expected", wq=i(4, 32, 15))
    bad("expected", wq=i(128, 16))
    bad("xq: dtype", xq=f(20, 16))
    bad("wq: dtype", wq=f(4, 32, 16))
    bad("sx", sx=f(19))
    bad("sw", sw=f(4, 31))
    bad("offsets", offsets=i(4))
    bad("offsets: dtype", offsets=f(5))
    bad("rows: dtype", rows=f(30))
    bad("bias", bias=f(4, 31))
    bad("out", out=f(29, 32) if call is ops.matmul_i8_grouped else f(29, 16))
    bad("out_dtype", out_dtype=torch.float16, out=None)
    bad("out: dtype", out_dtype=torch.bfloat16)
    bad("one GPU", wq=Fake(torch.zeros(4, 16, 32, dtype=torch.int32).transpose(1, 2)))
    bad("one GPU", rows=torch.zeros(30, dtype=torch.int32))
    bad("places", rows=big(PAST, dtype=torch.int32))
    bad("places", wq=big(PAST, 32, 16, dtype=torch.int32))
    bad("places", wq=big(4, PAST, 16, dtype=torch.int32))
    bad("places", xq=big(PAST, 16, dtype=torch.int32))
    bad("places", xq=big(20, 1 << 29, dtype=torch.int32), wq=big(4, 32, 1 << 29, dtype=torch.int32))
    if call is ops.matmul_i8_grouped_glu:
        bad("33 weight rows", wq=i(4, 33, 16), sw=f(4, 33))
        bad("out_dtype", out_dtype=torch.int32, out=None)


def test_ops_combine():
    ok = dict(y=f(8, 16), weights=f(4, 2), slots=i(4, 2), out=f(4, 16))

    def bad(word, **change):
        no(word, ops.moe_combine, **{**ok, **change})

    bad("moe_combine: y", y=f(8))
    bad("moe_combine: y", y=i(8, 16))
    bad("moe_combine: y", slots=i(8))
    bad("slots: dtype", slots=f(4, 2))
    bad("weights", weights=f(4, 1))
    bad("weights: dtype", weights=f(4, 2, dtype=torch.bfloat16))
    bad("out", out=f(3, 16))
    bad("out_dtype", out_dtype=torch.int32, out=None)
    bad("add", add=f(3, 16))
    bad("add: dtype", add=f(4, 16, dtype=torch.bfloat16))
    bad("one GPU", y=Fake(torch.zeros(16, 8).t()))
    bad("one GPU", weights=torch.zeros(4, 2))
    bad("places", y=big(PAST, 16))
    bad("places", slots=big(1 << 20, 1 << 12, dtype=torch.int32))


def test_layer_shapes():
    no("do not fit", moe.MoeInt8, i(4, 32, 16), f(4, 32), i(4, 63, 4), f(4, 64), 2)
    no("do not fit", moe.MoeInt8, i(4, 36, 16), f(4, 36), i(4, 64, 4), f(4, 64), 2)
    layer = moe.MoeInt8(i(4, 32, 16), f(4, 32), i(4, 64, 4), f(4, 64), 2)
    no("expected", layer, f(3, 60), f(3, 4))
    no("expected", layer, f(3, 64), f(3, 5))
    no("expected", layer, f(3, 64), f(2, 4))


def test_reference_plan():
    """The oracle itself, by hand."""
    offsets, rows, slots = moeref.plan(np.array([[2, 0], [0, 5], [-1, 2]]), 3)
    assert offsets.tolist() == [0, 2, 2, 4] and rows.tolist() == [0, 1, 0, 2] and slots.tolist() == [[2, 0], [1, -1], [-1, 3]]
    w, e = moeref.route(torch.tensor([[0.0, 3.0, 3.0, float("nan")]]), 2)
    assert e.tolist() == [[1, 2]] and np.allclose(w, 0.5)


def test_packed_descriptions():
    """What brain_amd.ops packs by hand is the C structure."""
    assert ops._route_pack(1, 2, 3, 4, 5, 6, 7, 8, 9, 1.5) == bytes(MoeRouterT(1, 2, 3, 4, 5, 6, 7, 8, 9, 1.5))
    assert ops._plan_pack(1, 2, 3) == bytes(MoePlanT(1, 2, 3))
    assert ops._group_pack(*range(1, 13)) == bytes(GroupedI8T(*range(1, 13)))
