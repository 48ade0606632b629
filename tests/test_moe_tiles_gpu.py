"""Grouped products on every kind of tile that launch_grouped chooses from, with more tiles than the chip holds at once wherever a workgroup stays for
more than one: all output types, gates, bias, rows that x does not have, row tiles partly filled and empty, K of a few stages and of
many. Which kernel a case gets is checked on the CPU (test_moe_dispatch.py)."""
import pytest
import torch

from test_moe_ops_gpu import check_products, gen, offsets_of, operands

pytestmark = pytest.mark.gpu

THIRD = [30, 65, 1, 0, 64, 33, 20, 31] * 5
MIDDLE = [190, 180, 130, 129, 300, 10, 0, 520]
TALL = [2100, 255, 0, 1800]

# (rows of each expert, n, k), and the tile: rows, columns, stages, bytes of a stage, through registers; whether workgroups come to a second one.
CASES = [
    (TALL, 4000, 128, (256, 256, 4, 64, False), True),
    (TALL, 3998, 384, (256, 256, 4, 64, False), True),
    ([300, 1, 2100, 700, 256, 33], 3874, 1152, (256, 256, 4, 64, False), True),
    ([1500] * 3, 3001, 640, (256, 256, 4, 64, False), False),
    (MIDDLE, 4300, 384, (128, 128, 4, 64, False), True),
    (MIDDLE, 4298, 1152, (128, 128, 4, 64, False), True),
    ([100, 200, 30, 129, 256, 127, 0, 158], 1500, 384, (128, 128, 4, 128, False), False),
    ([100, 200, 30, 129, 256, 127, 0, 158], 1502, 1152, (128, 128, 4, 128, False), False),
    ([128] * 8, 1501, 128, (128, 128, 4, 128, False), False),
    (THIRD, 1700, 384, (64, 128, 3, 128, False), True),
    (THIRD, 1702, 1152, (64, 128, 3, 128, False), True),
    ([1 + i % 3 for i in range(300)], 400, 384, (64, 128, 3, 128, False), True),
    ([10, 33, 0, 12, 9, 1, 8, 7] * 5, 1650, 1024, (32, 64, 4, 128, False), True),
    ([10, 33, 0, 12, 9, 1, 8, 7] * 5, 1654, 1152, (32, 64, 4, 128, False), True),
    ([1 + i % 3 for i in range(300)], 400, 1024, (32, 64, 4, 128, False), True),
    ([20, 0, 70, 64], 500, 1152, (64, 128, 6, 128, False), False),
    (THIRD, 1700, 1156, (64, 128, 3, 64, True), True),
    (THIRD, 1702, 60, (64, 128, 3, 64, True), True),
    (MIDDLE, 4300, 500, (128, 128, 3, 64, True), True),
    (MIDDLE, 4298, 1156, (128, 128, 3, 64, True), True),
]
ROWS_OF_X = 170


def places_of(counts):
    return sum(counts) + 5  # some of no group


@pytest.mark.parametrize("counts,n,k", [c[:3] for c in CASES])
def test_tiles(gpu, counts, n, k):
    places = places_of(counts)
    xq, wq, sx, sw, bias = operands(ROWS_OF_X, len(counts), n, k, k + n, gpu)
    rows = torch.randint(0, ROWS_OF_X, (places,), generator=gen(n), dtype=torch.int32)
    # The first expert's rows are all there (whole tiles go out another way then), of the last one's some are not.
    last = sum(counts[:-1]) + torch.randint(0, counts[-1], (1 + counts[-1] // 9,), generator=gen(k))
    rows[last] = torch.tensor([ROWS_OF_X, -1, 2 ** 31 - 1, -2 ** 31], dtype=torch.int32)[torch.arange(len(last)) % 4]
    check_products(gpu, xq, wq, sx, sw, bias, offsets_of(counts, gpu), rows.to(gpu))


@pytest.mark.parametrize("counts,n,k", [(TALL, 4000, 128), ([1500] * 3, 3002, 1152), (MIDDLE, 4300, 384)])
def test_tiles_without_rows(gpu, counts, n, k):
    xq, wq, sx, sw, bias = operands(places_of(counts), len(counts), n, k, k + n, gpu)
    check_products(gpu, xq, wq, sx, sw, bias, offsets_of(counts, gpu), None)


@pytest.mark.parametrize("counts,n,k", [(TALL, 4000, 1152), (MIDDLE, 4300, 1152), (THIRD, 1700, 1152)])
def test_tiles_repeat(gpu, counts, n, k):
    """The same call again and again, beside copies that keep the memory busy: the same bits."""
    from brain_amd import ops

    xq, wq, sx, sw, bias = operands(ROWS_OF_X, len(counts), n, k, 1, gpu)
    rows = torch.randint(0, ROWS_OF_X, (places_of(counts),), generator=gen(1), dtype=torch.int32).to(gpu)
    offsets = offsets_of(counts, gpu)
    want = ops.matmul_i8_grouped(xq, wq, sx, sw, offsets, rows, out_dtype=torch.int32)
    side, a = torch.cuda.Stream(), torch.randn(1 << 26, device=gpu)
    b = torch.empty_like(a)
    torch.cuda.synchronize()
    real = int(offsets[-1])
    for _ in range(20):
        with torch.cuda.stream(side):
            for _ in range(4):
                b.copy_(a)
        out = ops.matmul_i8_grouped(xq, wq, sx, sw, offsets, rows, out_dtype=torch.int32)
        torch.cuda.synchronize()
        assert torch.equal(out[:real], want[:real])
