"""Which kernel a grouped product gets, on the CPU (see test_dispatch.py for how): the cases of test_moe_tiles_gpu.py reach the tile that they are meant
for in every form, and few rows the kernel without tiles."""
import json
import os
import re
import subprocess
import sys

import pytest

from test_dispatch import FAKE, ROOT
from test_moe_tiles_gpu import CASES, ROWS_OF_X, places_of

CHILD = r"""
import ctypes as C, json, sys
fake = C.CDLL(sys.argv[1], mode=C.RTLD_GLOBAL)
from brain_amd import load
from brain_amd._lib import GroupedI8T
lib = load()
fake.fake_log.restype = C.c_char_p
A = 1 << 20
out = []
for rows, places, experts, n, k in json.loads(sys.stdin.read()):
    names = []
    for bias in (None, A):
        g = GroupedI8T(A, A, rows, A, A, places, experts, A, A, bias, k // 4, n)
        for fn, types in ((lib.bh_matmul_i8_grouped, (0, 1, 2)), (lib.bh_matmul_i8_grouped_glu, (0, 1) if n % 2 == 0 else ())):
            for t in types:
                fake.fake_clear()
                assert fn(None, C.byref(g), A, t) == 0
                names += fake.fake_log().decode().split()
    out.append(names)
print(json.dumps(out))
"""


@pytest.fixture(scope="module")
def kernels(tmp_path_factory):
    d = tmp_path_factory.mktemp("fakehip")
    src, so = d / "fake.cpp", d / "libfakehip.so"
    src.write_text(FAKE)
    subprocess.run(["g++", "-std=c++17", "-shared", "-fPIC", str(src), "-o", str(so), "-ldl"], check=True)

    def run(calls):
        p = subprocess.run([sys.executable, "-c", CHILD, str(so)], input=json.dumps(calls), capture_output=True, text=True, cwd=ROOT)
        assert p.returncode == 0, p.stderr
        return json.loads(p.stdout.splitlines()[-1])

    return run


def tile_of(name):
    """(rows, columns, stages, bytes, through registers) and the workgroups of a compute unit, of a kernel's name."""
    m = re.search(r"grouped_tile_kernelINS_7TileCfgI((?:L[ib]\d+E)+)EELi(\d)ELb(\d)ELb(\d)ELb(\d)E", name)
    cfg = [int(v) for v in re.findall(r"L[ib](\d+)E", m.group(1))]
    return (cfg[0], cfg[1], cfg[4], cfg[5], m.group(5) == "1"), cfg[6], m.groups()[1:4]


def test_cases_reach_their_tiles(kernels):
    got = kernels([(ROWS_OF_X, places_of(c[0]), len(c[0]), c[1], c[2]) for c in CASES])
    for (counts, n, k, want, again), names in zip(CASES, got):
        assert len(names) == (10 if n % 2 == 0 else 6)
        forms = set()
        for name in names:
            tile, per_unit, form = tile_of(name)
            assert tile == want, (counts, n, k, name)
            forms.add(form)
        # Types x gate x bias (raw sums have none).
        assert len(forms) == (9 if n % 2 == 0 else 5)
        tiles = sum(-(-c // want[0]) for c in counts) * -(-n // want[1])
        assert (tiles > 256 * per_unit) == again, (counts, n, k, tiles)


def test_every_tile_has_a_case():
    """The kinds of tile that launch_grouped names."""
    with open(os.path.join(ROOT, "brain_amd", "csrc", "bh_grouped.hip")) as f:
        text = f.read()
    kinds = {(int(a), int(b), int(s), int(d), reg == "true") for a, b, s, d, reg in re.findall(
        r"launch_tiles<TileCfg<(\d+), (\d+), \d+, \d+, (\d+), (\d+), \d+, \w+, \w+>, OUT, GLU, (\w+)>", text)}
    assert kinds == {c[3] for c in CASES}


def test_few_rows(kernels):
    for names in kernels([(1, 8, 128, 1536, 2048), (1, 8, 128, 2048, 768), (1, 1, 1, 64, 4), (20, 40, 8, 8184, 2044)]):
        assert all("grouped_step_kernel" in n for n in names)


def test_no_rows_of_x(kernels):
    assert all("grouped_zero_kernel" in n for n in kernels([(0, 5, 2, 8, 64)])[0])
