"""The tiles of the grouped product's workgroups (brain_amd/csrc/bh_tilespan.h), compiled alone: every tile is one workgroup's, and the loops over
them end whatever counts the offsets on the device add up to."""
import os
import subprocess

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "brain_amd", "csrc")

MAIN = r"""
#include "bh_tilespan.h"
#include <algorithm>
#include <cstdio>
#include <cstdlib>
#include <vector>
#define CHECK(x) do { if (!(x)) { std::printf("line %d: %s (%u x %u tiles, at most %u, workgroup %u of %u)\n", __LINE__, #x, rows, cols, most, w, wgs); std::exit(1); } } while (0)
int main() {
    uint32_t w = 0;
    const uint32_t counts[] = {0, 1, 2, 7, 8, 9, 63, 64, 65, 1000, 65535, 65536, 0x7fffffff, 0x80000000u, 0xfffffff0u, 0xffffffffu};
    const uint32_t columns[] = {1, 2, 3, 12, 257, 4096, 65536, 0xffffff};
    for (uint32_t rows : counts)
        for (uint32_t cols : columns)
            for (uint32_t most : {1u, 8u, 600u, 0x7fffffffu})
                for (uint32_t wgs : {8u, 16u, 256u, 512u, 768u}) {
                    const uint64_t tiles = std::min<uint64_t>((uint64_t)rows * cols, most);
                    std::vector<uint8_t> taken(tiles <= 5000 ? tiles : 0);
                    uint64_t before = 0;
                    for (w = 0; w < wgs; ++w) {
                        const bh::TileSpan s = bh::tile_span(rows, cols, most, w, wgs);
                        CHECK(s.step > 0 && s.end <= tiles);
                        if (s.at >= s.end) continue;
                        CHECK((uint64_t)s.end + s.step < 1ull << 32);  // the loop's last step does not wrap
                        before += (s.end - s.at + s.step - 1) / s.step;
                        if (tiles <= 5000)
                            for (uint32_t i = s.at; i < s.end; i += s.step) {
                                CHECK(!taken[i]);
                                taken[i] = 1;
                            }
                    }
                    CHECK(before == tiles);
                }
    return 0;
}
"""


def test_every_tile_once(tmp_path):
    src, exe = tmp_path / "span.cpp", tmp_path / "span"
    src.write_text(MAIN)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-I", CSRC, str(src), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True)
    assert out.returncode == 0, out.stdout
