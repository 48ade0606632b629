"""Lengths at their ends (brain_amd/csrc/bh_kvlen.h), compiled alone: whatever a program's seq_lens hold, a row sees no more keys
than the table has positions, the loops over them (64 or 128 at a time) end, and no sum wraps."""
import os
import subprocess

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "brain_amd", "csrc")

MAIN = r"""
#include "bh_kvlen.h"
#include <algorithm>
#include <cstdio>
#include <cstdlib>
#define CHECK(x) do { if (!(x)) { std::printf("line %d: %s (length %lld, row %u of %u)\n", __LINE__, #x, len, i, n); std::exit(1); } } while (0)
int main() {
    long long len = 0;
    uint32_t n = 1, i = 0;
    const long long lens[] = {0, 1, 2, 5, 63, 64, 65, 1 << 20, 0x7ffeffffll, 0x7fff0000ll, 0x7fffffffll, -1, -2, -5, -64, -(1ll << 31)};
    const uint32_t rows[] = {1, 2, 5, 64, 1000, 0x7fffffffu};
    const uint32_t tables[][2] = {{1, 1}, {4, 16}, {1, 0xffffffffu}, {0xffffffffu, 0xffffffffu}, {0xffffffffu, 1}, {0x7fff, 0x10000}};
    for (auto& t : tables) {
        const uint32_t reach = bh::kv_reach(t[0], t[1]);
        CHECK(reach == std::min<unsigned __int128>((unsigned __int128)t[0] * t[1], bh::KV_REACH));
        for (long long l : lens)
            for (uint32_t nn : rows)
                for (uint32_t ii : {0u, 1u, nn / 2, nn - 1}) {
                    len = l, n = nn, i = std::min(ii, nn - 1);
                    // The row's position is len - n + i; it sees the keys up to its own.
                    const long long want = std::min<long long>(std::max<long long>(0, std::max(0ll, len) - n + i + 1), reach);
                    const uint32_t seen = std::min(bh::kv_keys_seen(bh::kv_length((uint32_t)len), n, i), reach);
                    CHECK(seen == want);
                    for (uint32_t step : {64u, 128u}) {
                        const uint32_t last = seen ? (seen - 1) / step * step : 0;  // the loop's last start
                        CHECK(last + step >= seen && last + step > last);
                    }
                }
    }
    return 0;
}
"""


def test_lengths(tmp_path):
    src, exe = tmp_path / "len.cpp", tmp_path / "len"
    src.write_text(MAIN)
    subprocess.run(["g++", "-std=c++17", "-Wall", "-I", CSRC, str(src), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True)
    assert out.returncode == 0, out.stdout
