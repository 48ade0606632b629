"""The order of the 256 x 256 kernels' waves (brain_amd/csrc/bh_pingpong.h), compiled alone and walked: a wave reads a stage, or has it
overwritten, only behind a barrier that every wave has reached after what had to come first."""
import os
import re
import subprocess

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "brain_amd", "csrc")

MAIN = r"""
#include "bh_pingpong.h"
#include <cstdio>
#include <cstdlib>
#include <vector>
static int stages, nk;
#define CHECK(x) do { if (!(x)) { std::printf("line %d: %s (%d stages deep, %d of K)\n", __LINE__, #x, stages, nk); std::exit(1); } } while (0)
// What a wave of a group does, each with the barriers that the wave has passed by then.
struct Walk {
    int barriers = 0, products = 0, copied = 0;  // stages asked for
    std::vector<int> landed, asked, read;        // by stage
};
template <int STAGES>
static Walk walk(int group) {
    Walk w;
    w.landed.assign(nk, 1 << 30), w.asked.assign(nk, 1 << 30), w.read.assign(nk, 1 << 30);
    auto ask = [&](int s) {
        CHECK(s == w.copied);
        w.asked[w.copied++] = w.barriers;
    };
    for (int s = 0; s < STAGES - 1 && s < nk; ++s) ask(s);
    bh::ping_pong<STAGES>(
        group, nk,
        [&](auto most, int ahead) {
            CHECK(ahead <= decltype(most)::value);
            for (int s = 0; s < w.copied - (ahead > 0 ? ahead : 0); ++s)
                if (w.landed[s] > w.barriers) w.landed[s] = w.barriers;
        },
        [&] { ++w.barriers; },
        [&](int it) {
            CHECK(it == w.products);
            w.read[it] = w.barriers;
            if (it + STAGES - 1 < nk) ask(it + STAGES - 1);
        },
        [&] {
            CHECK(w.barriers > w.read[w.products]);  // read ends before the phase's barrier
            ++w.products;
        });
    CHECK(w.products == nk && w.copied == nk);
    return w;
}
template <int STAGES>
static void check() {
    stages = STAGES;
    for (nk = 0; nk < 40; ++nk) {
        const Walk w[2] = {walk<STAGES>(0), walk<STAGES>(1)};
        CHECK(w[0].barriers == w[1].barriers);
        // Any wave u reads, any wave v copies; both can be of one group.
        for (const Walk& u : w)
            for (const Walk& v : w)
                for (int s = 0; s < nk; ++s) {
                    CHECK(v.landed[s] < u.read[s]);  // v's share has landed before a barrier ahead of u's read
                    if (s >= STAGES) CHECK(u.read[s - STAGES] < v.asked[s]);  // and its buffer was read by then
                }
        // One group multiplies while the other reads.
        for (int s = 0; s < nk; ++s) CHECK(w[1].read[s] == w[0].read[s] + 1);
    }
}
int main() {
    check<3>();
    check<4>();
    check<5>();
    check<6>();
    return 0;
}
"""


def test_every_read_is_behind_every_copy(tmp_path):
    src, exe = tmp_path / "order.cpp", tmp_path / "order"
    src.write_text(MAIN)
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", "-I", CSRC, str(src), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True)
    assert out.returncode == 0, out.stdout


def test_the_kernels_take_their_order_from_there():
    """The two kernels that run their waves in two groups call ping_pong, and none has a group's barrier of its own."""
    callers = []
    for name in sorted(os.listdir(CSRC)):
        with open(os.path.join(CSRC, name)) as f:
            text = f.read()
        if name.endswith(".hip"):
            callers += [name] * len(re.findall(r"\bping_pong<", text))
            assert not re.search(r"if \((group|grp) == [01]\)", text), name
    assert callers == ["bh_gemm.hip", "bh_grouped.hip"]
