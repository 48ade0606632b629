// The order of a matrix kernel's waves, in plain C++ (no HIP in here: the CPU tests compile it alone and walk it).
//
// The waves of a workgroup form two groups, one wave of each on every SIMD, that run a phase apart: on
// every SIMD one multiplies while the other reads LDS and asks for copies. Each of nk stages
// takes a wave two phases, R (read the stage's fragments into registers, ask for the
// copies of stage + STAGES - 1, wait for the fragments) and M (multiply), each closed by a workgroup barrier.
// Group 1 starts a barrier late and group 0 ends one later.
//
//   barriers passed    1     2     3     4     5   ...
//   group 0           R(0)  M(0)  R(1)  M(1)  R(2)
//   group 1                 R(0)  M(0)  R(1)  M(1)
//
// A stage is copied by every wave of both groups, and a wave can wait for its own copies
// only. So whoever reads stage s does that behind a barrier that every wave has
// reached after its wait for s: group 0 waits at the end of its M(s - 1), group 1 at the beginning of its R(s - 1),
// both ahead of the barrier before group 0's R(s). For stage 0 all wait before a common first barrier.
//   The copies of R(s) go to the buffer of stage s - 1, whose fragments
// group 0 has in registers since a phase before and group 1 since the barrier just before group 0's R(s).
#pragma once
#include <type_traits>

namespace bh {

// wait(most, ahead): until at most `ahead` <= most stages of this wave's copies are on their way (below 0: none; `most` is an
// integral constant). Stages 0 .. STAGES - 2 have been asked for, as far as there are so many. group: of this wave, 0 or 1.
template <int STAGES, class Wait, class Barrier, class Read, class Multiply>
__attribute__((always_inline)) constexpr void ping_pong(int group, int nk, Wait wait, Barrier barrier, Read read, Multiply multiply) {
    static_assert(STAGES >= 3, "a stage that is read, one waited for, one asked for");
    // Stages behind the one waited for that may be on their way: group 1 waits before it asks for the last of them.
    constexpr std::integral_constant<int, STAGES - 2> asked{};
    constexpr std::integral_constant<int, STAGES - 3> unasked{};
    auto least = [](int a, int b) { return a < b ? a : b; };
    wait(asked, least(nk - 1, STAGES - 2));
    barrier();
    if (group == 1) barrier();
    for (int it = 0; it < nk; ++it) {
        if (group == 1) wait(unasked, least(nk - 2 - it, STAGES - 3));
        read(it);
        barrier();
        multiply();
        if (group == 0) wait(asked, least(nk - 2 - it, STAGES - 2));
        barrier();
    }
    if (group == 0) barrier();
}

}  // namespace bh
