// Lengths of the int8 paged cache's sequences as the kernels take them, plain
// C++ (constexpr: host and device alike), so that their ends can be tried on the
// host: what a length holds bounds the loops over a sequence's keys.
#pragma once
#include <stdint.h>

namespace bh {

// No table is taken to reach further: 64 positions past the last one still fit
// in 31 bits, so that loops over keys do not wrap.
constexpr uint32_t KV_REACH = 0x7fff0000u;

// Positions that a table of `blocks` blocks of `bs` has.
constexpr uint32_t kv_reach(uint32_t blocks, uint32_t bs) {
    return (uint64_t)blocks * bs < KV_REACH ? (uint32_t)((uint64_t)blocks * bs) : KV_REACH;
}

// A length as the program gives it: one below zero (as an int32) is none.
constexpr uint32_t kv_length(uint32_t len) { return len < 0x80000000u ? len : 0u; }

// The number of keys that row i < n of a sequence's chunk sees, which sits at
// position len - n + i. len from kv_length, n < 2^31: no sum here wraps.
constexpr uint32_t kv_keys_seen(uint32_t len, uint32_t n, uint32_t i) { return len + i + 1 > n ? len + i + 1 - n : 0u; }

}  // namespace bh
