// What the operators of the int8 paged KV cache share (bh_rope.hip,
// bh_pattn.hip, bh_evict.hip): the cache and the batch as the kernels take
// them, and their checks.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "../../include/brain_hip.h"
#include "bh_common.h"
#include "bh_kvlen.h"

namespace bh {

constexpr uint32_t NO_SLOT = 0xffffffffu;

// n / d for n < 2^31 without the division's dozen dependent steps: for d no
// power of two the upper half of n * m, m = ceil(2^(31 + l) / d) with
// l = ceil(log2 d), shifted by l - 1; n m / 2^(31 + l) is above n / d by less
// than 1 / d then (n < 2^31, m 2^-(31 + l) above 1 / d by less than 2^-(31 + l)).
struct Div {
    uint32_t m, s;  // m = 0: a shift
    static Div by(uint32_t d) {
        uint32_t l = 0;
        while (l < 32 && (1ull << l) < d) ++l;
        if ((1ull << l) == d) return Div{0, l};
        return Div{(uint32_t)(((1ull << (31 + l)) + d - 1) / d), l - 1};
    }
    __host__ __device__ __forceinline__ uint32_t of(uint32_t n) const {
        return (m ? (uint32_t)(((uint64_t)n * m) >> 32) : n) >> s;
    }
};

// A bh_kv8 whose geometry has been checked. Slots from `nslots` on lie outside
// the pool or the scales: a table entry that names one is skipped.
struct Kv8 {
    uint32_t* pool[2];  // codes of keys, values
    float* scales[2];
    const uint32_t* bt;
    uint32_t max_bt, bs, nkv, hd, nslots;
    Div by_bs;

    // Slot of position j of sequence b in a table of `cols` > 0 entries a row.
    // (Unconditional: the load is at an entry of the row in any case.)
    __device__ __forceinline__ uint32_t slot_in(const uint32_t* tables, uint32_t cols, uint32_t b, uint32_t j) const {
        const uint32_t blk = by_bs.of(j & 0x7fffffffu);
        const uint64_t s = (uint64_t)tables[(uint64_t)b * cols + min(blk, cols - 1)] * bs + (j - blk * bs);
        return blk < cols && j < 0x80000000u && s < nslots ? (uint32_t)s : NO_SLOT;
    }
    __device__ __forceinline__ uint32_t reach() const { return kv_reach(max_bt, bs); }
    __device__ __forceinline__ uint32_t slot(uint32_t b, uint32_t j) const { return slot_in(bt, max_bt, b, j); }
    __device__ __forceinline__ size_t row(uint32_t slot) const { return (size_t)slot * (nkv * hd); }  // bytes
};

// The rows of a ragged batch: sequence b has rows [start[b], start[b + 1]),
// the last ones of its len[b] cached positions.
struct Kv8Rows {
    const uint32_t* start;  // null: one row for each sequence
    const uint32_t* lens;
    uint32_t batch, rows;

    __device__ __forceinline__ uint32_t len(uint32_t b) const { return kv_length(lens[b]); }
    __device__ __forceinline__ uint32_t first(uint32_t b) const { return start ? min(start[b], rows) : min(b, rows); }
    __device__ __forceinline__ uint32_t end(uint32_t b) const { return start ? min(start[b + 1], rows) : min(b + 1, rows); }
};

// The last b < n for which below(b), a condition that holds up to some b and
// not behind it; NO_SLOT if there is none. For a whole wave; one load of the
// conditions' data for each factor of 64 in n. (Where the condition is not of
// that kind the answer is still below n.)
template <class F>
__device__ __forceinline__ uint32_t wave_last(uint32_t n, uint32_t lane, F below) {
    uint32_t lo = 0;
    while (n) {
        const uint32_t step = (n + 63) / 64, i = lane * step;
        const bool yes = i < n && below(lo + min(i, n - 1));
        const unsigned long long m = __ballot(yes);
        if (!m) return NO_SLOT;
        const uint32_t c = (63u - (uint32_t)__builtin_clzll(m)) * step;
        if (step == 1) return lo + c;
        lo += c;
        n = min(step, n - c);
    }
    return NO_SLOT;
}

// Inclusive sum over the lanes of a wave, by DPP row shifts and broadcasts.
__device__ __forceinline__ uint32_t lane_scan(uint32_t v) {
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x111, 0xf, 0xf, false);  // row_shr:1
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x112, 0xf, 0xf, false);  // row_shr:2
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x114, 0xf, 0xf, false);  // row_shr:4
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x118, 0xf, 0xf, false);  // row_shr:8
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x142, 0xa, 0xf, false);  // row_bcast:15 into rows 1, 3
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x143, 0xc, 0xf, false);  // row_bcast:31 into rows 2, 3
    return v;
}

// Host checks: BH_OK, or the error of `who`.
int check_kv8(const char* who, const bh_kv8* kv, Kv8* out);
int check_kv8_batch(const char* who, const bh_kv8_batch* bt, Kv8Rows* out);

inline bool aligned_to(const void* p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

// Element types of activations.
struct F32 {
    typedef float elem;
    static __device__ __forceinline__ float get(const float* p) { return *p; }
    typedef float raw4 __attribute__((ext_vector_type(4)));  // four elements as loaded
    static __device__ __forceinline__ void open4(raw4 v, float (&x)[4]) {
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = v[i];
    }
    static __device__ __forceinline__ void put(float* p, float v) { *p = v; }
    static __device__ __forceinline__ void put4(float* p, const float (&x)[4]) {
        *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
    }
};
struct Bf16 {
    typedef uint16_t elem;
    static __device__ __forceinline__ float get(const uint16_t* p) {
        return __builtin_bit_cast(float, (uint32_t)*p << 16);
    }
    typedef int raw4 __attribute__((ext_vector_type(2)));
    static __device__ __forceinline__ void open4(raw4 v, float (&x)[4]) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            x[2 * i] = __builtin_bit_cast(float, (uint32_t)v[i] << 16);
            x[2 * i + 1] = __builtin_bit_cast(float, (uint32_t)v[i] & 0xffff0000u);
        }
    }
    static __device__ __forceinline__ void put(uint16_t* p, float v) { *p = f32_to_bf16_rne(v); }
    static __device__ __forceinline__ void put4(uint16_t* p, const float (&x)[4]) {
        *reinterpret_cast<uint2*>(p) = make_uint2(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]));
    }
};

}  // namespace bh
