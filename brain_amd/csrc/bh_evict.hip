// Cutting sequences of the int8 paged KV cache down to a budget of positions:
// which ones each kv head keeps (its first, its last, and the ones that have
// received the most attention), and their move to the front.
#include "bh_kvops.h"

namespace bh {
namespace {

struct EvictArgs {
    const uint32_t* lens;
    const float* acc;
    float* acc_out;
    int32_t* keep;
    uint32_t* new_lens;
    const uint32_t* to;  // destination tables
    uint32_t to_cols, cap, cap_out, budget, sink, recent, in_place;
    Kv8 kv;
};

// A float's place in the order, ascending; -0 is +0, and NaN is -inf.
__device__ __forceinline__ uint32_t place(float v) {
    if (v != v) v = -INFINITY;
    const uint32_t u = __builtin_bit_cast(uint32_t, v + 0.0f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// One workgroup for each (sequence, kv head). The weight of the last entry
// kept is found digit by digit from the top (8 bits at a time, a histogram in
// LDS for each): 4 passes over the weights. A last pass in order writes the
// kept positions and their weights.
constexpr uint32_t ET = 1024;
__global__ __launch_bounds__(ET) void kv_evict_select_kernel(EvictArgs p) {
    __shared__ uint32_t hist[256], wtot[ET / 64], pick[2];
    const uint32_t b = blockIdx.x / p.kv.nkv, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const uint32_t len = min(p.lens[b], p.cap);
    const float* acc = p.acc + (uint64_t)blockIdx.x * p.cap;
    float* acc_out = p.acc_out ? p.acc_out + (uint64_t)blockIdx.x * p.cap_out : nullptr;
    int32_t* keep = p.keep + (uint64_t)blockIdx.x * p.budget;
    if (len <= p.budget) {
        for (uint32_t j = tid; j < p.budget; j += ET) keep[j] = j < len ? (int32_t)j : -1;
        if (acc_out && acc_out != acc)
            for (uint32_t j = tid; j < len; j += ET) acc_out[j] = acc[j];
        return;
    }
    // The candidates are positions [lo, hi); `need` of them stay.
    const uint32_t lo = p.sink, hi = len - p.recent, need = p.budget - p.sink - p.recent;
    uint32_t prefix = 0, left = need;  // of the digits found; how many of the weights that share them stay
    for (int shift = 24; shift >= 0; shift -= 8) {
        if (tid < 256) hist[tid] = 0;
        __syncthreads();
        const uint32_t mask = shift == 24 ? 0u : ~0u << (shift + 8);
        for (uint32_t j = lo + tid; j < hi; j += ET) {
            const uint32_t u = place(acc[j]);
            if ((u & mask) == prefix) atomicAdd(&hist[(u >> shift) & 255], 1u);
        }
        __syncthreads();
        // The highest digit d with at least `left` weights at or above it.
        if (tid < 64) {
            uint32_t c[4], mine = 0;
            for (int i = 3; i >= 0; --i) mine += c[i] = hist[4 * (63 - lane) + i];  // lane 0: the highest digits
            uint32_t upto = mine;
            for (int off = 1; off < 64; off *= 2) {
                const uint32_t o = __shfl_up(upto, off, 64);
                if ((int)lane >= off) upto += o;
            }
            const unsigned long long m = __ballot(upto >= left);
            const uint32_t first = m ? (uint32_t)__builtin_ctzll(m) : 63u;
            if (lane == first) {
                uint32_t above = upto - mine;
                int i = 3;
                while (i > 0 && above + c[i] < left) above += c[i--];
                pick[0] = 4 * (63 - lane) + i;
                pick[1] = left - above;
            }
        }
        __syncthreads();
        prefix |= pick[0] << shift;
        left = pick[1];
    }
    // All weights above `prefix` stay, and the first `left` equal to it.
    uint32_t kept = 0, equal = 0;  // before this chunk
    for (uint32_t j0 = 0; j0 < len; j0 += ET) {
        const uint32_t j = j0 + tid;
        const bool in = j < len, mid = in && j >= lo && j < hi;
        const float v = in ? acc[j] : 0.0f;
        const uint32_t u = place(v);
        const bool eq = mid && need && u == prefix;
        const unsigned long long below = (1ull << lane) - 1, em = __ballot(eq);
        __syncthreads();
        if (lane == 0) wtot[wave] = (uint32_t)__popcll(em);
        __syncthreads();
        uint32_t before = equal, all = 0;
        for (uint32_t w = 0; w < ET / 64; ++w) {
            if (w < wave) before += wtot[w];
            all += wtot[w];
        }
        const uint32_t rank = before + (uint32_t)__popcll(em & below);
        equal += all;
        const bool stay = in && (!mid || (need && (u > prefix || (eq && rank < left))));
        const unsigned long long km = __ballot(stay);
        __syncthreads();
        if (lane == 0) wtot[wave] = (uint32_t)__popcll(km);
        __syncthreads();
        before = kept, all = 0;
        for (uint32_t w = 0; w < ET / 64; ++w) {
            if (w < wave) before += wtot[w];
            all += wtot[w];
        }
        const uint32_t to = before + (uint32_t)__popcll(km & below);
        kept += all;
        // (acc_out may be acc: what is written lies at or before what this
        // chunk has read, and before all that is still to be read.)
        if (stay && to < p.budget) {
            keep[to] = (int32_t)j;
            if (acc_out) acc_out[to] = v;
        }
    }
}

// One workgroup for each (sequence, kv head, keys or values), MK entries at a
// time in order. Position i's entry comes from keep[i] >= i: what a step
// writes, in place, no later step reads, so a barrier between a step's reads
// and its writes is enough.
constexpr uint32_t MT = 256;
__global__ __launch_bounds__(MT) void kv_evict_move_kernel(EvictArgs p) {
    const uint32_t which = blockIdx.x & 1, bk = blockIdx.x >> 1, b = bk / p.kv.nkv, kvh = bk % p.kv.nkv;
    const uint32_t words = p.kv.hd / 4;
    const int32_t* keep = p.keep + (uint64_t)bk * p.budget;
    if (kvh == 0 && which == 0 && threadIdx.x == 0) p.new_lens[b] = min(min(p.lens[b], p.cap), p.budget);
    // A thread moves one word of an entry (lane groups of `words`).
    const uint32_t per = MT / words, e = threadIdx.x / words, w = threadIdx.x % words;
    for (uint32_t i0 = 0; i0 < p.budget; i0 += per) {
        const uint32_t i = i0 + e;
        const int32_t src = e < per && i < p.budget ? keep[i] : -1;
        uint32_t from = NO_SLOT, to = NO_SLOT;
        uint32_t c = 0;
        float s = 0.0f;
        if (src >= 0 && !(p.in_place && (uint32_t)src == i)) {
            from = p.kv.slot(b, (uint32_t)src);
            to = p.kv.slot_in(p.to, p.to_cols, b, i);
            if (from != NO_SLOT && to != NO_SLOT) {
                c = p.kv.pool[which][(p.kv.row(from) + (uint64_t)kvh * p.kv.hd) / 4 + w];
                if (w == 0) s = p.kv.scales[which][(uint64_t)from * p.kv.nkv + kvh];
            }
        }
        __syncthreads();
        if (from != NO_SLOT && to != NO_SLOT) {
            p.kv.pool[which][(p.kv.row(to) + (uint64_t)kvh * p.kv.hd) / 4 + w] = c;
            if (w == 0) p.kv.scales[which][(uint64_t)to * p.kv.nkv + kvh] = s;
        }
        __syncthreads();
    }
}

}  // namespace
}  // namespace bh

using namespace bh;

extern "C" int bh_paged_kv_evict_i8(void* stream, const bh_kv8* kv, const uint32_t* seq_lens, uint32_t batch,
                                    const float* acc, uint32_t acc_stride, uint32_t budget, uint32_t sink,
                                    uint32_t recent, const uint32_t* out_tables, uint32_t out_max_blocks,
                                    float* acc_out, uint32_t acc_out_stride, int32_t* keep, uint32_t* new_lens) {
    static const char* who = "bh_paged_kv_evict_i8";
    EvictArgs a{};
    const int rc = check_kv8(who, kv, &a.kv);
    if (rc) return rc;
    if (budget == 0 || (uint64_t)sink + recent > budget || budget > 0x7fffffffu || acc_stride > 0x7fffffffu)
        return fail(BH_ERR_INVALID, "%s: a budget of %u with %u first and %u last positions (acc_stride %u)", who, budget,
                    sink, recent, acc_stride);
    if (batch == 0) return BH_OK;
    if (!seq_lens || !acc || !keep || !new_lens) return fail(BH_ERR_INVALID, "%s: null buffer", who);
    if (acc_out && (acc_out_stride < std::min(budget, acc_stride) || (acc_out == acc && acc_out_stride != acc_stride)))
        return fail(BH_ERR_INVALID, "%s: rows of %u in acc_out for a budget of %u (acc_stride %u)", who, acc_out_stride,
                    budget, acc_stride);
    const uint64_t heads = (uint64_t)batch * kv->n_kv_heads;
    if (heads > 0x3fffffffull) return fail(BH_ERR_INVALID, "%s: grid too large", who);
    a.lens = seq_lens, a.acc = acc, a.acc_out = acc_out, a.keep = keep, a.new_lens = new_lens;
    a.in_place = !out_tables || out_tables == kv->block_tables;
    a.to = a.in_place ? kv->block_tables : out_tables;
    a.to_cols = a.in_place ? kv->max_blocks : out_max_blocks;
    a.cap = acc_stride, a.cap_out = acc_out_stride, a.budget = budget, a.sink = sink, a.recent = recent;
    const hipStream_t s = (hipStream_t)stream;
    kv_evict_select_kernel<<<(unsigned)heads, ET, 0, s>>>(a);
    hipError_t e = hipGetLastError();
    if (e == hipSuccess) {
        kv_evict_move_kernel<<<(unsigned)(2 * heads), MT, 0, s>>>(a);
        e = hipGetLastError();
    }
    return e == hipSuccess ? BH_OK : fail(BH_ERR_HIP, "%s: %s", who, hipGetErrorString(e));
}
