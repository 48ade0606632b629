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

constexpr uint32_t ET = 1024;
constexpr uint32_t CUS = 256;  // compute units

// A sequence within its budget keeps all.
__device__ __forceinline__ void keep_all(const EvictArgs& p, uint32_t len, const float* acc, float* acc_out, int32_t* keep) {
    for (uint32_t j = threadIdx.x; j < p.budget; j += ET) keep[j] = j < len ? (int32_t)j : -1;
    if (acc_out && acc_out != acc)
        for (uint32_t j = threadIdx.x; j < len; j += ET) acc_out[j] = acc[j];
}

// One workgroup for each (sequence, kv head), its weights in registers (VPT a
// thread, wave w those of positions 64 VPT w .. on): latency bounds it, so each
// weight is loaded once and the steps that the workgroup takes together are few.
// The weight of the last entry kept is found digit by digit from the top, 11, 11
// and 10 bits, a histogram in LDS for each (the first of 8 bits would hold little
// but exponents, a few bins for all weights to queue at); then a count of each
// wave's kept entries says where it writes them. 1024 threads of 4 entries up to
// 4096 positions (8 heads of 1111: 7.7 us), of 16 up to 16384 (16 sequences of up
// to 8192, 128 workgroups, half the chip: 12.6 to 15.8 us from run to run,
// histograms and barriers in turn).
template <int VPT>
__device__ __forceinline__ void select_entries(EvictArgs p) {
    constexpr int NW = ET / 64, BINS = 2048;
    __shared__ uint32_t hist[BINS], wtot[NW], pick[2];
    const uint32_t b = blockIdx.x / p.kv.nkv, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const uint32_t len = min(kv_length(p.lens[b]), p.cap);
    const float* acc = p.acc + (uint64_t)blockIdx.x * p.cap;
    float* acc_out = p.acc_out ? p.acc_out + (uint64_t)blockIdx.x * p.cap_out : nullptr;
    int32_t* keep = p.keep + (uint64_t)blockIdx.x * p.budget;
    if (len <= p.budget) return keep_all(p, len, acc, acc_out, keep);
    // The candidates are positions [lo, hi); `need` of them stay.
    const uint32_t lo = p.sink, hi = len - p.recent, need = p.budget - p.sink - p.recent;
    const uint32_t j0 = wave * 64 * VPT + lane;
    float v[VPT];
    uint32_t u[VPT];
#pragma unroll
    for (int i = 0; i < VPT; ++i) v[i] = j0 + 64 * i < len ? acc[j0 + 64 * i] : 0.0f;
    uint32_t prefix = 0, left = need;  // of the digits found; how many of the weights that share them stay
    if (need) {
#pragma unroll
        for (int i = 0; i < VPT; ++i) u[i] = place(v[i]);
#pragma unroll
        for (int d = 0; d < 3; ++d) {
            const int shift = d == 0 ? 21 : d == 1 ? 10 : 0;
            const uint32_t digit = d == 2 ? 1023u : 2047u, mask = d == 0 ? 0u : ~0u << (d == 1 ? 21 : 10);
            for (uint32_t i = tid; i < BINS; i += ET) hist[i] = 0;
            __syncthreads();
#pragma unroll
            for (int i = 0; i < VPT; ++i) {
                const uint32_t j = j0 + 64 * i;
                if (j >= lo && j < hi && (u[i] & mask) == prefix) atomicAdd(&hist[(u[i] >> shift) & digit], 1u);
            }
            __syncthreads();
            // The highest digit with at least `left` weights at or above it:
            // thread t looks at two, from the top.
            const uint32_t c1 = hist[BINS - 1 - 2 * tid], c0 = hist[BINS - 2 - 2 * tid];
            uint32_t upto = c1 + c0;
#pragma unroll
            for (int off = 1; off < 64; off *= 2) {
                const uint32_t o = __shfl_up(upto, off, 64);
                if ((int)lane >= off) upto += o;
            }
            if (lane == 63) wtot[wave] = upto;
            __syncthreads();
#pragma unroll
            for (int w = 0; w < NW; ++w)
                if (w < (int)wave) upto += wtot[w];
            const uint32_t above = upto - c1 - c0;
            if (above < left && left <= upto) {
                const bool first = above + c1 >= left;
                pick[0] = BINS - 2 - 2 * tid + (first ? 1 : 0);
                pick[1] = left - above - (first ? 0 : c1);
            }
            __syncthreads();
            prefix |= pick[0] << shift;
            left = pick[1];
        }
    }
    // All weights above `prefix` stay, and the first `left` equal to it.
    const unsigned long long below = (1ull << lane) - 1;
    uint32_t n = 0;
    if (need) {
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
            const uint32_t j = j0 + 64 * i;
            n += (uint32_t)__popcll(__ballot(j >= lo && j < hi && u[i] == prefix));
        }
    }
    if (lane == 0) wtot[wave] = n;
    __syncthreads();
    uint32_t before = 0, kept = 0, stay = 0;  // stay: bit i, entry i of this thread
#pragma unroll
    for (int w = 0; w < NW; ++w)
        if (w < (int)wave) before += wtot[w];
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
        const uint32_t j = j0 + 64 * i;
        const bool mid = j >= lo && j < hi, eq = need && mid && u[i] == prefix;
        const unsigned long long em = __ballot(eq);
        const bool s = j < len && (!mid || (need && (u[i] > prefix || (eq && before + (uint32_t)__popcll(em & below) < left))));
        before += (uint32_t)__popcll(em);
        kept += (uint32_t)__popcll(__ballot(s));
        stay |= (s ? 1u : 0u) << i;
    }
    __syncthreads();
    if (lane == 0) wtot[wave] = kept;
    __syncthreads();
    uint32_t to = 0;
#pragma unroll
    for (int w = 0; w < NW; ++w)
        if (w < (int)wave) to += wtot[w];
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
        const bool s = (stay >> i) & 1u;
        const unsigned long long km = __ballot(s);
        const uint32_t at = to + (uint32_t)__popcll(km & below);
        if (s && at < p.budget) {  // (acc_out may be acc: all of it has been read)
            keep[at] = (int32_t)(j0 + 64 * i);
            if (acc_out) acc_out[at] = v[i];
        }
        to += (uint32_t)__popcll(km);
    }
}

template <int VPT>
__global__ __launch_bounds__(ET) void kv_evict_select_kernel(EvictArgs p) {
    select_entries<VPT>(p);
}

// The same for any length, its weights read again for each digit (8 bits at a
// time) and for the last pass, which goes through them in order.
__global__ __launch_bounds__(ET) void kv_evict_select_long_kernel(EvictArgs p) {
    __shared__ uint32_t hist[256], wtot[ET / 64], pick[2];
    const uint32_t b = blockIdx.x / p.kv.nkv, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const uint32_t len = min(kv_length(p.lens[b]), p.cap);
    const float* acc = p.acc + (uint64_t)blockIdx.x * p.cap;
    float* acc_out = p.acc_out ? p.acc_out + (uint64_t)blockIdx.x * p.cap_out : nullptr;
    int32_t* keep = p.keep + (uint64_t)blockIdx.x * p.budget;
    if (len <= p.budget) return keep_all(p, len, acc, acc_out, keep);
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

// Moves the entries of a (sequence, kv head), keys or values, from entry i0 on, in
// strides of `step`, by threads tid of NT. A thread takes a piece of W, M entries of a
// pass at a time in flight. Position i's entry comes from keep[i] >= i, so in place a workgroup
// goes through all of them in order: what a pass writes no later pass reads, and a
// barrier between its reads and its writes is enough.
constexpr uint32_t MT = 256;
constexpr int MU = 4, SU = 8;  // M of the kernel for the move alone, and for both
template <class W, bool IN_PLACE, uint32_t NT, int M>
__device__ __forceinline__ void move_entries(const EvictArgs& p, uint32_t bk, uint32_t which, uint32_t tid, uint64_t i0,
                                             uint64_t step) {
    const uint32_t b = bk / p.kv.nkv, kvh = bk % p.kv.nkv;
    const uint32_t pieces = p.kv.hd / sizeof(W), per = NT / pieces, e = tid / pieces, w = tid % pieces;
    const int32_t* keep = p.keep + (uint64_t)bk * p.budget;
    uint8_t* pool = (uint8_t*)(which ? p.kv.pool[1] : p.kv.pool[0]) + (size_t)kvh * p.kv.hd + w * sizeof(W);
    float* scales = (which ? p.kv.scales[1] : p.kv.scales[0]) + kvh;
    for (; i0 < p.budget; i0 += step) {
        uint32_t from[M], to[M];
        W c[M];
        float s[M];
#pragma unroll
        for (int u = 0; u < M; ++u) {
            const uint64_t i = i0 + u * per + e;
            const int32_t src = e < per && i < p.budget ? keep[i] : -1;
            const bool move = src >= 0 && !(IN_PLACE && (uint32_t)src == (uint32_t)i);
            from[u] = move ? p.kv.slot(b, (uint32_t)src) : NO_SLOT;
            to[u] = move ? p.kv.slot_in(p.to, p.to_cols, b, (uint32_t)i) : NO_SLOT;
        }
#pragma unroll
        for (int u = 0; u < M; ++u) {
            if (to[u] == NO_SLOT) from[u] = NO_SLOT;
            c[u] = W{};
            s[u] = 0.0f;
            if (from[u] != NO_SLOT) {
                c[u] = *reinterpret_cast<const W*>(pool + p.kv.row(from[u]));
                if (w == 0) s[u] = scales[(uint64_t)from[u] * p.kv.nkv];
            }
        }
        if constexpr (IN_PLACE) __syncthreads();
#pragma unroll
        for (int u = 0; u < M; ++u) {
            if (from[u] == NO_SLOT) continue;
            *reinterpret_cast<W*>(pool + p.kv.row(to[u])) = c[u];
            if (w == 0) scales[(uint64_t)to[u] * p.kv.nkv] = s[u];
        }
        if constexpr (IN_PLACE) __syncthreads();
    }
}

// To other blocks the passes are spread over `steps` workgroups. 16 sequences cut
// to 2048 entries of 8 heads of 128: 138 MB in 26 us, 5.3 TB/s. In place a head's
// passes follow one another in one workgroup: the same eviction 72 us, 41 to other
// blocks (calls in a row, with the selection).
template <class W, bool IN_PLACE>
__global__ __launch_bounds__(MT) void kv_evict_move_kernel(EvictArgs p, uint32_t steps, uint32_t per) {
    const uint32_t group = blockIdx.x / steps, bk = group >> 1;
    if (bk % p.kv.nkv == 0 && blockIdx.x % (2 * steps * p.kv.nkv) == 0 && threadIdx.x == 0) {
        const uint32_t b = bk / p.kv.nkv;
        p.new_lens[b] = min(min(kv_length(p.lens[b]), p.cap), p.budget);
    }
    move_entries<W, IN_PLACE, MT, MU>(p, bk, group & 1, threadIdx.x, (uint64_t)(blockIdx.x % steps) * MU * per,
                                      (uint64_t)steps * MU * per);
}

// Selection and move of a (sequence, kv head) in one workgroup, half of it moving
// the keys and half the values.
template <class W, bool IN_PLACE>
__global__ __launch_bounds__(ET) void kv_evict_small_kernel(EvictArgs p) {
    select_entries<4>(p);
    __syncthreads();  // keep[] is written
    if (blockIdx.x % p.kv.nkv == 0 && threadIdx.x == 0) {
        const uint32_t b = blockIdx.x / p.kv.nkv;
        p.new_lens[b] = min(min(kv_length(p.lens[b]), p.cap), p.budget);
    }
    const uint32_t per = ET / 2 / (p.kv.hd / (uint32_t)sizeof(W));
    move_entries<W, IN_PLACE, ET / 2, SU>(p, blockIdx.x, threadIdx.x / (ET / 2), threadIdx.x % (ET / 2), 0, (uint64_t)SU * per);
}

template <class W>
hipError_t go_move(hipStream_t s, const EvictArgs& a, uint64_t heads) {
    const uint32_t per = MT / (a.kv.hd / sizeof(W));  // entries of a pass
    const uint64_t all = (a.budget + (uint64_t)per * MU - 1) / (per * MU);
    if (a.in_place) {
        kv_evict_move_kernel<W, true><<<(unsigned)(2 * heads), MT, 0, s>>>(a, 1, per);
    } else {
        const uint32_t steps = (uint32_t)std::max<uint64_t>(1, std::min<uint64_t>(all, 0x7fffffffull / (2 * heads)));
        kv_evict_move_kernel<W, false><<<(unsigned)(2 * heads * steps), MT, 0, s>>>(a, steps, per);
    }
    return hipGetLastError();
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
    const uint64_t most = std::min<uint64_t>({budget, acc_stride, (uint64_t)kv->max_blocks * kv->block_size});
    if (out_tables && (out_max_blocks == 0 || (uint64_t)out_max_blocks * kv->block_size < most))
        return fail(BH_ERR_INVALID, "%s: out_max_blocks %u, blocks of %u, for %llu positions", who, out_max_blocks,
                    kv->block_size, (unsigned long long)most);
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
    const bool wide = kv->head_dim % 16 == 0 && aligned_to(kv->k_pool, 16) && aligned_to(kv->v_pool, 16);
    // One launch where it is no slower. In place a workgroup of its own walks each
    // head's entries in two launches as well, with half the threads and a head's
    // keys and values apart: one launch up to a head for each compute unit (time in
    // a graph, us, one launch and two: 8 heads of 64, 1111 positions cut to 700, 14.0
    // and 18.4; 256 heads of 128, 4000 cut to 2048, 69 and 81; 512 heads of 64, 1111
    // cut to 700, 42 and 38). To other blocks two launches spread the move over the
    // chip, so one is for few pieces of few heads, where the second launch costs more
    // than it saves (the same, and between calls in a row: 32 heads of 64, 1111 cut
    // to 512, 12.1 and 12.8, 12.3 and 14.9; to 704, at the limit, 13.1 and 13.0, 13.1
    // and 14.9; to 896, 14.3 and 13.0, 14.4 and 15.3; 64 heads, 4000 cut to 640, 17.1
    // and 15.4, 16.9 and 15.7). Not where the new lengths may lie on the old ones,
    // which other workgroups still read.
    const bool apart = new_lens + batch <= seq_lens || seq_lens + batch <= new_lens;
    const uint64_t pieces = (uint64_t)budget * (kv->head_dim / (wide ? 16 : 4));
    if (acc_stride <= 4 * ET && apart && (a.in_place ? heads <= CUS : heads <= 32 && pieces <= 2816)) {
        if (wide && a.in_place) kv_evict_small_kernel<uint4, true><<<(unsigned)heads, ET, 0, s>>>(a);
        else if (wide) kv_evict_small_kernel<uint4, false><<<(unsigned)heads, ET, 0, s>>>(a);
        else if (a.in_place) kv_evict_small_kernel<uint32_t, true><<<(unsigned)heads, ET, 0, s>>>(a);
        else kv_evict_small_kernel<uint32_t, false><<<(unsigned)heads, ET, 0, s>>>(a);
        const hipError_t e = hipGetLastError();
        return e == hipSuccess ? BH_OK : fail(BH_ERR_HIP, "%s: %s", who, hipGetErrorString(e));
    }
    if (acc_stride <= 4 * ET) kv_evict_select_kernel<4><<<(unsigned)heads, ET, 0, s>>>(a);
    else if (acc_stride <= 16 * ET) kv_evict_select_kernel<16><<<(unsigned)heads, ET, 0, s>>>(a);
    else kv_evict_select_long_kernel<<<(unsigned)heads, ET, 0, s>>>(a);
    hipError_t e = hipGetLastError();
    if (e == hipSuccess) e = wide ? go_move<uint4>(s, a, heads) : go_move<uint32_t>(s, a, heads);
    return e == hipSuccess ? BH_OK : fail(BH_ERR_HIP, "%s: %s", who, hipGetErrorString(e));
}
