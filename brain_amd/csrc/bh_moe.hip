// The router of a sparse mixture of experts, the plan of which rows each
// expert has, and the weighted sum of the experts' rows (bh_moe_route,
// bh_moe_plan_rows, bh_moe_combine).
//
// Routing: a group of 16 lanes takes a token (the whole wave where there are more than 256 experts), its
// logits in registers (lane l of G holds experts l, l + G, ...), and finds the
// top_k largest one after another: the group's maximum, then the lowest index
// that has it.
//
// Plan: a stable counting sort of the (token, choice) entries by expert. A wave takes
// its entries 64 at a time; the lanes with the same expert are found with a
// ballot for each bit of its index, so an entry's rank among them is a
// popcount and the counts need no atomics: the plan is the same on every run.
// One token of 128 experts 5.1 us (a chain of 8 reductions behind one load); 16384 tokens 9.6 + 3.0 +
// 3.6 us (route, scan, place).
#include <cfloat>

#include "bh_kvops.h"

namespace bh {

constexpr uint32_t MOE_MAX_EXPERTS = 1024, MOE_MAX_TOP = 64;
constexpr uint32_t RW = 16, RT = RW * 64;  // most waves and threads of a routing workgroup
constexpr uint32_t MOE_ENTRIES = 4096;     // most entries of a workgroup (16 bits hold their ranks; LDS: 52 KB)

struct RouteArgs {
    const void* logits;
    uint64_t stride;
    const uint8_t* mask;
    uint32_t items, e, k, first, div;  // k entries an item; entry i is of token i / div
    int score, renormalize;
    float scale;
    float* weights;
    int32_t* experts;
    uint32_t *offsets, *rows;
    int32_t* slots;
    uint32_t* counts;  // [workgroups][e]: entries of each expert in each workgroup's items
    uint32_t per;      // items of a workgroup
};

// Reductions over G = 16 or 64 neighbouring lanes; every lane gets the result.
template <int CTRL>
__device__ __forceinline__ uint32_t turned(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_mov_dpp((int)v, CTRL, 0xf, 0xf, false);
}
template <int G, class F>
__device__ __forceinline__ uint32_t over_group(uint32_t v, F f) {
    v = f(v, turned<0x128>(v));  // row_ror 8, 4, 2, 1: all 16 lanes of a row
    v = f(v, turned<0x124>(v));
    v = f(v, turned<0x122>(v));
    v = f(v, turned<0x121>(v));
    if constexpr (G == 64) {
        v = f(v, xor_lane_u<16>(v));
        v = f(v, xor_lane_u<32>(v));
    }
    return v;
}
template <int G>
__device__ __forceinline__ float group_max(float v) {
    return __builtin_bit_cast(float, over_group<G>(__builtin_bit_cast(uint32_t, v), [](uint32_t a, uint32_t b) {
        return __builtin_bit_cast(uint32_t, fmaxf(__builtin_bit_cast(float, a), __builtin_bit_cast(float, b)));
    }));
}
template <int G>
__device__ __forceinline__ float group_sum(float v) {
    return __builtin_bit_cast(float, over_group<G>(__builtin_bit_cast(uint32_t, v), [](uint32_t a, uint32_t b) {
        return __builtin_bit_cast(uint32_t, __builtin_bit_cast(float, a) + __builtin_bit_cast(float, b));
    }));
}
template <int G>
__device__ __forceinline__ uint32_t group_min(uint32_t v) {
    return over_group<G>(v, [](uint32_t a, uint32_t b) { return min(a, b); });
}

// The top k experts of token t, of this lane's group (t >= items: of none): lane l of it gets choices l, l + G, ...
// (-1: none) and their weights. For a whole wave.
template <class T, int G, int NV, int NK>
__device__ __forceinline__ void route_token(const RouteArgs& a, uint32_t t, uint32_t l, int (&expert)[NK], float (&weight)[NK]) {
    const bool live = t < a.items && !(a.mask && !a.mask[min(t, a.items - 1)]);
    const typename T::elem* row = reinterpret_cast<const typename T::elem*>(a.logits) + (uint64_t)min(t, a.items - 1) * a.stride;
    float x[NV], logit[NK];
#pragma unroll
    for (int v = 0; v < NV; ++v) {
        const uint32_t i = v * G + l;
        const float f = T::get(row + min(i, a.e - 1));
        x[v] = live && i < a.e && f == f ? f : -INFINITY;
    }
#pragma unroll
    for (int n = 0; n < NK; ++n) expert[n] = -1, logit[n] = -INFINITY;
    float top = -INFINITY, total = 0.0f;
    for (uint32_t j = 0; j < a.k; ++j) {
        float m = x[0];
#pragma unroll
        for (int v = 1; v < NV; ++v) m = fmaxf(m, x[v]);
        m = group_max<G>(m);
        if (j == 0) {
            top = m;
            // exp(l - top), where equal infinities are no distance apart
            if (a.score == BH_MOE_SOFTMAX && !a.renormalize) {
                float s = 0.0f;
#pragma unroll
                for (int v = 0; v < NV; ++v) s += x[v] == top ? 1.0f : expf(x[v] - top);
                total = group_sum<G>(s);
            }
        }
        uint32_t at = ~0u;
#pragma unroll
        for (int v = NV - 1; v >= 0; --v) at = x[v] == m ? v * G + l : at;
        at = group_min<G>(at);
        const bool found = m > -INFINITY;
        if (!__any(found)) break;
#pragma unroll
        for (int v = 0; v < NV; ++v) x[v] = at == v * G + l ? -INFINITY : x[v];
#pragma unroll
        for (int n = 0; n < NK; ++n)
            if (found && j == n * G + l) expert[n] = (int)at, logit[n] = m;
    }
    float s[NK], sum = 0.0f;
#pragma unroll
    for (int n = 0; n < NK; ++n) {
        s[n] = 0.0f;
        if (expert[n] >= 0) {
            if (a.score == BH_MOE_SOFTMAX) s[n] = logit[n] == top ? 1.0f : expf(logit[n] - top);
            // sigmoid; for a sum that is divided out, of far negative logits, exp(-top) times it
            else if (a.renormalize && top < 0.0f) s[n] = expf(logit[n] - top) / (1.0f + expf(logit[n]));
            else s[n] = 1.0f / (1.0f + expf(-logit[n]));
        }
        sum += s[n];
    }
    if (a.renormalize) total = group_sum<G>(sum);
#pragma unroll
    for (int n = 0; n < NK; ++n) {
        if (a.score == BH_MOE_SOFTMAX || a.renormalize) s[n] = expert[n] >= 0 ? s[n] / total : 0.0f;
        weight[n] = s[n] * a.scale;
    }
}

// The lanes whose `key` is this lane's.
__device__ __forceinline__ unsigned long long same_key(uint32_t key, uint32_t bits) {
    unsigned long long same = ~0ull;
    for (uint32_t b = 0; b < bits; ++b) {
        const unsigned long long m = __ballot((key >> b) & 1);
        same &= (key >> b) & 1 ? m : ~m;
    }
    return same;
}

// LDS accesses of a wave's lanes stay in this order.
__device__ __forceinline__ void wave_order() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// Exclusive sums of n counts in LDS, by the first wave, to `to` (LDS; may be `from`) and, where given, `out`, the total behind them.
__device__ __forceinline__ void place_experts(const uint32_t* from, uint32_t n, uint32_t lane, uint32_t* to, uint32_t* out) {
    uint32_t base = 0;
    for (uint32_t e0 = 0; e0 < n; e0 += 64) {
        const uint32_t e = e0 + lane, c = e < n ? from[e] : 0, upto = lane_scan(c);
        if (e < n) {
            to[e] = base + upto - c;
            if (out) out[e] = base + upto - c;
        }
        base += (uint32_t)__builtin_amdgcn_readlane((int)upto, 63);
    }
    if (out && lane == 0) out[n] = base;
}

// LDS of a workgroup that plans: offsets [e], counts [waves][e], key and rank of each entry.
static size_t plan_lds(uint32_t e, uint32_t waves, uint32_t entries) {
    return (size_t)e * 4 + ((size_t)waves * e + 1) / 2 * 4 + (size_t)entries * 4;
}

// A workgroup's items: their experts (routed here, or read: NV = 0), and of each entry
// the rank among the entries of its expert in this workgroup. With one workgroup
// (ONE) the plan is complete at the end; else `slots` holds the ranks and
// `counts` the workgroup's counts, for moe_place_kernel. Some 13 vector instructions for each token and choice of 128
// experts are 2.8 us of the 9.6 that 16384 tokens take (8 choices); the rest is latency: the logits' way in, four tokens of
// a wave one choice after another, 16 waves' counts summed in turn between barriers, the results' way out.
template <class T, int G, int NV, int NK, bool PLAN, bool ONE>
__global__ __launch_bounds__(RT) void moe_route_kernel(RouteArgs a) {
    extern __shared__ uint32_t lds[];
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, waves = blockDim.x >> 6;
    const uint32_t t0 = min(blockIdx.x * a.per, a.items), t1 = min(t0 + a.per, a.items);
    // Wave w's items, in order: entries that follow each other. Whole groups of tokens.
    constexpr uint32_t TOKENS = 64 / G;
    uint32_t share = (t1 - t0 + waves - 1) / waves;
    if constexpr (NV > 0) share = (share + TOKENS - 1) / TOKENS * TOKENS;
    const uint32_t w0 = min(t0 + wave * share, t1), w1 = min(w0 + share, t1);
    uint32_t* off = lds;
    uint16_t *cnts = reinterpret_cast<uint16_t*>(off + a.e), *cnt = cnts + wave * a.e;
    // entry i of the workgroup: its key (low 16 bits) and its rank
    uint32_t* entry = off + a.e + (waves * a.e + 1) / 2;
    const uint32_t i0 = t0 * a.k;
    if constexpr (PLAN) {
        for (uint32_t i = lane; i < a.e; i += 64) cnt[i] = 0;
    }
    if constexpr (NV > 0) {
        for (uint32_t t = w0; t < w1; t += TOKENS) {
            const uint32_t mine = t + lane / G, l = lane % G;
            int expert[NK];
            float weight[NK];
            route_token<T, G, NV, NK>(a, mine < w1 ? mine : a.items, l, expert, weight);
#pragma unroll
            for (int n = 0; n < NK; ++n) {
                const uint32_t j = n * G + l;
                if (j < a.k && mine < w1) {
                    a.experts[(uint64_t)mine * a.k + j] = expert[n];
                    a.weights[(uint64_t)mine * a.k + j] = weight[n];
                    if constexpr (PLAN) entry[mine * a.k + j - i0] = min((uint32_t)expert[n], a.e);
                }
            }
        }
    }
    if constexpr (!PLAN) return;
    wave_order();
    const uint32_t bits = 32 - (uint32_t)__builtin_clz(a.e);  // of a key, e itself (routed nowhere) included
    const uint32_t from = w0 * a.k, to = w1 * a.k;
    for (uint32_t i = from + lane; i - lane < to; i += 64) {
        uint32_t key = a.e;
        if (i < to) key = NV > 0 ? entry[i - i0] : min((uint32_t)a.experts[i] - a.first, a.e);
        const unsigned long long same = same_key(key, bits), below = (1ull << lane) - 1;
        const uint32_t before = key < a.e ? cnt[key] : 0;
        wave_order();
        if (key < a.e && !(same & below)) cnt[key] = (uint16_t)(before + (uint32_t)__popcll(same));
        if (i < to) entry[i - i0] = key | (before + (uint32_t)__popcll(same & below)) << 16;
        wave_order();
    }
    __syncthreads();
    // Counts to where each wave's entries begin; the workgroup's counts.
    for (uint32_t e = tid; e < a.e; e += blockDim.x) {
        uint32_t sum = 0;
        for (uint32_t w = 0; w < waves; ++w) {
            const uint32_t c = cnts[w * a.e + e];
            cnts[w * a.e + e] = (uint16_t)sum;
            sum += c;
        }
        if constexpr (ONE) off[e] = sum;
        else a.counts[(uint64_t)blockIdx.x * a.e + e] = sum;
    }
    __syncthreads();
    if constexpr (ONE) {
        if (wave == 0) place_experts(off, a.e, lane, off, a.offsets);
        __syncthreads();
    }
    for (uint32_t i = from + lane; i < to; i += 64) {
        const uint32_t key = entry[i - i0] & 0xffff;
        if (key == a.e) {
            a.slots[i] = -1;
            continue;
        }
        const uint32_t at = (entry[i - i0] >> 16) + cnt[key] + (ONE ? off[key] : 0);
        a.slots[i] = (int32_t)at;
        if constexpr (ONE) a.rows[at] = i / a.div;
    }
}

// The counts of a call of many workgroups become the sums before each, and those of all go behind the last:
// a workgroup takes an expert.
__global__ __launch_bounds__(256) void moe_scan_kernel(RouteArgs a, uint32_t wgs) {
    __shared__ uint32_t part[4];
    const uint32_t e = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    uint32_t base = 0;
    for (uint32_t b0 = 0; b0 < wgs; b0 += 256) {
        const uint32_t b = b0 + tid, c = b < wgs ? a.counts[(uint64_t)b * a.e + e] : 0;
        const uint32_t upto = lane_scan(c);
        __syncthreads();
        if (lane == 63) part[wave] = upto;
        __syncthreads();
        uint32_t before = base;
        for (uint32_t w = 0; w < wave; ++w) before += part[w];
        if (b < wgs) a.counts[(uint64_t)b * a.e + e] = before + upto - c;
        base += part[0] + part[1] + part[2] + part[3];
    }
    if (tid == 0) a.counts[(uint64_t)wgs * a.e + e] = base;
}

// Ranks to places: workgroup b's entries of an expert come behind those of the
// workgroups before it. SUMMED: moe_scan_kernel has added them up; else every workgroup does.
template <bool SUMMED>
__global__ __launch_bounds__(RT) void moe_place_kernel(RouteArgs a) {
    extern __shared__ uint32_t lds[];  // [e] all, [e] before
    uint32_t *all = lds, *before = lds + a.e;
    const uint32_t tid = threadIdx.x, wgs = gridDim.x;
    // The thread's first entry is on its way beside the counts.
    const uint32_t t0 = min(blockIdx.x * a.per, a.items), t1 = min(t0 + a.per, a.items), end = t1 * a.k;
    uint32_t i = t0 * a.k + tid, e0 = ~0u, rank = 0;
    if (i < end) {
        e0 = (uint32_t)a.experts[i] - a.first;
        rank = (uint32_t)a.slots[i];
    }
    if constexpr (SUMMED) {
        for (uint32_t e = tid; e < a.e; e += RT) {
            all[e] = a.counts[(uint64_t)wgs * a.e + e];
            before[e] = a.counts[(uint64_t)blockIdx.x * a.e + e];
        }
    } else {
        for (uint32_t e = tid; e < 2 * a.e; e += RT) lds[e] = 0;
        __syncthreads();
        // A thread adds up an expert's counts in every parts-th workgroup. (Sums of integers: any order.)
        const uint32_t parts = a.e < RT ? RT / a.e : 1, part = tid / a.e, e = tid - part * a.e;
        if (part < parts) {
            uint32_t sum = 0, mine = 0;
#pragma unroll 16
            for (uint32_t b = part; b < wgs; b += parts) {
                const uint32_t c = a.counts[(uint64_t)b * a.e + e];
                sum += c;
                mine += b < blockIdx.x ? c : 0;
            }
            atomicAdd(&all[e], sum);
            atomicAdd(&before[e], mine);
        }
    }
    __syncthreads();
    if (tid < 64) place_experts(all, a.e, tid, all, blockIdx.x == 0 ? a.offsets : nullptr);
    __syncthreads();
    while (i < end) {
        if (e0 < a.e) {
            const uint32_t at = rank + before[e0] + all[e0];
            a.slots[i] = (int32_t)at;
            a.rows[at] = i / a.div;
        }
        i += RT;
        if (i < end) {
            e0 = (uint32_t)a.experts[i] - a.first;
            rank = (uint32_t)a.slots[i];
        }
    }
}

// Items of a workgroup: one workgroup up to 128 tokens or 4096 entries, else 256 or as
// many as it takes.
static uint32_t share_of(uint32_t items, uint32_t k, uint32_t one) {
    const uint32_t most = std::max(MOE_ENTRIES / std::max(k, 1u), 1u);
    if (items <= std::min(one, most)) return std::max(items, 1u);
    return std::min(most, std::max((items + 255) / 256, one / 4));
}
static uint32_t route_share(uint32_t tokens, uint32_t k) { return share_of(tokens, k, 128); }
static uint32_t plan_share(uint32_t entries) { return share_of(entries, 1, 4096); }
static uint32_t groups_of(uint32_t items, uint32_t per) { return std::max((items + per - 1) / per, 1u); }
// From this many workgroups on their counts are summed in a launch of its own (256 of them, 128 experts: 11.8 us
// of every workgroup adding up all, 3.8 + 3.5 us apart; 25 of them, 60 experts: 3.3 us in one).
constexpr uint32_t SCAN_GROUPS = 64;

template <class T, int G, int NV, int NK>
static hipError_t launch_route_as(hipStream_t s, const RouteArgs& a, bool plan) {
    const uint32_t wgs = groups_of(a.items, a.per);
    // (Four tokens of a wave at a time, or an entry a lane.)
    const uint32_t per_wave = NV > 0 ? 64 / G : 64;
    const uint32_t waves = std::min(RW, std::max(1u, (std::min(a.per, a.items) + per_wave - 1) / per_wave));
    if (!plan) {
        moe_route_kernel<T, G, NV, NK, false, false><<<wgs, waves * 64, 0, s>>>(a);
        return hipGetLastError();
    }
    const size_t lds = plan_lds(a.e, waves, a.per * a.k);
    if (wgs == 1) {
        moe_route_kernel<T, G, NV, NK, true, true><<<1, waves * 64, lds, s>>>(a);
        return hipGetLastError();
    }
    moe_route_kernel<T, G, NV, NK, true, false><<<wgs, waves * 64, lds, s>>>(a);
    hipError_t err = hipGetLastError();
    if (err != hipSuccess) return err;
    if (wgs < SCAN_GROUPS) {
        moe_place_kernel<false><<<wgs, RT, (size_t)2 * a.e * 4, s>>>(a);
        return hipGetLastError();
    }
    moe_scan_kernel<<<a.e, 256, 0, s>>>(a, wgs);
    if ((err = hipGetLastError()) != hipSuccess) return err;
    moe_place_kernel<true><<<wgs, RT, (size_t)2 * a.e * 4, s>>>(a);
    return hipGetLastError();
}

template <class T, int G, int NV>
static hipError_t launch_route(hipStream_t s, const RouteArgs& a, bool plan) {
    if (a.k <= G) return launch_route_as<T, G, NV, 1>(s, a, plan);
    return launch_route_as<T, G, NV, 64 / G>(s, a, plan);
}

template <class T>
static hipError_t launch_route_any(hipStream_t s, const RouteArgs& a, bool plan) {
    if (a.e <= 16) return launch_route<T, 16, 1>(s, a, plan);
    if (a.e <= 32) return launch_route<T, 16, 2>(s, a, plan);
    if (a.e <= 64) return launch_route<T, 16, 4>(s, a, plan);
    if (a.e <= 128) return launch_route<T, 16, 8>(s, a, plan);
    if (a.e <= 256) return launch_route<T, 16, 16>(s, a, plan);
    if (a.e <= 512) return launch_route<T, 64, 8>(s, a, plan);
    return launch_route<T, 64, 16>(s, a, plan);
}

static int check_plan(const char* who, uint32_t tokens, uint32_t top_k, uint32_t n_experts, const bh_moe_plan* plan,
                      const void* ws, uint64_t ws_bytes, RouteArgs* a) {
    if (n_experts == 0 || n_experts > MOE_MAX_EXPERTS)
        return fail(BH_ERR_INVALID, "%s: %u experts (1 to %u)", who, n_experts, MOE_MAX_EXPERTS);
    if ((uint64_t)tokens * top_k > 0x7fffffffu)
        return fail(BH_ERR_INVALID, "%s: %u tokens of %u choices", who, tokens, top_k);
    if (!plan) return BH_OK;
    if (!plan->offsets || ((uint64_t)tokens * top_k && (!plan->rows || !plan->slots)))
        return fail(BH_ERR_INVALID, "%s: null plan buffer", who);
    uint64_t need = 0;
    const int rc = bh_moe_workspace(tokens, top_k, n_experts, &need);
    if (rc) return rc;
    if (ws_bytes < need || (need && (!ws || !aligned_to(ws, 4))))
        return fail(BH_ERR_INVALID, "%s: a workspace of %llu bytes, needs %llu", who, (unsigned long long)(ws ? ws_bytes : 0),
                    (unsigned long long)need);
    a->offsets = plan->offsets, a->rows = plan->rows, a->slots = plan->slots;
    a->counts = static_cast<uint32_t*>(const_cast<void*>(ws));
    return BH_OK;
}

// ---------------------------------------------------------------- the weighted sum
struct CombineArgs {
    const void* y;
    const float* weights;
    const int32_t* slots;
    const void* add;
    void* out;
    uint32_t places, tokens, k, n, per;  // per: waves of a token's row
};

// W neighbouring elements, in registers as f32.
template <class T, int W>
struct Piece {
    static constexpr int BYTES = W * sizeof(typename T::elem), WORDS = BYTES >= 4 ? BYTES / 4 : 1;
    typedef uint32_t Part __attribute__((ext_vector_type(WORDS < 4 ? WORDS : 4)));
    static constexpr int PARTS = WORDS <= 4 ? 1 : WORDS / 4;
    Part part[PARTS];
    __device__ __forceinline__ void load(const typename T::elem* p) {
        if constexpr (BYTES == 2) {
            part[0] = *p;
        } else {
#pragma unroll
            for (int i = 0; i < PARTS; ++i) part[i] = reinterpret_cast<const Part*>(p)[i];
        }
    }
    __device__ __forceinline__ float get(int w) const {
        if constexpr (sizeof(typename T::elem) == 4) {
            return __builtin_bit_cast(float, (uint32_t)part[w / 4][w % 4]);
        } else {
            const uint32_t u = part[w / 8][w % 8 / 2];
            return __builtin_bit_cast(float, w % 2 ? u & 0xffff0000u : u << 16);
        }
    }
    __device__ __forceinline__ static void store(typename T::elem* p, const float (&v)[W]) {
        if constexpr (BYTES == 2) {
            T::put(p, v[0]);
        } else {
#pragma unroll
            for (int i = 0; i < PARTS; ++i) {
                Part o;
#pragma unroll
                for (int q = 0; q < (WORDS < 4 ? WORDS : 4); ++q) {
                    if constexpr (sizeof(typename T::elem) == 4) o[q] = __builtin_bit_cast(uint32_t, v[i * 4 + q]);
                    else o[q] = pack_bf16x2(v[i * 8 + 2 * q], v[i * 8 + 2 * q + 1]);
                }
                reinterpret_cast<Part*>(p)[i] = o;
            }
        }
    }
};

// A wave takes 64 W columns of a token; the slots and weights are in scalars, and the
// pieces of up to 8 of the token's rows are on their way together. Bound by memory: top_k rows read
// for one written (8192 tokens of 8 rows of 2048 bf16: 60 us, 5.6 TB/s; an element a thread, row by row, 268).
template <class Y, class O, int W>
__global__ __launch_bounds__(256) void moe_combine_kernel(CombineArgs a) {
    const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(blockIdx.x * 4 + (threadIdx.x >> 6)));
    const uint32_t t = wave / a.per, c = (wave - t * a.per) * (64 * W) + (threadIdx.x & 63) * W;
    if (t >= a.tokens || c >= a.n) return;
    const typename Y::elem* y = reinterpret_cast<const typename Y::elem*>(a.y) + c;
    const int32_t* slots = a.slots + (uint64_t)t * a.k;
    const float* weights = a.weights + (uint64_t)t * a.k;
    const uint64_t at = (uint64_t)t * a.n + c;
    Piece<O, W> extra;
    if (a.add) extra.load(reinterpret_cast<const typename O::elem*>(a.add) + at);
    float s[W];
#pragma unroll
    for (int w = 0; w < W; ++w) s[w] = 0.0f;
    for (uint32_t j0 = 0; j0 < a.k; j0 += 8) {
        uint32_t slot[8];
        Piece<Y, W> row[8];
#pragma unroll
        for (uint32_t j = 0; j < 8; ++j) slot[j] = j0 + j < a.k ? (uint32_t)slots[j0 + j] : ~0u;
        // (A row for every choice, so that no load waits for a branch; k > 0 here, so places > 0.)
#pragma unroll
        for (uint32_t j = 0; j < 8; ++j) row[j].load(y + (uint64_t)(slot[j] < a.places ? slot[j] : 0) * a.n);
#pragma unroll
        for (uint32_t j = 0; j < 8; ++j) {
            if (slot[j] >= a.places) continue;
            const float wt = weights[j0 + j];
#pragma unroll
            for (int w = 0; w < W; ++w) s[w] = fmaf(wt, row[j].get(w), s[w]);
        }
    }
    if (a.add) {
#pragma unroll
        for (int w = 0; w < W; ++w) s[w] += extra.get(w);
    }
    Piece<O, W>::store(reinterpret_cast<typename O::elem*>(a.out) + at, s);
}

template <class Y, class O, int W>
static bool combine_fits(const CombineArgs& a) {
    return a.n % W == 0 && aligned_to(a.y, std::min<size_t>(16, W * sizeof(typename Y::elem))) &&
           aligned_to(a.out, std::min<size_t>(16, W * sizeof(typename O::elem))) &&
           aligned_to(a.add, std::min<size_t>(16, W * sizeof(typename O::elem)));
}
template <class Y, class O, int W>
static hipError_t launch_combine_as(hipStream_t s, CombineArgs a) {
    a.per = (a.n + 64 * W - 1) / (64 * W);
    const uint64_t wgs = ((uint64_t)a.tokens * a.per + 3) / 4;
    if (wgs > 0x3fffffffu) return hipErrorInvalidConfiguration;
    moe_combine_kernel<Y, O, W><<<(unsigned)wgs, 256, 0, s>>>(a);
    return hipGetLastError();
}
template <class Y, class O>
static hipError_t launch_combine(hipStream_t s, CombineArgs a) {
    if (a.places == 0) a.k = 0;
    constexpr int most = sizeof(typename Y::elem) == 2 ? 8 : 4;  // 16 bytes of a row
    if (combine_fits<Y, O, most>(a)) return launch_combine_as<Y, O, most>(s, a);
    if (combine_fits<Y, O, 2>(a)) return launch_combine_as<Y, O, 2>(s, a);
    return launch_combine_as<Y, O, 1>(s, a);
}

}  // namespace bh

using namespace bh;

static int launched(hipError_t e, const char* who) {
    return e == hipSuccess ? BH_OK : fail(BH_ERR_HIP, "%s: %s", who, hipGetErrorString(e));
}

extern "C" int bh_moe_workspace(uint32_t tokens, uint32_t top_k, uint32_t n_experts, uint64_t* bytes) {
    if (!bytes) return fail(BH_ERR_INVALID, "bh_moe_workspace: null output");
    if (n_experts == 0 || n_experts > MOE_MAX_EXPERTS || (uint64_t)tokens * top_k > 0x7fffffffu)
        return fail(BH_ERR_INVALID, "bh_moe_workspace: %u tokens, %u choices, %u experts", tokens, top_k, n_experts);
    const uint32_t entries = tokens * top_k;
    const uint32_t wgs = std::max(groups_of(tokens, route_share(tokens, top_k)), groups_of(entries, plan_share(entries)));
    *bytes = wgs > 1 ? (uint64_t)(wgs + 1) * n_experts * 4 : 0;
    return BH_OK;
}

extern "C" int bh_moe_route(void* stream, const bh_moe_router* r, float* weights, int32_t* experts,
                            const bh_moe_plan* plan, void* ws, uint64_t ws_bytes) {
    static const char* who = "bh_moe_route";
    if (!r) return fail(BH_ERR_INVALID, "%s: null router", who);
    RouteArgs a{};
    const int rc = check_plan(who, r->tokens, r->top_k, r->n_experts, plan, ws, ws_bytes, &a);
    if (rc) return rc;
    if (r->top_k == 0 || r->top_k > MOE_MAX_TOP || r->top_k > r->n_experts)
        return fail(BH_ERR_INVALID, "%s: the top %u of %u experts (at most %u)", who, r->top_k, r->n_experts, MOE_MAX_TOP);
    if (r->dtype != BH_OUT_F32 && r->dtype != BH_OUT_BF16) return fail(BH_ERR_INVALID, "%s: dtype %d", who, r->dtype);
    if (r->score != BH_MOE_SOFTMAX && r->score != BH_MOE_SIGMOID) return fail(BH_ERR_INVALID, "%s: score %d", who, r->score);
    if (r->tokens > 1 && r->stride < r->n_experts)
        return fail(BH_ERR_INVALID, "%s: stride %llu below %u experts", who, (unsigned long long)r->stride, r->n_experts);
    if (r->tokens == 0 && !plan) return BH_OK;
    if (r->tokens && (!r->logits || !weights || !experts)) return fail(BH_ERR_INVALID, "%s: null buffer", who);
    a.logits = r->logits, a.stride = r->stride, a.mask = r->mask, a.items = r->tokens, a.e = r->n_experts;
    a.k = a.div = r->top_k;
    a.score = r->score, a.renormalize = r->renormalize, a.scale = r->scale, a.weights = weights, a.experts = experts;
    a.per = route_share(r->tokens, r->top_k);
    const hipStream_t s = (hipStream_t)stream;
    const hipError_t e = r->dtype == BH_OUT_F32 ? launch_route_any<F32>(s, a, plan) : launch_route_any<Bf16>(s, a, plan);
    return launched(e, who);
}

extern "C" int bh_moe_plan_rows(void* stream, const int32_t* experts, uint32_t tokens, uint32_t top_k, uint32_t first,
                                uint32_t n_experts, const bh_moe_plan* plan, void* ws, uint64_t ws_bytes) {
    static const char* who = "bh_moe_plan_rows";
    if (!plan) return fail(BH_ERR_INVALID, "%s: null plan", who);
    RouteArgs a{};
    const int rc = check_plan(who, tokens, top_k, n_experts, plan, ws, ws_bytes, &a);
    if (rc) return rc;
    // (The kernels take expert - first as an unsigned number: a negative expert, of none, stays outside up to here.)
    if ((uint64_t)first + n_experts > 1ull << 31)
        return fail(BH_ERR_INVALID, "%s: %u experts from first %u on pass 2^31", who, n_experts, first);
    if ((uint64_t)tokens * top_k && !experts) return fail(BH_ERR_INVALID, "%s: null experts", who);
    a.items = tokens * top_k, a.e = n_experts, a.k = 1, a.div = std::max(top_k, 1u), a.first = first;
    a.experts = const_cast<int32_t*>(experts);
    a.per = plan_share(a.items);
    return launched(launch_route_as<F32, 64, 0, 1>((hipStream_t)stream, a, true), who);
}

extern "C" int bh_moe_combine(void* stream, const void* y, int y_dtype, uint32_t places, const float* weights,
                              const int32_t* slots, uint32_t tokens, uint32_t top_k, uint32_t n, const void* add, void* out,
                              int out_dtype) {
    static const char* who = "bh_moe_combine";
    if ((y_dtype != BH_OUT_F32 && y_dtype != BH_OUT_BF16) || (out_dtype != BH_OUT_F32 && out_dtype != BH_OUT_BF16))
        return fail(BH_ERR_INVALID, "%s: dtypes %d and %d", who, y_dtype, out_dtype);
    if (places > 0x7fffffffu || tokens > 0x7fffffffu || n > 0x7fffffffu || (uint64_t)tokens * top_k > 0x7fffffffu)
        return fail(BH_ERR_INVALID, "%s: %u places, %u tokens of %u choices, rows of %u", who, places, tokens, top_k, n);
    if (tokens == 0 || n == 0) return BH_OK;
    if (!out || (top_k && (!weights || !slots || (places && !y)))) return fail(BH_ERR_INVALID, "%s: null buffer", who);
    const CombineArgs a{y, weights, slots, add, out, places, tokens, top_k, n, 0};
    const hipStream_t s = (hipStream_t)stream;
    hipError_t e;
    if (y_dtype == BH_OUT_F32) e = out_dtype == BH_OUT_F32 ? launch_combine<F32, F32>(s, a) : launch_combine<F32, Bf16>(s, a);
    else e = out_dtype == BH_OUT_F32 ? launch_combine<Bf16, F32>(s, a) : launch_combine<Bf16, Bf16>(s, a);
    if (e == hipErrorInvalidConfiguration) return fail(BH_ERR_INVALID, "%s: grid too large", who);
    return launched(e, who);
}
