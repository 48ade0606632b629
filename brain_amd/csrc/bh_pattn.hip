// Attention of a ragged batch's new rows over the int8 paged KV cache, and the
// weight that each cached key receives from it.
#include <type_traits>

#include "bh_kvops.h"

namespace bh {
namespace {

constexpr float LOG2E = 1.44269504088896341f, LN2 = 0.693147180559945309f;

typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef float v4f __attribute__((ext_vector_type(4)));

struct AttnArgs {
    const void* q;
    uint64_t qs;  // row stride, elements
    void* out;
    float* lse;
    Kv8 kv;
    Kv8Rows bt;
    uint32_t nh, group;
    Div by_group, by_nsplit, by_nkv;
    float scale2;  // scale * log2(e): softmax in base 2
    // The matrix kernels: blocks of query vectors, splits of the keys, what the
    // splits leave for the join.
    uint32_t blocks, nsplit, span;  // span: keys of a split
    float* part;                    // [row][head][split][hd], then
    float2* ml;                     // [row][head][split] maximum and sum
    uint32_t ovec;                  // outputs lie at multiples of 4 elements
};
struct SumsArgs {
    const void* q;
    uint64_t qs;
    const float* lse;
    float* acc;
    Kv8 kv;
    Kv8Rows bt;
    uint32_t nh, group, cap;
    Div by_group, by_nchunk, by_nkv;
    float scale2;
    uint32_t nchunk;  // workgroups of a (sequence, kv head)
};

__device__ __forceinline__ float code_f(uint32_t w, int e) { return (float)(int8_t)(uint8_t)(w >> (8 * e)); }

// Any head_dim: one wave for each row and query head. A lane takes a key for
// the score and four elements of the context for the weighted sum, 64 keys at
// a time, with a running maximum and sum. No matrix instructions, no split of the
// keys, and each query head reads its keys anew: 32 rows of 16 heads over 8 of 96,
// up to 4096 keys, bf16: 1.54 ms for traffic of 34 us; 256 rows 1.50 ms.
template <class T>
__global__ __launch_bounds__(64) void paged_attention_any_kernel(AttnArgs p) {
    typedef typename T::elem E;
    __shared__ float qv[256];
    const uint32_t r = blockIdx.x / p.nh, h = blockIdx.x % p.nh, kvh = h / p.group, lane = threadIdx.x;
    const uint32_t hd = p.kv.hd;
    uint32_t b = r;
    if (p.bt.start) b = wave_last(p.bt.batch, lane, [&](uint32_t i) { return p.bt.start[i] <= r; });
    if (b >= p.bt.batch) return;
    const uint32_t r0 = p.bt.first(b), e = p.bt.end(b), len = p.bt.len(b);
    if (r >= e) return;
    const uint32_t seen = min(kv_keys_seen(len, e - r0, r - r0), p.kv.reach());  // keys that the row sees
    for (uint32_t d = lane; d < hd; d += 64) qv[d] = T::get((const E*)p.q + r * p.qs + (uint64_t)h * hd + d);
    __syncthreads();
    const bool live = 4 * lane < hd;
    float m = -INFINITY, l = 0.0f, o[4] = {0.f, 0.f, 0.f, 0.f};
    for (uint32_t j0 = 0; j0 < seen; j0 += 64) {
        const uint32_t j = j0 + lane;
        const uint32_t slot = j < seen ? p.kv.slot(b, j) : NO_SLOT;
        float s = -INFINITY, vs = 0.0f;
        if (slot != NO_SLOT) {
            const uint32_t* k = p.kv.pool[0] + (p.kv.row(slot) + (uint64_t)kvh * hd) / 4;
            float acc = 0.0f;
            for (uint32_t d = 0; d < hd; d += 4) {
                const uint32_t w = k[d / 4];
                for (int i = 0; i < 4; ++i) acc = acc + qv[d + i] * code_f(w, i);
            }
            s = acc * p.kv.scales[0][(uint64_t)slot * p.kv.nkv + kvh] * p.scale2;
            vs = p.kv.scales[1][(uint64_t)slot * p.kv.nkv + kvh];
        }
        // fmaxf drops a NaN: it reaches the sum below.
        const float mn = fmaxf(m, xor_max<32>(s)), ref = mn == -INFINITY ? 0.0f : mn;
        const float alpha = __builtin_amdgcn_exp2f(m - ref), w = __builtin_amdgcn_exp2f(s - ref);
        l = l * alpha + xor_sum<32>(w);
        for (int i = 0; i < 4; ++i) o[i] = o[i] * alpha;
        const float wv = slot != NO_SLOT ? w * vs : 0.0f;
        const uint32_t n = min(64u, seen - j0);
        for (uint32_t u = 0; u < n; ++u) {
            const uint32_t su = (uint32_t)__builtin_amdgcn_readlane((int)slot, (int)u);
            if (su == NO_SLOT) continue;
            const float wu = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, wv), (int)u));
            if (live) {
                const uint32_t c = p.kv.pool[1][(p.kv.row(su) + (uint64_t)kvh * hd) / 4 + lane];
                for (int i = 0; i < 4; ++i) o[i] = o[i] + wu * code_f(c, i);
            }
        }
        m = mn;
    }
    E* dst = (E*)p.out + ((uint64_t)r * p.nh + h) * hd + 4 * lane;
    if (live)
        for (int i = 0; i < 4; ++i) T::put(dst + i, l == 0.0f ? 0.0f : o[i] / l);
    if (p.lse && lane == 0) p.lse[(uint64_t)r * p.nh + h] = l == 0.0f ? -INFINITY : (m + log2f(l)) * LN2;
}

// Any head_dim: a thread for each (sequence, kv head, key), which goes through the
// chunk's queries in order (the same batches: 200 us for 17 of traffic, 2.1 ms).
template <class T>
__global__ __launch_bounds__(64) void paged_weight_sums_any_kernel(SumsArgs p, uint32_t nchunk) {
    typedef typename T::elem E;
    const uint32_t bk = blockIdx.x / nchunk, j = (blockIdx.x % nchunk) * 64 + threadIdx.x;
    const uint32_t b = bk / p.kv.nkv, kvh = bk % p.kv.nkv, hd = p.kv.hd;
    const uint32_t len = p.bt.len(b);
    if (j >= len || j >= p.cap) return;
    const uint32_t r0 = p.bt.first(b), r1 = p.bt.end(b), n = r1 > r0 ? r1 - r0 : 0u;
    const uint32_t slot = p.kv.slot(b, j);
    float* dst = p.acc + ((uint64_t)b * p.kv.nkv + kvh) * p.cap + j;
    const bool old = n <= len && j < len - n;
    float sum = 0.0f;
    if (slot != NO_SLOT && n) {
        const uint32_t* k = p.kv.pool[0] + (p.kv.row(slot) + (uint64_t)kvh * hd) / 4;
        const float ks = p.kv.scales[0][(uint64_t)slot * p.kv.nkv + kvh];
        const uint32_t i0 = j + n > len ? j + n - len : 0;  // the first row that sees j
        for (uint32_t i = i0; i < n; ++i)
            for (uint32_t g = 0; g < p.group; ++g) {
                const uint32_t h = kvh * p.group + g;
                const E* q = (const E*)p.q + (r0 + i) * p.qs + (uint64_t)h * hd;
                float acc = 0.0f;
                for (uint32_t d = 0; d < hd; d += 4) {
                    const uint32_t w = k[d / 4];
                    for (int u = 0; u < 4; ++u) acc = acc + T::get(q + d + u) * code_f(w, u);
                }
                sum = sum + __builtin_amdgcn_exp2f(acc * ks * p.scale2 - p.lse[(uint64_t)(r0 + i) * p.nh + h] * LOG2E);
            }
    }
    *dst = old ? *dst + sum : sum;
}

constexpr uint32_t CUS = 256;  // compute units

// ---------------------------------------------------------------- few rows
//
// Up to 32 query vectors (rows x heads of one kv head) of a sequence at a time:
// the cache is read once and each code used for few products, so the stream of
// the codes bounds it (64 sequences of up to 8192 keys, one row of 32 heads over
// 8 of 128, bf16: 905 MB in 178 us, 5.1 TB/s, where a large copy moves 4.9 and a
// read alone 6.2). A wave takes 32 keys at a time straight into the operand
// layout of v_mfma_f32_16x16x32_bf16 (codes are exact in bf16), the next 32 in
// flight: no LDS, no barrier in the loop. Scores are computed transposed (keys x
// queries): lane (c, g) = (l % 16, l / 16) then holds the scores of query c and
// keys 4g..4g+3 and 16+4g..16+4g+3, which is the operand layout of the second
// product for an order of its 32 keys that V's loads follow.
//
// A query of f32 is the exact sum of three bf16 numbers, and so is a weight:
// three products each, 24 bits. With bf16 activations the query is exact, and
// the weight times its value scale is rounded to bf16, half a step 2^-9 of the
// next power of two: the size of the output's own rounding.
//
// A single sequence of 2000 keys (16 heads over 8, f32) takes 5.9 us, the chain
// of look-up, codes, products and the workgroup's sum; the join behind it 4 us.

__device__ __forceinline__ uint32_t fbits(float f) { return __builtin_bit_cast(uint32_t, f); }
__device__ __forceinline__ float bitsf(uint32_t u) { return __builtin_bit_cast(float, u); }
// The upper halves of two floats, packed (exact where they are bf16 numbers).
__device__ __forceinline__ uint32_t hi16x2(float lo, float hi) {
    return __builtin_amdgcn_perm(fbits(hi), fbits(lo), 0x07060302u);
}
// Eight floats as PARTS bf16 fragments: one, rounded to nearest, or three that
// add up to them: the first is cut, so that none rounds to infinity.
template <int PARTS>
__device__ __forceinline__ void split2(float x0, float x1, int i, v4i (&f)[PARTS]) {  // elements 2 i, 2 i + 1 of a fragment
    if constexpr (PARTS == 1) {
        f[0][i] = (int)pack_bf16x2(x0, x1);
    } else {
        f[0][i] = (int)hi16x2(x0, x1);
        const float r0 = x0 - bitsf(fbits(x0) & 0xffff0000u), r1 = x1 - bitsf(fbits(x1) & 0xffff0000u);
        const uint32_t q = pack_bf16x2(r0, r1);
        f[1][i] = (int)q;
        f[2][i] = (int)hi16x2(r0 - bitsf(q << 16), r1 - bitsf(q & 0xffff0000u));  // at most 8 bits are left
    }
}
template <int PARTS>
__device__ __forceinline__ void split8(const float (&x)[8], v4i (&f)[PARTS]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) split2<PARTS>(x[2 * i], x[2 * i + 1], i, f);
}
// Eight codes (along one key's dimensions) as a fragment.
__device__ __forceinline__ v4i codes8(uint32_t lo, uint32_t hi) {
    return v4i{(int)hi16x2(code_f(lo, 0), code_f(lo, 1)), (int)hi16x2(code_f(lo, 2), code_f(lo, 3)),
               (int)hi16x2(code_f(hi, 0), code_f(hi, 1)), (int)hi16x2(code_f(hi, 2), code_f(hi, 3))};
}
__device__ __forceinline__ v4f mfma16(v4i a, v4i b, v4f c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, a), __builtin_bit_cast(v8bf, b), c, 0, 0, 0);
}
// N times eight elements of a query, the n-th from p + at(n) on. (Wide loads all
// the same: the hardware takes them at any element's address.)
template <class T, int N, class At>
__device__ __forceinline__ void query8(const typename T::elem* p, float (&x)[N][8], At at) {
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
        for (int i = 0; i < 8; ++i) x[n][i] = T::get(p + at(n) + i);
}

// Where a workgroup works: sequence b, VB of its query vectors from v0 on (of
// nv = rows x group; vector v is head v % group of row v / group). Block numbers
// are given out so that sequence b's start at row_start[b] * group / VB + b:
// no list of them is needed, at the price of some that are empty.
struct Block {
    uint32_t b, r0, n, v0, nv, len;
};
template <int VB>
__device__ __forceinline__ uint32_t block_at(const Kv8Rows& bt, uint32_t group, uint32_t b, uint32_t r0) {
    return !bt.start && group <= VB ? b : r0 * group / VB + b;  // (without row_start and within VB: one block each)
}
template <int VB>
__device__ __forceinline__ bool find_block(const Kv8Rows& bt, uint32_t group, uint32_t blk, uint32_t lane, Block& o) {
    uint32_t b, r0, r1;
    if (bt.start && bt.batch < 64) {  // one round trip: lane i has row_start[i] and sequence i's length
        const uint32_t st = min(bt.start[min(lane, bt.batch)], bt.rows), ln = bt.len(min(lane, bt.batch - 1));
        asm volatile("" ::"v"(ln));  // both on their way before the branch
        const unsigned long long m = __ballot(lane < bt.batch && st * group / VB + lane <= blk);
        if (!m) return false;
        b = 63u - (uint32_t)__builtin_clzll(m);
        r0 = (uint32_t)__builtin_amdgcn_readlane((int)st, (int)b);
        r1 = (uint32_t)__builtin_amdgcn_readlane((int)st, (int)b + 1);
        o.len = (uint32_t)__builtin_amdgcn_readlane((int)ln, (int)b);
    } else {
        if (!bt.start && group <= VB) b = blk;
        else b = wave_last(bt.batch, lane, [&](uint32_t i) { return bt.first(i) * group / VB + i <= blk; });
        b = __builtin_amdgcn_readfirstlane((int)b);
        if (b >= bt.batch) return false;
        r0 = bt.first(b), r1 = bt.end(b), o.len = bt.len(b);
    }
    if (r1 <= r0) return false;
    o.b = b, o.r0 = r0, o.n = r1 - r0, o.nv = o.n * group;
    o.v0 = (blk - block_at<VB>(bt, group, b, r0)) * VB;
    return o.v0 < o.nv;
}
// The number of keys that row i of a block's sequence sees.
__device__ __forceinline__ uint32_t keys_seen(const Block& o, uint32_t i) {
    return kv_keys_seen(o.len, o.n, i);
}

constexpr int SW = 4;  // waves

// Waves per SIMD that the registers allow: queries, context and codes in flight.
template <class T, int HD, int NQ>
constexpr int stream_waves() {
    return (sizeof(typename T::elem) == 4 ? 3 : 1) * NQ * HD <= (sizeof(typename T::elem) == 4 ? 3 : 2) * 128 ? 2 : 1;
}

template <class T, int HD, int NQ, bool B16>
__global__ __launch_bounds__(SW * 64, (stream_waves<T, HD, NQ>())) void paged_attention_stream_kernel(AttnArgs p) {
    typedef typename T::elem E;
    constexpr int PARTS = sizeof(E) == 4 ? 3 : 1, VB = 16 * NQ, KT = HD / 64, VW = HD / 64;  // VW: words of V a lane takes of a key
    constexpr int OST = HD + 4;
    __shared__ __attribute__((aligned(16))) float so[SW][16][OST];
    __shared__ float sm[SW][VB], sl[SW][VB];
    __shared__ __attribute__((aligned(16))) float ssc[SW][64];
    const int tid = threadIdx.x, lane = tid & 63, c = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    // All kv heads of a unit run on one XCD (workgroups go round the eight):
    // their scales share cache lines.
    const uint32_t nkv = p.kv.nkv, turn = p.by_nkv.of(blockIdx.x / 8), unit = turn * 8 + blockIdx.x % 8, kvh = blockIdx.x / 8 - turn * nkv;
    if (unit >= p.blocks * p.nsplit) return;
    const uint32_t blk = p.by_nsplit.of(unit), split = unit - blk * p.nsplit;
    Block bl;
    if (!find_block<VB>(p.bt, p.group, blk, lane, bl)) return;
    const uint32_t reach = p.kv.reach();
    const uint32_t vend = min(bl.v0 + VB, bl.nv);
    const uint32_t kend = min(keys_seen(bl, p.by_group.of(vend - 1)), reach);  // keys that any of the vectors sees
    const uint32_t kall = min(keys_seen(bl, p.by_group.of(bl.v0)), reach);       // ... that all see
    const uint32_t k0 = split * p.span, k1 = split + 1 == p.nsplit ? kend : min(kend, k0 + p.span);
    if (k0 >= k1 && split) return;

    v4f o[NQ][HD / 16];
    float m[NQ], l[NQ];
#pragma unroll
    for (int q = 0; q < NQ; ++q) {
        m[q] = -INFINITY, l[q] = 0.0f;
#pragma unroll
        for (int j = 0; j < HD / 16; ++j) o[q][j] = v4f{0.f, 0.f, 0.f, 0.f};
    }

    const uint32_t kvs = nkv * HD;
    const uint8_t* kp = (const uint8_t*)p.kv.pool[0] + (size_t)kvh * HD;
    const uint8_t* vp = (const uint8_t*)p.kv.pool[1] + (size_t)kvh * HD;
    const float* sp = (lane < 32 ? p.kv.scales[0] : p.kv.scales[1]) + kvh;  // half the lanes take the keys' scales
    const uint32_t first = k0 + 32 * wave, step = 32 * SW;
    // Slots of the 32 keys of the wave's i-th tile. B16: the blocks hold whole
    // groups of 16 keys (and the pool as well), so two slots say where all are;
    // lane l looks those of tile l up, 64 tiles at a time (a look-up for each
    // tile would be waited for, tile by tile). Else lane l has that of key l % 32.
    // ok: which of the keys have a slot.
    struct Slots {
        uint32_t s0, s1, ok;
    };
    uint32_t mine0 = NO_SLOT, mine1 = NO_SLOT;
    auto slots_of = [&](uint32_t i) -> Slots {
        Slots r{0, 0, 0};
        if constexpr (B16) {
            if ((i & 63) == 0) {
                const uint32_t j = first + (i + lane) * step;
                uint32_t a = p.kv.slot(bl.b, j), b = p.kv.slot(bl.b, j + 16);
                asm volatile("" : "+v"(a), "+v"(b));  // both look-ups, then the comparisons
                mine0 = j < k1 ? a : NO_SLOT;
                mine1 = j + 16 < k1 ? b : NO_SLOT;
            }
            const uint32_t a = (uint32_t)__builtin_amdgcn_readlane((int)mine0, (int)(i & 63));
            const uint32_t b = (uint32_t)__builtin_amdgcn_readlane((int)mine1, (int)(i & 63));
            r.s0 = a != NO_SLOT ? a : 0u, r.s1 = b != NO_SLOT ? b : 0u;
            r.ok = (a != NO_SLOT ? 0xffffu : 0u) | (b != NO_SLOT ? 0xffff0000u : 0u);
        } else {
            const uint32_t j = first + i * step + (lane & 31), s = j < k1 ? p.kv.slot(bl.b, j) : NO_SLOT;
            r.s0 = s != NO_SLOT ? s : 0u;
            r.ok = (uint32_t)__ballot(s != NO_SLOT);
        }
        return r;
    };
    v4i kc[2][KT];       // codes of the keys in flight: lane (c, g) has key 16 u + c, bytes 16 (g + 4 i) ..+15
    uint32_t vc[8][VW];  // of the values: key 16 (e / 4) + 4 g + e % 4, bytes 4 VW c ..
    float sc;
    auto load_k = [&](const Slots& at) {
        const uint32_t lo = (uint32_t)c * kvs + 16 * g;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const uint8_t* k = B16 ? kp + (size_t)(u ? at.s1 : at.s0) * kvs + lo
                                   : kp + (size_t)(uint32_t)__shfl((int)at.s0, 16 * u + c, 64) * kvs + 16 * g;
#pragma unroll
            for (int i = 0; i < KT; ++i) kc[u][i] = *reinterpret_cast<const v4i*>(k + 64 * i);
        }
    };
    auto load_v = [&](const Slots& at) {
        const uint32_t lo = (uint32_t)(4 * g) * kvs + 4 * VW * c;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const uint8_t* v = B16 ? vp + (size_t)((e >> 2 ? at.s1 : at.s0) + (e & 3)) * kvs + lo
                                   : vp + (size_t)(uint32_t)__shfl((int)at.s0, 16 * (e >> 2) + 4 * g + (e & 3), 64) * kvs + 4 * VW * c;
            if constexpr (VW == 2) {
                const uint2 w = *reinterpret_cast<const uint2*>(v);
                vc[e][0] = w.x, vc[e][1] = w.y;
            } else {
                vc[e][0] = *reinterpret_cast<const uint32_t*>(v);
            }
        }
        const uint32_t a0 = at.s0, a1 = B16 ? at.s1 : 0u;
        sc = sp[(size_t)(B16 ? (lane & 16 ? a1 : a0) + c : a0) * nkv];
    };
    // The look-ups, the queries and the first tile go out before anything waits
    // for the queries.
    Slots at = slots_of(0);
    // Queries: fragment (t, half) holds d = 16 (g + 4t) + 8 half ..+7 of vector c.
    v4i qf[NQ][2 * KT][PARTS];
    float qx[NQ][2 * KT][8];
    uint32_t seen[NQ];
#pragma unroll
    for (int q = 0; q < NQ; ++q) {
        const uint32_t v = min(bl.v0 + 16 * q + c, vend - 1), i = p.by_group.of(v), h = kvh * p.group + (v - i * p.group);
        seen[q] = bl.v0 + 16 * q + c < vend ? min(keys_seen(bl, i), reach) : 0u;
        const E* src = (const E*)p.q + (bl.r0 + i) * p.qs + (uint64_t)h * HD;
        query8<T>(src, qx[q], [&](int t) { return 16 * (g + 4 * (t >> 1)) + 8 * (t & 1); });
    }
    load_k(at);
    load_v(at);
    Slots next = slots_of(1);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int q = 0; q < NQ; ++q)
#pragma unroll
        for (int t = 0; t < 2 * KT; ++t) split8<PARTS>(qx[q][t], qf[q][t]);
    uint32_t tile = 2;  // the one whose slots come next
#pragma unroll 1
    for (uint32_t j0 = first; j0 < k1; j0 += step) {
        const bool more = j0 + step < k1;
        uint32_t vt[8][VW];
#pragma unroll
        for (int e = 0; e < 8; ++e)
#pragma unroll
            for (int i = 0; i < VW; ++i) vt[e][i] = vc[e][i];
        // Scales by key: this wave's 64 floats, keys' then values'.
        ssc[wave][lane] = sc;
        const uint32_t ok = at.ok;
        if (more) load_v(next);
        __builtin_amdgcn_sched_barrier(0);
        v4f s[NQ][2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            v4i kf[2 * KT];
#pragma unroll
            for (int i = 0; i < KT; ++i) {
                kf[2 * i] = codes8((uint32_t)kc[u][i][0], (uint32_t)kc[u][i][1]);
                kf[2 * i + 1] = codes8((uint32_t)kc[u][i][2], (uint32_t)kc[u][i][3]);
            }
#pragma unroll
            for (int q = 0; q < NQ; ++q) {
                s[q][u] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int part = PARTS - 1; part >= 0; --part)  // small products first
#pragma unroll
                    for (int i = 0; i < 2 * KT; ++i) s[q][u] = mfma16(kf[i], qf[q][i][part], s[q][u]);
            }
        }
        __builtin_amdgcn_sched_barrier(0);
        if (more) {
            load_k(next);
            at = next;
            next = slots_of(tile++);
        }
        __builtin_amdgcn_wave_barrier();
        float ks[8], vs[8];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const float4 a = *reinterpret_cast<const float4*>(&ssc[wave][16 * u + 4 * g]);
            const float4 b = *reinterpret_cast<const float4*>(&ssc[wave][32 + 16 * u + 4 * g]);
            ks[4 * u] = a.x, ks[4 * u + 1] = a.y, ks[4 * u + 2] = a.z, ks[4 * u + 3] = a.w;
            vs[4 * u] = b.x, vs[4 * u + 1] = b.y, vs[4 * u + 2] = b.z, vs[4 * u + 3] = b.w;
        }
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int e = 0; e < 8; ++e) ks[e] = ks[e] * p.scale2;
        const bool masked = j0 + 32 > kall || ok != 0xffffffffu;
        v4i pf[NQ][PARTS];
#pragma unroll
        for (int q = 0; q < NQ; ++q) {
            float w[8], x[8], mx = -INFINITY;
            uint32_t unseen = 0;  // bit e: not a key of this query, whatever its scales are
#pragma unroll
            for (int e = 0; e < 8; ++e) w[e] = s[q][e >> 2][e & 3] * ks[e];
            if (masked) {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const uint32_t key = 16 * (e >> 2) + 4 * g + (e & 3);
                    if (j0 + key >= seen[q] || !((ok >> key) & 1u)) {
                        w[e] = -INFINITY;
                        unseen |= 1u << e;
                    }
                }
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) mx = fmaxf(mx, w[e]);
            mx = fmaxf(mx, xor_lane<16>(mx));
            mx = fmaxf(mx, xor_lane<32>(mx));
            if (__any(mx > m[q])) {
                const float mn = fmaxf(m[q], mx);
                const float alpha = mn == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m[q] - mn);
                l[q] = l[q] * alpha;
#pragma unroll
                for (int j = 0; j < HD / 16; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[q][j][e] = o[q][j][e] * alpha;
                m[q] = mn;
            }
            const float ref = m[q] == -INFINITY ? 0.0f : m[q];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                w[e] = __builtin_amdgcn_exp2f(w[e] - ref);
                l[q] = l[q] + w[e];
                x[e] = w[e] * vs[e];
            }
            if (masked) {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if ((unseen >> e) & 1u) x[e] = 0.0f;
            }
            split8<PARTS>(x, pf[q]);
        }
        __builtin_amdgcn_sched_barrier(0);
        // O^T: product j takes dimension 4 VW c + j of V for its row c.
#pragma unroll
        for (int j = 0; j < HD / 16; ++j) {
            float x[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = code_f(vt[e][j >> 2], j & 3);
            const v4i vf = v4i{(int)hi16x2(x[0], x[1]), (int)hi16x2(x[2], x[3]), (int)hi16x2(x[4], x[5]), (int)hi16x2(x[6], x[7])};
#pragma unroll
            for (int q = 0; q < NQ; ++q)
#pragma unroll
                for (int part = PARTS - 1; part >= 0; --part) o[q][j] = mfma16(vf, pf[q][part], o[q][j]);
        }
    }

    // The waves' parts, 16 vectors at a time: register (j, r) of lane (c, g) is
    // dimension 4 VW (4g + r) + j of vector c.
#pragma unroll
    for (int q = 0; q < NQ; ++q) {
        l[q] = l[q] + xor_lane<16>(l[q]);
        l[q] = l[q] + xor_lane<32>(l[q]);
        if (g == 0) sm[wave][16 * q + c] = m[q], sl[wave][16 * q + c] = l[q];
    }
    constexpr int DT = HD / 16;  // a thread's dimensions of vector tid / 16
    const int mv = tid >> 4, d0 = (tid & 15) * DT;
#pragma unroll
    for (int q = 0; q < NQ; ++q) {
        __syncthreads();
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int j = 0; j < HD / 16; j += 4)
                *reinterpret_cast<float4*>(&so[wave][c][DT * (4 * g + r) + j]) =
                    make_float4(o[q][j][r], o[q][j + 1][r], o[q][j + 2][r], o[q][j + 3][r]);
        __syncthreads();
        const uint32_t v = bl.v0 + 16 * q + mv;
        if (v >= vend) continue;
        float mm = -INFINITY, ll = 0.0f, acc[DT];
#pragma unroll
        for (int i = 0; i < DT; ++i) acc[i] = 0.0f;
#pragma unroll
        for (int w = 0; w < SW; ++w) mm = fmaxf(mm, sm[w][16 * q + mv]);
        const float ref = mm == -INFINITY ? 0.0f : mm;
#pragma unroll
        for (int w = 0; w < SW; ++w) {
            const float a = __builtin_amdgcn_exp2f(sm[w][16 * q + mv] - ref);
            ll = ll + sl[w][16 * q + mv] * a;
#pragma unroll
            for (int i = 0; i < DT; i += 4) {
                const float4 x = *reinterpret_cast<const float4*>(&so[w][mv][d0 + i]);
                acc[i] = acc[i] + x.x * a, acc[i + 1] = acc[i + 1] + x.y * a;
                acc[i + 2] = acc[i + 2] + x.z * a, acc[i + 3] = acc[i + 3] + x.w * a;
            }
        }
        const uint32_t iv = p.by_group.of(v);
        const uint64_t row = (uint64_t)(bl.r0 + iv) * p.nh + kvh * p.group + (v - iv * p.group);
        if (p.nsplit > 1) {
            const uint64_t at = row * p.nsplit + split;
#pragma unroll
            for (int i = 0; i < DT; i += 4)
                *reinterpret_cast<float4*>(p.part + at * HD + d0 + i) = make_float4(acc[i], acc[i + 1], acc[i + 2], acc[i + 3]);
            if (d0 == 0) p.ml[at] = make_float2(mm, ll);
        } else {
            E* dst = (E*)p.out + row * HD + d0;
#pragma unroll
            for (int i = 0; i < DT; ++i) T::put(dst + i, ll == 0.0f ? 0.0f : acc[i] / ll);
            if (p.lse && d0 == 0) p.lse[row] = ll == 0.0f ? -INFINITY : (mm + log2f(ll)) * LN2;
        }
    }
}

// ---------------------------------------------------------------- many rows
//
// NW waves of 32 query vectors each walk the keys 64 at a time, through LDS:
// codes go global -> registers -> bf16 -> LDS once for all, one tile in LDS
// and one in registers ahead of the products, with one barrier a tile.
// v_mfma_f32_32x32x16_bf16 on scores transposed (keys x queries), so that a lane
// has 16 keys of one query, which are the operand of the second product for the
// order of keys that V^T is stored in.
//
// The vector unit's work for each score is kept small, since it takes as long as
// the products: the key's scale goes into the exponent's fma, and the reference
// of the softmax is not the running maximum but below it by up to 2^ROOM, which
// floats hold as well (the exponent's rounding is that of the score itself). That
// a tile stays within ROOM is seen before it is computed, from |q| |k|, so that
// the loop of most tiles has no comparisons and no rescaling of the context (the
// registers of the two are what lets the products of one half tile run beside
// the exponentials of another). A tile for which the bound says nothing, such as
// a sequence's first, takes a step that looks at the scores and moves the
// reference where one lies more than 2^SLACK above it.
//
// A prompt's last 2048 rows over 32768 keys, 32 heads over 8 of 128, bf16: 1.10 to
// 1.17 ms by the card, 910 to 970 TFLOP/s, where a large library product reaches
// 1190 (the matrix unit is busy for 41 % of the cycles and the vector unit, with 32
// exponentials a lane and tile, for 65 %; 1.94 GHz under that load). f32, three products for one: 1000
// rows over 8000 keys in 407 us, 900 TFLOP/s of products. One kernel serves a call, chosen
// for its longest chunk, so that single tokens beside a chunk take a block each
// here: 63 of them and 256 rows over up to 8192 keys 550 us (bf16), where the
// 256 rows alone take 97 and 64 single tokens, streaming, 197.
constexpr int TK = 64;  // keys of a tile
// 2^(ROOM + 7) (codes) times value scales below VMOST times 2^28 keys is finite.
constexpr float SLACK = 6.0f, ROOM = 72.0f, VMOST = 1048576.0f;
typedef float v16f __attribute__((ext_vector_type(16)));

__device__ __forceinline__ v16f mfma32(v4i a, v4i b, v16f c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(v8bf, a), __builtin_bit_cast(v8bf, b), c, 0, 0, 0);
}

// Waves of a workgroup (one workgroup a compute unit: LDS), 32 query vectors
// each: four, so that each has a SIMD's registers, where f32 queries of 128 in
// three parts need them (1000 rows over 8000 keys 407 us; eight waves spilled,
// 470), else eight, which stage each tile for twice the queries (f32 of 64, 500
// rows of 4 sequences over 3000 keys: 36 us, with four 46).
template <class T, int HD>
constexpr int tile_waves() {
    return sizeof(typename T::elem) == 4 && HD == 128 ? 4 : 8;
}

template <class T, int HD>
__global__ __launch_bounds__((tile_waves<T, HD>() * 64), (tile_waves<T, HD>() / 4)) void paged_attention_tile_kernel(AttnArgs p) {
    typedef typename T::elem E;
    constexpr int TW = tile_waves<T, HD>(), TVB = 32 * TW;
    constexpr int PARTS = sizeof(E) == 4 ? 3 : 1, NT = TW * 64, NBUF = 3;
    // Bytes in LDS: a key, a line of values, those of 32 keys, a tile of each.
    constexpr int KROW = HD * 2 + 16, VROW = 256 + 16, VHALF = HD / 4 * VROW, KB = TK * KROW, VB = 2 * VHALF;
    __shared__ __attribute__((aligned(1024))) uint8_t kt[NBUF][KB], vt[NBUF][VB];
    __shared__ __attribute__((aligned(16))) float scs[NBUF][2][TK];  // keys', values' scales
    __shared__ int kn2[NBUF][TK];                                      // |codes|^2 of each key
    __shared__ __attribute__((aligned(16))) uint64_t ring[4][TK];      // bytes to each key's slot
    __shared__ unsigned long long okm[4];                              // which keys have one
    const int tid = threadIdx.x, lane = tid & 63, col = lane & 31, half = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t nkv = p.kv.nkv, kvs = nkv * HD, units = p.blocks * p.nsplit;
    const uint32_t turn = p.by_nkv.of(blockIdx.x / 8), kvh = blockIdx.x / 8 - turn * nkv;
    const uint32_t unit = turn * 8 + blockIdx.x % 8;
    if (unit >= units) return;
    const uint32_t blk = p.by_nsplit.of(unit), split = unit - blk * p.nsplit;
    Block bl;
    if (!find_block<TVB>(p.bt, p.group, blk, lane, bl)) return;
    const uint32_t reach = p.kv.reach();
    const uint32_t vend = min(bl.v0 + TVB, bl.nv);
    const uint32_t kend = min(keys_seen(bl, p.by_group.of(vend - 1)), reach);
    const uint32_t k0 = split * p.span, k1 = split + 1 == p.nsplit ? kend : min(kend, k0 + p.span);
    if (k0 >= k1 && split) return;
    const int nt = k1 > k0 ? (int)((k1 - k0 + TK - 1) / TK) : 0;

    // This wave's 32 vectors, and what its first and last see.
    const uint32_t wv0 = bl.v0 + 32 * wave, wv1 = min(wv0 + 32, vend);
    const bool wlive = wv0 < vend;
    const uint32_t wall = wlive ? min(keys_seen(bl, p.by_group.of(wv0)), reach) : 0u;
    const uint32_t wend = wlive ? min(keys_seen(bl, p.by_group.of(wv1 - 1)), reach) : 0u;
    v16f o[HD / 32];
    float m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int j = 0; j < HD / 32; ++j)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[j][e] = 0.0f;

    // ---- staging
    const uint8_t* kp = (const uint8_t*)p.kv.pool[0] + (size_t)kvh * HD;
    const uint8_t* vp = (const uint8_t*)p.kv.pool[1] + (size_t)kvh * HD;
    const uint8_t* sp = (const uint8_t*)((wave & 1 ? p.kv.scales[1] : p.kv.scales[0]) + kvh);  // even waves take the keys' scales
    auto barrier = [&]() {  // orders LDS only: loads in flight go on
        __builtin_amdgcn_sched_barrier(0);
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
    };
    // Where tile t's keys lie: wave t % TW looks the tables up, two steps before
    // the loads need it. A key behind the end or without a slot gets slot 0.
    auto slot_at = [&](int t) -> uint32_t {
        const uint32_t j = k0 + (uint32_t)t * TK + lane;
        return j < k1 ? p.kv.slot(bl.b, j) : NO_SLOT;
    };
    auto put_slots = [&](int t, uint32_t s) {
        ring[t & 3][lane] = s != NO_SLOT ? (uint64_t)s * kvs : 0u;
        okm[t & 3] = __ballot(s != NO_SLOT);
    };
    // The first look-ups, the queries and the first two tiles go out before
    // anything waits for the queries.
    const uint32_t sl_first = wave < 4 ? slot_at(wave) : NO_SLOT;
    uint32_t sl_next = wave == 4 % TW ? slot_at(4) : NO_SLOT;
    uint32_t seen;
    const bool dead = wv0 + col >= vend;  // no vector: computes the last one's again, its sums are not used
    float qx[HD / 16][8];  // step t: d = 16 t + 8 half ..+7 of vector col
    {
        const uint32_t v = min(wv0 + col, vend - 1), i = p.by_group.of(v), h = kvh * p.group + (v - i * p.group);
        seen = wv0 + col < vend ? min(keys_seen(bl, i), reach) : 0u;
        const E* src = (const E*)p.q + (bl.r0 + i) * p.qs + (uint64_t)h * HD + 8 * half;
        query8<T>(src, qx, [](int t) { return 16 * t; });
    }
    if (wave < 4) put_slots(wave, sl_first);
    barrier();
    // A thread takes 16 bytes of a key and four values' four bytes, PR times (8
    // waves and HD 64: one of the two).
    constexpr int CPK = HD / 16, DG = HD / 4, KP = TK * CPK, VP = TK / 4 * DG;  // pieces
    static_assert(KP == VP && (KP % NT == 0 || NT == 2 * KP), "whole pieces for each thread");
    constexpr int PR = KP > NT ? KP / NT : 1, VT = NT > VP ? NT - VP : 0;  // VT: the first thread with values
    const bool klive = KP >= NT || tid < KP, vlive = VT == 0 || tid >= VT;
    const int kkey = tid / CPK, kpc = tid % CPK, quad = (tid - VT) / DG, dg = (tid - VT) % DG;
    struct Raw {
        v4i k[PR];
        uint32_t v[PR][4];
        float s;
    };
    auto load = [&](int t, Raw& x) __attribute__((always_inline)) {
        const uint64_t* sl = ring[t & 3];
#pragma unroll
        for (int r = 0; r < PR; ++r) {
            if (klive) x.k[r] = *reinterpret_cast<const v4i*>(kp + sl[kkey + r * (NT / CPK)] + 16 * kpc);
            if (vlive) {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    x.v[r][i] = *reinterpret_cast<const uint32_t*>(vp + sl[4 * (quad + r * (NT / DG)) + i] + 4 * dg);
            }
        }
        x.s = *reinterpret_cast<const float*>(sp + sl[lane] / (HD / 4));
    };
    Raw raw, second;
    load(0, raw);
    load(1, second);
    __builtin_amdgcn_sched_barrier(0);
    float qn = 0.0f, qm = 0.0f;
    v4i qf[HD / 16][PARTS];
#pragma unroll
    for (int t = 0; t < HD / 16; ++t) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            qn = qn + qx[t][e] * qx[t][e];
            qm = fmaxf(qm, fabsf(qx[t][e]));
        }
        split8<PARTS>(qx[t], qf[t]);
    }
    // Above |q|, whatever the roundings: from 2^-100 on a sum of squares has lost
    // less than a 2^-18th to those below f32's range; one below that (1e-25 each:
    // all of it) gives way to HD times the largest. Infinite or NaN (no bound: a
    // NaN here would be lost in the maximum) becomes infinite.
    qn = qn + xor_lane<32>(qn);
    qm = fmaxf(qm, xor_lane<32>(qm));
    qn = (qn < 0x1p-100f ? qm * sqrtf((float)HD) : sqrtf(qn)) * 1.001f;
    qn = dead ? 0.0f : qn < INFINITY ? qn : INFINITY;
    // LDS images. K: chunk c (8 d) of key r. V^T: 32 keys at a time, lines of 256
    // bytes hold 4 d x 32 keys, 8 keys a chunk in the order of a lane's scores:
    // chunk 2u + h has keys 16u + 4h ..+3 and 16u + 8 + 4h ..+3. In both 16
    // bytes of padding send the 16 lanes that meet to different banks (and leave the
    // places of a lane's reads constants apart).
    auto kchunk = [&](int r, int c) -> int { return r * KROW + (c << 4); };
    auto vchunk = [&](int d, int oc) -> int {
        return (oc >> 2) * VHALF + (d >> 2) * VROW + ((4 * (d & 3) + (oc & 3)) << 4);
    };
    const int kst = klive ? kchunk(kkey, 2 * kpc) : 0;
    // quad: keys 4 quad ..+3 = 16 u' + 4 x: chunk (quad / 4) * 2 + (quad & 1), its half (quad >> 1) & 1
    const int vst = vlive ? vchunk(4 * dg, 2 * (quad >> 2) + (quad & 1)) + 8 * ((quad >> 1) & 1) : 0;
    // Piece r: 16 n keys on, and 16 n values: the same place of a later line.
    auto store_k = [&](int bu, int r) __attribute__((always_inline)) {
        if (!klive) return;
        uint8_t* at = kt[0] + bu * KB + r * (NT / CPK) * KROW;
        *reinterpret_cast<v4i*>(at + kst) = codes8((uint32_t)raw.k[r][0], (uint32_t)raw.k[r][1]);
        *reinterpret_cast<v4i*>(at + (kst + 16)) = codes8((uint32_t)raw.k[r][2], (uint32_t)raw.k[r][3]);
        int n2 = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) n2 = __builtin_amdgcn_sdot4(raw.k[r][i], raw.k[r][i], n2, false);
        n2 += (int)xor_lane_u<1>((uint32_t)n2);  // the CPK lanes of a key
        n2 += (int)xor_lane_u<2>((uint32_t)n2);
        if constexpr (CPK == 8) n2 += (int)xor_lane_u<4>((uint32_t)n2);
        kn2[bu][kkey + r * (NT / CPK)] = n2;
    };
    auto store_v = [&](int bu, unsigned long long ok, int r) __attribute__((always_inline)) {
        if (vlive) {
            uint8_t* at = vt[0] + bu * VB + r * (NT / DG / 8) * VHALF;
#pragma unroll
            for (int e = 0; e < 4; ++e)  // dimension 4 dg + e: chunk index + 4 e
                *reinterpret_cast<uint2*>(at + vst + (e << 6)) = make_uint2(
                    hi16x2(code_f(raw.v[r][0], e), code_f(raw.v[r][1], e)), hi16x2(code_f(raw.v[r][2], e), code_f(raw.v[r][3], e)));
        }
        if (r) return;
        // A key without a slot has scales of 0. (Waves of a kind write the same.)
        const float sc = (ok >> lane) & 1ull ? (wave & 1 ? raw.s : raw.s * p.scale2) : 0.0f;
        scs[bu][wave & 1][lane] = sc;
    };
    auto store = [&](int bu, unsigned long long ok) __attribute__((always_inline)) {
#pragma unroll
        for (int r = 0; r < PR; ++r) store_k(bu, r), store_v(bu, ok, r);
    };
    static_assert(PR == 1 || (NT / DG) % 8 == 0, "the pieces' places");
    // Scores of half kh of the tile in buffer bu. Register e: key 32 kh +
    // 8 (e / 4) + 4 half + e % 4.
    auto scores = [&](int bu, int kh, v16f& s) __attribute__((always_inline)) {
        const int ka = bu * KB + kh * (32 * KROW) + kchunk(col, half);
#pragma unroll
        for (int e = 0; e < 16; ++e) s[e] = 0.0f;
#pragma unroll
        for (int d = 0; d < HD / 16; ++d) {
            const v4i k = *reinterpret_cast<const v4i*>(kt[0] + ka + (d << 5));
#pragma unroll
            for (int part = PARTS - 1; part >= 0; --part) s = mfma32(k, qf[d][part], s);
        }
    };
    // Whether the tile in buffer bu stays within ROOM of every query's reference
    // (lane l looks at key l, for the longest query and the lowest reference; a
    // scale that is not a number says no).
    const float qmost = xor_max<32>(qn);
    float mleast = -INFINITY;
    auto within = [&](int bu) -> bool {
        const float size = __builtin_amdgcn_sqrtf((float)kn2[bu][lane]) * fabsf(scs[bu][0][lane]);
        return __all(qmost * size <= mleast + ROOM && fabsf(scs[bu][1][lane]) < VMOST);
    };
    // The keys (bit 8 (e / 4) + e % 4 of register e) that this lane's query sees in
    // half kh of the tile from j0 on.
    auto visible = [&](int kh, uint32_t j0, unsigned long long ok) -> uint32_t {
        const int lim = (int)(seen - j0) - 32 * kh - 4 * half;
        return (uint32_t)(ok >> (32 * kh)) >> (4 * half) & (lim >= 32 ? ~0u : (1u << max(lim, 0)) - 1u);
    };
    // Moves the reference to the largest score where that is more than SLACK
    // above it, each query for itself (ok: the keys that have a slot).
    auto refer = [&](int bu, int kh, uint32_t j0, unsigned long long ok, const v16f& s) __attribute__((always_inline)) {
        const float* kcp = &scs[bu][0][32 * kh + 4 * half];
        const uint32_t vis = visible(kh, j0, ok);
        float mx = -INFINITY;
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const float4 kc = *reinterpret_cast<const float4*>(kcp + 8 * g);
            float a[4] = {s[4 * g] * kc.x, s[4 * g + 1] * kc.y, s[4 * g + 2] * kc.z, s[4 * g + 3] * kc.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                asm volatile("" : "+v"(a[i]));  // no branch around each
                mx = fmaxf(mx, (vis >> (8 * g + i)) & 1u ? a[i] : -INFINITY);
            }
        }
        mx = fmaxf(mx, xor_lane<32>(mx));
        const bool up = mx > m + SLACK;
        if (!__any(up)) return;
        const float alpha = up ? __builtin_amdgcn_exp2f(m - mx) : 1.0f;
        l = l * alpha;
#pragma unroll
        for (int j = 0; j < HD / 32; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) o[j][e] = o[j][e] * alpha;
        m = up ? mx : m;
        const float none = dead ? 0.0f : m;
        mleast = -xor_max<32>(-none);
    };
    // Weights of registers 8 u ..+7 of a half's scores, times their values' scales.
    auto weights = [&](int bu, int kh, int u, uint32_t j0, unsigned long long ok, const v16f& s,
                       v4i (&pf)[PARTS]) __attribute__((always_inline)) {
        const float *kcp = &scs[bu][0][32 * kh + 4 * half], *vsp = &scs[bu][1][32 * kh + 4 * half];
        const uint32_t vis = visible(kh, j0, ok);
        const float ref = m == -INFINITY ? 0.0f : m;
        float x[8];
#pragma unroll
        for (int i4 = 0; i4 < 2; ++i4) {
            const int k_ = 16 * u + 8 * i4;
            const float4 kc = *reinterpret_cast<const float4*>(kcp + k_), vs = *reinterpret_cast<const float4*>(vsp + k_);
            const float kk[4] = {kc.x, kc.y, kc.z, kc.w}, vv[4] = {vs.x, vs.y, vs.z, vs.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const bool hid = !((vis >> (k_ + i)) & 1u);
                float a = __builtin_fmaf(s[8 * u + 4 * i4 + i], kk[i], -ref);
                if (hid) a = -INFINITY;
                const float w = __builtin_amdgcn_exp2f(a);
                l = l + w;
                x[4 * i4 + i] = hid ? 0.0f : w * vv[i];  // whatever its scale is
            }
        }
        split8<PARTS>(x, pf);
    };
    // Their product with the values.
    auto values = [&](int bu, int kh, int u, const v4i (&pf)[PARTS]) __attribute__((always_inline)) {
        const int va = bu * VB + kh * VHALF + vchunk(col, half) + (u << 5);  // vchunk(32 j + col, 2 u + half)
#pragma unroll
        for (int j = 0; j < HD / 32; ++j) {
            const v4i v = *reinterpret_cast<const v4i*>(vt[0] + va + j * (8 * VROW));
#pragma unroll
            for (int part = PARTS - 1; part >= 0; --part) o[j] = mfma32(v, pf[part], o[j]);
        }
    };

    auto ok_of = [&](int t) -> unsigned long long {
        const unsigned long long ok = okm[t & 3];
        return (unsigned long long)(uint32_t)__builtin_amdgcn_readfirstlane((int)(ok >> 32)) << 32 |
               (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)ok);
    };
    unsigned long long ok0 = ok_of(0), ok1 = ok_of(1), ok2 = ok_of(2);  // of tiles t .. t + 2
    store(0, ok0);
    raw = second;
    store(1, ok1);
    load(2, raw);
    barrier();
    // In step t tile t + 2 goes to LDS, whose buffer was last read in step t - 1.
    int b0 = 0, b1 = 1, b2 = 2;
    v16f s0, s1;
    bool calm = false;  // the next tile is within its bound and seen whole by all of the wave's queries
    auto rest = [&](int t) __attribute__((always_inline)) {
        const uint32_t j0 = k0 + (uint32_t)t * TK;
        load(t + 3, raw);
        calm = j0 + 2 * TK <= wall && ok1 == ~0ull && within(b1);
        ok0 = ok1, ok1 = ok2, ok2 = ok_of(t + 3);
        if (((t + 4) & (TW - 1)) == wave) put_slots(t + 4, sl_next);
        if (((t + 5) & (TW - 1)) == wave) sl_next = slot_at(t + 5);
        const int b = b0;
        b0 = b1, b1 = b2, b2 = b;
        barrier();
    };
    // Any tile, one thing after another.
    auto step = [&](int t) __attribute__((always_inline)) {
        const uint32_t j0 = k0 + (uint32_t)t * TK;
        store(b2, ok2);
        if (j0 < wend) {
#pragma unroll
            for (int kh = 0; kh < 2; ++kh) {
                v4i pf[PARTS];
                scores(b0, kh, s0);
                refer(b0, kh, j0, ok0, s0);
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    __builtin_amdgcn_sched_barrier(0);
                    weights(b0, kh, u, j0, ok0, s0, pf);
                    values(b0, kh, u, pf);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        rest(t);
    };
    // A calm tile. The products are laid out with the vector work that is to run
    // beside them, one product (32 cycles) and its share between two scheduling
    // barriers, and the operands of a product are read two products ahead. bf16:
    // beside the next half's scores go the weights of 8 of this half's keys;
    // beside their product with V the weights of the other 8; beside those'
    // product the conversion of a tile to come. f32: three products for each,
    // so that all weights fit beside the next scores; and since a wave has its
    // SIMD for itself, the vector work is dealt out product by product.
    constexpr int NS = HD / 16, NJ = HD / 32;
    constexpr bool WIDE = PARTS == 3;
    v4i ka_[2];     // the first two operands of the next scores
    float4 kc_, vs_;  // scales of the next 4 keys
    auto fence = [&]() { __builtin_amdgcn_sched_barrier(0); };
    auto kaddr = [&](int bu, int kh) -> int { return bu * KB + kh * (32 * KROW) + kchunk(col, half); };
    auto prime = [&](int kbase, int bu, int kh) __attribute__((always_inline)) {
        kc_ = *reinterpret_cast<const float4*>(&scs[bu][0][32 * kh + 4 * half]);
        vs_ = *reinterpret_cast<const float4*>(&scs[bu][1][32 * kh + 4 * half]);
        ka_[0] = *reinterpret_cast<const v4i*>(kt[0] + kbase);
        ka_[1] = *reinterpret_cast<const v4i*>(kt[0] + kbase + 32);
    };
    auto calm_half = [&](int kh, int kbase, const v16f& s, v16f& nx, int nbase, int nbu, int nkh) __attribute__((always_inline)) {
        const float* kcp = &scs[b0][0][32 * kh + 4 * half];  // values' scales: TK floats on
        const int va0 = b0 * VB + kh * VHALF + vchunk(col, half), va1 = va0 + 32;
        auto vread = [&](int va, int j) -> v4i { return *reinterpret_cast<const v4i*>(vt[0] + va + j * (8 * VROW)); };
        float x[16];
        float4 kc[4], vs[4];
        v4i kf[NS], vf[2][NJ], pf[PARTS], pg[PARTS];
        kc[0] = kc_, vs[0] = vs_, kf[0] = ka_[0], kf[1] = ka_[1];
        // Key register e: its weight's exponential, then (one product later) the rest.
        const float ref = dead ? 0.0f : m;  // (finite where not dead: mleast is)
        float w[16];
        auto at = [](const float4& v, int i) -> float { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; };
        auto raise = [&](int e) { w[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[e], at(kc[e >> 2], e & 3), -ref)); };
        auto finish = [&](int e) {
            l = l + w[e];
            x[e] = w[e] * at(vs[e >> 2], e & 3);
        };
        auto scales = [&](int g4) {  // of keys 8 g4 ..
            kc[g4] = *reinterpret_cast<const float4*>(kcp + 8 * g4);
            vs[g4] = *reinterpret_cast<const float4*>(kcp + TK + 8 * g4);
        };
        auto pair = [&](int k) { split2<PARTS>(x[2 * k], x[2 * k + 1], k & 3, k < 4 ? pf : pg); };
        auto products = [&](const v4i& a, const v4i (&b)[PARTS], v16f& c) {
#pragma unroll
            for (int part = PARTS - 1; part >= 0; --part) c = mfma32(a, b[part], c);
        };
        // f32: the vector work of a stretch of n products dealt out to each of them.
        auto deal = [&](auto n, auto each) __attribute__((always_inline)) {
#pragma unroll
            for (int i = 0; i < n(); ++i) {
                __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
                __builtin_amdgcn_sched_group_barrier(0x2, each(), 0);
            }
        };
        typedef std::integral_constant<int, 3> N3;
        typedef std::integral_constant<int, 7> N7;
        typedef std::integral_constant<int, 8> N8;
        typedef std::integral_constant<int, 3 * NJ> NV;
        constexpr int EP = WIDE ? 16 / NS : 8 / NS;
#pragma unroll
        for (int e = 0; e < 16; ++e) nx[e] = 0.0f;
#pragma unroll
        for (int d = 0; d < NS; ++d) {
            products(kf[d], qf[d], nx);
            if (d + 2 < NS) kf[d + 2] = *reinterpret_cast<const v4i*>(kt[0] + kbase + ((d + 2) << 5));
            if constexpr (WIDE) {  // (of the slot after next, or the next)
                if (EP * (d + 1) % 4 != 0 && EP * d / 4 < 3) scales(EP * d / 4 + 1);
                if (EP == 4 && d < 3) scales(d + 1);
            } else {
                if (d == 0) scales(1);
                if (d == NS - 2) scales(2);
            }
            if (d == NS - 2) vf[0][0] = vread(va0, 0);
            if (d == NS - 1) vf[0][1] = vread(va0, 1);
#pragma unroll
            for (int i = 0; i < EP; ++i) raise(EP * d + i);
            if (d)
#pragma unroll
                for (int i = 0; i < EP; ++i) {
                    const int e = EP * (d - 1) + i;
                    finish(e);
                    if (WIDE && e % 2) pair(e / 2);
                }
            if constexpr (WIDE) deal(N3{}, N7{});
            fence();
        }
        if constexpr (WIDE) {
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
                products(vf[0][j], pf, o[j]);
                if (j + 2 < NJ) vf[0][j + 2] = vread(va0, j + 2);
                else vf[1][j + 2 - NJ] = vread(va1, j + 2 - NJ);
            }
#pragma unroll
            for (int e = 16 - EP; e < 16; ++e) {
                finish(e);
                if (e % 2) pair(e / 2);
            }
            if (PR == 2) {
                if (kh == 0) store_k(b2, 1);
                else store_v(b2, ok2, 1);
            }
            deal(NV{}, N8{});
            fence();
        } else {
#pragma unroll
            for (int i = 0; i < EP; ++i) finish(8 - EP + i);
#pragma unroll
            for (int k = 0; k < 4; ++k) pair(k);
            fence();
            constexpr int EV = 8 / NJ;
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
                products(vf[0][j], pf, o[j]);
                if (j + 2 < NJ) vf[0][j + 2] = vread(va0, j + 2);
                else vf[1][j + 2 - NJ] = vread(va1, j + 2 - NJ);
                if (j == 0) scales(3);
#pragma unroll
                for (int i = 0; i < EV; ++i) raise(8 + EV * j + i);
                if (j)
#pragma unroll
                    for (int i = 0; i < EV; ++i) finish(8 + EV * (j - 1) + i);
                fence();
            }
#pragma unroll
            for (int i = 0; i < EV; ++i) finish(16 - EV + i);
#pragma unroll
            for (int k = 4; k < 8; ++k) pair(k);
            fence();
        }
        prime(nbase, nbu, nkh);
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            products(vf[1][j], pg, o[j]);
            if (j + 2 < NJ) vf[1][j + 2] = vread(va1, j + 2);
        }
        if (kh == 0) store_k(b2, 0);
        else store_v(b2, ok2, 0);
        if constexpr (WIDE) deal(NV{}, N8{});
        fence();
    };
    auto calm_step = [&](int t) __attribute__((always_inline)) {
        const int kb0 = kaddr(b0, 1), kb1 = kaddr(b1, 0), kb2 = kaddr(b1, 1);
        calm_half(0, kb0, s0, s1, kb1, b0, 1);
        calm_half(1, kb1, s1, s0, kb2, b1, 0);
        rest(t);
    };
    // (Each wave passes one barrier a tile in whichever loop it is.)
    for (int t = 0; t < nt;) {
        step(t++);
        if (t < nt && calm) {
            scores(b0, 0, s0);
            prime(kaddr(b0, 1), b0, 0);
        }
#pragma unroll 1
        while (t < nt && calm) calm_step(t++);
    }
    const uint32_t v = wv0 + col;
    l = l + xor_lane<32>(l);
    if (v >= vend) return;
    const uint32_t iv = p.by_group.of(v);
    const uint64_t row = (uint64_t)(bl.r0 + iv) * p.nh + kvh * p.group + (v - iv * p.group);
    if (p.nsplit > 1) {
        const uint64_t at = row * p.nsplit + split;
#pragma unroll
        for (int j = 0; j < HD / 32; ++j)
#pragma unroll
            for (int e4 = 0; e4 < 4; ++e4)
                *reinterpret_cast<float4*>(p.part + at * HD + 32 * j + 8 * e4 + 4 * half) =
                    make_float4(o[j][4 * e4], o[j][4 * e4 + 1], o[j][4 * e4 + 2], o[j][4 * e4 + 3]);
        if (half == 0) p.ml[at] = make_float2(m, l);
        return;
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    E* dst = (E*)p.out + row * HD;
#pragma unroll
    for (int j = 0; j < HD / 32; ++j)
#pragma unroll
        for (int e4 = 0; e4 < 4; ++e4) {
            const float y[4] = {o[j][4 * e4] * inv, o[j][4 * e4 + 1] * inv, o[j][4 * e4 + 2] * inv, o[j][4 * e4 + 3] * inv};
            if (p.ovec) T::put4(dst + 32 * j + 8 * e4 + 4 * half, y);
            else
#pragma unroll
                for (int i = 0; i < 4; ++i) T::put(dst + 32 * j + 8 * e4 + 4 * half + i, y[i]);
        }
    if (p.lse && half == 0) p.lse[row] = l == 0.0f ? -INFINITY : (m + log2f(l)) * LN2;
}

// Joins the splits of a row and head, one wave for each: lane s takes split s's
// maximum and sum (at most 64 splits), then all take their dimensions, eight
// splits' loads at once. Bound by the trip to memory, 4 us for few rows, and by
// the splits' bytes for many (1443 rows of 28 heads of 128, three splits: 24 us).
template <class T, int HD, int VB>
__global__ __launch_bounds__(256) void paged_attention_join_kernel(AttnArgs p) {
    typedef typename T::elem E;
    const uint32_t lane = threadIdx.x & 63;
    const uint32_t rh = __builtin_amdgcn_readfirstlane((int)(blockIdx.x * 4 + (threadIdx.x >> 6)));
    const uint32_t r = rh / p.nh, h = rh % p.nh;
    if (r >= p.bt.rows) return;
    uint32_t b = r;
    if (p.bt.start) b = wave_last(p.bt.batch, lane, [&](uint32_t i) { return p.bt.start[i] <= r; });
    b = __builtin_amdgcn_readfirstlane((int)b);
    if (b >= p.bt.batch) return;
    Block bl;
    bl.b = b, bl.r0 = p.bt.first(b);
    const uint32_t r1 = p.bt.end(b);
    if (r >= r1) return;
    bl.n = r1 - bl.r0, bl.nv = bl.n * p.group, bl.len = p.bt.len(b);
    const uint32_t v = (r - bl.r0) * p.group + h % p.group;
    const uint32_t reach = p.kv.reach();
    const uint32_t kend = min(keys_seen(bl, (min((v / VB + 1) * VB, bl.nv) - 1) / p.group), reach);  // of the vector's block
    const uint32_t live = max(1u, min(p.nsplit, (kend + p.span - 1) / p.span));                  // splits that had keys
    const uint64_t at = (uint64_t)rh * p.nsplit;
    const float2 ml = lane < live ? p.ml[at + lane] : make_float2(-INFINITY, 0.0f);
    const float mm = xor_max<32>(ml.x), ref = mm == -INFINITY ? 0.0f : mm;
    const float a = __builtin_amdgcn_exp2f(ml.x - ref);
    const float ll = xor_sum<32>(lane < live ? ml.y * a : 0.0f);
    constexpr int DL = HD / 64;
    float acc[DL];
#pragma unroll
    for (int i = 0; i < DL; ++i) acc[i] = 0.0f;
    const float* src = p.part + at * HD + lane * DL;
    for (uint32_t s0 = 0; s0 < live; s0 += 8) {
        float x[8][DL];
#pragma unroll
        for (int u = 0; u < 8; ++u)
#pragma unroll
            for (int i = 0; i < DL; ++i) x[u][i] = src[min(s0 + u, live - 1) * HD + i];
        __builtin_amdgcn_sched_barrier(0);  // all on their way
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            const float w = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, a), (int)min(s0 + u, 63u)));
#pragma unroll
            for (int i = 0; i < DL; ++i) acc[i] = s0 + u < live ? acc[i] + x[u][i] * w : acc[i];
        }
    }
    E* dst = (E*)p.out + (uint64_t)rh * HD + lane * DL;
#pragma unroll
    for (int i = 0; i < DL; ++i) T::put(dst + i, ll == 0.0f ? 0.0f : acc[i] / ll);
    if (p.lse && lane == 0) p.lse[rh] = ll == 0.0f ? -INFINITY : (mm + log2f(ll)) * LN2;
}

// ---------------------------------------------------------------- weight sums
//
// The keys stay, the queries pass by: a wave holds the codes of 16 KG keys as
// operands of v_mfma_f32_16x16x32_bf16, loaded straight in its layout, and the
// workgroup's queries go through LDS 32 at a time, two buffers. A lane then has
// four queries' scores of one key, so a key's sum needs no exchange until the
// end, and its order is that of the rows. A workgroup takes 64 KG keys of one
// kv head, and more of them when the grid (made for max_len) does not reach.
// 1024 rows over 16384 keys, 32 heads over 8 of 128, bf16: 170 us, 790 TFLOP/s,
// with an exponential, an fma and a sum for every 128 multiply-adds: the matrix
// unit's cycles and the vector unit's add up to the whole, one after the other.
template <class T, int HD, int KG>
__global__ __launch_bounds__(256, 2) void paged_weight_sums_kernel(SumsArgs p) {
    typedef typename T::elem E;
    constexpr int PARTS = sizeof(E) == 4 ? 3 : 1, TQ = 32, ST = HD / 32, PB = TQ * HD * 2;
    __shared__ __attribute__((aligned(1024))) uint8_t qt[2][PARTS][PB];
    __shared__ __attribute__((aligned(16))) float lses[2][TQ];
    __shared__ __attribute__((aligned(16))) uint32_t sees[2][TQ];
    const int tid = threadIdx.x, lane = tid & 63, c = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    // All kv heads of a unit on one XCD: their scales share cache lines.
    const uint32_t nkv = p.kv.nkv, turn = p.by_nkv.of(blockIdx.x / 8), unit = turn * 8 + blockIdx.x % 8, kvh = blockIdx.x / 8 - turn * nkv;
    if (unit >= p.bt.batch * p.nchunk) return;
    Block bl;
    bl.b = p.by_nchunk.of(unit);
    const uint32_t r1 = p.bt.end(bl.b);
    bl.r0 = p.bt.first(bl.b);
    bl.n = r1 > bl.r0 ? r1 - bl.r0 : 0u;
    bl.nv = bl.n * p.group, bl.v0 = 0, bl.len = p.bt.len(bl.b);
    const uint32_t end = min(bl.len, p.cap), kvs = nkv * HD;
    float* acc = p.acc + ((uint64_t)bl.b * nkv + kvh) * p.cap;
    auto kchunk = [&](int r, int ch) -> int { return r * (HD * 2) + ((HD == 128 ? ch ^ (r & 15) : ch ^ ((r >> 1) & 7)) << 4); };
    // A thread brings HD / 8 elements of vector tid / 8 of a tile.
    constexpr int QE = HD / 8;
    const int qv = tid >> 3, qd = (tid & 7) * QE;
    for (uint64_t j0 = (uint64_t)(unit - bl.b * p.nchunk) * (64 * KG); j0 < end; j0 += (uint64_t)p.nchunk * (64 * KG)) {
        // Keys: group k of the wave, key c of it.
        v4i kf[KG][2 * HD / 64];
        float kc[KG], sum[KG], old[KG];
        bool live[KG];
        const uint32_t jw = (uint32_t)j0 + 16 * KG * wave;
#pragma unroll
        for (int k = 0; k < KG; ++k) {
            const uint32_t j = jw + 16 * k + c, slot = j < end ? p.kv.slot(bl.b, j) : NO_SLOT, s = slot != NO_SLOT ? slot : 0u;
            live[k] = slot != NO_SLOT;
            const uint8_t* src = (const uint8_t*)p.kv.pool[0] + (size_t)s * kvs + kvh * HD + 16 * g;
#pragma unroll
            for (int i = 0; i < HD / 64; ++i) {
                const v4i w = *reinterpret_cast<const v4i*>(src + 64 * i);
                kf[k][2 * i] = codes8((uint32_t)w[0], (uint32_t)w[1]);
                kf[k][2 * i + 1] = codes8((uint32_t)w[2], (uint32_t)w[3]);
            }
            kc[k] = p.kv.scales[0][(size_t)s * nkv + kvh] * p.scale2;
            sum[k] = 0.0f;
            old[k] = j < end && (uint64_t)j + bl.n < bl.len ? acc[j] : 0.0f;
        }
        // The first row that sees the first key, from a whole tile on.
        const uint64_t i0 = j0 + bl.n > bl.len ? j0 + bl.n - bl.len : 0;
        const uint32_t v0 = (uint32_t)min(i0 * p.group, (uint64_t)bl.nv) / TQ * TQ;
        float x[QE / 8][8], xl = 0.0f;
        uint32_t xs = 0;
        auto load = [&](uint32_t v) {
            const uint32_t vv = min(v + qv, bl.nv - 1), i = p.by_group.of(vv), h = kvh * p.group + (vv - i * p.group);
            const E* src = (const E*)p.q + (bl.r0 + i) * p.qs + (uint64_t)h * HD + qd;
            query8<T>(src, x, [](int n) { return 8 * n; });
            xl = p.lse[(uint64_t)(bl.r0 + i) * p.nh + h] * LOG2E;
            xs = v + qv < bl.nv ? keys_seen(bl, i) : 0u;
        };
        auto store = [&](int bu) {
#pragma unroll
            for (int u = 0; u < QE; u += 8) {
                v4i f[PARTS];
                split8<PARTS>(x[u / 8], f);
#pragma unroll
                for (int part = 0; part < PARTS; ++part)
                    *reinterpret_cast<v4i*>(&qt[bu][part][kchunk(qv, (qd + u) / 8)]) = f[part];
            }
            if ((tid & 7) == 0) lses[bu][qv] = xl, sees[bu][qv] = xs;
        };
        __syncthreads();  // the buffers are free
        if (v0 < bl.nv) {
            load(v0);
            store(0);
        }
        __syncthreads();
        int bu = 0;
#pragma unroll 1
        for (uint32_t v = v0; v < bl.nv; v += TQ, bu ^= 1) {
            const bool more = v + TQ < bl.nv;
            if (more) load(v + TQ);
            // Every vector of the tile sees every key of the wave.
            const bool masked = v + TQ > bl.nv || keys_seen(bl, p.by_group.of(v)) < (uint64_t)jw + 16 * KG;
#pragma unroll
            for (int sub = 0; sub < 2; ++sub) {
                v4f s[KG];
#pragma unroll
                for (int k = 0; k < KG; ++k) s[k] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int part = PARTS - 1; part >= 0; --part)
#pragma unroll
                    for (int t = 0; t < ST; ++t) {
                        const v4i a = *reinterpret_cast<const v4i*>(&qt[bu][part][kchunk(16 * sub + c, 2 * (g + 4 * (t >> 1)) + (t & 1))]);
#pragma unroll
                        for (int k = 0; k < KG; ++k) s[k] = mfma16(a, kf[k][t], s[k]);
                    }
                const float4 l4 = *reinterpret_cast<const float4*>(&lses[bu][16 * sub + 4 * g]);
                const float ll[4] = {l4.x, l4.y, l4.z, l4.w};
                if (!masked) {
#pragma unroll
                    for (int k = 0; k < KG; ++k)
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            sum[k] = sum[k] + __builtin_amdgcn_exp2f(__builtin_fmaf(s[k][r], kc[k], -ll[r]));
                } else {
                    const uint4 n4 = *reinterpret_cast<const uint4*>(&sees[bu][16 * sub + 4 * g]);
                    const uint32_t nn[4] = {n4.x, n4.y, n4.z, n4.w};
#pragma unroll
                    for (int k = 0; k < KG; ++k)
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            const float w = __builtin_amdgcn_exp2f(__builtin_fmaf(s[k][r], kc[k], -ll[r]));
                            sum[k] = sum[k] + (jw + 16 * k + c < nn[r] ? w : 0.0f);
                        }
                }
            }
            if (more) store(bu ^ 1);
            __syncthreads();
        }
#pragma unroll
        for (int k = 0; k < KG; ++k) {
            float w = sum[k] + xor_lane<16>(sum[k]);
            w = w + xor_lane<32>(w);
            const uint32_t j = jw + 16 * k + c;
            if (g == k % 4 && j < end) acc[j] = (live[k] ? w : 0.0f) + old[k];
        }
    }
}

// Few query vectors (rows x heads of a kv head up to 32, or 32 at a time): they
// stay in LDS and the keys stream by, each wave with the next 64 in flight and no
// barrier between. 32 sequences of up to 4096 keys, one row of 16 heads over 8 of
// 128, f32: 113 MB in 39 us, 2.9 TB/s, with a table look-up before each step's
// loads. (Look-ups a step further ahead: 43 us.)
template <class T, int HD>
__global__ __launch_bounds__(256, 2) void paged_weight_sums_stream_kernel(SumsArgs p) {
    typedef typename T::elem E;
    constexpr int PARTS = sizeof(E) == 4 ? 3 : 1, TQ = 32, ST = HD / 32, PB = TQ * HD * 2, KG = 4;
    __shared__ __attribute__((aligned(1024))) uint8_t qt[PARTS][PB];
    __shared__ __attribute__((aligned(16))) float lses[TQ];
    __shared__ __attribute__((aligned(16))) uint32_t sees[TQ];
    const int tid = threadIdx.x, lane = tid & 63, c = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t nkv = p.kv.nkv, turn = p.by_nkv.of(blockIdx.x / 8), unit = turn * 8 + blockIdx.x % 8;
    const uint32_t kvh = blockIdx.x / 8 - turn * nkv;
    if (unit >= p.bt.batch * p.nchunk) return;
    Block bl;
    bl.b = p.by_nchunk.of(unit);
    const uint32_t r1 = p.bt.end(bl.b);
    bl.r0 = p.bt.first(bl.b), bl.len = p.bt.len(bl.b);
    if (r1 <= bl.r0) return;
    bl.n = r1 - bl.r0, bl.nv = bl.n * p.group, bl.v0 = 0;
    const uint32_t end = min(min(bl.len, p.cap), KV_REACH), kvs = nkv * HD;
    float* acc = p.acc + ((uint64_t)bl.b * nkv + kvh) * p.cap;
    auto kchunk = [&](int r, int ch) -> int { return r * (HD * 2) + ((HD == 128 ? ch ^ (r & 15) : ch ^ ((r >> 1) & 7)) << 4); };
    constexpr int QE = HD / 8;
    const int qv = tid >> 3, qd = (tid & 7) * QE;
    const uint32_t first = ((unit - bl.b * p.nchunk) * 4 + wave) * 64, step = p.nchunk * 256;
    v4i kr[KG][HD / 64];  // codes of the keys in flight: group k of the wave, key c of it, bytes 16 (g + 4 i)
    float sr[KG], ar[KG];
    uint32_t slot[KG];
    auto look = [&](uint32_t j) {
#pragma unroll
        for (int k = 0; k < KG; ++k) slot[k] = p.kv.slot(bl.b, j + 16 * k + c);
    };
    auto load = [&](uint32_t j) {
#pragma unroll
        for (int k = 0; k < KG; ++k) {
            const uint32_t s = slot[k] != NO_SLOT ? slot[k] : 0u;
            const uint8_t* src = (const uint8_t*)p.kv.pool[0] + (size_t)s * kvs + kvh * HD + 16 * g;
#pragma unroll
            for (int i = 0; i < HD / 64; ++i) kr[k][i] = *reinterpret_cast<const v4i*>(src + 64 * i);
            sr[k] = p.kv.scales[0][(size_t)s * nkv + kvh];
            ar[k] = acc[min(j + 16 * k + c, end - 1)];
        }
    };
    for (uint32_t v = 0; v < bl.nv; v += TQ) {
        if (first < end) {
            look(first);
            load(first);
        }
        {  // thread: HD / 8 elements of vector tid / 8
            const uint32_t vv = min(v + qv, bl.nv - 1), i = p.by_group.of(vv), h = kvh * p.group + (vv - i * p.group);
            const E* src = (const E*)p.q + (bl.r0 + i) * p.qs + (uint64_t)h * HD + qd;
            float x[QE / 8][8];
            query8<T>(src, x, [](int n) { return 8 * n; });
            const float xl = p.lse[(uint64_t)(bl.r0 + i) * p.nh + h] * LOG2E;
            if (v) __syncthreads();  // the last vectors are done with
#pragma unroll
            for (int u = 0; u < QE / 8; ++u) {
                v4i f[PARTS];
                split8<PARTS>(x[u], f);
#pragma unroll
                for (int part = 0; part < PARTS; ++part) *reinterpret_cast<v4i*>(&qt[part][kchunk(qv, qd / 8 + u)]) = f[part];
            }
            if ((tid & 7) == 0) lses[qv] = xl, sees[qv] = v + qv < bl.nv ? keys_seen(bl, i) : 0u;
        }
        __syncthreads();
        const uint32_t all = v + TQ <= bl.nv ? keys_seen(bl, p.by_group.of(v)) : 0u;  // keys that all of the vectors see
        const int subs = bl.nv - v > 16 ? 2 : 1;
#pragma unroll 1
        for (uint32_t j0 = first; j0 < end; j0 += step) {
            v4i kf[KG][ST];
            float kc[KG], sum[KG], old[KG];
            bool live[KG];
#pragma unroll
            for (int k = 0; k < KG; ++k) {
#pragma unroll
                for (int i = 0; i < HD / 64; ++i) {
                    asm volatile("" : "+v"(kr[k][i]));  // (else they are carried from step to step byte by byte)
                    kf[k][2 * i] = codes8((uint32_t)kr[k][i][0], (uint32_t)kr[k][i][1]);
                    kf[k][2 * i + 1] = codes8((uint32_t)kr[k][i][2], (uint32_t)kr[k][i][3]);
                }
                kc[k] = sr[k] * p.scale2, sum[k] = 0.0f, live[k] = slot[k] != NO_SLOT;
                // The chunk's own keys start from 0, at the first vectors.
                old[k] = v || (uint64_t)(j0 + 16 * k + c) + bl.n < bl.len ? ar[k] : 0.0f;
            }
            __builtin_amdgcn_sched_barrier(0);
            if (j0 + step < end) {
                look(j0 + step);
                load(j0 + step);
            }
            __builtin_amdgcn_sched_barrier(0);
            const bool masked = all < j0 + 64;
            for (int sub = 0; sub < subs; ++sub) {
                v4f s[KG];
#pragma unroll
                for (int k = 0; k < KG; ++k) s[k] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int part = PARTS - 1; part >= 0; --part)
#pragma unroll
                    for (int t = 0; t < ST; ++t) {
                        const v4i a = *reinterpret_cast<const v4i*>(&qt[part][kchunk(16 * sub + c, 2 * (g + 4 * (t >> 1)) + (t & 1))]);
#pragma unroll
                        for (int k = 0; k < KG; ++k) s[k] = mfma16(a, kf[k][t], s[k]);
                    }
                const float4 l4 = *reinterpret_cast<const float4*>(&lses[16 * sub + 4 * g]);
                const uint4 n4 = *reinterpret_cast<const uint4*>(&sees[16 * sub + 4 * g]);
                const float ll[4] = {l4.x, l4.y, l4.z, l4.w};
                const uint32_t nn[4] = {n4.x, n4.y, n4.z, n4.w};
#pragma unroll
                for (int k = 0; k < KG; ++k)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const float w = __builtin_amdgcn_exp2f(__builtin_fmaf(s[k][r], kc[k], -ll[r]));
                        sum[k] = sum[k] + (!masked || j0 + 16 * k + c < nn[r] ? w : 0.0f);
                    }
            }
#pragma unroll
            for (int k = 0; k < KG; ++k) {
                float w = sum[k] + xor_lane<16>(sum[k]);
                w = w + xor_lane<32>(w);
                const uint32_t j = j0 + 16 * k + c;
                if (g == k && j < end) acc[j] = (live[k] ? w : 0.0f) + old[k];
            }
        }
    }
}

// KG 0: the streaming kernel.
template <class T, int HD, int KG>
hipError_t go_sums(hipStream_t s, SumsArgs a, uint64_t len) {
    constexpr uint32_t keys = KG ? 64 * KG : 256;
    const uint64_t pairs = (uint64_t)a.bt.batch * a.kv.nkv, most = std::max<uint64_t>(1, 0x7fffffffull / 8 / pairs);
    uint64_t chunks = std::min<uint64_t>((len + keys - 1) / keys, most);
    if (KG == 0) chunks = std::min<uint64_t>(chunks, (2 * CUS + pairs - 1) / pairs);
    a.nchunk = (uint32_t)chunks, a.by_nchunk = Div::by(a.nchunk);
    const uint64_t grid = ((uint64_t)a.bt.batch * a.nchunk + 7) / 8 * 8 * a.kv.nkv;
    if (grid > 0x7fffffffull) return hipErrorInvalidConfiguration;
    if constexpr (KG) paged_weight_sums_kernel<T, HD, KG><<<(unsigned)grid, 256, 0, s>>>(a);
    else paged_weight_sums_stream_kernel<T, HD><<<(unsigned)grid, 256, 0, s>>>(a);
    return hipGetLastError();
}
template <class T>
hipError_t go_weight_sums(hipStream_t s, const SumsArgs& a, const bh_kv8_batch* hint) {
    if ((a.kv.hd != 64 && a.kv.hd != 128) || a.kv.nslots == 0 || !aligned_to(a.kv.pool[0], 16)) {
        const uint32_t nchunk = (a.cap - 1) / 64 + 1;
        const uint64_t grid = (uint64_t)a.bt.batch * a.kv.nkv * nchunk;
        if (grid > 0x7fffffffull) return hipErrorInvalidConfiguration;
        paged_weight_sums_any_kernel<T><<<(unsigned)grid, 64, 0, s>>>(a, nchunk);
        return hipGetLastError();
    }
    const uint64_t len = std::max<uint64_t>(1, hint->max_len ? std::min(hint->max_len, a.cap) : a.cap);
    const uint32_t most = a.bt.start ? (hint->max_rows ? std::min(hint->max_rows, a.bt.rows) : a.bt.rows) : 1;
    // One row of 32 sequences over 4096 keys: streaming 39 us, the tiles below 48;
    // 7 rows of 16 (28 vectors): 20 and 24; 16 rows (64 vectors, twice the keys'
    // stream): 32 and 25.
    if ((uint64_t)most * a.group <= 32) return a.kv.hd == 128 ? go_sums<T, 128, 0>(s, a, len) : go_sums<T, 64, 0>(s, a, len);
    // Keys for each wave: 16 where chunks of 256 would give no compute unit a
    // second workgroup (64 rows of 4 sequences over 2000 keys: 10.3 us, 13.4 with
    // 64 keys), else 64, which read a query's fragment a quarter as often (1024 rows
    // over 12000 keys: 178 us, 277 with 16; over 8192, at the limit, 165 and 164).
    const bool few = (uint64_t)a.bt.batch * a.kv.nkv * ((len + 255) / 256) <= CUS;
    if (a.kv.hd == 128) return few ? go_sums<T, 128, 1>(s, a, len) : go_sums<T, 128, 4>(s, a, len);
    return few ? go_sums<T, 64, 1>(s, a, len) : go_sums<T, 64, 4>(s, a, len);
}

// How a call is run. PLAIN: any head_dim, any alignment.
enum Kind { PLAIN, STREAM, TILE };
struct Plan {
    Kind kind;
    uint32_t vb, blocks, nsplit, span;  // vb: query vectors of a block
    uint64_t part_floats, ml_pairs;
};
Plan plan_attention(const Kv8& kv, const Kv8Rows& bt, const bh_kv8_batch* hint, uint32_t nh, int dtype) {
    Plan r{};
    const uint32_t group = nh / kv.nkv;
    if (bt.rows == 0 || bt.batch == 0) return r;
    if ((kv.hd != 64 && kv.hd != 128) || kv.nslots == 0 || !aligned_to(kv.pool[0], 16) || !aligned_to(kv.pool[1], 16)) return r;
    const uint32_t most = bt.start ? (hint->max_rows ? std::min(hint->max_rows, bt.rows) : bt.rows) : 1;
    const uint64_t vectors = (uint64_t)most * group, all = (uint64_t)bt.rows * group;
    const bool f32 = dtype == BH_OUT_F32;
    // By the bytes of a sequence's queries: up to 160 vectors of 128 in bf16 and 80
    // in f32, 32 to a block, whose blocks find the codes in the caches. Streaming
    // and tiles (kernel time): 63 vectors of 16 sequences over 8000 keys 42 and 92
    // us (bf16), 79 and 137 (f32); 80 of 8 sequences 37 and 84, 68 and 124; 128 of
    // one 23 and 22 (bf16), 41 and 28 (f32); 240 of 8 over 2000 keys 30 and 33
    // (bf16), 105 of 16 over 16000 225 and 204 (f32). Heads of 64: 300 vectors of 8
    // over 4000 keys 26 and 48 (bf16).
    r.kind = vectors * kv.hd * (f32 ? 4 : 2) <= 40960 ? STREAM : TILE;
    r.vb = r.kind == TILE ? (f32 && kv.hd == 128 ? 32 * tile_waves<F32, 128>() : 256) : vectors <= 16 ? 16 : 32;
    r.blocks = !bt.start && group <= r.vb ? bt.batch : (uint32_t)(all / r.vb) + bt.batch;
    const uint64_t reach = kv_reach(kv.max_bt, kv.bs);
    const uint64_t len = std::max<uint64_t>(1, hint->max_len ? std::min<uint64_t>(hint->max_len, reach) : reach);
    // Splits of whole rounds: 32 keys for each wave, or two tiles.
    const uint32_t round = 128;
    const uint64_t rounds = (len + round - 1) / round;
    uint64_t wgs = (uint64_t)r.blocks * kv.nkv, want;
    if (r.kind == STREAM) {
        // Workgroups a compute unit: of 16 vectors 16 (64 sequences of up to 8192
        // keys: 178 us; 8: 202, 32: 185), of 32, with twice the state to join, 4 (80
        // vectors of 8 sequences, f32: 68 us; 2: 73, 8: 91).
        want = std::min<uint64_t>({rounds, ((r.vb == 16 ? 16 : 4) * CUS + wgs - 1) / wgs, 64});
    } else {
        // Three workgroups a compute unit, or no splits where whole rounds of one
        // leave less than a quarter of the chip idle (1000 f32 rows over 8000 keys,
        // 250 workgroups: 407 us, 480 in three splits; a mixed batch's 312: 324 us
        // whole and 300 split).
        wgs = std::max<uint64_t>(1, all / r.vb) * kv.nkv;
        want = std::min<uint64_t>({(rounds + 1) / 2, (3 * CUS + wgs - 1) / wgs, 32});
        if ((wgs + CUS - 1) / CUS * CUS * 3 <= wgs * 4) want = 1;
    }
    want = std::max<uint64_t>(1, want);
    r.span = (uint32_t)std::min<uint64_t>((rounds + want - 1) / want * round, 0x40000000u);
    r.nsplit = (uint32_t)((len + r.span - 1) / r.span);
    // Partial sums have places by row and head, not by a block's vectors: a single
    // token beside a long chunk, whose block is nearly empty, needs its own row only
    // (63 single tokens and 256 rows of 32 heads of 128 over up to 8192 keys: 112
    // MiB, by blocks 1519).
    if (r.nsplit > 1) {
        r.ml_pairs = (uint64_t)bt.rows * nh * r.nsplit;
        r.part_floats = r.ml_pairs * kv.hd;
    }
    return r;
}

template <class T, int HD, int VB>
hipError_t go_matrix(hipStream_t s, const AttnArgs& a, bool b16) {
    const uint64_t units = ((uint64_t)a.blocks * a.nsplit + 7) / 8 * 8 * a.kv.nkv;
    const uint64_t joins = ((uint64_t)a.bt.rows * a.nh + 3) / 4;
    if (units > 0x7fffffffull || joins > 0x7fffffffull) return hipErrorInvalidConfiguration;
    if constexpr (VB > 32) paged_attention_tile_kernel<T, HD><<<(unsigned)units, tile_waves<T, HD>() * 64, 0, s>>>(a);
    else if (b16) paged_attention_stream_kernel<T, HD, VB / 16, true><<<(unsigned)units, SW * 64, 0, s>>>(a);
    else paged_attention_stream_kernel<T, HD, VB / 16, false><<<(unsigned)units, SW * 64, 0, s>>>(a);
    hipError_t e = hipGetLastError();
    if (e == hipSuccess && a.nsplit > 1) {
        paged_attention_join_kernel<T, HD, VB><<<(unsigned)joins, 256, 0, s>>>(a);
        e = hipGetLastError();
    }
    return e;
}
template <class T, int HD>
hipError_t go_hd(hipStream_t s, const AttnArgs& a, const Plan& pl) {
    const bool b16 = a.kv.bs % 16 == 0 && a.kv.nslots % 16 == 0;
    switch (pl.vb) {
        case 16: return go_matrix<T, HD, 16>(s, a, b16);
        case 32: return go_matrix<T, HD, 32>(s, a, b16);
    }
    return go_matrix<T, HD, 32 * tile_waves<T, HD>()>(s, a, b16);
}
template <class T>
hipError_t go_attention(hipStream_t s, const AttnArgs& a, const Plan& pl) {
    if (pl.kind == PLAIN) {
        paged_attention_any_kernel<T><<<a.bt.rows * a.nh, 64, 0, s>>>(a);
        return hipGetLastError();
    }
    return a.kv.hd == 128 ? go_hd<T, 128>(s, a, pl) : go_hd<T, 64>(s, a, pl);
}

int done(hipError_t e, const char* who) {
    return e == hipSuccess ? BH_OK : fail(BH_ERR_HIP, "%s: %s", who, hipGetErrorString(e));
}

// The arguments that both calls have in common.
int check_call(const char* who, const bh_kv8* kv, const bh_kv8_batch* batch, uint32_t n_heads, int dtype, uint64_t qs,
               Kv8* k, Kv8Rows* r) {
    int rc;
    if ((rc = check_kv8(who, kv, k)) || (rc = check_kv8_batch(who, batch, r))) return rc;
    if (dtype != BH_OUT_F32 && dtype != BH_OUT_BF16)
        return fail(BH_ERR_INVALID, "%s: dtype %d, expected f32 or bf16", who, dtype);
    if (n_heads == 0 || n_heads % kv->n_kv_heads)
        return fail(BH_ERR_INVALID, "%s: %u query heads over %u kv heads", who, n_heads, kv->n_kv_heads);
    if ((uint64_t)batch->rows * n_heads > 0x7fffffffull || (uint64_t)n_heads * kv->head_dim > 0x7fffffffull)
        return fail(BH_ERR_INVALID, "%s: %u rows of %u heads", who, batch->rows, n_heads);
    if (batch->rows > 1 && qs < (uint64_t)n_heads * kv->head_dim)
        return fail(BH_ERR_INVALID, "%s: row stride %llu is shorter than a row", who, (unsigned long long)qs);
    return BH_OK;
}

}  // namespace
}  // namespace bh

using namespace bh;

extern "C" int bh_paged_attention_i8_workspace(const bh_kv8* kv, const bh_kv8_batch* batch, uint32_t n_heads,
                                               uint64_t* bytes) {
    static const char* who = "bh_paged_attention_i8_workspace";
    Kv8 k;
    Kv8Rows r;
    if (!bytes) return fail(BH_ERR_INVALID, "%s: null result", who);
    const int rc = check_call(who, kv, batch, n_heads, BH_OUT_F32, (uint64_t)-1, &k, &r);
    if (rc) return rc;
    uint64_t need = 0;
    for (const int dtype : {BH_OUT_F32, BH_OUT_BF16}) {
        const Plan pl = plan_attention(k, r, batch, n_heads, dtype);
        need = std::max(need, pl.part_floats * 4 + pl.ml_pairs * 8);
    }
    *bytes = need;
    return BH_OK;
}

extern "C" int bh_paged_attention_i8(void* stream, const void* q, uint64_t q_stride, int dtype, uint32_t n_heads,
                                     const bh_kv8* kv, const bh_kv8_batch* batch, float scale, void* out, float* lse,
                                     void* ws, uint64_t ws_bytes) {
    static const char* who = "bh_paged_attention_i8";
    AttnArgs a{};
    const int rc = check_call(who, kv, batch, n_heads, dtype, q_stride, &a.kv, &a.bt);
    if (rc) return rc;
    if (batch->rows == 0 || batch->batch == 0) return BH_OK;
    if (!q || !out) return fail(BH_ERR_INVALID, "%s: null buffer", who);
    a.q = q, a.qs = q_stride, a.out = out, a.lse = lse;
    a.nh = n_heads, a.group = n_heads / kv->n_kv_heads, a.scale2 = scale * LOG2E;
    a.by_group = Div::by(a.group), a.by_nkv = Div::by(kv->n_kv_heads);
    const Plan pl = plan_attention(a.kv, a.bt, batch, n_heads, dtype);
    const uint64_t need = pl.part_floats * 4 + pl.ml_pairs * 8;
    if (ws_bytes < need || (need && (!ws || !aligned_to(ws, 16))))
        return fail(BH_ERR_INVALID, "%s: a workspace of %llu bytes, 16-byte aligned, is needed, %llu given", who,
                    (unsigned long long)need, (unsigned long long)ws_bytes);
    a.blocks = pl.blocks, a.nsplit = pl.nsplit, a.span = pl.span;
    if (pl.nsplit) a.by_nsplit = Div::by(pl.nsplit);
    a.part = (float*)ws, a.ml = (float2*)((float*)ws + pl.part_floats);
    const size_t es = dtype == BH_OUT_F32 ? 4 : 2;
    a.ovec = aligned_to(out, 4 * es);
    const hipStream_t s = (hipStream_t)stream;
    return done(dtype == BH_OUT_F32 ? go_attention<F32>(s, a, pl) : go_attention<Bf16>(s, a, pl), who);
}

extern "C" int bh_paged_weight_sums_i8(void* stream, const void* q, uint64_t q_stride, int dtype, uint32_t n_heads,
                                       const float* lse, const bh_kv8* kv, const bh_kv8_batch* batch, float scale,
                                       float* acc, uint32_t acc_stride) {
    static const char* who = "bh_paged_weight_sums_i8";
    SumsArgs a{};
    const int rc = check_call(who, kv, batch, n_heads, dtype, q_stride, &a.kv, &a.bt);
    if (rc) return rc;
    if (acc_stride > KV_REACH) return fail(BH_ERR_INVALID, "%s: acc_stride %u", who, acc_stride);
    if (batch->rows == 0 || batch->batch == 0 || acc_stride == 0) return BH_OK;
    if (!q || !lse || !acc) return fail(BH_ERR_INVALID, "%s: null buffer", who);
    a.q = q, a.qs = q_stride, a.lse = lse, a.acc = acc, a.cap = acc_stride;
    a.nh = n_heads, a.group = n_heads / kv->n_kv_heads, a.scale2 = scale * LOG2E;
    a.by_group = Div::by(a.group), a.by_nkv = Div::by(kv->n_kv_heads);
    const hipStream_t s = (hipStream_t)stream;
    return done(dtype == BH_OUT_F32 ? go_weight_sums<F32>(s, a, batch) : go_weight_sums<Bf16>(s, a, batch), who);
}
