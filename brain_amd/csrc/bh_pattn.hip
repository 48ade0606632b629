// Attention of a ragged batch's new rows over the int8 paged KV cache, and the
// weight that each cached key receives from it.
#include "bh_kvops.h"

namespace bh {
namespace {

constexpr float LOG2E = 1.44269504088896341f, LN2 = 0.693147180559945309f;

struct AttnArgs {
    const void* q;
    uint64_t qs;  // row stride, elements
    void* out;
    float* lse;
    Kv8 kv;
    Kv8Rows bt;
    uint32_t nh, group;
    float scale2;  // scale * log2(e): softmax in base 2
};
struct SumsArgs {
    const void* q;
    uint64_t qs;
    const float* lse;
    float* acc;
    Kv8 kv;
    Kv8Rows bt;
    uint32_t nh, group, cap;
    float scale2;
};

__device__ __forceinline__ float code_f(uint32_t w, int e) { return (float)(int8_t)(uint8_t)(w >> (8 * e)); }

// Any head_dim: one wave for each row and query head. A lane takes a key for
// the score and four elements of the context for the weighted sum, 64 keys at
// a time, with a running maximum and sum.
template <class T>
__global__ __launch_bounds__(64) void paged_attention_any_kernel(AttnArgs p) {
    typedef typename T::elem E;
    __shared__ float qv[256];
    const uint32_t r = blockIdx.x / p.nh, h = blockIdx.x % p.nh, kvh = h / p.group, lane = threadIdx.x;
    const uint32_t hd = p.kv.hd;
    uint32_t b = r;
    if (p.bt.start) b = wave_last(p.bt.batch, lane, [&](uint32_t i) { return p.bt.start[i] <= r; });
    if (b >= p.bt.batch) return;
    const uint32_t e = p.bt.end(b), len = p.bt.lens[b];
    if (r >= e) return;
    const uint32_t seen = len >= e - r ? len - (e - r) + 1 : 0;  // keys that the row sees
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

// Any head_dim: a thread for each (sequence, kv head, key).
template <class T>
__global__ __launch_bounds__(64) void paged_weight_sums_any_kernel(SumsArgs p, uint32_t nchunk) {
    typedef typename T::elem E;
    const uint32_t bk = blockIdx.x / nchunk, j = (blockIdx.x % nchunk) * 64 + threadIdx.x;
    const uint32_t b = bk / p.kv.nkv, kvh = bk % p.kv.nkv, hd = p.kv.hd;
    const uint32_t len = p.bt.lens[b];
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
    *bytes = 0;
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
    const hipStream_t s = (hipStream_t)stream;
    if (dtype == BH_OUT_F32) paged_attention_any_kernel<F32><<<batch->rows * n_heads, 64, 0, s>>>(a);
    else paged_attention_any_kernel<Bf16><<<batch->rows * n_heads, 64, 0, s>>>(a);
    return done(hipGetLastError(), who);
}

extern "C" int bh_paged_weight_sums_i8(void* stream, const void* q, uint64_t q_stride, int dtype, uint32_t n_heads,
                                       const float* lse, const bh_kv8* kv, const bh_kv8_batch* batch, float scale,
                                       float* acc, uint32_t acc_stride) {
    static const char* who = "bh_paged_weight_sums_i8";
    SumsArgs a{};
    const int rc = check_call(who, kv, batch, n_heads, dtype, q_stride, &a.kv, &a.bt);
    if (rc) return rc;
    if (batch->rows == 0 || batch->batch == 0 || acc_stride == 0) return BH_OK;
    if (!q || !lse || !acc) return fail(BH_ERR_INVALID, "%s: null buffer", who);
    a.q = q, a.qs = q_stride, a.lse = lse, a.acc = acc, a.cap = acc_stride;
    a.nh = n_heads, a.group = n_heads / kv->n_kv_heads, a.scale2 = scale * LOG2E;
    const uint32_t nchunk = (acc_stride - 1) / 64 + 1;
    const uint64_t grid = (uint64_t)batch->batch * kv->n_kv_heads * nchunk;
    if (grid > 0x7fffffffull) return fail(BH_ERR_INVALID, "%s: grid too large", who);
    const hipStream_t s = (hipStream_t)stream;
    if (dtype == BH_OUT_F32) paged_weight_sums_any_kernel<F32><<<(unsigned)grid, 64, 0, s>>>(a, nchunk);
    else paged_weight_sums_any_kernel<Bf16><<<(unsigned)grid, 64, 0, s>>>(a, nchunk);
    return done(hipGetLastError(), who);
}
