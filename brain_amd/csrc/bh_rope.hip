// Queries and keys of a layer's joined projection made ready for attention in
// one pass: per-head RMSNorm, rotation of the pairs (i, i + r/2), and, for the
// form with a cache, the rotated keys and the values as int8 codes in the paged
// pool. The reference runs these as separate dispatches (rope_paged.wgsl:27-38,
// paged_kv_append_i8_clipped_batched.wgsl:46-77); the arithmetic is theirs:
//   y = x * rsqrt(mean(x^2) + eps) * w
//   (y_i, y_{i+r/2}) -> (y_i c - y_{i+r/2} s, y_{i+r/2} c + y_i s), c, s of pos * freq_i
//   scale = min(max|y|, clip) / 127 (1 where that is 0), code = clamp(rne(y / scale), +-127)
// all in f32, rounded once to the output's type; the angle is reduced to a
// fraction of a turn in f64, since an f32 product is off by 2^-24 of itself,
// half a degree at position 131072.
#include "bh_kvops.h"

namespace bh {
namespace {

struct RopeRowsArgs {
    const void *q, *k, *v;
    void *qo, *ko;
    uint64_t qs, ks, vs, qos, kos;  // row strides, elements
    const uint32_t* pos;
    const double* freq;
    const float *qw, *kw;           // norm gains; null: no norm
    const float *kclip, *vclip;     // null: none
    uint32_t rows, nh, nkv, hd, rot;
    float eps;
    Kv8 kv;
    Kv8Rows bt;
};

// (cos, sin) of the rotation of pair i at position pos.
__device__ __forceinline__ void turn(uint32_t pos, double freq, float& c, float& s) {
    const double t = (double)pos * freq * 0.15915494309189533577;  // turns
    const float f = (float)(t - rint(t));
    sincospif(2.0f * f, &s, &c);
}

// Whether row r belongs to a sequence (rows behind the last one do not), and
// its cache slot: NO_SLOT where its position is before the sequence's first or
// has no block.
__device__ __forceinline__ bool row_slot(const Kv8& kv, const Kv8Rows& bt, uint32_t r, uint32_t lane, uint32_t& slot) {
    uint32_t b = r, e, len;
    if (bt.start && bt.batch < 64) {  // one round trip: lane i has row_start[i] and sequence i's length
        const uint32_t st = min(bt.start[min(lane, bt.batch)], bt.rows), ln = bt.len(min(lane, bt.batch - 1));
        asm volatile("" ::"v"(ln));  // both on their way before the branch
        const unsigned long long m = __ballot(lane < bt.batch && st <= r);
        if (!m) return false;
        b = 63u - (uint32_t)__builtin_clzll(m);
        e = (uint32_t)__builtin_amdgcn_readlane((int)st, (int)b + 1);
        len = (uint32_t)__builtin_amdgcn_readlane((int)ln, (int)b);
    } else {
        if (bt.start) b = wave_last(bt.batch, lane, [&](uint32_t i) { return bt.start[i] <= r; });
        if (b >= bt.batch) return false;
        e = bt.end(b), len = bt.len(b);
    }
    if (r >= e) return false;
    slot = len < e - r ? NO_SLOT : kv.slot(b, len - (e - r));
    return true;
}

// Without ceilings the largest finite one, as the appends of the decoder have it.
constexpr float NO_CLIP = 3.402823466e+38f;
__device__ __forceinline__ float code_scale(float mx, float clip) {
    const float s = fminf(mx, clip) / 127.0f;
    return s == 0.0f ? 1.0f : s;
}

// Any head_dim (a multiple of 4), any rotated part: one wave for each row and
// head, lane l holds elements 4l .. 4l + 3; partners meet in LDS. Every head
// computes its row's angles again, in f64, and that bounds it: 8192 rows of 32 + 8
// heads of 128, half of each turned, bf16: 146 us, where all turned take 28 in the
// kernel below; heads of 96: 139 us for traffic of 26.
template <class T, bool APPEND>
__global__ __launch_bounds__(64) void qk_norm_rope_any_kernel(RopeRowsArgs p) {
    typedef typename T::elem E;
    __shared__ float buf[256];
    const uint32_t heads = p.nh + p.nkv * (APPEND ? 2 : 1);
    const uint32_t r = blockIdx.x / heads, h = blockIdx.x % heads, lane = threadIdx.x;
    const uint32_t kind = h < p.nh ? 0 : h < p.nh + p.nkv ? 1 : 2;
    const uint32_t hh = kind == 0 ? h : kind == 1 ? h - p.nh : h - p.nh - p.nkv;
    uint32_t slot = 0;
    if constexpr (APPEND)
        if (!row_slot(p.kv, p.bt, r, lane, slot)) return;
    const E* src = (kind == 0 ? (const E*)p.q + r * p.qs : kind == 1 ? (const E*)p.k + r * p.ks
                                                                     : (const E*)p.v + r * p.vs) + (uint64_t)hh * p.hd;
    const bool live = 4 * lane < p.hd;
    float x[4] = {0.f, 0.f, 0.f, 0.f};
    if (live)
        for (int e = 0; e < 4; ++e) x[e] = T::get(src + 4 * lane + e);
    if (kind < 2) {
        const float* w = kind == 0 ? p.qw : p.kw;
        if (w) {
            float ss = x[0] * x[0] + x[1] * x[1] + (x[2] * x[2] + x[3] * x[3]);
            ss = xor_sum<32>(ss);
            const float rs = 1.0f / sqrtf(ss / (float)p.hd + p.eps);
            if (live)
                for (int e = 0; e < 4; ++e) x[e] = x[e] * rs * w[4 * lane + e];
        }
        for (int e = 0; e < 4; ++e) buf[4 * lane + e] = x[e];
        __syncthreads();
        const uint32_t half = p.rot / 2, pos = p.pos[r];
        for (int e = 0; e < 4; ++e) {
            const uint32_t d = 4 * lane + e;
            if (d >= p.rot) continue;
            const bool lo = d < half;
            float c, s;
            turn(pos, p.freq[lo ? d : d - half], c, s);
            const float y = buf[lo ? d + half : d - half];
            x[e] = lo ? x[e] * c - y * s : x[e] * c + y * s;
        }
    }
    if (kind == 0 || !APPEND) {
        E* dst = (kind == 0 ? (E*)p.qo + r * p.qos : (E*)p.ko + r * p.kos) + (uint64_t)hh * p.hd + 4 * lane;
        if (live)
            for (int e = 0; e < 4; ++e) T::put(dst + e, x[e]);
        return;
    }
    if (slot == NO_SLOT) return;
    float mx = fmaxf(fmaxf(fabsf(x[0]), fabsf(x[1])), fmaxf(fabsf(x[2]), fabsf(x[3])));
    mx = xor_max<32>(mx);
    const uint32_t which = kind - 1;
    const float* clip = which ? p.vclip : p.kclip;
    const float scale = code_scale(mx, clip ? clip[hh] : NO_CLIP);
    if (lane == 0) p.kv.scales[which][(uint64_t)slot * p.nkv + hh] = scale;
    if (live) {
        uint32_t w = 0;
        for (int e = 0; e < 4; ++e) w |= (uint32_t)kv8_code(x[e], scale) << (8 * e);
        p.kv.pool[which][(p.kv.row(slot) + (uint64_t)hh * p.hd) / 4 + lane] = w;
    }
}

// Heads of 64, 128 or 256 turned whole: HD / 8 lanes hold a head, lane i its
// elements 4i ..+3 of both halves, so a pair meets in a lane and a wave works on
// 512 / HD heads at once. Memory traffic bounds it: a wave takes one row (or a
// `part` of its heads, where there are few rows) and computes its angles once
// for all of them; the next heads' loads are in flight while it works. 8192 rows
// of 32 + 8 heads of 128, bf16: 168 MB in 28 us, 6.0 TB/s (a part of it from the
// last-level cache; a large copy moves 4.9). With the append, 2113 rows of 16 + 8 + 8
// heads: 15.6 us for traffic of 6; seven times the waves, each with a seventh of the
// steps, take the same, so neither bounds it, and what does is not known. One row of
// 16 + 8 heads 2.8 us, the latency of its loads and the angles.
template <class T, int HD, bool APPEND>
__global__ __launch_bounds__(256) void qk_norm_rope_kernel(RopeRowsArgs p, uint32_t parts) {
    typedef typename T::elem E;
    constexpr int LPH = HD / 8, HPW = 64 / LPH, HALF = HD / 2;
    const uint32_t lane = threadIdx.x & 63, li = lane % LPH;
    const uint32_t w = __builtin_amdgcn_readfirstlane((int)(blockIdx.x * 4 + (threadIdx.x >> 6)));
    const uint32_t r = w / parts, heads = p.nh + p.nkv * (APPEND ? 2 : 1);
    if (r >= p.rows) return;
    uint32_t h = (w % parts) * HPW + lane / LPH;
    struct In {
        typename T::raw4 a, b;
        float clip;
    };
    auto load = [&](uint32_t hh, In& x) {  // a head behind the last one reads the last
        hh = min(hh, heads - 1);
        const bool is_q = hh < p.nh, is_k = !is_q && hh < p.nh + p.nkv;
        const uint32_t kvh = is_q ? 0 : hh - p.nh - (is_k ? 0 : p.nkv);
        const E* src = is_q ? (const E*)p.q + r * p.qs + (uint64_t)hh * HD
                            : (is_k ? (const E*)p.k + r * p.ks : (const E*)p.v + r * p.vs) + (uint64_t)kvh * HD;
        x.a = *reinterpret_cast<const typename T::raw4*>(src + 4 * li);
        x.b = *reinterpret_cast<const typename T::raw4*>(src + 4 * li + HALF);
        // The ceiling goes out with the row: a load at its use would wait for the
        // stores and the next row as well.
        x.clip = 0.0f;
        if constexpr (APPEND) {
            const float* c = is_q ? nullptr : is_k ? p.kclip : p.vclip;
            x.clip = *(c ? c + kvh : (const float*)p.pos);  // (without one: any word)
        }
    };
    In x;
    load(h, x);
    const uint32_t pos = p.pos[r];
    double f[(HALF + 63) / 64];  // lane l: pairs l, l + 64
#pragma unroll
    for (int i = 0; i < (HALF + 63) / 64; ++i) f[i] = p.freq[min(64 * i + lane, (uint32_t)HALF - 1)];
    float cs[4], sn[4], qw[8], kw[8];
    auto gains = [&](const float* w, float (&g)[8]) {
#pragma unroll
        for (int e = 0; e < 8; ++e) g[e] = 1.0f;
        if (w) {
#pragma unroll
            for (int e = 0; e < 4; ++e) g[e] = w[4 * li + e], g[4 + e] = w[HALF + 4 * li + e];
        }
    };
    gains(p.qw, qw);
    gains(p.kw, kw);
    uint32_t slot = 0;
    if constexpr (APPEND)
        if (!row_slot(p.kv, p.bt, r, lane, slot)) return;
    // Each angle once for the wave (its lanes for different heads need the same).
    __shared__ __attribute__((aligned(16))) float turns[4][2][HALF];
    float(&tw)[2][HALF] = turns[threadIdx.x >> 6];
#pragma unroll
    for (int i = 0; i < (HALF + 63) / 64; ++i) {
        float c, s;
        turn(pos, f[i], c, s);
        if (HALF >= 64 || lane < HALF) tw[0][64 * i + lane] = c, tw[1][64 * i + lane] = s;
    }
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int e = 0; e < 4; ++e) cs[e] = tw[0][4 * li + e], sn[e] = tw[1][4 * li + e];
    // The whole wave stays for the exchanges.
    for (; __any(h < heads); h += parts * HPW) {
        struct {
            float a[4], b[4], clip;
        } cur;
        // (Opened here and not before: that would wait for the row's arrival, and
        // for all stores before it, a round early.)
        asm volatile("" : "+v"(x.a), "+v"(x.b), "+v"(x.clip));
        T::open4(x.a, cur.a);
        T::open4(x.b, cur.b);
        cur.clip = x.clip;
        load(h + parts * HPW, x);
        const bool real = h < heads, is_q = h < p.nh, rot = h < p.nh + p.nkv;
        if (__any(rot)) {
            float ss = 0.0f;
#pragma unroll
            for (int e = 0; e < 4; ++e) ss = ss + (cur.a[e] * cur.a[e] + cur.b[e] * cur.b[e]);
            ss = xor_sum<LPH / 2>(ss);
            const float rs = rsqrtf(ss * (1.0f / HD) + p.eps);
            const bool norm = is_q ? p.qw != nullptr : p.kw != nullptr;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                float a = cur.a[e], b = cur.b[e];
                if (norm) {
                    a = a * rs * (is_q ? qw[e] : kw[e]);
                    b = b * rs * (is_q ? qw[4 + e] : kw[4 + e]);
                }
                if (rot) {
                    cur.a[e] = a * cs[e] - b * sn[e];
                    cur.b[e] = b * cs[e] + a * sn[e];
                }
            }
        }
        if (is_q || (!APPEND && real)) {
            E* dst = (is_q ? (E*)p.qo + r * p.qos + (uint64_t)h * HD : (E*)p.ko + r * p.kos + (uint64_t)(h - p.nh) * HD) + 4 * li;
            T::put4(dst, cur.a);
            T::put4(dst + HALF, cur.b);
        }
        if constexpr (APPEND) {
            if (!__any(!is_q)) continue;
            float mx = 0.0f;
#pragma unroll
            for (int e = 0; e < 4; ++e) mx = fmaxf(mx, fmaxf(fabsf(cur.a[e]), fabsf(cur.b[e])));
            mx = xor_max<LPH / 2>(mx);
            if (real && !is_q && slot != NO_SLOT) {
                const uint32_t kvh = h - p.nh - (rot ? 0 : p.nkv);
                const float scale = code_scale(mx, (rot ? p.kclip : p.vclip) ? cur.clip : NO_CLIP);
                uint32_t wa = 0, wb = 0;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    wa |= (uint32_t)kv8_code(cur.a[e], scale) << (8 * e);
                    wb |= (uint32_t)kv8_code(cur.b[e], scale) << (8 * e);
                }
                uint32_t* pool = (rot ? p.kv.pool[0] : p.kv.pool[1]) + (p.kv.row(slot) + (uint64_t)kvh * HD) / 4 + li;
                pool[0] = wa;
                pool[HALF / 4] = wb;
                if (li == 0) (rot ? p.kv.scales[0] : p.kv.scales[1])[(uint64_t)slot * p.nkv + kvh] = scale;
            }
        }
    }
}

template <class T, int HD, bool APPEND>
hipError_t go_whole(hipStream_t s, const RopeRowsArgs& a) {
    const uint32_t heads = a.nh + a.nkv * (APPEND ? 2 : 1), groups = (heads + 512 / HD - 1) / (512 / HD);
    // Waves for the whole chip first, then rows whose angles are computed once:
    // 4096 waves (512 rows of 40 heads: 5.6 us, 6.2 with 1024 waves; 4 times more
    // are no faster).
    const uint32_t parts = std::min<uint32_t>(groups, std::max<uint32_t>(1, 4096 / a.rows));
    const uint64_t waves = (uint64_t)a.rows * parts;
    qk_norm_rope_kernel<T, HD, APPEND><<<(unsigned)((waves + 3) / 4), 256, 0, s>>>(a, parts);
    return hipGetLastError();
}

template <class T, bool APPEND>
hipError_t go(hipStream_t s, const RopeRowsArgs& a) {
    const uint32_t heads = a.nh + a.nkv * (APPEND ? 2 : 1);
    const size_t es = 4 * sizeof(typename T::elem);
    const bool whole = a.rot == a.hd && aligned_to(a.q, es) && aligned_to(a.k, es) && aligned_to(a.qo, es) &&
                       (a.qs | a.ks | a.qos) % 4 == 0 &&
                       (APPEND ? aligned_to(a.v, es) && a.vs % 4 == 0 : aligned_to(a.ko, es) && a.kos % 4 == 0);
    if (whole && a.hd == 64) return go_whole<T, 64, APPEND>(s, a);
    if (whole && a.hd == 128) return go_whole<T, 128, APPEND>(s, a);
    if (whole && a.hd == 256) return go_whole<T, 256, APPEND>(s, a);
    qk_norm_rope_any_kernel<T, APPEND><<<a.rows * heads, 64, 0, s>>>(a);
    return hipGetLastError();
}

int check_rows(const char* who, const bh_qk_rows* in, bool append, RopeRowsArgs* a) {
    if (!in) return fail(BH_ERR_INVALID, "%s: no rows", who);
    if (in->dtype != BH_OUT_F32 && in->dtype != BH_OUT_BF16)
        return fail(BH_ERR_INVALID, "%s: dtype %d, expected f32 or bf16", who, in->dtype);
    if (in->head_dim == 0 || in->head_dim % 4 || in->head_dim > 256)
        return fail(BH_ERR_INVALID, "%s: head_dim %u (a multiple of 4, <= 256)", who, in->head_dim);
    if (in->rotary_dim % 2 || in->rotary_dim > in->head_dim)
        return fail(BH_ERR_INVALID, "%s: rotary_dim %u (even, <= head_dim %u)", who, in->rotary_dim, in->head_dim);
    if (in->n_heads == 0 || in->n_kv_heads == 0)
        return fail(BH_ERR_INVALID, "%s: %u query heads, %u kv heads", who, in->n_heads, in->n_kv_heads);
    const uint64_t heads = (uint64_t)in->n_heads + (append ? 2ull : 1ull) * in->n_kv_heads;
    if (heads * in->rows > 0x7fffffffull)
        return fail(BH_ERR_INVALID, "%s: %u rows of %llu heads", who, in->rows, (unsigned long long)heads);
    const uint64_t qw = (uint64_t)in->n_heads * in->head_dim, kw = (uint64_t)in->n_kv_heads * in->head_dim;
    if (in->rows > 1 && (in->q_stride < qw || in->k_stride < kw || (append && in->v_stride < kw)))
        return fail(BH_ERR_INVALID, "%s: row strides %llu, %llu, %llu are shorter than the rows", who,
                    (unsigned long long)in->q_stride, (unsigned long long)in->k_stride,
                    (unsigned long long)in->v_stride);
    if (in->rows && (!in->q || !in->k || !in->positions || (append && !in->v) || (in->rotary_dim && !in->inv_freq)))
        return fail(BH_ERR_INVALID, "%s: null buffer", who);
    a->q = in->q, a->k = in->k, a->v = in->v;
    a->qs = in->q_stride, a->ks = in->k_stride, a->vs = in->v_stride;
    a->pos = in->positions, a->freq = in->inv_freq;
    a->qw = in->q_weight, a->kw = in->k_weight;
    a->rows = in->rows, a->nh = in->n_heads, a->nkv = in->n_kv_heads, a->hd = in->head_dim, a->rot = in->rotary_dim;
    a->eps = in->eps;
    return BH_OK;
}

int done(hipError_t e, const char* who) {
    return e == hipSuccess ? BH_OK : fail(BH_ERR_HIP, "%s: %s", who, hipGetErrorString(e));
}

}  // namespace

int check_kv8(const char* who, const bh_kv8* kv, Kv8* out) {
    if (!kv) return fail(BH_ERR_INVALID, "%s: no cache", who);
    if (kv->head_dim == 0 || kv->head_dim % 4 || kv->head_dim > 256 || kv->n_kv_heads == 0 || kv->block_size == 0 ||
        kv->max_blocks == 0 || (uint64_t)kv->n_kv_heads * kv->head_dim > 0x7fffffffull)
        return fail(BH_ERR_INVALID,
                    "%s: head_dim %u (a multiple of 4, <= 256), %u kv heads, block_size %u and max_blocks %u do not fit", who,
                    kv->head_dim, kv->n_kv_heads, kv->block_size, kv->max_blocks);
    if (!kv->k_pool || !kv->v_pool || !kv->k_scales || !kv->v_scales || !kv->block_tables)
        return fail(BH_ERR_INVALID, "%s: the cache has a null buffer", who);
    const uint64_t stride = (uint64_t)kv->n_kv_heads * kv->head_dim;
    const uint64_t n = std::min(kv->pool_words / (stride / 4), kv->n_scales / kv->n_kv_heads);
    *out = Kv8{{kv->k_pool, kv->v_pool}, {kv->k_scales, kv->v_scales}, kv->block_tables, kv->max_blocks,
               kv->block_size, kv->n_kv_heads, kv->head_dim, (uint32_t)std::min<uint64_t>(n, NO_SLOT),
               Div::by(kv->block_size)};
    return BH_OK;
}

int check_kv8_batch(const char* who, const bh_kv8_batch* bt, Kv8Rows* out) {
    if (!bt) return fail(BH_ERR_INVALID, "%s: no batch", who);
    if (bt->batch > 0x3fffffffu) return fail(BH_ERR_INVALID, "%s: %u sequences", who, bt->batch);
    if (bt->batch && bt->rows && !bt->seq_lens) return fail(BH_ERR_INVALID, "%s: no sequence lengths", who);
    if (!bt->row_start && bt->rows != bt->batch)
        return fail(BH_ERR_INVALID, "%s: %u rows of %u sequences need row_start", who, bt->rows, bt->batch);
    *out = Kv8Rows{bt->row_start, bt->seq_lens, bt->batch, bt->rows};
    return BH_OK;
}

}  // namespace bh

using namespace bh;

extern "C" int bh_qk_norm_rope(void* stream, const bh_qk_rows* in, void* q_out, uint64_t q_out_stride, void* k_out,
                               uint64_t k_out_stride) {
    static const char* who = "bh_qk_norm_rope";
    RopeRowsArgs a{};
    int rc = check_rows(who, in, false, &a);
    if (rc) return rc;
    if (in->rows == 0) return BH_OK;
    if (!q_out || !k_out) return fail(BH_ERR_INVALID, "%s: null buffer", who);
    if (in->rows > 1 && (q_out_stride < (uint64_t)a.nh * a.hd || k_out_stride < (uint64_t)a.nkv * a.hd))
        return fail(BH_ERR_INVALID, "%s: output row strides %llu, %llu are shorter than the rows", who,
                    (unsigned long long)q_out_stride, (unsigned long long)k_out_stride);
    a.qo = q_out, a.qos = q_out_stride, a.ko = k_out, a.kos = k_out_stride;
    const hipStream_t s = (hipStream_t)stream;
    return done(in->dtype == BH_OUT_F32 ? go<F32, false>(s, a) : go<Bf16, false>(s, a), who);
}

extern "C" int bh_qk_norm_rope_append_i8(void* stream, const bh_qk_rows* in, const bh_kv8* kv, const bh_kv8_batch* batch,
                                         const float* k_clip, const float* v_clip, void* q_out,
                                         uint64_t q_out_stride) {
    static const char* who = "bh_qk_norm_rope_append_i8";
    RopeRowsArgs a{};
    int rc;
    if ((rc = check_rows(who, in, true, &a)) || (rc = check_kv8(who, kv, &a.kv)) ||
        (rc = check_kv8_batch(who, batch, &a.bt)))
        return rc;
    if (kv->head_dim != in->head_dim || kv->n_kv_heads != in->n_kv_heads || batch->rows != in->rows)
        return fail(BH_ERR_INVALID, "%s: rows of %u kv heads of %u (%u of them) for a cache of %u of %u and a batch of %u",
                    who, in->n_kv_heads, in->head_dim, in->rows, kv->n_kv_heads, kv->head_dim, batch->rows);
    if (in->rows == 0 || batch->batch == 0) return BH_OK;
    if (!q_out) return fail(BH_ERR_INVALID, "%s: null buffer", who);
    if (in->rows > 1 && q_out_stride < (uint64_t)a.nh * a.hd)
        return fail(BH_ERR_INVALID, "%s: output row stride %llu is shorter than the rows", who,
                    (unsigned long long)q_out_stride);
    a.qo = q_out, a.qos = q_out_stride, a.kclip = k_clip, a.vclip = v_clip;
    const hipStream_t s = (hipStream_t)stream;
    return done(in->dtype == BH_OUT_F32 ? go<F32, true>(s, a) : go<Bf16, true>(s, a), who);
}
