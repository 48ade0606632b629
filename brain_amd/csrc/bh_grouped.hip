// Int8 products grouped by expert (bh_matmul_i8_grouped, bh_matmul_i8_grouped_glu):
//   y[p][n] = (f32(sum_k x[row(p)][k] * w[e][n][k]) * sx[row(p)]) * sw[e][n] (+ bias[e][n])
// for the places p of expert e, and silu(gate) * up of two such products.
//
// How many rows an expert has is known on the device only, so a launch has as many
// workgroups as any offsets could need and each finds its rows itself (find_tile); the
// ones too many end at once.
#include "bh_kvops.h"

namespace bh {

struct GroupedArgs {
    const uint32_t* xq;
    const float* sx;
    const uint32_t *rows, *offsets, *wq;
    const float *sw, *bias;
    void* out;
    uint32_t x_rows, places, experts, kg;
    uint32_t n, f;  // weight rows of an expert, columns of an output row (n, or n / 2: GLU)
};

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

struct Tile {
    uint32_t e, first, rows;  // expert, first place, rows from there to the group's end
};

// Row tile `tile` of the groups cut into tiles of TR rows, for a whole wave: lane l
// looks at experts 4 l .. 4 l + 3, 256 experts a pass. False: there are not so many.
template <uint32_t TR>
__device__ __forceinline__ bool find_tile(const GroupedArgs& a, uint32_t tile, Tile& out) {
    const uint32_t lane = threadIdx.x & 63;
    uint32_t base = 0;
    for (uint32_t e0 = 0; e0 < a.experts; e0 += 256) {
        uint32_t o[5], t[4], sum = 0;
#pragma unroll
        for (int j = 0; j < 5; ++j) o[j] = min(a.offsets[min(e0 + 4 * lane + j, a.experts)], a.places);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            t[j] = o[j + 1] > o[j] ? (o[j + 1] - o[j] + TR - 1) / TR : 0;
            sum += t[j];
        }
        const uint32_t upto = base + lane_scan(sum);
        const unsigned long long m = __ballot(upto > tile);
        if (m) {
            const int at = __builtin_ctzll(m);
            uint32_t rel = tile - (upto - sum), e = e0 + 4 * lane, first = o[0], end = o[1];
#pragma unroll
            for (int j = 0; j < 3; ++j)
                if (e == e0 + 4 * lane + j && rel >= t[j]) rel -= t[j], ++e, first = o[j + 1], end = o[j + 2];
            out.e = (uint32_t)__builtin_amdgcn_readlane((int)e, at);
            out.first = (uint32_t)__builtin_amdgcn_readlane((int)(first + rel * TR), at);
            end = (uint32_t)__builtin_amdgcn_readlane((int)end, at);
            out.rows = end - out.first;
            return out.first < end;  // (else offsets of no plan, whose counts wrapped)
        }
        base = (uint32_t)__builtin_amdgcn_readlane((int)upto, 63);
    }
    return false;
}

__device__ __forceinline__ float silu(float v) { return v / (1.0f + expf(-v)); }

// 16 bytes of a row at byte kb, zeros from kbytes on. Rows begin at words.
__device__ __forceinline__ v4i load_piece(const uint8_t* row, uint32_t kb, uint32_t kbytes) {
    typedef int v4iu __attribute__((ext_vector_type(4), aligned(4)));
    if (kb + 16 <= kbytes) return *reinterpret_cast<const v4iu*>(row + kb);
    v4i r = {0, 0, 0, 0};
#pragma unroll
    for (uint32_t d = 0; d < 3; ++d)
        if (kb + 4 * d < kbytes) r[d] = *reinterpret_cast<const int*>(row + kb + 4 * d);
    return r;
}

// ---------------------------------------------------------------- the plain kernel
// A workgroup takes up to 64 rows of an expert and 16 columns (of gate and up both)
// a wave, straight from memory: v_mfma_i32_16x16x64_i8 with rows of x as its
// first operand and weight rows as its second. Lane l feeds 16 bytes of row l % 16 at
// K piece l / 16 and gets column l % 16 of rows 4 (l / 16) .. + 3.
constexpr uint32_t GS_ROWS = 64;
template <int OUT, bool GLU, int NF>
__device__ __forceinline__ void stream_rows(const GroupedArgs& a, const Tile& tile, uint32_t col0) {
    constexpr int C = GLU ? 2 : 1;
    const uint32_t lane = threadIdx.x & 63, r16 = lane & 15, piece = lane >> 4;
    const uint32_t kbytes = a.kg * 4, rows = min(tile.rows, GS_ROWS);
    const uint8_t *xp[NF], *wp[C];
#pragma unroll
    for (int f = 0; f < NF; ++f) {
        const uint32_t p = tile.first + min(f * 16 + r16, rows - 1);
        const uint32_t row = min(a.rows ? a.rows[p] : p, a.x_rows - 1);
        xp[f] = reinterpret_cast<const uint8_t*>(a.xq) + (uint64_t)row * kbytes;
    }
    const uint32_t col = min(col0 + r16, a.f - 1);
#pragma unroll
    for (int c = 0; c < C; ++c)
        wp[c] = reinterpret_cast<const uint8_t*>(a.wq) + ((uint64_t)tile.e * a.n + (uint64_t)c * a.f + col) * kbytes;
    v4i acc[NF][C];
#pragma unroll
    for (int f = 0; f < NF; ++f)
#pragma unroll
        for (int c = 0; c < C; ++c) acc[f][c] = v4i{0, 0, 0, 0};
    for (uint32_t k0 = 0; k0 < kbytes; k0 += 64) {
        const uint32_t kb = k0 + piece * 16;
        v4i w[C];
#pragma unroll
        for (int c = 0; c < C; ++c) w[c] = load_piece(wp[c], kb, kbytes);
#pragma unroll
        for (int f = 0; f < NF; ++f) {
            const v4i x = load_piece(xp[f], kb, kbytes);
#pragma unroll
            for (int c = 0; c < C; ++c) acc[f][c] = __builtin_amdgcn_mfma_i32_16x16x64_i8(x, w[c], acc[f][c], 0, 0, 0);
        }
    }
    if (col0 + r16 >= a.f) return;
    float sw[C] = {}, bias[C] = {};
    if constexpr (OUT != OUT_I32) {
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const uint64_t at = (uint64_t)tile.e * a.n + (uint64_t)c * a.f + col;
            sw[c] = a.sw[at];
            if (a.bias) bias[c] = a.bias[at];
        }
    }
#pragma unroll
    for (int f = 0; f < NF; ++f)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t r = f * 16 + piece * 4 + i;
            if (r >= rows) continue;
            const uint32_t p = tile.first + r, row = a.rows ? a.rows[p] : p;
            const bool there = row < a.x_rows;
            const uint64_t at = (uint64_t)p * a.f + col;
            if constexpr (OUT == OUT_I32) {
                reinterpret_cast<int*>(a.out)[at] = there ? acc[f][0][i] : 0;
            } else {
                const float sx = a.sx[there ? row : 0];
                float v = dequant(acc[f][0][i], sx, sw[0]);
                if (a.bias) v = v + bias[0];
                if constexpr (GLU) {
                    float u = dequant(acc[f][C - 1][i], sx, sw[C - 1]);
                    if (a.bias) u = u + bias[C - 1];
                    v = silu(v) * u;
                }
                store_out<OUT>(a.out, (int64_t)at, there ? v : 0.0f);
            }
        }
}

template <int OUT, bool GLU>
__global__ __launch_bounds__(256) void grouped_stream_kernel(GroupedArgs a, uint32_t tiles_n) {
    const uint32_t wave = threadIdx.x >> 6, tn = blockIdx.x % tiles_n;
    Tile tile;
    if (!find_tile<GS_ROWS>(a, blockIdx.x / tiles_n, tile)) return;
    const uint32_t col0 = (tn * 4 + wave) * 16;
    if (col0 >= a.f) return;
    if (tile.rows <= 16) stream_rows<OUT, GLU, 1>(a, tile, col0);
    else if (tile.rows <= 32) stream_rows<OUT, GLU, 2>(a, tile, col0);
    else stream_rows<OUT, GLU, 4>(a, tile, col0);
}

// Rows that no x has: a launch whose x has no rows at all writes its zeros.
template <int OUT>
__global__ __launch_bounds__(256) void grouped_zero_kernel(GroupedArgs a) {
    uint32_t e = blockIdx.x;
    const uint32_t lo = min(a.offsets[e], a.places), hi = min(a.offsets[e + 1], a.places);
    const uint64_t end = (uint64_t)hi * a.f;
    for (uint64_t i = (uint64_t)lo * a.f + threadIdx.x; i < end; i += 256) {
        if constexpr (OUT == OUT_I32) reinterpret_cast<int*>(a.out)[i] = 0;
        else store_out<OUT>(a.out, (int64_t)i, 0.0f);
    }
}

// The most tiles of TR rows that `places` rows in up to `experts` groups can be.
static uint64_t most_tiles(uint64_t places, uint64_t experts, uint64_t tr) {
    return std::min(places, (places + std::min(experts, places) * (tr - 1)) / tr);
}

template <int OUT, bool GLU>
static hipError_t launch_grouped(hipStream_t s, const GroupedArgs& a) {
    if (a.x_rows == 0) {
        grouped_zero_kernel<OUT><<<a.experts, 256, 0, s>>>(a);
        return hipGetLastError();
    }
    const uint32_t tiles_n = (a.f + 63) / 64;
    const uint64_t wgs = most_tiles(a.places, a.experts, GS_ROWS) * tiles_n;
    if (wgs > 0x7fffffffu) return hipErrorInvalidConfiguration;
    grouped_stream_kernel<OUT, GLU><<<(unsigned)wgs, 256, 0, s>>>(a, tiles_n);
    return hipGetLastError();
}

static int check_grouped(const char* who, const bh_grouped_i8* g, const void* out, int out_dtype, bool glu, GroupedArgs* a) {
    if (!g) return fail(BH_ERR_INVALID, "%s: null group", who);
    if (out_dtype != OUT_F32 && out_dtype != OUT_BF16 && (glu || out_dtype != OUT_I32))
        return fail(BH_ERR_INVALID, "%s: out_dtype %d", who, out_dtype);
    if (g->places > 0x7fffffffu || g->n_experts > 0x7fffffffu || g->x_rows > 0x7fffffffu || g->n > 0x7fffffffu ||
        (uint64_t)g->kg * 4 > 0x7fffffffu)
        return fail(BH_ERR_INVALID, "%s: %u places, %u experts, %u rows, kg=%u n=%u out of range", who, g->places,
                    g->n_experts, g->x_rows, g->kg, g->n);
    if (glu && g->n % 2) return fail(BH_ERR_INVALID, "%s: n=%u rows of gate and up", who, g->n);
    if (!g->rows && g->places > g->x_rows)
        return fail(BH_ERR_INVALID, "%s: %u places of %u rows need `rows`", who, g->places, g->x_rows);
    if (g->places == 0 || g->n_experts == 0 || g->n == 0) return BH_OK;
    const bool scaled = out_dtype != OUT_I32;
    if (!out || !g->offsets || (scaled && (!g->sw || (g->x_rows && !g->sx))) || (g->kg && (!g->wq || (g->x_rows && !g->xq))))
        return fail(BH_ERR_INVALID, "%s: null buffer", who);
    *a = GroupedArgs{g->xq,      g->sx,     g->rows,   g->offsets,   g->wq, g->sw, g->bias, const_cast<void*>(out),
                     g->x_rows,  g->places, g->n_experts, g->kg, g->n, glu ? g->n / 2 : g->n};
    return BH_OK;
}

}  // namespace bh

using namespace bh;

static int grouped_done(hipError_t e, const char* who) {
    if (e == hipErrorInvalidConfiguration) return fail(BH_ERR_INVALID, "%s: grid too large", who);
    return e == hipSuccess ? BH_OK : fail(BH_ERR_HIP, "%s: %s", who, hipGetErrorString(e));
}

extern "C" int bh_matmul_i8_grouped(void* stream, const bh_grouped_i8* g, void* out, int out_dtype) {
    static const char* who = "bh_matmul_i8_grouped";
    GroupedArgs a{};
    const int rc = check_grouped(who, g, out, out_dtype, false, &a);
    if (rc || !a.out) return rc;
    const hipStream_t s = (hipStream_t)stream;
    switch (out_dtype) {
        case OUT_F32: return grouped_done(launch_grouped<OUT_F32, false>(s, a), who);
        case OUT_BF16: return grouped_done(launch_grouped<OUT_BF16, false>(s, a), who);
        default: return grouped_done(launch_grouped<OUT_I32, false>(s, a), who);
    }
}

extern "C" int bh_matmul_i8_grouped_glu(void* stream, const bh_grouped_i8* g, void* out, int out_dtype) {
    static const char* who = "bh_matmul_i8_grouped_glu";
    GroupedArgs a{};
    const int rc = check_grouped(who, g, out, out_dtype, true, &a);
    if (rc || !a.out) return rc;
    const hipStream_t s = (hipStream_t)stream;
    return grouped_done(out_dtype == OUT_F32 ? launch_grouped<OUT_F32, true>(s, a) : launch_grouped<OUT_BF16, true>(s, a),
                        who);
}
