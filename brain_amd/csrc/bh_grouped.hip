// Int8 products grouped by expert (bh_matmul_i8_grouped, bh_matmul_i8_grouped_glu):
//   y[p][n] = (f32(sum_k x[row(p)][k] * w[e][n][k]) * sx[row(p)]) * sw[e][n] (+ bias[e][n])
// for the places p of expert e, and silu(gate) * up of two such products.
//
// How many rows an expert has is known on the device only, so a launch has as many
// workgroups as any offsets could need, or as the chip holds, and each finds its rows itself
// (find_tile, Tiles); the ones too many end at once.
//
// Few rows are bound by the weights' way from memory, which every kernel here asks for once: 48 tokens
// through 126 of 128 experts (355 MB) 55 us, 6.5 TB/s, where a plain read of 1 GiB reaches 6.8. Many
// rows are bound by LDS and the matrix cores (1.9 POPS).
#include <cmath>
#include <type_traits>

#include "bh_kvops.h"
#include "bh_pingpong.h"
#include "bh_tilespan.h"

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

// The tiles of a launch over row tiles of TR rows and tiles_n column tiles, in an order in which neighbours
// share what they read: an expert's row tiles (8 at most) of one column tile, then the next
// columns. Each XCD has an L2 of its own, and gets an eighth of the tiles that follow each other (tile_span).
template <uint32_t TR>
struct Tiles {
    uint32_t o[5], upto;  // lane l: offsets of experts e0 + 4 l .. + 3; the tiles up to them
    uint32_t e0, tiles_n;
    TileSpan span;

    __device__ __forceinline__ void load(const GroupedArgs& a, uint32_t base) {
        const uint32_t lane = threadIdx.x & 63;
#pragma unroll
        for (int j = 0; j < 5; ++j) o[j] = min(a.offsets[min(e0 + 4 * lane + j, a.experts)], a.places);
        upto = base + lane_scan(tiles_of(0) + tiles_of(1) + tiles_of(2) + tiles_of(3));
    }
    __device__ __forceinline__ uint32_t tiles_of(int j) const { return o[j + 1] > o[j] ? (o[j + 1] - o[j] + TR - 1) / TR : 0; }
    __device__ __forceinline__ void begin(const GroupedArgs& a, uint32_t columns, uint32_t most) {
        tiles_n = columns;
        uint32_t total = 0;
        for (e0 = 0;; e0 += 256) {
            load(a, total);
            total = (uint32_t)__builtin_amdgcn_readlane((int)upto, 63);
            if (e0 + 256 >= a.experts) break;
        }
        span = tile_span(total, tiles_n, most, blockIdx.x, gridDim.x);
    }
    // The workgroup's next tile (for a whole wave); false: there is none.
    __device__ __forceinline__ bool next(const GroupedArgs& a, Tile& out, uint32_t& tn) {
        if (span.at >= span.end) return false;
        const uint32_t id = span.at, lane = threadIdx.x & 63;
        span.at += span.step;
        if (a.experts > 256) {
            uint32_t base = 0;
            for (e0 = 0;; e0 += 256) {
                load(a, base);
                base = (uint32_t)__builtin_amdgcn_readlane((int)upto, 63);
                if ((uint64_t)base * tiles_n > id || e0 + 256 >= a.experts) break;
            }
        }
        const unsigned long long m = __ballot((uint64_t)upto * tiles_n > id);
        if (!m) return false;
        const int l = __builtin_ctzll(m);
        const uint32_t t[4] = {tiles_of(0), tiles_of(1), tiles_of(2), tiles_of(3)};
        uint32_t rel = id - (upto - t[0] - t[1] - t[2] - t[3]) * tiles_n, e = e0 + 4 * lane, first = o[0], to = o[1], mine = t[0];
#pragma unroll
        for (int j = 0; j < 3; ++j)
            if (e == e0 + 4 * lane + j && rel >= t[j] * tiles_n)
                rel -= t[j] * tiles_n, ++e, first = o[j + 1], to = o[j + 2], mine = t[j + 1];
        out.e = (uint32_t)__builtin_amdgcn_readlane((int)e, l);
        first = (uint32_t)__builtin_amdgcn_readlane((int)first, l);
        to = (uint32_t)__builtin_amdgcn_readlane((int)to, l);
        rel = (uint32_t)__builtin_amdgcn_readlane((int)rel, l);
        mine = (uint32_t)__builtin_amdgcn_readlane((int)mine, l);
        // Row tiles in bands of 8, within a band the columns, within a column the band's rows.
        const uint32_t band = rel / (8 * tiles_n), in = rel - band * 8 * tiles_n;
        const uint32_t tall = max(min(mine - band * 8, 8u), 1u);
        tn = in / tall;
        out.first = first + (band * 8 + in % tall) * TR;
        out.rows = to - out.first;
        // (Else offsets of no plan, whose counts wrapped.)
        return out.e < a.experts && out.first >= first && out.first < to && tn < tiles_n;
    }
};

// v / (1 + exp(-v)) to 7 half steps: exp(-v) is 2^p, p = -v log2(e) rounded, by v_exp_f32 (1 ulp), times 1 + what p
// lost, to first order (2^-23 |p|: below 2^-16); the reciprocal is v_rcp_f32 (1 ulp). That is for |v| up
// to 87.3, where the reciprocal leaves the normal numbers; beyond 88 exp is held there (less than v 2^-126 is left of
// far negative ones).
// ROUGH, for a result of 8 bits: without that correction (p <= 126 is off by 2^-17 then).
template <bool ROUGH = false>
__device__ __forceinline__ float silu(float v) {
    constexpr float L = 1.44269502f, LO = 1.92596299e-8f, LN2 = 0.693147182f;  // log2(e) = L + LO
    if constexpr (ROUGH) return v * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-v * L));
    const float w = __builtin_amdgcn_fmed3f(v, -88.0f, 88.0f), p = -w * L;
    const float lost = fmaf(-w, LO, fmaf(-w, L, -p));
    const float x = __builtin_amdgcn_exp2f(p);
    return v * __builtin_amdgcn_rcpf(1.0f + fmaf(x, lost * LN2, x));
}

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

// ---------------------------------------------------------------- few rows
// A workgroup takes up to 16 rows of an expert and 16 columns (of gate and up both),
// straight from memory: v_mfma_i32_16x16x64_i8 with rows of x as its first operand
// and weight rows as its second. Lane l feeds 16 bytes of row l % 16 at K piece l / 16
// and gets column l % 16 of rows 4 (l / 16) .. + 3. Its waves share K, 128 bytes (a line
// of each weight row) at a time in turn, and their sums meet in LDS. What counts is how many bytes are
// on their way: a wave asks for 256 bytes of every row before it multiplies. WHOLE: K is a multiple of 64.
constexpr uint32_t GS_ROWS = 16, GS_WAVES = 8;
template <int OUT, bool GLU, bool WHOLE>
__global__ __launch_bounds__(GS_WAVES * 64) void grouped_step_kernel(GroupedArgs a, uint32_t tiles_n) {
    constexpr int C = GLU ? 2 : 1, U = 4;
    typedef int v4iu __attribute__((ext_vector_type(4), aligned(4)));
    __shared__ v4i sums[GS_WAVES][C][64];
    __shared__ uint32_t place_row[16];
    __shared__ float row_sx[16];
    const uint32_t lane = threadIdx.x & 63, r16 = lane & 15, piece = lane >> 4;
    const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)), waves = blockDim.x >> 6;
    const uint32_t kbytes = a.kg * 4, col0 = blockIdx.x % tiles_n * 16;
    Tile tile;
    if (!find_tile<GS_ROWS>(a, blockIdx.x / tiles_n, tile)) return;
    const uint32_t rows = min(tile.rows, GS_ROWS), col = min(col0 + r16, a.f - 1);
    const uint8_t* wp[C];
#pragma unroll
    for (int c = 0; c < C; ++c)
        wp[c] = reinterpret_cast<const uint8_t*>(a.wq) + ((uint64_t)tile.e * a.n + (uint64_t)c * a.f + col) * kbytes;
    const uint32_t p = tile.first + min(r16, rows - 1), x_row = a.rows ? a.rows[p] : p;
    const uint8_t* xp = reinterpret_cast<const uint8_t*>(a.xq) + (uint64_t)min(x_row, a.x_rows - 1) * kbytes;
    // Scales and bias, on their way beside the operands: a thread's results are all of column l % 16.
    float sx = 0.0f, sw[C], bias[C];
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const uint64_t n = (uint64_t)tile.e * a.n + (uint64_t)c * a.f + col;
        sw[c] = OUT != OUT_I32 ? a.sw[n] : 0.0f;
        bias[c] = OUT != OUT_I32 && a.bias ? a.bias[n] : 0.0f;
    }
    v4i acc[C];
#pragma unroll
    for (int c = 0; c < C; ++c) acc[c] = v4i{0, 0, 0, 0};
    for (uint32_t k0 = wave * 128; k0 < kbytes; k0 += waves * 128 * (U / 2)) {
        v4i w[U][C], x[U];
        auto load = [&](const uint8_t* row, int u) -> v4i {
            const uint32_t kb = k0 + (u / 2) * waves * 128 + (u % 2) * 64 + piece * 16;
            // (WHOLE: behind the row's end its last piece again, times zeros.)
            if constexpr (WHOLE) return *reinterpret_cast<const v4iu*>(row + min(kb, kbytes - 64 + piece * 16));
            else return load_piece(row, kb, kbytes);
        };
        // The weights first: where x lies is still being looked up.
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int c = 0; c < C; ++c) w[u][c] = load(wp[c], u);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int u = 0; u < U; ++u) x[u] = load(xp, u);
        if (OUT != OUT_I32 && k0 == 0) sx = a.sx[min(x_row, a.x_rows - 1)];  // (wave 0)
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const uint32_t kb = k0 + (u / 2) * waves * 128 + (u % 2) * 64;
            if (WHOLE && kb >= kbytes) x[u] = v4i{0, 0, 0, 0};
#pragma unroll
            for (int c = 0; c < C; ++c) acc[c] = __builtin_amdgcn_mfma_i32_16x16x64_i8(x[u], w[u][c], acc[c], 0, 0, 0);
        }
    }
#pragma unroll
    for (int c = 0; c < C; ++c) sums[wave][c][lane] = acc[c];
    if (OUT != OUT_I32 && kbytes == 0) sx = a.sx[min(x_row, a.x_rows - 1)];
    if (wave == 0) place_row[r16] = x_row, row_sx[r16] = sx;
    __syncthreads();
    // Thread t finishes register t / 64 of lane t % 64.
    for (uint32_t q = threadIdx.x; q < 256; q += blockDim.x) {
        const uint32_t i = q >> 6, l = q & 63, r = 4 * (l >> 4) + i;
        if (r >= rows || col0 + r16 >= a.f) continue;
        int y[C];
#pragma unroll
        for (int c = 0; c < C; ++c) {
            y[c] = 0;
            for (uint32_t w = 0; w < waves; ++w) y[c] += reinterpret_cast<const int*>(&sums[w][c][l])[i];
        }
        const bool there = place_row[r] < a.x_rows;
        const uint64_t at = (uint64_t)(tile.first + r) * a.f + col;
        if constexpr (OUT == OUT_I32) {
            reinterpret_cast<int*>(a.out)[at] = there ? y[0] : 0;
        } else {
            const float sx = row_sx[r];
            float v[C];
#pragma unroll
            for (int c = 0; c < C; ++c) {
                v[c] = dequant(y[c], sx, sw[c]);
                if (a.bias) v[c] = v[c] + bias[c];
            }
            if constexpr (GLU) v[0] = silu<OUT == OUT_BF16>(v[0]) * v[C - 1];
            store_out<OUT>(a.out, (int64_t)at, there ? v[0] : 0.0f);
        }
    }
}

// ---------------------------------------------------------------- tiles through LDS
// A workgroup takes BM rows of an expert and BN of its weight rows. K goes through LDS
// DK bytes at a time, STAGES buffers deep, copied there without registers
// (global_load_lds_dwordx4) where rows are 16-byte aligned and K is a multiple of DK, else (REG) loaded
// word-aligned into registers and stored, zeros behind K. 16-byte piece c of row r lies at place
// c ^ swizzle(r) of the row, so that the 16 lanes that LDS serves at a time, 16
// rows of one piece, find 16 different places of its 256-byte lines.
//   v_mfma_i32_32x32x32_i8 takes rows of x as its first operand: lane l gets column l % 32 and rows 8 (v / 4)
// + 4 (l / 32) + v % 4 in register v. Which weight row a column stands for is chosen so (`weight_row`) that a lane
// has the gate and the up product of the same column, and, with enough fragments, of two neighbouring
// columns: results leave as whole lines straight from the registers (through LDS, turned around, that
// took 65 us of 8192 tokens' 319, this way 27 of 292).
//   A workgroup stays for the next tile: its rows are looked up beside the products, and its first stages are
// asked for before the results of the tile before leave (4096 tokens, 128 experts: 187 us a workgroup a tile, 174 so). The
// first wait for a stage waits for those stores too: loads and stores are counted as one, in order, and the stores came later.
//   The group's last tile has fewer than BM rows: waves leave out the 32-row
// fragments that hold none.
template <int BM_, int BN_, int WM_, int WN_, int STAGES_, int DK_, int WGS_, bool PP_, bool ONCE_>
struct TileCfg {
    static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_, STAGES = STAGES_, DK = DK_;
    static constexpr bool PP = PP_;
    static constexpr bool ONCE = ONCE_;  // weights are read with the non-temporal hint
    static constexpr int WGS = WGS_;  // workgroups of a compute unit
    static constexpr int NT = WM * WN * 64, WTM = BM / WM, WTN = BN / WN, FM = WTM / 32, FN = WTN / 32;
    static constexpr int CPR = DK / 16, A_BYTES = BM * DK, B_BYTES = BN * DK, STAGE = A_BYTES + B_BYTES;
    static constexpr int A_LOADS = A_BYTES / 16 / NT, B_LOADS = B_BYTES / 16 / NT, LOADS = A_LOADS + B_LOADS;
    static constexpr int KSTEPS = DK / 32;
    static_assert(A_LOADS * 16 * NT == A_BYTES && B_LOADS * 16 * NT == B_BYTES, "whole loads");
    static_assert(KSTEPS % 2 == 0, "fragments alternate between two sets");
    static_assert(FN % 2 == 0 && (FN == 2 || FN % 4 == 0), "gate and up side by side, or pairs of them");
    static_assert(BM <= NT && BN <= NT, "a thread fetches a row's and a column's epilogue operands");
};

template <int DK>
__device__ __forceinline__ int lds_place(int r, int c) {
    return r * DK + ((c ^ (DK == 64 ? (r >> 2) & 3 : (r >> 1) & 7)) << 4);
}

// Waits until at most N of the wave's vector memory operations are outstanding.
template <int N>
__device__ __forceinline__ void wait_loads() {
    static_assert(N >= 0 && N < 64, "a 6-bit count");
    __builtin_amdgcn_s_waitcnt((N & 0xF) | (0x7 << 4) | (0xF << 8) | ((N >> 4) << 14));
}
// ... until at most `ahead` stages of N loads are, ahead <= MOST.
template <int N, int MOST>
__device__ __forceinline__ void wait_stages(int ahead) {
    if constexpr (MOST > 0) {
        if (ahead >= MOST) return wait_loads<MOST * N>();
        wait_stages<N, MOST - 1>(ahead);
    } else {
        wait_loads<0>();
    }
}
__device__ __forceinline__ void wait_lds() { __builtin_amdgcn_s_waitcnt(0xC07F); }
__device__ __forceinline__ void barrier_here() {
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
}

template <class C, int OUT, bool GLU, bool BIAS, bool REG>
__global__ __launch_bounds__(C::NT, C::WGS * C::NT / 256 > 1 ? C::WGS * C::NT / 256 : 1) void grouped_tile_kernel(GroupedArgs a, uint32_t tiles_n, uint32_t most) {
#if defined(__HIP_DEVICE_COMPILE__)
    constexpr int BNF = GLU ? C::BN / 2 : C::BN;  // output columns of a tile
    constexpr int DK = C::DK, JS = GLU ? 2 : 1;   // fragments of an output column
    constexpr int P = C::FN >= 2 * JS ? 2 : 1;    // neighbouring output columns of a lane
    constexpr int WCOLS = C::WTN / JS;
    __shared__ __attribute__((aligned(1024))) uint8_t lds[C::STAGES * C::STAGE];
    __shared__ float ep_sw[C::BN], ep_bias[BIAS ? C::BN : 1];
    __shared__ __attribute__((aligned(16))) float ep_sx[C::BM];
    __shared__ int ep_there[C::BM];

    const uint32_t kbytes = a.kg * 4;
    const int nk = (int)((kbytes + DK - 1) / DK);
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int wm = wave / C::WN, wn = wave % C::WN;

    Tiles<C::BM> tiles;
    Tile tile;
    uint32_t tn;
    tiles.begin(a, tiles_n, most);
    if (!tiles.next(a, tile, tn)) return;

    // Weight row, of the expert's, of tile row r. Lane c of a wave's fragments holds P neighbouring output
    // columns: fragment b * P * JS + p * JS + s is of columns P (32 b + c) + p, of the gate (s = 0) or
    // the up projection (1).
    auto weight_row = [&](int r) -> uint32_t {
        const int frag = r >> 5, s = frag % JS, p = frag / JS % P, b = frag / (JS * P);
        return (uint32_t)s * a.f + min(tn * BNF + P * (32 * b + (r & 31)) + p, a.f - 1);
    };
    // Row of x of tile row r.
    auto x_row = [&](int r) -> uint32_t {
        const uint32_t p = tile.first + min((uint32_t)r, tile.rows - 1);
        return a.rows ? a.rows[p] : p;
    };

    // Piece q = t + NT i of a stage: where it comes from. REG: its row and the piece's place in
    // a stage; else the two in one 32-bit offset (launch_grouped), the stage's part is in a scalar.
    using Src = std::conditional_t<REG, const uint8_t*, uint32_t>;
    const uint8_t* xbase = reinterpret_cast<const uint8_t*>(a.xq);
    const uint8_t* wbase;
    Src asrc[C::A_LOADS], bsrc[C::B_LOADS];
    uint32_t arow[C::A_LOADS + 1];  // rows of x of the next tile: of the thread's pieces, and of row t
    float r_sw = 0.0f, r_bias = 0.0f, r_sx = 0.0f;
    bool r_there = true;
    auto piece_of = [&](int i) -> uint32_t {
        const int q = t + C::NT * i, r = q / C::CPR;
        return (uint32_t)(lds_place<DK>(r, q % C::CPR) - r * DK);
    };
    auto fetch_rows = [&]() {
#pragma unroll
        for (int i = 0; i < C::A_LOADS; ++i) arow[i] = x_row((t + C::NT * i) / C::CPR);
        arow[C::A_LOADS] = x_row(min(t, C::BM - 1));
    };
    // Sources of the tile, and its scales and bias on their way.
    auto aim = [&]() {
        wbase = reinterpret_cast<const uint8_t*>(a.wq) + (uint64_t)tile.e * a.n * kbytes;
#pragma unroll
        for (int i = 0; i < C::A_LOADS; ++i) {
            const uint32_t row = min(arow[i], a.x_rows - 1);
            if constexpr (REG) asrc[i] = xbase + (uint64_t)row * kbytes;
            else asrc[i] = row * kbytes + piece_of(i);
        }
#pragma unroll
        for (int i = 0; i < C::B_LOADS; ++i) {
            const uint32_t row = weight_row((t + C::NT * i) / C::CPR);
            if constexpr (REG) bsrc[i] = wbase + (uint64_t)row * kbytes;
            else bsrc[i] = row * kbytes + piece_of(i);
        }
        r_there = arow[C::A_LOADS] < a.x_rows;
        if constexpr (OUT != OUT_I32) {
            if (t < C::BN) {
                const uint64_t w = (uint64_t)tile.e * a.n + weight_row(t);
                r_sw = a.sw[w];
                if constexpr (BIAS) r_bias = a.bias[w];
            }
            r_sx = a.sx[r_there ? arow[C::A_LOADS] : 0];
        }
    };

    // The copies go around the compiler's own accounting: only the waits below order them.
    const uint32_t lds_base = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)lds + wave * 64 * 16;
    auto copy = [&](auto once, const uint8_t* base, Src off, uint32_t to) {
        if constexpr (!REG && decltype(once)::value)
            asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1 nt"
                         :
                         : "v"(off), "s"(base), "s"(to)
                         : "memory", "m0");
        else if constexpr (!REG)
            asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1"
                         :
                         : "v"(off), "s"(base), "s"(to)
                         : "memory", "m0");
    };
    // Copy i of a stage: the rows of x first, then the weights.
    auto issue_one = [&](int kt, int buf, int i) {
        const uint32_t to = lds_base + buf * C::STAGE;
        const uint64_t k = (uint64_t)kt * DK;
        if (i < C::A_LOADS) copy(std::false_type{}, xbase + k, asrc[i < C::A_LOADS ? i : 0], to + i * C::NT * 16);
        else copy(std::bool_constant<C::ONCE>{}, wbase + k, bsrc[i < C::A_LOADS ? 0 : i - C::A_LOADS], to + C::A_BYTES + (i - C::A_LOADS) * C::NT * 16);
    };
    auto issue = [&](int kt, int buf) {
#pragma unroll
        for (int i = 0; i < C::LOADS; ++i) issue_one(kt, buf, i);
    };

    v16i acc[C::FM][C::FN];
    const int frow = lane & 31, fpiece = lane >> 5;
    // L: how many of the wave's row fragments hold rows.
    auto read_frags = [&](auto live, const uint8_t* A, int ks, v4i* fa, v4i* fb) {
        constexpr int L = decltype(live)::value;
#pragma unroll
        for (int i = 0; i < L; ++i)
            fa[i] = *reinterpret_cast<const v4i*>(A + lds_place<DK>(wm * C::WTM + i * 32 + frow, 2 * ks + fpiece));
#pragma unroll
        for (int j = 0; j < (L ? C::FN : 0); ++j)
            fb[j] = *reinterpret_cast<const v4i*>(A + C::A_BYTES + lds_place<DK>(wn * C::WTN + j * 32 + frow, 2 * ks + fpiece));
    };
    // Products q0 .. q1 - 1 of a k step.
    auto multiply = [&](auto live, const v4i* fa, const v4i* fb, int q0, int q1) {
        constexpr int L = decltype(live)::value;
#pragma unroll
        for (int q = 0; q < L * C::FN; ++q)
            if (q >= q0 && q < q1)
                acc[q / C::FN][q % C::FN] =
                    __builtin_amdgcn_mfma_i32_32x32x32_i8(fa[q / C::FN], fb[q % C::FN], acc[q / C::FN][q % C::FN], 0, 0, 0);
    };

    auto loop = [&](auto live) {
        constexpr int L = decltype(live)::value;
        if constexpr (REG) {
            // Two buffers: the next stage is loaded into registers while this one is multiplied.
            v4i ra[C::A_LOADS], rb[C::B_LOADS];
            auto load = [&](int kt) {
#pragma unroll
                for (int i = 0; i < C::A_LOADS; ++i) ra[i] = load_piece(asrc[i], (uint32_t)kt * DK + piece_of(i), kbytes);
#pragma unroll
                for (int i = 0; i < C::B_LOADS; ++i) rb[i] = load_piece(bsrc[i], (uint32_t)kt * DK + piece_of(i), kbytes);
            };
            auto store = [&](int buf) {
                uint8_t* base = lds + buf * C::STAGE + t * 16;
#pragma unroll
                for (int i = 0; i < C::A_LOADS; ++i) *reinterpret_cast<v4i*>(base + i * C::NT * 16) = ra[i];
#pragma unroll
                for (int i = 0; i < C::B_LOADS; ++i) *reinterpret_cast<v4i*>(base + C::A_BYTES + i * C::NT * 16) = rb[i];
            };
            if (nk > 0) {
                load(0);
                store(0);
            }
            __syncthreads();
            for (int it = 0; it < nk; ++it) {
                if (it + 1 < nk) load(it + 1);
                const uint8_t* A = lds + (it & 1) * C::STAGE;
#pragma unroll
                for (int ks = 0; ks < C::KSTEPS; ++ks) {
                    v4i fa[C::FM], fb[C::FN];
                    read_frags(live, A, ks, fa, fb);
                    multiply(live, fa, fb, 0, L * C::FN);
                }
                if (it + 1 < nk) store((it + 1) & 1);
                __syncthreads();
            }
        } else if constexpr (C::PP) {
            // Two groups of four waves a phase apart, in the order of ping_pong.
            static_assert(C::WM * C::WN == 8 && C::STAGES == 4, "two groups of four waves, four stages");
            const int group = __builtin_amdgcn_readfirstlane(wave) >> 2;
            v4i pa[C::KSTEPS][C::FM], pb[C::KSTEPS][C::FN];
            ping_pong<C::STAGES>(
                group, nk, [&](auto most, int ahead) { wait_stages<C::LOADS, decltype(most)::value>(ahead); }, [&]() { barrier_here(); },
                [&](int it) {
                    const uint8_t* A = lds + (it % C::STAGES) * C::STAGE;
#pragma unroll
                    for (int ks = 0; ks < C::KSTEPS; ++ks) read_frags(live, A, ks, pa[ks], pb[ks]);
                    const int next = it + C::STAGES - 1;
                    if (next < nk) issue(next, next % C::STAGES);
                    wait_lds();
                },
                [&]() {
#pragma unroll
                    for (int ks = 0; ks < C::KSTEPS; ++ks) multiply(live, pa[ks], pb[ks], 0, L * C::FN);
                    __builtin_amdgcn_sched_barrier(0);
                });
        } else {
            // The fragments of a k step are read while the step before is multiplied, those
            // of a stage's first step at the end of the stage before: stages it and
            // it + 1 have landed at the top of iteration it.
            static_assert(C::STAGES >= 3, "a stage is read one iteration early");
            v4i fa[2][C::FM], fb[2][C::FN];
            wait_stages<C::LOADS, C::STAGES - 2>(min(nk - 1, C::STAGES - 2));
            barrier_here();
            read_frags(live, lds, 0, fa[0], fb[0]);
            for (int it = 0; it < nk; ++it) {
                wait_stages<C::LOADS, C::STAGES - 3>(min(nk - 2 - it, C::STAGES - 3));
                wait_lds();
                barrier_here();
                const bool more = it + C::STAGES - 1 < nk;
                const int to = (it + C::STAGES - 1) % C::STAGES;
                const uint8_t* A = lds + (it % C::STAGES) * C::STAGE;
                const uint8_t* next = lds + ((it + 1) % C::STAGES) * C::STAGE;
#pragma unroll
                for (int ks = 0; ks < C::KSTEPS; ++ks) {
                    __builtin_amdgcn_sched_barrier(0);
                    // (Behind the last stage lies an older one, whose fragments are not used.)
                    const bool last = ks + 1 == C::KSTEPS;
                    read_frags(live, last ? next : A, last ? 0 : ks + 1, fa[(ks + 1) & 1], fb[(ks + 1) & 1]);
                    // A product, a read, a product, a read, ... then the stage's copies
                    // among the products that are left.
                    constexpr int READS = L ? L + C::FN : 0, PRODUCTS = L * C::FN, LEFT = PRODUCTS > READS ? PRODUCTS - READS : 0;
                    constexpr int D0 = (C::LOADS + C::KSTEPS - 1) / C::KSTEPS;
                    multiply(live, fa[ks & 1], fb[ks & 1], 0, PRODUCTS - LEFT);
                    if constexpr (LEFT > 0) {
#pragma unroll
                        for (int q = 0; q < READS; ++q) {
                            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
                        }
                    }
#pragma unroll
                    for (int d = 0; d < D0; ++d) {
                        __builtin_amdgcn_sched_barrier(0);
                        if (ks * D0 + d < C::LOADS && more) issue_one(it + C::STAGES - 1, to, ks * D0 + d);
                        __builtin_amdgcn_sched_barrier(0);
                        multiply(live, fa[ks & 1], fb[ks & 1], PRODUCTS - LEFT + LEFT * d / D0,
                                 PRODUCTS - LEFT + LEFT * (d + 1) / D0);
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
        }
    };

    auto first_stages = [&]() {
        if constexpr (!REG) {
#pragma unroll
            for (int s = 0; s < C::STAGES - 1; ++s)
                if (s < nk) issue(s, s);
        }
    };

    // Results: in register v lane l has row 8 (v / 4) + 4 (l / 32) + v % 4 of fragment row i, so a store of the P
    // columns writes two rows' 32 P neighbouring elements.
    typedef std::conditional_t<OUT == OUT_BF16, uint16_t, uint32_t> Elem;
    typedef Elem Elems __attribute__((ext_vector_type(P)));
    const int half = 4 * (lane >> 5);
    // Fragment row i of columns `col` .. (fragments j ..) to the rows from `out` on. FAST: as whole
    // vectors, every place has a row of x. FULL: all 32 rows are there.
    auto finish_block = [&](auto fast, auto full, int i, int j, uint32_t col, const float* sw, const float* bias, Elem* out,
                            int rows) {
        constexpr bool FAST = decltype(fast)::value, FULL = decltype(full)::value;
        const uint32_t lane_at = half * a.f + col;  // in elements, from a row that the wave shares
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const float4 sx4 = *reinterpret_cast<const float4*>(ep_sx + wm * C::WTM + i * 32 + 8 * g + half);
            const float sx[4] = {sx4.x, sx4.y, sx4.z, sx4.w};
#pragma unroll
            for (int v = 0; v < 4; ++v) {
                const int row = 8 * g + v;
                Elems e;
                float f[P];
#pragma unroll
                for (int p = 0; p < P; ++p) {
                    const int y = acc[i][j + p * JS][4 * g + v];
                    if constexpr (OUT == OUT_I32) {
                        e[p] = (uint32_t)y;
                    } else {
                        f[p] = dequant(y, sx[v], sw[p * JS]);
                        if constexpr (BIAS) f[p] = f[p] + bias[p * JS];
                        if constexpr (GLU) {
                            float u = dequant(acc[i][j + p * JS + JS - 1][4 * g + v], sx[v], sw[p * JS + JS - 1]);
                            if constexpr (BIAS) u = u + bias[p * JS + JS - 1];
                            f[p] = silu<OUT == OUT_BF16>(f[p]) * u;
                        }
                        if constexpr (OUT == OUT_F32) e[p] = __builtin_bit_cast(uint32_t, f[p]);
                    }
                }
                if constexpr (OUT == OUT_BF16) {
                    if constexpr (P == 2) e = __builtin_bit_cast(Elems, pack_bf16x2(f[0], f[P - 1]));
                    else e[0] = f32_to_bf16_rne(f[0]);
                }
                Elem* at = out + (uint64_t)row * a.f + lane_at;
                if constexpr (FAST) {
                    if (FULL || row + half < rows) *reinterpret_cast<Elems*>(at) = e;
                } else if (row + half < rows) {
                    const bool is = ep_there[wm * C::WTM + i * 32 + row + half];
#pragma unroll
                    for (int p = 0; p < P; ++p)
                        if (col + p < a.f) at[p] = is ? e[p] : (Elem)0;
                }
            }
        }
    };
    auto finish = [&](const Tile& tile, uint32_t tn, int live) {
        const int rows = (int)min(tile.rows, (uint32_t)C::BM) - wm * C::WTM;  // of the wave
        bool there = true;
#pragma unroll
        for (int r = 0; r < C::WTM; r += 64) there &= ep_there[wm * C::WTM + min(r + lane, C::WTM - 1)] != 0;
        const bool fast = __all(there) && (P == 1 || (a.f % P == 0 && (reinterpret_cast<uintptr_t>(a.out) & (P * sizeof(Elem) - 1)) == 0));
#pragma unroll
        for (int b = 0; b < C::FN / (JS * P); ++b) {
            const int j = b * P * JS;
            const uint32_t col = tn * BNF + wn * WCOLS + P * (32 * b + (lane & 31));
            if (col >= a.f) continue;
            float sw[P * JS], bias[P * JS];
#pragma unroll
            for (int q = 0; q < P * JS; ++q) {
                sw[q] = ep_sw[wn * C::WTN + (j + q) * 32 + (lane & 31)];
                bias[q] = BIAS ? ep_bias[wn * C::WTN + (j + q) * 32 + (lane & 31)] : 0.0f;
            }
#pragma unroll
            for (int i = 0; i < C::FM; ++i) {
                if (i >= live) break;
                Elem* out = static_cast<Elem*>(a.out) + ((uint64_t)tile.first + wm * C::WTM + i * 32) * a.f;
                const std::true_type yes;
                const std::false_type no;
                if (!fast) finish_block(no, no, i, j, col, sw, bias, out, rows - i * 32);
                else if (rows >= i * 32 + 32) finish_block(yes, yes, i, j, col, sw, bias, out, 32);
                else finish_block(yes, no, i, j, col, sw, bias, out, rows - i * 32);
            }
        }
    };

    fetch_rows();
    aim();
    first_stages();
    for (;;) {
        const Tile now = tile;
        const uint32_t now_n = tn;
        const int rows = (int)min(now.rows, (uint32_t)C::BM);
        const int live = __builtin_amdgcn_readfirstlane(min(max((rows - wm * C::WTM + 31) / 32, 0), C::FM));
        // The next tile's rows are looked up beside this one's products.
        const bool more = tiles.next(a, tile, tn);
        if constexpr (!REG) {
            if (more) fetch_rows();
        }
#pragma unroll
        for (int i = 0; i < C::FM; ++i)
#pragma unroll
            for (int j = 0; j < C::FN; ++j)
#pragma unroll
                for (int v = 0; v < 16; ++v) acc[i][j][v] = 0;
        if (nk > 0) {
            if constexpr (C::FM == 4) {
                if (live == 4) loop(std::integral_constant<int, 4>{});
                else if (live == 3) loop(std::integral_constant<int, 3>{});
                else if (live == 2) loop(std::integral_constant<int, 2>{});
                else if (live == 1) loop(std::integral_constant<int, 1>{});
                else loop(std::integral_constant<int, 0>{});
            } else if constexpr (C::FM == 2) {
                if (live == 2) loop(std::integral_constant<int, 2>{});
                else if (live == 1) loop(std::integral_constant<int, 1>{});
                else loop(std::integral_constant<int, 0>{});
            } else {
                static_assert(C::FM == 1, "row fragments of a wave");
                if (live) loop(std::integral_constant<int, 1>{});
                else loop(std::integral_constant<int, 0>{});
            }
        }
        // (Every wave has left the results before behind: the loop's barriers, or the one below, came after.)
        if (nk == 0) __syncthreads();
        if (t < C::BN) {
            ep_sw[t] = r_sw;
            if constexpr (BIAS) ep_bias[t] = r_bias;
        }
        if (t < C::BM) {
            ep_sx[t] = r_sx;
            ep_there[t] = r_there;
        }
        __builtin_amdgcn_s_waitcnt(0);  // every copy and fragment read has ended, in every wave
        barrier_here();
        // The next tile's first stages are on their way while this one's results leave.
        if (more) {
            if constexpr (REG) fetch_rows();
            aim();
            first_stages();
        }
        finish(now, now_n, live);
        if (!more) break;
        if constexpr (REG) __syncthreads();
    }
#endif
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

constexpr unsigned CUS = 256;  // compute units of the MI355X

// The most tiles of TR rows that `places` rows in up to `experts` groups without common places can be. No call takes
// more: where offsets give places to several groups, tiles behind them are left out.
static uint64_t most_tiles(uint64_t places, uint64_t experts, uint64_t tr) {
    return std::min(places, (places + std::min(experts, places) * (tr - 1)) / tr);
}

template <class C, int OUT, bool GLU, bool REG>
static hipError_t launch_tiles(hipStream_t s, const GroupedArgs& a) {
    constexpr uint32_t cols = GLU ? C::BN / 2 : C::BN;
    constexpr bool scaled = OUT != OUT_I32;
    const uint32_t tiles_n = (a.f + cols - 1) / cols;
    const uint64_t tiles = most_tiles(a.places, a.experts, C::BM) * tiles_n;
    if (tiles > 0x7fffffffu) return hipErrorInvalidConfiguration;
    const unsigned wgs = (unsigned)std::min<uint64_t>((tiles + 7) / 8 * 8, CUS * C::WGS);
    if (scaled && a.bias) grouped_tile_kernel<C, OUT, GLU, scaled, REG><<<wgs, C::NT, 0, s>>>(a, tiles_n, (uint32_t)tiles);
    else grouped_tile_kernel<C, OUT, GLU, false, REG><<<wgs, C::NT, 0, s>>>(a, tiles_n, (uint32_t)tiles);
    return hipGetLastError();
}

template <int OUT, bool GLU>
static hipError_t launch_grouped(hipStream_t s, const GroupedArgs& a) {
    if (a.x_rows == 0) {
        grouped_zero_kernel<OUT><<<a.experts, 256, 0, s>>>(a);
        return hipGetLastError();
    }
    // Copies to LDS: whole stages, aligned rows, 32-bit offsets.
    const uint64_t row = (uint64_t)a.kg * 4, per = a.places / a.experts;
    const bool copies = row % 128 == 0 && aligned_to(a.xq, 16) && aligned_to(a.wq, 16) &&
                        std::max(a.x_rows, a.n) * row < (1ull << 32) && a.f < (1u << 29);
    // How many tiles of 64 and of 128 rows there may be, for the compute units.
    constexpr uint32_t cols = GLU ? 64 : 128;
    const uint64_t wide = (a.f + cols - 1) / cols;
    const uint64_t t64 = most_tiles(a.places, a.experts, 64) * wide, t128 = most_tiles(a.places, a.experts, 128) * wide;
    // Which kernel, by the rows an expert has on average and by how many tiles there are, if every place is of a group: the
    // host knows the room only, so a rank's share of a plan is treated as all of it. Both sides of each line, of whole plans, in
    // us, weights from memory (several sets in turn), bf16 out; "128 experts": 8 of 128 a token, gate and up 2048 x
    // (2 x 768), down 768 x 2048; "8 experts": 2 of 8, 2048 x (2 x 4096), 4096 x 2048; "64 experts": 6 of 64,
    // 2048 x (2 x 1408), 1408 x 2048.
    if (copies && !(per < 8 && t64 <= 128)) {
        if (per < 56 || t64 <= CUS) {
            // 64 rows, weights once and around the caches (per 48, 64 experts: 79.5 and 43.7, of 128 rows 87.2 and 53.9;
            // per 64, 128 experts: 104.7 and 60.2, 100.7 and 59.3). 128-byte stages, whole lines, so that the hint helps: 128 tokens,
            // 128 experts, 62 with it and 72 without; with 64-byte stages, which fetch a line twice, 91 and 76.
            // A tile a unit: six stages deep instead of two workgroups of three (64 tokens, 8 experts, down: 19.0 and 29.7).
            if (t64 <= CUS) return launch_tiles<TileCfg<64, 128, 2, 2, 6, 128, 1, false, true>, OUT, GLU, false>(s, a);
            // Two workgroups of a unit with tiles of 128 columns, or three of one wave each with half of them: what
            // leaves less idle in the last round, where as many experts have rows as even chances give (8 tokens, 128
            // experts: 36.0 and 28.4; 16 tokens, 8 experts: 24.5 and 27.6). Short K has too little for so small a tile (256 experts of 512
            // x 1024, 48 tokens: 21.6 and 24.1).
            const double e = a.experts, busy = e * (1.0 - std::pow(1.0 - 1.0 / e, (double)a.places));
            const double w2 = 2 * CUS * std::ceil(busy * wide / (2 * CUS)), w3 = 1.5 * CUS * std::ceil(2 * busy * wide / (3 * CUS));
            if (per < 12 && row >= 1024 && w3 <= w2) return launch_tiles<TileCfg<32, 64, 1, 1, 4, 128, 3, false, true>, OUT, GLU, false>(s, a);
            return launch_tiles<TileCfg<64, 128, 2, 2, 3, 128, 2, false, true>, OUT, GLU, false>(s, a);
        }
        if (per < 192) {
            // 512 tokens, 8 experts, down: 27.0 four wide stages deep, 33.1 two workgroups of four narrow ones.
            if (t128 <= CUS) return launch_tiles<TileCfg<128, 128, 2, 2, 4, 128, 1, false, false>, OUT, GLU, false>(s, a);
            return launch_tiles<TileCfg<128, 128, 2, 2, 4, 64, 2, false, false>, OUT, GLU, false>(s, a);
        }
        // Per 128, 128 experts: 122 with 128 rows, 126 with 256; per 256: 182 and 155. 8192 tokens, 8 experts: 291 (1.9
        // POPS; a dense product of that size, bh_matmul_i8_dyn, takes 342), 254 without the results' way out, 183 the copies alone,
        // 205 the products alone: LDS carries 128 KB for the 1024 cycles of a stage's products.
        return launch_tiles<TileCfg<256, 256, 4, 2, 4, 64, 1, true, false>, OUT, GLU, false>(s, a);
    }
    // Other operands through registers (8 experts of 2044 x (2 x 4092), per 16: 41.0 and the step kernel 51.1; per 4: 38.8
    // and 38.1; per 64 and 256: 70.1 and 156.8 with 64 rows, 49.3 and 116.0 with 128; 7 of 500 x 332, per 292: 7.8 and 8.2).
    if (!copies && per >= 8 && a.f < (1u << 29)) {
        if (per < 48 || t64 <= CUS) return launch_tiles<TileCfg<64, 128, 2, 2, 3, 64, 2, false, false>, OUT, GLU, true>(s, a);
        return launch_tiles<TileCfg<128, 128, 2, 2, 3, 64, 2, false, false>, OUT, GLU, true>(s, a);
    }
    // Few tiles of few rows: one token, 128 experts 8.8 (deep tiles of 64 rows 10.6), down 6.9 (7.3); one token of 8 experts, down
    // 6.8 (14.8); 16 tokens 18.7 (18.0).
    const uint32_t tiles_n = (a.f + 15) / 16;
    const uint64_t wgs = most_tiles(a.places, a.experts, GS_ROWS) * tiles_n;
    if (wgs > 0x7fffffffu) return hipErrorInvalidConfiguration;
    // A wave for each 256 bytes of K, up to 8.
    const unsigned threads = 64 * (unsigned)std::min<uint64_t>(GS_WAVES, std::max<uint64_t>(1, (row + 255) / 256));
    if (row && row % 64 == 0) grouped_step_kernel<OUT, GLU, true><<<(unsigned)wgs, threads, 0, s>>>(a, tiles_n);
    else grouped_step_kernel<OUT, GLU, false><<<(unsigned)wgs, threads, 0, s>>>(a, tiles_n);
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
