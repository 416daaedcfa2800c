// moe_int8.hip -- the routed experts' FFN over 8-bit integer weights with a
// scale per output channel, for tokens whose expert ids and weights are given.
// The counterpart over block-quantized weights is chimere_moe_prefill
// (cs/src/qwen35_model/moe_ffn.rs:1081-1768 per token).
//
// Bound by the selected experts' weights: each byte of them is read from
// memory once.  A few pairs of (token, expert), two launches: gate and up of
// each pair (every work-group quantizes its token), then per token h to 8 bits,
// down and the weighted sum.  More, five or six: rows of x to 8 bits and the
// pairs of each expert together, with the list of tiles (above 4096 pairs that
// takes a launch more); gate and up product with h = silu(g) u; rows of h to 8
// bits; down product; each token's weighted sum.
#include <math.h>

#include <type_traits>

#include "api_internal.h"
#include "int8_gemm.h"
#include "int8_quant.h"
#include "moe_common.h"

namespace chimere {

struct MoeI8 {
    int H, F, E, K, T;
    const int8_t *gate, *up, *down;
    const float *gate_s, *up_s, *down_s;
    const int* ids;
    const float* wts;
    const void* x;
    int64_t ldx;
    int8_t* xq;            // [T][H]
    float* xs;             // [T]
    int *order, *rank;     // sorted position -> pair; pair -> rank among 1024 pairs' of its expert
    int* total;            // {pairs, tiles}
    int* cnt;              // pairs per expert of every 1024 pairs
    int4* tiles;           // {expert, first sorted pair, pairs, 0}
    float* h;              // [pairs][F], in sorted order (few pairs: by pair)
    int8_t* hq;
    float* hs;             // by pair
    void* y;               // [pairs][H], by pair: scaled f32, or sums in 24 bits
    void* out;
    int64_t ldo;
    int tile_pairs;
};

// ------------------------------------------------------------ few pairs

constexpr int FP_WAVES = 8, FP_KEEP = 16, FP_KEEP_H = 64, FP_AHEAD = 4;   // FP_AHEAD: a wave's pieces of work whose weights are loaded ahead

// Grid (F / 16, pairs): 16 columns of F of one pair, gate and up.  Steps of 128
// columns of H dealt to the eight waves; the one token is row 0 of the matrix
// instruction (the other rows repeat it: the weights' bytes are what counts),
// sums joined in LDS.
template <typename X>
__global__ __launch_bounds__(64 * FP_WAVES) void k_i8_pair_gate_up(MoeI8 a) {
    extern __shared__ __align__(16) uint8_t lds[];   // scale, integers of the token
    __shared__ int part[FP_WAVES][2][16];
    const int p = blockIdx.y, e = a.ids[p], t = p / a.K, f0 = blockIdx.x * 16;
    if ((unsigned)e >= (unsigned)a.E) return;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int S = (a.H + I8_BK - 1) / I8_BK, last = a.H / 16 - 1, r = lane & 15, pc = lane >> 4;
    const int64_t row = ((int64_t)e * a.F + f0 + r) * a.H;   // F is a multiple of 16
    v4i w[2][2];
    auto load_w = [&](int s) {
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const int at = min(8 * s + 4 * h + pc, last) * 16;
            w[0][h] = *(const v4i*)(a.gate + row + at);
            w[1][h] = *(const v4i*)(a.up + row + at);
        }
    };
    if (wave < S) load_w(wave);
    const float sg = tid < 16 ? a.gate_s[(int64_t)e * a.F + f0 + tid] : 0.0f;
    const float su = tid < 16 ? a.up_s[(int64_t)e * a.F + f0 + tid] : 0.0f;
    float* xs = (float*)lds;
    uint8_t* xq = lds + 16;
    const X* x = (const X*)a.x + t * a.ldx;
    i8_rows_to_lds<64 * FP_WAVES, FP_KEEP>(1, S * I8_BK, 0, xs, xq,
                                           [&](int, int c, auto& v) { i8_load(x, c, a.H, v); },
                                           std::integral_constant<int, 16 / sizeof(X)>{});
    v4i g = {}, u = {};
    for (int s = wave; s < S; s += FP_WAVES) {
        v4i now[2][2];
#pragma unroll
        for (int h = 0; h < 2; h++) {
            now[0][h] = w[0][h];
            now[1][h] = w[1][h];
        }
        if (s + FP_WAVES < S) load_w(s + FP_WAVES);
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const v4i f = *(const v4i*)(xq + (8 * s + 4 * h + pc) * 16);   // 0 behind H
            g = __builtin_amdgcn_mfma_i32_16x16x64_i8(f, now[0][h], g, 0, 0, 0);
            u = __builtin_amdgcn_mfma_i32_16x16x64_i8(f, now[1][h], u, 0, 0, 0);
        }
    }
    if (lane < 16) {   // row 0, column lane
        part[wave][0][lane] = g[0];
        part[wave][1][lane] = u[0];
    }
    __syncthreads();
    if (tid < 16) {
        int gs = 0, us = 0;
#pragma unroll
        for (int i = 0; i < FP_WAVES; i++) {
            gs += part[i][0][tid];
            us += part[i][1][tid];
        }
        a.h[(int64_t)p * a.F + f0 + tid] = silu((float)gs * *xs * sg) * ((float)us * *xs * su);
    }
}

// Grid (H / COLS, T): 16 or 8 columns of H of one token.  The token's rows of h
// to 8 bits in LDS; the (k, step of 128 columns of F) pieces dealt to the eight
// waves, whose sums meet in LDS integers; the weighted sum in ascending k.
// With 8 columns a matrix instruction takes two pieces, one in rows 0 .. 7 of
// the weights and row 0 of h, one in rows 8 .. 15 and row 1: twice the
// work-groups, where 16 columns would leave half of the CUs idle (one token
// of H = 2048: 7.3 us with 16, 6.6 with 8).
template <typename T, int COLS, int KEEP>
__global__ __launch_bounds__(64 * FP_WAVES) void k_i8_pair_down(MoeI8 a) {
    constexpr int PER = 16 / COLS;                   // pieces per instruction
    extern __shared__ __align__(16) uint8_t lds[];   // integers of h
    __shared__ float hs[MAX_K], wk[MAX_K], y[MAX_K][COLS];
    __shared__ int sum[MAX_K][COLS];
    const int t = blockIdx.y, n0 = blockIdx.x * COLS;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int S = (a.F + I8_BK - 1) / I8_BK, last = a.F / 16 - 1, r = lane & 15, pc = lane >> 4;
    const int pieces = a.K * S, n = (pieces + PER - 1) / PER;
    const int* ids = a.ids + (int64_t)t * a.K;
    v4i w[FP_AHEAD][2];
    auto load_w = [&](int u, v4i(&to)[2]) {
        const int at = min(u * PER + r / COLS, pieces - 1), k = at / S, s = at - k * S, e = ids[k];
        const int8_t* row = a.down + ((int64_t)((unsigned)e < (unsigned)a.E ? e : 0) * a.H + n0 + r % COLS) * a.F;
#pragma unroll
        for (int h = 0; h < 2; h++) to[h] = *(const v4i*)(row + min(8 * s + 4 * h + pc, last) * 16);
    };
#pragma unroll
    for (int i = 0; i < FP_AHEAD; i++)
        if (wave + i * FP_WAVES < n) load_w(wave + i * FP_WAVES, w[i]);
    // thread -> (k, column): its scale and weight, ahead of all that is waited for
    const int mk = tid / COLS, mc = tid % COLS, me = mk < a.K ? ids[mk] : -1;
    const bool mine = (unsigned)me < (unsigned)a.E;
    const float sd = mine ? a.down_s[(int64_t)me * a.H + n0 + mc] : 0.0f;
    const float wt = mine ? a.wts[(int64_t)t * a.K + mk] : 0.0f;
    if (tid < MAX_K * COLS) (&sum[0][0])[tid] = 0;
    // (a pair that was left out: whatever its row holds, its sums are not used)
    const int lda = S * I8_BK;
    i8_rows_to_lds<64 * FP_WAVES, KEEP>(
        a.K, S * I8_BK, lda, hs, lds,
        [&](int k, int c, auto& v) { i8_load(a.h + ((int64_t)t * a.K + k) * a.F, c, a.F, v); },
        std::integral_constant<int, 4>{});
    auto piece = [&](int u, const v4i(&now)[2]) {
        const int mine_at = min(u * PER + (r & (PER - 1)), pieces - 1), mk_ = mine_at / S, ms = mine_at - mk_ * S;
        v4i acc = {};
#pragma unroll
        for (int h = 0; h < 2; h++)
            acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(*(const v4i*)(lds + mk_ * lda + (8 * ms + 4 * h + pc) * 16),
                                                        now[h], acc, 0, 0, 0);
        // lane r < 16 holds column r of every row; its weights' piece is row r / COLS
        const int at = u * PER + r / COLS;
        if (lane < 16 && at < pieces) atomicAdd(&sum[at / S][r % COLS], PER == 2 && r >= COLS ? acc[1] : acc[0]);
    };
#pragma unroll
    for (int i = 0; i < FP_AHEAD; i++)
        if (wave + i * FP_WAVES < n) piece(wave + i * FP_WAVES, w[i]);
    for (int u = wave + FP_AHEAD * FP_WAVES; u < n; u += FP_WAVES) {
        load_w(u, w[0]);
        piece(u, w[0]);
    }
    __syncthreads();
    if (mk < a.K) {
        y[mk][mc] = mine ? (float)sum[mk][mc] * hs[mk] * sd : 0.0f;   // a pair that was left out: 0 times 0
        if (mc == 0) wk[mk] = wt;
    }
    __syncthreads();
    if (tid < COLS) {
        float acc = 0.0f;
        for (int k = 0; k < a.K; k++) acc = __builtin_fmaf(wk[k], y[k][tid], acc);
        store_f((T*)a.out + t * a.ldo + n0 + tid, acc);
    }
}

// ------------------------------------------------------------ many pairs

// Counting sort of the pairs by expert; a pair whose id is no expert is left
// out.  Pairs of one expert come in any order: each pair's row is computed on
// its own.  A work-group takes 1024 pairs: counts per expert and each pair's
// rank among them (PLAN 0); then every work-group adds up all counts, scans
// them and places its own pairs, the first one lists the tiles (PLAN 1).  Up to
// PLAN_ONE pairs: one work-group does both (PLAN 2), a launch less.  (One
// work-group for 32768 pairs, its atomics one after another: 31 us.)
constexpr int PLAN_ONE = 4096;
template <int PLAN>
__device__ __forceinline__ void i8_plan(const MoeI8& a, int groups) {
    constexpr int AT = PLAN == 2 ? PLAN_ONE / 1024 : 1;   // pairs of a thread
    __shared__ int first[MAX_E], wsum[16], tot[2];
    const int tid = threadIdx.x, P = a.T * a.K, TP = a.tile_pairs;
    int e[AT], rank[AT];
#pragma unroll
    for (int i = 0; i < AT; i++) {
        const int p = (blockIdx.x * AT + i) * 1024 + tid, id = p < P ? a.ids[p] : -1;
        e[i] = (unsigned)id < (unsigned)a.E ? id : -1;
        rank[i] = 0;
    }
    if constexpr (PLAN != 1) {
        first[tid] = 0;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < AT; i++)
            if (e[i] >= 0) rank[i] = atomicAdd(&first[e[i]], 1);
        __syncthreads();
        if constexpr (PLAN == 0) {
            if (tid < a.E) a.cnt[blockIdx.x * a.E + tid] = first[tid];
            if (e[0] >= 0) a.rank[blockIdx.x * 1024 + tid] = rank[0];
            return;
        }
    }
    int c = 0, before = 0;
    if constexpr (PLAN == 1) {
        if (e[0] >= 0) rank[0] = a.rank[blockIdx.x * 1024 + tid];
        if (tid < a.E) {
#pragma unroll 8
            for (int g = 0; g < groups; g++) {
                const int n = a.cnt[g * a.E + tid];
                c += n;
                before += g < (int)blockIdx.x ? n : 0;
            }
        }
    } else {
        c = first[tid];
    }
    const int nt = (c + TP - 1) / TP;
    const int at = excl_scan1024(c, wsum, &tot[0]);
    __syncthreads();
    const int tile = excl_scan1024(nt, wsum, &tot[1]);
    first[tid] = at + before;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < AT; i++)
        if (e[i] >= 0) a.order[first[e[i]] + rank[i]] = (blockIdx.x * AT + i) * 1024 + tid;
    if (blockIdx.x != 0) return;
    for (int s = 0; s < nt; s++) a.tiles[tile + s] = make_int4(tid, at + s * TP, min(TP, c - s * TP), 0);
    if (tid < 2) a.total[tid] = tot[tid];
}

// The first launch: `groups` work-groups plan, the others take rows of x to 8 bits.
template <int PLAN, typename X>
__global__ __launch_bounds__(1024) void k_i8_prepare(MoeI8 a, I8Rows<X> x, int groups) {
    if ((int)blockIdx.x < groups) i8_plan<PLAN>(a, groups);
    else if (a.H <= I8_WAVE_ROW) i8_quantize_rows<X, 1, 1024>(x, blockIdx.x - groups);
    else i8_quantize_rows<X, 4, 1024>(x, blockIdx.x - groups);
}
__global__ __launch_bounds__(1024) void k_i8_plan(MoeI8 a, int groups) { i8_plan<1>(a, groups); }

// rows of h, in sorted order, to 8 bits; their scales by pair
template <int W>
__global__ __launch_bounds__(256) void k_i8_hidden(I8Rows<float> h) { i8_quantize_rows<float, W, 256>(h, blockIdx.x); }

// Gate and up of a tile: its weight rows alternate in blocks of 16 between
// gate and up, so g and u of the same (pair, column) meet in a lane.
template <typename Tile>
__device__ __forceinline__ void i8_gate_up(const MoeI8& a, const int4& t, int f0, uint8_t* lds) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint32_t aoff[Tile::PM], woff[Tile::PN];
#pragma unroll
    for (int p = 0; p < Tile::PM; p++) {
        const int r = min((wave * Tile::PM + p) * 8 + (lane >> 3), t.z - 1);
        aoff[p] = (uint32_t)(a.order[t.y + r] / a.K) * (uint32_t)a.H;
    }
#pragma unroll
    for (int p = 0; p < Tile::PN; p++) {
        const int r = (wave * Tile::PN + p) * 8 + (lane >> 3);
        woff[p] = (uint32_t)min(f0 + (r >> 5) * 16 + (r & 15), a.F - 1) * (uint32_t)a.H;
    }
    const int64_t e = t.x;
    const float xs = threadIdx.x < Tile::BM ? a.xs[a.order[t.y + min((int)threadIdx.x, t.z - 1)] / a.K] : 0.0f;
    constexpr int VEC = 4;
    const int f = f0 + Tile::template first_col<VEC, true>();
    const bool in = f < a.F;   // F is a multiple of 16: all four columns or none
    const float4 sg = in ? *(const float4*)(a.gate_s + e * a.F + f) : float4{};
    const float4 su = in ? *(const float4*)(a.up_s + e * a.F + f) : float4{};
    v16i acc[Tile::MTILES][Tile::NTILES];
    Tile::run(a.xq, a.gate + e * a.F * a.H, a.up + e * a.F * a.H, aoff, woff, a.H, lds, acc);
    Tile::template rows<VEC, true>(lds, acc, make_float2(xs, 0.0f),
                                   [&](int r, const int(&g)[VEC], const int(&u)[VEC], float2 of_row) {
        if (r >= t.z || !in) return;
        const float s = of_row.x;
        float4 h;
        h.x = silu((float)g[0] * s * sg.x) * ((float)u[0] * s * su.x);
        h.y = silu((float)g[1] * s * sg.y) * ((float)u[1] * s * su.y);
        h.z = silu((float)g[2] * s * sg.z) * ((float)u[2] * s * su.z);
        h.w = silu((float)g[3] * s * sg.w) * ((float)u[3] * s * su.w);
        *(float4*)(a.h + (int64_t)(t.y + r) * a.F + f) = h;
    });
}

// Four sums of 24 bits each.  Sums of F products are 16256 F at most, so up to
// F = 512 nothing is lost, and an f32 output is the same as from f32 rows.
struct I24x4 {
    uint32_t w[3];
    __device__ __forceinline__ void pack(const int (&x)[4]) {
        w[0] = (x[0] & 0xFFFFFF) | (uint32_t)x[1] << 24;
        w[1] = ((uint32_t)x[1] >> 8 & 0xFFFF) | (uint32_t)x[2] << 16;
        w[2] = ((uint32_t)x[2] >> 16 & 0xFF) | (uint32_t)x[3] << 8;
    }
    __device__ __forceinline__ void unpack(int (&x)[4]) const {
        x[0] = (int)(w[0] << 8) >> 8;
        x[1] = (int)(w[1] << 16 | w[0] >> 24 << 8) >> 8;
        x[2] = (int)(w[2] << 24 | w[1] >> 16 << 8) >> 8;
        x[3] = (int)w[2] >> 8;
    }
};
constexpr int MAX_F24 = ((1 << 23) - 1) / (127 * 128);

// Down of a tile.  Y = float4: the scaled products.  Y = I24x4: the integer
// sums, which the weighted sum scales (the rows of 32768 pairs of 2048 columns
// are 201 MB instead of 268, written and read again: 4096 tokens of H 2048, F
// 512, top-8 of 256 take 343 us instead of 356).  An output is rounded once
// either way, whatever its type, and does not depend on the other tokens.
template <typename Tile, typename Y>
__device__ __forceinline__ void i8_down(const MoeI8& a, const int4& t, int n0, uint8_t* lds) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint32_t aoff[Tile::PM], woff[Tile::PN];
#pragma unroll
    for (int p = 0; p < Tile::PM; p++)
        aoff[p] = (uint32_t)min((wave * Tile::PM + p) * 8 + (lane >> 3), t.z - 1) * (uint32_t)a.F;
#pragma unroll
    for (int p = 0; p < Tile::PN; p++)
        woff[p] = (uint32_t)min(n0 + (wave * Tile::PN + p) * 8 + (lane >> 3), a.H - 1) * (uint32_t)a.F;
    const int64_t e = t.x;
    const int pair = threadIdx.x < Tile::BM ? a.order[t.y + min((int)threadIdx.x, t.z - 1)] : 0;
    constexpr bool SUMS = std::is_same<Y, I24x4>::value;
    const float2 mine = make_float2(SUMS ? 0.0f : a.hs[pair], __builtin_bit_cast(float, pair));
    constexpr int VEC = 4;
    const int n = n0 + Tile::template first_col<VEC>();
    const bool in = n < a.H;   // H is a multiple of 16: all columns or none
    const float4 sd = !SUMS && in ? *(const float4*)(a.down_s + e * a.H + n) : float4{};
    v16i acc[Tile::MTILES][Tile::NTILES];
    const int8_t* w = a.down + e * a.H * a.F;
    Tile::run(a.hq + (int64_t)t.y * a.F, w, w, aoff, woff, a.F, lds, acc);
    Tile::template rows<VEC>(lds, acc, mine, [&](int r, const int(&x)[VEC], float2 of_row) {
        if (r >= t.z || !in) return;
        const float s = of_row.x;
        Y y;
        if constexpr (SUMS) y.pack(x);
        else y = make_float4((float)x[0] * s * sd.x, (float)x[1] * s * sd.y, (float)x[2] * s * sd.z, (float)x[3] * s * sd.w);
        ((Y*)a.y)[((int64_t)__builtin_bit_cast(int, of_row.y) * a.H + n) / VEC] = y;
    });
}

// Tiles of up to 64 pairs (four waves) or 128 (eight waves) against BN weight
// rows; one that holds half of its pairs or less, the last of an expert,
// takes the code for half the rows: as many copies and matrix instructions less.
// (256 x 256 tiles, one work-group per CU, pairs' rows in 16 bits: 16 experts, 2811 tokens 109 us
// against 106, 8192 tokens of 256 experts 486 against 513.)
template <int ROWS>
struct MoeTile;
template <>
struct MoeTile<64> {
    typedef I8Tile<2, 2, 1, 2, 2, 2> Whole;
    typedef I8Tile<1, 4, 1, 1, 2, 2> Half;
    static constexpr int BN = 128, WAVES = 4, LDS = 48 << 10, GROUPS = 3;   // work-groups per CU
};
template <>
struct MoeTile<128> {
    typedef I8Tile<2, 4, 2, 1, 2, 2> Whole;
    typedef I8Tile<2, 4, 1, 1, 3, 2> Half;
    static constexpr int BN = 128, WAVES = 8, LDS = 64 << 10, GROUPS = 2;
};
template <int ROWS>
constexpr bool moe_tile_fits() {
    typedef MoeTile<ROWS> M;
    typedef typename M::Whole W;
    typedef typename M::Half H;
    return W::BM == ROWS && H::BM == ROWS / 2 && W::BN == M::BN && H::BN == M::BN && W::NW == M::WAVES &&
           H::NW == M::WAVES && W::LDS <= M::LDS && H::LDS <= M::LDS && M::LDS * M::GROUPS <= 160 << 10;
}
static_assert(moe_tile_fits<64>() && moe_tile_fits<128>(), "one grid and one LDS size per kernel");

// Work-group -> (tile, column block), in contiguous eighths for the XCDs, that
// work-groups are dealt to round-robin, so that the tiles of an expert and the
// column blocks of a tile share an L2; false: none.
__device__ __forceinline__ bool i8_tile_of(const MoeI8& a, int blocks, int4& t, int& block) {
    const int n = a.total[1] * blocks, per = (n + 7) / 8, at = blockIdx.x >> 3, id = (blockIdx.x & 7) * per + at;
    if (at >= per || id >= n) return false;
    t = a.tiles[id / blocks];
    block = id % blocks;
    return true;
}

template <int ROWS>
__global__ __launch_bounds__(64 * MoeTile<ROWS>::WAVES, MoeTile<ROWS>::WAVES / 4 * MoeTile<ROWS>::GROUPS)
void k_i8_gate_up(MoeI8 a) {
    typedef MoeTile<ROWS> M;
    __shared__ __align__(16) uint8_t lds[M::LDS];
    int4 t;
    int block;
    if (!i8_tile_of(a, (a.F + M::BN / 2 - 1) / (M::BN / 2), t, block)) return;
    if (t.z <= ROWS / 2) i8_gate_up<typename M::Half>(a, t, block * (M::BN / 2), lds);
    else i8_gate_up<typename M::Whole>(a, t, block * (M::BN / 2), lds);
}

template <int ROWS, typename Y>
__global__ __launch_bounds__(64 * MoeTile<ROWS>::WAVES, MoeTile<ROWS>::WAVES / 4 * MoeTile<ROWS>::GROUPS)
void k_i8_down(MoeI8 a) {
    typedef MoeTile<ROWS> M;
    __shared__ __align__(16) uint8_t lds[M::LDS];
    int4 t;
    int block;
    if (!i8_tile_of(a, (a.H + M::BN - 1) / M::BN, t, block)) return;
    if (t.z <= ROWS / 2) i8_down<typename M::Half, Y>(a, t, block * M::BN, lds);
    else i8_down<typename M::Whole, Y>(a, t, block * M::BN, lds);
}

// out[t] = sum over k, ascending, of w[t][k] y[t][k]; a pair that was left out
// adds nothing (its row of y, not written by this call, is read but not used).
// A thread takes four neighbouring columns, eight pairs' loads at a time.
template <typename Y, typename T>
__global__ __launch_bounds__(256) void k_i8_combine(MoeI8 a) {
    constexpr bool SUMS = std::is_same<Y, I24x4>::value;
    constexpr int VEC = 4, AT = 8;
    const int hb = (a.H / VEC + 255) / 256, t = blockIdx.x / hb, n = ((blockIdx.x - t * hb) * 256 + threadIdx.x) * VEC;
    if (n >= a.H) return;   // H is a multiple of 16
    const int64_t p0 = (int64_t)t * a.K;
    float acc[VEC] = {};
    for (int k0 = 0; k0 < a.K; k0 += AT) {
        Y y[AT];
        float4 sd[AT];
        float w[AT], hs[AT];
        int e[AT];
#pragma unroll
        for (int i = 0; i < AT; i++) {
            const int64_t p = p0 + min(k0 + i, a.K - 1);
            y[i] = ((const Y*)a.y)[(p * a.H + n) / VEC];
            e[i] = k0 + i < a.K ? a.ids[p] : -1;
            w[i] = a.wts[p];
            hs[i] = SUMS ? a.hs[p] : 0.0f;
        }
#pragma unroll
        for (int i = 0; i < AT; i++)
            if (SUMS && (unsigned)e[i] < (unsigned)a.E) sd[i] = *(const float4*)(a.down_s + (int64_t)e[i] * a.H + n);
#pragma unroll
        for (int i = 0; i < AT; i++) {
            if ((unsigned)e[i] < (unsigned)a.E) {
                float4 v;
                if constexpr (SUMS) {
                    int x[VEC];
                    y[i].unpack(x);
                    const float s = hs[i];
                    v = make_float4((float)x[0] * s * sd[i].x, (float)x[1] * s * sd[i].y, (float)x[2] * s * sd[i].z,
                                    (float)x[3] * s * sd[i].w);
                } else {
                    v = y[i];
                }
                acc[0] = __builtin_fmaf(w[i], v.x, acc[0]);
                acc[1] = __builtin_fmaf(w[i], v.y, acc[1]);
                acc[2] = __builtin_fmaf(w[i], v.z, acc[2]);
                acc[3] = __builtin_fmaf(w[i], v.w, acc[3]);
            }
        }
    }
    store_row((T*)a.out + t * a.ldo + n, acc, VEC);
}

// ------------------------------------------------------------ host

// Whether each pair is computed on its own: two launches read an expert's
// weights again for every pair of it, five read them once; the three more are
// worth about 50 MB.  Pairs that meet an expert again, by even routing, are P -
// E (1 - (1 - 1/E)^P).  Together / on its own, us (H, F, E, K; tokens):
//   2048, 512, 256, 8    1 24.5 / 13.1   4 32 / 24   8 42 / 40   16 60 / 73
//   2048, 512, 8, 2      4 22 / 12.6     8 22 / 16   16 21 / 26  64 23 / 86
//   1024, 1024, 64, 4    4 25 / 18       8 30 / 24   16 37 / 40
//   4096, 2048, 8, 1     4 30 / 29       8 35 / 50
constexpr double MOE_AGAIN = 50e6;
constexpr int MOE_PAIRS = 256;   // of small experts too (256, 128, 8, 2; 512 pairs: 23 / 38)
static bool moe_few(int H, int F, int E, int K, int64_t P) {
    const double again = P - E * (1.0 - pow(1.0 - 1.0 / E, (double)P));
    // rows that fit the work-groups' registers (a token's rows of h: 16, 32 or 64
    // elements of a thread; one token, together / on its own: H 2048, F 1536,
    // top-8 42 / 27 us, 4096, 4096, top-4 76 / 51, 2048, 4096, top-8 67 / 60; but
    // 2048, 2048, top-16 54 / 57, 1024, 2048, top-16 36 / 41)
    return P <= MOE_PAIRS && again * 3.0 * H * F <= MOE_AGAIN && pad_to(H, I8_BK) <= 64 * FP_WAVES * FP_KEEP &&
           K * pad_to(F, I8_BK) <= 64 * FP_WAVES * (K <= 8 ? FP_KEEP_H : FP_KEEP_H / 2);
}
// Pairs per tile: 128 instead of 64 where an expert meets more than 40 on
// average (us, tiles of 64 / 128; H, F, E, K: average):
//   2048, 512, 256, 8    16 185 / 196, 32 209 / 212, 48 231 / 234, 64 251 / 249, 128 354 / 345
//   2048, 1536, 64, 4    32 147 / 144, 64 180 / 171, 128 247 / 240
//   4096, 1024, 16, 2    38 52 / 50, 188 119 / 105        1024, 256, 60, 4    47 32 / 33, 133 48 / 50
static int moe_tile_pairs(double avg) { return avg <= 40 ? 64 : 128; }

struct MoeI8Plan {
    size_t xq, xs, order, rank, total, cnt, tiles, h, hq, hs, y, bytes;
    int max_tiles, tile_pairs;
    bool few;
};

static MoeI8Plan plan_moe_i8(int H, int F, int E, int K, int T) {
    MoeI8Plan p{};
    const size_t P = (size_t)T * K;
    p.few = moe_few(H, F, E, K, (int64_t)P);
    auto take = [&](size_t& at, size_t n) { at = p.bytes; p.bytes += al256(n); };
    take(p.h, P * F * 4);
    if (p.few) return p;
    p.tile_pairs = moe_tile_pairs((double)P / E);
    p.max_tiles = (int)(P / p.tile_pairs + (P < (size_t)E ? P : (size_t)E));
    take(p.xq, (size_t)T * H);
    take(p.xs, (size_t)T * 4);
    take(p.order, P * 4);
    take(p.rank, P * 4);
    take(p.total, 8);
    take(p.cnt, (P + 1023) / 1024 * E * 4);
    // the list for the smallest tile, so that more tokens never need less
    take(p.tiles, (P / 64 + (P < (size_t)E ? P : (size_t)E)) * sizeof(int4));
    take(p.hq, P * F);
    take(p.hs, P * 4);
    take(p.y, P * H * 4);
    return p;
}

template <int COLS, int KEEP = FP_KEEP>
static void launch_pair_down(const MoeI8& a, int out_type, hipStream_t s) {
    const dim3 grid(a.H / COLS, a.T), block(64 * FP_WAVES);
    const size_t lh = a.K * pad_to(a.F, I8_BK);
    if constexpr (KEEP < FP_KEEP_H)
        if (lh > 64 * FP_WAVES * KEEP) return launch_pair_down<COLS, 2 * KEEP>(a, out_type, s);
    if (out_type == T_F32) hipLaunchKernelGGL((k_i8_pair_down<float, COLS, KEEP>), grid, block, lh, s, a);
    else if (out_type == T_F16) hipLaunchKernelGGL((k_i8_pair_down<_Float16, COLS, KEEP>), grid, block, lh, s, a);
    else hipLaunchKernelGGL((k_i8_pair_down<__bf16, COLS, KEEP>), grid, block, lh, s, a);
}

static void launch_few_pairs(const MoeI8& a, int type, int out_type, hipStream_t s) {
    const dim3 gu(a.F / 16, a.T * a.K), block(64 * FP_WAVES);
    const size_t lx = 16 + pad_to(a.H, I8_BK);
    if (type == T_F32) hipLaunchKernelGGL(k_i8_pair_gate_up<float>, gu, block, lx, s, a);
    else if (type == T_F16) hipLaunchKernelGGL(k_i8_pair_gate_up<_Float16>, gu, block, lx, s, a);
    else hipLaunchKernelGGL(k_i8_pair_gate_up<__bf16>, gu, block, lx, s, a);
    if (a.T * (a.H / 16) <= 256) launch_pair_down<8>(a, out_type, s);
    else launch_pair_down<16>(a, out_type, s);
}

template <typename X>
static void launch_prepare(const MoeI8& a, hipStream_t s) {
    const int P = a.T * a.K, groups = P <= PLAN_ONE ? 1 : (P + 1023) / 1024, per = i8_rows_per_group<1024>(a.H);
    const I8Rows<X> x{(const X*)a.x, a.ldx, a.xq, a.H, a.xs, nullptr, nullptr, a.T, a.H};
    const dim3 grid(groups + (a.T + per - 1) / per);
    if (groups == 1) {
        hipLaunchKernelGGL((k_i8_prepare<2, X>), grid, dim3(1024), 0, s, a, x, groups);
    } else {
        hipLaunchKernelGGL((k_i8_prepare<0, X>), grid, dim3(1024), 0, s, a, x, groups);
        hipLaunchKernelGGL(k_i8_plan, dim3(groups), dim3(1024), 0, s, a, groups);
    }
}

static void launch_hidden(const MoeI8& a, hipStream_t s) {
    const I8Rows<float> h{a.h, a.F, a.hq, a.F, a.hs, a.order, a.total, 0, a.F};
    const int per = i8_rows_per_group<256>(a.F);
    const dim3 grid((a.T * a.K + per - 1) / per);
    if (a.F <= I8_WAVE_ROW) hipLaunchKernelGGL(k_i8_hidden<1>, grid, dim3(256), 0, s, h);
    else hipLaunchKernelGGL(k_i8_hidden<4>, grid, dim3(256), 0, s, h);
}

template <int ROWS>
static void launch_tiles(const MoeI8& a, int max_tiles, hipStream_t s) {
    constexpr int BN = MoeTile<ROWS>::BN;
    const dim3 block(64 * MoeTile<ROWS>::WAVES);
    const dim3 gu((unsigned)((max_tiles * ((a.F + BN / 2 - 1) / (BN / 2)) + 7) / 8 * 8));
    const dim3 dn((unsigned)((max_tiles * ((a.H + BN - 1) / BN) + 7) / 8 * 8));
    hipLaunchKernelGGL(k_i8_gate_up<ROWS>, gu, block, 0, s, a);
    launch_hidden(a, s);
    if (a.F <= MAX_F24) hipLaunchKernelGGL((k_i8_down<ROWS, I24x4>), dn, block, 0, s, a);
    else hipLaunchKernelGGL((k_i8_down<ROWS, float4>), dn, block, 0, s, a);
}

template <typename Y>
static void launch_combine(const MoeI8& a, int out_type, hipStream_t s) {
    const dim3 grid((unsigned)((a.H / 4 + 255) / 256) * a.T);
    if (out_type == T_F32) hipLaunchKernelGGL((k_i8_combine<Y, float>), grid, dim3(256), 0, s, a);
    else if (out_type == T_F16) hipLaunchKernelGGL((k_i8_combine<Y, _Float16>), grid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL((k_i8_combine<Y, __bf16>), grid, dim3(256), 0, s, a);
}

static void launch_many_pairs(const MoeI8& a, const MoeI8Plan& p, int type, int out_type, hipStream_t s) {
    if (type == T_F32) launch_prepare<float>(a, s);
    else if (type == T_F16) launch_prepare<_Float16>(a, s);
    else launch_prepare<__bf16>(a, s);
    if (p.tile_pairs == 64) launch_tiles<64>(a, p.max_tiles, s);
    else launch_tiles<128>(a, p.max_tiles, s);
    if (a.F <= MAX_F24) launch_combine<I24x4>(a, out_type, s);
    else launch_combine<float4>(a, out_type, s);
}

// Whether the tiles' grids have less than 2^32 threads
static bool moe_i8_grids(int H, int F, int E, int64_t P) {
    const int rows = moe_tile_pairs((double)P / E);   // 64 pairs: 256 threads, 128: 512
    const int64_t tiles = P / rows + (P < E ? P : E), blocks = (F + 63) / 64, down = (H + 127) / 128;
    return (tiles * (blocks > down ? blocks : down) + 7) / 8 * 8 * 4 * rows < (int64_t)1 << 32;
}
// Sizes whose offsets within a tensor of tokens or of one expert stay below 2^31
static bool moe_i8_shape(const chimere_moe_i8_layer* L, int K, int T) {
    const int64_t lim = (int64_t)1 << 31, P = (int64_t)T * K;
    const bool sizes = L->hidden >= 16 && L->hidden % 16 == 0 && L->hidden <= I8_MAX_C && L->ffn >= 16 && L->ffn % 16 == 0 &&
           L->ffn <= I8_MAX_C && (int64_t)L->hidden * L->ffn < lim && L->n_experts >= 1 && L->n_experts <= MAX_E &&
           K >= 1 && K <= MAX_K && T >= 0 && (int64_t)T * L->hidden < lim && P < (1 << 24);
    return sizes && moe_i8_grids(L->hidden, L->ffn, L->n_experts, P);
}

}  // namespace chimere

using namespace chimere;

extern "C" {

size_t chimere_moe_i8_workspace_size(const chimere_moe_i8_layer* L, int top_k, int max_ntok) {
    if (!L || max_ntok < 1 || !moe_i8_shape(L, top_k, max_ntok)) return 0;
    return plan_moe_i8(L->hidden, L->ffn, L->n_experts, top_k, max_ntok).bytes;
}

void chimere_moe_i8(const chimere_moe_i8_layer* L, int type, const void* x, int64_t x_stride, const int* ids,
                    const float* weights, int top_k, int out_type, void* out, int64_t out_stride, int ntok,
                    void* workspace, size_t workspace_bytes, hipStream_t stream) {
    CHIMERE_REQUIRE(L, CHIMERE_ERR_ARG, "moe_i8: null pointer");
    CHIMERE_REQUIRE(float_type(type) && float_type(out_type), CHIMERE_ERR_ARG, "moe_i8: unsupported type %d / %d",
                    type, out_type);
    CHIMERE_REQUIRE(moe_i8_shape(L, top_k, ntok), CHIMERE_ERR_ARG,
                    "moe_i8: hidden=%d / ffn=%d must be multiples of 16, n_experts=%d top_k=%d ntok=%d in range",
                    L->hidden, L->ffn, L->n_experts, top_k, ntok);
    CHIMERE_REQUIRE(L->gate && L->up && L->down && L->gate_scale && L->up_scale && L->down_scale, CHIMERE_ERR_ARG,
                    "moe_i8: null weight pointer");
    CHIMERE_REQUIRE((((uintptr_t)L->gate | (uintptr_t)L->up | (uintptr_t)L->down | (uintptr_t)L->gate_scale |
                      (uintptr_t)L->up_scale | (uintptr_t)L->down_scale) & 15) == 0, CHIMERE_ERR_ARG,
                    "moe_i8: weights and scales must be 16-byte aligned");
    if (ntok == 0) return;
    CHIMERE_REQUIRE(x && ids && weights && out && workspace, CHIMERE_ERR_ARG, "moe_i8: null pointer");
    CHIMERE_REQUIRE(x_stride >= 0 && out_stride >= L->hidden && float_aligned(type, x) && float_aligned(out_type, out),
                    CHIMERE_ERR_ARG, "moe_i8: bad strides %lld %lld, or rows not aligned to their elements",
                    (long long)x_stride, (long long)out_stride);
    const int H = L->hidden, F = L->ffn;
    const MoeI8Plan p = plan_moe_i8(H, F, L->n_experts, top_k, ntok);
    CHIMERE_REQUIRE(workspace_bytes >= p.bytes && ((uintptr_t)workspace & 255) == 0, CHIMERE_ERR_WORKSPACE,
                    "moe_i8: workspace %zu bytes < %zu (or not 256-byte aligned)", workspace_bytes, p.bytes);
    uint8_t* w = (uint8_t*)workspace;
    MoeI8 a{};
    a.H = H; a.F = F; a.E = L->n_experts; a.K = top_k; a.T = ntok;
    a.gate = L->gate; a.up = L->up; a.down = L->down;
    a.gate_s = L->gate_scale; a.up_s = L->up_scale; a.down_s = L->down_scale;
    a.ids = ids; a.wts = weights; a.x = x; a.ldx = x_stride; a.out = out; a.ldo = out_stride;
    a.h = (float*)(w + p.h);
    if (p.few) {
        launch_few_pairs(a, type, out_type, stream);
    } else {
        a.xq = (int8_t*)(w + p.xq); a.xs = (float*)(w + p.xs);
        a.order = (int*)(w + p.order); a.rank = (int*)(w + p.rank);
        a.total = (int*)(w + p.total); a.cnt = (int*)(w + p.cnt); a.tiles = (int4*)(w + p.tiles);
        a.hq = (int8_t*)(w + p.hq); a.hs = (float*)(w + p.hs); a.y = w + p.y;
        a.tile_pairs = p.tile_pairs;
        launch_many_pairs(a, p, type, out_type, stream);
    }
    check_launch("moe_i8");
}

}  // extern "C"
