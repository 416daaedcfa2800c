// int8_gemm.h -- tile product of 8-bit integer rows on the matrix cores.
//
// acc[m][n] = sum_c a[m][c] * w[n][c] for a tile of BM token rows and BN weight
// rows, in int32 (exact: at most 131071 columns of products up to 2^14).  Both
// operands are rows along c, so one v_mfma_i32_32x32x32_i8 takes 32 rows of
// each and 32 columns, every lane 16 consecutive bytes of one row.
//
// Staging: 128 columns of every row per step, copied global -> LDS in 16-byte
// pieces by asynchronous copies, two to four steps ahead.  A row's eight pieces
// are stored at piece ^ (row / 2 & 7), so the rows that a fragment read touches
// at the same piece spread over all banks.  Rows behind the last one and pieces
// behind the last column are read from clamped addresses: what a clamped row
// yields is not stored, and the columns behind C are cleared in the token
// fragments of the last step (their product with whatever the weight rows hold
// is 0).
#pragma once
#include <type_traits>

#include "float_rows.h"

namespace chimere {

constexpr int I8_BK = 128;              // columns per step
constexpr int I8_MAX_C = 131071;        // |sum| <= 131071 * 2^14 < 2^31
constexpr int I8_MAX_ROWS = 1 << 25;    // of either operand, and outputs: a grid has less than 2^32 threads
constexpr int64_t I8_MAX_OUT = (int64_t)1 << 38;
constexpr int I8_MAX_STRIDE = 1 << 23;  // bytes between rows: 256 rows of a tile stay within 32-bit offsets

typedef int v4i __attribute__((ext_vector_type(4)));
typedef int v16i __attribute__((ext_vector_type(16)));

// One 16-byte asynchronous copy per lane from base + off (off: 32 bits per
// lane) to LDS offset lds_wave + 16 * lane; not tracked by the compiler, as
// copy16_lds_untracked.
__device__ __forceinline__ void copy16_lds_base(const void* base, uint32_t off, uint32_t lds_wave) {
    uint32_t saved;
    __asm__ volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %3\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2\n\t"
                     "s_mov_b32 m0, %0"
                     : "=&s"(saved)
                     : "v"(off), "s"(base), "s"(lds_wave)
                     : "memory");
}

// a pointer that is the same for the whole wave, in scalar registers
__device__ __forceinline__ const int8_t* wave_uniform(const int8_t* p) {
    const uint64_t v = (uint64_t)(uintptr_t)p;
    const uint64_t lo = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)v);
    const uint64_t hi = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(v >> 32));
    return (const int8_t*)(uintptr_t)(hi << 32 | lo);
}

// `v` (columns k0 .. k0 + 15 of a row) with the columns from C on cleared
__device__ __forceinline__ v4i clear_tail(v4i v, int k0, int C) {
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const int n = C - k0 - 4 * j;
        v[j] = n >= 4 ? v[j] : n <= 0 ? 0 : v[j] & (int)((1u << (8 * n)) - 1u);
    }
    return v;
}

// WM x WN waves, each MT x NT blocks of 32 x 32; NS stages of weight rows and NA
// of token rows (these come from L2, the weights often from HBM: more of them
// in flight is what hides the longer way)
template <int WM, int WN, int MT, int NT, int NS = 2, int NA = NS>
struct I8Tile {
    static constexpr int BM = WM * MT * 32, BN = WN * NT * 32, NW = WM * WN;
    static constexpr int WAVES_N = WN, MTILES = MT, NTILES = NT;
    static constexpr int SA = BM * I8_BK, SW = BN * I8_BK, LDS = NA * SA + NS * SW;
    static_assert(NA >= 2 && NA <= NS, "stages");
    static constexpr int PM = BM / 8 / NW, PN = BN / 8 / NW;   // pieces of 8 rows that a wave copies
    static_assert(PM * 8 * NW == BM && PN * 8 * NW == BN, "tile rows over waves");

    // aoff[p] / woff[p]: this lane's row of piece p, as a byte offset from a / w
    // (row (wave * P + p) * 8 + lane / 8 of the tile).  Weight rows come in
    // blocks of 16 in turn from w and from w2 (the same matrix, or two).
    static __device__ __forceinline__ void run(const int8_t* a, const int8_t* w, const int8_t* w2,
                                               const uint32_t (&aoff)[PM], const uint32_t (&woff)[PN], int C,
                                               uint8_t* lds, v16i (&acc)[MT][NT]) {
        const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        const int wm = wave / WN, wn = wave % WN;
        a = wave_uniform(a);
        w = wave_uniform(w);
        w2 = wave_uniform(w2);
        const int S = (C + I8_BK - 1) / I8_BK, last = (C + 15) / 16 - 1, pc = (lane & 7) ^ (lane >> 4);
        const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_void_t*)lds;
        // copies of step s into stage `to`; past the last step the same columns
        // again, so that the count of copies in flight stays the same
        auto stage_a = [&](int s, int to) {
            const uint32_t k0 = (uint32_t)min(8 * s + pc, last) * 16u, k1 = (uint32_t)min(8 * s + (pc ^ 4), last) * 16u;
#pragma unroll
            for (int p = 0; p < PM; p++)
                copy16_lds_base(a, aoff[p] + ((wave * PM + p) & 1 ? k1 : k0), lds0 + to * SA + (wave * PM + p) * 1024);
        };
        auto stage_w = [&](int s, int to) {
            const uint32_t k0 = (uint32_t)min(8 * s + pc, last) * 16u, k1 = (uint32_t)min(8 * s + (pc ^ 4), last) * 16u;
#pragma unroll
            for (int p = 0; p < PN; p++)
                copy16_lds_base((wave * PN + p) & 2 ? w2 : w, woff[p] + ((wave * PN + p) & 1 ? k1 : k0),
                                lds0 + NA * SA + to * SW + (wave * PN + p) * 1024);
        };
#pragma unroll
        for (int i = 0; i < MT; i++)
#pragma unroll
            for (int j = 0; j < NT; j++) acc[i][j] = v16i{};
        // in the order of the steps below, which issue token rows first
#pragma unroll
        for (int s = 0; s < NS - 1; s++) {
            if (s >= NS - NA) stage_a(s - (NS - NA), s - (NS - NA));
            stage_w(s, s);
        }
        const int r = lane & 31, g = lane >> 5;
        int ca = 0, na = NA - 1, cw = 0, nw = NS - 1;
        auto step = [&](int s, auto tail) {
            // this wave's copies of step s have landed (issued later: the weights
            // of NS - NA steps more, and NA - 2 whole steps),
            wait_vm<(NA < NS ? PN : 0) + (NA - 2) * (PM + PN)>();
            lds_barrier();   // every wave's; and step s - 1 has been read by all
            stage_a(s + NA - 1, na);
            stage_w(s + NS - 1, nw);
            const uint8_t *at = lds + ca * SA, *wt = lds + NA * SA + cw * SW;
            ca = ca + 1 == NA ? 0 : ca + 1;
            na = na + 1 == NA ? 0 : na + 1;
            cw = cw + 1 == NS ? 0 : cw + 1;
            nw = nw + 1 == NS ? 0 : nw + 1;
            // the fragments of columns 32 (q + 1) are read while those of 32 q multiply
            v4i fa[2][MT], fw[2][NT];
            auto read = [&](int q) {
                const int c = 2 * q + g, piece = (c ^ (r >> 1 & 7)) * 16;
#pragma unroll
                for (int i = 0; i < MT; i++)
                    fa[q & 1][i] = *(const v4i*)(at + ((wm * MT + i) * 32 + r) * I8_BK + piece);
#pragma unroll
                for (int j = 0; j < NT; j++)
                    fw[q & 1][j] = *(const v4i*)(wt + ((wn * NT + j) * 32 + r) * I8_BK + piece);
                if (tail) {
#pragma unroll
                    for (int i = 0; i < MT; i++) fa[q & 1][i] = clear_tail(fa[q & 1][i], s * I8_BK + c * 16, C);
                }
            };
            read(0);
#pragma unroll
            for (int q = 0; q < 4; q++) {
                if (q < 3) read(q + 1);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int i = 0; i < MT; i++)
#pragma unroll
                    for (int j = 0; j < NT; j++)
                        acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(fa[q & 1][i], fw[q & 1][j], acc[i][j], 0, 0, 0);
                __builtin_amdgcn_sched_barrier(0);
            }
        };
        const int full = C / I8_BK;
        for (int s = 0; s < full; s++) step(s, std::false_type{});
        if (full < S) step(full, std::true_type{});
        wait_vm<0>();   // no copy may land in LDS that another work-group then owns
    }
    // The tile's sums, a row at a time: a wave lays 16 rows at a time of its
    // blocks out in LDS (in the stages, that run() is done with) and each lane
    // takes VEC neighbouring columns of one row, the same columns of every row
    // (first_col()), so that a row's stores are 16 bytes wide:
    // emit(row, sums, of_row) with the row counted within the tile and of_row the
    // value that thread `row` handed in (a scale that is loaded once, ahead of
    // the loop: loaded where it is used, each load's latency was paid 16 times
    // per tile, 17 us of a 256 x 256 tile).  PAIR (w and w2): columns are
    // those of w's rows and emit gets the sums of both,
    // emit(row, sums, sums2, of_row).
    static constexpr int PAD = NT * 32 + 8;   // dwords per row: the two half-waves write 4 rows apart, 32 banks apart
    static_assert(NW * 16 * PAD * 4 + BM * 8 <= LDS && 64 * NW >= BM, "the layout fits the stages, a thread per row");
    template <int VEC, bool PAIR = false>
    static __device__ __forceinline__ int first_col() {
        constexpr int COLS = PAIR ? NT * 16 : NT * 32;
        return (int)(threadIdx.x >> 6) % WN * COLS + (threadIdx.x & 63) % (COLS / VEC) * VEC;
    }
    template <int VEC, bool PAIR = false, typename Emit>
    static __device__ __forceinline__ void rows(uint8_t* lds, const v16i (&acc)[MT][NT], float2 of_row, Emit emit) {
        constexpr int COLS = PAIR ? NT * 16 : NT * 32, LANES = COLS / VEC, ROWS = 64 / LANES;
        static_assert(ROWS <= 16, "16 rows at a time");
        const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        const int wm = wave / WN;
        float2* each = (float2*)lds;
        int* at = (int*)(lds + BM * 8) + wave * 16 * PAD;
        lds_barrier();   // every wave has read its last stage
        if (threadIdx.x < BM) each[threadIdx.x] = of_row;
        lds_barrier();
#pragma unroll
        for (int h = 0; h < 2 * MT; h++) {
            // register v of a block: row 8 (v / 4) + 4 (lane / 32) + v % 4, column lane % 32
#pragma unroll
            for (int j = 0; j < NT; j++)
#pragma unroll
                for (int v = 0; v < 8; v++)
                    at[(8 * (v >> 2) + 4 * (lane >> 5) + (v & 3)) * PAD + j * 32 + (lane & 31)] =
                        acc[h >> 1][j][8 * (h & 1) + v];
#pragma unroll
            for (int q = 0; q < 16 / ROWS; q++) {
                const int r = q * ROWS + lane / LANES, c = lane % LANES * VEC, m = wm * MT * 32 + h * 16 + r;
                int x[VEC], y[VEC];
                const int* p = at + r * PAD + (PAIR ? (c >> 4) * 32 + (c & 15) : c);
#pragma unroll
                for (int k = 0; k < VEC; k += 4) {
                    *(v4i*)(x + k) = *(const v4i*)(p + k);
                    if constexpr (PAIR) *(v4i*)(y + k) = *(const v4i*)(p + 16 + k);
                }
                if constexpr (PAIR) emit(m, x, y, each[m]);
                else emit(m, x, each[m]);
            }
        }
    }
};

}  // namespace chimere
