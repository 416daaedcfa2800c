// int8_gemm.h -- tile product of 8-bit integer rows on the matrix cores.
//
// acc[m][n] = sum_c a[m][c] * w[n][c] for a tile of BM token rows and BN weight
// rows, in int32 (exact: at most 131071 columns of products up to 2^14).  Both
// operands are rows along c, so one v_mfma_i32_32x32x32_i8 takes 32 rows of
// each and 32 columns, every lane 16 consecutive bytes of one row.
//
// Staging: 128 columns of every row per step, copied global -> LDS in 16-byte
// pieces by asynchronous copies, two stages.  A row's eight pieces are stored
// at piece ^ (row & 7), so the 32 rows that a fragment read touches at the same
// piece spread over all banks.  Rows behind the last one and pieces behind the
// last column are read from clamped addresses: what a clamped row yields is
// not stored, and the columns behind C are cleared in the token fragments of
// the last step (their product with whatever the weight rows hold is 0).
#pragma once
#include "float_rows.h"

namespace chimere {

constexpr int I8_BK = 128;              // columns per step
constexpr int I8_MAX_C = 131071;        // |sum| <= 131071 * 2^14 < 2^31
constexpr int I8_MAX_STRIDE = 1 << 23;  // bytes between rows: 256 rows of a tile stay within 32-bit offsets

typedef int v4i __attribute__((ext_vector_type(4)));
typedef int v16i __attribute__((ext_vector_type(16)));

// One 16-byte asynchronous copy per lane from base + off (off: 32 bits per
// lane) to lds_wave + 16 * lane; see copy16_lds_untracked.
__device__ __forceinline__ void copy16_lds_base(const void* base, uint32_t off, void* lds_wave) {
    const uint32_t m = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)lds_wave);
    uint32_t saved;
    __asm__ volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %3\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2\n\t"
                     "s_mov_b32 m0, %0"
                     : "=&s"(saved)
                     : "v"(off), "s"(base), "s"(m)
                     : "memory");
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

// WM x WN waves, each MT x NT blocks of 32 x 32
template <int WM, int WN, int MT, int NT>
struct I8Tile {
    static constexpr int BM = WM * MT * 32, BN = WN * NT * 32, NW = WM * WN;
    static constexpr int WAVES_N = WN, MTILES = MT, NTILES = NT;
    static constexpr int STAGE = (BM + BN) * I8_BK, LDS = 2 * STAGE;
    static constexpr int PM = BM / 8 / NW, PN = BN / 8 / NW;   // pieces of 8 rows that a wave copies
    static_assert(PM * 8 * NW == BM && PN * 8 * NW == BN, "tile rows over waves");

    // aoff[p] / woff[p]: this lane's row of piece p, as a byte offset from a / w
    // (row (wave * P + p) * 8 + lane / 8 of the tile).  Weight rows come in
    // blocks of 32 in turn from w and from w2 (the same matrix, or two).
    static __device__ __forceinline__ void run(const int8_t* a, const int8_t* w, const int8_t* w2,
                                               const uint32_t (&aoff)[PM], const uint32_t (&woff)[PN], int C,
                                               uint8_t* lds, v16i (&acc)[MT][NT]) {
        const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        const int wm = wave / WN, wn = wave % WN;
        const int S = (C + I8_BK - 1) / I8_BK, last = (C + 15) / 16 - 1, pc = (lane & 7) ^ (lane >> 3);
        auto stage = [&](int s) {
            uint8_t* at = lds + (s & 1) * STAGE;
            const uint32_t k = (uint32_t)min(8 * s + pc, last) * 16u;
#pragma unroll
            for (int p = 0; p < PM; p++) copy16_lds_base(a, aoff[p] + k, at + (wave * PM + p) * 1024);
#pragma unroll
            for (int p = 0; p < PN; p++) 
                copy16_lds_base((wave * PN + p) & 4 ? w2 : w, woff[p] + k, at + BM * I8_BK + (wave * PN + p) * 1024);
        };
#pragma unroll
        for (int i = 0; i < MT; i++)
#pragma unroll
            for (int j = 0; j < NT; j++) acc[i][j] = v16i{};
        stage(0);
        const int r = lane & 31, g = lane >> 5;
        for (int s = 0; s < S; s++) {
            if (s + 1 < S) {
                stage(s + 1);
                wait_vm<PM + PN>();
            } else {
                wait_vm<0>();
            }
            lds_barrier();
            const uint8_t* at = lds + (s & 1) * STAGE;
            const bool tail = s + 1 == S && (C & (I8_BK - 1));
#pragma unroll
            for (int q = 0; q < 4; q++) {
                const int c = 2 * q + g, piece = (c ^ (r & 7)) * 16;
                v4i fa[MT], fw[NT];
#pragma unroll
                for (int i = 0; i < MT; i++) fa[i] = *(const v4i*)(at + ((wm * MT + i) * 32 + r) * I8_BK + piece);
#pragma unroll
                for (int j = 0; j < NT; j++)
                    fw[j] = *(const v4i*)(at + (BM + (wn * NT + j) * 32 + r) * I8_BK + piece);
                if (tail) {
#pragma unroll
                    for (int i = 0; i < MT; i++) fa[i] = clear_tail(fa[i], s * I8_BK + c * 16, C);
                }
#pragma unroll
                for (int i = 0; i < MT; i++)
#pragma unroll
                    for (int j = 0; j < NT; j++)
                        acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(fa[i], fw[j], acc[i][j], 0, 0, 0);
            }
            lds_barrier();   // the next step's copies write the stage that was read here
        }
    }
    // row of register i of a 32 x 32 block (column: lane & 31)
    static __device__ __forceinline__ int reg_row(int i) { return 8 * (i >> 2) + 4 * ((threadIdx.x & 63) >> 5) + (i & 3); }
};

// row quantizer (int8.hip), for float rows of a type on the device
void launch_i8_quantize(int type, const void* x, int64_t xs, int8_t* q, int64_t qs, float* scale, int64_t nrows,
                        int ncols, hipStream_t s);

}  // namespace chimere
