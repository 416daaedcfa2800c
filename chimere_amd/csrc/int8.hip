// int8.hip -- rows in 8-bit integers with one scale each, and their product.
// No counterpart in the reference, whose dense products of a prompt run one
// token at a time through the block-quantized GEMV.
#include "api_internal.h"
#include "int8_gemm.h"
#include "int8_quant.h"

namespace chimere {

// Row quantizer.  A row that holds an infinity or a NaN keeps it in the scale
// and 0 in its integers, so its products are NaN.  Bound by the rows' bytes.
template <typename T, int W>
__global__ __launch_bounds__(256) void k_i8_quantize(I8Rows<T> q) {
    i8_quantize_rows<T, W, 256>(q, blockIdx.x);
}

template <typename T>
static void launch_i8_quantize(const T* x, int64_t xs, int8_t* q, int64_t qs, float* scale, int64_t nrows, int ncols,
                               hipStream_t s) {
    i8_slices<256>(nrows, ncols, [&](int64_t r, int64_t n, int64_t groups) {
        const I8Rows<T> rows{x + r * xs, xs, q + r * qs, qs, scale + r, nullptr, nullptr, n, ncols};
        const dim3 grid((unsigned)groups);
        if (ncols <= I8_WAVE_ROW) hipLaunchKernelGGL((k_i8_quantize<T, 1>), grid, dim3(256), 0, s, rows);
        else hipLaunchKernelGGL((k_i8_quantize<T, 4>), grid, dim3(256), 0, s, rows);
    });
}

void launch_i8_quantize(int type, const void* x, int64_t xs, int8_t* q, int64_t qs, float* scale, int64_t nrows,
                        int ncols, hipStream_t s) {
    if (type == T_F32) launch_i8_quantize((const float*)x, xs, q, qs, scale, nrows, ncols, s);
    else if (type == T_F16) launch_i8_quantize((const _Float16*)x, xs, q, qs, scale, nrows, ncols, s);
    else launch_i8_quantize((const __bf16*)x, xs, q, qs, scale, nrows, ncols, s);
}

struct I8Gemm {
    const int8_t *a, *w;
    const float *as, *ws, *bias;
    void* out;
    int64_t lda, ldw, ldo;
    int M, N, C;
    const void* x;     // float tokens that the kernel quantizes itself, or null
    int64_t ldx;
};

// Many tokens: one tile per work-group.  Tiles go to the XCDs in contiguous
// eighths (work-groups are dealt round-robin), four token tiles against all
// weight tiles in turn, so the tiles that an XCD works on at a time share
// their rows in its L2.
template <typename T, typename Tile, int WAVES_PER_SIMD>
__global__ __launch_bounds__(64 * Tile::NW, WAVES_PER_SIMD) void k_i8_gemm(I8Gemm g) {
    __shared__ __align__(16) uint8_t lds[Tile::LDS];
    constexpr int VEC = sizeof(T) == 4 ? 4 : 8, GM = 4;
    const int tm = (g.M + Tile::BM - 1) / Tile::BM, tn = (g.N + Tile::BN - 1) / Tile::BN;
    const int per = (tm * tn + 7) / 8, tile = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
    if (tile >= tm * tn) return;
    const int grp = tile / (GM * tn), rows = min(GM, tm - grp * GM), at = tile - grp * GM * tn;
    const int m0 = (grp * GM + at % rows) * Tile::BM, n0 = at / rows * Tile::BN;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint32_t aoff[Tile::PM], woff[Tile::PN];
#pragma unroll
    for (int p = 0; p < Tile::PM; p++)
        aoff[p] = (uint32_t)(min((wave * Tile::PM + p) * 8 + (lane >> 3), g.M - 1 - m0) * g.lda);
#pragma unroll
    for (int p = 0; p < Tile::PN; p++)
        woff[p] = (uint32_t)(min((wave * Tile::PN + p) * 8 + (lane >> 3), g.N - 1 - n0) * g.ldw);
    const float as = threadIdx.x < Tile::BM ? g.as[min(m0 + (int)threadIdx.x, g.M - 1)] : 0.0f;
    const int n = n0 + Tile::template first_col<VEC>();
    float ws[VEC], b[VEC];
#pragma unroll
    for (int k = 0; k < VEC; k++) {
        const int nk = min(n + k, g.N - 1);
        ws[k] = g.ws[nk];
        b[k] = g.bias ? g.bias[nk] : 0.0f;
    }
    v16i acc[Tile::MTILES][Tile::NTILES];
    const int8_t* w = g.w + n0 * g.ldw;
    Tile::run(g.a + m0 * g.lda, w, w, aoff, woff, g.C, lds, acc);
    Tile::template rows<VEC>(lds, acc, make_float2(as, 0.0f), [&](int r, const int(&x)[VEC], float2 of_row) {
        if (m0 + r >= g.M || n >= g.N) return;
        float v[VEC];
#pragma unroll
        for (int k = 0; k < VEC; k++) v[k] = (float)x[k] * of_row.x * ws[k] + b[k];
        store_row((T*)g.out + (m0 + r) * g.ldo + n, v, g.N - n);
    });
}

// Few tokens: 16 MB of them against 16 NB weight rows per work-group, the
// columns in steps of 128 dealt to its eight waves (v_mfma_i32_16x16x64_i8,
// fragments straight from memory: no weight byte is used by two waves), whose
// int32 sums are joined in LDS.  With X, tokens are floats that every
// work-group quantizes for itself (one launch less); their integers lie in
// LDS, cleared up to whole steps.
constexpr int FEW_WAVES = 8;

// KEEP: elements that a thread quantizes at most
template <typename T, typename X, int MB, int NB, int KEEP = 16>
__global__ __launch_bounds__(64 * FEW_WAVES) void k_i8_few(I8Gemm g) {
    constexpr bool QUANT = !std::is_same<X, int8_t>::value;
    extern __shared__ __align__(16) uint8_t lds[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int m0 = blockIdx.y * 16 * MB, n0 = blockIdx.x * 16 * NB;
    const int S = (g.C + I8_BK - 1) / I8_BK, last = (g.C + 15) / 16 - 1;
    const int r = lane & 15, pc = lane >> 4;
    const int lda = S * I8_BK + 16;   // of the integers in LDS: rows 4 banks apart
    const int M = min(g.M - m0, 16 * MB);
    const int8_t* arow[MB];
    const int8_t* wrow[NB];
#pragma unroll
    for (int j = 0; j < NB; j++) wrow[j] = g.w + (int64_t)min(n0 + j * 16 + r, g.N - 1) * g.ldw;
    v4i fw[NB][2];
    auto load_w = [&](int s) {
#pragma unroll
        for (int j = 0; j < NB; j++)
#pragma unroll
            for (int h = 0; h < 2; h++) fw[j][h] = *(const v4i*)(wrow[j] + min(8 * s + 4 * h + pc, last) * 16);
    };
    if (wave < S) load_w(wave);
    // the scales of this thread's outputs (`at`), ahead of all that is waited for
    constexpr int OUTS = (MB * NB * 256 + 64 * FEW_WAVES - 1) / (64 * FEW_WAVES);
    float ws[OUTS], bias[OUTS];
    // register v of lane l in a block (i, j): token 4 (l / 16) + v, weight row l % 16
    auto at = [&](int q, int& m, int& n, int& from) {
        const int o = tid + q * 64 * FEW_WAVES, i = o / (NB * 256), v = o >> 6 & 3, l = o & 63, j = o / 256 % NB;
        m = i * 16 + 4 * (l >> 4) + v;
        n = n0 + j * 16 + (l & 15);
        from = (i * NB + j) * 256 + l * 4 + v;
        return o < MB * NB * 256 && m < M && n < g.N;
    };
#pragma unroll
    for (int q = 0; q < OUTS; q++) {
        int m, n, from;
        const bool in = at(q, m, n, from);
        ws[q] = in ? g.ws[n] : 0.0f;
        bias[q] = in && g.bias ? g.bias[n] : 0.0f;
    }
    float* as = (float*)lds;   // [16 MB]
    uint8_t* aq = lds + 16 * MB * 4;
    if constexpr (QUANT) {
        i8_rows_to_lds<64 * FEW_WAVES, KEEP>(M, S * I8_BK, lda, as, aq, [&](int m, int c, auto& v) {
            i8_load((const X*)g.x + (m0 + m) * g.ldx, c, g.C, v);
        }, std::integral_constant<int, 16 / sizeof(X)>{});
    } else {
        if (tid < 16 * MB) as[tid] = g.as[m0 + min(tid, M - 1)];
    }
#pragma unroll
    for (int i = 0; i < MB; i++) {
        const int m = min(i * 16 + r, M - 1);
        arow[i] = QUANT ? (const int8_t*)aq + m * lda : g.a + (m0 + m) * g.lda;
    }
    v4i acc[MB][NB] = {};
    for (int s = wave; s < S; s += FEW_WAVES) {
        v4i fa[MB][2], w[NB][2];
#pragma unroll
        for (int i = 0; i < MB; i++)
#pragma unroll
            for (int h = 0; h < 2; h++) {
                if constexpr (QUANT) {
                    fa[i][h] = *(const v4i*)(arow[i] + (8 * s + 4 * h + pc) * 16);
                } else {
                    fa[i][h] = *(const v4i*)(arow[i] + min(8 * s + 4 * h + pc, last) * 16);
                    if ((s + 1) * I8_BK > g.C) fa[i][h] = clear_tail(fa[i][h], (8 * s + 4 * h + pc) * 16, g.C);
                }
            }
#pragma unroll
        for (int j = 0; j < NB; j++)
#pragma unroll
            for (int h = 0; h < 2; h++) w[j][h] = fw[j][h];
        if (s + FEW_WAVES < S) load_w(s + FEW_WAVES);
#pragma unroll
        for (int i = 0; i < MB; i++)
#pragma unroll
            for (int j = 0; j < NB; j++)
#pragma unroll
                for (int h = 0; h < 2; h++)
                    acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(fa[i][h], w[j][h], acc[i][j], 0, 0, 0);
    }
    __syncthreads();   // aq has been read
    int* part = (int*)(lds + 16 * MB * 4);
#pragma unroll
    for (int i = 0; i < MB; i++)
#pragma unroll
        for (int j = 0; j < NB; j++) *(v4i*)(part + ((wave * MB + i) * NB + j) * 256 + lane * 4) = acc[i][j];
    __syncthreads();
#pragma unroll
    for (int q = 0; q < OUTS; q++) {
        int m, n, from, sum = 0;
        if (!at(q, m, n, from)) continue;
#pragma unroll
        for (int w = 0; w < FEW_WAVES; w++) sum += part[w * MB * NB * 256 + from];
        store_f((T*)g.out + (m0 + m) * g.ldo + n, (float)sum * as[m] * ws[q] + bias[q]);
    }
}

template <typename T, typename X, int MB, int NB, int KEEP = 16>
static void launch_few(const I8Gemm& g, hipStream_t s) {
    const size_t aq = std::is_same<X, int8_t>::value
                          ? 0 : (size_t)(g.M < 16 * MB ? g.M : 16 * MB) * (pad_to(g.C, I8_BK) + 16);
    const size_t part = (size_t)FEW_WAVES * MB * NB * 256 * 4;
    const dim3 grid((g.N + 16 * NB - 1) / (16 * NB), (g.M + 16 * MB - 1) / (16 * MB));
    hipLaunchKernelGGL((k_i8_few<T, X, MB, NB, KEEP>), grid, dim3(64 * FEW_WAVES), 16 * MB * 4 + (aq > part ? aq : part), s, g);
}

template <typename T, typename Tile, int WAVES_PER_SIMD>
static void launch_tiles(const I8Gemm& g, hipStream_t s) {
    const int64_t tiles = (int64_t)((g.M + Tile::BM - 1) / Tile::BM) * ((g.N + Tile::BN - 1) / Tile::BN);
    hipLaunchKernelGGL((k_i8_gemm<T, Tile, WAVES_PER_SIMD>), dim3((unsigned)((tiles + 7) / 8 * 8)), dim3(64 * Tile::NW),
                       0, s, g);
}

// Which kernel takes a product, by how many work-groups its tiles make for the
// 256 CUs: a larger tile reads its rows fewer times (all CUs together draw about
// 13 TB/s from L2: 128 x 128 tiles of 4096 x 8192 x 4096 take 160 us, 256 x 256
// 128), a smaller one puts more CUs to work, and where two work-groups fit a CU
// two stages are enough, with one the third hides the weights' way from HBM.
// Microseconds in a graph, each launch its own weights, from HBM (the same ones
// every time take up to a quarter less), tokens x rows x columns (bf16 out):
//   few tokens   16 x 1 / 16 x 2 rows   1x4096x2048 4.2 / 4.8  1x16384x4096 15.6 / 16.6 (the same weights 13.4 / 12.8)
//                1x151936x2048 51.0 / 51.6  16x16384x2048 10.3 / 9.1; 64 x 64 tiles 1x4096x2048 7.4
//   24x4096x2048     32 x 16 5.4, 32 x 32 6.4, 64 x 64 7.6    100x4096x2048  32 x 32 10.4, 64 x 64 7.9
//   100x2048x4096    32 x 16 13.6, 32 x 32 10.2, 64 x 64 11.6
//   512x2048x2048    64 x 64 with two stages 12.0, four 7.6; 64 x 128 9.5, 128 x 128 12.4
//   256x8192x4096    64 x 64 21.7, 64 x 128 20.1, 128 x 128 23.1    48x151936x2048 64 x 64 71, 64 x 128 64, 128 x 128 77
//   512x8192x2048    64 x 64 22, 64 x 128 18.2, 128 x 128 with two stages 20.1, three 15.4, 256 x 256 30
//   1000x8192x8192   128 x 128 with two stages 79, three 88, 256 x 256 93
constexpr int FEW_N = 8192;
template <typename T>
static void launch_gemm(const I8Gemm& g, hipStream_t s) {
    auto tiles = [&](int bm, int bn) { return (int64_t)((g.M + bm - 1) / bm) * ((g.N + bn - 1) / bn); };
    const bool short_rows = (g.M + 255) / 256 * 256 > (g.M + 127) / 128 * 160;   // over a quarter of 256-row tiles empty
    if (g.M <= 16) {
        if (g.N <= FEW_N) launch_few<T, int8_t, 1, 1>(g, s);
        else launch_few<T, int8_t, 1, 2>(g, s);
    } else if (tiles(64, 64) <= 64) {
        if (tiles(32, 16) <= 128) launch_few<T, int8_t, 1, 1>(g, s);
        else if (g.M <= 32) launch_few<T, int8_t, 2, 1>(g, s);
        else launch_few<T, int8_t, 2, 2>(g, s);
    } else if (tiles(64, 64) <= 256) {
        launch_tiles<T, I8Tile<2, 2, 1, 1, 4>, 1>(g, s);
    } else if (g.M <= 64 || tiles(64, 128) <= 256) {
        launch_tiles<T, I8Tile<2, 4, 1, 1, 3>, 2>(g, s);
    } else if (tiles(128, 128) <= 256) {
        launch_tiles<T, I8Tile<2, 4, 2, 1, 3>, 2>(g, s);
    } else if (tiles(128, 128) <= 512 || short_rows) {
        launch_tiles<T, I8Tile<2, 4, 2, 1, 2>, 4>(g, s);
    } else {
        launch_tiles<T, I8Tile<2, 4, 4, 2, 2>, 2>(g, s);
    }
}

// Float tokens that every work-group quantizes for itself, one launch instead
// of two (and nothing in the workspace): 16 tokens of a work-group as long as
// they fit its threads' registers, 32 KB.  One or two tokens always, more while
// the elements quantized by all work-groups together are 4 M at most (the
// calling thread 7.6 us instead of 10.2 then; GPU time in one / two launches,
// f32, bf16): 1x4096x2048 5.7 / 6.6, 1x151936x2048 51 / 55, 8x4096x1024 4.7 /
// 5.4, 4.0 / 5.0, 16x2048x512 4.6 / 4.9, 3.8 / 4.7, 64x2048x512 5.9 / 6.0, 4.7 /
// 5.9, 8x4096x2048 bf16 5.8 / 5.8; but 16x8192x1024 bf16 7.2 / 6.1, 32x8192x512
// 8.5 / 6.4, 6.7 / 6.1, 4x16384x2048 12.6 / 11.3.
static int few_elements(int ntok, int ncols) { return min(ntok, 16) * pad_to(ncols, I8_BK); }
static bool needs_no_workspace(int ntok, int ncols) { return ntok <= 2 && few_elements(ntok, ncols) <= 8192; }
static bool quantizes_itself(int type, int ntok, int nrows, int ncols) {
    if (needs_no_workspace(ntok, ncols)) return true;
    const int64_t groups = (int64_t)((ntok + 15) / 16) * ((nrows + 15) / 16), n = few_elements(ntok, ncols);
    return n <= (type == T_F32 ? 8192 : 16384) && groups * n <= 1 << 22 && (ntok <= 16 || groups <= 512);
}
template <typename T, typename X>
static void launch_few_quantizing(const I8Gemm& g, hipStream_t s) {
    if constexpr (sizeof(X) == 2)
        if (few_elements(g.M, g.C) > 8192) return launch_few<T, X, 1, 1, 32>(g, s);
    if (g.N <= FEW_N) launch_few<T, X, 1, 1>(g, s);
    else launch_few<T, X, 1, 2>(g, s);
}
template <typename T>
static void launch_few_quantizing(int type, const I8Gemm& g, hipStream_t s) {
    if (type == T_F32) launch_few_quantizing<T, float>(g, s);
    else if (type == T_F16) launch_few_quantizing<T, _Float16>(g, s);
    else launch_few_quantizing<T, __bf16>(g, s);
}

static void launch_gemm(int type, const I8Gemm& g, hipStream_t s) {
    if (type == T_F32) launch_gemm<float>(g, s);
    else if (type == T_F16) launch_gemm<_Float16>(g, s);
    else launch_gemm<__bf16>(g, s);
}

}  // namespace chimere

using namespace chimere;

extern "C" {

void chimere_quantize_i8(int type, const void* x, int64_t x_stride, int8_t* q, int64_t q_stride, float* scale,
                         int64_t nrows, int ncols, hipStream_t stream) {
    CHIMERE_REQUIRE(float_type(type), CHIMERE_ERR_ARG, "quantize_i8: unsupported type %d", type);
    CHIMERE_REQUIRE(nrows >= 0 && nrows <= 0x7FFFFFFF && ncols >= 1 && ncols <= I8_MAX_ROW, CHIMERE_ERR_ARG,
                    "quantize_i8: bad sizes nrows=%lld ncols=%d (at most %d)", (long long)nrows, ncols, I8_MAX_ROW);
    if (nrows == 0) return;
    CHIMERE_REQUIRE(x && q && scale, CHIMERE_ERR_ARG, "quantize_i8: null pointer");
    CHIMERE_REQUIRE(x_stride >= 0 && q_stride >= ncols, CHIMERE_ERR_ARG, "quantize_i8: bad strides %lld %lld",
                    (long long)x_stride, (long long)q_stride);
    CHIMERE_REQUIRE((((uintptr_t)q | (uintptr_t)q_stride) & 15) == 0 && ((uintptr_t)scale & 3) == 0 &&
                        float_aligned(type, x),
                    CHIMERE_ERR_ARG, "quantize_i8: rows of q must be 16-byte aligned, x and scale to their elements");
    launch_i8_quantize(type, x, x_stride, q, q_stride, scale, nrows, ncols, stream);
    check_launch("quantize_i8");
}

static bool gemm_args(const char* what, const int8_t* w, int64_t ldw, const float* ws, int out_type, const void* out,
                      int64_t ldo, int ntok, int nrows, int ncols) {
    if (!float_type(out_type)) {
        set_error(CHIMERE_ERR_ARG, "%s: unsupported output type %d", what, out_type);
    } else if (ntok < 0 || ntok > I8_MAX_ROWS || nrows < 1 || nrows > I8_MAX_ROWS || ncols < 1 || ncols > I8_MAX_C) {
        set_error(CHIMERE_ERR_ARG, "%s: bad sizes ntok=%d nrows=%d (at most %d) ncols=%d (at most %d)", what, ntok,
                  nrows, I8_MAX_ROWS, ncols, I8_MAX_C);
    } else if (ntok > 0 && !(w && ws && out)) {
        set_error(CHIMERE_ERR_ARG, "%s: null pointer", what);
    } else if (ldw < ncols || ldw > I8_MAX_STRIDE || ldo < nrows) {
        set_error(CHIMERE_ERR_ARG, "%s: bad strides w %lld out %lld", what, (long long)ldw, (long long)ldo);
    } else if ((((uintptr_t)w | (uintptr_t)ldw) & 15) || !float_aligned(out_type, out)) {
        set_error(CHIMERE_ERR_ARG, "%s: rows of 8-bit integers must be 16-byte aligned, out to its elements", what);
    } else if ((int64_t)ntok * nrows > I8_MAX_OUT) {
        set_error(CHIMERE_ERR_ARG, "%s: too many outputs (%d x %d)", what, ntok, nrows);
    } else {
        return true;
    }
    return false;
}

void chimere_gemm_i8(const int8_t* a, int64_t a_stride, const float* a_scale, const int8_t* w, int64_t w_stride,
                     const float* w_scale, const float* bias, int out_type, void* out, int64_t out_stride, int ntok,
                     int nrows, int ncols, hipStream_t stream) {
    if (!gemm_args("gemm_i8", w, w_stride, w_scale, out_type, out, out_stride, ntok, nrows, ncols) || ntok == 0) return;
    CHIMERE_REQUIRE(a && a_scale, CHIMERE_ERR_ARG, "gemm_i8: null pointer");
    CHIMERE_REQUIRE(a_stride >= ncols && a_stride <= I8_MAX_STRIDE, CHIMERE_ERR_ARG, "gemm_i8: bad stride %lld",
                    (long long)a_stride);
    CHIMERE_REQUIRE((((uintptr_t)a | (uintptr_t)a_stride) & 15) == 0, CHIMERE_ERR_ARG,
                    "gemm_i8: rows of 8-bit integers must be 16-byte aligned");
    launch_gemm(out_type, I8Gemm{a, w, a_scale, w_scale, bias, out, a_stride, w_stride, out_stride, ntok, nrows, ncols, nullptr, 0},
                stream);
    check_launch("gemm_i8");
}

size_t chimere_linear_i8_workspace_size(int max_ntok, int ncols) {
    if (max_ntok < 1 || ncols < 1 || ncols > I8_MAX_C || needs_no_workspace(max_ntok, ncols)) return 0;
    return al256((size_t)max_ntok * pad_to(ncols, 16)) + al256((size_t)max_ntok * 4);
}

void chimere_linear_i8(int type, const void* x, int64_t x_stride, const int8_t* w, int64_t w_stride,
                       const float* w_scale, const float* bias, int out_type, void* out, int64_t out_stride, int ntok,
                       int nrows, int ncols, void* workspace, size_t workspace_bytes, hipStream_t stream) {
    CHIMERE_REQUIRE(float_type(type), CHIMERE_ERR_ARG, "linear_i8: unsupported type %d", type);
    if (!gemm_args("linear_i8", w, w_stride, w_scale, out_type, out, out_stride, ntok, nrows, ncols) || ntok == 0) return;
    const size_t need = chimere_linear_i8_workspace_size(ntok, ncols);
    CHIMERE_REQUIRE(x && (workspace || !need), CHIMERE_ERR_ARG, "linear_i8: null pointer");
    CHIMERE_REQUIRE(x_stride >= 0 && float_aligned(type, x), CHIMERE_ERR_ARG,
                    "linear_i8: bad stride %lld, or x not aligned to its elements", (long long)x_stride);
    CHIMERE_REQUIRE(workspace_bytes >= need && ((uintptr_t)workspace & 255) == 0, CHIMERE_ERR_WORKSPACE,
                    "linear_i8: workspace %zu bytes < %zu (or not 256-byte aligned)", workspace_bytes, need);
    const int64_t lda = pad_to(ncols, 16);
    int8_t* q = (int8_t*)workspace;
    float* as = (float*)((uint8_t*)workspace + al256((size_t)ntok * lda));
    const I8Gemm g{q, w, as, w_scale, bias, out, lda, w_stride, out_stride, ntok, nrows, ncols, x, x_stride};
    if (quantizes_itself(type, ntok, nrows, ncols)) {
        if (out_type == T_F32) launch_few_quantizing<float>(type, g, stream);
        else if (out_type == T_F16) launch_few_quantizing<_Float16>(type, g, stream);
        else launch_few_quantizing<__bf16>(type, g, stream);
    } else {
        launch_i8_quantize(type, x, x_stride, q, lda, as, ntok, ncols, stream);
        if (!check_launch("linear_i8: quantizer")) return;   // no product of rows that were not written
        launch_gemm(out_type, g, stream);
    }
    check_launch("linear_i8");
}

}  // extern "C"
