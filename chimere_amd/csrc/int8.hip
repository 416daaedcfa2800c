// int8.hip -- rows in 8-bit integers with one scale each, and their product.
// No counterpart in the reference, whose dense products of a prompt run one
// token at a time through the block-quantized GEMV.
#include "api_internal.h"
#include "int8_gemm.h"

namespace chimere {

// Row quantizer: scale = max |x| / 127, q = x / scale rounded to the nearest
// integer, ties to even (IEEE divisions).  A row that holds an infinity or a
// NaN keeps it in the scale and 0 in its integers, so its products are NaN.
// One work-group per row, two passes over it.
template <typename T>
__global__ __launch_bounds__(256) void k_i8_quantize(const T* __restrict__ x, int64_t xs, int8_t* __restrict__ q,
                                                     int64_t qs, float* __restrict__ scale, int ncols) {
    __shared__ uint32_t part[4];
    const T* row = x + (int64_t)blockIdx.x * xs;
    // |x| as bits: a NaN is larger than an infinity, and both than any number
    uint32_t m = 0;
    for (int c = threadIdx.x; c < ncols; c += 256)
        m = max(m, __builtin_bit_cast(uint32_t, load_f(row + c)) & 0x7FFFFFFFu);
    m = max(m, (uint32_t)xlane<32>((int)m));
    m = max(m, (uint32_t)xlane<16>((int)m));
    m = max(m, (uint32_t)xlane<8>((int)m));
    m = max(m, (uint32_t)xlane<4>((int)m));
    m = max(m, (uint32_t)xlane<2>((int)m));
    m = max(m, (uint32_t)xlane<1>((int)m));
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = m;
    __syncthreads();
    m = max(max(part[0], part[1]), max(part[2], part[3]));
    const float d = __builtin_bit_cast(float, m) / 127.0f;
    const bool zero = m >= 0x7F800000u || d == 0.0f;
    for (int c = threadIdx.x; c < ncols; c += 256)
        q[(int64_t)blockIdx.x * qs + c] = zero ? 0 : (int8_t)(int)__builtin_rintf(load_f(row + c) / d);
    if (threadIdx.x == 0) scale[blockIdx.x] = d;
}

void launch_i8_quantize(int type, const void* x, int64_t xs, int8_t* q, int64_t qs, float* scale, int64_t nrows,
                        int ncols, hipStream_t s) {
    const dim3 grid((unsigned)nrows);
    if (type == T_F32)
        hipLaunchKernelGGL(k_i8_quantize<float>, grid, dim3(256), 0, s, (const float*)x, xs, q, qs, scale, ncols);
    else if (type == T_F16)
        hipLaunchKernelGGL(k_i8_quantize<_Float16>, grid, dim3(256), 0, s, (const _Float16*)x, xs, q, qs, scale, ncols);
    else
        hipLaunchKernelGGL(k_i8_quantize<__bf16>, grid, dim3(256), 0, s, (const __bf16*)x, xs, q, qs, scale, ncols);
}

struct I8Gemm {
    const int8_t *a, *w;
    const float *as, *ws, *bias;
    void* out;
    int64_t lda, ldw, ldo;
    int M, N, C;
};

template <typename T, typename Tile>
__global__ __launch_bounds__(64 * Tile::NW) void k_i8_gemm(I8Gemm g) {
    extern __shared__ __align__(16) uint8_t lds[];
    const int tm = (g.M + Tile::BM - 1) / Tile::BM;
    const int m0 = blockIdx.x % tm * Tile::BM, n0 = blockIdx.x / tm * Tile::BN;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint32_t aoff[Tile::PM], woff[Tile::PN];
#pragma unroll
    for (int p = 0; p < Tile::PM; p++)
        aoff[p] = (uint32_t)(min((wave * Tile::PM + p) * 8 + (lane >> 3), g.M - 1 - m0) * g.lda);
#pragma unroll
    for (int p = 0; p < Tile::PN; p++)
        woff[p] = (uint32_t)(min((wave * Tile::PN + p) * 8 + (lane >> 3), g.N - 1 - n0) * g.ldw);
    constexpr int MT = Tile::MTILES, NT = Tile::NTILES;
    v16i acc[MT][NT];
    const int8_t* w = g.w + n0 * g.ldw;
    Tile::run(g.a + m0 * g.lda, w, w, aoff, woff, g.C, lds, acc);
    const int wm = wave / Tile::WAVES_N, wn = wave % Tile::WAVES_N;
#pragma unroll
    for (int j = 0; j < NT; j++) {
        const int n = n0 + (wn * NT + j) * 32 + (lane & 31);
        if (n >= g.N) continue;
        const float s = g.ws[n], b = g.bias ? g.bias[n] : 0.0f;
#pragma unroll
        for (int i = 0; i < MT; i++)
#pragma unroll
            for (int v = 0; v < 16; v++) {
                const int m = m0 + (wm * MT + i) * 32 + Tile::reg_row(v);
                if (m < g.M) store_f((T*)g.out + m * g.ldo + n, (float)acc[i][j][v] * g.as[m] * s + b);
            }
    }
}

template <typename T>
static void launch_gemm(const I8Gemm& g, hipStream_t s) {
    typedef I8Tile<2, 2, 1, 1> Tile;
    const int64_t tiles = (int64_t)((g.M + Tile::BM - 1) / Tile::BM) * ((g.N + Tile::BN - 1) / Tile::BN);
    hipLaunchKernelGGL((k_i8_gemm<T, Tile>), dim3((unsigned)tiles), dim3(64 * Tile::NW), Tile::LDS, s, g);
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
    CHIMERE_REQUIRE(nrows >= 0 && nrows <= 0x7FFFFFFF && ncols >= 1, CHIMERE_ERR_ARG,
                    "quantize_i8: bad sizes nrows=%lld ncols=%d", (long long)nrows, ncols);
    if (nrows == 0) return;
    CHIMERE_REQUIRE(x && q && scale, CHIMERE_ERR_ARG, "quantize_i8: null pointer");
    CHIMERE_REQUIRE(x_stride >= 0 && q_stride >= ncols, CHIMERE_ERR_ARG, "quantize_i8: bad strides %lld %lld",
                    (long long)x_stride, (long long)q_stride);
    CHIMERE_REQUIRE((((uintptr_t)q | (uintptr_t)q_stride) & 15) == 0 && ((uintptr_t)scale & 3) == 0, CHIMERE_ERR_ARG,
                    "quantize_i8: rows of q must be 16-byte aligned");
    launch_i8_quantize(type, x, x_stride, q, q_stride, scale, nrows, ncols, stream);
    check_launch("quantize_i8");
}

static bool gemm_args(const char* what, const int8_t* w, int64_t ldw, const float* ws, int out_type, const void* out,
                      int64_t ldo, int ntok, int nrows, int ncols) {
    if (!float_type(out_type)) {
        set_error(CHIMERE_ERR_ARG, "%s: unsupported output type %d", what, out_type);
    } else if (ntok < 0 || nrows < 1 || ncols < 1 || ncols > I8_MAX_C) {
        set_error(CHIMERE_ERR_ARG, "%s: bad sizes ntok=%d nrows=%d ncols=%d (ncols at most %d)", what, ntok, nrows,
                  ncols, I8_MAX_C);
    } else if (ntok > 0 && !(w && ws && out)) {
        set_error(CHIMERE_ERR_ARG, "%s: null pointer", what);
    } else if (ldw < ncols || ldw > I8_MAX_STRIDE || ldo < nrows) {
        set_error(CHIMERE_ERR_ARG, "%s: bad strides w %lld out %lld", what, (long long)ldw, (long long)ldo);
    } else if (((uintptr_t)w | (uintptr_t)ldw) & 15) {
        set_error(CHIMERE_ERR_ARG, "%s: rows of 8-bit integers must be 16-byte aligned", what);
    } else if (((int64_t)ntok + 31) / 32 * (((int64_t)nrows + 15) / 16) > 0x7FFFFFFF) {
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
    launch_gemm(out_type, I8Gemm{a, w, a_scale, w_scale, bias, out, a_stride, w_stride, out_stride, ntok, nrows, ncols},
                stream);
    check_launch("gemm_i8");
}

size_t chimere_linear_i8_workspace_size(int max_ntok, int ncols) {
    if (max_ntok < 1 || ncols < 1 || ncols > I8_MAX_C) return 0;
    return al256((size_t)max_ntok * pad_to(ncols, 16)) + al256((size_t)max_ntok * 4);
}

void chimere_linear_i8(int type, const void* x, int64_t x_stride, const int8_t* w, int64_t w_stride,
                       const float* w_scale, const float* bias, int out_type, void* out, int64_t out_stride, int ntok,
                       int nrows, int ncols, void* workspace, size_t workspace_bytes, hipStream_t stream) {
    CHIMERE_REQUIRE(float_type(type), CHIMERE_ERR_ARG, "linear_i8: unsupported type %d", type);
    if (!gemm_args("linear_i8", w, w_stride, w_scale, out_type, out, out_stride, ntok, nrows, ncols) || ntok == 0) return;
    CHIMERE_REQUIRE(x && workspace, CHIMERE_ERR_ARG, "linear_i8: null pointer");
    CHIMERE_REQUIRE(x_stride >= 0, CHIMERE_ERR_ARG, "linear_i8: bad stride %lld", (long long)x_stride);
    const size_t need = chimere_linear_i8_workspace_size(ntok, ncols);
    CHIMERE_REQUIRE(workspace_bytes >= need && ((uintptr_t)workspace & 255) == 0, CHIMERE_ERR_WORKSPACE,
                    "linear_i8: workspace %zu bytes < %zu (or not 256-byte aligned)", workspace_bytes, need);
    const int64_t lda = pad_to(ncols, 16);
    int8_t* q = (int8_t*)workspace;
    float* as = (float*)((uint8_t*)workspace + al256((size_t)ntok * lda));
    launch_i8_quantize(type, x, x_stride, q, lda, as, ntok, ncols, stream);
    launch_gemm(out_type, I8Gemm{q, w, as, w_scale, bias, out, lda, w_stride, out_stride, ntok, nrows, ncols}, stream);
    check_launch("linear_i8");
}

}  // extern "C"
