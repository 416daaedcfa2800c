// norm.h -- root-mean-square norm of rows with the residual's addition before
// it, an output in floats or in 8 bits with a scale per row, and the gradient.
//
// h = x + residual, y = h w / sqrt(mean h^2 + eps).  A row stays in registers
// between its sum and its output: it is read once and written once, and bytes
// bound all of it from a few hundred rows on (2^25 bf16 elements with a residual
// and h, 268 MB, part of it still in the last-level cache: 42 to 46 us at 512 to
// 16384 columns, 5.8 to 6.4 TB/s; 1 to 512 rows of 512: 2.9 us).  What is read
// is held in its own type until it is used, which leaves registers for more
// waves.
#pragma once
#include <type_traits>

#include "float_rows.h"

namespace chimere {

struct Norm {
    const void *x, *res, *w;
    void *h, *out;     // h: the sum, in the residual's type, or null
    float* scale;
    int64_t xs, rs, hs, os;
    double eps;
    int wtype, otype, rows, cols;
};
struct NormGrad {
    const void *h, *gy, *gh, *w;
    void* gx;
    float* part;       // [groups][pitch]: gradient of the weight, work-group by work-group; or null
    int64_t hs, ys, gs, xs;
    double eps;
    int wtype, rows, cols, pitch;
};

// Rows of up to 64 WAVES EL columns: lane l of a row's WAVES waves holds the
// columns i STEP + V l .. + V - 1 for i < N, in accesses of 16 bytes.
template <typename T, int WAVES, int EL>
struct NormRow {
    static constexpr int V = 16 / sizeof(T), N = EL / V, STEP = 64 * WAVES * V;
    static constexpr int THREADS = WAVES == 16 ? 1024 : 256, ROWS = THREADS / 64 / WAVES;
    static __device__ __forceinline__ int col() { return (threadIdx.x & (64 * WAVES - 1)) * V; }
    static __device__ __forceinline__ int row() { return threadIdx.x / (64 * WAVES); }
};

// V elements of a row at column c, 0 behind its end
template <int V, typename T>
__device__ __forceinline__ void norm_load(const T* row, int c, int cols, float (&v)[V]) {
    typedef typename VecOf<T, V>::type vec;
    if (c + V <= cols) {
        const vec x = *(const vec*)(row + c);
#pragma unroll
        for (int k = 0; k < V; k++) v[k] = (float)x[k];
    } else {
#pragma unroll
        for (int k = 0; k < V; k++) v[k] = c + k < cols ? load_f(row + c + k) : 0.0f;
    }
}
// as they are, for a kernel that holds several rows' elements
template <int V, typename T>
__device__ __forceinline__ void norm_load(const T* row, int c, int cols, typename VecOf<T, V>::type& v) {
    if (c + V <= cols) {
        v = *(const typename VecOf<T, V>::type*)(row + c);
    } else {
#pragma unroll
        for (int k = 0; k < V; k++) v[k] = c + k < cols ? row[c + k] : (T)0.0f;
    }
}
// the same of a type known at run time (a branch that the whole wave takes); 1 where there is no weight
template <int V>
__device__ __forceinline__ void norm_weight(const void* w, int type, int c, int cols, float (&v)[V]) {
    if (!w) {
#pragma unroll
        for (int k = 0; k < V; k++) v[k] = 1.0f;
    } else if (type == T_F32) norm_load((const float*)w, c, cols, v);
    else if (type == T_F16) norm_load((const _Float16*)w, c, cols, v);
    else norm_load((const __bf16*)w, c, cols, v);
}
template <int V>
__device__ __forceinline__ void norm_store(void* row, int type, int c, int cols, const float (&v)[V]) {
    if (type == T_F32) store_row((float*)row + c, v, cols - c);
    else if (type == T_F16) store_row((_Float16*)row + c, v, cols - c);
    else store_row((__bf16*)row + c, v, cols - c);
}
__host__ __device__ inline int64_t type_bytes(int type) { return type == T_F32 ? 4 : 2; }

// A row's two values joined over its WAVES waves, the same in every lane.
// `part`: [2][THREADS / 64] of this row; one row after another they take turns
// with two of them, so one barrier per row is enough.
template <int WAVES, typename A, typename B, typename F, typename G>
__device__ __forceinline__ void norm_join(A& a, B& b, A* pa, B* pb, F f, G g) {
    a = wave_join(a, f);
    b = wave_join(b, g);
    if constexpr (WAVES > 1) {
        const int wave = threadIdx.x >> 6, first = wave & ~(WAVES - 1);
        if ((threadIdx.x & 63) == 0) {
            pa[wave] = a;
            pb[wave] = b;
        }
        __syncthreads();
        a = pa[first];
        b = pb[first];
#pragma unroll
        for (int i = 1; i < WAVES; i++) {
            a = f(a, pa[first + i]);
            b = g(b, pb[first + i]);
        }
    }
}
// the larger by its bits without the sign: a NaN above an infinity above any number
__device__ __forceinline__ double norm_amax(double a, double b) {
    return __builtin_bit_cast(uint64_t, a) > __builtin_bit_cast(uint64_t, b) ? a : b;
}

// What makes y of a row's sums (64 bits): y = h w `by`, in 8 bits y / scale = h w `to`.
struct NormScale {
    double by, to;
    float scale;
    bool ok;
    __device__ __forceinline__ NormScale(double ss, double top, int cols, double eps) {
        by = 1.0 / __builtin_sqrt(ss / (double)cols + eps);
        scale = (float)(top * by / 127.0);
        ok = scale > 0.0f && scale < __builtin_huge_valf();
        to = ok ? by / (double)scale : 0.0;
    }
    // V integers of h w at column c of a row
    template <int V>
    __device__ __forceinline__ void store(int8_t* q, int c, int cols, const double (&hw)[V]) const {
        uint32_t p[V / 4];
#pragma unroll
        for (int j = 0; j < V / 4; j++) {
            p[j] = 0;
#pragma unroll
            for (int k = 0; k < 4; k++) {
                // (held to 127: a subnormal scale can be rounded down by up to a third)
                const int b = max(-127, min(127, (int)__builtin_rint(hw[4 * j + k] * to)));
                p[j] |= (uint32_t)(b & 255) << (8 * k);
            }
            if (!ok) p[j] = 0;
        }
        if (c + V <= cols) {
            typedef uint32_t words __attribute__((ext_vector_type(V / 4), aligned(4)));
            words o;
#pragma unroll
            for (int j = 0; j < V / 4; j++) o[j] = p[j];
            *(words*)(q + c) = o;
        } else {
#pragma unroll
            for (int k = 0; k < V; k++)
                if (c + k < cols) q[c + k] = (int8_t)(p[k / 4] >> (8 * (k & 3)));
        }
    }
};
__device__ __forceinline__ float norm_by(float ss, int cols, double eps) {
    return 1.0f / __builtin_sqrtf(ss / (float)cols + (float)eps);
}

// RES: no residual, one of x's type, one of f32.  In 8 bits a row is worked on
// in 64 bits up to its integers: one that is next to a border is then the
// formula's, not that of the last places of a 32-bit sum.  It costs little
// at the bytes' rate: 235 MB of 2^25 elements in 47 us (rows of 2048 columns, 5
// TB/s), 44 (4096), 62 (8192), 47 (16384); 256 rows of 4096 4.8 us.
template <typename T, int RES, bool I8, int WAVES, int EL>
__global__ __launch_bounds__((NormRow<T, WAVES, EL>::THREADS)) void k_rms_norm(Norm n) {
    typedef NormRow<T, WAVES, EL> Row;
    constexpr int V = Row::V, N = Row::N;
    typedef std::conditional_t<I8, double, float> Wide;
    typedef std::conditional_t<RES == 2, float, T> R;
    __shared__ Wide part[2][2][Row::THREADS / 64];
    const int c0 = Row::col(), cols = n.cols;
    float w[N][V];
#pragma unroll
    for (int i = 0; i < N; i++) norm_weight(n.w, n.wtype, c0 + i * Row::STEP, cols, w[i]);
    const int64_t step = (int64_t)gridDim.x * Row::ROWS;
    // the next row is on its way while 16 waves join the sums of this one (8192 columns: 48 -> 43 us, 8 bits 66 -> 62)
    constexpr bool AHEAD = WAVES == 16 && (EL == 8 || (I8 && sizeof(T) == 2));
    typename VecOf<T, V>::type x[N];
    typename VecOf<R, V>::type u[N];
    auto fetch = [&](int64_t r) {
#pragma unroll
        for (int i = 0; i < N; i++) norm_load<V>((const T*)n.x + r * n.xs, c0 + i * Row::STEP, cols, x[i]);
        if constexpr (RES != 0)
#pragma unroll
            for (int i = 0; i < N; i++) norm_load<V>((const R*)n.res + r * n.rs, c0 + i * Row::STEP, cols, u[i]);
    };
    if (AHEAD && (int64_t)blockIdx.x < n.rows) fetch(blockIdx.x);
    int turn = 0;
    for (int64_t r0 = (int64_t)blockIdx.x * Row::ROWS; r0 < n.rows; r0 += step, turn ^= 1) {
        const int64_t r = r0 + Row::row();
        if (WAVES == 1 && r >= n.rows) return;   // no barrier follows; elsewhere a work-group has one row
        Wide h[N][V], ss = 0, top = 0;
        float v[N][V];
        if (!AHEAD) fetch(r);
#pragma unroll
        for (int i = 0; i < N; i++)
#pragma unroll
            for (int k = 0; k < V; k++) h[i][k] = RES != 0 ? (Wide)(float)x[i][k] + (Wide)(float)u[i][k] : (Wide)(float)x[i][k];
        if (AHEAD && r0 + step < n.rows) fetch(r0 + step);
#pragma unroll
        for (int i = 0; i < N; i++) {
#pragma unroll
            for (int k = 0; k < V; k++) v[i][k] = (float)h[i][k];
            if constexpr (RES != 0)
                if (n.h) store_row((R*)n.h + r * n.hs + c0 + i * Row::STEP, v[i], cols - c0 - i * Row::STEP);
#pragma unroll
            for (int k = 0; k < V; k++) {
                if constexpr (I8) {
                    ss = __builtin_fma(h[i][k], h[i][k], ss);
                    h[i][k] *= (double)w[i][k];
                    top = norm_amax(top, __builtin_fabs(h[i][k]));
                } else {
                    ss = __builtin_fmaf(h[i][k], h[i][k], ss);
                }
            }
        }
        if constexpr (I8) {
            norm_join<WAVES>(ss, top, part[turn][0], part[turn][1], [](double a, double b) { return a + b; }, norm_amax);
            const NormScale by(ss, top, cols, n.eps);
            if (c0 == 0) n.scale[r] = by.scale;
#pragma unroll
            for (int i = 0; i < N; i++)
                if (c0 + i * Row::STEP < cols) by.store((int8_t*)n.out + r * n.os, c0 + i * Row::STEP, cols, h[i]);
        } else {
            auto add = [](float a, float b) { return a + b; };
            norm_join<WAVES>(ss, top, part[turn][0], part[turn][1], add, add);
            const float by = norm_by(ss, cols, n.eps);
            uint8_t* out = (uint8_t*)n.out + r * n.os * type_bytes(n.otype);
#pragma unroll
            for (int i = 0; i < N; i++) {
#pragma unroll
                for (int k = 0; k < V; k++) v[i][k] = v[i][k] * by * w[i][k];
                norm_store(out, n.otype, c0 + i * Row::STEP, cols, v[i]);
            }
        }
    }
}

// Rows that do not fit a work-group's registers: read twice, the second time
// from L2.  h is written in the second pass, by the lane that has read its
// place last, so that it may lie where the residual does.  (1024 rows of
// 32768 bf16 with residual: 69 us, in 8 bits 80; rows of 16384 this way 61 and
// 81 us, kept in registers 46 and 47.)
template <typename T, int RES, bool I8>
__global__ __launch_bounds__(1024) void k_rms_norm_long(Norm n) {
    typedef NormRow<T, 16, 16> Row;
    constexpr int V = Row::V;
    typedef std::conditional_t<I8, double, float> Wide;
    typedef std::conditional_t<RES == 2, float, T> R;
    __shared__ Wide part[2][2][16];
    const int cols = n.cols;
    int turn = 0;
    for (int64_t r = blockIdx.x; r < n.rows; r += gridDim.x, turn ^= 1) {
        auto load = [&](int c, Wide(&h)[V], float(&v)[V], float(&w)[V]) {
            norm_load((const T*)n.x + r * n.xs, c, cols, v);
            norm_weight(n.w, n.wtype, c, cols, w);
            float u[V] = {};
            if constexpr (RES != 0) norm_load((const R*)n.res + r * n.rs, c, cols, u);
#pragma unroll
            for (int k = 0; k < V; k++) {
                h[k] = RES != 0 ? (Wide)v[k] + (Wide)u[k] : (Wide)v[k];
                v[k] = (float)h[k];
            }
        };
        Wide ss = 0, top = 0, h[V];
        float v[V], w[V];
        for (int c = Row::col(); c < cols; c += Row::STEP) {
            load(c, h, v, w);
#pragma unroll
            for (int k = 0; k < V; k++) {
                if constexpr (I8) {
                    ss = __builtin_fma(h[k], h[k], ss);
                    top = norm_amax(top, __builtin_fabs(h[k] * (double)w[k]));
                } else {
                    ss = __builtin_fmaf(h[k], h[k], ss);
                }
            }
        }
        auto add = [](Wide a, Wide b) { return a + b; };
        auto larger = [](Wide a, Wide b) { return I8 ? (Wide)norm_amax(a, b) : a; };
        norm_join<16>(ss, top, part[turn][0], part[turn][1], add, larger);
        const NormScale eight(I8 ? ss : 1.0, top, cols, n.eps);
        const float by = I8 ? 0.0f : norm_by((float)ss, cols, n.eps);
        if (I8 && threadIdx.x == 0) n.scale[r] = eight.scale;
        for (int c = Row::col(); c < cols; c += Row::STEP) {
            load(c, h, v, w);
            if constexpr (RES != 0)
                if (n.h) store_row((R*)n.h + r * n.hs + c, v, cols - c);
            if constexpr (I8) {
#pragma unroll
                for (int k = 0; k < V; k++) h[k] *= (double)w[k];
                eight.store((int8_t*)n.out + r * n.os, c, cols, h);
            } else {
#pragma unroll
                for (int k = 0; k < V; k++) v[k] = v[k] * by * w[k];
                norm_store((uint8_t*)n.out + r * n.os * type_bytes(n.otype), n.otype, c, cols, v);
            }
        }
    }
}

// g = gy w, r = 1 / sqrt(mean h^2 + eps): gx = r (g - h r^2 mean(g h)) + gh and
// the weight's gradient, sum over rows of gy h r.  Nothing is kept from the
// forward pass but h: the sum of its squares is formed again with the other
// one.  A lane adds up its columns of the weight's gradient over the
// work-group's rows; the work-groups' sums are joined by k_norm_gw, all in a
// fixed order.  The rows' elements are held in their own types:
// as floats those of 16384 columns spill, and such rows, read twice, took 109
// us for 55.  Bytes bound it (2^25 bf16 elements with grad_h, 268 MB: rows of
// 2048 columns 50 us, 5.4 TB/s, and 4 for the join, 4096 48 + 4.5, 8192 52 +
// 4.5, 16384 54 + 7).
template <typename T, typename G, int WAVES, int EL>
__global__ __launch_bounds__((NormRow<T, WAVES, EL>::THREADS)) void k_rms_norm_grad(NormGrad n) {
    typedef NormRow<T, WAVES, EL> Row;
    constexpr int V = Row::V, N = Row::N;
    __shared__ float part[2][2][Row::THREADS / 64];
    const int c0 = Row::col(), cols = n.cols;
    float w[N][V], sum[N][V] = {};
#pragma unroll
    for (int i = 0; i < N; i++) norm_weight(n.w, n.wtype, c0 + i * Row::STEP, cols, w[i]);
    const int64_t step = (int64_t)gridDim.x * Row::ROWS;
    int turn = 0;
    for (int64_t r0 = (int64_t)blockIdx.x * Row::ROWS; r0 < n.rows; r0 += step, turn ^= 1) {
        const int64_t r = r0 + Row::row();
        if (WAVES == 1 && r >= n.rows) break;    // no barrier within the loop; elsewhere a work-group has one row
        typename VecOf<T, V>::type h[N], add[N];
        typename VecOf<G, V>::type g[N];
        float ss = 0.0f, gh = 0.0f;
#pragma unroll
        for (int i = 0; i < N; i++) norm_load<V>((const T*)n.h + r * n.hs, c0 + i * Row::STEP, cols, h[i]);
#pragma unroll
        for (int i = 0; i < N; i++) norm_load<V>((const G*)n.gy + r * n.ys, c0 + i * Row::STEP, cols, g[i]);
        if (n.gh)
#pragma unroll
            for (int i = 0; i < N; i++) norm_load<V>((const T*)n.gh + r * n.gs, c0 + i * Row::STEP, cols, add[i]);
#pragma unroll
        for (int i = 0; i < N; i++)
#pragma unroll
            for (int k = 0; k < V; k++) {
                const float x = (float)h[i][k];
                ss = __builtin_fmaf(x, x, ss);
                gh = __builtin_fmaf((float)g[i][k] * w[i][k], x, gh);
            }
        auto plus = [](float a, float b) { return a + b; };
        norm_join<WAVES>(ss, gh, part[turn][0], part[turn][1], plus, plus);
        const float by = norm_by(ss, cols, n.eps), mean = by * by * (gh / (float)cols);
        T* gx = (T*)n.gx + r * n.xs;
#pragma unroll
        for (int i = 0; i < N; i++) {
            float o[V];
#pragma unroll
            for (int k = 0; k < V; k++) {
                const float x = (float)h[i][k], y = (float)g[i][k];
                o[k] = by * __builtin_fmaf(-x, mean, y * w[i][k]);
                if (n.gh) o[k] += (float)add[i][k];
                sum[i][k] = __builtin_fmaf(y, x * by, sum[i][k]);
            }
            store_row(gx + c0 + i * Row::STEP, o, cols - c0 - i * Row::STEP);
        }
    }
    if (!n.part) return;
    float* to = n.part + (int64_t)blockIdx.x * n.pitch;
    if constexpr (Row::ROWS > 1) {       // the rows that the work-group has at a time
        __shared__ float join[Row::ROWS][64 * EL];
#pragma unroll
        for (int i = 0; i < N; i++)
#pragma unroll
            for (int k = 0; k < V; k++) join[Row::row()][c0 + i * Row::STEP + k] = sum[i][k];
        __syncthreads();
        for (int c = threadIdx.x; c < cols; c += Row::THREADS) {
            float s = 0.0f;
#pragma unroll
            for (int j = 0; j < Row::ROWS; j++) s += join[j][c];
            to[c] = s;
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; i++) store_row(to + c0 + i * Row::STEP, sum[i], cols - c0 - i * Row::STEP);
    }
}

// Rows past a work-group's registers: read twice, the weight's gradient added
// up where the work-group's sums lie, every column by one lane.  (1024 rows of
// 32768 bf16: 112 us and 12 for the join.)
template <typename T, typename G>
__global__ __launch_bounds__(1024) void k_rms_norm_grad_long(NormGrad n) {
    typedef NormRow<T, 16, 16> Row;
    constexpr int V = Row::V;
    __shared__ float part[2][2][16];
    const int cols = n.cols;
    float* sums = n.part ? n.part + (int64_t)blockIdx.x * n.pitch : nullptr;
    int turn = 0;
    for (int64_t r = blockIdx.x; r < n.rows; r += gridDim.x, turn ^= 1) {
        const T* hr = (const T*)n.h + r * n.hs;
        const G* gr = (const G*)n.gy + r * n.ys;
        float h[V], g[V], w[V], ss = 0.0f, gh = 0.0f;
        for (int c = Row::col(); c < cols; c += Row::STEP) {
            norm_load(hr, c, cols, h);
            norm_load(gr, c, cols, g);
            norm_weight(n.w, n.wtype, c, cols, w);
#pragma unroll
            for (int k = 0; k < V; k++) {
                ss = __builtin_fmaf(h[k], h[k], ss);
                gh = __builtin_fmaf(g[k] * w[k], h[k], gh);
            }
        }
        auto plus = [](float a, float b) { return a + b; };
        norm_join<16>(ss, gh, part[turn][0], part[turn][1], plus, plus);
        const float by = norm_by(ss, cols, n.eps), mean = by * by * (gh / (float)cols);
        for (int c = Row::col(); c < cols; c += Row::STEP) {
            float add[V] = {}, sum[V] = {}, o[V];
            norm_load(hr, c, cols, h);
            norm_load(gr, c, cols, g);
            norm_weight(n.w, n.wtype, c, cols, w);
            if (n.gh) norm_load((const T*)n.gh + r * n.gs, c, cols, add);
            if (sums && r != blockIdx.x) norm_load(sums, c, cols, sum);
#pragma unroll
            for (int k = 0; k < V; k++) {
                o[k] = by * __builtin_fmaf(-h[k], mean, g[k] * w[k]) + add[k];
                sum[k] = __builtin_fmaf(g[k], h[k] * by, sum[k]);
            }
            store_row((T*)n.gx + r * n.xs + c, o, cols - c);
            if (sums) store_row(sums + c, sum, cols - c);
        }
    }
}

// f(WAVES, EL) of rows of `cols` columns: the fewest waves that hold a row in
// 8 or 16 elements of a lane (2^25 bf16 elements, float output, 8 bits and
// gradient without its join in us.  1024 columns by one wave of 16: 44, 43, 47,
// by four of 8: 55, 82, 87; 2048 by four of 8: 41, 49, 49, by one of 32: 43, 46,
// 53; 4096 by four of 16: 43, 44, 49, by 16 of 8: 45, 107, 68; 8192 by 16 of 8:
// 43, 62, 52, by four of 32: 43, 50, 59.  2^24 f32 elements of 8192: 43, 41, 49
// and 43, 43, 53.  So 8-bit output of 16-bit rows alone goes better by four waves
// of 32, at 8192 columns.)  Up to 512 columns a wave has a row, below that with
// idle lanes: 128 columns 130, 164, 205.
constexpr int NORM_MAX_COLS = 1 << 20;
constexpr int NORM_LONG = 16384;        // columns that are kept in registers
template <typename T>
constexpr int NORM_GRAD_LONG = sizeof(T) == 2 ? 16384 : 8192;     // (three rows of f32 at 16384 spill)
template <typename F>
inline void norm_kind(int cols, F f) {
    std::integral_constant<int, 1> one;
    std::integral_constant<int, 4> four;
    std::integral_constant<int, 8> e8;
    std::integral_constant<int, 16> sixteen;
    if (cols <= 512) f(one, e8);
    else if (cols <= 1024) f(one, sixteen);
    else if (cols <= 2048) f(four, e8);
    else if (cols <= 4096) f(four, sixteen);
    else if (cols <= 8192) f(sixteen, e8);
    else f(sixteen, sixteen);
}
// Work-groups at most: no more than keep the memory busy, so that each loads its weights once for many rows (float output of
// 2^25 bf16 elements, rows of 2048 / 4096 / 8192 columns: 1024 work-groups 42 / 44 / 45 us, 512 51 / 42 / 43, 2048 43 / 44 / 46).
// In 8 bits short rows go better by more, which evens out what a row takes (2048 columns: 4096 work-groups 47 us, 1024 57), and
// of 16 waves one work-group fits a CU (16384 columns: 256 work-groups 47 us, 512 52).
constexpr int norm_groups(int waves, int el, bool i8) { return waves == 16 ? (i8 ? 256 : 512) : el == 8 && i8 ? 4096 : 1024; }
constexpr int NORM_LONG_GROUPS = 2048;

template <typename T, bool I8>
void launch_norm(const Norm& n, int res, hipStream_t s) {
    auto go = [&](auto plain, auto same, auto wide, int at_once, int threads, int most) {
        const int64_t groups = ((int64_t)n.rows + at_once - 1) / at_once;
        const dim3 grid((unsigned)(groups < most ? groups : most)), block(threads);
        if (res == 0) hipLaunchKernelGGL(plain, grid, block, 0, s, n);
        else if (res == 1) hipLaunchKernelGGL(same, grid, block, 0, s, n);
        else hipLaunchKernelGGL(wide, grid, block, 0, s, n);
    };
    constexpr int WIDE = std::is_same_v<T, float> ? 1 : 2;    // (f32 rows have no other residual)
    if (n.cols > NORM_LONG) {
        go(k_rms_norm_long<T, 0, I8>, k_rms_norm_long<T, 1, I8>, k_rms_norm_long<T, WIDE, I8>, 1, 1024, NORM_LONG_GROUPS);
        return;
    }
    norm_kind(n.cols, [&](auto waves, auto el) {
        constexpr int W = decltype(waves)::value, EL = decltype(el)::value;
        typedef NormRow<T, W, EL> Row;
        go(k_rms_norm<T, 0, I8, W, EL>, k_rms_norm<T, 1, I8, W, EL>, k_rms_norm<T, WIDE, I8, W, EL>, Row::ROWS, Row::THREADS,
           norm_groups(W, EL, I8));
    });
}
template <typename T, typename G>
void launch_norm_grad(const NormGrad& n, int groups, hipStream_t s) {
    if (n.cols > NORM_GRAD_LONG<T>) {
        hipLaunchKernelGGL((k_rms_norm_grad_long<T, G>), dim3(groups), dim3(1024), 0, s, n);
        return;
    }
    norm_kind(n.cols, [&](auto waves, auto el) {
        constexpr int W = decltype(waves)::value, EL = W == 16 && sizeof(T) == 4 ? 8 : decltype(el)::value;
        hipLaunchKernelGGL((k_rms_norm_grad<T, G, W, EL>), dim3(groups), dim3(NormRow<T, W, EL>::THREADS), 0, s, n);
    });
}
// The gradient's, of which each leaves its sums of a row's length: no more than keep the memory busy (2^25 bf16 elements, rows
// of 2048 / 4096 / 8192 columns, with the join: 1536 work-groups 57 / 62 / 78 us, 768 54 / 57 / 66, 512 58 / 53 / 61, 256 89 /
// 64 / 57)
inline int norm_grad_groups(int rows, int cols) {
    const int64_t at_once = cols <= 1024 ? 4 : 1, groups = ((int64_t)rows + at_once - 1) / at_once;
    const int64_t most = cols <= 512 || (cols > 1024 && cols <= 2048) ? 768 : cols <= 4096 ? 512 : cols <= 65536 ? 256 : 64;
    return (int)(groups < most ? groups : most);
}

// the kernels of one type of rows, compiled in a file of their own each
template <typename T> void norm_rows(const Norm& n, int res, bool i8, hipStream_t s);
template <typename T> void norm_grad_rows(const NormGrad& n, int gtype, int groups, hipStream_t s);

}  // namespace chimere
