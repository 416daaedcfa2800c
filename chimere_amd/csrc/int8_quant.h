// int8_quant.h -- rows of floats as 8-bit integers with one scale: scale =
// max |x| times 1/127 (its f32 value: what torch computes for a division by
// the number 127, so that rows quantized there have the same scales), q =
// x / scale (IEEE) rounded to the nearest integer, ties to even.
#pragma once
#include "float_rows.h"
#include "int8_slices.h"

namespace chimere {

// a row's scale from its max |x| as bits
__device__ __forceinline__ float i8_scale(uint32_t amax) {
    return __builtin_bit_cast(float, amax) * (1.0f / 127.0f);
}
// x / d as IEEE rounds it, with what a row's divisions share worked out once:
// from y = 1 / d (rounded to nearest) the product x y is off by two units in
// the last place at most, one correction q + (x - q d) y makes that less than
// one and a second the nearest (Markstein, "Computation of elementary functions
// on the IBM RISC System/6000 processor", 1990); the remainders are exact in an
// fma as long as nothing leaves f32's normal range, so rows of scale under 2^-90
// divide.  With the packing below 8 operations an element, where a division and
// conversions take about 20: rows of 512 bf16, 32768 of them, 14.4 -> 11.8 us,
// 4096 rows of 2048 8.4 -> 7.0.
struct I8Scale {
    float d, y;
    bool ok, near;
    __device__ __forceinline__ explicit I8Scale(float scale)
        : d(scale), y(1.0f / scale), ok(scale > 0.0f && scale < __builtin_huge_valf()), near(scale >= 0x1p-90f) {}
    __device__ __forceinline__ float quotient(float x) const {
        const float q = x * y, u = __builtin_fmaf(__builtin_fmaf(-q, d, x), y, q);
        return __builtin_fmaf(__builtin_fmaf(-u, d, x), y, u);
    }
    // The integer of a quotient in the low byte: the sum's unit is 1, so the
    // addition rounds to the nearest integer, ties to even.  Held to +-127: a
    // subnormal scale can be rounded down by up to a third.
    __device__ __forceinline__ uint32_t byte(float q) const {
        return __float_as_uint(__builtin_amdgcn_fmed3f(q, -127.0f, 127.0f) + 12582912.0f);
    }
};

// N integers packed into bytes; 0 where the scale is 0, infinite or NaN
template <int N>
__device__ __forceinline__ void i8_pack(const float (&x)[N], const I8Scale& s, uint32_t (&q)[N / 4]) {
    float u[N];
#pragma unroll
    for (int k = 0; k < N; k++) u[k] = s.quotient(x[k]);
    if (__builtin_expect(!s.near, 0))
#pragma unroll
        for (int k = 0; k < N; k++) u[k] = x[k] / s.d;
#pragma unroll
    for (int k = 0; k < N; k += 4) {
        const uint32_t lo = __builtin_amdgcn_perm(s.byte(u[k + 1]), s.byte(u[k]), 0x0c0c0400);
        const uint32_t hi = __builtin_amdgcn_perm(s.byte(u[k + 3]), s.byte(u[k + 2]), 0x04000c0c);
        q[k / 4] = s.ok ? lo | hi : 0;
    }
}

// Elements c .. c + V - 1 of a row as f32, those from ncols on 0
template <typename T, int V>
__device__ __forceinline__ void i8_load(const T* row, int c, int ncols, float (&x)[V]) {
    typedef typename VecOf<T, V>::type vec;
    if (c + V <= ncols) {
        const vec v = *(const vec*)(row + c);
#pragma unroll
        for (int k = 0; k < V; k++) x[k] = (float)v[k];
    } else {
#pragma unroll
        for (int k = 0; k < V; k++) x[k] = c + k < ncols ? load_f(row + c + k) : 0.0f;
    }
}

// max |x| as bits: a NaN is larger than an infinity, and both than any number
template <int V>
__device__ __forceinline__ uint32_t i8_amax(uint32_t m, const float (&x)[V]) {
#pragma unroll
    for (int k = 0; k < V; k++) m = max(m, __builtin_bit_cast(uint32_t, x[k]) & 0x7FFFFFFFu);
    return m;
}
__device__ __forceinline__ uint32_t wave_amax(uint32_t m) {
    m = max(m, (uint32_t)xlane<32>((int)m));
    m = max(m, (uint32_t)xlane<16>((int)m));
    m = max(m, (uint32_t)xlane<8>((int)m));
    m = max(m, (uint32_t)xlane<4>((int)m));
    m = max(m, (uint32_t)xlane<2>((int)m));
    return max(m, (uint32_t)xlane<1>((int)m));
}

// M rows of `cols` columns (a multiple of V) as integers in LDS, by all THREADS
// threads: pieces of V elements, row by row, KEEP elements of a thread at most
// in registers between the rows' maxima (through LDS atomics: any order gives
// the same) and the integers.  load(m, c, v) gives the elements c .. c + V - 1 of row m
// (0 behind its end); as[m] receives the scale, aq + m * lda the integers.
// M * cols <= THREADS * KEEP; a barrier follows the last write.
template <int THREADS, int KEEP, int V, typename Load>
__device__ __forceinline__ void i8_rows_to_lds(int M, int cols, int lda, float* as, uint8_t* aq, Load load,
                                               std::integral_constant<int, V>) {
    const int tid = threadIdx.x, per = cols / V, n = M * per;
    uint32_t* bits = (uint32_t*)as;
    for (int m = tid; m < M; m += THREADS) bits[m] = 0;
    __syncthreads();
    float v[KEEP / V][V];
#pragma unroll
    for (int i = 0; i < KEEP / V; i++) {
        const int at = tid + i * THREADS, m = min(at / per, M - 1);
        uint32_t top = 0;
        if (at < n) {
            load(m, (at - m * per) * V, v[i]);
            top = i8_amax(0u, v[i]);
        }
        if (__all(m == __builtin_amdgcn_readfirstlane(m))) {   // a wave within one row: one atomic
            top = wave_amax(top);
            if ((tid & 63) == 0) atomicMax(&bits[m], top);
        } else if (at < n) {
            atomicMax(&bits[m], top);
        }
    }
    __syncthreads();
    for (int m = tid; m < M; m += THREADS) as[m] = i8_scale(bits[m]);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < KEEP / V; i++) {
        const int at = tid + i * THREADS, m = min(at / per, M - 1);
        if (at < n) {
            uint32_t p[V / 4];
            i8_pack(v[i], I8Scale(as[m]), p);
#pragma unroll
            for (int k = 0; k < V / 4; k++) *(uint32_t*)(aq + m * lda + (at - m * per) * V + 4 * k) = p[k];
        }
    }
    __syncthreads();
}

template <typename T>
struct I8Rows {
    const T* x;
    int64_t xs;
    int8_t* q;
    int64_t qs;
    float* scale;
    const int* to;      // scale of row r at scale[to[r]], or null: scale[r]
    const int* count;   // rows, where the device has counted them, or null: nrows
    int64_t nrows;
    int ncols;
};

// The rows of work-group `group` of THREADS threads, W waves each: 16 elements
// of each lane stay in registers between the maximum and the integers; columns
// past those (1024 or 4096) are read twice.
template <typename T, int W, int THREADS>
__device__ __forceinline__ void i8_quantize_rows(const I8Rows<T>& g, int64_t group) {
    constexpr int V = 16 / sizeof(T), KEEP = 16 / V, STEP = 64 * W * V;
    __shared__ uint32_t part[THREADS / 64];
    const int wave = threadIdx.x >> 6;
    const int64_t r = group * (THREADS / 64 / W) + wave / W;
    const bool on = r < (g.count ? *g.count : g.nrows);
    if (W == 1 && !on) return;   // no barrier follows
    const T* row = g.x + (on ? r : 0) * g.xs;
    const int c0 = (threadIdx.x & (64 * W - 1)) * V, ncols = g.ncols;
    float v[KEEP][V];
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < KEEP; i++) {
        i8_load(row, c0 + i * STEP, ncols, v[i]);
        m = i8_amax(m, v[i]);
    }
    for (int c = c0 + KEEP * STEP; c < ncols; c += STEP) {
        float u[V];
        i8_load(row, c, ncols, u);
        m = i8_amax(m, u);
    }
    m = wave_amax(m);
    if constexpr (W == 4) {
        if ((threadIdx.x & 63) == 0) part[wave] = m;
        __syncthreads();
        const uint32_t* p = part + wave / 4 * 4;
        m = max(max(p[0], p[1]), max(p[2], p[3]));
        if (!on) return;
    }
    const float d = i8_scale(m);
    const I8Scale by(d);
    if (c0 == 0) g.scale[g.to ? g.to[r] : r] = d;
    int8_t* to = g.q + r * g.qs;
    auto put = [&](int c, const float(&u)[V]) {
        uint32_t p[V / 4];
        i8_pack(u, by, p);
        if (c + V <= ncols) {
            typedef uint32_t words __attribute__((ext_vector_type(V / 4)));
            words o;
#pragma unroll
            for (int k = 0; k < V / 4; k++) o[k] = p[k];
            *(words*)(to + c) = o;
        } else {
#pragma unroll
            for (int k = 0; k < V; k++)
                if (c + k < ncols) to[c + k] = (int8_t)(p[k / 4] >> (8 * (k & 3)));
        }
    };
#pragma unroll
    for (int i = 0; i < KEEP; i++)
        if (c0 + i * STEP < ncols) put(c0 + i * STEP, v[i]);
    for (int c = c0 + KEEP * STEP; c < ncols; c += STEP) {
        float u[V];
        i8_load(row, c, ncols, u);
        put(c, u);
    }
}

// rows of a float type (int8.hip)
void launch_i8_quantize(int type, const void* x, int64_t xs, int8_t* q, int64_t qs, float* scale, int64_t nrows,
                        int ncols, hipStream_t s);

}  // namespace chimere
