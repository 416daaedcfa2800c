// int8_quant.h -- rows of floats as 8-bit integers with one scale: scale =
// max |x| / 127, q = x / scale rounded to the nearest integer, ties to even
// (IEEE divisions).
#pragma once
#include "float_rows.h"

namespace chimere {

// the integer of x in a row of scale d
__device__ __forceinline__ int i8_quant(float x, float d) {
    return d > 0.0f && d < __builtin_huge_valf() ? (int)__builtin_rintf(x / d) : 0;
}

// N integers packed into bytes
template <int N>
__device__ __forceinline__ void i8_pack(const float (&x)[N], float d, uint32_t (&q)[N / 4]) {
#pragma unroll
    for (int k = 0; k < N; k += 4)
        q[k / 4] = (uint32_t)(uint8_t)i8_quant(x[k], d) | (uint32_t)(uint8_t)i8_quant(x[k + 1], d) << 8 |
                   (uint32_t)(uint8_t)i8_quant(x[k + 2], d) << 16 | (uint32_t)(uint8_t)i8_quant(x[k + 3], d) << 24;
}

// Elements c .. c + V - 1 of a row as f32, one 16-byte load where `wide`; those
// from ncols on are 0
template <typename T, int V>
__device__ __forceinline__ void i8_load(const T* row, int c, int ncols, bool wide, float (&x)[V]) {
    typedef T vec __attribute__((ext_vector_type(V)));
    if (wide && c + V <= ncols) {
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
        if (M == 1) {
            top = wave_amax(top);
            if ((tid & 63) == 0) atomicMax(&bits[0], top);
        } else if (at < n) {
            atomicMax(&bits[m], top);
        }
    }
    __syncthreads();
    for (int m = tid; m < M; m += THREADS) as[m] = __builtin_bit_cast(float, bits[m]) / 127.0f;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < KEEP / V; i++) {
        const int at = tid + i * THREADS, m = min(at / per, M - 1);
        if (at < n) {
            uint32_t p[V / 4];
            i8_pack(v[i], as[m], p);
#pragma unroll
            for (int k = 0; k < V / 4; k++) *(uint32_t*)(aq + m * lda + (at - m * per) * V + 4 * k) = p[k];
        }
    }
    __syncthreads();
}

}  // namespace chimere
