// float_rows.h -- the float types of rows that callers hand in (ggml ids) and
// their loads and stores as f32 (stores round to nearest even).
#pragma once
#include "common.h"

namespace chimere {

enum : int { T_F32 = 0, T_F16 = 1, T_BF16 = 30 };

inline bool float_type(int t) { return t == T_F32 || t == T_F16 || t == T_BF16; }
// whether rows of a float type at p start on whole elements
inline bool float_aligned(int t, const void* p) { return ((uintptr_t)p & (t == T_F32 ? 3 : 1)) == 0; }
inline size_t al256(size_t n) { return (n + 255) & ~(size_t)255; }

// N elements in one access.  Rows start on any element (odd strides, slices):
// global memory takes vectors at any address, and where they are not a
// multiple of their size only lines that are crossed cost more (1987 rows of
// 8226 f32 outputs, tokens of 361 columns: 60 us element by element, 38 so).
template <typename T, int N>
struct VecOf {
    typedef T type __attribute__((ext_vector_type(N), aligned(sizeof(T))));
};

__device__ __forceinline__ float load_f(const float* p) { return *p; }
__device__ __forceinline__ float load_f(const _Float16* p) { return (float)*p; }
__device__ __forceinline__ float load_f(const __bf16* p) { return (float)*p; }
__device__ __forceinline__ void store_f(float* p, float v) { *p = v; }
__device__ __forceinline__ void store_f(_Float16* p, float v) { *p = (_Float16)v; }
__device__ __forceinline__ void store_f(__bf16* p, float v) { *p = (__bf16)v; }

// N values at p, of which the first `count` are inside the row
template <int N, typename T>
__device__ __forceinline__ void store_row(T* p, const float (&v)[N], int count) {
    typedef typename VecOf<T, N>::type vec;
    if (count >= N) {
        vec o;
#pragma unroll
        for (int k = 0; k < N; k++) o[k] = (T)v[k];
        *(vec*)p = o;
    } else {
#pragma unroll
        for (int k = 0; k < N; k++)
            if (k < count) store_f(p + k, v[k]);
    }
}

// e^x for x <= 88: 2^(x log2 e) by the hardware's exponential, with what the
// product x log2 e is off by (known exactly from the fma, log2 e in two parts)
// put right to first order: about 2 units in the last place, at half of
// det_exp's instructions, for sums that are bound by these.  Below e^-87 it
// comes to 0; a NaN stays one.
__device__ __forceinline__ float fast_exp(float x) {
    constexpr float HI = 0x1.715476p+0f, LO = 0x1.4ae0cp-26f, LN2 = 0x1.62e430p-1f;
    x = x < -120.0f ? -120.0f : x;   // (not a maximum: a NaN stays)
    const float t = x * HI, off = __builtin_fmaf(x, LO, __builtin_fmaf(x, HI, -t));
    const float e = __builtin_amdgcn_exp2f(t);
    return __builtin_fmaf(e, off * LN2, e);
}
// g / (1 + e^-g), the exponential of the device library (1 unit in the last
// place) and an IEEE division: its result is requantized, and an h that is off
// by a few units more moves integers (with the hardware's exponential and
// reciprocal 6e-5 of 4096 tokens' outputs, at 343 against 345 us).
__device__ __forceinline__ float silu(float g) { return g / (1.0f + expf(-g)); }

}  // namespace chimere
