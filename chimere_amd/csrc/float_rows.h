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

__device__ __forceinline__ float load_f(const float* p) { return *p; }
__device__ __forceinline__ float load_f(const _Float16* p) { return (float)*p; }
__device__ __forceinline__ float load_f(const __bf16* p) { return (float)*p; }
__device__ __forceinline__ void store_f(float* p, float v) { *p = v; }
__device__ __forceinline__ void store_f(_Float16* p, float v) { *p = (_Float16)v; }
__device__ __forceinline__ void store_f(__bf16* p, float v) { *p = (__bf16)v; }

}  // namespace chimere
