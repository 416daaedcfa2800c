// balance.hip -- per-expert counts and the balance loss of a router's choice,
// and the gradient of its logits.  No counterpart in the reference.
#include "api_internal.h"
#include "float_rows.h"
#include "moe_common.h"

namespace chimere {

constexpr int BAL_COLS = MAX_E / 64;    // columns per lane

struct Balance {
    const int* ids;
    const uint8_t* mask;
    const int *counts, *tokens;
    const float* grad_loss;
    int64_t ld, ldg;
    int E, K, T, groups;
    float* psum;     // [groups][E]
    int *pcnt, *pn;  // [groups][E], [groups]
    float *loss, *probs;
    int *counts_out, *tokens_out;
};

__device__ __forceinline__ float wave_sum(float v) {
    v += xlane<32>(v);
    v += xlane<16>(v);
    v += xlane<8>(v);
    v += xlane<4>(v);
    v += xlane<2>(v);
    return v + xlane<1>(v);
}
__device__ __forceinline__ float wave_max(float v) {
    v = __builtin_fmaxf(v, xlane<32>(v));
    v = __builtin_fmaxf(v, xlane<16>(v));
    v = __builtin_fmaxf(v, xlane<8>(v));
    v = __builtin_fmaxf(v, xlane<4>(v));
    v = __builtin_fmaxf(v, xlane<2>(v));
    return __builtin_fmaxf(v, xlane<1>(v));
}

// softmax of one row by one wave (lane l: columns l, l + 64, ...); a row of
// -inf alone has no probabilities: zeros
template <typename T>
__device__ __forceinline__ void softmax_row(const T* row, int E, float (&p)[BAL_COLS]) {
    const int lane = threadIdx.x & 63;
    float m = -__builtin_huge_valf();
#pragma unroll
    for (int i = 0; i < BAL_COLS; i++) {
        p[i] = lane + 64 * i < E ? load_f(row + lane + 64 * i) : -__builtin_huge_valf();
        m = __builtin_fmaxf(m, p[i]);
    }
    m = wave_max(m);
    float s = 0.0f;
    bool nan = false;
#pragma unroll
    for (int i = 0; i < BAL_COLS; i++) nan |= p[i] != p[i];
    const bool none = m == -__builtin_huge_valf() && !__any(nan);
#pragma unroll
    for (int i = 0; i < BAL_COLS; i++) {
        p[i] = lane + 64 * i < E && !none ? det_exp(p[i] - m) : 0.0f;
        s += p[i];
    }
    s = wave_sum(s);
    const float r = none ? 0.0f : 1.0f / s;
#pragma unroll
    for (int i = 0; i < BAL_COLS; i++) p[i] *= r;
}

template <typename T>
__global__ __launch_bounds__(256) void k_balance_sums(Balance b, const T* __restrict__ logits) {
    __shared__ float part[4][MAX_E];
    __shared__ int cnt[MAX_E], n;
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    for (int e = tid; e < b.E; e += 256) cnt[e] = 0;
    if (tid == 0) n = 0;
    __syncthreads();
    float sum[BAL_COLS] = {};
    int rows = 0;
    for (int t = blockIdx.x * 4 + wave; t < b.T; t += b.groups * 4) {
        if (b.mask && !b.mask[t]) continue;
        rows++;
        float p[BAL_COLS];
        softmax_row(logits + t * b.ld, b.E, p);
#pragma unroll
        for (int i = 0; i < BAL_COLS; i++) sum[i] += p[i];
        for (int k = lane; k < b.K; k += 64) {
            const int e = b.ids[(int64_t)t * b.K + k];
            if ((unsigned)e < (unsigned)b.E) atomicAdd(&cnt[e], 1);
        }
    }
#pragma unroll
    for (int i = 0; i < BAL_COLS; i++) part[wave][lane + 64 * i] = sum[i];
    if (lane == 0) atomicAdd(&n, rows);
    __syncthreads();
    for (int e = tid; e < b.E; e += 256) {
        b.psum[(int64_t)blockIdx.x * b.E + e] = (part[0][e] + part[1][e]) + (part[2][e] + part[3][e]);
        b.pcnt[(int64_t)blockIdx.x * b.E + e] = cnt[e];
    }
    if (tid == 0) b.pn[blockIdx.x] = n;
}

__global__ __launch_bounds__(1024) void k_balance_loss(Balance b) {
    __shared__ float part[16];
    __shared__ int n;
    const int e = threadIdx.x;
    if (e == 0) {
        n = 0;
        for (int g = 0; g < b.groups; g++) n += b.pn[g];
    }
    __syncthreads();
    float s = 0.0f;
    int c = 0;
    if (e < b.E) {
        for (int g = 0; g < b.groups; g++) {
            s += b.psum[(int64_t)g * b.E + e];
            c += b.pcnt[(int64_t)g * b.E + e];
        }
        s = n ? s / (float)n : 0.0f;
        b.probs[e] = s;
        b.counts_out[e] = c;
    }
    const float l = wave_sum(n ? (float)c / ((float)n * (float)b.K) * s : 0.0f);
    if ((e & 63) == 0) part[e >> 6] = l;
    __syncthreads();
    if (e == 0) {
        float v = 0.0f;
        for (int i = 0; i < 16; i++) v += part[i];
        *b.loss = (float)b.E * v;
        *b.tokens_out = n;
    }
}

template <typename T>
__global__ __launch_bounds__(256) void k_balance_grad(Balance b, const T* __restrict__ logits, T* __restrict__ grad) {
    const int lane = threadIdx.x & 63;
    const int n = *b.tokens;
    const float all = n ? 1.0f / ((float)n * (float)b.K) : 0.0f;
    const float c = n ? *b.grad_loss * (float)b.E / (float)n : 0.0f;
    float f[BAL_COLS];
#pragma unroll
    for (int i = 0; i < BAL_COLS; i++) f[i] = lane + 64 * i < b.E ? (float)b.counts[lane + 64 * i] * all : 0.0f;
    for (int t = blockIdx.x * 4 + (threadIdx.x >> 6); t < b.T; t += gridDim.x * 4) {
        float p[BAL_COLS] = {}, d = 0.0f;
        if (!b.mask || b.mask[t]) softmax_row(logits + t * b.ld, b.E, p);
#pragma unroll
        for (int i = 0; i < BAL_COLS; i++) d = __builtin_fmaf(f[i], p[i], d);
        d = wave_sum(d);
#pragma unroll
        for (int i = 0; i < BAL_COLS; i++)
            if (lane + 64 * i < b.E) store_f(grad + t * b.ldg + lane + 64 * i, c * p[i] * (f[i] - d));
    }
}

static int balance_groups(int T) { return T < 1024 ? (T + 3) / 4 : 256; }

}  // namespace chimere

using namespace chimere;

extern "C" {

size_t chimere_balance_loss_workspace_size(int n_experts, int max_ntok) {
    if (n_experts < 1 || n_experts > MAX_E || max_ntok < 0) return 0;
    const size_t g = balance_groups(max_ntok) + 1;
    return 2 * al256(g * n_experts * 4) + al256(g * 4);
}

static bool balance_args(const char* what, int type, const void* logits, int64_t ld, int E, int K, int T) {
    if (!float_type(type))
        set_error(CHIMERE_ERR_ARG, "%s: unsupported type %d", what, type);
    else if (E < 1 || E > MAX_E || K < 1 || T < 0)
        set_error(CHIMERE_ERR_ARG, "%s: n_experts=%d top_k=%d ntok=%d out of range", what, E, K, T);
    else if (T > 0 && (!logits || ld < 0))
        set_error(CHIMERE_ERR_ARG, "%s: null pointer or bad stride", what);
    else
        return true;
    return false;
}

void chimere_balance_loss(int type, const void* logits, int64_t logits_stride, const int* ids, int top_k,
                          const uint8_t* mask, float* loss, float* probs, int* counts, int* tokens, int n_experts,
                          int ntok, void* workspace, size_t workspace_bytes, hipStream_t stream) {
    if (!balance_args("balance_loss", type, logits, logits_stride, n_experts, top_k, ntok)) return;
    CHIMERE_REQUIRE(loss && probs && counts && tokens && workspace && (ids || ntok == 0), CHIMERE_ERR_ARG,
                    "balance_loss: null pointer");
    const size_t need = chimere_balance_loss_workspace_size(n_experts, ntok);
    CHIMERE_REQUIRE(workspace_bytes >= need && ((uintptr_t)workspace & 255) == 0, CHIMERE_ERR_WORKSPACE,
                    "balance_loss: workspace %zu bytes < %zu (or not 256-byte aligned)", workspace_bytes, need);
    Balance b{};
    b.ids = ids; b.mask = mask; b.ld = logits_stride;
    b.E = n_experts; b.K = top_k; b.T = ntok; b.groups = balance_groups(ntok);
    uint8_t* w = (uint8_t*)workspace;
    const size_t one = al256((size_t)(b.groups + 1) * n_experts * 4);
    b.psum = (float*)w; b.pcnt = (int*)(w + one); b.pn = (int*)(w + 2 * one);
    b.loss = loss; b.probs = probs; b.counts_out = counts; b.tokens_out = tokens;
    if (b.groups) {
        if (type == T_F32)
            hipLaunchKernelGGL(k_balance_sums<float>, dim3(b.groups), dim3(256), 0, stream, b, (const float*)logits);
        else if (type == T_F16)
            hipLaunchKernelGGL(k_balance_sums<_Float16>, dim3(b.groups), dim3(256), 0, stream, b, (const _Float16*)logits);
        else
            hipLaunchKernelGGL(k_balance_sums<__bf16>, dim3(b.groups), dim3(256), 0, stream, b, (const __bf16*)logits);
    }
    hipLaunchKernelGGL(k_balance_loss, dim3(1), dim3(1024), 0, stream, b);
    check_launch("balance_loss");
}

void chimere_balance_loss_grad(int type, const void* logits, int64_t logits_stride, const uint8_t* mask,
                               const int* counts, const int* tokens, const float* grad_loss, int top_k, void* grad,
                               int64_t grad_stride, int n_experts, int ntok, hipStream_t stream) {
    if (!balance_args("balance_loss_grad", type, logits, logits_stride, n_experts, top_k, ntok) || ntok == 0) return;
    CHIMERE_REQUIRE(counts && tokens && grad_loss && grad && grad_stride >= n_experts, CHIMERE_ERR_ARG,
                    "balance_loss_grad: null pointer or bad stride");
    Balance b{};
    b.mask = mask; b.counts = counts; b.tokens = tokens; b.grad_loss = grad_loss;
    b.ld = logits_stride; b.ldg = grad_stride; b.E = n_experts; b.K = top_k; b.T = ntok;
    const dim3 grid(ntok < 8192 ? (ntok + 3) / 4 : 2048);
    if (type == T_F32)
        hipLaunchKernelGGL(k_balance_grad<float>, grid, dim3(256), 0, stream, b, (const float*)logits, (float*)grad);
    else if (type == T_F16)
        hipLaunchKernelGGL(k_balance_grad<_Float16>, grid, dim3(256), 0, stream, b, (const _Float16*)logits, (_Float16*)grad);
    else
        hipLaunchKernelGGL(k_balance_grad<__bf16>, grid, dim3(256), 0, stream, b, (const __bf16*)logits, (__bf16*)grad);
    check_launch("balance_loss_grad");
}

}  // extern "C"
