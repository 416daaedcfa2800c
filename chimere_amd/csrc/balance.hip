// balance.hip -- per-expert counts and the balance loss of a router's choice,
// and the gradient of its logits.  No counterpart in the reference.
#include <type_traits>

#include "api_internal.h"
#include "float_rows.h"
#include "moe_common.h"

namespace chimere {

struct Balance {
    const int* ids;
    const uint8_t* mask;
    const int *counts, *tokens;
    const float* grad_loss;
    int64_t ld, ldg;
    int E, K, T, groups;
    float* psum;     // [groups][E]
    int *pcnt, *pn;  // [groups][E], [groups]
    float* lpart;    // parts of the loss, one per work-group of k_balance_loss
    int* done;       // how many of them have ended
    float *loss, *probs;
    int *counts_out, *tokens_out;
};

// LANES lanes per row, lane l of them the columns 4 LANES i + 4 l .. + 3 for
// i < NV.  Sixteen up to 512 columns: a row of 256 is four loads of 16 bytes
// per lane, and the sums over a row are four DPP steps for four rows at once;
// above, the whole wave, so that a lane keeps 16 values and as many sums.
template <int LANES, int NV>
struct BalRow {
    float v[4 * NV];
    static __device__ __forceinline__ int lane() { return threadIdx.x & (LANES - 1); }
    static __device__ __forceinline__ int col(int i) { return 4 * LANES * i + 4 * lane(); }
    static __device__ __forceinline__ float sum(float x) {
        x = slot_reduce16(x);
        if constexpr (LANES == 64) {
            x += xlane<16>(x);
            x += xlane<32>(x);
        }
        return x;
    }

    template <typename T>
    __device__ __forceinline__ void load(const T* row, int E) {
        typedef typename VecOf<T, 4>::type vec;
#pragma unroll
        for (int i = 0; i < NV; i++) {
            const int c = col(i);
            if (c + 4 <= E) {
                const vec x = *(const vec*)(row + c);
#pragma unroll
                for (int k = 0; k < 4; k++) v[4 * i + k] = (float)x[k];
            } else {
#pragma unroll
                for (int k = 0; k < 4; k++) v[4 * i + k] = c + k < E ? load_f(row + c + k) : -__builtin_huge_valf();
            }
        }
    }
    // softmax of the loaded row; one of -inf alone has no probabilities: zeros
    __device__ __forceinline__ void softmax() {
        float m = v[0];
#pragma unroll
        for (int i = 1; i < 4 * NV; i++) m = __builtin_fmaxf(m, v[i]);
        m = __builtin_fmaxf(m, xlane<8>(m));
        m = __builtin_fmaxf(m, xlane<4>(m));
        m = __builtin_fmaxf(m, xlane<2>(m));
        m = __builtin_fmaxf(m, xlane<1>(m));
        if constexpr (LANES == 64) {
            m = __builtin_fmaxf(m, xlane<16>(m));
            m = __builtin_fmaxf(m, xlane<32>(m));
        }
        // where all are -inf: 0 instead, so that every exponential is 0 (a NaN among them stays one)
        const float from = m == -__builtin_huge_valf() ? 0.0f : m;
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < NV; i++) {
#pragma unroll
            for (int k = 0; k < 4; k++) v[4 * i + k] = fast_exp(v[4 * i + k] - from);
            s += (v[4 * i] + v[4 * i + 1]) + (v[4 * i + 2] + v[4 * i + 3]);
        }
        s = sum(s);
        const float r = s == 0.0f ? 0.0f : 1.0f / s;
#pragma unroll
        for (int i = 0; i < 4 * NV; i++) v[i] *= r;
    }
};

// Columns past E hold exponentials of -inf: 0.

constexpr int BAL_THREADS = 1024;   // of a work-group of the sums

// Probabilities and pairs summed over the rows of each work-group (row t of
// round i: (i * groups + group) * 64 + ..), every sum in a fixed order: a lane
// over its rows, four rows of a wave, the waves.  Counts are integers: LDS
// atomics in any order.  With one work-group the results follow at once.
template <typename T, int LANES, int NV, bool ONE>
__global__ __launch_bounds__(BAL_THREADS) void k_balance_sums(Balance b, const T* __restrict__ logits) {
    constexpr int THREADS = BAL_THREADS, ROWS = THREADS / LANES, COLS = 4 * LANES * NV;
    __shared__ float part[THREADS / 64][COLS];
    __shared__ float lpart[THREADS / 64];
    __shared__ int cnt[COLS], n;
    const int tid = threadIdx.x, wave = tid >> 6;
    for (int e = tid; e < COLS; e += THREADS) cnt[e] = 0;
    if (tid == 0) n = 0;
    if (!ONE && blockIdx.x == 0 && tid == 0) *b.done = 0;   // for k_balance_loss, that follows
    __syncthreads();
    float sum[4 * NV] = {};
    int rows = 0;
    for (int t0 = blockIdx.x * ROWS; t0 < b.T; t0 += b.groups * ROWS) {
        const int t = t0 + tid / LANES;
        const bool on = t < b.T && (!b.mask || b.mask[t]);
        BalRow<LANES, NV> row;
        if (on) row.load(logits + t * b.ld, b.E);
        const int pairs = min(ROWS, b.T - t0) * b.K;
        const int* ids = b.ids + (int64_t)t0 * b.K;
        for (int p = tid; p < pairs; p += THREADS) {
            const int e = ids[p];
            if ((unsigned)e < (unsigned)b.E && (!b.mask || b.mask[t0 + p / b.K])) atomicAdd(&cnt[e], 1);
        }
        if (on) {
            row.softmax();
#pragma unroll
            for (int i = 0; i < 4 * NV; i++) sum[i] += row.v[i];
            rows += row.lane() == 0;
        }
    }
    if constexpr (LANES == 16) {
#pragma unroll
        for (int i = 0; i < 4 * NV; i++) {
            sum[i] += xlane<16>(sum[i]);
            sum[i] += xlane<32>(sum[i]);
        }
    }
    if ((tid & 63) < LANES)
#pragma unroll
        for (int i = 0; i < NV; i++)
            *(float4*)&part[wave][BalRow<LANES, NV>::col(i)] =
                make_float4(sum[4 * i], sum[4 * i + 1], sum[4 * i + 2], sum[4 * i + 3]);
    if (rows) atomicAdd(&n, rows);
    __syncthreads();
    auto psum = [&](int e) {
        float v = 0.0f;
#pragma unroll
        for (int w = 0; w < THREADS / 64; w++) v += part[w][e];
        return v;
    };
    if constexpr (ONE) {
        float l = 0.0f;
        for (int e = tid; e < b.E; e += THREADS) {
            const float p = n ? psum(e) / (float)n : 0.0f;
            b.probs[e] = p;
            b.counts_out[e] = cnt[e];
            l += n ? (float)cnt[e] / ((float)n * (float)b.K) * p : 0.0f;
        }
        l = slot_reduce16(l);
        l += xlane<16>(l);
        l += xlane<32>(l);
        if ((tid & 63) == 0) lpart[wave] = l;
        __syncthreads();
        if (tid == 0) {
            float v = 0.0f;
            for (int i = 0; i < THREADS / 64; i++) v += lpart[i];
            *b.loss = (float)b.E * v;
            *b.tokens_out = n;
        }
    } else {
        for (int e = tid; e < b.E; e += THREADS) {
            b.psum[(int64_t)blockIdx.x * b.E + e] = psum(e);
            b.pcnt[(int64_t)blockIdx.x * b.E + e] = cnt[e];
        }
        if (tid == 0) b.pn[blockIdx.x] = n;
    }
}

// The work-groups' sums joined, 32 experts per work-group by eight segments of
// them (one work-group for all experts read 256 x 256 sums in 7 us); the last
// work-group to end adds up the parts of the loss, in their order.
constexpr int BAL_JOIN = 32;
__global__ __launch_bounds__(256) void k_balance_loss(Balance b) {
    __shared__ float ps[256], part[MAX_E / BAL_JOIN];
    __shared__ int pc[256], n, last;
    const int tid = threadIdx.x, seg = tid / BAL_JOIN, e = blockIdx.x * BAL_JOIN + tid % BAL_JOIN;
    if (tid == 0) n = 0;
    __syncthreads();
    float s = 0.0f;
    int c = 0;
    if (e < b.E) {
#pragma unroll 8
        for (int g = seg; g < b.groups; g += 256 / BAL_JOIN) {
            s += b.psum[(int64_t)g * b.E + e];
            c += b.pcnt[(int64_t)g * b.E + e];
        }
    }
    ps[tid] = s;
    pc[tid] = c;
    for (int g = tid; g < b.groups; g += 256) atomicAdd(&n, b.pn[g]);
    __syncthreads();
    float l = 0.0f;
    if (tid < BAL_JOIN && e < b.E) {
#pragma unroll
        for (int i = 1; i < 256 / BAL_JOIN; i++) {
            s += ps[i * BAL_JOIN + tid];
            c += pc[i * BAL_JOIN + tid];
        }
        s = n ? s / (float)n : 0.0f;
        b.probs[e] = s;
        b.counts_out[e] = c;
        l = n ? (float)c / ((float)n * (float)b.K) * s : 0.0f;
    }
    l = slot_reduce16(l);
    l += xlane<16>(l);
    if (tid == 0) {
        // visible to the whole device before the count says so
        __hip_atomic_store(&b.lpart[blockIdx.x], l, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        last = __hip_atomic_fetch_add(b.done, 1, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT) == (int)gridDim.x - 1;
    }
    __syncthreads();
    if (!last) return;
    if (tid < gridDim.x) part[tid] = __hip_atomic_load(&b.lpart[tid], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    if (tid == 0) {
        float v = 0.0f;
        for (int i = 0; i < (int)gridDim.x; i++) v += part[i];
        *b.loss = (float)b.E * v;
        *b.tokens_out = n;
    }
}

template <typename T, int LANES, int NV>
__global__ __launch_bounds__(256) void k_balance_grad(Balance b, const T* __restrict__ logits, T* __restrict__ grad) {
    typedef BalRow<LANES, NV> Row;
    constexpr int ROWS = 256 / LANES;
    const int n = *b.tokens;
    const float all = n ? 1.0f / ((float)n * (float)b.K) : 0.0f;
    const float c = n ? *b.grad_loss * (float)b.E / (float)n : 0.0f;
    float f[4 * NV];
#pragma unroll
    for (int i = 0; i < NV; i++) {
        typedef typename VecOf<int, 4>::type vec;
        const int e = Row::col(i);
        vec x = {};
        if (e + 4 <= b.E) {
            x = *(const vec*)(b.counts + e);
        } else {
#pragma unroll
            for (int k = 0; k < 4; k++) x[k] = e + k < b.E ? b.counts[e + k] : 0;
        }
#pragma unroll
        for (int k = 0; k < 4; k++) f[4 * i + k] = (float)x[k] * all;
    }
    // the next round's row is loaded while this one's gradient is formed
    Row p, next;
    auto fetch = [&](int t, Row& r) {
        const bool on = t < b.T && (!b.mask || b.mask[t]);
        if (on) r.load(logits + t * b.ld, b.E);
        return on;
    };
    const int first = blockIdx.x * ROWS + threadIdx.x / LANES;
    bool on = fetch(first, p);
    for (int t = first; t < b.T; t += gridDim.x * ROWS) {
        const bool more = fetch(t + gridDim.x * ROWS, next);
        float d = 0.0f;
        if (on) {
            p.softmax();
#pragma unroll
            for (int i = 0; i < 4 * NV; i += 4)
                d += __builtin_fmaf(f[i], p.v[i], f[i + 1] * p.v[i + 1]) +
                     __builtin_fmaf(f[i + 2], p.v[i + 2], f[i + 3] * p.v[i + 3]);
            d = Row::sum(d);
        }
        T* to = grad + t * b.ldg;
#pragma unroll
        for (int i = 0; i < NV; i++) {
            const int e = Row::col(i);
            float o[4];
#pragma unroll
            for (int k = 0; k < 4; k++) o[k] = on ? c * p.v[4 * i + k] * (f[4 * i + k] - d) : 0.0f;
            store_row(to + e, o, b.E - e);
        }
        p = next;
        on = more;
    }
}

// Work-groups of the sums of T rows: one, that also finishes, up to BAL_ONE
// rounds of its rows.
constexpr int BAL_ONE = 4, BAL_GROUPS = 256, BAL_GRAD = 1024;
static int balance_groups(int T, int E) {
    const int rows = E > 512 ? 16 : 64, n = (T + rows - 1) / rows;
    return n <= BAL_ONE ? 1 : n < BAL_GROUPS ? n : BAL_GROUPS;
}

template <typename T, int LANES, int NV>
static void launch_balance(const Balance& b, const void* logits, hipStream_t s) {
    const dim3 block(BAL_THREADS);
    if (b.groups == 1) {
        hipLaunchKernelGGL((k_balance_sums<T, LANES, NV, true>), dim3(1), block, 0, s, b, (const T*)logits);
    } else {
        hipLaunchKernelGGL((k_balance_sums<T, LANES, NV, false>), dim3(b.groups), block, 0, s, b, (const T*)logits);
        hipLaunchKernelGGL(k_balance_loss, dim3((b.E + BAL_JOIN - 1) / BAL_JOIN), dim3(256), 0, s, b);
    }
}

template <typename T, int LANES, int NV>
static void launch_balance_grad(const Balance& b, const void* logits, void* grad, hipStream_t s) {
    const int rows = 256 / LANES, n = (b.T + rows - 1) / rows;
    hipLaunchKernelGGL((k_balance_grad<T, LANES, NV>), dim3(n < BAL_GRAD ? n : BAL_GRAD), dim3(256), 0, s, b,
                       (const T*)logits, (T*)grad);
}

// f(type of the rows, LANES, NV of E columns)
template <typename F>
static void balance_kind(int type, int E, F f) {
    auto width = [&](auto t) {
        std::integral_constant<int, 16> few;
        if (E <= 64) f(t, few, std::integral_constant<int, 1>{});
        else if (E <= 128) f(t, few, std::integral_constant<int, 2>{});
        else if (E <= 256) f(t, few, std::integral_constant<int, 4>{});
        else if (E <= 512) f(t, few, std::integral_constant<int, 8>{});
        else f(t, std::integral_constant<int, 64>{}, std::integral_constant<int, 4>{});
    };
    if (type == T_F32) width((float*)nullptr);
    else if (type == T_F16) width((_Float16*)nullptr);
    else width((__bf16*)nullptr);
}

}  // namespace chimere

using namespace chimere;

extern "C" {

size_t chimere_balance_loss_workspace_size(int n_experts, int max_ntok) {
    if (n_experts < 1 || n_experts > MAX_E || max_ntok < 0) return 0;
    const size_t g = balance_groups(max_ntok, n_experts);
    if (g == 1) return 0;
    return 2 * al256(g * n_experts * 4) + al256(g * 4) + 256;
}

static bool balance_args(const char* what, int type, const void* logits, int64_t ld, int E, int K, int T) {
    if (!float_type(type))
        set_error(CHIMERE_ERR_ARG, "%s: unsupported type %d", what, type);
    else if (E < 1 || E > MAX_E || K < 1 || K > MAX_E || T < 0 || (int64_t)T * K >= (1 << 30))
        set_error(CHIMERE_ERR_ARG, "%s: n_experts=%d top_k=%d ntok=%d out of range", what, E, K, T);
    else if (T > 0 && (!logits || ld < 0 || !float_aligned(type, logits)))
        set_error(CHIMERE_ERR_ARG, "%s: null or misaligned pointer, or bad stride", what);
    else
        return true;
    return false;
}

void chimere_balance_loss(int type, const void* logits, int64_t logits_stride, const int* ids, int top_k,
                          const uint8_t* mask, float* loss, float* probs, int* counts, int* tokens, int n_experts,
                          int ntok, void* workspace, size_t workspace_bytes, hipStream_t stream) {
    if (!balance_args("balance_loss", type, logits, logits_stride, n_experts, top_k, ntok)) return;
    const size_t need = chimere_balance_loss_workspace_size(n_experts, ntok);
    CHIMERE_REQUIRE(loss && probs && counts && tokens && (workspace || !need) && (ids || ntok == 0), CHIMERE_ERR_ARG,
                    "balance_loss: null pointer");
    CHIMERE_REQUIRE(workspace_bytes >= need && ((uintptr_t)workspace & 255) == 0, CHIMERE_ERR_WORKSPACE,
                    "balance_loss: workspace %zu bytes < %zu (or not 256-byte aligned)", workspace_bytes, need);
    Balance b{};
    b.ids = ids; b.mask = mask; b.ld = logits_stride;
    b.E = n_experts; b.K = top_k; b.T = ntok; b.groups = balance_groups(ntok, n_experts);
    uint8_t* w = (uint8_t*)workspace;
    const size_t one = al256((size_t)b.groups * n_experts * 4);
    b.psum = (float*)w; b.pcnt = (int*)(w + one); b.pn = (int*)(w + 2 * one);
    b.lpart = (float*)(w + 2 * one + al256((size_t)b.groups * 4));
    b.done = (int*)(b.lpart + MAX_E / BAL_JOIN);
    b.loss = loss; b.probs = probs; b.counts_out = counts; b.tokens_out = tokens;
    balance_kind(type, n_experts, [&](auto t, auto lanes, auto nv) {
        launch_balance<std::remove_pointer_t<decltype(t)>, decltype(lanes)::value, decltype(nv)::value>(b, logits, stream);
    });
    check_launch("balance_loss");
}

void chimere_balance_loss_grad(int type, const void* logits, int64_t logits_stride, const uint8_t* mask,
                               const int* counts, const int* tokens, const float* grad_loss, int top_k, void* grad,
                               int64_t grad_stride, int n_experts, int ntok, hipStream_t stream) {
    if (!balance_args("balance_loss_grad", type, logits, logits_stride, n_experts, top_k, ntok) || ntok == 0) return;
    CHIMERE_REQUIRE(counts && tokens && grad_loss && grad && grad_stride >= n_experts && float_aligned(type, grad),
                    CHIMERE_ERR_ARG, "balance_loss_grad: null or misaligned pointer, or bad stride");
    Balance b{};
    b.mask = mask; b.counts = counts; b.tokens = tokens; b.grad_loss = grad_loss;
    b.ld = logits_stride; b.ldg = grad_stride; b.E = n_experts; b.K = top_k; b.T = ntok;
    balance_kind(type, n_experts, [&](auto t, auto lanes, auto nv) {
        launch_balance_grad<std::remove_pointer_t<decltype(t)>, decltype(lanes)::value, decltype(nv)::value>(b, logits, grad, stream);
    });
    check_launch("balance_loss_grad");
}

}  // extern "C"
