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
    int E, K, T, groups, threads;   // threads per work-group of the sums
    int ep, lanes, joins;   // columns of a work-group's sums; lanes of four columns to join them, and work-groups
    float* psum;     // [groups][ep]
    int *pcnt, *pn;  // [groups][ep], [groups]
    float* lpart;    // parts of the loss, one per work-group of k_balance_loss
    int* done;       // how many of them have ended
    float *loss, *probs;
    int *counts_out, *tokens_out;
};

// LANES lanes per row, lane l of them the columns 4 LANES i + 4 l .. + 3 for
// i < NV.  Sixteen up to 256 columns: a row of 256 is four loads of 16 bytes
// per lane, and the sums over a row are four DPP steps for four rows at once;
// above, the whole wave, 8 or 16 values and as many sums per lane (2048 rows
// of 384: 15.0 us for loss and gradient, with 16 lanes 20.0).
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

// Probabilities and pairs summed over the rows of each work-group (row t of
// round i: (i * groups + group) * ROWS + ..), every sum in a fixed order: a lane
// over its rows, four rows of a wave, the waves.  Counts are integers: LDS
// atomics in any order.  With one work-group the results follow at once.
template <typename T, int LANES, int NV, int THREADS, bool ONE>
__global__ __launch_bounds__(THREADS) void k_balance_sums(Balance b, const T* __restrict__ logits) {
    constexpr int ROWS = THREADS / LANES, COLS = 4 * LANES * NV;
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
            b.psum[(int64_t)blockIdx.x * b.ep + e] = psum(e);
            b.pcnt[(int64_t)blockIdx.x * b.ep + e] = cnt[e];
        }
        if (tid == 0) b.pn[blockIdx.x] = n;
    }
}

// The work-groups' sums joined: LANES lanes of four experts each by the segments
// of the groups that fit in 1024 threads (32 at most), a wave's segments added
// up first.  Where one work-group does not take all experts, the last to end
// adds up the parts of the loss.
constexpr int BAL_GROUPS = 256;   // of the sums at most
constexpr int BAL_JOIN = 8;   // lanes where there are several work-groups
constexpr int bal_join_threads(int lanes) { return lanes < 32 ? 32 * lanes : 1024; }
template <int LANES>
__global__ __launch_bounds__(bal_join_threads(LANES)) void k_balance_loss(Balance b) {
    constexpr int THREADS = bal_join_threads(LANES), SEGS = THREADS / LANES, COLS = 4 * LANES;
    constexpr int PARTS = LANES < 64 ? THREADS / 64 : SEGS, LOSSES = COLS <= 64 ? 1 : COLS / 64;
    __shared__ float ps[PARTS][COLS], part[LOSSES];
    __shared__ int pc[PARTS][COLS], n, last;
    const int tid = threadIdx.x, seg = tid / LANES, c = tid % LANES * 4, e0 = blockIdx.x * COLS, e = e0 + tid;
    if (tid == 0) n = 0;
    __syncthreads();
    float s[4] = {};
    int k[4] = {};
    if (e0 + c < b.ep) {
#pragma unroll 8
        for (int g = seg; g < b.groups; g += SEGS) {
            const float4 v = *(const float4*)(b.psum + (int64_t)g * b.ep + e0 + c);
            const int4 u = *(const int4*)(b.pcnt + (int64_t)g * b.ep + e0 + c);
            s[0] += v.x; s[1] += v.y; s[2] += v.z; s[3] += v.w;
            k[0] += u.x; k[1] += u.y; k[2] += u.z; k[3] += u.w;
        }
    }
    static_assert(THREADS >= BAL_GROUPS);
    const int tokens = tid < b.groups ? b.pn[tid] : 0;
    if (tokens) atomicAdd(&n, tokens);
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if constexpr (LANES <= 8) {
            s[i] += xlane<8>(s[i]);
            k[i] += xlane<8>(k[i]);
        }
        if constexpr (LANES <= 16) {
            s[i] += xlane<16>(s[i]);
            k[i] += xlane<16>(k[i]);
        }
        if constexpr (LANES <= 32) {
            s[i] += xlane<32>(s[i]);
            k[i] += xlane<32>(k[i]);
        }
    }
    if (LANES >= 64 || (tid & 63) < LANES) {
        *(float4*)&ps[LANES < 64 ? tid / 64 : seg][c] = make_float4(s[0], s[1], s[2], s[3]);
        *(int4*)&pc[LANES < 64 ? tid / 64 : seg][c] = make_int4(k[0], k[1], k[2], k[3]);
    }
    __syncthreads();
    float l = 0.0f;
    if (tid < COLS && e < b.E) {
        float v = 0.0f;
        int u = 0;
#pragma unroll
        for (int i = 0; i < PARTS; i++) {
            v += ps[i][tid];
            u += pc[i][tid];
        }
        v = n ? v / (float)n : 0.0f;
        b.probs[e] = v;
        b.counts_out[e] = u;
        l = n ? (float)u / ((float)n * (float)b.K) * v : 0.0f;
    }
    l = slot_reduce16(l);
    l += xlane<16>(l);
    l += xlane<32>(l);
    if constexpr (LOSSES > 1) {
        if ((tid & 63) == 0 && tid / 64 < LOSSES) part[tid / 64] = l;
        __syncthreads();
        l = 0.0f;
#pragma unroll
        for (int i = 0; i < LOSSES; i++) l += part[i];
    }
    if constexpr (LANES == BAL_JOIN) {
        if (b.joins > 1) {
            if (tid == 0) {
                // visible to the whole device before the count says so
                __hip_atomic_store(&b.lpart[blockIdx.x], l, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                last = __hip_atomic_fetch_add(b.done, 1, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT) == b.joins - 1;
            }
            __syncthreads();
            if (!last || tid >= 64) return;
            l = tid < b.joins ? __hip_atomic_load(&b.lpart[tid], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : 0.0f;
            l = slot_reduce16(l);
            l += xlane<16>(l);
        }
    }
    if (tid == 0) {
        *b.loss = (float)b.E * l;
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

// How T rows are shared out.  Work-groups of the sums have 1024 threads, 64 rows
// (16 above 256 experts) at once.  One alone, that finishes by itself, while the
// rounds of its rows cost less than a second launch, about 4 us (64 tokens of
// 256 experts 5.9 us, another 1.4 us for every 64 more; 160 of 72 6.0, against
// 4.0 + 3.0 and the launch).  256 threads while the sums of a quarter of the
// rows per work-group are still joined by one work-group, which takes 3 to 5.6 us
// for up to BAL_JOIN_MAX sums where several take 6 to 7 (2219 tokens of 143
// experts: 4.8 + 5.6 us, before 7.2 + 6.3).
constexpr int BAL_ONE = 4, BAL_ONE_MAX = 32768;   // rounds and logits of a single work-group
constexpr int BAL_GRAD = 1024, BAL_JOIN_MAX = 32768;
static void balance_plan(Balance& b) {
    const int rows = b.E > 256 ? 16 : 64;
    auto groups = [&](int r) { return b.T / r + (b.T % r != 0); };
    b.ep = (b.E + 3) & ~3;
    b.threads = 1024;
    b.groups = groups(rows);
    if (b.groups <= BAL_ONE && b.T * b.ep <= BAL_ONE_MAX) {
        b.groups = 1;
    } else if (groups(rows / 4) <= BAL_GROUPS && groups(rows / 4) * b.ep <= BAL_JOIN_MAX) {
        b.threads = 256;
        b.groups = groups(rows / 4);
    } else if (b.groups > BAL_GROUPS) {
        b.groups = BAL_GROUPS;
    }
    b.lanes = BAL_JOIN;
    while (b.groups * b.ep <= BAL_JOIN_MAX && 4 * b.lanes < b.ep) b.lanes *= 2;
    b.joins = (b.ep + 4 * b.lanes - 1) / (4 * b.lanes);
}

template <int LANES>
static void launch_join(const Balance& b, hipStream_t s) {
    if (b.lanes == LANES)
        hipLaunchKernelGGL(k_balance_loss<LANES>, dim3(b.joins), dim3(bal_join_threads(LANES)), 0, s, b);
    else if constexpr (LANES < MAX_E / 4)
        launch_join<2 * LANES>(b, s);
}

template <typename T, int LANES, int NV>
static void launch_balance(const Balance& b, const void* logits, hipStream_t s) {
    const T* x = (const T*)logits;
    if (b.groups == 1) {
        hipLaunchKernelGGL((k_balance_sums<T, LANES, NV, 1024, true>), dim3(1), dim3(1024), 0, s, b, x);
        return;
    }
    if (b.threads == 256)
        hipLaunchKernelGGL((k_balance_sums<T, LANES, NV, 256, false>), dim3(b.groups), dim3(256), 0, s, b, x);
    else
        hipLaunchKernelGGL((k_balance_sums<T, LANES, NV, 1024, false>), dim3(b.groups), dim3(1024), 0, s, b, x);
    launch_join<BAL_JOIN>(b, s);
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
        std::integral_constant<int, 64> all;
        if (E <= 64) f(t, few, std::integral_constant<int, 1>{});
        else if (E <= 128) f(t, few, std::integral_constant<int, 2>{});
        else if (E <= 256) f(t, few, std::integral_constant<int, 4>{});
        else if (E <= 512) f(t, all, std::integral_constant<int, 2>{});
        else f(t, all, std::integral_constant<int, 4>{});
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
    Balance b{};
    b.E = n_experts; b.T = max_ntok;
    balance_plan(b);
    if (b.groups == 1) return 0;
    // of any smaller number of tokens, too
    const int64_t quarter = min(BAL_JOIN_MAX / b.ep, BAL_GROUPS);
    const size_t g = b.threads == 256 ? b.groups : max((int64_t)b.groups, quarter);
    return 2 * al256(g * b.ep * 4) + al256(g * 4) + 256;
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
    b.E = n_experts; b.K = top_k; b.T = ntok;
    balance_plan(b);
    uint8_t* w = (uint8_t*)workspace;
    const size_t one = al256((size_t)b.groups * b.ep * 4);
    b.psum = (float*)w; b.pcnt = (int*)(w + one); b.pn = (int*)(w + 2 * one);
    b.lpart = (float*)(w + 2 * one + al256((size_t)b.groups * 4));
    b.done = (int*)(b.lpart + MAX_E / (4 * BAL_JOIN));
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
