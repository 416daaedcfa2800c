// pairs.hip -- a router's (token, expert) pairs sorted by expert, the tokens'
// rows copied into that order and the experts' rows summed back, with the
// gradients.  No counterpart in the reference, which runs one token at a time.
#include <type_traits>

#include "api_internal.h"
#include "float_rows.h"
#include "moe_common.h"

namespace chimere {

struct Pairs {
    const int* ids;
    const uint8_t* mask;
    int *order, *position, *offsets;
    int* counts;    // [groups][E]: pairs of each work-group's chunk
    int E, K, P, groups, chunk;
};

constexpr int PAIR_THREADS = 1024, PAIR_WAVES = PAIR_THREADS / 64;
constexpr int PAIR_CHUNK = 2048, PAIR_GROUPS = 256;   // pairs of a work-group at least, work-groups at most
constexpr int PAIR_ONE = 8192;    // that one work-group sorts by itself (4948 of 60 experts 6.6 us, two launches 3.4 + 4.7; 8192 of 256 9.3, 3.6 + 4.8; 16384 17.6, 4.2 + 5.2)
constexpr int PAIR_AHEAD = 8;     // ids of a lane on their way at a time (131072 pairs, both launches: 10 us, one at a time 13.2)

// the expert of pair p, -1 where it has none
__device__ __forceinline__ int pair_expert(const Pairs& s, int p, int end) {
    if (p >= end) return -1;
    const int e = s.ids[p];
    const bool kept = !s.mask || s.mask[p / s.K];     // (on its way with the id)
    return (unsigned)e < (unsigned)s.E && kept ? e : -1;
}

__global__ __launch_bounds__(PAIR_THREADS) void k_pairs_count(Pairs s) {
    __shared__ int cnt[MAX_E];
    for (int e = threadIdx.x; e < s.E; e += PAIR_THREADS) cnt[e] = 0;
    __syncthreads();
    const int p0 = blockIdx.x * s.chunk, end = min(s.P - p0, s.chunk) + p0;
#pragma unroll 2
    for (int p = p0 + threadIdx.x; p < end; p += PAIR_THREADS) {
        const int e = pair_expert(s, p, end);
        if (e >= 0) atomicAdd(&cnt[e], 1);
    }
    __syncthreads();
    for (int e = threadIdx.x; e < s.E; e += PAIR_THREADS) s.counts[(int64_t)blockIdx.x * s.E + e] = cnt[e];
}

// A counting sort, stable: a wave has a contiguous piece of its work-group's
// chunk and counters of its own that start where its pairs of each expert
// start; 64 pairs at a time find their place among those of the same expert by
// comparing ballots of the id's bits.  Every work-group adds up the counts of
// those before it (64 KB of L2 at 64 work-groups of 256 experts); with one
// work-group there is no launch before.  Latency bounds it: two passes over a
// lane's ids, which stay in registers if there are eight or fewer (131072 pairs
// of 256 experts: 5.8 us after 4.3 for the counts; 4096 pairs in one launch 5.8).
template <int EMAX, bool ONE>
__global__ __launch_bounds__(PAIR_THREADS) void k_pairs_place(Pairs s) {
    constexpr int BITS = EMAX == 256 ? 8 : 10, SEGS = PAIR_THREADS / EMAX;
    __shared__ int cnt[PAIR_WAVES][EMAX];
    __shared__ int before[SEGS][EMAX], total[SEGS][EMAX], wsum[PAIR_WAVES];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    for (int i = tid; i < PAIR_WAVES * EMAX; i += PAIR_THREADS) (&cnt[0][0])[i] = 0;
    __syncthreads();
    const int p0 = blockIdx.x * s.chunk, end = min(s.P - p0, s.chunk) + p0;
    const int piece = (s.chunk + PAIR_THREADS - 1) / PAIR_THREADS * 64, w0 = p0 + wave * piece, w1 = min(w0 + piece, end);
    // PAIR_AHEAD ids of a lane at a time; the first ones stay for the second pass
    int x[PAIR_AHEAD];
    auto load = [&](int q) {
#pragma unroll
        for (int i = 0; i < PAIR_AHEAD; i++) x[i] = pair_expert(s, q + 64 * i + lane, w1);
    };
    for (int q = w0; q < w1; q += 64 * PAIR_AHEAD) {
        load(q);
#pragma unroll
        for (int i = 0; i < PAIR_AHEAD; i++)
            if (x[i] >= 0) atomicAdd(&cnt[wave][x[i]], 1);
    }
    // pairs of expert e in all and in the work-groups before this one
    const int seg = tid / EMAX, e = tid % EMAX;
    if constexpr (!ONE) {
        int b = 0, t = 0;
        if (e < s.E) {
#pragma unroll 8
            for (int g = seg; g < s.groups; g += SEGS) {
                const int c = s.counts[(int64_t)g * s.E + e];
                t += c;
                b += g < (int)blockIdx.x ? c : 0;
            }
        }
        before[seg][e] = b;
        total[seg][e] = t;
    }
    __syncthreads();
    int all = 0, base = 0;
    if (tid < EMAX) {
        if constexpr (ONE) {
            for (int w = 0; w < PAIR_WAVES; w++) all += cnt[w][tid];
        } else {
            for (int i = 0; i < SEGS; i++) {
                all += total[i][tid];
                base += before[i][tid];
            }
        }
    }
    const int incl = wave_incl_scan(all);
    if (lane == 63) wsum[wave] = incl;
    __syncthreads();
    int first = incl - all, n = 0;
    for (int w = 0; w < PAIR_WAVES; w++) {
        if (w < wave) first += wsum[w];
        n += wsum[w];
    }
    if (tid < EMAX) {
        if (blockIdx.x == 0 && tid < s.E) s.offsets[tid] = first;
        int at = first + base;
        for (int w = 0; w < PAIR_WAVES; w++) {
            const int c = cnt[w][tid];
            cnt[w][tid] = at;
            at += c;
        }
    }
    if (blockIdx.x == 0 && tid == 0) s.offsets[s.E] = n;
    __syncthreads();
    for (int q0 = w0; q0 < w1; q0 += 64 * PAIR_AHEAD) {
        if (w1 - w0 > 64 * PAIR_AHEAD) load(q0);
#pragma unroll
        for (int i = 0; i < PAIR_AHEAD; i++) {
            const int p = q0 + 64 * i + lane, e = x[i];
            if (q0 + 64 * i >= w1) break;
            uint64_t same = __ballot(e >= 0);
#pragma unroll
            for (int b = 0; b < BITS; b++) {
                const uint64_t set = __ballot((e >> b) & 1);
                same &= (e >> b) & 1 ? set : ~set;
            }
            const int rank = __popcll(same & ((1ull << lane) - 1)), lead = __ffsll((unsigned long long)same) - 1;
            int at = 0;
            if (e >= 0 && rank == 0) at = atomicAdd(&cnt[wave][e], __popcll(same));
            at = __shfl(at, e >= 0 ? lead : lane) + rank;
            if (p < w1) s.position[p] = e >= 0 ? at : -1;
            if (e >= 0) s.order[at] = p;
        }
    }
    // rows behind the last pair: of this work-group's part of them
    for (int p = max(p0, n) + tid; p < end; p += PAIR_THREADS) s.order[p] = -1;
}

static void pairs_plan(Pairs& s) {
    if (s.P <= PAIR_ONE) {
        s.chunk = s.P;
        s.groups = 1;
        return;
    }
    const int64_t one = (int64_t)PAIR_CHUNK * PAIR_GROUPS;
    s.chunk = (int)(PAIR_CHUNK * (((int64_t)s.P + one - 1) / one));
    s.groups = (int)(((int64_t)s.P + s.chunk - 1) / s.chunk);
}

struct Rows {
    const void *x, *gout;     // rows that are read; gradient of the sums
    void* out;
    const float *scale, *weights;
    float *out_scale, *gw;
    const int *position, *count;
    int64_t xs, os, gs;
    int T, K, H, R, otype, gtype;     // R: rows in the experts' order
};

// The row of the token's pair k0 + lane, -1 where there is none: one load for all of them.
__device__ __forceinline__ int pair_row(const Rows& d, int64_t t, int k0) {
    const int k = k0 + (threadIdx.x & 63), r = k < d.K ? d.position[t * d.K + k] : -1;
    return (unsigned)r < (unsigned)d.R ? r : -1;
}

// A token's row of H elements is read once and written at its pairs' rows;
// rows behind the last pair are cleared.  W waves per token, four pieces of 16
// bytes of a lane at a time.  Bytes bound it (16384 tokens, top-8, 2048 bf16:
// 604 MB in 112 us, 5.4 TB/s, the rate of a large copy; 512 tokens 5.4 us).
template <typename T, int W>
__global__ __launch_bounds__(256) void k_dispatch(Rows d) {
    constexpr int V = 16 / sizeof(T), N = 4, STEP = 64 * W * V;
    typedef typename VecOf<T, V>::type vec;
    const int c0 = (threadIdx.x & (64 * W - 1)) * V;
    const int64_t items = (int64_t)gridDim.x * (4 / W);
    const T* x = (const T*)d.x;
    T* out = (T*)d.out;
    const int64_t first = (int64_t)blockIdx.x * (4 / W) + threadIdx.x / (64 * W), end = max(*d.count, 0);
    for (int64_t t = first; t < d.T; t += items) {
        // (64 pairs at a time: more are a rare choice, and read the row again)
        for (int k0 = 0; k0 < d.K; k0 += 64) {
            const int mine = pair_row(d, t, k0);
            const uint64_t on = __ballot(mine >= 0);
            if (!on) continue;           // (what a mask has left out is not read)
            for (int c1 = 0; c1 < d.H; c1 += N * STEP) {     // (all lanes go round: one has the row of each pair)
                const int c = c1 + c0;
                vec v[N];
#pragma unroll
                for (int i = 0; i < N; i++) {
                    const int at = c + i * STEP;
                    if (at + V <= d.H) {
                        v[i] = *(const vec*)(x + t * d.xs + at);
                    } else if (at < d.H) {
#pragma unroll
                        for (int j = 0; j < V; j++) v[i][j] = at + j < d.H ? x[t * d.xs + at + j] : T{};
                    }
                }
                for (uint64_t m = on; m; m &= m - 1) {
                    T* to = out + __builtin_amdgcn_readlane(mine, __ffsll((unsigned long long)m) - 1) * d.os;
#pragma unroll
                    for (int i = 0; i < N; i++) {
                        const int at = c + i * STEP;
                        if (at + V <= d.H) {
                            *(vec*)(to + at) = v[i];
                        } else if (at < d.H) {
#pragma unroll
                            for (int j = 0; j < V; j++)
                                if (at + j < d.H) to[at + j] = v[i][j];
                        }
                    }
                }
            }
            if (d.scale && threadIdx.x % (64 * W) < 64 && mine >= 0) d.out_scale[mine] = d.scale[t];
        }
    }
    for (int64_t r = end + first; r < d.R; r += items) {
        T* to = out + r * d.os;
        for (int c = c0; c < d.H; c += STEP) {
            if (c + V <= d.H) {
                *(vec*)(to + c) = vec{};
            } else {
                for (int j = 0; c + j < d.H; j++) to[c + j] = T{};
            }
        }
        if (d.out_scale && c0 == 0) d.out_scale[r] = 0.0f;     // (of no tokens there is no scale to read)
    }
}

template <int V, typename T>
__device__ __forceinline__ void rows_load(const T* row, int c, int cols, typename VecOf<T, V>::type& v) {
    if (c + V <= cols) {
        v = *(const typename VecOf<T, V>::type*)(row + c);
    } else {
#pragma unroll
        for (int k = 0; k < V; k++) v[k] = c + k < cols ? row[c + k] : (T)0.0f;
    }
}
template <int V>
__device__ __forceinline__ void rows_store(void* row, int type, int c, int cols, const float (&v)[V]) {
    if (type == T_F32) store_row((float*)row + c, v, cols - c);
    else if (type == T_F16) store_row((_Float16*)row + c, v, cols - c);
    else store_row((__bf16*)row + c, v, cols - c);
}
template <int V>
__device__ __forceinline__ void rows_load_as(const void* row, int type, int c, int cols, float (&v)[V]) {
    auto of = [&](auto* p) {
        typedef std::remove_const_t<std::remove_pointer_t<decltype(p)>> U;
        typename VecOf<U, V>::type x;
        rows_load<V>(p, c, cols, x);
#pragma unroll
        for (int k = 0; k < V; k++) v[k] = (float)x[k];
    };
    if (type == T_F32) of((const float*)row);
    else if (type == T_F16) of((const _Float16*)row);
    else of((const __bf16*)row);
}
__device__ __forceinline__ int64_t rows_bytes(int type) { return type == T_F32 ? 4 : 2; }

constexpr int ROWS_K = 8;   // pairs of a token whose rows are on their way at a time

// out[t] = sum over k, ascending, of weights[t][k] y[position[t][k]] in f32:
// every row is read once, by the waves of its token, eight rows on their way
// at a time; no atomics, so sums repeat bit for bit.  Bytes bound it (4096
// tokens, top-8, 2048 bf16: 151 MB in 23.5 us, 6.4 TB/s, part of it from the
// last-level cache; 16384: 604 MB in 122 us, 5.0 TB/s; 512: 4.4 us).
template <typename T>
__global__ __launch_bounds__(256) void k_combine(Rows d) {
    constexpr int V = 16 / sizeof(T), STEP = 256 * V;
    typedef typename VecOf<T, V>::type vec;
    const int c0 = threadIdx.x * V;
    const int64_t items = gridDim.x;
    const T* y = (const T*)d.x;
    for (int64_t t = blockIdx.x; t < d.T; t += items) {
        uint8_t* out = (uint8_t*)d.out + t * d.os * rows_bytes(d.otype);
        for (int c1 = 0; c1 < d.H; c1 += STEP) {     // (all lanes go round: one has the row of each pair)
            const int c = c1 + c0;
            float s[V] = {};
            for (int k0 = 0; k0 < d.K; k0 += 64) {
                const int row = pair_row(d, t, k0), lane = threadIdx.x & 63;
                const float weight = row >= 0 && d.weights ? d.weights[t * d.K + k0 + lane] : 1.0f;
                uint64_t on = __ballot(row >= 0);
                while (on) {
                    vec v[ROWS_K];
                    float w[ROWS_K];
                    int n = 0;
#pragma unroll
                    for (int k = 0; k < ROWS_K; k++) {
                        if (!on) break;
                        const int at = __ffsll((unsigned long long)on) - 1;
                        on &= on - 1;
                        n++;
                        w[k] = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, weight), at));
                        rows_load<V>(y + __builtin_amdgcn_readlane(row, at) * d.xs, c, d.H, v[k]);
                    }
#pragma unroll
                    for (int k = 0; k < ROWS_K; k++)
                        if (k < n)
#pragma unroll
                            for (int j = 0; j < V; j++) s[j] = __builtin_fmaf(w[k], (float)v[k][j], s[j]);
                }
            }
            rows_store(out, d.otype, c, d.H, s);
        }
    }
}

// gy[position[t][k]] = weights[t][k] gout[t], gw[t][k] = <gout[t], y[position[t][k]]>:
// gout's row is read once (again for every further eight pairs), y's read and
// gy's written once.  Rows of gy behind the last pair are cleared.  Bytes bound
// it (4096 tokens, top-8, 2048 bf16: 285 MB in 54 us, 5.2 TB/s; 16384: 1.14 GB
// in 240 us, 4.8 TB/s).
template <typename T>
__global__ __launch_bounds__(256) void k_combine_grad(Rows d) {
    constexpr int V = 16 / sizeof(T), STEP = 256 * V;
    typedef typename VecOf<T, V>::type vec;
    __shared__ float part[4][ROWS_K];
    const int c0 = threadIdx.x * V, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t items = gridDim.x;
    const T* y = (const T*)d.x;
    T* gy = (T*)d.out;
    const int64_t first = blockIdx.x, end = gy ? max(*d.count, 0) : 0;
    for (int64_t t = first; t < d.T; t += items) {
        const uint8_t* gout = (const uint8_t*)d.gout + t * d.gs * rows_bytes(d.gtype);
        for (int k0 = 0; k0 < d.K; k0 += ROWS_K) {
            float w[ROWS_K], dot[ROWS_K] = {};
            int r[ROWS_K];
            bool any = false;
            const int row = pair_row(d, t, k0);
            const float weight = lane < ROWS_K && row >= 0 && d.weights ? d.weights[t * d.K + k0 + lane] : 1.0f;
#pragma unroll
            for (int k = 0; k < ROWS_K; k++) {
                r[k] = __builtin_amdgcn_readlane(row, k);
                w[k] = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, weight), k));
                any |= r[k] >= 0;
            }
            if (any)
                for (int c = c0; c < d.H; c += STEP) {
                    vec v[ROWS_K];
                    float g[V];
                    if (d.gw)
#pragma unroll
                        for (int k = 0; k < ROWS_K; k++)
                            if (r[k] >= 0) rows_load<V>(y + r[k] * d.xs, c, d.H, v[k]);
                    rows_load_as(gout, d.gtype, c, d.H, g);
#pragma unroll
                    for (int k = 0; k < ROWS_K; k++) {
                        if (r[k] < 0) continue;
                        if (gy) {
                            float o[V];
#pragma unroll
                            for (int j = 0; j < V; j++) o[j] = w[k] * g[j];
                            store_row(gy + r[k] * d.os + c, o, d.H - c);
                        }
                        if (d.gw)
#pragma unroll
                            for (int j = 0; j < V; j++) dot[k] = __builtin_fmaf(g[j], (float)v[k][j], dot[k]);
                    }
                }
            if (d.gw) {
#pragma unroll
                for (int k = 0; k < ROWS_K; k++) {
                    float v = slot_reduce16(dot[k]);
                    v += xlane<16>(v);
                    v += xlane<32>(v);
                    dot[k] = v;
                }
                __syncthreads();        // the sums of the round before have been read
                if (lane == 0)
#pragma unroll
                    for (int k = 0; k < ROWS_K; k++) part[wave][k] = dot[k];
                __syncthreads();
                if (threadIdx.x < ROWS_K && k0 + (int)threadIdx.x < d.K)
                    d.gw[t * d.K + k0 + threadIdx.x] = (part[0][threadIdx.x] + part[1][threadIdx.x]) + (part[2][threadIdx.x] + part[3][threadIdx.x]);
            }
        }
    }
    if (!gy) return;
    for (int64_t r = end + first; r < d.R; r += items) {
        T* to = gy + r * d.os;
        const float none[V] = {};
        for (int c = c0; c < d.H; c += STEP) store_row(to + c, none, d.H - c);
    }
}

// Sums take four waves per token, one token per work-group (4096 tokens, top-8, 2048 bf16: gradient 54 us, with a wave per
// token 58.5).  Copies take one wave per token where it has the row at a time, four pieces of 1 KB: it loads the token's places
// once, and its stores run on while the next token's are loaded (4096 tokens, top-8, 2048 int8: 13.5 us, with four waves 34;
// bf16 23 and 24).  Longer rows take four (256 tokens of 4096 bf16: 5.3 us, with one wave 8.2; 1024 12.8 and 13.1; 16384 243 both).
constexpr int ROWS_GROUPS = 4096;           // work-groups at most
constexpr int ROWS_WAVE_BYTES = 4096;       // of a row that one wave copies
static dim3 rows_grid(int64_t T, bool wave) {
    const int64_t groups = wave ? (T + 3) / 4 : T;
    return dim3((unsigned)(groups < 1 ? 1 : groups < ROWS_GROUPS ? groups : ROWS_GROUPS));
}
template <typename F>
static void rows_type(int type, F f) {
    if (type == T_F32) f((float*)nullptr);
    else if (type == T_F16) f((_Float16*)nullptr);
    else f((__bf16*)nullptr);
}

constexpr int TYPE_I8 = CHIMERE_TYPE_I8;

static bool pairs_size(const char* what, int E, int K, int T) {
    if (E >= 1 && E <= MAX_E && K >= 1 && K <= MAX_E && T >= 0 && (int64_t)T * K < (1 << 30)) return true;
    set_error(CHIMERE_ERR_ARG, "%s: n_experts=%d top_k=%d ntok=%d out of range", what, E, K, T);
    return false;
}
static bool at_float_rows(int type, const void* p, int64_t ld, int least) {
    return p && float_aligned(type, p) && ld >= least;
}

}  // namespace chimere

using namespace chimere;

extern "C" {

size_t chimere_sort_pairs_workspace_size(int n_experts, int top_k, int max_ntok) {
    if (n_experts < 1 || n_experts > MAX_E || top_k < 1 || top_k > MAX_E || max_ntok < 0 || (int64_t)max_ntok * top_k >= (1 << 30))
        return 0;
    Pairs s{};
    s.P = max_ntok * top_k;
    pairs_plan(s);
    // (of any smaller number of tokens, too: fewer pairs can be more work-groups of shorter chunks)
    return s.groups <= 1 ? 0 : al256((size_t)(s.chunk > PAIR_CHUNK ? PAIR_GROUPS : s.groups) * n_experts * 4);
}

void chimere_sort_pairs(const int* ids, const uint8_t* mask, int* order, int* position, int* offsets, int n_experts,
                        int top_k, int ntok, void* workspace, size_t workspace_bytes, hipStream_t stream) {
    if (!pairs_size("sort_pairs", n_experts, top_k, ntok)) return;
    const size_t need = chimere_sort_pairs_workspace_size(n_experts, top_k, ntok);
    CHIMERE_REQUIRE(offsets && (ntok == 0 || (ids && order && position)) && (workspace || !need), CHIMERE_ERR_ARG,
                    "sort_pairs: null pointer");
    CHIMERE_REQUIRE(workspace_bytes >= need && ((uintptr_t)workspace & 255) == 0, CHIMERE_ERR_WORKSPACE,
                    "sort_pairs: workspace %zu bytes < %zu (or not 256-byte aligned)", workspace_bytes, need);
    Pairs s{ids, mask, order, position, offsets, (int*)workspace, n_experts, top_k, ntok * top_k, 0, 0};
    pairs_plan(s);
    const dim3 threads(PAIR_THREADS);
    if (s.groups <= 1) {
        if (n_experts <= 256) hipLaunchKernelGGL((k_pairs_place<256, true>), dim3(1), threads, 0, stream, s);
        else hipLaunchKernelGGL((k_pairs_place<1024, true>), dim3(1), threads, 0, stream, s);
    } else {
        hipLaunchKernelGGL(k_pairs_count, dim3(s.groups), threads, 0, stream, s);
        if (n_experts <= 256) hipLaunchKernelGGL((k_pairs_place<256, false>), dim3(s.groups), threads, 0, stream, s);
        else hipLaunchKernelGGL((k_pairs_place<1024, false>), dim3(s.groups), threads, 0, stream, s);
    }
    check_launch("sort_pairs");
}

void chimere_dispatch(int type, const void* x, int64_t x_stride, const float* scale, const int* position, const int* offsets,
                      void* out, int64_t out_stride, float* out_scale, int nrows, int n_experts, int top_k, int ntok,
                      int ncols, hipStream_t stream) {
    if (!pairs_size("dispatch", n_experts, top_k, ntok)) return;
    CHIMERE_REQUIRE(float_type(type) || type == TYPE_I8, CHIMERE_ERR_ARG, "dispatch: unsupported type %d", type);
    CHIMERE_REQUIRE(ncols >= 1 && ncols <= (1 << 24) && nrows >= 0, CHIMERE_ERR_ARG, "dispatch: nrows=%d ncols=%d out of range", nrows, ncols);
    if (nrows == 0) return;
    CHIMERE_REQUIRE(offsets && out && out_stride >= ncols && (type == TYPE_I8 || float_aligned(type, out)), CHIMERE_ERR_ARG,
                    "dispatch: null or misaligned pointer, or bad stride");
    CHIMERE_REQUIRE(ntok == 0 || (x && position && x_stride >= 0 && (type == TYPE_I8 || float_aligned(type, x))), CHIMERE_ERR_ARG,
                    "dispatch: null or misaligned pointer, or bad stride");
    CHIMERE_REQUIRE((scale && out_scale) || (!scale && !out_scale) || ntok == 0, CHIMERE_ERR_ARG, "dispatch: scales of one side only");
    Rows d{};
    d.x = x; d.out = out; d.scale = out_scale ? scale : nullptr; d.out_scale = out_scale; d.position = position; d.count = offsets + n_experts;
    d.xs = x_stride; d.os = out_stride; d.T = ntok; d.K = top_k; d.H = ncols; d.R = nrows;
    const int64_t bytes = (int64_t)ncols * (type == TYPE_I8 ? 1 : type == T_F32 ? 4 : 2);
    const bool wave = bytes <= ROWS_WAVE_BYTES;
    const dim3 grid = rows_grid(ntok, wave);
    auto go = [&](auto t) {
        typedef std::remove_pointer_t<decltype(t)> U;
        if (wave) hipLaunchKernelGGL((k_dispatch<U, 1>), grid, dim3(256), 0, stream, d);
        else hipLaunchKernelGGL((k_dispatch<U, 4>), grid, dim3(256), 0, stream, d);
    };
    if (type == TYPE_I8) go((uint8_t*)nullptr);
    else if (type == T_F32) go((uint32_t*)nullptr);
    else go((uint16_t*)nullptr);
    check_launch("dispatch");
}

void chimere_combine(int type, const void* y, int64_t y_stride, const int* position, const float* weights, int out_type,
                     void* out, int64_t out_stride, int nrows, int top_k, int ntok, int ncols, hipStream_t stream) {
    if (!pairs_size("combine", 1, top_k, ntok)) return;
    CHIMERE_REQUIRE(float_type(type) && float_type(out_type), CHIMERE_ERR_ARG, "combine: unsupported type %d or %d", type, out_type);
    CHIMERE_REQUIRE(ncols >= 1 && ncols <= (1 << 24) && nrows >= 0, CHIMERE_ERR_ARG, "combine: nrows=%d ncols=%d out of range", nrows, ncols);
    if (ntok == 0) return;
    CHIMERE_REQUIRE(position && at_float_rows(out_type, out, out_stride, ncols) && (nrows == 0 || at_float_rows(type, y, y_stride, 0)),
                    CHIMERE_ERR_ARG, "combine: null or misaligned pointer, or bad stride");
    Rows d{};
    d.x = y; d.out = out; d.weights = weights; d.position = position;
    d.xs = y_stride; d.os = out_stride; d.T = ntok; d.K = top_k; d.H = ncols; d.R = nrows; d.otype = out_type;
    rows_type(type, [&](auto t) {
        hipLaunchKernelGGL(k_combine<std::remove_pointer_t<decltype(t)>>, rows_grid(ntok, false), dim3(256), 0, stream, d);
    });
    check_launch("combine");
}

void chimere_combine_grad(int grad_type, const void* grad_out, int64_t grad_out_stride, int type, const void* y,
                          int64_t y_stride, const int* position, const float* weights, const int* offsets, void* grad_y,
                          int64_t grad_y_stride, float* grad_weights, int nrows, int n_experts, int top_k, int ntok, int ncols,
                          hipStream_t stream) {
    if (!pairs_size("combine_grad", n_experts, top_k, ntok)) return;
    CHIMERE_REQUIRE(float_type(type) && float_type(grad_type), CHIMERE_ERR_ARG, "combine_grad: unsupported type %d or %d", type, grad_type);
    CHIMERE_REQUIRE(ncols >= 1 && ncols <= (1 << 24) && nrows >= 0, CHIMERE_ERR_ARG, "combine_grad: nrows=%d ncols=%d out of range", nrows, ncols);
    CHIMERE_REQUIRE(ntok == 0 || (position && at_float_rows(grad_type, grad_out, grad_out_stride, 0)), CHIMERE_ERR_ARG,
                    "combine_grad: null or misaligned pointer, or bad stride");
    CHIMERE_REQUIRE(nrows == 0 || ((!grad_y || (offsets && at_float_rows(type, grad_y, grad_y_stride, ncols))) &&
                                   (!grad_weights || at_float_rows(type, y, y_stride, 0))),
                    CHIMERE_ERR_ARG, "combine_grad: null or misaligned pointer, or bad stride");
    if ((!grad_y || nrows == 0) && (!grad_weights || ntok == 0)) return;
    Rows d{};
    d.x = y; d.gout = grad_out; d.out = nrows ? grad_y : nullptr; d.weights = weights; d.gw = grad_weights; d.position = position;
    d.count = offsets ? offsets + n_experts : nullptr;
    d.xs = y_stride; d.os = grad_y_stride; d.gs = grad_out_stride; d.gtype = grad_type;
    d.T = ntok; d.K = top_k; d.H = ncols; d.R = nrows;
    rows_type(type, [&](auto t) {
        hipLaunchKernelGGL(k_combine_grad<std::remove_pointer_t<decltype(t)>>, rows_grid(ntok, false), dim3(256), 0, stream, d);
    });
    check_launch("combine_grad");
}

}  // extern "C"
