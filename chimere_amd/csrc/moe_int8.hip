// moe_int8.hip -- the routed experts' FFN over 8-bit integer weights with a
// scale per output channel, for tokens whose expert ids and weights are given.
// The counterpart over block-quantized weights is chimere_moe_prefill
// (cs/src/qwen35_model/moe_ffn.rs:1081-1768 per token).
//
// Launches: rows of x to 8 bits; the pairs of each expert together, with the
// list of tiles; gate and up product with h = silu(g) u; rows of h to 8 bits;
// down product; each token's weighted sum.
#include "api_internal.h"
#include "int8_gemm.h"
#include "moe_common.h"

namespace chimere {

struct MoeI8 {
    int H, F, E, K, T;
    const int8_t *gate, *up, *down;
    const float *gate_s, *up_s, *down_s;
    const int* ids;
    const float* wts;
    const int8_t* xq;      // [T][H]
    const float* xs;       // [T]
    int *order, *total;    // pairs by expert; {pairs, tiles}
    int4* tiles;           // {expert, first sorted pair, pairs, 0}
    float* h;              // [pairs][F], in sorted order
    int8_t* hq;
    float* hs;
    float* y;              // [T * K][H], by pair
    void* out;
    int64_t ldo;
    int tile_pairs;
};

// Counting sort of the pairs by expert; a pair whose id is no expert is left
// out.  Pairs of one expert come in any order: each pair's row is computed on
// its own.
__global__ __launch_bounds__(1024) void k_i8_plan(MoeI8 a) {
    __shared__ int cnt[MAX_E], first[MAX_E], tile0[MAX_E];
    const int tid = threadIdx.x, P = a.T * a.K, TP = a.tile_pairs;
    cnt[tid] = 0;
    __syncthreads();
    for (int p = tid; p < P; p += 1024) {
        const int e = a.ids[p];
        if ((unsigned)e < (unsigned)a.E) atomicAdd(&cnt[e], 1);
    }
    __syncthreads();
    if (tid == 0) {
        int n = 0, t = 0;
        for (int e = 0; e < a.E; e++) {
            first[e] = n;
            tile0[e] = t;
            n += cnt[e];
            t += (cnt[e] + TP - 1) / TP;
        }
        a.total[0] = n;
        a.total[1] = t;
    }
    __syncthreads();
    if (tid < a.E)
        for (int s = 0; s * TP < cnt[tid]; s++)
            a.tiles[tile0[tid] + s] = make_int4(tid, first[tid] + s * TP, min(TP, cnt[tid] - s * TP), 0);
    __syncthreads();
    for (int p = tid; p < P; p += 1024) {
        const int e = a.ids[p];
        if ((unsigned)e < (unsigned)a.E) a.order[atomicAdd(&first[e], 1)] = p;
    }
}

typedef I8Tile<2, 2, 2, 2> GuTile;    // 128 pairs x 64 columns of F, gate and up
typedef I8Tile<2, 2, 2, 2> DnTile;    // 128 pairs x 128 columns of H

// Gate and up: the weight rows of a tile alternate in blocks of 32 between
// gate and up, so g and u of the same (pair, column) meet in a lane.
__global__ __launch_bounds__(64 * GuTile::NW) void k_i8_gate_up(MoeI8 a) {
    typedef GuTile Tile;
    __shared__ __align__(16) uint8_t lds[Tile::LDS];
    const int fb = (a.F + Tile::BN / 2 - 1) / (Tile::BN / 2), tile = blockIdx.x / fb;
    if (tile >= a.total[1]) return;
    const int4 t = a.tiles[tile];
    const int f0 = (blockIdx.x - tile * fb) * (Tile::BN / 2), lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint32_t aoff[Tile::PM], woff[Tile::PN];
#pragma unroll
    for (int p = 0; p < Tile::PM; p++) {
        const int r = min((wave * Tile::PM + p) * 8 + (lane >> 3), t.z - 1);
        aoff[p] = (uint32_t)(a.order[t.y + r] / a.K) * (uint32_t)a.H;
    }
#pragma unroll
    for (int p = 0; p < Tile::PN; p++) {
        const int r = (wave * Tile::PN + p) * 8 + (lane >> 3);
        woff[p] = (uint32_t)(min(f0 + (r >> 6) * 32 + (r & 31), a.F - 1)) * (uint32_t)a.H;
    }
    const int64_t e = t.x;
    const float xs = threadIdx.x < Tile::BM ? a.xs[a.order[t.y + min((int)threadIdx.x, t.z - 1)] / a.K] : 0.0f;
    v16i acc[Tile::MTILES][Tile::NTILES];
    Tile::run(a.xq, a.gate + e * a.F * a.H, a.up + e * a.F * a.H, aoff, woff, a.H, lds, acc);
    constexpr int VEC = 4;
    const int f = f0 + Tile::first_col<VEC, true>();
    const bool in = f < a.F;   // F is a multiple of 16: all four columns or none
    const float4 sg = in ? *(const float4*)(a.gate_s + e * a.F + f) : float4{};
    const float4 su = in ? *(const float4*)(a.up_s + e * a.F + f) : float4{};
    Tile::rows<VEC, true>(lds, acc, make_float2(xs, 0.0f),
                          [&](int r, const int(&g)[VEC], const int(&u)[VEC], float2 of_row) {
        if (r >= t.z || !in) return;
        const float s = of_row.x;
        float4 h;
        h.x = det_silu((float)g[0] * s * sg.x) * ((float)u[0] * s * su.x);
        h.y = det_silu((float)g[1] * s * sg.y) * ((float)u[1] * s * su.y);
        h.z = det_silu((float)g[2] * s * sg.z) * ((float)u[2] * s * su.z);
        h.w = det_silu((float)g[3] * s * sg.w) * ((float)u[3] * s * su.w);
        *(float4*)(a.h + (int64_t)(t.y + r) * a.F + f) = h;
    });
}

__global__ __launch_bounds__(64 * DnTile::NW) void k_i8_down(MoeI8 a) {
    typedef DnTile Tile;
    __shared__ __align__(16) uint8_t lds[Tile::LDS];
    const int hb = (a.H + Tile::BN - 1) / Tile::BN, tile = blockIdx.x / hb;
    if (tile >= a.total[1]) return;
    const int4 t = a.tiles[tile];
    const int n0 = (blockIdx.x - tile * hb) * Tile::BN, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint32_t aoff[Tile::PM], woff[Tile::PN];
#pragma unroll
    for (int p = 0; p < Tile::PM; p++)
        aoff[p] = (uint32_t)min((wave * Tile::PM + p) * 8 + (lane >> 3), t.z - 1) * (uint32_t)a.F;
#pragma unroll
    for (int p = 0; p < Tile::PN; p++)
        woff[p] = (uint32_t)min(n0 + (wave * Tile::PN + p) * 8 + (lane >> 3), a.H - 1) * (uint32_t)a.F;
    const int64_t e = t.x;
    const int row = t.y + min((int)threadIdx.x, t.z - 1);
    const float2 mine = threadIdx.x < Tile::BM ? make_float2(a.hs[row], __builtin_bit_cast(float, a.order[row]))
                                               : float2{};
    v16i acc[Tile::MTILES][Tile::NTILES];
    const int8_t* w = a.down + e * a.H * a.F;
    Tile::run(a.hq + (int64_t)t.y * a.F, w, w, aoff, woff, a.F, lds, acc);
    constexpr int VEC = 4;
    const int n = n0 + Tile::first_col<VEC>();
    const bool in = n < a.H;   // H is a multiple of 16: all four columns or none
    const float4 sd = in ? *(const float4*)(a.down_s + e * a.H + n) : float4{};
    Tile::rows<VEC>(lds, acc, mine, [&](int r, const int(&x)[VEC], float2 of_row) {
        if (r >= t.z || !in) return;
        const float s = of_row.x;
        *(float4*)(a.y + (int64_t)__builtin_bit_cast(int, of_row.y) * a.H + n) =
            make_float4((float)x[0] * s * sd.x, (float)x[1] * s * sd.y, (float)x[2] * s * sd.z, (float)x[3] * s * sd.w);
    });
}

// out[t] = sum over k, ascending, of w[t][k] y[t][k]; a pair whose id is no
// expert adds nothing.
template <typename T>
__global__ __launch_bounds__(256) void k_i8_combine(MoeI8 a) {
    const int hb = (a.H + 255) / 256, t = blockIdx.x / hb, h = (blockIdx.x - t * hb) * 256 + threadIdx.x;
    if (h >= a.H) return;
    float acc = 0.0f;
    for (int k = 0; k < a.K; k++) {
        const int64_t p = (int64_t)t * a.K + k;
        if ((unsigned)a.ids[p] < (unsigned)a.E) acc = __builtin_fmaf(a.wts[p], a.y[p * a.H + h], acc);
    }
    store_f((T*)a.out + t * a.ldo + h, acc);
}

struct MoeI8Plan {
    size_t xq, xs, order, total, tiles, h, hq, hs, y, bytes;
    int max_tiles;
};

static MoeI8Plan plan_moe_i8(int H, int F, int E, int K, int T) {
    MoeI8Plan p{};
    const size_t P = (size_t)T * K;
    p.max_tiles = (int)(P / GuTile::BM + (P < (size_t)E ? P : (size_t)E));
    auto take = [&](size_t& at, size_t n) { at = p.bytes; p.bytes += al256(n); };
    take(p.xq, (size_t)T * H);
    take(p.xs, (size_t)T * 4);
    take(p.order, P * 4);
    take(p.total, 8);
    take(p.tiles, (size_t)p.max_tiles * sizeof(int4));
    take(p.h, P * F * 4);
    take(p.hq, P * F);
    take(p.hs, P * 4);
    take(p.y, P * H * 4);
    return p;
}

static bool moe_i8_shape(const chimere_moe_i8_layer* L, int K, int T) {
    const int64_t lim = (int64_t)1 << 31;
    return L->hidden >= 16 && L->hidden % 16 == 0 && L->hidden <= I8_MAX_C && L->ffn >= 16 && L->ffn % 16 == 0 &&
           L->ffn <= I8_MAX_C && (int64_t)L->hidden * L->ffn < lim && L->n_experts >= 1 && L->n_experts <= MAX_E &&
           K >= 1 && K <= MAX_K && T >= 0 && (int64_t)T * L->hidden < lim && (int64_t)T * K < (1 << 24);
}

}  // namespace chimere

using namespace chimere;

extern "C" {

size_t chimere_moe_i8_workspace_size(const chimere_moe_i8_layer* L, int top_k, int max_ntok) {
    if (!L || max_ntok < 1 || !moe_i8_shape(L, top_k, max_ntok)) return 0;
    return plan_moe_i8(L->hidden, L->ffn, L->n_experts, top_k, max_ntok).bytes;
}

void chimere_moe_i8(const chimere_moe_i8_layer* L, int type, const void* x, int64_t x_stride, const int* ids,
                    const float* weights, int top_k, int out_type, void* out, int64_t out_stride, int ntok,
                    void* workspace, size_t workspace_bytes, hipStream_t stream) {
    CHIMERE_REQUIRE(L, CHIMERE_ERR_ARG, "moe_i8: null pointer");
    CHIMERE_REQUIRE(float_type(type) && float_type(out_type), CHIMERE_ERR_ARG, "moe_i8: unsupported type %d / %d",
                    type, out_type);
    CHIMERE_REQUIRE(moe_i8_shape(L, top_k, ntok), CHIMERE_ERR_ARG,
                    "moe_i8: hidden=%d / ffn=%d must be multiples of 16, n_experts=%d top_k=%d ntok=%d in range",
                    L->hidden, L->ffn, L->n_experts, top_k, ntok);
    CHIMERE_REQUIRE(L->gate && L->up && L->down && L->gate_scale && L->up_scale && L->down_scale, CHIMERE_ERR_ARG,
                    "moe_i8: null weight pointer");
    CHIMERE_REQUIRE((((uintptr_t)L->gate | (uintptr_t)L->up | (uintptr_t)L->down | (uintptr_t)L->gate_scale |
                      (uintptr_t)L->up_scale | (uintptr_t)L->down_scale) & 15) == 0, CHIMERE_ERR_ARG,
                    "moe_i8: weights and scales must be 16-byte aligned");
    if (ntok == 0) return;
    CHIMERE_REQUIRE(x && ids && weights && out && workspace, CHIMERE_ERR_ARG, "moe_i8: null pointer");
    CHIMERE_REQUIRE(x_stride >= 0 && out_stride >= L->hidden, CHIMERE_ERR_ARG, "moe_i8: bad strides %lld %lld",
                    (long long)x_stride, (long long)out_stride);
    const int H = L->hidden, F = L->ffn;
    const MoeI8Plan p = plan_moe_i8(H, F, L->n_experts, top_k, ntok);
    CHIMERE_REQUIRE(workspace_bytes >= p.bytes && ((uintptr_t)workspace & 255) == 0, CHIMERE_ERR_WORKSPACE,
                    "moe_i8: workspace %zu bytes < %zu (or not 256-byte aligned)", workspace_bytes, p.bytes);
    uint8_t* w = (uint8_t*)workspace;
    MoeI8 a{};
    a.H = H; a.F = F; a.E = L->n_experts; a.K = top_k; a.T = ntok;
    a.gate = L->gate; a.up = L->up; a.down = L->down;
    a.gate_s = L->gate_scale; a.up_s = L->up_scale; a.down_s = L->down_scale;
    a.ids = ids; a.wts = weights; a.out = out; a.ldo = out_stride;
    a.xq = (int8_t*)(w + p.xq); a.xs = (float*)(w + p.xs);
    a.order = (int*)(w + p.order); a.total = (int*)(w + p.total); a.tiles = (int4*)(w + p.tiles);
    a.h = (float*)(w + p.h); a.hq = (int8_t*)(w + p.hq); a.hs = (float*)(w + p.hs); a.y = (float*)(w + p.y);
    a.tile_pairs = GuTile::BM;
    launch_i8_quantize(type, x, x_stride, (int8_t*)a.xq, H, (float*)a.xs, ntok, H, stream);
    hipLaunchKernelGGL(k_i8_plan, dim3(1), dim3(1024), 0, stream, a);
    const int fb = (F + GuTile::BN / 2 - 1) / (GuTile::BN / 2), hb = (H + DnTile::BN - 1) / DnTile::BN;
    hipLaunchKernelGGL(k_i8_gate_up, dim3((unsigned)(p.max_tiles * fb)), dim3(64 * GuTile::NW), 0, stream, a);
    launch_i8_quantize(T_F32, a.h, F, a.hq, F, a.hs, (int64_t)ntok * top_k, F, stream);
    hipLaunchKernelGGL(k_i8_down, dim3((unsigned)(p.max_tiles * hb)), dim3(64 * DnTile::NW), 0, stream, a);
    const dim3 grid((unsigned)((H + 255) / 256) * ntok);
    if (out_type == T_F32) hipLaunchKernelGGL(k_i8_combine<float>, grid, dim3(256), 0, stream, a);
    else if (out_type == T_F16) hipLaunchKernelGGL(k_i8_combine<_Float16>, grid, dim3(256), 0, stream, a);
    else hipLaunchKernelGGL(k_i8_combine<__bf16>, grid, dim3(256), 0, stream, a);
    check_launch("moe_i8");
}

}  // extern "C"
