// sample.hip -- one token per row of logits by temperature, top-k, top-p and
// min-p from a given uniform number.  The reference samples on the host
// (chimere_sampler.cpp:127-392, through libllama's chain); this is a form of
// its own, whose definition stands in chimere_hip.h.
#include <math.h>

#include <type_traits>

#include "api_internal.h"
#include "float_rows.h"

namespace chimere {

struct Sample {
    const void* logits;
    const float *u, *temperature, *top_p, *min_p;
    const int* top_k;
    int* token;
    float* logprob;
    int64_t ld;
    float temperature_all, top_p_all, min_p_all;
    int top_k_all, V, bits;     // weights are multiples of 2^-bits
    int chunks;                 // of a row
    struct SampleChunk* chunk;  // [rows][chunks]
    float* tops;                // [rows][chunks][SAMPLE_CHUNK / 256]: the largest logit of each piece
    uint64_t* bins;             // [rows][chunks][SAMPLE_BINS]
};

// Order of the logits as unsigned numbers (-0 as 0; NaN as -inf, which is never
// taken: smaller than KEY_LOW, the key of the lowest number).
constexpr uint32_t KEY_LOW = 0x00800000u;
__device__ __forceinline__ uint32_t logit_key(float x) {
    const uint32_t b = __float_as_uint(x + 0.0f);
    return x != x ? 0u : b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float key_logit(uint32_t k) {
    return __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k);
}

// Weights are powers of two: 2^(k / 128 + f / 128) with k the nearest whole
// number of 128ths of an octave to d per (so that it grows with d) and |f| <=
// 1/2, both exact to the last place of f through the fma.  A table has the
// 2^(j / 128), Taylor's polynomial of degree 4 of e^(f ln 2 / 128) the rest, to
// 2e-15; k's upper bits go into the exponent.
constexpr double SAMPLE_MAGIC = 6755399441055744.0;     // 1.5 * 2^52: a sum with it has its nearest integer in the low bits
constexpr int SAMPLE_TABLE = 128;
__device__ __forceinline__ int low_word(double m) { return (int)(uint32_t)__builtin_bit_cast(uint64_t, m); }
// The polynomial's coefficients: each held in registers of its own, so that none is copied for every power (first launch of
// 256 rows of 151936 f32: 52.8 us for 55.0).
struct PowerSeries {
    double c1, c2, c3, c4;
    __device__ __forceinline__ PowerSeries() {
        constexpr double L = 0.69314718055994530942 / SAMPLE_TABLE;
        c1 = L; c2 = L * L / 2; c3 = L * L * L / 6; c4 = L * L * L * L / 24;
        __asm__("" : "+v"(c1), "+v"(c2), "+v"(c3), "+v"(c4));
    }
};
// k counts from `magic` - SAMPLE_MAGIC; at -1000 octaves and below the exponent wraps round
__device__ __forceinline__ double power_of(double d, double per, double magic, const double* table, int& k, const PowerSeries& c) {
    const double m = __builtin_fma(d, per, magic);
    k = low_word(m);
    const double f = __builtin_fma(d, per, magic - m);
    double p = __builtin_fma(c.c4, f, c.c3);
    p = __builtin_fma(p, f, c.c2);
    p = __builtin_fma(p, f, c.c1);
    p = __builtin_fma(p, f, 1.0);
    const uint64_t v = __builtin_bit_cast(uint64_t, table[k & (SAMPLE_TABLE - 1)] * p);
    return __builtin_bit_cast(double, (uint64_t)((uint32_t)(v >> 32) + ((uint32_t)(k & ~(SAMPLE_TABLE - 1)) << 13)) << 32 | (uint32_t)v);
}
// the nearest integer of a power below 2^52
__device__ __forceinline__ uint64_t whole_of(double v) {
    return __builtin_bit_cast(uint64_t, v + 4503599627370496.0) & 0xFFFFFFFFFFFFFull;
}
// the table's entries by the first threads: Taylor's polynomial of degree 13 of e^(ln 2 j / 128 - ln 2 / 2)
__device__ __forceinline__ void octave_table(double* table) {
    if (threadIdx.x < SAMPLE_TABLE) {
        const double g = ((double)(int)threadIdx.x - SAMPLE_TABLE / 2) * (0.69314718055994530942 / SAMPLE_TABLE);
        double p = 1.0 / 6227020800;
        p = __builtin_fma(p, g, 1.0 / 479001600);
        p = __builtin_fma(p, g, 1.0 / 39916800);
        p = __builtin_fma(p, g, 1.0 / 3628800);
        p = __builtin_fma(p, g, 1.0 / 362880);
        p = __builtin_fma(p, g, 1.0 / 40320);
        p = __builtin_fma(p, g, 1.0 / 5040);
        p = __builtin_fma(p, g, 1.0 / 720);
        p = __builtin_fma(p, g, 1.0 / 120);
        p = __builtin_fma(p, g, 1.0 / 24);
        p = __builtin_fma(p, g, 1.0 / 6);
        p = __builtin_fma(p, g, 0.5);
        p = __builtin_fma(p, g, 1.0);
        p = __builtin_fma(p, g, 1.0);
        table[threadIdx.x] = threadIdx.x == 0 ? 1.0 : p * 1.41421356237309504880;       // 2^(1/2)
    }
}

// log of a weight of 2^octaves, `whole` as an integer, among weights of `all`
__device__ __noinline__ float weight_logprob(double octaves, uint64_t whole, uint64_t all) {
    const uint64_t rest = all - whole;
    if (rest == 0) return 0.0f;
    if (rest < whole) return (float)log1p(-((double)rest / (double)all));
    return (float)(octaves * 0.69314718055994530942 - log((double)all));
}

// Weights as integers, 2^bits for the power of two above the largest: their sums
// are exact in any order, so a cut and the sums on both sides of it agree, and
// results repeat bit for bit.  64 bits hold 2^20 weights of 42 bits or, of
// 151936, 44: a weight is off by 2^-45, where 32 bits would be off by 2^-24 of
// it and move a token of one row in ten thousand.  In chunks of a row the power
// of two is the one above the chunk's largest, in what the first launch adds up
// and in what the second adds up and draws from of the chunk: what a chunk
// keeps, rounded down to the row's last bit, is its share of the row, and the
// token is where its own weights reach the same part of their sum, so that it
// is always found and never a logit of weight 0.
struct Weights {
    float top;                  // the largest logit, at d = d_top; others at d = x - from
    double d_top, from, per;    // d per: 128ths of an octave
    double most;                // of |d|: k's 32 bits
    double magic;               // SAMPLE_MAGIC + 128 (bits - less), less: the octaves of the power of two above all weights
    const double* table;
    __device__ __forceinline__ Weights(float top_, double d_top_, double from_, double per_, int less, int bits, const double* table_)
        : top(top_), d_top(d_top_), from(from_), per(per_), most(__builtin_fmin(0x1p30 / per_, 0x1p1000)), magic(SAMPLE_MAGIC + SAMPLE_TABLE * (double)(bits - less)), table(table_) {}
    __device__ __forceinline__ double d(float x) const {
        return x == top ? d_top : __builtin_fmin(__builtin_fmax((double)x - from, -most), most);
    }
    __device__ __forceinline__ uint64_t whole(float x) const {
        int k;
        const double v = power_of(d(x), per, magic, table, k, PowerSeries());
        return k < -30 * SAMPLE_TABLE ? 0 : whole_of(v);
    }
    // and in a chunk whose power of two lies that many octaves lower: what of_chunk(octaves).whole(x) is
    __device__ __forceinline__ uint64_t whole(float x, int octaves, uint64_t& in_chunk) const {
        int k;
        const double v = power_of(d(x), per, magic, table, k, PowerSeries());
        const uint64_t b = __builtin_bit_cast(uint64_t, v) + ((uint64_t)(uint32_t)octaves << 52);
        in_chunk = k + octaves * SAMPLE_TABLE < -30 * SAMPLE_TABLE ? 0 : whole_of(__builtin_bit_cast(double, b));
        return k < -30 * SAMPLE_TABLE ? 0 : whole_of(v);
    }
    // relative to the largest
    __device__ __forceinline__ double real(float x) const {
        if (x == top) return 1.0;
        int k;
        const double v = power_of(__builtin_fmax((double)x - (double)top, -most), per, SAMPLE_MAGIC, table, k, PowerSeries());
        return k < -1000 * SAMPLE_TABLE ? 0.0 : v;
    }
    // of a chunk, below a power of two that lies that many octaves lower
    __device__ __forceinline__ Weights of_chunk(int octaves) const {
        Weights v = *this;
        v.magic += SAMPLE_TABLE * (double)octaves;
        return v;
    }
    // sixteenths of an octave
    __device__ __forceinline__ int level(float x) const { return low_word(__builtin_fma(d(x), per, magic)) >> 3; }
    __device__ __forceinline__ float logprob(float x, uint64_t all) const {
        return weight_logprob((d(x) * per + (magic - SAMPLE_MAGIC)) * (1.0 / SAMPLE_TABLE), whole(x), all);
    }
};

constexpr int SAMPLE_THREADS = 1024, SAMPLE_WAVES = 16;
// Logits of a work-group of the first launch, 32 of each of its threads (256 rows of 151936 f32, when this took 65 us in all: 16
// of 1024 threads 75, 64 of 256 72; one row 7.9, 7.4 and 12.4)
constexpr int SAMPLE_CHUNK = 16384, SCAN_THREADS = 512;
constexpr int SAMPLE_CHUNKS = 64;        // of a row at most
constexpr int SAMPLE_MAX_VOCAB = SAMPLE_CHUNK * SAMPLE_CHUNKS;
constexpr int SAMPLE_BINS = 1024;        // of a chunk, a sixteenth of an octave each; the last: all below
constexpr int SAMPLE_CUT_BINS = 2048;    // of find_key
constexpr int SAMPLE_EARLY = 16;         // chunks whose bins are loaded before anything else is known
constexpr int SAMPLE_LIST = 8192;        // logits around a cut that are kept in LDS
constexpr int SAMPLE_TOP_K = 2048;       // that a list is made for
constexpr int SAMPLE_WHOLE = 1024;       // logits of a row that is all in the list (2000 by one launch: 32 us, by two 20)
constexpr int SAMPLE_SORT = 1024;       // that are sorted, one of each thread
constexpr int SAMPLE_PIECES = SAMPLE_MAX_VOCAB / 256;     // of 64 accesses of 16 bytes, of a row at most
constexpr int SAMPLE_FEW = 128;          // of which each adds up those before it by itself (one row, 64: second launch 15.2 us, by a second order 16.0; 128: 18.3 and 18.2; 190: 21.2 and 20.0)
constexpr int SAMPLE_SEG = 1024, SAMPLE_SEGS = SAMPLE_MAX_VOCAB / SAMPLE_SEG;

// What a row asks for.  ALL: nothing is left out; TOP: a top_k, found by counts;
// SHARE: top_p or min_p of all, found by sums; ROW: anything else, by the row itself.
enum { GREEDY, ALL, TOP, SHARE, ROW };
struct Settings {
    float t, p;
    int k, mode;
    double least;
    __device__ __forceinline__ Settings(const Sample& a, int64_t r) {
        t = a.temperature ? a.temperature[r] : a.temperature_all;
        k = a.top_k ? a.top_k[r] : a.top_k_all;
        p = a.top_p ? a.top_p[r] : a.top_p_all;
        const float low = a.min_p ? a.min_p[r] : a.min_p_all;
        least = low > 0.0f ? (low < 1.0f ? (double)low : 1.0) : 0.0;
        const bool some = k > 0 && k < a.V;
        mode = !(t > 0.0f) ? GREEDY : some ? (k <= SAMPLE_TOP_K ? TOP : ROW) : p < 1.0f || least > 0.0 ? SHARE : ALL;
    }
};

// What the first launch leaves of a chunk, next to its bins (counts or sums).
struct SampleChunk {
    uint64_t best, mass;    // key of the largest above the complement of its index (GREEDY) or 0; sum of the weights below 2^less
    uint32_t top;           // key of the largest, 0 where there is none, or none that could matter to a row without +inf
    int k, less;            // its octave in 128ths; the power of two above it
    int unused;
};
// Octaves from 0 that rows in chunks are done with (a temperature of a hundred
// thousandth at usual logits), and that a chunk of such a row can lie below it.
constexpr double SAMPLE_NEAR = 0x1p20, SAMPLE_FAR = 0x1p21;
constexpr double SAMPLE_LEAST_PER = 1e-30;      // 70 octaves are inside f32's range

__device__ __forceinline__ uint64_t shfl_xor64(uint64_t v, int d) {
    return (uint64_t)(uint32_t)__shfl_xor((int)(v >> 32), d) << 32 | (uint32_t)__shfl_xor((int)v, d);
}
template <int M>
__device__ __forceinline__ uint64_t xlane64(uint64_t v) {
    return (uint64_t)(uint32_t)xlane<M>((int)(v >> 32)) << 32 | (uint32_t)xlane<M>((int)v);
}
template <int CTRL, int ROWS>
__device__ __forceinline__ uint64_t dpp_add64(uint64_t v) {
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xF, false);
    const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(v >> 32), CTRL, ROWS, 0xF, false);
    return v + ((uint64_t)hi << 32 | lo);
}
// inclusive sums over the wave (the steps of wave_incl_scan)
__device__ __forceinline__ uint64_t wave_scan64(uint64_t v) {
    v = dpp_add64<0x111, 0xF>(v);
    v = dpp_add64<0x112, 0xF>(v);
    v = dpp_add64<0x114, 0xF>(v);
    v = dpp_add64<0x118, 0xF>(v);
    v = dpp_add64<0x142, 0xA>(v);
    return dpp_add64<0x143, 0xC>(v);
}
__device__ __forceinline__ uint64_t readlane64(uint64_t v, int lane) {
    return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), lane) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)v, lane);
}
__device__ __forceinline__ uint64_t last_lane64(uint64_t v) { return readlane64(v, 63); }
// Sums and maxima over a work-group, one barrier each: they take turns with two rows of LDS.
template <int WAVES>
struct BlockOf {
    uint64_t (*part)[WAVES];
    int turn = 0;
    // inclusive sums over the threads; `all`: the last
    __device__ __forceinline__ uint64_t scan(uint64_t v, uint64_t& all) {
        v = wave_scan64(v);
        uint64_t* p = part[turn ^= 1];
        if ((threadIdx.x & 63) == 63) p[threadIdx.x >> 6] = v;
        __syncthreads();
        uint64_t first = 0;
        all = 0;
#pragma unroll
        for (int w = 0; w < WAVES; w++) {
            if (w < (int)(threadIdx.x >> 6)) first += p[w];
            all += p[w];
        }
        return v + first;
    }
    __device__ __forceinline__ uint64_t sum(uint64_t v) {
        uint64_t all;
        scan(v, all);
        return all;
    }
    __device__ __forceinline__ uint64_t max(uint64_t v) {
        auto larger = [](uint64_t x, uint64_t y) { return x > y ? x : y; };
        v = larger(v, xlane64<32>(v));
        v = larger(v, xlane64<16>(v));
        v = larger(v, xlane64<8>(v));
        v = larger(v, xlane64<4>(v));
        v = larger(v, xlane64<2>(v));
        v = larger(v, xlane64<1>(v));
        uint64_t* p = part[turn ^= 1];
        if ((threadIdx.x & 63) == 0) p[threadIdx.x >> 6] = v;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < WAVES; w++) v = larger(v, p[w]);
        return v;
    }
};
typedef BlockOf<SAMPLE_WAVES> Block;
__device__ __forceinline__ float no_nan(float x) { return x == x ? x + 0.0f : -__builtin_huge_valf(); }

template <typename T, int V>
__device__ __forceinline__ void logits_load(const T* row, int i, int end, float (&x)[V]) {
    typedef typename VecOf<T, V>::type vec;
    if (i + V <= end) {
        const vec v = *(const vec*)(row + i);
#pragma unroll
        for (int j = 0; j < V; j++) x[j] = no_nan((float)v[j]);
    } else {
#pragma unroll
        for (int j = 0; j < V; j++) x[j] = i + j < end ? no_nan(load_f(row + i + j)) : -__builtin_huge_valf();
    }
}

// First launch: a chunk's largest logit, then, with its weights relative to the
// power of two above that, their sum and how much of it (or how many) lies in
// each sixteenth of an octave (the last bin has all below: it is not used).
// The bins lie at the same places in all chunks of a row, since octaves are
// counted from 0: no launch before it has to find the row's largest logit.
// The largest alone (temperature 0) takes 27 us of 256 rows of 151936 f32, 156
// MB, 5.8 TB/s; counts (top-k) 39.  With weights it takes 47 to 50 us: seven
// operations in 64 bits and an atomic addition in LDS per logit, in bf16 too (45
// us where bytes are half).  One row: 7.6 us.
template <typename T>
__global__ __launch_bounds__(SCAN_THREADS, 8) void k_sample_scan(Sample a, int64_t row0) {
    constexpr int THREADS = SCAN_THREADS;
    __shared__ uint64_t hist[SAMPLE_BINS], part[2][THREADS / 64];
    BlockOf<THREADS / 64> block{part};
    __shared__ double table[SAMPLE_TABLE];
    constexpr int V = 16 / sizeof(T), N = SAMPLE_CHUNK / THREADS / V;
    const int tid = threadIdx.x, c = blockIdx.x % a.chunks;
    const int64_t local = blockIdx.x / a.chunks, r = row0 + local;
    const T* row = (const T*)a.logits + r * a.ld;
    const int i0 = c * SAMPLE_CHUNK + tid * V;
    float x[N][V], top = -__builtin_huge_valf();
#pragma unroll
    for (int i = 0; i < N; i++) logits_load(row, i0 + i * THREADS * V, a.V, x[i]);
    const Settings s(a, r);
    if (s.mode == ROW) return;
    octave_table(table);
    for (int b = tid; b < SAMPLE_BINS; b += THREADS) hist[b] = 0;
#pragma unroll
    for (int i = 0; i < N; i++)
#pragma unroll
        for (int j = 0; j < V; j++) top = __builtin_fmaxf(top, x[i][j]);
    // of a wave's piece of 64 accesses, for the second launch to see which of them to read again
    if (s.mode == TOP) {
#pragma unroll
        for (int i = 0; i < N; i++) {
            float m = x[i][0];
#pragma unroll
            for (int j = 1; j < V; j++) m = __builtin_fmaxf(m, x[i][j]);
            m = wave_join(m, [](float u, float v) { return __builtin_fmaxf(u, v); });
            if ((tid & 63) == 0) a.tops[(int64_t)blockIdx.x * (SAMPLE_CHUNK / 256) + i * (THREADS / 64) + (tid >> 6)] = m;
        }
    }
    // with the largest of each lane above it 64 logits are: none below it is among the first 64
    float least = -3.402823466e38f;
    if (s.mode == TOP && s.k <= 64) least = __builtin_fmaxf(least, wave_join(top, [](float u, float v) { return __builtin_fminf(u, v); }));
    uint64_t best = (uint64_t)logit_key(top) << 32;
    if (s.mode == GREEDY) {
#pragma unroll
        for (int i = N - 1; i >= 0; i--)
#pragma unroll
            for (int j = V - 1; j >= 0; j--)
                if (x[i][j] == top) best = (best & ~0xFFFFFFFFull) | (uint32_t)~(i0 + i * THREADS * V + j);
    }
    best = block.max(best);
    SampleChunk* to = a.chunk + blockIdx.x;
    const uint32_t key = (uint32_t)(best >> 32);
    const double per = 1.44269504088896340736 * SAMPLE_TABLE / (double)s.t, d = (double)key_logit(key);
    const bool near = key >= KEY_LOW && per >= SAMPLE_LEAST_PER && __builtin_fabs(d * per) < SAMPLE_FAR * SAMPLE_TABLE;
    const int k = near ? low_word(__builtin_fma(d, per, SAMPLE_MAGIC)) : 0, less = (k >> 7) + 1;
    uint64_t mass = 0, all = 0;
    if (s.mode != GREEDY && near) {
        const double magic = SAMPLE_MAGIC + SAMPLE_TABLE * (double)(a.bits - less);
        const int low = (k + SAMPLE_TABLE * (a.bits - less)) & ~7, end = 8 * (SAMPLE_BINS - 1);    // bins of eight bytes
        // 70 octaves below the chunk's largest a weight is 0, and no further down the octaves' 32 bits hold: a mask's -1e9 would
        // wrap round to any bin.  (-inf and what is behind the row's end would all be added to the last bin, one after the
        // other, too: 80 us for 256 rows instead of 57, then.)
        least = __builtin_fmaxf(least, (float)((double)(k - 70 * SAMPLE_TABLE) / per));
        if (s.mode == TOP) {
#pragma unroll
            for (int i = 0; i < N; i++)
#pragma unroll
                for (int j = 0; j < V; j++)
                    if (x[i][j] >= least) {
                        const int at = min(low - (low_word(__builtin_fma((double)x[i][j], per, magic)) & ~7), end);
                        atomicAdd((unsigned long long*)((uint8_t*)hist + at), 1ull);
                    }
            __syncthreads();
        } else {
            const PowerSeries series;
#pragma unroll
            for (int i = 0; i < N; i++)
#pragma unroll
                for (int j = 0; j < V; j++) {
                    if (!(x[i][j] >= least)) continue;
                    int o;
                    const uint64_t w = whole_of(power_of((double)x[i][j], per, magic, table, o, series));
                    mass += w;
                    atomicAdd((unsigned long long*)((uint8_t*)hist + min(low - (o & ~7), end)), (unsigned long long)w);
                }
            all = block.sum(mass);
        }
        uint64_t* bins = a.bins + (int64_t)blockIdx.x * SAMPLE_BINS;
        for (int b = tid; b < SAMPLE_BINS; b += THREADS) {
            if (s.mode != ALL) bins[b] = hist[b];
        }
    }
    if (tid == 0) *to = SampleChunk{best, all, near ? key : 0, k, less, 0};
}

// What is kept of a row: keys above `key` and the first `ties` (by index) of those equal to it
struct Cut {
    uint32_t key;
    int64_t ties;
};

// The first key above lo, which is none of them, whose logit is one of those that on(x) says, which go up to all above; hi, where
// no key below it is one.  By a wave, 64 at a time.
template <typename On>
__device__ __forceinline__ uint32_t first_key(uint32_t lo, uint32_t hi, On on) {
    while (hi - lo > 1) {
        const uint32_t step = (hi - lo + 63) / 64, k = min(lo + ((threadIdx.x & 63) + 1) * step, hi);
        const int f = __ffsll((unsigned long long)__ballot((k == hi) | on(key_logit(k)))) - 1;
        hi = min(lo + (uint32_t)(f + 1) * step, hi);
        lo += (uint32_t)f * step;
    }
    return hi;
}
// of logits of that level or above
__device__ __forceinline__ uint32_t level_start(const Weights& w, int level, uint32_t lo, uint32_t hi) {
    return first_key(lo, hi, [&](float x) { return w.level(x) >= level; });
}
// of logits whose probability is at least `least` of the largest: the comparison of each is what counts, around the logit that it
// comes to by the logarithm
__device__ __forceinline__ uint32_t least_start(const Weights& w, double least, uint32_t top) {
    const double below = SAMPLE_TABLE * log2(least) / w.per, v = (double)w.top + below;
    const double far = __builtin_fabs(v) * 1e-6 + (__builtin_fabs((double)w.top) - below) * 1e-12 + 1e-9 / w.per;
    const uint32_t lo = logit_key((float)__builtin_fmax(v - far, -3.402823466e38)), hi = logit_key((float)__builtin_fmin(v + far, (double)w.top));
    return first_key(lo - 1, min(hi, top), [&](float x) { return w.real(x) >= least; });
}

struct SampleLds {
    Sample args;
    uint64_t part[2][SAMPLE_WAVES], kept[SAMPLE_CHUNKS];
    double table[SAMPLE_TABLE];
    SampleChunk head[SAMPLE_CHUNKS];
    int ties[SAMPLE_CHUNKS];    // of each chunk: equals at the cut in it
    int shift[SAMPLE_CHUNKS], less[SAMPLE_CHUNKS];     // bins and octaves that it lies below the row's
    uint64_t above, found, with;
    uint32_t edge[2];
    int bin, n;
    union {
        uint64_t hist[SAMPLE_CUT_BINS];
        uint64_t sorted[2][SAMPLE_SORT];
        struct {
            uint64_t mass[SAMPLE_SEGS];
            int ties[SAMPLE_SEGS];
        } seg;
    };
    uint32_t key[SAMPLE_LIST], index[SAMPLE_LIST];      // the list, in any order
    uint16_t read[SAMPLE_PIECES];                       // the pieces of the row that are read
};

// The key at which the sum over the elements in descending order of their keys reaches `need`, and the sum above it; 0 where
// all of them do not.  A histogram of 2048 parts of the keys' range, then of the part where it does, until that is a single
// key.  each(f): f(key, what it adds) for every element of this thread with a key from lo to hi.
struct Found {
    uint32_t key;
    uint64_t above;
};
template <typename Each>
__device__ __forceinline__ Found find_key(SampleLds& s, Block& block, uint32_t lo, uint32_t hi, uint64_t need, Each each) {
    const int tid = threadIdx.x;
    uint64_t above = 0;
    for (;;) {
        const int width = 32 - __clz((int)(hi - lo)), shift = hi == lo || width < 11 ? 0 : width - 11;
        __syncthreads();
        for (int b = tid; b < SAMPLE_CUT_BINS; b += SAMPLE_THREADS) s.hist[b] = 0;
        if (tid == 0) s.bin = -1;
        __syncthreads();
        each([&](uint32_t k, uint64_t v) {
            if (k >= lo && k <= hi) atomicAdd((unsigned long long*)&s.hist[(k - lo) >> shift], (unsigned long long)v);
        });
        __syncthreads();
        // two bins of each thread, from the top
        const int b1 = SAMPLE_CUT_BINS - 1 - 2 * tid, b0 = b1 - 1;
        const uint64_t h1 = s.hist[b1], h0 = s.hist[b0];
        uint64_t all;
        const uint64_t upto = above + block.scan(h1 + h0, all);
        const uint64_t past1 = upto - h0, past0 = past1 - h1;
        if (past0 < need && upto >= need) {
            const bool second = past1 < need;
            s.bin = second ? b0 : b1;
            s.above = second ? past1 : past0;
        }
        __syncthreads();
        if (s.bin < 0) return {0u, above};
        above = s.above;
        lo += (uint32_t)s.bin << shift;
        if (shift == 0) return {lo, above};
        hi = lo + min(hi - lo, (1u << shift) - 1);
    }
}
// The cut after the first k of the elements each(f): f(logit, index); keys are lo to hi.
template <typename Each>
__device__ __forceinline__ Cut count_cut(SampleLds& s, Block& block, uint32_t lo, uint32_t hi, uint64_t k, Each each) {
    const Found f = find_key(s, block, lo, hi, k, [&](auto g) { each([&](float x, uint32_t) { g(logit_key(x), 1); }); });
    return f.key ? Cut{f.key, (int64_t)(k - f.above)} : Cut{lo - 1, 0};
}
// And where their weights reach `need`.
template <typename Each>
__device__ __forceinline__ Cut mass_cut(SampleLds& s, Block& block, const Weights& w, uint32_t lo, uint32_t hi, uint64_t need, Each each) {
    const Found f = find_key(s, block, lo, hi, need, [&](auto g) {
        each([&](float x, uint32_t) {
            const uint32_t key = logit_key(x);
            if (key >= lo && key <= hi) g(key, w.whole(x));
        });
    });
    if (!f.key) return {lo - 1, 0};
    const uint64_t one = w.whole(key_logit(f.key));
    return {f.key, (int64_t)((need - f.above + one - 1) / one)};
}

// The wave's, then the work-group's elements in descending order: a bitonic
// network over the first `size` threads (a power of two, 64 at least), an
// element each; within a wave by lane exchanges, else through LDS.
template <int M>
__device__ __forceinline__ uint64_t sort_step(uint64_t v, bool first) {
    const uint64_t u = xlane64<M>(v);
    return (u > v) == first ? u : v;
}
__device__ __forceinline__ uint64_t sort_wave(uint64_t v, int k) {
    const int t = threadIdx.x;
    const bool down = !(t & k);     // this run of k is in descending order
    switch (k) {
    default: v = sort_step<32>(v, down == !(t & 32)); [[fallthrough]];
    case 32: v = sort_step<16>(v, down == !(t & 16)); [[fallthrough]];
    case 16: v = sort_step<8>(v, down == !(t & 8)); [[fallthrough]];
    case 8: v = sort_step<4>(v, down == !(t & 4)); [[fallthrough]];
    case 4: v = sort_step<2>(v, down == !(t & 2)); [[fallthrough]];
    case 2: v = sort_step<1>(v, down == !(t & 1));
    }
    return v;
}
__device__ __forceinline__ uint64_t sort_down(SampleLds& s, uint64_t v, int size) {
    const int t = threadIdx.x;
    v = sort_wave(v, 2);
    v = sort_wave(v, 4);
    v = sort_wave(v, 8);
    v = sort_wave(v, 16);
    v = sort_wave(v, 32);
    v = sort_wave(v, 64);
    int turn = 0;
    for (int k = 128; k <= size; k *= 2) {
        const bool down = !(t & k);
        for (int j = k / 2; j >= 64; j /= 2) {
            s.sorted[turn][t] = v;
            __syncthreads();
            const uint64_t u = s.sorted[turn][t ^ j];
            turn ^= 1;
            v = (u > v) == (down == !(t & j)) ? u : v;
        }
        v = sort_wave(v, k);
    }
    return v;
}

// the smallest whole sum that is at least the share p of `all`, one at least
__device__ __forceinline__ uint64_t share_of(float p, uint64_t all) {
    const double want = p > 0.0f ? __builtin_ceil((double)p * (double)all) : 1.0;
    const uint64_t need = want < 1.0 ? 1 : (uint64_t)want;
    return need < all ? need : all;
}
// the largest whole sum that is at most u of `all`, below all
__device__ __forceinline__ uint64_t part_of(float u, uint64_t all) {
    const uint64_t want = u > 0.0f ? (uint64_t)__builtin_floor((double)(u < 1.0f ? u : 1.0f) * (double)all) : 0;
    return want < all ? want : all - 1;
}

// of the first k (0: all), then of the share p of these (1 and more: all)
template <typename Each>
__device__ __forceinline__ Cut find_cuts(SampleLds& s, Block& block, const Weights& w, uint32_t top, int k, float p, Each each) {
    Cut cut{KEY_LOW - 1, 0};
    if (k > 0) cut = count_cut(s, block, KEY_LOW, top, (uint64_t)k, each);
    if (p < 1.0f) {
        uint64_t mass = 0;
        each([&](float x, uint32_t) {
            if (logit_key(x) > cut.key) mass += w.whole(x);
        });
        uint64_t all = block.sum(mass);
        if (cut.ties) all += (uint64_t)cut.ties * w.whole(key_logit(cut.key));
        const Cut c = mass_cut(s, block, w, cut.ties ? cut.key : cut.key + 1, top, share_of(p, all), each);
        cut = c.key == cut.key && cut.ties && cut.ties < c.ties ? cut : c;
    }
    return cut;
}
// The cut where probabilities come below `least` of the largest, if that is the shorter one
template <typename Each>
__device__ __forceinline__ Cut least_cut(Block& block, const Weights& w, const Cut& cut, double least, Each each) {
    uint64_t low = 0;       // complement of the smallest key that stays
    each([&](float x, uint32_t) {
        const uint32_t key = logit_key(x);
        if ((key > cut.key || (cut.ties && key == cut.key)) && (uint64_t)(uint32_t)~key > low && w.real(x) >= least) low = (uint32_t)~key;
    });
    low = block.max(low);
    const uint32_t end = low ? (uint32_t)~(uint32_t)low - 1 : ~0u;
    return end >= cut.key ? Cut{end, 0} : cut;
}

// The token among `count` elements in the order of their indexes: the first at which the kept weights, summed up, exceed
// want(their sum).  get(e, x, i): element e, false where it is none; kept(x): whether it is, equals at the cut apart, of which
// the first `ties` are.  w: the weights; row, all_of_row: what the probability is formed by (0: their sum).
template <typename Want, typename Get, typename Kept>
__device__ __forceinline__ void pick(SampleLds& s, Block& block, const Sample& a, int64_t r, const Weights& w, const Weights& row, const Cut& cut,
                                     int64_t ties, int count, bool equals_stay, uint64_t all_of_row, Want want_of, Get get, Kept kept) {
    const int tid = threadIdx.x, lane = tid & 63, segs = (count + SAMPLE_SEG - 1) / SAMPLE_SEG;
    const uint64_t of_tie = cut.ties && equals_stay ? w.whole(key_logit(cut.key)) : 0;
    // weight of an element; equals at the cut apart
    auto weigh = [&](bool on, float x, bool& tie) -> uint64_t {
        tie = on && cut.ties && logit_key(x) == cut.key;
        return on && !tie && kept(x) ? w.whole(x) : 0;
    };
    float x = 0.0f;
    int i = 0;
    bool tie;
    __syncthreads();
#pragma unroll 1
    for (int g = tid >> 6; g < segs; g += SAMPLE_WAVES) {
        uint64_t mass = 0;
        int equals = 0;
#pragma unroll 1
        for (int e = g * SAMPLE_SEG + lane; e < (g + 1) * SAMPLE_SEG; e += 256) {
            float y[4];
            bool on[4];
#pragma unroll
            for (int j = 0; j < 4; j++) on[j] = e + 64 * j < count && get(e + 64 * j, y[j], i);
#pragma unroll
            for (int j = 0; j < 4; j++) {
                mass += weigh(on[j], y[j], tie);
                equals += __popcll(__ballot(tie));
            }
        }
        mass = wave_scan64(mass);
        if (lane == 63) {
            s.seg.mass[g] = mass;
            s.seg.ties[g] = equals;
        }
    }
    __syncthreads();
    uint64_t all;
    const int mine = tid < segs ? s.seg.ties[tid] : 0;
    int64_t room = ties;
    if (cut.ties) room -= (int64_t)block.scan(mine, all) - mine;
    const uint64_t some = room <= 0 ? 0 : room < mine ? room : mine;
    const uint64_t mass = (tid < segs ? s.seg.mass[tid] : 0) + some * of_tie;
    const uint64_t upto = block.scan(mass, all), want = want_of(all);
    if (all_of_row == 0) all_of_row = all;
    if (upto > want && upto - mass <= want) {
        s.bin = tid;
        s.above = upto - mass;
        s.found = (uint64_t)(room <= 0 ? 0 : room);
    }
    __syncthreads();
    const int e = s.bin * SAMPLE_SEG + tid;
    const bool on = e < count && get(e, x, i);
    const uint64_t v0 = weigh(on, x, tie);
    int64_t rank = 0;
    if (cut.ties) rank = (int64_t)block.scan(tie, all) - tie;
    const uint64_t v = tie ? (rank < (int64_t)s.found ? of_tie : 0) : v0;
    const uint64_t past = s.above + block.scan(v, all) - v;
    if (past <= want && past + v > want) {
        a.token[r] = i;
        a.logprob[r] = row.logprob(x, all_of_row);
    }
}

// A row by itself, read again for every step: for what the launches below have no list for.  (The kernel's arguments from
// LDS, where the caller has put them: a reference to the others would keep them in scratch memory.)
template <typename T>
__device__ __noinline__ void sample_row(SampleLds& s, int64_t r) {
    const Sample& a = s.args;
    const Settings o(a, r);
    const int tid = threadIdx.x, V = a.V;
    const T* row = (const T*)a.logits + r * a.ld;
    Block block{s.part};
    auto each = [&](auto f) {
#pragma unroll 4
        for (int i = tid; i < V; i += SAMPLE_THREADS) f(no_nan(load_f(row + i)), (uint32_t)i);
    };
    uint64_t best = 0;
    each([&](float x, uint32_t i) {
        const uint64_t v = (uint64_t)logit_key(x) << 32 | ~i;
        best = v > best ? v : best;
    });
    __syncthreads();
    best = block.max(best);
    const uint32_t top = (uint32_t)(best >> 32);
    if (top < KEY_LOW || o.mode == GREEDY) {
        if (tid == 0) {
            a.token[r] = top < KEY_LOW ? -1 : (int)~(uint32_t)best;
            a.logprob[r] = top < KEY_LOW ? -__builtin_huge_valf() : 0.0f;
        }
        return;
    }
    const float most = key_logit(top);
    const Weights w(most, 0.0, most, 1.44269504088896340736 * SAMPLE_TABLE / (double)o.t, 0, a.bits, s.table);
    const Cut cut = find_cuts(s, block, w, top, o.k < V ? o.k : 0, o.p, each);
    const float u = a.u[r];
    pick(s, block, a, r, w, w, cut, cut.ties, V, cut.ties && w.real(key_logit(cut.key)) >= o.least, 0, [&](uint64_t all) { return part_of(u, all); },
         [&](int e, float& x, int& i) {
             x = no_nan(load_f(row + e));
             i = e;
             return x > -__builtin_huge_valf();
         },
         [&](float x) { return logit_key(x) > cut.key && w.real(x) >= o.least; });
}

// hit(on, x, index) of a row's logits from lo to hi, by whole waves: `on` where the lane has one.  Pieces of 64 accesses of
// 16 bytes, SAMPLE_AHEAD of them on their way at a time.  Only pieces of `chunks` are read (bits), and only those whose
// largest, in `tops` unless that is null, is not below lo.  What is found is marked by bits and taken up one of each lane at
// a time, read again (from the first cache), so that there is one place in the code for it: a work-group runs all of this
// once, and every 64 bytes of code that it comes to it waits for.
constexpr int SAMPLE_AHEAD = 8;
template <typename T, typename Hit>
__device__ __forceinline__ void scan_row(SampleLds& s, Block& block, const T* row, int vocab, const float* tops, uint64_t chunks, float lo, float hi, Hit hit) {
    constexpr int V = 16 / sizeof(T), PIECE = 64 * V, U = SAMPLE_AHEAD, CHUNK = SAMPLE_CHUNK / PIECE;
    typedef typename VecOf<T, V>::type vec;
    typedef std::conditional_t<U * V == 32, uint32_t, uint64_t> bits;
    const int tid = threadIdx.x, lane = tid & 63, pieces = (vocab + PIECE - 1) / PIECE;
    const int each = (pieces + SAMPLE_THREADS - 1) / SAMPLE_THREADS;
    uint32_t reads = 0;
#pragma unroll 1
    for (int j = 0; j < each; j++) {
        const int p = tid * each + j;
        if (p < pieces && (chunks >> (p / CHUNK) & 1) && (!tops || tops[p / CHUNK * (SAMPLE_CHUNK / 256) + p % CHUNK] >= lo)) reads |= 1u << j;
    }
    uint64_t all;
    int at = (int)block.scan(__popc(reads), all) - __popc(reads);
    for (; reads; reads &= reads - 1) s.read[at++] = (uint16_t)(tid * each + __ffs((int)reads) - 1);
    __syncthreads();
    const int n = (int)all;
#pragma unroll 1
    for (int q0 = (tid >> 6) * U; q0 < n; q0 += SAMPLE_WAVES * U) {
        vec v[U];
        int from[U];        // the logits that v has, where it is moved to stay inside the row
#pragma unroll
        for (int u = 0; u < U; u++) {
            from[u] = (int)s.read[min(q0 + u, n - 1)] * PIECE + lane * V;
            const int i = max(min(from[u], vocab - V), 0);
            if (vocab >= V) {
                v[u] = *(const vec*)(row + i);
            } else {
#pragma unroll
                for (int j = 0; j < V; j++) v[u][j] = row[min(j, vocab - 1)];
            }
        }
        bits found = 0;
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int moved = from[u] - max(min(from[u], vocab - V), 0);
#pragma unroll
            for (int j = 0; j < V; j++)
                found |= (float)v[u][j] >= lo && (float)v[u][j] <= hi && j >= moved && j < vocab ? (bits)1 << (u * V + j) : 0;
            if (q0 + u >= n) found &= ((bits)1 << (u * V)) - 1;
        }
        while (__any(found != 0)) {
            const bool on = found != 0;
            const int b = on ? __ffsll((unsigned long long)found) - 1 : 0;
            const int i = max(min((int)s.read[min(q0 + b / V, n - 1)] * PIECE + lane * V, vocab - V), 0) + b % V;
            hit(on, on ? no_nan(load_f(row + i)) : 0.0f, (uint32_t)i);
            found &= found - 1;
        }
    }
}

// The logits of a row from lo to hi as a list in LDS, in any order: their number, or -1 where they are too many.
template <typename T>
__device__ __forceinline__ int gather(SampleLds& s, Block& block, const T* row, int vocab, const float* tops, uint64_t chunks, float lo, float hi) {
    const int tid = threadIdx.x, lane = tid & 63;
    if (tid == 0) s.n = 0;
    __syncthreads();
    scan_row(s, block, row, vocab, tops, chunks, lo, hi, [&](bool on, float x, uint32_t i) {
        const uint64_t has = __ballot(on);
        int start = 0;
        if (lane == 0) start = atomicAdd(&s.n, __popcll(has));
        start = __builtin_amdgcn_readfirstlane(start);
        const int at = start + (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(has >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)has, 0));
        if (on && at < SAMPLE_LIST) {
            s.key[at] = logit_key(x);
            s.index[at] = i;
        }
    });
    __syncthreads();
    return s.n > SAMPLE_LIST ? -1 : s.n;
}

// The token of a list that holds all that may be kept.
__device__ __forceinline__ void pick_of_list(SampleLds& s, Block& block, const Sample& a, int64_t r, const Settings& o, const Weights& w,
                                             uint32_t top, int n) {
    const int tid = threadIdx.x;
    const float u = a.u[r];
    if (n <= SAMPLE_SORT) {
        // sorted: what is kept is a first part, up to where any of the three ends it
        int size = 64;
        while (size < n) size *= 2;
        uint64_t v = sort_down(s, tid < n ? (uint64_t)s.key[tid] << 32 | ~s.index[tid] : 0, size);
        const float x = key_logit((uint32_t)(v >> 32));
        const uint32_t index = ~(uint32_t)v;
        const bool first = tid < n && (o.k <= 0 || tid < o.k);
        const uint64_t weight = first ? w.whole(x) : 0;
        uint64_t all;
        const uint64_t upto = block.scan(weight, all);
        const uint64_t need = o.p < 1.0f ? share_of(o.p, all) : ~0ull;
        const bool keep = first && upto - weight < need && (o.least <= 0.0 || w.real(x) >= o.least);
        uint64_t mine = keep ? weight : 0, past = 0;
        s.sorted[0][tid] = mine;        // (what sort_down has read there lies before the scan's barrier)
        s.index[tid] = index;
        const int m = __syncthreads_count(keep);
        // the kept weights up to each of them by index: added up by each for itself, or, of many, in a second order
        if (m <= SAMPLE_FEW) {
            all = 0;
            if (tid < m)
                for (int j = 0; j < m; j++) {
                    const uint64_t q = s.sorted[0][j];
                    all += q;
                    past += s.index[j] < index ? q : 0;
                }
            const uint64_t want = part_of(u, all);
            if (mine && past <= want && past + mine > want) {
                a.token[r] = (int)index;
                a.logprob[r] = w.logprob(x, all);
            }
            return;
        }
        s.key[tid] = (uint32_t)(v >> 32);
        size = 64;
        while (size < m) size *= 2;
        const int rank = (int)(uint32_t)sort_down(s, keep ? (uint64_t)~index << 32 | tid : 0, size);
        __syncthreads();
        const float y = key_logit(s.key[rank]);
        mine = tid < m ? w.whole(y) : 0;
        past = block.scan(mine, all) - mine;
        const uint64_t want = part_of(u, all);
        if (mine && past <= want && past + mine > want) {
            a.token[r] = (int)s.index[rank];
            a.logprob[r] = w.logprob(y, all);
        }
        return;
    }
    auto each = [&](auto f) {
#pragma unroll 1
        for (int i = tid; i < n; i += SAMPLE_THREADS) f(key_logit(s.key[i]), s.index[i]);
    };
    Cut cut = find_cuts(s, block, w, top, o.k < n ? o.k : 0, o.p, each);
    if (o.least > 0.0) cut = least_cut(block, w, cut, o.least, each);
    // the last of the equals that stay, then the token, by index: keys that fall with it
    uint32_t end = 0;
    if (cut.ties)
        end = find_key(s, block, ~(uint32_t)(a.V - 1), ~0u, (uint64_t)cut.ties, [&](auto g) {
                  each([&](float x, uint32_t i) {
                      if (logit_key(x) == cut.key) g(~i, 1);
                  });
              }).key;
    auto kept = [&](float x, uint32_t i) { return logit_key(x) > cut.key || (cut.ties && logit_key(x) == cut.key && ~i >= end); };
    uint64_t mass = 0;
    each([&](float x, uint32_t i) {
        if (kept(x, i)) mass += w.whole(x);
    });
    const uint64_t all = block.sum(mass);
    const uint32_t token = ~find_key(s, block, ~(uint32_t)(a.V - 1), ~0u, part_of(u, all) + 1, [&](auto g) {
                                each([&](float x, uint32_t i) {
                                    if (kept(x, i)) g(~i, w.whole(x));
                                });
                            }).key;
    each([&](float x, uint32_t i) {
        if (i == token) {
            a.token[r] = (int)i;
            a.logprob[r] = w.logprob(x, all);
        }
    });
}

// Second launch, a work-group per row: its chunks joined, the cut found by
// their bins, the logits around it gathered (the row is read a second time, from
// L2 or the memory-side cache, where a piece's largest or a chunk's bins do not
// rule it out), the cut's place among them, the token.  WHOLE: a short row, all
// of it as the list, with no launch before.  A chain of dependent steps bounds
// it, a dozen or two barriers of 16 waves: one row of 151936 13.3 us by top-k,
// 25 by top-p; 256 rows, one per CU, 17 us by top-k, 20 without limits, 52 to 59
// by top-p (which adds up all chunks' bins, 20 MB, and reads the cut's).  A row
// that has a top_k above SAMPLE_TOP_K, or no list, is done by sample_row (one
// row, top_k 2048: 43 us with the scan, 2049 186; 256 rows 88 and 366).
template <typename T, bool WHOLE>
__global__ __launch_bounds__(SAMPLE_THREADS) void k_sample_pick(Sample a, int64_t row0) {
    __shared__ SampleLds s;
    Block block{s.part};
    const int tid = threadIdx.x;
    const int64_t r = row0 + blockIdx.x;
    const T* row = (const T*)a.logits + r * a.ld;
    const Settings o(a, r);
    const float lowest = -3.402823466e38f, inf = __builtin_huge_valf();
    auto alone = [&] {
        if (tid == 0) s.args = a;
        __syncthreads();
        sample_row<T>(s, r);
    };
    octave_table(s.table);
    if constexpr (WHOLE) {
        const int n = gather(s, block, row, a.V, nullptr, ~0ull, lowest, inf);
        uint64_t best = 0;
        for (int i = tid; i < n; i += SAMPLE_THREADS) {
            const uint64_t v = (uint64_t)s.key[i] << 32 | (uint32_t)~s.index[i];
            best = v > best ? v : best;
        }
        best = block.max(best);
        const uint32_t top = (uint32_t)(best >> 32);
        if (n == 0 || o.mode == GREEDY) {
            if (tid == 0) {
                a.token[r] = n == 0 ? -1 : (int)~(uint32_t)best;
                a.logprob[r] = n == 0 ? -inf : 0.0f;
            }
            return;
        }
        const float most = key_logit(top);
        pick_of_list(s, block, a, r, o, Weights(most, 0.0, most, 1.44269504088896340736 * SAMPLE_TABLE / (double)o.t, 0, a.bits, s.table), top, n);
        return;
    }
    const uint64_t* bins = a.bins + (int64_t)blockIdx.x * a.chunks * SAMPLE_BINS;
    const float* tops = a.tops + (int64_t)blockIdx.x * a.chunks * (SAMPLE_CHUNK / 256);
    // the chunks' bins are on their way before it is known where they go
    uint64_t v[SAMPLE_EARLY];
#pragma unroll
    for (int c = 0; c < SAMPLE_EARLY; c++) v[c] = c < a.chunks ? bins[(int64_t)c * SAMPLE_BINS + tid] : 0;
    if (tid < a.chunks) {
        s.head[tid] = a.chunk[(int64_t)blockIdx.x * a.chunks + tid];
        s.kept[tid] = 0;
        s.ties[tid] = 0;
    }
    s.hist[tid] = 0;
    __syncthreads();
    if (o.mode == ROW) {
        alone();
        return;
    }
    // the row's largest logit and the power of two above its weights, by every wave for itself
    const bool mine = (tid & 63) < a.chunks;
    const SampleChunk head = s.head[mine ? tid & 63 : 0];
    auto larger = [](uint64_t x, uint64_t y) { return x > y ? x : y; };
    uint64_t best = mine ? head.best : 0;
    best = larger(best, xlane64<32>(best));
    best = larger(best, xlane64<16>(best));
    best = larger(best, xlane64<8>(best));
    best = larger(best, xlane64<4>(best));
    best = larger(best, xlane64<2>(best));
    best = larger(best, xlane64<1>(best));
    const int less = wave_join(mine && head.top ? head.less : -(1 << 30), [](int x, int y) { return max(x, y); });
    const uint32_t top = (uint32_t)(best >> 32);
    if (top < KEY_LOW || o.mode == GREEDY) {
        if (tid == 0) {
            a.token[r] = top < KEY_LOW ? -1 : (int)~(uint32_t)best;
            a.logprob[r] = top < KEY_LOW ? -inf : 0.0f;
        }
        return;
    }
    const float most = key_logit(top);
    const double per = 1.44269504088896340736 * SAMPLE_TABLE / (double)o.t;
    if (!(per >= SAMPLE_LEAST_PER && __builtin_fabs((double)most * per) < SAMPLE_NEAR * SAMPLE_TABLE)) {
        alone();
        return;
    }
    const Weights w(most, (double)most, 0.0, per, less, a.bits, s.table);
    const int top_k = w.level(most);
    if (tid < a.chunks) {
        const int none = head.top ? 0 : SAMPLE_BINS;
        s.shift[tid] = none ? none : top_k - (head.k >> 3) - 16 * (a.bits - less);
        s.less[tid] = none ? 0 : min(less - head.less, 63);
        if (none) s.head[tid].mass = 0;
    }
    __syncthreads();
    // About where a bin is (the middle, and a little more than half a bin away), then its least and its largest logit: the
    // first keys of its level and of the next one, each by a wave.
    const double of_bin = 8.0 / per, first = (double)(8 * (top_k - 16 * (a.bits - less)) + 4) / per;
    auto edges = [&](int bin) {
        const double v = first - bin * of_bin, far = __builtin_fabs(v) * 1e-6 + of_bin * 0.75;
        const uint32_t lo = logit_key((float)__builtin_fmax(v - far, (double)lowest)), hi = logit_key((float)__builtin_fmin(v + far, (double)inf));
        if (tid < 64) s.edge[0] = level_start(w, top_k - bin, lo - 1, min(hi, top));
        else if (tid < 128) s.edge[1] = bin == 0 ? top : level_start(w, top_k - bin + 1, lo - 1, min(hi, top)) - 1;
        else if (tid < 192) {       // the chunks that have weight in the bin
            const int c = tid - 128, b = c < a.chunks ? bin - s.shift[c] : -1;
            const uint64_t with = __ballot(b >= 0 && bins[(int64_t)c * SAMPLE_BINS + b] != 0);
            if (c == 0) s.with = with;
        }
        __syncthreads();
    };
    // the bins joined: a chunk's lie s.shift[c] below the row's, its sums are below a power of two s.less[c] octaves lower (and are
    // rounded down bin by bin: a share's cut is off by less than a sixteenth of the row's last bit per logit)
    auto join = [&](int c, uint64_t x) {
        const int to = tid + s.shift[c];
        if (x && to < SAMPLE_BINS - 1) atomicAdd((unsigned long long*)&s.hist[to], (unsigned long long)(o.mode == SHARE ? x >> s.less[c] : x));
    };
    if (o.mode != ALL) {
#pragma unroll
        for (int c = 0; c < SAMPLE_EARLY; c++)
            if (c < a.chunks) join(c, v[c]);
        for (int c = SAMPLE_EARLY; c < a.chunks; c++) join(c, bins[(int64_t)c * SAMPLE_BINS + tid]);
        __syncthreads();
    }
    if (o.mode == TOP) {
        uint64_t all;
        const uint64_t count = s.hist[tid];
        const uint64_t upto = block.scan(count, all);
        if (all < (uint64_t)o.k ? tid == 0 : upto >= (uint64_t)o.k && upto - count < (uint64_t)o.k)
            s.bin = all < (uint64_t)o.k ? SAMPLE_BINS - 2 : tid;
        __syncthreads();
        const int last = s.bin;
        edges(last);
        const int n = gather(s, block, row, a.V, tops, ~0ull, key_logit(s.edge[0]), inf);
        if (n < 0) alone();
        else pick_of_list(s, block, a, r, o, w, top, n);
        return;
    }
    Cut cut{KEY_LOW - 1, 0};
    int last = SAMPLE_BINS - 1;
    if (o.mode == SHARE) {
        uint64_t all = 0, sum;
        for (int c = 0; c < a.chunks; c++) all += s.head[c].mass >> s.less[c];
        const uint64_t mass = s.hist[tid];
        const uint64_t need = o.p < 1.0f ? share_of(o.p, all) : ~0ull;
        if (tid == 0) s.bin = SAMPLE_BINS - 1;
        const uint64_t upto = block.scan(mass, sum);
        if (upto >= need && upto - mass < need) {
            s.bin = tid;
            s.above = upto - mass;
        }
        __syncthreads();
        last = s.bin;
        bool shares = last < SAMPLE_BINS - 1;
        const uint64_t rest = shares ? need - s.above : 0;
        // (a key, so that its bin and what of that bin stays agree: of min_p 1 the largest logit's)
        const uint32_t at_least = o.least > 0.0 ? least_start(w, o.least, top) : 0;
        if (o.least > 0.0) {
            const int low = top_k - w.level(key_logit(at_least));
            if (low < last) shares = false;
            last = min(last, low);
        }
        if (last < SAMPLE_BINS - 1) {
            edges(last);
            const uint32_t from = s.edge[0], to = s.edge[1];
            const float lo = key_logit(from), hi = key_logit(to);
            const int n = from <= to ? gather(s, block, row, a.V, nullptr, s.with, lo, hi) : 0;
            // the bin's logits, from the list or, where they are more, from the row
            auto each = [&](auto f) {
                if (n >= 0) {
#pragma unroll 1
                    for (int i = tid; i < n; i += SAMPLE_THREADS) f(key_logit(s.key[i]), s.index[i]);
                } else {
                    scan_row(s, block, row, a.V, nullptr, s.with, lo, hi, [&](bool on, float x, uint32_t i) {
                        if (on) f(x, i);
                    });
                }
            };
            if (n >= 0 && n <= SAMPLE_SORT) {
                int size = 64;
                while (size < n) size *= 2;
                const uint64_t v = sort_down(s, tid < n ? (uint64_t)s.key[tid] << 32 | ~s.index[tid] : 0, size);
                const uint32_t key = (uint32_t)(v >> 32), chunk = ~(uint32_t)v / SAMPLE_CHUNK;
                uint64_t weight = 0, in_chunk = 0;
                if (tid < n) weight = w.whole(key_logit(key), s.less[chunk], in_chunk);
                const uint64_t upto = block.scan(weight, sum);
                const bool keep = tid < n && (!shares || upto - weight < rest) && key >= at_least;
                if (keep) atomicAdd((unsigned long long*)&s.kept[chunk], (unsigned long long)in_chunk);
                const int m = __syncthreads_count(keep);
                if (tid == m - 1) s.bin = (int)key;
                __syncthreads();
                cut.key = m ? (uint32_t)s.bin : to;      // (of none: nothing of the bin)
                const bool tie = m && tid < n && key == cut.key;
                if (tie) atomicAdd(&s.ties[chunk], 1);
                cut.ties = __syncthreads_count(tie && keep);
            } else {
                cut = Cut{0u, 0};
                if (shares) {
                    uint64_t here = 0;
                    each([&](float x, uint32_t) { here += w.whole(x); });
                    here = block.sum(here);
                    cut = mass_cut(s, block, w, from, to, rest < here ? rest : here, each);
                }
                if (at_least > cut.key) cut = Cut{at_least - 1, 0};
                cut.key = min(cut.key, to);     // (of none: nothing of the bin)
                // what the chunks keep of this bin, and their equals at the cut
                each([&](float x, uint32_t i) {
                    const uint32_t key = logit_key(x);
                    if (cut.ties && key == cut.key) atomicAdd(&s.ties[i / SAMPLE_CHUNK], 1);
                    if (key > cut.key) atomicAdd((unsigned long long*)&s.kept[i / SAMPLE_CHUNK], (unsigned long long)w.of_chunk(s.less[i / SAMPLE_CHUNK]).whole(x));
                });
                __syncthreads();
                if (cut.ties && tid < a.chunks) {
                    int64_t room = cut.ties;
                    for (int c = 0; c < tid; c++) room -= s.ties[c];
                    const int64_t ties = room <= 0 ? 0 : room < s.ties[tid] ? room : s.ties[tid];
                    atomicAdd((unsigned long long*)&s.kept[tid], (unsigned long long)ties * w.of_chunk(s.less[tid]).whole(key_logit(cut.key)));
                }
            }
        }
    }
    // and of the bins above it
    const int lane = tid & 63;
    for (int c = tid >> 6; c < a.chunks; c += SAMPLE_WAVES) {
        uint64_t v = 0;
        if (last >= SAMPLE_BINS - 1) {
            v = lane == 0 ? s.head[c].mass : 0;
        } else {
#pragma unroll 4
            for (int b = lane; b < last - s.shift[c]; b += 64) v += bins[(int64_t)c * SAMPLE_BINS + b];
        }
        v = last_lane64(wave_scan64(v));
        if (lane == 0) atomicAdd((unsigned long long*)&s.kept[c], (unsigned long long)v);
    }
    __syncthreads();
    // the token's chunk, by every wave for itself: a chunk of each lane
    const uint64_t share = lane < a.chunks ? s.kept[lane] >> s.less[lane] : 0, upto = wave_scan64(share), all = last_lane64(upto);
    const uint64_t want = part_of(a.u[r], all);
    const int c = __ffsll((unsigned long long)__ballot(upto > want)) - 1;
    const uint64_t past = readlane64(upto - share, c);
    int64_t ties = cut.ties;
    if (ties) {
        const uint64_t equals = lane < a.chunks ? s.ties[lane] : 0;
        ties -= (int64_t)readlane64(wave_scan64(equals) - equals, c);
    }
    // its chunk in LDS, where the lists have been
    constexpr int V = 16 / sizeof(T);
    const int i0 = c * SAMPLE_CHUNK;
    float* logit = (float*)s.key;
    static_assert(sizeof s.key + sizeof s.index >= SAMPLE_CHUNK * sizeof(float));
    {
        float x[SAMPLE_CHUNK / SAMPLE_THREADS / V][V];
#pragma unroll
        for (int i = 0; i < SAMPLE_CHUNK / SAMPLE_THREADS / V; i++) logits_load(row, i0 + (i * SAMPLE_THREADS + tid) * V, a.V, x[i]);
#pragma unroll
        for (int i = 0; i < SAMPLE_CHUNK / SAMPLE_THREADS / V; i++)
#pragma unroll
            for (int j = 0; j < V; j++) logit[(i * SAMPLE_THREADS + tid) * V + j] = x[i][j];
    }
    pick(s, block, a, r, w.of_chunk(s.less[c]), w, cut, ties < 0 ? 0 : ties, min(SAMPLE_CHUNK, a.V - i0), true, all,
         [&](uint64_t) { return (want - past) << s.less[c]; },
         [&](int e, float& y, int& i) {
             y = logit[e];
             i = i0 + e;
             return y > -inf;
         },
         [&](float y) { return logit_key(y) > cut.key; });
}

static inline int sample_chunks(int vocab) { return (vocab + SAMPLE_CHUNK - 1) / SAMPLE_CHUNK; }
// rows whose chunks are kept at a time: 4096 chunks of 8 KB
static inline int sample_rows(int vocab) { return 4096 / sample_chunks(vocab); }

template <typename T>
static void launch_sample(Sample& a, int nrows, hipStream_t s) {
    const dim3 threads(SAMPLE_THREADS);
    if (a.V <= SAMPLE_WHOLE) {
        hipLaunchKernelGGL((k_sample_pick<T, true>), dim3(nrows), threads, 0, s, a, (int64_t)0);
        return;
    }
    const int most = sample_rows(a.V);
    for (int64_t r = 0; r < nrows; r += most) {
        const int rows = (int)(nrows - r < most ? nrows - r : most);
        hipLaunchKernelGGL((k_sample_scan<T>), dim3(rows * a.chunks), dim3(SCAN_THREADS), 0, s, a, r);
        hipLaunchKernelGGL((k_sample_pick<T, false>), dim3(rows), threads, 0, s, a, r);
    }
}

}  // namespace chimere

using namespace chimere;

extern "C" {

size_t chimere_sample_workspace_size(int vocab, int max_rows) {
    if (vocab <= SAMPLE_WHOLE || vocab > SAMPLE_MAX_VOCAB || max_rows < 1) return 0;
    const int most = sample_rows(vocab), rows = max_rows < most ? max_rows : most;
    const size_t chunks = (size_t)rows * sample_chunks(vocab);
    return al256(chunks * sizeof(SampleChunk)) + al256(chunks * (SAMPLE_CHUNK / 256) * 4) + chunks * SAMPLE_BINS * 8;
}

void chimere_sample(int type, const void* logits, int64_t logits_stride, const float* uniform,
                    const chimere_sampling* settings, int* token, float* logprob, int nrows, int vocab, void* workspace,
                    size_t workspace_bytes, hipStream_t stream) {
    CHIMERE_REQUIRE(float_type(type), CHIMERE_ERR_ARG, "sample: unsupported type %d", type);
    CHIMERE_REQUIRE(settings, CHIMERE_ERR_ARG, "sample: null settings");
    CHIMERE_REQUIRE(vocab >= 1 && vocab <= SAMPLE_MAX_VOCAB && nrows >= 0 && nrows <= (1 << 21), CHIMERE_ERR_ARG,
                    "sample: nrows=%d vocab=%d out of range", nrows, vocab);
    if (nrows == 0) return;
    CHIMERE_REQUIRE(logits && uniform && token && logprob && logits_stride >= 0 && float_aligned(type, logits), CHIMERE_ERR_ARG,
                    "sample: null or misaligned pointer, or bad stride");
    const size_t need = chimere_sample_workspace_size(vocab, nrows);
    CHIMERE_REQUIRE(workspace || !need, CHIMERE_ERR_ARG, "sample: null workspace");
    CHIMERE_REQUIRE(workspace_bytes >= need && ((uintptr_t)workspace & 255) == 0, CHIMERE_ERR_WORKSPACE,
                    "sample: workspace %zu bytes < %zu (or not 256-byte aligned)", workspace_bytes, need);
    Sample a{logits, uniform, settings->temperature, settings->top_p, settings->min_p, settings->top_k, token, logprob,
             logits_stride, settings->temperature_all, settings->top_p_all, settings->min_p_all, settings->top_k_all, vocab, 62,
             sample_chunks(vocab), nullptr, nullptr, nullptr};
    for (int v = 1; v < vocab; v *= 2) a.bits--;
    if (a.bits > 51) a.bits = 51;
    if (need) {
        const int most = sample_rows(vocab), rows = nrows < most ? nrows : most;
        a.chunk = (SampleChunk*)workspace;
        const size_t chunks = (size_t)rows * a.chunks;
        a.tops = (float*)((uint8_t*)workspace + al256(chunks * sizeof(SampleChunk)));
        a.bins = (uint64_t*)((uint8_t*)a.tops + al256(chunks * (SAMPLE_CHUNK / 256) * 4));
    }
    if (type == T_F32) launch_sample<float>(a, nrows, stream);
    else if (type == T_F16) launch_sample<_Float16>(a, nrows, stream);
    else launch_sample<__bf16>(a, nrows, stream);
    check_launch("sample");
}

}  // extern "C"
