// sample.hip — tokens from rows of logits and given random numbers: temperature, top-k, top-p
// and min-p, exactly, without a sort of the vocabulary.
//
// Math, per row l with temperature T > 0 and M = max l. Order the tokens by logit, equal ones by
// index; w_i = 2^((l_i - M) log2(e) / T). Kept are the first k; of them those before which the sum of w is
// under p of all of the k's; of them those with w >= m. Each of the three keeps a head of that order. The token
// is the first one, by index, at which the running sum of the kept w passes u of their total.
//
// Split. scan_kernel reads the logits once: a wave takes a part of 2048 of a row into registers and leaves
// their maximum, the sum of their weights (where it will be needed) and the maximum of every 32 (a group).
// pick_kernel has a workgroup a row. Where nothing is cut off, it finds the part by the parts' sums and reads
// that part again. Else it finds a border from the groups' maxima alone: k groups above it hold k tokens
// above it, and the weights of groups' maxima that sum to p of all do as well. The few groups above
// the border are read again; their tokens above it hold all that is kept. Where that is too many (a flat
// distribution, most of the vocabulary), the whole row takes their place.
//
// A cut is found in bins of the weight, among the candidates or the whole row: the one that reaches k, or p, is
// known by the sums of the bins, and the few tokens in it are compared with each other.
//
// Precision. Weights are fp64 (a table of 64 and a polynomial: off by 2^-44), since the index of a running
// sum over a vocabulary is compared with a given border. Sums are fp64 in a fixed order, or, where
// histograms add in any order, whole numbers in steps of 2^-45 of the largest weight.
//
// What bounds it. The scan: bytes where no row needs a sum (256 rows of 129280 bf16, 66 MB: 12.0 us, 5.5 TB/s, as a
// large copy), the weights' 18 instructions a logit where all do (30 us; filters that differ: 21). The pick: a chain of
// loads that wait for each other (parameters and maxima 1.3 us, the border 2, the candidates' groups 3.4, their
// comparison 1 and up, the sums 0.7), and in a flat row the fp64 weights of all its logits, twice, on one CU: one row of
// 129280 of which thousands stay adds 110 us to a call of any number of rows (256 rows 36 us without such a row, 145 to 153 with).

#include "ds4hip_common.h"
#include "scan.h"
#include "../../include/ds4hip.h"

#include <algorithm>

using namespace ds4hip;

// (A call in a kernel of this file, anywhere, costs each launch of it 4 us: the stack that calls need.)
#define DS4_INLINE __attribute__((always_inline))

namespace {

constexpr int kPart = 2048, kGroup = 32;   // logits of a part (a wave's), of a group
constexpr int kMaxVocab = 1 << 18;         // (sums of 2^45 stay in 64 bits)
constexpr int kScanThreads = 256, kScanParts = kScanThreads / 64;
constexpr int kThreads = 512, kWaves = kThreads / 64;   // (1024: one row 9.2 us and not 8.6, flat rows 79 and not 85)
constexpr int kRow = 8192;       // logits of a row that has one launch: all a workgroup's registers take, 16 a thread
constexpr int kBins = 2048;
constexpr int kList = 4096;      // candidates in LDS: a larger share of the vocabulary is read again from memory
constexpr int kFew = 256;        // candidates that are all compared with each other, four a lane; more go through bins
constexpr int kNear = 512;       // tokens of a bin that are compared with each other
constexpr double kLog2e = 1.4426950408889634074;

struct Args {
    const void *logits;
    long long stride;
    int n_rows, n_vocab, parts, groups;   // of a row, whole workgroups of the scan
    const float *temperature, *top_p, *min_p, *u;
    const int32_t *top_k;
    float all_temperature, all_top_p, all_min_p;
    int all_top_k;
    int32_t *tokens;
    float *probs;
    // workspace
    float *part_max;     // [rows][parts]; NaN: a logit that is NaN or +inf
    double *part_sum;    // [rows][parts] of 2^((l - part's maximum) log2(e) / T)
    float *group_max;    // [rows][groups]
};

// A row's parameters.
struct Row {
    double c;        // 64 log2(e) / T; 0: the largest logit
    int k;           // 0: all
    double p, m, u;
    bool valid;
};

__device__ __forceinline__ Row row_of(const Args &A, int row) {
    Row R;
    const float t = A.temperature ? A.temperature[row] : A.all_temperature;
    const float p = A.top_p ? A.top_p[row] : A.all_top_p, m = A.min_p ? A.min_p[row] : A.all_min_p;
    const int k = A.top_k ? A.top_k[row] : A.all_top_k;
    const float u = A.u[row];
    R.valid = t >= 0.0f && t < INFINITY && p == p && m == m && u >= 0.0f && u < 1.0f;
    R.c = t > 0.0f ? 64.0 * kLog2e / t : 0.0;
    R.k = m > 1.0f ? 1 : k > 0 && k < A.n_vocab ? k : 0;   // (a weight over 1: the first one alone)
    R.p = p > 0.0f ? p : 0.0;
    R.m = m > 1.0f ? 0.0 : m;
    R.u = u;
    return R;
}

__device__ __forceinline__ bool cuts_p(const Row &R) { return R.p < 1.0; }
__device__ __forceinline__ bool cuts_m(const Row &R) { return R.m > 0.0; }
// Whether the sum of all weights is needed.
__device__ __forceinline__ bool needs_sum(const Row &R) { return R.c > 0.0 && R.k == 0 && (cuts_p(R) || !cuts_m(R)); }

// 2^(t / 64) for t <= 0 (2^-1000 for all under -64000), from 2^(j/64) in LDS and the Taylor series of
// 2^(r/64), |r| <= 1/2, up to r^4. Adding 1.5 x 2^52 rounds t to a whole number and leaves it in the low bits: 18
// instructions, eight or more of them side by side (26 with the rounding and conversion instructions and a test).
__device__ __forceinline__ double pow2(double t, const double *table) {
    constexpr double round = 6755399441055744.0, l = 0.69314718055994530942 / 64.0;
    t = fmax(t, -64000.0);
    const double s = t + round, r = t - (s - round);
    const int n = (int)(uint32_t)__double_as_longlong(s);
    double y = l * l * l * l / 24.0;
    y = fma(y, r, l * l * l / 6.0);
    y = fma(y, r, l * l / 2.0);
    y = fma(y, r, l);
    y = fma(y, r, 1.0);
    uint2_t x = __builtin_bit_cast(uint2_t, table[n & 63] * y);
    x[1] += (uint32_t)(n >> 6) << 20;
    return __builtin_bit_cast(double, x);
}

// 2^(j/64), by the exponential series.
struct Table {
    double v[64];
    constexpr Table() : v{} {
        for (int j = 0; j < 64; ++j) {
            const double x = j * (0.69314718055994530942 / 64.0);
            double sum = 0.0;
            for (int k = 24; k > 0; --k) sum = (sum + 1.0) * x / k;
            v[j] = 1.0 + sum;
        }
    }
};
__constant__ const Table kTable = Table();

// Weight of logit x where the row's largest is `top`; some_weight: 2^-1000 at least, also for -inf.
__device__ __forceinline__ double some_weight(float x, float top, double c, const double *table) {
    return pow2(((double)x - (double)top) * c, table);
}
__device__ __forceinline__ double weight(float x, float top, double c, const double *table) {
    const double w = some_weight(x, top, c, table);
    return w > 0x1p-999 ? w : 0.0;
}

// Order of the logits as whole numbers (-0 is 0).
__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t u = __float_as_uint(x + 0.0f);
    return u >> 31 ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t k) { return __uint_as_float(k >> 31 ? k & 0x7FFFFFFFu : ~k); }

// Eight logits of a row from e on (-inf past its end), as they lie in memory. Rows start at any multiple of
// a logit's size.
template <bool kF32>
struct Eight {
    uint4_t v[kF32 ? 2 : 1];
    __device__ __forceinline__ void load(const Args &A, int row, int e) {
        if (kF32) {
            const float *src = static_cast<const float *>(A.logits) + row * A.stride + e;
            if (e + 8 <= A.n_vocab) {
                __builtin_memcpy(v, src, 32);
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) v[kF32 ? i >> 2 : 0][i & 3] = e + i < A.n_vocab ? __float_as_uint(src[i]) : 0xFF800000u;
            }
        } else {
            const uint16_t *src = static_cast<const uint16_t *>(A.logits) + row * A.stride + e;
            if (e + 8 <= A.n_vocab) {
                __builtin_memcpy(v, src, 16);
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    v[0][i] = (e + 2 * i < A.n_vocab ? src[2 * i] : 0xFF80u) | (e + 2 * i + 1 < A.n_vocab ? src[2 * i + 1] : 0xFF80u) << 16;
            }
        }
    }
    __device__ __forceinline__ float operator[](int i) const {
        return __uint_as_float(kF32 ? v[kF32 ? i >> 2 : 0][i & 3] : i & 1 ? v[0][i >> 1] & 0xFFFF0000u : v[0][i >> 1] << 16);
    }
};

template <bool kF32>
__device__ __forceinline__ float load_one(const Args &A, int row, int e) {
    return kF32 ? static_cast<const float *>(A.logits)[row * A.stride + e]
                : bf16_to_f32(static_cast<const uint16_t *>(A.logits)[row * A.stride + e]);
}

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v = fmaxf(v, __shfl_xor(v, off));
    return v;
}

// Waves on their own: four times 512 logits of a part each, all of their loads ahead of the first use, no barrier.
// 256 rows of 129280 bf16: 12 us without sums, 21 with those of filters that differ, 30 with all. One row: 4.1.
template <bool kF32>
__global__ __launch_bounds__(kScanThreads) void scan_kernel(const Args A) {
    __shared__ double tables[kScanParts][64];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wgs = A.parts / kScanParts, row = blockIdx.x / wgs, part = (blockIdx.x - row * wgs) * kScanParts + w;
    const size_t at = (size_t)row * A.parts + part;
    double *table = tables[w];
    const double entry = kTable.v[lane];
    Eight<kF32> x[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j].load(A, row, min(part * kPart + j * 512 + lane * 8, A.n_vocab));
    const Row R = row_of(A, row);
    bool odd = false;
    float top = -INFINITY, *group_max = A.group_max + at * (kPart / kGroup);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        float m = -INFINITY;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            m = fmaxf(m, x[j][i]);
            odd = odd || !(x[j][i] < INFINITY);
        }
        top = fmaxf(top, m);
        m = fmaxf(m, __shfl_xor(m, 1));
        m = fmaxf(m, __shfl_xor(m, 2));
        if ((lane & 3) == 0) group_max[16 * j + (lane >> 2)] = m;
    }
    top = wave_max(top);
    odd = __any(odd);   // (all lanes take part)
    if (lane == 0) A.part_max[at] = odd ? __builtin_nanf("") : top;
    if (!needs_sum(R)) return;
    table[lane] = entry;   // (a wave's LDS accesses are in order)
    __builtin_amdgcn_wave_barrier();
    double sum = 0.0;
    if (top > -INFINITY) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int i = 0; i < 8; ++i) sum += some_weight(x[j][i], top, R.c, table);
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) sum += __shfl_xor(sum, off);
    if (lane == 0) A.part_sum[at] = sum;
}

// ---- pick ------------------------------------------------------------------------

struct Pick {
    double table[64];
    double sums[kWaves];
    float tops[kWaves];
    unsigned long long scans[kWaves];
    int counts[kWaves];
    unsigned long long bins[kBins];        // weights, or numbers, of tokens
    uint16_t groups[kMaxVocab / kGroup];   // those with a candidate, by index
    float logit[kList];                    // the candidates, by index
    uint32_t index[kList];
    unsigned long long near[kNear], near_w[kNear];   // the places and weights in a cut's bin
    int rank[kFew];
    double wave_sum[kMaxVocab / 512];      // of 512 tokens of the row each
    int n_near, n_list, found;
    unsigned long long found_above, place;
    double before;
};

// A token's place in the order of logits, as a whole number: the highest first, equal logits by index.
__device__ __forceinline__ unsigned long long place_of(uint32_t key, uint32_t index) { return (unsigned long long)key << 32 | ~index; }

template <typename T>
__device__ __forceinline__ T block_scan(T v, T *sums, T *total) {
    return wg_scan<kWaves>(v, sums, total);
}

__device__ __forceinline__ void give(const Args &A, int row, int token, double share) {
    A.tokens[row] = token;
    A.probs[row] = (float)share;
}

// Tokens in the order of their indexes: the logits of kEach from the i-th on (-inf past the last), and a
// token's index.
struct ListSource {
    const Pick &S;
    int n;
    static constexpr int kDeep = 1;
    static constexpr bool kList = true;
    template <int kEach>
    struct Some {
        float x[kEach];
        __device__ __forceinline__ void load(const ListSource &L, int i) {
#pragma unroll
            for (int u = 0; u < kEach; ++u) x[u] = i + u < L.n ? L.S.logit[i + u] : -INFINITY;
        }
        __device__ __forceinline__ float operator()(const ListSource &, int, int u) const { return x[u]; }
    };
    __device__ __forceinline__ int index(int i) const { return S.index[i]; }
};
template <bool kF32, int kAhead>
struct RowSource {
    const Args &A;
    int row, first, n;   // logits first .. first + n - 1 of the row
    static constexpr int kDeep = kAhead;
    static constexpr bool kList = false;
    __device__ __forceinline__ RowSource<kF32, 1> slow() const { return {A, row, first, n}; }   // (less code)
    template <int kEach>
    struct Some {
        static_assert(kEach == 8, "as the loads are");
        Eight<kF32> x;
        __device__ __forceinline__ void load(const RowSource &L, int i) { x.load(L.A, L.row, min(L.first + i, L.A.n_vocab)); }   // (past the end: nothing is read)
        __device__ __forceinline__ float operator()(const RowSource &L, int i, int u) const { return i + u < L.n ? x[u] : -INFINITY; }
    };
    __device__ __forceinline__ int index(int i) const { return first + i; }
};

// use(i, logits) for all of a source, kEach * kThreads at a time. kDeep of them are loaded while those before
// are used (memory is 2 us away: with one of them ahead, converted as it came, a pass of 65536 took 28 us).
template <int kEach, typename Source, typename Use>
__device__ __forceinline__ void each_tile(const Source &src, Use use) {
    constexpr int kStep = kEach * kThreads, kDeep = Source::kDeep;
    typename Source::template Some<kEach> next[kDeep];
    int i = kEach * threadIdx.x;
#pragma unroll
    for (int d = 0; d < kDeep; ++d) next[d].load(src, i + d * kStep);
    for (int i0 = 0; i0 < src.n; i0 += kDeep * kStep, i += kDeep * kStep) {
        typename Source::template Some<kEach> now[kDeep];
#pragma unroll
        for (int d = 0; d < kDeep; ++d) now[d] = next[d];
        if (i0 + kDeep * kStep < src.n)
#pragma unroll
            for (int d = 0; d < kDeep; ++d) next[d].load(src, i + (kDeep + d) * kStep);
        __builtin_amdgcn_sched_barrier(0);   // (in flight before the others are used)
#pragma unroll
        for (int d = 0; d < kDeep; ++d) {
            if (i0 + d * kStep >= src.n) break;
            float x[kEach];
#pragma unroll
            for (int u = 0; u < kEach; ++u) x[u] = now[d](src, i + d * kStep, u);
            use(i + d * kStep, x);
        }
    }
}

constexpr double kUnit = 35184372088832.0;   // 2^45
// (adding 2^52 rounds to a whole number and leaves it in the low bits)
__device__ __forceinline__ unsigned long long units(double w) {
    return (unsigned long long)__double_as_longlong(fma(w, kUnit, 4503599627370496.0)) & 0xFFFFFFFFFFFFFull;
}

// A row's bins, 32 for each halving of the weight: kBins - 1 has the largest logit, 0 all whose weight is under
// 2^-63.9. What is rounded on the way grows with the distance, so the bins keep the order of logits.
struct Bins {
    float top, scale;
    float half = 0.5f * top, twice = 2.0f * scale;   // (half the difference of two logits stays in fp32's range, and twice the scale does)
    __device__ __forceinline__ float steps(float x) const { return fminf(fmaf(x, -0.5f, half) * twice, (float)(kBins - 1)); }
    __device__ __forceinline__ int operator()(float x) const { return kBins - 1 - (int)steps(x); }
    // of x in its bin: the part of kBins that it lies in
    __device__ __forceinline__ int part(float x) const {
        const float d = steps(x);
        return kBins - 1 - (int)((d - floorf(d)) * (float)kBins);
    }
};

__device__ __forceinline__ void clear_bins(Pick &S) {
#pragma unroll
    for (int i = 0; i < kBins; i += kThreads) S.bins[i + threadIdx.x] = 0;
    __syncthreads();
}

// After a barrier: the first bin, from the highest down, at which the bins' sum reaches need (-1: none), and in
// S.found_above the sum of those above it. share: need is that of the bins' sum instead.
__device__ __forceinline__ int find_bin(Pick &S, unsigned long long *need, double share = 0.0) {
    constexpr int kEach = kBins / kThreads;
    const int hi = kBins - 1 - kEach * (int)threadIdx.x;
    unsigned long long x[kEach], sum = 0, all;
#pragma unroll
    for (int u = 0; u < kEach; ++u) sum += x[u] = S.bins[hi - u];
    const unsigned long long upto = block_scan(sum, S.scans, &all);
    if (share > 0.0) *need = max((unsigned long long)ceil(share * (double)all), 1ull);
    if (all < *need) return -1;
    unsigned long long above = upto - sum;
    if (above < *need && upto >= *need) {   // one thread's
        int u = 0;
#pragma unroll
        for (int v = 0; v < kEach - 1; ++v)
            if (u == v && above + x[v] < *need) {
                above += x[v];
                u = v + 1;
            }
        S.found = hi - u;
        S.found_above = above;
    }
    __syncthreads();
    return S.found;
}

// Which tokens of a source a cut is looked for in, and where: the place of the last of the first `need` of them
// (kWeigh: the first one with which the sum of units reaches it), from place `within` up.
struct Search {
    unsigned long long need, within, prefix;
    int level, below;   // levels of bins behind it, bits of the places below those that are found
    int bin[2];         // bins of the first two levels: of the weight, parts of one of them
};

template <bool kWeigh>
__device__ __forceinline__ unsigned long long amount(const Pick &S, const Row &R, const Bins &bins, float x) {
    return kWeigh ? units(weight(x, bins.top, R.c, S.table)) : 1;
}

// Whether a token lies in the bins of `levels` levels.
template <typename Source>
__device__ __forceinline__ bool inside(const Search &Q, const Bins &bins, const Source &src, float x, int i, int levels) {
    const int b = bins(x);
    if (b == 0 || (levels > 0 && b != Q.bin[0]) || (levels > 1 && bins.part(x) != Q.bin[1])) return false;
    if (!Q.within && Q.below == 64) return true;
    const unsigned long long place = place_of(key_of(x), src.index(i));
    return place >= Q.within && (Q.below == 64 || place >> Q.below == Q.prefix);
}

// use(item, logit) for the tokens of a source that are inside the found bins, one of a lane at a time: they are few, and
// in different lanes. Most of the others are known by two comparisons.
template <int kEach, typename Source, typename Use>
__device__ __forceinline__ void each_inside(const Search &Q, const Bins &bins, const Source &src, Use use) {
    const float near = (float)(kBins - 1 - Q.bin[0]) / bins.scale, far = (float)(kBins - Q.bin[0]) / bins.scale,
                slack = 1e-6f * (fabsf(bins.top) + far), from = bins.top - far - slack, to = bins.top - near + slack;
    each_tile<kEach>(src, [&](int i, const float *x) DS4_INLINE {
        uint32_t mine = 0;
#pragma unroll
        for (int u = 0; u < kEach; ++u) mine |= x[u] < from || x[u] > to ? 0 : 1u << u;
        while (__any(mine != 0)) {
            const int u = mine ? __builtin_ctz(mine) : 0;
            float y = x[0];
#pragma unroll
            for (int v = 1; v < kEach; ++v) y = u == v ? x[v] : y;
            if (mine && inside(Q, bins, src, y, i + u, Q.level)) use(i + u, y);
            mine &= mine - 1;
        }
    });
}

// The place, among the n <= kNear tokens in S.near.
template <bool kWeigh>
__device__ __forceinline__ unsigned long long cut_near(Pick &S, int n, const Row &R, const Bins &bins, unsigned long long need) {
    const int tid = threadIdx.x;
    if (kWeigh) {
        if (tid < n) S.near_w[tid] = amount<true>(S, R, bins, value_of((uint32_t)(S.near[tid] >> 32)));
        __syncthreads();
    }
    if (tid < n) {   // what lies before each of them
        const unsigned long long mine = S.near[tid];
        unsigned long long before = 0;
#pragma unroll 4
        for (int j = 0; j < n; ++j) {
            const unsigned long long w = kWeigh ? S.near_w[j] : 1;   // (read whether it counts or not: no branch)
            before += S.near[j] > mine ? w : 0;
        }
        if (before < need && before + (kWeigh ? S.near_w[tid] : 1) >= need) S.place = mine;
    }
    __syncthreads();
    return S.place;
}

// The tokens that are inside, counted in S.n_near; the first kNear of them in S.near.
template <int kEach, typename Source>
__device__ __forceinline__ int gather_near(Pick &S, const Search &Q, const Bins &bins, const Source &src) {
    __syncthreads();
    if (threadIdx.x == 0) S.n_near = 0;
    __syncthreads();
    each_inside<kEach>(Q, bins, src, [&](int at, float x) DS4_INLINE {
        const int to = atomicAdd(&S.n_near, 1);
        if (to < kNear) S.near[to] = place_of(key_of(x), src.index(at));
    });
    __syncthreads();
    return S.n_near;
}

// From the second level on: parts of the weight's bin, then digits of the places, which all differ, until kNear are left.
template <bool kWeigh, int kEach, typename Source>
__device__ __forceinline__ unsigned long long cut_inside(Pick &S, Search Q, const Row &R, const Bins &bins, const Source &src) {
    while (true) {
        const int n = gather_near<kEach>(S, Q, bins, src);
        if (n <= kNear) return cut_near<kWeigh>(S, n, R, bins, Q.need);
        const int shift = Q.level == 1 ? 64 : Q.below - min(Q.below, 11);
        clear_bins(S);
        each_inside<kEach>(Q, bins, src, [&](int at, float x) DS4_INLINE {
            const int b = shift == 64 ? bins.part(x)
                                      : (int)(place_of(key_of(x), src.index(at)) >> shift & ((1ull << (Q.below - shift)) - 1));
            atomicAdd(&S.bins[b], amount<kWeigh>(S, R, bins, x));
        });
        __syncthreads();
        const int found = find_bin(S, &Q.need);
        Q.need -= S.found_above;
        if (Q.level == 1) {
            Q.bin[1] = found;
        } else {
            Q.prefix = Q.prefix << (Q.below - shift) | (unsigned)found;
            Q.below = shift;
        }
        ++Q.level;
    }
}

// The cut of a source: the place of the last of the first k tokens from place `within` up (kWeigh: of those before which
// their weights' sum is under the share p of `all` units; all 0: of their sum). 0: all of them. What is in the
// weight's bin that has it goes to the list, where that is not the source and holds it.
template <bool kWeigh, int kEach, typename Source>
__device__ __forceinline__ unsigned long long cut_at(Pick &S, const Source &src, const Row &R, const Bins &bins, int k,
                                            unsigned long long within, double all) {
    Search Q = {kWeigh ? max((unsigned long long)ceil(R.p * all), 1ull) : (unsigned long long)k, within, 0, 0, 64, {0, 0}};
    clear_bins(S);
    each_tile<kEach>(src, [&](int i, const float *x) DS4_INLINE {
        unsigned long long w[kEach];
#pragma unroll
        for (int u = 0; u < kEach; ++u) w[u] = amount<kWeigh>(S, R, bins, x[u]);
#pragma unroll
        for (int u = 0; u < kEach; ++u)
            if (w[u] && inside(Q, bins, src, x[u], i + u, 0)) atomicAdd(&S.bins[bins(x[u])], w[u]);
    });
    if (threadIdx.x == 0) S.n_list = 0;
    __syncthreads();
    const int found = find_bin(S, &Q.need, kWeigh && !(all > 0.0) ? fmax(R.p, 1e-300) : 0.0);
    if (found < 0) return 0;
    Q.need -= S.found_above;
    Q.bin[0] = found;
    Q.level = 1;
    if constexpr (Source::kList) {
        return cut_inside<kWeigh, kEach>(S, Q, R, bins, src);
    } else {
        each_inside<kEach>(Q, bins, src, [&](int at, float x) DS4_INLINE {
            const int to = atomicAdd(&S.n_list, 1);
            if (to < kList) S.logit[to] = x, S.index[to] = src.index(at);
        });
        __syncthreads();
        const int n = S.n_list;
        return n <= kList ? cut_inside<kWeigh, 1>(S, Q, R, bins, ListSource{S, n}) : cut_inside<kWeigh, kEach>(S, Q, R, bins, src.slow());
    }
}

// Gives the token: the first by index at which the sum of the weights that are kept (from place `cut` up, R.m
// at least) passes the target, u of their sum, or the one given with the sum of all. A wave's kEach * 64 tokens
// are summed together; the wave in which the target lies is looked through again.
template <int kEach, typename Source>
__device__ __forceinline__ void draw(const Args &A, Pick &S, const Source &src, const Row &R, int row, float top, unsigned long long cut,
                            double target, double all) {
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    const float cut_logit = cut ? value_of((uint32_t)(cut >> 32)) : -INFINITY;
    const int cut_index = (int)~(uint32_t)cut;
    const double least = fmax(R.m, 0x1p-999);   // (weight()'s 0)
    auto weights = [&](int i, const float *logit, double *x) DS4_INLINE {
        double sum = 0.0;
#pragma unroll
        for (int u = 0; u < kEach; ++u) {
            const bool in = logit[u] > cut_logit || (logit[u] == cut_logit && src.index(i + u) <= cut_index);
            const double y = some_weight(logit[u], top, R.c, S.table);
            x[u] = in && y >= least ? y : 0.0;
            sum += x[u];
        }
        return sum;
    };
    double x[kEach], sum = 0.0;
    int n_sums = 0;
    each_tile<kEach>(src, [&](int i, const float *logit) DS4_INLINE {
        sum = weights(i, logit, x);
        const double upto = wave_scan(sum);
        if (lane == 63) S.wave_sum[n_sums + w] = upto;
        n_sums += kWaves;
    });
    if (tid == 0) S.found = 0x7FFFFFFF, S.n_near = -1;
    __syncthreads();
    const double mine = tid < n_sums ? S.wave_sum[tid] : 0.0;
    double total;
    const double upto = block_scan(mine, S.sums, &total);
    if (!(all > 0.0)) {
        all = total;
        target = R.u * total;
    }
    if (mine > 0.0) {
        if (upto > target) atomicMin(&S.found, tid);
        atomicMax(&S.n_near, tid);
    }
    __syncthreads();
    // (none: sums that were rounded otherwise; then the last that is kept)
    const int at = S.found < 0x7FFFFFFF ? S.found : max(S.n_near, 0);   // (the largest logit is always kept)
    if (tid == at) S.before = upto - mine;
    __syncthreads();
    if (S.n_near < 0 || w != at % kWaves) return;
    const int i = (at / kWaves * kThreads + tid) * kEach;
    if (n_sums > kWaves) {   // (else x and sum are what they were)
        typename Source::template Some<kEach> again;
        again.load(src, i);
        float logit[kEach];
#pragma unroll
        for (int u = 0; u < kEach; ++u) logit[u] = again(src, i, u);
        sum = weights(i, logit, x);
    }
    const double incl = S.before + wave_scan(sum);
    const uint64_t over = __ballot(sum > 0.0 && incl > target), any = __ballot(sum > 0.0);
    if (lane != (over ? __builtin_ctzll(over) : 63 - __builtin_clzll(any))) return;
    double run = incl - sum, share = 0.0;
    int hit = -1;
    bool done = false;
#pragma unroll
    for (int u = 0; u < kEach; ++u) {
        run += x[u];
        if (x[u] > 0.0 && !done) {
            hit = i + u;
            share = x[u];
            done = run > target;
        }
    }
    give(A, row, src.index(hit), share / all);
}

// The same and the cuts for a list of at most kFew candidates: all are compared with all, which gives each one's rank and
// the weights before it at once. A lane holds four of them and a wave has an eighth of the others to compare with, so that
// what is read from LDS serves 256 comparisons (a read for each 64 took 4 us for 212 candidates). All sums are units: that of
// all that is kept is off by 2^-38 of itself at most.
__device__ __forceinline__ void pick_few(const Args &A, Pick &S, int n, const Row &R, int row, float top, double all) {
    constexpr int kHeld = kFew / 64;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    if (tid < n) {
        S.near[tid] = place_of(key_of(S.logit[tid]), S.index[tid]);
        S.near_w[tid] = units(weight(S.logit[tid], top, R.c, S.table));
    }
    if (tid < kFew) S.rank[tid] = 0, S.bins[tid] = 0;   // (bins: the weights before each)
    __syncthreads();
    if (R.k || cuts_p(R)) {
        unsigned long long place[kHeld], before[kHeld];
        int rank[kHeld];
#pragma unroll
        for (int t = 0; t < kHeld; ++t) {
            place[t] = S.near[min(lane + 64 * t, n - 1)];
            rank[t] = 0;
            before[t] = 0;
        }
        const int each = (n + kWaves - 1) / kWaves, end = min(n, (wave + 1) * each);
#pragma unroll 2
        for (int j = wave * each; j < end; ++j) {
            const unsigned long long other = S.near[j], w = S.near_w[j];
#pragma unroll
            for (int t = 0; t < kHeld; ++t) {
                if (64 * t >= n) break;
                const bool is = other > place[t];
                rank[t] += is;
                before[t] += is ? w : 0;
            }
        }
#pragma unroll
        for (int t = 0; t < kHeld; ++t)
            if (rank[t]) {
                atomicAdd(&S.rank[lane + 64 * t], rank[t]);
                atomicAdd(&S.bins[lane + 64 * t], before[t]);
            }
        __syncthreads();
    }
    const int i = min(tid, n - 1), rank = S.rank[min(i, kFew - 1)];
    const unsigned long long mine = S.near[i], w = S.near_w[i], before = S.bins[i];
    bool in = tid < n && (!R.k || rank < R.k);
    unsigned long long total;
    if (cuts_p(R)) {
        double sum = all * kUnit;
        if (R.k) {
            block_scan(in ? w : 0, S.scans, &total);
            sum = (double)total;
        }
        in = in && before < max((unsigned long long)ceil(R.p * sum), 1ull);
    }
    // (min-p as a share of the largest weight, in doubles as everywhere)
    if (cuts_m(R)) in = in && (rank == 0 && (R.k || cuts_p(R)) ? true : weight(value_of((uint32_t)(mine >> 32)), top, R.c, S.table) >= R.m);
    const unsigned long long upto = block_scan(in ? w : 0, S.scans, &total);
    const unsigned long long target = (unsigned long long)(R.u * (double)total);   // the sum passes it: at least one more
    // (the token's own weight not in units: of a small one they keep only the leading bits)
    if (in && upto > target && upto - w <= target)
        give(A, row, (int)~(uint32_t)mine, weight(value_of((uint32_t)(mine >> 32)), top, R.c, S.table) * kUnit / (double)total);
}

// The least logit of a candidate, from the lowest bin that all that is kept lies in (as one logit, with room for what is
// rounded: more candidates do no harm). min-p gives a border too (the exact test comes later), but for
// those that top-p counts among the first k.
__device__ __forceinline__ float least_of(const Row &R, const Bins &bins, int border) {
    const float top = bins.top, floor_m = cuts_m(R) ? top + (float)(64.0 * log2(R.m) / R.c) : -INFINITY;
    const float least = floor_m > -INFINITY && !(R.k && cuts_p(R)) ? fminf(floor_m - 1e-5f * (fabsf(top) + fabsf(floor_m) + 1e-30f), top) : -INFINITY;
    const float reach = (float)(kBins - border) / bins.scale;
    return fmaxf(least, top - reach - 1e-6f * (fabsf(top) + reach));
}

// The n candidates in the list, or where it does not hold them the whole row: cut, and the token.
template <bool kF32>
__device__ __forceinline__ void settle(const Args &A, Pick &S, const Row &R, int row, const Bins &bins, int n, double all) {
    const float top = bins.top;
    if (n <= kFew) {
        pick_few(A, S, n, R, row, top, all);
    } else if (n <= kList) {
        const ListSource src{S, n};
        unsigned long long cut = 0;
        if (R.k) cut = cut_at<false, 1>(S, src, R, bins, R.k, 0, 0.0);
        if (cuts_p(R)) cut = cut_at<true, 1>(S, src, R, bins, 0, cut, all * kUnit);
        draw<1>(A, S, src, R, row, top, cut, 0.0, 0.0);
    } else {
        const RowSource<kF32, 2> src{A, row, 0, A.n_vocab};
        unsigned long long cut = 0;
        if (R.k) cut = cut_at<false, 8>(S, src, R, bins, R.k, 0, 0.0);
        if (cuts_p(R)) cut = cut_at<true, 8>(S, src, R, bins, 0, cut, all * kUnit);
        draw<8>(A, S, src, R, row, top, cut, 0.0, 0.0);
    }
}

// Rows of up to kRow logits, a workgroup each and one launch: sixteen logits of a thread in registers.
template <bool kF32>
__global__ __launch_bounds__(kThreads) void row_kernel(const Args A) {
    static_assert(kRow == 16 * kThreads, "sixteen a thread");
    __shared__ Pick S;
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, row = blockIdx.x;
    Eight<kF32> x[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) x[j].load(A, row, min(j * (kRow / 2) + 8 * tid, A.n_vocab));
    const Row R = row_of(A, row);
    if (tid < 64) S.table[tid] = kTable.v[tid];
    if (tid == 0) S.found = 0x7FFFFFFF;
    float top = -INFINITY;
    bool odd = false;
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            top = fmaxf(top, x[j][u]);
            odd = odd || !(x[j][u] < INFINITY);
        }
    odd = __any(odd);
    top = wave_max(top);
    if (lane == 0) S.tops[w] = odd ? __builtin_nanf("") : top;
    clear_bins(S);
#pragma unroll
    for (int i = 0; i < kWaves; ++i) {
        odd = odd || S.tops[i] != S.tops[i];
        top = fmaxf(top, S.tops[i]);
    }
    if (odd || !(top > -INFINITY) || !R.valid) {
        if (tid == 0) give(A, row, -1, __builtin_nan(""));
        return;
    }
    if (R.c == 0.0) {
#pragma unroll
        for (int j = 1; j >= 0; --j)
#pragma unroll
            for (int u = 7; u >= 0; --u)
                if (x[j][u] == top) atomicMin(&S.found, j * (kRow / 2) + 8 * tid + u);
        __syncthreads();
        if (tid == 0) give(A, row, S.found, 1.0);
        return;
    }
    if (!R.k && !cuts_p(R) && !cuts_m(R)) {   // nothing is cut off
        draw<8>(A, S, RowSource<kF32, 2>{A, row, 0, A.n_vocab}, R, row, top, 0, 0.0, 0.0);
        return;
    }
    const Bins bins{top, (float)fmin(R.c * 0.5, 1e30)};
    double all = 0.0;   // of all weights
    int border = 1;
    if (R.k || cuts_p(R)) {   // as in pick_kernel, with the tokens themselves
        double sum = 0.0;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            unsigned long long n[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                const double y = R.k ? 0.0 : weight(x[j][u], top, R.c, S.table);
                sum += y;
                n[u] = R.k ? 1 : units(y);
            }
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                const int b = bins(x[j][u]);
                if (b && n[u]) atomicAdd(&S.bins[b], n[u]);
            }
        }
        if (!R.k) block_scan(sum, S.sums, &all);
        __syncthreads();
        unsigned long long need = R.k ? R.k : (unsigned long long)(R.p * all * kUnit) + kRow;
        border = max(find_bin(S, &need), 1);
    }
    const float from = least_of(R, bins, border);
    // the candidates, by index: first those of the first half
    uint32_t mine[2] = {0, 0};
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int u = 0; u < 8; ++u) mine[j] |= x[j][u] >= from && x[j][u] > -INFINITY ? 1u << u : 0;
    const int both = (int)(__popc(mine[0]) | __popc(mine[1]) << 16);
    int found;
    const int before = block_scan(both, S.counts, &found) - both, n = (found & 0xFFFF) + (found >> 16);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        int at = j ? (found & 0xFFFF) + (before >> 16) : before & 0xFFFF;
#pragma unroll
        for (int u = 0; u < 8; ++u)
            if (mine[j] >> u & 1) {
                if (at < kList) S.logit[at] = x[j][u], S.index[at] = j * (kRow / 2) + 8 * tid + u;
                ++at;
            }
    }
    __syncthreads();
    settle<kF32>(A, S, R, row, bins, n, all);
}

// A workgroup a row, the groups' maxima in registers. One row of 129280 with k and p: 9.0 us; 256 rows with filters of
// their own: 15 (k = 200: 13 alone); 24 flat rows of 65536 with p: 86, of which bins of all weights 25, the cut's
// bin gathered 10, the draw 27 (a row on one CU: the host does not know which rows are flat, and
// further launches for them would cost the others about 3 us each).
template <bool kF32>
__global__ __launch_bounds__(kThreads) void pick_kernel(const Args A) {
    __shared__ Pick S;
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, row = blockIdx.x;
    const Row R = row_of(A, row);
    // the thread's groups: `each` next to each other, a multiple of four as a row's are
    constexpr int kMost = kMaxVocab / kGroup / kThreads;
    const int each = (A.groups / 4 + kThreads - 1) / kThreads * 4, g0 = each * tid;
    const float *group_max = A.group_max + (size_t)row * A.groups;
    float g[kMost];
#pragma unroll
    for (int u = 0; u < kMost; ++u) g[u] = -INFINITY;
#pragma unroll
    for (int u = 0; u < kMost; u += 4)
        if (u < each && g0 + u < A.groups) __builtin_memcpy(g + u, group_max + g0 + u, 16);
    // (every wave for itself: a lane has two parts, of 128 at most and a multiple of four)
    float pm[2] = {-INFINITY, -INFINITY};
    double ps[2] = {0.0, 0.0};
    if (2 * lane < A.parts) {
        __builtin_memcpy(pm, A.part_max + (size_t)row * A.parts + 2 * lane, 8);
        if (needs_sum(R)) __builtin_memcpy(ps, A.part_sum + (size_t)row * A.parts + 2 * lane, 16);
    }
    const float top = wave_max(fmaxf(pm[0], pm[1]));
    if (__any(pm[0] != pm[0] || pm[1] != pm[1]) || !(top > -INFINITY) || !R.valid) {
        if (tid == 0) give(A, row, -1, __builtin_nan(""));
        return;
    }
    if (tid < 64) S.table[tid] = kTable.v[tid];
    if (tid == 0) S.found = 0x7FFFFFFF;
    clear_bins(S);
    if (R.c == 0.0) {   // the first group that has the largest, the first of its logits that is it
#pragma unroll
        for (int u = 0; u < kMost; ++u)
            if (u < each && g[u] == top) atomicMin(&S.found, g0 + u);
        __syncthreads();
        if (w == 0 && S.found < A.groups) {
            const int e = S.found * kGroup + lane;
            const uint64_t is = __ballot(lane < kGroup && e < A.n_vocab && load_one<kF32>(A, row, min(e, A.n_vocab - 1)) == top);
            if (lane == 0) give(A, row, S.found * kGroup + __builtin_ctzll(is), 1.0);
        }
        return;
    }
    double all = 0.0;   // of all weights
    if (needs_sum(R)) {
#pragma unroll
        for (int u = 0; u < 2; ++u) ps[u] = pm[u] > -INFINITY ? ps[u] * weight(pm[u], top, R.c, S.table) : 0.0;
        const double mine = ps[0] + ps[1], upto = wave_scan(mine);
        all = lane_of(upto, 63);
        if (!cuts_p(R) && !cuts_m(R)) {   // nothing is cut off
            const double target = R.u * all;
            const uint64_t over = __ballot(mine > 0.0 && upto > target), any = __ballot(mine > 0.0);
            if (!any) return;   // (the largest logit's part weighs something)
            const int pair = over ? __builtin_ctzll(over) : 63 - __builtin_clzll(any);
            const double first = lane_of(ps[0], pair), begin = lane_of(upto - mine, pair);
            const bool second = !(first > 0.0 && begin + first > target) && lane_of(ps[1], pair) > 0.0;
            const int part = 2 * pair + second;
            draw<8>(A, S, RowSource<kF32, 1>{A, row, part * kPart, min(kPart, A.n_vocab - part * kPart)}, R, row, top, 0,
                    target - (second ? begin + first : begin), all);
            return;
        }
    }

    // The border: a bin that holds, with those above it, k groups' maxima, or p of all in their weights
    // (and a unit for each group's rounding). All that is kept lies in it or above it.
    const Bins bins{top, (float)fmin(R.c * 0.5, 1e30)};
    int border = 1;
    if (R.k || cuts_p(R)) {
#pragma unroll
        for (int j = 0; j < kMost; j += 4)
            if (j < each) {
                unsigned long long x[4];
#pragma unroll
                for (int u = 0; u < 4; ++u) x[u] = bins(g[j + u]) == 0 ? 0 : R.k ? 1 : units(weight(g[j + u], top, R.c, S.table));
#pragma unroll
                for (int u = 0; u < 4; ++u)
                    if (x[u]) atomicAdd(&S.bins[bins(g[j + u])], x[u]);
            }
        __syncthreads();
        unsigned long long need = R.k ? R.k : (unsigned long long)(R.p * all * kUnit) + A.groups;
        border = max(find_bin(S, &need), 1);
    }
    const float from = least_of(R, bins, border);
    auto in = [&](float x) DS4_INLINE { return x >= from && x > -INFINITY; };
    // the groups that have a candidate, by index
    int n_groups = 0;
    {
        int mine = 0;
#pragma unroll
        for (int u = 0; u < kMost; ++u) mine += u < each && in(g[u]) ? 1 << u : 0;
        int at = block_scan((int)__popc(mine), S.counts, &n_groups) - __popc(mine);
        for (; mine; mine &= mine - 1) S.groups[at++] = (uint16_t)(g0 + __builtin_ctz(mine));
        __syncthreads();
    }
    // their candidates, by index: a thread a group
    int n = 0;
    for (int i0 = 0; i0 < n_groups && n <= kList; i0 += kThreads) {
        Eight<kF32> x[kGroup / 8];
        uint32_t mine = 0;
        int e = 0, found;
        if (i0 + 64 * w < n_groups) {   // (waves without a group skip the work)
            e = i0 + tid < n_groups ? S.groups[i0 + tid] * kGroup : A.n_vocab;
#pragma unroll
            for (int j = 0; j < kGroup / 8; ++j) x[j].load(A, row, min(e + 8 * j, A.n_vocab));
#pragma unroll
            for (int u = 0; u < kGroup; ++u) mine |= in(x[u >> 3][u & 7]) ? 1u << u : 0;
        }
        int at = n + block_scan((int)__popc(mine), S.counts, &found) - __popc(mine);
        if (__any(mine != 0)) {
#pragma unroll
            for (int u = 0; u < kGroup; ++u)
                if (mine >> u & 1) {
                    if (at < kList) S.logit[at] = x[u >> 3][u & 7], S.index[at] = e + u;
                    ++at;
                }
        }
        n += found;
    }
    __syncthreads();
    settle<kF32>(A, S, R, row, bins, n, all);
}

size_t up256(size_t b) { return (b + 255) & ~(size_t)255; }

// The workspace, laid out from `base` (or only measured).
size_t lay_out(Args *A, char *base, int n_rows, int n_vocab) {
    const size_t parts = (n_vocab + kPart * kScanParts - 1) / (kPart * kScanParts) * kScanParts, groups = parts * (kPart / kGroup);
    const size_t sums = up256(sizeof(double) * n_rows * parts), tops = up256(sizeof(float) * n_rows * parts);
    if (A) {
        A->parts = (int)parts;
        A->groups = (int)groups;
        A->part_sum = reinterpret_cast<double *>(base);
        A->part_max = reinterpret_cast<float *>(base + sums);
        A->group_max = reinterpret_cast<float *>(base + sums + tops);
    }
    return sums + tops + up256(sizeof(float) * n_rows * groups);
}

bool aligned(const void *p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

constexpr int kMaxRows = 1 << 16;

}  // namespace

extern "C" size_t ds4hip_sample_workspace_bytes(int n_rows, int n_vocab) {
    if (n_rows <= 0 || n_rows > kMaxRows || n_vocab <= 0 || n_vocab > kMaxVocab) return 0;
    return lay_out(nullptr, nullptr, n_rows, n_vocab);
}

extern "C" int ds4hip_sample_tokens(const ds4hip_sample *a, void *workspace, size_t workspace_bytes, void *stream) {
    if (!a || a->n_rows < 0 || a->n_rows > kMaxRows || a->n_vocab <= 0 || a->n_vocab > kMaxVocab ||
        (a->logits_f32 != 0 && a->logits_f32 != 1) || (a->n_rows > 1 && a->row_stride < a->n_vocab))
        return ds4hip_set_last_error(kEINVAL);
    if (a->n_rows == 0) return 0;
    Args A = {};
    if (!a->logits || !a->u || !a->tokens || !a->probs || !workspace || !aligned(a->logits, a->logits_f32 ? 4 : 2) ||
        !aligned(workspace, 8) || workspace_bytes < lay_out(&A, static_cast<char *>(workspace), a->n_rows, a->n_vocab))
        return ds4hip_set_last_error(kEINVAL);
    A.logits = a->logits;
    A.stride = a->row_stride;
    A.n_rows = a->n_rows;
    A.n_vocab = a->n_vocab;
    A.temperature = a->temperature;
    A.top_k = a->top_k;
    A.top_p = a->top_p;
    A.min_p = a->min_p;
    A.u = a->u;
    A.all_temperature = a->all_temperature;
    A.all_top_k = a->all_top_k;
    A.all_top_p = a->all_top_p;
    A.all_min_p = a->all_min_p;
    A.tokens = a->tokens;
    A.probs = a->probs;
    const hipStream_t st = (hipStream_t)stream;
    const dim3 grid((unsigned)a->n_rows * (A.parts / kScanParts));
    if (a->n_vocab <= kRow) {
        hipLaunchKernelGGL(a->logits_f32 ? row_kernel<true> : row_kernel<false>, dim3(a->n_rows), dim3(kThreads), 0, st, A);
        return ds4hip_set_last_error(hip_status(hipGetLastError()));
    }
    if (a->logits_f32) {
        hipLaunchKernelGGL(scan_kernel<true>, grid, dim3(kScanThreads), 0, st, A);
        hipLaunchKernelGGL(pick_kernel<true>, dim3(a->n_rows), dim3(kThreads), 0, st, A);
    } else {
        hipLaunchKernelGGL(scan_kernel<false>, grid, dim3(kScanThreads), 0, st, A);
        hipLaunchKernelGGL(pick_kernel<false>, dim3(a->n_rows), dim3(kThreads), 0, st, A);
    }
    return ds4hip_set_last_error(hip_status(hipGetLastError()));
}
