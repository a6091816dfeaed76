// sample.hip — tokens from rows of logits and given random numbers: temperature, top-k, top-p
// and min-p, exactly, without a sort of the vocabulary.
//
// Math, per row l with temperature T > 0 and M = max l. Order the tokens by logit, equal ones by
// index; w_i = 2^((l_i - M) log2(e) / T). Kept are the first k; of them those before which the sum of w is
// under p of all of the k's; of them those with w >= m. Each of the three keeps a head of that order. The token
// is the first one, by index, at which the running sum of the kept w passes u of their total.
//
// Split. scan_kernel reads the logits once: a workgroup takes 8192 of a row into registers and leaves
// their maximum, the sum of their weights (where it will be needed) and the maximum of every 32 (a group).
// pick_kernel has a workgroup a row. Where nothing is cut off, it finds the part by the parts' sums and reads
// that part again. Else it finds a border from the groups' maxima alone: k groups above it hold k tokens
// above it, and the weights of groups' maxima that sum to p of all do as well. The few groups above
// the border are read again; their tokens above it hold all that is kept. Where that is too many (a flat
// distribution, most of the vocabulary), the row is read again, in four or more passes.
//
// Precision. Weights are fp64 (a table of 64 and a polynomial: off by 2^-51), since the index of a running
// sum over a vocabulary is compared with a given border. Sums are fp64 in a fixed order, or, where
// histograms add in any order, whole numbers in steps of 2^-45 of the largest weight.

#include "ds4hip_common.h"
#include "../../include/ds4hip.h"

#include <algorithm>

using namespace ds4hip;

namespace {

constexpr int kPart = 8192, kGroup = 32;   // logits of a workgroup, of a group
constexpr int kMaxVocab = 1 << 18;         // (sums of 2^45 stay in 64 bits)
constexpr int kScanThreads = 256;
constexpr int kThreads = 1024, kWaves = kThreads / 64;
constexpr int kBins = 2048;
constexpr int kList = 4096;      // candidates in LDS
constexpr int kRanked = 512;     // candidates that are put in order by counting
constexpr double kLog2e64 = 1.4426950408889634074;

struct Args {
    const void *logits;
    long long stride;
    int n_rows, n_vocab, parts, groups;   // groups of all parts of a row
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
    double c;        // log2(e) / T; 0: the largest logit
    int k;           // 0: all
    double p, m, u;
    bool valid;
};

__device__ inline Row row_of(const Args &A, int row) {
    Row R;
    const float t = A.temperature ? A.temperature[row] : A.all_temperature;
    const float p = A.top_p ? A.top_p[row] : A.all_top_p, m = A.min_p ? A.min_p[row] : A.all_min_p;
    const int k = A.top_k ? A.top_k[row] : A.all_top_k;
    const float u = A.u[row];
    R.valid = t >= 0.0f && t < INFINITY && p == p && m == m && u >= 0.0f && u < 1.0f;
    R.c = t > 0.0f ? kLog2e64 / t : 0.0;
    R.k = m > 1.0f ? 1 : k > 0 && k < A.n_vocab ? k : 0;   // (a weight over 1: the first one alone)
    R.p = p > 0.0f ? p : 0.0;
    R.m = m > 1.0f ? 0.0 : m;
    R.u = u;
    return R;
}

__device__ inline bool cuts_p(const Row &R) { return R.p < 1.0; }
__device__ inline bool cuts_m(const Row &R) { return R.m > 0.0; }
// Whether the sum of all weights is needed.
__device__ inline bool needs_sum(const Row &R) { return R.c > 0.0 && R.k == 0 && (cuts_p(R) || !cuts_m(R)); }

// 2^t for t <= 0, from 2^(j/64) in LDS and the Taylor series of 2^r, |r| <= 2^-7, up to r^5.
__device__ inline double pow2(double t, const double *table) {
    if (!(t > -1000.0)) return 0.0;
    const double n = rint(t * 64.0), r = fma(n, -1.0 / 64.0, t);
    const int i = (int)n;
    constexpr double l = 0.69314718055994530942;
    double y = l * l * l * l * l / 120.0;
    y = fma(y, r, l * l * l * l / 24.0);
    y = fma(y, r, l * l * l / 6.0);
    y = fma(y, r, l * l / 2.0);
    y = fma(y, r, l);
    y = fma(y, r, 1.0);
    return __longlong_as_double(__double_as_longlong(table[i & 63] * y) + ((long long)(i >> 6) << 52));
}

__device__ inline void fill_table(double *table) {
    if (threadIdx.x < 64) table[threadIdx.x] = exp2((double)threadIdx.x / 64.0);
}

// Weight of logit x where the row's largest is `top`.
__device__ inline double weight(float x, float top, double c, const double *table) {
    return pow2(((double)x - (double)top) * c, table);
}

// Order of the logits as whole numbers (-0 is 0).
__device__ inline uint32_t key_of(float x) {
    const uint32_t u = __float_as_uint(x + 0.0f);
    return u >> 31 ? ~u : u | 0x80000000u;
}
__device__ inline float value_of(uint32_t k) { return __uint_as_float(k >> 31 ? k & 0x7FFFFFFFu : ~k); }

// Eight logits of a row from e on (-inf past its end). Rows start at any multiple of a logit's size.
template <bool kF32>
__device__ inline void load_eight(const Args &A, int row, int e, float *x) {
    if (kF32) {
        const float *src = static_cast<const float *>(A.logits) + row * A.stride + e;
        if (e + 8 <= A.n_vocab) {
            __builtin_memcpy(x, src, 32);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = e + i < A.n_vocab ? src[i] : -INFINITY;
        }
    } else {
        const uint16_t *src = static_cast<const uint16_t *>(A.logits) + row * A.stride + e;
        if (e + 8 <= A.n_vocab) {
            uint4_t v;
            __builtin_memcpy(&v, src, 16);
#pragma unroll
            for (int i = 0; i < 4; ++i) x[2 * i] = __uint_as_float(v[i] << 16), x[2 * i + 1] = __uint_as_float(v[i] & 0xFFFF0000u);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = e + i < A.n_vocab ? bf16_to_f32(src[i]) : -INFINITY;
        }
    }
}

template <bool kF32>
__device__ inline float load_one(const Args &A, int row, int e) {
    return kF32 ? static_cast<const float *>(A.logits)[row * A.stride + e]
                : bf16_to_f32(static_cast<const uint16_t *>(A.logits)[row * A.stride + e]);
}

__device__ inline float wave_max(float v) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v = fmaxf(v, __shfl_xor(v, off));
    return v;
}

template <bool kF32>
__global__ __launch_bounds__(kScanThreads) void scan_kernel(const Args A) {
    __shared__ double table[64], sum_s[kScanThreads / 64];
    __shared__ float max_s[kScanThreads / 64];
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    const int row = blockIdx.x / A.parts, part = blockIdx.x - row * A.parts;
    float x[4][8], top = -INFINITY;
#pragma unroll
    for (int j = 0; j < 4; ++j) load_eight<kF32>(A, row, part * kPart + j * 2048 + tid * 8, x[j]);
    fill_table(table);
    const Row R = row_of(A, row);
    bool odd = false;
    float *group_max = A.group_max + (size_t)row * A.groups + part * (kPart / kGroup);
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
        if ((lane & 3) == 0) group_max[64 * j + (tid >> 2)] = m;
    }
    top = wave_max(top);
    if (__any(odd)) top = __builtin_nanf("");
    if (lane == 0) max_s[w] = top;
    __syncthreads();
    top = max_s[0];
    odd = top != top;
#pragma unroll
    for (int i = 1; i < kScanThreads / 64; ++i) {
        odd = odd || max_s[i] != max_s[i];
        top = fmaxf(top, max_s[i]);
    }
    if (odd) top = __builtin_nanf("");
    if (tid == 0) A.part_max[(size_t)row * A.parts + part] = top;
    if (!needs_sum(R)) return;
    double sum = 0.0;
    if (top > -INFINITY) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int i = 0; i < 8; ++i) sum += weight(x[j][i], top, R.c, table);
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) sum += __shfl_xor(sum, off);
    if (lane == 0) sum_s[w] = sum;
    __syncthreads();
    if (tid == 0) {
#pragma unroll
        for (int i = 1; i < kScanThreads / 64; ++i) sum += sum_s[i];
        A.part_sum[(size_t)row * A.parts + part] = sum;
    }
}

// ---- pick ------------------------------------------------------------------------

struct Pick {
    double table[64];
    double sums[kWaves];
    int counts[kWaves];
    // the border's and the radix search's histogram
    uint32_t bin_n[kBins];
    unsigned long long bin_w[kBins];
    uint16_t groups[kMaxVocab / kGroup];   // those above the border, by index
    // the candidates, by index
    uint32_t key[kList], index[kList];
    unsigned long long order[kRanked];     // in order of their keys (equal ones by index)
    int found, found_n;
    unsigned long long found_w;
    float top;
};

// Inclusive sum over the workgroup's threads, in their order; *total: of all.
template <typename T>
__device__ inline T block_scan(T v, T *sums, T *total) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    T x = v;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const T y = __shfl_up(x, off);
        if (lane >= off) x += y;
    }
    __syncthreads();
    if (lane == 63) sums[w] = x;
    __syncthreads();
    T before = 0, all = 0;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) {
        before += i < w ? sums[i] : 0;
        all += sums[i];
    }
    *total = all;
    return before + x;
}

__device__ inline void give(const Args &A, int row, int token, float prob) {
    A.tokens[row] = token;
    A.probs[row] = prob;
}

// What is kept, in the order of logits: keys over `key`, and the first `ties` of equal ones.
struct Cut {
    uint32_t key;
    int ties;
};

// A source of tokens in the order of their indexes: item(i, key, index) for i < n.
struct ListSource {
    const Pick &S;
    int n;
    __device__ void eight(int i, uint32_t *key) const {
#pragma unroll
        for (int u = 0; u < 8; ++u) key[u] = i + u < n ? S.key[i + u] : 0;
    }
    __device__ int index(int i) const { return S.index[i]; }
};
template <bool kF32>
struct RowSource {
    const Args &A;
    int row, n;
    __device__ void eight(int i, uint32_t *key) const {
        float x[8];
        load_eight<kF32>(A, row, i, x);
#pragma unroll
        for (int u = 0; u < 8; ++u) key[u] = i + u < n ? key_of(x[u]) : 0;   // (0 is no logit's)
    }
    __device__ int index(int i) const { return i; }
};

// The token: the first by index at which the kept weights' sum passes u of their total. Two passes
// of 8192 items at a time; all threads.
template <typename Source>
__device__ inline void draw(const Args &A, Pick &S, const Source &src, const Row &R, int row, Cut cut) {
    const int tid = threadIdx.x;
    const float top = S.top;
    double total = 0.0, target = 0.0;
    for (int pass = 0; pass < 2; ++pass) {
        if (pass == 1) {
            target = R.u * total;
            if (tid == 0) S.found = 0x7FFFFFFF;
            __syncthreads();
        }
        double sum = 0.0;
        int ties = 0, last = -1;      // last: an item of this thread that is kept
        double last_w = 0.0;
        for (int i0 = 0; i0 < src.n; i0 += 8 * kThreads) {
            const int i = i0 + 8 * tid;
            uint32_t key[8];
            if (i < src.n) {
                src.eight(i, key);
            } else {
#pragma unroll
                for (int u = 0; u < 8; ++u) key[u] = 0;
            }
            int equal = 0, all_equal = 0;
#pragma unroll
            for (int u = 0; u < 8; ++u) equal += key[u] == cut.key;
            const int upto = block_scan(equal, S.counts, &all_equal);
            int tie = ties + upto - equal;
            double w[8], mine = 0.0, all;
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                bool in = key[u] > cut.key || (key[u] == cut.key && tie < cut.ties);
                tie += key[u] == cut.key;
                w[u] = 0.0;
                if (in) {
                    const double x = weight(value_of(key[u]), top, R.c, S.table);
                    w[u] = x >= R.m ? x : 0.0;
                }
                mine += w[u];
            }
            const double incl = sum + block_scan(mine, S.sums, &all);
            if (pass == 1) {
                double at = incl - mine;
                int hit = -1;
                double hit_w = 0.0;
#pragma unroll
                for (int u = 0; u < 8; ++u) {
                    at += w[u];
                    if (w[u] > 0.0) {
                        last = i + u;
                        last_w = w[u];
                        if (hit < 0 && at > target) {
                            hit = i + u;
                            hit_w = w[u];
                        }
                    }
                }
                if (hit >= 0) atomicMin(&S.found, hit);
                __syncthreads();
                const int found = S.found;
                if (found < 0x7FFFFFFF) {
                    if (hit == found) give(A, row, src.index(hit), (float)(hit_w / total));
                    return;
                }
            }
            sum += all;
            ties += all_equal;
        }
        total = sum;
        if (pass == 1) {   // (a rounding of the last sum: the last kept one)
            __syncthreads();
            if (tid == 0) S.found = -1;
            __syncthreads();
            if (last >= 0) atomicMax(&S.found, last);
            __syncthreads();
            if (last >= 0 && last == S.found) give(A, row, src.index(last), (float)(last_w / total));
        }
    }
}

// Of the bins, from the highest key on, the first at which `need` is reached (by counts, or by weights);
// S.found: the bin (-1: none), S.found_n and S.found_w: what lies above it. Two bins a thread.
__device__ inline void find_bin(Pick &S, bool by_weight, unsigned long long need) {
    const int tid = threadIdx.x, hi = kBins - 1 - 2 * tid;
    const unsigned long long n0 = S.bin_n[hi], n1 = S.bin_n[hi - 1], w0 = S.bin_w[hi], w1 = S.bin_w[hi - 1];
    unsigned long long all_n, all_w;
    __shared__ unsigned long long scratch[kWaves];
    const unsigned long long upto_n = block_scan(n0 + n1, scratch, &all_n);
    const unsigned long long upto_w = block_scan(w0 + w1, scratch, &all_w);
    if (tid == 0) S.found = -1;
    __syncthreads();
    const unsigned long long a = by_weight ? upto_w - w0 - w1 : upto_n - n0 - n1, x0 = by_weight ? w0 : n0,
                             x1 = by_weight ? w1 : n1;
    if (a < need && a + x0 + x1 >= need) {
        const bool first = a + x0 >= need;
        S.found = first ? hi : hi - 1;
        S.found_n = (int)(upto_n - n0 - n1 + (first ? 0 : n0));
        S.found_w = upto_w - w0 - w1 + (first ? 0 : w0);
    }
    __syncthreads();
}

constexpr double kUnit = 35184372088832.0;   // 2^45
__device__ inline unsigned long long units(double w) { return (unsigned long long)rint(w * kUnit); }

// The cut of the first k items (by_weight: of the items whose weights before them are under the share
// R.p of `all`, or where that is 0 of all that `within` keeps), by the digits of the keys, highest first.
template <typename Source>
__device__ inline Cut radix(Pick &S, const Source &src, const Row &R, bool by_weight, int k, Cut within, double all) {
    const int tid = threadIdx.x;
    const float top = S.top;
    uint32_t prefix = 0;   // the digits found
    unsigned long long need = k;
    const unsigned long long tie_w = by_weight ? units(weight(value_of(within.key), top, R.c, S.table)) : 0;
    const bool bounded = by_weight && within.key;
    constexpr int kBits[3] = {11, 11, 10};
    int shift = 32;
#pragma unroll 1
    for (int level = 0; level < 3; ++level) {
        const int bits = kBits[level], below = shift;
        shift -= bits;
        for (int i = tid; i < kBins; i += kThreads) S.bin_n[i] = 0, S.bin_w[i] = 0;
        __syncthreads();
        for (int i0 = 0; i0 < src.n; i0 += 8 * kThreads) {
            const int i = i0 + 8 * tid;
            if (i >= src.n) break;
            uint32_t key[8];
            src.eight(i, key);
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                if (key[u] == 0 || (level && key[u] >> below != prefix)) continue;
                if (bounded && key[u] <= within.key) continue;   // (equal ones: below)
                const uint32_t bin = key[u] >> shift & ((1u << bits) - 1);
                atomicAdd(&S.bin_n[bin], 1u);
                if (by_weight) {
                    const unsigned long long w = units(weight(value_of(key[u]), top, R.c, S.table));
                    if (w) atomicAdd(&S.bin_w[bin], w);
                }
            }
        }
        if (bounded && tid == 0 && (!level || within.key >> below == prefix)) {
            const uint32_t bin = within.key >> shift & ((1u << bits) - 1);
            atomicAdd(&S.bin_n[bin], (uint32_t)within.ties);
            atomicAdd(&S.bin_w[bin], within.ties * tie_w);
        }
        __syncthreads();
        if (by_weight && level == 0) {   // the total is known now
            unsigned long long here;
            __shared__ unsigned long long scratch[kWaves];
            block_scan(S.bin_w[2 * tid] + S.bin_w[2 * tid + 1], scratch, &here);
            need = (unsigned long long)ceil(R.p * (all > 0.0 ? all * kUnit : (double)here));
            need = need < 1 ? 1 : need > here ? here : need;
        }
        find_bin(S, by_weight, need);
        prefix = prefix << bits | (uint32_t)S.found;
        need -= by_weight ? S.found_w : S.found_n;
        __syncthreads();
    }
    // all in the last bin are equal: as many of them as are needed
    Cut cut;
    cut.key = prefix;
    if (by_weight) {
        const unsigned long long w = units(weight(value_of(prefix), top, R.c, S.table));
        cut.ties = (int)((need + w - 1) / w);   // (w > 0: its bin reached what was needed)
        if (bounded && prefix == within.key) cut.ties = min(cut.ties, within.ties);
    } else {
        cut.ties = (int)need;
    }
    return cut;
}

// Any number of items; all: the sum of the row's weights, where its share is asked for.
template <typename Source>
__device__ inline void pick_radix(const Args &A, Pick &S, const Source &src, const Row &R, int row, double all) {
    Cut cut = {0, 0};   // all
    if (R.k) cut = radix(S, src, R, false, min(R.k, src.n), cut, 0.0);
    if (cuts_p(R)) cut = radix(S, src, R, true, 0, cut, all);
    draw(A, S, src, R, row, cut);
}

template <bool kF32>
__global__ __launch_bounds__(kThreads) void pick_kernel(const Args A) {
    __shared__ Pick S;
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, row = blockIdx.x;
    const Row R = row_of(A, row);
    fill_table(S.table);
    const float *part_max = A.part_max + (size_t)row * A.parts;
    const double *part_sum = A.part_sum + (size_t)row * A.parts;
    const float *group_max = A.group_max + (size_t)row * A.groups;
    // (every wave for itself; at most 32 parts)
    const float pm = lane < A.parts ? part_max[lane] : -INFINITY;
    const float top = wave_max(pm);
    if (__any(pm != pm) || !(top > -INFINITY) || !R.valid) {
        if (tid == 0) give(A, row, -1, __builtin_nanf(""));
        return;
    }
    if (tid == 0) S.top = top, S.found = 0x7FFFFFFF;
    __syncthreads();
    if (R.c == 0.0) {   // the first group that has the largest, the first of its logits that is it
        for (int i = tid; i < A.groups; i += kThreads)
            if (group_max[i] == top) {
                atomicMin(&S.found, i);
                break;
            }
        __syncthreads();
        if (w == 0) {
            const int e = S.found * kGroup + lane;
            const uint64_t is = __ballot(lane < kGroup && e < A.n_vocab && load_one<kF32>(A, row, min(e, A.n_vocab - 1)) == top);
            if (lane == 0) give(A, row, S.found * kGroup + __builtin_ctzll(is), 1.0f);
        }
        return;
    }
    double all = 0.0;   // of all weights
    if (needs_sum(R)) {
        const double mine = lane < A.parts && pm > -INFINITY ? part_sum[lane] * weight(pm, top, R.c, S.table) : 0.0;
        double upto = mine;
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
            const double y = __shfl_up(upto, off);
            if (lane >= off) upto += y;
        }
        all = __shfl(upto, 63);
        if (!cuts_p(R) && !cuts_m(R)) {   // nothing is cut off
            const double target = R.u * all;
            const uint64_t over = __ballot(mine > 0.0 && upto > target), any = __ballot(mine > 0.0);
            const int part = over ? __builtin_ctzll(over) : 63 - __builtin_clzll(any);
            const double before = __shfl(upto - mine, part);
            float x[8];
            const int e = part * kPart + 8 * tid;
            load_eight<kF32>(A, row, min(e, A.n_vocab), x);   // (past the end: -inf, nothing is read)
            double wt[8], sum = 0.0, ignored;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                wt[i] = weight(x[i], top, R.c, S.table);
                sum += wt[i];
            }
            double at = before + block_scan(sum, S.sums, &ignored) - sum;
            int hit = -1, last = -1;
            double hit_w = 0.0, last_w = 0.0;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                at += wt[i];
                if (wt[i] > 0.0) {
                    last = e + i;
                    last_w = wt[i];
                    if (hit < 0 && at > target) {
                        hit = e + i;
                        hit_w = wt[i];
                    }
                }
            }
            if (hit >= 0) atomicMin(&S.found, hit);
            __syncthreads();
            const int found = S.found;
            if (found < 0x7FFFFFFF) {
                if (hit == found) give(A, row, hit, (float)(hit_w / all));
                return;
            }
            __syncthreads();   // (a rounding of the part's sum: its last one)
            if (tid == 0) S.found = -1;
            __syncthreads();
            if (last >= 0) atomicMax(&S.found, last);
            __syncthreads();
            if (last >= 0 && last == S.found) give(A, row, last, (float)(last_w / all));
            return;
        }
    }

    // The border, as a bin of the distance from the largest logit: `scale` bins per unit, up to the lowest
    // group's maximum. Bins grow with the distance for logits and groups alike, whatever is rounded.
    constexpr int kSteps = kMaxVocab / kGroup / kThreads;
    float g[kSteps], low = INFINITY;
#pragma unroll
    for (int u = 0; u < kSteps; ++u) {
        const int i = u * kThreads + tid;
        g[u] = i < A.groups ? group_max[i] : -INFINITY;
        if (g[u] > -INFINITY) low = fminf(low, g[u]);
    }
    for (int i = tid; i < kBins; i += kThreads) S.bin_n[i] = 0, S.bin_w[i] = 0;
    __shared__ float low_s[kWaves];
    low = -wave_max(-low);
    if (lane == 0) low_s[w] = low;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kWaves; ++i) low = fminf(low, low_s[i]);
    const float span = top - low, scale = span > 0.0f && span < INFINITY ? (kBins - 1) / span : 0.0f;
    auto bin_of = [&](float x) {   // kBins - 1: the largest
        const float d = (top - x) * scale;
        return x > -INFINITY ? kBins - 1 - min((int)fminf(d, (float)kBins), kBins - 1) : -1;
    };
    int border = 0;   // lowest bin of the candidates
    bool enough = true;
    if (R.k || cuts_p(R)) {
#pragma unroll
        for (int u = 0; u < kSteps; ++u) {
            const int b = bin_of(g[u]);
            if (b < 0) continue;
            atomicAdd(&S.bin_n[b], 1u);
            if (!R.k) {
                const unsigned long long x = units(weight(g[u], top, R.c, S.table));
                if (x) atomicAdd(&S.bin_w[b], x);
            }
        }
        __syncthreads();
        // (a step of 2^-44 more for each group than the share asks for: the groups' roundings)
        const unsigned long long need = R.k ? R.k : (unsigned long long)(R.p * all * kUnit) + 2 * A.groups;
        find_bin(S, !R.k, need < 1 ? 1 : need);
        border = S.found;
        enough = border >= 0;
    }
    int n = 0;
    if (enough) {
        // min-p alone gives a border too; exact tests follow
        const float floor_m = cuts_m(R) ? top + (float)(log2(R.m) / R.c) : -INFINITY;
        const float slack = 1e-5f * (fabsf(top) + fabsf(floor_m) + 1e-30f);
        // (not where top-p asks for the sum of the first k, those under the floor among them)
        const float least = floor_m > -INFINITY && !(R.k && cuts_p(R)) ? fminf(floor_m - slack, top) : -INFINITY;
        auto in = [&](float x) { return bin_of(x) >= border && x >= least && x > -INFINITY; };
        // the groups that have a candidate, by index: a thread takes kSteps next to each other
        int n_groups = 0, mine = 0, taken;
        float h[kSteps];
#pragma unroll
        for (int u = 0; u < kSteps; ++u) {
            const int i = tid * kSteps + u;
            h[u] = i < A.groups ? group_max[i] : -INFINITY;
            mine += in(h[u]);
        }
        taken = block_scan(mine, S.counts, &n_groups) - mine;
#pragma unroll
        for (int u = 0; u < kSteps; ++u)
            if (in(h[u])) S.groups[taken++] = (uint16_t)(tid * kSteps + u);
        __syncthreads();
        // their candidates, by index
        for (int i0 = 0; i0 < n_groups * kGroup && n <= kList; i0 += kThreads) {
            const int i = i0 + tid;
            const int e = i < n_groups * kGroup ? S.groups[i >> 5] * kGroup + (i & 31) : A.n_vocab;
            const float x = e < A.n_vocab ? load_one<kF32>(A, row, e) : -INFINITY;
            const bool is = in(x);
            int found;
            const int at = n + block_scan((int)is, S.counts, &found) - 1;
            if (is && at < kList) S.key[at] = key_of(x), S.index[at] = e;
            n += found;
        }
        __syncthreads();
    }
    if (!enough || n > kList) {
        pick_radix(A, S, RowSource<kF32>{A, row, A.n_vocab}, R, row, all);
        return;
    }
    const ListSource list{S, n};
    if (n > kRanked) {
        pick_radix(A, S, list, R, row, all);
        return;
    }
    // Each one's place in the order: how many come before it. Two threads count for one.
    {
        const int i = tid >> 1, half = tid & 1;
        const unsigned long long mine = i < n ? (unsigned long long)S.key[i] << 32 | ~S.index[i] : 0;
        int rank = 0;
        if (i < n)
            for (int j = half; j < n; j += 2) rank += ((unsigned long long)S.key[j] << 32 | ~S.index[j]) > mine;
        rank += __shfl_xor(rank, 1);
        if (i < n && half == 0) S.order[rank] = mine;
    }
    __syncthreads();
    const uint32_t my_key = tid < n ? (uint32_t)(S.order[tid] >> 32) : 0;
    const double mine = tid < n ? weight(value_of(my_key), top, R.c, S.table) : 0.0;
    double total;
    const bool among = tid < n && (!R.k || tid < R.k);
    const double upto = block_scan(among ? mine : 0.0, S.sums, &total);
    if (R.k) all = total;
    const bool stays = among && (tid == 0 || ((!cuts_p(R) || upto - mine < R.p * all) && mine >= R.m));
    int kept;
    block_scan((int)stays, S.counts, &kept);
    // equal ones of the last that stays, among those that do
    const uint32_t last_key = (uint32_t)(S.order[kept - 1] >> 32);
    int ties;
    block_scan((int)(stays && my_key == last_key), S.counts, &ties);
    draw(A, S, list, R, row, Cut{last_key, ties});
}

size_t up256(size_t b) { return (b + 255) & ~(size_t)255; }

// The workspace, laid out from `base` (or only measured).
size_t lay_out(Args *A, char *base, int n_rows, int n_vocab) {
    const size_t parts = (n_vocab + kPart - 1) / kPart, groups = parts * (kPart / kGroup);
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
    const dim3 grid((unsigned)a->n_rows * A.parts);
    if (a->logits_f32) {
        hipLaunchKernelGGL(scan_kernel<true>, grid, dim3(kScanThreads), 0, st, A);
        hipLaunchKernelGGL(pick_kernel<true>, dim3(a->n_rows), dim3(kThreads), 0, st, A);
    } else {
        hipLaunchKernelGGL(scan_kernel<false>, grid, dim3(kScanThreads), 0, st, A);
        hipLaunchKernelGGL(pick_kernel<false>, dim3(a->n_rows), dim3(kThreads), 0, st, A);
    }
    return ds4hip_set_last_error(hip_status(hipGetLastError()));
}
