// window_attn.hip — attention of packed queries over the pages of their
// sequences' FP8 rows: a sliding window and a few first rows that stay visible,
// for prompts and for single tokens, on gfx950 MFMA.
//
// Math, per query at position p and head h over the rows k it sees
// (k <= p and (k > p - window or k < first)):
//   out = sum_k exp(s_k - M) V_k / (exp(sink_h - M) + sum_k exp(s_k - M)),
//   s_k = (q_h . K_k) / sqrt(512), K == V (one latent KV head).
//
// Work split. A problem is 64 rows (queries x heads of one sequence) and the
// key tiles any of them sees. The tiles of all problems are one line that is cut
// into equal parts, one per workgroup, so that ragged lengths, few long
// sequences and many short ones all fill the chip; a problem that a cut falls
// into leaves its parts' (O, m, l) to a merge. The lengths live on the device: a
// plan kernel lays the line out.

#include "attn_tile.h"
#include "ds4hip_common.h"
#include "../../include/ds4hip_pages.h"

#include <algorithm>

using namespace ds4hip;

namespace {

constexpr int kM = 64;               // rows (queries x heads) of a problem
constexpr int kWgs = 512;            // workgroups the line of tiles is cut for
constexpr int kMinTiles = 4;         // tiles of a part
constexpr int kMaxSeqs = 4096;
// P = 2^((s - m) kq + kTop) with s and the row's reference m as the matrix
// instructions leave them and kq its scale to log2: their difference is exact where P
// is large, at any magnitude. The reference moves only where P would pass 2^(kTop +
// kLazy) = 2^15 (f16 ends at 2^16), so outputs are rescaled on few tiles.
constexpr float kTop = 8.0f;
constexpr float kLazy = 7.0f;

struct WinArgs {
    const void *q;
    void *out;
    const float *sinks;
    const uint8_t *codes;
    const int8_t *sexp;
    const uint16_t *tail;
    const int32_t *table, *rows, *q_start, *seq_ids;
    int n_seqs, n_slots, n_q, log_head, window, first, stride, shift, n_pages;
    // workspace
    int prob_cap;
    int *n_prob;
    int2 *prob;              // [prob_cap] sequence and tile of its rows
    long long *pre;          // [prob_cap + 1] tiles before each problem
    long long *wg_tile;      // [kWgs + 1] first tile of each workgroup
    int *wg_prob;            // [kWgs + 1] the problem it lies in
    float *part_ml;          // [2 kWgs][3][kM] references, sums and scales to log2
    float *part_o;           // [2 kWgs][kM][kD] unnormalized outputs
};

// The queries of sequence s: their first packed index and their number, whatever
// q_start holds.
__device__ inline int2 queries_of(const WinArgs &A, int s) {
    if (!A.q_start) return make_int2(s, 1);
    const int b = min(max(A.q_start[s], 0), A.n_q), e = min(max(A.q_start[s + 1], 0), A.n_q);
    return make_int2(b, max(e - b, 0));
}

struct Problem {
    int slot;       // table row; -1: not a sequence of the table
    int q0, n;      // first packed query and the queries of the tile
    int head0;      // first head
    int pos0, pos1; // positions of the first and the last query
    int n_first, t_window, tiles;   // tiles of the first rows, first tile of the window, all tiles
    bool bad;       // names rows that the table does not hold
};

// The rows of a tile: hpt heads (a power of two) of kM / hpt queries.
__device__ inline int log_hpt(const WinArgs &A) { return min(A.log_head, 6); }

__device__ inline Problem problem_of(const WinArgs &A, int s, int tile) {
    Problem P;
    const int lh = log_hpt(A), groups = 1 << (A.log_head - lh), qpt = kM >> lh;
    const int2 qs = queries_of(A, s);
    const int q = (tile >> (A.log_head - lh)) * qpt;
    P.q0 = qs.x + q;
    P.n = min(qpt, qs.y - q);
    P.head0 = (tile & (groups - 1)) << lh;
    P.slot = A.seq_ids ? A.seq_ids[s] : s;
    P.bad = P.slot < 0 || P.slot >= A.n_slots;
    const int rows = P.bad ? 0 : max(A.rows[P.slot], 0);
    P.bad = P.bad || ((rows - 1) >> A.shift) >= A.stride;
    P.pos0 = rows - qs.y + q;
    P.pos1 = P.pos0 + P.n - 1;
    if (P.bad || P.pos1 < 0) {   // one tile that sees nothing
        P.pos1 = -1;
        P.n_first = P.t_window = 0;
        P.tiles = 1;
        return P;
    }
    const int lo = A.window > 0 ? max(0, max(P.pos0, 0) - A.window + 1) : 0;
    P.n_first = (min(A.first, lo) + kTile - 1) / kTile;
    P.t_window = lo / kTile;
    if (P.n_first >= P.t_window) P.n_first = P.t_window = 0;   // they meet: one run of tiles from row 0
    P.tiles = P.n_first + P.pos1 / kTile - P.t_window + 1;
    return P;
}

// First key of the problem's tile i.
__device__ inline int tile_key(const Problem &P, int i) {
    return kTile * (i < P.n_first ? i : P.t_window + i - P.n_first);
}

__device__ inline bool sees(const WinArgs &A, int pos, int key) {
    return key <= pos && (A.window <= 0 || key > pos - A.window || key < A.first);
}

// ---- plan ------------------------------------------------------------------------

// Exclusive sum of v over the 1024 threads; *total receives the sum.
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
    for (int i = 0; i < 16; ++i) {
        const T y = sums[i];
        before += i < w ? y : 0;
        all += y;
    }
    *total = all;
    return before + x - v;
}

__global__ __launch_bounds__(1024) void plan_kernel(const WinArgs A) {
    __shared__ int first_s[kMaxSeqs];   // problems before each sequence
    __shared__ int sums_i[16];
    __shared__ long long sums_l[16];
    const int tid = threadIdx.x;
    const int lh = log_hpt(A), qpt = kM >> lh;
    int n_prob = 0;
    for (int s0 = 0; s0 < A.n_seqs; s0 += 1024) {
        const int s = s0 + tid;
        int n = s < A.n_seqs ? ((queries_of(A, s).y + qpt - 1) / qpt) << (A.log_head - lh) : 0;
        int all;
        const int before = n_prob + block_scan(n, sums_i, &all);
        if (s < A.n_seqs) first_s[s] = before;
        n_prob += all;
    }
    __syncthreads();
    n_prob = min(n_prob, A.prob_cap);   // (only a q_start that goes back names more)
    long long tiles = 0;
    for (int i0 = 0; i0 < n_prob; i0 += 1024) {
        const int i = i0 + tid;
        int n = 0;
        if (i < n_prob) {
            int lo = 0, hi = A.n_seqs;   // the last sequence whose first problem is at most i
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if (first_s[mid] <= i) lo = mid; else hi = mid;
            }
            A.prob[i] = make_int2(lo, i - first_s[lo]);
            n = problem_of(A, lo, i - first_s[lo]).tiles;
        }
        long long all;
        const long long before = tiles + block_scan<long long>(n, sums_l, &all);
        if (i < n_prob) A.pre[i] = before;
        tiles += all;
    }
    if (tid == 0) {
        A.pre[n_prob] = tiles;
        *A.n_prob = n_prob;
    }
    __syncthreads();
    const long long per = max((tiles + kWgs - 1) / kWgs, (long long)kMinTiles);
    for (int b = tid; b <= kWgs; b += 1024) {
        const long long t = min(b * per, tiles);
        int lo = 0, hi = n_prob;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (A.pre[mid] <= t) lo = mid; else hi = mid;
        }
        A.wg_tile[b] = t;
        A.wg_prob[b] = lo;
    }
}

// ---- attention -------------------------------------------------------------------

// One of the workgroup's 16-row query tiles as f16 fragments (hi, and for fp32
// queries lo): lane (n16, g) holds row n16's dims 32 s + 8 g .. + 8. Each row is
// scaled by a power of two that brings its largest value to [2^7, 2^8), so that f16
// keeps what bf16 and fp32 rows of any magnitude hold: hi + lo are off by 2^-22 of
// a value, or 2^-32 of the row's largest. Returns the power's inverse.
template <bool kF32>
__device__ inline float load_q(const WinArgs &A, const Problem &P, int row, int g, half8_t *hi, half8_t *lo) {
    const int lh = log_hpt(A);
    const int qi = row >> lh, head = P.head0 + (row & ((1 << lh) - 1));
    const bool ok = qi < P.n;
    const size_t at = (((size_t)(P.q0 + (ok ? qi : 0)) << A.log_head) + head) * kD + 8 * g;
    float x[16][8];
    float amax = 0.0f;
#pragma unroll
    for (int s = 0; s < 16; ++s) {
        if (kF32) {
            const float *src = static_cast<const float *>(A.q) + at + 32 * s;
            const float4_t a = *reinterpret_cast<const float4_t *>(src), b = *reinterpret_cast<const float4_t *>(src + 4);
#pragma unroll
            for (int i = 0; i < 4; ++i) x[s][i] = a[i], x[s][4 + i] = b[i];
        } else {
            const uint4_t v = *reinterpret_cast<const uint4_t *>(static_cast<const uint16_t *>(A.q) + at + 32 * s);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                x[s][2 * i] = bf16_to_f32((uint16_t)(v[i] & 0xFFFF));
                x[s][2 * i + 1] = bf16_to_f32((uint16_t)(v[i] >> 16));
            }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) amax = fmaxf(amax, fabsf(x[s][i]));
    }
    amax = xmax_16_32(amax);
    // (a row of zeros, or with an infinity, is left as it is)
    const int e = amax > 0.0f && amax < INFINITY ? 7 - ilogbf(amax) : 0;
#pragma unroll
    for (int s = 0; s < 16; ++s)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float v = ok ? ldexpf(x[s][i], e) : 0.0f;
            hi[s][i] = (half_t)v;
            if (kF32) lo[s][i] = (half_t)(v - (float)hi[s][i]);
        }
    return ldexpf(1.0f, -e);
}

// The sink's part of a denominator with reference m.
__device__ inline float sink_term(const WinArgs &A, int head, float m, float kq) {
    return A.sinks ? __builtin_amdgcn_exp2f(fmaf(-m, kq, fmaf(A.sinks[head], kLog2e, kTop))) : 0.0f;
}

template <bool kF32>
__global__ __launch_bounds__(256) void window_kernel(const WinArgs A) {
    __shared__ __attribute__((aligned(16))) uint8_t stage[kStageB];
    __shared__ __attribute__((aligned(16))) half8_t pb[2][4][64];   // [hi, lo][row tile][lane]
    __shared__ float fac_s[kM], m_s[kM], l_s[kM], kq_s[kM];
    __shared__ uint32_t odd_s[4];   // keys whose scores are not finite, per wave
    __shared__ int bad_s;

    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    const int n16 = lane & 15, g = lane >> 4;
    const int wg = blockIdx.x;
    const int n_prob = *A.n_prob;
    long long t = A.wg_tile[wg];
    const long long t_end = A.wg_tile[wg + 1];
    uint32_t ka[2], va[2];
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) {
        const int r = pi_key(16 * kt + n16);
        ka[kt] = r * kRowB + ((16 * g) ^ row_swz(r));
        const int v = pi_key(16 * kt + 4 * g + (n16 >> 2));
        va[kt] = lds_addr(stage) + v * kRowB + 256 * w + ((8 * (n16 & 3)) ^ row_swz(v));
    }

    for (int pi = A.wg_prob[wg]; t < t_end && pi < n_prob; ++pi) {
        const long long p_begin = A.pre[pi], p_end = A.pre[pi + 1];
        const int2 id = A.prob[pi];
        const Problem P = problem_of(A, id.x, id.y);
        const bool begins = t == p_begin, ends = p_end <= t_end;
        const int i0 = (int)(t - p_begin), i1 = (int)(min(p_end, t_end) - p_begin);
        t = min(p_end, t_end);
        const int row = 16 * w + n16, lh = log_hpt(A);
        const int pos = P.pos0 + min(row >> lh, P.n - 1);   // (rows past the queries repeat the last one's)
        half8_t qh[16], ql[16];
        const float unit = load_q<kF32>(A, P, row, g, qh, ql);
        const float kq = unit * (kLog2e / 22.62741699796952f);   // 1 / sqrt(512), in the exp2 domain
        float4_t o[4][8];
#pragma unroll
        for (int a = 0; a < 4; ++a)
#pragma unroll
            for (int b = 0; b < 8; ++b) o[a][b] = float4_t{0, 0, 0, 0};
        float m = -INFINITY, l = 0.0f;
        bool bad = P.bad;
        if (tid == 0) bad_s = 0;
        for (int i = i0; i < i1 && P.pos1 >= 0; ++i) {
            const int key0 = tile_key(P, i);
            {
                const int r = min(key0 + (tid >> 3), P.pos1);
                int page = A.table[(long long)P.slot * A.stride + (r >> A.shift)];
                if (page < 0 || page >= A.n_pages) {
                    bad = true;
                    page = 0;
                }
                Raw R;
                load_raw_row(A.codes, A.sexp, A.tail,
                             ((long long)page << A.shift) + (r & ((1 << A.shift) - 1)), tid & 7, R);
                __syncthreads();   // the last tile's readers are done
                store_tile(stage, tid, R);
            }
            __syncthreads();
            float4_t acc[2];
#pragma unroll
            for (int kt = 0; kt < 2; ++kt) {
                acc[kt] = float4_t{0, 0, 0, 0};
#pragma unroll
                for (int s = 0; s < 16; ++s) {
                    const half8_t k = *reinterpret_cast<const half8_t *>(stage + ka[kt] + 64 * s);
                    acc[kt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, qh[s], acc[kt], 0, 0, 0);
                    if (kF32) acc[kt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, ql[s], acc[kt], 0, 0, 0);
                }
            }
            const bool edge = !(key0 + kTile - 1 <= P.pos0 &&
                                (A.window <= 0 || key0 > P.pos1 - A.window || key0 + kTile - 1 < A.first));
            float mx = -INFINITY;
            if (edge) {
                uint32_t odd = 0;
#pragma unroll
                for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const int k = pi_key(16 * kt + 4 * g + r);
                        const uint64_t b = __ballot(!(fabsf(acc[kt][r]) < INFINITY));
                        if (((b >> (16 * g)) & 0xFFFF) == 0xFFFF) odd |= 1u << k;
                        if (!sees(A, pos, key0 + k))
                            acc[kt][r] = -INFINITY;
                        else if (!(fabsf(acc[kt][r]) < INFINITY))
                            acc[kt][r] = __builtin_nanf("");
                    }
                odd |= __shfl_xor(odd, 16);
                odd |= __shfl_xor(odd, 32);
                if (lane == 0) odd_s[w] = odd;
            }
#pragma unroll
            for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                for (int r = 0; r < 4; ++r) mx = fmaxf(mx, acc[kt][r]);
            mx = xmax_16_32(mx);
            float fac = 1.0f;
            if ((mx - m) * kq > kLazy) {   // (m is -inf before the first key seen)
                fac = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((m - mx) * kq);
                m = mx;
            }
            l *= fac;
            half8_t ph, pl;
#pragma unroll
            for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const float p = acc[kt][r] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(fmaf(acc[kt][r] - m, kq, kTop));
                    const half_t h = (half_t)p;
                    ph[4 * kt + r] = h;
                    if (kF32) pl[4 * kt + r] = (half_t)(p - (float)h);
                    l += kF32 ? p : (float)h;
                }
            pb[0][w][lane] = ph;
            if (kF32) pb[1][w][lane] = pl;
            if (g == 0) fac_s[row] = fac;
            __syncthreads();
            if (edge) {
                uint32_t odd = odd_s[0] & odd_s[1] & odd_s[2] & odd_s[3];
                // A row that is not finite and that some query must not see: zeroed in this
                // wave's own dims (0 x inf would reach it). Queries that see it have a P that is not finite.
                while (odd) {
                    const int k = __builtin_ctz(odd);
                    odd &= odd - 1;
                    *reinterpret_cast<uint32_t *>(stage + k * kRowB + 256 * w + ((4 * lane) ^ row_swz(k))) = 0;
                }
                asm volatile("" ::: "memory");   // before the reads below, which are asm
            }
            half8_t vb[8];
            read_vt4<0>(va[0], va[1], vb);
            read_vt4<4>(va[0], va[1], vb + 4);
#pragma unroll
            for (int rt = 0; rt < 4; ++rt) {
                const half8_t h = pb[0][rt][lane];
                float f[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) f[r] = fac_s[16 * rt + 4 * g + r];
#pragma unroll
                for (int dt = 0; dt < 8; ++dt) {
#pragma unroll
                    for (int r = 0; r < 4; ++r) o[rt][dt][r] *= f[r];
                    o[rt][dt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(h, vb[dt], o[rt][dt], 0, 0, 0);
                    if (kF32)
                        o[rt][dt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(pb[1][rt][lane], vb[dt], o[rt][dt], 0, 0, 0);
                }
            }
        }
        __syncthreads();
        l = xsum_16_32(l);
        if (g == 0) {
            m_s[row] = m;
            l_s[row] = l;
            kq_s[row] = kq;
        }
        if (__any(bad) && lane == 0) bad_s = 1;
        __syncthreads();
        const float nan = bad_s ? __builtin_nanf("") : 0.0f;
        if (begins && ends) {
#pragma unroll
            for (int rt = 0; rt < 4; ++rt)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int rr = 16 * rt + 4 * g + r, qi = rr >> lh, head = P.head0 + (rr & ((1 << lh) - 1));
                    if (qi >= P.n) continue;
                    const float mm = m_s[rr];
                    const float sink = sink_term(A, head, mm, kq_s[rr]);
                    const float inv = mm == -INFINITY ? nan : 1.0f / (l_s[rr] + sink) + nan;
                    const size_t at = (((size_t)(P.q0 + qi) << A.log_head) + head) * kD + 128 * w + n16;
#pragma unroll
                    for (int dt = 0; dt < 8; ++dt) {
                        const float v = o[rt][dt][r] * inv;
                        if (kF32)
                            static_cast<float *>(A.out)[at + 16 * dt] = v;
                        else
                            static_cast<__bf16 *>(A.out)[at + 16 * dt] = (__bf16)v;
                    }
                }
        } else {
            const int slot = 2 * wg + (begins ? 1 : 0);
            if (tid < kM) {
                float *ml = A.part_ml + (size_t)slot * 3 * kM + tid;
                ml[0] = m_s[tid];
                ml[kM] = l_s[tid] + nan;
                ml[2 * kM] = kq_s[tid];
            }
            float *dst = A.part_o + ((size_t)slot * kM + 4 * g) * kD + 128 * w + n16;
#pragma unroll
            for (int rt = 0; rt < 4; ++rt)
#pragma unroll
                for (int dt = 0; dt < 8; ++dt)
#pragma unroll
                    for (int r = 0; r < 4; ++r) dst[(16 * rt + r) * kD + 16 * dt] = o[rt][dt][r];
        }
        __syncthreads();   // bad_s, m_s and l_s are free again
    }
}

// The parts of each problem that a cut falls into, in order, and the sink. One
// workgroup per four rows and first cut of a problem; a lane's eight dims.
template <bool kF32>
__global__ __launch_bounds__(256) void window_merge_kernel(const WinArgs A) {
    const int b = blockIdx.x / (kM / 4), row = 4 * (blockIdx.x % (kM / 4)) + (threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int n_prob = *A.n_prob, pi = A.wg_prob[b + 1];
    if (pi >= n_prob) return;
    const long long begin = A.pre[pi], end = A.pre[pi + 1], cut = A.wg_tile[b + 1];
    if (cut <= begin || cut >= end || A.wg_tile[b] > begin) return;
    const int2 id = A.prob[pi];
    const Problem P = problem_of(A, id.x, id.y);
    const int lh = log_hpt(A), qi = row >> lh, head = P.head0 + (row & ((1 << lh) - 1));
    if (qi >= P.n) return;
    int last = b + 1;
    while (last + 1 < kWgs && A.wg_tile[last + 1] < end) ++last;
    float mx = -INFINITY;
    for (int c = b; c <= last; ++c) mx = fmaxf(mx, A.part_ml[(size_t)(c == b ? 2 * c + 1 : 2 * c) * 3 * kM + row]);
    const float kq = A.part_ml[(size_t)(2 * b + 1) * 3 * kM + 2 * kM + row];
    float den = 0.0f, o[8] = {};
    for (int c = b; c <= last; ++c) {
        const size_t slot = c == b ? 2 * c + 1 : 2 * c;
        const float m = A.part_ml[slot * 3 * kM + row], l = A.part_ml[slot * 3 * kM + kM + row];
        const float f = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((m - mx) * kq);
        den += l * f;
        const float *src = A.part_o + (slot * kM + row) * kD + 8 * lane;
#pragma unroll
        for (int i = 0; i < 8; ++i) o[i] += src[i] * f;
    }
    const float sink = sink_term(A, head, mx, kq);
    // (a part whose rows could not be read has a NaN sum)
    const float inv = mx == -INFINITY && den == 0.0f ? 0.0f : 1.0f / (den + sink);
    const size_t at = (((size_t)(P.q0 + qi) << A.log_head) + head) * kD + 8 * lane;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        if (kF32)
            static_cast<float *>(A.out)[at + i] = o[i] * inv;
        else
            static_cast<__bf16 *>(A.out)[at + i] = (__bf16)(o[i] * inv);
    }
}

size_t up256(size_t b) { return (b + 255) & ~(size_t)255; }

int log2_heads(int n_head) {
    for (int i = 3; i <= 7; ++i)
        if (n_head == 1 << i) return i;
    return -1;
}

// Problems that n_seqs sequences of n_q queries in all can make.
long long prob_cap(int n_seqs, int n_q, int log_head) {
    const int lh = std::min(log_head, 6);
    return ((long long)n_q / (kM >> lh) + n_seqs) << (log_head - lh);
}

// The workspace, laid out from `base` (or only measured).
size_t lay_out(WinArgs *A, char *base, long long cap) {
    size_t at = 0;
    auto take = [&](size_t bytes) {
        char *p = base + at;
        at += up256(bytes);
        return p;
    };
    char *n_prob = take(sizeof(int)), *prob = take(sizeof(int2) * cap), *pre = take(sizeof(long long) * (cap + 1)),
         *wg_tile = take(sizeof(long long) * (kWgs + 1)), *wg_prob = take(sizeof(int) * (kWgs + 1)),
         *ml = take(sizeof(float) * 2 * kWgs * 3 * kM), *o = take(sizeof(float) * 2 * kWgs * kM * kD);
    if (A) {
        A->prob_cap = (int)cap;
        A->n_prob = reinterpret_cast<int *>(n_prob);
        A->prob = reinterpret_cast<int2 *>(prob);
        A->pre = reinterpret_cast<long long *>(pre);
        A->wg_tile = reinterpret_cast<long long *>(wg_tile);
        A->wg_prob = reinterpret_cast<int *>(wg_prob);
        A->part_ml = reinterpret_cast<float *>(ml);
        A->part_o = reinterpret_cast<float *>(o);
    }
    return at;
}

bool aligned(const void *p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

}  // namespace

extern "C" size_t ds4hip_flash_attn_window_fp8_workspace_bytes(int n_seqs, int n_q, int n_head) {
    const int lh = log2_heads(n_head);
    if (lh < 0 || n_seqs <= 0 || n_seqs > kMaxSeqs || n_q <= 0 || n_q > (1 << 24)) return 0;
    return lay_out(nullptr, nullptr, prob_cap(n_seqs, n_q, lh));
}

extern "C" int ds4hip_flash_attn_window_fp8(const ds4hip_window_attn *a, void *workspace, size_t workspace_bytes,
                                            void *stream) {
    if (!a) return ds4hip_set_last_error(kEINVAL);
    const int lh = log2_heads(a->n_head);
    const int shift = a->page_rows > 0 ? __builtin_ctz(a->page_rows) : 0;
    if (lh < 0 || a->n_seqs < 0 || a->n_seqs > kMaxSeqs || a->n_q < 0 || a->n_q > (1 << 24) || a->window < 0 ||
        a->n_first < 0 || (a->io_f32 != 0 && a->io_f32 != 1) || a->page_rows <= 0 || a->page_rows != 1 << shift)
        return ds4hip_set_last_error(kEINVAL);
    if (a->n_seqs == 0 || a->n_q == 0) return 0;
    if (!a->q || !a->out || !a->codes || !a->sexp || !a->tail || !a->table || !a->rows || a->table_stride <= 0 ||
        a->n_slots <= 0 || a->n_cache_rows < a->page_rows || (a->n_cache_rows >> shift) > 0x7FFFFFFF || !workspace ||
        (!a->q_start && a->n_q < a->n_seqs) || (!a->seq_ids && a->n_slots < a->n_seqs) || !aligned(a->q, 16) ||
        !aligned(a->out, a->io_f32 ? 16 : 8) || !aligned(a->codes, 8) || !aligned(a->sexp, 8) || !aligned(a->tail, 16) ||
        !aligned(workspace, 16))
        return ds4hip_set_last_error(kEINVAL);
    WinArgs A = {};
    if (workspace_bytes < lay_out(&A, static_cast<char *>(workspace), prob_cap(a->n_seqs, a->n_q, lh)))
        return ds4hip_set_last_error(kEINVAL);
    A.q = a->q;
    A.out = a->out;
    A.sinks = a->sinks;
    A.codes = a->codes;
    A.sexp = a->sexp;
    A.tail = a->tail;
    A.table = a->table;
    A.rows = a->rows;
    A.q_start = a->q_start;
    A.seq_ids = a->seq_ids;
    A.n_seqs = a->n_seqs;
    A.n_slots = a->n_slots;
    A.n_q = a->n_q;
    A.log_head = lh;
    A.window = a->window;
    A.first = a->n_first;
    A.stride = a->table_stride;
    A.shift = shift;
    A.n_pages = (int)(a->n_cache_rows >> shift);
    const hipStream_t st = (hipStream_t)stream;
    hipLaunchKernelGGL(plan_kernel, dim3(1), dim3(1024), 0, st, A);
    const dim3 merge((kWgs - 1) * (kM / 4));
    if (a->io_f32) {
        hipLaunchKernelGGL(window_kernel<true>, dim3(kWgs), dim3(256), 0, st, A);
        hipLaunchKernelGGL(window_merge_kernel<true>, merge, dim3(256), 0, st, A);
    } else {
        hipLaunchKernelGGL(window_kernel<false>, dim3(kWgs), dim3(256), 0, st, A);
        hipLaunchKernelGGL(window_merge_kernel<false>, merge, dim3(256), 0, st, A);
    }
    return ds4hip_set_last_error(hip_status(hipGetLastError()));
}
