// window_attn.hip — attention of packed queries over the pages of their
// sequences' FP8 rows: a sliding window and a few first rows that stay visible,
// for prompts, for single tokens and for trees of drafted tokens, on gfx950 MFMA.
//
// Math, per query at position p and head h over the rows k it sees
// (k <= p and (k > p - window or k < first)):
//   out = sum_k exp(s_k - M) V_k / (exp(sink_h - M) + sum_k exp(s_k - M)),
//   s_k = (q_h . K_k) / sqrt(512), K == V (one latent KV head).
// The nodes of a tree are the last rows of their sequence. Node i at depth d sees of them its line to the root
// alone, has position p = (rows before the tree's) + d, and sees an ancestor by that one's position.
//
// Work split. A problem is 64 rows (queries x heads of one sequence), or 16 where the
// sequences have no more on the average, and the key tiles any of them sees. The tiles
// of all problems are one line that is cut into equal parts, one per workgroup, so that
// ragged lengths, few long sequences and many short ones all fill the chip; a problem
// that a cut falls into leaves its parts' (O, m, l) to a merge. The lengths live on the
// device: where problems are few every workgroup lays the line out for itself, else a plan
// kernel does.
//
// What bounds it. In a tile of 64 rows the matrix instructions (0.4 us at peak, 0.9 at a
// library product's rate), 150 or 228 KB through LDS (0.5, 0.7) and the weights take turns: 1.4 us, 1.9
// over a long prompt whose references move, where counters have the matrix units busy for 22% of the cycles and
// the LDS for 23% (8% of those bank conflicts); lists that come from memory wait for it too (2.0: 14%, 15%). Calls
// of a few tiles are launch, the queries, the first rows and the outputs one after the other (about 20 us).
// (A workgroup's place on the line by XCD, so that neighbours share an L2, changed nothing:
// the rows come from there already.)
// Trees of 64 heads: 16 of up to 24 nodes after up to 8192 rows (80 GFLOP) 159 us a call (traced, one after the other,
// 164 and 14 to merge), 75 tiles a workgroup in 1.7 parts on the average; 512 nodes after 60000 rows 0.88 PFLOP/s; 48 of up to 13 in a window of 128 rows
// 30 us, one of 7 after 1500 rows 28 and 6.4 to merge: launch, line (4), queries and first rows (7), tiles (1.6), outputs (3).

#include "attn_tile.h"
#include "ds4hip_common.h"
#include "scan.h"
#include "../../include/ds4hip_pages.h"

#include <algorithm>
#include <cmath>

using namespace ds4hip;

namespace {

constexpr int kMaxWgs = 512;         // workgroups the line of tiles is cut for: one or two per CU
constexpr int kMinTiles = 4;         // tiles of a part
constexpr int kWhole = 8;            // tiles of a problem that is never cut
constexpr int kPart = 12;            // tiles whose time a cut costs: its parts' 256 KB and their merge
constexpr int kSecond = 4;           // tiles whose time a workgroup's second problem costs
constexpr int kHead = 10;            // tiles whose time a problem of trees costs besides its own
constexpr int kMaxSeqs = 4096;
constexpr int kMaxRows = 0x7FFFFF00; // rows of a sequence: a tile's keys stay in 32 bits
constexpr int kFewProbs = 512, kFewProbs16 = 128;   // problems of 64, 16 rows that a workgroup lays out itself
constexpr int kMaxNodes = DS4HIP_TREE_MAX_NODES;     // drafted nodes of a tree
// P = 2^((s - m) kq + top) with s and the row's reference m as the matrix
// instructions leave them and kq its scale to log2: their difference is exact where P is
// large, at any magnitude. The reference moves only where P would pass 2^15 (f16 ends at
// 2^16): a row gains 15 - top bits before it moves. An f16 under 2^-14 is off by up to 2^-25. The largest P
// is 2^top at least, so the small weights of n rows are off by up to n 2^-(25 + top) of it together, in
// the sum and in the outputs, and many that each are little count. So the start grows with the tiles of
// a stretch (the parts of a cut problem have references of their own): with one f16 they are off by
// 2^-16 of the largest together, with hi + lo by 2^-22 (up to 2^18, 2^12 tiles, where it stays at 2^14).
// Moving costs up to half a tile: 4096 queries over windows of 1024 rows, 1% of them eight times as large, took
// 1017 us from 2^-8 on, 1083 from the 2^2 that their 34 tiles ask for; 16 tokens of up to 32768 rows 67 and 69.5.
template <bool kF32>
__device__ inline float start_of(int tiles) {
    const int log_up = 32 - __clz(tiles - 1);   // (of one tile: 0)
    const int top = min(14, kF32 ? max(8, log_up + 2) : max(0, log_up - 4));
    return __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint((float)top)));
}

struct WinArgs {
    const void *q;
    void *out;
    const float *sinks;
    const uint8_t *codes;
    const int8_t *sexp;
    const uint16_t *tail;
    const int32_t *table, *rows, *q_start, *seq_ids;
    const int32_t *parents;  // of the queries' nodes (trees)
    int n_seqs, n_slots, n_q, log_head, window, first, stride, shift, n_pages;
    int log_rows;            // a problem has 2^log_rows rows (queries x heads)
    int n_wg;                // workgroups that the line is cut for
    int uncut;               // 1: no problem is cut, however long
    // workspace
    int prob_cap;
    long long *line;         // [3] tiles per workgroup, tiles of a problem that stays whole, of a problem's head (trees)
    int *n_prob;
    int4 *prob;              // [prob_cap] records
    long long *pre;          // [prob_cap + 1] tiles before each problem
    long long *wg_tile;      // [n_wg + 1] first tile of each workgroup
    int *wg_prob;            // [n_wg + 1] the problem it lies in
    float *part_ml;          // [2 n_wg][3][rows] references, sums and scales to log2
    float *part_o;           // [2 n_wg][rows][kD] unnormalized outputs
};

// The queries of sequence s: their first packed index and their number, whatever
// q_start holds.
__device__ inline int2 queries_of(const WinArgs &A, int s) {
    if (!A.q_start) return make_int2(s, 1);
    const int b = min(max(A.q_start[s], 0), A.n_q), e = min(max(A.q_start[s + 1], 0), A.n_q);
    return make_int2(b, max(e - b, 0));
}

// The heads of a query in one problem.
__device__ inline int log_hpt(const WinArgs &A) { return min(A.log_head, A.log_rows); }

// Sequence s of the call: its first packed query and their number, its table row (-1: not a sequence of
// the table, or one with more rows than its table row holds; of a tree also one with more nodes than a tree may have, or
// than it has rows) and the rows before its queries.
template <bool kTree>
__device__ inline int4 sequence_of(const WinArgs &A, int s) {
    const int slot = A.seq_ids ? A.seq_ids[s] : s;
    const int2 qs = queries_of(A, s);
    const bool in = slot >= 0 && slot < A.n_slots;
    const int rows = in ? max(A.rows[slot], 0) : 0;
    const bool fits = in && rows <= kMaxRows && ((rows - 1) >> A.shift) < A.stride &&
                      (!kTree || (qs.y <= kMaxNodes && qs.y <= rows));
    return make_int4(qs.x, qs.y, fits ? slot : -1, rows - qs.y);
}

// Its problem `tile` as the plan keeps it: table row, first packed query, number of queries, first head
// (times 256) and, of a tree, first node (times 65536), position (of a tree: row) of its first query.
template <bool kTree>
__device__ inline int4 record_of(const WinArgs &A, int4 seq, int tile) {
    const int lh = log_hpt(A), lg = A.log_head - lh, qpt = (1 << A.log_rows) >> lh;
    const int q = (tile >> lg) * qpt;
    return make_int4(seq.z, seq.x + q,
                     min(qpt, seq.y - q) | ((tile & ((1 << lg) - 1)) << lh) << 8 | (kTree && seq.z >= 0 ? q << 16 : 0),
                     seq.w + q);
}

struct Problem {
    int slot;       // table row; -1: names rows that the table does not hold
    int q0, n;      // first packed query and the queries of the tile
    int head0;      // first head
    int pos0, pos1; // positions of the first and the last query; pos1 < 0: it sees nothing
    int n_first, t_window, tiles;   // tiles of the first rows, first tile of the window, all tiles
    int whole_a, whole_b, whole_c;  // tiles t < a, or b <= t, of those t < c, are seen whole by every query
    int node0, base;   // of a tree: the first query's node, the rows before the tree's
};

// A tree's node sees rows before the tree's from its position on backwards, which is base at least and
// no more than its own row's place; rows of the tree as its ancestors are (so no tile of them is whole).
template <bool kTree>
__device__ inline Problem problem_of(const WinArgs &A, int4 rec) {
    Problem P;
    P.slot = rec.x;
    P.q0 = rec.y;
    P.n = rec.z & 255;
    P.head0 = rec.z >> 8 & 255;
    P.node0 = kTree ? rec.z >> 16 : 0;
    P.pos0 = rec.w;
    P.pos1 = P.pos0 + P.n - 1;
    P.base = P.pos0 - P.node0;
    P.n_first = P.t_window = P.whole_a = P.whole_b = P.whole_c = 0;
    if (P.slot < 0 || P.pos1 < 0) {   // one tile that sees nothing
        P.pos1 = -1;
        P.tiles = 1;
        return P;
    }
    const int lo = A.window > 0 ? max(0, max(kTree ? P.base : P.pos0, 0) - A.window + 1) : 0;
    P.n_first = (min(A.first, lo) + kTile - 1) / kTile;
    P.t_window = lo / kTile;
    if (P.n_first >= P.t_window) P.n_first = P.t_window = 0;   // they meet: one run of tiles from row 0
    P.tiles = P.n_first + P.pos1 / kTile - P.t_window + 1;
    P.whole_a = A.first / kTile;
    P.whole_b = A.window > 0 && P.pos1 >= A.window ? (P.pos1 - A.window) / kTile + 1 : 0;
    P.whole_c = kTree ? P.base / kTile : max(P.pos0 + 1, 0) / kTile;
    return P;
}

// Tile of the keys that the problem's i-th one is.
__device__ inline int tile_at(const Problem &P, int i) { return i < P.n_first ? i : P.t_window + i - P.n_first; }

__device__ inline bool sees(const WinArgs &A, int pos, int key) {
    return key <= pos && (A.window <= 0 || key > pos - A.window || key < A.first);
}

// ---- trees -----------------------------------------------------------------------

// What the queries of a problem see of their tree: each one's position (the rows before the tree's
// and its depth), and a bit for each node that is its own or an ancestor's and lies in the window or
// among the first rows.
template <bool kTree, int kRows>
struct Tree {};
template <int kRows>
struct Tree<true, kRows> {
    static constexpr int kWords = kMaxNodes / 32 + 2;
    uint32_t mask[kRows / 8][kWords];   // (8 heads at least) words 1 ..; a word of zeros at each end
    int pos[kRows / 8], base;
};

// All threads of the workgroup, after a barrier of it; false in the threads whose query has an ancestor
// whose parent is none. A thread walks one query's line to the root in LDS, 64 cycles a step (again, where rows before the
// tree's are fewer than the first ones, for what those keep visible); parents come before their children, so every walk
// ends. parent: LDS that nothing else uses up to the second barrier from here (the stage of a later tile).
template <int kThreads, int kRows>
__device__ inline bool plant(const WinArgs &A, const Problem &P, Tree<true, kRows> &T, uint8_t *stage) {
    static_assert(2 * kMaxNodes <= kStageB, "a node's parent takes two bytes");
    const int tid = threadIdx.x, n = P.node0 + P.n;
    short *parent = reinterpret_cast<short *>(stage);   // -1: a child of the last row before the tree's; -2: not a parent
    const int32_t *parents = A.parents + (P.q0 - P.node0);
    for (int i = tid; i < n; i += kThreads) {
        const int p = parents[i];
        parent[i] = (short)(p >= -1 && p < i ? p : -2);
    }
    for (int i = tid; i < P.n * T.kWords; i += kThreads) T.mask[0][i] = 0;
    if (tid == 0) T.base = P.base;
    lds_barrier();
    if (tid >= P.n) return true;
    // the words of the line, from the node's own down; a word is written when the line leaves it
    int v = P.node0 + tid, depth = 0, word = v >> 5;
    uint32_t bits = 0;
    for (; v >= 0; v = parent[v], ++depth) {
        if (v >> 5 != word) {
            T.mask[tid][1 + word] = bits;
            word = v >> 5;
            bits = 0;
        }
        if (A.window <= 0 || depth < A.window) bits |= 1u << (v & 31);
    }
    T.mask[tid][1 + word] = bits;
    const int pos = P.base + depth - 1;
    T.pos[tid] = pos;
    if (A.window > 0 && P.base < A.first)
        for (int u = P.node0 + tid, at = pos; u >= 0; u = parent[u], --at)
            if (at < A.first) T.mask[tid][1 + (u >> 5)] |= 1u << (u & 31);
    return v == -1;
}

// Whether the stretch of tiles up to i1 has any that the masks and positions are needed for.
__device__ inline bool needs_tree(const WinArgs &A, const Problem &P, int i1) {
    return A.window > 0 || tile_at(P, i1 - 1) >= P.whole_c;
}

// What a query sees of the tile from key0 on, for its rows k = 0 .. 31. Of a tree: as bits.
struct TreeSight {
    uint32_t seen;
    __device__ bool operator()(const WinArgs &, int, int k) const { return seen >> k & 1; }
};
struct RowSight {
    int pos;
    __device__ bool operator()(const WinArgs &A, int key0, int k) const { return sees(A, pos, key0 + k); }
};
// The lowest n of 32 bits, of any n.
__device__ inline uint32_t lowest(int n) { return n <= 0 ? 0u : n >= 32 ? ~0u : (1u << n) - 1; }
template <int kRows>
__device__ inline TreeSight sight_of(const WinArgs &A, const Tree<true, kRows> &T, int, int qi, int key0) {
    const int at = __builtin_amdgcn_readfirstlane(key0 - T.base);   // of the tile in the tree's rows
    uint32_t seen = lowest(-at);
    if (A.window > 0) seen &= ~lowest(T.pos[qi] - A.window + 1 - key0) | lowest(A.first - key0);
    if (at > -32) {
        const uint32_t *m = &T.mask[qi][1 + (at >> 5)];
        seen |= (uint32_t)((((uint64_t)m[1] << 32) | m[0]) >> (at & 31));
    }
    return {seen};
}
template <int kRows>
__device__ inline RowSight sight_of(const WinArgs &, const Tree<false, kRows> &, int pos, int, int) { return {pos}; }

// ---- plan ------------------------------------------------------------------------

// Exclusive sum of v over the workgroup's kThreads threads; *total receives the sum.
template <int kThreads>
__device__ inline long long block_scan(long long v, long long *sums, long long *total) {
    return wg_scan<kThreads / 64>(v, sums, total) - v;
}

// put(i, record, tiles before) for every problem; returns their number, *tiles and, in
// *longest (shared, 0 before), the most of one. All threads of the workgroup; first_s, seq_s: [n_seqs] (what the problems
// need of their sequences is loaded once and at once: three loads that wait for each other less).
template <bool kTree, int kThreads, int kEach, typename First, typename Put>
__device__ inline int lay_line(const WinArgs &A, First *first_s, int4 *seq_s, long long *sums, int *longest, long long *tiles, Put put) {
    const int tid = threadIdx.x;
    const int lh = log_hpt(A), lg = A.log_head - lh, qpt = (1 << A.log_rows) >> lh;
    long long n_all = 0, t_all = 0;
    if (A.q_start) {
        for (int s0 = 0; s0 < A.n_seqs; s0 += kThreads) {
            const int s = s0 + tid;
            int4 seq = make_int4(0, 0, 0, 0);
            if (s < A.n_seqs) seq_s[s] = seq = sequence_of<kTree>(A, s);
            const long long n = (long long)((seq.y + qpt - 1) / qpt) << lg;
            long long all;
            const long long before = n_all + block_scan<kThreads>(n, sums, &all);
            if (s < A.n_seqs) first_s[s] = (First)min(before, (long long)A.prob_cap);
            n_all += all;
        }
        __syncthreads();
    } else {
        n_all = (long long)A.n_seqs << lg;
    }
    const int n_prob = (int)min(n_all, (long long)A.prob_cap);   // (only a q_start that goes back names more)
    for (int i0 = 0; i0 < n_prob; i0 += kThreads * kEach) {
        int4 rec[kEach];
        int n[kEach], sum = 0, most = 0;
#pragma unroll
        for (int u = 0; u < kEach; ++u) {
            const int i = i0 + kEach * tid + u;
            n[u] = 0;
            if (i < n_prob) {
                int s = i >> lg, first = s << lg;
                if (A.q_start) {
                    int hi = A.n_seqs;   // the last sequence whose first problem is at most i
                    s = 0;
                    while (hi - s > 1) {
                        const int mid = (s + hi) >> 1;
                        if (first_s[mid] <= i) s = mid; else hi = mid;
                    }
                    first = first_s[s];
                }
                rec[u] = record_of<kTree>(A, A.q_start ? seq_s[s] : sequence_of<kTree>(A, s), i - first);
            }
        }
#pragma unroll
        for (int u = 0; u < kEach; ++u)
            if (i0 + kEach * tid + u < n_prob) {
                n[u] = problem_of<kTree>(A, rec[u]).tiles;
                sum += n[u];   // (four problems have under 2^30)
                most = max(most, n[u]);
            }
        long long all;
        long long before = t_all + block_scan<kThreads>(sum, sums, &all);
#pragma unroll
        for (int u = 0; u < kEach; ++u)
            if (i0 + kEach * tid + u < n_prob) {
                put(i0 + kEach * tid + u, rec[u], before);
                before += n[u];
            }
        t_all += all;
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) most = max(most, __shfl_xor(most, off));
        if ((tid & 63) == 0 && most) atomicMax(longest, most);
    }
    __syncthreads();
    *tiles = t_all;
    return n_prob;
}

// How the line is cut. Where every workgroup can have a problem of its own and the longest
// costs less than parts and their merge would (about kPart tiles), nothing is cut; else at
// every `per` tiles, but not through short problems.
struct Cuts {
    long long tiles, per;
    int whole;   // tiles of a problem that stays whole; < 0: workgroup b has problem b
    int head;    // tiles that the line counts for a problem besides its own
};

// Trees: the line counts kHead tiles more for a problem, the time of its queries, mask and outputs, where workgroups have
// several of them; else one with many short ones ends last. Problems of 64 rows, us with and without, tiles of a
// workgroup in brackets: 12 to 16 trees of up to 32 nodes after 128 to 8192 rows 131, 178 [45], 135, 236 [53], 182, 335 [84];
// after 32 to 2048 rows 79, 121 [13], 107, 212 [26]; 16 of up to 24 after up to 8192 164, 185 [75]; fp32 250, 391 [49]; of
// 16 rows 68, 72 [31]. (14 tiles: 0 to 5% more, 18: up to 30%, 6: up to 10%.) Cuts lie further apart than a head is long, so that every part has a tile.
__device__ inline int head_of(const WinArgs &A, const Cuts &C, int n_prob) {
    const long long per = (C.tiles + (long long)kHead * n_prob + A.n_wg - 1) / A.n_wg;
    return C.whole >= 0 && !A.uncut && per > kHead + 2 ? kHead : 0;
}
__device__ inline void add_heads(const WinArgs &A, Cuts &C, int n_prob) {
    C.tiles += (long long)C.head * n_prob;
    C.per = max(C.per, (C.tiles + A.n_wg - 1) / A.n_wg);
    C.whole += C.head;   // (so what is cut has nine tiles or more)
}

__device__ inline Cuts cuts_of(const WinArgs &A, long long tiles, int n_prob, int longest) {
    const int n_wg = A.n_wg;
    Cuts C;
    C.tiles = tiles;
    C.head = 0;
    // at least sqrt(longest / 16) tiles: a long problem's merge takes 0.09 us a part, a tile 1.5
    C.per = max((tiles + n_wg - 1) / n_wg, (long long)max(kMinTiles, (int)sqrtf((float)longest * 0.0625f)));
    C.whole = A.uncut ? 1 << 30 : (int)min(max((long long)kWhole, C.per / 8), 1LL << 30);
    if (n_prob <= n_wg && longest <= C.per + kPart) {
        C.whole = -1;
        C.per = tiles + 1;   // (no cut inside the line)
    }
    return C;
}

// Tile and problem at which workgroup b begins.
template <typename Pre>
__device__ inline long long begin_of(const Cuts &C, int b, int n_prob, Pre pre, int *prob) {
    if (C.whole < 0) {
        *prob = min(b, n_prob);
        return pre(*prob);
    }
    const long long t = b * C.per;
    *prob = n_prob;
    if (t >= C.tiles) return C.tiles;
    int lo = 0, hi = n_prob;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (pre(mid) <= t) lo = mid; else hi = mid;
    }
    *prob = lo;
    const long long begin = pre(lo), end = pre(lo + 1);
    if (end - begin > C.whole) return t;
    if (2 * t <= begin + end) return begin;   // a short problem goes to the side that has more of it
    *prob = lo + 1;
    return end;
}

// What the merge needs of the plan, besides the problems.
__device__ inline void leave(const WinArgs &A, const Cuts &C, int n_prob) {
    *A.n_prob = n_prob;
    A.line[0] = C.per;
    A.line[1] = C.whole;
    A.line[2] = C.head;
}

// One workgroup, for lines of many problems: latency of a few loads, scans and a search in LDS,
// 10 us for 3840 problems and 12 for 4096 of one sequence.
template <bool kTree>
__global__ __launch_bounds__(1024) void plan_kernel(const WinArgs A) {
    __shared__ int first_s[kMaxSeqs];   // problems before each sequence
    __shared__ int4 seq_s[kMaxSeqs];
    __shared__ long long sums[16];
    long long tiles;
    __shared__ int longest;
    if (threadIdx.x == 0) longest = 0;
    constexpr int kHeld = 8192;   // (64 KB; the search below took half the kernel's time in memory)
    __shared__ long long pre_s[kHeld];
    // four problems a thread: their loads and one sum for 4096 (12 us; with one a thread 17)
    const int n_prob = lay_line<kTree, 1024, 4>(A, first_s, seq_s, sums, &longest, &tiles, [&](int i, int4 rec, long long before) {
        A.prob[i] = rec;
        A.pre[i] = before;
        if (i < kHeld) pre_s[i] = before;
    });
    Cuts C = cuts_of(A, tiles, n_prob, longest);
    if constexpr (kTree) {
        C.head = head_of(A, C, n_prob);
        if (C.head) {
            add_heads(A, C, n_prob);
            for (int i = threadIdx.x; i < n_prob; i += 1024) {
                const long long before = (i < kHeld ? pre_s[i] : A.pre[i]) + (long long)C.head * i;
                A.pre[i] = before;
                if (i < kHeld) pre_s[i] = before;
            }
        }
    }
    if (threadIdx.x == 0) {
        A.pre[n_prob] = C.tiles;
        if (n_prob < kHeld) pre_s[n_prob] = C.tiles;
        leave(A, C, n_prob);
    }
    __syncthreads();
    const int b = threadIdx.x;
    if (b > A.n_wg) return;
    int prob;
    A.wg_tile[b] = begin_of(C, b, n_prob, [&](int i) { return i < kHeld ? pre_s[i] : A.pre[i]; }, &prob);
    A.wg_prob[b] = prob;
}

// The workgroup's own copy of a line of at most kFew problems (0: none).
template <int kFew>
struct Line {
    int4 prob[kFew ? kFew : 1];
    long long pre[kFew + 1], sums[8];
    int4 seq[kFew ? kFew : 1];
    uint16_t first[kFew ? kFew : 1];   // (at most kFew)
    int longest;
};

// Where a workgroup stands: its first problem, and the tiles [t, end) of the line.
struct Place {
    int n_prob, prob;
    long long t, end;
    int part;   // > 0: even parts of that many tiles at most
    int head;   // tiles that the line counts before each problem's own
};

// Few problems: every workgroup lays out the line itself (a launch and a wait less), and
// the first one leaves it to the merge; else the plan kernel did.
template <bool kTree, int kFew, int kThreads>
__device__ inline Place take_place(const WinArgs &A, Line<kFew> &L) {
    const int tid = threadIdx.x, wg = blockIdx.x;
    Place at;
    at.part = at.head = 0;
    if constexpr (kFew != 0) {
        if (tid == 0) L.longest = 0;
        long long tiles;
        at.n_prob = lay_line<kTree, kThreads, 1>(A, L.first, L.seq, L.sums, &L.longest, &tiles, [&](int i, int4 rec, long long before) {
            L.prob[i] = rec;
            L.pre[i] = before;
        });
        if (tid == 0) L.pre[at.n_prob] = tiles;
        __syncthreads();
        Cuts C = cuts_of(A, tiles, at.n_prob, L.longest);
        // Even parts: a problem is cut into equal ones and no workgroup has parts of two (the second's
        // queries and stores take as long as about kSecond tiles); the line then counts a problem as
        // a whole number of cuts. 16 long sequences: 70 us with parts that pass from one to the
        // next, 63 with even ones. Where the parts would be much longer for it (one long sequence among
        // a hundred short ones, whose workgroups are lost to it) they pass.
        if (C.whole >= 0 && !A.uncut && at.n_prob < A.n_wg) {
            const long long per = max(C.per, (tiles + A.n_wg - at.n_prob - 1) / (A.n_wg - at.n_prob));
            if (per <= C.per + kSecond) {   // (a sum over problems of tiles / per, rounded up, is at most n_wg)
                const long long n = tid < at.n_prob ? L.pre[tid + 1] - L.pre[tid] : 0;
                long long all;
                const long long before = block_scan<kThreads>((n + per - 1) / per * per, L.sums, &all);
                if (tid < at.n_prob) L.pre[tid] = before;
                if (tid == 0) L.pre[at.n_prob] = all;
                __syncthreads();
                C.tiles = all;
                C.per = per;
                C.whole = 0;
                at.part = (int)per;
            }
        }
        if constexpr (kTree) {
            C.head = at.part ? 0 : head_of(A, C, at.n_prob);
            if (C.head) {
                add_heads(A, C, at.n_prob);
                for (int i = tid; i <= at.n_prob; i += kThreads) L.pre[i] += (long long)C.head * i;
                __syncthreads();
            }
            at.head = C.head;
        }
        if (wg == 0) {
            for (int i = tid; i <= at.n_prob; i += kThreads) {
                if (i < at.n_prob) A.prob[i] = L.prob[i];
                A.pre[i] = L.pre[i];
            }
            if (tid == 0) leave(A, C, at.n_prob);
        }
        auto pre = [&](int i) { return L.pre[i]; };
        at.end = begin_of(C, wg + 1, at.n_prob, pre, &at.prob);
        at.t = begin_of(C, wg, at.n_prob, pre, &at.prob);
    } else {
        at.n_prob = *A.n_prob;
        at.prob = A.wg_prob[wg];
        at.t = A.wg_tile[wg];
        at.end = A.wg_tile[wg + 1];
        if constexpr (kTree) at.head = (int)A.line[2];
    }
    return at;
}

// Its next stretch of one problem: tiles [i0, i1) of P; false at the end.
struct Stretch {
    Problem P;
    bool begins, ends;
    int i0, i1;
    float top;   // P starts at 2^top
};
template <bool kTree, bool kF32, int kFew>
__device__ inline bool next_stretch(const WinArgs &A, const Line<kFew> &L, Place &at, Stretch &S) {
    if (__builtin_amdgcn_readfirstlane(at.t >= at.end || at.prob >= at.n_prob)) return false;
    const int pi = at.prob++;
    const long long begin = kFew ? L.pre[kFew ? pi : 0] : A.pre[pi], end = kFew ? L.pre[kFew ? pi + 1 : 0] : A.pre[pi + 1];
    const int4 rec = kFew ? L.prob[kFew ? pi : 0] : A.prob[pi];
    S.P = problem_of<kTree>(A, make_int4(__builtin_amdgcn_readfirstlane(rec.x), __builtin_amdgcn_readfirstlane(rec.y),
                                  __builtin_amdgcn_readfirstlane(rec.z), __builtin_amdgcn_readfirstlane(rec.w)));
    S.begins = at.t == begin;
    S.ends = end <= at.end;
    int i0 = (int)(at.t - begin), i1 = (int)(min(end, at.end) - begin);
    if constexpr (kTree) {   // (a cut leaves both sides a tile; cuts lie further apart than heads are long)
        const int last = S.P.tiles - 1;
        if (at.head) {
            i0 = S.begins ? 0 : min(max(i0 - at.head, 1), last);
            i1 = S.ends ? last + 1 : min(max(i1 - at.head, 1), last);
        }
    }
    if (kFew && at.part) {
        const int parts = (int)(end - begin) / at.part, k = i0 / at.part, n = S.P.tiles / parts, more = S.P.tiles - n * parts;
        i0 = n * k + min(k, more);
        i1 = i0 + n + (k < more);
    }
    S.i0 = __builtin_amdgcn_readfirstlane(i0);
    S.i1 = __builtin_amdgcn_readfirstlane(i1);
    S.top = start_of<kF32>(S.i1 - S.i0);
    at.t = min(end, at.end);
    return true;
}

// ---- queries and rows ------------------------------------------------------------

// The order of dims in an LDS row: the first dim of 8-dim granule p. A
// thread's 16-byte code chunk becomes two granules; the first ones of 16 threads lie
// side by side and so do the second ones, so that no LDS write meets another's banks.
__device__ inline int dim_of(int p) {
    const int i = p >> 5, h = p >> 4 & 1, j = p & 15;
    return i == 0 || j < 12 ? 256 * i + 16 * j + 8 * h : kNope + 8 * (j - 12) + 32 * h;
}

// v, as a value the compiler does not know: what rare paths derive from it is computed
// there again, not kept in registers through the loop (where a spilled one's reload would
// wait for every copy in flight).
__device__ inline int again(int v) {
    asm volatile("" : "+v"(v));
    return v;
}

// The largest of the lanes 16 and 32 apart.
__device__ inline uint32_t umax_16_32(uint32_t v) {
    v = max(v, (uint32_t)__shfl_xor((int)v, 16));
    return max(v, (uint32_t)__shfl_xor((int)v, 32));
}

// The power of two that brings a row's largest value, of bits `top`, to [2^7, 2^8); none where
// it is 0 or not finite. (At most 2^120, itself an fp32 value: scores of rows under 2^-113 are
// 0 to all that is done with them, |s| < 2^-88.)
__device__ inline int power_of(uint32_t top) {
    return top && top < 0x7F800000u ? min(7 - ilogbf(__uint_as_float(top)), 120) : 0;
}

// Eight query values from element `at` on.
template <bool kF32>
__device__ inline void load_eight(const void *q, size_t at, float *x) {
    if (kF32) {
        const float *src = static_cast<const float *>(q) + at;
        const float4_t a = *reinterpret_cast<const float4_t *>(src), b = *reinterpret_cast<const float4_t *>(src + 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = a[i], x[4 + i] = b[i];
    } else {
        const uint4_t v = *reinterpret_cast<const uint4_t *>(static_cast<const uint16_t *>(q) + at);
#pragma unroll
        for (int i = 0; i < 4; ++i) x[2 * i] = __uint_as_float(v[i] << 16), x[2 * i + 1] = __uint_as_float(v[i] & 0xFFFF0000u);
    }
}

// A lane's part of a 16-row query tile: lane (n16, g) has row n16's granules g, 4 + g, ..
template <bool kF32>
struct QRow {
    uint4_t x[kF32 ? 32 : 16];
};
// (rows past the queries repeat the last one's)
template <bool kF32>
__device__ inline void load_row(const WinArgs &A, const Problem &P, int row, int g, QRow<kF32> &q) {
    const int lh = log_hpt(A);
    const size_t at = (((size_t)(P.q0 + min(row >> lh, P.n - 1)) << A.log_head) + P.head0 + (row & ((1 << lh) - 1))) * kD;
    const uint8_t *src = static_cast<const uint8_t *>(A.q) + at * (kF32 ? 4 : 2);
#pragma unroll
    for (int s = 0; s < 16; ++s) {
        const uint4_t *from = reinterpret_cast<const uint4_t *>(src + dim_of(4 * s + g) * (kF32 ? 4 : 2));
        if (kF32) {
            q.x[kF32 ? 2 * s : 0] = from[0];
            q.x[kF32 ? 2 * s + 1 : 0] = from[1];
        } else {
            q.x[s] = from[0];
        }
    }
    __builtin_amdgcn_sched_barrier(0);   // all in flight before the first is used
}

// It as f16 fragments (hi, and for fp32 queries lo). Each row is
// scaled by a power of two that brings its largest value to [2^7, 2^8), so that f16
// keeps what bf16 and fp32 rows of any magnitude hold: hi + lo are off by 2^-22 of
// a value, or 2^-32 of the row's largest; hi alone, from bf16, by 2^-31 of the largest (values that become
// subnormal, rounded toward zero: one instruction for two; the others are exact). Returns the power's inverse.
template <bool kF32>
__device__ inline float fragments_of(const QRow<kF32> &q, half8_t *hi, half8_t *lo) {
    if constexpr (kF32) {
        float top = 0.0f;
#pragma unroll
        for (int s = 0; s < 32; ++s)
#pragma unroll
            for (int i = 0; i < 4; ++i) top = fmaxf(top, fabsf(__uint_as_float(q.x[s][i])));
        const int e = power_of(umax_16_32(__float_as_uint(top)));
        const float scale = ldexpf(1.0f, e);
#pragma unroll
        for (int s = 0; s < 16; ++s)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float v = __uint_as_float(q.x[2 * s + (i >> 2)][i & 3]) * scale;
                hi[s][i] = (half_t)v;
                lo[s][i] = (half_t)(v - (float)hi[s][i]);
            }
        return ldexpf(1.0f, -e);
    } else {
        typedef uint16_t ushort2_t __attribute__((ext_vector_type(2)));
        ushort2_t top = {0, 0};   // bits of |x| compare as the values do
#pragma unroll
        for (int s = 0; s < 16; ++s)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                top = __builtin_elementwise_max(top, __builtin_bit_cast(ushort2_t, q.x[s][i] & 0x7FFF7FFFu));
        const int e = power_of(umax_16_32((uint32_t)max(top[0], top[1]) << 16));
        const float scale = ldexpf(1.0f, e);
#pragma unroll
        for (int s = 0; s < 16; ++s)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const auto two = __builtin_amdgcn_cvt_pkrtz(__uint_as_float(q.x[s][i] << 16) * scale,
                                                            __uint_as_float(q.x[s][i] & 0xFFFF0000u) * scale);
                hi[s][2 * i] = (half_t)two[0];
                hi[s][2 * i + 1] = (half_t)two[1];
            }
        return ldexpf(1.0f, -e);
    }
}

// The sink's part of a denominator with reference m, whose weights start at 2^top.
__device__ inline float sink_term(const WinArgs &A, int head, float m, float kq, float top) {
    return A.sinks ? __builtin_amdgcn_exp2f(fmaf(-m, kq, fmaf(A.sinks[head], kLog2e, top))) : 0.0f;
}

// Four outputs, rounded to bf16 unless the call's type is fp32.
template <bool kF32>
__device__ inline void store_out(void *out, size_t at, float4_t v) {
    if (kF32) {
        *reinterpret_cast<float4_t *>(static_cast<float *>(out) + at) = v;
    } else {
        typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
        *reinterpret_cast<bf16x4 *>(static_cast<__bf16 *>(out) + at) = __builtin_convertvector(v, bf16x4);
    }
}

// ---- 64 rows ----------------------------------------------------------------------
//
// bf16: eight waves, two per SIMD, so that one's matrix instructions run under the other's
// vector instructions and waits (four waves of twice the work each: 2.07 us a tile, eight
// 1.6). fp32: four waves, whose queries' hi and lo halves and outputs take the registers of
// two. Wave w has rows 16 (w % 4) .. + 16 and one half of the tile's keys (of eight waves; else both) for
// scores and softmax, and an equal share of the dims of all rows for O += P V.

// The thread's share of a tile: of row tid / 16, code chunks j and (j < 12) j + 16 of 16
// bytes, j = tid % 16, the row's exponents and its tail's dims 4 j .. + 4.
struct Part {
    uint4_t c[2];
    uint2_t t, e;
};

__device__ inline void load_part(const WinArgs &A, long long row, int j, Part &R) {
    const uint8_t *cp = A.codes + row * kNope + 16 * j;
    R.c[0] = *reinterpret_cast<const uint4_t *>(cp);
    // (every thread loads, so that the counts of loads in flight are the same on all paths)
    R.c[1] = *reinterpret_cast<const uint4_t *>(cp + (j < 12 ? 256 : 0));
    R.e = *reinterpret_cast<const uint2_t *>(A.sexp + row * 8);
    R.t = *reinterpret_cast<const uint2_t *>(A.tail + row * kRot + 4 * j);
}

__device__ inline void store_part(uint8_t *stage, int tid, const Part &R) {
    const int row = tid >> 4, j = tid & 15;   // (of the 16 or 32 rows at stage)
    uint8_t *rp = stage + row * kRowB;
    uint8_t *p = rp + 16 * j;   // dim_of's order
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        if (i == 1 && j >= 12) break;
        const int e = (int)(int8_t)(R.e[i] >> (8 * (j >> 2)));   // block j / 4 + 4 i
        const float sc = __uint_as_float((uint32_t)(e + 127) << 23);
        half2_t h[8];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            h[2 * k] = cvt2<false>(R.c[i][k], sc);
            h[2 * k + 1] = cvt2<true>(R.c[i][k], sc);
        }
        *reinterpret_cast<half8_t *>(p + 512 * i) = half8_t{h[0][0], h[0][1], h[1][0], h[1][1], h[2][0], h[2][1], h[3][0], h[3][1]};
        *reinterpret_cast<half8_t *>(p + 512 * i + 256) = half8_t{h[4][0], h[4][1], h[5][0], h[5][1], h[6][0], h[6][1], h[7][0], h[7][1]};
    }
    const int u = j >> 1;   // tail granule
    *reinterpret_cast<uint2_t *>(rp + 512 + 16 * (12 + (u & 3)) + 256 * (u >> 2) + 8 * (j & 1)) = R.t;
}

// Iteration i, with one barrier: scores of tile i | tile i + 1 dequantized, a later one
// fetched | P of tile i | O += P V of tile i - 1. P is computed against the references of the
// tile before. Where a row outgrows its reference, P's tile is marked, and before it is
// used all waves agree on new references, rescale and compute it again from its scores:
// always on the first tile, seldom after it.
//
// Eight waves of two key halves x four row tiles for the scores, 64 dims each for the outputs;
// fp32's hi and lo fragments fill 512 registers a lane, so it has four waves. One tile in flight: two
// gained 7% on lists that come from memory alone and lost on all others. 128 rows a workgroup, which
// would halve the rows read, spilled.
//
// Measured. Six prompts of up to 640 queries of 64 heads over windows of 128 rows and 4: 165 us, 11 a
// problem of six tiles, three of them with masks; the queries and outputs take 3 (212 MB, 1.3
// TB/s). 3 x 501 queries of 16 heads over windows of 500 rows in fp32 (13 GFLOP, issued twice): 90 us.
template <bool kTree, bool kF32, bool kInline>
__global__ __launch_bounds__(kF32 ? 256 : 512, kF32 ? 1 : 2) void window_kernel(const WinArgs A) {
    constexpr int kRT = 4, kRows = 16 * kRT;   // row tiles and rows of a problem
    constexpr int kW = kF32 ? 4 : 8;     // waves
    constexpr int kN = 8 / kW;           // key halves of a wave, and thread rows of a tile
    constexpr int kDT = 4 * kN;          // dim tiles of a wave
    constexpr int kDB = 1024 / kW;       // its bytes of an f16 row
    __shared__ __attribute__((aligned(16))) uint8_t stages[3][kStageB];
    __shared__ __attribute__((aligned(16))) half4_t pb[2][kF32 ? 2 : 1][kRT][64][2];   // [buffer][hi, lo][row tile][lane][key half]
    __shared__ float top_s[2][kRows], l_s[2][kRows], m_s[kRows], kq_s[kRows];
    __shared__ uint32_t odd_s[2][8];   // keys whose scores are not finite, per wave
    __shared__ __attribute__((aligned(16))) int moved_s[2][8];   // whether a row of the wave's outgrew its reference
    __shared__ int bad_s;

    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n16 = lane & 15, g = lane >> 4, row = 16 * (w & 3) + n16;
    const int kh = w >> 2;   // the wave's (first) key half
    const int wg = blockIdx.x;
    constexpr int kFew = kInline ? kFewProbs : 0;
    __shared__ Line<kFew> line;
    __shared__ Tree<kTree, kRows> tree;
    Place at = take_place<kTree, kFew, 64 * kW>(A, line);
    const int lh = log_hpt(A);
    // (the other key half is kHalf further. With a register for it, and one for that of va, the fp32 kernels read three
    // spilled fragments a tile and not two, in one form or the other: 16 queries of 64 heads over 20000 rows 180 us and not 174)
    constexpr uint32_t kHalf = 16 * kRowB;
    const uint32_t ka = pi_key(16 * kh + n16) * kRowB + 16 * g;
    uint32_t va[2];
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) {
        const int v = pi_key(16 * kt + 4 * g + (n16 >> 2));
        va[kt] = lds_addr(stages[0]) + v * kRowB + kDB * w + 8 * (n16 & 3);
    }

    // The page of the thread's u-th row of the first tile is looked up before the outputs of the
    // problem before are stored. (Loading the queries there as well spills 47 registers.)
    Stretch S;
    int page[kN];
    auto next = [&]() {
        if (!next_stretch<kTree, kF32>(A, line, at, S)) return false;
        const int t = again(tid);
#pragma unroll
        for (int u = 0; u < kN; ++u) {
            const int key = min(kTile * tile_at(S.P, S.i0) + (t >> 4) + 16 * u, S.P.pos1);
            page[u] = S.P.pos1 < 0 ? -1 : A.table[(long long)S.P.slot * A.stride + (key >> A.shift)];
        }
        return true;
    };
    bool more = next();
    while (more) {
        const Problem P = S.P;
        const bool begins = S.begins, ends = S.ends;
        const int i0 = S.i0, i1 = S.i1;
        const float start = S.top;
        bool bad = P.slot < 0;
        float4_t o[kRT][kDT];
#pragma unroll
        for (int a = 0; a < kRT; ++a)
#pragma unroll
            for (int b = 0; b < kDT; ++b) o[a][b] = float4_t{0, 0, 0, 0};
        if (tid == 0) bad_s = 0;
        if (P.pos1 >= 0) {   // else its one tile sees nothing
            // row tiles in use; the waves of the others only share the rest
            const int n_rt = ((P.n << lh) + 15) >> 4;
            const bool scores_mine = (w & 3) < n_rt;
            // the thread's u-th row of tile i (past the last row seen: that row again, masked), and its page
            auto row_of = [&](int i, int u) { return min(kTile * tile_at(P, min(i, i1 - 1)) + (tid >> 4) + 16 * u, P.pos1); };
            auto page_of = [&](int i, int u) { return A.table[(long long)P.slot * A.stride + (row_of(i, u) >> A.shift)]; };
            Part R[kN];
            // fetches tile i + 2 (the pages after it first: waiting for a page must not wait for the
            // rows). An entry outside the pool reads row 0
            auto advance = [&](int i) {
                int next[kN];
#pragma unroll
                for (int u = 0; u < kN; ++u) next[u] = page_of(i + 3, u);
#pragma unroll
                for (int u = 0; u < kN; ++u) {
                    if (page[u] < 0 || page[u] >= A.n_pages) {
                        bad = true;
                        page[u] = 0;
                    }
                    load_part(A, ((long long)page[u] << A.shift) + (row_of(i + 2, u) & ((1 << A.shift) - 1)), tid & 15, R[u]);
                    page[u] = next[u];
                }
            };
            auto store = [&](int stage) {
#pragma unroll
                for (int u = 0; u < kN; ++u) store_part(stages[0] + stage + 16 * u * kRowB, tid, R[u]);
            };
            advance(i0 - 2);
            half8_t qh[16], ql[kF32 ? 16 : 1];
            float kq = 0.0f;
            if (scores_mine) {
                QRow<kF32> q;
                load_row<kF32>(A, P, row, g, q);
                kq = fragments_of<kF32>(q, qh, ql) * (kLog2e / 22.62741699796952f);   // 1 / sqrt(512)
            }
            if constexpr (kTree)   // (under the first tile's loads; read after the tiles' first barrier)
                if (needs_tree(A, P, i1)) bad |= !plant<64 * kW>(A, P, tree, stages[2]);
            const int pos = P.pos0 + min(row >> lh, P.n - 1);   // (rows past the queries repeat the last one's)
            float m = -INFINITY, l = 0.0f, sum = 0.0f;
            float ref = 0.0f;   // m, or 0 while there is none
            store(0);
            advance(i0 - 1);
            int sp = 2 * kStageB, sc = 0, sn = kStageB;   // stages of tiles i - 1, i, i + 1
            int buf = 0;                                  // P's of tile i
            float4_t acc[kN];                             // scores of the tile whose P is the newest

            // P of the scores in acc into buffer b
            auto weights = [&](int b) {
                sum = 0.0f;
#pragma unroll
                for (int u = 0; u < kN; ++u) {
                    half4_t ph, pl;
                    float p[4];
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        p[r] = __builtin_amdgcn_exp2f(fmaf(acc[u][r] - ref, kq, start));
                        ph[r] = (half_t)p[r];
                        if (kF32) pl[r] = (half_t)(p[r] - (float)ph[r]);
                    }
                    if (kF32) {
                        sum += (p[0] + p[1]) + (p[2] + p[3]);
                    } else {   // of the rounded values: the output stays an average
                        const half2_t one = {(half_t)1.0f, (half_t)1.0f};
                        sum = __builtin_amdgcn_fdot2(half2_t{ph[0], ph[1]}, one, sum, false);
                        sum = __builtin_amdgcn_fdot2(half2_t{ph[2], ph[3]}, one, sum, false);
                    }
                    pb[b][0][w & 3][lane][kh + u] = ph;
                    if (kF32) pb[b][kF32 ? 1 : 0][w & 3][lane][kh + u] = pl;
                }
            };
            auto top_of = [&]() {
                float x = -INFINITY;
#pragma unroll
                for (int u = 0; u < kN; ++u) x = fmaxf(x, fmaxf(fmaxf(acc[u][0], acc[u][1]), fmaxf(acc[u][2], acc[u][3])));
                return x;
            };

            // O += P V of the tile in stage sp, whose P lies in buffer b (after a barrier)
            auto settle = [&](int b, int4 f0, int4 f1) {
                int any = f0.x | f0.y | f0.z | f0.w;
                if (kW == 8) any |= f1.x | f1.y | f1.z | f1.w;
                if (__builtin_amdgcn_readfirstlane(any)) {
                    const int lane_r = again(lane), n_r = lane_r & 15, row_r = 16 * (w & 3) + n_r;
                    const float top = xmax_16_32(top_of());   // (all lanes take part)
                    if (lane_r < 16 && scores_mine) top_s[kh][row_r] = top;
                    lds_barrier();
                    // every lane: its own row's reference, and those of its output rows
                    auto renew = [&](int r, float &old, float scale) {
                        const float top = kW == 8 ? fmaxf(top_s[0][r], top_s[1][r]) : top_s[0][r];
                        float f = 1.0f;
                        if ((top - old) * scale > 15.0f - start) {   // (-inf before the first key seen)
                            f = old == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((old - top) * scale);
                            old = top;
                        }
                        return f;
                    };
#pragma unroll
                    for (int rt = 0; rt < kRT; ++rt) {
                        if (rt >= n_rt) break;
                        float old = m_s[16 * rt + n_r];
                        const float f = renew(16 * rt + n_r, old, kq_s[16 * rt + n_r]);
                        if (!__any(f != 1.0f)) continue;
#pragma unroll
                        for (int dt = 0; dt < kDT; ++dt) o[rt][dt] *= f;
                    }
                    if (scores_mine) {
                        const float f = renew(row_r, m, kq);
                        if (__any(f != 1.0f)) {   // (the same in both waves of a row tile)
                            l *= f;
                            ref = m == -INFINITY ? 0.0f : m;
                            weights(b);
                        }
                    }
                    lds_barrier();
                    if (scores_mine && kh == 0 && lane_r < 16) m_s[row_r] = m;   // (read again after more barriers)
                }
                l += sum;
            };
            auto add = [&](int b, bool edge) {
                if (edge) {
                    uint32_t odd = odd_s[b][0] & odd_s[b][1] & odd_s[b][2] & odd_s[b][3];
                    if (kW == 8) odd |= odd_s[b][4] & odd_s[b][5] & odd_s[b][6] & odd_s[b][7];
                    odd = __builtin_amdgcn_readfirstlane(odd);
                    // A row that is not finite and that some query must not see: zeroed in this wave's own
                    // dims (0 x inf would reach it). Queries that see it have a P that is not finite.
                    while (odd) {
                        const int k = __builtin_ctz(odd);
                        odd &= odd - 1;
                        if (4 * lane < kDB)
                            *reinterpret_cast<uint32_t *>(stages[0] + sp + k * kRowB + kDB * w + 4 * lane) = 0;
                    }
                    asm volatile("" ::: "memory");   // before the reads below, which are asm
                }
#pragma unroll
                for (int d0 = 0; d0 < kDT; d0 += 4) {
                    half8_t vb[4];
                    if (d0 == 0)
                        read_vt4<0>(va[0] + sp, va[1] + sp, vb);
                    else
                        read_vt4<4>(va[0] + sp, va[1] + sp, vb);
#pragma unroll
                    for (int rt = 0; rt < kRT; ++rt) {
                        if (rt >= n_rt) break;
                        const half8_t h = *reinterpret_cast<const half8_t *>(&pb[b][0][rt][lane][0]);
#pragma unroll
                        for (int dt = 0; dt < 4; ++dt)
                            o[rt][d0 + dt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vb[dt], h, o[rt][d0 + dt], 0, 0, 0);
                        if (kF32) {
                            const half8_t lo = *reinterpret_cast<const half8_t *>(&pb[b][kF32 ? 1 : 0][rt][lane][0]);
#pragma unroll
                            for (int dt = 0; dt < 4; ++dt)
                                o[rt][d0 + dt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vb[dt], lo, o[rt][d0 + dt], 0, 0, 0);
                        }
                    }
                }
            };

            if (kh == 0 && g == 0 && scores_mine) {
                m_s[row] = m;
                kq_s[row] = kq;
            }
            bool edge_before = false;
            auto step = [&](int i) {
                const bool live = i < i1;
                lds_barrier();
                const int4 f0 = *reinterpret_cast<const int4 *>(&moved_s[buf ^ 1][0]), f1 = *reinterpret_cast<const int4 *>(&moved_s[buf ^ 1][4]);
                float4_t a[kN][2];   // two chains each
                if (live && scores_mine) {
                    const uint8_t *st = stages[0] + sc;
#pragma unroll
                    for (int u = 0; u < kN; ++u) a[u][0] = a[u][1] = float4_t{0, 0, 0, 0};
                    half8_t k[2][kN][2];   // K fragments, read two steps ahead
#pragma unroll
                    for (int u = 0; u < kN; ++u)
#pragma unroll
                        for (int v = 0; v < 2; ++v) k[0][u][v] = *reinterpret_cast<const half8_t *>(st + ka + kHalf * u + 64 * v);
#pragma unroll
                    for (int s0 = 0; s0 < 16; s0 += 2) {
                        const int now = (s0 / 2) & 1;
#pragma unroll
                        for (int u = 0; u < kN; ++u)
#pragma unroll
                            for (int v = 0; v < 2; ++v)
                                if (s0 < 14) k[now ^ 1][u][v] = *reinterpret_cast<const half8_t *>(st + ka + kHalf * u + 64 * (s0 + 2 + v));
#pragma unroll
                        for (int u = 0; u < kN; ++u)
#pragma unroll
                            for (int v = 0; v < 2; ++v)
                                a[u][v] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k[now][u][v], qh[s0 + v], a[u][v], 0, 0, 0);
                        if (kF32)
#pragma unroll
                            for (int u = 0; u < kN; ++u)
#pragma unroll
                                for (int v = 0; v < 2; ++v)
                                    a[u][v] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k[now][u][v], ql[kF32 ? s0 + v : 0], a[u][v], 0, 0, 0);
                        __builtin_amdgcn_sched_barrier(0);
                    }
                }
                if (i > i0) {
                    settle(buf ^ 1, f0, f1);   // (acc: still the scores of the tile before)
                    add(buf ^ 1, edge_before);
                }
                if (!live) return;
                store(sn);
                advance(i);
#pragma unroll
                for (int u = 0; u < kN; ++u) acc[u] = a[u][0] + a[u][1];
                const int tile = tile_at(P, i), key0 = kTile * tile;
                const bool edge = !(tile < P.whole_c && (tile >= P.whole_b || tile < P.whole_a));
                if (edge) {
                    uint32_t odd = 0;
                    const int lane_r = again(lane), g_r = lane_r >> 4;
                    const auto sight = sight_of(A, tree, pos, min((16 * (w & 3) + (lane_r & 15)) >> lh, P.n - 1), key0);
#pragma unroll
                    for (int u = 0; u < kN; ++u)
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            const int k = pi_key(16 * (kh + u) + 4 * g_r + r);
                            const bool fine = fabsf(acc[u][r]) < INFINITY;
                            if (((__ballot(!fine) >> (16 * g_r)) & 0xFFFF) == 0xFFFF) odd |= 1u << k;
                            acc[u][r] = !sight(A, key0, k) ? -INFINITY : fine ? acc[u][r] : __builtin_nanf("");
                        }
                    odd |= __shfl_xor(odd, 16);
                    odd |= __shfl_xor(odd, 32);
                    if (lane_r == 0) odd_s[buf][w] = scores_mine ? odd : ~0u;
                }
                const bool moved = scores_mine && __any((top_of() - m) * kq > 15.0f - start);
                if (lane == 0) moved_s[buf][w] = moved;
                if (scores_mine) weights(buf);
                edge_before = edge;
                buf ^= 1;
                const int free = sp;
                sp = sc;
                sc = sn;
                sn = free;
            };
            // the last step only adds the tile before: the code of settle and add stands once
            for (int i = i0; i <= i1; ++i) step(i);
            l = xsum_16_32(l);
            if (g == 0 && scores_mine) l_s[kh][row] = l;
        } else if (tid < kRows) {
            m_s[tid] = -INFINITY;
        }
        if (__any(bad) && lane == 0) bad_s = 1;
        more = next();
        lds_barrier();
        const float nan = bad_s ? __builtin_nanf("") : 0.0f;
        const int lane_e = again(lane), n_e = lane_e & 15, g_e = lane_e >> 4;
        // first of the lane's four dims of the wave's dim tile dt
        auto out_dim = [&](int dt) { return dim_of(kDB / 16 * w + 2 * dt + (g_e >> 1)) + 4 * (g_e & 1); };
        if (begins && ends) {
            constexpr int kOutB = 2 * kD + 16;   // a bf16 row in LDS
#pragma unroll
            for (int rt = 0; rt < kRT; ++rt) {
                const int rr = 16 * rt + n_e, qi = rr >> lh, head = P.head0 + (rr & ((1 << lh) - 1));
                if (qi >= P.n) continue;
                const float mm = m_s[rr];
                const float sum = kW == 8 ? l_s[0][rr] + l_s[1][rr] : l_s[0][rr];
                const float inv = mm == -INFINITY ? nan : 1.0f / (sum + sink_term(A, head, mm, kq_s[rr], start)) + nan;
                const size_t to = (((size_t)(P.q0 + qi) << A.log_head) + head) * kD;
#pragma unroll
                for (int dt = 0; dt < kDT; ++dt) {
                    if (kF32)
                        store_out<true>(A.out, to + out_dim(dt), o[rt][dt] * inv);
                    else
                        store_out<false>(stages[0], (rr * kOutB) / 2 + out_dim(dt), o[rt][dt] * inv);
                }
            }
            if (!kF32) {   // whole rows of 1 KB (eight bytes a lane from the accumulators: 2 us more)
                lds_barrier();
                for (int rr = w; rr < P.n << lh; rr += kW) {
                    const size_t to = (((size_t)(P.q0 + (rr >> lh)) << A.log_head) + P.head0 + (rr & ((1 << lh) - 1))) * kD + 8 * lane_e;
                    *reinterpret_cast<uint4_t *>(static_cast<uint16_t *>(A.out) + to) =
                        *reinterpret_cast<const uint4_t *>(stages[0] + rr * kOutB + 16 * lane_e);
                }
            }
        } else {
            // (as if they had started at 2^0: the parts of a problem need not agree)
            const float down = ldexpf(1.0f, -(int)start);
            const int slot = 2 * wg + (begins ? 1 : 0);
            if (tid < kRows) {
                float *ml = A.part_ml + (size_t)slot * 3 * kRows + tid;
                ml[0] = m_s[tid];
                ml[kRows] = (kW == 8 ? l_s[0][tid] + l_s[1][tid] : l_s[0][tid]) * down + nan;
                ml[2 * kRows] = kq_s[tid];
            }
            float *dst = A.part_o + ((size_t)slot * kRows + n_e) * kD;
#pragma unroll
            for (int rt = 0; rt < kRT; ++rt) {
                if (16 * rt >= P.n << lh) break;
#pragma unroll
                for (int dt = 0; dt < kDT; ++dt) *reinterpret_cast<float4_t *>(dst + 16 * rt * kD + out_dim(dt)) = o[rt][dt] * down;
            }
        }
        lds_barrier();   // what is shared is free again
    }
}

// A thread's share of the tiles of a stretch: its row of each, and the row's page.
struct Fetch {
    Part R;
    int page;
    bool bad;   // a page lay outside the pool
    // (past the last row seen: that row again, masked)
    __device__ int row_of(const Stretch &T, int i, int tid) const {
        return min(kTile * tile_at(T.P, min(i, T.i1 - 1)) + (tid >> 4), T.P.pos1);
    }
    __device__ int page_of(const WinArgs &A, const Stretch &T, int i, int tid) const {
        return A.table[(long long)T.P.slot * A.stride + (row_of(T, i, tid) >> A.shift)];
    }
    // Tile i (the page after it first: waiting for a page must not wait for the rows). An entry
    // outside the pool reads row 0.
    __device__ void tile(const WinArgs &A, const Stretch &T, int i, int tid) {
        const int after = page_of(A, T, i + 1, tid);
        if (page < 0 || page >= A.n_pages) {
            bad = true;
            page = 0;
        }
        load_part(A, ((long long)page << A.shift) + (row_of(T, i, tid) & ((1 << A.shift) - 1)), tid & 15, R);
        page = after;
    }
};

// Whether some query of the problem must not see some row of tile i.
__device__ inline bool edge_at(const Problem &P, int i) {
    const int tile = tile_at(P, i);
    return !(tile < P.whole_c && (tile >= P.whole_b || tile < P.whole_a));
}

// The stages of tiles i - 1, i, i + 1 (bytes from the first), and the P buffer of tile i.
struct Ring {
    int sp = 2 * kStageB, sc = 0, sn = kStageB, buf = 0;
    __device__ void turn() {
        buf ^= 1;
        const int free = sp;
        sp = sc;
        sc = sn;
        sn = free;
    }
};

// ---- 64 rows of bf16, long problems --------------------------------------------------
//
// Four waves make the scores and weights (two row tiles by one key half each, their queries in
// 128 registers), four the outputs (128 dims each, in as many): a K fragment read from LDS
// serves two row tiles, 150 KB a tile and not 228. Iteration i, with one barrier: the first four
// have scores and P of tile i, the others O += P V of tile i - 1; all dequantize tile i + 1
// and fetch a later one. P, its marks and the references are the eight equal waves' ones above. Both
// roles pass the same barriers: one a tile, two more where a tile is marked, which both read
// from the same words.
//
// Measured. 4096 queries of 64 heads over windows of 1024 rows (584 GFLOP): 1.08 ms, 0.54 PFLOP/s,
// half of a library f16 product's 1.1 here. 4096 queries over 32768 rows and their own (18.7 TFLOP):
// 22.7 ms, 0.82 PFLOP/s. 16 single tokens of 64 heads over 105 MB of rows: 63
// us, 1.7 TB/s of the 5.1 that a copy reaches: a tile's chain (wait for its rows, to f16,
// scores, weights, outputs, one barrier) bounds it, 2 us where memory alone would take 0.9.
template <bool kTree, bool kInline>
__global__ __launch_bounds__(512, 2) void roles_kernel(const WinArgs A) {
    constexpr int kRT = 4, kRows = 16 * kRT, kDT = 8;
    constexpr int kFew = kInline ? kFewProbs : 0;
    constexpr int kOutB = 2 * kD + 16;   // a bf16 row in LDS
    __shared__ __attribute__((aligned(16))) uint8_t stages[3][kStageB];
    __shared__ __attribute__((aligned(16))) half4_t pb[2][kRT][64][2];   // [buffer][row tile][lane][key half]
    __shared__ float top_s[2][kRows], l_s[2][kRows], m_s[kRows], kq_s[kRows];
    __shared__ uint32_t odd_s[2][4];   // keys whose scores are not finite, per wave
    __shared__ __attribute__((aligned(16))) int moved_s[2][4];   // whether a row of the wave's outgrew its reference
    __shared__ int bad_s;
    __shared__ Line<kFew> line;
    __shared__ Tree<kTree, kRows> tree;

    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    Place at = take_place<kTree, kFew, 512>(A, line);
    const int lh = log_hpt(A);
    Stretch S;
    Fetch F;
    // (the next problem's first page is looked up before the outputs of this one are stored)
    auto next = [&]() {
        if (!next_stretch<kTree, false>(A, line, at, S)) return false;
        F.page = S.P.pos1 < 0 ? -1 : F.page_of(A, S, S.i0, again(tid));
        return true;
    };
    auto marked = [&](int4 f) { return __builtin_amdgcn_readfirstlane(f.x | f.y | f.z | f.w); };
    // bf16 outputs from LDS, whole rows of 1 KB (eight bytes a lane from the accumulators: 2 us more)
    auto rows_out = [&](const Problem &P) {
        lds_barrier();
        const int lane_e = again(lane);
        for (int row = w; row < P.n << lh; row += 8) {
            const size_t to = (((size_t)(P.q0 + (row >> lh)) << A.log_head) + P.head0 + (row & ((1 << lh) - 1))) * kD + 8 * lane_e;
            *reinterpret_cast<uint4_t *>(static_cast<uint16_t *>(A.out) + to) =
                *reinterpret_cast<const uint4_t *>(stages[0] + row * kOutB + 16 * lane_e);
        }
    };
    if (w < 4) {
        const int n16 = lane & 15, g = lane >> 4, rg = w & 1, kh = w >> 1;
        QRow<false> q[2];   // of the problem to come: no outputs here, so there are registers for them
        auto load_next = [&]() {
            if (!next()) {   // (else their last values would be kept for it)
                q[0] = q[1] = {};
                return false;
            }
            const int lane_q = again(lane);
#pragma unroll
            for (int j = 0; j < 2; ++j) load_row<false>(A, S.P, 32 * rg + 16 * j + (lane_q & 15), lane_q >> 4, q[j]);
            return true;
        };
        bool more = load_next();
        while (more) {
            const Stretch T = S;
            const Problem &P = T.P;
            const bool whole = T.begins && T.ends;
            const int slot = 2 * blockIdx.x + (T.begins ? 1 : 0), i0 = T.i0, i1 = T.i1;
            const int n_rt = ((P.n << lh) + 15) >> 4;   // row tiles in use
            F.bad = P.slot < 0;
            Ring G;
            if (tid == 0) bad_s = 0;
            const bool mine = 2 * rg < n_rt;   // else the wave only shares the rest
            if (P.pos1 >= 0) {
                const uint32_t ka = pi_key(16 * kh + n16) * kRowB + 16 * g;
                F.tile(A, T, i0, tid);
                if constexpr (kTree)   // (with the other role's waves, under the tile's loads)
                    if (needs_tree(A, P, i1)) F.bad |= !plant<512>(A, P, tree, stages[2]);
                half8_t qh[2][16];
                float kq[2] = {0.0f, 0.0f}, m[2], l[2], ref[2], sum[2];   // ref: m, or 0 while there is none
                int pos[2];
                // (not under `mine`: the compiler then spilled 118 registers)
#pragma unroll
                for (int j = 0; j < 2; ++j)
                    kq[j] = fragments_of<false>(q[j], qh[j], nullptr) * (kLog2e / 22.62741699796952f);   // 1 / sqrt(512)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const int row = 32 * rg + 16 * j + n16;
                    pos[j] = P.pos0 + min(row >> lh, P.n - 1);   // (rows past the queries repeat the last one's)
                    m[j] = -INFINITY;
                    l[j] = ref[j] = sum[j] = 0.0f;
                    if (kh == 0 && g == 0) {
                        m_s[row] = -INFINITY;
                        kq_s[row] = kq[j];
                    }
                }
                store_part(stages[0], tid, F.R);
                F.tile(A, T, i0 + 1, tid);
                float4_t acc[2];   // scores of the tile whose P is the newest
                auto weights = [&](int b) {
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        half4_t ph;
#pragma unroll
                        for (int r = 0; r < 4; ++r) ph[r] = (half_t)__builtin_amdgcn_exp2f(fmaf(acc[j][r] - ref[j], kq[j], T.top));
                        // of the rounded values: the output stays an average
                        const half2_t one = {(half_t)1.0f, (half_t)1.0f};
                        sum[j] = __builtin_amdgcn_fdot2(half2_t{ph[0], ph[1]}, one, 0.0f, false);
                        sum[j] = __builtin_amdgcn_fdot2(half2_t{ph[2], ph[3]}, one, sum[j], false);
                        pb[b][2 * rg + j][lane][kh] = ph;
                    }
                };
                auto top_of = [&](int j) { return fmaxf(fmaxf(acc[j][0], acc[j][1]), fmaxf(acc[j][2], acc[j][3])); };
                for (int i = i0;; ++i) {
                    const bool live = i < i1;
                    lds_barrier();
                    const int4 f = *reinterpret_cast<const int4 *>(&moved_s[G.buf ^ 1][0]);
                    float4_t a[2][2];   // two chains each
                    if (live) {
                        const uint8_t *st = stages[0] + G.sc + ka;
#pragma unroll
                        for (int j = 0; j < 2; ++j) a[j][0] = a[j][1] = float4_t{0, 0, 0, 0};
                        half8_t k[2][2];   // K fragments, read two steps ahead
#pragma unroll
                        for (int v = 0; v < 2; ++v) k[0][v] = *reinterpret_cast<const half8_t *>(st + 64 * v);
#pragma unroll
                        for (int s0 = 0; s0 < 16; s0 += 2) {
                            const int now = (s0 / 2) & 1;
#pragma unroll
                            for (int v = 0; v < 2; ++v)
                                if (s0 < 14) k[now ^ 1][v] = *reinterpret_cast<const half8_t *>(st + 64 * (s0 + 2 + v));
#pragma unroll
                            for (int v = 0; v < 2; ++v)
#pragma unroll
                                for (int j = 0; j < 2; ++j)
                                    a[j][v] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k[now][v], qh[j][s0 + v], a[j][v], 0, 0, 0);
                            __builtin_amdgcn_sched_barrier(0);
                        }
                    }
                    if (i > i0) {
                        if (marked(f)) {   // (acc: still the scores of the tile before)
                            const int lane_r = again(lane), n_r = lane_r & 15;
#pragma unroll
                            for (int j = 0; j < 2; ++j) {
                                const float top = xmax_16_32(top_of(j));   // (all lanes take part)
                                if (lane_r < 16 && mine) top_s[kh][32 * rg + 16 * j + n_r] = top;
                            }
                            lds_barrier();
                            if (mine) {
                                bool moves = false;
#pragma unroll
                                for (int j = 0; j < 2; ++j) {
                                    const int row = 32 * rg + 16 * j + n_r;
                                    const float top = fmaxf(top_s[0][row], top_s[1][row]);
                                    if ((top - m[j]) * kq[j] > 15.0f - T.top) {   // (-inf before the first key seen)
                                        l[j] *= m[j] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((m[j] - top) * kq[j]);
                                        ref[j] = m[j] = top;
                                        moves = true;
                                    }
                                }
                                if (__any(moves)) weights(G.buf ^ 1);   // (the same in both waves of a row tile)
                            }
                            lds_barrier();
                            if (mine && kh == 0 && lane_r < 16) {   // (read again after more barriers)
                                m_s[32 * rg + n_r] = m[0];
                                m_s[32 * rg + 16 + n_r] = m[1];
                            }
                        }
                        l[0] += sum[0];
                        l[1] += sum[1];
                    }
                    if (!live) break;
                    store_part(stages[0] + G.sn, tid, F.R);
                    F.tile(A, T, i + 2, tid);
#pragma unroll
                    for (int j = 0; j < 2; ++j) acc[j] = a[j][0] + a[j][1];
                    if (edge_at(P, i)) {
                        const int key0 = kTile * tile_at(P, i), lane_r = again(lane), g_r = lane_r >> 4;
                        uint32_t odd = 0;
                        const decltype(sight_of(A, tree, 0, 0, 0)) sight[2] = {
                            sight_of(A, tree, pos[0], min((32 * rg + (lane_r & 15)) >> lh, P.n - 1), key0),
                            sight_of(A, tree, pos[1], min((32 * rg + 16 + (lane_r & 15)) >> lh, P.n - 1), key0)};
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            const int k = pi_key(16 * kh + 4 * g_r + r);
                            bool any = false;
#pragma unroll
                            for (int j = 0; j < 2; ++j) {
                                const bool fine = fabsf(acc[j][r]) < INFINITY;
                                any = any || fine;
                                acc[j][r] = !sight[j](A, key0, k) ? -INFINITY : fine ? acc[j][r] : __builtin_nanf("");
                            }
                            if (((__ballot(!any) >> (16 * g_r)) & 0xFFFF) == 0xFFFF) odd |= 1u << k;
                        }
                        odd |= __shfl_xor(odd, 16);
                        odd |= __shfl_xor(odd, 32);
                        if (lane_r == 0) odd_s[G.buf][w] = mine ? odd : ~0u;
                    }
                    const bool moved = mine && __any((top_of(0) - m[0]) * kq[0] > 15.0f - T.top || (top_of(1) - m[1]) * kq[1] > 15.0f - T.top);
                    if (lane == 0) moved_s[G.buf][w] = moved;
                    if (mine) weights(G.buf);
                    G.turn();
                }
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    l[j] = xsum_16_32(l[j]);
                    if (g == 0 && mine) l_s[kh][32 * rg + 16 * j + n16] = l[j];
                }
            } else if (tid < kRows) {
                m_s[tid] = -INFINITY;
            }
            if (__any(F.bad) && lane == 0) bad_s = 1;
            more = load_next();
            lds_barrier();
            if (!whole && tid < kRows) {
                float *ml = A.part_ml + (size_t)slot * 3 * kRows + tid;
                ml[0] = m_s[tid];
                ml[kRows] = (l_s[0][tid] + l_s[1][tid]) * ldexpf(1.0f, -(int)T.top) + (bad_s ? __builtin_nanf("") : 0.0f);
                ml[2 * kRows] = kq_s[tid];
            }
            if (whole) rows_out(P);
            lds_barrier();   // what is shared is free again
        }
    } else {
        bool more = next();
        while (more) {
            const Stretch T = S;
            const Problem &P = T.P;
            const bool whole = T.begins && T.ends;
            const int slot = 2 * blockIdx.x + (T.begins ? 1 : 0), i0 = T.i0, i1 = T.i1;
            const int n_rt = ((P.n << lh) + 15) >> 4;   // row tiles in use
            F.bad = P.slot < 0;
            Ring G;
            float4_t o[kRT][kDT];
#pragma unroll
            for (int a = 0; a < kRT; ++a)
#pragma unroll
                for (int b = 0; b < kDT; ++b) o[a][b] = float4_t{0, 0, 0, 0};
            if (P.pos1 >= 0) {
                uint32_t va[2];
#pragma unroll
                for (int kt = 0; kt < 2; ++kt)
                    va[kt] = lds_addr(stages[0]) + pi_key(16 * kt + 4 * (lane >> 4) + ((lane & 15) >> 2)) * kRowB + 256 * (w - 4) + 8 * (lane & 3);
                F.tile(A, T, i0, tid);
                if constexpr (kTree)
                    if (needs_tree(A, P, i1)) F.bad |= !plant<512>(A, P, tree, stages[2]);
                store_part(stages[0], tid, F.R);
                F.tile(A, T, i0 + 1, tid);
                for (int i = i0;; ++i) {
                    lds_barrier();
                    if (i > i0) {
                        const int b = G.buf ^ 1;
                        if (marked(*reinterpret_cast<const int4 *>(&moved_s[b][0]))) {
                            lds_barrier();
                            const int n_r = again(lane) & 15;
#pragma unroll
                            for (int rt = 0; rt < kRT; ++rt) {
                                if (rt >= n_rt) break;
                                const int row = 16 * rt + n_r;
                                const float old = m_s[row], top = fmaxf(top_s[0][row], top_s[1][row]), scale = kq_s[row];
                                const float f = (top - old) * scale > 15.0f - T.top
                                                    ? old == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((old - top) * scale) : 1.0f;
                                if (!__any(f != 1.0f)) continue;
#pragma unroll
                                for (int dt = 0; dt < kDT; ++dt) o[rt][dt] *= f;
                            }
                            lds_barrier();
                        }
                        if (edge_at(P, i - 1)) {
                            // a row that is not finite and that some query must not see: zeroed in this wave's own
                            // dims (0 x inf would reach it). Queries that see it have a P that is not finite.
                            uint32_t odd = __builtin_amdgcn_readfirstlane((odd_s[b][0] & odd_s[b][1]) | (odd_s[b][2] & odd_s[b][3]));
                            for (; odd; odd &= odd - 1)
                                *reinterpret_cast<uint32_t *>(stages[0] + G.sp + __builtin_ctz(odd) * kRowB + 256 * (w - 4) + 4 * lane) = 0;
                            asm volatile("" ::: "memory");   // before the reads below, which are asm
                        }
#pragma unroll
                        for (int d0 = 0; d0 < kDT; d0 += 4) {
                            half8_t vb[4];
                            if (d0 == 0)
                                read_vt4<0>(va[0] + G.sp, va[1] + G.sp, vb);
                            else
                                read_vt4<4>(va[0] + G.sp, va[1] + G.sp, vb);
#pragma unroll
                            for (int rt = 0; rt < kRT; ++rt) {
                                if (rt >= n_rt) break;
                                const half8_t h = *reinterpret_cast<const half8_t *>(&pb[b][rt][lane][0]);
#pragma unroll
                                for (int dt = 0; dt < 4; ++dt)
                                    o[rt][d0 + dt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vb[dt], h, o[rt][d0 + dt], 0, 0, 0);
                            }
                        }
                    }
                    if (i >= i1) break;
                    store_part(stages[0] + G.sn, tid, F.R);
                    F.tile(A, T, i + 2, tid);
                    G.turn();
                }
            }
            if (__any(F.bad) && lane == 0) bad_s = 1;
            more = next();
            lds_barrier();
            const int lane_e = again(lane), n_e = lane_e & 15, g_e = lane_e >> 4;
            // first of the lane's four dims of the wave's dim tile dt
            auto out_dim = [&](int dt) { return dim_of(16 * (w - 4) + 2 * dt + (g_e >> 1)) + 4 * (g_e & 1); };
            if (whole) {
                const float nan = bad_s ? __builtin_nanf("") : 0.0f;
#pragma unroll
                for (int rt = 0; rt < kRT; ++rt) {
                    const int row = 16 * rt + n_e;
                    if (row >> lh >= P.n) continue;
                    const float mm = m_s[row], head_sink = sink_term(A, P.head0 + (row & ((1 << lh) - 1)), mm, kq_s[row], T.top);
                    const float inv = mm == -INFINITY ? nan : 1.0f / (l_s[0][row] + l_s[1][row] + head_sink) + nan;
#pragma unroll
                    for (int dt = 0; dt < kDT; ++dt) store_out<false>(stages[0], (row * kOutB) / 2 + out_dim(dt), o[rt][dt] * inv);
                }
            } else {
                const float down = ldexpf(1.0f, -(int)T.top);   // (as if it had started at 2^0)
                float *dst = A.part_o + ((size_t)slot * kRows + n_e) * kD;
#pragma unroll
                for (int rt = 0; rt < kRT; ++rt) {
                    if (rt >= n_rt) break;
#pragma unroll
                    for (int dt = 0; dt < kDT; ++dt) *reinterpret_cast<float4_t *>(dst + 16 * rt * kD + out_dim(dt)) = o[rt][dt] * down;
                }
            }
            if (whole) rows_out(P);
            lds_barrier();   // what is shared is free again
        }
    }
}

// ---- 16 rows -----------------------------------------------------------------------
//
// Single tokens of a slice of the heads: too few rows to share a key tile's scores out by
// rows (one wave of four would have them all: 3.5 us a tile of fp32). Wave w has dims
// 128 w .. + 128 of the scores' sums and of the outputs; the four partial sums meet in LDS, and
// then every wave has all weights in registers, as its matrix instructions take them, with
// references and sums of its own that agree bit for bit. Two workgroups a CU.
//
// Measured: 4 tokens of 16 heads over 112 MB of rows, fp32: 44 us, 2.5 TB/s (101 us on 64-row
// problems). The same chain bounds it, two of them a CU.
template <bool kTree, bool kF32, bool kInline>
__global__ __launch_bounds__(256, 2) void few_rows_kernel(const WinArgs A) {
    constexpr int kRT = 1, kRows = 16 * kRT;
    constexpr int kFew = kInline ? kFewProbs16 : 0;
    __shared__ __attribute__((aligned(16))) uint8_t stages[2][kStageB];
    __shared__ __attribute__((aligned(16))) float4_t sum_s[4][kRT][2][64];   // [wave][row tile][key half][lane]
    __shared__ uint32_t top_s[4][kRows];   // bits of the largest query value
    __shared__ int bad_s;
    __shared__ Line<kFew> line;
    __shared__ Tree<kTree, kRows> tree;
    // (each on 16 bytes at most)
    static_assert(sizeof(stages) + sizeof(sum_s) + sizeof(top_s) + sizeof(bad_s) + sizeof(line) + sizeof(tree) + 6 * 16 <= 160 * 1024 / 2,
                  "two workgroups a CU");
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    const int n16 = lane & 15, g = lane >> 4;
    Place at = take_place<kTree, kFew, 256>(A, line);
    const int lh = log_hpt(A);
    uint32_t ka[2], va[2];
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) {
        ka[kt] = pi_key(16 * kt + n16) * kRowB + 256 * w + 16 * g;
        va[kt] = lds_addr(stages[0]) + pi_key(16 * kt + 4 * g + (n16 >> 2)) * kRowB + 256 * w + 8 * (n16 & 3);
    }
    Stretch S;
    while (next_stretch<kTree, kF32>(A, line, at, S)) {
        const Problem P = S.P;
        const int i0 = S.i0, i1 = S.i1;
        bool bad = P.slot < 0;
        float4_t o[kRT][8];
#pragma unroll
        for (int a = 0; a < kRT; ++a)
#pragma unroll
            for (int b = 0; b < 8; ++b) o[a][b] = float4_t{0, 0, 0, 0};
        float m[kRT], l[kRT], kq[kRT];
#pragma unroll
        for (int rt = 0; rt < kRT; ++rt) m[rt] = -INFINITY, l[rt] = kq[rt] = 0.0f;
        if (tid == 0) bad_s = 0;
        if (P.pos1 >= 0) {   // else its one tile sees nothing
            // the thread's u-th row of tile i (past the last row seen: that row again, masked), and its page
            auto row_of = [&](int i, int u) { return min(kTile * tile_at(P, min(i, i1 - 1)) + (tid >> 4) + 16 * u, P.pos1); };
            auto page_of = [&](int i, int u) { return A.table[(long long)P.slot * A.stride + (row_of(i, u) >> A.shift)]; };
            Part R[2];
            int page[2] = {page_of(i0, 0), page_of(i0, 1)};
            // fetches tile i (the next one's pages first: waiting for a page must not wait for the
            // rows). An entry outside the pool reads row 0
            auto fetch = [&](int i) {
                const int next[2] = {page_of(i + 1, 0), page_of(i + 1, 1)};
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    if (page[u] < 0 || page[u] >= A.n_pages) {
                        bad = true;
                        page[u] = 0;
                    }
                    load_part(A, ((long long)page[u] << A.shift) + (row_of(i, u) & ((1 << A.shift) - 1)), tid & 15, R[u]);
                    page[u] = next[u];
                }
            };
            auto store = [&](int stage) {
#pragma unroll
                for (int u = 0; u < 2; ++u) store_part(stages[stage] + 16 * u * kRowB, tid, R[u]);
            };
            fetch(i0);
            if constexpr (kTree)   // (under the tile's loads; read after the tiles' first barrier)
                if (needs_tree(A, P, i1)) bad |= !plant<256>(A, P, tree, stages[1]);
            // the wave's quarter of the rows' dims, and its power of two from all quarters' largest values
            float x[kRT][4][8];
            int pos[kRT];
#pragma unroll
            for (int rt = 0; rt < kRT; ++rt) {
                const int row = 16 * rt + n16, qi = min(row >> lh, P.n - 1);   // (rows past the queries repeat the last one's)
                pos[rt] = P.pos0 + qi;
                const size_t from = (((size_t)(P.q0 + qi) << A.log_head) + P.head0 + (row & ((1 << lh) - 1))) * kD;
                uint32_t top = 0;
#pragma unroll
                for (int s = 0; s < 4; ++s) {
                    load_eight<kF32>(A.q, from + dim_of(4 * (4 * w + s) + g), x[rt][s]);
#pragma unroll
                    for (int k = 0; k < 8; ++k) top = max(top, __float_as_uint(x[rt][s][k]) & 0x7FFFFFFFu);
                }
                top = umax_16_32(top);
                if (g == 0) top_s[w][row] = top;
            }
            store(0);
            fetch(i0 + 1);
            lds_barrier();
            half8_t qh[kRT][4], ql[kRT][kF32 ? 4 : 1];
#pragma unroll
            for (int rt = 0; rt < kRT; ++rt) {
                const int row = 16 * rt + n16;
                const int e = power_of(max(max(top_s[0][row], top_s[1][row]), max(top_s[2][row], top_s[3][row])));
                kq[rt] = ldexpf(kLog2e / 22.62741699796952f, -e);   // 1 / sqrt(512)
#pragma unroll
                for (int s = 0; s < 4; ++s)
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        const float v = ldexpf(x[rt][s][k], e);
                        qh[rt][s][k] = (half_t)v;
                        if (kF32) ql[rt][kF32 ? s : 0][k] = (half_t)(v - (float)qh[rt][s][k]);
                    }
            }
            for (int i = i0; i < i1; ++i) {
                const int cur = (i - i0) & 1;
                if (i > i0) lds_barrier();   // the tile is whole, the last one's V and sums are read
                float4_t acc[kRT][2];
                {
                    const uint8_t *st = stages[cur];
#pragma unroll
                    for (int rt = 0; rt < kRT; ++rt) acc[rt][0] = acc[rt][1] = float4_t{0, 0, 0, 0};
#pragma unroll
                    for (int s = 0; s < 4; ++s)
#pragma unroll
                        for (int kt = 0; kt < 2; ++kt) {
                            const half8_t k = *reinterpret_cast<const half8_t *>(st + ka[kt] + 64 * s);
#pragma unroll
                            for (int rt = 0; rt < kRT; ++rt) {
                                acc[rt][kt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, qh[rt][s], acc[rt][kt], 0, 0, 0);
                                if (kF32) acc[rt][kt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, ql[rt][kF32 ? s : 0], acc[rt][kt], 0, 0, 0);
                            }
                        }
                }
#pragma unroll
                for (int rt = 0; rt < kRT; ++rt)
#pragma unroll
                    for (int kt = 0; kt < 2; ++kt) sum_s[w][rt][kt][lane] = acc[rt][kt];
                if (i + 1 < i1) store(cur ^ 1);
                fetch(i + 2);
                lds_barrier();
#pragma unroll
                for (int rt = 0; rt < kRT; ++rt)
#pragma unroll
                    for (int kt = 0; kt < 2; ++kt)
                        acc[rt][kt] = (sum_s[0][rt][kt][lane] + sum_s[1][rt][kt][lane]) + (sum_s[2][rt][kt][lane] + sum_s[3][rt][kt][lane]);
                const int tile = tile_at(P, i), key0 = kTile * tile;
                if (!(tile < P.whole_c && (tile >= P.whole_b || tile < P.whole_a))) {
                    uint32_t odd = 0;   // keys whose scores are not finite in any row
                    const int lane_r = again(lane), g_r = lane_r >> 4;
                    decltype(sight_of(A, tree, 0, 0, 0)) sight[kRT];
#pragma unroll
                    for (int rt = 0; rt < kRT; ++rt)
                        sight[rt] = sight_of(A, tree, pos[rt], min((16 * rt + (lane_r & 15)) >> lh, P.n - 1), key0);
#pragma unroll
                    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            const int k = pi_key(16 * kt + 4 * g_r + r);
                            bool all = true;
#pragma unroll
                            for (int rt = 0; rt < kRT; ++rt) {
                                const bool fine = fabsf(acc[rt][kt][r]) < INFINITY;
                                all = all && !fine;
                                acc[rt][kt][r] = !sight[rt](A, key0, k) ? -INFINITY : fine ? acc[rt][kt][r] : __builtin_nanf("");
                            }
                            if (((__ballot(all) >> (16 * g_r)) & 0xFFFF) == 0xFFFF) odd |= 1u << k;
                        }
                    odd |= __shfl_xor(odd, 16);
                    odd |= __shfl_xor(odd, 32);
                    odd = __builtin_amdgcn_readfirstlane(odd);
                    // such a row is zeroed in this wave's own dims (0 x inf would reach queries that must not
                    // see it). Queries that see it have a P that is not finite.
                    for (; odd; odd &= odd - 1)
                        *reinterpret_cast<uint32_t *>(stages[cur] + __builtin_ctz(odd) * kRowB + 256 * w + 4 * lane) = 0;
                    asm volatile("" ::: "memory");   // before the reads below, which are asm
                }
                half8_t ph[kRT], pl[kRT];
#pragma unroll
                for (int rt = 0; rt < kRT; ++rt) {
                    float top = -INFINITY;
#pragma unroll
                    for (int kt = 0; kt < 2; ++kt)
                        top = fmaxf(top, fmaxf(fmaxf(acc[rt][kt][0], acc[rt][kt][1]), fmaxf(acc[rt][kt][2], acc[rt][kt][3])));
                    top = xmax_16_32(top);
                    const bool moves = (top - m[rt]) * kq[rt] > 15.0f - S.top;   // (m is -inf before the first key seen)
                    if (__any(moves)) {
                        const float f = !moves ? 1.0f : m[rt] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((m[rt] - top) * kq[rt]);
                        if (moves) m[rt] = top;
                        l[rt] *= f;
#pragma unroll
                        for (int dt = 0; dt < 8; ++dt) o[rt][dt] *= f;
                    }
                    const float ref = m[rt] == -INFINITY ? 0.0f : m[rt];
                    float sum[2];   // a tile's before l's: one rounding to l's size a tile, not eight
#pragma unroll
                    for (int kt = 0; kt < 2; ++kt) {
                        float p[4];
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            p[r] = __builtin_amdgcn_exp2f(fmaf(acc[rt][kt][r] - ref, kq[rt], S.top));
                            const half_t h = (half_t)p[r];
                            ph[rt][4 * kt + r] = h;
                            if (kF32) pl[rt][4 * kt + r] = (half_t)(p[r] - (float)h);
                            else p[r] = (float)h;   // (of the rounded values: the output stays an average)
                        }
                        sum[kt] = (p[0] + p[1]) + (p[2] + p[3]);
                    }
                    l[rt] += sum[0] + sum[1];
                }
                const uint32_t v0 = va[0] + cur * kStageB, v1 = va[1] + cur * kStageB;
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    half8_t vb[4];
                    if (half == 0)
                        read_vt4<0>(v0, v1, vb);
                    else
                        read_vt4<4>(v0, v1, vb);
#pragma unroll
                    for (int rt = 0; rt < kRT; ++rt)
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            float4_t &c = o[rt][4 * half + k];
                            c = __builtin_amdgcn_mfma_f32_16x16x32_f16(vb[k], ph[rt], c, 0, 0, 0);
                            if (kF32) c = __builtin_amdgcn_mfma_f32_16x16x32_f16(vb[k], pl[rt], c, 0, 0, 0);
                        }
                }
            }
#pragma unroll
            for (int rt = 0; rt < kRT; ++rt) l[rt] = xsum_16_32(l[rt]);
        }
        if (__any(bad) && lane == 0) bad_s = 1;
        lds_barrier();
        const float nan = bad_s ? __builtin_nanf("") : 0.0f;
        const int slot = 2 * blockIdx.x + (S.begins ? 1 : 0);
#pragma unroll
        for (int rt = 0; rt < kRT; ++rt) {
            const int row = 16 * rt + n16, qi = row >> lh, head = P.head0 + (row & ((1 << lh) - 1));
            if (qi >= P.n) continue;
            if (S.begins && S.ends) {
                const float inv = m[rt] == -INFINITY ? nan : 1.0f / (l[rt] + sink_term(A, head, m[rt], kq[rt], S.top)) + nan;
                const size_t to = (((size_t)(P.q0 + qi) << A.log_head) + head) * kD;
#pragma unroll
                for (int dt = 0; dt < 8; ++dt)
                    store_out<kF32>(A.out, to + dim_of(16 * w + 2 * dt + (g >> 1)) + 4 * (g & 1), o[rt][dt] * inv);
            } else {
                const float down = ldexpf(1.0f, -(int)S.top);   // (as if it had started at 2^0)
                if (w == 0 && g == 0) {
                    float *ml = A.part_ml + (size_t)slot * 3 * kRows + row;
                    ml[0] = m[rt];
                    ml[kRows] = l[rt] * down + nan;
                    ml[2 * kRows] = kq[rt];
                }
                float *to = A.part_o + ((size_t)slot * kRows + row) * kD;
#pragma unroll
                for (int dt = 0; dt < 8; ++dt)
                    *reinterpret_cast<float4_t *>(to + dim_of(16 * w + 2 * dt + (g >> 1)) + 4 * (g & 1)) = o[rt][dt] * down;
            }
        }
        lds_barrier();   // bad_s and the stages are free again
    }
}

// The parts of a problem that cuts fall into, in order, and the sink. A workgroup has
// kShare rows: one, whose parts its four or eight waves share (parts w, w + 4, .., then their sums in
// order), or four, a wave each; a lane has eight dims, eight parts in flight.
// kInline: the workgroups' problems are 0, 1, ..; else those that cuts 1, 2, .. fall into, each
// at its first cut. Measured: 16 problems of 64 rows in 15 parts each, 31 MB: 9.6 us, 3.3 TB/s.
template <bool kF32, bool kInline, int kWaves, int kShare>
__global__ __launch_bounds__(64 * kWaves) void window_merge_kernel(const WinArgs A) {
    constexpr int kStep = kShare == 1 ? kWaves : 1;
    const int rows = 1 << A.log_rows, wgs = rows / kShare;   // workgroups of a problem
    __shared__ float f_s[kWaves][kMaxWgs];   // each wave's parts' factors
    __shared__ float4_t o_s[kShare == 1 ? kWaves - 1 : 1][64][2];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, n_prob = *A.n_prob;
    const int row = kShare == 1 ? blockIdx.x % wgs : 4 * (blockIdx.x % wgs) + w;
    const long long per = A.line[0], whole = A.line[1];
    int pi = blockIdx.x / wgs;
    if (!kInline) pi = A.wg_prob[pi + 1];
    if (pi >= n_prob) return;
    const long long begin = A.pre[pi], end = A.pre[pi + 1];
    const long long b0 = begin / per;   // the workgroup of its first tile; the first cut is the next one's
    if (end - begin <= whole || (b0 + 1) * per >= end) return;
    if (!kInline && b0 != blockIdx.x / wgs) return;
    const Problem P = problem_of<false>(A, A.prob[pi]);   // (its queries and heads)
    const int lh = log_hpt(A), qi = row >> lh, head = P.head0 + (row & ((1 << lh) - 1));
    if (qi >= P.n) return;   // (of four rows, whole waves; one row's waves leave together)
    const int parts = (int)((end - 1) / per - b0) + 1;
    // (the first part is its workgroup's last one, the others their workgroups' first)
    auto slot = [&](int c) { return (size_t)(2 * (b0 + c) + (c == 0)); };
    const float *ml = A.part_ml + row;
    float mx = -INFINITY;
    for (int c = lane; c < parts; c += 64) mx = fmaxf(mx, ml[slot(c) * 3 * rows]);
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) mx = fmaxf(mx, __shfl_xor(mx, off));
    const float kq = ml[slot(0) * 3 * rows + 2 * rows];
    float den = 0.0f;
    for (int c = lane; c < parts; c += 64) {
        const float *x = ml + slot(c) * 3 * rows;
        const float f = x[0] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((x[0] - mx) * kq);
        den += x[rows] * f;
        f_s[w][c] = f;
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) den += __shfl_xor(den, off);
    float4_t o[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
    const float *src = A.part_o + (size_t)row * kD + 8 * lane;
    for (int c0 = kShare == 1 ? w : 0; c0 < parts; c0 += 8 * kStep) {
        float4_t v[8][2];
#pragma unroll
        for (int u = 0; u < 8; ++u)
#pragma unroll
            for (int h = 0; h < 2; ++h)
                v[u][h] = *reinterpret_cast<const float4_t *>(src + slot(min(c0 + kStep * u, parts - 1)) * rows * kD + 4 * h);
#pragma unroll
        for (int u = 0; u < 8; ++u)
            if (c0 + kStep * u < parts) {
                const float f = f_s[w][c0 + kStep * u];
                o[0] += v[u][0] * f;
                o[1] += v[u][1] * f;
            }
    }
    if (kShare == 1) {
        if (w > 0) {
            o_s[w - 1][lane][0] = o[0];
            o_s[w - 1][lane][1] = o[1];
        }
        __syncthreads();
        if (w > 0) return;
#pragma unroll
        for (int k = 0; k < kWaves - 1; ++k) {
            o[0] += o_s[k][lane][0];
            o[1] += o_s[k][lane][1];
        }
    }
    // (a part whose rows could not be read has a NaN sum)
    const float inv = mx == -INFINITY && den == 0.0f ? 0.0f : 1.0f / (den + sink_term(A, head, mx, kq, 0.0f));
    const size_t at = (((size_t)(P.q0 + qi) << A.log_head) + head) * kD + 8 * lane;
    store_out<kF32>(A.out, at, o[0] * inv);
    store_out<kF32>(A.out, at + 4, o[1] * inv);
}

size_t up256(size_t b) { return (b + 255) & ~(size_t)255; }

int log2_heads(int n_head) {
    for (int i = 3; i <= 7; ++i)
        if (n_head == 1 << i) return i;
    return -1;
}

// Problems that n_seqs sequences of n_q queries in all can make.
long long prob_cap(int n_seqs, int n_q, int log_head, int log_rows) {
    const int lh = std::min(log_head, log_rows);
    return ((long long)(n_q >> (log_rows - lh)) + n_seqs) << (log_head - lh);
}

// The workspace, laid out from `base` (or only measured).
size_t lay_out(WinArgs *A, char *base, long long cap, int log_rows) {
    const size_t rows = (size_t)1 << log_rows;
    const int n_wg = log_rows == 6 ? 256 : 512;
    size_t at = 0;
    auto take = [&](size_t bytes) {
        char *p = base + at;
        at += up256(bytes);
        return p;
    };
    char *line = take(3 * sizeof(long long)), *n_prob = take(sizeof(int)), *prob = take(sizeof(int4) * cap),
         *pre = take(sizeof(long long) * (cap + 1)), *wg_tile = take(sizeof(long long) * (n_wg + 1)),
         *wg_prob = take(sizeof(int) * (n_wg + 1)), *ml = take(sizeof(float) * 2 * n_wg * 3 * rows),
         *o = take(sizeof(float) * 2 * n_wg * rows * kD);
    if (A) {
        A->log_rows = log_rows;
        A->n_wg = n_wg;
        A->prob_cap = (int)cap;
        A->line = reinterpret_cast<long long *>(line);
        A->n_prob = reinterpret_cast<int *>(n_prob);
        A->prob = reinterpret_cast<int4 *>(prob);
        A->pre = reinterpret_cast<long long *>(pre);
        A->wg_tile = reinterpret_cast<long long *>(wg_tile);
        A->wg_prob = reinterpret_cast<int *>(wg_prob);
        A->part_ml = reinterpret_cast<float *>(ml);
        A->part_o = reinterpret_cast<float *>(o);
    }
    return at;
}

// Rows of a problem: 64, so that a key tile serves as many as it can; 16 where the sequences
// have no more on the average. Both for 16 heads, one token each, us (16 rows, 64): 4 sequences of up to
// 131072 rows bf16 45, 50, fp32 48, 88; 128 of 1000 bf16 30, 44, fp32 33, 70; one of 4000
// 17.5, 19.9 and 18.6, 28.5; 200 of 100, which need the plan kernel, 16.3, 14.2 and 17.6, 24.0.
int rows_log(int n_seqs, int n_q, int log_head) {
    const long long rows = (long long)n_q << log_head;
    return rows <= 16LL * n_seqs ? 4 : 6;
}

bool aligned(const void *p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

}  // namespace

extern "C" size_t ds4hip_flash_attn_window_fp8_workspace_bytes(int n_seqs, int n_q, int n_head) {
    const int lh = log2_heads(n_head);
    if (lh < 0 || n_seqs <= 0 || n_seqs > kMaxSeqs || n_q <= 0 || n_q > (1 << 24)) return 0;
    // (of either split: what is enough for some sizes is enough for smaller ones)
    size_t most = 0;
    for (int log_rows : {4, 6}) most = std::max(most, lay_out(nullptr, nullptr, prob_cap(n_seqs, n_q, lh, log_rows), log_rows));
    return most;
}

// Trees: the queries are the nodes of their sequences' trees.
template <bool kTree>
static int attend(const ds4hip_window_attn *a, const int32_t *parents, void *workspace, size_t workspace_bytes, void *stream) {
    if (!a) return ds4hip_set_last_error(kEINVAL);
    const int lh = log2_heads(a->n_head);
    const int shift = a->page_rows > 0 ? __builtin_ctz(a->page_rows) : 0;
    if (lh < 0 || a->n_seqs < 0 || a->n_seqs > kMaxSeqs || a->n_q < 0 || a->n_q > (1 << 24) || a->window < 0 ||
        a->n_first < 0 || (a->io_f32 != 0 && a->io_f32 != 1) || a->page_rows <= 0 || a->page_rows != 1 << shift)
        return ds4hip_set_last_error(kEINVAL);
    if (a->n_seqs == 0 || a->n_q == 0) return 0;
    if (!a->q || !a->out || !a->codes || !a->sexp || !a->tail || !a->table || !a->rows || a->table_stride <= 0 ||
        a->n_slots <= 0 || a->n_cache_rows < a->page_rows || (a->n_cache_rows >> shift) > 0x7FFFFFFF || !workspace ||
        (!a->q_start && a->n_q < a->n_seqs) || (kTree && !parents) || (!a->seq_ids && a->n_slots < a->n_seqs) || !aligned(a->q, 16) ||
        !aligned(a->out, 16) || !aligned(a->codes, 16) || !aligned(a->sexp, 8) || !aligned(a->tail, 16) ||
        !aligned(workspace, 16))
        return ds4hip_set_last_error(kEINVAL);
    WinArgs A = {};
    const int log_rows = rows_log(a->n_seqs, a->n_q, lh);
    if (workspace_bytes < lay_out(&A, static_cast<char *>(workspace), prob_cap(a->n_seqs, a->n_q, lh, log_rows), log_rows))
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
    A.parents = parents;
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
    // (one query each: exactly as many problems)
    if (!a->q_start) A.prob_cap = a->n_seqs << (lh - std::min(lh, log_rows));
    const bool f32 = a->io_f32, in = A.prob_cap <= (log_rows == 4 ? kFewProbs16 : kFewProbs);
    // tiles that a problem can have: of rows that the table can name, or of the window, the queries'
    // own span (a tree's: twice the average one's) and the first rows, with their ends inside tiles
    const long long held = (long long)a->table_stride << shift;
    const long long own = kTree ? std::min(kMaxNodes, 2 * (a->n_q / a->n_seqs + 1)) : (1 << log_rows) >> std::min(lh, log_rows);
    const long long span = std::min<long long>(held, (long long)a->window + own);
    const long long most = a->window > 0 ? span / kTile + 2 + (std::min<long long>(a->n_first, held) + kTile - 1) / kTile : held / kTile + 1;
    // A tree in a short window is not cut: its problems have a tile more for 32 nodes before theirs, of which the
    // host knows the average alone, and then need no merge (48 trees of up to 13 nodes: 37 us with it, 30 without).
    A.uncut = kTree && a->window > 0 && most <= 16;
    if (!in) hipLaunchKernelGGL(plan_kernel<kTree>, dim3(1), dim3(1024), 0, st, A);
    // Waves with roles for long problems of bf16 (us a call, with roles and without: problems of 34 tiles 1083, 1122,
    // of 1025 to 1152 22700, 24800, 16 sequences of up to 32768 rows 69.5, 72; problems of 6 tiles 176, 166; one
    // token over 4000 rows, in parts of 4 tiles, 30.5, 29.1)
    auto *main = log_rows == 4 ? f32 ? in ? few_rows_kernel<kTree, true, true> : few_rows_kernel<kTree, true, false>
                                     : in ? few_rows_kernel<kTree, false, true> : few_rows_kernel<kTree, false, false>
                 : f32         ? in ? window_kernel<kTree, true, true> : window_kernel<kTree, true, false>
                 : most > 16   ? in ? roles_kernel<kTree, true> : roles_kernel<kTree, false>
                               : in ? window_kernel<kTree, false, true> : window_kernel<kTree, false, false>;
    hipLaunchKernelGGL(main, dim3(A.n_wg), dim3(log_rows < 6 || f32 ? 256 : 512), 0, st, A);
    if (most > kWhole && !A.uncut) {   // (else nothing is cut)
        const int n = in ? A.prob_cap : A.n_wg - 1;
        // parts that a problem can have: its share of the workgroups, or as many as `per` leaves. Four rows a
        // workgroup from 17 problems on; a row's parts are shared by four waves, by eight from
        // 65 parts on (128 parts: 16.0 us with four, 12.0 with eight; 16 parts: 10.1 and 12.5)
        const int parts = std::min(A.n_wg / std::max(n, 1), 4 * (int)std::sqrt((double)most));
        const bool shared = n <= 16, eight = shared && parts > 64;
        auto *merge = eight    ? f32 ? window_merge_kernel<true, true, 8, 1> : window_merge_kernel<false, true, 8, 1>
                      : shared ? f32 ? window_merge_kernel<true, true, 4, 1> : window_merge_kernel<false, true, 4, 1>
                      : f32    ? in ? window_merge_kernel<true, true, 4, 4> : window_merge_kernel<true, false, 4, 4>
                               : in ? window_merge_kernel<false, true, 4, 4> : window_merge_kernel<false, false, 4, 4>;
        hipLaunchKernelGGL(merge, dim3(n << (shared ? log_rows : log_rows - 2)), dim3(eight ? 512 : 256), 0, st, A);
    }
    return ds4hip_set_last_error(hip_status(hipGetLastError()));
}

extern "C" int ds4hip_flash_attn_window_fp8(const ds4hip_window_attn *a, void *workspace, size_t workspace_bytes,
                                            void *stream) {
    return attend<false>(a, nullptr, workspace, workspace_bytes, stream);
}

extern "C" int ds4hip_flash_attn_tree_fp8(const ds4hip_window_attn *a, const int32_t *parents, void *workspace,
                                          size_t workspace_bytes, void *stream) {
    return attend<true>(a, parents, workspace, workspace_bytes, stream);
}
