// pages.hip — the pages of a paged FP8 KV cache: extended, forked, freed and
// compacted on the device, so that no call waits for the host.
//
// The state is the reference count of each page, the sequences' tables and
// their row counts. One workgroup plans a call: it checks every job before it
// changes anything, finds the lowest free pages (a page is free where its count
// is 0) with ballots over the counts, and so gives the same pages for the same pool
// every time. What moves rows is a second launch over all the chip that reads the
// plan's list: 584 bytes a row and layer, read and written once.
//
// What bounds them. A plan is a chain of loads that wait for each other (jobs, rows, table
// entries, counts) and of barriers: 4.0 us to extend 6 sequences, 8.2 to fork 6, 3.4 to free
// them, 7.4 to compact a pool of 352 pages, 4.8 to accept 2 trees of up to 9 nodes, 8.1 for 64 of
// up to 48. The moves run at memory speed: deep copies of four sequences of 7001 rows in 43 layers
// (647 MB read and written) 140 us, 4.6 TB/s of the 5.1 that a large copy reaches.

#include "ds4hip_common.h"
#include "node_range.h"
#include "step_bodies.h"
#include "../../include/ds4hip_pages.h"

#include <algorithm>
#include <type_traits>

using namespace ds4hip;

namespace {

constexpr int kENOSPC = -28;
constexpr int kJobs = DS4HIP_PAGES_MAX_JOBS;
constexpr int kThreads = 1024;
constexpr int kWaves = kThreads / 64;
constexpr int kScan = 8;   // counts per thread and step of a search
constexpr int kDim = 512, kRotD = 64, kCodes = kDim - kRotD;

// The workspace: what the plan leaves to the copy.
struct Moves {
    int *n;        // pages to copy
    int *n_live;   // held pages (compact)
    int *src, *dst, *count;   // [n_pages] pages, and the rows of each
    int *now;      // [n_pages] where a page went (compact)
};

size_t moves_bytes(int n_pages) { return sizeof(int) * (64 + 4 * (size_t)n_pages); }

Moves moves_at(void *ws, int n_pages) {
    int *p = static_cast<int *>(ws);
    return {p, p + 1, p + 64, p + 64 + (size_t)n_pages, p + 64 + 2 * (size_t)n_pages, p + 64 + 3 * (size_t)n_pages};
}

struct Plan {
    int base[kJobs + 1];   // sums over the jobs before each
    int more[kJobs + 1];
    int at[kJobs];         // their sequences, pages held before, or the like
    int sums[kScan * kWaves];
    uint32_t seen[DS4HIP_PAGES_MAX_SEQS / 32];
    int fail;
};

// Exclusive sums of v over the jobs (one per thread) in out[0 .. n_jobs], saturating
// far above any pool's size.
__device__ inline void scan_jobs(Plan &S, long long v, int *out, int n_jobs) {
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    constexpr long long kMost = 1 << 30;
    long long x = v < kMost ? v : kMost;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const long long y = __shfl_up(x, off);
        if (lane >= off) x += y;
    }
    x = x < kMost ? x : kMost;
    if (n_jobs > 64) {   // (else the first wave has all)
        __syncthreads();
        if (lane == 63) S.sums[w] = (int)x;
        __syncthreads();
        for (int i = 0; i < w; ++i) x += S.sums[i];
        x = x < kMost ? x : kMost;
    }
    if (tid < n_jobs) out[tid + 1] = (int)x;
    if (tid == 0) out[0] = 0;
    __syncthreads();
}

// The job that item i of the sums `base` belongs to.
__device__ inline int job_of(const int *base, int n_jobs, int i) {
    int lo = 0, hi = n_jobs;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (base[mid] <= i) lo = mid; else hi = mid;
    }
    return lo;
}

// Marks sequence s; false where another job of this call named it.
__device__ inline bool first_named(Plan &S, int s) { return !(atomicOr(&S.seen[s >> 5], 1u << (s & 31)) >> (s & 31) & 1); }

__device__ inline void start(Plan &S, int n_seqs) {
    for (int i = threadIdx.x; i < (n_seqs + 31) / 32; i += kThreads) S.seen[i] = 0;
    if (threadIdx.x == 0) S.fail = 0;
    __syncthreads();
}

// All threads; true where a job failed (-22 before -28, whatever their order).
__device__ inline bool failed(Plan &S, const ds4hip_kv_pages &P) {
    __syncthreads();
    const int f = S.fail;
    __syncthreads();   // all have read it before a job of the next check fails: all take the same way
    if (f && threadIdx.x == 0) *P.status = f & 1 ? kEINVAL : kENOSPC;
    return f != 0;
}

__device__ inline void fail(Plan &S, int code) { atomicOr(&S.fail, code == kEINVAL ? 1 : 2); }

// The thread's counts of a step of the search below, from page p0 on. A kernel loads the
// first ones before anything else: they arrive while it checks its jobs.
struct Counts {
    int c[kScan];
};
__device__ inline Counts counts_from(const ds4hip_kv_pages &P, int p0) {
    Counts C;
#pragma unroll
    for (int u = 0; u < kScan; ++u) {
        const int p = p0 + u * kThreads + (int)threadIdx.x;
        C.c[u] = p < P.n_pages ? P.refs[p] : 1;
    }
    return C;
}

// use(k, page) for the `want` lowest free pages, k = 0, 1, ... in order; false where
// there are fewer. 8192 counts a step, from the front, until there are enough.
template <typename Use>
__device__ inline bool lowest_free(Plan &S, const ds4hip_kv_pages &P, Counts C, int want, Use use) {
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    int found = 0;
    for (int p0 = 0; p0 < P.n_pages && found < want; p0 += kScan * kThreads) {
        if (p0) C = counts_from(P, p0);
        const int (&c)[kScan] = C.c;
        uint64_t b[kScan];
        __syncthreads();
#pragma unroll
        for (int u = 0; u < kScan; ++u) {
            b[u] = __ballot(c[u] <= 0);
            if (lane == 0) S.sums[u * kWaves + w] = __popcll(b[u]);
        }
        __syncthreads();
        int before = found;
#pragma unroll
        for (int u = 0; u < kScan; ++u) {
            int mine = before, all = 0;
#pragma unroll
            for (int i = 0; i < kWaves; ++i) {
                const int n = S.sums[u * kWaves + i];
                mine += i < w ? n : 0;
                all += n;
            }
            mine += __popcll(b[u] & ((1ull << lane) - 1));
            if (c[u] <= 0 && mine < want) use(mine, p0 + u * kThreads + tid);
            before += all;
        }
        found = before;
    }
    __syncthreads();
    return found >= want;
}

__device__ inline int pages_of(const ds4hip_kv_pages &P, long long rows) {
    const int shift = __builtin_ctz(P.page_rows);
    return (int)((rows + P.page_rows - 1) >> shift);
}

__device__ inline int32_t *entry(const ds4hip_kv_pages &P, int seq, int i) {
    return P.table + (long long)seq * P.table_stride + i;
}

// A page that the pool has and a sequence holds.
__device__ inline bool held(const ds4hip_kv_pages &P, int page) {
    return page >= 0 && page < P.n_pages && P.refs[page] > 0;
}

__global__ __launch_bounds__(256) void init_kernel(const ds4hip_kv_pages P) {
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x, step = (long long)gridDim.x * 256;
    for (long long k = i; k < (long long)P.n_seqs * P.table_stride; k += step) P.table[k] = -1;
    for (long long k = i; k < P.n_pages; k += step) P.refs[k] = 0;
    for (long long k = i; k < P.n_seqs; k += step) P.rows[k] = 0;
    if (i == 0) *P.status = 0;
}

__global__ __launch_bounds__(kThreads) void extend_kernel(const ds4hip_kv_pages P, const int32_t *seqs, const int32_t *n_new,
                                                          int n_jobs, long long *dst_rows, int n_dst) {
    __shared__ Plan S;
    __shared__ int rows_s[kJobs];
    const int tid = threadIdx.x;
    const Counts counts = counts_from(P, 0);
    start(S, P.n_seqs);
    int seq = -1, n = 0, r0 = 0, need = 0;
    if (tid < n_jobs) {
        seq = seqs[tid];
        n = n_new[tid];
        if (seq < 0 || seq >= P.n_seqs || n < 0 || !first_named(S, seq) || P.rows[seq] < 0) {
            fail(S, kEINVAL);
            n = 0;
        } else {
            r0 = P.rows[seq];
            const int had = pages_of(P, r0);
            const long long rows = (long long)r0 + n;
            if (had > P.table_stride) {
                fail(S, kEINVAL);
            } else {
                if (n > 0 && (r0 & (P.page_rows - 1))) {
                    const int last = *entry(P, seq, had - 1);
                    if (!held(P, last) || P.refs[last] != 1) fail(S, kEINVAL);
                }
                if (rows > 0x7FFFFFFF || pages_of(P, rows) > P.table_stride)
                    fail(S, kENOSPC);
                else
                    need = pages_of(P, rows) - had;
            }
        }
        S.at[tid] = seq;
        rows_s[tid] = r0;
    }
    scan_jobs(S, need, S.base, n_jobs);
    scan_jobs(S, n, S.more, n_jobs);
    const int want = S.base[n_jobs], total = S.more[n_jobs];
    if (tid == 0 && total > n_dst) fail(S, kEINVAL);
    bool refused = failed(S, P);
    if (!refused) {
        // into the tables, where entries past the rows mean nothing yet
        const bool enough = lowest_free(S, P, counts, want, [&](int k, int page) {
            const int j = job_of(S.base, n_jobs, k);
            *entry(P, S.at[j], pages_of(P, rows_s[j]) + k - S.base[j]) = page;
        });
        if (!enough && tid == 0) fail(S, kENOSPC);
        refused = failed(S, P);
    }
    if (!refused) {
        if (tid < n_jobs) P.rows[seq] = r0 + n;
        for (int k = tid; k < want; k += kThreads) {
            const int j = job_of(S.base, n_jobs, k);
            P.refs[*entry(P, S.at[j], pages_of(P, rows_s[j]) + k - S.base[j])] = 1;
        }
    }
    const int shift = __builtin_ctz(P.page_rows);
    for (int i = tid; i < n_dst; i += kThreads) {
        long long to = -1;
        if (!refused && i < total) {
            const int j = job_of(S.more, n_jobs, i), r = rows_s[j] + i - S.more[j];
            to = ((long long)*entry(P, S.at[j], r >> shift) << shift) + (r & (P.page_rows - 1));
        }
        dst_rows[i] = to;
    }
}

__global__ __launch_bounds__(256) void append_kernel(const ds4hip_kv_pages P, long long layer_row, const float *kv, int n_rows,
                                                     const long long *dst_rows) {
    const int row = blockIdx.x * 4 + (threadIdx.x >> 6), t = threadIdx.x & 63;
    if (row >= n_rows) return;
    const long long to = dst_rows[row];
    if (to < 0 || to >= (long long)P.n_pages * P.page_rows) return;
    fp8_row_body<false>(kv, nullptr, P.codes, P.sexp, P.tail, row, kDim, kRotD, layer_row + to, t);
}

__global__ __launch_bounds__(kThreads) void fork_kernel(const ds4hip_kv_pages P, const int32_t *parents, const int32_t *children,
                                                        const int32_t *n_rows, int n_jobs, int deep, const Moves M) {
    __shared__ Plan S;
    __shared__ int child_s[kJobs], rows_s[kJobs];
    const int tid = threadIdx.x, page_rows = P.page_rows;
    const Counts counts = counts_from(P, 0);
    start(S, P.n_seqs);
    int child = -1, r = 0;
    if (tid < n_jobs) {
        const int parent = parents[tid];
        child = children[tid];
        r = n_rows ? n_rows[tid] : -1;
        if (parent < 0 || parent >= P.n_seqs || child < 0 || child >= P.n_seqs || !first_named(S, child) ||
            P.rows[child] != 0 || P.rows[parent] < 0 || r > P.rows[parent] ||
            pages_of(P, P.rows[parent]) > P.table_stride) {
            fail(S, kEINVAL);
            r = 0;
        } else if (r < 0) {
            r = P.rows[parent];
        }
        S.at[tid] = parent;
        child_s[tid] = child;
        rows_s[tid] = r;
    }
    // fresh pages: every one of a deep copy, else a partly filled last one
    scan_jobs(S, deep ? pages_of(P, r) : (r & (page_rows - 1)) != 0, S.base, n_jobs);
    scan_jobs(S, pages_of(P, r), S.more, n_jobs);
    const int want = S.base[n_jobs], total = S.more[n_jobs];
    bool refused = failed(S, P);
    if (!refused) {
        for (int i = tid; i < total; i += kThreads) {
            const int j = job_of(S.more, n_jobs, i), k = i - S.more[j];
            const int page = *entry(P, S.at[j], k);
            if (!held(P, page)) fail(S, kEINVAL);
            *entry(P, child_s[j], k) = page;   // (the child holds nothing yet: this means nothing)
        }
        refused = failed(S, P);
    }
    if (!refused) {
        const bool enough = lowest_free(S, P, counts, want, [&](int k, int page) {
            const int j = job_of(S.base, n_jobs, k);
            const int i = deep ? k - S.base[j] : pages_of(P, rows_s[j]) - 1;
            M.src[k] = *entry(P, S.at[j], i);
            M.dst[k] = page;
            M.count[k] = min(page_rows, rows_s[j] - i * page_rows);
            *entry(P, child_s[j], i) = page;
        });
        if (!enough && tid == 0) fail(S, kENOSPC);
        refused = failed(S, P);
    }
    if (tid == 0) *M.n = refused ? 0 : want;
    if (refused) return;
    for (int k = tid; k < want; k += kThreads) P.refs[M.dst[k]] = 1;
    if (tid < n_jobs) P.rows[child] = r;
    if (!deep)
        for (int i = tid; i < total; i += kThreads) {
            const int j = job_of(S.more, n_jobs, i), k = i - S.more[j];
            if ((k + 1) * (long long)page_rows <= rows_s[j]) atomicAdd(&P.refs[*entry(P, S.at[j], k)], 1);
        }
}

__global__ __launch_bounds__(kThreads) void free_kernel(const ds4hip_kv_pages P, const int32_t *seqs, const int32_t *keep,
                                                        int n_jobs) {
    __shared__ Plan S;
    __shared__ int first_s[kJobs];
    const int tid = threadIdx.x;
    start(S, P.n_seqs);
    int seq = -1, kept = 0, n = 0;
    if (tid < n_jobs) {
        seq = seqs[tid];
        kept = keep ? keep[tid] : 0;
        if (seq < 0 || seq >= P.n_seqs || !first_named(S, seq) || kept < 0 || kept > P.rows[seq] ||
            pages_of(P, P.rows[seq]) > P.table_stride) {
            fail(S, kEINVAL);
        } else {
            n = pages_of(P, P.rows[seq]) - pages_of(P, kept);
            // a page cut short has room: no other sequence may hold it
            if (kept < P.rows[seq] && (kept & (P.page_rows - 1))) {
                const int last = *entry(P, seq, pages_of(P, kept) - 1);
                if (!held(P, last) || P.refs[last] != 1) fail(S, kEINVAL);
            }
        }
        S.at[tid] = seq;
        first_s[tid] = pages_of(P, kept);
    }
    scan_jobs(S, n, S.base, n_jobs);
    if (failed(S, P)) return;
    const int total = S.base[n_jobs];
    for (int i = tid; i < total; i += kThreads) {
        const int j = job_of(S.base, n_jobs, i);
        if (!held(P, *entry(P, S.at[j], first_s[j] + i - S.base[j]))) fail(S, kEINVAL);
    }
    if (failed(S, P)) return;
    for (int i = tid; i < total; i += kThreads) {
        const int j = job_of(S.base, n_jobs, i);
        atomicSub(&P.refs[*entry(P, S.at[j], first_s[j] + i - S.base[j])], 1);
    }
    if (tid < n_jobs) P.rows[seq] = kept;
}

__global__ __launch_bounds__(kThreads) void compact_kernel(const ds4hip_kv_pages P, const Moves M, int32_t *n_live) {
    __shared__ int sums[kScan * kWaves];
    __shared__ int live_s;
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    if (tid == 0) live_s = 0;
    __syncthreads();
    int n = 0;
    for (int p = tid; p < P.n_pages; p += kThreads) n += P.refs[p] > 0;
    if (n) atomicAdd(&live_s, n);
    __syncthreads();
    const int live = live_s;
    int n_src = 0, n_dst = 0;
    for (int p0 = 0; p0 < P.n_pages; p0 += kScan * kThreads) {
        uint64_t from[kScan], to[kScan];
        __syncthreads();
#pragma unroll
        for (int u = 0; u < kScan; ++u) {
            const int p = p0 + u * kThreads + tid;
            const bool in = p < P.n_pages, holds = in && P.refs[p] > 0;
            from[u] = __ballot(holds && p >= live);
            to[u] = __ballot(in && !holds && p < live);
            // both counts (at most 8192 a step) in one word
            if (lane == 0) sums[u * kWaves + w] = __popcll(from[u]) << 16 | __popcll(to[u]);
            if (in && p >= live) M.now[p] = -1;
        }
        __syncthreads();
#pragma unroll
        for (int u = 0; u < kScan; ++u) {
            int mine = 0, all = 0;
#pragma unroll
            for (int i = 0; i < kWaves; ++i) {
                const int c = sums[u * kWaves + i];
                mine += i < w ? c : 0;
                all += c;
            }
            const uint64_t below = (1ull << lane) - 1;
            const int p = p0 + u * kThreads + tid;
            if (from[u] >> lane & 1) M.src[n_src + (mine >> 16) + __popcll(from[u] & below)] = p;
            if (to[u] >> lane & 1) M.dst[n_dst + (mine & 0xFFFF) + __popcll(to[u] & below)] = p;
            n_src += all >> 16;
            n_dst += all & 0xFFFF;
        }
    }
    __syncthreads();
    for (int k = tid; k < n_src; k += kThreads) {
        const int s = M.src[k], d = M.dst[k];
        M.count[k] = P.page_rows;
        M.now[s] = d;
        P.refs[d] = P.refs[s];
        P.refs[s] = 0;
    }
    if (tid == 0) {
        *M.n = n_src;
        *M.n_live = live;
        *n_live = live;
    }
}

// The list's pages, all layers: a workgroup takes 64 rows of one page and layer,
// every load before the first store. kMoved: the tables name the new places too.
template <bool kMoved>
__global__ __launch_bounds__(256) void move_kernel(const ds4hip_kv_pages P, const Moves M) {
    const int tid = threadIdx.x;
    const int n = *M.n;
    if (kMoved) {
        const int live = *M.n_live;
        const long long entries = (long long)P.n_seqs * P.table_stride;
        for (long long k = (long long)blockIdx.x * 256 + tid; n > 0 && k < entries; k += (long long)gridDim.x * 256) {
            const int page = P.table[k];
            if (page < live || page >= P.n_pages) continue;
            const int seq = (int)(k / P.table_stride);
            if (k - (long long)seq * P.table_stride < pages_of(P, P.rows[seq]) && M.now[page] >= 0) P.table[k] = M.now[page];
        }
    }
    const int slices = (P.page_rows + 63) / 64;
    const long long units = (long long)n * P.n_layers * slices;
    for (long long u = blockIdx.x; u < units; u += gridDim.x) {
        const int k = (int)(u / (P.n_layers * slices)), rest = (int)(u - (long long)k * P.n_layers * slices);
        const int layer = rest / slices, row0 = 64 * (rest - layer * slices), rows = min(64, M.count[k] - row0);
        if (rows <= 0) continue;
        const long long from = layer * P.layer_rows + (long long)M.src[k] * P.page_rows + row0;
        const long long to = layer * P.layer_rows + (long long)M.dst[k] * P.page_rows + row0;
        const uint4_t *c0 = reinterpret_cast<const uint4_t *>(P.codes + from * kCodes);
        const uint4_t *t0 = reinterpret_cast<const uint4_t *>(P.tail + from * kRotD);
        uint4_t *c1 = reinterpret_cast<uint4_t *>(P.codes + to * kCodes);
        uint4_t *t1 = reinterpret_cast<uint4_t *>(P.tail + to * kRotD);
        uint4_t c[7], t[2];
        uint2_t e;
#pragma unroll
        for (int i = 0; i < 7; ++i)
            if (tid + 256 * i < 28 * rows) c[i] = c0[tid + 256 * i];
#pragma unroll
        for (int i = 0; i < 2; ++i)
            if (tid + 256 * i < 8 * rows) t[i] = t0[tid + 256 * i];
        if (tid < rows) e = *reinterpret_cast<const uint2_t *>(P.sexp + (from + tid) * 8);
#pragma unroll
        for (int i = 0; i < 7; ++i)
            if (tid + 256 * i < 28 * rows) c1[tid + 256 * i] = c[i];
#pragma unroll
        for (int i = 0; i < 2; ++i)
            if (tid + 256 * i < 8 * rows) t1[tid + 256 * i] = t[i];
        if (tid < rows) *reinterpret_cast<uint2_t *>(P.sexp + (to + tid) * 8) = e;
    }
}

// ---- drafted trees ---------------------------------------------------------------

constexpr int kNodes = DS4HIP_TREE_MAX_NODES;

// What walks read and write.
struct Walk {
    const int32_t *parents, *tokens, *targets;
    int32_t *path, *n_path, *next;
};

// One wave: job j's path, from node 0 to the first child whose token is its parent's target, and so on; returns its
// length. The tree's nodes lie in LDS at parent, token and target; a step is a look at 64 of them at a time behind
// the last one (children follow their parents).
__device__ inline int walk(const Walk &W, int j, int a, int n, const int *parent, const int *token, const int *target) {
    const int lane = threadIdx.x & 63;
    int at = 0, length = 0, says;
    while (true) {
        if (lane == 0) W.path[a + length] = at;
        ++length;
        says = target[at];
        int child = -1;
        for (int c0 = at + 1; says >= 0 && c0 < n; c0 += 64) {
            const int c = min(c0 + lane, n - 1);
            const uint64_t fits = __ballot(c0 + lane < n && parent[c] == at && token[c] == says);
            if (fits) {
                child = c0 + __builtin_ctzll(fits);
                break;
            }
        }
        if (child < 0) break;
        at = child;
    }
    for (int i = length + lane; i < n; i += 64) W.path[a + i] = -1;
    if (lane == 0) {
        W.n_path[j] = length;
        W.next[j] = says;
    }
    return length;
}

// -1 for the nodes that no job names, before the first job's and behind the last one's.
__device__ inline void clear_path(const Walk &W, const int32_t *q_start, int n_jobs, int n_nodes, int tid, int threads) {
    for (int i = tid; i < start_in(q_start[0], n_nodes); i += threads) W.path[i] = -1;
    for (int i = start_in(q_start[n_jobs], n_nodes) + tid; i < n_nodes; i += threads) W.path[i] = -1;
}

// A call without jobs: its nodes are no job's.
__global__ __launch_bounds__(256) void no_path_kernel(int32_t *path, int n_nodes) {
    const int i = blockIdx.x * 256 + threadIdx.x;
    if (i < n_nodes) path[i] = -1;
}

// A workgroup a job, of one wave, for calls of many nodes (the planning workgroup walks the others itself).
__global__ __launch_bounds__(64) void walk_kernel(const int32_t *q_start, int n_jobs, int n_nodes, const Walk W) {
    __shared__ int parent_s[kNodes], token_s[kNodes], target_s[kNodes];
    const int j = blockIdx.x, lane = threadIdx.x;
    const NodeRange own = nodes_between(q_start[j], q_start[j + 1], n_nodes, kNodes);
    const int a = own.first, n = own.n;
    if (j == 0) clear_path(W, q_start, n_jobs, n_nodes, lane, 64);
    if (n == 0) {   // (the plan refuses starts that do not say so)
        if (lane == 0) W.n_path[j] = 0, W.next[j] = -1;
        return;
    }
    for (int i = lane; i < n; i += 64) {
        parent_s[i] = W.parents[a + i];
        token_s[i] = W.tokens[a + i];
        target_s[i] = W.targets[a + i];
    }
    __syncthreads();
    walk(W, j, a, n, parent_s, token_s, target_s);
}

// Nodes of a call whose planning workgroup finds the paths itself: a launch less, all nodes loaded at once, and
// all jobs' paths followed at once, a thread each, through the one child of each node that agrees. (64 jobs of 1195
// nodes: the plan with it 9 us, with a wave a tree there 16, with walk_kernel before it 4.7 + 7.1.)
constexpr int kWalkNodes = 4096;

struct Trees {
    int parent[kWalkNodes], token[kWalkNodes], target[kWalkNodes], next[kWalkNodes], start[kJobs + 1];
};

// All threads; length[j] receives the nodes of job j's path.
__device__ inline void walk_all(const Walk &W, Trees &T, const int32_t *q_start, int n_jobs, int n_nodes, int *length) {
    const int tid = threadIdx.x;
    for (int i = tid; i < n_nodes; i += kThreads) {
        T.parent[i] = W.parents[i];
        T.token[i] = W.tokens[i];
        T.target[i] = W.targets[i];
        T.next[i] = kWalkNodes;
    }
    for (int i = tid; i <= n_jobs; i += kThreads) T.start[i] = start_in(q_start[i], n_nodes);
    __syncthreads();
    // (the plan looks at the starts as they are, and refuses those that were moved here)
    auto nodes_of = [&](int j) { return nodes_between(T.start[j], T.start[j + 1], n_nodes, kNodes).n; };
    for (int i = tid; i < n_nodes; i += kThreads) {
        const int j = job_of(T.start, n_jobs, i), a = T.start[j], v = i - a, p = T.parent[i];
        if (v > 0 && v < nodes_of(j) && p >= 0 && p < v && T.target[a + p] >= 0 && T.token[i] == T.target[a + p]) atomicMin(&T.next[a + p], v);
    }
    __syncthreads();
    if (tid < n_jobs) {
        const int a = T.start[tid], n = nodes_of(tid);
        int k = 0, at = 0, says = -1;
        while (at < n) {   // (kWalkNodes: no child agrees)
            W.path[a + k++] = at;
            says = T.target[a + at];
            const int to = T.next[a + at];
            at = to > at ? to : n;   // (a child comes later; where q_start goes back, trees lie over each other)
        }
        length[tid] = k;
        W.n_path[tid] = k;
        W.next[tid] = says;
    }
    __syncthreads();
    for (int i = tid; i < n_nodes; i += kThreads) {
        const int j = job_of(T.start, n_jobs, i), v = i - T.start[j];
        if (v < 0 || v >= length[j]) W.path[i] = -1;   // (before the first job's nodes, behind a path, or behind the last job's)
    }
}

// Checks the jobs' paths, cuts their sequences and releases the pages behind them. kAccept: a refused call
// takes back what the walks wrote; kWalk: they are walked here.
template <bool kAccept, bool kWalk>
__global__ __launch_bounds__(kThreads) void keep_kernel(const ds4hip_kv_pages P, const int32_t *seqs, const int32_t *q_start,
                                                        int n_jobs, int n_nodes, const Walk W, const Moves M) {
    __shared__ Plan S;
    __shared__ int kept_s[kJobs], nodes_s[kJobs];
    __shared__ std::conditional_t<kWalk, Trees, int> T;
    const int tid = threadIdx.x, shift = __builtin_ctz(P.page_rows);
    start(S, P.n_seqs);
    if constexpr (kWalk) walk_all(W, T, q_start, n_jobs, n_nodes, kept_s);
    int seq = -1, base = -1, n = 0, kept = 0, held_pages = 0;
    if (tid < n_jobs) {
        const int a = q_start[tid], b = q_start[tid + 1];
        seq = seqs[tid];
        kept = kWalk ? kept_s[tid] : W.n_path[tid];
        const long long count = (long long)b - a;
        if (a < 0 || count < 0 || b > n_nodes || seq < 0 || seq >= P.n_seqs || !first_named(S, seq) || kept < 0 || kept > count ||
            count > P.rows[seq] || (kAccept && count > kNodes) || pages_of(P, P.rows[seq]) > P.table_stride) {
            fail(S, kEINVAL);
        } else {
            n = (int)count;
            base = P.rows[seq] - n;
            if (n > 0) held_pages = pages_of(P, P.rows[seq]) - (base >> shift);
        }
        S.at[tid] = seq;
        nodes_s[tid] = a;
        kept_s[tid] = kept;
    }
    scan_jobs(S, held_pages, S.base, n_jobs);   // pages with drafts in them
    scan_jobs(S, n > 0 ? kept : 0, S.more, n_jobs);
    if (failed(S, P)) {
        if (kAccept) goto refuse;
        if (tid == 0) *M.n = 0;
        return;
    }
    {
        const int pages = S.base[n_jobs], rows = S.more[n_jobs];
        // this sequence's alone: its rows move, or are cut
        for (int i = tid; i < pages; i += kThreads) {
            const int j = job_of(S.base, n_jobs, i), s = S.at[j];
            const int page = *entry(P, s, pages_of(P, P.rows[s]) - (S.base[j + 1] - i));
            if (!held(P, page) || P.refs[page] != 1) fail(S, kEINVAL);
        }
        if (!kAccept)
            for (int i = tid; i < rows; i += kThreads) {   // nodes in order
                const int j = job_of(S.more, n_jobs, i), k = i - S.more[j];
                const int v = W.path[nodes_s[j] + k], before = k ? W.path[nodes_s[j] + k - 1] : -1;
                if (v <= before || v >= q_start[j + 1] - nodes_s[j]) fail(S, kEINVAL);
            }
        if (failed(S, P)) {
            if (kAccept) goto refuse;
            if (tid == 0) *M.n = 0;
            return;
        }
        for (int i = tid; i < pages; i += kThreads) {
            const int j = job_of(S.base, n_jobs, i), s = S.at[j];
            const int had = pages_of(P, P.rows[s]), k = had - (S.base[j + 1] - i);
            // (its rows are still those before the call)
            const int now = P.rows[s] - (q_start[j + 1] - nodes_s[j]) + kept_s[j];
            if (k >= pages_of(P, now)) P.refs[*entry(P, s, k)] = 0;
        }
        __syncthreads();
        if (tid < n_jobs) P.rows[seq] = base + kept;
        if (tid == 0) *M.n = n_jobs;
        return;
    }
refuse:
    if (tid == 0) *M.n = 0;
    for (int i = tid; i < n_nodes; i += kThreads) W.path[i] = -1;
    if (tid < n_jobs) W.n_path[tid] = 0, W.next[tid] = -1;
}

// The paths' rows: row path[i] of the drafts becomes row i, from the first that moves on (those before it, which are
// their own places, lie together). Every load comes before the first store, 64 rows at a time in order (path[i] >= i:
// a row that is read later lies behind those already written). A job's layers go to `split` workgroups, each with as many
// layers at once as make 64 rows: the places are looked up once for all of them, and little is left to wait for.
// (64 jobs of 5 rows in 43 layers, 4.8 MB: 5.6 us, of loads that wait for each other; a workgroup for each job and
// layer took 10.8.)
__global__ __launch_bounds__(256) void keep_rows_kernel(const ds4hip_kv_pages P, const int32_t *seqs, const int32_t *q_start,
                                                        const int32_t *path, const int32_t *n_path, int split, const Moves M) {
    constexpr int kRows = 64;
    __shared__ long long from_s[kRows], to_s[kRows];
    const int tid = threadIdx.x, lane = tid & 63, shift = __builtin_ctz(P.page_rows);
    const int j = blockIdx.x / split, part = blockIdx.x - j * split;
    const int l0 = (int)((long long)P.n_layers * part / split), l1 = (int)((long long)P.n_layers * (part + 1) / split);
    const int kept = n_path[j], seq = seqs[j], a = q_start[j];
    // (the plan has cut the sequence; asked for before it is known whether the call was refused: 0.3 us less)
    const int base = P.rows[min(max(seq, 0), P.n_seqs - 1)] - kept;
    if (*M.n == 0) return;   // refused
    for (int i0 = 0; i0 < kept; i0 += kRows) {
        const int i = i0 + lane, node = i < kept ? path[a + i] : i;
        const uint64_t moved = __ballot(node != i);   // (the same in every wave)
        if (!moved) continue;
        const int first = __builtin_ctzll(moved), rows = min(kRows, kept - i0) - first;
        __syncthreads();   // (the places before are read)
        if (tid >= first && tid < first + rows) {
            const int f = base + node, t = base + i;
            from_s[tid - first] = ((long long)*entry(P, seq, f >> shift) << shift) + (f & (P.page_rows - 1));
            to_s[tid - first] = ((long long)*entry(P, seq, t >> shift) << shift) + (t & (P.page_rows - 1));
        }
        __syncthreads();
        const int per = kRows / rows;
        for (int l = l0; l < l1; l += per) {
            const int all = rows * min(per, l1 - l);   // rows of these layers
            constexpr int kUnits = 36, kEach = kRows * kUnits / 256;   // 16 bytes each: 28 of codes, 8 of the tail
            auto place = [&](const long long *at, int r) {
                const int layer = r / rows;
                return (l + layer) * P.layer_rows + at[r - layer * rows];
            };
            uint4_t v[kEach];
            uint2_t e = {0, 0};
#pragma unroll
            for (int u = 0; u < kEach; ++u) {
                const int x = tid + 256 * u, r = x / kUnits, k = x - r * kUnits;
                if (r < all) {
                    const long long from = place(from_s, r);
                    v[u] = k < 28 ? reinterpret_cast<const uint4_t *>(P.codes + from * kCodes)[k]
                                  : reinterpret_cast<const uint4_t *>(P.tail + from * kRotD)[k - 28];
                }
            }
            if (tid < all) e = *reinterpret_cast<const uint2_t *>(P.sexp + place(from_s, tid) * 8);
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // no other wave's store overtakes a load
            __syncthreads();
#pragma unroll
            for (int u = 0; u < kEach; ++u) {
                const int x = tid + 256 * u, r = x / kUnits, k = x - r * kUnits;
                if (r < all) {
                    const long long to = place(to_s, r);
                    if (k < 28)
                        reinterpret_cast<uint4_t *>(P.codes + to * kCodes)[k] = v[u];
                    else
                        reinterpret_cast<uint4_t *>(P.tail + to * kRotD)[k - 28] = v[u];
                }
            }
            if (tid < all) *reinterpret_cast<uint2_t *>(P.sexp + place(to_s, tid) * 8) = e;
        }
    }
}

// Workgroups of a job's rows: two for each CU in all.
int keep_split(const ds4hip_kv_pages *p, int n_jobs) { return std::max(1, std::min(p->n_layers, 512 / n_jobs)); }

bool aligned(const void *p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

bool pool_ok(const ds4hip_kv_pages *p) {
    return p && p->n_layers > 0 && p->n_pages > 0 && p->n_pages <= (1 << 28) && p->page_rows > 0 &&
           (p->page_rows & (p->page_rows - 1)) == 0 && p->table_stride > 0 && p->n_seqs > 0 &&
           p->n_seqs <= DS4HIP_PAGES_MAX_SEQS && p->layer_rows >= (long long)p->n_pages * p->page_rows && p->codes &&
           p->sexp && p->tail && p->refs && p->table && p->rows && p->status && aligned(p->codes, 16) &&
           aligned(p->tail, 16) && aligned(p->sexp, 8);
}

// Workgroups for the copy of up to n pages: whole rounds of the chip at most.
unsigned move_grid(const ds4hip_kv_pages *p, long long n) {
    const long long units = n * p->n_layers * ((p->page_rows + 63) / 64);
    return (unsigned)std::min<long long>(std::max<long long>(units, 1), 256 * 8);
}

}  // namespace

extern "C" int ds4hip_kv_pages_init(const ds4hip_kv_pages *p, void *stream) {
    if (!pool_ok(p)) return ds4hip_set_last_error(kEINVAL);
    hipLaunchKernelGGL(init_kernel, dim3(256), dim3(256), 0, (hipStream_t)stream, *p);
    return ds4hip_set_last_error(hip_status(hipGetLastError()));
}

extern "C" size_t ds4hip_kv_pages_workspace_bytes(const ds4hip_kv_pages *p) {
    return p && p->n_pages > 0 ? moves_bytes(p->n_pages) : 0;
}

extern "C" int ds4hip_kv_pages_extend(const ds4hip_kv_pages *p, const int32_t *seqs, const int32_t *n_new, int n_jobs,
                                      long long *dst_rows, int n_dst, void *stream) {
    if (!pool_ok(p) || n_jobs < 0 || n_jobs > kJobs || n_dst < 0 || n_dst > (1 << 28) || (n_jobs && (!seqs || !n_new)) ||
        (n_dst && !dst_rows))
        return ds4hip_set_last_error(kEINVAL);
    if (n_jobs == 0 && n_dst == 0) return 0;
    hipLaunchKernelGGL(extend_kernel, dim3(1), dim3(kThreads), 0, (hipStream_t)stream, *p, seqs, n_new, n_jobs, dst_rows,
                       n_dst);
    return ds4hip_set_last_error(hip_status(hipGetLastError()));
}

extern "C" int ds4hip_kv_pages_append(const ds4hip_kv_pages *p, int layer, const float *kv, int n_rows,
                                      const long long *dst_rows, void *stream) {
    if (!pool_ok(p) || layer < 0 || layer >= p->n_layers || n_rows < 0 || (n_rows && (!kv || !dst_rows || !aligned(kv, 16))))
        return ds4hip_set_last_error(kEINVAL);
    if (n_rows == 0) return 0;
    hipLaunchKernelGGL(append_kernel, dim3((unsigned)(n_rows / 4 + (n_rows % 4 != 0))), dim3(256), 0, (hipStream_t)stream, *p,
                       layer * p->layer_rows, kv, n_rows, dst_rows);
    return ds4hip_set_last_error(hip_status(hipGetLastError()));
}

extern "C" int ds4hip_kv_pages_fork(const ds4hip_kv_pages *p, const int32_t *parents, const int32_t *children,
                                    const int32_t *n_rows, int n_jobs, int deep, void *workspace, size_t workspace_bytes,
                                    void *stream) {
    if (!pool_ok(p) || n_jobs < 0 || n_jobs > kJobs || (deep != 0 && deep != 1) ||
        (n_jobs && (!parents || !children || !workspace || !aligned(workspace, 8) || workspace_bytes < moves_bytes(p->n_pages))))
        return ds4hip_set_last_error(kEINVAL);
    if (n_jobs == 0) return 0;
    const Moves M = moves_at(workspace, p->n_pages);
    const hipStream_t st = (hipStream_t)stream;
    hipLaunchKernelGGL(fork_kernel, dim3(1), dim3(kThreads), 0, st, *p, parents, children, n_rows, n_jobs, deep, M);
    const unsigned grid = move_grid(p, deep ? p->n_pages : n_jobs);
    hipLaunchKernelGGL(move_kernel<false>, dim3(grid), dim3(256), 0, st, *p, M);
    return ds4hip_set_last_error(hip_status(hipGetLastError()));
}

extern "C" int ds4hip_kv_pages_free(const ds4hip_kv_pages *p, const int32_t *seqs, const int32_t *keep, int n_jobs,
                                    void *stream) {
    if (!pool_ok(p) || n_jobs < 0 || n_jobs > kJobs || (n_jobs && !seqs)) return ds4hip_set_last_error(kEINVAL);
    if (n_jobs == 0) return 0;
    hipLaunchKernelGGL(free_kernel, dim3(1), dim3(kThreads), 0, (hipStream_t)stream, *p, seqs, keep, n_jobs);
    return ds4hip_set_last_error(hip_status(hipGetLastError()));
}

extern "C" int ds4hip_kv_pages_compact(const ds4hip_kv_pages *p, int32_t *n_live, void *workspace, size_t workspace_bytes,
                                       void *stream) {
    if (!pool_ok(p) || !n_live || !workspace || !aligned(workspace, 8) || workspace_bytes < moves_bytes(p->n_pages))
        return ds4hip_set_last_error(kEINVAL);
    const Moves M = moves_at(workspace, p->n_pages);
    const hipStream_t st = (hipStream_t)stream;
    hipLaunchKernelGGL(compact_kernel, dim3(1), dim3(kThreads), 0, st, *p, M, n_live);
    hipLaunchKernelGGL(move_kernel<true>, dim3(256 * 8), dim3(256), 0, st, *p, M);
    return ds4hip_set_last_error(hip_status(hipGetLastError()));
}

extern "C" int ds4hip_kv_pages_keep(const ds4hip_kv_pages *p, const int32_t *seqs, const int32_t *q_start, int n_jobs,
                                    const int32_t *path, int n_nodes, const int32_t *n_path, void *workspace,
                                    size_t workspace_bytes, void *stream) {
    if (!pool_ok(p) || n_jobs < 0 || n_jobs > kJobs || n_nodes < 0 || n_nodes > (1 << 24) ||
        (n_jobs && (!seqs || !q_start || !n_path || (n_nodes && !path) || !workspace || !aligned(workspace, 8) ||
                    workspace_bytes < moves_bytes(p->n_pages))))
        return ds4hip_set_last_error(kEINVAL);
    if (n_jobs == 0) return 0;
    const Moves M = moves_at(workspace, p->n_pages);
    const hipStream_t st = (hipStream_t)stream;
    const Walk W = {nullptr, nullptr, nullptr, const_cast<int32_t *>(path), const_cast<int32_t *>(n_path), nullptr};   // (only read)
    hipLaunchKernelGGL((keep_kernel<false, false>), dim3(1), dim3(kThreads), 0, st, *p, seqs, q_start, n_jobs, n_nodes, W, M);
    const int split = keep_split(p, n_jobs);
    hipLaunchKernelGGL(keep_rows_kernel, dim3(n_jobs * split), dim3(256), 0, st, *p, seqs, q_start, path, n_path, split, M);
    return ds4hip_set_last_error(hip_status(hipGetLastError()));
}

extern "C" int ds4hip_kv_pages_accept(const ds4hip_kv_pages *p, const int32_t *seqs, const int32_t *q_start, int n_jobs,
                                      const int32_t *parents, const int32_t *tokens, const int32_t *targets, int n_nodes,
                                      int32_t *path, int32_t *n_path, int32_t *next, void *workspace, size_t workspace_bytes,
                                      void *stream) {
    if (!pool_ok(p) || n_jobs < 0 || n_jobs > kJobs || n_nodes < 0 || n_nodes > (1 << 24) || (n_nodes && !path) ||
        (n_jobs && (!seqs || !q_start || !n_path || !next || (n_nodes && (!parents || !tokens || !targets)) ||
                    !workspace || !aligned(workspace, 8) || workspace_bytes < moves_bytes(p->n_pages))))
        return ds4hip_set_last_error(kEINVAL);
    const hipStream_t st = (hipStream_t)stream;
    if (n_jobs == 0) {
        if (n_nodes == 0) return 0;
        hipLaunchKernelGGL(no_path_kernel, dim3((unsigned)(n_nodes + 255) / 256), dim3(256), 0, st, path, n_nodes);
        return ds4hip_set_last_error(hip_status(hipGetLastError()));
    }
    const Moves M = moves_at(workspace, p->n_pages);
    const Walk W = {parents, tokens, targets, path, n_path, next};
    const bool here = n_nodes <= kWalkNodes;
    if (!here) hipLaunchKernelGGL(walk_kernel, dim3(n_jobs), dim3(64), 0, st, q_start, n_jobs, n_nodes, W);
    auto *plan = here ? keep_kernel<true, true> : keep_kernel<true, false>;
    hipLaunchKernelGGL(plan, dim3(1), dim3(kThreads), 0, st, *p, seqs, q_start, n_jobs, n_nodes, W, M);
    const int split = keep_split(p, n_jobs);
    hipLaunchKernelGGL(keep_rows_kernel, dim3(n_jobs * split), dim3(256), 0, st, *p, seqs, q_start, path, n_path, split, M);
    return ds4hip_set_last_error(hip_status(hipGetLastError()));
}
