// Pages of the paged cache as shared, counted objects: fork, extend, free, copy, compact.
//
// refcount[p] is the number of sequences whose table names page p; a page is free when it is 0. New
// pages are the lowest free ones, handed out in the order of the call's list, so the tables are the
// same on every run. Every page lies in each of the pools (K and V of all layers) at p * page_bytes.
//
// What bounds it: the bytes of the pages moved (read and written once, 16 bytes per thread and
// access), and for small calls the launches: planning needs an ordered scan over the counts, which
// one CTA does; table rows, counts and page contents then follow in one launch over all of the GPU.
// Measured on a B200: 15 forks of an 8191-position prompt over 64 pools 16 us (4.4 TB/s with its three
// launches, 6.0 in the last), compaction of 302 MB 114 us (5.3 TB/s, 82 % of the measured copy rate).
#include <cuda_runtime.h>

#include "common.cuh"
#include "launch.cuh"

namespace vsl {

constexpr int KP_MAX_POOLS = 256;
constexpr int KP_THREADS = 256;
constexpr int KP_PLAN_THREADS = 1024;
constexpr int KP_COPY_BYTES = 16384;  // bytes of a page one CTA moves at a time

struct KpPools {
    unsigned char* base[KP_MAX_POOLS];
};
struct KpParams {
    int32_t* table;
    int n_seq, max_pages, page_size;
    int32_t* lens;
    int32_t* ref;
    int n_pages, n_pools;
    size_t page_bytes;
    int* status;
};

__device__ __forceinline__ int kp_held(const KpParams& p, int len) {
    return min((max(len, 0) + p.page_size - 1) / p.page_size, p.max_pages);
}

// Give back the pages of sequence s (one CTA).
__device__ __forceinline__ void kp_release(const KpParams& p, int s) {
    const int held = kp_held(p, p.lens[s]);
    for (int i = threadIdx.x; i < held; i += blockDim.x) {
        const int pg = p.table[(size_t)s * p.max_pages + i];
        if (pg >= 0 && pg < p.n_pages) atomicSub(p.ref + pg, 1);
        else set_status(p.status, VSL_ERR_BOUNDS);
    }
}

// Exclusive scan of v over the CTA's KP_PLAN_THREADS threads; *total gets the sum.
__device__ __forceinline__ int kp_scan(int v, int* total) {
    __shared__ int warp_sum_s[32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int n = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += n;
    }
    __syncthreads();
    if (lane == 31) warp_sum_s[warp] = x;
    __syncthreads();
    if (warp == 0) {
        int y = warp_sum_s[lane];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int n = __shfl_up_sync(0xffffffffu, y, o);
            if (lane >= o) y += n;
        }
        warp_sum_s[lane] = y;
    }
    __syncthreads();
    *total = warp_sum_s[31];
    return x - v + (warp ? warp_sum_s[warp - 1] : 0);
}

// The lowest `want` free pages, ascending, into list; returns how many there are (at most want).
__device__ __forceinline__ int kp_find_free(const KpParams& p, int want, int32_t* list) {
    constexpr int PER = 4;
    int found = 0;
    for (int c0 = 0; c0 < p.n_pages && found < want; c0 += KP_PLAN_THREADS * PER) {
        const int i0 = c0 + threadIdx.x * PER;
        bool free_[PER];
        int n = 0;
#pragma unroll
        for (int i = 0; i < PER; i++) {
            free_[i] = i0 + i < p.n_pages && __ldcg(p.ref + i0 + i) == 0;
            n += free_[i];
        }
        int total;
        int at = found + kp_scan(n, &total);
#pragma unroll
        for (int i = 0; i < PER; i++)
            if (free_[i]) {
                if (at < want) list[at] = i0 + i;
                at++;
            }
        found += total;
    }
    __syncthreads();
    return min(found, want);
}

// Copy bytes [lo, hi) of page src to page dst of one pool (one CTA; multiples of 16).
__device__ __forceinline__ void kp_copy(unsigned char* pool, size_t page_bytes, int src, int dst, size_t lo, size_t hi) {
    const uint4* a = reinterpret_cast<const uint4*>(pool + (size_t)src * page_bytes + lo);
    uint4* d = reinterpret_cast<uint4*>(pool + (size_t)dst * page_bytes + lo);
    const int n = (int)((hi - lo) / 16);
    int i = threadIdx.x;
    for (; i + 3 * KP_THREADS < n; i += 4 * KP_THREADS) {
        const uint4 v0 = __ldcs(a + i), v1 = __ldcs(a + i + KP_THREADS), v2 = __ldcs(a + i + 2 * KP_THREADS),
                    v3 = __ldcs(a + i + 3 * KP_THREADS);
        d[i] = v0;
        d[i + KP_THREADS] = v1;
        d[i + 2 * KP_THREADS] = v2;
        d[i + 3 * KP_THREADS] = v3;
    }
    for (; i < n; i += KP_THREADS) d[i] = __ldcs(a + i);
}

// ---- fork ----
// ok[k]: fork k names two sequences of the table, its source is no longer than its table row, its
// target is no fork's source and no earlier fork's target. A target gives its pages back.
__global__ void __launch_bounds__(KP_THREADS) vsl_kv_fork_release_kernel(KpParams p, const int32_t* src,
                                                                          const int32_t* dst, int n, int32_t* ok) {
    pdl_wait();
    pdl_launch_dependents();
    const int k = blockIdx.x, s = src[k], d = dst[k];
    bool bad = s < 0 || s >= p.n_seq || d < 0 || d >= p.n_seq;
    bad = bad || p.lens[s] > p.max_pages * p.page_size;
    for (int j = threadIdx.x; j < n; j += KP_THREADS) bad = bad || src[j] == d || (j < k && dst[j] == d);
    bad = __syncthreads_or(bad);
    if (threadIdx.x == 0) {
        ok[k] = !bad;
        if (bad) set_status(p.status, VSL_ERR_BOUNDS);
    }
    if (!bad) kp_release(p, d);
}

// fresh[k]: the page that takes the content of fork k's unfinished last page (-1: it has none, -2:
// no page was left). tails: scratch [n], the forks that need one, in order.
__global__ void __launch_bounds__(KP_PLAN_THREADS) vsl_kv_fork_plan_kernel(KpParams p, const int32_t* src, int n,
                                                                           const int32_t* ok, int32_t* fresh,
                                                                           int32_t* tails, int32_t* list) {
    pdl_wait();
    pdl_launch_dependents();
    int n_tails = 0;
    for (int k0 = 0; k0 < n; k0 += KP_PLAN_THREADS) {
        const int k = k0 + threadIdx.x;
        const bool need = k < n && ok[k] && max(p.lens[src[k]], 0) % p.page_size != 0;
        int total;
        const int at = n_tails + kp_scan(need, &total);
        if (need) tails[at] = k;
        if (k < n) fresh[k] = need ? -2 : -1;
        n_tails += total;
    }
    __syncthreads();
    const int found = kp_find_free(p, n_tails, list);
    for (int i = threadIdx.x; i < found; i += KP_PLAN_THREADS) fresh[tails[i]] = list[i];
    if (found < n_tails && threadIdx.x == 0) set_status(p.status, VSL_ERR_OOM);
}

// CTA (piece, pool, k): its piece of the unfinished page's copy in that pool; CTA (0, 0, k) writes
// the target's table row and the counts as well.
__global__ void __launch_bounds__(KP_THREADS) vsl_kv_fork_kernel(KpParams p, const __grid_constant__ KpPools pools,
                                                                 const int32_t* src, const int32_t* dst,
                                                                 const int32_t* ok, const int32_t* fresh) {
    pdl_wait();
    pdl_launch_dependents();
    const int k = blockIdx.z;
    if (!ok[k]) return;
    const int s = src[k], d = dst[k], f = fresh[k], len = max(p.lens[s], 0);
    const int full = f == -2 ? 0 : min(len / p.page_size, p.max_pages);  // whole pages to share
    const int tail = f >= 0 && full < p.max_pages ? p.table[(size_t)s * p.max_pages + full] : -1;
    const bool has_tail = tail >= 0 && tail < p.n_pages;  // else there is nothing to copy: f stays free, the entry is the source's
    if (blockIdx.x == 0 && blockIdx.y == 0) {
        for (int i = threadIdx.x; i < p.max_pages; i += KP_THREADS) {
            int pg = i < full ? p.table[(size_t)s * p.max_pages + i] : i == full && f >= 0 ? (has_tail ? f : tail) : -1;
            if (i < full) {
                if (pg >= 0 && pg < p.n_pages) atomicAdd(p.ref + pg, 1);
                else set_status(p.status, VSL_ERR_BOUNDS);
            }
            p.table[(size_t)d * p.max_pages + i] = pg;
        }
        if (threadIdx.x == 0) {
            if (has_tail) p.ref[f] = 1;
            p.lens[d] = f == -2 ? 0 : len;
        }
    }
    if (f < 0) return;
    if (!has_tail) {
        if (threadIdx.x == 0) set_status(p.status, VSL_ERR_BOUNDS);
        return;
    }
    const size_t lo = (size_t)blockIdx.x * KP_COPY_BYTES;
    kp_copy(pools.base[blockIdx.y], p.page_bytes, tail, f, lo, min(lo + KP_COPY_BYTES, p.page_bytes));
}

// ---- free ----
__global__ void __launch_bounds__(KP_THREADS) vsl_kv_free_kernel(KpParams p, const int32_t* seqs, int n) {
    pdl_wait();
    pdl_launch_dependents();
    const int k = blockIdx.x, s = seqs[k];
    bool bad = s < 0 || s >= p.n_seq;
    for (int j = threadIdx.x; j < k; j += KP_THREADS) bad = bad || seqs[j] == s;
    bad = __syncthreads_or(bad);
    if (bad) {
        if (threadIdx.x == 0) set_status(p.status, VSL_ERR_BOUNDS);
        return;
    }
    kp_release(p, s);
    __syncthreads();
    for (int i = threadIdx.x; i < p.max_pages; i += KP_THREADS) p.table[(size_t)s * p.max_pages + i] = -1;
    if (threadIdx.x == 0) p.lens[s] = 0;
}

// ---- extend ----
// Sequence seqs[k] grows by add[k] positions: the pages they need, then its length. One CTA; a
// sequence that cannot have all of its pages gets none and keeps its length, as do those after it.
__global__ void __launch_bounds__(KP_PLAN_THREADS) vsl_kv_extend_kernel(KpParams p, const int32_t* seqs,
                                                                        const int32_t* add, int n, int32_t* start,
                                                                        int32_t* list) {
    pdl_wait();
    pdl_launch_dependents();
    int want = 0;
    for (int k0 = 0; k0 < n; k0 += KP_PLAN_THREADS) {  // start[k]: its first page in the list; -1: refused
        const int k = k0 + threadIdx.x;
        int need = 0;
        bool bad = false;
        if (k < n) {
            const int s = seqs[k], a = add[k];
            bad = s < 0 || s >= p.n_seq || a < 0;
            for (int j = 0; j < k && !bad; j++) bad = seqs[j] == s;
            if (!bad) {
                const long long end = (long long)max(p.lens[s], 0) + a;
                bad = end > (long long)p.max_pages * p.page_size;
                if (!bad) need = (int)((end + p.page_size - 1) / p.page_size) - kp_held(p, p.lens[s]);
            }
            if (bad) set_status(p.status, VSL_ERR_BOUNDS);
        }
        // more pages than the pool has (2^20 at most) cannot be found: the sums stay inside an int
        int total;
        const int at = kp_scan(min(need, p.n_pages + 1), &total);
        if (k < n) start[k] = bad ? -1 : min(want + at, p.n_pages + 1);
        want = min(want + total, p.n_pages + 1);
    }
    __syncthreads();
    const int found = kp_find_free(p, min(want, p.n_pages), list);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int k = warp; k < n; k += KP_PLAN_THREADS / 32) {
        const int at = start[k];
        if (at < 0) continue;
        const int s = seqs[k], len = max(p.lens[s], 0), held = kp_held(p, len);
        const int need = (len + add[k] + p.page_size - 1) / p.page_size - held;
        if ((long long)at + need > found) {
            if (lane == 0) set_status(p.status, VSL_ERR_OOM);
            continue;
        }
        for (int i = lane; i < need; i += 32) {
            p.table[(size_t)s * p.max_pages + held + i] = list[at + i];
            p.ref[list[at + i]] = 1;
        }
        __syncwarp();
        if (lane == 0) p.lens[s] = len + add[k];
    }
}

// ---- copy ----
__global__ void __launch_bounds__(KP_THREADS) vsl_kv_copy_kernel(KpParams p, const __grid_constant__ KpPools pools,
                                                                 const int32_t* src, const int32_t* dst) {
    pdl_wait();
    pdl_launch_dependents();
    const int s = src[blockIdx.z], d = dst[blockIdx.z];
    if (s < 0 || s >= p.n_pages || d < 0 || d >= p.n_pages) {
        if (threadIdx.x == 0) set_status(p.status, VSL_ERR_BOUNDS);
        return;
    }
    const size_t lo = (size_t)blockIdx.x * KP_COPY_BYTES;
    kp_copy(pools.base[blockIdx.y], p.page_bytes, s, d, lo, min(lo + KP_COPY_BYTES, p.page_bytes));
}

// ---- compact ----
// n_live pages are in use: those at n_live and above ("movers") go, in order, to the free pages
// below it ("holes"). to[p]: the new place of a page p >= n_live, -1 for one that is not in use.
__global__ void __launch_bounds__(KP_PLAN_THREADS) vsl_kv_compact_plan_kernel(KpParams p, int32_t* counts,
                                                                              int32_t* holes, int32_t* movers,
                                                                              int32_t* to) {
    pdl_wait();
    pdl_launch_dependents();
    int mine = 0;
    for (int i = threadIdx.x; i < p.n_pages; i += KP_PLAN_THREADS) mine += p.ref[i] > 0;
    int n_live;
    kp_scan(mine, &n_live);
    int n_holes = 0, n_movers = 0;
    for (int c0 = 0; c0 < p.n_pages; c0 += KP_PLAN_THREADS) {
        const int i = c0 + threadIdx.x;
        const bool used = i < p.n_pages && p.ref[i] > 0;
        const bool hole = i < n_live && !used, mover = i >= n_live && used;
        int total;
        // a chunk's holes and movers in one scan: both counts fit 16 bits (1024 threads)
        const int at = kp_scan((int)hole + ((int)mover << 16), &total);
        if (hole) holes[n_holes + (at & 0xffff)] = i;
        if (mover) movers[n_movers + (at >> 16)] = i;
        if (i >= n_live && i < p.n_pages && !used) to[i] = -1;
        n_holes += total & 0xffff;
        n_movers += total >> 16;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < n_movers; i += KP_PLAN_THREADS) to[movers[i]] = holes[i];
    if (threadIdx.x == 0) {
        counts[0] = n_live;
        counts[1] = n_movers;
    }
}

__global__ void __launch_bounds__(KP_THREADS) vsl_kv_compact_kernel(KpParams p, const __grid_constant__ KpPools pools,
                                                                    int32_t* table_out, int32_t* ref_out,
                                                                    const int32_t* counts, const int32_t* holes,
                                                                    const int32_t* movers, const int32_t* to) {
    pdl_wait();
    pdl_launch_dependents();
    const int n_live = counts[0], moved = counts[1];
    const long long t0 = (long long)blockIdx.x * KP_THREADS + threadIdx.x, step = (long long)gridDim.x * KP_THREADS;
    for (long long i = t0; i < (long long)p.n_seq * p.max_pages; i += step) {
        int pg = p.table[i];
        if (pg >= p.n_pages) {
            set_status(p.status, VSL_ERR_BOUNDS);
            pg = -1;
        }
        table_out[i] = pg < n_live ? pg : to[pg];
    }
    // counts: a hole takes its mover's (one thread reads the one and writes both: ref_out may be ref)
    for (long long i = t0; i < moved; i += step) {
        const int32_t n = p.ref[movers[i]];
        ref_out[holes[i]] = n;
        ref_out[movers[i]] = 0;
    }
    if (ref_out != p.ref)
        for (long long i = t0; i < p.n_pages; i += step) {
            const int32_t n = p.ref[i];
            if (i < n_live ? n > 0 : n <= 0) ref_out[i] = n;
        }
    const int pieces = (int)((p.page_bytes + KP_COPY_BYTES - 1) / KP_COPY_BYTES);
    const long long work = (long long)moved * p.n_pools * pieces;
    for (long long w = blockIdx.x; w < work; w += gridDim.x) {
        const int piece = (int)(w % pieces), pool = (int)(w / pieces % p.n_pools), i = (int)(w / pieces / p.n_pools);
        const size_t lo = (size_t)piece * KP_COPY_BYTES;
        kp_copy(pools.base[pool], p.page_bytes, movers[i], holes[i], lo, min(lo + KP_COPY_BYTES, p.page_bytes));
    }
}

// ---------------------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------------------

static size_t kp_workspace(int n_seq, int n_pages) {
    return (size_t)4 * (n_seq > n_pages ? n_seq : n_pages) * sizeof(int32_t);
}

// Checks the handle; `lens` and `pools`: whether the call uses them.
static int kp_params(const char* what, const vsl_kv_pages* kv, bool lens, bool pools, int* status, KpParams* p, KpPools* q) {
    if (!kv) return set_error(VSL_ERR_INVALID, "%s: null handle", what);
    if (!kv->page_table || !kv->refcount || (lens && !kv->lens) || (pools && kv->n_pools > 0 && !kv->pools))
        return set_error(VSL_ERR_INVALID, "%s: null pointer in the handle", what);
    if (kv->n_seq <= 0 || kv->max_pages <= 0 || kv->n_pages <= 0 || kv->page_size <= 0 || kv->n_pages > (1 << 20) ||
        (long long)kv->max_pages * kv->page_size > (1 << 30))
        return set_error(VSL_ERR_INVALID, "%s: %d sequences of %d pages of %d positions, pool of %d pages", what, kv->n_seq,
                         kv->max_pages, kv->page_size, kv->n_pages);
    *p = KpParams{kv->page_table, kv->n_seq, kv->max_pages, kv->page_size, kv->lens, kv->refcount,
                  kv->n_pages, 0, 0, status};
    if (!pools) return VSL_OK;
    if (kv->n_pools < 0 || kv->n_pools > KP_MAX_POOLS)
        return set_error(VSL_ERR_UNSUPPORTED, "%s: %d pools (at most %d)", what, kv->n_pools, KP_MAX_POOLS);
    if (kv->n_pools && (kv->page_bytes == 0 || kv->page_bytes % 16 || kv->page_bytes > ((size_t)1 << 30)))
        return set_error(VSL_ERR_INVALID, "%s: page_bytes %zu (a multiple of 16, at most 2^30)", what, kv->page_bytes);
    for (int i = 0; i < kv->n_pools; i++) {
        if (!kv->pools[i] || ((uintptr_t)kv->pools[i] & 15))
            return set_error(VSL_ERR_INVALID, "%s: pool %d is null or not 16-byte aligned", what, i);
        q->base[i] = static_cast<unsigned char*>(kv->pools[i]);
    }
    p->n_pools = kv->n_pools;
    p->page_bytes = kv->page_bytes;
    return VSL_OK;
}
static int kp_check_ws(const char* what, const KpParams& p, const void* ws, size_t bytes) {
    const size_t need = kp_workspace(p.n_seq, p.n_pages);
    if (!ws || bytes < need || ((uintptr_t)ws & 3))
        return set_error(VSL_ERR_INVALID, "%s: workspace %zu bytes < %zu, null or misaligned", what, bytes, need);
    return VSL_OK;
}
static int kp_check_list(const char* what, const KpParams& p, int n, const void* a, const void* b) {
    if (n < 0 || n > p.n_seq) return set_error(VSL_ERR_INVALID, "%s: %d entries for %d sequences", what, n, p.n_seq);
    if (n && (!a || !b)) return set_error(VSL_ERR_INVALID, "%s: null list", what);
    return VSL_OK;
}
static unsigned kp_pieces(const KpParams& p) {
    return p.n_pools ? (unsigned)((p.page_bytes + KP_COPY_BYTES - 1) / KP_COPY_BYTES) : 1u;
}

}  // namespace vsl

using namespace vsl;

extern "C" int vsl_kv_pages_workspace_size(int n_seq, int n_pages, size_t* bytes) {
    if (!bytes || n_seq <= 0 || n_pages <= 0)
        return set_error(VSL_ERR_INVALID, "kv_pages_workspace_size: %d sequences, %d pages", n_seq, n_pages);
    *bytes = kp_workspace(n_seq, n_pages);
    return VSL_OK;
}

extern "C" int vsl_kv_fork(const vsl_kv_pages* kv, const int32_t* src, const int32_t* dst, int n, void* workspace,
                           size_t workspace_bytes, int* status, void* stream) {
    KpParams p;
    KpPools pools = {};
    if (int rc = kp_params("kv_fork", kv, true, true, status, &p, &pools)) return rc;
    if (int rc = kp_check_list("kv_fork", p, n, src, dst)) return rc;
    if (int rc = kp_check_ws("kv_fork", p, workspace, workspace_bytes)) return rc;
    if (n > 65535) return set_error(VSL_ERR_UNSUPPORTED, "kv_fork: %d forks in one call (at most 65535)", n);
    if (n == 0) return VSL_OK;
    cudaStream_t st = (cudaStream_t)stream;
    const size_t m = (size_t)(p.n_seq > p.n_pages ? p.n_seq : p.n_pages);
    int32_t* ok = static_cast<int32_t*>(workspace);
    int32_t *fresh = ok + m, *tails = ok + 2 * m, *list = ok + 3 * m;
    if (int rc = launch_status(launch_k(vsl_kv_fork_release_kernel, dim3(n), dim3(KP_THREADS), 0, st, p, src, dst, n, ok),
                               "kv_fork release"))
        return rc;
    if (int rc = launch_status(launch_k(vsl_kv_fork_plan_kernel, dim3(1), dim3(KP_PLAN_THREADS), 0, st, p, src, n, ok,
                                        fresh, tails, list),
                               "kv_fork plan"))
        return rc;
    const dim3 grid(kp_pieces(p), (unsigned)(p.n_pools ? p.n_pools : 1), (unsigned)n);
    if (!p.n_pools) p.page_bytes = 0;
    return launch_status(launch_k(vsl_kv_fork_kernel, grid, dim3(KP_THREADS), 0, st, p, pools, src, dst, ok, fresh),
                         "kv_fork");
}

extern "C" int vsl_kv_free(const vsl_kv_pages* kv, const int32_t* seqs, int n, int* status, void* stream) {
    KpParams p;
    if (int rc = kp_params("kv_free", kv, true, false, status, &p, nullptr)) return rc;
    if (int rc = kp_check_list("kv_free", p, n, seqs, seqs)) return rc;
    if (n == 0) return VSL_OK;
    return launch_status(launch_k(vsl_kv_free_kernel, dim3(n), dim3(KP_THREADS), 0, (cudaStream_t)stream, p, seqs, n),
                         "kv_free");
}

extern "C" int vsl_kv_extend(const vsl_kv_pages* kv, const int32_t* seqs, const int32_t* add, int n, void* workspace,
                             size_t workspace_bytes, int* status, void* stream) {
    KpParams p;
    if (int rc = kp_params("kv_extend", kv, true, false, status, &p, nullptr)) return rc;
    if (int rc = kp_check_list("kv_extend", p, n, seqs, add)) return rc;
    if (int rc = kp_check_ws("kv_extend", p, workspace, workspace_bytes)) return rc;
    if (n == 0) return VSL_OK;
    const size_t m = (size_t)(p.n_seq > p.n_pages ? p.n_seq : p.n_pages);
    int32_t* start = static_cast<int32_t*>(workspace);
    return launch_status(launch_k(vsl_kv_extend_kernel, dim3(1), dim3(KP_PLAN_THREADS), 0, (cudaStream_t)stream, p, seqs,
                                  add, n, start, start + m),
                         "kv_extend");
}

extern "C" int vsl_kv_copy_pages(const vsl_kv_pages* kv, const int32_t* src, const int32_t* dst, int n, int* status,
                                 void* stream) {
    KpParams p;
    KpPools pools = {};
    if (int rc = kp_params("kv_copy_pages", kv, false, true, status, &p, &pools)) return rc;
    if (n < 0 || n > p.n_pages) return set_error(VSL_ERR_INVALID, "kv_copy_pages: %d copies in a pool of %d pages", n, p.n_pages);
    if (n && (!src || !dst)) return set_error(VSL_ERR_INVALID, "kv_copy_pages: null list");
    if (!p.n_pools) return VSL_OK;
    for (int k = 0; k < n; k += 65535) {
        const unsigned m = (unsigned)(n - k < 65535 ? n - k : 65535);
        if (int rc = launch_status(launch_k(vsl_kv_copy_kernel, dim3(kp_pieces(p), (unsigned)p.n_pools, m), dim3(KP_THREADS),
                                            0, (cudaStream_t)stream, p, pools, src + k, dst + k),
                                   "kv_copy_pages"))
            return rc;
    }
    return VSL_OK;
}

extern "C" int vsl_kv_compact(const vsl_kv_pages* kv, int32_t* page_table_out, int32_t* refcount_out, int32_t* counts,
                              void* workspace, size_t workspace_bytes, int* status, void* stream) {
    KpParams p;
    KpPools pools = {};
    if (int rc = kp_params("kv_compact", kv, false, true, status, &p, &pools)) return rc;
    if (!page_table_out || !refcount_out || !counts) return set_error(VSL_ERR_INVALID, "kv_compact: null output");
    if (int rc = kp_check_ws("kv_compact", p, workspace, workspace_bytes)) return rc;
    cudaStream_t st = (cudaStream_t)stream;
    const size_t m = (size_t)(p.n_seq > p.n_pages ? p.n_seq : p.n_pages);
    int32_t* holes = static_cast<int32_t*>(workspace);
    int32_t *movers = holes + m, *to = holes + 2 * m;
    if (int rc = launch_status(launch_k(vsl_kv_compact_plan_kernel, dim3(1), dim3(KP_PLAN_THREADS), 0, st, p, counts, holes,
                                        movers, to),
                               "kv_compact plan"))
        return rc;
    return launch_status(launch_k(vsl_kv_compact_kernel, dim3(sm_count() * 8), dim3(KP_THREADS), 0, st, p, pools,
                                  page_table_out, refcount_out, counts, holes, movers, to),
                         "kv_compact");
}
