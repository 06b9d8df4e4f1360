// kv4_pages.cu -- pages of the paged 4-bit KV cache: allocation, forks,
// release, compaction and copies, all decided on the device.
//
// A fork or a compaction is two launches: one CTA makes the plan (prefix sums
// over refs, 4096 pages a step: the lowest free pages, or the pairs to move),
// then a grid over all SMs copies the pages in every layer and rewrites tables
// and refs; where there is little to copy (512 KB at most) the one CTA does that
// too, which for a small model takes 18 us for fork, release, compaction and a copy
// instead of 24.  Free pages go to the sequences in the order of the list, so
// the result does not depend on timing.  The copies read and write each moved byte
// once, at 5.5 TB/s in both directions together (80 layers, pages of 64 positions of 8 heads of 128).
#include "kv4.cuh"

namespace {

constexpr int PLAN_THREADS = 1024;
constexpr int PLAN_STEP = 4 * PLAN_THREADS;   // pages a step of the plan
constexpr int COPY_THREADS = 256;

// the plan's words: [0] moves of a compaction; lists from word 16 on
constexpr int PLAN_LISTS = 16;

__device__ __forceinline__ int warp_inclusive(int v) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, v, o);
        if ((threadIdx.x & 31) >= o) v += u;
    }
    return v;
}

// inclusive prefix sum over the CTA's PLAN_THREADS threads; total: of all
__device__ __forceinline__ int block_inclusive(int v, int *sh, int &total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    v = warp_inclusive(v);
    __syncthreads();
    if (lane == 31) sh[warp] = v;
    __syncthreads();
    const int w = warp_inclusive(sh[lane]);   // PLAN_THREADS / 32 = 32 warps
    total = __shfl_sync(0xffffffffu, w, 31);
    const int before = __shfl_sync(0xffffffffu, w, (warp + 31) & 31);
    return v + (warp ? before : 0);
}

// four refs from page p on; pages past the end count as held
__device__ __forceinline__ int4 four_refs(const Kv4View &c, int p) {
    int4 r;
    r.x = p < c.n_pages ? c.refs[p] : 1;
    r.y = p + 1 < c.n_pages ? c.refs[p + 1] : 1;
    r.z = p + 2 < c.n_pages ? c.refs[p + 2] : 1;
    r.w = p + 3 < c.n_pages ? c.refs[p + 3] : 1;
    return r;
}

// the lowest `want` free pages into list; returns how many there are
__device__ int find_free(const Kv4View &c, int want, int *list, int *sh) {
    int found = 0;
    for (int p0 = 0; p0 < c.n_pages && found < want; p0 += PLAN_STEP) {
        const int p = p0 + 4 * threadIdx.x;
        const int4 r = four_refs(c, p);
        const int f[4] = {r.x == 0, r.y == 0, r.z == 0, r.w == 0};
        const int mine = f[0] + f[1] + f[2] + f[3];
        int total, at = found + block_inclusive(mine, sh, total) - mine;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (f[i]) {
                if (at < want) list[at] = p + i;
                ++at;
            }
        found += total;
    }
    __syncthreads();   // the list is read by other threads
    return min(found, want);
}

__device__ __forceinline__ int pages_of(const Kv4View &c, int len) { return len / c.page_tokens + (len % c.page_tokens != 0); }
// whether a length is one that a row of the tables can hold: no other is followed into them
__device__ __forceinline__ bool len_ok(const Kv4View &c, int len) {
    return len >= 0 && len <= (long long)c.max_pages * c.page_tokens;
}

// ---- extend -----------------------------------------------------------------
// A sequence's need is at most n_pages + 1 (<= 2^20 + 1) in the sums, and the
// sum before a step of 1024 sequences at most 2^29: no int overflows.
constexpr int PLAN_SUM_MAX = 1 << 29;

__global__ void __launch_bounds__(PLAN_THREADS, 1)
extend_kernel(const __grid_constant__ Kv4View c, const int *seqs, const int *counts,
              int *start, int n, int *list) {
    early_wait();
    early_next();
    __shared__ int sh[32];
    // pages that the list's sequences need, in order
    int need_all = 0;
    for (int i0 = 0; i0 < n; i0 += PLAN_THREADS) {
        const int i = i0 + threadIdx.x;
        int need = 0;
        if (i < n) {
            const int s = seqs ? seqs[i] : i, add = counts[i];
            if (s >= 0 && s < c.max_seqs && add > 0) {
                const long long len = c.lens[s], after = len + add;
                if (len >= 0 && after <= (long long)c.max_pages * c.page_tokens)
                    need = min(pages_of(c, (int)after) - pages_of(c, (int)len), c.n_pages + 1);
            }
        }
        int total;
        block_inclusive(need, sh, total);
        need_all = min(need_all + total, PLAN_SUM_MAX);
    }
    const int have = find_free(c, need_all, list, sh);
    int base = 0;
    for (int i0 = 0; i0 < n; i0 += PLAN_THREADS) {
        const int i = i0 + threadIdx.x;
        int need = 0, s = -1, add = 0, len = 0, err = 0;
        if (i < n) {
            s = seqs ? seqs[i] : i;
            add = counts[i];
            if (s < 0 || s >= c.max_seqs || add < 0) {
                err = HOLO_E_ARG;
            } else {
                len = c.lens[s];
                if (!len_ok(c, len)) err = HOLO_E_ARG;
                else if ((long long)len + add > (long long)c.max_pages * c.page_tokens) err = HOLO_E_NOMEM;
                else need = min(pages_of(c, len + add) - pages_of(c, len), c.n_pages + 1);
            }
        }
        int total;
        const int end = base + block_inclusive(need, sh, total);
        base = min(base + total, PLAN_SUM_MAX);
        if (i < n) {
            if (!err && need > 0 && end > have) err = HOLO_E_NOMEM;
            if (!err) {
                const int first = pages_of(c, len);
                for (int j = 0; j < need; ++j) {
                    const int page = list[end - need + j];
                    c.tables[(size_t)s * c.max_pages + first + j] = page;
                    c.refs[page] = 1;
                }
                c.lens[s] = len + add;
                start[i] = len;
            } else {
                start[i] = -1;
                kv4_report(c.status, err);
            }
        }
    }
}

// ---- copies ---------------------------------------------------------------------
// The threads that share a unit of work, one of `teams`: a CTA of a grid, or a
// warp of the one CTA that does everything.
struct Team {
    int team, teams, thread, threads;
};
__device__ __forceinline__ Team cta_team() { return {(int)blockIdx.x, (int)gridDim.x, (int)threadIdx.x, (int)blockDim.x}; }
__device__ __forceinline__ Team warp_team() { return {(int)threadIdx.x / 32, PLAN_THREADS / 32, (int)threadIdx.x % 32, 32}; }

// One page of one layer; four loads under way a thread.
__device__ __forceinline__ void copy_page(const Team &t, uint8_t *pool, size_t page_bytes, int src, int dst) {
    const uint4 *s = reinterpret_cast<const uint4 *>(pool + (size_t)src * page_bytes);
    uint4 *d = reinterpret_cast<uint4 *>(pool + (size_t)dst * page_bytes);
    const int words = (int)(page_bytes / 16), step = t.threads;
    int i = t.thread;
    for (; i + 3 * step < words; i += 4 * step) {
        uint4 v[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = __ldcs(s + i + k * step);
#pragma unroll
        for (int k = 0; k < 4; ++k) __stcs(d + i + k * step, v[k]);
    }
    for (; i < words; i += step) d[i] = s[i];
}

__global__ void __launch_bounds__(COPY_THREADS)
copy_kernel(const __grid_constant__ Kv4View c, size_t page_bytes, size_t layer_bytes, int layers,
            const int *src, const int *dst, int n) {
    early_wait();
    early_next();
    const long long total = (long long)n * layers;
    for (long long u = blockIdx.x; u < total; u += gridDim.x) {
        const int i = (int)(u / layers), layer = (int)(u % layers);
        const int s = src[i], d = dst[i];
        if (s < 0 || s >= c.n_pages || d < 0 || d >= c.n_pages) {
            if (threadIdx.x == 0) kv4_report(c.status, HOLO_E_ARG);
            continue;
        }
        copy_page(cta_team(), c.pool + layer * layer_bytes, page_bytes, s, d);
    }
}

// ---- fork ------------------------------------------------------------------------
// the children's rows, the pages' counts and the copies; the plan has looked at the parents' entries
__device__ __forceinline__ void fork_apply(const Kv4View &c, size_t page_bytes, size_t layer_bytes, int layers,
                                           const int *parents, const int *children, int n, const int *page, const Team &t) {
    const long long total = (long long)n * layers;
    for (long long u = t.team; u < total; u += t.teams) {
        const int i = (int)(u / layers), layer = (int)(u % layers);
        const int fresh = page[i];
        if (fresh == -2) continue;
        const int p = parents[i], k = children[i], len = c.lens[p], full = len / c.page_tokens;
        const int *from = c.tables + (size_t)p * c.max_pages;
        if (layer == 0) {   // the child's row and the pages' counts, once
            int *to = c.tables + (size_t)k * c.max_pages;
            for (int j = t.thread; j < c.max_pages; j += t.threads) {
                int e = -1;
                if (j < full) {
                    e = from[j];
                    atomicAdd(c.refs + e, 1);
                } else if (j == full) {
                    e = fresh;   // -1: the parent ends with a full page
                    if (e >= 0) c.refs[e] = 1;
                }
                to[j] = e;
            }
            if (t.thread == 0) c.lens[k] = len;
        }
        if (fresh >= 0) copy_page(t, c.pool + layer * layer_bytes, page_bytes, from[full], fresh);
    }
}

// page[i]: the new page of child i; -1: it needs none, -2: it is left out.
// ALL: the rest of the work too, where it is little
template <bool ALL>
__global__ void __launch_bounds__(PLAN_THREADS, 1)
fork_plan_kernel(const __grid_constant__ Kv4View c, size_t page_bytes, size_t layer_bytes, int layers, const int *parents,
                 const int *children, int n, int *page, int *list) {
    early_wait();
    early_next();
    __shared__ int sh[32];
    // which children there can be: a warp each looks at the parent's pages
    for (int i = threadIdx.x / 32; i < n; i += PLAN_THREADS / 32) {
        const int p = parents[i], k = children[i];
        bool good = p >= 0 && p < c.max_seqs && k >= 0 && k < c.max_seqs && p != k && c.lens[k] == 0 && len_ok(c, c.lens[p]);
        if (good) {
            const int *from = c.tables + (size_t)p * c.max_pages;
            const int held = pages_of(c, c.lens[p]);
            for (int j = threadIdx.x % 32; j < held; j += 32) good &= (unsigned)from[j] < (unsigned)c.n_pages;
        }
        good = __all_sync(0xffffffffu, good);
        if (threadIdx.x % 32 == 0) {
            page[i] = good ? -1 : -2;
            if (!good) kv4_report(c.status, HOLO_E_ARG);
        }
    }
    __syncthreads();
    int need_all = 0;
    for (int i0 = 0; i0 < n; i0 += PLAN_THREADS) {
        const int i = i0 + threadIdx.x;
        const int need = i < n && page[i] == -1 ? c.lens[parents[i]] % c.page_tokens != 0 : 0;
        int total;
        block_inclusive(need, sh, total);
        need_all += total;
    }
    const int have = find_free(c, need_all, list, sh);
    int base = 0;
    for (int i0 = 0; i0 < n; i0 += PLAN_THREADS) {
        const int i = i0 + threadIdx.x;
        const int need = i < n && page[i] == -1 ? c.lens[parents[i]] % c.page_tokens != 0 : 0;
        int total;
        const int end = base + block_inclusive(need, sh, total);
        base += total;
        if (need) {
            if (end <= have) {
                page[i] = list[end - 1];
            } else {
                page[i] = -2;
                kv4_report(c.status, HOLO_E_NOMEM);
            }
        }
    }
    if (ALL) {
        __syncthreads();
        fork_apply(c, page_bytes, layer_bytes, layers, parents, children, n, page, warp_team());
    }
}

__global__ void __launch_bounds__(COPY_THREADS)
fork_kernel(const __grid_constant__ Kv4View c, size_t page_bytes, size_t layer_bytes, int layers, const int *parents,
            const int *children, int n, const int *page) {
    early_wait();
    early_next();
    fork_apply(c, page_bytes, layer_bytes, layers, parents, children, n, page, cta_team());
}

// ---- release ----------------------------------------------------------------------
__global__ void __launch_bounds__(COPY_THREADS)
release_kernel(const __grid_constant__ Kv4View c, const int *seqs, int n) {
    early_wait();
    early_next();
    __shared__ int len_s;
    for (int i = blockIdx.x; i < n; i += gridDim.x) {
        const int s = seqs ? seqs[i] : i;
        if (s < 0 || s >= c.max_seqs) {
            if (threadIdx.x == 0) kv4_report(c.status, HOLO_E_ARG);
            continue;
        }
        __syncthreads();
        if (threadIdx.x == 0) {
            len_s = atomicExch(c.lens + s, 0);
            if (!len_ok(c, len_s)) {          // left as it was
                c.lens[s] = len_s;
                kv4_report(c.status, HOLO_E_ARG);
            }
        }
        __syncthreads();
        if (!len_ok(c, len_s)) continue;
        const int held = pages_of(c, len_s);
        int *row = c.tables + (size_t)s * c.max_pages;
        for (int j = threadIdx.x; j < c.max_pages; j += COPY_THREADS) {
            if (j < held) {
                const int e = row[j];
                if (e >= 0 && e < c.n_pages) atomicSub(c.refs + e, 1);
                else kv4_report(c.status, HOLO_E_ARG);
            }
            row[j] = -1;
        }
    }
}

// ---- compact ------------------------------------------------------------------------
// the counts, the tables and the copies
__device__ __forceinline__ void compact_apply(const Kv4View &c, size_t page_bytes, size_t layer_bytes, int layers, int moves,
                                              const int *src, const int *dst, const int *to, const Team &t) {
    if (moves == 0) return;
    const long long me = (long long)t.team * t.threads + t.thread, all = (long long)t.teams * t.threads;
    for (long long i = me; i < moves; i += all) {   // sources and targets are disjoint
        c.refs[dst[i]] = c.refs[src[i]];
        c.refs[src[i]] = 0;
    }
    for (long long i = me; i < (long long)c.max_seqs * c.max_pages; i += all) {
        const int e = c.tables[i];
        if (e >= 0 && e < c.n_pages && to[e] != e) c.tables[i] = to[e];
    }
    const long long total = (long long)moves * layers;
    for (long long u = t.team; u < total; u += t.teams)
        copy_page(t, c.pool + (u % layers) * layer_bytes, page_bytes, src[u / layers], dst[u / layers]);
}

// plan[0] moves: src, dst (ascending both); to[page]: its number afterwards.
// ALL: the rest of the work too, where it is little
template <bool ALL>
__global__ void __launch_bounds__(PLAN_THREADS, 1)
compact_plan_kernel(const __grid_constant__ Kv4View c, size_t page_bytes, size_t layer_bytes, int layers, int *plan, int *src,
                    int *dst, int *to) {
    early_wait();
    early_next();
    __shared__ int sh[32];
    int live = 0;
    int4 r;                                   // (a pool of one step is read once)
    for (int p0 = 0; p0 < c.n_pages; p0 += PLAN_STEP) {
        const int p = p0 + 4 * threadIdx.x;
        r = four_refs(c, p);
        const int held[4] = {r.x != 0 && p < c.n_pages, r.y != 0 && p + 1 < c.n_pages, r.z != 0 && p + 2 < c.n_pages,
                             r.w != 0 && p + 3 < c.n_pages};
        int total;
        block_inclusive(held[0] + held[1] + held[2] + held[3], sh, total);
        live += total;
    }
    int movers = 0, holes = 0;
    for (int p0 = 0; p0 < c.n_pages; p0 += PLAN_STEP) {
        const int p = p0 + 4 * threadIdx.x;
        if (c.n_pages > PLAN_STEP) r = four_refs(c, p);
        const int ref[4] = {r.x, r.y, r.z, r.w};
        // movers in the low half of a sum, holes in the high half
        int mine = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (p + i < c.n_pages) {
                if (ref[i] != 0 && p + i >= live) mine += 1;
                if (ref[i] == 0 && p + i < live) mine += 1 << 16;
            }
        int total;
        const int before = block_inclusive(mine, sh, total) - mine;
        int m = movers + (before & 0xffff), h = holes + (before >> 16);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (p + i < c.n_pages) {
                if (ref[i] != 0 && p + i >= live) src[m++] = p + i;
                if (ref[i] == 0 && p + i < live) dst[h++] = p + i;
                to[p + i] = p + i;
            }
        movers += total & 0xffff;
        holes += total >> 16;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < movers; i += PLAN_THREADS) to[src[i]] = dst[i];
    if (threadIdx.x == 0) plan[0] = movers;   // as many holes as movers
    if (ALL) {
        __syncthreads();
        compact_apply(c, page_bytes, layer_bytes, layers, movers, src, dst, to, warp_team());
    }
}

__global__ void __launch_bounds__(COPY_THREADS)
compact_kernel(const __grid_constant__ Kv4View c, size_t page_bytes, size_t layer_bytes, int layers, const int *plan,
               const int *src, const int *dst, const int *to) {
    early_wait();
    early_next();
    compact_apply(c, page_bytes, layer_bytes, layers, plan[0], src, dst, to, cta_team());
}

struct Pages {
    Kv4View view;
    Kv4Work work;
    cudaStream_t st;
    size_t page_bytes, layer_bytes;
    int sms;
};

bool begin(const holo_kv4 *c, const char *what, Pages &p, bool refs) {
    if (!kv4_begin(c, 0, what, p.view, p.st, &p.work)) return false;
    if (refs && !c->refs) {
        holo_set_status(HOLO_E_ARG, what);
        return false;
    }
    p.page_bytes = (size_t)c->n_kv_heads * p.view.page_blocks * kv4_block_bytes(c->head_dim);
    p.layer_bytes = p.page_bytes * c->n_pages;
    p.sms = holo_dev()->sms;
    return true;
}

int refuse(const char *what) {
    holo_set_status(HOLO_E_ARG, what);
    return HOLO_E_ARG;
}

// so little to copy (page-layers) that one CTA does it sooner than a second launch would begin
bool little(const Pages &p, long long units) { return units * (long long)p.page_bytes <= (512 << 10); }

unsigned copy_grid(const Pages &p, long long units) {
    const long long most = (long long)p.sms * 8;
    return (unsigned)(units < 1 ? 1 : units < most ? units : most);
}

}  // namespace

extern "C" {

int cuda_kv4_extend(const holo_kv4 *c, const int *seqs, const int *counts, int *start, int n) {
    Pages p;
    if (!begin(c, "cuda_kv4_extend", p, true)) return cuda_last_status();
    if (n < 0 || n > c->max_seqs || (n > 0 && (!counts || !start))) return refuse("cuda_kv4_extend");
    if (n == 0) return HOLO_OK;
    holo_launch_early(extend_kernel, 1, PLAN_THREADS, 0, p.st, p.view, seqs, counts, start, n, p.work.plan + PLAN_LISTS);
    return kv4_end("cuda_kv4_extend");
}

int cuda_kv4_fork(const holo_kv4 *c, const int *parents, const int *children, int n) {
    Pages p;
    if (!begin(c, "cuda_kv4_fork", p, true)) return cuda_last_status();
    if (n < 0 || n > c->max_seqs || (n > 0 && (!parents || !children))) return refuse("cuda_kv4_fork");
    if (n == 0) return HOLO_OK;
    int *page = p.work.plan + PLAN_LISTS, *list = page + c->max_seqs;
    if (little(p, (long long)n * c->n_layers)) {
        holo_launch_early(fork_plan_kernel<true>, 1, PLAN_THREADS, 0, p.st, p.view, p.page_bytes, p.layer_bytes, c->n_layers,
                          parents, children, n, page, list);
    } else {
        holo_launch_early(fork_plan_kernel<false>, 1, PLAN_THREADS, 0, p.st, p.view, p.page_bytes, p.layer_bytes,
                          c->n_layers, parents, children, n, page, list);
        holo_launch_early(fork_kernel, copy_grid(p, (long long)n * c->n_layers), COPY_THREADS, 0, p.st, p.view, p.page_bytes,
                          p.layer_bytes, c->n_layers, parents, children, n, page);
    }
    return kv4_end("cuda_kv4_fork");
}

int cuda_kv4_release(const holo_kv4 *c, const int *seqs, int n) {
    Pages p;
    if (!begin(c, "cuda_kv4_release", p, true)) return cuda_last_status();
    if (n < 0 || n > c->max_seqs) return refuse("cuda_kv4_release");
    if (n == 0) return HOLO_OK;
    holo_launch_early(release_kernel, copy_grid(p, n), COPY_THREADS, 0, p.st, p.view, seqs, n);
    return kv4_end("cuda_kv4_release");
}

int cuda_kv4_compact(const holo_kv4 *c) {
    Pages p;
    if (!begin(c, "cuda_kv4_compact", p, true)) return cuda_last_status();
    int *src = p.work.plan + PLAN_LISTS, *dst = src + c->n_pages, *to = dst + c->n_pages;
    // at most half of the pages move
    if (little(p, (long long)(c->n_pages / 2) * c->n_layers) && (long long)c->max_seqs * c->max_pages <= 64 * PLAN_THREADS) {
        holo_launch_early(compact_plan_kernel<true>, 1, PLAN_THREADS, 0, p.st, p.view, p.page_bytes, p.layer_bytes,
                          c->n_layers, p.work.plan, src, dst, to);
    } else {
        holo_launch_early(compact_plan_kernel<false>, 1, PLAN_THREADS, 0, p.st, p.view, p.page_bytes, p.layer_bytes,
                          c->n_layers, p.work.plan, src, dst, to);
        holo_launch_early(compact_kernel, copy_grid(p, (long long)c->n_pages * c->n_layers), COPY_THREADS, 0, p.st, p.view,
                          p.page_bytes, p.layer_bytes, c->n_layers, p.work.plan, src, dst, to);
    }
    return kv4_end("cuda_kv4_compact");
}

int cuda_kv4_copy_pages(const holo_kv4 *c, const int *src, const int *dst, int n) {
    Pages p;
    if (!begin(c, "cuda_kv4_copy_pages", p, false)) return cuda_last_status();
    if (n < 0 || (n > 0 && (!src || !dst))) return refuse("cuda_kv4_copy_pages");
    if (n == 0) return HOLO_OK;
    holo_launch_early(copy_kernel, copy_grid(p, (long long)n * c->n_layers), COPY_THREADS, 0, p.st, p.view, p.page_bytes, p.layer_bytes, c->n_layers, src, dst, n);
    return kv4_end("cuda_kv4_copy_pages");
}

}  // extern "C"
