/* kv_pages.cu - the page bookkeeping of a paged cache on the device:
 * growth, fork (beam reorder, release) and compaction.
 *
 * A call is a plan (one CTA: validation, the ordered choice of pages) and,
 * where pages are moved or tables rewritten, an apply over the whole GPU.
 * The choice is a compaction of {p : refs[p] == 0} (or of live and free
 * pages around the live count) in page order, so its result depends on the
 * state alone, never on timing; reference counts change by integer atomics,
 * whose order does not show.  Everything that a plan refuses leaves the
 * state as it was: the apply kernels return on its first word.
 *
 * The copies are bound by bytes, the rest by latency (a plan reads rows,
 * lengths, marks and counts one behind the other).  Measured on the device:
 * compaction of 128 sequences, 335 MB read and written, 66 us (53 of them the
 * copies, 6.2 TB/s); fork of 32 x 8 beams with 63 MB of copies, and growth,
 * 22 us; of 2 x 4 beams 13 us. */
#include "pk_common.h"

__device__ uint32_t pk_err_word_dev;

uint32_t *pk_err_word() {
    static uint32_t *word[64];
    const int dev = pm_cur_device();
    if (dev < 64 && word[dev]) return word[dev];
    void *p = nullptr;
    if (cudaGetSymbolAddress(&p, pk_err_word_dev) != cudaSuccess) return nullptr;
    if (dev < 64) word[dev] = (uint32_t *)p;
    return (uint32_t *)p;
}

extern "C" uint32_t pulsar_kv_error(void) {
    uint32_t v = 0, zero = 0;
    uint32_t *w = pk_err_word();
    /* the calls' streams need not be ones that a copy waits for */
    if (!w || !pm_ok(cudaDeviceSynchronize(), "kv error word") || !pm_ok(cudaMemcpy(&v, w, 4, cudaMemcpyDeviceToHost), "kv error word") ||
        (v && !pm_ok(cudaMemcpy(w, &zero, 4, cudaMemcpyHostToDevice), "kv error word")))
        return 0xffffffffu;
    return v;
}

#define PK_PLAN 1024u /* threads of a plan CTA */
#define PK_FORK_COLS 8u

/* -------------------------------------------------- ordered choice of pages */

struct pk_scan {
    uint32_t warp[32];
    uint32_t total;
};

/* exclusive prefix of v over the CTA's threads; *total = their sum */
__device__ __forceinline__ uint32_t pk_block_scan(uint32_t v, pk_scan &s, uint32_t *total) {
    const uint32_t lane = threadIdx.x & 31u, w = threadIdx.x >> 5;
    uint32_t x = v;
#pragma unroll
    for (uint32_t o = 1; o < 32; o <<= 1) {
        const uint32_t y = __shfl_up_sync(~0u, x, o);
        if (lane >= o) x += y;
    }
    __syncthreads(); /* the previous scan's readers are done */
    if (lane == 31) s.warp[w] = x;
    __syncthreads();
    if (w == 0) {
        const uint32_t mine = lane < (blockDim.x >> 5) ? s.warp[lane] : 0u;
        uint32_t y = mine;
#pragma unroll
        for (uint32_t o = 1; o < 32; o <<= 1) {
            const uint32_t z = __shfl_up_sync(~0u, y, o);
            if (lane >= o) y += z;
        }
        s.warp[lane] = y - mine;
        if (lane == 31) s.total = y;
    }
    __syncthreads();
    *total = s.total;
    return s.warp[w] + x - v;
}

/* Each warp walks its own run of [lo, hi) in page order, 32 pages a step; the
 * pages for which refs[p] > 0 equals `live` get the ranks 0, 1, ... in page
 * order.  want(total) is asked once their number is known (by every thread
 * alike), and emit(p, rank) is called for the ranks below it.  Returns the
 * total.  The counts are read twice; an SM takes them from the caches at some
 * 64 bytes a cycle. */
template <class W, class F>
__device__ uint32_t pk_choose(const int32_t *refs, uint32_t lo, uint32_t hi, bool live, pk_scan &s, W want, F emit) {
    const uint32_t lane = threadIdx.x & 31u, w = threadIdx.x >> 5, nw = blockDim.x >> 5;
    const uint32_t n = hi - lo;
    const uint32_t run = ((n + nw - 1) / nw + 31u) & ~31u;
    const uint64_t b64 = (uint64_t)lo + (uint64_t)w * run;
    const uint32_t b = b64 < hi ? (uint32_t)b64 : hi, e = hi - b < run ? hi : b + run;
    uint32_t count = 0;
#pragma unroll 8
    for (uint32_t p = b + lane; p < e; p += 32) count += (refs[p] > 0) == live;
    uint32_t total;
    uint32_t at = pk_block_scan(count, s, &total);
    at = __shfl_sync(~0u, at, 0); /* the warp's first rank */
    const uint32_t most = want(total);
    for (uint32_t p0 = b; p0 < e && at < most; p0 += 32) {
        const uint32_t p = p0 + lane;
        const bool hit = p < e && (refs[p] > 0) == live;
        const uint32_t m = __ballot_sync(~0u, hit);
        const uint32_t rank = at + __popc(m & ((1u << lane) - 1u));
        if (hit && rank < most) emit(p, rank);
        at += __popc(m);
    }
    return total;
}

/* words that a plan keeps in shared memory (row marks, offsets, ranks: what it looks up at random); more rows than
 * that use the workspace */
#define PK_MARKS 8192u

__device__ __forceinline__ uint32_t pk_ceil(uint32_t a, uint32_t b) { return (a + b - 1u) / b; }

/* ------------------------------------------------------------------ growth */

/* One CTA.  ws: u32 mark[n_rows], offset[n]; the pages go straight into the
 * tables: a page's rank finds its row by binary search over the offsets. */
__global__ void __launch_bounds__(PK_PLAN) pk_grow_kernel(pulsar_kv_pool P, const int32_t *rows, const int32_t *n_new,
                                                          uint32_t n, int32_t *status, uint32_t *ws) {
    __shared__ pk_scan scan;
    __shared__ uint32_t bad, marks[PK_MARKS];
    __shared__ unsigned long long wanted; /* need_all could wrap: nothing is taken from it unless this fits */
    pk_enter();
    const bool near = (uint64_t)P.n_rows + n <= PK_MARKS;
    uint32_t *mark = near ? marks : ws, *off = mark + P.n_rows;
    const uint32_t tid = threadIdx.x;
    const uint32_t cap = P.max_pages * P.page_size;
    if (tid == 0) {
        bad = 0;
        wanted = 0;
    }
    for (uint32_t r = tid; r < P.n_rows; r += PK_PLAN) mark[r] = 0;
    __syncthreads();
    uint32_t need_all = 0;
    for (uint32_t i0 = 0; i0 < n; i0 += PK_PLAN) {
        const uint32_t i = i0 + tid;
        uint32_t need = 0;
        if (i < n) {
            const int32_t r = rows ? rows[i] : (int32_t)i;
            const int32_t more = n_new[i];
            if (r < 0 || (uint32_t)r >= P.n_rows || more < 0 || atomicExch(&mark[r], 1u)) {
                atomicOr(&bad, 1u);
            } else {
                const int32_t len = P.len[r];
                if (len < 0 || (uint32_t)len > cap) atomicOr(&bad, 1u);
                else if ((uint32_t)more > cap - (uint32_t)len) atomicOr(&bad, 2u);
                else need = pk_ceil((uint32_t)len + more, P.page_size) - pk_ceil(len, P.page_size);
            }
        }
        if (need) atomicAdd(&wanted, (unsigned long long)need);
        uint32_t total;
        const uint32_t at = pk_block_scan(need, scan, &total);
        if (i < n) off[i] = need_all + at;
        need_all += total;
    }
    __syncthreads();
    if (bad) {
        if (tid == 0) *(int4 *)status = make_int4(bad & 1u ? PULSAR_KV_INVALID : PULSAR_KV_WIDE, 0, 0, 0);
        return;
    }
    bool ok = false;
    const uint32_t free_pages = pk_choose(
        P.refs, 0, P.n_pages, false, scan,
        [&](uint32_t total) {
            ok = wanted <= total;
            return ok ? need_all : 0u;
        },
        [&](uint32_t page, uint32_t rank) {
            uint32_t a = 0, b = n; /* the last i with off[i] <= rank */
            while (b - a > 1) {
                const uint32_t m = (a + b) >> 1;
                if (off[m] <= rank) a = m;
                else b = m;
            }
            const uint32_t r = rows ? (uint32_t)rows[a] : a;
            P.table[r * P.table_stride + pk_ceil(P.len[r], P.page_size) + (rank - off[a])] = (int32_t)page;
            P.refs[page] = 1;
        });
    if (tid == 0)
        *(int4 *)status = make_int4(ok ? PULSAR_KV_OK : PULSAR_KV_SHORT, ok ? (int32_t)need_all : 0, (int32_t)free_pages, 0);
    if (!ok) return;
    __syncthreads(); /* the lengths above are read before they change */
    for (uint32_t i = tid; i < n; i += PK_PLAN) P.len[rows ? rows[i] : (int32_t)i] += n_new[i];
}

/* -------------------------------------------------------------------- fork */

/* what the plan hands to the apply kernel */
struct pk_fork_ws {
    uint32_t *head;           /* [0] go, [1] copies, [2] widest row touched, in pages */
    uint32_t *mark, *first;   /* [n_rows] */
    uint32_t *was, *now;      /* [n] tokens of dst[i] before and after */
    int32_t *fresh;           /* [n] the page of i's copy, or -1 */
    int32_t *pair;            /* [n][2] copies: from, to */
    uint32_t *rank;           /* [n] */
};

__host__ __device__ static inline pk_fork_ws pk_fork_layout(void *ws, uint32_t n_rows, uint32_t n) {
    pk_fork_ws w;
    uint32_t *p = (uint32_t *)ws;
    w.head = p;
    w.mark = p + 4;
    w.first = w.mark + n_rows;
    w.was = w.first + n_rows;
    w.now = w.was + n;
    w.fresh = (int32_t *)(w.now + n);
    w.rank = (uint32_t *)(w.fresh + n);
    w.pair = (int32_t *)(w.rank + n);
    return w;
}

#define PK_IS_DST 1u
#define PK_STAYS 2u /* continues itself */

/* by one CTA */
__device__ void pk_fork_plan(const pulsar_kv_pool &P, const int32_t *dst, const int32_t *src, uint32_t n,
                             int32_t *status, void *wsp) {
    __shared__ pk_scan scan;
    __shared__ uint32_t bad, wide, marks[PK_MARKS];
    pk_fork_ws w = pk_fork_layout(wsp, P.n_rows, n);
    const uint32_t tid = threadIdx.x, threads = blockDim.x;
    const uint32_t cap = P.max_pages * P.page_size;
    if (2ull * P.n_rows + n <= PK_MARKS) {
        w.mark = marks;
        w.first = marks + P.n_rows;
        w.rank = w.first + P.n_rows; /* the apply kernel does not read these */
    }
    if (tid == 0) bad = wide = 0;
    for (uint32_t r = tid; r < P.n_rows; r += threads) {
        w.mark[r] = 0;
        w.first[r] = ~0u;
    }
    __syncthreads();
    for (uint32_t i = tid; i < n; i += threads) {
        const int32_t d = dst[i], s = src[i];
        if (d < 0 || (uint32_t)d >= P.n_rows || s < -1 || s >= (int32_t)P.n_rows ||
            (atomicOr(&w.mark[d], s == d ? PK_IS_DST | PK_STAYS : PK_IS_DST) & PK_IS_DST)) {
            atomicOr(&bad, 1u);
            continue;
        }
        const int32_t was = P.len[d], now = s < 0 ? 0 : P.len[s];
        if (was < 0 || now < 0 || (uint32_t)was > cap || (uint32_t)now > cap) {
            atomicOr(&bad, 1u);
            continue;
        }
        if (s >= 0) atomicMin(&w.first[s], i);
        w.was[i] = was;
        w.now[i] = now;
        atomicMax(&wide, pk_ceil(was > now ? was : now, P.page_size));
    }
    __syncthreads();
    if (bad) {
        if (tid == 0) {
            w.head[0] = 0;
            *(int4 *)status = make_int4(PULSAR_KV_INVALID, 0, 0, 0);
        }
        return;
    }
    uint32_t copies = 0;
    for (uint32_t i0 = 0; i0 < n; i0 += threads) {
        const uint32_t i = i0 + tid;
        uint32_t need = 0;
        if (i < n) {
            const int32_t s = src[i];
            if (s >= 0 && s != dst[i] && w.now[i] % P.page_size) {
                const uint32_t m = w.mark[s];
                const bool stays = !(m & PK_IS_DST) || (m & PK_STAYS);
                need = stays || w.first[s] != i;
            }
        }
        uint32_t total;
        const uint32_t at = pk_block_scan(need, scan, &total);
        if (i < n) {
            w.fresh[i] = -1;
            if (need) w.rank[copies + at] = i;
        }
        copies += total;
    }
    __syncthreads(); /* rank[] is whole */
    bool ok = false;
    const uint32_t free_pages = pk_choose(
        P.refs, 0, P.n_pages, false, scan,
        [&](uint32_t total) {
            ok = copies <= total;
            return ok ? copies : 0u;
        },
        [&](uint32_t page, uint32_t rank) {
            const uint32_t i = w.rank[rank];
            w.fresh[i] = (int32_t)page;
            w.pair[2 * rank] = P.table[src[i] * P.table_stride + w.now[i] / P.page_size];
            w.pair[2 * rank + 1] = (int32_t)page;
        });
    if (tid == 0) {
        w.head[0] = ok;
        w.head[1] = copies;
        w.head[2] = wide;
        *(int4 *)status = make_int4(ok ? PULSAR_KV_OK : PULSAR_KV_SHORT, ok ? (int32_t)copies : 0, (int32_t)free_pages, 0);
    }
}

__global__ void __launch_bounds__(PK_PLAN) pk_fork_plan_kernel(pulsar_kv_pool P, const int32_t *dst,
                                                               const int32_t *src, uint32_t n, int32_t *status,
                                                               void *wsp) {
    pk_enter();
    pk_fork_plan(P, dst, src, n, status, wsp);
}

/* Pages from -> to of every slab.  A warp moves 4 KB at a time (16 bytes a
 * lane, eight loads in flight); pages of other sizes or alignment go by bytes. */
#define PK_COPY 4096u
__device__ void pk_copy_pages(const pulsar_kv_pool &P, const int32_t *from, const int32_t *to, uint32_t step,
                              uint32_t n, uint32_t block, uint32_t blocks, uint32_t *err) {
    const uint32_t lane = threadIdx.x & 31u;
    const uint32_t warps = blocks * (blockDim.x >> 5);
    const uint64_t per = (P.page_bytes + PK_COPY - 1) / PK_COPY;
    const uint64_t all = per * P.n_slab * n;
    const bool wide = (((uintptr_t)P.data | P.slab_stride | P.page_bytes) & 15u) == 0;
    for (uint64_t u = block * (blockDim.x >> 5) + (threadIdx.x >> 5); u < all; u += warps) {
        uint64_t part, ps;
        if (all >> 32) {
            part = u % per;
            ps = u / per;
        } else {
            part = (uint32_t)u % (uint32_t)per;
            ps = (uint32_t)u / (uint32_t)per;
        }
        const uint32_t slab = (uint32_t)(ps >> 32 ? ps % P.n_slab : (uint32_t)ps % P.n_slab);
        const uint32_t pr = (uint32_t)(ps >> 32 ? ps / P.n_slab : (uint32_t)ps / P.n_slab);
        const uint32_t a = (uint32_t)from[pr * step], b = (uint32_t)to[pr * step];
        if (a >= P.n_pages || b >= P.n_pages) {
            if (lane == 0) atomicOr(err, PULSAR_KV_ERR_PAGE);
            continue;
        }
        const uint8_t *x = (const uint8_t *)P.data + slab * P.slab_stride + a * P.page_bytes;
        uint8_t *y = (uint8_t *)P.data + slab * P.slab_stride + b * P.page_bytes;
        const uint64_t o0 = part * PK_COPY, left = P.page_bytes - o0;
        const uint32_t m = left < PK_COPY ? (uint32_t)left : PK_COPY;
        if (wide) {
            uint4 v[PK_COPY / 512];
#pragma unroll
            for (uint32_t k = 0; k < PK_COPY / 512; k++) {
                const uint32_t o = (k * 32 + lane) * 16;
                if (o < m) v[k] = __ldcs((const uint4 *)(x + o0 + o));
            }
#pragma unroll
            for (uint32_t k = 0; k < PK_COPY / 512; k++) {
                const uint32_t o = (k * 32 + lane) * 16;
                if (o < m) *(uint4 *)(y + o0 + o) = v[k];
            }
        } else {
            for (uint32_t o = lane; o < m; o += 32) y[o0 + o] = x[o0 + o];
        }
    }
}

/* Block `block` of `blocks` rewrites its part of the tables, up to
 * PK_FORK_COLS columns at a time (one, while there are CTAs enough): it reads
 * its columns of every source row into shared memory before it writes any
 * row, so rows may trade places without a second buffer.  The page copies
 * read live pages and write pages that were free: they and the tables do not
 * touch, nor do the copies among themselves. */
__device__ void pk_fork_tables(const pulsar_kv_pool &P, const pk_fork_ws &w, const int32_t *dst, const int32_t *src,
                               uint32_t n, uint32_t block, uint32_t blocks, int32_t *stage, uint32_t *err) {
    if (block == 0)
        for (uint32_t i = threadIdx.x; i < n; i += blockDim.x) P.len[dst[i]] = (int32_t)w.now[i];
    const uint32_t wide = w.head[2], even = pk_ceil(wide, blocks);
    const uint32_t cols = even < 1 ? 1 : even < PK_FORK_COLS ? even : PK_FORK_COLS;
    for (uint32_t c0 = block * cols; c0 < wide; c0 += blocks * cols) {
        for (uint32_t u = threadIdx.x; u < n * cols; u += blockDim.x) {
            const uint32_t i = u / cols, c = c0 + u % cols;
            const int32_t s = src[i], d = dst[i], copy = w.fresh[i];
            const uint32_t now = w.now[i], was = w.was[i];
            const bool holds = s != d && c < pk_ceil(now, P.page_size), held = s != d && c < pk_ceil(was, P.page_size);
            int32_t page = -1, old = -1;
            if (holds) page = copy >= 0 && c == now / P.page_size ? copy : P.table[s * P.table_stride + c];
            if (held) old = P.table[d * P.table_stride + c];
            if (holds) {
                if ((uint32_t)page >= P.n_pages) atomicOr(err, PULSAR_KV_ERR_PAGE);
                else atomicAdd(&P.refs[page], 1);
            }
            if (held) {
                if ((uint32_t)old >= P.n_pages) atomicOr(err, PULSAR_KV_ERR_PAGE);
                else atomicSub(&P.refs[old], 1);
            }
            stage[u] = page;
        }
        __syncthreads();
        for (uint32_t u = threadIdx.x; u < n * cols; u += blockDim.x) {
            const uint32_t i = u / cols, c = c0 + u % cols;
            const uint32_t now = w.now[i], was = w.was[i];
            if (src[i] != dst[i] && c < pk_ceil(was > now ? was : now, P.page_size))
                P.table[dst[i] * P.table_stride + c] = stage[u];
        }
        __syncthreads();
    }
}

/* the first table_blocks CTAs do the tables, the others the copies */
__global__ void __launch_bounds__(256) pk_fork_apply_kernel(pulsar_kv_pool P, const int32_t *dst, const int32_t *src,
                                                            uint32_t n, uint32_t table_blocks, const void *wsp,
                                                            uint32_t *err) {
    extern __shared__ int32_t stage[]; /* [n][PK_FORK_COLS] */
    const pk_fork_ws w = pk_fork_layout((void *)wsp, P.n_rows, n);
    pk_enter();
    if (!w.head[0]) return;
    if (blockIdx.x >= table_blocks)
        pk_copy_pages(P, w.pair, w.pair + 1, 2, w.head[1], blockIdx.x - table_blocks, gridDim.x - table_blocks, err);
    else
        pk_fork_tables(P, w, dst, src, n, blockIdx.x, table_blocks, stage, err);
}

/* A small fork in one launch: a cluster, whose first CTA plans, and which then
 * does both: it saves the host a launch and does the copies and tables slower.
 * So it takes up to 32 rows, 512 table entries and 512 KB of copies.  Measured
 * with a growth behind it, in a stream, one launch against two, us: 8 rows of
 * 64 pages 10.1 / 12.8 without copies, 11.5 / 12.7 with 512 KB, 12.9 / 12.7 with 1 MB;
 * 32 rows of 16 pages 10.2 / 12.8, 12.2 / 12.8, 13.3 / 12.6; 1024 entries and 512 KB:
 * 8 rows 14.8 / 13.0, 32 rows 13.3 / 12.9; 2048 entries 16.0 / 12.7; 256 rows of 8 pages
 * (in a graph, the fork alone) 21.1 / 8.8. */
#define PK_CLUSTER 8
#define PK_SMALL_ROWS 32u
#define PK_SMALL_ENTRIES 512u
#define PK_SMALL_BYTES (512u << 10)
static_assert(4 * PK_MARKS + sizeof(pk_scan) + 64 + PK_SMALL_ROWS * PK_FORK_COLS * 4 <= 48 * 1024,
              "a small fork needs no more shared memory than any kernel may have");
__global__ void __cluster_dims__(PK_CLUSTER, 1, 1) __launch_bounds__(512)
    pk_fork_small_kernel(pulsar_kv_pool P, const int32_t *dst, const int32_t *src, uint32_t n, int32_t *status,
                         void *wsp, uint32_t *err) {
    extern __shared__ int32_t stage[]; /* [n][PK_FORK_COLS] */
    const pk_fork_ws w = pk_fork_layout(wsp, P.n_rows, n);
    pk_enter();
    if (blockIdx.x == 0) pk_fork_plan(P, dst, src, n, status, wsp);
    asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
    if (!w.head[0]) return;
    pk_fork_tables(P, w, dst, src, n, blockIdx.x, PK_CLUSTER, stage, err);
    pk_copy_pages(P, w.pair, w.pair + 1, 2, w.head[1], blockIdx.x, PK_CLUSTER, err);
}

/* -------------------------------------------------------------- compaction */

/* ws: u32 head[4] (moves, live pages), from[n_pages / 2 + 1], to[..], map[n_pages] */
__global__ void __launch_bounds__(PK_PLAN) pk_compact_plan_kernel(pulsar_kv_pool P, int32_t *status, uint32_t *ws) {
    __shared__ pk_scan scan;
    const uint32_t half = P.n_pages / 2 + 1;
    uint32_t *head = ws;
    int32_t *from = (int32_t *)ws + 4, *to = from + half, *map = to + half;
    pk_enter();
    const auto none = [](uint32_t) { return 0u; };
    const auto every = [](uint32_t total) { return total; };
    const uint32_t live = pk_choose(P.refs, 0, P.n_pages, true, scan, none, [](uint32_t, uint32_t) {});
    const uint32_t moves = pk_choose(P.refs, 0, live, false, scan, every,
                                     [&](uint32_t page, uint32_t rank) { to[rank] = (int32_t)page; });
    for (uint32_t p = live + threadIdx.x; p < P.n_pages; p += PK_PLAN) map[p] = -1; /* but for the pages that move */
    __syncthreads();
    pk_choose(P.refs, live, P.n_pages, true, scan, every, [&](uint32_t page, uint32_t rank) {
        from[rank] = (int32_t)page;
        map[page] = to[rank];
    });
    if (threadIdx.x == 0) {
        head[0] = moves;
        head[1] = live;
        *(int4 *)status = make_int4(PULSAR_KV_OK, (int32_t)moves, (int32_t)live, 0);
    }
}

__global__ void __launch_bounds__(256) pk_compact_apply_kernel(pulsar_kv_pool P, uint32_t table_blocks,
                                                               const uint32_t *ws, uint32_t *err) {
    pk_enter();
    const uint32_t half = P.n_pages / 2 + 1, moves = ws[0], live = ws[1];
    const int32_t *from = (const int32_t *)ws + 4, *to = from + half, *map = to + half;
    if (blockIdx.x >= table_blocks) {
        const uint32_t block = blockIdx.x - table_blocks, blocks = gridDim.x - table_blocks;
        for (uint32_t m = block * blockDim.x + threadIdx.x; m < moves; m += blocks * blockDim.x) {
            P.refs[to[m]] = P.refs[from[m]];
            P.refs[from[m]] = 0;
        }
        pk_copy_pages(P, from, to, 1, moves, block, blocks, err);
        return;
    }
    if (!moves) return;
    const uint32_t warps = table_blocks * (blockDim.x >> 5), lane = threadIdx.x & 31u;
    const uint32_t cap = P.max_pages * P.page_size;
    for (uint32_t r = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5); r < P.n_rows; r += warps) {
        int32_t len = P.len[r];
        if (len < 0 || (uint32_t)len > cap) {
            if (lane == 0) atomicOr(err, PULSAR_KV_ERR_SPAN);
            len = len < 0 ? 0 : (int32_t)cap;
        }
        int32_t *row = P.table + r * P.table_stride;
        for (uint32_t c = lane; c < pk_ceil(len, P.page_size); c += 32) {
            const int32_t e = row[c];
            if ((uint32_t)e >= P.n_pages) atomicOr(err, PULSAR_KV_ERR_PAGE);
            else if ((uint32_t)e >= live) {
                const int32_t m = map[e];
                if (m >= 0) row[c] = m;
                else atomicOr(err, PULSAR_KV_ERR_PAGE); /* a page that no reference count holds */
            }
        }
    }
}

/* -------------------------------------------------------------------- host */

static const char *pk_pool_fault(const pulsar_kv_pool *p) {
    if (!p || !p->table || !p->len || !p->refs) return "kv pool: null descriptor, table, lengths or counts";
    if (!p->n_rows || !p->max_pages || !p->n_pages || !p->page_size) return "kv pool: a zero size";
    if (p->n_rows > 0x3fffffffu || p->n_pages > 0x3fffffffu || (uint64_t)p->max_pages * p->page_size > 0x7fffffffull)
        return "kv pool: too many rows or pages, or rows above 2^31 - 1 tokens";
    if (p->table_stride < p->max_pages) return "kv pool: table rows overlap";
    if (p->n_slab && (!p->data || !p->page_bytes)) return "kv pool: slabs without bytes";
    return nullptr;
}

extern "C" size_t pulsar_kv_pool_workspace(const pulsar_kv_pool *p, uint32_t n) {
    if (pk_pool_fault(p)) return 0;
    const uint64_t fork = 4ull + 2ull * p->n_rows + 6ull * n;
    const uint64_t compact = 4ull + 2ull * (p->n_pages / 2 + 1) + p->n_pages;
    return 4ull * (fork > compact ? fork : compact);
}

/* what the three entries have in common; 1 = go on */
static int pk_pool_check(const pulsar_kv_pool *p, const int32_t *status, const void *ws, size_t ws_bytes, uint32_t n) {
    const char *f = pk_pool_fault(p);
    if (f) return pk_refuse(f);
    if (!status || !ws || (((uintptr_t)ws | (uintptr_t)status) & 15u))
        return pk_refuse("kv pool: status and workspace are there and aligned to 16 bytes");
    if (ws_bytes < pulsar_kv_pool_workspace(p, n)) return pk_refuse("kv pool: workspace too small");
    return pk_err_word() ? 1 : pk_refuse("kv pool: no error word on this device");
}

extern "C" int pulsar_kv_grow(const pulsar_kv_pool *p, const int32_t *rows, const int32_t *n_new, uint32_t n,
                              int32_t *status, void *ws, size_t ws_bytes, void *stream) {
    if (!pk_pool_check(p, status, ws, ws_bytes, n)) return 0;
    if (!n_new || !n || n > p->n_rows) return pk_refuse("kv grow: between 1 and n_rows rows, each with a count");
    return pm_ok(pk_launch(pk_grow_kernel, 1, PK_PLAN, 0, pk_stream(stream), *p, rows, n_new, n, status, (uint32_t *)ws),
                 "kv grow launch");
}

extern "C" int pulsar_kv_fork(const pulsar_kv_pool *p, const int32_t *dst, const int32_t *src, uint32_t n,
                              int32_t *status, void *ws, size_t ws_bytes, void *stream) {
    static uint64_t done = 0;
    if (!pk_pool_check(p, status, ws, ws_bytes, n)) return 0;
    if (!dst || !src || !n || n > p->n_rows || n > PULSAR_KV_MAX_FORK)
        return pk_refuse("kv fork: between 1 and min(n_rows, 4096) rows, each with a source");
    const uint32_t smem = n * PK_FORK_COLS * 4u;
    const cudaStream_t st = pk_stream(stream);
    if (n <= PK_SMALL_ROWS && (uint64_t)n * p->max_pages <= PK_SMALL_ENTRIES &&
        p->page_bytes <= PK_SMALL_BYTES && (uint64_t)n * p->n_slab * p->page_bytes <= PK_SMALL_BYTES)
        return pm_ok(pk_launch(pk_fork_small_kernel, PK_CLUSTER, 512, smem, st, *p, dst, src, n, status, ws, pk_err_word()),
                     "kv fork launch");
    if (!pm_smem_attr(pk_fork_apply_kernel, smem, &done)) return 0;
    if (!pm_ok(pk_launch(pk_fork_plan_kernel, 1, PK_PLAN, 0, st, *p, dst, src, n, status, ws), "kv fork plan launch"))
        return 0;
    const uint32_t sms = pk_sm_count();
    const uint32_t tb = p->max_pages < 2 * sms ? p->max_pages : 2 * sms;
    const uint32_t cb = p->n_slab ? 4 * sms : 0;
    return pm_ok(pk_launch(pk_fork_apply_kernel, tb + cb, 256, smem, st, *p, dst, src, n, tb, (const void *)ws,
                           pk_err_word()),
                 "kv fork launch");
}

extern "C" int pulsar_kv_compact(const pulsar_kv_pool *p, int32_t *status, void *ws, size_t ws_bytes, void *stream) {
    if (!pk_pool_check(p, status, ws, ws_bytes, 0)) return 0;
    const cudaStream_t st = pk_stream(stream);
    if (!pm_ok(pk_launch(pk_compact_plan_kernel, 1, PK_PLAN, 0, st, *p, status, (uint32_t *)ws), "kv compact plan launch"))
        return 0;
    const uint32_t sms = pk_sm_count();
    uint32_t tb = (p->n_rows + 7) / 8;
    if (tb > 2 * sms) tb = 2 * sms;
    return pm_ok(pk_launch(pk_compact_apply_kernel, tb + 4 * sms, 256, 0, st, *p, tb, (const uint32_t *)ws,
                           pk_err_word()),
                 "kv compact launch");
}
