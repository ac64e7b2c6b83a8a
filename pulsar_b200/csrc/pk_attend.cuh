/* pk_attend.cuh - attention of new tokens over a paged cache.
 *
 *   o = sum_j e^(s_j - m) v_j / (sum_j e^(s_j - m) + e^(sink - m)),  s_j = scale q.k_j
 *
 * The cache's bytes are the bound: each visible key and value is read once
 * for up to 16 query heads that share it, and 2 x 16 x head_dim multiply-adds
 * per key are far below what the warp matrix instructions do in that time.
 * Measured: 256 sequences of up to 4096 keys, bf16, 32 / 8 heads of 128:
 * 389 to 410 us, 6.4 to 6.7 TB/s (a copy's rate); 4 of up to 131071 in e4m3,
 * 64 / 8 heads: 113 to 128 us, 5.0 to 5.7 TB/s (the loads alone 105 us); one
 * of 100 keys: 7.1 us, all of it latency.
 *
 * Work.  The query rows of a key head are its n_q * (n_head / n_kv) (token,
 * head) pairs; a tile is HEADS of them.  All (sequence, key head, tile)
 * segments lie one behind the other on a line, counted in chunks of CK keys,
 * and the workers take equal slices of it: no length, batch or head count
 * leaves SMs idle, and the host needs no lengths (it only sees to it that the
 * line stays below 2^32 chunks).  Long segments: a worker is a CTA, whose four
 * warps take the chunks of its slice in turn, each with its own running
 * maximum, sum and output tile, and meet at a segment's end; a segment that a
 * slice cuts is joined through the workspace by the CTA that arrives last, in
 * the order of the slices (a fixed order: the same call gives the same bits),
 * 32 parts at a time.  Few segments are cut evenly among CTAs of their own (8
 * sequences of up to 4001 keys: 16.9 us against 21.9 with slices across
 * segments).  Many short segments (8 chunks or fewer on average, more of them
 * than CTAs): a worker is a warp, which takes whole segments and meets nobody
 * (64 windows of 128 keys, 8 key heads: 13.6 us against 19.0).
 *
 * Each warp fills a ring of its own with 16-byte asynchronous copies: no
 * barrier in the stream, and keys out of the span are filled with zeros, so
 * that stale bytes never meet the arithmetic.
 *
 * Products.  q and the probabilities p are taken in 16-bit parts (leading 16
 * bits, the next, ...), keys and values as they are, sums in f32.
 *   R = 1 (up to 8 query rows): the 16 rows of a matrix tile are 8 query rows
 *   twice, the leading part in row g and the next in row g + 8: the tile is
 *   16 rows high anyway, so the second part costs nothing.
 *   R = 2: 16 query rows a tile, one product per part.
 * Two f16 parts hold 22 bits (q's rows and p are first scaled by a power of
 * two, so that nothing of weight falls among f16's subnormals: weights are lost
 * below 2^-32 of the row's largest), two bf16 parts 16, which is more than
 * their bf16 results have; QP = 3 adds a third where a bf16 cache meets wider q,
 * so that f32 results are f32 results.  QP = 1: q has the cache's type or fewer bits. */
#pragma once
#include "pk_common.h"

#define PK_WARPS 4
/* keys per chunk, by the bytes of a row in shared memory: 32 while their keys fit 8 KB */
#define PK_CK(row_bytes) ((row_bytes) > 256 ? 16 : 32)
#define PK_SM_BYTES (228 * 1024) /* shared memory of an SM; each CTA takes 1 KB more than it asks for */
#define PK_GROUP 32u          /* parts joined at a time */
#define PK_MAX_WORKERS 1024u  /* 2 x 2 counters of each fill PULSAR_KV_WS_ZEROED / 2 */
#define PK_LOG2E 1.4426950408889634f

/* q_type is read at run time (it costs a few loads a segment) */
struct pk_attend_job {
    pulsar_kv_desc D;
    pulsar_kv_attend_args A;
    uint32_t group;      /* query heads per key head */
    uint32_t rows;       /* query rows per key head: n_q * group */
    uint32_t tiles;      /* tiles per key head */
    uint32_t segs;       /* segments per sequence: n_kv * tiles */
    int32_t page_shift;  /* log2(page_size), or -1 */
    uint32_t pairs;      /* q's rows are aligned for loads of two values */
    uint32_t least;      /* least chunks in a slice, where segments are long */
    uint32_t *counters;  /* [2][2 * PK_MAX_WORKERS] */
    float *parts;        /* [workers][2] parts of HEADS * (DP + 2) floats */
    uint32_t *err;
};

template <uint32_t CT, int DP, int R, int QP>
struct pk_shape {
    static constexpr int ELT = CT == PULSAR_TYPE_E4M3 ? 1 : 2;
    static constexpr int ROW = (DP == 96 ? 128 : DP) * ELT; /* bytes of a key in shared memory: whole 64s or 128s */
    static constexpr int UNITS = ROW / 16;
    static constexpr int CK = PK_CK(ROW);
    /* A stage of the ring is a chunk's keys and values; at rows of 256 bytes or more its keys or its values,
     * which take turns: stages stay at 4 to 8 KB, a warp's ring at 18 to 24. */
    static constexpr bool SPLIT = ROW >= 256;
    static constexpr int STAGE = (SPLIT ? 1 : 2) * CK * ROW;
    static constexpr int STAGES = STAGE <= 4096 ? 6 : 3;
    static constexpr int RING = STAGES * STAGE;           /* per warp */
    static constexpr bool QSM = DP > 128;                 /* q's parts wait in shared memory, not registers */
    static constexpr int QW = R == 1 ? 2 * QP : 4 * QP;   /* their words per lane and k-step */
    static constexpr int XROW = 64 + 4;                   /* floats of 64 columns in the warps' meeting; no bank conflicts */
    static constexpr int MEET = PK_WARPS * 8 * XROW * 4, QALL = QSM ? DP / 16 * QW * 128 : 0;
    static constexpr int SIDE = MEET > QALL ? MEET : QALL; /* bytes beside the rings: both, at different times */
    static constexpr int OCC = 2 * (PK_WARPS * RING + SIDE + 4096) <= PK_SM_BYTES ? 2 : 1; /* CTAs that an SM holds */
};

__device__ __forceinline__ uint32_t pk_saddr(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }

/* 16 bytes global -> shared, or 16 zero bytes */
__device__ __forceinline__ void pk_cp16(uint32_t dst, const void *src, bool real) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(real ? 16 : 0) : "memory");
}
__device__ __forceinline__ void pk_cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void pk_cp_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ void pk_ldm4(uint32_t *r, uint32_t a) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(a)
                 : "memory");
}
__device__ __forceinline__ void pk_ldm4t(uint32_t *r, uint32_t a) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(a)
                 : "memory");
}

template <bool BF>
__device__ __forceinline__ void pk_mma(float *c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                       uint32_t b1) {
    if constexpr (BF)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
                     "{%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
                     "{%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

/* x, y rounded to 16 bits and packed, x low; x, y become what is left (SAFE:
 * 0 where the value is not finite) */
template <bool BF, bool SAFE>
__device__ __forceinline__ uint32_t pk_split(float &x, float &y) {
    uint32_t r;
    float a, b;
    if constexpr (BF) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
        r = *(const uint32_t *)&h;
        a = x - __low2float(h);
        b = y - __high2float(h);
    } else {
        const __half2 h = __floats2half2_rn(x, y);
        r = *(const uint32_t *)&h;
        a = x - __low2float(h);
        b = y - __high2float(h);
    }
    x = !SAFE || isfinite(x) ? a : 0.0f;
    y = !SAFE || isfinite(y) ? b : 0.0f;
    return r;
}

/* two e4m3 bytes (low half of v) -> f16x2, exact */
__device__ __forceinline__ uint32_t pk_e4m3x2(uint32_t v) {
    uint32_t r;
    asm("{\n\t.reg .b16 t;\n\tcvt.u16.u32 t, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, t;\n\t}" : "=r"(r) : "r"(v));
    return r;
}

/* 2^x: the hardware's, within 2 ulp; below 2^-126 it is 0 */
__device__ __forceinline__ float pk_exp2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

/* a warp zeroes the rows of CK values in shared memory that hold an infinity or
 * NaN; returns which (of those that are there) */
template <uint32_t CT, int CK, int ROW>
__device__ __noinline__ uint32_t pk_take_odd(uint32_t rows, uint32_t there) {
    constexpr uint32_t ONES = CT == PULSAR_TYPE_E4M3 ? 0x7f7f7f7fu : CT == PULSAR_TYPE_BF16 ? 0x7f807f80u : 0x7c007c00u;
    const uint32_t lane = threadIdx.x & 31u, at = rows + lane % CK * ROW;
    uint32_t hit = 0;
#pragma unroll 1
    for (uint32_t u = 0; u < ROW / 16; u++) {
        const uint32_t x = at + (u ^ (lane & (ROW >= 128 ? 7u : 3u))) * 16;
        uint32_t v[4];
        asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(x) : "memory");
#pragma unroll
        for (int e = 0; e < 4; e++)
            hit |= CT == PULSAR_TYPE_E4M3 ? __vcmpeq4(v[e] & ONES, ONES) : __vcmpeq2(v[e] & ONES, ONES);
    }
    const uint32_t odd = __ballot_sync(~0u, hit && (there >> lane & 1u));
    if (odd >> lane & 1u)
#pragma unroll 1
        for (uint32_t u = 0; u < ROW / 16; u++)
            asm volatile("st.shared.v4.u32 [%0], {%1,%1,%1,%1};" ::"r"(at + u * 16), "r"(0) : "memory");
    __syncwarp();
    return CK == 32 ? odd : odd & ((1u << (CK & 31)) - 1u);
}

/* the leading sum, plus the rest where the rest is a number: a key or value
 * of +-inf makes the lower parts' products NaN, the leading one's +-inf */
__device__ __forceinline__ float pk_fold(float lead, float rest) { return isfinite(rest) ? lead + rest : lead; }

/* ------------------------------------------------------------ the line */

#define PK_CACHED 256u /* sequences whose length and table row are kept in shared memory */

/* what a sequence's length, window and table row say */
struct pk_row {
    int32_t len, c0, n; /* keys; first chunk; chunks (at least 1) */
    const int32_t *table;
};

/* (keys, table row) of sequence b, checked */
__device__ __forceinline__ int2 pk_len_of(const pk_attend_job &J, uint32_t b, bool tell) {
    int32_t row = J.A.seq ? J.A.seq[b] : (int32_t)b, len = J.A.lens[b];
    const int32_t cap = (int32_t)(J.D.max_pages * J.D.page_size);
    uint32_t bad = 0;
    if (row < 0 || len < 0) len = 0;
    if (row >= 0 && (uint32_t)row >= J.D.n_rows) {
        bad = PULSAR_KV_ERR_ROW;
        len = 0;
    }
    if (len > cap) {
        bad |= PULSAR_KV_ERR_SPAN;
        len = cap;
    }
    if (bad && tell) atomicOr(J.err, bad);
    return make_int2(len, len ? row : 0);
}

template <int CK>
__device__ __forceinline__ pk_row pk_row_of(const pk_attend_job &J, int2 lr) {
    pk_row r;
    r.len = lr.x;
    const int64_t lo = J.A.window ? (int64_t)lr.x - (J.A.n_q - 1) - J.A.window : 0;
    r.c0 = lo > 0 ? (int32_t)lo / CK : 0;
    const int32_t end = (int32_t)(((uint32_t)lr.x + CK - 1) / CK);
    r.n = end > r.c0 ? end - r.c0 : 1;
    r.table = J.D.table + (uint64_t)lr.y * J.D.table_stride;
    return r;
}

/* keys [lo, hi) that token i of a sequence of len keys sees */
__device__ __forceinline__ void pk_span(const pk_attend_job &J, int32_t len, uint32_t i, int32_t &lo, int32_t &hi) {
    const int64_t h = (int64_t)len - (J.A.n_q - 1 - i);
    hi = h > 0 ? (int32_t)h : 0;
    lo = J.A.window && (uint32_t)hi > J.A.window ? hi - (int32_t)J.A.window : 0;
}

/* a warp's place on the line: chunk pos of tile `tile` of key head hk of
 * sequence b, and the keys that the tile's rows see between them */
template <int CK, int HEADS>
struct pk_cursor {
    uint32_t b, hk, tile;
    int32_t pos, lo, hi;
    uint64_t head; /* byte offset of the key head */
    pk_row row;
    __device__ __forceinline__ void enter(const pk_attend_job &J) {
        head = hk * J.D.head_stride * (J.D.dtype == PULSAR_TYPE_E4M3 ? 1 : 2);
        uint32_t i0 = 0, i1 = 0;
        if (J.A.n_q > 1) {
            const uint32_t v0 = tile * HEADS, v1 = v0 + HEADS < J.rows ? v0 + HEADS - 1 : J.rows - 1;
            i0 = v0 / J.group;
            i1 = v1 / J.group;
        }
        int32_t x;
        pk_span(J, row.len, i0, lo, x);
        pk_span(J, row.len, i1, x, hi);
    }
    __device__ __forceinline__ void step(const pk_attend_job &J, const int2 *cached, int32_t by) {
        pos += by;
        if (pos < row.n) return;
        do {
            pos -= row.n;
            if (++tile == J.tiles) {
                tile = 0;
                if (++hk == J.D.n_kv) {
                    hk = 0;
                    if (++b >= J.A.n_rows) return; /* past the line's end: not used again */
                    row = pk_row_of<CK>(J, J.A.n_rows <= PK_CACHED ? cached[b] : pk_len_of(J, b, false));
                }
            }
        } while (pos >= row.n);
        enter(J);
    }
};

/* chunks of sequence r in one segment, in units of `per` */
template <int CK>
__device__ __forceinline__ uint32_t pk_units(const pk_attend_job &J, const int2 *cached, uint32_t r, uint32_t per) {
    const uint32_t n = (uint32_t)pk_row_of<CK>(J, J.A.n_rows <= PK_CACHED ? cached[r] : pk_len_of(J, r, false)).n;
    return per == 1 ? n : (n + per - 1) / per;
}

/* inclusive prefix over the CTA's threads -> upto[]; returns their sum */
__device__ __forceinline__ uint32_t pk_prefix(uint32_t mine, uint32_t *upto) {
    const uint32_t lane = threadIdx.x & 31u, w = threadIdx.x >> 5;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t y = __shfl_up_sync(~0u, mine, o);
        if (lane >= o) mine += y;
    }
    if (lane == 31) upto[PK_WARPS * 32 + w] = mine;
    __syncthreads();
    uint32_t all = 0;
#pragma unroll
    for (uint32_t k = 0; k < PK_WARPS; k++) {
        const uint32_t x = upto[PK_WARPS * 32 + k];
        if (k < w) mine += x;
        all += x;
    }
    upto[threadIdx.x] = mine;
    __syncthreads();
    return all;
}

/* a warp finds the sequence that holds unit `at` of the line: upto[t] are the
 * units of one segment each up to the rows of thread t (`run` rows a
 * thread), to which every segment adds `extra`; before = the units of all
 * earlier rows without that */
template <int CK>
__device__ __forceinline__ uint32_t pk_locate(const pk_attend_job &J, const int2 *cached, const uint32_t *upto,
                                              uint32_t run, uint32_t per, uint32_t extra, uint32_t at, uint32_t *before) {
    const uint32_t lane = threadIdx.x & 31u;
    uint32_t t = 0;
#pragma unroll
    for (uint32_t k = 0; k < PK_WARPS; k++) {
        const uint32_t x = k * 32 + lane, rows = (x + 1) * run < J.A.n_rows ? (x + 1) * run : J.A.n_rows;
        t += __popc(__ballot_sync(~0u, (upto[x] + extra * rows) * J.segs <= at));
    }
    uint32_t sum = t ? upto[t - 1] : 0;
    if (run == 1) {
        *before = sum;
        return t;
    }
    for (uint32_t r0 = t * run;; r0 += 32) {
        const uint32_t r = r0 + lane;
        const bool in = r < (t + 1) * run && r < J.A.n_rows;
        const uint32_t n = in ? pk_units<CK>(J, cached, r, per) : 0;
        uint32_t x = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t y = __shfl_up_sync(~0u, x, o);
            if (lane >= o) x += y;
        }
        const uint32_t hit = __ballot_sync(~0u, in && (sum + x + extra * (r + 1)) * J.segs > at);
        if (hit || r0 + 32 >= (t + 1) * run || r0 + 32 >= J.A.n_rows) {
            const uint32_t k = hit ? __ffs(hit) - 1 : 0;
            *before = sum + __shfl_sync(~0u, x - n, k);
            return r0 + k;
        }
        sum += __shfl_sync(~0u, x, 31);
    }
}

/* ------------------------------------------------------------ q, results */

/* N k-steps of a lane's q values of one row: runs x[n][0..1], x[n][2..3] at
 * 16 (k0 + n) + d0 and d1 further on.  No load waits for another: the type is
 * settled outside the loop, and a row or column that is not there reads one
 * that is.  pairs: q is aligned for loads of two. */
template <uint32_t QT, int N>
__device__ __forceinline__ void pk_q_load(const pk_attend_job &J, uint64_t at, uint32_t k0, uint32_t d0, uint32_t d1,
                                          float (*x)[4]) {
    typedef typename pk_type<QT>::t T;
    struct __align__(2 * sizeof(T)) two {
        T v[2];
    };
    const T *q = (const T *)J.A.q + at + d0;
    if (J.pairs) {
#pragma unroll
        for (int n = 0; n < N; n++)
#pragma unroll
            for (int e = 0; e < 4; e += 2) {
                const uint32_t d = (k0 + n) * 16u < J.D.head_dim ? (k0 + n) * 16u : 0u;
                const two r = *(const two *)(q + d + (e ? d1 : 0));
                x[n][e] = pk_type<QT>::get(r.v[0]);
                x[n][e + 1] = pk_type<QT>::get(r.v[1]);
            }
    } else {
#pragma unroll
        for (int n = 0; n < N; n++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const uint32_t d = (k0 + n) * 16u < J.D.head_dim ? (k0 + n) * 16u : 0u;
                x[n][e] = pk_type<QT>::get(q[d + (e & 2 ? d1 : 0) + (e & 1)]);
            }
    }
}

/* what query row v's output sums are multiplied with, given its maximum
 * (log2 units) and sum; writes its lse */
__device__ __forceinline__ float pk_finish(const pk_attend_job &J, uint32_t b, int32_t len, uint32_t hk, uint32_t v,
                                           float top, float sum, bool tell = true) {
    const uint32_t i = v / J.group, h = hk * J.group + v % J.group;
    int32_t lo, hi;
    pk_span(J, len, i, lo, hi);
    const bool empty = hi <= lo;
    float by = 1.0f;
    if (J.A.sinks && !empty) {
        const float sink = __ldg(J.A.sinks + h) * PK_LOG2E, t = fmaxf(top, sink);
        if (t != -INFINITY) {
            by = pk_exp2(top - t);
            sum = sum * by + pk_exp2(sink - t);
            top = t;
        }
    }
    if (J.A.lse && tell)
        J.A.lse[((uint64_t)b * J.A.n_q + i) * J.A.n_head + h] =
            empty ? -INFINITY : logf(sum) + top * 0.6931471805599453f;
    by = sum == 0.0f ? 0.0f : by / sum;
    return J.D.v_scale ? by * __ldg(J.D.v_scale + hk) : by;
}

/* N neighbouring columns of query row v's output */
template <int N>
__device__ __forceinline__ void pk_put(const pk_attend_job &J, uint32_t b, uint32_t hk, uint32_t v, uint32_t col,
                                       const float *y) {
    const uint64_t tok = (uint64_t)b * J.A.n_q + v / J.group;
    const uint64_t at = tok * J.A.out_stride + (uint64_t)(hk * J.group + v % J.group) * J.D.head_dim + col;
    if (J.A.q_type == PULSAR_TYPE_F32) {
        float *d = (float *)J.A.out + at;
#pragma unroll
        for (int e = 0; e < N; e++) d[e] = y[e];
    } else if (J.A.q_type == PULSAR_TYPE_BF16) {
        __nv_bfloat16 *d = (__nv_bfloat16 *)J.A.out + at;
#pragma unroll
        for (int e = 0; e < N; e++) d[e] = __float2bfloat16_rn(y[e]);
    } else {
        __half *d = (__half *)J.A.out + at;
#pragma unroll
        for (int e = 0; e < N; e++) d[e] = __float2half_rn(y[e]);
    }
}

/* ------------------------------------------------------------ joins */

/* a segment that several workers share */
struct pk_joint {
    uint32_t b, hk, v0, w0, w1;
    int32_t len;
    bool inside; /* it begins inside w0's slice: w0's part is in slot 2 w0 + 1, others' (w) in 2 w */
    __device__ __forceinline__ uint32_t slot(uint32_t k) const { return 2 * (w0 + k) + (k == 0 && inside); }
};

/* one more part of a counter's `of` is in the workspace; true for the CTA
 * whose part completes them (which leaves the counter at zero).  Every thread
 * of the CTA calls it. */
__device__ __forceinline__ bool pk_arrive(uint32_t *counter, uint32_t of, uint32_t *last) {
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) {
        *last = atomicAdd(counter, 1u) == of - 1;
        if (*last) *counter = 0;
    }
    __syncthreads();
    const bool yes = *last;
    __threadfence();
    return yes;
}

/* the parts meet PK_GROUP at a time, then the groups */
__device__ __forceinline__ bool pk_joint_arrive(const pk_attend_job &J, const pk_joint &S, uint32_t *last) {
    const uint32_t n = S.w1 - S.w0 + 1, first = (blockIdx.x - S.w0) / PK_GROUP * PK_GROUP;
    return pk_arrive(J.counters + S.slot(first), n - first < PK_GROUP ? n - first : PK_GROUP, last);
}

/* sums of `count` parts (step apart) from `first` on, in their order; done by
 * the CTA that completed them.  The parts come through `room` (PARTS of them
 * at a time) by asynchronous copies, so that one latency serves many. */
template <int DP, int HEADS, int PARTS>
__device__ void pk_join(const pk_attend_job &J, const pk_joint &S, uint32_t first, uint32_t step, uint32_t count,
                        bool final, float (*ml)[2], float *room) {
    constexpr uint32_t FLOATS = HEADS * (DP + 2), THREADS = PK_WARPS * 32;
    constexpr uint32_t RUNS = HEADS * DP / 4;                 /* of four columns */
    constexpr int NX = (RUNS + THREADS - 1) / THREADS;        /* that a thread sums */
    static_assert(PARTS > 0, "a part fits");
    float4 acc[NX];
#pragma unroll
    for (int n = 0; n < NX; n++) acc[n] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (threadIdx.x < HEADS) {
        ml[threadIdx.x][0] = -INFINITY;
        ml[threadIdx.x][1] = 0.0f;
    }
    for (uint32_t k0 = 0; k0 < count; k0 += PARTS) {
        const uint32_t m = count - k0 < PARTS ? count - k0 : PARTS;
        for (uint32_t k = 0; k < m; k++) {
            const float *p = J.parts + S.slot(first + (k0 + k) * step) * (uint64_t)FLOATS;
            for (uint32_t x = threadIdx.x; x < FLOATS / 4; x += THREADS)
                pk_cp16(pk_saddr(room + k * FLOATS + 4 * x), p + 4 * x, true);
        }
        pk_cp_commit();
        pk_cp_wait<0>();
        __syncthreads();
        /* each part's maximum becomes its factor, part 0's sum what is kept of the sums so far */
        if (threadIdx.x < HEADS) {
            float *f = room + 2 * threadIdx.x, old = ml[threadIdx.x][0], top = old, sum;
            for (uint32_t k = 0; k < m; k++) top = fmaxf(top, f[k * FLOATS]);
            const float zero = top == -INFINITY ? 0.0f : top;
            sum = ml[threadIdx.x][1] * pk_exp2(old - zero);
            for (uint32_t k = 0; k < m; k++) {
                const float by = pk_exp2(f[k * FLOATS] - zero);
                sum += by * f[k * FLOATS + 1];
                f[k * FLOATS] = by;
            }
            f[1] = pk_exp2(old - zero);
            ml[threadIdx.x][0] = top;
            ml[threadIdx.x][1] = sum;
        }
        __syncthreads();
#pragma unroll
        for (int n = 0; n < NX; n++) {
            const uint32_t x = n * THREADS + threadIdx.x;
            if (RUNS % THREADS && x >= RUNS) break;
            const float keep = room[2 * (x / (DP / 4)) + 1];
            acc[n].x *= keep;
            acc[n].y *= keep;
            acc[n].z *= keep;
            acc[n].w *= keep;
        }
#pragma unroll 2
        for (uint32_t k = 0; k < m; k++)
#pragma unroll
            for (int n = 0; n < NX; n++) {
                const uint32_t x = n * THREADS + threadIdx.x;
                if (RUNS % THREADS && x >= RUNS) break;
                const float by = room[k * FLOATS + 2 * (x / (DP / 4))];
                const float4 v = *(const float4 *)(room + k * FLOATS + 2 * HEADS + 4 * x);
                acc[n].x += v.x * by;
                acc[n].y += v.y * by;
                acc[n].z += v.z * by;
                acc[n].w += v.w * by;
            }
        __syncthreads();
    }
    if (final) {
        const uint32_t v = S.v0 + threadIdx.x;
        if (threadIdx.x < HEADS && v < J.rows)
            ml[threadIdx.x][0] = pk_finish(J, S.b, S.len, S.hk, v, ml[threadIdx.x][0], ml[threadIdx.x][1]);
        __syncthreads();
    }
#pragma unroll
    for (int n = 0; n < NX; n++) {
        const uint32_t x = n * THREADS + threadIdx.x, head = x / (DP / 4), col = x % (DP / 4) * 4, v = S.v0 + head;
        if (RUNS % THREADS && x >= RUNS) break;
        if (!final) {
            __stcg((float4 *)(J.parts + S.slot(first) * (uint64_t)FLOATS + 2 * HEADS + 4 * x), acc[n]);
        } else if (v < J.rows && col < J.D.head_dim) {
            const float by = ml[head][0], y[4] = {acc[n].x * by, acc[n].y * by, acc[n].z * by, acc[n].w * by};
            pk_put<4>(J, S.b, S.hk, v, col, y);
        }
    }
}

/* the join of a segment by the CTA that completed its group */
template <int DP, int HEADS, int PARTS>
__device__ void pk_joint_finish(const pk_attend_job &J, const pk_joint &S, uint32_t *last, float (*ml)[2], float *room) {
    const uint32_t n = S.w1 - S.w0 + 1, groups = (n + PK_GROUP - 1) / PK_GROUP;
    const uint32_t first = (blockIdx.x - S.w0) / PK_GROUP * PK_GROUP;
    __syncthreads();
    pk_join<DP, HEADS, PARTS>(J, S, first, 1, n - first < PK_GROUP ? n - first : PK_GROUP, groups == 1, ml, room);
    if (groups == 1) return;
    if (threadIdx.x < HEADS)
        __stcg((float2 *)(J.parts + S.slot(first) * (uint64_t)(HEADS * (DP + 2)) + 2 * threadIdx.x),
               make_float2(ml[threadIdx.x][0], ml[threadIdx.x][1]));
    if (pk_arrive(J.counters + 2 * PK_MAX_WORKERS + S.slot(0), groups, last))
        pk_join<DP, HEADS, PARTS>(J, S, 0, PK_GROUP, groups, true, ml, room);
}

/* ------------------------------------------------------------ the kernel */

template <uint32_t CT, int DP, int R, int QP>
__global__ void __launch_bounds__(PK_WARPS * 32, pk_shape<CT, DP, R, QP>::OCC) pk_attend_kernel(const __grid_constant__ pk_attend_job J) {
    typedef pk_shape<CT, DP, R, QP> S;
    constexpr bool BF = CT == PULSAR_TYPE_BF16;
    constexpr bool F8 = CT == PULSAR_TYPE_E4M3;
    constexpr int CK = S::CK, KS = DP / 16, NT = DP / 8, KT = CK / 8;
    constexpr int HEADS = 8 * R;                          /* query rows of a tile; a lane's are R */
    constexpr bool QSM = S::QSM;
    constexpr int QW = S::QW;
    constexpr int PP = QP == 3 ? 3 : 2;                   /* parts of p */
    constexpr int PW = R == 1 ? (PP == 3 ? 6 : 4) : 4 * PP;
    constexpr bool REST = R == 1 ? QP == 3 : QP > 1;      /* lower parts of q have sums of their own */
    constexpr float LIFT = BF ? 0.0f : 7.0f, SLACK = 8.0f; /* see the running maximum below */

    extern __shared__ __align__(128) uint8_t smem[];
    uint8_t *ring = smem + (threadIdx.x >> 5) * S::RING;
    float *side = (float *)(smem + PK_WARPS * S::RING);
    uint32_t *upto = (uint32_t *)side;                    /* in the beginning */
    uint32_t *qsm = (uint32_t *)side;                     /* QSM: [KS][QW / 2][32][2], until a segment's warps meet */
    static_assert((PK_WARPS * 32 + PK_WARPS) * 4 <= S::SIDE, "the line's sums fit");
    __shared__ float wml[PK_WARPS][HEADS][2];             /* each warp's maximum and sum */
    __shared__ float fml[HEADS][2];
    __shared__ uint32_t vmask[PK_WARPS][S::STAGES];       /* keys of a stage that are there */
    __shared__ int2 cached[PK_CACHED];
    __shared__ uint32_t last;

    const uint32_t tid = threadIdx.x, lane = tid & 31u, w = tid >> 5;
    const uint32_t g = lane >> 2, c = lane & 3u;          /* row and column pair of a fragment */

    pk_enter();
    /* ---- the line's length */
    const uint32_t B = J.A.n_rows;
    const uint32_t run = (B + PK_WARPS * 32 - 1) / (PK_WARPS * 32);
    uint32_t mine = 0;
    for (uint32_t r = tid * run; r < (tid + 1) * run && r < B; r++) {
        const int2 lr = pk_len_of(J, r, blockIdx.x == 0);
        if (B <= PK_CACHED) cached[r] = lr;
        mine += (uint32_t)pk_row_of<CK>(J, lr).n;
    }
    /* columns from head_dim to DP stay zero: copies never write them */
    const uint32_t units = J.D.head_dim * S::ELT / 16;
    if (units < S::UNITS)
        for (uint32_t o = tid * 16; o < PK_WARPS * S::RING; o += PK_WARPS * 32 * 16)
            *(uint4 *)(smem + o) = make_uint4(0, 0, 0, 0);
    const uint32_t all = pk_prefix(mine, upto);

    /* ---- the worker's slice of it */
    const uint32_t total = all * J.segs, segs = B * J.segs;
    const bool brief = all <= 8u * B;                     /* 8 chunks a segment or fewer, on average */
    const bool solo = !QSM && brief && segs > gridDim.x;
    /* a warp's slice is cut by cost: beside its chunks a segment costs about three (q, the results) */
    const uint32_t extra = solo ? 3 : 0;
    const uint32_t workers = solo ? gridDim.x * PK_WARPS : gridDim.x, me = solo ? blockIdx.x * PK_WARPS + w : blockIdx.x;
    const uint32_t cost = total + extra * segs;
    uint32_t per = (cost + workers - 1) / workers;
    /* Few segments: each is cut evenly among CTAs of its own, so that no CTA takes parts of two.  That makes
     * slices longer by segs / (CTAs - segs); a second segment in a slice costs its CTA about 14 chunks' time
     * (q, the warps' meeting, the join: 5 us). */
    const bool own = !solo && segs < workers && (uint64_t)per * segs < 14ull * (workers - segs);
    /* a segment of up to 8 chunks is not cut to fill idle SMs: joining it costs more than reading it */
    const uint32_t least = !brief ? J.least : B == 1 ? all : (all + B - 1) / B;
    if (own) per = (total + workers - segs - 1) / (workers - segs);
    if (!solo) per = per < least ? least : (per + PK_WARPS - 1) & ~(PK_WARPS - 1);
    uint32_t lo, hi, in, at, piece = 0, pieces = 1;         /* slice [lo, hi); piece of `pieces` of an own segment */
    pk_cursor<CK, HEADS> cons;
    if (own) {
        __syncthreads();
        mine = 0;
        for (uint32_t r = tid * run; r < (tid + 1) * run && r < B; r++) mine += pk_units<CK>(J, cached, r, per);
        if (me >= pk_prefix(mine, upto) * J.segs) return; /* more CTAs than pieces */
        cons.b = pk_locate<CK>(J, cached, upto, run, per, 0, me, &at);
        cons.row = pk_row_of<CK>(J, B <= PK_CACHED ? cached[cons.b] : pk_len_of(J, cons.b, false));
        pieces = ((uint32_t)cons.row.n + per - 1) / per;
        in = (me - at * J.segs) / pieces;
        piece = me - at * J.segs - in * pieces;
        const uint32_t each = (uint32_t)cons.row.n / pieces, more = (uint32_t)cons.row.n - each * pieces;
        lo = each * piece + (piece < more ? piece : more);
        hi = lo + each + (piece < more);
        cons.pos = (int32_t)lo;
    } else {
        /* where the line position x lies: sequence, segment, chunk; solo: the first segment that begins at or
         * behind it.  Returns the chunk's place on the line. */
        auto place = [&](uint32_t x, uint32_t &b, uint32_t &seg, int32_t &pos) {
            b = pk_locate<CK>(J, cached, upto, run, 1, extra, x, &at);
            const uint32_t n = pk_units<CK>(J, cached, b, 1), off = x - (at + extra * b) * J.segs;
            if (solo) {
                seg = (off + n + extra - 1) / (n + extra);
                pos = 0;
                return at * J.segs + seg * n;
            }
            seg = off / n;
            pos = (int32_t)(off - seg * n);
            return x;
        };
        lo = per * me;
        hi = total;
        if ((per && lo / per != me) || lo >= cost) {      /* past 2^32: past the end */
            lo = total;
        } else {
            uint32_t b2, seg2;
            int32_t pos2;
            if (cost - lo > per) hi = solo ? place(lo + per, b2, seg2, pos2) : lo + per;
            lo = place(lo, cons.b, in, cons.pos);
            if (in == J.segs) { /* solo: behind the row's last segment */
                in = 0;
                cons.b++;
            }
            if (lo < hi) cons.row = pk_row_of<CK>(J, B <= PK_CACHED ? cached[cons.b] : pk_len_of(J, cons.b, false));
        }
    }
    if (lo < hi) {
        cons.hk = J.tiles == 1 ? in : in / J.tiles;
        cons.tile = in - cons.hk * J.tiles;
        cons.enter(J);
    }
    __syncthreads(); /* `upto` has been read */
    if (lo >= hi) return; /* a CTA's four warps alike, but for solo ones, which meet no more */

    /* ---- cursors: cons walks the worker's segments, prod runs ahead by the warp's chunks */
    const uint32_t stride = solo ? 1 : PK_WARPS, lead = solo ? 0 : w;
    const uint32_t slice = hi - lo;                       /* chunks in the slice */
    pk_cursor<CK, HEADS> prod = cons;
    uint32_t ahead = lead;                                /* slice offset of prod */
    if (lead) prod.step(J, cached, (int32_t)lead);
    const uint32_t kbase = pk_saddr(ring);

    /* the page of each lane's key of prod's chunk is loaded a chunk ahead */
    uint32_t page = 0, slot = 0, there = 0;
    bool real = false, values = false;                    /* values: prod's chunk has its keys issued (SPLIT) */
    uint64_t at_key = 0;                                  /* byte offset of the lane's key */
    auto fetch = [&]() {
        const int32_t j = (prod.row.c0 + prod.pos) * CK + (int32_t)(lane % CK);
        real = j >= prod.lo && j < prod.hi;
        if (real) {
            const uint32_t pi = J.page_shift >= 0 ? (uint32_t)j >> J.page_shift : (uint32_t)j / J.D.page_size;
            slot = (uint32_t)j - pi * J.D.page_size;
            page = (uint32_t)__ldcg(prod.row.table + pi); /* a kernel that this one overlapped may have written it */
        }
    };
    constexpr uint32_t RPI = 32 / S::UNITS;               /* keys per copy instruction of a warp */
    const uint32_t cu = lane % S::UNITS, cr = lane / S::UNITS; /* a lane's 16 bytes and first key in it */
    const bool runs = J.D.page_size % 8 == 0;             /* 8 aligned keys are in one page */
    const bool copies = cr < RPI && cu < units;
    const uint32_t tok_bytes = (uint32_t)J.D.tok_stride * S::ELT;
    const uint64_t page_bytes = J.D.page_stride * S::ELT;
    /* what does not change of the copies' addresses: a lane's first source less its key's offset, its targets in
     * the first 8 keys of a stage */
    const uint64_t lane_at = (uint64_t)J.D.k + (uint64_t)cr * tok_bytes + cu * 16;
    const uint64_t key_step = (uint64_t)RPI * tok_bytes;
    uint32_t lane_to[8 / RPI];
#pragma unroll
    for (uint32_t i = 0; i < 8 / RPI; i++) {
        const uint32_t r = i * RPI + cr;
        lane_to[i] = kbase + r * S::ROW + (S::ROW >= 128 ? cu ^ (r & 7u) : cu ^ ((r >> 1) & 3u)) * 16;
    }
    const uint64_t k_to_v = (uint64_t)((const uint8_t *)J.D.v - (const uint8_t *)J.D.k);
    if (ahead < slice) fetch();

    auto issue = [&](uint32_t st) {
        if (ahead < slice) {
            if (!S::SPLIT || !values) {
                if (real && page >= J.D.n_pages) {
                    real = false;
                    atomicOr(J.err, PULSAR_KV_ERR_PAGE);
                }
                there = __ballot_sync(~0u, real);
                if (lane == 0) vmask[w][st] = there;
                at_key = real ? page * page_bytes + prod.head + (uint64_t)slot * tok_bytes : 0;
            }
            const uint64_t base = lane_at + (S::SPLIT && values ? k_to_v : 0);
            const uint32_t to = st * S::STAGE;
            if (there == ~0u && runs) {
                /* every key: within 8 of them addresses go up by a constant */
#pragma unroll
                for (uint32_t h = 0; h < CK; h += 8) {
                    const uint32_t lo32 = __shfl_sync(~0u, (uint32_t)at_key, h), hi32 = __shfl_sync(~0u, (uint32_t)(at_key >> 32), h);
                    if (copies) {
                        uint64_t k = base + ((uint64_t)hi32 << 32 | lo32);
#pragma unroll
                        for (uint32_t i = 0; i < 8 / RPI; i++) {
                            pk_cp16(lane_to[i] + to + h * S::ROW, (const void *)k, true);
                            if constexpr (!S::SPLIT) pk_cp16(lane_to[i] + to + (h + CK) * S::ROW, (const void *)(k + k_to_v), true);
                            k += key_step;
                        }
                    }
                }
            } else if (there) {
#pragma unroll 1
                for (uint32_t h = 0; h < CK; h += 8)
#pragma unroll
                    for (uint32_t i = 0; i < 8 / RPI; i++) {
                        const uint32_t r = h + i * RPI + (cr < RPI ? cr : 0);
                        const uint32_t lo32 = __shfl_sync(~0u, (uint32_t)at_key, r), hi32 = __shfl_sync(~0u, (uint32_t)(at_key >> 32), r);
                        const uint64_t k = base - (uint64_t)cr * tok_bytes + ((uint64_t)hi32 << 32 | lo32);
                        const bool ok = there >> r & 1u;
                        if (copies) {
                            pk_cp16(lane_to[i] + to + h * S::ROW, (const void *)k, ok);
                            if constexpr (!S::SPLIT) pk_cp16(lane_to[i] + to + (h + CK) * S::ROW, (const void *)(k + k_to_v), ok);
                        }
                    }
            }
            if (S::SPLIT) values = !values;
            if (!values) {
                ahead += stride;
                if (ahead < slice) {
                    prod.step(J, cached, (int32_t)stride);
                    fetch();
                }
            }
        }
        pk_cp_commit();
    };

    uint32_t stage = 0;
    uint32_t done = 0;                                    /* slice offset where the segment at hand begins */
    uint32_t next = lead;                                 /* slice offset of this warp's next chunk */
    pk_joint owed, joint;                                 /* joins that this CTA completed (a slice cuts two
                                                           * segments at most), put off to the slice's end */
    bool owes = false, also = false;

    while (done < slice) {
        const int32_t from = cons.pos;                    /* chunks [from, to) of this segment are ours */
        const int32_t to = (uint32_t)(cons.row.n - from) <= slice - done ? cons.row.n : from + (int32_t)(slice - done);
        const uint32_t v0 = cons.tile * HEADS;

        /* ---- q of this tile, in 16-bit parts; row 8 y + g of it is the lane's row y.  In shared memory the
         * warps' shares (KN k-steps each) meet; in registers each warp has all. */
        constexpr int KN = QSM ? KS / PK_WARPS : KS;
        const uint32_t k0 = QSM ? w * KN : 0;
        uint32_t qr[QSM ? 1 : KS][QW];
        float unit[R];                                   /* score units: log2, the power of two taken from q */
        int32_t slo[R], shi[R];
        {
            float x[R][KN][4];
#pragma unroll
            for (int y = 0; y < R; y++) {
                const uint32_t v = v0 + y * 8 + g;
                const bool have = v < J.rows;
                const uint32_t i = have ? v / J.group : 0, h = cons.hk * J.group + (have ? v % J.group : 0);
                pk_span(J, cons.row.len, i, slo[y], shi[y]);
                if (!have) shi[y] = 0;
                const uint64_t at = ((uint64_t)cons.b * J.A.n_q + i) * J.A.q_stride + (uint64_t)h * J.D.head_dim;
                /* e4m3 rows come as four neighbouring values a lane, 16-bit ones as two pairs */
                const uint32_t d0 = F8 ? 4 * c : 2 * c, d1 = F8 ? 2 : 8;
                if (J.A.q_type == PULSAR_TYPE_BF16) pk_q_load<PULSAR_TYPE_BF16, KN>(J, at, k0, d0, d1, x[y]);
                else if (J.A.q_type == PULSAR_TYPE_F16) pk_q_load<PULSAR_TYPE_F16, KN>(J, at, k0, d0, d1, x[y]);
                else pk_q_load<PULSAR_TYPE_F32, KN>(J, at, k0, d0, d1, x[y]);
                unit[y] = J.A.scale * PK_LOG2E * (F8 && J.D.k_scale ? __ldg(J.D.k_scale + cons.hk) : 1.0f);
            }
            if (done == 0) /* behind q's loads in the queue, not before them */
#pragma unroll 1
                for (uint32_t st = 0; st < S::STAGES - 1; st++) issue(st);
            float most[R];
#pragma unroll
            for (int y = 0; y < R; y++) {
                most[y] = 0.0f;
#pragma unroll
                for (int n = 0; n < KN; n++)
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        if (v0 + y * 8 + g >= J.rows || (k0 + n) * 16u >= J.D.head_dim) x[y][n][e] = 0.0f;
                        most[y] = fmaxf(most[y], fabsf(x[y][n][e]));
                    }
                if (!BF) {
                    most[y] = fmaxf(most[y], __shfl_xor_sync(~0u, most[y], 1));
                    most[y] = fmaxf(most[y], __shfl_xor_sync(~0u, most[y], 2));
                    if (QSM && c == 0) wml[w][y * 8 + g][0] = most[y];
                }
            }
            if (!BF) {
                if (QSM) __syncthreads();
#pragma unroll
                for (int y = 0; y < R; y++) {
                    if (QSM)
#pragma unroll
                        for (uint32_t k = 0; k < PK_WARPS; k++) most[y] = fmaxf(most[y], wml[k][y * 8 + g][0]);
                    /* the row's largest value to [2^14, 2^15): small ones stay clear of f16's subnormals */
                    uint32_t ex = __float_as_uint(most[y]) >> 23;
                    ex = ex < 15 ? 15 : ex > 253 ? 253 : ex;
                    const float up = __uint_as_float((268u - ex) << 23);
                    unit[y] *= __uint_as_float((ex - 14u) << 23);
#pragma unroll
                    for (int n = 0; n < KN; n++)
#pragma unroll
                        for (int e = 0; e < 4; e++) x[y][n][e] *= up;
                }
            }
#pragma unroll
            for (int n = 0; n < KN; n++) {
                uint32_t p[QW];
#pragma unroll
                for (int e = 0; e < QW; e++) {
                    /* R = 1: parts of (row g, low columns), (row g, high); R = 2: (g, low), (g + 8, low), (g, high), (g + 8, high) */
                    float *z = R == 1 ? x[0][n] + 2 * (e & 1) : x[(e & 1) * (R - 1)][n] + (e & 2);
                    p[e] = pk_split<BF, true>(z[0], z[1]);
                }
#pragma unroll
                for (int e = 0; e < QW; e++) {
                    if constexpr (QSM) qsm[(((k0 + n) * (QW / 2) + e / 2) * 32 + lane) * 2 + (e & 1)] = p[e];
                    else qr[n][e] = p[e];
                }
            }
        }
        if constexpr (QSM) __syncthreads();
        auto q_words = [&](int ks, uint32_t *a) {
#pragma unroll
            for (int e = 0; e < QW; e += 2) {
                if constexpr (QSM) {
                    const uint2 z = ((const uint2 *)qsm)[(ks * (QW / 2) + e / 2) * 32 + lane];
                    a[e] = z.x;
                    a[e + 1] = z.y;
                } else {
                    a[e] = qr[ks][e];
                    a[e + 1] = qr[ks][e + 1];
                }
            }
        };

        float o[NT][4], m[R], l[R];
#pragma unroll
        for (int y = 0; y < R; y++) {
            m[y] = -INFINITY;
            l[y] = 0.0f;
        }
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
            for (int e = 0; e < 4; e++) o[t][e] = 0.0f;

        /* the next stage, with the one after next issued behind it; *mask: which of its keys are there */
        auto turn = [&](uint32_t *mask) {
            pk_cp_wait<S::STAGES - 2>();
            __syncwarp();
            issue(stage == 0 ? S::STAGES - 1 : stage - 1);
            const uint32_t at = kbase + stage * S::STAGE;
            if (mask) *mask = vmask[w][stage];
            stage = stage + 1 == S::STAGES ? 0 : stage + 1;
            return at;
        };

        /* ---- the warp's chunks of this segment */
        const uint32_t end = done + (uint32_t)(to - from);
#pragma unroll 1
        for (; next < end; next += stride) {
            uint32_t mask;
            const uint32_t ka = turn(&mask);
            if (!mask) {
                if (S::SPLIT) turn(nullptr);
                continue;
            }
            /* the lane's ldmatrix rows; 16-byte unit u of row r sits at unit u ^ swizzle(r), the swizzle within
             * 128 aligned bytes, so that unit u + v (no carry) is an exclusive or away */
            auto unit_at = [](uint32_t x, int u) { return (x ^ ((u & 7) * 16)) + (u >> 3) * 128; };
            const uint32_t kr = F8 ? lane : (lane >> 4) * 8 + (lane & 7u), ku = F8 ? 0u : (lane >> 3) & 1u;
            const uint32_t kx = ka + kr * S::ROW + (S::ROW >= 128 ? ku ^ (kr & 7u) : ku ^ ((kr >> 1) & 3u)) * 16;
            const int32_t key0 = (cons.row.c0 + from + (int32_t)(next - done)) * CK;

            /* scores: keys are the columns */
            float s[KT][4], rest[REST ? KT : 1][4];
#pragma unroll
            for (int t = 0; t < KT; t++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    s[t][e] = 0.0f;
                    if constexpr (REST) rest[t][e] = 0.0f;
                }
            auto score = [&](int t, const uint32_t *a, uint32_t b0, uint32_t b1) {
                float *sum = s[t];
                if constexpr (R == 1) pk_mma<BF>(sum, a[0], QP > 1 ? a[QW > 2 ? 2 : 0] : 0, a[1], QP > 1 ? a[QW > 2 ? 3 : 1] : 0, b0, b1);
                else pk_mma<BF>(sum, a[0], a[1], a[2], a[3], b0, b1);
                if constexpr (R == 1 && QP == 3) pk_mma<BF>(rest[REST ? t : 0], a[4], 0, a[5], 0, b0, b1);
                if constexpr (R == 2 && QP > 1) pk_mma<BF>(rest[REST ? t : 0], a[4], a[5], a[6], a[7], b0, b1);
                if constexpr (R == 2 && QP > 2) pk_mma<BF>(rest[REST ? t : 0], a[8], a[9], a[10], a[11], b0, b1);
            };
#pragma unroll
            for (int ks = 0; ks < KS; ks++) {
                uint32_t a[QW], b[4];
                q_words(ks, a);
                if constexpr (!F8) {
                    /* matrices (keys 0-7, d 0-7), (0-7, 8-15), (8-15, 0-7), (8-15, 8-15) */
#pragma unroll
                    for (int t = 0; t < KT; t += 2) {
                        pk_ldm4(b, unit_at(kx, 2 * ks) + t * 8 * S::ROW);
                        score(t, a, b[0], b[1]);
                        score(t + 1, a, b[2], b[3]);
                    }
                } else {
                    /* a matrix is 8 keys x 16 bytes */
                    pk_ldm4(b, unit_at(kx, ks));
#pragma unroll
                    for (int t = 0; t < KT; t++) score(t, a, pk_e4m3x2(b[t]), pk_e4m3x2(b[t] >> 16));
                }
            }

            /* Fold the parts and mask (a lane has columns 2c, 2c + 1 of its rows).  m is the running maximum but
             * for SLACK: it moves, and the sums with it, only where the maximum has outgrown it by 2^SLACK.
             * Weights are relative to m less LIFT: at most 2^15, so that f16 holds them, and small ones stay
             * clear of its subnormals.  p's parts are the left factors of the output products in the layout that
             * they already have. */
            float top[R];
            bool moved = false;
#pragma unroll
            for (int y = 0; y < R; y++) {
#pragma unroll
                for (int t = 0; t < KT; t++)
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        float &x = s[t][2 * y + e];
                        if constexpr (R == 1 && QP > 1) {
                            const float low = s[t][e + 2];
                            x = pk_fold(x, QP == 3 ? low + rest[REST ? t : 0][e] : low);
                        }
                        if constexpr (R == 2 && QP > 1) x = pk_fold(x, rest[REST ? t : 0][2 * y + e]);
                        x *= unit[y];
                    }
                if (__builtin_expect(mask != ~0u || key0 < slo[y] || key0 + CK > shi[y], 0))
#pragma unroll
                    for (int t = 0; t < KT; t++)
#pragma unroll
                        for (int e = 0; e < 2; e++) {
                            const int32_t k = t * 8 + 2 * (int32_t)c + e;
                            if (!(mask >> k & 1u) || key0 + k < slo[y] || key0 + k >= shi[y]) s[t][2 * y + e] = -INFINITY;
                        }
                float half[KT];
#pragma unroll
                for (int t = 0; t < KT; t++) half[t] = fmaxf(s[t][2 * y], s[t][2 * y + 1]);
                top[y] = fmaxf(fmaxf(half[0], half[1]), fmaxf(half[KT - 2], half[KT - 1]));
            }
#pragma unroll
            for (int o2 = 1; o2 < 4; o2 <<= 1)
#pragma unroll
                for (int y = 0; y < R; y++) top[y] = fmaxf(top[y], __shfl_xor_sync(~0u, top[y], o2));
#pragma unroll
            for (int y = 0; y < R; y++) moved |= top[y] > m[y] + SLACK;
            if (__builtin_expect(__any_sync(~0u, moved), 0)) {
#pragma unroll
                for (int y = 0; y < R; y++) {
                    const float to = top[y] > m[y] + SLACK ? top[y] : m[y];
                    const float keep = to == m[y] ? 1.0f : pk_exp2(m[y] - to);
                    m[y] = to;
                    l[y] *= keep;
#pragma unroll
                    for (int t = 0; t < NT; t++) {
                        if constexpr (R == 1) {
#pragma unroll
                            for (int e = 0; e < 4; e++) o[t][e] *= keep;
                        } else {
                            o[t][2 * y] *= keep;
                            o[t][2 * y + 1] *= keep;
                        }
                    }
                }
            }
            uint32_t pa[KT / 2][PW];
#pragma unroll
            for (int y = 0; y < R; y++) {
                const float zero = (m[y] == -INFINITY ? 0.0f : m[y]) - LIFT; /* nothing seen yet: every weight is 0 */
#pragma unroll
                for (int t = 0; t < KT; t++)
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        float &x = s[t][2 * y + e];
                        x = pk_exp2(x - zero);
                    }
#pragma unroll
                for (int t = 0; t < KT; t += 2)
                    l[y] += s[t][2 * y] + s[t][2 * y + 1] + (s[t + 1][2 * y] + s[t + 1][2 * y + 1]);
            }
#pragma unroll
            for (int kt = 0; kt < KT / 2; kt++) {
                uint32_t *a = pa[kt];
                float *p0 = s[2 * kt], *p1 = s[2 * kt + 1];
                if constexpr (R == 1) {
                    a[0] = pk_split<BF, false>(p0[0], p0[1]);
                    a[2] = pk_split<BF, false>(p1[0], p1[1]);
                    a[1] = pk_split<BF, false>(p0[0], p0[1]);
                    a[3] = pk_split<BF, false>(p1[0], p1[1]);
                    if constexpr (PP == 3) {
                        a[4] = pk_split<BF, false>(p0[0], p0[1]);
                        a[5] = pk_split<BF, false>(p1[0], p1[1]);
                    }
                } else {
#pragma unroll
                    for (int q = 0; q < PP; q++)
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            float *z = (e < 2 ? p0 : p1) + 2 * (e & 1);
                            a[4 * q + e] = pk_split<BF, false>(z[0], z[1]);
                        }
                }
            }
            const uint32_t vr = lane & 15u, vu = lane >> 4;
            const uint32_t va = S::SPLIT ? turn(nullptr) : ka + CK * S::ROW;
            const uint32_t vx = va + vr * S::ROW + (S::ROW >= 128 ? vu ^ (vr & 7u) : vu ^ ((vr >> 1) & 3u)) * 16;
            if (J.A.n_q > 1) {
                /* rows of several tokens: a value that is not a number, seen by some of them, would reach the
                 * others as 0 * NaN.  Where the tile's spans end in this chunk, such values are taken out and
                 * a weight of the rows that see them becomes NaN, and with it their outputs (not their sums of
                 * weights, which make the lse). */
                bool edge = false;
#pragma unroll
                for (int y = 0; y < R; y++)
                    edge |= v0 + y * 8 + g < J.rows && (key0 < slo[y] || key0 + CK > shi[y]);
                if (__any_sync(~0u, edge)) {
                    const uint32_t odd = pk_take_odd<CT, CK, S::ROW>(va, mask);
#pragma unroll
                    for (int y = 0; y < R; y++) {
                        const int32_t a = slo[y] - key0, z = shi[y] - key0;
                        const uint32_t from = a <= 0 ? ~0u : a >= 32 ? 0u : ~0u << a, to = z <= 0 ? 0u : z >= 32 ? ~0u : ~(~0u << z);
                        if (odd & from & to) pa[0][y] = 0x7fff7fffu; /* two NaN weights of row 8 y + g, in either type */
                    }
                }
            }
#pragma unroll
            for (int kt = 0; kt < KT / 2; kt++)
#pragma unroll
                for (int t0 = 0; t0 < NT; t0 += 4) {
                    /* four output tiles' right factors, from matrices (keys 0-7, unit u), (keys 8-15, u),
                     * (0-7, u + 1), (8-15, u + 1) */
                    uint32_t b[8];
                    if constexpr (!F8) {
                        pk_ldm4t(b, unit_at(vx, t0) + kt * 16 * S::ROW);
                        pk_ldm4t(b + 4, unit_at(vx, t0 + 2) + kt * 16 * S::ROW);
                    } else {
                        /* a 16-bit column is two values: the even ones to tile 2u, the odd ones to 2u + 1 */
                        uint32_t v[4];
                        pk_ldm4t(v, unit_at(vx, t0 / 2) + kt * 16 * S::ROW);
#pragma unroll
                        for (int x = 0; x < 4; x++) {
                            b[4 * (x >> 1) + (x & 1)] = pk_e4m3x2(__byte_perm(v[x], 0, 0x0020));
                            b[4 * (x >> 1) + 2 + (x & 1)] = pk_e4m3x2(__byte_perm(v[x], 0, 0x0031));
                        }
                    }
                    /* a part's products for all tiles before the next part's, which add to the same sums */
#pragma unroll
                    for (int q = 0; q < (R == 1 ? PP - 1 : PP); q++)
#pragma unroll
                        for (int x = 0; x < 4; x++) {
                            const uint32_t *a = pa[kt] + 4 * q;
                            if (R == 1 && q == 1) pk_mma<BF>(o[t0 + x], a[0], 0, a[PW > 5 ? 1 : 0], 0, b[2 * x], b[2 * x + 1]);
                            else pk_mma<BF>(o[t0 + x], a[0], a[1], a[2], a[3], b[2 * x], b[2 * x + 1]);
                        }
                }
        }

        /* ---- the segment's end */
        const uint32_t took = (uint32_t)(to - from);
        constexpr int RUN = F8 ? 4 : 2;                   /* a lane's run of columns */
        /* RUN neighbouring columns of row y at tile t: folded parts, times by */
        auto columns = [&](int y, int t, float by, float *x) {
            const float *a = o[t], *b2 = o[F8 ? t + 1 : t];
            if constexpr (R == 1) {
                x[0] = pk_fold(a[0], a[2]);
                x[RUN - 2 > 0 ? 2 : 1] = pk_fold(a[1], a[3]);
                if constexpr (F8) {
                    x[1] = pk_fold(b2[0], b2[2]);
                    x[RUN - 1] = pk_fold(b2[1], b2[3]);
                }
            } else {
                x[0] = a[2 * y];
                x[RUN - 2 > 0 ? 2 : 1] = a[2 * y + 1];
                if constexpr (F8) {
                    x[1] = b2[2 * y];
                    x[RUN - 1] = b2[2 * y + 1];
                }
            }
#pragma unroll
            for (int e = 0; e < RUN; e++) x[e] *= by;
        };
#pragma unroll
        for (int y = 0; y < R; y++) {
            l[y] += __shfl_xor_sync(~0u, l[y], 1);
            l[y] += __shfl_xor_sync(~0u, l[y], 2);
        }
        const float drop = BF ? 1.0f : 1.0f / 128.0f;     /* 2^-LIFT */
        if (solo) {
#pragma unroll
            for (int y = 0; y < R; y++) {
                const uint32_t v = v0 + y * 8 + g;
                if (v >= J.rows) continue;
                const float by = drop * pk_finish(J, cons.b, cons.row.len, cons.hk, v, m[y], l[y] * drop, c == 0);
#pragma unroll
                for (int t = 0; t < NT; t += RUN / 2) {
                    const uint32_t col = t * 8 + RUN * c;
                    float x[RUN];
                    columns(y, t, by, x);
                    if (col < J.D.head_dim) pk_put<RUN>(J, cons.b, cons.hk, v, col, x);
                }
            }
        } else {
            /* the four warps meet: maxima, then the sums of 64 columns at a time */
            const bool cut = from != 0 || to != cons.row.n;
            float *part = J.parts + (uint64_t)(2 * blockIdx.x + (done != 0)) * (HEADS * (DP + 2));
#pragma unroll
            for (int y = 0; y < R; y++)
                if (c == 0) *(float2 *)wml[w][y * 8 + g] = make_float2(m[y], l[y] * drop);
            __syncthreads();
#pragma unroll
            for (int y = 0; y < R; y++) {
                float top = -INFINITY, sum = 0.0f;
#pragma unroll
                for (uint32_t k = 0; k < PK_WARPS; k++) top = fmaxf(top, wml[k][y * 8 + g][0]);
                const float zero = top == -INFINITY ? 0.0f : top;
#pragma unroll
                for (uint32_t k = 0; k < PK_WARPS; k++) sum += wml[k][y * 8 + g][1] * pk_exp2(wml[k][y * 8 + g][0] - zero);
                const float keep = drop * pk_exp2(m[y] - zero);
                if (w == 0 && c == 0) {
                    const uint32_t v = v0 + y * 8 + g;
                    if (!cut && v < J.rows) top = pk_finish(J, cons.b, cons.row.len, cons.hk, v, top, sum);
                    *(float2 *)fml[y * 8 + g] = make_float2(top, sum); /* uncut: [0] is the output's factor */
                }
#pragma unroll
                for (int c0 = 0; c0 < DP; c0 += 64) {
                    if (y || c0) __syncthreads(); /* the previous columns have been read */
#pragma unroll
                    for (int t = 0; t < (NT - c0 / 8 < 8 ? NT - c0 / 8 : 8); t += RUN / 2) {
                        float x[RUN], *d = side + (w * 8 + g) * S::XROW + t * 8 + RUN * c;
                        columns(y, c0 / 8 + t, keep, x);
                        if constexpr (F8) *(float4 *)d = make_float4(x[0], x[1], x[RUN - 2], x[RUN - 1]);
                        else *(float2 *)d = make_float2(x[0], x[1]);
                    }
                    __syncthreads();
                    /* four columns of a row a thread: out, or into the workspace */
                    static_assert(PK_WARPS * 32 == 8 * 64 / 4, "one run of four columns a thread");
                    const uint32_t head = y * 8 + tid / 16, col = c0 + tid % 16 * 4;
                    float4 z = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
                    for (uint32_t k = 0; k < PK_WARPS; k++) {
                        const float4 v = *(const float4 *)(side + (k * 8 + tid / 16) * S::XROW + tid % 16 * 4);
                        z.x += v.x;
                        z.y += v.y;
                        z.z += v.z;
                        z.w += v.w;
                    }
                    if (DP % 64 && col >= DP) {
                    } else if (cut) {
                        __stcg((float4 *)(part + 2 * HEADS + head * DP + col), z);
                        if (col == 0) __stcg((float2 *)(part + 2 * head), make_float2(fml[head][0], fml[head][1]));
                    } else if (v0 + head < J.rows && col < J.D.head_dim) {
                        const float by = fml[head][0], q4[4] = {z.x * by, z.y * by, z.z * by, z.w * by};
                        pk_put<4>(J, cons.b, cons.hk, v0 + head, col, q4);
                    }
                }
            }
            if (cut) {
                /* a join that falls to this CTA waits for its slice's end: other joins may wait for the rest of it */
                pk_joint S2;
                S2.b = cons.b;
                S2.hk = cons.hk;
                S2.v0 = v0;
                S2.len = cons.row.len;
                if (own) {
                    S2.w0 = me - piece;
                    S2.w1 = S2.w0 + pieces - 1;
                    S2.inside = false;
                } else {
                    const uint32_t seg0 = lo + done - (uint32_t)from;
                    S2.w0 = seg0 / per;
                    S2.w1 = (seg0 + (uint32_t)cons.row.n - 1) / per;
                    S2.inside = seg0 > per * S2.w0;
                }
                if (pk_joint_arrive(J, S2, &last)) {
                    if (owes) {
                        also = true;
                        joint = S2;
                    } else {
                        owes = true;
                        owed = S2;
                    }
                }
            }
            __syncthreads(); /* wml, fml and side are free again */
        }
        done += took;
        if (done < slice) cons.step(J, cached, (int32_t)took);
    }
    pk_cp_wait<0>();
    /* the ring is free now */
    constexpr int PARTS = PK_WARPS * S::RING / (HEADS * (DP + 2) * 4);
    if (owes) pk_joint_finish<DP, HEADS, PARTS>(J, owed, &last, fml, (float *)smem);
    if (also) pk_joint_finish<DP, HEADS, PARTS>(J, joint, &last, fml, (float *)smem);
}

template <uint32_t CT, int DP, int R, int QP>
static int pk_attend_launch(const pk_attend_job &J, uint32_t grid, cudaStream_t st) {
    typedef pk_shape<CT, DP, R, QP> S;
    static uint64_t done = 0;
    constexpr uint32_t smem = PK_WARPS * S::RING + S::SIDE;
    auto kernel = pk_attend_kernel<CT, DP, R, QP>;
    if (!pm_smem_attr(kernel, smem, &done)) return 0;
    const uint32_t most = S::OCC * pk_sm_count(); /* one wave */
    return pm_ok(pk_launch(kernel, grid < most ? grid : most, PK_WARPS * 32, smem, st, J), "kv attend launch");
}

/* one translation unit per cache type (kv_attend_*.cu); r as the kernel's R,
 * wide: q has more bits than one part holds */
typedef int (*pk_attend_fn)(const pk_attend_job &, uint32_t, cudaStream_t);
pk_attend_fn pk_attend_bf16(int dp, int r, bool wide);
pk_attend_fn pk_attend_f16(int dp, int r, bool wide);
pk_attend_fn pk_attend_e4m3(int dp, int r, bool wide);

template <uint32_t CT, int DP>
static pk_attend_fn pk_attend_pick_at(int r, bool wide) {
    constexpr int MOST = CT == PULSAR_TYPE_BF16 ? 3 : 2; /* parts of wide q */
    if (r == 1) return wide ? pk_attend_launch<CT, DP, 1, MOST> : pk_attend_launch<CT, DP, 1, 1>;
    return wide ? pk_attend_launch<CT, DP, 2, MOST> : pk_attend_launch<CT, DP, 2, 1>;
}

template <uint32_t CT>
static pk_attend_fn pk_attend_pick(int dp, int r, bool wide) {
    if (dp == 64) return pk_attend_pick_at<CT, 64>(r, wide);
    if (dp == 96) return pk_attend_pick_at<CT, 96>(r, wide);
    if (dp == 128) return pk_attend_pick_at<CT, 128>(r, wide);
    if constexpr (CT != PULSAR_TYPE_E4M3) /* rows of 192 bytes would break the swizzle's 128 */
        if (dp == 192) return pk_attend_pick_at<CT, 192>(r, wide);
    return pk_attend_pick_at<CT, 256>(r, wide);
}
