/* pk_attend.cuh - attention of new tokens over a paged cache.
 *
 *   o = sum_j e^(s_j - m) v_j / (sum_j e^(s_j - m) + e^(sink - m)),  s_j = scale q.k_j
 *
 * The cache's bytes are the bound: each visible key and value is read once
 * for all the query heads that share it, and 2 x 16 x head_dim multiply-adds
 * per key are far below what the warp matrix instructions do in that time.
 *
 * Work.  The query rows of a key head are its n_q * (n_head / n_kv) (token,
 * head) pairs; a tile is 8 * MT of them.  All (sequence, key head, tile)
 * segments lie one behind the other on a line, counted in chunks of CK keys,
 * and the CTAs take equal slices of it: no length, batch or head count leaves
 * SMs idle, and the host needs no lengths.  A segment that a slice cuts is
 * joined through the workspace by the CTA that arrives last, in the order of
 * the slices (a fixed order: the same call gives the same bits), 32 parts at
 * a time.
 *
 * Inside a CTA four warps take the chunks of its slice in turn.  Each warp
 * fills a ring of its own with 16-byte asynchronous copies (no barrier in the
 * stream; keys out of the span are filled with zeros, so stale bytes never
 * meet the arithmetic) and keeps its own running maximum, sum and output
 * tile; the four meet at a segment's end.
 *
 * Products.  A 16-row matrix tile holds 8 query rows twice: the leading 16
 * bits of each value in row g and the next 16 in row g + 8, of q for the
 * scores and of the probabilities for the output.  The tile is 16 rows high
 * anyway, so the second half costs nothing and the sums keep 22 bits of each
 * factor (f16 parts; q's rows are first scaled by a power of two) or 16 (bf16
 * parts); THREE adds a third bf16 part where a bf16 cache meets wider q, so
 * that f32 results are f32 results.  Sums, maxima and outputs are f32. */
#pragma once
#include "pk_common.h"

#define PK_WARPS 4u
#define PK_STAGES 3u
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
    uint32_t least;      /* least chunks in a slice, where segments are long */
    uint32_t *counters;  /* [2][2 * PK_MAX_WORKERS] */
    float *parts;        /* [workers][2] parts of 8 * MT * (DP + 2) floats */
    uint32_t *err;
};

template <uint32_t CT, int DP>
struct pk_shape {
    static constexpr int ELT = CT == PULSAR_TYPE_E4M3 ? 1 : 2;
    static constexpr int ROW = DP * ELT;                  /* bytes of a key in shared memory */
    static constexpr int UNITS = ROW / 16;
    static constexpr int CK = ROW >= 256 ? 16 : 32;       /* keys per chunk: about 8 KB of keys and values */
    static constexpr int STAGE = 2 * CK * ROW;
    static constexpr int RING = PK_STAGES * STAGE;        /* per warp */
    static constexpr int QROW = DP / 4 + 4;               /* floats; padded against bank conflicts */
    static constexpr int JOIN = 4 * 3 * 8 * QROW * 4;     /* bytes: each quarter of the columns, from three warps */
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
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
                     "{%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
                     "{%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

/* x, y rounded to 16 bits and packed, x low; x, y become what is left (0
 * where the value is not finite) */
template <bool BF>
__device__ __forceinline__ uint32_t pk_split(float &x, float &y) {
    uint32_t r;
    if constexpr (BF) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
        r = *(const uint32_t *)&h;
        x = isfinite(x) ? x - __low2float(h) : 0.0f;
        y = isfinite(y) ? y - __high2float(h) : 0.0f;
    } else {
        const __half2 h = __floats2half2_rn(x, y);
        r = *(const uint32_t *)&h;
        x = isfinite(x) ? x - __low2float(h) : 0.0f;
        y = isfinite(y) ? y - __high2float(h) : 0.0f;
    }
    return r;
}

/* two e4m3 bytes (low half of v) -> f16x2, exact */
__device__ __forceinline__ uint32_t pk_e4m3x2(uint32_t v) {
    uint32_t r;
    asm("{\n\t.reg .b16 t;\n\tcvt.u16.u32 t, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, t;\n\t}" : "=r"(r) : "r"(v));
    return r;
}

/* the leading sum, plus the rest where the rest is a number: a key or value
 * of +-inf makes the lower parts' products NaN, the leading one's +-inf */
__device__ __forceinline__ float pk_fold(float lead, float rest) { return isfinite(rest) ? lead + rest : lead; }

/* what a sequence's length, window and row say */
struct pk_row {
    int32_t len, c0, n;       /* keys; first chunk; chunks (at least 1) */
    const int32_t *table;
};

template <int CK>
__device__ __forceinline__ pk_row pk_row_of(const pk_attend_job &J, uint32_t b, bool tell) {
    pk_row r;
    const int32_t row = J.A.seq ? J.A.seq[b] : (int32_t)b;
    int32_t len = J.A.lens[b];
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
    r.len = len;
    const int64_t lo = J.A.window ? (int64_t)len - (J.A.n_q - 1) - J.A.window : 0;
    r.c0 = lo > 0 ? (int32_t)(lo / CK) : 0;
    const int32_t end = (int32_t)(((int64_t)len + CK - 1) / CK);
    r.n = end > r.c0 ? end - r.c0 : 1;
    r.table = J.D.table + (uint64_t)(len ? row : 0) * J.D.table_stride;
    return r;
}

/* keys [lo, hi) that token i of a sequence of len keys sees */
__device__ __forceinline__ void pk_span(const pk_attend_job &J, int32_t len, uint32_t i, int32_t &lo, int32_t &hi) {
    const int64_t h = (int64_t)len - (J.A.n_q - 1 - i);
    hi = h > 0 ? (int32_t)h : 0;
    lo = J.A.window && (uint32_t)hi > J.A.window ? hi - (int32_t)J.A.window : 0;
}

__device__ __forceinline__ float pk_q_at(const pk_attend_job &J, uint64_t at) {
    if (J.A.q_type == PULSAR_TYPE_BF16) return __bfloat162float(((const __nv_bfloat16 *)J.A.q)[at]);
    if (J.A.q_type == PULSAR_TYPE_F16) return __half2float(((const __half *)J.A.q)[at]);
    return ((const float *)J.A.q)[at];
}

/* A warp's place on the line: the chunk `pos` of segment `seg` of sequence b */
template <int CK>
struct pk_cursor {
    uint32_t b, seg;
    int32_t pos;
    pk_row row;
    __device__ __forceinline__ void step(const pk_attend_job &J, int32_t by) {
        pos += by;
        while (pos >= row.n) {
            pos -= row.n;
            if (++seg == J.segs) {
                seg = 0;
                if (++b >= J.A.n_rows) return; /* past the line's end: not used again */
                row = pk_row_of<CK>(J, b, false);
            }
        }
    }
};

/* columns col .. col + 3 of query row v (of key head hk, sequence b): top
 * and sum are the row's maximum (log2 units) and sum, x its output sums */
template <int DP>
__device__ __forceinline__ void pk_attend_out(const pk_attend_job &J, uint32_t b, int32_t len, uint32_t hk, uint32_t v,
                                              uint32_t col, float top, float sum, float4 x) {
    if (v >= J.rows || col >= J.D.head_dim) return;
    const uint32_t i = v / J.group, h = hk * J.group + v % J.group;
    int32_t lo, hi;
    pk_span(J, len, i, lo, hi);
    const bool empty = hi <= lo;
    float by = 1.0f;
    if (J.A.sinks && !empty) {
        const float sink = __ldg(J.A.sinks + h) * PK_LOG2E, t = fmaxf(top, sink);
        if (t != -INFINITY) {
            by = exp2f(top - t);
            sum = sum * by + exp2f(sink - t);
            top = t;
        }
    }
    const uint64_t tok = (uint64_t)b * J.A.n_q + i;
    if (J.A.lse && col == 0) J.A.lse[tok * J.A.n_head + h] = empty ? -INFINITY : logf(sum) + top * 0.6931471805599453f;
    by = sum == 0.0f ? 0.0f : by / sum;
    if (J.D.v_scale) by *= __ldg(J.D.v_scale + hk);
    if (sum == 0.0f) x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    const uint64_t at = tok * J.A.out_stride + (uint64_t)h * J.D.head_dim + col;
    const float y[4] = {x.x * by, x.y * by, x.z * by, x.w * by};
    if (J.A.q_type == PULSAR_TYPE_F32) {
        float *d = (float *)J.A.out + at;
#pragma unroll
        for (int e = 0; e < 4; e++) d[e] = y[e];
    } else if (J.A.q_type == PULSAR_TYPE_BF16) {
        __nv_bfloat16 *d = (__nv_bfloat16 *)J.A.out + at;
#pragma unroll
        for (int e = 0; e < 4; e++) d[e] = __float2bfloat16_rn(y[e]);
    } else {
        __half *d = (__half *)J.A.out + at;
#pragma unroll
        for (int e = 0; e < 4; e++) d[e] = __float2half_rn(y[e]);
    }
}

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

/* The join of a cut segment, which the workers w0 .. w1 share; worker w's
 * part is in slot 2 w, but in 2 w0 + 1 where the segment begins inside w0's
 * slice.  The parts meet PK_GROUP at a time (the group's sum replaces its
 * first part), then the groups; the sums run in the order of the workers. */
template <int DP, int MT>
__device__ void pk_attend_join(const pk_attend_job &J, uint32_t b, int32_t len, uint32_t hk, uint32_t v0, uint32_t w0,
                               uint32_t w1, bool inside, uint32_t *last, float (*ml)[2]) {
    constexpr uint32_t HEADS = 8 * MT;
    constexpr uint64_t FLOATS = (uint64_t)HEADS * (DP + 2);
    const uint32_t n = w1 - w0 + 1, groups = (n + PK_GROUP - 1) / PK_GROUP;
    const uint32_t mine = (blockIdx.x - w0) / PK_GROUP;
    uint32_t first = mine * PK_GROUP, step = 1, count = n - first < PK_GROUP ? n - first : PK_GROUP;
    const uint32_t name = 2 * w0 + inside; /* no other segment's first slot */
    bool final = groups == 1;
    if (!pk_arrive(J.counters + (final ? name : 2 * (w0 + first) + (first == 0 && inside)), count, last)) return;
    for (;;) {
        for (uint32_t x = threadIdx.x; x < HEADS * DP / 4; x += PK_WARPS * 32) {
            const uint32_t head = x / (DP / 4), col = x % (DP / 4) * 4;
            auto part = [&](uint32_t k) {
                const uint32_t at = first + k * step;
                return J.parts + (2ull * (w0 + at) + (at == 0 && inside)) * FLOATS;
            };
            float top = -INFINITY, sum = 0.0f;
#pragma unroll 4
            for (uint32_t k = 0; k < count; k++) top = fmaxf(top, __ldcg(part(k) + 2 * head));
            const float zero = top == -INFINITY ? 0.0f : top;
            float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
            for (uint32_t k = 0; k < count; k++) {
                const float2 x2 = __ldcg((const float2 *)(part(k) + 2 * head));
                const float4 v = __ldcg((const float4 *)(part(k) + 2 * HEADS + head * DP + col));
                const float f = exp2f(x2.x - zero);
                sum += x2.y * f;
                acc.x += v.x * f;
                acc.y += v.y * f;
                acc.z += v.z * f;
                acc.w += v.w * f;
            }
            if (final) {
                pk_attend_out<DP>(J, b, len, hk, v0 + head, col, top, sum, acc);
            } else {
                __stcg((float4 *)(part(0) + 2 * HEADS + head * DP + col), acc);
                if (col == 0) {
                    ml[head][0] = top;
                    ml[head][1] = sum;
                }
            }
        }
        if (final) return;
        __syncthreads(); /* part 0's maxima and sums have been read */
        if (threadIdx.x < HEADS)
            __stcg((float2 *)(J.parts + (2ull * (w0 + first) + (first == 0 && inside)) * FLOATS + 2 * threadIdx.x),
                   make_float2(ml[threadIdx.x][0], ml[threadIdx.x][1]));
        if (!pk_arrive(J.counters + 2 * PK_MAX_WORKERS + name, groups, last)) return;
        first = 0;
        step = PK_GROUP;
        count = groups;
        final = true;
    }
}

template <uint32_t CT, int DP, int MT, bool THREE>
__global__ void __launch_bounds__(PK_WARPS * 32, 1) pk_attend_kernel(const __grid_constant__ pk_attend_job J) {
    typedef pk_shape<CT, DP> S;
    constexpr bool BF = CT == PULSAR_TYPE_BF16;
    constexpr bool F8 = CT == PULSAR_TYPE_E4M3;
    constexpr int CK = S::CK, KS = DP / 16, NT = DP / 8, KT = CK / 8;
    constexpr int HEADS = 8 * MT;
    constexpr bool QSM = MT * DP > 128 || THREE;          /* q's parts wait in shared memory, not registers */
    constexpr float LIFT = BF ? 0.0f : 15.0f;
    constexpr int QPARTS = THREE ? 6 : 4;                 /* words per lane and k-step */

    extern __shared__ __align__(128) uint8_t smem[];
    uint8_t *ring = smem + (threadIdx.x >> 5) * S::RING;
    float *join = (float *)(smem + PK_WARPS * S::RING);
    /* QSM: [MT][KS][QPARTS][32], in the same bytes: q is done with when a segment's warps meet */
    uint32_t *qsm = (uint32_t *)join;
    static_assert(!QSM || MT * KS * QPARTS * 128 <= S::JOIN, "q's parts fit beside the ring");
    __shared__ float wml[PK_WARPS][HEADS][2];             /* each warp's maximum and sum */
    __shared__ float fml[HEADS][2];
    __shared__ uint32_t vmask[PK_WARPS][PK_STAGES];       /* keys of a stage that are there */
    __shared__ unsigned long long scan[PK_WARPS + 2];
    __shared__ uint32_t found[2], last;

    const uint32_t tid = threadIdx.x, lane = tid & 31u, w = tid >> 5;
    const uint32_t g = lane >> 2, c = lane & 3u;          /* row and column pair of a fragment */

    /* ---- the line's length, this CTA's slice, and where that begins */
    const uint32_t B = J.A.n_rows;
    const uint32_t run = (B + PK_WARPS * 32 - 1) / (PK_WARPS * 32);
    const uint32_t r0 = tid * run < B ? tid * run : B, r1 = B - r0 < run ? B : r0 + run;
    unsigned long long mine = 0;
    for (uint32_t r = r0; r < r1; r++) mine += (unsigned long long)pk_row_of<CK>(J, r, blockIdx.x == 0).n;
    unsigned long long upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const unsigned long long y = __shfl_up_sync(~0u, upto, o);
        if (lane >= o) upto += y;
    }
    if (lane == 31) scan[w] = upto;
    __syncthreads();
    unsigned long long before = 0, all = 0;
#pragma unroll
    for (uint32_t k = 0; k < PK_WARPS; k++) {
        if (k < w) before += scan[k];
        all += scan[k];
    }
    upto += before;
    const unsigned long long total = all * J.segs;
    unsigned long long per = (total + gridDim.x - 1) / gridDim.x;
    /* a segment of up to 16 chunks is not cut to fill idle SMs: joining it costs more than reading it */
    const unsigned long long least = all <= 16ull * B ? (all + B - 1) / B : J.least;
    if (per < least) per = least;
    const unsigned long long lo = per * blockIdx.x;
    if (lo >= total) return;
    const unsigned long long hi = total - lo < per ? total : lo + per;
    if ((upto - mine) * J.segs <= lo && lo < upto * J.segs) { /* one thread: lo is in its rows */
        unsigned long long at = upto - mine;
        for (uint32_t r = r0; r < r1; r++) {
            const uint32_t n = (uint32_t)pk_row_of<CK>(J, r, false).n;
            if (lo < (at + n) * J.segs) {
                found[0] = r;
                scan[PK_WARPS] = at * J.segs;
                break;
            }
            at += n;
        }
    }
    /* columns from head_dim to DP stay zero: copies never write them */
    const uint32_t units = J.D.head_dim * S::ELT / 16;
    if (units < S::UNITS)
        for (uint32_t o = tid * 16; o < PK_WARPS * S::RING; o += PK_WARPS * 32 * 16)
            *(uint4 *)(smem + o) = make_uint4(0, 0, 0, 0);
    __syncthreads();

    /* ---- cursors: cons walks the CTA's segments, prod runs ahead by the warp's chunks */
    pk_cursor<CK> cons;
    cons.b = found[0];
    cons.row = pk_row_of<CK>(J, cons.b, false);
    {
        const unsigned long long in = lo - scan[PK_WARPS];
        cons.seg = (uint32_t)(in / (uint32_t)cons.row.n);
        cons.pos = (int32_t)(in % (uint32_t)cons.row.n);
    }
    pk_cursor<CK> prod = cons;
    prod.step(J, (int32_t)w);
    const uint32_t slice = (uint32_t)(hi - lo);           /* chunks in this CTA's slice */
    uint32_t ahead = w;                                   /* slice offset of prod */

    const uint32_t kbase = pk_saddr(ring);
    const uint64_t elt = S::ELT;

    auto issue = [&](uint32_t st) {
        if (ahead < slice) {
            const uint32_t hk = prod.seg / J.tiles, tile = prod.seg % J.tiles;
            int32_t tlo, thi, x;
            {
                const uint32_t v0 = tile * HEADS, v1 = v0 + HEADS < J.rows ? v0 + HEADS - 1 : J.rows - 1;
                pk_span(J, prod.row.len, v0 / J.group, tlo, x);
                pk_span(J, prod.row.len, v1 / J.group, x, thi);
            }
            const int32_t j = (prod.row.c0 + prod.pos) * CK + (int32_t)(lane % CK);
            uint64_t off = 0;
            bool real = j >= tlo && j < thi;
            if (real) {
                const uint32_t pi = J.page_shift >= 0 ? (uint32_t)j >> J.page_shift : (uint32_t)j / J.D.page_size;
                const uint32_t slot = (uint32_t)j - pi * J.D.page_size;
                const uint32_t page = (uint32_t)__ldg(prod.row.table + pi);
                if (page < J.D.n_pages) {
                    off = ((uint64_t)page * J.D.page_stride + hk * J.D.head_stride + slot * J.D.tok_stride) * elt;
                } else {
                    real = false;
                    atomicOr(J.err, PULSAR_KV_ERR_PAGE);
                }
            }
            const uint32_t there = __ballot_sync(~0u, real);
            if (lane == 0) vmask[w][st] = CK == 32 ? there : there & ((1u << (CK & 31)) - 1u);
            if (there) {
                const uint32_t lo32 = (uint32_t)off, hi32 = (uint32_t)(off >> 32);
                constexpr uint32_t RPI = 32 / S::UNITS ? 32 / S::UNITS : 1; /* rows per instruction */
                const uint32_t u = lane % S::UNITS, rr = lane / S::UNITS;
                const uint32_t dst = kbase + st * S::STAGE;
#pragma unroll
                for (uint32_t i = 0; i < CK / RPI; i++) {
                    const uint32_t r = i * RPI + rr;
                    const uint64_t o = (uint64_t)__shfl_sync(~0u, hi32, r) << 32 | __shfl_sync(~0u, lo32, r);
                    const uint32_t sw = S::ROW >= 128 ? u ^ (r & 7u) : u ^ ((r >> 1) & 3u);
                    const bool ok = there >> r & 1u;
                    if (u < units) {
                        pk_cp16(dst + r * S::ROW + sw * 16, (const uint8_t *)J.D.k + o + u * 16, ok);
                        pk_cp16(dst + CK * S::ROW + r * S::ROW + sw * 16, (const uint8_t *)J.D.v + o + u * 16, ok);
                    }
                }
            }
            prod.step(J, PK_WARPS);
            ahead += PK_WARPS;
        }
        pk_cp_commit();
    };
#pragma unroll
    for (uint32_t st = 0; st < PK_STAGES - 1; st++) issue(st);

    uint32_t stage = 0;
    uint32_t done = 0;                                    /* slice offset where the segment at hand begins */
    uint32_t next = w;                                    /* slice offset of this warp's next chunk */
    unsigned long long base = lo;                         /* line position of `done` */

    while (done < slice) {
        const int32_t from = cons.pos;                    /* chunks [from, to) of this segment are ours */
        const int32_t to = (uint32_t)(cons.row.n - from) <= slice - done ? cons.row.n : from + (int32_t)(slice - done);
        const uint32_t hk = cons.seg / J.tiles, tile = cons.seg % J.tiles;
        const uint32_t v0 = tile * HEADS;

        /* ---- q of this tile, in 16-bit parts */
        uint32_t qr[QSM ? 1 : MT][QSM ? 1 : KS][4];
        float unit[MT];                                   /* score units: log2, the power of two taken from q */
        int32_t slo[MT], shi[MT];
#pragma unroll
        for (int mt = 0; mt < MT; mt++) {
            const uint32_t v = v0 + mt * 8 + g;
            const bool have = v < J.rows;
            const uint32_t i = have ? v / J.group : 0, h = hk * J.group + (have ? v % J.group : 0);
            pk_span(J, cons.row.len, i, slo[mt], shi[mt]);
            if (!have) shi[mt] = 0;
            const uint64_t at = ((uint64_t)cons.b * J.A.n_q + i) * J.A.q_stride + (uint64_t)h * J.D.head_dim;
            float x[KS][4], most = 0.0f;
#pragma unroll
            for (int ks = 0; ks < KS; ks++) {
                /* e4m3 rows come as four neighbouring values a lane, 16-bit ones as two pairs */
                const uint32_t d0 = ks * 16 + (F8 ? 4 * c : 2 * c), d1 = d0 + (F8 ? 2 : 8);
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const uint32_t d = (e < 2 ? d0 : d1) + (e & 1);
                    x[ks][e] = have && d < J.D.head_dim ? pk_q_at(J, at + d) : 0.0f;
                    most = fmaxf(most, fabsf(x[ks][e]));
                }
            }
            unit[mt] = J.A.scale * PK_LOG2E * (F8 && J.D.k_scale ? __ldg(J.D.k_scale + hk) : 1.0f);
            if (!BF) {
                most = fmaxf(most, __shfl_xor_sync(~0u, most, 1));
                most = fmaxf(most, __shfl_xor_sync(~0u, most, 2));
                uint32_t ex = __float_as_uint(most) >> 23;
                ex = ex < 15 ? 15 : ex > 253 ? 253 : ex;
                /* the row's largest value to [2^14, 2^15): small ones stay clear of f16's subnormals */
                const float down = __uint_as_float((268u - ex) << 23);
                unit[mt] *= __uint_as_float((ex - 14u) << 23);
#pragma unroll
                for (int ks = 0; ks < KS; ks++)
#pragma unroll
                    for (int e = 0; e < 4; e++) x[ks][e] *= down;
            }
#pragma unroll
            for (int ks = 0; ks < KS; ks++) {
                uint32_t p[QPARTS];
                p[0] = pk_split<BF>(x[ks][0], x[ks][1]);
                p[2] = pk_split<BF>(x[ks][2], x[ks][3]);
                p[1] = pk_split<BF>(x[ks][0], x[ks][1]);
                p[3] = pk_split<BF>(x[ks][2], x[ks][3]);
                if constexpr (THREE) {
                    p[4] = pk_split<BF>(x[ks][0], x[ks][1]);
                    p[5] = pk_split<BF>(x[ks][2], x[ks][3]);
                }
                if constexpr (QSM) {
                    if (ks % PK_WARPS == w)
#pragma unroll
                        for (int e = 0; e < QPARTS; e++) qsm[((mt * KS + ks) * QPARTS + e) * 32 + lane] = p[e];
                } else {
#pragma unroll
                    for (int e = 0; e < 4; e++) qr[mt][ks][e] = p[e];
                }
            }
        }
        if constexpr (QSM) __syncthreads();

        float o[MT][NT][4], m[MT], l[MT];
#pragma unroll
        for (int mt = 0; mt < MT; mt++) {
            m[mt] = -INFINITY;
            l[mt] = 0.0f;
#pragma unroll
            for (int t = 0; t < NT; t++)
#pragma unroll
                for (int e = 0; e < 4; e++) o[mt][t][e] = 0.0f;
        }

        /* ---- the warp's chunks of this segment */
        const uint32_t end = done + (uint32_t)(to - from);
        for (; next < end; next += PK_WARPS) {
            pk_cp_wait<PK_STAGES - 2>();
            __syncwarp();
            issue(stage + PK_STAGES - 1 < PK_STAGES ? stage + PK_STAGES - 1 : stage - 1);
            const uint32_t there = vmask[w][stage];
            const uint32_t ka = kbase + stage * S::STAGE, va = ka + CK * S::ROW;
            stage = stage + 1 == PK_STAGES ? 0 : stage + 1;
            if (!there) continue;
            const int32_t key0 = (cons.row.c0 + from + (int32_t)(next - done)) * CK;

#pragma unroll
            for (int mt = 0; mt < MT; mt++) {
                /* scores: keys are the columns */
                float s[KT][4], s3[THREE ? KT : 1][4];
#pragma unroll
                for (int t = 0; t < KT; t++)
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        s[t][e] = 0.0f;
                        if constexpr (THREE) s3[t][e] = 0.0f;
                    }
#pragma unroll
                for (int ks = 0; ks < KS; ks++) {
                    uint32_t a[QPARTS];
                    if constexpr (QSM) {
#pragma unroll
                        for (int e = 0; e < QPARTS; e++) a[e] = qsm[((mt * KS + ks) * QPARTS + e) * 32 + lane];
                    } else {
#pragma unroll
                        for (int e = 0; e < 4; e++) a[e] = qr[mt][ks][e];
                    }
                    if constexpr (!F8) {
                        /* 16 keys x 16 values at a time: matrices (keys 0-7, d 0-7), (0-7, 8-15), (8-15, 0-7), (8-15, 8-15) */
#pragma unroll
                        for (int t = 0; t < KT; t += 2) {
                            uint32_t b[4];
                            const uint32_t r = t * 8 + (lane >> 4) * 8 + (lane & 7u), u = ks * 2 + ((lane >> 3) & 1u);
                            pk_ldm4(b, ka + r * S::ROW + (u ^ (r & 7u)) * 16);
                            pk_mma<BF>(s[t], a[0], a[1], a[2], a[3], b[0], b[1]);
                            pk_mma<BF>(s[t + 1], a[0], a[1], a[2], a[3], b[2], b[3]);
                            if constexpr (THREE) {
                                pk_mma<BF>(s3[t], a[4], 0, a[5], 0, b[0], b[1]);
                                pk_mma<BF>(s3[t + 1], a[4], 0, a[5], 0, b[2], b[3]);
                            }
                        }
                    } else {
                        /* a matrix is 8 keys x 16 bytes; 16-key chunks take two k-steps at a time */
                        if constexpr (KT == 4) {
                            uint32_t b[4];
                            const uint32_t sw = S::ROW >= 128 ? (uint32_t)ks ^ (lane & 7u) : (uint32_t)ks ^ ((lane >> 1) & 3u);
                            pk_ldm4(b, ka + lane * S::ROW + sw * 16);
#pragma unroll
                            for (int t = 0; t < 4; t++)
                                pk_mma<BF>(s[t], a[0], a[1], a[2], a[3], pk_e4m3x2(b[t]), pk_e4m3x2(b[t] >> 16));
                        } else if (ks % 2 == 0) {
                            uint32_t b[4], a2[4];
                            const uint32_t r = lane & 15u, u = ks + (lane >> 4);
                            pk_ldm4(b, ka + r * S::ROW + (u ^ (r & 7u)) * 16);
#pragma unroll
                            for (int e = 0; e < 4; e++) {
                                if constexpr (QSM) a2[e] = qsm[((mt * KS + ks + 1) * QPARTS + e) * 32 + lane];
                                else a2[e] = qr[mt][ks + 1 < KS ? ks + 1 : ks][e];
                            }
#pragma unroll
                            for (int t = 0; t < 2; t++) {
                                pk_mma<BF>(s[t], a[0], a[1], a[2], a[3], pk_e4m3x2(b[t]), pk_e4m3x2(b[t] >> 16));
                                pk_mma<BF>(s[t], a2[0], a2[1], a2[2], a2[3], pk_e4m3x2(b[2 + t]),
                                           pk_e4m3x2(b[2 + t] >> 16));
                            }
                        }
                    }
                }
                /* fold the parts, mask, running maximum and sum: a lane has columns 2c, 2c + 1 of row g */
                const bool whole = there == (CK == 32 ? ~0u : (1u << (CK & 31)) - 1u) && key0 >= slo[mt] &&
                                   key0 + CK <= shi[mt];
                float p[KT][2], top = -INFINITY;
#pragma unroll
                for (int t = 0; t < KT; t++)
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        float x = pk_fold(s[t][e], THREE ? s[t][e + 2] + s3[t][e] : s[t][e + 2]) * unit[mt];
                        if (!whole) {
                            const int32_t k = t * 8 + 2 * (int32_t)c + e;
                            if (!(there >> k & 1u) || key0 + k < slo[mt] || key0 + k >= shi[mt]) x = -INFINITY;
                        }
                        p[t][e] = x;
                        top = fmaxf(top, x);
                    }
                top = fmaxf(top, __shfl_xor_sync(~0u, top, 1));
                top = fmaxf(top, __shfl_xor_sync(~0u, top, 2));
                top = fmaxf(top, m[mt]);
                /* weights are relative to the maximum less LIFT, so that small ones stay clear of f16's
                 * subnormals; nothing seen yet: every weight is 0 */
                const float zero = (top == -INFINITY ? 0.0f : top) - LIFT;
                const float keep = exp2f(m[mt] - LIFT - zero);
                if (__any_sync(~0u, top != m[mt])) {
                    l[mt] *= keep;
#pragma unroll
                    for (int t = 0; t < NT; t++)
#pragma unroll
                        for (int e = 0; e < 4; e++) o[mt][t][e] *= keep;
                }
                m[mt] = top;
#pragma unroll
                for (int t = 0; t < KT; t++)
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        p[t][e] = exp2f(p[t][e] - zero);
                        l[mt] += p[t][e];
                    }
                /* output: the weights are the left factor in the layout that they already have */
#pragma unroll
                for (int kt = 0; kt < KT; kt += 2) {
                    uint32_t a[6];
                    a[0] = pk_split<BF>(p[kt][0], p[kt][1]);
                    a[2] = pk_split<BF>(p[kt + 1][0], p[kt + 1][1]);
                    a[1] = pk_split<BF>(p[kt][0], p[kt][1]);
                    a[3] = pk_split<BF>(p[kt + 1][0], p[kt + 1][1]);
                    if constexpr (THREE) {
                        a[4] = pk_split<BF>(p[kt][0], p[kt][1]);
                        a[5] = pk_split<BF>(p[kt + 1][0], p[kt + 1][1]);
                    }
                    /* matrices (keys 0-7, unit u), (keys 8-15, u), (0-7, u + 1), (8-15, u + 1) */
                    const uint32_t r = kt * 8 + (lane & 15u), up = lane >> 4;
#pragma unroll
                    for (int u = 0; u < S::UNITS; u += 2) {
                        uint32_t b[4];
                        const uint32_t sw = S::ROW >= 128 ? (u + up) ^ (r & 7u) : (u + up) ^ ((r >> 1) & 3u);
                        pk_ldm4t(b, va + r * S::ROW + sw * 16);
                        if constexpr (!F8) {
                            pk_mma<BF>(o[mt][u], a[0], a[1], a[2], a[3], b[0], b[1]);
                            pk_mma<BF>(o[mt][u + 1], a[0], a[1], a[2], a[3], b[2], b[3]);
                            if constexpr (THREE) {
                                pk_mma<BF>(o[mt][u], a[4], 0, a[5], 0, b[0], b[1]);
                                pk_mma<BF>(o[mt][u + 1], a[4], 0, a[5], 0, b[2], b[3]);
                            }
                        } else {
                            /* a 16-bit column is two values: the even ones to tile 2u, the odd ones to 2u + 1 */
#pragma unroll
                            for (int y = 0; y < 2; y++) {
                                const uint32_t x0 = b[2 * y], x1 = b[2 * y + 1];
                                pk_mma<BF>(o[mt][2 * (u + y)], a[0], a[1], a[2], a[3], pk_e4m3x2(__byte_perm(x0, 0, 0x0020)),
                                           pk_e4m3x2(__byte_perm(x1, 0, 0x0020)));
                                pk_mma<BF>(o[mt][2 * (u + y) + 1], a[0], a[1], a[2], a[3],
                                           pk_e4m3x2(__byte_perm(x0, 0, 0x0031)), pk_e4m3x2(__byte_perm(x1, 0, 0x0031)));
                            }
                        }
                    }
                }
            }
        }

        /* ---- the four warps meet: maxima, then each quarter of the columns goes to one warp */
        const bool cut = from != 0 || to != cons.row.n;
        const uint32_t slot = 2 * blockIdx.x + (done != 0);
        const uint64_t part_floats = (uint64_t)HEADS * (DP + 2);
#pragma unroll
        for (int mt = 0; mt < MT; mt++) {
            l[mt] += __shfl_xor_sync(~0u, l[mt], 1);
            l[mt] += __shfl_xor_sync(~0u, l[mt], 2);
            if (c == 0) {
                wml[w][mt * 8 + g][0] = m[mt];
                wml[w][mt * 8 + g][1] = l[mt];
            }
        }
        __syncthreads();
#pragma unroll
        for (int mt = 0; mt < MT; mt++) {
            if (mt) __syncthreads(); /* the previous tile's sums are out of `join` */
            float top = -INFINITY, sum = 0.0f;
#pragma unroll
            for (uint32_t k = 0; k < PK_WARPS; k++) top = fmaxf(top, wml[k][mt * 8 + g][0]);
            const float zero = top == -INFINITY ? 0.0f : top;
#pragma unroll
            for (uint32_t k = 0; k < PK_WARPS; k++) sum += wml[k][mt * 8 + g][1] * exp2f(wml[k][mt * 8 + g][0] - LIFT - zero);
            const float keep = exp2f(m[mt] - LIFT - zero);
            if (w == 0 && c == 0) {
                fml[mt * 8 + g][0] = top;
                fml[mt * 8 + g][1] = sum;
            }
#pragma unroll
            for (int t = 0; t < NT; t++) {
                o[mt][t][0] = pk_fold(o[mt][t][0], o[mt][t][2]) * keep;
                o[mt][t][1] = pk_fold(o[mt][t][1], o[mt][t][3]) * keep;
            }
            /* column of (tile t, element e) within its quarter: a lane's run of 2 (16-bit) or 4 (e4m3) columns */
            constexpr int QT = NT / 4, RUN = F8 ? 4 : 2;
            auto place = [&](uint32_t owner, uint32_t source, int tq) {
                return join + ((owner * 3 + source) * 8 + g) * S::QROW + (F8 ? tq * 8 + 4 * c : tq * 8 + 2 * c);
            };
#pragma unroll
            for (uint32_t q = 0; q < 4; q++)
                if (q != w)
#pragma unroll
                    for (int t = 0; t < QT; t += RUN / 2) {
                        float *d = place(q, w < q ? w : w - 1, t);
                        const float *x = o[mt][q * QT + t];
                        if constexpr (F8) {
                            const float *y = o[mt][q * QT + t + 1];
                            *(float4 *)d = make_float4(x[0], y[0], x[1], y[1]);
                        } else {
                            *(float2 *)d = make_float2(x[0], x[1]);
                        }
                    }
            __syncthreads();
#pragma unroll
            for (uint32_t q = 0; q < 4; q++)
                if (q == w)
#pragma unroll
                    for (int t = 0; t < QT; t += RUN / 2) {
                        const float *x = o[mt][q * QT + t];
                        float own[RUN], sum4[RUN];
                        own[0] = x[0];
                        if constexpr (F8) {
                            const float *y = o[mt][q * QT + t + 1];
                            own[1] = y[0];
                            own[2] = x[1];
                            own[3] = y[1];
                        } else {
                            own[1] = x[1];
                        }
#pragma unroll
                        for (int e = 0; e < RUN; e++) sum4[e] = 0.0f;
#pragma unroll
                        for (uint32_t k = 0; k < 4; k++)
#pragma unroll
                            for (int e = 0; e < RUN; e++) sum4[e] += k == q ? own[e] : place(q, k < q ? k : k - 1, t)[e];
                        float *d = place(q, 0, t);
#pragma unroll
                        for (int e = 0; e < RUN; e++) d[e] = sum4[e];
                    }
            __syncthreads();

            /* ---- out, or into the workspace */
            for (uint32_t x = tid; x < 8 * DP / 4; x += PK_WARPS * 32) {
                const uint32_t hh = x / (DP / 4), col = x % (DP / 4) * 4, q = col / (DP / 4);
                const float4 v = *(const float4 *)(join + ((q * 3) * 8 + hh) * S::QROW + col % (DP / 4));
                const uint32_t head = mt * 8 + hh;
                if (cut) {
                    float *part = J.parts + slot * part_floats;
                    __stcg((float4 *)(part + 2 * HEADS + head * DP + col), v);
                    if (col == 0) __stcg((float2 *)(part + 2 * head), make_float2(fml[head][0], fml[head][1]));
                } else {
                    pk_attend_out<DP>(J, cons.b, cons.row.len, hk, v0 + head, col, fml[head][0], fml[head][1], v);
                }
            }
        }
        if (cut) {
            const unsigned long long seg0 = base - (uint32_t)from, seg1 = seg0 + (uint32_t)cons.row.n;
            const uint32_t w0 = (uint32_t)(seg0 / per), w1 = (uint32_t)((seg1 - 1) / per);
            pk_attend_join<DP, MT>(J, cons.b, cons.row.len, hk, v0, w0, w1, seg0 > per * w0, &last, fml);
        }
        __syncthreads(); /* wml, fml, join and qsm are free again */

        const uint32_t took = (uint32_t)(to - from);
        done += took;
        base += took;
        if (done < slice) cons.step(J, (int32_t)took);
    }
    pk_cp_wait<0>();
}

template <uint32_t CT, int DP, int MT, bool THREE>
static int pk_attend_launch(const pk_attend_job &J, uint32_t grid, cudaStream_t st) {
    typedef pk_shape<CT, DP> S;
    static uint64_t done = 0;
    constexpr uint32_t smem = PK_WARPS * S::RING + S::JOIN;
    auto kernel = pk_attend_kernel<CT, DP, MT, THREE>;
    if (!pm_smem_attr(kernel, smem, &done)) return 0;
    kernel<<<grid, PK_WARPS * 32, smem, st>>>(J);
    return pm_ok(cudaGetLastError(), "kv attend launch");
}

/* one translation unit per cache type (kv_attend_*.cu) */
typedef int (*pk_attend_fn)(const pk_attend_job &, uint32_t, cudaStream_t);
pk_attend_fn pk_attend_bf16(int dp, int mt, bool three);
pk_attend_fn pk_attend_f16(int dp, int mt, bool three);
pk_attend_fn pk_attend_e4m3(int dp, int mt, bool three);

template <uint32_t CT, bool THREE>
static pk_attend_fn pk_attend_pick(int dp, int mt) {
    if (dp == 64) return mt == 2 ? pk_attend_launch<CT, 64, 2, THREE> : pk_attend_launch<CT, 64, 1, THREE>;
    if (dp == 128) return mt == 2 ? pk_attend_launch<CT, 128, 2, THREE> : pk_attend_launch<CT, 128, 1, THREE>;
    return pk_attend_launch<CT, 256, 1, THREE>;
}
