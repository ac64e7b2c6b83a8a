/* kv_attend.cu - attention over a paged cache: arguments, the choice of a
 * kernel, the workspace (the kernels are in pk_attend.cuh). */
#include "pk_attend.cuh"

/* what a call's sizes settle */
struct pk_attend_plan {
    int dp, r;               /* padded head width; the kernel's R */
    bool wide;               /* q has more bits than one 16-bit part of the cache's kind holds */
    uint32_t workers, rows;  /* CTAs and sequences of a launch */
    size_t bytes;            /* of the workspace */
};

static uint32_t pk_attend_width(const pulsar_kv_desc *d) {
    return d->head_dim <= 64    ? 64
           : d->head_dim <= 96  ? 96
           : d->head_dim <= 128 ? 128
           : d->head_dim <= 192 && d->dtype != PULSAR_TYPE_E4M3 ? 192 : 256;
}

/* two CTAs an SM (pk_shape's OCC; one where q's parts at 256 columns leave no
 * room for two) */
static uint32_t pk_attend_workers() {
    const uint32_t n = pk_sm_count() * 2;
    return n < PK_MAX_WORKERS ? n : PK_MAX_WORKERS;
}

/* a worker has two parts of `heads` rows */
static size_t pk_attend_bytes(uint32_t workers, uint32_t heads, uint32_t dp) {
    return PULSAR_KV_WS_ZEROED + 4ull * workers * 2 * heads * (dp + 2);
}

static int pk_attend_prepare(const pulsar_kv_desc *d, const pulsar_kv_attend_args *a, pk_attend_job *J,
                             pk_attend_plan *p) {
    const char *f = pk_desc_fault(d);
    if (f) return pk_refuse(f);
    if (!a) return pk_refuse("kv attend: null arguments");
    if (a->q_type > PULSAR_TYPE_F16) return pk_refuse("kv attend: values are f32, bf16 or f16");
    if (!a->n_head || a->n_head > 0xffffu || a->n_head % d->n_kv)
        return pk_refuse("kv attend: n_head is a multiple of n_kv, at most 65535");
    if (!a->n_rows || !a->n_q || (uint64_t)a->n_rows * a->n_q > 0x7fffffffull ||
        (uint64_t)a->n_q * a->n_head > 0x7fffffffull)
        return pk_refuse("kv attend: between 1 and 2^31 - 1 tokens");
    J->D = *d;
    J->A = *a;
    J->group = a->n_head / d->n_kv;
    J->rows = a->n_q * J->group;
    p->dp = (int)pk_attend_width(d);
    /* q in one part: the cache's own 16-bit type, or bf16 (8 bits) beside f16 and e4m3 */
    p->wide = a->q_type == PULSAR_TYPE_F32 || (d->dtype == PULSAR_TYPE_BF16 && a->q_type == PULSAR_TYPE_F16);
    /* a tile of 16 query rows, or of 8 where there are no more.  (32, with two
     * matrix tiles to a reading of the keys, measured the same as two tiles of
     * 16: 70 us at 16 sequences of up to 9001 keys and 28 rows.) */
    p->r = J->rows > 8 ? 2 : 1;
    const uint32_t heads = 8u * p->r;
    J->tiles = (J->rows + heads - 1) / heads;
    if ((uint64_t)J->tiles * d->n_kv > 0x7fffffffull) return pk_refuse("kv attend: too many heads and tokens");
    J->segs = J->tiles * d->n_kv;
    J->page_shift = d->page_size & (d->page_size - 1) ? -1 : __builtin_ctz(d->page_size);
    const uint32_t qe = pk_type_bytes(a->q_type);
    J->pairs = (((uintptr_t)a->q | a->q_stride * qe) % (2 * qe)) == 0;
    const uint32_t ck = PK_CK((p->dp == 96 ? 128 : p->dp) * pk_type_bytes(d->dtype));
    J->least = 128 / ck;
    p->workers = pk_attend_workers();
    /* no more CTAs than the longest rows could feed; no more rows in a launch
     * than a line of less than 2^32 chunks holds */
    uint64_t keys = (uint64_t)d->max_pages * d->page_size;
    if (a->window && keys > (uint64_t)a->window + a->n_q - 1) keys = (uint64_t)a->window + a->n_q - 1;
    const uint64_t row = (uint64_t)J->segs * (keys / ck + 2 + 3); /* 3: the kernel's cost of a segment */
    if (row > 0x7fffffffull) return pk_refuse("kv attend: a row too long for its heads");
    p->rows = 0xffffffffull / row < a->n_rows ? (uint32_t)(0xffffffffull / row) : a->n_rows;
    if (p->workers > row * p->rows) p->workers = (uint32_t)(row * p->rows);
    p->bytes = pk_attend_bytes(p->workers, heads, p->dp);
    return 1;
}
static_assert(4 * 2 * 2 * PK_MAX_WORKERS <= PULSAR_KV_WS_ZEROED, "the counters are in the zeroed bytes");

extern "C" size_t pulsar_kv_attend_workspace(const pulsar_kv_desc *d, const pulsar_kv_attend_args *a) {
    pk_attend_job J;
    pk_attend_plan p;
    if (!a) {
        if (const char *f = pk_desc_fault(d)) return (size_t)pk_refuse(f);
        const uint32_t dp = pk_attend_width(d);
        return pk_attend_bytes(pk_attend_workers(), 16, dp);
    }
    return pk_attend_prepare(d, a, &J, &p) ? p.bytes : 0;
}

extern "C" int pulsar_kv_attend(const pulsar_kv_desc *d, const pulsar_kv_attend_args *a, void *ws, size_t ws_bytes,
                                void *stream) {
    pk_attend_job J;
    pk_attend_plan p;
    if (!pk_attend_prepare(d, a, &J, &p)) return 0;
    if (!a->q || !a->out || !a->lens || !ws || ((uintptr_t)ws & 15u)) return pk_refuse("kv attend: null arguments");
    if (!a->seq && a->n_rows > d->n_rows) return pk_refuse("kv attend: more rows than the table has");
    const uint64_t w = (uint64_t)a->n_head * d->head_dim;
    if ((uint64_t)a->n_rows * a->n_q > 1 && (a->q_stride < w || a->out_stride < w))
        return pk_refuse("kv attend: tokens overlap");
    if (ws_bytes < p.bytes) return pk_refuse("kv attend: workspace too small");
    J.counters = (uint32_t *)ws;
    J.parts = (float *)((uint8_t *)ws + PULSAR_KV_WS_ZEROED);
    J.err = pk_err_word();
    if (!J.err) return pk_refuse("kv: no error word on this device");
    const pk_attend_fn f = d->dtype == PULSAR_TYPE_BF16  ? pk_attend_bf16(p.dp, p.r, p.wide)
                           : d->dtype == PULSAR_TYPE_F16 ? pk_attend_f16(p.dp, p.r, p.wide)
                                                         : pk_attend_e4m3(p.dp, p.r, p.wide);
    for (uint32_t r = 0; r < a->n_rows; r += p.rows) {
        J.A.n_rows = a->n_rows - r < p.rows ? a->n_rows - r : p.rows;
        if (!f(J, p.workers, pk_stream(stream))) return 0;
        const uint64_t tok = (uint64_t)p.rows * a->n_q;
        J.A.q = (const uint8_t *)J.A.q + tok * a->q_stride * pk_type_bytes(a->q_type);
        J.A.out = (uint8_t *)J.A.out + tok * a->out_stride * pk_type_bytes(a->q_type);
        if (J.A.lse) J.A.lse += tok * a->n_head;
        J.A.lens += p.rows;
        if (J.A.seq) {
            J.A.seq += p.rows;
        } else {
            J.D.table += p.rows * J.D.table_stride;
            J.D.n_rows -= p.rows;
        }
    }
    return 1;
}
