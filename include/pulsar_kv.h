/* pulsar_kv.h - C ABI of the paged key/value cache in libpulsar_moe.so:
 * rotary positions with the cache write, attention of new tokens over the
 * cache, and the page bookkeeping (growth, fork, compaction), all on the
 * device.  With the expert layer of pulsar_moe.h they make a decoder layer.
 *
 * Conventions are those of pulsar_moe.h: 1 = launched, 0 = refused (invalid
 * arguments or a launch error, with a message on stderr); every pointer is
 * device memory of the caller on the current device; launches go to `stream`
 * (cudaStream_t, NULL = the calling thread's default stream); nothing
 * allocates or synchronises, so the calls can be captured into a graph (the
 * first call on a device loads the kernels there: make it before a capture).
 *
 * What only the device sees (page ids, lengths, positions, rows) is checked
 * there: an entry that is out of range is not followed, and a bit of the
 * family's error word says so (pulsar_kv_error).
 */
#ifndef PULSAR_KV_H
#define PULSAR_KV_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define PULSAR_TYPE_F32 0u
#define PULSAR_TYPE_BF16 1u
#define PULSAR_TYPE_F16 2u
#define PULSAR_TYPE_E4M3 3u /* caches only */

/* error word bits */
#define PULSAR_KV_ERR_PAGE 1u /* a page id outside [0, n_pages); compact: a page that no count holds, behind the live ones */
#define PULSAR_KV_ERR_SPAN 2u /* a length or position past the table's width or the position table's end */
#define PULSAR_KV_ERR_ROW 4u  /* a table row outside [0, n_rows) */

/* One layer's cache.  Token t of sequence row r and key head h is the
 * head_dim values at page table[r * table_stride + t / page_size]:
 *   k + page * page_stride + h * head_stride + (t % page_size) * tok_stride
 * (strides in values; v alike).  Each token's row of a head is contiguous;
 * k, v and the strides are multiples of 16 bytes.  head_dim: a multiple of
 * 16, at most 256.  page_size: any.  dtype: BF16, F16 or E4M3; an e4m3
 * value of key head h stands for value * k_scale[h] (v_scale[h]); NULL
 * scales are 1 (and must be NULL for the other types). */
typedef struct pulsar_kv_desc {
    void *k, *v;
    const int32_t *table;
    const float *k_scale, *v_scale; /* [n_kv] or NULL */
    uint64_t page_stride, head_stride, tok_stride;
    uint64_t table_stride; /* entries between table rows */
    uint32_t n_pages, page_size, n_kv, head_dim;
    uint32_t n_rows, max_pages; /* table rows, entries used of each */
    uint32_t dtype;
} pulsar_kv_desc;

/* Rotary positions fused with the cache write.  For each token t, with
 * position p = pos[t] and angle table row (c, s) = cos_sin[p]:
 *   half layout:        pairs (x[i], x[i + rot_dim/2]),  i < rot_dim/2
 *   interleaved layout: pairs (x[2i], x[2i + 1])
 *   (a, b) -> (a c_i - b s_i, b c_i + a s_i); values from rot_dim on stay
 * q's heads are turned into q_out; k's heads are turned and written with
 * v's at token p of table row seq[t].  The arithmetic is in 32 bits,
 * rounded once on the way out (e4m3: value / scale, saturating).
 * A token with pos < 0 or seq < 0 is padding: nothing of it is written.
 * Two tokens of one call may not name the same place.
 * cos_sin: f32 [n_pos][2][rot_dim / 2], cosines first (a longer context's
 * scaling is in the table).  rot_dim even, 0 = no rotation (cos_sin NULL).
 * q NULL with n_head 0: keys and values only.  q_out may be q where types
 * and strides agree.  Strides in values between tokens, heads head_dim
 * apart. */
typedef struct pulsar_kv_append_args {
    const void *q, *k, *v;
    void *q_out;
    const int32_t *seq, *pos; /* [n_tok] */
    const float *cos_sin;
    uint64_t q_stride, k_stride, v_stride, q_out_stride;
    uint32_t n_tok, n_head, rot_dim, n_pos;
    uint32_t x_type, q_out_type; /* F32, BF16 or F16: of q, k, v; of q_out */
    uint32_t interleaved;
} pulsar_kv_append_args;
int pulsar_kv_append(const pulsar_kv_desc *d, const pulsar_kv_append_args *a, void *stream);

/* Attention of n_q new tokens of each of n_rows sequences over their
 * cached keys (the new tokens' own, already appended, among them).  Row b
 * reads table row seq[b] (NULL: b) and has lens[b] keys; its token i sees
 * the keys j with
 *   lo <= j < hi,  hi = lens[b] - (n_q - 1 - i),  lo = window ? max(0, hi - window) : 0
 *   o = sum_j e^(scale q.k_j - m) v_j / (sum_j e^(scale q.k_j - m) + e^(sinks[h] - m))
 * (the last term only with sinks).  A token that sees no key gets zeros and
 * lse -inf; seq[b] < 0 marks a padding row, which sees none.  lse, if not
 * NULL: f32 [n_rows][n_q][n_head], the logarithm of the denominator plus m.
 * q, out: [n_rows * n_q] tokens of n_head heads of head_dim values of
 * q_type, q_stride / out_stride values apart.  n_head is a multiple of
 * n_kv; query head h reads key head h / (n_head / n_kv).  Keys beyond a
 * token's span have no influence, whatever their bytes are; an infinite or
 * NaN score or value that is seen gives what the formula gives, or NaN.  (Where
 * a value that some of a sequence's n_q tokens see and others do not is
 * infinite or NaN, the outputs of those that see it are NaN throughout; lse,
 * which no value enters, is what the formula gives.)
 * ws: pulsar_kv_attend_workspace bytes (with a NULL: enough for any
 * arguments over this cache), aligned to 16; its first PULSAR_KV_WS_ZEROED bytes
 * are zero before the first call and are zero again after every call.  One
 * ws serves any sequence of calls on one stream. */
typedef struct pulsar_kv_attend_args {
    const void *q;
    void *out;
    float *lse;
    const int32_t *lens, *seq;
    const float *sinks; /* [n_head] or NULL */
    uint64_t q_stride, out_stride;
    float scale;
    uint32_t n_rows, n_q, n_head, window, q_type;
} pulsar_kv_attend_args;
#define PULSAR_KV_WS_ZEROED 32768u
size_t pulsar_kv_attend_workspace(const pulsar_kv_desc *d, const pulsar_kv_attend_args *a);
int pulsar_kv_attend(const pulsar_kv_desc *d, const pulsar_kv_attend_args *a, void *ws, size_t ws_bytes, void *stream);

/* The bookkeeping of a cache's pages, shared by all its layers: row r holds
 * len[r] tokens in the pages table[r * table_stride + 0 .. ceil(len[r] /
 * page_size) - 1]; refs[p] rows hold page p (0 = free).  The bytes of page p
 * are those at data + s * slab_stride + p * page_bytes for every slab s
 * (keys and values of each layer).  A page that is not full has one holder:
 * fork keeps that so. */
typedef struct pulsar_kv_pool {
    int32_t *table, *len, *refs;
    void *data;
    uint64_t slab_stride, page_bytes; /* bytes */
    uint64_t table_stride;            /* entries */
    uint32_t n_rows, max_pages, n_pages, page_size, n_slab;
} pulsar_kv_pool;

/* status words (int32[4], device, 16-byte aligned like ws) of the three calls: [0] what happened,
 * [1] pages taken or moved, [2] pages that were free before (grow, fork) or
 * are live (compact).  Unless [0] is PULSAR_KV_OK nothing was changed. */
#define PULSAR_KV_OK 0
#define PULSAR_KV_SHORT 1   /* fewer free pages than the call needs */
#define PULSAR_KV_WIDE 2    /* a row would outgrow max_pages */
#define PULSAR_KV_INVALID 3 /* a row out of range or named twice, a length or count out of range */

/* Row rows[i] (NULL: i) grows by n_new[i] >= 0 tokens: len grows, and the
 * pages that it lacks are the lowest free ones, in the order of i. */
int pulsar_kv_grow(const pulsar_kv_pool *p, const int32_t *rows, const int32_t *n_new, uint32_t n, int32_t *status,
                   void *ws, size_t ws_bytes, void *stream);

/* Row dst[i] becomes what row src[i] was before the call (src -1: empty),
 * for all i at once, so that any reordering of beams is one call; dst rows
 * are distinct, rows not in dst stay.  Pages are shared, but for a partly
 * filled last page: it stays with src[i] itself if that row stays (or
 * continues itself), else with the first i that names it, and every other i
 * gets a copy in the lowest page free before the call, in the order of i. */
int pulsar_kv_fork(const pulsar_kv_pool *p, const int32_t *dst, const int32_t *src, uint32_t n, int32_t *status,
                   void *ws, size_t ws_bytes, void *stream);

/* With n live pages, the live pages from n on move to the free ones below
 * it, lowest to lowest; tables and reference counts follow. */
int pulsar_kv_compact(const pulsar_kv_pool *p, int32_t *status, void *ws, size_t ws_bytes, void *stream);

/* bytes of workspace of the three calls (n: rows named in one call, at most
 * PULSAR_KV_MAX_FORK for fork); its contents carry nothing between calls */
#define PULSAR_KV_MAX_FORK 4096u
size_t pulsar_kv_pool_workspace(const pulsar_kv_pool *p, uint32_t n);

/* reads and clears the family's error word on the current device (waits for the device) */
uint32_t pulsar_kv_error(void);

#ifdef __cplusplus
}
#endif
#endif
