/* kv_append.cu - rotary positions fused with the cache write.
 *
 *   (a, b) -> (a c - b s, b c + a s)   pairs of q's and k's heads,
 * q' to q_out, k' and v to token pos % page_size of page table[seq][pos /
 * page_size].  Every value is read once and written once (bytes bound: a
 * handful of operations per value), so the kernel is a copy with addresses:
 * a thread owns one item of a token - V pairs of a head, or V values that
 * only pass through (the unrotated part, v) - works its place out once and
 * takes that item of many tokens.  V = 8 moves 16 bytes of a 16-bit type per
 * load; 4, 2 and 1 serve rotary widths, strides and addresses that are not
 * multiples of that. */
#include "pk_common.h"

struct pk_append_geo {
    uint32_t pairs;  /* items of V pairs per rotated head */
    uint32_t head;   /* items per q or k head */
    uint32_t vhead;  /* items per v head */
    uint32_t items;  /* items per token */
};

template <class T, int V>
struct __align__(sizeof(T) * V > 16 ? 16 : sizeof(T) * V) pk_vec {
    T v[V];
};

template <uint32_t X, int V>
__device__ __forceinline__ void pk_load(const void *base, uint64_t at, float *x) {
    typedef typename pk_type<X>::t T;
    const pk_vec<T, V> r = *(const pk_vec<T, V> *)((const T *)base + at);
#pragma unroll
    for (int i = 0; i < V; i++) x[i] = pk_type<X>::get(r.v[i]);
}

template <uint32_t Y, int V>
__device__ __forceinline__ void pk_store_as(void *base, uint64_t at, const float *x) {
    typedef typename pk_type<Y>::t T;
    pk_vec<T, V> r;
#pragma unroll
    for (int i = 0; i < V; i++) r.v[i] = pk_type<Y>::put(x[i]);
    *(pk_vec<T, V> *)((T *)base + at) = r;
}

template <int V>
__device__ __forceinline__ void pk_store(void *base, uint32_t type, uint64_t at, const float *x) {
    if (type == PULSAR_TYPE_BF16) pk_store_as<PULSAR_TYPE_BF16, V>(base, at, x);
    else if (type == PULSAR_TYPE_F16) pk_store_as<PULSAR_TYPE_F16, V>(base, at, x);
    else if (type == PULSAR_TYPE_E4M3) pk_store_as<PULSAR_TYPE_E4M3, V>(base, at, x);
    else pk_store_as<PULSAR_TYPE_F32, V>(base, at, x);
}

/* blockDim (items, tokens); grid (item blocks, token blocks) */
template <uint32_t X, int V>
__global__ void __launch_bounds__(256)
    pk_append_kernel(const pulsar_kv_desc D, const pulsar_kv_append_args A, const pk_append_geo G, uint32_t *err) {
    const uint32_t it = blockIdx.x * blockDim.x + threadIdx.x;
    if (it >= G.items) return;
    const uint32_t n_turn = (A.n_head + D.n_kv) * G.head;
    const bool is_v = it >= n_turn;
    const uint32_t per = is_v ? G.vhead : G.head;
    const uint32_t h_all = (is_v ? it - n_turn : it) / per, j = (is_v ? it - n_turn : it) % per;
    const bool is_q = !is_v && h_all < A.n_head;
    const uint32_t h = is_v || is_q ? h_all : h_all - A.n_head; /* head within q, k or v */
    const bool turn = !is_v && j < G.pairs;
    const uint32_t half = A.rot_dim / 2;
    /* first value of the item; a turned item has a second run of V values at o1 */
    const uint32_t o0 = is_v ? j * V : !turn ? A.rot_dim + (j - G.pairs) * V : A.interleaved ? j * 2 * V : j * V;
    const uint32_t o1 = A.interleaved ? o0 + V : o0 + half;
    const void *in = is_v ? A.v : is_q ? A.q : A.k;
    const uint64_t in_stride = is_v ? A.v_stride : is_q ? A.q_stride : A.k_stride;
    void *cache = is_v ? D.v : D.k;
    const float *scale = is_v ? D.v_scale : D.k_scale;
    const float sc = !is_q && scale ? scale[h] : 1.0f;

    /* one latency a token: x's loads wait for nothing, and the token's
     * position and row were loaded a token ahead */
    const uint32_t step = gridDim.y * blockDim.y;
    uint32_t t = blockIdx.y * blockDim.y + threadIdx.y;
    int32_t pos = -1, seq = -1;
    if (t < A.n_tok) {
        pos = __ldg(A.pos + t);
        seq = __ldg(A.seq + t);
    }
    for (int32_t pos2 = -1, seq2 = -1; t < A.n_tok; t += step, pos = pos2, seq = seq2) {
        float x[2 * V];
        const uint64_t from = t * in_stride + (uint64_t)h * D.head_dim;
        pk_load<X, V>(in, from + o0, x);
        if (turn) pk_load<X, V>(in, from + o1, x + V);
        if (A.n_tok - t > step) {
            pos2 = __ldg(A.pos + t + step);
            seq2 = __ldg(A.seq + t + step);
        }
        if (pos < 0 || seq < 0) continue;
        if (turn) {
            if ((uint32_t)pos >= A.n_pos) {
                atomicOr(err, PULSAR_KV_ERR_SPAN);
                continue;
            }
            const float *cs = A.cos_sin + (uint64_t)pos * A.rot_dim + (uint64_t)j * V;
            const pk_vec<float, V> c4 = *(const pk_vec<float, V> *)cs, s4 = *(const pk_vec<float, V> *)(cs + half);
            const float *c = c4.v, *s = s4.v;
            if (A.interleaved) {
#pragma unroll
                for (int i = 0; i < V; i++) {
                    const float a = x[2 * i], b = x[2 * i + 1];
                    x[2 * i] = a * c[i] - b * s[i];
                    x[2 * i + 1] = b * c[i] + a * s[i];
                }
            } else {
#pragma unroll
                for (int i = 0; i < V; i++) {
                    const float a = x[i], b = x[V + i];
                    x[i] = a * c[i] - b * s[i];
                    x[V + i] = b * c[i] + a * s[i];
                }
            }
        }
        uint64_t to;
        void *out;
        uint32_t type;
        if (is_q) {
            out = A.q_out;
            type = A.q_out_type;
            to = t * A.q_out_stride + (uint64_t)h * D.head_dim;
        } else {
            const uint32_t slot = (uint32_t)pos / D.page_size;
            if ((uint32_t)seq >= D.n_rows || slot >= D.max_pages) {
                atomicOr(err, (uint32_t)seq >= D.n_rows ? PULSAR_KV_ERR_ROW : PULSAR_KV_ERR_SPAN);
                continue;
            }
            const int32_t page = __ldg(D.table + (uint64_t)seq * D.table_stride + slot);
            if ((uint32_t)page >= D.n_pages) {
                atomicOr(err, PULSAR_KV_ERR_PAGE);
                continue;
            }
            out = cache;
            type = D.dtype;
            to = (uint64_t)page * D.page_stride + h * D.head_stride + ((uint32_t)pos % D.page_size) * D.tok_stride;
            if (scale) {
#pragma unroll
                for (int i = 0; i < 2 * V; i++) x[i] /= sc;
            }
        }
        pk_store<V>(out, type, to + o0, x);
        if (turn) pk_store<V>(out, type, to + o1, x + V);
    }
}

template <uint32_t X, int V>
static int pk_append_launch(const pulsar_kv_desc *d, const pulsar_kv_append_args *a, cudaStream_t st) {
    pk_append_geo g;
    g.pairs = a->rot_dim / 2 / V;
    g.head = g.pairs + (d->head_dim - a->rot_dim) / V;
    g.vhead = d->head_dim / V;
    g.items = (a->n_head + d->n_kv) * g.head + d->n_kv * g.vhead;
    dim3 block(g.items >= 256 ? 256 : (g.items + 31u) & ~31u, 1), grid((g.items + block.x - 1) / block.x);
    block.y = 256 / block.x;
    /* about 16 CTAs to an SM where there are that many tokens: past that a
     * thread takes more tokens of its item */
    uint32_t y = (a->n_tok + block.y - 1) / block.y;
    const uint32_t most = (16 * pk_sm_count() + grid.x - 1) / grid.x;
    grid.y = y < most ? y : most;
    pk_append_kernel<X, V><<<grid, block, 0, st>>>(*d, *a, g, pk_err_word());
    return pm_ok(cudaGetLastError(), "kv append launch");
}

template <uint32_t X>
static int pk_append_by_width(const pulsar_kv_desc *d, const pulsar_kv_append_args *a, cudaStream_t st) {
    /* the widest run of values that every part of a head and every address
     * is a multiple of (head_dim is a multiple of 16, cache rows of 16 bytes) */
    const uint32_t xe = pk_type_bytes(a->x_type), qe = pk_type_bytes(a->q_out_type);
    for (uint32_t v = 8; v > 1; v /= 2) {
        const uint32_t xb = xe * v > 16 ? 16 : xe * v, qb = qe * v > 16 ? 16 : qe * v;
        const uint32_t cb = v < 4 ? 4 * v : 16; /* the angles' loads */
        uint64_t odd = (uintptr_t)a->cos_sin % cb;
        odd |= ((uintptr_t)a->k | (uintptr_t)a->v | a->k_stride * xe | a->v_stride * xe) % xb;
        if (a->n_head)
            odd |= ((uintptr_t)a->q | a->q_stride * xe) % xb | ((uintptr_t)a->q_out | a->q_out_stride * qe) % qb;
        if (odd || a->rot_dim / 2 % v) continue;
        if (v == 8) return pk_append_launch<X, 8>(d, a, st);
        if (v == 4) return pk_append_launch<X, 4>(d, a, st);
        return pk_append_launch<X, 2>(d, a, st);
    }
    return pk_append_launch<X, 1>(d, a, st);
}

extern "C" int pulsar_kv_append(const pulsar_kv_desc *d, const pulsar_kv_append_args *a, void *stream) {
    const char *f = pk_desc_fault(d);
    if (f) return pk_refuse(f);
    if (!a || !a->k || !a->v || !a->seq || !a->pos) return pk_refuse("kv append: null arguments");
    if (a->n_head && (!a->q || !a->q_out)) return pk_refuse("kv append: query heads without q or q_out");
    if (a->x_type > PULSAR_TYPE_F16 || a->q_out_type > PULSAR_TYPE_F16)
        return pk_refuse("kv append: values are f32, bf16 or f16");
    if (a->rot_dim % 2 || a->rot_dim > d->head_dim) return pk_refuse("kv append: rot_dim is even and within the head");
    if (a->rot_dim && (!a->cos_sin || !a->n_pos)) return pk_refuse("kv append: a rotation without its table");
    if (a->n_head > 0xffffu || d->n_kv > 0xffffu) return pk_refuse("kv append: too many heads");
    if (!a->n_tok || a->n_tok > 0x7fffffffu) return pk_refuse("kv append: between 1 and 2^31 - 1 tokens");
    const uint64_t kv = (uint64_t)d->n_kv * d->head_dim, q = (uint64_t)a->n_head * d->head_dim;
    if (a->n_tok > 1 && (a->k_stride < kv || a->v_stride < kv || (a->n_head && (a->q_stride < q || a->q_out_stride < q))))
        return pk_refuse("kv append: tokens overlap");
    if (!pk_err_word()) return pk_refuse("kv: no error word on this device");
    const cudaStream_t st = pk_stream(stream);
    if (a->x_type == PULSAR_TYPE_F32) return pk_append_by_width<PULSAR_TYPE_F32>(d, a, st);
    if (a->x_type == PULSAR_TYPE_BF16) return pk_append_by_width<PULSAR_TYPE_BF16>(d, a, st);
    return pk_append_by_width<PULSAR_TYPE_F16>(d, a, st);
}
