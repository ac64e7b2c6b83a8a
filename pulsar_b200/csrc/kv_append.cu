/* kv_append.cu - rotary positions fused with the cache write.
 *
 *   (a, b) -> (a c - b s, b c + a s)   pairs of q's and k's heads,
 * q' to q_out, k' and v to token pos % page_size of page table[seq][pos /
 * page_size].  Every value is read once and written once (bytes bound: a
 * handful of operations per value), so the kernel is a copy with addresses:
 * a thread owns one item of a token, works its place out once and takes that
 * item of many tokens.  An item is a run of V values at the same place of HU
 * neighbouring heads, values that only pass through (the unrotated part, v)
 * or V / 2 interleaved pairs, or, in the half layout, V values and their V
 * partners.  V values are 16 bytes (8 of a 16-bit type, 4 of f32), so that a
 * warp's loads and stores are whole runs; 4, 2 and 1 serve rotary widths,
 * strides and addresses that are not multiples of that.  HU = 4 (2 in the half
 * layout, whose items are twice as wide) has four loads in flight per thread
 * and reads a token's angles once for its heads; where there are too few
 * tokens for that, HU = 1 spreads a token wider.  Measured: 8 x 2048 tokens of
 * 64 + 8 + 8 f16 heads of 128, interleaved: 122 to 127 us, 5.5 TB/s (with one 16-byte
 * run a thread 211 us: too few loads in flight); one token: 2.2 us. */
#include "pk_common.h"

struct pk_append_geo {
    uint32_t turned; /* items of a head that rotate */
    uint32_t head;   /* items per q or k head group */
    uint32_t vhead;  /* items per v head group */
    uint32_t q, kv;  /* head groups of q; of k, and of v */
    uint32_t items;  /* items per token */
};

template <class T, int V>
struct __align__(sizeof(T) * V > 16 ? 16 : sizeof(T) * V) pk_vec {
    T v[V];
};

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
template <uint32_t X, int V, bool NEAR, int HU>
__global__ void __launch_bounds__(256, V == 8 && !NEAR && HU > 1 ? 3 : 4) /* 64 KB of loads in flight an SM; no spills to speak of */
    pk_append_kernel(const pulsar_kv_desc D, const pulsar_kv_append_args A, const pk_append_geo G, uint32_t *err) {
    typedef typename pk_type<X>::t T;
    constexpr int P = NEAR ? V / 2 : V;                    /* pairs of an item */
    const uint32_t it = blockIdx.x * blockDim.x + threadIdx.x;
    pk_enter();
    if (it >= G.items) return;
    const uint32_t n_turn = (G.q + G.kv) * G.head;
    const bool is_v = it >= n_turn;
    const uint32_t per = is_v ? G.vhead : G.head;
    const uint32_t group = (is_v ? it - n_turn : it) / per, j = (is_v ? it - n_turn : it) % per;
    const bool is_q = !is_v && group < G.q;
    const uint32_t h0 = HU * (is_v || is_q ? group : group - G.q); /* first head within q, k or v */
    const uint32_t heads = is_q ? A.n_head : D.n_kv;
    const bool turn = !is_v && j < G.turned;
    const uint32_t half = A.rot_dim / 2;
    /* first value of the item; partners elsewhere are a second run of V values at o1 */
    const uint32_t o0 = is_v ? j * V : !turn ? A.rot_dim + (j - G.turned) * V : A.interleaved && !NEAR ? 2 * j : j * V;
    const uint32_t o1 = A.interleaved ? o0 + 1 : o0 + half;
    const bool second = turn && !NEAR;
    const uint32_t angle = j * P;                          /* its first pair */
    const T *in = (const T *)(is_v ? A.v : is_q ? A.q : A.k) + (uint64_t)h0 * D.head_dim;
    const uint64_t in_stride = is_v ? A.v_stride : is_q ? A.q_stride : A.k_stride;
    void *out = is_v ? D.v : is_q ? A.q_out : D.k;
    const uint32_t type = is_q ? A.q_out_type : D.dtype;
    const uint64_t head_stride = is_q ? D.head_dim : D.head_stride;
    const float *scale = is_q ? nullptr : is_v ? D.v_scale : D.k_scale;

    const uint32_t step = gridDim.y * blockDim.y;
    uint32_t t = blockIdx.y * blockDim.y + threadIdx.y;
    int32_t pos = -1, seq = -1;
    if (t < A.n_tok) { /* plain loads: a kernel that this one overlapped may have written them (a pool's lengths) */
        pos = A.pos[t];
        seq = A.seq[t];
    }
    while (t < A.n_tok) {
        /* the values wait for nothing, angles and page for the position, which came a token ahead */
        pk_vec<T, V> r0[HU], r1[NEAR ? 1 : HU];
        const T *from = in + t * in_stride;
#pragma unroll
        for (int u = 0; u < HU; u++)
            if (HU == 1 || h0 + u < heads) {
                r0[u] = *(const pk_vec<T, V> *)(from + u * D.head_dim + o0);
                if constexpr (!NEAR)
                    if (second) r1[u] = *(const pk_vec<T, V> *)(from + u * D.head_dim + o1);
            }
        const uint32_t now = t;
        int32_t p = seq < 0 ? -1 : pos;
        const int32_t row = seq;
        const bool more = A.n_tok - t > step;
        t = more ? t + step : A.n_tok;
        if (more) {
            pos = A.pos[t];
            seq = A.seq[t];
        }
        if (p >= 0 && A.rot_dim && (uint32_t)p >= A.n_pos) { /* no angles: nothing of the token is written */
            atomicOr(err, PULSAR_KV_ERR_SPAN);
            p = -1;
        }
        if (p < 0) continue;
        uint64_t to;
        if (is_q) {
            to = now * A.q_out_stride;
        } else {
            const uint32_t slot = (uint32_t)p / D.page_size;
            if ((uint32_t)row >= D.n_rows || slot >= D.max_pages) {
                atomicOr(err, (uint32_t)row >= D.n_rows ? PULSAR_KV_ERR_ROW : PULSAR_KV_ERR_SPAN);
                continue;
            }
            /* a kernel that this one overlapped may have written the table */
            const uint32_t page = (uint32_t)__ldcg(D.table + (uint64_t)row * D.table_stride + slot);
            if (page >= D.n_pages) {
                atomicOr(err, PULSAR_KV_ERR_PAGE);
                continue;
            }
            to = (uint64_t)page * D.page_stride + ((uint32_t)p - slot * D.page_size) * D.tok_stride;
        }
        pk_vec<float, P> c, s;
        if (turn) {
            const float *cs = A.cos_sin + (uint64_t)p * A.rot_dim + angle;
            c = *(const pk_vec<float, P> *)cs;
            s = *(const pk_vec<float, P> *)(cs + half);
        }
        to += h0 * head_stride;
#pragma unroll
        for (int u = 0; u < HU; u++) {
            if (HU > 1 && h0 + u >= heads) break;
            float x[V], y[V]; /* y: the partners' run */
#pragma unroll
            for (int i = 0; i < V; i++) {
                x[i] = pk_type<X>::get(r0[u].v[i]);
                if constexpr (!NEAR) y[i] = second ? pk_type<X>::get(r1[u].v[i]) : 0.0f;
            }
            if (turn) {
#pragma unroll
                for (int i = 0; i < P; i++) {
                    float &a = NEAR ? x[2 * i] : x[i], &b = NEAR ? x[2 * i + 1] : y[i];
                    const float a0 = a;
                    a = a0 * c.v[i] - b * s.v[i];
                    b = b * c.v[i] + a0 * s.v[i];
                }
            }
            if (scale) {
                const float sc = __ldg(scale + h0 + u);
#pragma unroll
                for (int i = 0; i < V; i++) {
                    x[i] /= sc;
                    if constexpr (!NEAR) y[i] /= sc;
                }
            }
            pk_store<V>(out, type, to + u * head_stride + o0, x);
            if constexpr (!NEAR)
                if (second) pk_store<V>(out, type, to + u * head_stride + o1, y);
        }
    }
}

template <uint32_t X, int V, bool NEAR, int HU>
static int pk_append_grid(const pulsar_kv_desc *d, const pulsar_kv_append_args *a, cudaStream_t st) {
    pk_append_geo g;
    g.turned = NEAR ? a->rot_dim / V : a->rot_dim / 2 / V;
    g.head = g.turned + (d->head_dim - a->rot_dim) / V;
    g.vhead = d->head_dim / V;
    g.q = (a->n_head + HU - 1) / HU;
    g.kv = (d->n_kv + HU - 1) / HU;
    g.items = (g.q + g.kv) * g.head + g.kv * g.vhead;
    dim3 block(g.items >= 256 ? 256 : (g.items + 31u) & ~31u, 1), grid((g.items + block.x - 1) / block.x);
    block.y = 256 / block.x;
    /* 16 CTAs to an SM where there are that many tokens (a thread then takes
     * its item of more of them), a token a thread where there are fewer */
    const uint32_t y = (a->n_tok + block.y - 1) / block.y, most = (16 * pk_sm_count() + grid.x - 1) / grid.x;
    grid.y = y < most ? y : most;
    return pm_ok(pk_launch(pk_append_kernel<X, V, NEAR, HU>, grid, block, 0, st, *d, *a, g, pk_err_word()), "kv append launch");
}

template <uint32_t X, int V>
static int pk_append_launch(const pulsar_kv_desc *d, const pulsar_kv_append_args *a, cudaStream_t st) {
    /* one head a thread until the GPU is full of threads */
    const uint64_t runs = (uint64_t)a->n_tok * (a->n_head + 2 * d->n_kv) * (d->head_dim / V);
    const bool few = runs < 2048ull * pk_sm_count();
    if constexpr (V > 1)
        if (a->interleaved)
            return few ? pk_append_grid<X, V, true, 1>(d, a, st) : pk_append_grid<X, V, true, 4>(d, a, st);
    return few ? pk_append_grid<X, V, false, 1>(d, a, st) : pk_append_grid<X, V, false, 2>(d, a, st);
}

template <uint32_t X>
static int pk_append_by_width(const pulsar_kv_desc *d, const pulsar_kv_append_args *a, cudaStream_t st) {
    /* the widest run of values, up to 16 bytes, that every part of a head and
     * every address is a multiple of (head_dim is a multiple of 16, cache rows
     * of 16 bytes); the angles' runs are of f32, half as many of near pairs */
    const uint32_t xe = pk_type_bytes(a->x_type), qe = pk_type_bytes(a->q_out_type);
    for (uint32_t v = 16 / xe; v > 1; v /= 2) {
        const uint32_t ab = 4 * (a->interleaved ? v / 2 : v), qb = qe * v;
        uint64_t odd = (uintptr_t)a->cos_sin % (ab < 16 ? ab : 16);
        odd |= ((uintptr_t)a->k | (uintptr_t)a->v | a->k_stride * xe | a->v_stride * xe) % (xe * v);
        if (a->n_head)
            odd |= ((uintptr_t)a->q | a->q_stride * xe) % (xe * v) |
                   ((uintptr_t)a->q_out | a->q_out_stride * qe) % (qb < 16 ? qb : 16);
        if (odd || (a->interleaved ? a->rot_dim : a->rot_dim / 2) % v) continue;
        if constexpr (X != PULSAR_TYPE_F32)
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
