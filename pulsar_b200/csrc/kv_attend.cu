/* kv_attend.cu - attention of new tokens over a paged cache.
 *
 *   o = sum_j e^(s_j - m) v_j / (sum_j e^(s_j - m) + e^(sink - m)),  s_j = scale q.k_j
 * One warp per (token, query head); lanes hold 8 values of the head each,
 * the keys pass once with the running maximum and sum. */
#include "pk_common.h"

template <uint32_t T>
__device__ __forceinline__ float pk_get(const void *p, uint64_t at) {
    return pk_type<T>::get(((const typename pk_type<T>::t *)p)[at]);
}

template <uint32_t Q, uint32_t C>
__global__ void __launch_bounds__(32) pk_attend_kernel(const pulsar_kv_desc D, const pulsar_kv_attend_args A,
                                                       uint32_t *err) {
    const uint32_t lane = threadIdx.x, h = blockIdx.y, hk = h / (A.n_head / D.n_kv);
    const uint32_t b = blockIdx.x / A.n_q, i = blockIdx.x % A.n_q;
    const int32_t row = A.seq ? A.seq[b] : (int32_t)b;
    int64_t len = A.lens[b];
    if (row < 0 || len < 0) len = 0;
    else if ((uint32_t)row >= D.n_rows) {
        if (lane == 0) atomicOr(err, PULSAR_KV_ERR_ROW);
        len = 0;
    }
    if (len > (int64_t)D.max_pages * D.page_size) {
        if (lane == 0) atomicOr(err, PULSAR_KV_ERR_SPAN);
        len = (int64_t)D.max_pages * D.page_size;
    }
    const int64_t hi = len - (int64_t)(A.n_q - 1 - i), lo = A.window && hi > A.window ? hi - A.window : 0;
    const float ks = D.k_scale ? D.k_scale[hk] : 1.0f, vs = D.v_scale ? D.v_scale[hk] : 1.0f;
    float q[8], o[8];
    const uint64_t at = blockIdx.x * A.q_stride + (uint64_t)h * D.head_dim;
    for (int x = 0; x < 8; x++) {
        const uint32_t c = lane + 32 * x;
        q[x] = c < D.head_dim ? pk_get<Q>(A.q, at + c) * A.scale * ks : 0.0f;
        o[x] = 0.0f;
    }
    float m = -INFINITY, l = 0.0f;
    for (int64_t j = lo; j < hi; j++) {
        const int32_t page = D.table[(uint64_t)row * D.table_stride + j / D.page_size];
        if ((uint32_t)page >= D.n_pages) {
            if (lane == 0) atomicOr(err, PULSAR_KV_ERR_PAGE);
            continue;
        }
        const uint64_t e = (uint64_t)page * D.page_stride + hk * D.head_stride + (j % D.page_size) * D.tok_stride;
        float s = 0.0f;
        for (int x = 0; x < 8; x++)
            if (lane + 32 * x < D.head_dim) s += q[x] * pk_get<C>(D.k, e + lane + 32 * x);
        for (int w = 16; w; w >>= 1) s += __shfl_xor_sync(~0u, s, w);
        const float m2 = fmaxf(m, s), base = m2 == -INFINITY ? 0.0f : m2;
        const float keep = expf(m - base), p = expf(s - base);
        m = m2;
        l = l * keep + p;
        for (int x = 0; x < 8; x++)
            o[x] = o[x] * keep +
                   (lane + 32 * x < D.head_dim ? p * pk_get<C>(D.v, e + lane + 32 * x) : 0.0f);
    }
    const bool empty = hi <= lo;
    if (A.sinks && !empty) {
        const float m2 = fmaxf(m, A.sinks[h]), keep = expf(m - m2);
        l = l * keep + expf(A.sinks[h] - m2);
        for (int x = 0; x < 8; x++) o[x] *= keep;
        m = m2;
    }
    typedef typename pk_type<Q>::t T;
    T *out = (T *)A.out + blockIdx.x * A.out_stride + (uint64_t)h * D.head_dim;
    for (int x = 0; x < 8; x++)
        if (lane + 32 * x < D.head_dim) out[lane + 32 * x] = pk_type<Q>::put(l > 0.0f || isnan(l) ? o[x] * vs / l : 0.0f);
    if (A.lse && lane == 0)
        A.lse[(uint64_t)blockIdx.x * A.n_head + h] = empty ? -INFINITY : logf(l) + m;
}

extern "C" size_t pulsar_kv_attend_workspace(const pulsar_kv_desc *d, const pulsar_kv_attend_args *a) {
    return pk_desc_fault(d) || !a ? 0 : PULSAR_KV_WS_ZEROED;
}

template <uint32_t Q>
static int pk_attend_by_cache(const pulsar_kv_desc *d, const pulsar_kv_attend_args *a, cudaStream_t st) {
    const dim3 grid(a->n_rows * a->n_q, a->n_head);
    if (d->dtype == PULSAR_TYPE_BF16)
        pk_attend_kernel<Q, PULSAR_TYPE_BF16><<<grid, 32, 0, st>>>(*d, *a, pk_err_word());
    else if (d->dtype == PULSAR_TYPE_F16)
        pk_attend_kernel<Q, PULSAR_TYPE_F16><<<grid, 32, 0, st>>>(*d, *a, pk_err_word());
    else
        pk_attend_kernel<Q, PULSAR_TYPE_E4M3><<<grid, 32, 0, st>>>(*d, *a, pk_err_word());
    return pm_ok(cudaGetLastError(), "kv attend launch");
}

extern "C" int pulsar_kv_attend(const pulsar_kv_desc *d, const pulsar_kv_attend_args *a, void *ws, size_t ws_bytes,
                                void *stream) {
    const char *f = pk_desc_fault(d);
    if (f) return pk_refuse(f);
    if (!a || !a->q || !a->out || !a->lens || !ws) return pk_refuse("kv attend: null arguments");
    if (a->q_type > PULSAR_TYPE_F16) return pk_refuse("kv attend: values are f32, bf16 or f16");
    if (!a->n_head || a->n_head > 0xffffu || a->n_head % d->n_kv)
        return pk_refuse("kv attend: n_head is a multiple of n_kv, at most 65535");
    if (!a->n_rows || !a->n_q || (uint64_t)a->n_rows * a->n_q > 0x7fffffffull)
        return pk_refuse("kv attend: between 1 and 2^31 - 1 tokens");
    if (!a->seq && a->n_rows > d->n_rows) return pk_refuse("kv attend: more rows than the table has");
    const uint64_t w = (uint64_t)a->n_head * d->head_dim;
    if ((uint64_t)a->n_rows * a->n_q > 1 && (a->q_stride < w || a->out_stride < w))
        return pk_refuse("kv attend: tokens overlap");
    if (ws_bytes < pulsar_kv_attend_workspace(d, a)) return pk_refuse("kv attend: workspace too small");
    if (!pk_err_word()) return pk_refuse("kv: no error word on this device");
    const cudaStream_t st = pk_stream(stream);
    if (a->q_type == PULSAR_TYPE_F32) return pk_attend_by_cache<PULSAR_TYPE_F32>(d, a, st);
    if (a->q_type == PULSAR_TYPE_BF16) return pk_attend_by_cache<PULSAR_TYPE_BF16>(d, a, st);
    return pk_attend_by_cache<PULSAR_TYPE_F16>(d, a, st);
}
