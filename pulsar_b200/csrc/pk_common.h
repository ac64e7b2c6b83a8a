/* pk_common.h - what the paged-cache translation units share: argument
 * checks, type conversion, the error word. */
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <stdint.h>
#include <stdio.h>

#include "../../include/pulsar_kv.h"
#include "pm_host.h"

/* the family's error word on the current device (kv_pages.cu) */
uint32_t *pk_err_word();

static inline int pk_refuse(const char *what) {
    fprintf(stderr, "pulsar-b200: %s\n", what);
    return 0;
}

static inline cudaStream_t pk_stream(void *s) { return s ? (cudaStream_t)s : cudaStreamPerThread; }

static inline uint32_t pk_type_bytes(uint32_t t) {
    return t == PULSAR_TYPE_F32 ? 4u : t == PULSAR_TYPE_E4M3 ? 1u : 2u;
}

/* SMs of the current device, looked up once per device */
static inline uint32_t pk_sm_count() {
    static int sms[64];
    const int dev = pm_cur_device();
    if (dev < 64 && sms[dev]) return (uint32_t)sms[dev];
    int n = 0;
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n < 1) n = 1;
    if (dev < 64) sms[dev] = n;
    return (uint32_t)n;
}

/* what pulsar_kv_desc says of itself; NULL = sound, else what is wrong */
static inline const char *pk_desc_fault(const pulsar_kv_desc *d) {
    if (!d || !d->k || !d->v || !d->table) return "kv: null descriptor, cache or table";
    if (d->dtype != PULSAR_TYPE_BF16 && d->dtype != PULSAR_TYPE_F16 && d->dtype != PULSAR_TYPE_E4M3)
        return "kv: caches are bf16, f16 or e4m3";
    if (!d->n_pages || !d->page_size || !d->n_kv || !d->n_rows || !d->max_pages) return "kv: a zero size";
    if (d->n_pages > 0x7fffffffu || (uint64_t)d->max_pages * d->page_size > 0x7fffffffull)
        return "kv: pages or row length above 2^31 - 1";
    if (!d->head_dim || d->head_dim % 16 || d->head_dim > 256) return "kv: head_dim is a multiple of 16 up to 256";
    if (d->table_stride < d->max_pages) return "kv: table rows overlap";
    const uint64_t e = pk_type_bytes(d->dtype);
    if (((uintptr_t)d->k | (uintptr_t)d->v | d->page_stride * e | d->head_stride * e | d->tok_stride * e) % 16)
        return "kv: cache pointers and strides are multiples of 16 bytes";
    if (d->tok_stride > 0x0fffffffull) return "kv: tokens are less than 2^28 values apart";
    if (d->dtype != PULSAR_TYPE_E4M3 && (d->k_scale || d->v_scale)) return "kv: scales belong to e4m3 caches";
    return nullptr;
}

/* ------------------------------------------------------ launches */

/* A kernel of the family may be launched while the one before it in its
 * stream, if that is of the family too, still runs: its CTAs take the places
 * that come free and wait at pk_enter (in the hardware, for the end and the
 * writes of what came before), which saves the launch's latency.  Each kernel
 * enters before its first access to global memory. */
__device__ __forceinline__ void pk_enter() {
    asm volatile("griddepcontrol.wait;\n\tgriddepcontrol.launch_dependents;" ::: "memory");
}

template <class... P, class... A>
static cudaError_t pk_launch(void (*kernel)(P...), dim3 grid, dim3 block, uint32_t smem, cudaStream_t st, A... args) {
    cudaLaunchAttribute early;
    early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    early.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t c = {};
    c.gridDim = grid;
    c.blockDim = block;
    c.dynamicSmemBytes = smem;
    c.stream = st;
    c.attrs = &early;
    c.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&c, kernel, (P)args...);
    if (e != cudaSuccess) (void)cudaGetLastError(); /* the caller's next check of a launch is not about this one */
    return e;
}

/* ------------------------------------------------------ values by type */

template <uint32_t T> struct pk_type;
template <> struct pk_type<PULSAR_TYPE_F32> {
    typedef float t;
    static __device__ __forceinline__ float get(t v) { return v; }
    static __device__ __forceinline__ t put(float v) { return v; }
};
template <> struct pk_type<PULSAR_TYPE_BF16> {
    typedef __nv_bfloat16 t;
    static __device__ __forceinline__ float get(t v) { return __bfloat162float(v); }
    static __device__ __forceinline__ t put(float v) { return __float2bfloat16_rn(v); }
};
template <> struct pk_type<PULSAR_TYPE_F16> {
    typedef __half t;
    static __device__ __forceinline__ float get(t v) { return __half2float(v); }
    static __device__ __forceinline__ t put(float v) { return __float2half_rn(v); }
};
template <> struct pk_type<PULSAR_TYPE_E4M3> {
    typedef __nv_fp8_storage_t t;
    static __device__ __forceinline__ float get(t v) {
        return __half2float(__half(__nv_cvt_fp8_to_halfraw(v, __NV_E4M3)));
    }
    static __device__ __forceinline__ t put(float v) { return __nv_cvt_float_to_fp8(v, __NV_SATFINITE, __NV_E4M3); }
};
