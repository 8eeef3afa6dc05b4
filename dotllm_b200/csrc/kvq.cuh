// kvq.cuh -- pool of 8-bit KV pages: argument checks and the device-side lookups shared by the
// write, read and attention kernels.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp8.h>

#include "common.cuh"

namespace llmdot {

constexpr int KVQ_PAGE = LLMDOT_KV_PAGE;

// Host checks; the error names the calling entry point.
int kvq_check(const char *who, const llmdot_kvq_pool *pool, const llmdot_kvq_batch *batch);
bool kvq_type_ok(uint32_t type);
inline int kvq_type_size(uint32_t type) { return type == T_F32 ? 4 : 2; }

// An exception (a failed allocation of an error message) must not cross the C boundary.
template <typename F> inline int c_boundary(F f) noexcept
{
    try {
        return f();
    } catch (...) {
        return LLMDOT_E_NOMEM;
    }
}

// The sequence that holds packed row r: the last b with row_start[b] <= r, skipping empty ones; -1
// when r is outside every sequence.
__device__ __forceinline__ int kvq_seq_of(const int32_t *__restrict__ row_start, int batch, int r)
{
    int lo = 0, hi = batch;  // first b with row_start[b + 1] > r
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (row_start[mid + 1] > r) hi = mid;
        else lo = mid + 1;
    }
    return lo < batch && row_start[lo] <= r ? lo : -1;
}

// Index of (page, kv head 0, slot) of sequence b's position pos in units of one head's row, or -1.
__device__ __forceinline__ int64_t kvq_place(const llmdot_kvq_pool &pool, const llmdot_kvq_batch &bt, int b, int pos)
{
    const int pi = pos / KVQ_PAGE;
    if (pos < 0 || pi >= bt.max_pages) return -1;
    const int page = bt.pages[(int64_t)b * bt.max_pages + pi];
    if ((unsigned)page >= (unsigned)pool.n_pages) return -1;
    return (int64_t)page * pool.heads_kv * KVQ_PAGE + pos % KVQ_PAGE;
}

template <typename T> __device__ __forceinline__ T from_f32(float x);
template <> __device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <> __device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// Eight consecutive values; `wide`: the address is a multiple of 16 bytes.
template <typename T> __device__ __forceinline__ void store8(T *__restrict__ p, bool wide, const float (&x)[8])
{
    __align__(16) T t[8];
#pragma unroll
    for (int i = 0; i < 8; i++) t[i] = from_f32<T>(x[i]);
    if (wide) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; i++) ((uint4 *)p)[i] = ((const uint4 *)t)[i];
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) p[i] = t[i];
    }
}

// Value of one code byte (without its scale).
template <int FMT> __device__ __forceinline__ float code_value(uint8_t c)
{
    if (FMT == LLMDOT_KVQ_I8) return (float)(int8_t)c;
    __nv_fp8_e4m3 f;
    f.__x = c;
    return (float)f;
}

}  // namespace llmdot
