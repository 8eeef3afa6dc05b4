// kvq.cu -- writing K/V rows into the 8-bit paged pool and reading them back.
//
// Per row and head: a = max |x|, scale = a / M, code = rne(x * (M * (1 / a))), M = 127 (int8) or 448
// (e4m3), every operation rounded to fp32 by itself, so the codes are a function of the inputs alone.
//
// Bound: HBM (each input value read once, one byte written for it) for long prompts, launch latency for a
// decode step.  A (row, head) item is held by a group of D / 8 lanes
// (rounded up to a power of two), eight values per lane: one 16-byte load per lane for 16-bit
// inputs, one 8-byte store of codes, the maximum by shuffles inside the group.  A group takes K and V
// of one or two items, so a lane has up to four loads in flight while the rows' places are looked up.
// Instructions come next to bytes: the maxima are taken on packed 16-bit pairs, and the two IEEE
// divisions of an item are done by one lane per item.
//
// Measured on a B200 (copy bandwidth 6457 GB/s): writing 16381 rows of 8 x 128 bf16 values to e4m3 22.8 us,
// 4460 GB/s (51 us with every lane dividing and 64-bit index divisions); reading 15988 such rows to fp32 30.8 us,
// 5360 GB/s (43 us with eight neighbouring values per lane); a decode step of 8 rows of 8 x 64 4.2 us.
#include "kvq.cuh"

namespace llmdot {

bool kvq_type_ok(uint32_t type) { return type == T_F32 || type == T_F16 || type == T_BF16; }

int kvq_check(const char *who, const llmdot_kvq_pool *p, const llmdot_kvq_batch *b)
{
    auto bad = [&](const char *what) { return fail(LLMDOT_E_INVALID, std::string(who) + ": " + what); };
    if (!p || !b) return bad("null pool or batch");
    if (p->format != LLMDOT_KVQ_I8 && p->format != LLMDOT_KVQ_E4M3) return bad("unknown pool format");
    if (p->head_dim != 64 && p->head_dim != 96 && p->head_dim != 128 && p->head_dim != 256)
        return fail(LLMDOT_E_UNSUPPORTED, std::string(who) + ": head_dim must be 64, 96, 128 or 256");
    if (p->heads_kv <= 0 || p->heads_kv > 4096 || p->n_pages < 0) return bad("bad heads_kv or n_pages");
    if (p->n_pages > 0 && (!p->k || !p->v || !p->k_scale || !p->v_scale)) return bad("null pool memory");
    if (((uintptr_t)p->k | (uintptr_t)p->v) & 15) return bad("pool codes must be 16-byte aligned");
    if (((uintptr_t)p->k_scale | (uintptr_t)p->v_scale) & 3) return bad("pool scales must be 4-byte aligned");
    if (b->batch < 0 || b->rows < 0 || b->max_rows < 0 || b->max_pages < 0) return bad("negative size in the batch");
    if (b->max_pages > (1 << 24)) return bad("max_pages exceeds 2^24 (positions are 32-bit)");
    if (b->batch > 0 && (!b->row_start || !b->seq_len)) return bad("null row_start or seq_len");
    if (b->batch > 0 && b->max_pages > 0 && !b->pages) return bad("null pages");
    if (((uintptr_t)b->row_start | (uintptr_t)b->seq_len | (uintptr_t)b->pages) & 3) return bad("row_start, seq_len and pages must be 4-byte aligned");
    if (b->rows > 0 && b->batch == 0) return bad("rows without a sequence");
    return LLMDOT_OK;
}

namespace {

// Lanes per (row, head): D / 8, rounded up to a power of two (96 leaves 4 of 16 idle).
template <int D> constexpr int kvq_lanes() { return D == 64 ? 8 : D == 256 ? 32 : 16; }
constexpr int KVQ_THREADS = 256;
// Items of a group where there are enough for four blocks per SM: two, so that more loads are in flight, but one for
// fp32 heads of 128 and more, where a lane's own loads do.  Some 16000 rows of 8 heads, us with one / two:
// reading bf16 128 22.6 / 18.7, fp32 64 17.2 / 16.5, fp32 128 30.9 / 32.3; writing bf16 256 42.7 / 39.1, fp32 128 29.9 / 30.8.
template <typename T, int D> constexpr int kvq_each() { return sizeof(T) == 2 || D < 128 ? 2 : 1; }
template <int D, int EACH> constexpr int kvq_items() { return KVQ_THREADS / kvq_lanes<D>() * EACH; }

// Where a block's rows lie: for each row of the block's items the pool row of (page, head 0, slot), or -1
// for no position, -2 for no sequence.  One thread per row, so that the chain of dependent loads (row ->
// sequence -> length, page) is walked once per row and not once per head.
template <int N> __device__ __forceinline__ void kvq_find(const llmdot_kvq_pool &pool, const llmdot_kvq_batch &bt, int row0,
                                                          int64_t (&place)[N])
{
    const int r = row0 + threadIdx.x;
    if (threadIdx.x < N && r < bt.rows) {
        const int b = kvq_seq_of(bt.row_start, bt.batch, r);
        place[threadIdx.x] = b < 0 ? -2 : kvq_place(pool, bt, b, bt.seq_len[b] - bt.row_start[b + 1] + r);
    }
}

// Maxima that a NaN survives: a row is finite when its maximum is.
__device__ __forceinline__ float max_nan(float a, float b)
{
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}
// Eight values of one lane as they were loaded, their largest magnitude, and as floats.
template <typename T> struct Raw8;
template <> struct Raw8<float> {
    float x[8];
    __device__ __forceinline__ float top() const
    {
        float a = fabsf(x[0]);
#pragma unroll
        for (int e = 1; e < 8; e++) a = max_nan(a, fabsf(x[e]));
        return a;
    }
    __device__ __forceinline__ void floats(float (&f)[8]) const
    {
#pragma unroll
        for (int e = 0; e < 8; e++) f[e] = x[e];
    }
};
template <> struct Raw8<__half> {
    __half2 x[4];
    __device__ __forceinline__ float top() const
    {
        const __half2 m = __hmax2_nan(__hmax2_nan(__habs2(x[0]), __habs2(x[1])), __hmax2_nan(__habs2(x[2]), __habs2(x[3])));
        return __half2float(__hmax_nan(__low2half(m), __high2half(m)));
    }
    __device__ __forceinline__ void floats(float (&f)[8]) const
    {
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const float2 y = __half22float2(x[e]);
            f[2 * e] = y.x;
            f[2 * e + 1] = y.y;
        }
    }
};
template <> struct Raw8<__nv_bfloat16> {
    __nv_bfloat162 x[4];
    __device__ __forceinline__ float top() const
    {
        const __nv_bfloat162 m = __hmax2_nan(__hmax2_nan(__habs2(x[0]), __habs2(x[1])), __hmax2_nan(__habs2(x[2]), __habs2(x[3])));
        return __bfloat162float(__hmax_nan(__low2bfloat16(m), __high2bfloat16(m)));
    }
    __device__ __forceinline__ void floats(float (&f)[8]) const
    {
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const float2 y = __bfloat1622float2(x[e]);
            f[2 * e] = y.x;
            f[2 * e + 1] = y.y;
        }
    }
};
template <typename T> __device__ __forceinline__ void load_raw(Raw8<T> &r, const T *__restrict__ p, bool on, bool wide)
{
    if (!on) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; i++) ((uint4 *)&r)[i] = make_uint4(0, 0, 0, 0);
    } else if (wide) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; i++) ((uint4 *)&r)[i] = __ldg((const uint4 *)p + i);
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) ((T *)&r)[i] = p[i];
    }
}
// Codes of eight values.  int8: adding 1.5 * 2^23 rounds to an integer (ties to even) that stands in the
// low byte; |y| <= 127 (1 + 2^-22) rounds to at most 127.
template <int FMT> __device__ __forceinline__ uint2 codes8(const float (&f)[8], float inv)
{
    uint32_t w[2];
#pragma unroll
    for (int i = 0; i < 2; i++) {
        if (FMT == LLMDOT_KVQ_I8) {
            uint32_t y[4];
#pragma unroll
            for (int e = 0; e < 4; e++) y[e] = __float_as_uint(__fadd_rn(__fmul_rn(f[4 * i + e], inv), 12582912.0f));
            w[i] = __byte_perm(__byte_perm(y[0], y[1], 0x0040), __byte_perm(y[2], y[3], 0x0040), 0x5410);
        } else {
            uint16_t h[2];
#pragma unroll
            for (int e = 0; e < 2; e++)
                asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;"
                    : "=h"(h[e])
                    : "f"(__fmul_rn(f[4 * i + 2 * e + 1], inv)), "f"(__fmul_rn(f[4 * i + 2 * e], inv)));
            w[i] = (uint32_t)h[0] | (uint32_t)h[1] << 16;
        }
    }
    return make_uint2(w[0], w[1]);
}

template <typename T, int D, int FMT, int EACH>
__global__ void __launch_bounds__(KVQ_THREADS)
kvq_write_kernel(const llmdot_kvq_pool pool, const llmdot_kvq_batch bt, const T *__restrict__ xk,
                 const T *__restrict__ xv, int64_t ldk, int64_t ldv, int wide)
{
    constexpr int L = kvq_lanes<D>(), GR = KVQ_THREADS / L, N = kvq_items<D, EACH>();
    __shared__ int64_t s_place[N];  // N consecutive items are of at most N rows
    const uint32_t Hk = pool.heads_kv, items = bt.rows * Hk, item0 = blockIdx.x * N, row0 = item0 / Hk;
    const int lane = threadIdx.x % L, grp = threadIdx.x / L;
    const bool on = lane * 8 < D;
    Raw8<T> x[EACH][2];
    uint32_t row[EACH], head[EACH];
#pragma unroll
    for (int i = 0; i < EACH; i++) {
        const uint32_t item = item0 + i * GR + grp;
        row[i] = item / Hk;
        head[i] = item - row[i] * Hk;
        const int64_t o = head[i] * D + lane * 8;
        load_raw(x[i][0], xk + row[i] * ldk + o, on && item < items, wide != 0);
        load_raw(x[i][1], xv + row[i] * ldv + o, on && item < items, wide != 0);
    }
    kvq_find(pool, bt, (int)row0, s_place);
    constexpr float M = FMT == LLMDOT_KVQ_I8 ? 127.0f : 448.0f;
    // the groups' maxima; lane c of a group then divides for combination c (item, K or V)
    float mine = 0.0f;
#pragma unroll
    for (int c = 0; c < 2 * EACH; c++) {
        float a = x[c >> 1][c & 1].top();
#pragma unroll
        for (int o = L / 2; o > 0; o >>= 1) a = max_nan(a, __shfl_xor_sync(0xffffffffu, a, o));
        if (lane == c) mine = a;
    }
    const bool fine = mine < INFINITY, some = fine && mine >= 1e-30f;
    const float scale = some ? __fdiv_rn(mine, M) : fine ? 0.0f : NAN;
    const float inv_mine = some ? __fmul_rn(M, __frcp_rn(mine)) : 0.0f;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < EACH; i++) {
        const bool real = item0 + i * GR + grp < items;
        const int64_t at0 = real ? s_place[row[i] - row0] : -2, at = at0 + (int64_t)head[i] * KVQ_PAGE;
#pragma unroll
        for (int v = 0; v < 2; v++) {
            const float inv = __shfl_sync(0xffffffffu, inv_mine, 2 * i + v, L);
            if (at0 < 0) continue;
            if (lane == 2 * i + v) (v ? pool.v_scale : pool.k_scale)[at] = scale;
            if (!on) continue;
            float f[8];
            x[i][v].floats(f);
            const uint2 w = inv == 0.0f ? make_uint2(0, 0) : codes8<FMT>(f, inv);
            *(uint2 *)((uint8_t *)(v ? pool.v : pool.k) + at * D + lane * 8) = w;
        }
    }
}

// Four codes of a word as floats.
template <int FMT> __device__ __forceinline__ void floats4(uint32_t w, float s, float (&f)[4])
{
    if (FMT == LLMDOT_KVQ_I8) {  // the byte, sign bit flipped, under the exponent of 2^23: an exact difference
        w ^= 0x80808080u;
        f[0] = __fmul_rn(__uint_as_float(__byte_perm(w, 0x4B000000u, 0x7440)) - 8388736.0f, s);
        f[1] = __fmul_rn(__uint_as_float(__byte_perm(w, 0x4B000000u, 0x7441)) - 8388736.0f, s);
        f[2] = __fmul_rn(__uint_as_float(__byte_perm(w, 0x4B000000u, 0x7442)) - 8388736.0f, s);
        f[3] = __fmul_rn(__uint_as_float(__byte_perm(w, 0x4B000000u, 0x7443)) - 8388736.0f, s);
    } else {
#pragma unroll
        for (int e = 0; e < 4; e++) f[e] = __fmul_rn(code_value<FMT>((uint8_t)(w >> (8 * e))), s);
    }
}
template <typename T> __device__ __forceinline__ void store4v(T *p, bool wide, const float (&f)[4])
{
    __align__(16) T t[4];
#pragma unroll
    for (int e = 0; e < 4; e++) t[e] = from_f32<T>(f[e]);
    if (wide) {
        if (sizeof(T) == 4) *(uint4 *)p = *(const uint4 *)t;
        else *(uint2 *)p = *(const uint2 *)t;
    } else {
#pragma unroll
        for (int e = 0; e < 4; e++) p[e] = t[e];
    }
}

// A lane's eight values: neighbours for 16-bit outputs (one 16-byte store); for fp32 four in each half of
// the row, so that the lanes of a store write consecutive bytes.
template <typename T, int D, int FMT, int EACH>
__global__ void __launch_bounds__(KVQ_THREADS)
kvq_read_kernel(const llmdot_kvq_pool pool, const llmdot_kvq_batch bt, T *__restrict__ xk, T *__restrict__ xv,
                int64_t ldk, int64_t ldv, int wide)
{
    constexpr int L = kvq_lanes<D>(), GR = KVQ_THREADS / L, N = kvq_items<D, EACH>();
    __shared__ int64_t s_place[N];
    const uint32_t Hk = pool.heads_kv, items = bt.rows * Hk, item0 = blockIdx.x * N, row0 = item0 / Hk;
    const int lane = threadIdx.x % L, grp = threadIdx.x / L;
    kvq_find(pool, bt, (int)row0, s_place);
    __syncthreads();
    if (lane * 8 >= D) return;
    constexpr int d0 = sizeof(T) == 4 ? 4 : 8, d1 = sizeof(T) == 4 ? D / 2 : 4;  // lane's first value, its second four
    uint2 c[EACH][2];
    float s[EACH][2];
    int64_t at0[EACH], o[EACH];
    uint32_t row[EACH];
#pragma unroll
    for (int i = 0; i < EACH; i++) {
        const uint32_t item = item0 + i * GR + grp;
        row[i] = item / Hk;
        const uint32_t head = item - row[i] * Hk;
        o[i] = head * D + lane * d0;
        at0[i] = item < items ? s_place[row[i] - row0] : -2;
        const int64_t at = at0[i] + (int64_t)head * KVQ_PAGE;
#pragma unroll
        for (int v = 0; v < 2; v++) {
            c[i][v] = make_uint2(0, 0);
            s[i][v] = 0.0f;
            if (at0[i] >= 0) {
                const uint8_t *p = (const uint8_t *)(v ? pool.v : pool.k) + at * D + lane * d0;
                if (sizeof(T) == 4) c[i][v] = make_uint2(__ldg((const uint32_t *)p), __ldg((const uint32_t *)(p + d1)));
                else c[i][v] = __ldg((const uint2 *)p);
                s[i][v] = __ldg((v ? pool.v_scale : pool.k_scale) + at);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < EACH; i++) {
        if (at0[i] == -2) continue;  // no item, or a row of no sequence
#pragma unroll
        for (int v = 0; v < 2; v++) {
            T *to = (v ? xv + row[i] * ldv : xk + row[i] * ldk) + o[i];
            float f[4], h[4];
            floats4<FMT>(c[i][v].x, s[i][v], f);
            floats4<FMT>(c[i][v].y, s[i][v], h);
            if (at0[i] < 0)
#pragma unroll
                for (int e = 0; e < 4; e++) f[e] = h[e] = 0.0f;
            if (sizeof(T) == 4) {
                store4v(to, wide != 0, f);
                store4v(to + d1, wide != 0, h);
            } else {
                const float x[8] = {f[0], f[1], f[2], f[3], h[0], h[1], h[2], h[3]};
                store8(to, wide != 0, x);
            }
        }
    }
}

// The kernel instance for a type, head dimension and format.
template <template <typename, int, int> class Op, typename... A>
cudaError_t dispatch(uint32_t type, int dim, int fmt, A... a)
{
#define LLMDOT_KVQ_D(T, F)                                   \
    switch (dim) {                                           \
    case 64: return Op<T, 64, F>::launch(a...);              \
    case 96: return Op<T, 96, F>::launch(a...);              \
    case 128: return Op<T, 128, F>::launch(a...);            \
    default: return Op<T, 256, F>::launch(a...);             \
    }
#define LLMDOT_KVQ_T(F)                                      \
    switch (type) {                                          \
    case T_F32: LLMDOT_KVQ_D(float, F)                       \
    case T_F16: LLMDOT_KVQ_D(__half, F)                      \
    default: LLMDOT_KVQ_D(__nv_bfloat16, F)                  \
    }
    if (fmt == LLMDOT_KVQ_I8) LLMDOT_KVQ_T(LLMDOT_KVQ_I8)
    LLMDOT_KVQ_T(LLMDOT_KVQ_E4M3)
#undef LLMDOT_KVQ_T
#undef LLMDOT_KVQ_D
}

// Two items per group once that still gives every SM a few blocks; one for small calls, where the
// groups' work in sequence is the latency.
template <typename T, int D, int FMT> struct WriteOp {
    static cudaError_t launch(const llmdot_kvq_pool &p, const llmdot_kvq_batch &b, const void *k, const void *v, int64_t ldk,
                              int64_t ldv, int wide, cudaStream_t st)
    {
        const int64_t items = (int64_t)b.rows * p.heads_kv;
        constexpr int EACH = kvq_each<T, D>(), N1 = kvq_items<D, 1>(), N2 = kvq_items<D, EACH>();
        if (items >= 148 * 4 * N2)
            kvq_write_kernel<T, D, FMT, EACH><<<(unsigned)((items + N2 - 1) / N2), KVQ_THREADS, 0, st>>>(p, b, (const T *)k, (const T *)v,
                                                                                                         ldk, ldv, wide);
        else
            kvq_write_kernel<T, D, FMT, 1><<<(unsigned)((items + N1 - 1) / N1), KVQ_THREADS, 0, st>>>(p, b, (const T *)k, (const T *)v,
                                                                                                      ldk, ldv, wide);
        return cudaGetLastError();
    }
};
template <typename T, int D, int FMT> struct ReadOp {
    static cudaError_t launch(const llmdot_kvq_pool &p, const llmdot_kvq_batch &b, void *k, void *v, int64_t ldk, int64_t ldv,
                              int wide, cudaStream_t st)
    {
        const int64_t items = (int64_t)b.rows * p.heads_kv;
        constexpr int EACH = kvq_each<T, D>(), N1 = kvq_items<D, 1>(), N2 = kvq_items<D, EACH>();
        if (items >= 148 * 4 * N2)
            kvq_read_kernel<T, D, FMT, EACH><<<(unsigned)((items + N2 - 1) / N2), KVQ_THREADS, 0, st>>>(p, b, (T *)k, (T *)v, ldk, ldv, wide);
        else
            kvq_read_kernel<T, D, FMT, 1><<<(unsigned)((items + N1 - 1) / N1), KVQ_THREADS, 0, st>>>(p, b, (T *)k, (T *)v, ldk, ldv, wide);
        return cudaGetLastError();
    }
};

int check_rows(const char *who, const llmdot_kvq_pool *p, const llmdot_kvq_batch *b, const void *k, const void *v, uint32_t type,
               int64_t ldk, int64_t ldv, int *wide)
{
    LLMDOT_TRY(kvq_check(who, p, b));
    auto bad = [&](const char *what) { return fail(LLMDOT_E_INVALID, std::string(who) + ": " + what); };
    if (!kvq_type_ok(type)) return fail(LLMDOT_E_UNSUPPORTED, std::string(who) + ": type must be F32, F16 or BF16");
    const int64_t row = (int64_t)p->heads_kv * p->head_dim;
    if (b->rows > 0 && (!k || !v)) return bad("null K or V rows");
    if (b->rows > 1 && (ldk < row || ldv < row)) return bad("row stride below heads_kv * head_dim");
    if ((int64_t)b->rows * p->heads_kv > (int64_t)1 << 31) return bad("rows * heads_kv exceeds 2^31");
    const int es = kvq_type_size(type);
    if (((uintptr_t)k | (uintptr_t)v) % es) return bad("K or V rows are not aligned to their type");
    *wide = (((uintptr_t)k | (uintptr_t)v) & 15) == 0 && (b->rows <= 1 || (ldk * es % 16 == 0 && ldv * es % 16 == 0));
    return LLMDOT_OK;
}

}  // namespace
}  // namespace llmdot

using namespace llmdot;

extern "C" int llmdot_cuda_kvq_write(const llmdot_kvq_pool *pool, const llmdot_kvq_batch *batch, const void *d_k, const void *d_v,
                                     uint32_t type, int64_t ld_k, int64_t ld_v, void *stream)
{
    return c_boundary([&]() -> int {
        int wide = 0;
        LLMDOT_TRY(check_rows("kvq_write", pool, batch, d_k, d_v, type, ld_k, ld_v, &wide));
        if (batch->rows == 0 || pool->n_pages == 0) return LLMDOT_OK;
        LLMDOT_CUDA_TRY((dispatch<WriteOp>(type, pool->head_dim, pool->format, *pool, *batch, d_k, d_v, ld_k, ld_v, wide,
                                           (cudaStream_t)stream)));
        return LLMDOT_OK;
    });
}

extern "C" int llmdot_cuda_kvq_read(const llmdot_kvq_pool *pool, const llmdot_kvq_batch *batch, void *d_k, void *d_v,
                                    uint32_t type, int64_t ld_k, int64_t ld_v, void *stream)
{
    return c_boundary([&]() -> int {
        int wide = 0;
        LLMDOT_TRY(check_rows("kvq_read", pool, batch, d_k, d_v, type, ld_k, ld_v, &wide));
        if (batch->rows == 0) return LLMDOT_OK;
        LLMDOT_CUDA_TRY((dispatch<ReadOp>(type, pool->head_dim, pool->format, *pool, *batch, d_k, d_v, ld_k, ld_v, wide,
                                          (cudaStream_t)stream)));
        return LLMDOT_OK;
    });
}
