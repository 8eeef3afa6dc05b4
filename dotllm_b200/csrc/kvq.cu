// kvq.cu -- writing K/V rows into the 8-bit paged pool and reading them back.
//
// Per row and head: a = max |x|, scale = a / M, code = rne(x * (M * (1 / a))), M = 127 (int8) or 448
// (e4m3), every operation rounded to fp32 by itself, so the codes are a function of the inputs alone.  Bound: HBM (each input value read once, one byte written for it) for long
// prompts, launch latency for a decode step.  A (row, head) item is held by a group of D / 8 lanes
// (rounded up to a power of two), eight values per lane: one 16-byte load per lane for 16-bit
// inputs, one 8-byte store of codes, the maximum by shuffles inside the group.  A group takes K and V
// of two items, so a lane has four loads in flight while the rows' places are looked up.
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
    if (b->rows > 0 && b->batch == 0) return bad("rows without a sequence");
    return LLMDOT_OK;
}

namespace {

// Lanes per (row, head): D / 8, rounded up to a power of two (96 leaves 4 of 16 idle).
template <int D> constexpr int kvq_lanes() { return D == 64 ? 8 : D == 256 ? 32 : 16; }
constexpr int KVQ_THREADS = 256, KVQ_EACH = 2;
template <int D> constexpr int kvq_items() { return KVQ_THREADS / kvq_lanes<D>() * KVQ_EACH; }

// Where a block's rows lie: for each row of the block's items the pool row of (page, head 0, slot), or -1.
// One thread per row, so that the chain of dependent loads (row -> sequence -> length, page) is walked
// once per row and not once per head, and while the values are already on their way.
template <int D> __device__ __forceinline__ void kvq_find(const llmdot_kvq_pool &pool, const llmdot_kvq_batch &bt, int64_t item0,
                                                          int64_t (&place)[kvq_items<D>()])
{
    const int r = (int)(item0 / pool.heads_kv) + threadIdx.x;
    if (threadIdx.x < kvq_items<D>() && r < bt.rows) {
        const int b = kvq_seq_of(bt.row_start, bt.batch, r);
        place[threadIdx.x] = b < 0 ? -2 : kvq_place(pool, bt, b, bt.seq_len[b] - bt.row_start[b + 1] + r, 0);
    }
}

template <typename T, int D, int FMT>
__global__ void __launch_bounds__(KVQ_THREADS)
kvq_write_kernel(const llmdot_kvq_pool pool, const llmdot_kvq_batch bt, const T *__restrict__ xk,
                 const T *__restrict__ xv, int64_t ldk, int64_t ldv, int wide)
{
    constexpr int L = kvq_lanes<D>(), GR = KVQ_THREADS / L, N = kvq_items<D>();
    // the rows of N consecutive items are at most N (an item more can begin another row only if heads_kv > 1)
    __shared__ int64_t s_place[N];
    const int64_t item0 = (int64_t)blockIdx.x * N, items = (int64_t)bt.rows * pool.heads_kv;
    const int lane = threadIdx.x % L, grp = threadIdx.x / L, row0 = (int)(item0 / pool.heads_kv);
    const bool on = lane * 8 < D;
    float f[KVQ_EACH][2][8];
#pragma unroll
    for (int i = 0; i < KVQ_EACH; i++) {
        const int64_t item = item0 + i * GR + grp;
#pragma unroll
        for (int v = 0; v < 2; v++) {
#pragma unroll
            for (int e = 0; e < 8; e++) f[i][v][e] = 0.0f;
            if (item < items && on) {
                const int r = (int)(item / pool.heads_kv), h = (int)(item % pool.heads_kv);
                load8((v ? xv + r * ldv : xk + r * ldk) + h * D + lane * 8, wide != 0, f[i][v]);
            }
        }
    }
    kvq_find<D>(pool, bt, item0, s_place);
    __syncthreads();
    // lanes of one group are neighbours
    const unsigned mask = L == 32 ? 0xffffffffu : ((1u << (L & 31)) - 1u) << (threadIdx.x & 31 & ~(L - 1));
#pragma unroll
    for (int i = 0; i < KVQ_EACH; i++) {
        const int64_t item = item0 + i * GR + grp;
        if (item >= items) break;  // a whole group alike
        const int64_t at0 = s_place[(int)(item / pool.heads_kv) - row0];
        const int64_t at = at0 + item % pool.heads_kv * KVQ_PAGE;
#pragma unroll
        for (int v = 0; v < 2; v++) {
            float a = 0.0f;
            bool fine = true;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                a = fmaxf(a, fabsf(f[i][v][e]));
                fine = fine && fabsf(f[i][v][e]) < INFINITY;
            }
#pragma unroll
            for (int o = L / 2; o > 0; o >>= 1) a = fmaxf(a, __shfl_xor_sync(mask, a, o));
            fine = __all_sync(mask, fine);
            if (at0 < 0) continue;
            constexpr float M = FMT == LLMDOT_KVQ_I8 ? 127.0f : 448.0f;
            const bool some = fine && a >= 1e-30f;
            if (lane == 0) (v ? pool.v_scale : pool.k_scale)[at] = some ? __fdiv_rn(a, M) : fine ? 0.0f : NAN;
            if (!on) continue;
            const float inv = some ? __fmul_rn(M, __frcp_rn(a)) : 0.0f;
            __align__(8) uint8_t c[8];
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const float y = some ? fminf(fmaxf(__fmul_rn(f[i][v][e], inv), -M), M) : 0.0f;
                if (FMT == LLMDOT_KVQ_I8) c[e] = (uint8_t)(int8_t)__float2int_rn(y);
                else c[e] = __nv_cvt_float_to_fp8(y, __NV_SATFINITE, __NV_E4M3);
            }
            *(uint2 *)((uint8_t *)(v ? pool.v : pool.k) + at * D + lane * 8) = *(const uint2 *)c;
        }
    }
}

template <typename T, int D, int FMT>
__global__ void __launch_bounds__(KVQ_THREADS)
kvq_read_kernel(const llmdot_kvq_pool pool, const llmdot_kvq_batch bt, T *__restrict__ xk, T *__restrict__ xv,
                int64_t ldk, int64_t ldv, int wide)
{
    constexpr int L = kvq_lanes<D>(), GR = KVQ_THREADS / L, N = kvq_items<D>();
    __shared__ int64_t s_place[N];
    const int64_t item0 = (int64_t)blockIdx.x * N, items = (int64_t)bt.rows * pool.heads_kv;
    const int lane = threadIdx.x % L, grp = threadIdx.x / L, row0 = (int)(item0 / pool.heads_kv);
    kvq_find<D>(pool, bt, item0, s_place);
    __syncthreads();
    if (lane * 8 >= D) return;
    uint2 c[KVQ_EACH][2];
    float s[KVQ_EACH][2];
    int64_t at0[KVQ_EACH];
#pragma unroll
    for (int i = 0; i < KVQ_EACH; i++) {
        const int64_t item = item0 + i * GR + grp;
        at0[i] = item < items ? s_place[(int)(item / pool.heads_kv) - row0] : -2;
        const int64_t at = at0[i] + item % pool.heads_kv * KVQ_PAGE;
#pragma unroll
        for (int v = 0; v < 2; v++) {
            c[i][v] = make_uint2(0, 0);
            s[i][v] = 0.0f;
            if (at0[i] >= 0) {
                c[i][v] = __ldg((const uint2 *)((const uint8_t *)(v ? pool.v : pool.k) + at * D + lane * 8));
                s[i][v] = __ldg((v ? pool.v_scale : pool.k_scale) + at);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < KVQ_EACH; i++) {
        if (at0[i] == -2) continue;  // no item, or a row of no sequence
        const int64_t item = item0 + i * GR + grp;
        const int r = (int)(item / pool.heads_kv), h = (int)(item % pool.heads_kv);
#pragma unroll
        for (int v = 0; v < 2; v++) {
            __align__(8) uint8_t b[8];
            *(uint2 *)b = c[i][v];
            float f[8];
#pragma unroll
            for (int e = 0; e < 8; e++) f[e] = at0[i] < 0 ? 0.0f : __fmul_rn(code_value<FMT>(b[e]), s[i][v]);
            store8((v ? xv + r * ldv : xk + r * ldk) + h * D + lane * 8, wide != 0, f);
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

template <int D> unsigned kvq_grid(const llmdot_kvq_pool &p, const llmdot_kvq_batch &b)
{
    return (unsigned)(((int64_t)b.rows * p.heads_kv + kvq_items<D>() - 1) / kvq_items<D>());
}

template <typename T, int D, int FMT> struct WriteOp {
    static cudaError_t launch(const llmdot_kvq_pool &p, const llmdot_kvq_batch &b, const void *k, const void *v, int64_t ldk,
                              int64_t ldv, int wide, cudaStream_t st)
    {
        kvq_write_kernel<T, D, FMT><<<kvq_grid<D>(p, b), KVQ_THREADS, 0, st>>>(
            p, b, (const T *)k, (const T *)v, ldk, ldv, wide);
        return cudaGetLastError();
    }
};
template <typename T, int D, int FMT> struct ReadOp {
    static cudaError_t launch(const llmdot_kvq_pool &p, const llmdot_kvq_batch &b, void *k, void *v, int64_t ldk, int64_t ldv,
                              int wide, cudaStream_t st)
    {
        kvq_read_kernel<T, D, FMT><<<kvq_grid<D>(p, b), KVQ_THREADS, 0, st>>>(
            p, b, (T *)k, (T *)v, ldk, ldv, wide);
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
    if ((int64_t)b->rows * p->heads_kv > (int64_t)1 << 33) return bad("rows * heads_kv exceeds 2^33");
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
