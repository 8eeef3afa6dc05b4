// kvq_attn.cu -- attention of a batch over a shared prefix and its own pages, K and V in 8 bits.
//
// s_j = scale * (q . code_j) * k_scale_j, optionally capped; out = sum_j softmax(s)_j v_scale_j code_j.
// One warp per (row, head): lanes over the head dimension, running maximum and sum over positions.
#include "kvq.cuh"

namespace llmdot {
namespace {

template <typename T, int D, int FMT>
__global__ void __launch_bounds__(128)
kvq_attn_kernel(const llmdot_kvq_pool pool, const llmdot_kvq_batch bt, const llmdot_kvq_attn at, const T *__restrict__ q,
                int64_t ldq, T *__restrict__ out, int64_t ldo, float *__restrict__ lse)
{
    constexpr int N = D / 32;
    const int64_t item = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    if (item >= (int64_t)bt.rows * at.heads) return;
    const int r = (int)(item / at.heads), h = (int)(item % at.heads), hk = h / (at.heads / pool.heads_kv);
    const int b = kvq_seq_of(bt.row_start, bt.batch, r);
    if (b < 0 || r - bt.row_start[b] >= bt.max_rows) return;
    const int P = at.prefix_len, S = bt.seq_len[b];
    const int64_t pos = (int64_t)P + S - bt.row_start[b + 1] + r, first = at.window > 0 ? pos - at.window + 1 : 0;
    float x[N], o[N] = {}, m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int i = 0; i < N; i++) x[i] = to_f32<T>(q[r * ldq + h * D + i * 32 + lane]);
    for (int64_t j = first > 0 ? first : 0; j <= pos; j++) {
        int64_t place;
        if (j < P) {
            const int page = at.prefix_pages[j / KVQ_PAGE];
            place = (unsigned)page < (unsigned)pool.n_pages ? ((int64_t)page * pool.heads_kv + hk) * KVQ_PAGE + j % KVQ_PAGE : -1;
        } else {
            place = kvq_place(pool, bt, b, (int)(j - P), hk);
        }
        if (place < 0) continue;
        const uint8_t *kc = (const uint8_t *)pool.k + place * D, *vc = (const uint8_t *)pool.v + place * D;
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < N; i++) s = fmaf(x[i], code_value<FMT>(kc[i * 32 + lane]), s);
        s = warp_sum(s) * pool.k_scale[place] * at.scale;
        if (at.softcap > 0.0f) s = at.softcap * tanhf(s / at.softcap);
        const float mn = fmaxf(m, s), f = m == -INFINITY ? 0.0f : expf(m - mn), p = expf(s - mn);
        l = l * f + p;
#pragma unroll
        for (int i = 0; i < N; i++) o[i] = fmaf(p * pool.v_scale[place], code_value<FMT>(vc[i * 32 + lane]), o[i] * f);
        m = mn;
    }
#pragma unroll
    for (int i = 0; i < N; i++) out[r * ldo + h * D + i * 32 + lane] = from_f32<T>(l == 0.0f ? 0.0f : o[i] / l);
    if (lse && lane == 0) lse[(int64_t)r * at.heads + h] = l == 0.0f ? -INFINITY : m + logf(l);
}

template <typename T, int D, int FMT>
cudaError_t launch(const llmdot_kvq_pool &p, const llmdot_kvq_batch &b, const llmdot_kvq_attn &a, const void *q, int64_t ldq,
                   void *out, int64_t ldo, float *lse, cudaStream_t st)
{
    kvq_attn_kernel<T, D, FMT><<<(unsigned)(((int64_t)b.rows * a.heads + 3) / 4), 128, 0, st>>>(p, b, a, (const T *)q, ldq, (T *)out,
                                                                                              ldo, lse);
    return cudaGetLastError();
}

template <typename T, int FMT, typename... A> cudaError_t by_dim(int dim, A... a)
{
    switch (dim) {
    case 64: return launch<T, 64, FMT>(a...);
    case 96: return launch<T, 96, FMT>(a...);
    case 128: return launch<T, 128, FMT>(a...);
    default: return launch<T, 256, FMT>(a...);
    }
}

int check_attn(const char *who, const llmdot_kvq_pool *p, const llmdot_kvq_batch *b, const llmdot_kvq_attn *a)
{
    LLMDOT_TRY(kvq_check(who, p, b));
    auto bad = [&](const char *what) { return fail(LLMDOT_E_INVALID, std::string(who) + ": " + what); };
    if (!a) return bad("null attention arguments");
    if (!kvq_type_ok(a->type)) return fail(LLMDOT_E_UNSUPPORTED, std::string(who) + ": type must be F32, F16 or BF16");
    if (a->heads <= 0 || a->heads % p->heads_kv || a->heads > (1 << 16)) return bad("heads must be a multiple of heads_kv, at most 65536");
    if (a->prefix_len < 0 || a->prefix_len > (1 << 30) || a->window < 0) return bad("bad prefix_len or window");
    if (a->prefix_len > 0 && !a->prefix_pages) return bad("null prefix_pages");
    if (!(a->softcap >= 0.0f) || !(a->softcap < INFINITY) || !(fabsf(a->scale) < INFINITY)) return bad("bad scale or softcap");
    if ((int64_t)b->rows * a->heads > (int64_t)1 << 30) return bad("rows * heads exceeds 2^30");
    return LLMDOT_OK;
}

}  // namespace
}  // namespace llmdot

using namespace llmdot;

extern "C" int llmdot_cuda_kvq_attention_workspace(const llmdot_kvq_pool *pool, const llmdot_kvq_batch *batch,
                                                   const llmdot_kvq_attn *attn, size_t *bytes)
{
    return c_boundary([&]() -> int {
        LLMDOT_TRY(check_attn("kvq_attention_workspace", pool, batch, attn));
        if (!bytes) return fail(LLMDOT_E_INVALID, "kvq_attention_workspace: bytes is null");
        *bytes = 0;
        return LLMDOT_OK;
    });
}

extern "C" int llmdot_cuda_kvq_attention(const llmdot_kvq_pool *pool, const llmdot_kvq_batch *batch, const llmdot_kvq_attn *attn,
                                         const void *d_q, int64_t ld_q, void *d_out, int64_t ld_out, float *d_lse, void *d_work,
                                         size_t work_bytes, void *stream)
{
    return c_boundary([&]() -> int {
        LLMDOT_TRY(check_attn("kvq_attention", pool, batch, attn));
        auto bad = [&](const char *what) { return fail(LLMDOT_E_INVALID, std::string("kvq_attention: ") + what); };
        if (batch->rows == 0) return LLMDOT_OK;
        const int64_t row = (int64_t)attn->heads * pool->head_dim;
        if (!d_q || !d_out) return bad("null q or output");
        if (batch->rows > 1 && (ld_q < row || ld_out < row)) return bad("row stride below heads * head_dim");
        if (((uintptr_t)d_q | (uintptr_t)d_out) % kvq_type_size(attn->type)) return bad("q or output is not aligned to its type");
        (void)d_work;
        (void)work_bytes;
        cudaError_t e;
        auto go = [&](auto t) {
            using T = decltype(t);
            return pool->format == LLMDOT_KVQ_I8
                       ? by_dim<T, LLMDOT_KVQ_I8>(pool->head_dim, *pool, *batch, *attn, d_q, ld_q, d_out, ld_out, d_lse, (cudaStream_t)stream)
                       : by_dim<T, LLMDOT_KVQ_E4M3>(pool->head_dim, *pool, *batch, *attn, d_q, ld_q, d_out, ld_out, d_lse, (cudaStream_t)stream);
        };
        if (attn->type == T_F32) e = go(float{});
        else if (attn->type == T_F16) e = go(__half{});
        else e = go(__nv_bfloat16{});
        if (e != cudaSuccess) return cuda_fail(e, "kvq_attention");
        return LLMDOT_OK;
    });
}
