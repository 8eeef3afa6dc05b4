// verify.cu -- verification of drafted tokens from given uniform numbers.
//
// Draft i of a sequence is accepted when all before it were and u_i q_i(x_i) < p_i(x_i); the token after
// the accepted ones is drawn from the residual max(p - q, 0) of the refused position (or from p after
// the last draft) by inverting its running sum.  The weights are summed as 64-bit integers
// floor(w * 2^40), so the drawn token does not depend on how the sum is split over threads.
//
// Bound: HBM, one row of p and one of q per sequence (the accepted positions cost two gathers each).
// One CTA per sequence: every thread finds the accepted count for itself, the CTA sums the weights
// (one contiguous span per warp), then the warp whose span holds the threshold walks it again.
#include "common.cuh"

namespace llmdot {
namespace {

constexpr int VT = 1024, VW = VT / 32;

__device__ __forceinline__ unsigned long long weight(float w)
{
    // fmaxf(NaN, 0) = 0; at most 2^40 each, so 2^22 of them stay below 2^62
    return (unsigned long long)__fmul_rn(fminf(fmaxf(w, 0.0f), 1.0f), 1099511627776.0f);
}
__device__ __forceinline__ unsigned long long warp_add(unsigned long long v)
{
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

__global__ void __launch_bounds__(VT) verify_kernel(const llmdot_verify a)
{
    __shared__ unsigned long long part[VW];
    __shared__ int pick;
    const int b = blockIdx.x, k = a.drafts, V = a.vocab, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int32_t *draft = a.draft + (int64_t)b * k;
    const float *u = a.uniform + (int64_t)b * (k + 1);
    int n = k;
    if (a.n_draft) n = min(max(a.n_draft[b], 0), k);
    // the first refused draft (two per lane)
    unsigned ok[2];
#pragma unroll
    for (int h = 0; h < 2; h++) {
        const int i = 32 * h + lane;
        bool acc = false;
        if (i < n) {
            const int x = draft[i];
            if ((unsigned)x < (unsigned)V) {
                const float px = a.p[((int64_t)b * (k + 1) + i) * a.ld_p + x];
                const float qx = a.q ? a.q[((int64_t)b * k + i) * a.ld_q + x] : 1.0f;
                acc = __fmul_rn(u[i], qx) < px;
            }
        }
        ok[h] = __ballot_sync(0xffffffffu, acc);
    }
    const int acc = ok[0] != 0xffffffffu ? __ffs(~ok[0]) - 1 : ok[1] != 0xffffffffu ? 31 + __ffs(~ok[1]) : 64;
    const float *p = a.p + ((int64_t)b * (k + 1) + acc) * a.ld_p;
    const bool refused = acc < n;
    const float *q = refused && a.q ? a.q + ((int64_t)b * k + acc) * a.ld_q : nullptr;
    const int out = refused && !a.q ? draft[acc] : -1;  // one-hot draft: its own weight goes

    // spans of whole 32-element steps per warp
    const int steps = (V + 31) / 32, per = (steps + VW - 1) / VW;
    const int lo = min(warp * per, steps), hi = min(lo + per, steps);
    for (int pass = 0; pass < 2; pass++) {  // the second only when the residual weighs nothing
        auto w = [&](int j) -> unsigned long long {
            if (j >= V) return 0ull;
            float x = p[j];
            if (pass == 0 && q) x = __fsub_rn(x, q[j]);
            if (pass == 0 && j == out) x = __fsub_rn(x, 1.0f);
            return weight(x);
        };
        unsigned long long s = 0;
        for (int i = lo; i < hi; i++) s += w(i * 32 + lane);
        s = warp_add(s);
        if (lane == 0) part[warp] = s;
        if (threadIdx.x == 0) pick = 0;
        __syncthreads();
        unsigned long long total = 0, before = 0;
        for (int i = 0; i < VW; i++) {
            if (i == warp) before = total;
            total += part[i];
        }
        const unsigned long long m = (unsigned long long)__fmul_rn(fminf(fmaxf(u[k], 0.0f), 0.99999994f), 16777216.0f);
        const unsigned long long t = (total >> 24) * m + (((total & 0xFFFFFFull) * m) >> 24);
        if (total > 0 && before <= t && t < before + s) {  // the one warp whose span holds the threshold
            unsigned long long run = before;
            for (int i = lo; i < hi; i++) {
                const unsigned long long x = w(i * 32 + lane), sum = warp_add(x);
                if (t < run + sum) {
                    unsigned long long inc = x;
#pragma unroll
                    for (int o = 1; o < 32; o <<= 1) {
                        const unsigned long long y = __shfl_up_sync(0xffffffffu, inc, o);
                        if (lane >= o) inc += y;
                    }
                    const unsigned hit = __ballot_sync(0xffffffffu, run + inc > t);
                    if (lane == 0) pick = i * 32 + __ffs(hit) - 1;
                    break;
                }
                run += sum;
            }
        }
        __syncthreads();
        if (total > 0 || !refused) break;
        __syncthreads();
    }
    int32_t *tok = a.tokens + (int64_t)b * (k + 1);
    for (int i = threadIdx.x; i <= k; i += VT) tok[i] = i < acc ? draft[i] : i == acc ? pick : -1;
    if (threadIdx.x == 0) a.accepted[b] = acc;
}

}  // namespace
}  // namespace llmdot

using namespace llmdot;

extern "C" int llmdot_cuda_verify_draft(const llmdot_verify *a, void *stream)
{
    try {
        auto bad = [&](const char *what) { return fail(LLMDOT_E_INVALID, std::string("verify_draft: ") + what); };
        if (!a) return bad("null arguments");
        if (a->batch < 0 || a->drafts < 0 || a->vocab <= 0) return bad("bad batch, drafts or vocab");
        if (a->drafts > 64 || a->vocab > (1 << 22))
            return fail(LLMDOT_E_UNSUPPORTED, "verify_draft: more than 64 drafts or 4194304 tokens");
        if (a->batch == 0) return LLMDOT_OK;
        if (!a->p || !a->uniform || !a->tokens || !a->accepted) return bad("null device pointer");
        if (a->drafts > 0 && !a->draft) return bad("null drafts");
        if (((uintptr_t)a->p | (uintptr_t)a->q) & 3) return bad("probabilities must be 4-byte aligned");
        if (a->ld_p < a->vocab || (a->q && a->ld_q < a->vocab)) return bad("row stride below the vocabulary");
        verify_kernel<<<a->batch, VT, 0, (cudaStream_t)stream>>>(*a);
        LLMDOT_CUDA_TRY(cudaGetLastError());
        return LLMDOT_OK;
    } catch (...) {
        return LLMDOT_E_NOMEM;
    }
}
