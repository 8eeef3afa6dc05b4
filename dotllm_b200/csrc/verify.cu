// verify.cu -- verification of drafted tokens from given uniform numbers.
//
// Draft i of a sequence is accepted when all before it were and u_i q_i(x_i) < p_i(x_i); the token after
// the accepted ones is drawn from the residual max(p - q, 0) of the refused position (or from p after
// the last draft) by inverting its running sum.  The weights are summed as 64-bit integers
// floor(w * 2^40), so the drawn token does not depend on how the sum is split over threads.
//
// Bound: HBM, one row of p and one of q per sequence (the accepted positions cost two gathers each);
// for few sequences the latency of one pass.  A cluster of CTAs per sequence, every thread finding the
// accepted count for itself; each CTA sums its contiguous span of the vocabulary by blocks of 256
// elements (one warp, eight coalesced loads of p and of q per lane in flight; 4-byte loads, since the rows
// of an odd vocabulary have every alignment and p's differs from q's), keeps the blocks' sums in shared
// memory and pushes its total into the other CTAs' shared memory.  After one cluster barrier every CTA
// knows the total and what lies before its span; the one that holds the threshold finds the block among
// its sums and reads that block alone a second time.
//
// Measured on a B200: 96 sequences, 7 drafts, 256000 tokens 45 us for the 196 MB that their rows take
// (4.3 TB/s; one CTA per sequence took 281 us); 24 sequences, 128255 tokens 13 us; one, 32000 tokens 8.2 us.
// Tried and slower: the next block's loads ahead of this one's sum (54 us), 16 elements per lane (51), 256
// threads (51), the weight's integer by shifts in place of the 64-bit conversion (57 with the loads ahead).
#include <algorithm>

#include "common.cuh"

namespace llmdot {
namespace {

constexpr int VT = 512, VW = VT / 32, VE = 8, VBLOCK = 32 * VE, VCLUSTER = 8;
constexpr int VSPAN = (1 << 22) / VCLUSTER;  // most elements of one CTA
typedef unsigned long long u64;

__device__ __forceinline__ u64 weight(float w)
{
    // fmaxf(NaN, 0) = 0; at most 2^40 each, so 2^22 of them stay below 2^62
    return (u64)__fmul_rn(fminf(fmaxf(w, 0.0f), 1.0f), 1099511627776.0f);
}
__device__ __forceinline__ u64 warp_add(u64 v)
{
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
// The lane whose inclusive running sum (on top of `run`) is the first to exceed t; run becomes the sum
// before it.  Some lane's does.
__device__ __forceinline__ int first_over(u64 x, u64 &run, u64 t)
{
    const int lane = threadIdx.x & 31;
    u64 inc = x;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const u64 y = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += y;
    }
    const int at = __ffs(__ballot_sync(0xffffffffu, run + inc > t)) - 1;
    run += __shfl_sync(0xffffffffu, inc - x, at);
    return at;
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ void push(u64 *local, int rank, u64 v)  // into the same variable of CTA `rank`
{
    uint32_t a = (uint32_t)__cvta_generic_to_shared(local), r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(rank));
    asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(r), "l"(v) : "memory");
}

// blockIdx.x = sequence * cluster size + rank; the cluster is gridDim.x / batch CTAs.
__global__ void __launch_bounds__(VT) verify_kernel(const llmdot_verify a, int C)
{
    extern __shared__ u64 sums[];               // one per block of the span
    __shared__ u64 totals[2][VCLUSTER], s_warp[VW];
    const int b = blockIdx.x / C, rank = blockIdx.x % C, k = a.drafts, V = a.vocab;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    cluster_arrive();  // every CTA of the cluster runs before anything is pushed into it
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
    const float ul = u[k];

    const int blocks = (V + VBLOCK - 1) / VBLOCK, lo = (int)((int64_t)rank * blocks / C), nb = (int)((int64_t)(rank + 1) * blocks / C) - lo;
    int32_t *tok = a.tokens + (int64_t)b * (k + 1);
    auto write = [&](int pick) {
        for (int i = lane; i <= k; i += 32) tok[i] = i < acc ? draft[i] : i == acc ? pick : -1;
        if (lane == 0) a.accepted[b] = acc;
    };
    for (int pass = 0; pass < 2; pass++) {  // the second only when the residual weighs nothing
        const float *qq = pass == 0 ? q : nullptr;
        const int hot = pass == 0 ? out : -1;
        u64 mine = 0;
        for (int i = warp; i < nb; i += VW) {
            const int j0 = (lo + i) * VBLOCK + lane;
            float x[VE], y[VE];
#pragma unroll
            for (int e = 0; e < VE; e++) x[e] = j0 + 32 * e < V ? __ldg(p + j0 + 32 * e) : 0.0f;
#pragma unroll
            for (int e = 0; e < VE; e++) y[e] = qq && j0 + 32 * e < V ? __ldg(qq + j0 + 32 * e) : j0 + 32 * e == hot ? 1.0f : 0.0f;
            u64 s = 0;
#pragma unroll
            for (int e = 0; e < VE; e++) s += weight(__fsub_rn(x[e], y[e]));
            s = warp_add(s);
            if (lane == 0) sums[i] = s;
            mine += s;
        }
        if (lane == 0) s_warp[warp] = mine;
        __syncthreads();
        u64 own = warp_add(lane < VW ? s_warp[lane] : 0ull);
        if (pass == 0) cluster_wait();
        if (warp == 0 && lane < C) push(&totals[pass][rank], lane, own);
        cluster_arrive();
        cluster_wait();
        u64 total = 0, before = 0;
        for (int r = 0; r < C; r++) {
            if (r == rank) before = total;
            total += totals[pass][r];
        }
        if (total == 0) {
            if (refused && pass == 0) continue;  // every CTA of the cluster alike
            if (rank == 0 && warp == 0) write(0);
            return;
        }
        const u64 m = (u64)__fmul_rn(fminf(fmaxf(ul, 0.0f), 0.99999994f), 16777216.0f);
        const u64 t = (total >> 24) * m + (((total & 0xFFFFFFull) * m) >> 24);
        if (warp != 0 || t < before || t >= before + own) return;  // the one CTA whose span holds the threshold
        u64 run = before;
        int blk = 0;
        for (int i0 = 0; i0 < nb; i0 += 32) {
            const u64 s = i0 + lane < nb ? sums[i0 + lane] : 0ull, all = warp_add(s);
            if (t < run + all) {
                blk = i0 + first_over(s, run, t);
                break;
            }
            run += all;
        }
        const int j0 = (lo + blk) * VBLOCK;
        u64 w[VE];
#pragma unroll
        for (int e = 0; e < VE; e++) {
            const int j = j0 + 32 * e + lane;
            w[e] = j < V ? weight(__fsub_rn(p[j], qq ? qq[j] : j == hot ? 1.0f : 0.0f)) : 0ull;
        }
        int pick = 0;
        bool found = false;
#pragma unroll
        for (int e = 0; e < VE; e++) {
            const u64 all = warp_add(w[e]);
            if (!found && t < run + all) {
                pick = j0 + 32 * e + first_over(w[e], run, t);
                found = true;
            }
            if (!found) run += all;
        }
        write(pick);
        return;
    }
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
        if (((uintptr_t)a->draft | (uintptr_t)a->uniform | (uintptr_t)a->n_draft | (uintptr_t)a->tokens | (uintptr_t)a->accepted) & 3)
            return bad("drafts, uniform numbers, counts and results must be 4-byte aligned");
        if (a->ld_p < a->vocab || (a->q && a->ld_q < a->vocab)) return bad("row stride below the vocabulary");
        // CTAs per sequence: as many as still give each warp a block, until the SMs hold two each
        const int blocks = (a->vocab + VBLOCK - 1) / VBLOCK;
        int C = VCLUSTER;
        while (C > 1 && (blocks < C * VW / 2 || (int64_t)a->batch * C > 148 * 4) && a->vocab <= VSPAN / 16 * C) C >>= 1;
        if ((int64_t)a->batch * C > 0x7fffffff) return bad("too many sequences");
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3((unsigned)(a->batch * C));
        cfg.blockDim = dim3(VT);
        cfg.dynamicSmemBytes = (size_t)(blocks / C + 1) * sizeof(u64);
        cfg.stream = (cudaStream_t)stream;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = (unsigned)C;
        attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        LLMDOT_CUDA_TRY(cudaLaunchKernelEx(&cfg, verify_kernel, *a, C));
        return LLMDOT_OK;
    } catch (...) {
        return LLMDOT_E_NOMEM;
    }
}
