// kvq_attn_tc.cu -- shared-prefix attention for segments with many rows, on tcgen05.
//
// Same mathematics as kvq_attn.cu (codes exact in fp16, the key's scale on the score, the value's scale
// in the weight), for 16-bit queries; leaves partials (m, l, O) that the joining kernel adds.
//
// Bound: with hundreds of rows per kv head the products, the exponentials (16 per clock and SM) and
// the conversion of codes to fp16 take about the same time, and HBM little.  So one CTA takes two tiles of
// 128 rows (one for head_dim 256) over the same positions -- each code is converted once for 256 rows --
// and its roles overlap, 64 positions (a page) at a time:
//   warps of a tile (4 each)  a thread per row: S from TMEM, scale, mask, running maximum, exponentials,
//                             the weights as fp16 back into TMEM over S; rescales O in TMEM only when
//                             its maximum rose by more than 2^8 (fp16 holds weights up to 2^13)
//   4 converting warps        codes from global memory (next page's loads in flight) to fp16 K and V^T
//                             operands in shared memory (three stages), scales beside them
//   1 warp                    one thread issues tcgen05.mma: S = Q K^T and O += P V with Q, P and the
//                             accumulators in TMEM; while one tile's rows are in their softmax, the other
//                             tile's products run
// Operands in shared memory are unswizzled K-major core matrices (8 rows x 16 bytes).  K: cores adjacent
// along head_dim 128 bytes apart.  V is transposed on conversion (a lane holds eight positions of eight
// dimensions and permutes bytes): cores adjacent along positions are 144 bytes apart, which spreads
// the eight lanes that write one dimension's pieces over all banks.
// Every wait is bounded; one that gives up leaves NaN partials, so the output shows it.
#include "kvq_attn.cuh"

namespace llmdot {
namespace {

constexpr int UN = KVQ_PAGE;  // positions per unit
constexpr int STAGES = 3;
constexpr unsigned long long WAIT_NS = 2000000000ull;
constexpr float RAISE = 8.0f;  // the maximum may lag by this power of two

template <int D> struct Wide {
    static constexpr int TILES = D == 256 ? 1 : 2;
    static constexpr int THREADS = TILES * 128 + 128 + 32;
    static constexpr uint32_t K_SBO = D / 8 * 128, V_LBO = 144, V_SBO = 8 * V_LBO;
    static constexpr uint32_t K_BYTES = 8 * K_SBO, V_BYTES = D / 8 * V_SBO;
    static constexpr uint32_t STAGE = K_BYTES + V_BYTES;
    static constexpr uint32_t OFF_SC = STAGES * STAGE;  // per stage: K scales, V scales, {rescale, 2^E, bad, -}
    static constexpr uint32_t SC_STAGE = 2 * UN * 4 + 16;
    static constexpr uint32_t OFF_BAR = OFF_SC + STAGES * SC_STAGE;
    static constexpr int B_FULL = 0, B_EMPTY = STAGES, B_S = 2 * STAGES, B_P = B_S + 2, B_O = B_P + 2, B_DRAIN = B_O + 2,
                         B_COUNT = B_DRAIN + 1;
    static constexpr uint32_t SMEM = OFF_BAR + B_COUNT * 8 + 16;
    static constexpr int QC = D / 2;  // TMEM columns of Q
    static constexpr int TILE_COLS = (D + UN + QC + 31) / 32 * 32;
    static constexpr int C_O = 0, C_S = D, C_Q = D + UN;
    static_assert(TILES * TILE_COLS <= 512, "TMEM columns");
    static_assert(SMEM <= 227 * 1024, "shared memory");
};

__device__ __forceinline__ uint32_t su32(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ unsigned long long gtime()
{
    unsigned long long t;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
    return t;
}
__device__ __forceinline__ void bar_init(uint32_t b, uint32_t count)
{
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(b), "r"(count) : "memory");
}
__device__ __forceinline__ void bar_arrive(uint32_t b)
{
    asm volatile("mbarrier.arrive.release.cta.shared::cta.b64 _, [%0];" ::"r"(b) : "memory");
}
__device__ __forceinline__ bool bar_try(uint32_t b, uint32_t parity)
{
    uint32_t ok;
    asm volatile("{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
                 : "=r"(ok)
                 : "r"(b), "r"(parity)
                 : "memory");
    return ok != 0;
}
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
// shared-memory matrix descriptor: no swizzle, K-major cores; lbo: K-adjacent cores, sbo: 8-row groups
__device__ __forceinline__ uint64_t sdesc(uint32_t addr, uint32_t lbo, uint32_t sbo)
{
    return (uint64_t)((addr >> 4) & 0x3FFFu) | ((uint64_t)((lbo >> 4) & 0x3FFFu) << 16) |
           ((uint64_t)((sbo >> 4) & 0x3FFFu) << 32) | (1ull << 46);
}
// kind::f16, fp32 accumulator, fp16 A (TMEM) and B (shared memory), M = 128
template <int N> __device__ __forceinline__ void umma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t acc)
{
    constexpr uint32_t idesc = (1u << 4) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
    asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
                 " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d),
                 "r"(a), "l"(b), "r"(idesc), "r"(acc)
                 : "memory");
}
__device__ __forceinline__ void umma_commit(uint32_t b)
{
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(b) : "memory");
}
// 32 consecutive 32-bit TMEM columns of this thread's lane
__device__ __forceinline__ void tmem_ld32(uint32_t ta, uint32_t *v)
{
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
                 "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
                   "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]),
                   "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]),
                   "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
                 : "r"(ta));
}
__device__ __forceinline__ void tmem_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_st16(uint32_t ta, const uint32_t *v)
{
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(ta),
                 "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
                 "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
                 : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void sts128(uint32_t a, uint32_t x, uint32_t y, uint32_t z, uint32_t w)
{
    asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(a), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}

template <typename T> __device__ __forceinline__ float query_top(const T *q, bool wide, int D)
{
    float top = 0.0f;
    for (int c = 0; c < D; c += 8) {
        float f[8];
        load8(q + c, wide, f);
#pragma unroll
        for (int e = 0; e < 8; e++) top = fmaxf(top, fabsf(f[e]));
    }
    return top;
}
// 32 scaled values of the row as 16 fp16 pairs
template <typename T> __device__ __forceinline__ void query_pairs(const T *q, bool wide, float up, uint32_t (&v)[16])
{
#pragma unroll
    for (int c = 0; c < 4; c++) {
        float f[8];
        load8(q + 8 * c, wide, f);
#pragma unroll
        for (int e = 0; e < 4; e++) v[4 * c + e] = pack(f[2 * e] * up, f[2 * e + 1] * up);
    }
}

template <int D, int FMT>
__global__ void __launch_bounds__(Wide<D>::THREADS, 1) kvq_wide_kernel(const __grid_constant__ AttnArgs a, const int qwide)
{
    using W = Wide<D>;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ int s_lo[8], s_hi[8], s_abort;
    __shared__ uint32_t s_tmem;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int G = a.group, Hk = a.pool.heads_kv;
    const uint32_t base = su32(smem), bars = base + W::OFF_BAR;
    pdl_launch();
    Segment sg;
    if (!segment_of(a, W::TILES * 128, sg)) {
        if (a.chained) pdl_wait();
        return;
    }
    const int row_first = sg.tile * W::TILES * 128, len = sg.len;
    const int nact = min(W::TILES, (sg.nrows * G - row_first + 127) / 128);  // tiles with rows

    auto wait = [&](int bi, uint32_t parity) -> bool {  // bounded; gives up with another role too
        const uint32_t b = bars + 8 * bi;
        if (bar_try(b, parity)) return true;
        const unsigned long long t0 = gtime();
        while (!bar_try(b, parity)) {
            if (*(volatile int *)&s_abort || gtime() - t0 > WAIT_NS) {
                *(volatile int *)&s_abort = 1;
                return false;
            }
        }
        return true;
    };

    // ---- set-up: barriers, TMEM, the rows' ranges
    constexpr int SOFT = W::TILES * 128;
    if (tid == SOFT) {
        for (int i = 0; i < W::B_COUNT; i++)
            bar_init(bars + 8 * i, i < STAGES || (i >= W::B_P && i < W::B_P + 2) ? 128u : 1u);
        s_abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == SOFT / 32 + 4) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(su32(&s_tmem)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    int row = -1, lo = 0, hi = 0x7fffffff;
    if (tid < SOFT) {
        row_range(a, sg, row_first + tid, row, lo, hi);
        const int wlo = __reduce_min_sync(0xffffffffu, row >= 0 ? lo : 0x7fffffff);
        const int whi = __reduce_max_sync(0xffffffffu, row >= 0 ? hi : -1);
        if (lane == 0) {
            s_lo[warp] = wlo;
            s_hi[warp] = whi;
        }
    }
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = s_tmem;
    int lo_min = 0x7fffffff, hi_max = -1;
#pragma unroll
    for (int w = 0; w < SOFT / 32; w++) {
        lo_min = min(lo_min, s_lo[w]);
        hi_max = max(hi_max, s_hi[w]);
    }
    const int u0 = max(sg.chunk * sg.ch, lo_min / UN);
    const int u1 = min((sg.chunk + 1) * sg.ch, hi_max < 0 ? 0 : hi_max / UN + 1), n = max(u1 - u0, 0);

    if (warp < SOFT / 32) {
        // ------------------------------------------------------------ a row per thread
        const int tile = warp >> 2, head = sg.kvh * G + (row_first + tid) % G;
        const uint32_t tm = tmem + tile * W::TILE_COLS + ((uint32_t)(32 * (warp & 3)) << 16);
        // the query, scaled by a power of two, into TMEM (zeros for rows that do not exist)
        float qf;
        {
            const int64_t at = row < 0 ? 0 : row * a.ldq + (int64_t)head * D;
            const bool half = a.at.type == T_F16;
            float top = 0.0f;
            if (row >= 0) top = half ? query_top((const __half *)a.q + at, qwide != 0, D) : query_top((const __nv_bfloat16 *)a.q + at, qwide != 0, D);
            const int e = row_exponent(top);
            const float up = a.at.scale < 0.0f ? -pow2(e) : pow2(e);
            for (int c = 0; c < D / 32; c++) {
                uint32_t v[16] = {};
                if (row >= 0) {
                    if (half) query_pairs((const __half *)a.q + at + 32 * c, qwide != 0, up, v);
                    else query_pairs((const __nv_bfloat16 *)a.q + at + 32 * c, qwide != 0, up, v);
                }
                __syncwarp();
                tmem_st16(tm + W::C_Q + 16 * c, v);
            }
            qf = fabsf(a.at.scale) * code_unit<FMT>() * (a.at.softcap > 0.0f ? 1.0f : 1.4426950408889634f) * pow2(-e);
        }
        tmem_st_wait();
        fence_before();
        __syncthreads();
        const int lo_max = __reduce_max_sync(0xffffffffu, row >= 0 ? lo : 0);
        const int hi_min = __reduce_min_sync(0xffffffffu, row >= 0 ? hi : 0x7fffffff);
        const bool cap = a.at.softcap > 0.0f;
        const float inv_cap2 = cap ? 2.0f * 1.4426950408889634f / a.at.softcap : 0.0f;
        float m = -INFINITY, l = 0.0f, vpow = 0.0f;  // maximum in base 2
        bool ok = tile < nact;
        for (int i = 0; i < n && ok; i++) {
            const int st = i % STAGES;
            ok = wait(W::B_S + tile, i & 1) && wait(W::B_FULL + st, (i / STAGES) & 1);
            if (!(ok = __all_sync(0xffffffffu, ok))) break;
            fence_after();
            const float *ks = (const float *)(smem + W::OFF_SC + st * W::SC_STAGE), *vs = ks + UN, *ex = vs + UN;
            uint32_t s[UN];
            tmem_ld32(tm + W::C_S, s);
            tmem_ld32(tm + W::C_S + 32, s + 32);
            tmem_ld_wait();
            const int t0 = (u0 + i) * UN;
            const bool whole = t0 >= lo_max && t0 + UN - 1 <= hi_min && ex[2] == 0.0f;
            float x[UN], mx = -INFINITY, qx = qf;
#pragma unroll
            for (int j = 0; j < UN; j += 4) {
                const float4 k4 = *(const float4 *)(ks + j);
                x[j] = __uint_as_float(s[j]) * k4.x;
                x[j + 1] = __uint_as_float(s[j + 1]) * k4.y;
                x[j + 2] = __uint_as_float(s[j + 2]) * k4.z;
                x[j + 3] = __uint_as_float(s[j + 3]) * k4.w;
            }
            if (cap) {
#pragma unroll
                for (int j = 0; j < UN; j++) x[j] = capped<false>(x[j] * qf, a.at.softcap, inv_cap2) * 1.4426950408889634f;
                qx = 1.0f;
            }
            if (!whole) {
                const bool bad = ex[2] != 0.0f;
#pragma unroll
                for (int j = 0; j < UN; j++)
                    if (bad || t0 + j < lo || t0 + j > hi || t0 + j >= len) x[j] = -INFINITY;
            }
#pragma unroll
            for (int j = 0; j < UN; j++) mx = fmaxf(mx, x[j]);
            const float top = mx == -INFINITY ? -INFINITY : mx * qx;
            const bool raise = top > m + RAISE || (m == -INFINITY && top > -INFINITY);
            const float f = raise ? ex2(m - top) : 1.0f, ve = ex[0];
            if (raise) m = top;
            l *= f;
            vpow = ex[1];
            if (i > 0 && __any_sync(0xffffffffu, raise || ve != 1.0f)) {
                ok = wait(W::B_O + tile, (i - 1) & 1);
                if (!(ok = __all_sync(0xffffffffu, ok))) break;
                fence_after();
                const float fo = f * ve;
#pragma unroll 1
                for (int c = 0; c < D / 32; c++) {
                    uint32_t v[32];
                    tmem_ld32(tm + W::C_O + 32 * c, v);
                    tmem_ld_wait();
#pragma unroll
                    for (int j = 0; j < 32; j++) v[j] = __float_as_uint(__uint_as_float(v[j]) * fo);
                    tmem_st16(tm + W::C_O + 32 * c, v);
                    tmem_st16(tm + W::C_O + 32 * c + 16, v + 16);
                }
            }
            const float off = m == -INFINITY ? 0.0f : m;
            uint32_t p[UN / 2];
#pragma unroll
            for (int j = 0; j < UN; j += 4) {
                const float4 v4 = *(const float4 *)(vs + j);
                float y[4], w[4];
#pragma unroll
                for (int e = 0; e < 4; e++) y[e] = ex2(fmaf(x[j + e], qx, -off));
                w[0] = y[0] * v4.x;
                w[1] = y[1] * v4.y;
                w[2] = y[2] * v4.z;
                w[3] = y[3] * v4.w;
                if (!whole) {
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        if (x[j + e] == -INFINITY) y[e] = w[e] = 0.0f;  // whatever the unseen position holds
                }
                l += (y[0] + y[1]) + (y[2] + y[3]);
                p[j / 2] = pack(w[0], w[1]);
                p[j / 2 + 1] = pack(w[2], w[3]);
            }
            tmem_st16(tm + W::C_S, p);
            tmem_st16(tm + W::C_S + 16, p + 16);
            tmem_st_wait();
            fence_before();
            bar_arrive(bars + 8 * (W::B_P + tile));
        }
        if (ok && n > 0) {
            ok = wait(W::B_O + tile, (n - 1) & 1);
            ok = __all_sync(0xffffffffu, ok);
        }
        const int64_t RH = (int64_t)a.bt.rows * a.at.heads, slot = sg.pre ? sg.chunk : a.nsp + sg.chunk;
        const int64_t at = slot * RH + (int64_t)row * a.at.heads + head;
        if (ok && n > 0) {
            fence_after();
#pragma unroll 1
            for (int c = 0; c < D / 32; c++) {
                uint32_t v[32];
                tmem_ld32(tm + W::C_O + 32 * c, v);
                tmem_ld_wait();
                if (row >= 0) {
                    float4 *o = (float4 *)(a.part_o + at * D + 32 * c);
#pragma unroll
                    for (int j = 0; j < 8; j++)
                        o[j] = make_float4(__uint_as_float(v[4 * j]) * vpow, __uint_as_float(v[4 * j + 1]) * vpow,
                                           __uint_as_float(v[4 * j + 2]) * vpow, __uint_as_float(v[4 * j + 3]) * vpow);
                }
            }
        }
        if (row >= 0) a.part_ml[at] = ok ? make_float2(m, l) : make_float2(0.0f, NAN);
    } else if (warp < SOFT / 32 + 4) {
        // ------------------------------------------------------------ codes to operands
        const int dt = tid - SOFT, dw = dt >> 5;
        constexpr int KT = D / 32, VT = (D + 127) / 128;
        struct Codes {
            uint4 k[KT];
            uint2 v[VT][8];
            float sc[2];
            bool bad;
        };
        auto page_of = [&](int u) { return u < u1 ? __ldg(sg.pages + u) : -1; };
        auto load = [&](int page, Codes &c) {
            c.bad = (unsigned)page >= (unsigned)a.pool.n_pages;
            if (c.bad) {
#pragma unroll
                for (int i = 0; i < KT; i++) c.k[i] = make_uint4(0, 0, 0, 0);
#pragma unroll
                for (int i = 0; i < VT; i++)
#pragma unroll
                    for (int j = 0; j < 8; j++) c.v[i][j] = make_uint2(0, 0);
                c.sc[0] = c.sc[1] = 0.0f;
                return;
            }
            const int64_t at = ((int64_t)page * Hk + sg.kvh) * KVQ_PAGE;
            const uint8_t *k = (const uint8_t *)a.pool.k + at * D, *v = (const uint8_t *)a.pool.v + at * D;
#pragma unroll
            for (int i = 0; i < KT; i++) {
                const int t = dt + 128 * i, r7 = t & 7, ch = (t >> 3) % (D / 16), rg = (t >> 3) / (D / 16);
                c.k[i] = __ldg((const uint4 *)(k + (rg * 8 + r7) * D + ch * 16));
            }
#pragma unroll
            for (int i = 0; i < VT; i++) {
                const int t = dt + 128 * i, tk = t & 7, c8 = t >> 3;
                if (t < D)
#pragma unroll
                    for (int j = 0; j < 8; j++) c.v[i][j] = __ldg((const uint2 *)(v + (tk * 8 + j) * D + c8 * 8));
            }
            if (dw < 2) {  // warp 0: V's scales, warp 1: K's
                const float *s = (dw == 0 ? a.pool.v_scale : a.pool.k_scale) + at;
                c.sc[0] = __ldg(s + lane);
                c.sc[1] = __ldg(s + lane + 32);
            }
        };
        Codes cur, nxt;
        load(page_of(u0), cur);
        int page = page_of(u0 + 1);
        __syncthreads();
        float vp = 0.0f;  // 2^E (warp 0)
        bool ok = true;
        for (int i = 0; i < n && ok; i++) {
            const int st = i % STAGES;
            load(page, nxt);
            page = page_of(u0 + i + 2);
            if (i >= STAGES) {
                ok = wait(W::B_EMPTY + st, (i / STAGES - 1) & 1);
                if (!(ok = __all_sync(0xffffffffu, ok))) break;
            }
            const uint32_t ka = base + st * W::STAGE, va = ka + W::K_BYTES;
#pragma unroll
            for (int x = 0; x < KT; x++) {
                const int t = dt + 128 * x, r7 = t & 7, ch = (t >> 3) % (D / 16), rg = (t >> 3) / (D / 16);
                const uint32_t w[4] = {cur.k[x].x ^ code_flip<FMT>(), cur.k[x].y ^ code_flip<FMT>(), cur.k[x].z ^ code_flip<FMT>(),
                                       cur.k[x].w ^ code_flip<FMT>()};
                const uint32_t d = ka + rg * W::K_SBO + ch * 256 + r7 * 16;
                sts128(d, codes2<FMT, 0, 1>(w[0]), codes2<FMT, 2, 3>(w[0]), codes2<FMT, 0, 1>(w[1]), codes2<FMT, 2, 3>(w[1]));
                sts128(d + 128, codes2<FMT, 0, 1>(w[2]), codes2<FMT, 2, 3>(w[2]), codes2<FMT, 0, 1>(w[3]), codes2<FMT, 2, 3>(w[3]));
            }
#pragma unroll
            for (int x = 0; x < VT; x++) {
                const int t = dt + 128 * x, tk = t & 7, c8 = t >> 3;
                if (t < D) {
                    const uint32_t d = va + c8 * W::V_SBO + tk * W::V_LBO;
#pragma unroll
                    for (int wd = 0; wd < 2; wd++)
#pragma unroll
                        for (int h = 0; h < 2; h++) {
                            uint32_t ab[4];
#pragma unroll
                            for (int j = 0; j < 4; j++) {
                                const uint32_t r0 = (wd ? cur.v[x][2 * j].y : cur.v[x][2 * j].x) ^ code_flip<FMT>();
                                const uint32_t r1 = (wd ? cur.v[x][2 * j + 1].y : cur.v[x][2 * j + 1].x) ^ code_flip<FMT>();
                                ab[j] = __byte_perm(r0, r1, h ? 0x7362 : 0x5140);
                            }
                            const int dd = wd * 4 + h * 2;
                            sts128(d + dd * 16, codes2<FMT, 0, 1>(ab[0]), codes2<FMT, 0, 1>(ab[1]), codes2<FMT, 0, 1>(ab[2]),
                                   codes2<FMT, 0, 1>(ab[3]));
                            sts128(d + dd * 16 + 16, codes2<FMT, 2, 3>(ab[0]), codes2<FMT, 2, 3>(ab[1]), codes2<FMT, 2, 3>(ab[2]),
                                   codes2<FMT, 2, 3>(ab[3]));
                        }
                }
            }
            float *ks = (float *)(smem + W::OFF_SC + st * W::SC_STAGE), *vs = ks + UN, *ex = vs + UN;
            if (dw == 0) {
                const int t0 = (u0 + i) * UN + lane;
                const float v0 = cur.sc[0] * code_unit<FMT>(), v1 = cur.sc[1] * code_unit<FMT>();
                float top = 0.0f;  // of positions that exist; a NaN does not count
                if (t0 < len) top = fmaxf(top, v0);
                if (t0 + 32 < len) top = fmaxf(top, v1);
                const float pw = scale_pow(warp_max(top));
                float ve = 1.0f;
                if (i == 0) {
                    vp = pw;
                } else if (pw > vp * 8.0f) {  // weights stay below 2^8 * 2 * 8
                    ve = vp * pow_inverse(pw);
                    vp = pw;
                }
                const float inv = pow_inverse(vp);
                vs[lane] = v0 * inv;
                vs[lane + 32] = v1 * inv;
                if (lane == 0) {
                    ex[0] = ve;
                    ex[1] = vp;
                    ex[2] = cur.bad ? 1.0f : 0.0f;
                }
            } else if (dw == 1) {
                ks[lane] = cur.sc[0];
                ks[lane + 32] = cur.sc[1];
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // operands: generic writes -> tensor core
            bar_arrive(bars + 8 * (W::B_FULL + st));
            cur = nxt;
        }
    } else {
        // ------------------------------------------------------------ products
        __syncthreads();
        if (lane == 0 && n > 0) {
            fence_after();
            auto qk = [&](int t, int st) {
                const uint32_t k = base + st * W::STAGE, tm = tmem + t * W::TILE_COLS;
#pragma unroll
                for (int kk = 0; kk < D / 16; kk++)
                    umma_ts<UN>(tm + W::C_S, tm + W::C_Q + 8 * kk, sdesc(k + kk * 256, 128, W::K_SBO), kk != 0);
                umma_commit(bars + 8 * (W::B_S + t));
            };
            bool ok = wait(W::B_FULL, 0);
            fence_after();
            for (int t = 0; t < nact && ok; t++) qk(t, 0);
            for (int i = 0; i < n && ok; i++) {
                const int st = i % STAGES, nx = (i + 1) % STAGES;
                for (int t = 0; t < nact; t++) {
                    if (!(ok = wait(W::B_P + t, i & 1))) break;
                    fence_after();
                    const uint32_t v = base + st * W::STAGE + W::K_BYTES, tm = tmem + t * W::TILE_COLS;
#pragma unroll
                    for (int kk = 0; kk < UN / 16; kk++)
                        umma_ts<D>(tm + W::C_O, tm + W::C_S + 8 * kk, sdesc(v + kk * 2 * W::V_LBO, W::V_LBO, W::V_SBO), i != 0 || kk != 0);
                    umma_commit(bars + 8 * (W::B_O + t));
                    if (t == nact - 1) umma_commit(bars + 8 * (W::B_EMPTY + st));
                    if (i + 1 < n) {
                        if (t == 0) {
                            if (!(ok = wait(W::B_FULL + nx, ((i + 1) / STAGES) & 1))) break;
                            fence_after();
                        }
                        qk(t, nx);
                    }
                }
            }
            // every product issued completes before the TMEM is released
            umma_commit(bars + 8 * W::B_DRAIN);
            const unsigned long long t0 = gtime();
            while (!bar_try(bars + 8 * W::B_DRAIN, 0) && gtime() - t0 < WAIT_NS) {}
        }
        __syncwarp();
    }
    fence_before();
    __syncthreads();
    fence_after();
    if (warp == SOFT / 32 + 4)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
    if (a.chained) pdl_wait();
}

template <int D, int FMT> cudaError_t launch(const AttnArgs &a, int64_t ctas, bool pdl, cudaStream_t st)
{
    using W = Wide<D>;
    static std::atomic<unsigned long long> done{0};
    cudaError_t e = smem_attr_once(done, kvq_wide_kernel<D, FMT>, W::SMEM);
    if (e != cudaSuccess) return e;
    const int qwide = ((uintptr_t)a.q & 15) == 0 && (a.bt.rows <= 1 || a.ldq * 2 % 16 == 0);
    return launch_kernel(pdl, kvq_wide_kernel<D, FMT>, dim3((unsigned)ctas), dim3(W::THREADS), W::SMEM, st, a, qwide);
}
template <int FMT> cudaError_t by_dim(const AttnArgs &a, int64_t ctas, bool pdl, cudaStream_t st)
{
    switch (a.pool.head_dim) {
    case 64: return launch<64, FMT>(a, ctas, pdl, st);
    case 96: return launch<96, FMT>(a, ctas, pdl, st);
    case 128: return launch<128, FMT>(a, ctas, pdl, st);
    default: return launch<256, FMT>(a, ctas, pdl, st);
    }
}

}  // namespace

int kvq_wide_rows(int head_dim) { return head_dim == 256 ? 128 : 256; }
cudaError_t launch_kvq_wide(const AttnArgs &a, int64_t ctas, bool pdl, cudaStream_t st)
{
    return a.pool.format == LLMDOT_KVQ_I8 ? by_dim<LLMDOT_KVQ_I8>(a, ctas, pdl, st) : by_dim<LLMDOT_KVQ_E4M3>(a, ctas, pdl, st);
}

}  // namespace llmdot
