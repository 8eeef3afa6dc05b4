// kvq_attn_tc.cu -- shared-prefix attention for segments with many rows, on tcgen05.
//
// Same mathematics as kvq_attn.cu (codes exact in fp16, the key's scale on the score, the value's scale
// in the weight), for 16-bit queries; leaves partials (m, l, O) that the joining kernel adds.
//
// Bound: with hundreds of rows per kv head the products, the exponentials (16 per clock and SM) and
// the conversion of codes to fp16 take about the same time, and HBM little.  So one CTA takes two tiles of
// 128 rows (one for head_dim 256) over the same positions -- each code is converted once for 256 rows --
// and its roles overlap, 64 positions (a page) at a time:
//   warps of a tile (4 each)  S from TMEM 64 columns at a time in fragments of 4 rows by 2 columns a lane
//                             (a lane so needs a quarter of the columns' scales), weights as fp16 back
//                             into TMEM over S.  The weights are taken relative to a row's two references,
//                             one for the exponentials and one with the values' scales (raise_refs); only when a
//                             weight comes near fp16's limit are the maxima searched, the references of the
//                             rows that need it raised, and their sums and O rescaled, which after the first
//                             positions is rare
//   4 converting warps        codes from global memory (three K or V pages' loads in flight) to fp16 K
//                             and V operands in shared memory, scales beside them
//   1 warp per tile           one thread issues tcgen05.mma: S = Q K^T and O += P V with P and the
//                             accumulators in TMEM.  S has two places per tile, so that the scores of the next
//                             page are there when a page's weights are done.  (With one place of two pages the
//                             products with N = 128 need half the time -- N = 64 takes as long, measured 62
//                             clocks against 65 -- but a tile's products and its softmax then take turns, and
//                             the kernel took 1.5 times as long.)
// Operands in shared memory are rows of 64 values (128 bytes) of one position in 8-row groups, the
// 16-byte pieces swizzled by the row (piece ^ row % 8), which spreads the converting lanes' stores over all
// banks: K-major for Q and K, and the same layout read as N-major for V, which so needs no transposing.
// Shared memory and L1 are one data path that the tensor core's operands already fill by half, so a warp
// loads 512 consecutive bytes of codes at once (loads of 8 separate rows at a time held the whole kernel
// at a third of this speed).
// Every wait is bounded; one that gives up leaves NaN partials, so the output shows it.
//
// Measured on a B200, 1536 rows per kv head over 8192 positions of 8 kv heads of 128: 74 us, 690 TFLOP/s; a
// page takes 2500 clocks, of which the exponentials need 1024 and the products as issued 1500; the start
// (queries, tables, registers handed over) takes about 5 us, the end 2.  The steps: registers
// spilled by the issuing thread 128 us; split without spills and fragments in place of a row per thread
// 87; two places for S and a thread per tile 75.  (With a row's unit as a second product in the inner
// loop the whole call took 175.1 us, with it in the exponent's offset 173.7.)
#include <type_traits>

#include "kvq_attn.cuh"

namespace llmdot {
namespace {

constexpr long long WAIT_CLOCKS = 4000000000ll;  // about two seconds

template <int D> struct Wide {
    static constexpr int TILES = D == 256 ? 1 : 2;
    static constexpr int UN = KVQ_PAGE;               // positions of a unit
    static constexpr int STAGES = D == 256 ? 2 : 4;
    static constexpr int THREADS = TILES * 128 + 256;  // rows, converters, products (a warp per tile, of four)
    static constexpr uint32_t ROW = 128, GROUP = 8 * ROW;  // bytes of an operand's row, of eight
    static constexpr int KBLK = (D + 63) / 64;             // 64-wide blocks along the head dimension (Q, K)
    static constexpr uint32_t Q_BLK = 128 * ROW, K_BLK = UN * ROW;
    static constexpr uint32_t Q_BYTES = KBLK * Q_BLK, K_BYTES = KBLK * K_BLK;
    static constexpr uint32_t STAGE = 2 * K_BYTES;  // K, then V alike
    static constexpr uint32_t OFF_Q = STAGES * STAGE;
    static constexpr uint32_t OFF_SC = OFF_Q + TILES * Q_BYTES;  // per stage: K scales, V scales, 1 where there is no page
    static constexpr uint32_t SC_STAGE = 2 * UN * 4 + 16;
    static constexpr uint32_t OFF_BAR = OFF_SC + STAGES * SC_STAGE;
    // barriers: a stage is converted, read; S, P and P V of a tile's two places; the drain
    static constexpr int B_FULL = 0, B_EMPTY = STAGES, B_S = 2 * STAGES, B_P = B_S + 2 * TILES, B_O = B_P + 2 * TILES,
                         B_DRAIN = B_O + 2 * TILES, B_COUNT = B_DRAIN + TILES;
    static constexpr uint32_t SMEM = OFF_BAR + B_COUNT * 8 + 1024;  // and up to 1 KB to align the operands
    static constexpr int TILE_COLS = D + 2 * UN, C_O = 0, C_S = D;  // TMEM columns
    static_assert(TILES * TILE_COLS <= 512, "TMEM columns");
    static_assert(SMEM <= 227 * 1024, "shared memory");
};

__device__ __forceinline__ uint32_t su32(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }
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
// shared-memory matrix descriptor: rows of 128 bytes, 128-byte swizzle, 8-row groups of 1024 bytes.  lbo: bytes
// between blocks of 64 along N (N-major operands; K-major ones have a block per descriptor)
__device__ __forceinline__ uint64_t sdesc(uint32_t addr, uint32_t lbo = 16)
{
    return (uint64_t)((addr >> 4) & 0x3FFFu) | ((uint64_t)(lbo >> 4) << 16) | (64ull << 32) | (1ull << 46) | (2ull << 61);
}
// kind::f16, fp32 accumulator, fp16 A (TMEM) and N-major B (shared memory), M = 128
template <int N> __device__ __forceinline__ void umma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t acc)
{
    constexpr uint32_t idesc = (1u << 4) | (1u << 16) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
    asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
                 " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d),
                 "r"(a), "l"(b), "r"(idesc), "r"(acc)
                 : "memory");
}
// both operands in shared memory
template <int N> __device__ __forceinline__ void umma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t acc)
{
    constexpr uint32_t idesc = (1u << 4) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
    asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
                 " tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
                 "l"(a), "l"(b), "r"(idesc), "r"(acc)
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
// 16 lanes x 64 columns: register 4 i + 2 h + e of a lane is row lane / 4 + 8 h, column 8 i + 2 (lane % 4) + e
__device__ __forceinline__ void tmem_ld_frag(uint32_t ta, uint32_t *v)
{
    asm volatile("tcgen05.ld.sync.aligned.16x256b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
                 "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
                   "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]),
                   "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]),
                   "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
                 : "r"(ta));
}
// 16 lanes x 32 columns: register 2 i + h is row lane / 4 + 8 h, column 4 i + lane % 4
__device__ __forceinline__ void tmem_st_frag(uint32_t ta, const uint32_t *v)
{
    asm volatile("tcgen05.st.sync.aligned.16x128b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(ta),
                 "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
                 "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
                 : "memory");
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
// Loads that stay where they are written, ahead of the waits: the next page's codes.
__device__ __forceinline__ uint4 ldg128(const void *p)
{
    uint4 v;
    asm volatile("ld.global.nc.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}
__device__ __forceinline__ uint4 lds128(uint32_t a)
{
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ void sts128(uint32_t a, uint32_t x, uint32_t y, uint32_t z, uint32_t w)
{
    asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(a), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}

// Two fp32 values at once (one instruction each).
struct F2 {
    unsigned long long v;
};
__device__ __forceinline__ F2 f2(float x, float y)
{
    F2 r;
    asm("mov.b64 %0, {%1,%2};" : "=l"(r.v) : "f"(x), "f"(y));
    return r;
}
__device__ __forceinline__ void un2(F2 a, float &x, float &y) { asm("mov.b64 {%0,%1}, %2;" : "=f"(x), "=f"(y) : "l"(a.v)); }
__device__ __forceinline__ F2 mul2(F2 a, F2 b)
{
    F2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}
__device__ __forceinline__ F2 add2(F2 a, F2 b)
{
    F2 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c)
{
    F2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
    return r;
}
// TWO: the weights as hi + lo (fp16 queries, whose outputs have 11 bits); one fp16 else.
template <int D, int FMT, bool TWO>
__global__ void __launch_bounds__(Wide<D>::THREADS, 1) kvq_wide_kernel(const __grid_constant__ AttnArgs a, const int qwide)
{
    using W = Wide<D>;
    constexpr int STAGES = W::STAGES, UN = W::UN;
    extern __shared__ __align__(16) uint8_t smem_raw[];
    uint8_t *smem = smem_raw + (1024 - (su32(smem_raw) & 1023)) % 1024;
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
        const long long t0 = clock64();  // a few clocks; %globaltimer takes hundreds
        while (!bar_try(b, parity)) {
            if (*(volatile int *)&s_abort || clock64() - t0 > WAIT_CLOCKS) {
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
            bar_init(bars + 8 * i, i < STAGES || (i >= W::B_P && i < W::B_O) ? 128u : i < 2 * STAGES ? (uint32_t)nact : 1u);
        s_abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == SOFT / 32 + 4) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(su32(&s_tmem)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    // The queries of this warp's 32 rows go into their operand as they are, 16 bytes at a time, while the
    // rest is set up; rows that do not exist are zeros.
    if (tid < SOFT) {
        const uint32_t rho = row_first + tid;
        const int i = rho / (uint32_t)G;
        const int64_t mine = i < sg.nrows ? (sg.r0 + i) * a.ldq + (int64_t)(sg.kvh * G + (rho - i * G)) * D : -1;
        const uint32_t dst = base + W::OFF_Q + (warp >> 2) * W::Q_BYTES + (warp & 3) * 32 * W::ROW;
#pragma unroll 2
        for (int x = lane; x < 4 * D; x += 32) {  // 32 rows of D / 8 pieces
            const int r = x / (D / 8), c = x % (D / 8);
            const int64_t from = __shfl_sync(0xffffffffu, mine, r);
            const uint32_t to = dst + (c >> 3) * W::Q_BLK + r * W::ROW + ((c & 7) ^ (r & 7)) * 16;
            const uint16_t *src = (const uint16_t *)a.q + (from < 0 ? 0 : from + c * 8);
            if (qwide) {
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(src), "r"(from < 0 ? 0 : 16) : "memory");
            } else {
                uint32_t w[4] = {};
                if (from >= 0)
#pragma unroll
                    for (int k = 0; k < 4; k++) w[k] = src[2 * k] | (uint32_t)src[2 * k + 1] << 16;
                sts128(to, w[0], w[1], w[2], w[3]);
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    }
    // (the operands' memory holds the sequences' tables meanwhile)
    const SeqTable seqs = load_seqs(a, sg, (int32_t *)smem, W::THREADS);
    int row = -1, lo = 0, hi = 0x7fffffff;
    if (tid < SOFT) {
        row_range(a, sg, seqs, row_first + tid, row, lo, hi);
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
    // pages [u0, u1)
    const int u0 = max(sg.chunk * sg.ch, lo_min / KVQ_PAGE);
    const int u1 = min((sg.chunk + 1) * sg.ch, hi_max < 0 ? 0 : hi_max / KVQ_PAGE + 1), n = max(u1 - u0, 0);

    // Registers: 16 warps start with 128 each (2048 warp-registers in all); the row warps hold two pieces of
    // scores and need more: 8 * 152 + 4 * 128 + 4 * 80 = 2048.
    if (warp < SOFT / 32) {
        // ------------------------------------------------------------ a row per thread
        if (W::TILES == 2) asm volatile("setmaxnreg.inc.sync.aligned.u32 152;");
        const int tile = warp >> 2, head = sg.kvh * G + (row_first + tid) % G;
        const uint32_t tm = tmem + tile * W::TILE_COLS + ((uint32_t)(32 * (warp & 3)) << 16);
        // bf16 queries become fp16 ones, scaled by a power of two per row; a negative scale's sign goes into the query
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        __syncwarp();
        int e = 0;
        if (a.at.type != T_F16 || a.at.scale < 0.0f) {
            const uint32_t mine = base + W::OFF_Q + tile * W::Q_BYTES + (tid & 127) * W::ROW;
            const uint32_t flip = a.at.scale < 0.0f ? 0x80008000u : 0u;
            auto piece = [&](int c) { return mine + (c >> 3) * W::Q_BLK + ((c & 7) ^ (lane & 7)) * 16; };
            if (a.at.type == T_F16) {
#pragma unroll 4
                for (int c = 0; c < D / 8; c++) {
                    const uint4 v = lds128(piece(c));
                    sts128(piece(c), v.x ^ flip, v.y ^ flip, v.z ^ flip, v.w ^ flip);
                }
            } else {
                __nv_bfloat162 top2 = __float2bfloat162_rn(0.0f);  // a NaN survives the maxima
#pragma unroll 8
                for (int c = 0; c < D / 8; c++) {
                    const uint4 v = lds128(piece(c));
                    const __nv_bfloat162 *h = reinterpret_cast<const __nv_bfloat162 *>(&v);
                    top2 = __hmax2_nan(top2, __hmax2_nan(__hmax2_nan(__habs2(h[0]), __habs2(h[1])), __hmax2_nan(__habs2(h[2]), __habs2(h[3]))));
                }
                const float top = __bfloat162float(__hmax_nan(__low2bfloat16(top2), __high2bfloat16(top2)));
                e = row_exponent(top);
                const float up = pow2(e);
#pragma unroll 8
                for (int c = 0; c < D / 8; c++) {
                    const uint4 v = lds128(piece(c));
                    const uint32_t w[4] = {v.x ^ flip, v.y ^ flip, v.z ^ flip, v.w ^ flip};
                    uint32_t h[4];
#pragma unroll
                    for (int k = 0; k < 4; k++) h[k] = pack(__uint_as_float(w[k] << 16) * up, __uint_as_float(w[k] & 0xFFFF0000u) * up);
                    sts128(piece(c), h[0], h[1], h[2], h[3]);
                }
            }
        }
        const float qf = fabsf(a.at.scale) * code_unit<FMT>() * (a.at.softcap > 0.0f ? 1.0f : 1.4426950408889634f) * pow2(-e);
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncthreads();
        // this warp's rows: positions that all of them see, and that any does
        const int lo_max = __reduce_max_sync(0xffffffffu, row >= 0 ? lo : 0), hi_end = s_hi[warp];
        lo_min = s_lo[warp];
        const int hi_min = __reduce_min_sync(0xffffffffu, row >= 0 ? hi : 0x7fffffff);
        const bool cap = a.at.softcap > 0.0f;
        const float inv_cap2 = cap ? 2.0f * 1.4426950408889634f / a.at.softcap : 0.0f;
        // ---- fragments: this lane's four rows (of the warp's 32) are g + 8 k, its columns 8 i + 2 t and the next
        const int g = lane >> 2, t = lane & 3;
        int flo[4], fhi[4];
        float fq[4], ref[4], unit[4];  // ref: base 2; -infinity until the row has seen a position
        F2 l[4];
#pragma unroll
        for (int k = 0; k < 4; k++) {
            flo[k] = __shfl_sync(0xffffffffu, lo, g + 8 * k);
            fhi[k] = __shfl_sync(0xffffffffu, hi, g + 8 * k);
            fq[k] = __shfl_sync(0xffffffffu, qf, g + 8 * k);
            ref[k] = -INFINITY;
            unit[k] = 1.0f;
            l[k] = f2(0.0f, 0.0f);
        }
        bool ok = tile < nact, wild = false;  // wild: some row's unit is too large or small to go through an exponential
        // O times f (lane = row), once the products that add to it (through unit i) are complete.
        auto rescale_o = [&](int i, float f) {
            ok = wait(W::B_O + tile * 2 + (i & 1), (i >> 1) & 1);
            if (!(ok = __all_sync(0xffffffffu, ok))) return;
            fence_after();
            const F2 ff = f2(f, f);
#pragma unroll 1
            for (int c = 0; c < D / 32; c++) {
                uint32_t v[32];
                tmem_ld32(tm + W::C_O + 32 * c, v);
                tmem_ld_wait();
#pragma unroll
                for (int j = 0; j < 32; j += 2) {
                    float p, q;
                    un2(mul2(f2(__uint_as_float(v[j]), __uint_as_float(v[j + 1])), ff), p, q);
                    v[j] = __float_as_uint(p);
                    v[j + 1] = __float_as_uint(q);
                }
                tmem_st16(tm + W::C_O + 32 * c, v);
                tmem_st16(tm + W::C_O + 32 * c + 16, v + 16);
            }
            tmem_st_wait();
        };
        // A page's weights, hi and lo in 32 columns each, over scores that were read.
        constexpr int NP = TWO ? 2 : 1;
        auto hand_over = [&](int buf, const uint32_t (&p)[NP][2][16]) {
#pragma unroll
            for (int x = 0; x < NP; x++)
#pragma unroll
                for (int h = 0; h < 2; h++) tmem_st_frag(tm + ((uint32_t)(16 * h) << 16) + W::C_S + 64 * buf + 32 * x, p[x][h]);
            tmem_st_wait();
            fence_before();
            bar_arrive(bars + 8 * (W::B_P + tile * 2 + buf));
        };
        auto split = [&](float y, float z, uint32_t (&p)[NP][2][16], int h, int at) {
            const uint32_t hi = pack(y, z);
            p[0][h][at] = hi;
            if (TWO) {
                const float2 b = __half22float2(*reinterpret_cast<const __half2 *>(&hi));
                p[NP - 1][h][at] = pack(y - b.x, z - b.y);
            }
            return hi;
        };
        // Whether a page's sums or weights have passed the limits for a row of the warp (or are NaN).
        auto passed = [&](const F2 (&sum)[4], uint32_t any) {
            bool over = too_large(any);
#pragma unroll
            for (int k = 0; k < 4; k++) {
                float x, y;
                un2(sum[k], x, y);
                over |= !(x + y < SUM_LIMIT);
            }
            return __any_sync(0xffffffffu, over) != 0;
        };
        // A page that the rows see whole, without a cap: false (and nothing done) when a weight comes too near
        // the limit and the references have to rise.  `unit` goes into the exponent (so not where a row is `wild`), and
        // comes out of the page's sums.
        auto plain_page = [&](const float *ks, const float *vs, int buf) -> bool {
            uint32_t s[2][32], p[NP][2][16], any = 0;
            tmem_ld_frag(tm + W::C_S + 64 * buf, s[0]);
            tmem_ld_frag(tm + (16u << 16) + W::C_S + 64 * buf, s[1]);
            F2 q2[4], off[4], sum[4];
#pragma unroll
            for (int k = 0; k < 4; k++) {
                q2[k] = f2(fq[k], fq[k]);
                const float at = pow_exponent(unit[k]) - ref[k];
                off[k] = f2(at, at);
                sum[k] = f2(0.0f, 0.0f);
            }
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const float2 kf = *(const float2 *)(ks + 8 * i + 2 * t), vf = *(const float2 *)(vs + 8 * i + 2 * t);
                const F2 k2 = f2(kf.x, kf.y), v2 = f2(vf.x, vf.y);
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const uint32_t *x = s[k >> 1] + 4 * i + 2 * (k & 1);
                    float y, z;
                    un2(fma2(f2(__uint_as_float(x[0]), __uint_as_float(x[1])), mul2(k2, q2[k]), off[k]), y, z);
                    const F2 e = f2(ex2(y), ex2(z));
                    sum[k] = add2(sum[k], e);
                    un2(mul2(e, v2), y, z);
                    const uint32_t hi = split(y, z, p, k >> 1, 2 * i + (k & 1));
                    any = hadd2(any, hi);
                }
            }
#pragma unroll
            for (int k = 0; k < 4; k++) sum[k] = mul2(sum[k], f2(pow_inverse(unit[k]), pow_inverse(unit[k])));
            if (passed(sum, any)) return false;
#pragma unroll
            for (int k = 0; k < 4; k++) l[k] = add2(l[k], sum[k]);
            hand_over(buf, p);
            return true;
        };
        // The search for the rows' maxima over a page, of the scores and with the values' scales, and the references raised
        // where they stand too low.  MASKED: scores of positions that a row does not see do not count.
        auto search = [&](int i, const float *ks, const float *vs, int buf, auto masked) {
            constexpr bool MASKED = decltype(masked)::value;
            const int j0 = u0 * KVQ_PAGE + i * UN + 2 * t;
            float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY}, topv[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int h = 0; h < 2; h++) {
                uint32_t s[32];
                tmem_ld_frag(tm + ((uint32_t)(16 * h) << 16) + W::C_S + 64 * buf, s);
                tmem_ld_wait();
#pragma unroll
                for (int c = 0; c < 8; c++) {
                    const float2 kf = *(const float2 *)(ks + 8 * c + 2 * t), vf = *(const float2 *)(vs + 8 * c + 2 * t);
                    const float lx = log2_abs(vf.x), ly = log2_abs(vf.y);
                    const int j = j0 + 8 * c;
#pragma unroll
                    for (int r = 0; r < 2; r++) {
                        const int k = 2 * h + r;
                        float x = __uint_as_float(s[4 * c + 2 * r]) * (kf.x * fq[k]), y = __uint_as_float(s[4 * c + 2 * r + 1]) * (kf.y * fq[k]);
                        if (cap) {
                            x = capped<false>(x, a.at.softcap, inv_cap2) * 1.4426950408889634f;
                            y = capped<false>(y, a.at.softcap, inv_cap2) * 1.4426950408889634f;
                        }
                        if (MASKED && (j < flo[k] || j > fhi[k])) x = -INFINITY;
                        if (MASKED && (j + 1 < flo[k] || j + 1 > fhi[k])) y = -INFINITY;
                        top[k] = fmaxf(top[k], fmaxf(x, y));  // (a NaN does not count)
                        topv[k] = fmaxf(topv[k], fmaxf(x + lx, y + ly));
                    }
                }
            }
            float f[4];
            bool moved = false;
#pragma unroll
            for (int k = 0; k < 4; k++) {
#pragma unroll
                for (int d = 1; d < 4; d <<= 1) {
                    top[k] = fmaxf(top[k], __shfl_xor_sync(0xffffffffu, top[k], d));
                    topv[k] = fmaxf(topv[k], __shfl_xor_sync(0xffffffffu, topv[k], d));
                }
                float fl = 1.0f;
                f[k] = 1.0f;
                if (raise_refs(top[k], topv[k], ref[k], unit[k], fl, f[k])) moved = true;
                l[k] = mul2(l[k], f2(fl, fl));
            }
            wild = __any_sync(0xffffffffu, max(max(abs(pow_exponent(unit[0])), abs(pow_exponent(unit[1]))),
                                               max(abs(pow_exponent(unit[2])), abs(pow_exponent(unit[3])))) > 60);
            if (i > 0 && __any_sync(0xffffffffu, moved)) {
                float mine = 1.0f;  // of the row that is this lane
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const float x = __shfl_sync(0xffffffffu, f[k], (lane & 7) * 4);
                    if (lane >> 3 == k) mine = x;
                }
                rescale_o(i - 1, mine);
            }
        };
        // The weights of a page, with masks and cap: false (and nothing done) as above, unless `last`.
        auto masked_page = [&](int i, const float *ks, const float *vs, int buf, bool last) -> bool {
            const int j0 = u0 * KVQ_PAGE + i * UN + 2 * t;
            uint32_t p[NP][2][16], any = 0;
            F2 sum[4];
#pragma unroll
            for (int k = 0; k < 4; k++) sum[k] = f2(0.0f, 0.0f);
#pragma unroll
            for (int h = 0; h < 2; h++) {
                uint32_t s[32];
                tmem_ld_frag(tm + ((uint32_t)(16 * h) << 16) + W::C_S + 64 * buf, s);
                tmem_ld_wait();
#pragma unroll
                for (int c = 0; c < 8; c++) {
                    const float2 kf = *(const float2 *)(ks + 8 * c + 2 * t), vf = *(const float2 *)(vs + 8 * c + 2 * t);
#pragma unroll
                    for (int r = 0; r < 2; r++) {
                        const int k = 2 * h + r, j = j0 + 8 * c;
                        const float off = ref[k] == -INFINITY ? 0.0f : ref[k];
                        float x = __uint_as_float(s[4 * c + 2 * r]) * (kf.x * fq[k]), y = __uint_as_float(s[4 * c + 2 * r + 1]) * (kf.y * fq[k]);
                        if (cap) {
                            x = capped<false>(x, a.at.softcap, inv_cap2) * 1.4426950408889634f;
                            y = capped<false>(y, a.at.softcap, inv_cap2) * 1.4426950408889634f;
                        }
                        x = ex2(x - off);
                        y = ex2(y - off);
                        const bool gx = j < flo[k] || j > fhi[k], gy = j + 1 < flo[k] || j + 1 > fhi[k];
                        sum[k] = add2(sum[k], f2(gx ? 0.0f : x, gy ? 0.0f : y));
                        // whatever an unseen position holds
                        const uint32_t hi = split(gx ? 0.0f : x * vf.x * unit[k], gy ? 0.0f : y * vf.y * unit[k], p, h, 2 * c + r);
                        any = hadd2(any, hi);
                    }
                }
            }
            if (passed(sum, any) && !last) return false;
#pragma unroll
            for (int k = 0; k < 4; k++) l[k] = add2(l[k], sum[k]);
            hand_over(buf, p);
            return true;
        };
        bool known = false;  // every row of the warp has seen a position
        for (int i = 0; i < n && ok; i++) {
            const int st = i % STAGES, buf = i & 1, p0 = u0 * KVQ_PAGE + i * UN;
            ok = wait(W::B_S + tile * 2 + buf, (i >> 1) & 1) && wait(W::B_FULL + st, (i / STAGES) & 1);
            if (!(ok = __all_sync(0xffffffffu, ok))) break;
            fence_after();
            const float *ks = (const float *)(smem + W::OFF_SC + st * W::SC_STAGE), *vs = ks + UN;
            if (vs[UN] != 0.0f || p0 > hi_end || p0 + KVQ_PAGE <= lo_min) {  // nothing for this warp's rows
                const uint32_t zero[NP][2][16] = {};
                hand_over(buf, zero);
            } else if (!cap && !wild && p0 >= lo_max && p0 + KVQ_PAGE - 1 <= hi_min) {  // everything
                if (known && plain_page(ks, vs, buf)) continue;
                search(i, ks, vs, buf, std::false_type{});
                known = true;
                if (ok && (wild || !plain_page(ks, vs, buf))) masked_page(i, ks, vs, buf, true);  // (a NaN stays one)
            } else {
                if (known && masked_page(i, ks, vs, buf, false)) continue;
                search(i, ks, vs, buf, std::true_type{});
                if (ok) masked_page(i, ks, vs, buf, true);
                known = __all_sync(0xffffffffu, fminf(fminf(ref[0], ref[1]), fminf(ref[2], ref[3])) > -INFINITY);
            }
        }
        if (ok && n > 0) {
            ok = wait(W::B_O + tile * 2 + ((n - 1) & 1), ((n - 1) >> 1) & 1);
            ok = __all_sync(0xffffffffu, ok);
        }
        const int64_t RH = (int64_t)a.bt.rows * a.at.heads, slot = sg.pre ? sg.chunk : a.nsp + sg.chunk;
        const int at = row < 0 ? -1 : row * a.at.heads + head;  // rows * heads fits 2^30
        int to[4];
        __syncwarp();
#pragma unroll
        for (int k = 0; k < 4; k++) {
            to[k] = __shfl_sync(0xffffffffu, at, g + 8 * k);
            // a row's sum lies in four lanes, its reference in each of them
            float x, y;
            un2(l[k], x, y);
            x += y;
            x += __shfl_xor_sync(0xffffffffu, x, 1);
            x += __shfl_xor_sync(0xffffffffu, x, 2);
            if (t == 0 && to[k] >= 0) a.part_ml[slot * RH + to[k]] = ok ? make_float2(ref[k], x) : make_float2(0.0f, NAN);
        }
        if (ok && n > 0) {  // O: four lanes write 32 consecutive bytes of a row
            fence_after();
            F2 u2[4];
#pragma unroll
            for (int k = 0; k < 4; k++) u2[k] = f2(pow_inverse(unit[k]), pow_inverse(unit[k]));
#pragma unroll 1
            for (int c = 0; c < (D + 63) / 64; c++) {
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    uint32_t v[32];
                    tmem_ld_frag(tm + ((uint32_t)(16 * h) << 16) + W::C_O + 64 * c, v);
                    tmem_ld_wait();
#pragma unroll
                    for (int r = 0; r < 2; r++) {
                        const int k = 2 * h + r;
                        float2 *o = (float2 *)(a.part_o + (slot * RH + to[k]) * D + 64 * c + 2 * t);
#pragma unroll
                        for (int i = 0; i < 8; i++) {
                            float x, y;
                            un2(mul2(f2(__uint_as_float(v[4 * i + 2 * r]), __uint_as_float(v[4 * i + 2 * r + 1])), u2[k]), x, y);
                            if (to[k] >= 0 && 64 * c + 8 * i < D) o[4 * i] = make_float2(x, y);
                        }
                    }
                }
            }
        }
    } else if (warp < SOFT / 32 + 4) {
        // ------------------------------------------------------------ codes to operands
        const int dt = tid - SOFT, dw = dt >> 5;
        // a page's K or V: 4 D pieces of 16 codes, T per thread, a warp's at consecutive addresses
        constexpr int T = D / 32;
        struct Codes {
            uint4 c[T];
        };
        auto page_of = [&](int u) { return u < u1 ? __ldg(sg.pages + u) : -1; };
        auto none = [&](int page) { return (unsigned)page >= (unsigned)a.pool.n_pages; };
        auto load = [&](int page, bool v, Codes &x) {
            if (none(page)) {
#pragma unroll
                for (int i = 0; i < T; i++) x.c[i] = make_uint4(0, 0, 0, 0);
                return;
            }
            const uint8_t *p = (const uint8_t *)(v ? a.pool.v : a.pool.k) + (((int64_t)page * Hk + sg.kvh) * KVQ_PAGE) * D + dt * 16;
#pragma unroll
            for (int i = 0; i < T; i++) x.c[i] = ldg128(p + 2048 * i);
        };
        // a page's scales: warp 0 V's, warp 1 K's; lane: positions lane and lane + 32
        auto load_scales = [&](int page, float (&c)[2]) {
            if (dw >= 2) return;
            const float *s = (dw == 0 ? a.pool.v_scale : a.pool.k_scale) + ((int64_t)page * Hk + sg.kvh) * KVQ_PAGE + lane;
            c[0] = none(page) ? 0.0f : __ldg(s);
            c[1] = none(page) ? 0.0f : __ldg(s + 32);
        };
        bool ok = true;
        auto put_scales = [&](int i, int page, const float (&c)[2]) {
            float *ks = (float *)(smem + W::OFF_SC + i % STAGES * W::SC_STAGE), *vs = ks + UN;
            if (dw == 0) {
                vs[lane] = c[0] * code_unit<FMT>();
                vs[lane + 32] = c[1] * code_unit<FMT>();
                if (lane == 0) vs[UN] = none(page) ? 1.0f : 0.0f;
            } else if (dw == 1) {
                ks[lane] = c[0];
                ks[lane + 32] = c[1];
            }
        };
        // K or V of unit i
        auto convert = [&](int i, bool v, const Codes &x) {
            const uint32_t d = base + i % STAGES * W::STAGE + (v ? W::K_BYTES : 0u);
#pragma unroll
            for (int k = 0; k < T; k++) {
                // piece t: position r, codes 16 ch ..: two operand pieces of 8.  Lanes of the upper half of a
                // 128-code row write them in the other order, so that eight lanes meet eight banks.
                const int t = dt + 128 * k, ch = t % (D / 16), r = t / (D / 16), pc = (ch & 3) * 2, swap = (ch >> 2) & 1;
                const uint32_t to = d + (ch >> 2) * W::K_BLK + r * W::ROW;
                const uint4 c = x.c[k];
                const uint32_t w[4] = {(swap ? c.z : c.x) ^ code_flip<FMT>(), (swap ? c.w : c.y) ^ code_flip<FMT>(),
                                       (swap ? c.x : c.z) ^ code_flip<FMT>(), (swap ? c.y : c.w) ^ code_flip<FMT>()};
                sts128(to + ((pc + swap) ^ (r & 7)) * 16, codes2<FMT, 0, 1>(w[0]), codes2<FMT, 2, 3>(w[0]), codes2<FMT, 0, 1>(w[1]),
                       codes2<FMT, 2, 3>(w[1]));
                sts128(to + ((pc + 1 - swap) ^ (r & 7)) * 16, codes2<FMT, 0, 1>(w[2]), codes2<FMT, 2, 3>(w[2]),
                       codes2<FMT, 0, 1>(w[3]), codes2<FMT, 2, 3>(w[3]));
            }
        };
        // four sets of registers in turn, three loads ahead (a copy between sets would wait for them)
        Codes k0, v0, k1, v1;
        float sc[2];
        int p0 = page_of(u0), p1 = page_of(u0 + 1), p2 = page_of(u0 + 2), p3 = page_of(u0 + 3);
        load(p0, false, k0);
        load(p0, true, v0);
        load(p1, false, k1);
        load_scales(p0, sc);
        __syncthreads();
        auto slot = [&](int i) {
            if (i < STAGES) return true;
            ok = wait(W::B_EMPTY + i % STAGES, (i / STAGES - 1) & 1);
            return ok = __all_sync(0xffffffffu, ok);
        };
        auto done = [&](int i) {
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // operands: generic writes -> tensor core
            bar_arrive(bars + 8 * (W::B_FULL + i % STAGES));
        };
        for (int i = 0; i < n && ok; i += 2) {  // two pages a round
            const int p4 = page_of(u0 + i + 4), p5 = page_of(u0 + i + 5);
            load(p1, true, v1);
            if (!slot(i)) break;
            put_scales(i, p0, sc);
            load_scales(p1, sc);
            convert(i, false, k0);
            load(p2, false, k0);
            convert(i, true, v0);
            done(i);
            if (i + 1 >= n) break;
            load(p2, true, v0);
            if (!slot(i + 1)) break;
            put_scales(i + 1, p1, sc);
            load_scales(p2, sc);
            convert(i + 1, false, k1);
            load(p3, false, k1);
            convert(i + 1, true, v1);
            done(i + 1);
            p0 = p2;
            p1 = p3;
            p2 = p4;
            p3 = p5;
        }
    } else {
        // ------------------------------------------------------------ products
        if (W::TILES == 2) asm volatile("setmaxnreg.dec.sync.aligned.u32 80;");
        __syncthreads();
        const int t = warp - (SOFT / 32 + 4);  // each tile's products are issued by a thread of its own
        if (t < nact && lane == 0 && n > 0) {
            fence_after();
            // descriptors differ in their address field (units of 16 bytes): one addition each
            const uint64_t qd = sdesc(base + W::OFF_Q + t * W::Q_BYTES), kd = sdesc(base), vd = sdesc(base + W::K_BYTES, W::K_BLK);
            const uint32_t tm = tmem + t * W::TILE_COLS, bs = bars + 8 * (W::B_S + t * 2), bo = bars + 8 * (W::B_O + t * 2);
            bool ok = true;
            auto qk = [&](int i) {
                ok = wait(W::B_FULL + i % STAGES, (i / STAGES) & 1);
                if (!ok) return;
                fence_after();
                const uint64_t k = kd + i % STAGES * (W::STAGE / 16);
#pragma unroll
                for (int kk = 0; kk < D / 16; kk++)
                    umma_ss<UN>(tm + W::C_S + 64 * (i & 1), qd + (kk / 4 * W::Q_BLK + kk % 4 * 32) / 16,
                                k + (kk / 4 * W::K_BLK + kk % 4 * 32) / 16, kk != 0);
                umma_commit(bs + 8 * (i & 1));
            };
            qk(0);
            if (n > 1 && ok) qk(1);
            for (int i = 0; i < n && ok; i++) {
                if (!(ok = wait(W::B_P + t * 2 + (i & 1), (i >> 1) & 1))) break;
                fence_after();
                const uint64_t v = vd + i % STAGES * (W::STAGE / 16);
#pragma unroll
                for (int kk = 0; kk < (TWO ? 2 : 1) * UN / 16; kk++)  // hi, then lo, on the same values
                    umma_ts<D>(tm + W::C_O, tm + W::C_S + 64 * (i & 1) + 8 * kk, v + kk % (UN / 16) * 2 * W::GROUP / 16, i != 0 || kk != 0);
                umma_commit(bo + 8 * (i & 1));
                umma_commit(bars + 8 * (W::B_EMPTY + i % STAGES));
                if (i + 2 < n) qk(i + 2);  // the scores that this page's weights leave room for
            }
            // every product issued completes before the TMEM is released
            umma_commit(bars + 8 * (W::B_DRAIN + t));
            const long long t0 = clock64();
            while (!bar_try(bars + 8 * (W::B_DRAIN + t), 0) && clock64() - t0 < WAIT_CLOCKS) {}
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

template <int D, int FMT, bool TWO> cudaError_t launch_one(const AttnArgs &a, int64_t ctas, bool pdl, cudaStream_t st)
{
    using W = Wide<D>;
    static std::atomic<unsigned long long> done{0};
    cudaError_t e = smem_attr_once(done, kvq_wide_kernel<D, FMT, TWO>, W::SMEM);
    if (e != cudaSuccess) return e;
    const int qwide = ((uintptr_t)a.q & 15) == 0 && (a.bt.rows <= 1 || a.ldq * 2 % 16 == 0);
    return launch_kernel(pdl, kvq_wide_kernel<D, FMT, TWO>, dim3((unsigned)ctas), dim3(W::THREADS), W::SMEM, st, a, qwide);
}
template <int D, int FMT> cudaError_t launch(const AttnArgs &a, int64_t ctas, bool pdl, cudaStream_t st)
{
    return a.at.type == T_F16 ? launch_one<D, FMT, true>(a, ctas, pdl, st) : launch_one<D, FMT, false>(a, ctas, pdl, st);
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
