// kvq_attn.cu -- attention of a batch over a shared prefix and its own pages, K and V in 8 bits.
//
// s_j = scale * (q . k_j), optionally capped; out = sum_j softmax(s)_j v_j, with k_j = code * scale_j
// (one fp32 scale per position and head).
//
// Mathematics.  A code is an integer of at most 7 bits and sign, or an e4m3 value: exact in fp16.  The
// query row is scaled by a power of two into fp16 (fp32 queries: as hi + lo, two products), so q . code
// is a sum of exact products in fp32, and the key's scale multiplies the score.  The value's scale goes
// into the weight: P_j = exp2(s_j - ref) * v_scale_j / 2^E.  ref and E are a row's own, from the positions that it
// sees: ref was its maximum when it was set, E brought its largest exp2(s_j - ref) * v_scale_j into fp16's upper
// range, and both rise (the sums rescaled by powers of two) when a later product of the row nears fp16's limit.
// So neither a value that a row does not see nor one that it gives no weight costs it bits, whatever
// the scales' size.  P is hi + lo, or with bf16 queries, whose output has 8 bits, one fp16 (with fp16 outputs its
// rounding would add as much error again as the output's own).
// The sum of exponentials, the maxima, both products' sums and the outputs are fp32.  The tensor core truncates what it
// adds into its accumulators, half a unit of the sum lost per addition, so with fp32 queries a chain of such additions
// ends after a K piece (64 dimensions or fewer) and after a page, and its sum is added with rounding: 60 drawn
// cases against 64 bits, 0.73 of the error of 32-bit torch operations in the geometric mean, 4.5e-7 at most (1.23 and 2.9e-6
// with one chain).
//
// Work is cut into segments -- the prefix with every row of the batch, each sequence's own pages with
// its rows -- times kv heads, row tiles and chunks of pages.  The prefix is read once per row tile of
// the whole batch, not once per sequence.  Each CTA leaves a partial (m, l, O) of its chunk; a second kernel
// (programmatic dependent launch) joins a row's partials in chunk order.  A call with one chunk in
// all writes its output directly.  Segments with many rows go to kvq_attn_tc.cu.
//
// This kernel, for few rows per kv head, is bound by HBM (the codes), and below that by instructions: the
// codes of a page become fp16 fragments with about 1.3 instructions a code.  Four warps share a page of 64
// positions.  For S^T = K Q^T (mma.m16n8k16; positions and head dimensions take the 16-wide side, rows
// the 8-wide side, so one token of a group of 4 heads wastes half a tile, not three quarters) each
// warp has 16 positions; the weights pass through shared memory, one barrier per page; and for O^T = V^T P^T
// each warp has 32 head dimensions and all positions, so that O needs a quarter of the registers (many
// CTAs per SM hide the latencies) and no joining of warps at the end.  The order of k inside a tile is free
// as long as both operands agree; it is chosen so that a lane's K bytes are 16 consecutive ones, and its V
// bytes four positions of four consecutive dimensions, which byte permutes turn into fragments.
// While no weight comes near fp16's limit no maximum is searched, and the barrier's vote tells all warps when one
// does; then only the rows that need it take new references, so that a row's result does not depend on its neighbours.
//
// Measured on a B200, the own pages of 96 sequences with 3 to 5 drafted rows of 4 heads each, 64 to 2048
// positions of 8 kv heads of 128: 94 us for 224 MB (2.4 TB/s; 0.58 instructions per clock and scheduler).
// With a page per warp, maxima and O of all dimensions in each warp: 124 us.  Left out in turn (same sizes),
// the scores' product saved 15 us, the output's 15, the loads 14, all of these 63.
#include <algorithm>

#include "kvq_attn.cuh"

namespace llmdot {
namespace {

constexpr int NW = 4;  // warps per CTA

__device__ __forceinline__ uint32_t su32(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void cp16(uint32_t dst, const void *src)
{
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp4(uint32_t dst, const void *src)
{
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
{
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8(uint32_t a)
{
    uint32_t d;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
    return d;
}
// Shapes of the kernel for a head dimension D.
template <int D> struct Shape {
    static constexpr int CPR = D / 16;                         // 16-byte pieces of a position's codes
    static constexpr int SLOT = KVQ_PAGE * D;                  // bytes of a page's K or V
    static constexpr int KB = D == 96 ? 8 : 16, KC = D / (4 * KB);  // K bytes a lane takes at once; such pieces
    static constexpr int GPW = D == 256 ? 2 : 1;               // 32-dimension groups of O per warp (64: two warps share one, 96: three have one)
    static constexpr int QPAD = D == 96 ? 0 : 8;               // halves between query rows against bank conflicts
    static constexpr int OFF_SC = 4 * SLOT, OFF_Q = OFF_SC + 4 * KVQ_PAGE * 4;  // K 0, K 1, V 0, V 1, scales, queries, weights
};
constexpr int PS = 80;  // halves from one row's weights to the next (64 and 16 against bank conflicts)
// An instance's resources, for its launch, its compilation and the plan alike.  CTAs per SM that its registers are
// limited to leave room for: what its accumulators and query fragments take with few spills.
constexpr int narrow_regs_ctas(int d, int nt) { return d == 256 ? (nt <= 2 ? 3 : 2) : nt == 1 ? 5 : nt <= 3 ? 4 : 2; }
// Bytes of dynamic shared memory with nq terms per query and np per weight; 48 bytes per row and 1 KB of the system's beside it.
constexpr int narrow_smem(int d, int nt, int nq, int np) { return 4 * KVQ_PAGE * d + 1024 + nt * 8 * (nq * (d + (d == 96 ? 0 : 8)) + np * 2 * PS) * 2; }
constexpr int narrow_ctas(int d, int nt, int nq, int np)
{
    const int room = 228 * 1024 / (narrow_smem(d, nt, nq, np) + nt * 8 * 48 + 1024), regs = narrow_regs_ctas(d, nt);
    return room < 1 ? 1 : room < regs ? room : regs;
}
// Where 16-byte piece c of position r lies in its slot: chosen so that the lanes of one shared-memory
// access (K: 8 or 16 lanes on positions a, a + 4, ...; V: on positions 4 i .. 4 i + 3) meet distinct banks.
template <int D> __device__ __forceinline__ int k_piece(int r, int c)
{
    if (D == 64) return (r ^ ((r >> 2) & 1)) * 4 + c;
    if (D == 96) return (r ^ ((r >> 1) & 2)) * 6 + c;
    return r * (D / 16) + (c ^ (r & 4));
}
template <int D> __device__ __forceinline__ int v_piece(int r, int c)
{
    if (D == 64) return r * 4 + (c ^ (r & 2));
    if (D == 96) return (r ^ ((r >> 1) & 2)) * 6 + c;
    return r * (D / 16) + (c ^ ((r & 3) << 1));
}
// The position (of 16) that row r of an S^T tile stands for: row 2 t' -> t', 2 t' + 1 -> 4 + t', + 8 alike.
__device__ __forceinline__ int row_position(int r) { return ((r & 7) >> 1) + 4 * (r & 1) + (r & 8); }

template <int N> struct Bytes;
template <> struct Bytes<8> { using T = uint2; };
template <> struct Bytes<16> { using T = uint4; };
template <int N> __device__ __forceinline__ void lds(const uint8_t *p, uint32_t (&w)[N / 4])
{
    const typename Bytes<N>::T v = *(const typename Bytes<N>::T *)p;
    const uint32_t *x = reinterpret_cast<const uint32_t *>(&v);
#pragma unroll
    for (int i = 0; i < N / 4; i++) w[i] = x[i];
}

__device__ __forceinline__ void store4(void *p, int64_t i, uint32_t type, bool wide, const float (&x)[4])
{
    if (type == T_F32) {
        float *o = (float *)p + i;
        if (wide) *(float4 *)o = make_float4(x[0], x[1], x[2], x[3]);
        else
#pragma unroll
            for (int e = 0; e < 4; e++) o[e] = x[e];
    } else {
        __align__(8) uint16_t h[4];
#pragma unroll
        for (int e = 0; e < 4; e++)
            h[e] = type == T_F16 ? __half_as_ushort(__float2half_rn(x[e])) : __bfloat16_as_ushort(__float2bfloat16_rn(x[e]));
        uint16_t *o = (uint16_t *)p + i;
        if (wide) *(uint2 *)o = *(const uint2 *)h;
        else
#pragma unroll
            for (int e = 0; e < 4; e++) o[e] = h[e];
    }
}

// PREC 0 (bf16): one fp16 for query and weight; 1 (fp16): hi + lo weights; 2 (fp32): hi + lo queries too.
template <int D, int FMT, int NT, int PREC>
__global__ void __launch_bounds__(NW * 32, narrow_regs_ctas(D, NT)) kvq_attn_kernel(const __grid_constant__ AttnArgs a)
{
    using Sh = Shape<D>;
    constexpr int RT = 8 * NT, QS = D + Sh::QPAD, NQ = PREC == 2 ? 2 : 1, NP = PREC > 0 ? 2 : 1;
    constexpr bool QREG = NT * NQ * D / 8 <= 32;  // the query's fragments stay in registers
    constexpr bool ROUNDED = PREC == 2;           // short chains of tensor-core additions
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ float s_qf[RT], s_max[NW][RT], s_l[NW][RT];  // s_l: at the end; before, maxima with the values' scales
    __shared__ int s_lo[RT], s_hi[RT], s_row[RT];
    __half *sq = (__half *)(smem + Sh::OFF_Q);  // [NQ][RT][QS]
    __half *sp = sq + NQ * RT * QS;             // [2][NP][RT][PS]
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int G = a.group, Hk = a.pool.heads_kv;

    pdl_launch();  // the joining kernel may be set up while this one runs
    Segment sg;
    if (!segment_of(a, RT, sg)) {
        if (a.chained) pdl_wait();
        return;
    }
    const int kvh = sg.kvh, chunk = sg.chunk, ch = sg.ch, len = sg.len, row_first = sg.tile * RT;
    const int32_t *pages = sg.pages;
    const uint32_t smem_s = su32(smem);
    // ---- pages [u0, u1) of the segment's list; those outside a window are left out once the rows' ranges are
    // known, without one the first pages are on their way before that
    int u0 = chunk * ch, u1 = min((chunk + 1) * ch, (max(len, 0) + KVQ_PAGE - 1) / KVQ_PAGE);
    auto place = [&](int u) -> int64_t {  // the page's first position in rows of one head, or -1
        const int page = u < u1 ? __ldg(pages + u) : -1;
        return (unsigned)page < (unsigned)a.pool.n_pages ? ((int64_t)page * Hk + kvh) * KVQ_PAGE : -1;
    };
    auto fetch = [&](int64_t at, int slot, bool v) {  // K with both scales, or V, into slot 0 or 1
        if (at >= 0) {
            const uint8_t *src = (const uint8_t *)(v ? a.pool.v : a.pool.k) + at * D + tid * 16;
            const uint32_t dst = smem_s + ((v ? 2 : 0) + slot) * Sh::SLOT;
#pragma unroll
            for (int i = 0; i < Sh::SLOT / 2048; i++) {
                const int idx = i * 128 + tid, r = idx / Sh::CPR, c = idx % Sh::CPR;
                cp16(dst + 16 * (v ? v_piece<D>(r, c) : k_piece<D>(r, c)), src + i * 2048);
            }
            if (!v) cp4(smem_s + Sh::OFF_SC + (slot * 128 + tid) * 4, (tid < 64 ? a.pool.k_scale + at : a.pool.v_scale + at - 64) + tid);
        }
        cp_commit();
    };
    int64_t at = -1, at1 = -1, at2 = -1;
    auto begin = [&]() {
        at = place(u0);
        at1 = place(u0 + 1);
        at2 = place(u0 + 2);
        fetch(at, 0, false);
        fetch(at, 0, true);
        fetch(at1, 1, false);
    };
    if (a.at.window == 0) begin();
    // ---- rows: place, visible range [lo, hi] in the segment's positions, query as fp16
    const SeqTable seqs = load_seqs(a, sg, (int32_t *)sq, NW * 32);  // (the queries' memory, not in use yet)
    if (tid < RT) row_range(a, sg, seqs, row_first + tid, s_row[tid], s_lo[tid], s_hi[tid]);
    __syncthreads();
    // the tile's ranges (rows that do not exist see everything and are not written)
    int lo_min = 0x7fffffff, lo_max = 0, hi_min = 0x7fffffff, hi_max = -1;
#pragma unroll
    for (int n = lane; n < (RT + 31) / 32 * 32; n += 32) {
        const bool on = n < RT && s_row[n < RT ? n : 0] >= 0;
        const int lo = on ? s_lo[n] : 0, hi = on ? s_hi[n] : 0;
        lo_min = min(lo_min, __reduce_min_sync(0xffffffffu, on ? lo : 0x7fffffff));
        lo_max = max(lo_max, __reduce_max_sync(0xffffffffu, on ? lo : 0));
        hi_min = min(hi_min, __reduce_min_sync(0xffffffffu, on ? hi : 0x7fffffff));
        hi_max = max(hi_max, __reduce_max_sync(0xffffffffu, on ? hi : -1));
    }
    if (a.at.window > 0) {
        u0 = max(u0, lo_min / KVQ_PAGE);
        u1 = min(u1, hi_max < 0 ? 0 : hi_max / KVQ_PAGE + 1);
        begin();
    }

    for (int n = warp; n < RT; n += NW) {
        const int row = s_row[n];
        float x[D / 32], mx = 0.0f;
#pragma unroll
        for (int i = 0; i < D / 32; i++) {
            x[i] = row < 0 ? 0.0f : load_any(a.q, row * a.ldq + (kvh * G + (row_first + n) % G) * D + i * 32 + lane, a.at.type);
            mx = fmaxf(mx, fabsf(x[i]));
        }
        mx = warp_max(mx);
        const int e = row_exponent(mx);
        const float up = pow2(e);
#pragma unroll
        for (int i = 0; i < D / 32; i++) {
            const float y = x[i] * up;
            const __half h = __float2half_rn(y);
            sq[n * QS + i * 32 + lane] = h;
            if (NQ > 1) sq[(RT + n) * QS + i * 32 + lane] = __float2half_rn(y - __half2float(h));
        }
        // scores in base 2, or natural ones for the cap
        if (lane == 0)
            s_qf[n] = a.at.scale * code_unit<FMT>() * (a.at.softcap > 0.0f ? 1.0f : 1.4426950408889634f) * pow2(-e);
    }
    cp_wait<0>();
    __syncthreads();
    // this lane's rows are nt * 8 + 2 t and the next
    float qf[NT][2], ref[NT][2], unit[NT][2], l[NT][2], o[Sh::GPW][2][NT][4];  // unit: 2^-E
    int clo[NT][2], chi[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
#pragma unroll
        for (int c = 0; c < 2; c++) {
            const int n = nt * 8 + 2 * t + c;
            qf[nt][c] = s_qf[n];
            clo[nt][c] = s_lo[n];
            chi[nt][c] = s_hi[n];
            ref[nt][c] = -INFINITY;
            unit[nt][c] = 1.0f;
            l[nt][c] = 0.0f;
        }
#pragma unroll
        for (int q = 0; q < Sh::GPW; q++)
#pragma unroll
            for (int e = 0; e < 4; e++) o[q][0][nt][e] = o[q][1][nt][e] = 0.0f;
    }
    const bool cap = a.at.softcap > 0.0f;
    const float inv_cap2 = cap ? 2.0f * 1.4426950408889634f / a.at.softcap : 0.0f;
    auto query = [&](int c, uint32_t (&qb)[NQ][NT][Sh::KB / 2]) {  // B fragments of piece c
#pragma unroll
        for (int h = 0; h < NQ; h++)
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
                const uint8_t *p = (const uint8_t *)(sq + (h * RT + nt * 8 + g) * QS + (c * 4 + t) * Sh::KB);
#pragma unroll
                for (int i = 0; i < Sh::KB / 8; i++) {
                    uint32_t w[4];
                    lds<16>(p + 16 * i, w);
#pragma unroll
                    for (int x = 0; x < 4; x++) qb[h][nt][4 * i + x] = w[x];
                }
            }
    };
    uint32_t qr[QREG ? Sh::KC : 1][NQ][NT][Sh::KB / 2];
    if (QREG)
#pragma unroll
        for (int c = 0; c < Sh::KC; c++) query(c, qr[QREG ? c : 0]);

    const int j16 = warp * 16 + row_position(g);  // this lane's positions of a page in S^T: j16 and j16 + 8
    const int grp = D == 64 ? warp & 1 : warp, mt0 = D == 64 ? (warp >> 1) * 2 : 0;
    for (int u = u0, sl = 0; u < u1; u++, sl ^= 1) {
        const int64_t now = at;
        at = at1;
        at1 = at2;
        at2 = place(u + 3);
        bool again = false;
        const int t0 = u * KVQ_PAGE + j16;
        __half *pw = sp + sl * NP * RT * PS;
        float s[NT][4], ln[NT][2], vf[2] = {0.0f, 0.0f};
        const bool whole = u * KVQ_PAGE >= lo_max && u * KVQ_PAGE + KVQ_PAGE - 1 <= hi_min;
        // the weights of this warp's positions into shared memory, relative to the references
        auto weights = [&]() {
            uint32_t any = 0;
            bool over = false;
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
                float p[4];
                ln[nt][0] = ln[nt][1] = 0.0f;
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const float x = s[nt][e];
                    float y = ex2(x - ref[nt][e & 1]);
                    p[e] = y * vf[e >> 1] * unit[nt][e & 1];
                    if (!whole && x == -INFINITY) y = p[e] = 0.0f;  // whatever the unseen position holds
                    ln[nt][e & 1] += y;
                }
                over |= !(fmaxf(ln[nt][0], ln[nt][1]) < SUM_LIMIT);  // (not set yet: infinite)
                uint32_t b[NP][2];
#pragma unroll
                for (int hf = 0; hf < 2; hf++) {
                    const uint32_t hi = pack(p[2 * hf], p[2 * hf + 1]);
                    any = hadd2(any, hi);
                    b[0][hf] = transpose8(hi);
                    if (NP > 1) {
                        const float2 back = __half22float2(*reinterpret_cast<const __half2 *>(&hi));
                        b[NP - 1][hf] = transpose8(pack(p[2 * hf] - back.x, p[2 * hf + 1] - back.y));
                    }
                }
#pragma unroll
                for (int h = 0; h < NP; h++)
                    *(uint2 *)(pw + (h * RT + nt * 8 + g) * PS + warp * 16 + t * 4) = make_uint2(b[h][0], b[h][1]);
            }
            return over || too_large(any);
        };
        if (now >= 0) {
            // ---- S^T = K Q^T: 16 positions
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int e = 0; e < 4; e++) s[nt][e] = 0.0f;
            const uint8_t *kslot = smem + sl * Sh::SLOT;
            const float *ksc = (const float *)(smem + Sh::OFF_SC) + sl * 128;
            const float kf[2] = {ksc[j16], ksc[j16 + 8]};
            vf[0] = ksc[64 + j16] * code_unit<FMT>();
            vf[1] = ksc[64 + j16 + 8] * code_unit<FMT>();
#pragma unroll
            for (int c = 0; c < Sh::KC; c++) {
                uint32_t ql[NQ][NT][Sh::KB / 2];
                if (!QREG) query(c, ql);
                const uint32_t (&qb)[NQ][NT][Sh::KB / 2] = QREG ? qr[QREG ? c : 0] : ql;
                float piece[NT][4] = {};
                float (&acc)[NT][4] = ROUNDED && Sh::KC > 1 ? piece : s;
                uint32_t w[2][Sh::KB / 4];
#pragma unroll
                for (int hf = 0; hf < 2; hf++) {
                    const int r = j16 + hf * 8, byte = (c * 4 + t) * Sh::KB;
                    lds<Sh::KB>(kslot + 16 * k_piece<D>(r, byte / 16) + byte % 16, w[hf]);
                }
#pragma unroll
                for (int k = 0; k < Sh::KB / 4; k++) {
                    const uint32_t x0 = w[0][k] ^ code_flip<FMT>(), x1 = w[1][k] ^ code_flip<FMT>();
                    const uint32_t f[4] = {codes2<FMT, 0, 1>(x0), codes2<FMT, 0, 1>(x1), codes2<FMT, 2, 3>(x0), codes2<FMT, 2, 3>(x1)};
#pragma unroll
                    for (int nt = 0; nt < NT; nt++)
#pragma unroll
                        for (int h = 0; h < NQ; h++) mma(acc[nt], f, qb[h][nt][2 * k], qb[h][nt][2 * k + 1]);
                }
                if (ROUNDED && Sh::KC > 1)
#pragma unroll
                    for (int nt = 0; nt < NT; nt++)
#pragma unroll
                        for (int e = 0; e < 4; e++) s[nt][e] += piece[nt][e];
            }
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    s[nt][e] *= kf[e >> 1] * qf[nt][e & 1];
                    if (cap) s[nt][e] = capped<PREC == 2>(s[nt][e], a.at.softcap, inv_cap2) * 1.4426950408889634f;
                }
            if (!whole)
#pragma unroll
                for (int nt = 0; nt < NT; nt++)
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const int j = t0 + (e >> 1) * 8;
                        if (j < clo[nt][e & 1] || j > chi[nt][e & 1] || j >= len) s[nt][e] = -INFINITY;
                    }
            again = weights();
        }
        cp_wait<0>();                  // V of this page and K of the next, this thread's part
        again = __syncthreads_or(again);  // everybody's, and all weights
        fetch(at, sl ^ 1, true);
        fetch(at1, sl, false);
        if (now < 0) continue;
        if (again) {
            // ---- some weight is near the limit (or a reference is not set): search the rows' maxima over the page, of
            // the scores and with the values' scales, and raise the references of the rows that need it
            const float lv[2] = {log2_abs(vf[0]), log2_abs(vf[1])};
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int c = 0; c < 2; c++) {  // (a NaN does not count)
                    float mx = fmaxf(s[nt][c], s[nt][c + 2]), mv = fmaxf(s[nt][c] + lv[0], s[nt][c + 2] + lv[1]);
#pragma unroll
                    for (int d = 4; d < 32; d <<= 1) {
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
                        mv = fmaxf(mv, __shfl_xor_sync(0xffffffffu, mv, d));
                    }
                    if (g == 0) {
                        s_max[warp][nt * 8 + 2 * t + c] = mx;
                        s_l[warp][nt * 8 + 2 * t + c] = mv;
                    }
                }
            __syncthreads();
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int c = 0; c < 2; c++) {
                    const int n = nt * 8 + 2 * t + c;
                    const float top = fmaxf(fmaxf(s_max[0][n], s_max[1][n]), fmaxf(s_max[2][n], s_max[3][n]));
                    const float topv = fmaxf(fmaxf(s_l[0][n], s_l[1][n]), fmaxf(s_l[2][n], s_l[3][n]));
                    float fl, fo;
                    if (!raise_refs(top, topv, ref[nt][c], unit[nt][c], fl, fo)) continue;
                    l[nt][c] *= fl;
#pragma unroll
                    for (int q = 0; q < Sh::GPW; q++)
#pragma unroll
                        for (int j = 0; j < 2; j++) {
                            o[q][j][nt][c] *= fo;
                            o[q][j][nt][c + 2] *= fo;
                        }
                }
            weights();
            __syncthreads();
        }
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            l[nt][0] += ln[nt][0];
            l[nt][1] += ln[nt][1];
        }
        // ---- O^T += V^T P^T: 32 dimensions
        if (D != 96 || warp < 3) {
            const uint8_t *vslot = smem + (2 + sl) * Sh::SLOT;
            float page[Sh::GPW][2][NT][4] = {};
            float (&acc)[Sh::GPW][2][NT][4] = ROUNDED ? page : o;
#pragma unroll
            for (int m = 0; m < (D == 64 ? 2 : 4); m++) {
                const int mt = mt0 + m;
                uint2 pb[NP][NT];
#pragma unroll
                for (int h = 0; h < NP; h++)
#pragma unroll
                    for (int nt = 0; nt < NT; nt++) pb[h][nt] = *(const uint2 *)(pw + (h * RT + nt * 8 + g) * PS + mt * 16 + t * 4);
#pragma unroll
                for (int q = 0; q < Sh::GPW; q++) {
                    uint32_t x[4];
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const int r = mt * 16 + 4 * i + t, byte = (grp + 4 * q) * 32 + g * 4;
                        x[i] = *(const uint32_t *)(vslot + 16 * v_piece<D>(r, byte / 16) + byte % 16) ^ code_flip<FMT>();
                    }
#pragma unroll
                    for (int hf = 0; hf < 2; hf++) {  // dimensions 0, 1 and 2, 3 of the four bytes
                        const uint32_t ab = __byte_perm(x[0], x[1], hf ? 0x7362 : 0x5140), cd = __byte_perm(x[2], x[3], hf ? 0x7362 : 0x5140);
                        const uint32_t fr[4] = {codes2<FMT, 0, 1>(ab), codes2<FMT, 2, 3>(ab), codes2<FMT, 0, 1>(cd), codes2<FMT, 2, 3>(cd)};
#pragma unroll
                        for (int nt = 0; nt < NT; nt++)
#pragma unroll
                            for (int h = 0; h < NP; h++) mma(acc[q][hf][nt], fr, pb[h][nt].x, pb[h][nt].y);
                    }
                }
            }
            if (ROUNDED)
#pragma unroll
                for (int q = 0; q < Sh::GPW; q++)
#pragma unroll
                    for (int hf = 0; hf < 2; hf++)
#pragma unroll
                        for (int nt = 0; nt < NT; nt++)
#pragma unroll
                            for (int e = 0; e < 4; e++) o[q][hf][nt][e] += page[q][hf][nt][e];
        }
    }
    cp_wait<0>();

    // ---- the rows' sums over the warps; with head_dim 64 the two warps of a group
#pragma unroll
    for (int nt = 0; nt < NT; nt++)
#pragma unroll
        for (int c = 0; c < 2; c++) {
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) l[nt][c] += __shfl_xor_sync(0xffffffffu, l[nt][c], d);
            if (g == 0) s_l[warp][nt * 8 + 2 * t + c] = l[nt][c];
        }
    __syncthreads();
    float4 *so = (float4 *)smem;  // [warp & 1][nt, column][lane]
    if (D == 64 && warp >= 2) {
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int c = 0; c < 2; c++)
                so[((warp & 1) * NT * 2 + nt * 2 + c) * 32 + lane] = make_float4(o[0][0][nt][c], o[0][0][nt][c + 2], o[0][1][nt][c], o[0][1][nt][c + 2]);
    }
    if (D == 64) __syncthreads();
    const int64_t RH = (int64_t)a.bt.rows * a.at.heads, slot = sg.pre ? chunk : a.nsp + chunk;
    if (warp < (D == 64 ? 2 : D == 96 ? 3 : 4)) {
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int c = 0; c < 2; c++) {
                const int n = nt * 8 + 2 * t + c, row = s_row[n];
                if (row < 0) continue;
                const float L = (s_l[0][n] + s_l[1][n]) + (s_l[2][n] + s_l[3][n]);
                const int head = kvh * G + (row_first + n) % G;
                const int64_t rh = (int64_t)row * a.at.heads + head;
#pragma unroll
                for (int q = 0; q < Sh::GPW; q++) {
                    float x[4] = {o[q][0][nt][c], o[q][0][nt][c + 2], o[q][1][nt][c], o[q][1][nt][c + 2]};
                    if (D == 64) {
                        const float4 v = so[(warp * NT * 2 + nt * 2 + c) * 32 + lane];
                        x[0] += v.x;
                        x[1] += v.y;
                        x[2] += v.z;
                        x[3] += v.w;
                    }
                    const int d = (grp + 4 * q) * 32 + g * 4;
                    const float f = a.direct ? 1.0f / L : 1.0f, u = pow_inverse(unit[nt][c]);
#pragma unroll
                    for (int e = 0; e < 4; e++) x[e] = a.direct && L == 0.0f ? 0.0f : x[e] * f * u;
                    if (a.direct) store4(a.out, row * a.ldo + (int64_t)head * D + d, a.at.type, a.wide != 0, x);
                    else *(float4 *)(a.part_o + (slot * RH + rh) * D + d) = make_float4(x[0], x[1], x[2], x[3]);
                }
                if (warp == 0 && g == 0) {
                    if (!a.direct) a.part_ml[slot * RH + rh] = make_float2(ref[nt][c], L);
                    else if (a.lse) a.lse[rh] = L == 0.0f ? -INFINITY : (ref[nt][c] + log2f(L)) * 0.6931471805599453f;
                }
            }
    }
    if (a.chained) pdl_wait();
}

// Joins a row's partials in chunk order: W warps per (row, head), each every W-th chunk, then the prefix's
// chunks first.  One warp where there are many rows or few chunks; four else, since a warp has only
// a few loads in flight.
template <int D, int W> __global__ void __launch_bounds__(128) kvq_join_kernel(const __grid_constant__ AttnArgs a)
{
    constexpr int N = D / 32;
    __shared__ float s_x[W > 1 ? 4 : 1][W > 1 ? D : 1], s_l[4];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, part = warp % W;
    const int64_t item = (int64_t)blockIdx.x * (4 / W) + warp / W, RH = (int64_t)a.bt.rows * a.at.heads;
    if (item >= RH) return;  // with W = 4 a whole CTA
    const int row = (uint32_t)item / (uint32_t)a.at.heads, head = (uint32_t)item - row * a.at.heads;
    const int b = kvq_seq_of(a.bt.row_start, a.bt.batch, row);
    int nown = 0;
    if (b >= 0) {
        const int len = (int)min((int64_t)a.bt.seq_len[b], (int64_t)a.bt.max_pages * KVQ_PAGE);
        nown = len > 0 ? (len - 1) / (a.ch_s * KVQ_PAGE) + 1 : 0;
    }
    pdl_wait();
    if (b < 0 || row - a.bt.row_start[b] >= a.bt.max_rows) return;
    const int slots = a.nsp + nown;
    const float2 *ml = a.part_ml + item;
    float M = -INFINITY;
    for (int s = lane; s < slots; s += 32) M = fmaxf(M, __ldcg(ml + s * RH).x);
    M = warp_max(M);
    float L = 0.0f, x[N] = {};
    for (int s0 = 0; s0 < slots; s0 += 32 * W) {
        float w = 0.0f;
        const int mine = s0 + lane * W + part;
        if (mine < slots) {
            const float2 v = __ldcg(ml + mine * RH);
            if (v.x != -INFINITY || v.y != v.y) {
                w = ex2(v.x - M);
                L = fmaf(v.y, w, L);
            }
        }
        const int n = min(32, (slots - s0 - part + W - 1) / W);
#pragma unroll 4
        for (int s = 0; s < n; s++) {
            const float f = __shfl_sync(0xffffffffu, w, s);
            const float *p = a.part_o + ((int64_t)(s0 + s * W + part) * RH + item) * D + lane;
            float v[N];
#pragma unroll
            for (int i = 0; i < N; i++) v[i] = __ldcg(p + 32 * i);
#pragma unroll
            for (int i = 0; i < N; i++) x[i] = f == 0.0f ? x[i] : fmaf(v[i], f, x[i]);  // a chunk that saw nothing wrote nothing
        }
    }
    L = warp_sum(L);
    if (W > 1) {
#pragma unroll
        for (int i = 0; i < N; i++) s_x[warp][32 * i + lane] = x[i];
        if (lane == 0) s_l[warp] = L;
        __syncthreads();
        L = (s_l[0] + s_l[1]) + (s_l[2] + s_l[3]);
    }
    const float inv = 1.0f / L;
#pragma unroll
    for (int i = 0; i < N; i++) {
        if (W > 1 && i % W != part) continue;
        if (W > 1) x[i] = (s_x[0][32 * i + lane] + s_x[1][32 * i + lane]) + (s_x[2][32 * i + lane] + s_x[3][32 * i + lane]);
        const float y = L == 0.0f ? 0.0f : x[i] * inv;
        const int64_t at = row * a.ldo + (int64_t)head * D + 32 * i + lane;
        if (a.at.type == T_F32) ((float *)a.out)[at] = y;
        else if (a.at.type == T_F16) ((__half *)a.out)[at] = __float2half_rn(y);
        else ((__nv_bfloat16 *)a.out)[at] = __float2bfloat16_rn(y);
    }
    if (a.lse && part == 0 && lane == 0) a.lse[item] = L == 0.0f ? -INFINITY : (M + log2f(L)) * 0.6931471805599453f;
}

// ------------------------------------------------------------------ launch
template <int D, int FMT, int NT, int PREC> cudaError_t launch_tiles(const AttnArgs &a, int64_t grid, cudaStream_t st)
{
    using Sh = Shape<D>;
    constexpr int NQ = PREC == 2 ? 2 : 1, NP = PREC > 0 ? 2 : 1, smem = narrow_smem(D, NT, NQ, NP);
    static_assert(smem == Sh::OFF_Q + NT * 8 * (NQ * (D + Sh::QPAD) + NP * 2 * PS) * 2, "the kernel's layout");
    static_assert(smem - Sh::OFF_Q >= (2 * SEQ_TABLE + 1) * 4, "the sequences' tables fit into the queries' and weights' memory");
    static_assert(D != 64 || 4 * Sh::SLOT >= 2 * NT * 2 * 512, "two warps' outputs fit into the slots");
    static std::atomic<unsigned long long> done{0};
    cudaError_t e = smem_attr_once(done, kvq_attn_kernel<D, FMT, NT, PREC>, smem);
    if (e != cudaSuccess) return e;
    return launch_kernel(a.chained != 0, kvq_attn_kernel<D, FMT, NT, PREC>, dim3((unsigned)grid), dim3(NW * 32), smem, st, a);
}
template <int D, int FMT, int PREC> cudaError_t launch_nt(int nt, const AttnArgs &a, int64_t grid, cudaStream_t st)
{
    switch (nt) {
    case 1: return launch_tiles<D, FMT, 1, PREC>(a, grid, st);
    case 2: return launch_tiles<D, FMT, 2, PREC>(a, grid, st);
    case 3: return launch_tiles<D, FMT, 3, PREC>(a, grid, st);
    default: return launch_tiles<D, FMT, D == 256 && PREC == 2 ? 3 : 4, PREC>(a, grid, st);
    }
}
template <int D, int FMT> cudaError_t launch_prec(int nt, const AttnArgs &a, int64_t grid, cudaStream_t st)
{
    if (a.at.type == T_F32) return launch_nt<D, FMT, 2>(nt, a, grid, st);
    if (a.at.type == T_F16) return launch_nt<D, FMT, 1>(nt, a, grid, st);
    return launch_nt<D, FMT, 0>(nt, a, grid, st);
}
template <int D> cudaError_t launch_dim(int nt, const AttnArgs &a, int64_t grid, cudaStream_t st)
{
    if (a.pool.format == LLMDOT_KVQ_I8) return launch_prec<D, LLMDOT_KVQ_I8>(nt, a, grid, st);
    return launch_prec<D, LLMDOT_KVQ_E4M3>(nt, a, grid, st);
}
cudaError_t launch_narrow(int nt, const AttnArgs &a, int64_t grid, cudaStream_t st)
{
    switch (a.pool.head_dim) {
    case 64: return launch_dim<64>(nt, a, grid, st);
    case 96: return launch_dim<96>(nt, a, grid, st);
    case 128: return launch_dim<128>(nt, a, grid, st);
    default: return launch_dim<256>(nt, a, grid, st);
    }
}
template <int D> cudaError_t launch_join_dim(const AttnArgs &a, cudaStream_t st)
{
    const int64_t items = (int64_t)a.bt.rows * a.at.heads;
    if (a.nsp + a.nss <= 4 || items > 148 * 32)
        return launch_kernel(true, kvq_join_kernel<D, 1>, dim3((unsigned)((items + 3) / 4)), dim3(128), 0, st, a);
    return launch_kernel(true, kvq_join_kernel<D, 4>, dim3((unsigned)items), dim3(128), 0, st, a);
}
cudaError_t launch_join(const AttnArgs &a, cudaStream_t st)
{
    switch (a.pool.head_dim) {
    case 64: return launch_join_dim<64>(a, st);
    case 96: return launch_join_dim<96>(a, st);
    case 128: return launch_join_dim<128>(a, st);
    default: return launch_join_dim<256>(a, st);
    }
}

// How a call is cut.  From the sizes the host knows; lengths on the device only decide which CTAs find
// nothing to do.
struct Plan {
    int wide_p, wide_s;  // the segment kind goes to the wide kernel
    int nt_p, nt_s;      // 8-row tiles of the narrow kernel
    int ch_p, ch_s, nsp, nss, ptiles, rtiles, direct;
    int64_t ctas_p, ctas_s;
    size_t o_bytes, ml_bytes;
};
// 8-row tiles per CTA, 1 to 4.  16-bit queries of more than 32 rows go to the wide kernel; fp32 ones take several CTAs: a tile of
// 64 rows leaves two CTAs per SM and spills (512 rows, heads of 64 / 96 / 128: 263 / 424 / 447 us; 32: 221 / 286 / 310).  fp32 and
// head_dim 256, where 32 rows fill an SM's shared memory: 16 up to 32 rows, else 24 (4 x 4 rows on a prefix of 6144: 16 28.9, 24
// 33.5, 32 39.0; 80 rows on 3000: 39.1, 31.6, 53.0; 512 rows: 634, 522, 669).
int tiles_of(int dim, int64_t rows, uint32_t type)
{
    const int64_t n = std::max<int64_t>(1, (rows + 7) / 8);
    return (int)std::min<int64_t>(n, type != T_F32 || dim != 256 ? 4 : n <= 4 ? 2 : 3);
}
// Whether `rows` rows (times heads) per kv head over `items` pages and heads in all go to the wide kernel.  It takes
// the same time for 1 to 256 rows, the narrow one grows with every 8 (above 32 rows measured with a tile of 64).  Some thousand
// positions, 8 kv heads (or as said), bf16, heads of 64 / 96 / 128 / 256, us, wide : narrow.
//   Work enough for all SMs, so that only throughput counts, own pages of 24 sequences, 4608 items: 32 rows 62 : 46 / 68 : 64 /
//   72 : 72 / 128 : 115, 40 rows 62 : 68 / 68 : 92 / 72 : 103 / 128 : 161; 96 sequences, fp16, heads of 64: 40 rows 165 : 160.
//   2048 items or fewer, where the latency of one CTA's chunk counts.  Own pages, 2048 items: 16 rows 28 : 27 / 31 : 33 / 31 : 35 /
//   52 : 54, 20 rows 29 : 35 / 31 : 39 / 32 : 42 / 52 : 66; 188 items, 20 rows 19 : 18 / 21 : 21 / 21 : 21 / 24 : 27.
//   A prefix, 2048 items: 24 rows 29 : 30 / 34 : 37 / 34 : 37 / 58 : 56, with 32 kv heads 33 : 27 / 38 : 33 / 39 : 35 / 62 : 73, and with
//   32 rows 33 : 39 / 39 : 46 / 39 : 51 / 64 : 86; 256 items, 20 rows of 256 27 : 35.  3000 items: 24 rows 37 : 33 / 43 : 41 / 44 : 43 / 79 : 64.
bool wide_pays(const llmdot_kvq_pool &p, int64_t rows, int64_t items, bool own)
{
    return rows >= 33 || (items <= 2048 && rows >= (own || p.head_dim == 256 ? 17 : 25));
}

// Product of counts, at most 2^60: batch, max_pages and heads may each be large without any being too large.
int64_t times(int64_t a, int64_t b)
{
    const int64_t most = (int64_t)1 << 60;
    return b > 0 && a > most / b ? most : std::min(a * b, most);
}

constexpr int64_t PART_BYTES = 128 << 20;  // of the prefix's partials, and of the own pages'

Plan make_plan(const llmdot_kvq_pool &p, const llmdot_kvq_batch &b, const llmdot_kvq_attn &a)
{
    Plan x = {};
    // max_rows is a bound: no sequence has more rows than the call
    const int64_t G = a.heads / p.heads_kv, Hk = p.heads_kv, own_rows = std::min(b.max_rows, b.rows) * G, all_rows = (int64_t)b.rows * G;
    const int64_t npp = (a.prefix_len + KVQ_PAGE - 1) / KVQ_PAGE, wide = kvq_wide_rows(p.head_dim);
    auto up = [](int64_t x, int64_t y) { return (x + y - 1) / y; };
    x.wide_p = a.type != T_F32 && npp > 0 && wide_pays(p, all_rows, Hk * npp, false);
    x.wide_s = a.type != T_F32 && wide_pays(p, own_rows, times(Hk * b.batch, b.max_pages), true);
    x.nt_p = tiles_of(p.head_dim, all_rows, a.type);
    x.nt_s = tiles_of(p.head_dim, own_rows, a.type);
    if (npp == 0) x.nt_p = x.nt_s;
    x.ptiles = (int)up(all_rows, x.wide_p ? wide : 8 * x.nt_p);
    x.rtiles = (int)std::max<int64_t>(1, up(own_rows, x.wide_s ? wide : 8 * x.nt_s));
    // Chunks.  Narrow: about one CTA per place on the SMs for the prefix, two for the sequences' own pages
    // (max_pages is a bound: ragged sequences leave some without work), at most 32 pages, so that long
    // and short sequences balance.  Wide: one CTA per SM, at least two pages.  At most 256 chunks of either, even ones,
    // and no more than PART_BYTES of partials unless one chunk takes them: with rows enough for that a chunk has
    // CTAs enough for all SMs, and the partials of a table much longer than the sequences, or of a long prompt
    // chunk of fp32 rows (2 GB with 2048 rows of 32 heads and 2048 pages), stay in L2.
    const int64_t part = std::max<int64_t>(1, (int64_t)b.rows * a.heads * (p.head_dim * 4 + 8));  // bytes of one chunk's
    const int64_t most = std::min<int64_t>(256, std::max<int64_t>(1, PART_BYTES / part));
    auto places = [&](int nt) {  // CTAs on the SMs
        return (int64_t)148 * narrow_ctas(p.head_dim, nt, a.type == T_F32 ? 2 : 1, a.type == T_BF16 ? 1 : 2);
    };
    auto chunk = [&](int64_t pages, int64_t ctas, int64_t least) { return std::min<int64_t>(32, std::max<int64_t>(least, up(pages, ctas))); };
    auto bounded = [&](int64_t ch, int64_t pages) {
        ch = std::max(ch, up(pages, most));
        return (int)std::max<int64_t>(1, up(pages, std::max<int64_t>(1, up(pages, ch))));
    };
    auto wide_ch = [&](int64_t ctas, int64_t pages) { return std::max<int64_t>(2, up(pages, std::max<int64_t>(1, 148 / std::max<int64_t>(1, ctas)))); };
    x.ch_p = bounded(x.wide_p ? wide_ch(Hk * x.ptiles, npp) : chunk(Hk * x.ptiles * npp, places(x.nt_p), 1), npp);
    x.ch_s = bounded(x.wide_s ? wide_ch(times(Hk * x.rtiles, b.batch), b.max_pages)
                              : chunk(times(times(Hk * x.rtiles, b.batch), b.max_pages), 2 * places(x.nt_s), 2), b.max_pages);
    x.nsp = (int)up(npp, x.ch_p);
    x.nss = (int)std::max<int64_t>(1, up(b.max_pages, x.ch_s));
    x.direct = x.nsp == 0 && x.nss == 1 && !x.wide_s;
    x.ctas_p = Hk * x.ptiles * x.nsp;
    x.ctas_s = times(times(Hk * x.rtiles, x.nss), b.batch);
    if (!x.direct) {
        const size_t rh = (size_t)b.rows * a.heads * (x.nsp + x.nss);
        x.o_bytes = rh * p.head_dim * 4;
        x.ml_bytes = rh * 8;
    }
    return x;
}

// One to two kernels over the segments (the second over the first, which it outlives), then the join.
cudaError_t run_plan(const Plan &x, AttnArgs &a, cudaStream_t st)
{
    cudaError_t e = cudaSuccess;
    const bool together = !x.wide_p && !x.wide_s && x.nt_p == x.nt_s;
    if (!together && x.ctas_p > 0) {
        a.prefix_ctas = (int)x.ctas_p;
        e = x.wide_p ? launch_kvq_wide(a, x.ctas_p, false, st) : launch_narrow(x.nt_p, a, x.ctas_p, st);
        if (e != cudaSuccess) return e;
        a.chained = 1;
    }
    a.prefix_ctas = together ? (int)x.ctas_p : 0;
    e = x.wide_s ? launch_kvq_wide(a, x.ctas_s, a.chained != 0, st) : launch_narrow(x.nt_s, a, a.prefix_ctas + x.ctas_s, st);
    if (e != cudaSuccess || x.direct) return e;
    return launch_join(a, st);
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
    if ((uintptr_t)a->prefix_pages & 3) return bad("prefix_pages must be 4-byte aligned");
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
        const Plan x = make_plan(*pool, *batch, *attn);
        *bytes = x.o_bytes + x.ml_bytes;
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
        const int es = kvq_type_size(attn->type);
        if (((uintptr_t)d_q | (uintptr_t)d_out) % es) return bad("q or output is not aligned to its type");
        if ((uintptr_t)d_lse & 3) return bad("lse must be 4-byte aligned");
        const Plan x = make_plan(*pool, *batch, *attn);
        if (x.o_bytes + x.ml_bytes > 0 && (!d_work || work_bytes < x.o_bytes + x.ml_bytes || ((uintptr_t)d_work & 15)))
            return bad("workspace is null, too small or not 16-byte aligned");
        if (x.ctas_p + x.ctas_s > 0x7fffffff) return bad("too many sequences, rows or pages for one call");
        AttnArgs a = {};
        a.pool = *pool;
        a.bt = *batch;
        a.at = *attn;
        a.q = d_q;
        a.out = d_out;
        a.ldq = ld_q;
        a.ldo = ld_out;
        a.lse = d_lse;
        a.part_o = (float *)d_work;
        a.part_ml = (float2 *)((uint8_t *)d_work + x.o_bytes);
        a.group = attn->heads / pool->heads_kv;
        a.ch_p = x.ch_p;
        a.ch_s = x.ch_s;
        a.nsp = x.nsp;
        a.nss = x.nss;
        a.ptiles = x.ptiles;
        a.rtiles = x.rtiles;
        a.direct = x.direct;
        a.wide = ((uintptr_t)d_out & 15) == 0 && (batch->rows <= 1 || ld_out * es % 16 == 0);
        const cudaError_t e = run_plan(x, a, (cudaStream_t)stream);
        if (e != cudaSuccess) return cuda_fail(e, "kvq_attention");
        return LLMDOT_OK;
    });
}
