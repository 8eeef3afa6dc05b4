// kvq_attn.cu -- attention of a batch over a shared prefix and its own pages, K and V in 8 bits.
//
// s_j = scale * (q . k_j), optionally capped; out = sum_j softmax(s)_j v_j, with k_j = code * scale_j
// (one fp32 scale per position and head).
//
// Mathematics.  A code is an integer of at most 7 bits and sign, or an e4m3 value: exact in fp16.  The
// query row is scaled by a power of two into fp16 (fp32 queries: as hi + lo, two products), so q . code
// is a sum of exact products in fp32, and the key's scale multiplies the score.  The value's scale goes
// into the weight: P_j = exp2(s_j - m) * (v_scale_j / 2^E), 2^E the largest power of two not above the
// v_scales seen so far (raised with the running maximum, the sums rescaled by both), so that P stays in
// fp16's normal range whatever the scales' size; P is rounded to fp16 once (fp32 queries: hi + lo).
// The sum of exponentials, the maxima, both products' sums and the outputs are fp32.
//
// Work is cut into segments -- the prefix with every row of the batch, each sequence's own pages with
// its rows -- times kv heads, row tiles and chunks of pages.  The prefix is read once per row tile of
// the whole batch, not once per sequence.  Each CTA leaves a partial (m, l, O) of its chunk; a second kernel
// (programmatic dependent launch) joins a row's partials in chunk order.  A call with one chunk in
// all writes its output directly.
//
// Bound: HBM (the codes) while a kv head has few rows.  Inside a CTA each of four warps streams its own
// units of LT positions (cp.async, one K and one V slot in flight per warp, no block barrier in
// the loop) and forms S^T = K Q^T and O^T = V^T P^T with mma.m16n8k16: positions and head dimensions
// take the 16-wide side and the rows the 8-wide side, so 4 rows (one token of a group of 4 heads) waste
// half a tile rather than three quarters.  The order of k inside a tile is free as long as both
// operands agree; it is chosen so that a lane's K bytes are 16 consecutive ones, and its V bytes four
// positions of 16 (4, 8) consecutive dimensions, which shuffle into A fragments by byte permutes.
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
// Shapes of the kernel for a head dimension D and NT tiles of 8 rows.
template <int D> struct Shape {
    static constexpr int LT = D == 256 ? 32 : 64;   // positions of one unit (slot)
    static constexpr int CPR = D / 16;              // 16-byte pieces of a position's codes
    static constexpr int SLOT = LT * D;             // bytes of a K or V slot
    static constexpr int KB = D == 96 ? 8 : 16;     // K bytes a lane takes at once
    static constexpr int KC = D / (4 * KB);         // such pieces
    static constexpr int VB = D == 64 ? 8 : D == 96 ? 4 : 16;  // V bytes a lane takes at once
    static constexpr int VC = D / (8 * VB);
    static constexpr int MAX_NT = D == 256 ? 2 : D == 128 ? 3 : 4;  // O^T in registers: D / 4 * NT of them
    static constexpr int QPAD = D == 96 ? 0 : 8;    // halves between query rows against bank conflicts
    static constexpr int WARP = 2 * SLOT + 2 * LT * 4;  // bytes per warp: K, V and their scales
};
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
template <> struct Bytes<4> { using T = uint32_t; };
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

template <int D, int FMT, int NT, bool SPLIT>
__global__ void __launch_bounds__(NW * 32) kvq_attn_kernel(const __grid_constant__ AttnArgs a)
{
    using Sh = Shape<D>;
    constexpr int LT = Sh::LT, MT = LT / 16, RT = 8 * NT, QS = D + Sh::QPAD, NQ = SPLIT ? 2 : 1;
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ float s_qf[RT], s_m[NW][RT], s_l[NW][RT];
    __shared__ float s_e[NW];
    __shared__ int s_lo[RT], s_hi[RT], s_row[RT];
    __half *sq = (__half *)(smem + NW * Sh::WARP);  // [NQ][RT][QS]
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
    // ---- rows: place, visible range [lo, hi] in the segment's positions, query as fp16
    const SeqTable seqs = load_seqs(a, sg, (int32_t *)smem, NW * 32);  // (the slots' memory, not in use yet)
    if (tid < RT) row_range(a, sg, seqs, row_first + tid, s_row[tid], s_lo[tid], s_hi[tid]);
    __syncthreads();
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
            if (SPLIT) sq[(RT + n) * QS + i * 32 + lane] = __float2half_rn(y - __half2float(h));
        }
        // scores in base 2, or natural ones for the cap
        if (lane == 0)
            s_qf[n] = a.at.scale * code_unit<FMT>() * (a.at.softcap > 0.0f ? 1.0f : 1.4426950408889634f) *
                      pow2(-e);
    }
    __syncthreads();
    // the tile's ranges (rows that do not exist see everything and are not written)
    int lo_min = 0x7fffffff, lo_max = 0, hi_min = 0x7fffffff, hi_max = -1;
    {
        const bool on = lane < RT && s_row[lane < RT ? lane : 0] >= 0;
        const int lo = on ? s_lo[lane] : 0, hi = on ? s_hi[lane] : 0;
        lo_min = __reduce_min_sync(0xffffffffu, on ? lo : 0x7fffffff);
        lo_max = __reduce_max_sync(0xffffffffu, on ? lo : 0);
        hi_min = __reduce_min_sync(0xffffffffu, on ? hi : 0x7fffffff);
        hi_max = __reduce_max_sync(0xffffffffu, on ? hi : -1);
    }
    float qf[NT][2];
    int clo[NT][2], chi[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; nt++)
#pragma unroll
        for (int c = 0; c < 2; c++) {
            const int n = nt * 8 + 2 * t + c;
            qf[nt][c] = s_qf[n];
            clo[nt][c] = s_lo[n];
            chi[nt][c] = s_hi[n];
        }

    // ---- this warp's units: u0 + warp, + NW, ...
    constexpr int UPP = KVQ_PAGE / LT;
    int u0 = max(chunk * ch * UPP, lo_min / LT);
    const int u1 = (int)min((int64_t)(chunk + 1) * ch * UPP, hi_max < 0 ? 0 : (int64_t)hi_max / LT + 1);
    uint8_t *kslot = smem + warp * Sh::WARP, *vslot = kslot + Sh::SLOT;
    float *ksc = (float *)(vslot + Sh::SLOT), *vsc = ksc + LT;
    const uint32_t kslot_s = su32(kslot), vslot_s = su32(vslot), ksc_s = su32(ksc), vsc_s = su32(vsc);
    auto place = [&](int u) -> int64_t {  // first position of unit u in rows of one head, or -1
        if (u >= u1) return -1;
        const int page = __ldg(pages + u / UPP);
        if ((unsigned)page >= (unsigned)a.pool.n_pages) return -1;
        return ((int64_t)page * Hk + kvh) * KVQ_PAGE + (u % UPP) * LT;
    };
    auto fetch = [&](int64_t at, bool v) {
        if (at >= 0) {
            const uint8_t *src = (const uint8_t *)(v ? a.pool.v : a.pool.k) + at * D + lane * 16;
            const uint32_t dst = v ? vslot_s : kslot_s;
#pragma unroll
            for (int i = 0; i < Sh::SLOT / 512; i++) {
                const int idx = i * 32 + lane, r = idx / Sh::CPR, c = idx % Sh::CPR;
                cp16(dst + 16 * (v ? v_piece<D>(r, c) : k_piece<D>(r, c)), src + i * 512);
            }
            const float *sc = (v ? a.pool.v_scale : a.pool.k_scale) + at + lane;
#pragma unroll
            for (int i = 0; i < LT / 32; i++) cp4((v ? vsc_s : ksc_s) + 4 * (lane + 32 * i), sc + 32 * i);
        }
        cp_commit();
    };
    float o[NT][D / 16][4], m[NT][2], l[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
#pragma unroll
        for (int j = 0; j < D / 16; j++)
#pragma unroll
            for (int e = 0; e < 4; e++) o[nt][j][e] = 0.0f;
        m[nt][0] = m[nt][1] = -INFINITY;
        l[nt][0] = l[nt][1] = 0.0f;
    }
    float vpow = 1.17549435e-38f;  // 2^E: O is in units of it
    const bool cap = a.at.softcap > 0.0f;
    const float inv_cap2 = cap ? 2.0f * 1.4426950408889634f / a.at.softcap : 0.0f;

    int u = u0 + warp;
    int64_t at = place(u), at_next = place(u + NW);
    fetch(at, false);
    fetch(at, true);
    for (; u < u1; u += NW) {
        const int64_t after = place(u + 2 * NW);
        cp_wait<1>();
        __syncwarp();
        // ---- S^T = K Q^T
        float s[MT][NT][4];
#pragma unroll
        for (int mt = 0; mt < MT; mt++)
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int e = 0; e < 4; e++) s[mt][nt][e] = 0.0f;
        if (at >= 0) {
            const int kr = (g >> 1) + 4 * (g & 1);
#pragma unroll
            for (int c = 0; c < Sh::KC; c++) {
                uint32_t qb[NQ][NT][Sh::KB / 2];
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
#pragma unroll
                for (int mt = 0; mt < MT; mt++) {
                    uint32_t w[2][Sh::KB / 4];
#pragma unroll
                    for (int hf = 0; hf < 2; hf++) {
                        const int r = mt * 16 + hf * 8 + kr, byte = (c * 4 + t) * Sh::KB;
                        lds<Sh::KB>(kslot + 16 * k_piece<D>(r, byte / 16) + byte % 16, w[hf]);
                    }
#pragma unroll
                    for (int k = 0; k < Sh::KB / 4; k++) {
                        const uint32_t x0 = w[0][k] ^ code_flip<FMT>(), x1 = w[1][k] ^ code_flip<FMT>();
                        const uint32_t f[4] = {codes2<FMT, 0, 1>(x0), codes2<FMT, 0, 1>(x1), codes2<FMT, 2, 3>(x0),
                                               codes2<FMT, 2, 3>(x1)};
#pragma unroll
                        for (int nt = 0; nt < NT; nt++)
#pragma unroll
                            for (int h = 0; h < NQ; h++) mma(s[mt][nt], f, qb[h][nt][2 * k], qb[h][nt][2 * k + 1]);
                    }
                }
            }
        }
        float kf[MT][2];
#pragma unroll
        for (int mt = 0; mt < MT; mt++)
#pragma unroll
            for (int hf = 0; hf < 2; hf++) kf[mt][hf] = ksc[mt * 16 + hf * 8 + row_position(g)];
        __syncwarp();
        const int64_t now = at;
        fetch(at_next, false);
        // ---- softmax over the unit
        const int t0 = u * LT;
        const bool whole = t0 >= lo_max && t0 + LT - 1 <= hi_min;
        if (now >= 0) {
            float mx[NT][2];
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int c = 0; c < 2; c++) mx[nt][c] = -INFINITY;
#pragma unroll
            for (int mt = 0; mt < MT; mt++)
#pragma unroll
                for (int nt = 0; nt < NT; nt++)
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        float x = s[mt][nt][e] * (kf[mt][e >> 1] * qf[nt][e & 1]);
                        if (cap) x = capped<SPLIT>(x, a.at.softcap, inv_cap2) * 1.4426950408889634f;
                        if (!whole) {
                            const int j = t0 + mt * 16 + (e >> 1) * 8 + row_position(g);
                            if (j < clo[nt][e & 1] || j > chi[nt][e & 1] || j >= len) x = -INFINITY;
                        }
                        s[mt][nt][e] = x;
                        mx[nt][e & 1] = fmaxf(mx[nt][e & 1], x);
                    }
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int c = 0; c < 2; c++) {
#pragma unroll
                    for (int d = 4; d < 32; d <<= 1) mx[nt][c] = fmaxf(mx[nt][c], __shfl_xor_sync(0xffffffffu, mx[nt][c], d));
                    mx[nt][c] = fmaxf(mx[nt][c], m[nt][c]);
                }
            cp_wait<1>();  // V and its scales
            __syncwarp();
            float vf[MT][2], vmax = 0.0f;
#pragma unroll
            for (int mt = 0; mt < MT; mt++)
#pragma unroll
                for (int hf = 0; hf < 2; hf++) {
                    const int j = mt * 16 + hf * 8 + row_position(g);
                    vf[mt][hf] = vsc[j] * code_unit<FMT>();
                    if (t0 + j < len) vmax = fmaxf(vmax, vf[mt][hf]);  // a NaN scale does not count
                }
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) vmax = fmaxf(vmax, __shfl_xor_sync(0xffffffffu, vmax, d));
            const float vp = fmaxf(vpow, scale_pow(vmax)), inv = pow_inverse(vp), ve = vpow * inv;
            vpow = vp;
            bool moved = ve != 1.0f;
            float f[NT][2], base[NT][2];
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int c = 0; c < 2; c++) {
                    base[nt][c] = mx[nt][c] == -INFINITY ? 0.0f : mx[nt][c];
                    f[nt][c] = ex2(m[nt][c] - base[nt][c]);  // nothing seen before: exp2(-inf) = 0
                    m[nt][c] = mx[nt][c];
                    l[nt][c] *= f[nt][c];
                    f[nt][c] *= ve;
                    moved = moved || f[nt][c] != 1.0f;
                }
            if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
                for (int nt = 0; nt < NT; nt++)
#pragma unroll
                    for (int j = 0; j < D / 16; j++)
#pragma unroll
                        for (int e = 0; e < 4; e++) o[nt][j][e] *= f[nt][e & 1];
            }
            // ---- P^T fragments: the S^T tile transposed
            uint32_t pb[NQ][MT][NT][2];
#pragma unroll
            for (int mt = 0; mt < MT; mt++) {
                const float w0 = vf[mt][0] * inv, w1 = vf[mt][1] * inv;
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
                    float p[4];
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const float x = s[mt][nt][e], y = ex2(x - base[nt][e & 1]);
                        l[nt][e & 1] += y;
                        p[e] = y * (e < 2 ? w0 : w1);
                        if (!whole && x == -INFINITY) p[e] = 0.0f;  // whatever the unseen position holds
                    }
#pragma unroll
                    for (int hf = 0; hf < 2; hf++) {
                        const uint32_t hi = pack(p[2 * hf], p[2 * hf + 1]);
                        pb[0][mt][nt][hf] = transpose8(hi);
                        if (SPLIT) {
                            const float2 back = __half22float2(*reinterpret_cast<const __half2 *>(&hi));
                            pb[NQ - 1][mt][nt][hf] = transpose8(pack(p[2 * hf] - back.x, p[2 * hf + 1] - back.y));
                        }
                    }
                }
            }
            // ---- O^T += V^T P^T
#pragma unroll
            for (int mt = 0; mt < MT; mt++)
#pragma unroll
                for (int c = 0; c < Sh::VC; c++) {
                    uint32_t w[4][Sh::VB / 4];
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const int r = mt * 16 + 4 * i + t, byte = (c * 8 + g) * Sh::VB;
                        lds<Sh::VB>(vslot + 16 * v_piece<D>(r, byte / 16) + byte % 16, w[i]);
                    }
#pragma unroll
                    for (int k = 0; k < Sh::VB / 4; k++) {
                        const uint32_t x0 = w[0][k] ^ code_flip<FMT>(), x1 = w[1][k] ^ code_flip<FMT>();
                        const uint32_t x2 = w[2][k] ^ code_flip<FMT>(), x3 = w[3][k] ^ code_flip<FMT>();
#pragma unroll
                        for (int hf = 0; hf < 2; hf++) {  // dimensions 0, 1 and 2, 3 of the four bytes
                            const uint32_t ab = __byte_perm(x0, x1, hf ? 0x7362 : 0x5140), cd = __byte_perm(x2, x3, hf ? 0x7362 : 0x5140);
                            const uint32_t fr[4] = {codes2<FMT, 0, 1>(ab), codes2<FMT, 2, 3>(ab), codes2<FMT, 0, 1>(cd),
                                                    codes2<FMT, 2, 3>(cd)};
                            const int j = (c * Sh::VB / 4 + k) * 2 + hf;
#pragma unroll
                            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                                for (int h = 0; h < NQ; h++) mma(o[nt][j], fr, pb[h][mt][nt][0], pb[h][mt][nt][1]);
                        }
                    }
                }
        } else {
            cp_wait<1>();
        }
        __syncwarp();
        fetch(at_next, true);
        at = at_next;
        at_next = after;
    }
    cp_wait<0>();
    __syncthreads();

    // ---- join the warps: sums over the lanes that share a row, then O through shared memory in
    // register order (one float4 of four consecutive dimensions per lane)
#pragma unroll
    for (int nt = 0; nt < NT; nt++)
#pragma unroll
        for (int c = 0; c < 2; c++) {
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) l[nt][c] += __shfl_xor_sync(0xffffffffu, l[nt][c], d);
            if (g == 0) {
                s_m[warp][nt * 8 + 2 * t + c] = m[nt][c];
                s_l[warp][nt * 8 + 2 * t + c] = l[nt][c];
            }
        }
    if (lane == 0) s_e[warp] = vpow;
    constexpr int PIECES = NT * 2 * (D / 32);  // float4 pieces of a lane: (nt, column, four dimensions)
    float4 *so = (float4 *)smem;               // [NW][PIECES][32]
#pragma unroll
    for (int nt = 0; nt < NT; nt++)
#pragma unroll
        for (int c = 0; c < 2; c++)
#pragma unroll
            for (int k = 0; k < D / 32; k++)
                so[(warp * PIECES + (nt * 2 + c) * (D / 32) + k) * 32 + lane] =
                    make_float4(o[nt][2 * k][c], o[nt][2 * k][2 + c], o[nt][2 * k + 1][c], o[nt][2 * k + 1][2 + c]);
    __syncthreads();
    const int64_t RH = (int64_t)a.bt.rows * a.at.heads, slot = sg.pre ? chunk : a.nsp + chunk;
    for (int pc = warp; pc < PIECES; pc += NW) {
        const int nc = pc / (D / 32), k = pc % (D / 32), n = (nc >> 1) * 8 + 2 * t + (nc & 1), row = s_row[n];
        if (row < 0) continue;
        float M = -INFINITY;
#pragma unroll
        for (int w = 0; w < NW; w++) M = fmaxf(M, s_m[w][n]);
        float L = 0.0f, x[4] = {};
#pragma unroll
        for (int w = 0; w < NW; w++) {
            if (s_m[w][n] == -INFINITY && !(s_l[w][n] != s_l[w][n])) continue;  // this warp saw nothing
            const float f = ex2(s_m[w][n] - M), fo = f * s_e[w];
            L = fmaf(s_l[w][n], f, L);
            const float4 v = so[(w * PIECES + pc) * 32 + lane];
            x[0] = fmaf(v.x, fo, x[0]);
            x[1] = fmaf(v.y, fo, x[1]);
            x[2] = fmaf(v.z, fo, x[2]);
            x[3] = fmaf(v.w, fo, x[3]);
        }
        const int head = kvh * G + (row_first + n) % G, word = k;  // four dimensions of this lane
        const int d = word / (Sh::VB / 4) * 8 * Sh::VB + g * Sh::VB + word % (Sh::VB / 4) * 4;
        if (a.direct) {
            const float inv = L == 0.0f ? 0.0f : 1.0f / L;
            float y[4];
#pragma unroll
            for (int e = 0; e < 4; e++) y[e] = L == 0.0f ? 0.0f : x[e] * inv;
            store4(a.out, row * a.ldo + (int64_t)head * D + d, a.at.type, a.wide != 0, y);
            if (a.lse && g == 0 && k == 0)
                a.lse[(int64_t)row * a.at.heads + head] = L == 0.0f ? -INFINITY : (M + log2f(L)) * 0.6931471805599453f;
        } else {
            const int64_t rh = (int64_t)row * a.at.heads + head;
            *(float4 *)(a.part_o + (slot * RH + rh) * D + d) = make_float4(x[0], x[1], x[2], x[3]);
            if (g == 0 && k == 0) a.part_ml[slot * RH + rh] = make_float2(M, L);
        }
    }
    if (a.chained) pdl_wait();
}

// Joins a row's partials: one warp per (row, head); the prefix's chunks, then the sequence's.
template <int D> __global__ void __launch_bounds__(128) kvq_join_kernel(const __grid_constant__ AttnArgs a)
{
    constexpr int N = D / 32;
    const int64_t item = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5), RH = (int64_t)a.bt.rows * a.at.heads;
    const int lane = threadIdx.x & 31;
    if (item >= RH) return;
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
    for (int s0 = 0; s0 < slots; s0 += 32) {
        float w = 0.0f;
        if (s0 + lane < slots) {
            const float2 v = __ldcg(ml + (s0 + lane) * RH);
            if (v.x != -INFINITY || v.y != v.y) {
                w = ex2(v.x - M);
                L = fmaf(v.y, w, L);
            }
        }
        const int n = min(32, slots - s0);
#pragma unroll 4
        for (int s = 0; s < n; s++) {
            const float f = __shfl_sync(0xffffffffu, w, s);
            if (f == 0.0f) continue;
            const float *p = a.part_o + ((s0 + s) * RH + item) * D + lane;
#pragma unroll
            for (int i = 0; i < N; i++) x[i] = fmaf(__ldcg(p + 32 * i), f, x[i]);
        }
    }
    L = warp_sum(L);
    const float inv = 1.0f / L;
#pragma unroll
    for (int i = 0; i < N; i++) {
        const float y = L == 0.0f ? 0.0f : x[i] * inv;
        const int64_t at = row * a.ldo + (int64_t)head * D + 32 * i + lane;
        if (a.at.type == T_F32) ((float *)a.out)[at] = y;
        else if (a.at.type == T_F16) ((__half *)a.out)[at] = __float2half_rn(y);
        else ((__nv_bfloat16 *)a.out)[at] = __float2bfloat16_rn(y);
    }
    if (a.lse && lane == 0) a.lse[item] = L == 0.0f ? -INFINITY : (M + log2f(L)) * 0.6931471805599453f;
}

// ------------------------------------------------------------------ launch
template <int D, int FMT, int NT, bool SPLIT> cudaError_t launch_tiles(const AttnArgs &a, int64_t grid, cudaStream_t st)
{
    using Sh = Shape<D>;
    static_assert(NW * Sh::WARP >= (2 * SEQ_TABLE + 1) * 4, "the sequences' tables fit into the slots");
    constexpr int smem = NW * Sh::WARP + (SPLIT ? 2 : 1) * NT * 8 * (D + Sh::QPAD) * 2;
    static_assert(NT * 8 * D * 4 <= Sh::WARP, "the warps' outputs fit into their slots");
    static std::atomic<unsigned long long> done{0};
    cudaError_t e = smem_attr_once(done, kvq_attn_kernel<D, FMT, NT, SPLIT>, smem);
    if (e != cudaSuccess) return e;
    return launch_kernel(a.chained != 0, kvq_attn_kernel<D, FMT, NT, SPLIT>, dim3((unsigned)grid), dim3(NW * 32), smem, st, a);
}
template <int D, int FMT, bool SPLIT> cudaError_t launch_nt(int nt, const AttnArgs &a, int64_t grid, cudaStream_t st)
{
    constexpr int MX = Shape<D>::MAX_NT;
    if (nt == 1) return launch_tiles<D, FMT, 1, SPLIT>(a, grid, st);
    if (nt == 2 || MX == 2) return launch_tiles<D, FMT, 2, SPLIT>(a, grid, st);
    if (nt == 3 || MX == 3) return launch_tiles<D, FMT, MX < 3 ? 2 : 3, SPLIT>(a, grid, st);
    return launch_tiles<D, FMT, MX < 4 ? 2 : 4, SPLIT>(a, grid, st);
}
template <int D> cudaError_t launch_dim(int nt, const AttnArgs &a, int64_t grid, cudaStream_t st)
{
    const bool split = a.at.type == T_F32;
    if (a.pool.format == LLMDOT_KVQ_I8)
        return split ? launch_nt<D, LLMDOT_KVQ_I8, true>(nt, a, grid, st) : launch_nt<D, LLMDOT_KVQ_I8, false>(nt, a, grid, st);
    return split ? launch_nt<D, LLMDOT_KVQ_E4M3, true>(nt, a, grid, st) : launch_nt<D, LLMDOT_KVQ_E4M3, false>(nt, a, grid, st);
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
cudaError_t launch_join(const AttnArgs &a, cudaStream_t st)
{
    const dim3 grid((unsigned)(((int64_t)a.bt.rows * a.at.heads + 3) / 4)), block(128);
    switch (a.pool.head_dim) {
    case 64: return launch_kernel(true, kvq_join_kernel<64>, grid, block, 0, st, a);
    case 96: return launch_kernel(true, kvq_join_kernel<96>, grid, block, 0, st, a);
    case 128: return launch_kernel(true, kvq_join_kernel<128>, grid, block, 0, st, a);
    default: return launch_kernel(true, kvq_join_kernel<256>, grid, block, 0, st, a);
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
int max_nt(int dim) { return dim == 256 ? 2 : dim == 128 ? 3 : 4; }
// From this many rows (times heads) per kv head a segment is worth the wide kernel.
constexpr int64_t WIDE_FROM = 48;

Plan make_plan(const llmdot_kvq_pool &p, const llmdot_kvq_batch &b, const llmdot_kvq_attn &a)
{
    Plan x = {};
    const int64_t G = a.heads / p.heads_kv, Hk = p.heads_kv, own_rows = (int64_t)b.max_rows * G, all_rows = (int64_t)b.rows * G;
    const int64_t npp = (a.prefix_len + KVQ_PAGE - 1) / KVQ_PAGE, wide = kvq_wide_rows(p.head_dim);
    auto nt_of = [&](int64_t rows) { return (int)std::min<int64_t>(max_nt(p.head_dim), std::max<int64_t>(1, (rows + 7) / 8)); };
    auto up = [](int64_t x, int64_t y) { return (x + y - 1) / y; };
    x.wide_p = a.type != T_F32 && npp > 0 && all_rows >= WIDE_FROM;
    x.wide_s = a.type != T_F32 && own_rows >= WIDE_FROM;
    x.nt_p = nt_of(all_rows);
    x.nt_s = nt_of(own_rows);
    if (npp == 0) x.nt_p = x.nt_s;
    x.ptiles = (int)up(all_rows, x.wide_p ? wide : 8 * x.nt_p);
    x.rtiles = (int)std::max<int64_t>(1, up(own_rows, x.wide_s ? wide : 8 * x.nt_s));
    // Chunks.  Narrow: enough CTAs to fill the SMs about four times (ragged sequences leave some without
    // work), at least one page per warp, at most 32 pages, so that long and short sequences balance.
    // Wide: one CTA per SM, at least four pages each.
    const int64_t np = x.wide_p ? 0 : Hk * x.ptiles * npp, ns = x.wide_s ? 0 : Hk * b.batch * x.rtiles * b.max_pages;
    const int64_t ch = std::min<int64_t>(32, std::max<int64_t>(NW, up(up(np + ns, 148 * 4), NW) * NW));
    auto wide_ch = [&](int64_t ctas, int64_t pages) { return std::max<int64_t>(4, up(pages, std::max<int64_t>(1, 148 / std::max<int64_t>(1, ctas)))); };
    x.ch_p = (int)(x.wide_p ? wide_ch(Hk * x.ptiles, npp) : ch);
    x.ch_s = (int)(x.wide_s ? wide_ch(Hk * x.rtiles * b.batch, b.max_pages) : ch);
    x.nsp = (int)up(npp, x.ch_p);
    x.nss = (int)std::max<int64_t>(1, up(b.max_pages, x.ch_s));
    x.direct = x.nsp == 0 && x.nss == 1 && !x.wide_s;
    x.ctas_p = Hk * x.ptiles * x.nsp;
    x.ctas_s = Hk * x.rtiles * x.nss * b.batch;
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
