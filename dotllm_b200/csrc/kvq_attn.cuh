// kvq_attn.cuh -- what the kernels of the shared-prefix attention have in common: the cut of a call into
// segments, row tiles and chunks, the rows' visible ranges, and small arithmetic.
#pragma once
#include "kvq.cuh"

namespace llmdot {

struct AttnArgs {
    llmdot_kvq_pool pool;
    llmdot_kvq_batch bt;
    llmdot_kvq_attn at;
    const void *q;
    void *out;
    int64_t ldq, ldo;
    float *lse;
    float *part_o;     // [slots][rows * heads][D]
    float2 *part_ml;   // [slots][rows * heads]: reference (base 2), sum of the exponentials
    int group;         // query heads per kv head
    int ch_p, ch_s;    // pages per chunk: prefix, own pages
    int nsp, nss;      // chunks of the prefix; most chunks of a sequence
    int ptiles, rtiles;  // row tiles of the launch: prefix, own pages
    int prefix_ctas;   // the launch's first CTAs, which attend the prefix
    int direct;        // one slot: write the output itself
    int wide;          // the output's rows are 16-byte aligned
    int chained;       // launched over a kernel that still runs: end only after it
};

// Scores of many rows over one segment on the 5th-generation tensor cores (kvq_attn_tc.cu): 16-bit
// queries, partials only.  Rows per CTA:
int kvq_wide_rows(int head_dim);
cudaError_t launch_kvq_wide(const AttnArgs &a, int64_t ctas, bool pdl, cudaStream_t st);

// One CTA's share of a call.
struct Segment {
    bool pre;
    int kvh, tile, chunk;
    int r0, nrows;   // first packed row, rows
    int own, n_all;  // the sequence's positions and rows (own segments)
    int len;         // positions of the segment
    int ch;          // pages per chunk
    const int32_t *pages;
};
// False when the CTA has nothing to do.  rows: rows (times heads) of a row tile.
__device__ __forceinline__ bool segment_of(const AttnArgs &a, int rows, Segment &s)
{
    const int Hk = a.pool.heads_kv;
    s.pre = (int)blockIdx.x < a.prefix_ctas;
    int rest = s.pre ? blockIdx.x : blockIdx.x - a.prefix_ctas;
    s.kvh = rest % Hk;
    rest /= Hk;
    const int tiles = s.pre ? a.ptiles : a.rtiles;
    s.tile = rest % tiles;
    rest /= tiles;
    s.own = s.n_all = s.r0 = 0;
    if (s.pre) {
        s.chunk = rest;
        s.nrows = a.bt.rows;
        s.len = a.at.prefix_len;
        s.pages = a.at.prefix_pages;
        s.ch = a.ch_p;
    } else {
        s.chunk = rest % a.nss;
        const int b = rest / a.nss;
        s.r0 = a.bt.row_start[b];
        s.n_all = a.bt.row_start[b + 1] - s.r0;
        s.nrows = min(min(s.n_all, a.bt.max_rows), a.bt.rows - s.r0);
        s.own = a.bt.seq_len[b];
        s.len = (int)min((int64_t)s.own, (int64_t)a.bt.max_pages * KVQ_PAGE);
        s.pages = a.bt.pages + (int64_t)b * a.bt.max_pages;
        s.ch = a.ch_s;
        if (s.r0 < 0) return false;
    }
    if ((int64_t)s.tile * rows >= (int64_t)s.nrows * a.group) return false;
    // the joining kernel does not look for a chunk that begins behind the end
    return a.direct || s.chunk * s.ch * KVQ_PAGE < s.len;
}
// row_start and seq_len of the batch, in shared memory when they fit: a row's search for its sequence is
// a chain of dependent loads, half a microsecond each from global memory.
struct SeqTable {
    const int32_t *row_start, *seq_len;
};
constexpr int SEQ_TABLE = 448;  // sequences
// Called by all threads; `room`: 2 * SEQ_TABLE + 1 ints of shared memory.  The prefix's rows need it alone.
__device__ __forceinline__ SeqTable load_seqs(const AttnArgs &a, const Segment &s, int32_t *room, int threads)
{
    SeqTable t = {a.bt.row_start, a.bt.seq_len};
    if (!s.pre || a.bt.batch > SEQ_TABLE) return t;
    for (int i = threadIdx.x; i <= a.bt.batch; i += threads) {
        room[i] = a.bt.row_start[i];
        if (i < a.bt.batch) room[SEQ_TABLE + 1 + i] = a.bt.seq_len[i];
    }
    __syncthreads();
    t.row_start = room;
    t.seq_len = room + SEQ_TABLE + 1;
    return t;
}
// Row rho (of rows times the group's heads): its packed row (-1: none) and visible positions [lo, hi].
// Rows that do not exist see everything, so that they hide nothing.
__device__ __forceinline__ void row_range(const AttnArgs &a, const Segment &s, const SeqTable &q, uint32_t rho, int &row, int &lo, int &hi)
{
    row = -1;
    lo = 0;
    hi = 0x7fffffff;
    if (rho >= (uint32_t)s.nrows * a.group) return;  // rows * heads fits 2^30
    const int i = rho / (uint32_t)a.group, win = a.at.window;
    row = s.r0 + i;
    int64_t pos = (int64_t)s.own - s.n_all + i;  // in the segment's positions
    if (s.pre) {
        const int b = kvq_seq_of(q.row_start, a.bt.batch, row);
        pos = b >= 0 ? (int64_t)a.at.prefix_len + q.seq_len[b] - q.row_start[b + 1] + row : -1;
    }
    hi = pos < 0 ? -1 : (int)min(pos, (int64_t)s.len - 1);
    if (win > 0) lo = (int)max((int64_t)0, min(pos - win + 1, (int64_t)0x7fffffff));
}

__device__ __forceinline__ float ex2(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float rcp(float x)
{
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// cap * tanh(s / cap).  16-bit activations: 1 - 2 / (1 + e^{2x}), a few 1e-7 of the cap off, which
// the hardware's own tanh (2^-11) would not reach; fp32 ones: tanhf, exact to the last places of s.
template <bool FULL> __device__ __forceinline__ float capped(float s, float cap, float inv_cap2)
{
    if (FULL) return cap * tanhf(s * (inv_cap2 * 0.34657359027997264f));
    return cap - 2.0f * cap * rcp(1.0f + ex2(s * inv_cap2));
}
__device__ __forceinline__ uint32_t pack(float lo, float hi)
{
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ uint32_t hadd2(uint32_t a, uint32_t b)
{
    uint32_t d;
    asm("add.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
}
__device__ __forceinline__ uint32_t hsub2(uint32_t a, uint32_t b)
{
    uint32_t d;
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
}

// Two codes, bytes LO and HI of x, as an fp16 pair.  int8 (x with its sign bits flipped): the byte
// under the exponent of 1024, minus 1152.  e4m3: sign, exponent and mantissa moved into fp16's places,
// the value times 2^-8 (which the scale makes good), subnormals included.
template <int FMT, int LO, int HI> __device__ __forceinline__ uint32_t codes2(uint32_t x)
{
    if (FMT == LLMDOT_KVQ_I8) return hsub2(__byte_perm(x, 0x64646464u, LO | 0x40 | (HI << 8) | 0x4000), 0x64806480u);
    const uint32_t v = __byte_perm(x, 0u, 0x4 | (LO << 4) | 0x400 | (HI << 12));
    return (v & 0x80008000u) | ((v >> 1) & 0x3F803F80u);
}
template <int FMT> constexpr uint32_t code_flip() { return FMT == LLMDOT_KVQ_I8 ? 0x80808080u : 0u; }
template <int FMT> constexpr float code_unit() { return FMT == LLMDOT_KVQ_I8 ? 1.0f : 256.0f; }

// Exponent that brings a row's largest magnitude into [2^14, 2^15); 0 for zero and non-finite rows.
__device__ __forceinline__ int row_exponent(float top)
{
    const int b = __float_as_int(top);
    return b > 0 && b < 0x7f800000 ? min(14 + 127 - (b >> 23), 126) : 0;
}
__device__ __forceinline__ float pow2(int e) { return __int_as_float((e + 127) << 23); }
__device__ __forceinline__ float pow_inverse(float p) { return __int_as_float(0x7f000000 - __float_as_int(p)); }  // p a power of two
__device__ __forceinline__ int pow_exponent(float p) { return (__float_as_int(p) >> 23) - 127; }
__device__ __forceinline__ float log2_abs(float x)  // -infinity for 0 and subnormal numbers
{
    float y;
    asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(fabsf(x)));
    return y;
}

// A row's two references.  Its exponentials are exp2(s - ref); its weights those times the values' scales times `unit`,
// a power of two, as fp16.  When they are set, `ref` is the row's maximum and `unit` brings its largest weight into
// (2^3, 2^4], so that weights of 2^-17 of the largest are still normal numbers (the lo of a hi + lo pair, those of 2^-6).
// They are set again where a weight has reached 2^8, which a lane notices when its at most 32 packed weights sum to 2^13
// (an addition of two halves costs less than a test, and an infinity or NaN stays one), or when the exponentials grow
// without their values (scales of nearly 0) and their sum reaches SUM_LIMIT.
constexpr float REF_HEAD = 4.0f, REF_LIMIT = 8.0f;
constexpr float SUM_LIMIT = 18446744073709551616.0f, SUM_LIMIT_LOG = 64.0f;
// Whether either half of such a sum is 2^13 or more, infinite or NaN, or negative (by a negative scale).
__device__ __forceinline__ bool too_large(uint32_t p) { return (((p & 0x70007000u) + 0x10001000u) | p) & 0x80008000u; }
// top: the largest score (base 2) that the row sees in a page; topv: with the logs of the values' scales.  False where the
// references hold for them; else they rise, and fl and fo are the (exact) factors for what was summed before: the
// exponentials, and the products.  The margins keep the logs' rounding from leaving a weight past the limit unanswered.
__device__ __forceinline__ bool raise_refs(float top, float topv, float &ref, float &unit, float &fl, float &fo)
{
    if (top == -INFINITY) return false;
    const bool first = ref == -INFINITY;
    const float E = -pow_exponent(unit);
    if (!first && topv - ref - E < REF_LIMIT - 0.01f && top - ref < SUM_LIMIT_LOG - 7.0f) return false;
    const float d = first ? 0.0f : ceilf(fmaxf(top - ref, 0.0f)), to = first ? top : ref + d;
    const float least = fminf(fmaxf(ceilf(topv - to) - REF_HEAD, -126.0f), 126.0f), Eo = first ? least : fmaxf(E - d, least);
    fl = d > 126.0f ? 0.0f : pow2(-(int)d);  // (both 1 for a row that has summed nothing)
    fo = first || Eo - E + d > 126.0f ? (float)first : pow2((int)(E - d - Eo));
    ref = to;
    unit = __int_as_float((127 - (int)Eo) << 23);
    return true;
}

__device__ __forceinline__ float load_any(const void *p, int64_t i, uint32_t type)
{
    if (type == T_F32) return __ldg((const float *)p + i);
    if (type == T_F16) return __half2float(__ldg((const __half *)p + i));
    return __bfloat162float(__ldg((const __nv_bfloat16 *)p + i));
}

}  // namespace llmdot
