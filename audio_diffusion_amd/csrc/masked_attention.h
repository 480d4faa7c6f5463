// Shared parts of the masked attention kernels (masked_attention_fwd.inc, _step.inc, _bwd.inc): the mask of a query row as a key
// limit and a document, the score transform, LDS tiles of keys (or query rows) and their fragments.
//
// All kernels keep ONE index of a score tile on the lane: a 32 x 32 tile of S^T = K Q^T (or S = Q K^T) comes out of
// v_mfma_f32_32x32x16 with column = lane & 31 and rows (r & 3) + 8 (r >> 2) + 4 (lane >> 5), r = 0..15, and those 16 registers,
// rounded to 16 bits, are the B operand of the next product as they stand: neither scores nor probabilities touch LDS.
#pragma once
#include "adk_common.h"
#include <stddef.h>
#include <string.h>
#include <cmath>

// adk_attention_args as the kernels take it: without its last member, o_low, which only some of them use and get beside it.  (The second backward
// kernel at D = 64 with bias fills its registers to the last one; 8 bytes more of arguments made hipcc spill in its loop.)
struct AttArgs {
    int32_t dtype, B, Nq, Nk, Hq, Hk, D, causal;
    float scale, softcap;
    const void *q, *k, *v;
    int64_t q_stride_b, q_stride_n, q_stride_h, k_stride_b, k_stride_n, k_stride_h, v_stride_b, v_stride_n, v_stride_h;
    const float* slopes;
    const int32_t *prefix, *lengths, *starts, *documents;
    int64_t documents_stride;
    void* o;
    float* lse;
    const void* o_grad;
    int64_t og_stride_b, og_stride_n, og_stride_h;
    void *q_grad, *k_grad, *v_grad;
};
static_assert(sizeof(AttArgs) == offsetof(adk_attention_args, o_low) && offsetof(AttArgs, v_stride_h) == offsetof(adk_attention_args, v_stride_h)
              && offsetof(AttArgs, documents) == offsetof(adk_attention_args, documents) && offsetof(AttArgs, lse) == offsetof(adk_attention_args, lse)
              && offsetof(AttArgs, v_grad) == offsetof(adk_attention_args, v_grad), "the same members in the same places");
static inline AttArgs att_args_of(const adk_attention_args& a)
{
    AttArgs k;
    memcpy(&k, &a, sizeof k);
    return k;
}
typedef __attribute__((ext_vector_type(4))) short att_s16x4;

constexpr int AT_KT = 64;                    // keys of one LDS tile, and of one entry of the document ranges
constexpr float AT_LOG2E = 1.44269504088896340736f;

template <typename T> struct SeqMma;
template <> struct SeqMma<bf16_t> {
    typedef bf16x8 Frag;
    static __device__ __forceinline__ f32x16 run(const Frag& a, const Frag& b, const f32x16& c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
};
template <> struct SeqMma<f16_t> {
    typedef f16x8 Frag;
    static __device__ __forceinline__ f32x16 run(const Frag& a, const Frag& b, const f32x16& c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
};

__device__ __forceinline__ f32x16 at_zero16()
{
    f32x16 z;
#pragma unroll
    for (int r = 0; r < 16; ++r) z[r] = 0.f;
    return z;
}
// row of register r of a 32 x 32 tile, less the lane half's 4 h
__device__ __forceinline__ constexpr int at_row(int r) { return (r & 3) + 8 * (r >> 2); }

__device__ __forceinline__ float at_xhalf_max(float x)
{
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float at_xhalf_sum(float x)
{
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// ---- masks ---------------------------------------------------------------------------------------------------------------
// Causal, prefix and length masks together are one limit per row: key j is seen if j <= lim.  lim grows with the row, so
// the first and last row of a tile bound it.  Documents are an equality on top; a row without one gets the limit -1.
struct AtSample { int klen, start, prefix; };

__device__ __forceinline__ AtSample at_sample(const AttArgs& a, int b)
{
    AtSample s;
    s.klen = a.lengths ? min(max(a.lengths[b], 0), a.Nk) : a.Nk;
    s.start = a.starts ? min(max(a.starts[b], -(1 << 29)), 1 << 29) : a.Nk - a.Nq;
    s.prefix = a.prefix ? max(a.prefix[b], 0) : 0;
    return s;
}
__device__ __forceinline__ int at_limit(const AttArgs& a, const AtSample& s, int i)
{
    return a.causal ? min(s.klen - 1, max(s.start + i, s.prefix - 1)) : s.klen - 1;
}
// The position a distance is taken from: outside the keys the distances differ from those of the nearest end by a constant
// of the row, which the softmax does not see.  Whole numbers: their difference is rounded to f32, not they (behind key 2^24 f32 skips keys).
__device__ __forceinline__ int at_bias_pos(const AttArgs& a, const AtSample& s, int i) { return min(max(s.start + i, 0), a.Nk - 1); }
// The bias -slope |pos - j| of a tile of 64 keys from k0 is side * (j - pos) where all keys stand on one side of the positions first .. last
// (0: they do not, or there is no bias).
__device__ __forceinline__ float at_side(float slope, int k0, int first, int last)
{
    return k0 + AT_KT - 1 <= first ? slope : k0 >= last ? -slope : 0.f;
}
__device__ __forceinline__ int at_row_doc(const AttArgs& a, const AtSample& s, int b, int i)       // negative: none
{
    const int p = s.start + i;
    if (p < 0 || p >= a.Nk) return -1;
    return a.documents[(long long)b * a.documents_stride + p];
}
// smallest and largest document of the rows that have one (empty: lo > hi), over all 64 lanes; and whether all 64 have it
struct AtDocs { int lo, hi; bool one; };
__device__ __forceinline__ AtDocs at_doc_range(int doc)
{
    AtDocs d;
    d.lo = doc < 0 ? 0x7fffffff : doc;
    d.hi = doc < 0 ? -1 : doc;
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) {
        d.lo = min(d.lo, __shfl_xor(d.lo, m, 64));
        d.hi = max(d.hi, __shfl_xor(d.hi, m, 64));
    }
    d.lo = __builtin_amdgcn_readfirstlane(d.lo);
    d.hi = __builtin_amdgcn_readfirstlane(d.hi);
    d.one = __ballot(doc != d.lo) == 0ull;
    return d;
}
// [lo, hi] of documents; entry t of the ranges of the 64-key tiles by a scalar load (t is wave-uniform)
struct AtRange { int lo, hi; };
__device__ __forceinline__ AtRange at_range(const int* ranges, int t)
{
    const auto* p = (const __attribute__((address_space(4))) int*)(ranges + 2 * (long long)t);
    return {p[0], p[1]};
}
__device__ __forceinline__ bool at_meet(const AtRange& r, int lo, int hi) { return r.lo <= hi && r.hi >= lo; }

// ---- scores --------------------------------------------------------------------------------------------------------------
// base-2 scores: x = score * log2(e).  Plain (CAP = 0): x = qk * c.  Capped: c tanh(t), t = qk * scale / cap, in two forms.
//   CAP = 1, caps up to AT_NEAR_CAP: cap - 2 cap / (exp(2 t) + 1).  Its error is that of a difference of numbers as large as the cap: the
//   exponential and the reciprocal are off by a step of 2^-23, the sums by half of one, 2.4e-7 cap of the score together, 3e-5 at most here.
//   CAP = 2, larger caps: where |t| < 0.35 the Taylor series of tanh (to t^11; the next term is 1.2e-8 of the first), which multiplies the
//   score and has an error relative to it; elsewhere the same difference, there 2.4e-7 cap < 7e-7 |score|.
//   The second form has kernels of its own, since it takes longer (2 x 16 heads on 4 of 8192 x 8192 at D = 128, causal, bf16: forward 655 -> 1053 us,
//   backward 2158 -> 2778).
// Caps whose factors leave the range of f32 are refused (at_scores_finite).
struct AtScore { float c, k1, capl2, t; };   // scale * log2 e;  2 log2 e scale / cap;  cap * log2 e;  scale / cap

constexpr float AT_NEAR_CAP = 128.f;
static inline int at_cap_of(const AttArgs& a) { return a.softcap == 0.f ? 0 : a.softcap <= AT_NEAR_CAP ? 1 : 2; }
static inline AtScore at_score_of(const AttArgs& a)
{
    AtScore s;
    s.c = a.scale * AT_LOG2E;
    s.k1 = a.softcap > 0.f ? 2.f * AT_LOG2E * (a.scale / a.softcap) : 0.f;
    s.capl2 = a.softcap * AT_LOG2E;
    s.t = a.softcap > 0.f ? a.scale / a.softcap : 0.f;
    return s;
}
static inline bool at_scores_finite(const AttArgs& a)
{
    const AtScore s = at_score_of(a);
    return std::isfinite(s.c) && std::isfinite(s.k1) && std::isfinite(2.f * s.capl2);
}
__device__ __forceinline__ float at_tanh(float qk, float k1)
{
    return 1.f - 2.f * __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(qk * k1) + 1.f);
}
// tanh(t) / t for |t| < 0.35
__device__ __forceinline__ float at_tanh_series(float t)
{
    const float u = t * t;
    float p = __builtin_fmaf(u, -1382.f / 155925.f, 62.f / 2835.f);
    p = __builtin_fmaf(u, p, -17.f / 315.f);
    p = __builtin_fmaf(u, p, 2.f / 15.f);
    p = __builtin_fmaf(u, p, -1.f / 3.f);
    return __builtin_fmaf(u, p, 1.f);
}
// a score less y, and the tanh for its derivative
template <int CAP> __device__ __forceinline__ float at_score(const AtScore& sc, float qk, float y, float& th)
{
    if constexpr (CAP == 0) {
        th = 0.f;
        return __builtin_fmaf(qk, sc.c, -y);
    } else if constexpr (CAP == 1) {
        th = at_tanh(qk, sc.k1);
        return __builtin_fmaf(th, sc.capl2, -y);
    } else {
        const float t = qk * sc.t, p = at_tanh_series(t), far = at_tanh(qk, sc.k1);
        const bool near = fabsf(t) < 0.35f;
        th = near ? t * p : far;
        return __builtin_fmaf(near ? qk * sc.c : sc.capl2, near ? p : far, -y);
    }
}
// the capped score alone: in the first form cap tanh as one multiply-add of the reciprocal
template <int CAP> __device__ __forceinline__ float at_capped(float qk, const AtScore& sc)
{
    if constexpr (CAP == 1) return __builtin_fmaf(-2.f * sc.capl2, __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(qk * sc.k1) + 1.f), sc.capl2);
    float th;
    return at_score<CAP>(sc, qk, 0.f, th);
}

// The running maximum of the forward kernels is kept this much lower, so that a probability is at most 2^(8 + this) before it is rounded (8: see
// masked_attention_fwd.inc).  f16 ends at 2^16 and has its smallest step at 2^-24: taken relative to the maximum itself, the keys of a long row that
// hold 2^-25 each are counted in the sum and lost in the product (65536 of them: 0.2 % of the row).  bf16 has f32's range.
template <typename T> __device__ __forceinline__ constexpr float at_raised() { return 0.f; }
template <> __device__ __forceinline__ constexpr float at_raised<f16_t>() { return 7.f; }

// ---- LDS tiles -----------------------------------------------------------------------------------------------------------
// A tile is [rows][D] 16-bit, rows of 2 D bytes, filled by LDS-DMA (1 KiB per wave instruction, lane l at + 16 l).  Piece p
// (16 bytes) of row r sits in slot p ^ swz(r): reading one piece of 8 consecutive rows (row fragments) and 4 pieces of
// 4 consecutive rows (transposed fragments) then both cover the banks evenly.
template <int D> __device__ __forceinline__ int at_swz(int row)
{
    constexpr int hi_shift = D == 128 ? 0 : D == 64 ? 1 : 2;
    const int hi = (row >> hi_shift) & (D / 32 - 1), lo = (row >> 2) & 3;
    return (hi << 2) | lo;
}
// The DMA instructions are written out: hipcc orders every later LDS read it cannot tell apart behind the builtin's transfers
// (an s_waitcnt vmcnt(0) in front of the transposed reads of the CURRENT tile, which waited for the next one), and does not put
// that wait in front of a barrier, where it belongs.  at_landed() is that wait: every wave calls it in front of the barrier after
// which the tile is read.  The statements have no register results, so nothing can be reused under a transfer in flight.
// Program order of memory accesses, no instruction.  (Not an empty asm statement: hipcc counts every asm statement as a wait state behind a
// matrix instruction, whatever it holds; statements below that only pin a value therefore hold an s_nop.)
__device__ __forceinline__ void at_order() { __atomic_signal_fence(__ATOMIC_SEQ_CST); }
__device__ __forceinline__ void at_scalars() { asm volatile("s_nop 4" ::: "memory"); }
__device__ __forceinline__ uint32_t at_lds_addr(const unsigned char* lds) { return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) unsigned char*)lds; }
template <int PLUS> __device__ __forceinline__ void at_dma16(const unsigned char* base, uint32_t offset, uint32_t lds)  // lane l: 16 bytes of base + offset to lds + PLUS + 16 l
{
    asm volatile("s_add_u32 m0, %0, %3\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" :: "s"(lds), "v"(offset), "s"(base), "i"(PLUS) : "memory", "scc");
}
__device__ __forceinline__ void at_dma4(const void* src, uint32_t lds)             // lane l: 4 bytes to lds + 4 l
{
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" :: "s"(lds), "v"(src) : "memory");
}
// (The builtin, not asm: hipcc then knows that its own loads in front of the loop have landed too, and puts no wait for them
// into the loop, where it would also wait for the tile in flight.)
template <int YOUNGER = 0> __device__ __forceinline__ void at_landed()      // all but the YOUNGER last requests
{
    at_order();
    __builtin_amdgcn_s_waitcnt((YOUNGER & 15) | ((YOUNGER >> 4) << 14) | 0x0f70);        // vmcnt; the other counters as they are
    at_order();
}
// A barrier that orders LDS accesses in the program but waits for none of them (reads are consumed before their buffer is
// asked for again, and DMA has its own wait).
__device__ __forceinline__ void at_barrier()
{
    at_order();
    __builtin_amdgcn_s_barrier();
    at_order();
}
// Loads of 64-row tiles of two tensors x and y (K and V, or Q and dO), one tile behind the other in LDS.  Wave `wave` of NW issues
// its share, the same number of instructions as every other, all of one tensor.  The 64-bit part of an address (first row of the
// tile) is scalar and moves with the walk; a lane keeps the 32-bit offsets of its rows in the tile (64 rows of a 2^24-element stride at
// most).  Scalar instructions take their turn in a wave's stream like any other: an address worked out afresh cost about 100 cycles per
// request, as much as three products.
template <int D, int NW> struct AtPair {
    static constexpr int PPR = D / 8, RPI = 64 / PPR, NI = 64 / RPI, PER = 2 * NI / NW;  // pieces per row, rows per instruction
    static_assert(2 * NI % NW == 0 && NI % PER == 0, "a wave's share lies in one tile");
    const unsigned char* at;         // first row of the tile to ask for
    long long step;                  // bytes of 64 rows
    uint32_t stride, off[PER], lds;  // bytes of a row; per lane; the wave's part of a stage
    int wave, lane;
    __device__ __forceinline__ AtPair(const void* x, long long xs, const void* y, long long ys, uint32_t lds0, int wave_, int lane_) : wave(wave_), lane(lane_)
    {
        const bool second = wave * PER >= NI;
        at = reinterpret_cast<const unsigned char*>(second ? y : x);
        stride = (uint32_t)(second ? ys : xs) * 2;
        step = (second ? ys : xs) * 128;
        lds = lds0 + wave * PER * 1024;
#pragma unroll
        for (int t = 0; t < PER; ++t) off[t] = (uint32_t)row(t) * stride + piece(t);
    }
    __device__ __forceinline__ int row(int t) const { return ((wave * PER + t) % NI) * RPI + lane / PPR; }
    __device__ __forceinline__ uint32_t piece(int t) const { return ((lane % PPR) ^ at_swz<D>(row(t))) * 16; }
    __device__ __forceinline__ void move(int tiles) { at += tiles * step; }
    // the tile at hand holds rows 0 .. left of the tensor's last: rows past them repeat it.  Only ever the last tile of a walk.
    __device__ __forceinline__ void clip(int left)
    {
        if (left < 63) {
#pragma unroll
            for (int t = 0; t < PER; ++t) off[t] = (uint32_t)min(row(t), left) * stride + piece(t);
        }
    }
    // request I of PER into the stage at byte `stage`
    template <int I> __device__ __forceinline__ void part(uint32_t stage) const
    {
        if constexpr (I < PER) at_dma16<I * 1024>(at, off[I], lds + stage);
    }
    // the same by a number that is known once its loop is unrolled
    __device__ __forceinline__ void ask(int i, uint32_t stage) const
    {
        switch (i) {
        case 0: return part<0>(stage); case 1: return part<1>(stage); case 2: return part<2>(stage); case 3: return part<3>(stage);
        case 4: return part<4>(stage); case 5: return part<5>(stage); case 6: return part<6>(stage); default: return part<7>(stage);
        }
    }
    __device__ __forceinline__ void load(uint32_t stage) const
    {
        at_scalars();
        part<0>(stage); part<1>(stage); part<2>(stage); part<3>(stage);
        part<4>(stage); part<5>(stage); part<6>(stage); part<7>(stage);
    }
};
// Row fragment (A or B operand, contraction over d): lane (row = lane & 31, h) gets elements 16 ks + 8 h .. + 7 of row
// row0 + (lane & 31).  `addr` = at_row_addr(lane), kept by the caller.
template <int D> __device__ __forceinline__ int at_row_addr(int lane) { const int r = lane & 31; return r * 2 * D + (((lane >> 5) ^ at_swz<D>(r)) << 4); }
template <int D, typename Frag> __device__ __forceinline__ Frag at_row_frag(const unsigned char* tile, int addr, int row0, int ks)
{
    return *reinterpret_cast<const Frag*>(tile + row0 * 2 * D + (addr ^ (ks << 5)));     // row0 a multiple of 32
}
// Transposed fragment (A operand X^T, contraction over the tile's rows): lane (d = 32 dt + (lane & 31), h) gets rows
// row0 + 16 s + {4 h + 0..3, 8 + 4 h + 0..3}: the order in which the score registers 8 s .. 8 s + 7 hold them.
template <int D> __device__ __forceinline__ int at_tr_addr(int lane, int u)
{
    const int r = 8 * u + 4 * (lane >> 5) + ((lane & 15) >> 2);
    const int piece = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
    return r * 2 * D + ((piece ^ at_swz<D>(r)) << 4) + (lane & 1) * 8;
}
template <int D, typename Frag> union AtTr { att_s16x4 v[2]; Frag f; };
// its half u, for reads that are spread out one by one
template <int D> __device__ __forceinline__ att_s16x4 at_tr_half(const unsigned char* tile, const int (&addr)[2], int row0, int s, int dt, int u)
{
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (__attribute__((address_space(3))) att_s16x4*)(tile + (row0 + 16 * s) * 2 * D + (addr[u] ^ (dt << 6))));
}
template <int D, typename Frag> __device__ __forceinline__ Frag at_tr_frag(const unsigned char* tile, const int (&addr)[2], int row0, int s, int dt)
{
    AtTr<D, Frag> cv;
#pragma unroll
    for (int u = 0; u < 2; ++u) cv.v[u] = at_tr_half<D>(tile, addr, row0, s, dt, u);
    return cv.f;
}

// NM products with NR other instructions (LDS reads, mostly) spread between them, in exactly this order: an LDS instruction takes its
// 16 or so cycles to issue while the matrix unit works on the product in front of it.  Issued in a bunch they leave it idle.
template <int NM, int NR, typename F, typename R> __device__ __forceinline__ void at_weave(F product, R other)
{
#pragma unroll
    for (int x = 0; x < NM; ++x) {
        product(x);
#pragma unroll
        for (int r = x * NR / NM; r < (x + 1) * NR / NM; ++r) other(r);
        __builtin_amdgcn_sched_barrier(0);
    }
}

// 16 f32 -> two B operands (registers 0..7, 8..15)
template <typename T> __device__ __forceinline__ void at_pack(const f32x16& p, typename SeqMma<T>::Frag (&f)[2])
{
#pragma unroll
    for (int s = 0; s < 2; ++s) {
        union { uint32_t w[4]; typename SeqMma<T>::Frag f; } cv;
#pragma unroll
        for (int e = 0; e < 4; ++e) cv.w[e] = pack2v(f32x2{p[8 * s + 2 * e], p[8 * s + 2 * e + 1]}, T());
        f[s] = cv.f;
    }
}

// Four elements of a result row from element `at` on, and, where the call wants it (low), what their rounding lost (nothing where they are not finite)
template <typename T> __device__ __forceinline__ void at_store_o(void* o, void* low, long long at, float x0, float x1, float x2, float x3)
{
    uint2 w;
    w.x = pack2v(f32x2{x0, x1}, T());
    w.y = pack2v(f32x2{x2, x3}, T());
    *reinterpret_cast<uint2*>(reinterpret_cast<T*>(o) + at) = w;
    if (low) {
        const f32x2 p = unpack2(w.x, T()), q = unpack2(w.y, T());
        auto lost = [](float x, float r) { const float l = x - r; return l * 0.f == 0.f ? l : 0.f; };
        w.x = pack2v(f32x2{lost(x0, p.x), lost(x1, p.y)}, T());
        w.y = pack2v(f32x2{lost(x2, q.x), lost(x3, q.y)}, T());
        *reinterpret_cast<uint2*>(reinterpret_cast<T*>(low) + at) = w;
    }
}

// ---- the key tiles that a block of query rows walks (forward and dQ) -----------------------------------------------------------
// First and last tile that any row of the block sees, found by all threads over the ranges of documents; tiles between them
// that miss the block's documents are stepped over.
template <int NW> struct AtWalk {
    const int* ranges;          // of the sample, or nullptr: no documents
    int t0, t1, lo, hi;
    __device__ __forceinline__ int next(int t) const       // t1 or more: none
    {
        if (t >= t1) return t;
        ++t;
        if (ranges) while (t < t1 && !at_meet(at_range(ranges, t), lo, hi)) ++t;
        return t;
    }
};
template <int NW>
__device__ __forceinline__ AtWalk<NW> at_walk(const AttArgs& a, const int* all_ranges, int b, int last_limit, int lo, int hi, int* red)
{
    AtWalk<NW> w;
    const int tid = threadIdx.x;
    w.ranges = nullptr; w.t0 = 0; w.lo = lo; w.hi = hi;
    w.t1 = last_limit < 0 ? 0 : last_limit / AT_KT + 1;
    if (a.documents && w.t1) {
        w.ranges = all_ranges + (long long)b * ((a.Nk + AT_KT - 1) / AT_KT) * 2;
        if ((tid & 63) == 0) { red[2 * (tid >> 6)] = lo; red[2 * (tid >> 6) + 1] = hi; }
        if (tid == 0) { red[2 * NW] = 0x7fffffff; red[2 * NW + 1] = 0; }
        __syncthreads();
        for (int v = 0; v < NW; ++v) { lo = min(lo, red[2 * v]); hi = max(hi, red[2 * v + 1]); }
        int first = 0x7fffffff, end = 0;
        for (int t = tid; t < w.t1; t += 64 * NW)
            if (w.ranges[2 * (long long)t] <= hi && w.ranges[2 * (long long)t + 1] >= lo) { first = min(first, t); end = t + 1; }
        if (end) { atomicMin(&red[2 * NW], first); atomicMax(&red[2 * NW + 1], end); }       // min and max: any order, one result
        __syncthreads();
        w.t0 = __builtin_amdgcn_readfirstlane(red[2 * NW]);
        w.t1 = __builtin_amdgcn_readfirstlane(red[2 * NW + 1]);
        w.lo = __builtin_amdgcn_readfirstlane(lo); w.hi = __builtin_amdgcn_readfirstlane(hi);
    }
    return w;
}

// ---- which forward kernel --------------------------------------------------------------------------------------------------
// The step kernel splits keys over waves and blocks, the other one only query rows.  It takes over where most of a block's rows would be missing
// (128 rows over 4096 keys, 32 heads of 64: 22 us, otherwise 58), and where those rows alone give too few blocks for 256 CUs.  bf16, step kernel /
// the other, 8 heads, as many keys as rows: D = 32, 128 blocks 17.9 / 29.7 us, 248 blocks 41.9 / 51.8; D = 64, 128 blocks 20.7 / 34.4, 192 blocks
// 47.6 / 48.7, 248 blocks 61.7 / 60.6; D = 128, 64 blocks 44.8 / 56.4, 80 blocks 78.3 / 69.2, 128 blocks 149 / 105.  With 32 heads, hence a quarter of the
// rows, the blocks at which they meet are fewer (D = 64, 128 blocks 11.8 / 12.9, 192 blocks 25.9 / 16.8; D = 128, 64 blocks 31 / 23): the count of blocks
// is not all of it (profiles/token_ops/forward_kernels.txt).
// Its own blocks are split over the keys to fill the card once, at least 512 keys each (below that the joining costs more than it gains:
// 4096 keys, 8 key heads of 128: 13.8 us, split to 256 keys 15.6) and, so that caches of unequal fill come out even, at most about 4096 (8 caches of 32 to
// 64 Ki keys: 289 us, four splits of each 316); 2^16 blocks are even enough for any cache, and bound the partial sums.
struct AtStepPlan { bool use; int nsplit; };
static inline AtStepPlan at_step_plan(const AttArgs& a)
{
    const int rows = a.D == 128 ? 256 : 128;
    const long long NR = (long long)a.Nq * (a.Hq / a.Hk), blocks = (long long)a.B * a.Hq * ((a.Nq + rows - 1) / rows);
    AtStepPlan p = {blocks < (a.D == 128 ? 85 : 256) || a.Nq <= rows / 4, 1};
    const long long items = (long long)a.B * a.Hk * ((NR + 31) / 32);
    if (p.use && items > 0) {
        const long long fill = 256 / items, even = items < 2048 ? a.Nk / 4096 : 0, most = a.Nk / 512;
        long long n = fill > even ? fill : even;
        n = n < most ? n : most;
        n = n < 65536 / items ? n : 65536 / items;
        p.nsplit = n < 1 ? 1 : (int)n;
    }
    return p;
}
// A launch has fewer than 2^32 threads.  (The backward kernels are split, at most 2048 blocks of them, only where their blocks are few.)
static inline bool att_grids_fit(const AttArgs& a, bool grad)
{
    const long long rows = (long long)a.B * a.Hq * ((a.Nq + 255LL) / 256) * 512, G = a.Hq / a.Hk, most = 1LL << 32;
    if (grad) return rows < most && (long long)a.B * a.Hk * ((a.Nk + 127LL) / 128) * 256 < most;
    return at_step_plan(a).use ? (long long)a.B * a.Hk * ((a.Nq * G + 31) / 32) * 256 < most : rows < most;
}

// ---- launchers (one translation unit per type) -----------------------------------------------------------------------------
int att_forward_bf16(const AttArgs& a, void* o_low, void* ws, hipStream_t st);
int att_forward_f16(const AttArgs& a, void* o_low, void* ws, hipStream_t st);
int att_backward_bf16(const AttArgs& a, const void* o_low, void* ws, hipStream_t st);
int att_backward_f16(const AttArgs& a, const void* o_low, void* ws, hipStream_t st);
int att_launch_doc_ranges(const AttArgs& a, int* ranges, hipStream_t st);
static inline int att_key_tiles(const AttArgs& a) { return (a.Nk + AT_KT - 1) / AT_KT; }
constexpr int AT_DOC_LDS = AT_KT * 4;        // documents of a tile, behind its rows
static inline long long att_doc_bytes(const AttArgs& a) { return a.documents ? (((long long)a.B * att_key_tiles(a) * 8 + 255) & ~255LL) : 0; }
