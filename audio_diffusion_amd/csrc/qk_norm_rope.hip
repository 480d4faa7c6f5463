// Queries and keys of an attention layer: RMS norm of every head and the position rotation in ONE pass, and its gradient.
//
//   r = 1 / sqrt(mean_d x_d^2 + eps)      n_d = x_d r      u_d = n_d w_d
//   (y_a, y_b) = (u_a cos - u_b sin, u_a sin + u_b cos)    with the angle position * frequency[p] of pair p = (a, b),
//   pairs (p, p + R/2), or (2p, 2p + 1) interleaved, over the first R elements; elements R.. are normed only.
// Gradient: g = the gradient of y turned back by the angle;  dw = sum_rows g n;  h = g w;  dx = r (h - n mean_d(h n)).
//
// Measured, bf16, the kernels alone: 4 x 8191 tokens, 32 + 8 heads of 128: 127 to 138 us forwards, 215 to 229 us gradients (5.3 to 4.9 and 4.7 to 4.4 TB/s;
// a copy of 2 GiB runs at 4.9 here); one token of each of 32 sequences: 5.7 us.
// Bound by HBM: every element is read once and written once (gradient: two reads, one write), with 16-byte accesses.
// A wave takes one TOKEN and walks its heads: the angles of a token are the same for all heads, so each lane computes one of
// them (in 64 bits up to the fraction of a turn: exact for any position a 64-bit product holds), the wave shares them through
// LDS, and every lane then keeps the NV cosines and sines of its own pairs in registers for all heads.  A head's row is spread over
// D / (2 NV) lanes, each holding BOTH elements of its NV pairs: no cross-lane traffic for the rotation, only the few
// DPP additions of the sum of squares.  Sums are held in 32 bits; the one rounding to 16 bits is the store.
#include "adk_common.h"

typedef adk_qk_norm_rope_args QkArgs;

constexpr int QK_MAX_PAIRS = 128;            // D <= 256
constexpr int QK_WAVES = 4;
constexpr int QK_BWD_BLOCKS = 2048;          // blocks of the gradient, each leaves one row of weight-gradient partials (1024: 256 us where 2048 take 212)

template <typename T> __device__ __forceinline__ float to_f(T v) { return (float)v; }

// One lane's share of a head row: P pairs, x[2P].  VEC: two 16-byte pieces; otherwise single elements, pairs lane + 64 j.
template <typename T, bool VEC> struct QkRow {
    static constexpr int NV = ElemTraits<T>::NV;
    static constexpr int P = VEC ? NV : QK_MAX_PAIRS / 64;
    int ea, eb;              // VEC: first elements of the two pieces
    int slot, D, R;
    bool inter, on;          // on: this lane holds a part of the row

    __device__ __forceinline__ QkRow(const QkArgs& a, int slot_) : slot(slot_), D(a.D), R(a.R), inter(a.interleaved != 0) {
        if (VEC) {
            on = slot < D / (2 * NV);
            const int rs = R / (2 * NV);
            if (inter || slot >= rs) { ea = 2 * slot * NV; eb = ea + NV; }     // untouched elements: pairs of no meaning
            else { ea = slot * NV; eb = R / 2 + slot * NV; }
            if (!on) ea = eb = 0;
        } else {
            on = true; ea = eb = 0;
        }
    }
    // pair index of pair j, and whether it is rotated / exists
    __device__ __forceinline__ int pair(int j) const { return VEC ? slot * NV + j : slot + 64 * j; }
    __device__ __forceinline__ int elem(int j, int second) const {             // !VEC: element of the row
        const int p = pair(j);
        if (inter || p >= R / 2) return 2 * p + second;
        return p + second * (R / 2);
    }
    // the lane's part of a row as it stands in memory, so that the next rows can be on their way while these are worked on
    struct Raw { uint4 a, b; };
    __device__ __forceinline__ Raw fetch(const T* row, bool ok) const {
        Raw w;
        w.a = w.b = make_uint4(0, 0, 0, 0);
        if (VEC) {
            if (ok) { w.a = *reinterpret_cast<const uint4*>(row + ea); w.b = *reinterpret_cast<const uint4*>(row + eb); }
        } else {
            union { Raw r; T v[32 / sizeof(T)]; } u;
            u.r = w;
#pragma unroll
            for (int j = 0; j < P; ++j)
#pragma unroll
                for (int s = 0; s < 2; ++s)
                    if (ok && pair(j) < D / 2) u.v[2 * j + s] = row[elem(j, s)];
            w = u.r;
        }
        return w;
    }
    __device__ __forceinline__ void value(const Raw& w, float (&x)[2 * P]) const {
        if (VEC) {
            float f[NV], g[NV];
            piece_to_float(w.a, f, T()); piece_to_float(w.b, g, T());
#pragma unroll
            for (int e = 0; e < NV; ++e) { x[e] = f[e]; x[NV + e] = g[e]; }
        } else {
            union { Raw r; T v[32 / sizeof(T)]; } u;
            u.r = w;
#pragma unroll
            for (int e = 0; e < 2 * P; ++e) x[e] = to_f(u.v[e]);
        }
    }
    __device__ __forceinline__ void load_f32(const float* w, float (&x)[2 * P]) const {      // a weight row; 1 where there is none
        if (VEC) {
#pragma unroll
            for (int e = 0; e < NV; ++e) { x[e] = w ? w[ea + e] : 1.f; x[NV + e] = w ? w[eb + e] : 1.f; }
        } else {
#pragma unroll
            for (int j = 0; j < P; ++j)
#pragma unroll
                for (int s = 0; s < 2; ++s) x[2 * j + s] = w && pair(j) < D / 2 ? w[elem(j, s)] : 1.f;
        }
    }
    __device__ __forceinline__ void store(T* row, const float (&x)[2 * P], bool ok) const {
        if (!ok) return;
        if (VEC) {
            float f[NV], g[NV];
#pragma unroll
            for (int e = 0; e < NV; ++e) { f[e] = x[e]; g[e] = x[NV + e]; }
            *reinterpret_cast<uint4*>(row + ea) = float_to_piece(f, T());
            *reinterpret_cast<uint4*>(row + eb) = float_to_piece(g, T());
        } else {
#pragma unroll
            for (int j = 0; j < P; ++j)
#pragma unroll
                for (int s = 0; s < 2; ++s)
                    if (pair(j) < D / 2) row[elem(j, s)] = (T)x[2 * j + s];
        }
    }
    __device__ __forceinline__ void add_f32(float* w, const float (&x)[2 * P]) const {       // w[element] += x, LDS or global
        if (VEC) {
            if (!on) return;
#pragma unroll
            for (int e = 0; e < NV; ++e) { w[ea + e] += x[e]; w[eb + e] += x[NV + e]; }
        } else {
#pragma unroll
            for (int j = 0; j < P; ++j)
#pragma unroll
                for (int s = 0; s < 2; ++s)
                    if (pair(j) < D / 2) w[elem(j, s)] += x[2 * j + s];
        }
    }
};

// Pairs of the interleaved and the split form lie differently in x[]: turned by a template constant so that x[] keeps to
// registers.
// Pairs past R / 2 are left alone, not turned by (1, 0): an element must not meet its neighbour's infinity.
template <typename Row, bool VEC, bool INTER>
__device__ __forceinline__ void turn(const Row& row, float (&x)[2 * Row::P], const float (&c)[Row::P], const float (&s)[Row::P], float sign)
{
    constexpr int P = Row::P;
#pragma unroll
    for (int j = 0; j < P; ++j) {
        const int ia = VEC && !INTER ? j : 2 * j, ib = VEC && !INTER ? P + j : 2 * j + 1;
        const float a = x[ia], b = x[ib], sj = sign * s[j];
        if (row.pair(j) < row.R / 2) {
            x[ia] = a * c[j] - b * sj;
            x[ib] = a * sj + b * c[j];
        }
    }
}

// The two halves (32 lanes), or the rows of a half (16 lanes), of a wave added up: a swap of the value with itself gives both.
__device__ __forceinline__ float add_halves(float v)
{
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float add_rows(float v)
{
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
// sum over each group of lpr (a power of two, the same for the whole grid) neighbouring lanes
__device__ __forceinline__ float group_sum(float v, int lpr)
{
    if (lpr > 1) v += dpp_mov<DPP_QUAD_XOR1>(v);
    if (lpr > 2) v += dpp_mov<DPP_QUAD_XOR2>(v);
    if (lpr > 4) v += dpp_mov<DPP_ROW_HALF_MIRROR>(v);
    if (lpr > 8) v += dpp_mov<DPP_ROW_MIRROR>(v);
    if (lpr > 16) v = add_rows(v);
    if (lpr > 32) v = add_halves(v);
    return v;
}
// sum over the groups: lane l gets the lanes equal to l modulo lpr
__device__ __forceinline__ float across_groups(float v, int lpr)
{
    if (lpr <= 8) v += dpp_mov<DPP_ROW_ROR8>(v);
    if (lpr <= 4) v += dpp_mov<DPP_ROW_ROR4>(v);
    if (lpr <= 2) v += dpp_mov<0x122>(v);          // row_ror:2
    if (lpr <= 1) v += dpp_mov<0x121>(v);          // row_ror:1
    if (lpr <= 16) v = add_rows(v);
    if (lpr <= 32) v = add_halves(v);
    return v;
}

// cos / sin of the wave's token for every pair, one per lane, into the wave's LDS row: (1, 0) for pairs that do not turn
__device__ __forceinline__ void token_angles(const QkArgs& a, int b, int n, float2* cs)
{
    const int lane = threadIdx.x & 63;
    double pos;
    const long long at = (long long)b * a.pos_stride_b + (long long)n * a.pos_stride_n;
    if (a.pos_bytes == 8) pos = (double)reinterpret_cast<const long long*>(a.positions)[at];
    else pos = (double)reinterpret_cast<const int*>(a.positions)[at];
    for (int p = lane; p < a.D / 2; p += 64) {
        float2 v = make_float2(1.f, 0.f);
        if (p < a.R / 2) {
            // the 64-bit product's fraction of a turn: 1 / (2 pi) in two parts, the rounding of the first product kept by an fma
            // (and no contraction: an fma in place of hi - rint(hi) would count that rounding twice)
#pragma clang fp contract(off)
            const double rad = pos * a.frequencies[p], hi = rad * 0.15915494309189535, lo = fma(rad, 0.15915494309189535, -hi) + rad * -9.839338337591243e-18;
            sincospif(2.0f * (float)((hi - rint(hi)) + lo), &v.y, &v.x);
        }
        cs[p] = v;
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
}

struct QkGrid { int lpr, groups, chunk, chunks, qblocks; long long tokens; };

template <typename T, bool VEC, bool INTER>
__global__ __launch_bounds__(64 * QK_WAVES) void qk_fwd_kernel(const QkArgs a, const QkGrid gr)
{
    typedef QkRow<T, VEC> Row;
    __shared__ float2 cs_all[QK_WAVES][QK_MAX_PAIRS];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const long long item = ((long long)blockIdx.y * gridDim.x + blockIdx.x) * QK_WAVES + wave;
    if (item >= gr.tokens * gr.chunks) return;                     // wave-uniform; no block barrier in this kernel
    const long long token = item / gr.chunks;
    const int ch = (int)(item % gr.chunks), b = (int)(token / a.N), n = (int)(token % a.N);
    const Row row(a, lane & (gr.lpr - 1));
    const int group = lane / gr.lpr;
        // units of `groups` heads (one row per lane; two need registers that cost more waves than they gain), first those of q, then those of k
    const int h0 = ch * gr.chunk, h1 = min(h0 + gr.chunk, a.Hq + a.Hk), step = gr.groups;
    const int q1 = min(h1, a.Hq), k0 = max(h0, a.Hq);
    const int nq = q1 > h0 ? (q1 - h0 + step - 1) / step : 0, units = nq + (h1 > k0 ? (h1 - k0 + step - 1) / step : 0);
    const T* qx = reinterpret_cast<const T*>(a.q) + (long long)b * a.q_stride_b + (long long)n * a.q_stride_n;
    const T* kx = reinterpret_cast<const T*>(a.k) + (long long)b * a.k_stride_b + (long long)n * a.k_stride_n;
    auto head = [&](int u) { return (u < nq ? h0 + u * step : k0 - a.Hq + (u - nq) * step) + group; };     // of q or k
    auto live = [&](int u) { return row.on && head(u) < (u < nq ? q1 : h1 - a.Hq); };
    auto fetch = [&](int u) { return row.fetch((u < nq ? qx : kx) + (long long)head(u) * (u < nq ? a.q_stride_h : a.k_stride_h), live(u)); };
    typename Row::Raw raw = fetch(0);           // on its way during the angles
    float2* cs = cs_all[wave];
    token_angles(a, b, n, cs);
    float c[Row::P], s[Row::P], w[2 * Row::P];
#pragma unroll
    for (int j = 0; j < Row::P; ++j) {
        const float2 v = row.pair(j) < a.D / 2 ? cs[row.pair(j)] : make_float2(1.f, 0.f);
        c[j] = v.x; s[j] = v.y;
    }
    const float inv_d = 1.0f / a.D;
    for (int u = 0; u < units; ++u) {
        if (u == 0 || u == nq) row.load_f32(u < nq ? a.q_weight : a.k_weight, w);
        float x[2 * Row::P], ss = 0.f;
        row.value(raw, x);
        if (u + 1 < units) raw = fetch(u + 1);
        T* y0 = u < nq ? reinterpret_cast<T*>(a.q_out) + token * a.Hq * a.D : reinterpret_cast<T*>(a.k_out) + token * a.Hk * a.D;
#pragma unroll
        for (int e = 0; e < 2 * Row::P; ++e) ss += x[e] * x[e];
        ss = group_sum(ss, gr.lpr);
        const float rs = 1.0f / sqrtf(ss * inv_d + a.eps);
#pragma unroll
        for (int e = 0; e < 2 * Row::P; ++e) x[e] = x[e] * rs * w[e];
        turn<Row, VEC, INTER>(row, x, c, s, 1.0f);
        row.store(y0 + (long long)head(u) * a.D, x, live(u));
    }
}

template <typename T, bool VEC, bool INTER>
__global__ __launch_bounds__(64 * QK_WAVES) void qk_bwd_kernel(const QkArgs a, const QkGrid gr, float* partial)
{
    typedef QkRow<T, VEC> Row;
    __shared__ float2 cs_all[QK_WAVES][QK_MAX_PAIRS];
    __shared__ float dw_all[QK_WAVES][2 * QK_MAX_PAIRS];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const Row row(a, lane & (gr.lpr - 1));
    const int group = lane / gr.lpr;
    float2* cs = cs_all[wave];
    const float inv_d = 1.0f / a.D;
    // a block works on q or on k alone (each its share of the blocks): one set of weights and of sums in registers
    const int which = (int)blockIdx.x >= gr.qblocks, H = which ? a.Hk : a.Hq;
    const int blk = which ? blockIdx.x - gr.qblocks : blockIdx.x, nblk = which ? gridDim.x - gr.qblocks : gr.qblocks;
    const T* x0 = reinterpret_cast<const T*>(which ? a.k : a.q);
    const T* g0 = reinterpret_cast<const T*>(which ? a.k_grad : a.q_grad);
    T* y0 = reinterpret_cast<T*>(which ? a.k_out : a.q_out);
    const long long xb = which ? a.k_stride_b : a.q_stride_b, xn = which ? a.k_stride_n : a.q_stride_n, xh = which ? a.k_stride_h : a.q_stride_h;
    const long long gb = which ? a.kg_stride_b : a.qg_stride_b, gn = which ? a.kg_stride_n : a.qg_stride_n, gh = which ? a.kg_stride_h : a.qg_stride_h;
    float acc[2 * Row::P], w[2 * Row::P];
#pragma unroll
    for (int e = 0; e < 2 * Row::P; ++e) acc[e] = 0.f;
    row.load_f32(which ? a.k_weight : a.q_weight, w);

    const long long waves = (long long)nblk * QK_WAVES;
    for (long long token = (long long)blk * QK_WAVES + wave; token < gr.tokens; token += waves) {
        const int b = (int)(token / a.N), n = (int)(token % a.N);
        const T* xr = x0 + (long long)b * xb + (long long)n * xn;
        const T* gr_ = g0 + (long long)b * gb + (long long)n * gn;
        typename Row::Raw rx = row.fetch(xr + (long long)group * xh, row.on && group < H), rg = row.fetch(gr_ + (long long)group * gh, row.on && group < H);
        token_angles(a, b, n, cs);                                 // rows on their way
        float c[Row::P], s[Row::P];
#pragma unroll
        for (int j = 0; j < Row::P; ++j) {
            const float2 v = row.pair(j) < a.D / 2 ? cs[row.pair(j)] : make_float2(1.f, 0.f);
            c[j] = v.x; s[j] = v.y;
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");     // the next token's angles go to the same LDS row
        for (int hb = 0; hb < H; hb += gr.groups) {
            const int h = hb + group, hn = h + gr.groups;
            const bool ok = h < H && row.on;
            float x[2 * Row::P], g[2 * Row::P];
            row.value(rx, x);
            row.value(rg, g);
            if (hb + gr.groups < H) {
                rx = row.fetch(xr + (long long)hn * xh, hn < H && row.on);
                rg = row.fetch(gr_ + (long long)hn * gh, hn < H && row.on);
            }
            float ss = 0.f, dot = 0.f;
            turn<Row, VEC, INTER>(row, g, c, s, -1.0f);
#pragma unroll
            for (int e = 0; e < 2 * Row::P; ++e) { ss += x[e] * x[e]; dot += g[e] * w[e] * x[e]; }
            ss = group_sum(ss, gr.lpr);
            dot = group_sum(dot, gr.lpr);
            const float r = 1.0f / sqrtf(ss * inv_d + a.eps);
            const float m = dot * r * inv_d;                       // mean_d(h n), n = x r
#pragma unroll
            for (int e = 0; e < 2 * Row::P; ++e) {
                const float nx = x[e] * r;
                if (ok) acc[e] += g[e] * nx;
                x[e] = r * (g[e] * w[e] - nx * m);
            }
            row.store(y0 + (token * H + h) * a.D, x, ok);
        }
    }
    // this block's sums, in a fixed order: over the lane groups of a wave, then over the waves through LDS
    if (!(which ? a.k_weight_grad : a.q_weight_grad)) return;      // uniform over the block
#pragma unroll
    for (int e = 0; e < 2 * Row::P; ++e) acc[e] = across_groups(acc[e], gr.lpr);
    for (int e = lane; e < 2 * QK_MAX_PAIRS; e += 64) dw_all[wave][e] = 0.f;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    if (group == 0) row.add_f32(dw_all[wave], acc);
    __syncthreads();
    for (int e = threadIdx.x; e < a.D; e += 64 * QK_WAVES) {
        float t = 0.f;
#pragma unroll
        for (int v = 0; v < QK_WAVES; ++v) t += dw_all[v][e];
        partial[(long long)blockIdx.x * a.D + e] = t;
    }
}

// weight gradients: element e of q's or k's weight summed over the partials of its blocks, one block per element, fixed order
__global__ __launch_bounds__(256) void qk_weight_grad_kernel(const float* partial, int qblocks, int nblk, int D, float* dq_w, float* dk_w)
{
    const int which = blockIdx.x / D, e = blockIdx.x % D;
    float* out = which ? dk_w : dq_w;
    if (!out) return;                                              // block-uniform
    __shared__ float red[16];
    float t = 0.f, z = 0.f;
    for (int i = (which ? qblocks : 0) + threadIdx.x; i < (which ? nblk : qblocks); i += 256) t += partial[(long long)i * D + e];
    block_sum2(t, z, red);
    if (threadIdx.x == 0) out[e] = t;
}

static bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// blocks for q and for k: every token a wave of its own up to QK_BWD_BLOCKS blocks in all, shared out by heads
struct QkBlocks { int q, k; };
static QkBlocks qk_bwd_blocks(const QkArgs& a)
{
    const long long tokens = (long long)a.B * a.N, need = (tokens + QK_WAVES - 1) / QK_WAVES;
    const int kmost = QK_BWD_BLOCKS * a.Hk / (a.Hq + a.Hk), k = kmost < 1 ? 1 : kmost, q = QK_BWD_BLOCKS - k < 1 ? 1 : QK_BWD_BLOCKS - k;
    return {(int)(need < q ? need : q), (int)(need < k ? need : k)};
}

long long qk_norm_rope_workspace(const QkArgs& a)
{
    const QkBlocks n = qk_bwd_blocks(a);
    return (long long)(n.q + n.k) * a.D * (long long)sizeof(float);
}

template <typename T> static int launch_qk_t(const QkArgs& a, void* ws, hipStream_t st, bool grad)
{
    constexpr int NV = ElemTraits<T>::NV;
    // 16-byte form: whole pieces on both sides of every pair, 16-byte rows.  Anything else goes element by element.
    auto strides_ok = [&](long long x, long long y, long long z) { return x % NV == 0 && y % NV == 0 && z % NV == 0; };
    bool vec = a.D % (2 * NV) == 0 && (a.interleaved || a.R % (2 * NV) == 0) && aligned16(a.q) && aligned16(a.k)
               && aligned16(a.q_out) && aligned16(a.k_out) && strides_ok(a.q_stride_b, a.q_stride_n, a.q_stride_h)
               && strides_ok(a.k_stride_b, a.k_stride_n, a.k_stride_h);
    if (grad)
        vec = vec && aligned16(a.q_grad) && aligned16(a.k_grad) && strides_ok(a.qg_stride_b, a.qg_stride_n, a.qg_stride_h)
              && strides_ok(a.kg_stride_b, a.kg_stride_n, a.kg_stride_h);
    QkGrid g;
    g.lpr = 64;
    if (vec) for (g.lpr = 1; g.lpr < a.D / (2 * NV); g.lpr <<= 1) {}
    g.groups = 64 / g.lpr;
    g.tokens = (long long)a.B * a.N;
    const int H = a.Hq + a.Hk;
    g.chunk = H; g.chunks = 1; g.qblocks = 0;
    if (grad) {
        const QkBlocks n = qk_bwd_blocks(a);
        const int nblk = n.q + n.k;
        g.qblocks = n.q;
        float* partial = reinterpret_cast<float*>(ws);
        if (vec) {
            if (a.interleaved) hipLaunchKernelGGL((qk_bwd_kernel<T, true, true>), dim3(nblk), dim3(64 * QK_WAVES), 0, st, a, g, partial);
            else hipLaunchKernelGGL((qk_bwd_kernel<T, true, false>), dim3(nblk), dim3(64 * QK_WAVES), 0, st, a, g, partial);
        } else hipLaunchKernelGGL((qk_bwd_kernel<T, false, true>), dim3(nblk), dim3(64 * QK_WAVES), 0, st, a, g, partial);
        if (hipGetLastError() != hipSuccess) return ADK_ELAUNCH;
        if (a.q_weight_grad || a.k_weight_grad)
            hipLaunchKernelGGL(qk_weight_grad_kernel, dim3(2 * a.D), dim3(256), 0, st, partial, n.q, nblk, a.D, a.q_weight_grad, a.k_weight_grad);
    } else {
        // few tokens: a token's heads are split over several waves (2 * groups heads each), so that a single step's launch
        // is one round of loads deep
        if (g.tokens < 4096) {
            g.chunk = 2 * g.groups;
            g.chunks = (H + g.chunk - 1) / g.chunk;
        }
        const long long items = g.tokens * g.chunks;
        // (a row of the grid has fewer than 2^32 threads)
        const long long blocks = (items + QK_WAVES - 1) / QK_WAVES, row = 1LL << 22;
        const dim3 grid((unsigned)(blocks < row ? blocks : row), (unsigned)((blocks + row - 1) / row));
        if (vec) {
            if (a.interleaved) hipLaunchKernelGGL((qk_fwd_kernel<T, true, true>), grid, dim3(64 * QK_WAVES), 0, st, a, g);
            else hipLaunchKernelGGL((qk_fwd_kernel<T, true, false>), grid, dim3(64 * QK_WAVES), 0, st, a, g);
        } else hipLaunchKernelGGL((qk_fwd_kernel<T, false, true>), grid, dim3(64 * QK_WAVES), 0, st, a, g);
    }
    return hipGetLastError() == hipSuccess ? ADK_OK : ADK_ELAUNCH;
}

int launch_qk_norm_rope(const QkArgs& a, void* ws, hipStream_t st, bool grad)
{
    if (a.dtype == ADK_F32) return launch_qk_t<float>(a, ws, st, grad);
    if (a.dtype == ADK_BF16) return launch_qk_t<bf16_t>(a, ws, st, grad);
    return launch_qk_t<f16_t>(a, ws, st, grad);
}
