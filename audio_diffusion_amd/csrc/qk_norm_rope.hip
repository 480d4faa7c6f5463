// Queries and keys of an attention layer: RMS norm of every head and the position rotation in ONE pass, and its gradient.
//
//   r = 1 / sqrt(mean_d x_d^2 + eps)      n_d = x_d r      u_d = n_d w_d
//   (y_a, y_b) = (u_a cos - u_b sin, u_a sin + u_b cos)    with the angle position * frequency[p] of pair p = (a, b),
//   pairs (p, p + R/2), or (2p, 2p + 1) interleaved, over the first R elements; elements R.. are normed only.
// Gradient: g = the gradient of y turned back by the angle;  dw = sum_rows g n;  h = g w;  dx = r (h - n mean_d(h n)).
//
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
constexpr int QK_BWD_BLOCKS = 1024;          // blocks of the gradient: each leaves one row of weight-gradient partials

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
    __device__ __forceinline__ void load(const T* row, float (&x)[2 * P], bool ok) const {
        if (VEC) {
            uint4 u = make_uint4(0, 0, 0, 0), v = u;
            if (ok) { u = *reinterpret_cast<const uint4*>(row + ea); v = *reinterpret_cast<const uint4*>(row + eb); }
            float f[NV], g[NV];
            piece_to_float(u, f, T()); piece_to_float(v, g, T());
#pragma unroll
            for (int e = 0; e < NV; ++e) { x[e] = f[e]; x[NV + e] = g[e]; }
        } else {
#pragma unroll
            for (int j = 0; j < P; ++j)
#pragma unroll
                for (int s = 0; s < 2; ++s) x[2 * j + s] = ok && pair(j) < D / 2 ? to_f(row[elem(j, s)]) : 0.f;
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
    for (int p = lane; p < QK_MAX_PAIRS; p += 64) {
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

struct QkGrid { int lpr, groups, chunk, chunks; long long tokens; };

template <typename T, bool VEC, bool INTER>
__global__ __launch_bounds__(64 * QK_WAVES) void qk_fwd_kernel(const QkArgs a, const QkGrid gr)
{
    typedef QkRow<T, VEC> Row;
    __shared__ float2 cs_all[QK_WAVES][QK_MAX_PAIRS];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const long long item = (long long)blockIdx.x * QK_WAVES + wave;
    if (item >= gr.tokens * gr.chunks) return;                     // wave-uniform; no block barrier in this kernel
    const long long token = item / gr.chunks;
    const int ch = (int)(item % gr.chunks), b = (int)(token / a.N), n = (int)(token % a.N);
    const Row row(a, lane & (gr.lpr - 1));
    const int group = lane / gr.lpr;
    float2* cs = cs_all[wave];
    token_angles(a, b, n, cs);
    float c[Row::P], s[Row::P];
#pragma unroll
    for (int j = 0; j < Row::P; ++j) {
        const float2 v = row.pair(j) < QK_MAX_PAIRS ? cs[row.pair(j)] : make_float2(1.f, 0.f);
        c[j] = v.x; s[j] = v.y;
    }
    const float inv_d = 1.0f / a.D;
    const int h0 = ch * gr.chunk, h1 = min(h0 + gr.chunk, a.Hq + a.Hk);
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        const int H = which ? a.Hk : a.Hq, off = which ? a.Hq : 0;
        const int lo = max(h0 - off, 0), hi = min(h1 - off, H);
        if (lo >= hi) continue;
        const T* x0 = reinterpret_cast<const T*>(which ? a.k : a.q) + (long long)b * (which ? a.k_stride_b : a.q_stride_b)
                      + (long long)n * (which ? a.k_stride_n : a.q_stride_n);
        const long long sh = which ? a.k_stride_h : a.q_stride_h;
        T* y0 = reinterpret_cast<T*>(which ? a.k_out : a.q_out) + token * H * a.D;
        float w[2 * Row::P];
        row.load_f32(which ? a.k_weight : a.q_weight, w);
        for (int hb = lo; hb < hi; hb += 2 * gr.groups) {          // two heads per lane in flight
            float x[2][2 * Row::P];
            bool ok[2];
            int h[2];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                h[u] = hb + u * gr.groups + group;
                ok[u] = h[u] < hi && row.on;
                row.load(x0 + (long long)h[u] * sh, x[u], ok[u]);
            }
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                float ss = 0.f;
#pragma unroll
                for (int e = 0; e < 2 * Row::P; ++e) ss += x[u][e] * x[u][e];
                ss = group_sum(ss, gr.lpr);
                const float r = 1.0f / sqrtf(ss * inv_d + a.eps);
#pragma unroll
                for (int e = 0; e < 2 * Row::P; ++e) x[u][e] = x[u][e] * r * w[e];
                turn<Row, VEC, INTER>(row, x[u], c, s, 1.0f);
                row.store(y0 + (long long)h[u] * a.D, x[u], ok[u]);
            }
        }
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
    float acc[2][2 * Row::P];
#pragma unroll
    for (int which = 0; which < 2; ++which)
#pragma unroll
        for (int e = 0; e < 2 * Row::P; ++e) acc[which][e] = 0.f;

    const long long waves = (long long)gridDim.x * QK_WAVES;
    for (long long token = (long long)blockIdx.x * QK_WAVES + wave; token < gr.tokens; token += waves) {
        const int b = (int)(token / a.N), n = (int)(token % a.N);
        token_angles(a, b, n, cs);
        float c[Row::P], s[Row::P];
#pragma unroll
        for (int j = 0; j < Row::P; ++j) {
            const float2 v = row.pair(j) < QK_MAX_PAIRS ? cs[row.pair(j)] : make_float2(1.f, 0.f);
            c[j] = v.x; s[j] = v.y;
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");     // the next token's angles go to the same LDS row
#pragma unroll
        for (int which = 0; which < 2; ++which) {
            const int H = which ? a.Hk : a.Hq;
            const T* x0 = reinterpret_cast<const T*>(which ? a.k : a.q) + (long long)b * (which ? a.k_stride_b : a.q_stride_b)
                          + (long long)n * (which ? a.k_stride_n : a.q_stride_n);
            const T* g0 = reinterpret_cast<const T*>(which ? a.k_grad : a.q_grad) + (long long)b * (which ? a.kg_stride_b : a.qg_stride_b)
                          + (long long)n * (which ? a.kg_stride_n : a.qg_stride_n);
            const long long sh = which ? a.k_stride_h : a.q_stride_h, gsh = which ? a.kg_stride_h : a.qg_stride_h;
            T* y0 = reinterpret_cast<T*>(which ? a.k_out : a.q_out) + token * H * a.D;
            float w[2 * Row::P];
            row.load_f32(which ? a.k_weight : a.q_weight, w);
            for (int hb = 0; hb < H; hb += gr.groups) {
                const int h = hb + group;
                const bool ok = h < H && row.on;
                float x[2 * Row::P], g[2 * Row::P];
                row.load(x0 + (long long)h * sh, x, ok);
                row.load(g0 + (long long)h * gsh, g, ok);
                float ss = 0.f, hn = 0.f;
                turn<Row, VEC, INTER>(row, g, c, s, -1.0f);
#pragma unroll
                for (int e = 0; e < 2 * Row::P; ++e) { ss += x[e] * x[e]; hn += g[e] * w[e] * x[e]; }
                ss = group_sum(ss, gr.lpr);
                hn = group_sum(hn, gr.lpr);
                const float r = 1.0f / sqrtf(ss * inv_d + a.eps);
                const float m = hn * r * inv_d;                    // mean_d(h n), n = x r
#pragma unroll
                for (int e = 0; e < 2 * Row::P; ++e) {
                    const float nx = x[e] * r;
                    if (ok) acc[which][e] += g[e] * nx;
                    x[e] = r * (g[e] * w[e] - nx * m);
                }
                row.store(y0 + (long long)h * a.D, x, ok);
            }
        }
    }
    // this block's sums, in a fixed order: over the lane groups of a wave, then over the waves through LDS
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        if (!(which ? a.k_weight_grad : a.q_weight_grad)) continue;            // uniform over the grid
#pragma unroll
        for (int e = 0; e < 2 * Row::P; ++e) acc[which][e] = across_groups(acc[which][e], gr.lpr);
        __syncthreads();
        for (int e = lane; e < 2 * QK_MAX_PAIRS; e += 64) dw_all[wave][e] = 0.f;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        if (group == 0) row.add_f32(dw_all[wave], acc[which]);
        __syncthreads();
        for (int e = threadIdx.x; e < a.D; e += 64 * QK_WAVES) {
            float t = 0.f;
#pragma unroll
            for (int v = 0; v < QK_WAVES; ++v) t += dw_all[v][e];
            partial[((long long)blockIdx.x * 2 + which) * a.D + e] = t;
        }
    }
}

// weight gradients: column (which, e) summed over the blocks' partials, one block per column, fixed order
__global__ __launch_bounds__(256) void qk_weight_grad_kernel(const float* partial, int nblk, int D, float* dq_w, float* dk_w)
{
    const int which = blockIdx.x / D, e = blockIdx.x % D;
    float* out = which ? dk_w : dq_w;
    if (!out) return;                                              // block-uniform
    __shared__ float red[16];
    float t = 0.f, z = 0.f;
    for (int i = threadIdx.x; i < nblk; i += 256) t += partial[((long long)i * 2 + which) * D + e];
    block_sum2(t, z, red);
    if (threadIdx.x == 0) out[e] = t;
}

static bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

static int qk_bwd_blocks(const QkArgs& a)
{
    const long long tokens = (long long)a.B * a.N, need = (tokens + QK_WAVES - 1) / QK_WAVES;
    return (int)(need < QK_BWD_BLOCKS ? need : QK_BWD_BLOCKS);
}

long long qk_norm_rope_workspace(const QkArgs& a)
{
    return (long long)qk_bwd_blocks(a) * 2 * a.D * (long long)sizeof(float);
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
    g.chunk = H; g.chunks = 1;
    if (grad) {
        const int nblk = qk_bwd_blocks(a);
        float* partial = reinterpret_cast<float*>(ws);
        if (vec) {
            if (a.interleaved) hipLaunchKernelGGL((qk_bwd_kernel<T, true, true>), dim3(nblk), dim3(64 * QK_WAVES), 0, st, a, g, partial);
            else hipLaunchKernelGGL((qk_bwd_kernel<T, true, false>), dim3(nblk), dim3(64 * QK_WAVES), 0, st, a, g, partial);
        } else hipLaunchKernelGGL((qk_bwd_kernel<T, false, true>), dim3(nblk), dim3(64 * QK_WAVES), 0, st, a, g, partial);
        if (hipGetLastError() != hipSuccess) return ADK_ELAUNCH;
        if (a.q_weight_grad || a.k_weight_grad)
            hipLaunchKernelGGL(qk_weight_grad_kernel, dim3(2 * a.D), dim3(256), 0, st, partial, nblk, a.D, a.q_weight_grad, a.k_weight_grad);
    } else {
        // few tokens: a token's heads are split over several waves (2 * groups heads each), so that a single step's launch
        // is one round of loads deep
        if (g.tokens < 4096) {
            g.chunk = 2 * g.groups;
            g.chunks = (H + g.chunk - 1) / g.chunk;
        }
        const long long items = g.tokens * g.chunks;
        const dim3 grid((unsigned)((items + QK_WAVES - 1) / QK_WAVES));
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
