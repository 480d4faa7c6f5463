// Infinities and NaN at places that a mask hides.  The products of the fast kernels multiply every element of a tile: a hidden key's
// probability of zero times an infinite v is NaN, and would reach rows that do not see the key (likewise k in dQ, and the q and dO of
// other rows in dK and dV).  Scores are not concerned: hidden ones are replaced, not multiplied.  So every wave looks at its sums when it is
// done (a zero times a non-finite sum is not zero), and works rows (or keys) with a non-finite sum out again, one after the other,
// over what they see alone.  A row that does see a NaN keeps it.  Costs one multiply-add per sum; slow where it strikes (a wave per row).
#pragma once
#include "masked_attention.h"

template <int DT> __device__ __forceinline__ bool at_not_finite(const f32x16 (&o)[DT])
{
    float t = 0.f;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int r = 0; r < 16; ++r) t = __builtin_fmaf(o[dt][r], 0.f, t);
    return !(t == 0.f);
}
// bit q: one of the two lanes of column q says so
__device__ __forceinline__ uint32_t at_columns(bool bad)
{
    const unsigned long long m = __ballot(bad);
    return (uint32_t)m | (uint32_t)(m >> 32);
}

template <typename T, int D> __device__ __forceinline__ float at_dot(const T* x, const T* y)
{
    float s = 0.f;
    for (int e = 0; e < D; e += 8) {
        float f[8], g[8];
        piece_to_float(*reinterpret_cast<const uint4*>(x + e), f, T());
        piece_to_float(*reinterpret_cast<const uint4*>(y + e), g, T());
#pragma unroll
        for (int j = 0; j < 8; ++j) s = __builtin_fmaf(f[j], g[j], s);
    }
    return s;
}
template <int CAP, bool BIAS> __device__ __forceinline__ float at_base2(const AtScore& sc, float qk, float slope2, float dist, float& th)
{
    float x = at_score<CAP>(sc, qk, 0.f, th);
    if (BIAS) x = __builtin_fmaf(-slope2, fabsf(dist), x);
    return x;
}
__device__ __forceinline__ float at_lane(float v, int lane) { return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(v), lane)); }
__device__ __forceinline__ float at_wave_max(float v)
{
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) v = __builtin_elementwise_maximum(v, __shfl_xor(v, m, 64));
    return v;
}

// Everything below is computed by a whole wave, all arguments the same on its lanes; lane l gets elements l and l + 64 of the results.

template <typename T> struct AtOperands { const T *q, *k, *v, *g; };           // row 0 of the head (g: gradient of o)
template <typename T> __device__ __forceinline__ AtOperands<T> at_operands(const AttArgs& a, int b, int head)
{
    const int kh = head / (a.Hq / a.Hk);
    return {reinterpret_cast<const T*>(a.q) + (long long)b * a.q_stride_b + (long long)head * a.q_stride_h,
            reinterpret_cast<const T*>(a.k) + (long long)b * a.k_stride_b + (long long)kh * a.k_stride_h,
            reinterpret_cast<const T*>(a.v) + (long long)b * a.v_stride_b + (long long)kh * a.v_stride_h,
            reinterpret_cast<const T*>(a.o_grad) + (long long)b * a.og_stride_b + (long long)head * a.og_stride_h};
}

// forward: row i over the keys j0 .. j1 - 1 that it sees
template <typename T, int D, int CAP, bool BIAS>
__device__ __forceinline__ void at_exact_row(const AttArgs& a, const AtScore& sc, const AtSample& sm, int b, int head, int i, int j0, int j1,
                                             float& m, float& l, float (&o)[2])
{
    const int lane = threadIdx.x & 63;
    const AtOperands<T> p = at_operands<T>(a, b, head);
    const T* qr = p.q + (long long)i * a.q_stride_n;
    const int doc = a.documents ? at_row_doc(a, sm, b, i) : 0, lim = doc < 0 ? -1 : min(at_limit(a, sm, i), j1 - 1);
    const int pos = at_bias_pos(a, sm, i);
    const float slope2 = BIAS ? a.slopes[head] * AT_LOG2E : 0.f;
    m = -INFINITY; l = 0.f; o[0] = o[1] = 0.f;
    for (int jb = j0; jb <= lim; jb += 64) {
        const int j = jb + lane;
        const bool see = j <= lim && (!a.documents || a.documents[(long long)b * a.documents_stride + j] == doc);
        float x = -INFINITY, th;
        if (see) x = at_base2<CAP, BIAS>(sc, at_dot<T, D>(qr, p.k + (long long)j * a.k_stride_n), slope2, (float)(pos - j), th);
        unsigned long long seen = __ballot(see);
        if (!seen) continue;
        const float mn = __builtin_elementwise_maximum(m, at_wave_max(x)), f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - mn);
        const float pr = see ? __builtin_amdgcn_exp2f(mn == -INFINITY ? x : x - mn) : 0.f;
        m = mn;
        l = l * f + wave_sum(pr);
        o[0] *= f; o[1] *= f;
        for (; seen; seen &= seen - 1) {
            const int s = __builtin_ctzll(seen);
            const float ps = at_lane(pr, s);
            const T* vr = p.v + (long long)(jb + s) * a.v_stride_n;
            if (lane < D) o[0] = __builtin_fmaf(ps, (float)vr[lane], o[0]);
            if (lane + 64 < D) o[1] = __builtin_fmaf(ps, (float)vr[lane + 64], o[1]);
        }
    }
}

// dQ of row i, without the scale
template <typename T, int D, int CAP, bool BIAS>
__device__ __forceinline__ void at_exact_dq(const AttArgs& a, const AtScore& sc, const AtSample& sm, int b, int head, int i, float lse, float delta, float (&dq)[2])
{
    const int lane = threadIdx.x & 63;
    const AtOperands<T> p = at_operands<T>(a, b, head);
    const T *qr = p.q + (long long)i * a.q_stride_n, *gr = p.g + (long long)i * a.og_stride_n;
    const int doc = a.documents ? at_row_doc(a, sm, b, i) : 0, lim = doc < 0 ? -1 : at_limit(a, sm, i);
    const int pos = at_bias_pos(a, sm, i);
    const float slope2 = BIAS ? a.slopes[head] * AT_LOG2E : 0.f;
    dq[0] = dq[1] = 0.f;
    for (int jb = 0; jb <= lim; jb += 64) {
        const int j = jb + lane;
        const bool see = j <= lim && (!a.documents || a.documents[(long long)b * a.documents_stride + j] == doc);
        float ds = 0.f, th;
        if (see) {
            const float x = at_base2<CAP, BIAS>(sc, at_dot<T, D>(qr, p.k + (long long)j * a.k_stride_n), slope2, (float)(pos - j), th);
            ds = __builtin_amdgcn_exp2f(x - lse) * (at_dot<T, D>(gr, p.v + (long long)j * a.v_stride_n) - delta) * (1.f - th * th);
        }
        for (unsigned long long seen = __ballot(see); seen; seen &= seen - 1) {
            const int s = __builtin_ctzll(seen);
            const float w = at_lane(ds, s);
            const T* kr = p.k + (long long)(jb + s) * a.k_stride_n;
            if (lane < D) dq[0] = __builtin_fmaf(w, (float)kr[lane], dq[0]);
            if (lane + 64 < D) dq[1] = __builtin_fmaf(w, (float)kr[lane + 64], dq[1]);
        }
    }
}

// dK (without the scale) and dV of key j over the rows `first` .. `end` - 1 of every head that reads it
template <typename T, int D, int CAP, bool BIAS>
__device__ __forceinline__ void at_exact_dkv(const AttArgs& a, const AtScore& sc, const AtSample& sm, const float* delta, int b, int khead, int j, int first, int end,
                                             float (&dk)[2], float (&dv)[2])
{
    const int lane = threadIdx.x & 63, G = a.Hq / a.Hk;
    const int doc = a.documents ? a.documents[(long long)b * a.documents_stride + j] : 0;
    dk[0] = dk[1] = dv[0] = dv[1] = 0.f;
    if (doc < 0) return;
    for (int gi = 0; gi < G; ++gi) {
        const int head = khead * G + gi;
        const AtOperands<T> p = at_operands<T>(a, b, head);
        const T *kr = p.k + (long long)j * a.k_stride_n, *vr = p.v + (long long)j * a.v_stride_n;
        const float slope2 = BIAS ? a.slopes[head] * AT_LOG2E : 0.f;
        const long long at = ((long long)b * a.Hq + head) * a.Nq;
        for (int ib = max(first, 0); ib < end; ib += 64) {
            const int i = ib + lane;
            const bool see = i < end && (!a.documents || at_row_doc(a, sm, b, i) == doc);
            float ds = 0.f, pr = 0.f, th;
            if (see) {
                const float x = at_base2<CAP, BIAS>(sc, at_dot<T, D>(p.q + (long long)i * a.q_stride_n, kr), slope2, (float)(at_bias_pos(a, sm, i) - j), th);
                pr = __builtin_amdgcn_exp2f(x - a.lse[at + i]);
                ds = pr * (at_dot<T, D>(p.g + (long long)i * a.og_stride_n, vr) - delta[at + i]) * (1.f - th * th);
            }
            for (unsigned long long seen = __ballot(see); seen; seen &= seen - 1) {
                const int s = __builtin_ctzll(seen);
                const float w = at_lane(ds, s), u = at_lane(pr, s);
                const T *qr = p.q + (long long)(ib + s) * a.q_stride_n, *gr = p.g + (long long)(ib + s) * a.og_stride_n;
                if (lane < D) { dk[0] = __builtin_fmaf(w, (float)qr[lane], dk[0]); dv[0] = __builtin_fmaf(u, (float)gr[lane], dv[0]); }
                if (lane + 64 < D) { dk[1] = __builtin_fmaf(w, (float)qr[lane + 64], dk[1]); dv[1] = __builtin_fmaf(u, (float)gr[lane + 64], dv[1]); }
            }
        }
    }
}

// o, and what its rounding lost: see at_store_o
template <typename T, int D> __device__ __forceinline__ void at_store_o_row(void* o, void* low, long long at, const float (&x)[2], float f)
{
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        const int e = lane + 64 * u;
        if (e >= D) break;
        const float y = x[u] * f;
        const T r = (T)y;
        reinterpret_cast<T*>(o)[at + e] = r;
        if (low) {
            const float l = y - (float)r;
            reinterpret_cast<T*>(low)[at + e] = (T)(l * 0.f == 0.f ? l : 0.f);
        }
    }
}
template <typename T, int D> __device__ __forceinline__ void at_store_row(T* row, const float (&x)[2], float f)
{
    const int lane = threadIdx.x & 63;
    if (lane < D) row[lane] = (T)(x[0] * f);
    if (lane + 64 < D) row[lane + 64] = (T)(x[1] * f);
}
