// f16 instantiations of masked_attention_bwd.inc, and the scale of every key's dS
#include "masked_attention_bwd.inc"

int att_backward_f16(const AttArgs& a, const void* o_low, void* ws, hipStream_t st) { return att_backward_t<f16_t>(a, o_low, ws, st); }

// The largest |dO| of the rows, of all heads that share the keys, that see each key.  A wave takes 32 keys (key on the lane, half of a
// tile's rows on each half of the lanes) and looks at the 64-row tiles, first a tile per lane: those that all its keys see whole give their maximum
// to all; those of one document that no key's first row divides, to the keys that see them; the others (a causal mask's corner,
// the edges of documents) are gone through row by row.  A kernel of its own: inside the second kernel it cost 15 % with documents, in that kernel's few
// waves and registers.
__global__ __launch_bounds__(256) void att_key_amax_kernel(const AttArgs a, const BwdGeo g)
{
    __shared__ __attribute__((aligned(16))) float row_max[4][AT_QT];
    __shared__ __attribute__((aligned(16))) int row_doc[4][AT_QT];
    const int lane = threadIdx.x & 63, hh = lane >> 5, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), G = a.Hq / a.Hk;
    const int bh = blockIdx.x % g.nbh, b = bh / a.Hk, khead = bh % a.Hk;
    const AtSample sm = at_sample(a, b);
    const int j0 = blockIdx.x / g.nbh * 128 + wave * 32, j = j0 + (lane & 31);
    if (j0 >= sm.klen) return;                 // wave-uniform; no block barrier here
    const int jc = min(j, sm.klen - 1), ntile = (a.Nq + AT_QT - 1) / AT_QT;
    int imin = at_first_row(a, sm, jc), iend = a.Nq, kdoc = 0;
    const int wfirst = at_first_row(a, sm, j0), wall = at_first_row(a, sm, min(j0 + 31, sm.klen - 1));
    AtDocs docs = {0, 0, true};
    const int* ranges = nullptr;
    if (a.documents) {
        ranges = g.ranges + (long long)b * ((a.Nk + AT_KT - 1) / AT_KT) * 2;
        kdoc = a.documents[(long long)b * a.documents_stride + jc];
        docs = at_doc_range(kdoc);
        imin = kdoc < 0 ? 0x7fffffff : max(imin, -sm.start);
        iend = min(iend, a.Nk - sm.start);
    }
    const long long heads = (long long)b * a.Hq + khead * G;
    float amax = 0.f;
    for (int tb = max(wfirst, 0) / AT_QT; tb < ntile; tb += 64) {
        const int t = tb + lane;
        AtRange r = {0, 0};
        if (ranges && t < ntile) r = at_row_docs(a, sm, ranges, t);
        const bool some = t < ntile && at_meet(r, docs.lo, docs.hi), all = some && t * AT_QT >= wall && docs.one && r.lo == docs.lo && r.hi == docs.lo;
        float tile = 0.f;
        if (some)
            for (int gi = 0; gi < G; ++gi) {
                const float* groups = g.gmax + (heads + gi) * g.ngroup;
                tile = fmaxf(tile, fmaxf(groups[2 * t], groups[min(2 * t + 1, g.ngroup - 1)]));
            }
        amax = fmaxf(amax, at_wave_max(all ? tile : 0.f));
        for (unsigned long long todo = __ballot(some && !all); todo; todo &= todo - 1) {
            const int l = __builtin_ctzll(todo), i0 = (tb + l) * AT_QT, i = i0 + lane;
            const int lo = __builtin_amdgcn_readlane(r.lo, l), hi = __builtin_amdgcn_readlane(r.hi, l);
            if (lo == hi && !__ballot(imin > i0 && imin < i0 + AT_QT)) {
                const float m = at_lane(tile, l);
                amax = fmaxf(amax, imin <= i0 && kdoc == lo ? m : 0.f);
                continue;
            }
            float m = 0.f;
            if (i < iend) for (int gi = 0; gi < G; ++gi) m = fmaxf(m, g.amax[(heads + gi) * a.Nq + i]);
            row_max[wave][lane] = m;
            row_doc[wave][lane] = ranges ? at_row_doc(a, sm, b, i) : 0;
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            const int from = imin - i0 - 32 * hh;
#pragma unroll
            for (int s = 0; s < 32; s += 4) {
                const float4 x = *reinterpret_cast<const float4*>(&row_max[wave][32 * hh + s]);
                const int4 d = *reinterpret_cast<const int4*>(&row_doc[wave][32 * hh + s]);
                amax = fmaxf(amax, s >= from && d.x == kdoc ? x.x : 0.f);
                amax = fmaxf(amax, s + 1 >= from && d.y == kdoc ? x.y : 0.f);
                amax = fmaxf(amax, s + 2 >= from && d.z == kdoc ? x.z : 0.f);
                amax = fmaxf(amax, s + 3 >= from && d.w == kdoc ? x.w : 0.f);
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");             // the next tile's go to the same place
        }
    }
    amax = at_xhalf_max(amax);
    if (hh == 0 && j < sm.klen) g.kmax[(long long)bh * a.Nk + j] = amax;
}

int att_launch_key_amax(const AttArgs& a, const BwdGeo& geo, hipStream_t st)
{
    BwdGeo g = geo;
    g.nbh = a.B * a.Hk;
    hipLaunchKernelGGL(att_key_amax_kernel, dim3((unsigned)((a.Nk + 127) / 128 * g.nbh)), dim3(256), 0, st, a, g);
    return hipGetLastError() == hipSuccess ? ADK_OK : ADK_ELAUNCH;
}
