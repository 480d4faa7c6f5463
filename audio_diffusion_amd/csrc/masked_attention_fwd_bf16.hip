// bf16 instantiations of masked_attention_fwd.inc, and the document ranges that every kernel of the family reads
#include "masked_attention_fwd.inc"

int att_forward_bf16(const AttArgs& a, void* o_low, void* ws, hipStream_t st) { return att_forward_t<bf16_t>(a, o_low, ws, st); }

// smallest and largest document of every 64 keys (padding counts as -1): a tile whose range misses a block's documents is
// skipped without being loaded
__global__ __launch_bounds__(64) void att_doc_ranges_kernel(const AttArgs a, int2* out, int tiles)
{
    const int t = blockIdx.x, b = blockIdx.y, j = min(t * AT_KT + (int)threadIdx.x, a.Nk - 1);
    const int doc = a.documents[(long long)b * a.documents_stride + j];
    int lo = max(doc, -1), hi = lo;
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) { lo = min(lo, __shfl_xor(lo, m, 64)); hi = max(hi, __shfl_xor(hi, m, 64)); }
    if (threadIdx.x == 0) out[(long long)b * tiles + t] = make_int2(lo, hi);
}

int att_launch_doc_ranges(const AttArgs& a, int* ranges, hipStream_t st)
{
    const int tiles = att_key_tiles(a);
    hipLaunchKernelGGL(att_doc_ranges_kernel, dim3(tiles, a.B), dim3(64), 0, st, a, reinterpret_cast<int2*>(ranges), tiles);
    return hipGetLastError() == hipSuccess ? ADK_OK : ADK_ELAUNCH;
}

long long att_forward_workspace(const AttArgs& a)
{
    const AtStepPlan p = at_step_plan(a);
    return att_doc_bytes(a) + (p.nsplit > 1 ? (long long)a.B * a.Nq * a.Hq * p.nsplit * (a.D + 2) * 4 : 0);
}
