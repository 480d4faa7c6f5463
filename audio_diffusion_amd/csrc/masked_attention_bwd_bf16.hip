// bf16 instantiations of masked_attention_bwd.inc
#include "masked_attention_bwd.inc"

int att_backward_bf16(const AttArgs& a, const void* o_low, void* ws, hipStream_t st) { return att_backward_t<bf16_t>(a, o_low, ws, st); }

long long att_backward_workspace(const AttArgs& a)
{
    const long long rows = att_round((long long)a.B * a.Hq * a.Nq * 4);
    const long long f16 = 2 * rows + att_round((long long)a.B * a.Hq * att_bwd_groups(a) * 4) + att_round((long long)a.B * a.Hk * a.Nk * 4);
    return att_doc_bytes(a) + rows + (a.dtype == ADK_F16 ? f16 : 0) + att_bwd_part(a);
}
