// bf16 instantiations of masked_attention_bwd.inc
#include "masked_attention_bwd.inc"

int att_backward_bf16(const AttArgs& a, void* ws, hipStream_t st) { return att_backward_t<bf16_t>(a, ws, st); }

long long att_backward_workspace(const AttArgs& a)
{
    return att_doc_bytes(a) + att_round((long long)a.B * a.Hq * a.Nq * 4) * (a.dtype == ADK_F16 ? 2 : 1) + att_round((long long)a.B * a.Hq * att_bwd_qtiles(a) * 4) + att_bwd_part(a);
}
