// f16 instantiations of masked_attention_bwd.inc
#include "masked_attention_bwd.inc"

int att_backward_f16(const AttArgs& a, void* ws, hipStream_t st) { return att_backward_t<f16_t>(a, ws, st); }
