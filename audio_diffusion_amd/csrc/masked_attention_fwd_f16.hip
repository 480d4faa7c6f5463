// f16 instantiations of masked_attention_fwd.inc
#include "masked_attention_fwd.inc"

int att_forward_f16(const AttArgs& a, void* o_low, void* ws, hipStream_t st) { return att_forward_t<f16_t>(a, o_low, ws, st); }
