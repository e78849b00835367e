#include "attn_bwd.inc"

template int attn::bwd_launch<re_bf16>(const args&, const bwd_io&, const bwd_plan&, hipStream_t);
