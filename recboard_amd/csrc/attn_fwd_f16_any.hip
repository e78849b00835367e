#include "attn_fwd.inc"

template int attn::fwd_launch<re_f16, false>(const args&, const fwd_out&, const fwd_plan&, hipStream_t);
