#include "attn_bwd.inc"

template int attn::bwd_launch<float>(const args&, const bwd_io&, const bwd_plan&, hipStream_t);
