// The launch of attention's forward kernels, between the entry point (attn_fwd.hip) and the instances for each type, aligned and
// not (attn_fwd_*.hip).
#pragma once
#include "attn_common.h"

namespace attn {

struct fwd_out {
    void* o;
    int64_t os[3];                 // batch, head, row
    float* stats;                  // [reference score, log sum relative to it][B][Hq][Sq]
    void* low;                     // [B][Hq][Sq][low_len(D)]: what rounding took from o; null: not wanted
    float* part;                   // [splits][B][Hq][Sq][D], then [splits][B][Hq][Sq][2]; null: one split
    order ord;                     // units: workgroup heads of all sequences; tiles: query tiles x splits
    int32_t splits, tiles, heads, pg;        // heads: workgroup heads per sequence; pg: query heads that share a workgroup's rows
};

struct fwd_plan {
    int wq, wk, pg, tiles, heads, splits, bk;
    bool mod, vec;
    int dp;
    size_t lds, part;     // bytes of LDS; of workspace
};

template <class T, bool VEC>
int fwd_launch(const args& a, const fwd_out& f, const fwd_plan& p, hipStream_t st);

}  // namespace attn
