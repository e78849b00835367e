// The launch of attention's backward kernels, between the entry point (attn_bwd.hip) and the instances for each type (attn_bwd_*.hip).
#pragma once
#include "attn_common.h"

namespace attn {

struct bwd_io {
    const void *o, *low, *dout;    // low: what rounding took from o (attn_common.h); null: nothing is known of it
    void *dq, *dk, *dv;
    int64_t os[3], dos[3], dqs[3], dks[3], dvs[3];
    const float* stats;            // the forward's [max, log sum][B][Hq][Sq]
    float* delta;                  // [B][Hq][Sq]: rowsum(dO O), written by the dq kernel, read by the dk / dv kernel
    float* kv_part;                // [splits][dk, dv][B][Hkv][Sk][D], fp32; null: one split
    int32_t splits;                // parts of the queries (of all heads that share a key head)
    float* q_part;                 // [qsplits][B][Hq][Sq][D], fp32; null: one split
    int32_t qsplits;               // parts of the keys for dq
    float* part;                   // [B][Hq][tiles x qsplits][buckets]: the bias gradient of a workgroup; null: none wanted
};
struct bwd_plan {
    int wq, wk;                    // waves of the dq / of the dk, dv kernel: 32 queries / 32 keys each
    int dp;
    bool mod, vec;
    int64_t qtiles, ktiles;
    int splits, qsplits;           // of the queries for dk, dv; of the keys for dq
    size_t lds_q, lds_k;
};

template <class T>
int bwd_launch(const args& a, const bwd_io& io, const bwd_plan& p, hipStream_t st);

}  // namespace attn
