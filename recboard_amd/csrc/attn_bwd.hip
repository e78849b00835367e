// Attention, backward: the entry point, its workspace and the rule that chooses the kernels' shapes (the kernels: attn_bwd.inc).
#include "attn_bwd.h"

namespace attn {

static bwd_plan make_bwd_plan(const args& a, int dtype, bool vec, bool want_table) {
    bwd_plan p{};
    p.vec = vec;
    p.mod = attn_mod(a);
    p.dp = a.D <= 32 ? 32 : a.D <= 64 ? 64 : a.D <= 96 ? 96 : 128;
    p.wq = a.Sq <= 64 ? 2 : 4;
    p.wk = a.Sk <= 64 ? 2 : 4;
    p.qtiles = re_cdiv(a.Sq, 32 * p.wq);
    p.ktiles = re_cdiv(a.Sk, 32 * p.wk);
    const int rows = dtype == RE_F32 ? 32 : 64;                                      // keys of a dq tile
    const bool v_lds = dtype != RE_F32 && p.dp > 64;
    const int qrows = dtype == RE_F32 || v_lds ? 32 : 64;                            // queries of a dk, dv tile
    // dq: two workgroups a compute unit, each with four tiles of keys at least
    const int64_t qwgs = (int64_t)a.B * a.Hq * p.qtiles, qmost = re_cdiv(a.Sk, 256);
    int64_t qs = qwgs >= 384 ? 1 : re_cdiv(512, qwgs);
    qs = qs < qmost ? qs : qmost;
    p.qsplits = (int)(qs < 1 ? 1 : qs > 16 ? 16 : qs);
    // dk, dv: enough workgroups to fill the card twice over (with a triangle, whose workgroups are uneven, four times), each with 512 queries
    // at least
    const int64_t wgs = (int64_t)a.B * a.Hkv * p.ktiles, want = a.causal ? 1024 : 512;
    int64_t splits = p.ktiles == 0 || wgs >= want ? 1 : re_cdiv(want, wgs);
    const int64_t most = (int64_t)a.group * re_cdiv(a.Sq, 64) / 8;
    splits = splits < most ? splits : most;
    p.splits = (int)(splits < 1 ? 1 : splits > 16 ? 16 : splits);
    const int ch = p.dp * (int)re_dtype_size(dtype) / 16;
    const int chp = dtype == RE_F32 ? ch + 1 : ch <= 4 ? 4 : ch <= 8 ? 8 : 16;
    const size_t tiles = (size_t)4 * rows * chp * 16, n_line = 2 * a.R + 1;
    const size_t line = a.table ? line_len(a.R) * sizeof(float) : 0;
    // (the sums by distance; behind the loop a distance's bucket each and a float a lane)
    const size_t by_wave = p.wq * (n_line + 124), by_lane = n_line + 64 * p.wq;
    p.lds_q = tiles + line + (want_table ? (by_wave > by_lane ? by_wave : by_lane) * sizeof(float) : 0);
    p.lds_k = (size_t)(4 * qrows + (v_lds ? 32 * p.wk : 0)) * chp * 16 + 6 * qrows * sizeof(float) + line;
    return p;
}
static size_t delta_bytes(const args& a) { return re_align((size_t)a.B * a.Hq * a.Sq * sizeof(float)); }
static size_t kv_bytes(const args& a, const bwd_plan& p) {
    return p.splits > 1 ? re_align((size_t)p.splits * 2 * a.B * a.Hkv * a.Sk * a.D * sizeof(float)) : 0;
}
static size_t q_bytes(const args& a, const bwd_plan& p) {
    return p.qsplits > 1 ? re_align((size_t)p.qsplits * a.B * a.Hq * a.Sq * a.D * sizeof(float)) : 0;
}
static size_t part_bytes(const args& a, const bwd_plan& p) { return (size_t)a.B * a.Hq * p.qtiles * p.qsplits * a.buckets * sizeof(float); }

}  // namespace attn

extern "C" size_t re_attention_bwd_workspace_bytes(const re_attention* d) {
    attn::args a;
    if (attn_args(d, a) != RE_OK || attn_empty(a)) return 0;
    const attn::bwd_plan p = attn::make_bwd_plan(a, d->dtype, false, true);
    return attn::delta_bytes(a) + attn::kv_bytes(a, p) + attn::q_bytes(a, p) + (a.table ? attn::part_bytes(a, p) : 0);
}

extern "C" int re_attention_bwd(const re_attention* d, const void* out, const int64_t* out_stride, const float* stats, const void* out_low, const void* dout,
                                const int64_t* dout_stride, void* dq, const int64_t* dq_stride, void* dk, const int64_t* dk_stride, void* dv,
                                const int64_t* dv_stride, void* dtable, void* ws, size_t ws_bytes, re_stream_t stream) {
    attn::args a;
    const int rc = attn_args(d, a);
    if (rc != RE_OK) return rc;
    if ((reinterpret_cast<uintptr_t>(out_low) & 15) || !out_stride || !dout_stride || !dq_stride || !dk_stride || !dv_stride || (dtable && !a.table)) return RE_EINVAL;
    if (attn_empty(a)) return (a.B && a.Hq && a.Sk) || (dtable && a.Hq) ? RE_EUNSUPPORTED : RE_OK;      // (no row, but gradients to write: the caller's zeros)
    if (!a.q || !out || !stats || !dout || !dq || (a.Sk > 0 && (!a.k || !a.v || !dk || !dv))) return RE_EINVAL;
    const bool vec = attn_aligned(a, d->dtype, {{a.q, a.qs}, {a.k, a.ks}, {a.v, a.vs}, {out, out_stride}, {dout, dout_stride}, {dq, dq_stride},
                                                {dk, dk_stride}, {dv, dv_stride}});
    const attn::bwd_plan p = attn::make_bwd_plan(a, d->dtype, vec, dtable != nullptr);
    if ((int64_t)a.B * a.Hq * p.qtiles * p.qsplits >= (1ll << 23) || (int64_t)a.B * a.Hkv * p.ktiles * p.splits >= (1ll << 23)) return RE_EUNSUPPORTED;
    const size_t kv = attn::kv_bytes(a, p), qb = attn::q_bytes(a, p), need = attn::delta_bytes(a) + kv + qb + (dtable ? attn::part_bytes(a, p) : 0);
    if (!ws || ws_bytes < need) return RE_EWORKSPACE;
    char* at = (char*)ws + attn::delta_bytes(a);
    attn::bwd_io io{out, d->dtype == RE_F32 ? nullptr : out_low, dout, dq, dk, dv, {}, {}, {}, {}, {}, stats, (float*)ws, kv ? (float*)at : nullptr, p.splits, qb ? (float*)(at + kv) : nullptr,
                    p.qsplits, dtable ? (float*)(at + kv + qb) : nullptr};
    for (int x = 0; x < 3; ++x) {
        io.os[x] = out_stride[x];
        io.dos[x] = dout_stride[x];
        io.dqs[x] = dq_stride[x];
        io.dks[x] = dk_stride[x];
        io.dvs[x] = dv_stride[x];
    }
    re_clear_error();
    hipStream_t st = (hipStream_t)stream;
    const int r = d->dtype == RE_F32 ? attn::bwd_launch<float>(a, io, p, st) : d->dtype == RE_BF16 ? attn::bwd_launch<re_bf16>(a, io, p, st)
                                                                                              : attn::bwd_launch<re_f16>(a, io, p, st);
    if (r != RE_OK) return r;
    if (dtable)
        hipLaunchKernelGGL(rb_reduce_k, dim3((unsigned)a.Hq), dim3(1024), 0, st, io.part, (int64_t)a.B, (int64_t)a.Hq, p.qtiles * p.qsplits, a.buckets, dtable,
                           a.tdtype);
    return re_launch_status();
}
