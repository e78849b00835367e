// Attention, forward: the entry point and the rule that chooses a kernel's shape (the kernels: attn_fwd.inc).
#include "attn_fwd.h"

namespace attn {

static size_t lds_bytes(int dtype, int dp, int bk, const args& a, int pg) {
    const int ch = dp * (int)re_dtype_size(dtype) / 16;
    const int chp = dtype == RE_F32 ? ch + 1 : ch <= 4 ? 4 : ch <= 8 ? 8 : 16;
    size_t n = (size_t)4 * bk * chp * 16;
    if (a.table) n += (size_t)pg * line_len(a.R) * sizeof(float);
    return n;
}

static fwd_plan make_plan(const args& a, int dtype, bool vec) {
    fwd_plan p{};
    p.vec = vec;
    p.mod = attn_mod(a);
    p.dp = a.D <= 32 ? 32 : a.D <= 64 ? 64 : a.D <= 96 ? 96 : 128;
    // few rows: the heads that share keys are one workgroup's rows and its waves go along the keys
    const int64_t packed = (int64_t)a.group * a.Sq;
    const bool few = packed <= 32 && (!a.table || (int64_t)a.group * line_len(a.R) <= 4096);
    p.pg = few ? a.group : 1;
    p.wk = !few && a.Sq > 32 ? 1 : 2;
    p.wq = p.wk > 1 ? 1 : a.Sq <= 64 ? 2 : 4;
    p.bk = 32 * (dtype == RE_F32 || p.wk > 1 ? 1 : 2) * p.wk;
    p.heads = p.pg > 1 ? a.Hkv : a.Hq;
    p.tiles = (int)re_cdiv((int64_t)p.pg * a.Sq, 32 * p.wq);
    // keys are split until two workgroups a compute unit are there, each with at least two tiles
    const int64_t wgs = (int64_t)a.B * p.heads * p.tiles;
    int64_t splits = wgs >= 512 ? 1 : re_cdiv(512, wgs);
    const int64_t most = re_cdiv(a.Sk, 2 * p.bk);
    splits = splits < most ? splits : most;
    p.splits = (int)(splits < 1 ? 1 : splits > 128 ? 128 : splits);
    p.lds = lds_bytes(dtype, p.dp, p.bk, a, p.pg);
    p.part = p.splits > 1 ? (size_t)p.splits * a.B * a.Hq * a.Sq * (a.D + 2) * sizeof(float) : 0;
    return p;
}

template <class T>
static int fwd_any(const args& a, const fwd_out& f, const fwd_plan& p, hipStream_t st) {
    return p.vec ? fwd_launch<T, true>(a, f, p, st) : fwd_launch<T, false>(a, f, p, st);
}

}  // namespace attn

extern "C" size_t re_attention_fwd_workspace_bytes(const re_attention* d) {
    attn::args a;
    if (attn_args(d, a) != RE_OK || attn_empty(a)) return 0;
    return attn::make_plan(a, d->dtype, false).part;
}

extern "C" int re_attention_fwd(const re_attention* d, void* out, const int64_t* out_stride, float* stats, void* out_low, void* ws, size_t ws_bytes,
                                re_stream_t stream) {
    attn::args a;
    const int rc = attn_args(d, a);
    if (rc != RE_OK) return rc;
    if (!out_stride || (reinterpret_cast<uintptr_t>(out_low) & 15)) return RE_EINVAL;
    if (attn_empty(a)) return RE_OK;
    if (!a.q || !out || !stats || (a.Sk > 0 && (!a.k || !a.v))) return RE_EINVAL;
    const bool vec = attn_aligned(a, d->dtype, {{a.q, a.qs}, {a.k, a.ks}, {a.v, a.vs}, {out, out_stride}});
    const attn::fwd_plan p = attn::make_plan(a, d->dtype, vec);
    if ((int64_t)a.B * p.heads * p.tiles * p.splits >= (1ll << 23)) return RE_EUNSUPPORTED;
    if (p.part && (!ws || ws_bytes < p.part)) return RE_EWORKSPACE;
    const attn::fwd_out f{out, {out_stride[0], out_stride[1], out_stride[2]}, stats, d->dtype == RE_F32 ? nullptr : out_low, p.part ? (float*)ws : nullptr,
                          attn_order((int64_t)a.B * p.heads, (int64_t)p.tiles * p.splits, p.pg > 1 ? 1 : a.group), p.splits, p.tiles, p.heads, p.pg};
    re_clear_error();
    hipStream_t st = (hipStream_t)stream;
    const int r = d->dtype == RE_F32 ? attn::fwd_any<float>(a, f, p, st) : d->dtype == RE_BF16 ? attn::fwd_any<re_bf16>(a, f, p, st) : attn::fwd_any<re_f16>(a, f, p, st);
    return r != RE_OK ? r : re_launch_status();
}
