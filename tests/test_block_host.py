"""CPU: what the transformer-block entry points refuse, and their workspace sizes: host logic, nothing is launched."""
import ctypes

import pytest
import torch

from recboard_amd import lib, ops

EINVAL, EWORKSPACE, EUNSUPPORTED = -1, -2, -4
P = ctypes.c_void_p(4096)                      # a pointer that nothing reads


def desc(**kw):
    d = ops._Attention()
    d.q = d.k = d.v = 4096
    d.B, d.Hq, d.Hkv, d.Sq, d.Sk, d.D = 2, 8, 2, 100, 100, 64
    for s in (d.q_stride, d.k_stride, d.v_stride):
        s[0], s[1], s[2] = 6400 * 8, 6400, 64
    d.scale, d.dtype = 0.125, 1
    for k, v in kw.items():
        setattr(d, k, v)
    return d


def fwd(d, out=P, stats=P, ws=P, n=1 << 40, low=None):
    st = (ctypes.c_int64 * 3)(51200, 64, 512)
    return lib.load().re_attention_fwd(ctypes.addressof(d), out, st, stats, low, ws, n, None)


def bwd(d, n=1 << 40, dtable=None):
    st = (ctypes.c_int64 * 3)(51200, 64, 512)
    return lib.load().re_attention_bwd(ctypes.addressof(d), P, st, P, None, P, st, P, st, P, st, P, st, dtable, P, n, None)


@pytest.mark.parametrize("bad,code", [({"D": 0}, EINVAL), ({"D": 129}, EUNSUPPORTED), ({"Hkv": 3}, EINVAL), ({"Hkv": 0}, EINVAL), ({"B": -1}, EINVAL), ({"dtype": 3}, EINVAL),
                                      ({"scale": 0.0}, EINVAL), ({"scale": float("nan")}, EINVAL), ({"scale": -1.0}, EINVAL), ({"Sk": 1 << 30}, EUNSUPPORTED),
                                      ({"mask_kind": 1}, EINVAL), ({"mask": 4096}, EINVAL), ({"mask": 4096, "mask_kind": 5}, EINVAL), ({"table": 4096}, EINVAL),
                                      ({"table": 4096, "bucket_map": 4096, "buckets": 257, "max_distance": 8}, EUNSUPPORTED),
                                      ({"table": 4096, "bucket_map": 4096, "buckets": 8, "max_distance": 1025}, EUNSUPPORTED),
                                      ({"table": 4096, "bucket_map": 4096, "buckets": 8, "max_distance": 8, "table_dtype": 9}, EINVAL), ({"q": None}, EINVAL),
                                      ({"k": None}, EINVAL)])
def test_attention_refuses_what_it_cannot_do(bad, code):
    assert fwd(desc(**bad)) == code and bwd(desc(**bad)) == code


def test_attention_refuses_missing_outputs_and_short_workspaces():
    L = lib.load()
    assert fwd(desc(), out=None) == EINVAL and fwd(desc(), stats=None) == EINVAL
    assert L.re_attention_fwd(None, P, None, P, None, P, 0, None) == EINVAL
    assert fwd(desc(), low=ctypes.c_void_p(4104)) == EINVAL
    one = desc(Sq=1, Sk=16384)
    need = L.re_attention_fwd_workspace_bytes(ctypes.addressof(one))
    assert need > 0 and fwd(one, n=need - 1) == EWORKSPACE and fwd(one, ws=None) == EWORKSPACE
    assert L.re_attention_fwd_workspace_bytes(ctypes.addressof(desc(B=64, Sq=2048))) == 0
    need = L.re_attention_bwd_workspace_bytes(ctypes.addressof(desc()))
    assert need >= 2 * 8 * 100 * 4 and bwd(desc(), n=need - 1) == EWORKSPACE
    assert bwd(desc(), dtable=P) == EINVAL                     # a bias gradient without a bias
    assert fwd(desc(B=0)) == 0 and fwd(desc(Sq=0)) == 0 and bwd(desc(B=0)) == 0


def test_norm_and_bias_refuse_what_they_cannot_do():
    L = lib.load()
    assert L.re_layer_norm_fwd(P, None, None, None, 4, 0, 1e-5, 0, 0, P, None, None, None, None) == EINVAL
    assert L.re_layer_norm_fwd(P, None, None, None, 4, 8, 1e-5, 7, 0, P, None, None, None, None) == EINVAL
    assert L.re_layer_norm_fwd(P, None, None, None, 4, (1 << 24) + 1, 1e-5, 0, 0, P, None, None, None, None) == EUNSUPPORTED
    assert L.re_layer_norm_fwd(None, None, None, None, 4, 8, 1e-5, 0, 0, P, None, None, None, None) == EINVAL
    assert L.re_layer_norm_fwd(None, None, None, None, 0, 8, 1e-5, 0, 0, None, None, None, None, None) == 0
    n = L.re_layer_norm_bwd_workspace_bytes(100, 64)
    assert n > 0 and L.re_layer_norm_bwd(P, P, None, P, P, None, 100, 64, 0, 0, P, P, P, P, n - 1, None) == EWORKSPACE
    assert L.re_relative_bias_fwd(P, P, 257, 128, 4, 8, 8, 0, 0, P, None) == EUNSUPPORTED
    assert L.re_relative_bias_fwd(P, P, 32, 0, 4, 8, 8, 0, 0, P, None) == EINVAL
    assert L.re_relative_bias_fwd(None, P, 32, 128, 4, 8, 8, 0, 0, P, None) == EINVAL
    n = L.re_relative_bias_bwd_workspace_bytes(4, 100, 32)
    assert n > 0 and L.re_relative_bias_bwd(P, P, 32, 128, 4, 100, 8, 0, 0, P, 0, P, n - 1, None) == EWORKSPACE


def test_python_front_end_refuses_cpu_tensors():
    x = torch.randn(2, 2, 4, 8)
    for call in (lambda: ops.attention_fwd(x, x, x), lambda: ops.layer_norm_fwd(x), lambda: ops.relative_bias_fwd(x[0, 0], torch.zeros(3, dtype=torch.int32), 2, 2)):
        with pytest.raises(RuntimeError):
            call()


def test_relative_buckets_against_exact_fractions():
    """A bucket's first distance is the least n with (n / exact)^steps >= (max / exact)^m."""
    from fractions import Fraction
    for nb, far, both in ((32, 128, True), (8, 40, False), (64, 256, True), (16, 100, True), (2, 5, False), (4, 2, True)):
        m = ops.relative_buckets(nb, far, both, device="cpu").tolist()
        side = nb // 2 if both else nb
        exact, steps = side // 2, side - side // 2
        for n in range(far + 1):
            want = n if n < exact else exact + max(x for x in range(steps) if Fraction(n, exact) ** steps >= Fraction(far, exact) ** x)
            assert m[far - n] == want
            if n:
                assert m[far + n] == (side + want if both else 0)
