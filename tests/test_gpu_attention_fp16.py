"""GPU: attention's fp16 forms where probabilities and gradients are small: fp16 has no normal numbers below 2^-14, fp32 sums do.

Bound: in the 2-norm a result may be off by what rounding the 64-bit value to fp16 costs (its subnormal steps counted), and by one rounding of each
factor on the way, u = 2^-11, independent of each other: sum_j (1 + e_j) x_j y_j with |e_j| <= u is off by u sqrt(sum_j x_j^2 y_j^2) at the most in the root mean square (a uniform rounding's own is
1 / sqrt(3) of u: the rest is left for the fp32 sums)."""
import math

import pytest
import torch

from test_gpu_attention import make, rel

pytestmark = pytest.mark.gpu
U = 2.0 ** -11


def parts(q, k, v, dout, scale, extra=0.0):
    """64 bits, one batch, as many key heads as query heads."""
    q, k, v, g = (x.double() for x in (q, k, v, dout))
    T = lambda x: x.transpose(2, 3).contiguous()  # noqa: E731
    p = torch.softmax(q @ T(k) * scale + extra, 3)
    out = p @ v
    ds = p * (g @ T(v) - (g * out).sum(3, keepdim=True))
    return {"out": (out, (p * p) @ (v * v), 1.0), "dq": (ds @ k * scale, (ds * ds) @ (k * k), scale), "dk": (T(ds) @ q * scale, T(ds * ds) @ (q * q), scale),
            "dv": (T(p) @ g, T(p * p) @ (g * g), 1.0)}


def near(got, want, name):
    value, squares, scale = want
    assert torch.isfinite(got).all(), name
    off = (got.double() - value).norm()
    tol = (value.half().double() - value).norm() + U * scale * squares.sqrt().norm()
    assert off <= tol, (name, float(off / tol), float(off / value.norm()))


@pytest.mark.parametrize("small", [0, 10, 14, 17])
@pytest.mark.parametrize("Sq,Sk,D", [(2048, 2048, 64), (60, 60, 16), (500, 700, 128), (300, 3000, 20)])
def test_gradients_of_a_small_output_gradient(Sq, Sk, D, small):
    """A loss of fp16 training without a large loss scale: dout about 2^-small, dS about 2^-small / Sk."""
    from recboard_amd import ops
    q, k, v, dout = make(1, 2, 2, Sq, Sk, D, torch.float16)
    dout = (dout.float() * 2.0 ** -small).half()
    out, stats = ops.attention_fwd(q, k, v)
    got = ops.attention_bwd(dout, q, k, v, out, stats)
    want = parts(q, k, v, dout, D ** -0.5)
    for g, name in zip(got, ("dq", "dk", "dv")):
        near(g, want[name], name)


@pytest.mark.parametrize("bias", [False, True])
def test_gradients_whose_size_differs_from_row_to_row_and_from_key_to_key(bias):
    """Rows of dout and keys' values over 2^20: each row of dq, each key of dk has a size of its own; the largest are near what fp16 holds."""
    from recboard_amd import ops
    Sq, Sk, D = 333, 700, 64
    q, k, v, dout = make(1, 2, 2, Sq, Sk, D, torch.float16)
    dout = (dout.float() * 2.0 ** -torch.randint(0, 21, (1, 1, Sq, 1), device="cuda")).half()
    v = (v.float() * 2.0 ** (6 - torch.randint(0, 15, (1, 1, Sk, 1), device="cuda"))).half()
    how = rel(2, torch.float32, 8, 16) if bias else {}
    out, stats = ops.attention_fwd(q, k, v, **how)
    got = ops.attention_bwd(dout, q, k, v, out, stats, **how)
    extra = 0.0
    if bias:
        d = (torch.arange(Sk, device="cuda") - torch.arange(Sq, device="cuda").unsqueeze(1) - (Sk - Sq)).clamp(-16, 16) + 16
        extra = how["rel_table"].double()[how["bucket_map"][d].long()].permute(2, 0, 1)
    want = parts(q, k, v, dout, D ** -0.5, extra)
    for g, name in zip(got, ("dq", "dk", "dv")):
        near(g, want[name], name)
        value, squares, scale = want[name]              # ... and row by row, where the rows are long enough for a 2-norm: a row's own rounding and 4 u
        off = (g.double() - value).norm(dim=3)
        tol = (value.half().double() - value).norm(dim=3) + 4 * U * scale * squares.sum(3).sqrt() + 2.0 ** -25 * math.sqrt(D)
        assert (off <= tol).all(), (name, float((off / tol).max()))


def test_a_gradient_too_large_for_fp16_is_infinite_and_its_neighbours_are_not():
    from recboard_amd import ops
    q, k, v, dout = make(1, 1, 1, 100, 120, 64, torch.float16)
    v = v * 200
    dout = dout.clone()
    dout[0, 0, 7] *= 4000
    out, stats = ops.attention_fwd(q, k, v)
    dq, dk, dv, _ = ops.attention_bwd(dout, q, k, v, out, stats)
    want = parts(q, k, v, dout, 0.125)
    value = want["dq"][0]
    assert value[0, 0, 7].abs().max() > 2 * 65504
    rows = torch.arange(100, device="cuda") != 7
    near(dq[:, :, rows], (value[:, :, rows], want["dq"][1][:, :, rows], 0.125), "dq")
    big = value[0, 0, 7].abs() > 1.01 * 65504
    assert torch.equal(dq[0, 0, 7][big].double(), value[0, 0, 7][big].sign() * math.inf) and torch.isfinite(dq[0, 0, 7][value[0, 0, 7].abs() < 0.99 * 65504]).all()


@pytest.mark.parametrize("Sq,Sk", [(64, 16384), (100, 40000)])
def test_value_gradients_of_keys_with_small_probabilities(Sq, Sk):
    """Key by key: P is about 1 / Sk, and for the second half of the keys exp(-6) of that."""
    from recboard_amd import ops
    q, k, v, dout = make(1, 1, 1, Sq, Sk, 64, torch.float16)
    q, k, dout = q.clone(), k.clone(), dout * 64
    q[..., 0], k[:, :, Sk // 2:, 0], k[:, :, :Sk // 2, 0] = 4.0, -12.0, 0.0
    out, stats = ops.attention_fwd(q, k, v)
    dv = ops.attention_bwd(dout, q, k, v, out, stats)[2]
    want = parts(q, k, v, dout, 0.125)["dv"]
    near(dv, want, "dv")
    value, squares, _ = want
    off = (dv.double() - value).norm(dim=3)
    assert (off <= (value.half().double() - value).norm(dim=3) + 4 * U * squares.sum(3).sqrt()).all()


@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("Sq,Sk,D", [(150, 2048, 64), (64, 700, 128), (1, 3000, 64), (3, 1500, 20), (700, 700, 16)])
def test_rows_with_one_key_far_above_the_others(Sq, Sk, D, bias):
    """The first key takes nearly all of every row and has the value 0 (what a trained causal model does with its first token): the output is
    made of the others' probabilities, about exp(-13) = 2^-19 each."""
    from recboard_amd import ops
    q, k, v, dout = make(1, 2, 2, Sq, Sk, D, torch.float16)
    q, k, v = q.clone(), k.clone(), v.clone()
    q[..., 0], k[..., 0], k[:, :, 0] = 4.0, 0.0, 0.0
    k[:, :, 0, 0] = 13.0 / 4.0 * math.sqrt(D)
    v[:, :, 0] = 0.0
    how = {"rel_table": torch.zeros(8, 2, device="cuda"), "bucket_map": ops.relative_buckets(8, 16)} if bias else {}
    want = parts(q, k, v, dout, D ** -0.5)
    out, stats = ops.attention_fwd(q, k, v, **how)
    near(out, want["out"], "out")
    lse = (q.double() @ k.double().transpose(2, 3).contiguous() * D ** -0.5).logsumexp(3)
    assert ((stats[0] + stats[1]).double() - lse).abs().max() < 1e-4
    got = ops.attention_bwd(dout, q, k, v, out, stats, **how)
    near(got[2][:, :, 1:], tuple(x[:, :, 1:] if torch.is_tensor(x) else x for x in want["dv"]), "dv")
