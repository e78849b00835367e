"""GPU: attention and its backward pass against the definition in 64 bits (materialised, one sequence and head at a time).

Tolerances, per element, from the arithmetic.  u = eps / 2 of the inputs' type (fp32: 2^-24), f = 2^-24.
A score is a chain of D <= 128 fp32 products and sums, the exponent's scaling and a 1-ulp-class exponential: its error e_s <= (D + 8) f (|q| . |k|) scale
+ 4 f (|bias| + |mask| + |lse| + 2), and P is off by the factor e_s + 4 f.  P (and dS) are rounded once, u, before their products, and a
product sums at most n = Sk (Sq, Sq * group) terms in fp32: n f of the sum of magnitudes at the worst, (64 + n / 64) f as the tiles add them.
A result is rounded once more, u.  fp16 has a floor: a rounding below 2^-14 is off by half of 2^-24.
Every bound is evaluated with the 64-bit magnitudes of the very inputs."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]
F = 2.0 ** -24


def visible(B, H, Sq, Sk, causal, mask, lens, offs, dev):
    at = torch.arange(Sk, device=dev)
    seen = torch.ones(B, H, Sq, Sk, dtype=torch.bool, device=dev)
    if causal:
        seen &= at <= (offs.view(B, 1, 1, 1) + torch.arange(Sq, device=dev).view(1, 1, Sq, 1))
    if lens is not None:
        seen &= at < lens.view(B, 1, 1, 1)
    if mask is not None:
        seen &= (mask if mask.dtype == torch.bool else mask != -math.inf).expand(B, H, Sq, Sk)
    return seen


def reference(q, k, v, scale=None, causal=False, mask=None, key_lengths=None, q_offset=None, rel_table=None, bucket_map=None, dout=None):
    """64 bits: a dict of (value, bound) pairs."""
    t, dev = q.dtype, q.device
    u = torch.finfo(t).eps / 2
    tiny = 2.0 ** -25 if t == torch.float16 else 2.0 ** -130
    B, H, Sq, D = q.shape
    Sk, G = k.shape[2], H // k.shape[1]
    scale = D ** -0.5 if scale is None else scale
    if not torch.is_tensor(q_offset):
        q_offset = torch.full((B,), Sk - Sq if q_offset is None else q_offset, device=dev)
    seen = visible(B, H, Sq, Sk, causal, mask, key_lengths, q_offset, dev)
    q, k, v = q.double(), k.double().repeat_interleave(G, 1), v.double().repeat_interleave(G, 1)
    any_row = seen.any(2).unsqueeze(-1)                                     # keys that no row sees may hold anything
    k, v = torch.where(any_row, k, 0.0), torch.where(any_row, v, 0.0)
    kT, vT = k.transpose(2, 3).contiguous(), v.transpose(2, 3).contiguous()
    s = q @ kT * scale
    es = (D + 8) * F * scale * (q.abs() @ kT.abs())
    extra = torch.zeros_like(s)
    if rel_table is not None:
        far = bucket_map.numel() // 2
        d = (torch.arange(Sk, device=dev) - torch.arange(Sq, device=dev).unsqueeze(1)).unsqueeze(0) - q_offset.view(B, 1, 1)
        ids = bucket_map[d.clamp(-far, far) + far].long()
        extra = extra + rel_table.double()[ids].permute(0, 3, 1, 2)
    es = es + 4 * F * extra.abs()
    if mask is not None and mask.dtype != torch.bool:
        m = torch.where(seen, mask.double().expand_as(s), 0.0)
        extra, es = extra + m, es + 4 * F * m.abs()
    s = torch.where(seen, s + extra, -math.inf)
    none = ~seen.any(3, keepdim=True)
    lse = torch.logsumexp(s.masked_fill(none, 0.0), 3, keepdim=True)
    p = torch.where(seen & ~none, torch.exp(s - lse), 0.0)
    out = p @ v
    es = torch.where(seen, es, 0.0) + 4 * F * (lse.abs() + 2)
    es = es + (p * es).sum(3, keepdim=True)                                 # (the sum that p is divided by is off by its terms' errors)
    n = (64 + Sk / 64) * F
    pe = p * torch.expm1(es.clamp_max(1.0))                                 # P's own error
    out_tol = u * out.abs() + pe @ v.abs() + (u + n) * (p @ v.abs()) + tiny * (1 + v.abs().sum(2, keepdim=True))
    r = {"out": (out, out_tol), "lse": (torch.where(none, -math.inf, lse).squeeze(3), (es.amax(3) + n) + F * lse.abs().squeeze(3))}
    if dout is None:
        return r
    g = torch.where(none, 0.0, dout.double())
    dp = g @ vT
    delta = (p * dp).sum(3, keepdim=True)
    ds = p * (dp - delta)
    # delta comes from the output and what rounding took from it (u^2 is left): dO . (out + its error before rounding)
    e_delta = (g.abs() * (out_tol - u * out.abs() * (1 - u))).sum(3, keepdim=True) + D * F * (g.abs() * out.abs()).sum(3, keepdim=True)
    e_dp = (D + 4) * F * (g.abs() @ vT.abs())
    dse = pe * (dp - delta).abs() + (p + pe) * (e_dp + e_delta)
    mag_s = ds.abs() + dse
    Gk = lambda x: x.view(B, H // G, G, Sk, D).sum(2)  # noqa: E731
    nq = (64 + Sq * G / 64) * F
    dq = ds @ k * scale
    r["dq"] = (dq, u * dq.abs() + scale * (dse @ k.abs() + (u + n) * (mag_s @ k.abs()) + tiny * k.abs().sum(2, keepdim=True)) + tiny)
    T = lambda x: x.transpose(2, 3).contiguous()  # noqa: E731
    dk, dv = Gk(T(ds) @ q) * scale, Gk(T(p) @ g)
    r["dk"] = (dk, u * dk.abs() + scale * Gk(T(dse) @ q.abs() + (u + nq) * (T(mag_s) @ q.abs()) + tiny * q.abs().sum(2, keepdim=True)) + tiny)
    r["dv"] = (dv, u * dv.abs() + Gk(T(pe) @ g.abs() + (u + nq) * (T(p + pe) @ g.abs()) + tiny * g.abs().sum(2, keepdim=True)) + tiny)
    if rel_table is not None:
        member = [(ids == b).unsqueeze(1) for b in range(rel_table.shape[0])]
        dt = torch.stack([(ds * m).sum((0, 2, 3)) for m in member])
        # (a chain: diagonals of 32, a wave's blocks, 2 R + 1 distances, the workgroups: at most 2^12 serial additions)
        mag = torch.stack([(dse * m).sum((0, 2, 3)) + 2.0 ** -12 * (mag_s * m).sum((0, 2, 3)) for m in member])
        r["dtable"] = (dt, torch.finfo(rel_table.dtype).eps / 2 * dt.abs() + mag + tiny)
    return r


def compare(got, want, name):
    value, tol = want
    assert got.shape == value.shape, name
    finite = torch.isfinite(value)
    assert torch.equal(got[~finite].double(), value[~finite]), name
    off = (got.double() - value).abs()[finite]
    assert (off <= tol[finite]).all(), (name, float((off - tol[finite]).max()), float((off / tol[finite].clamp_min(1e-300)).max()))


def check(q, k, v, dout=None, **how):
    from recboard_amd import ops
    out, stats = ops.attention_fwd(q, k, v, **how)
    want = reference(q, k, v, dout=dout, **how)
    compare(out, want["out"], "out")
    lse = stats[0] + stats[1]
    lean, two = ops.attention_fwd(q, k, v, need_backward=False, **how)
    assert torch.equal(lean, out) or not torch.isfinite(out).all()
    assert two.shape[0] == 2 and torch.equal(two, stats[:2])
    compare(lse, want["lse"], "lse")
    if dout is None:
        return out, lse
    grads = ops.attention_bwd(dout, q, k, v, out, stats, **how)
    for name, g in zip(("dq", "dk", "dv", "dtable"), grads):
        if g is not None:
            compare(g, want[name], name)
    return (out, lse) + tuple(grads)


def make(B, H, Hkv, Sq, Sk, D, t, seed=0, packed=False):
    g = torch.Generator(device="cuda").manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=g, device="cuda").to(t)  # noqa: E731
    if packed:
        q, k, v = n(B, Sq, H + 2 * Hkv, D).transpose(1, 2).split([H, Hkv, Hkv], 1)
    else:
        q, k, v = n(B, H, Sq, D), n(B, Hkv, Sk, D), n(B, Hkv, Sk, D)
    return q, k, v, n(B, Sq, H, D).transpose(1, 2)


def rel(H, t, buckets=32, distance=128, bidirectional=True):
    from recboard_amd import ops
    g = torch.Generator(device="cuda").manual_seed(5)
    return {"rel_table": torch.randn(buckets, H, generator=g, device="cuda").to(t), "bucket_map": ops.relative_buckets(buckets, distance, bidirectional)}


@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("B,H,Hkv,Sq,Sk,D", [(1, 1, 1, 1, 1, 1), (2, 2, 2, 50, 50, 16), (1, 2, 1, 33, 65, 32), (2, 4, 2, 129, 129, 64), (1, 3, 1, 70, 200, 80), (1, 2, 2, 257, 300, 128),
                                             (1, 2, 2, 40, 31, 20), (1, 1, 1, 64, 7, 7), (1, 6, 2, 5, 100, 96), (1, 2, 1, 200, 190, 33)])
def test_attention_matches_the_definition(t, causal, B, H, Hkv, Sq, Sk, D):
    q, k, v, dout = make(B, H, Hkv, Sq, Sk, D, t, seed=D + Sq)
    check(q, k, v, dout, causal=causal)


@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("Sq,D", [(50, 16), (150, 64), (70, 20)])
def test_attention_on_a_joint_projection_with_padding_that_leaves_rows_empty(t, Sq, D):
    q, k, v, dout = make(3, 4, 2, Sq, Sq, D, t, packed=True)
    n = torch.tensor([Sq, 1, Sq // 2], device="cuda")
    left = (torch.arange(Sq, device="cuda") >= (Sq - n).unsqueeze(1)).view(3, 1, 1, Sq)
    out, lse, dq, dk, dv, _ = check(q, k, v, dout, causal=True, mask=left)
    assert not out[1, :, :Sq - 1].any() and lse[1, :, 0].isinf().all() and not dq[1, :, :Sq - 1].any() and not dk[1, :, :Sq - 1].any()
    check(q, k, v, dout, mask=left)
    none = torch.zeros(3, 1, 1, Sq, dtype=torch.bool, device="cuda")
    out, lse, dq, dk, dv, _ = check(q, k, v, dout, mask=none)
    assert not out.any() and not dq.any() and not dk.any() and not dv.any()


@pytest.mark.parametrize("t", TYPES, ids=str)
def test_attention_masks_of_every_kind(t):
    q, k, v, dout = make(2, 4, 2, 75, 130, 64, t)
    g = torch.Generator(device="cuda").manual_seed(1)
    rand = lambda *s: torch.rand(*s, generator=g, device="cuda")  # noqa: E731
    check(q, k, v, dout, mask=rand(2, 4, 75, 130) < 0.5)
    check(q, k, v, dout, mask=(rand(1, 4, 1, 130) < 0.5))
    check(q, k, v, dout, mask=(rand(75, 1) < 0.7))                           # rows that see nothing
    check(q, k, v, dout, mask=(rand(130, 75) < 0.5).t())                      # a transposed view
    add = rand(2, 1, 75, 130) * 4 - 2
    for mt in TYPES:
        check(q, k, v, dout, mask=add.to(mt))
        low = torch.where(rand(75, 130) < 0.3, torch.finfo(mt).min, 0.0).to(mt)
        low[3] = 0.0
        low[:, 5] = 0.0                                                       # (each row keeps a key: the others are exact zeros)
        check(q, k, v, dout, mask=low)
        check(q, k, v, dout, mask=torch.where(rand(2, 1, 75, 130) < 0.3, -math.inf, 0.5).to(mt), causal=True)


def test_attention_rows_whose_additive_mask_is_the_lowest_value_everywhere_are_uniform():
    """score + lowest = lowest for every key (the score is below half a step of it): the mean of v, in 32 and in 64 bits."""
    q, k, v, dout = make(1, 2, 2, 40, 70, 32, torch.float32)
    mask = torch.zeros(40, 70, device="cuda")
    mask[7] = torch.finfo(torch.float32).min
    from recboard_amd import ops
    out, stats = ops.attention_fwd(q, k, v, mask=mask)
    assert (out[:, :, 7].double() - v.double().mean(2)).abs().max() < 1e-5
    assert torch.isfinite(out).all()
    # a row of zeros in q has the same probabilities: its gradients, except that dk takes the true row of q with a weight of dS
    q0 = q.clone()
    q0[:, :, 7] = 0.0
    want = reference(q0, k, v, dout=dout)
    dq, dk, dv, _ = ops.attention_bwd(dout, q, k, v, out, stats, mask=mask)
    compare(out, want["out"], "out")
    compare(dq, want["dq"], "dq")
    compare(dv, want["dv"], "dv")


@pytest.mark.parametrize("t", TYPES, ids=str)
def test_attention_ignores_whatever_lies_behind_lengths_and_shut_keys(t):
    q, k, v, dout = make(3, 4, 2, 70, 200, 64, t)
    lens = torch.tensor([200, 0, 77], device="cuda")
    off = torch.tensor([130, 0, 7], device="cuda")
    how = {"causal": True, "key_lengths": lens, "q_offset": off}
    clean = check(q, k, v, dout, **how)
    for bad in (float("nan"), float("inf")):
        k2, v2 = k.clone(), v.clone()
        for x in (k2, v2):
            x[1] = bad
            x[2, :, 77:] = bad
        again = check(q, k2, v2, dout, **how)
        assert all(torch.equal(p, r) for p, r in zip(clean[:5], again[:5]))
        mask = torch.ones(3, 1, 1, 200, dtype=torch.bool, device="cuda")
        mask[0, ..., 100:110] = False
        k2[0, :, 100:110] = bad
        v2[0, :, 100:110] = bad
        check(q, k2, v2, dout, mask=mask, **how)
        check(q, k2, v2, dout, mask=torch.where(mask, 0.0, -math.inf), **how)
        # shut for some rows, seen by others: those alone are not finite
        from recboard_amd import ops
        k3, v3 = k.clone(), v.clone()
        v3[0, :, 150] = bad
        out, _ = ops.attention_fwd(q, k3, v3, causal=True)
        sees = torch.arange(70, device="cuda") + 130 >= 150
        want = ops.attention_fwd(q, k, v, causal=True)[0]
        assert torch.isfinite(out[0][:, ~sees]).all() and not torch.isfinite(out[0][:, sees]).any()
        assert (out[0][:, ~sees].double() - want[0][:, ~sees].double()).abs().max() < 0.02


@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("Sq,Sk,D,R", [(50, 50, 16, 128), (150, 333, 64, 40), (90, 90, 20, 1024), (260, 260, 128, 24)])
def test_attention_with_the_position_bias_and_its_gradient(t, Sq, Sk, D, R):
    q, k, v, dout = make(2, 4, 2, Sq, Sk, D, t, seed=R)
    for bidirectional, causal, tt in ((True, False, t), (False, True, torch.float32)):
        check(q, k, v, dout, causal=causal, **rel(4, tt, 32, R, bidirectional))
    mask = (torch.rand(2, 1, 1, Sk, device="cuda") < 0.8)
    check(q, k, v, dout, mask=mask, q_offset=3, **rel(4, t, 256 if R > 128 else 8, R))


@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("B,H,Hkv,Sk,D", [(2, 8, 2, 1000, 128), (1, 4, 4, 2500, 64), (3, 32, 1, 700, 80), (1, 3, 1, 64, 20), (1, 1, 1, 1, 64)])
def test_attention_of_single_tokens_over_a_cache(t, B, H, Hkv, Sk, D):
    for Sq in (1, 3):
        q, k, v, _ = make(B, H, Hkv, Sq, Sk, D, t)
        check(q, k, v)
        lens = torch.randint(min(Sq, Sk), Sk + 1, (B,), device="cuda")
        how = {"causal": True, "key_lengths": lens, "q_offset": lens - Sq}
        check(q, k, v, **how)
        check(q, k, v, **how, **rel(H, t, 32, 128, False))
        k[:, :, Sk // 2], v[:, :, Sk // 2] = float("nan"), float("inf")
        mask = torch.ones(Sk, dtype=torch.bool, device="cuda")
        mask[Sk // 2] = False
        check(q, k, v, mask=mask, **how)


def test_attention_of_a_cache_whose_offsets_pass_32_bits():
    """k and v as views of one long cache: the last sequence's rows lie behind 2^31 elements (and 2^32 bytes)."""
    big = torch.zeros(2 ** 31 + 2 ** 20, dtype=torch.bfloat16, device="cuda")
    Sk, D = 300, 64
    k = big.as_strided((2, 2, Sk, D), (2 ** 31, Sk * D, D, 1))
    v = big.as_strided((2, 2, Sk, D), (2 ** 31, Sk * D, D, 1), 100000)
    for x in (k, v):
        x.copy_(torch.randn(2, 2, Sk, D, device="cuda"))
    q, _, _, dout = make(2, 4, 2, 70, Sk, D, torch.bfloat16)
    check(q, k, v, dout, causal=True)
    check(q[:, :, :1], k, v)
    row = big.as_strided((1, 1, 3, D), (0, 0, 2 ** 30, 1))                    # rows far apart
    row.copy_(torch.randn(1, 1, 3, D, device="cuda"))
    check(q[:1, :1, :40].contiguous(), row, row, dout[:1, :1, :40], causal=False)


def test_attention_strides_broadcasts_and_misalignment():
    q, k, v, dout = make(2, 4, 4, 60, 90, 64, torch.float16)
    a = check(q, k, v, dout)
    off = lambda t: torch.cat([t.new_zeros(1), t.reshape(-1)])[1:].view(t.shape)  # noqa: E731
    b = check(off(q), off(k), off(v), off(dout))
    assert all((x.float() - y.float()).abs().max() < 0.01 for x, y in zip(a[:5], b[:5]))
    one = k[:, :1].expand(2, 4, 90, 64)                                       # a head that all share, by stride 0
    c = check(q, one, one, dout)
    d = check(q, k[:, :1], k[:, :1], dout)
    assert torch.equal(c[0], d[0])
    every = q[..., ::1].permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3)
    assert torch.equal(check(every, k, v, dout)[0], a[0])


def test_attention_of_nothing():
    from recboard_amd import ops
    q, k, v, dout = make(2, 4, 2, 5, 6, 32, torch.bfloat16)
    out, lse = ops.attention_fwd(q, k[:, :, :0], v[:, :, :0])
    assert not out.any() and lse[0].isinf().all()
    dq, dk, dv, _ = ops.attention_bwd(dout, q, k[:, :, :0], v[:, :, :0], out, lse)
    assert not dq.any() and dk.shape == (2, 2, 0, 32)
    out, lse = ops.attention_fwd(q[:, :, :0], k, v)
    assert out.shape == (2, 4, 0, 32)
    dq, dk, dv, _ = ops.attention_bwd(dout[:, :, :0], q[:, :, :0], k, v, out, lse)
    assert not dk.any() and not dv.any()
    out, lse = ops.attention_fwd(q[:0], k[:0], v[:0])
    assert out.shape == (0, 4, 5, 32)


@pytest.mark.parametrize("t", [torch.bfloat16, torch.float16], ids=str)
def test_attention_position_gradient_is_as_exact_as_the_scores(t):
    """The rows of dS sum to zero, so an error of delta does not average out of the bias's gradient: with delta from the rounded output it was 2^-9 of
    |dO| |out| per row.  What is left is the scores' fp32 error and the rounding of P in the output, n * u / sqrt(n) of its terms at random: within
    1.5 roundings of the result in the 2-norm."""
    from recboard_amd import ops
    q, k, v, dout = make(2, 4, 4, 512, 512, 64, t)
    how = rel(4, t)
    out, stats = ops.attention_fwd(q, k, v, **how)
    got = ops.attention_bwd(dout, q, k, v, out, stats, **how)[3].double()
    want = reference(q, k, v, dout=dout, **how)["dtable"][0]
    plain = ops.attention_bwd(dout, q, k, v, out, stats[:2].contiguous(), **how)[3].double()
    near, far = ((x - want).norm() / want.norm() for x in (got, plain))
    assert near < far and near <= 1.5 * torch.finfo(t).eps / 2, (float(near), float(far))


@pytest.mark.parametrize("t", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("Sq,Sk,D", [(150, 333, 64), (50, 50, 16), (260, 260, 128), (1, 700, 80), (90, 90, 20)])
def test_attention_with_a_position_table_rounds_its_output_once(t, Sq, Sk, D):
    """P is carried in two pieces there (u^2 of it is lost), so of the reference's bound the term u (P |v|) becomes u^2 (P |v|)."""
    from recboard_amd import ops
    u = torch.finfo(t).eps / 2
    q, k, v, _ = make(2, 4, 2, Sq, Sk, D, t, seed=Sk)
    for causal in (False, True):
        how = dict(rel(4, t, 32, 40), causal=causal)
        want, tol = reference(q, k, v, **how)["out"]
        tol = tol - (u - u * u) * reference(q, k, v.abs(), **how)["out"][0]
        for train in (False, True):
            out = ops.attention_fwd(q, k, v, need_backward=train, **how)[0]
            assert ((out.double() - want).abs() <= tol).all()


@pytest.mark.parametrize("t", [torch.bfloat16, torch.float16], ids=str)
def test_attention_position_gradient_is_off_by_its_last_rounding(t):
    """Long rows and few buckets: the last rounding is u of each value at most; a tenth of that is left for the 32-bit sums and u^2 in delta."""
    from recboard_amd import ops
    q, k, v, dout = make(2, 1, 1, 2050, 2050, 32, t)
    how = rel(1, t, 32, 64)
    out, stats = ops.attention_fwd(q, k, v, **how)
    got = ops.attention_bwd(dout, q, k, v, out, stats, **how)[3].double()
    want = reference(q, k, v, dout=dout, **how)["dtable"][0]
    assert (got - want).norm() <= 1.1 * torch.finfo(t).eps / 2 * want.norm()


@pytest.mark.parametrize("R", [24, 40, 100])
def test_attention_with_the_position_bias_run_to_run(R):
    q, k, v, _ = make(1, 4, 2, 150, 333, 64, torch.bfloat16)
    from recboard_amd import ops
    how = rel(4, torch.bfloat16, 16, R)
    first = ops.attention_fwd(q, k, v, **how)[0]
    assert all(torch.equal(first, ops.attention_fwd(q, k, v, **how)[0]) for _ in range(20))


@pytest.mark.parametrize("D", [64, 128])
def test_attention_same_bits_again_on_another_stream_and_in_graphs(D):
    from recboard_amd import ops
    from recboard_amd.capture import recording
    q, k, v, dout = make(2, 4, 2, 200, 200, D, torch.bfloat16)
    how = {"causal": True, **rel(4, torch.float32, 32, 64, False)}
    one = q[:, :, :1].contiguous()

    def step():
        out, lse = ops.attention_fwd(q, k, v, **how)
        return (out, ops.attention_fwd(one, k, v)[0]) + ops.attention_bwd(dout, q, k, v, out, lse, **how)
    first = [t.clone() for t in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(p, r) for p, r in zip(first, again))
    graphs, outs = [], []
    for _ in range(2):                                                        # two graphs of the same calls: workspaces of their own
        graphs.append(torch.cuda.CUDAGraph())
        with recording(graphs[-1]):
            outs.append(step())
    for x in range(3):
        q.copy_(torch.randn_like(q))
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        want = step()
        for o in outs:
            assert all(torch.equal(p, r) for p, r in zip(o, want)), x


def test_attention_gradient_against_differences():
    """Central differences of the 64-bit definition along random directions (h = 1e-5: truncation below 1e-8 of the value): the fp32 gradient's
    own bound summed over the direction's magnitudes."""
    q, k, v, dout = make(1, 2, 1, 20, 30, 16, torch.float32)
    how = {"causal": True, **rel(2, torch.float32, 8, 16, False)}
    out, lse, dq, dk, dv, dt = check(q, k, v, dout, **how)
    tols = reference(q, k, v, dout=dout, **how)
    h = 1e-5
    for name, x, g in (("dq", q, dq), ("dk", k, dk), ("dv", v, dv), ("dtable", how["rel_table"], dt)):
        d = torch.randn_like(x).double()

        def loss(c):
            a = [y.double() + c * d if y is x else y.double() for y in (q, k, v, how["rel_table"])]
            return float((reference(*a[:3], **dict(how, rel_table=a[3]))["out"][0] * dout.double()).sum())
        want = (loss(h) - loss(-h)) / (2 * h)
        tol = float((tols[name][1] * d.abs()).sum()) + 1e-6 * (1 + abs(want))
        assert abs(float((g.double() * d).sum()) - want) <= tol, name


def test_attention_refusals():
    from recboard_amd import ops
    q, k, v, dout = make(2, 4, 2, 5, 6, 32, torch.bfloat16)
    m = ops.relative_buckets(32, 128)
    for bad in (lambda: ops.attention_fwd(q, k, v[:, :, :5]), lambda: ops.attention_fwd(q, k[:1], v[:1]), lambda: ops.attention_fwd(q[:, :3], k, v),
                lambda: ops.attention_fwd(q[0], k, v), lambda: ops.attention_fwd(q.transpose(2, 3).contiguous().transpose(2, 3), k, v),
                lambda: ops.attention_fwd(torch.cat([q] * 5, 3), torch.cat([k] * 5, 3), torch.cat([v] * 5, 3)),
                lambda: ops.attention_fwd(q, k, v, scale=0.0), lambda: ops.attention_fwd(q, k, v, mask=torch.ones(7, dtype=torch.bool, device="cuda")),
                lambda: ops.attention_fwd(q, k, v, mask=torch.ones(6, dtype=torch.bool)),
                lambda: ops.attention_fwd(q, k, v, key_lengths=torch.ones(3, dtype=torch.int64, device="cuda")),
                lambda: ops.attention_fwd(q, k, v, q_offset=torch.ones(3, dtype=torch.int64, device="cuda")),
                lambda: ops.attention_fwd(q, k, v, rel_table=torch.ones(32, 4, device="cuda")),
                lambda: ops.attention_fwd(q, k, v, rel_table=torch.ones(32, 3, device="cuda"), bucket_map=m)):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: ops.attention_fwd(q, k.float(), v), lambda: ops.attention_fwd(q.double(), k.double(), v.double()),
                lambda: ops.attention_fwd(q, k, v, mask=torch.ones(6, dtype=torch.int32, device="cuda")),
                lambda: ops.attention_fwd(q, k, v, key_lengths=torch.ones(2, dtype=torch.int32, device="cuda"))):
        with pytest.raises(TypeError):
            bad()
    with pytest.raises(RuntimeError):
        ops.attention_fwd(q.cpu(), k.cpu(), v.cpu())
    out, lse = ops.attention_fwd(q, k, v)
    with pytest.raises(ValueError):
        ops.attention_bwd(dout, q, k, v, out, lse[:1].contiguous())
    with pytest.raises(ValueError):
        ops.attention_bwd(dout[:, :2], q, k, v, out, lse)
