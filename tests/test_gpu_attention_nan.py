"""GPU: attention where a NaN lies in a place that a row may see: that row's results are NaN, whatever way its keys are cut into parts, and no other
row's results change."""
import pytest
import torch

from test_gpu_attention import TYPES, make, reference, rel

pytestmark = pytest.mark.gpu
NAN = float("nan")


@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("B,H,Hkv,Sq,Sk,D", [(2, 4, 2, 1, 1000, 64), (1, 8, 2, 1, 3001, 128), (2, 2, 2, 3, 700, 20), (1, 2, 2, 150, 900, 64), (2, 4, 2, 1, 60, 64), (2, 4, 2, 70, 60, 64)],
                         ids=lambda x: str(x))
def test_nan_in_a_row_of_q_stays_in_that_row(t, B, H, Hkv, Sq, Sk, D):
    """Long caches are cut into parts and joined, short ones are not: the answer is the same either way."""
    from recboard_amd import ops
    q, k, v, _ = make(B, H, Hkv, Sq, Sk, D, t)
    clean, stats = ops.attention_fwd(q, k, v)
    q2 = q.clone()
    q2[0, 1, Sq - 1, D // 2] = NAN
    out, st = ops.attention_fwd(q2, k, v)
    hit = torch.zeros(B, H, Sq, dtype=torch.bool, device="cuda")
    hit[0, 1, Sq - 1] = True
    assert out[hit].isnan().all()
    # the neighbours in a tile may be made again row by row: another order of the same sums, so the definition's own bound
    value, tol = reference(q, k, v)["out"]
    assert ((out.double() - value).abs() <= tol)[~hit].all()
    assert torch.isfinite(st[:2][:, ~hit]).all()


@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("Sq,Sk,D,first,last", [(1, 1000, 64, 0, 128), (1, 3001, 128, 2900, 3001), (1, 3001, 128, 0, 3001), (3, 700, 20, 128, 256), (150, 900, 64, 0, 300),
                                                (1, 60, 64, 0, 60)])
def test_nan_in_every_key_of_a_stretch_reaches_the_rows_that_see_it(t, Sq, Sk, D, first, last):
    from recboard_amd import ops
    q, k, v, _ = make(2, 4, 2, Sq, Sk, D, t)
    clean, stats = ops.attention_fwd(q, k, v)
    k2 = k.clone()
    k2[0, 0, first:last] = NAN
    out, st = ops.attention_fwd(q, k2, v)
    assert out[0, :2].isnan().all()
    assert torch.equal(out[0, 2:], clean[0, 2:]) and torch.equal(out[1], clean[1]) and torch.equal(st[:2, 1], stats[:2, 1])


@pytest.mark.parametrize("t", TYPES, ids=str)
def test_nan_in_a_part_whose_other_scores_are_negligible(t):
    """The part's weight in the join is exp(-640) = 0: it is still not a part that saw nothing."""
    from recboard_amd import ops
    q, k, v = torch.ones(1, 1, 1, 64, device="cuda", dtype=t), torch.zeros(1, 1, 1000, 64, device="cuda", dtype=t), torch.ones(1, 1, 1000, 64, device="cuda", dtype=t)
    k[:, :, :128] = -10.0
    # 872 equal terms, exact in 32 bits; one rounding of 1 / 872 and one of the product, 2^-24 each (rounded to 16 bits: 1 itself)
    assert ((ops.attention_fwd(q, k, v, scale=1.0)[0].double() - 1).abs() <= 2.0 ** -23).all()
    k[:, :, 7] = NAN
    assert ops.attention_fwd(q, k, v, scale=1.0)[0].isnan().all()


@pytest.mark.parametrize("t", TYPES, ids=str)
def test_rows_and_parts_that_see_nothing_stay_zero_beside_nan(t):
    from recboard_amd import ops
    q, k, v, _ = make(3, 4, 2, 1, 1000, 64, t)
    lens = torch.tensor([0, 1000, 100], device="cuda")
    k[0], v[0], k[2, :, 100:], v[2, :, 100:] = NAN, NAN, NAN, NAN
    q[0] = NAN
    out, st = ops.attention_fwd(q, k, v, key_lengths=lens)
    assert not out[0].any() and (st[0, 0] == -float("inf")).all() and not st[1, 0].any()
    assert torch.isfinite(out[1:]).all() and torch.isfinite(st[:2, 1:]).all()


@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("Sq,Sk,D,row,bias", [(50, 50, 16, 20, False), (150, 150, 64, 100, False), (90, 200, 20, 10, False), (300, 300, 128, 40, False), (600, 2100, 64, 3, False),
                                              (150, 150, 64, 100, True)])
def test_nan_in_a_row_of_q_reaches_the_gradients_of_the_keys_that_it_sees(t, Sq, Sk, D, row, bias):
    """Causal: dq of the row itself and dk, dv of the keys up to its own place are NaN, everything else is what it is without that row's NaN."""
    from recboard_amd import ops
    q, k, v, dout = make(2, 2, 1, Sq, Sk, D, t)
    how = dict(rel(2, t, 32, 40) if bias else {}, causal=True)
    want = reference(q, k, v, dout=dout, **how)
    q2 = q.clone()
    q2[1, 0, row, 0] = NAN
    out, stats = ops.attention_fwd(q2, k, v, **how)
    dq, dk, dv, dtable = ops.attention_bwd(dout, q2, k, v, out, stats, **how)
    hit = torch.zeros(2, 2, Sq, dtype=torch.bool, device="cuda")
    hit[1, 0, row] = True
    seen = torch.zeros(2, 1, Sk, dtype=torch.bool, device="cuda")
    seen[1, 0, :Sk - Sq + row + 1] = True
    for g, name, where in ((dq, "dq", hit), (dk, "dk", seen), (dv, "dv", seen)):
        assert g[where].isnan().all(), name
        value, tol = want[name]
        assert ((g.double() - value).abs() <= tol)[~where].all(), name
    if bias:
        assert dtable[:, 0].isnan().any() and torch.isfinite(dtable[:, 1]).all()


@pytest.mark.parametrize("t", TYPES, ids=str)
def test_gradients_of_rows_that_see_nothing_are_zero_whatever_they_hold(t):
    from recboard_amd import ops
    q, k, v, dout = make(2, 2, 2, 70, 70, 64, t)
    mask = torch.ones(2, 1, 70, 70, dtype=torch.bool, device="cuda")
    mask[0, :, 5] = False
    want = reference(q, k, v, dout=dout, mask=mask)
    q[0, :, 5] = NAN
    out, stats = ops.attention_fwd(q, k, v, mask=mask)
    assert not out[0, :, 5].any()
    for g, name in zip(ops.attention_bwd(dout, q, k, v, out, stats, mask=mask), ("dq", "dk", "dv")):
        value, tol = want[name]
        assert ((g.double() - value).abs() <= tol).all(), name


@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("Sq,Sk", [(1, 60), (1, 1000), (70, 60), (150, 900)])
def test_statistics_of_a_row_whose_scores_are_nan_add_up_to_nan(t, Sq, Sk):
    """... and not to those of a row that sees nothing, -inf and 0."""
    from recboard_amd import ops
    q, k, v, _ = make(2, 4, 2, Sq, Sk, 64, t)
    q[1, 2, 0, 3] = NAN
    k[0, 0] = NAN
    st = ops.attention_fwd(q, k, v)[1]
    hit = torch.zeros(2, 4, Sq, dtype=torch.bool, device="cuda")
    hit[1, 2, 0] = True
    hit[0, :2] = True
    assert (st[0] + st[1])[hit].isnan().all() and torch.isfinite(st[:2][:, ~hit]).all()


@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("D", [64, 20])
def test_keys_behind_a_length_take_no_gradient_where_rows_are_made_again(t, D):
    """A tile that holds the length's end, a NaN in front of it, shut for every row but one (which sends the whole tile to the row-by-row form), and NaN
    behind: a row behind is not read there, its gradient is 0."""
    from recboard_amd import ops
    q, k, v, dout = make(2, 2, 1, 90, 200, D, t)
    lens = torch.tensor([77, 200], device="cuda")
    mask = torch.ones(2, 1, 90, 200, dtype=torch.bool, device="cuda")
    mask[0, :, 1:, 70] = False
    how = {"mask": mask, "key_lengths": lens}
    want = reference(q, k, v, dout=dout, **how)
    k, v = k.clone(), v.clone()
    k[0, :, 70], v[0, :, 70], k[0, :, 77:], v[0, :, 77:] = NAN, NAN, NAN, NAN
    out, stats = ops.attention_fwd(q, k, v, **how)
    dq, dk, dv, _ = ops.attention_bwd(dout, q, k, v, out, stats, **how)
    assert not dk[0, :, 77:].any() and not dv[0, :, 77:].any()
    assert dq[0, :, 0].isnan().all() and torch.isfinite(dq[0, :, 1:]).all() and torch.isfinite(dq[1]).all()
    for g, name in ((dk, "dk"), (dv, "dv")):                    # the row that saw the NaN has a part in every key of the length
        value, tol = want[name]
        assert g[0, :, :77].isnan().all() and ((g.double() - value).abs() <= tol)[1].all(), name
    value, tol = want["dq"]
    assert ((dq.double() - value).abs() <= tol)[0, :, 1:].all()


@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("Sq,Sk,D", [(2048, 2048, 128), (1, 5000, 64), (70, 300, 20)])
def test_a_batch_that_is_nan_throughout(t, Sq, Sk, D):
    """Every row is made again; each stops at its first keys."""
    from recboard_amd import ops
    q, k, v, dout = make(1, 8, 2, Sq, Sk, D, t)
    for poison in ("q", "k", "dout"):
        x = {"q": q.clone(), "k": k.clone(), "v": v, "dout": dout.clone()}
        x[poison].fill_(NAN)
        out, stats = ops.attention_fwd(x["q"], x["k"], x["v"], causal=True)
        dq, dk, dv, _ = ops.attention_bwd(x["dout"], x["q"], x["k"], x["v"], out, stats, causal=True)
        assert dq.isnan().all() and dk.isnan().all() and dv.isnan().all()
        assert out.isnan().all() if poison != "dout" else torch.isfinite(out).all()


@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("D", [40, 128])
def test_nan_in_single_columns_of_v_stays_in_them(t, D):
    """A row is made again to its end while any of its sums is not NaN."""
    from recboard_amd import ops
    q, k, v, dout = make(1, 2, 1, 90, 300, D, t)
    for cols in (range(0, 1), range(D // 2, D), range(0, D - 1)):
        cols = list(cols)
        rest = [c for c in range(D) if c not in cols]
        v2 = v.clone()
        v2[:, :, 3:70, cols] = NAN
        out, _ = ops.attention_fwd(q, k, v2)
        value, tol = reference(q, k, v)["out"]
        assert out[..., cols].isnan().all() and ((out.double() - value).abs() <= tol)[..., rest].all()
        one = ops.attention_fwd(q[:, :, :1], k, v2)[0]
        assert one[..., cols].isnan().all() and torch.isfinite(one[..., rest]).all()
    dout2 = dout.clone()
    dout2[:, :, 5:9, 0] = NAN                                     # delta of those rows is NaN: dq of the rows, dk everywhere, dv in that column
    out, stats = ops.attention_fwd(q, k, v)
    dq, dk, dv, _ = ops.attention_bwd(dout2, q, k, v, out, stats)
    want = reference(q, k, v, dout=dout)
    rows = torch.ones(90, dtype=torch.bool, device="cuda")
    rows[5:9] = False
    assert dq[:, :, ~rows].isnan().all() and dk.isnan().all() and dv[..., 0].isnan().all()
    assert ((dq.double() - want["dq"][0]).abs() <= want["dq"][1])[:, :, rows].all() and ((dv.double() - want["dv"][0]).abs() <= want["dv"][1])[..., 1:].all()
