"""The engine's LayerNorm module in the place of torch's: its class, arguments and state dict (CPU), and the norm itself (GPU)."""
import pytest
import torch

from recboard_amd import nn as rnn


@pytest.mark.parametrize("how", [{}, {"eps": 1e-12}, {"elementwise_affine": False}, {"bias": False}, {"dtype": torch.bfloat16}])
@pytest.mark.parametrize("shape", [8, (8,), [3, 8], torch.Size([2, 3, 8])])
def test_module_has_what_torchs_has(shape, how):
    a, b = rnn.LayerNorm(shape, **how), torch.nn.LayerNorm(shape, **how)
    assert isinstance(a, torch.nn.LayerNorm) and repr(a) == repr(b) and a.normalized_shape == b.normalized_shape and a.eps == b.eps
    assert {k: (v.shape, v.dtype) for k, v in a.state_dict().items()} == {k: (v.shape, v.dtype) for k, v in b.state_dict().items()}
    if a.weight is not None:
        with torch.no_grad():
            a.weight.zero_()
        a.reset_parameters()
        assert (a.weight == 1).all()


def test_module_refuses_other_shapes():
    with pytest.raises(ValueError):
        rnn.LayerNorm(8, elementwise_affine=False)(torch.zeros(4, 7))
    with pytest.raises(ValueError):
        rnn.LayerNorm((3, 8))(torch.zeros(4, 8, 3))


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(64,), (5, 20), (2, 3, 7)])
@pytest.mark.parametrize("how", [{}, {"bias": False}, {"elementwise_affine": False}])
def test_module_is_the_norm_over_its_dimensions(shape, how):
    torch.manual_seed(0)
    a = rnn.LayerNorm(shape, device="cuda", **how)
    if a.weight is not None:
        torch.nn.init.normal_(a.weight)
    b = torch.nn.LayerNorm(shape, device="cuda", dtype=torch.float64, **how)
    b.load_state_dict(a.state_dict())
    x, r, g, gs = (torch.randn(4, 6, *shape, device="cuda") for _ in range(4))
    for residual in (None, r):
        xa, xb = x.clone().requires_grad_(), x.double().requires_grad_()
        if residual is None:
            y, z = a(xa), b(xb)
            (y * g).sum().backward()
            (z * g.double()).sum().backward()
        else:
            (y, s), t = a(xa, residual), xb + residual.double()
            z = b(t)
            ((y * g).sum() + (s * gs).sum()).backward()
            ((z * g.double()).sum() + (t * gs.double()).sum()).backward()
            assert (s.double() - t).abs().max() <= 2.0 ** -23 * t.abs().max()
        assert y.shape == x.shape
        # fp32 sums of up to 100 terms and 24 rows: 1e-5 of the largest value
        for have, want in [(y, z), (xa.grad, xb.grad)] + [(p.grad, q.grad) for p, q in zip(a.parameters(), b.parameters())]:
            assert (have.double() - want).abs().max() <= 1e-5 * want.abs().max()
        a.zero_grad(), b.zero_grad()
