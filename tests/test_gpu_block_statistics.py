"""GPU: what the block's operators return beside their result -- a row's mean, rstd, softmax statistics -- has no gradient, and a loss made of it fails
instead of training on a part of itself."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_statistics_do_not_require_a_gradient():
    import recboard_amd.torch_ops  # noqa: F401
    R = torch.ops.recengine
    r = lambda *s: torch.randn(*s, device="cuda", requires_grad=True)  # noqa: E731
    x, w, b = r(6, 64), r(64), r(64)
    y, mean, rstd = R.layer_norm(x, w, b, 1e-5)
    y2, total, mean2, rstd2 = R.add_layer_norm(x, r(6, 64), w, b, 1e-5)
    out, stats = R.attention(r(2, 4, 5, 16), r(2, 2, 7, 16), r(2, 2, 7, 16), 0.0, False, None, None, None, 2, None, None)
    assert y.requires_grad and y2.requires_grad and total.requires_grad and out.requires_grad
    for t in (mean, rstd, mean2, rstd2, stats):
        assert not t.requires_grad
        with pytest.raises(RuntimeError):
            t.sum().backward()
    (y.sum() + y2.sum() + total.sum() + out.sum() + (stats[0] + stats[1]).sum() + mean.sum()).backward()
    assert torch.isfinite(x.grad).all() and w.grad is not None and b.grad is not None
