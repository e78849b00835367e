"""GPU: layer norm, alone and behind a residual sum, forward and backward, against the definition in 64 bits.

Tolerances, from the arithmetic: u = eps / 2 of the tensor's type is the one rounding of a result; fp32 sums over a row are trees of at most
64 levels and serial steps per lane, so a sum is off by at most 64 * 2^-24 of the sum of magnitudes; e_x is what that leaves on xhat (with a
residual and a 16-bit type also the rounding of the stored sum, which the backward reads)."""
import pytest
import torch

pytestmark = pytest.mark.gpu
EPS = 1e-5
F = 64 * 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def definition(x, r, w, b, dy=None, ds=None):
    """64 bits: y, s and, with dy, (dx, dw, db)."""
    s = x.double() if r is None else x.double() + r.double()
    w64 = torch.ones(x.shape[-1], dtype=torch.float64, device=x.device) if w is None else w.double()
    b64 = torch.zeros_like(w64) if b is None else b.double()
    mean = s.mean(-1, keepdim=True)
    rstd = 1.0 / torch.sqrt(((s - mean) ** 2).mean(-1, keepdim=True) + EPS)
    xhat = (s - mean) * rstd
    y = xhat * w64 + b64
    if dy is None:
        return y, s, mean, rstd, xhat
    g = dy.double() * w64
    dx = rstd * (g - g.mean(-1, keepdim=True) - xhat * (g * xhat).mean(-1, keepdim=True))
    if ds is not None:
        dx = dx + ds.double()
    return y, s, mean, rstd, xhat, g, dx, (dy.double() * xhat).reshape(-1, x.shape[-1]).sum(0), dy.double().reshape(-1, x.shape[-1]).sum(0)


def check(x, r, w, b, dy, ds):
    from recboard_amd import ops
    t = x.dtype
    u = torch.finfo(t).eps / 2
    uw = u if w is None and t == torch.float32 else torch.finfo(torch.float32 if w is None else w.dtype).eps / 2
    y, s, mean, rstd = ops.layer_norm_fwd(x, w, b, EPS, residual=r)
    dx, dw, db = ops.layer_norm_bwd(dy, s, w, mean, rstd, dsum=ds)
    y64, s64, mean64, rstd64, xhat, g, dx64, dw64, db64 = definition(x, r, w, b, dy, ds)
    top = s64.abs().amax(-1, keepdim=True)
    # fp32 on xhat: the mean's error, the deviation's rounding, rstd's relative error (half of the variance's)
    e = (F * top * rstd64 + F * xhat.abs()) * 1.5
    w64 = 1.0 if w is None else w.double()
    b64 = 0.0 if b is None else b.double().abs()
    tol = u * y64.abs() + (e * abs(w64) if w is None else e * w64.abs()) + 2.0 ** -23 * (y64.abs() + b64) + torch.finfo(t).tiny
    assert ((y.double() - y64).abs() <= tol).all(), ((y.double() - y64).abs() - tol).max()
    if r is not None:
        assert s.dtype == t and ((s.double() - s64).abs() <= (u + 2.0 ** -24) * s64.abs() + torch.finfo(t).tiny).all()
        if t != torch.float32:
            e = e + u * s64.abs() * rstd64
    assert ((mean.double().unsqueeze(-1) - mean64).abs() <= F * top).all()
    mg, ma = g.abs().mean(-1, keepdim=True), (g * xhat).mean(-1, keepdim=True).abs()
    # c1, c2: F of the means of magnitudes; c2 also through xhat's own error
    e_c2 = F * (g * xhat).abs().mean(-1, keepdim=True) + (g.abs() * e).mean(-1, keepdim=True)
    tol = u * dx64.abs() + rstd64 * (F * mg + 2.0 ** -22 * (g.abs() + mg) + e * ma + (xhat.abs() + e) * e_c2) + F * rstd64 * (g.abs() + mg + xhat.abs() * ma)
    tol = tol + 2.0 ** -23 * dx64.abs() + torch.finfo(t).tiny
    assert ((dx.double() - dx64).abs() <= tol).all(), ((dx.double() - dx64).abs() - tol).max()
    D = x.shape[-1]
    mag = (dy.double().abs() * (xhat.abs() * (1 + F) + e) ).reshape(-1, D).sum(0)
    tol = uw * dw64.abs() + (dy.double().abs() * e).reshape(-1, D).sum(0) + 2 * F * mag + torch.finfo(torch.float16).tiny
    assert ((dw.double() - dw64).abs() <= tol).all(), ((dw.double() - dw64).abs() - tol).max()
    tol = uw * db64.abs() + 2 * F * dy.double().abs().reshape(-1, D).sum(0) + torch.finfo(torch.float16).tiny
    assert ((db.double() - db64).abs() <= tol).all()
    return y, s, dx, dw, db


def make(shape, t, residual, seed=0, wtype=None, scale=1.0, shift=0.3):
    g = torch.Generator(device="cuda").manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    x, r = (n(*shape) * scale + shift).to(t), (n(*shape) * 2 - shift).to(t) if residual else None
    w, b = (1 + 0.1 * n(shape[-1])).to(wtype or t), (0.1 * n(shape[-1])).to(wtype or t)
    return x, r, w, b, n(*shape).to(t), n(*shape).to(t) if residual else None


@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("rows,D", [(1, 1), (5, 2), (3, 7), (1, 64), (257, 64), (700, 50), (33, 128), (18, 130), (9, 200), (5, 512), (7, 1001), (3, 1024),
                                    (2, 2048), (2, 2050), (600, 4096), (2, 5000), (2, 8192), (1, 16384), (3, 16390), (2, 40003)])
def test_layer_norm_matches_the_definition(t, rows, D):
    for residual in (False, True):
        check(*make((rows, D), t, residual, seed=rows * 7 + D))


@pytest.mark.parametrize("t", [torch.bfloat16, torch.float16], ids=str)
def test_layer_norm_takes_fp32_weights_and_none(t):
    check(*make((37, 96), t, True, wtype=torch.float32))
    x, r, w, b, dy, ds = make((37, 96), t, False)
    check(x, None, None, None, dy, None)
    check(x, None, w, None, dy, None)


def test_layer_norm_on_misaligned_rows_and_leading_dimensions():
    x, r, w, b, dy, ds = make((2, 3, 5, 64), torch.bfloat16, True)
    off = lambda t: torch.cat([t.new_zeros(1), t.reshape(-1)])[1:].view(t.shape)  # noqa: E731   (contiguous, two bytes off a 16-byte boundary)
    a = check(x, r, w, b, dy, ds)
    c = check(off(x), off(r), off(w), off(b), off(dy), off(ds))
    assert all(p.shape == q.shape for p, q in zip(a, c))


def test_layer_norm_with_a_mean_far_from_zero_and_constant_rows():
    check(*make((20, 256), torch.float32, False, scale=1.0, shift=3000.0))       # a sum of squares would cancel here
    x, r, w, b, dy, ds = make((4, 64), torch.float32, False)
    x[1] = 5.0
    x[2] = 0.0
    y, s, dx, dw, db = check(x, None, w, b, dy, None)
    assert torch.equal(y[2], b) and torch.isfinite(dx).all()


def test_layer_norm_keeps_a_bad_row_to_itself():
    x, r, w, b, dy, ds = make((6, 64), torch.float32, False)
    from recboard_amd import ops
    clean = ops.layer_norm_fwd(x, w, b)[0]
    x[3, 7] = float("nan")
    y = ops.layer_norm_fwd(x, w, b)[0]
    assert y[3].isnan().all()
    keep = [0, 1, 2, 4, 5]
    assert torch.equal(y[keep], clean[keep])


def test_layer_norm_of_no_rows():
    from recboard_amd import ops
    x = torch.empty(0, 64, device="cuda")
    w = torch.ones(64, device="cuda")
    y, s, mean, rstd = ops.layer_norm_fwd(x, w, w)
    dx, dw, db = ops.layer_norm_bwd(x, x, w, mean, rstd)
    assert y.shape == (0, 64) and dx.shape == (0, 64) and not dw.any() and not db.any()


def test_layer_norm_same_bits_again_on_another_stream_and_in_a_graph():
    from recboard_amd import ops
    from recboard_amd.capture import recording
    x, r, w, b, dy, ds = make((1500, 256), torch.bfloat16, True)

    def step():
        y, s, mean, rstd = ops.layer_norm_fwd(x, w, b, residual=r)
        return (y, s) + ops.layer_norm_bwd(dy, s, w, mean, rstd, dsum=ds)
    first = [t.clone() for t in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(p, q) for p, q in zip(first, again))
    graph = torch.cuda.CUDAGraph()
    with recording(graph):
        out = step()
    for k in range(3):
        x.copy_(torch.randn_like(x))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, step())), k


def test_layer_norm_gradient_against_differences():
    """<dx, v> against the central difference of the 64-bit definition along v: error h^2 of the third derivative (h = 1e-5: below 1e-8 of the
    value) plus dx's own fp32 error, bounded by sum |v| * 1e-5 * max|dx| generously above what `check` allows per element."""
    from recboard_amd import ops
    x, r, w, b, dy, ds = make((4, 48), torch.float32, True)
    y, s, mean, rstd = ops.layer_norm_fwd(x, w, b, residual=r)
    dx, dw, db = ops.layer_norm_bwd(dy, s, w, mean, rstd, dsum=ds)
    v, h = torch.randn_like(x).double(), 1e-5

    def loss(d):
        out = definition(x.double() + d, r, w, b)
        return (out[0] * dy.double()).sum() + (out[1] * ds.double()).sum()
    want = (loss(h * v) - loss(-h * v)) / (2 * h)
    assert abs(float((dx.double() * v).sum() - want)) <= 1e-5 * float(v.abs().sum() * dx.abs().max())


def test_layer_norm_refusals():
    from recboard_amd import ops
    x, w = torch.randn(4, 64, device="cuda"), torch.ones(64, device="cuda")
    with pytest.raises(ValueError):
        ops.layer_norm_fwd(x.t(), w, w)                       # not contiguous
    with pytest.raises(ValueError):
        ops.layer_norm_fwd(x, w[:32].contiguous(), None)
    with pytest.raises(TypeError):
        ops.layer_norm_fwd(x.double(), w, w)
    with pytest.raises(TypeError):
        ops.layer_norm_fwd(x, w, w.half())
    with pytest.raises(TypeError):
        ops.layer_norm_fwd(x, w, w, residual=x.half())
    with pytest.raises(ValueError):
        ops.layer_norm_fwd(x, w, w, residual=x[:2].contiguous())
    y, s, mean, rstd = ops.layer_norm_fwd(x, w, w)
    with pytest.raises(ValueError):
        ops.layer_norm_bwd(x, s, w, mean[:2].contiguous(), rstd)
    with pytest.raises(RuntimeError):
        ops.layer_norm_fwd(x.cpu(), w, w)
