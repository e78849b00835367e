"""GPU: attention through the C entry with rows (heads, sequences) that go backwards in memory: strides that torch has no tensors for."""
import ctypes

import pytest
import torch

from test_gpu_attention import TYPES, make

pytestmark = pytest.mark.gpu


def back(t, dims):
    """A tensor's copy with the given dimensions reversed in memory: -> (what keeps it, the address of element [0, 0, 0, 0], its strides)."""
    kept = t.contiguous().flip(dims).contiguous()
    st = list(kept.stride())
    at = kept.data_ptr() + sum((t.shape[d] - 1) * st[d] for d in dims) * t.element_size()
    return kept, at, (ctypes.c_int64 * 3)(*(-s if d in dims else s for d, s in enumerate(st[:3])))


@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("dims", [(2,), (0, 1), (0, 1, 2)])
@pytest.mark.parametrize("Sq,Sk,D", [(70, 200, 64), (1, 1000, 128), (50, 50, 16)])
def test_reversed_dimensions(t, dims, Sq, Sk, D):
    from recboard_amd import lib, ops
    q, k, v, dout = make(2, 4, 2, Sq, Sk, D, t)
    want_out, want_stats = ops.attention_fwd(q, k, v, causal=True)
    want = ops.attention_bwd(dout, q, k, v, want_out, want_stats, causal=True)
    kept = [back(x, dims) for x in (q, k, v, torch.zeros_like(q), dout, torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v))]
    d = ops._attention_args(q, k, v, None, True, None, None, None, None, None)
    for name, (_, at, st) in zip("qkv", kept):
        setattr(d, name, at)
        setattr(d, name + "_stride", st)
    stats = torch.zeros_like(want_stats[:2])
    L, p = lib.load(), ctypes.addressof(d)
    n = L.re_attention_fwd_workspace_bytes(p)
    ws = torch.empty(max(n, L.re_attention_bwd_workspace_bytes(p)), dtype=torch.uint8, device="cuda")
    stream = torch.cuda.current_stream().cuda_stream
    (_, o, o_st), (_, g, g_st) = kept[3:5]
    assert L.re_attention_fwd(p, o, o_st, stats.data_ptr(), None, ws.data_ptr(), ws.numel(), stream) == 0
    outs = [x for _, at, st in kept[5:] for x in (at, st)]
    assert L.re_attention_bwd(p, o, o_st, stats.data_ptr(), None, g, g_st, *outs, None, ws.data_ptr(), ws.numel(), stream) == 0
    torch.cuda.synchronize()
    # the same operator; another form of it, and without what rounding took from the output: a few roundings of the largest values
    u = 8 * torch.finfo(t).eps
    for (have, _, _), w in zip([kept[3]] + kept[5:], (want_out,) + want[:3]):
        assert (have.flip(dims).double() - w.double()).abs().max() <= u * w.double().abs().max()
    assert (stats.sum(0) - want_stats[:2].sum(0)).abs().max() <= 1e-5 * want_stats[:2].sum(0).abs().max()
