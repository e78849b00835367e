"""GPU: the relative position bias by buckets and its gradient, against plain indexing and 64-bit sums.

The forward copies table entries: equal to the bit.  A gradient sum in fp32 of n terms in chains of at most 2^12 (a lane's diagonal over 16 rows,
a bucket's diagonals, the workgroups) is off by at most 2^12 * 2^-24 of the sum of magnitudes, plus the one rounding to the table's type."""
import pytest
import torch

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def ids_of(bucket_map, queries, keys, offset):
    far = bucket_map.numel() // 2
    d = torch.arange(keys, device="cuda") - torch.arange(queries, device="cuda").unsqueeze(1) - offset
    return bucket_map[d.clamp(-far, far) + far].long()


def check(t, H, queries, keys, offset, buckets=32, distance=128, bidirectional=True, seed=0):
    from recboard_amd import ops
    g = torch.Generator(device="cuda").manual_seed(seed)
    table = torch.randn(buckets, H, generator=g, device="cuda").to(t)
    m = ops.relative_buckets(buckets, distance, bidirectional)
    off = keys - queries if offset is None else offset
    ids = ids_of(m, queries, keys, off)
    bias = ops.relative_bias_fwd(table, m, queries, keys, offset)
    assert bias.dtype == t and torch.equal(bias, table.t()[:, ids])
    d = torch.randn(H, queries, keys, generator=g, device="cuda").to(t)
    got = ops.relative_bias_bwd(d, m, buckets, offset)
    member = ids.reshape(-1, 1) == torch.arange(buckets, device="cuda")
    want = (d.double().reshape(H, -1) @ member.double()).t()
    mag = (d.double().abs().reshape(H, -1) @ member.double()).t()
    tol = torch.finfo(t).eps / 2 * want.abs() + 2.0 ** -12 * mag + torch.finfo(t).tiny
    assert got.shape == (buckets, H) and got.dtype == t
    assert ((got.double() - want).abs() <= tol).all(), ((got.double() - want).abs() - tol).max()
    wide = ops.relative_bias_bwd(d, m, buckets, offset, dtype=torch.float32)
    assert ((wide.double() - want).abs() <= 2.0 ** -12 * mag + 1e-30).all()


@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("H,queries,keys,offset", [(1, 1, 1, None), (3, 1, 700, None), (4, 50, 50, None), (2, 17, 16, None), (2, 33, 257, 5), (1, 300, 8, -290),
                                                   (2, 64, 1024, None), (2, 5, 64, 100000), (2, 5, 64, -100000), (5, 130, 1000, 7)])
def test_bias_and_gradient(t, H, queries, keys, offset):
    check(t, H, queries, keys, offset)


@pytest.mark.parametrize("buckets,distance,bidirectional", [(2, 5, False), (4, 2, True), (8, 40, False), (64, 256, True), (256, 1024, True), (100, 1000, False)])
def test_bias_of_other_tables(buckets, distance, bidirectional):
    check(torch.float32, 3, 70, 1100, 40, buckets, distance, bidirectional)


def test_bucket_map_is_the_logarithmic_rule_and_borders_are_whole():
    from recboard_amd import ops
    m = ops.relative_buckets(32, 128, True, device="cpu").tolist()
    far = 128
    assert m[far] == 0 and m[far - 7] == 7 and m[far + 7] == 23
    # exact = 8, 8 steps: bucket 8 + m begins at ceil(8 * 2^(m / 2)) = 8, 12, 16, 23, 32, 46, 64, 91
    for k, n in enumerate([8, 12, 16, 23, 32, 46, 64, 91]):
        assert m[far - n] == 8 + k and m[far - n + 1] == 7 + k
    one = ops.relative_buckets(32, 128, False, device="cpu").tolist()
    assert one[far:] == [0] * 129 and one[far - 15] == 15 and one[0] == 31


def test_entries_of_a_map_that_are_no_bucket_read_as_zero_and_take_nothing():
    from recboard_amd import ops
    m = torch.tensor([0, -1, 1, 7, 2], dtype=torch.int32, device="cuda")
    table = torch.randn(3, 2, device="cuda")
    bias = ops.relative_bias_fwd(table, m, 6, 6)
    d = torch.arange(6, device="cuda") - torch.arange(6, device="cuda").unsqueeze(1)
    assert not bias[:, d == -1].any() and not bias[:, d == 1].any()
    g = ops.relative_bias_bwd(torch.ones(2, 6, 6, device="cuda"), m, 3)
    assert g[:, 0].tolist() == [10.0, 6.0, 10.0]


def test_bias_of_no_rows_and_gradient_of_nothing():
    from recboard_amd import ops
    m = ops.relative_buckets(8, 16)
    assert ops.relative_bias_fwd(torch.randn(8, 2, device="cuda"), m, 0, 5).shape == (2, 0, 5)
    assert not ops.relative_bias_bwd(torch.empty(2, 0, 5, device="cuda"), m, 8).any()


def test_bias_in_a_graph_and_run_to_run():
    from recboard_amd import ops
    from recboard_amd.capture import recording
    m = ops.relative_buckets(32, 128)
    table, d = torch.randn(32, 4, device="cuda"), torch.randn(4, 130, 256, device="cuda")
    graph = torch.cuda.CUDAGraph()
    ops.relative_bias_bwd(d, m, 32)
    with recording(graph):
        out = (ops.relative_bias_fwd(table, m, 130, 256), ops.relative_bias_bwd(d, m, 32))
    for _ in range(3):
        table.normal_()
        d.normal_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out[0], ops.relative_bias_fwd(table, m, 130, 256)) and torch.equal(out[1], ops.relative_bias_bwd(d, m, 32))


def test_bias_refusals():
    from recboard_amd import ops
    m = ops.relative_buckets(32, 128)
    table = torch.randn(32, 4, device="cuda")
    for bad in (dict(num_buckets=2), dict(num_buckets=512), dict(max_distance=8), dict(max_distance=2000)):
        with pytest.raises(ValueError):
            ops.relative_buckets(**bad)
    with pytest.raises(ValueError):
        ops.relative_bias_fwd(table, m[:-1], 4, 4)
    with pytest.raises(TypeError):
        ops.relative_bias_fwd(table, m.long(), 4, 4)
    with pytest.raises(ValueError):
        ops.relative_bias_fwd(table.t(), m, 4, 4)
    with pytest.raises(ValueError):
        ops.relative_bias_bwd(torch.randn(2, 4, 4, device="cuda").transpose(1, 2), m, 32)
    with pytest.raises(RuntimeError):
        ops.relative_bias_fwd(table.cpu(), m, 4, 4)
    with pytest.raises(RuntimeError):
        ops.relative_bias_fwd(table, m, -1, 4)
