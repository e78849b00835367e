"""GPU: the block's operators together, through the torch surface: position bias -> attention -> residual norm, trained, captured, and served a
token at a time; the registered ops; the models that call them."""
import copy

import pytest
import torch

pytestmark = pytest.mark.gpu


class Block(torch.nn.Module):
    """A transformer block's attention half on the engine (`plain`: the same in elementary torch operations, any type)."""

    def __init__(self, D=64, H=4, Hkv=2, plain=False, causal=True):
        super().__init__()
        from recboard_amd import nn as rnn
        self.H, self.Hkv, self.dh, self.plain, self.causal = H, Hkv, D // H, plain, causal
        self.qkv = torch.nn.Linear(D, (H + 2 * Hkv) * self.dh, device="cuda")
        self.out = torch.nn.Linear(D, D, device="cuda")
        self.position = rnn.RelativePositionBias(H, 32, 64, bidirectional=not causal)
        self.norm = rnn.LayerNorm(D, device="cuda")
        with torch.no_grad():
            self.position.weight.normal_()
            self.norm.weight.normal_(1.0, 0.1)

    def forward(self, x, mask=None):
        from recboard_amd import nn as rnn
        B, S, D = x.shape
        qkv = self.qkv(x).view(B, S, self.H + 2 * self.Hkv, self.dh).transpose(1, 2)
        q, k, v = qkv.split([self.H, self.Hkv, self.Hkv], 1)
        if not self.plain:
            a = rnn.attention(q, k, v, causal=self.causal, mask=mask, position=self.position)
            return self.norm(self.out(a.transpose(1, 2).reshape(B, S, D)), x)
        k, v = (t.repeat_interleave(self.H // self.Hkv, 1) for t in (k, v))
        far = self.position.bucket_map.numel() // 2
        d = torch.arange(S, device="cuda") - torch.arange(S, device="cuda").unsqueeze(1)
        s = q @ k.transpose(2, 3) / self.dh ** 0.5 + self.position.weight[self.position.bucket_map[d.clamp(-far, far) + far].long()].permute(2, 0, 1)
        seen = torch.ones(B, 1, S, S, dtype=torch.bool, device="cuda")
        if self.causal:
            seen = seen.tril()
        if mask is not None:
            seen = seen & mask
        none = ~seen.any(3, keepdim=True)
        p = torch.softmax(s.masked_fill(~seen, float("-inf")).masked_fill(none, 0.0), 3).masked_fill(none, 0.0)
        total = self.out((p @ v).transpose(1, 2).reshape(B, S, D)) + x
        u = total.mean(-1, keepdim=True)
        return (total - u) / torch.sqrt(((total - u) ** 2).mean(-1, keepdim=True) + self.norm.eps) * self.norm.weight + self.norm.bias, total


@pytest.mark.parametrize("causal", [True, False])
def test_block_matches_itself_in_64_bits_with_every_gradient(causal):
    torch.manual_seed(0)
    m = Block(causal=causal)
    ref = copy.deepcopy(m).double()
    ref.plain = True
    x = torch.randn(3, 50, 64, device="cuda", requires_grad=True)
    x64 = x.detach().double().requires_grad_()
    mask = (torch.arange(50, device="cuda") >= torch.tensor([[0], [13], [49]], device="cuda")).view(3, 1, 1, 50)
    w = torch.randn(2, 3, 50, 64, device="cuda")
    y, total = m(x, mask)
    ((y * w[0]).sum() + (total * w[1]).sum()).backward()
    y64, total64 = ref(x64, mask)
    ((y64 * w[0]).sum() + (total64 * w[1]).sum()).backward()
    # fp32 end to end, ~300-term sums: 1e-5 of each tensor's largest value (2^-24 times a chain of 64 products and sums, three layers deep)
    close = lambda a, b: (a.double() - b).abs().max() <= 1e-5 * b.abs().max()  # noqa: E731
    assert close(y, y64) and close(total, total64) and close(x.grad, x64.grad)
    for (n, p), q in zip(m.named_parameters(), ref.parameters()):
        assert close(p.grad, q.grad), n


def test_block_trains_in_a_graph_as_it_does_eagerly():
    from recboard_amd import nn as rnn
    torch.manual_seed(1)
    a = Block()
    b = copy.deepcopy(a)
    batches = [(torch.randn(4, 40, 64, device="cuda"), torch.randn(4, 40, 64, device="cuda")) for _ in range(4)]
    loss = lambda m: lambda x, t: ((m(x)[0] - t) ** 2).mean()  # noqa: E731
    oa, ob = (torch.optim.Adam(m.parameters(), lr=1e-3, capturable=True) for m in (a, b))
    step = rnn.GraphedStep(a, loss(a), oa, batches[0])
    for x, t in batches:
        got = step(x, t).clone()
        ob.zero_grad(set_to_none=True)
        want = loss(b)(x, t)
        want.backward()
        ob.step()
        torch.cuda.synchronize()
        assert torch.allclose(got, want, rtol=1e-5)
    for p, q in zip(a.parameters(), b.parameters()):
        assert torch.allclose(p, q, rtol=1e-4, atol=1e-6)


@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16], ids=str)
def test_tokens_served_one_by_one_from_a_cache_repeat_the_whole_sequence(t):
    """A prompt, then single tokens, ragged: each step's row is the whole causal pass's row (fp32: the order of sums; bf16: two roundings of values
    below 4, 2^-8 each, of P and of the result)."""
    from recboard_amd import nn as rnn, ops
    torch.manual_seed(2)
    B, H, Hkv, D, S = 3, 8, 2, 64, 90
    q, k, v = (torch.randn(B, h, S, D, device="cuda").to(t) for h in (H, Hkv, Hkv))
    pos = rnn.RelativePositionBias(H, 32, 64, bidirectional=False)
    torch.nn.init.normal_(pos.weight)
    whole = rnn.attention(q, k, v, causal=True, position=pos)
    cache_k, cache_v = (torch.full((B, Hkv, 128, D), float("nan"), device="cuda").to(t) for _ in range(2))
    start = torch.tensor([60, 17, 1], device="cuda")
    tol = 1e-5 if t == torch.float32 else 2.0 ** -5
    with torch.no_grad():
        for b in range(B):
            n = int(start[b])
            cache_k[b, :, :n], cache_v[b, :, :n] = k[b, :, :n], v[b, :, :n]
        first = rnn.attention(q[:, :, :60], cache_k, cache_v, causal=True, key_lengths=start, q_offset=torch.zeros_like(start), position=pos)
        for b in range(B):
            n = int(start[b])
            assert (first[b, :, :n].float() - whole[b, :, :n].float()).abs().max() <= tol
        for step in range(12):
            at = start + step
            idx = at.view(B, 1, 1, 1).expand(B, Hkv, 1, D)
            cache_k.scatter_(2, idx, k.gather(2, idx))
            cache_v.scatter_(2, idx, v.gather(2, idx))
            qi = q.gather(2, at.view(B, 1, 1, 1).expand(B, H, 1, D))
            one = rnn.attention(qi, cache_k, cache_v, causal=True, key_lengths=at + 1, q_offset=at, position=pos)
            want = whole.gather(2, at.view(B, 1, 1, 1).expand(B, H, 1, D))
            assert (one.float() - want.float()).abs().max() <= tol, step


def test_norm_with_an_unused_output_and_with_the_same_tensor_twice():
    from recboard_amd import nn as rnn
    x = torch.randn(6, 64, device="cuda", requires_grad=True)
    ln = rnn.LayerNorm(64, device="cuda")
    y, total = ln(x, x)
    y.sum().backward(retain_graph=True)
    assert x.grad.abs().max() < 1e-4                      # a constant shift of a row leaves its norm
    x.grad = None
    total.sum().backward()
    assert torch.equal(x.grad, torch.full_like(x, 2.0)) and ln.weight.grad is not None
    plain = rnn.LayerNorm(64, elementwise_affine=False)
    g = torch.autograd.grad(plain(x).pow(2).sum(), x)[0]
    assert torch.isfinite(g).all() and not list(plain.parameters())
    b = torch.zeros(64, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    xb = x.detach().bfloat16()
    db = torch.autograd.grad(rnn.layer_norm(xb, None, b).sum(), b)[0]
    assert db.dtype == torch.bfloat16 and torch.equal(db, torch.full_like(db, 6.0))


def test_bias_module_materialised_and_its_gradient():
    from recboard_amd import nn as rnn
    pos = rnn.RelativePositionBias(4, 8, 16)
    torch.nn.init.normal_(pos.weight)
    w = torch.randn(4, 20, 20, device="cuda")
    (pos(20, 20) * w).sum().backward()
    d = torch.arange(20, device="cuda") - torch.arange(20, device="cuda").unsqueeze(1)
    ids = pos.bucket_map[d.clamp(-16, 16) + 16].long()
    want = torch.stack([w[:, ids == b].sum(1) for b in range(8)])
    torch.testing.assert_close(pos.weight.grad, want, rtol=1e-5, atol=1e-5)
    assert "bucket_map" not in pos.state_dict()


def test_every_new_op_passes_opcheck_and_refuses_the_cpu():
    import recboard_amd.torch_ops  # noqa: F401
    from recboard_amd import nn as rnn, ops
    R = torch.ops.recengine
    tests = ("test_schema", "test_faketensor", "test_autograd_registration")
    r = lambda *s: torch.randn(*s, device="cuda", requires_grad=True)  # noqa: E731
    x, w, b = r(6, 64), r(64), r(64)
    torch.library.opcheck(R.layer_norm.default, (x, w, b, 1e-5), test_utils=tests)
    torch.library.opcheck(R.layer_norm.default, (x, None, None, 1e-5), test_utils=tests)
    torch.library.opcheck(R.add_layer_norm.default, (x, r(6, 64), w, b, 1e-5), test_utils=tests)
    m = ops.relative_buckets(8, 16)
    table = r(8, 4)
    torch.library.opcheck(R.relative_bias.default, (table, m, 5, 7, 2), test_utils=tests)
    q, k, v = r(2, 4, 5, 16), r(2, 2, 7, 16), r(2, 2, 7, 16)
    mask = torch.rand(2, 1, 1, 7, device="cuda") < 0.8
    torch.library.opcheck(R.attention.default, (q, k, v, 0.0, False, mask, None, None, 2, table, m), test_utils=tests)
    lens = torch.tensor([3, 7], device="cuda")
    torch.library.opcheck(R.attention.default, (q, k, v, 0.3, True, None, lens, lens - 2, 0, None, None, True), test_utils=tests)
    for call in (lambda: R.layer_norm(x.cpu(), None, None), lambda: R.attention(q.cpu(), k.cpu(), v.cpu(), 0.0, False, None, None, None, 0, None, None),
                 lambda: R.relative_bias(table.cpu(), m.cpu(), 2, 2, 0)):
        with pytest.raises(RuntimeError):
            call()
    with pytest.raises(ValueError):
        rnn.attention(q, k, v, mask=torch.zeros(5, 7, device="cuda", requires_grad=True))
    with pytest.raises(ValueError):
        rnn.attention(q, k, v, scale=-1.0)


def test_bsarec_attention_is_the_products_it_replaces():
    """The additive -1e4 of a left-padded causal history, padding rows (every key at -1e4) among them: engine attention against the model's own
    products with dropped probabilities switched off.  fp32 at scores of -1e4: half a step is 2^-11, so P may be off by 2 * 2^-11 of itself."""
    from recboard_amd.siblings import _BSAAttention
    torch.manual_seed(3)
    m = _BSAAttention(64, 2, 0.0, 0.0, "cuda")
    x = torch.randn(4, 50, 64, device="cuda")
    seqs = torch.where(torch.arange(50, device="cuda") >= torch.tensor([[0], [10], [30], [49]], device="cuda"), 1, 0)
    mask = torch.where((seqs != 0).view(4, 1, 1, 50).expand(-1, -1, 50, -1).tril(), 0.0, -1.0e4)
    got = m(x, mask)
    q, k, v = (l(x.reshape(-1, 64)).view(4, 50, 2, 32).permute(0, 2, 1, 3).double() for l in (m.query, m.key, m.value))
    p = torch.softmax(q @ k.transpose(-1, -2) / 32 ** 0.5 + mask.double(), -1)
    ctx = (p @ v).permute(0, 2, 1, 3).reshape(200, 64)
    want = torch.nn.functional.layer_norm((ctx @ m.dense.weight.double().t() + m.dense.bias.double()).view(4, 50, 64)
                                          + x.double(), (64,), m.LayerNorm.weight.double(), m.LayerNorm.bias.double(), 1e-12)
    assert (got.double() - want).abs().max() <= 2 * 2.0 ** -10 * want.abs().max()
