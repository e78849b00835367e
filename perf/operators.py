"""The transformer-block operators of the sequence recommenders, as workloads: layer norm (alone, and behind a residual sum), the
learned relative position bias by buckets, and attention with its recomputing backward pass.

`own = False`: every operator in its plain form, elementary torch operations in 32 bits (the bucket sums in 64), rounded once at the
end.  `own = True`: the framework's calls (`recboard_amd.ops`).  A case is a dict of plain values:

    op = "layer_norm"     rows, dim, type, residual, train         y = (s - mean) / sqrt(var + eps) * w + b,  s = x (+ r)
    op = "relative_bias"  heads, queries, keys, type, buckets, distance, causal       bias[h, i, j] = table[bucket(j - i - offset), h]
    op = "attention"      batch, heads, kv_heads, queries, keys, dim, type, causal, padding, buckets, distance, train
                          out = softmax(q k^T / sqrt(dim) + bias, over the keys that the row may see) v
                          padding: "none"; "left" / "mixed" -- a truth value for each key of each sequence; "cache" -- a length for each sequence

With `train` the pass is forward and backward, its outputs are the results and the gradients of every input.
"""
import math

import torch

own = False

_TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
_BYTES = {"fp32": 4, "bf16": 2, "fp16": 2}
_EPS = 1e-5


# ------------------------------------------------------------------------------------------------ the cases
def _ln(name, rows, dim, type, residual, train):
    return {"name": name, "op": "layer_norm", "rows": rows, "dim": dim, "type": type, "residual": residual, "train": train}


def _rel(name, heads, queries, keys, type, buckets, distance, causal):
    return {"name": name, "op": "relative_bias", "heads": heads, "queries": queries, "keys": keys, "type": type, "buckets": buckets,
            "distance": distance, "causal": causal}


def _attn(name, batch, heads, kv_heads, queries, keys, dim, type, causal, padding, buckets, distance, train):
    return {"name": name, "op": "attention", "batch": batch, "heads": heads, "kv_heads": kv_heads, "queries": queries, "keys": keys, "dim": dim,
            "type": type, "causal": causal, "padding": padding, "buckets": buckets, "distance": distance, "train": train}


def listed():
    return [
        # one new token of a served model: the residual sum and the norm in front of the next projection
        _ln("norm_token", 1, 4096, "bf16", True, False),
        # the norm behind a block of the sequence models: a batch of 512 histories of 50 items, 64 features
        _ln("norm_items", 512 * 50, 64, "fp32", True, True),
        # a packed ragged batch with a width that no vector divides evenly
        _ln("norm_odd", 3001, 1001, "fp16", False, True),
        # a training step of a wide text encoder of the items: 16 sequences of 1024 tokens
        _ln("norm_wide", 16 * 1024, 4096, "bf16", True, True),
        # the position bias of a history of 50 items, four heads, in training
        _rel("bias_items", 4, 50, 50, "fp32", 32, 128, False),
        # the same for a long bidirectional encoder
        _rel("bias_long", 16, 4096, 4096, "bf16", 32, 128, False),
        # BERT4Rec's encoder in training: 256 left-padded histories of 50 items, four heads of 16
        _attn("attn_items", 256, 4, 4, 50, 50, 16, "fp32", False, "left", 0, 0, True),
        # a ragged left-padded batch, causal (its padding queries see nothing), shared heads, a bias, an unusual head size
        _attn("attn_ragged", 5, 12, 4, 777, 777, 80, "fp16", True, "left", 32, 128, True),
        # a bidirectional encoder with the position bias over long histories
        _attn("attn_bias", 2, 8, 8, 2048, 2048, 64, "bf16", False, "mixed", 32, 128, True),
        # a training step of a causal decoder
        _attn("attn_train", 2, 16, 4, 4096, 4096, 128, "bf16", True, "none", 0, 0, True),
        # a piece of a prompt behind a cached prefix, ragged
        _attn("attn_prefill", 3, 32, 8, 333, 4429, 128, "bf16", True, "cache", 0, 0, False),
        # one new token for each of 16 sequences against their caches
        _attn("attn_decode", 16, 32, 8, 1, 16384, 128, "bf16", True, "cache", 0, 0, False),
    ]


def _spread(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(["norm", "token", "bias", "train", "items", "prefill", "decode"])
    type = rng.choice(["fp32", "bf16", "fp16"])
    if kind in ("norm", "token"):
        while True:
            rows = _spread(rng, 1, 16384) if kind == "norm" else rng.randint(1, 8)
            dim = _spread(rng, 16, 8192)
            if rows * dim * _BYTES[type] <= 16384 * 4096 * 2:
                return _ln(None, rows, dim, type, rng.random() < 0.5, kind == "norm")
    buckets, distance = rng.choice([8, 16, 32, 64]), rng.choice([40, 64, 128, 200, 256])
    if kind == "bias":
        while True:
            heads, queries = _spread(rng, 1, 32), _spread(rng, 1, 4096)
            keys = _spread(rng, queries, 4096)
            if heads * queries * keys * _BYTES[type] <= 16 * 4096 * 4096 * 2:
                return _rel(None, heads, queries, keys, type, buckets, distance, rng.random() < 0.5)
    group, kv_heads = rng.choice([1, 1, 2, 3, 4, 8]), rng.choice([1, 2, 3, 4, 8])
    dim = rng.choice([16, 20, 32, 40, 64, 80, 96, 128])
    if rng.random() < 0.5:
        buckets = distance = 0
    if kind == "items":
        batch, length = _spread(rng, 16, 256), _spread(rng, 2, 200)
        return _attn(None, batch, 4, 4, length, length, rng.choice([16, 20, 32, 64]), "fp32", rng.random() < 0.5, "left", buckets, distance, True)
    if kind == "train":
        if type == "fp32":                # an fp32 product costs many times a 16-bit one: shorter
            top = 1024
        else:
            top = 4096
        while True:
            batch, length = _spread(rng, 1, 16), _spread(rng, 64, top)
            if batch * kv_heads * group * length * length * dim <= 2 * 16 * 2048 * 4096 * 128:
                return _attn(None, batch, kv_heads * group, kv_heads, length, length, dim, type, rng.random() < 0.6, rng.choice(["none", "left", "mixed"]),
                             buckets, distance, True)
    while True:
        batch, keys = _spread(rng, 1, 32), _spread(rng, 16, 16384)
        queries = min(keys, _spread(rng, 2, 512)) if kind == "prefill" else 1
        heads = kv_heads * group
        if batch * kv_heads * keys * dim * _BYTES[type] <= 16 * 8 * 16384 * 128 * 2 and batch * heads * queries * keys <= 3 * 32 * 333 * 4429:
            return _attn(None, batch, heads, kv_heads, queries, keys, dim, type, True, "cache", buckets, distance, False)


# ------------------------------------------------------------------------------------------------ the inputs
def _bucket_of(distance, buckets, max_distance, causal):
    """Bucket of the signed distance key - query: small distances have one each, larger ones share on a logarithmic scale."""
    side, first = (buckets, 0) if causal else (buckets // 2, buckets // 2 if distance > 0 else 0)
    n = max(-distance, 0) if causal else abs(distance)
    exact = side // 2
    if n < exact:
        return first + n
    steps, m = side - exact, 0
    # floor(log(n / exact) / log(max_distance / exact) * steps), in whole numbers
    while m < steps - 1 and max_distance ** (m + 1) * exact ** (steps - m - 1) <= n ** steps:
        m += 1
    return first + exact + m


def _bucket_map(case):
    far = case["distance"]
    return torch.tensor([_bucket_of(d, case["buckets"], far, case["causal"]) for d in range(-far, far + 1)], dtype=torch.int32, device="cuda")


def _lengths(case, gen):
    """Keys that each sequence has: at least its new tokens, at most `keys`, the first sequence all of them."""
    batch, keys, least = case["batch"], case["keys"], case["queries"] if case["padding"] == "cache" else 1
    least = max(least, keys // 4)
    n = least + (torch.rand(batch, generator=gen, device="cuda") * (keys - least + 1)).long().clamp_(max=keys - least)
    n[0] = keys
    return n


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    t = _TYPES[case["type"]]

    def normal(*shape, scale=1.0, shift=0.0):
        return (torch.randn(*shape, generator=gen, device="cuda") * scale + shift).to(t)

    s = {"case": case}
    if case["op"] == "layer_norm":
        rows, dim = case["rows"], case["dim"]
        s["x"] = normal(rows, dim)
        s["residual"] = normal(rows, dim, scale=2.0, shift=0.25) if case["residual"] else None
        s["weight"], s["bias"] = normal(dim, scale=0.1, shift=1.0), normal(dim, scale=0.1)
        if case["train"]:
            s["dy"] = normal(rows, dim)
            s["ds"] = normal(rows, dim) if case["residual"] else None        # the residual stream's own gradient
        return s
    if case["op"] == "relative_bias":
        heads, queries, keys = case["heads"], case["queries"], case["keys"]
        s["table"] = normal(case["buckets"], heads, scale=0.5)
        s["map"] = _bucket_map(case)
        s["dbias"] = normal(heads, queries, keys)
        return s
    batch, heads, kv_heads, queries, keys, dim = (case[k] for k in ("batch", "heads", "kv_heads", "queries", "keys", "dim"))
    if case["padding"] == "cache":
        s["q"] = normal(batch, queries, heads, dim).transpose(1, 2)
        s["k"], s["v"] = normal(batch, kv_heads, keys, dim), normal(batch, kv_heads, keys, dim)
        s["lengths"] = _lengths(case, gen)
        s["offset"] = s["lengths"] - queries
    else:
        packed = normal(batch, queries, heads + 2 * kv_heads, dim).transpose(1, 2)         # one projection makes all three
        s["q"], s["k"], s["v"] = packed.split([heads, kv_heads, kv_heads], dim=1)
        s["lengths"] = s["offset"] = None
    s["mask"] = None
    if case["padding"] in ("left", "mixed"):
        n = _lengths(case, gen)
        at = torch.arange(keys, device="cuda")
        keep = at >= (keys - n).unsqueeze(1)
        if case["padding"] == "mixed":
            keep &= torch.rand(batch, keys, generator=gen, device="cuda") < 0.9
        s["mask"] = keep.view(batch, 1, 1, keys)
    s["table"] = s["map"] = None
    if case["buckets"]:
        s["table"], s["map"] = normal(case["buckets"], heads, scale=0.5), _bucket_map(case)
    if case["train"]:
        s["dout"] = normal(batch, queries, heads, dim).transpose(1, 2)
    return s


# ------------------------------------------------------------------------------------------------ one pass, as a user calls it
def run(state):
    case = state["case"]
    f = {"layer_norm": (_norm_plain, _norm_own), "relative_bias": (_bias_plain, _bias_own), "attention": (_attention_plain, _attention_own)}
    return f[case["op"]][1 if own else 0](case, state)


def _norm_own(case, s):
    from recboard_amd import ops
    y, total, mean, rstd = ops.layer_norm_fwd(s["x"], s["weight"], s["bias"], _EPS, residual=s["residual"])
    out = {"y": y}
    if case["residual"]:
        out["sum"] = total
    if case["train"]:
        out["dx"], out["dweight"], out["dbias"] = ops.layer_norm_bwd(s["dy"], total, s["weight"], mean, rstd, dsum=s["ds"])
    return out


def _norm_plain(case, s):
    t = s["x"].dtype
    x = s["x"].float()
    if case["residual"]:
        x = x + s["residual"].float()
    w, b = s["weight"].float(), s["bias"].float()
    centred = x - x.mean(dim=1, keepdim=True)
    rstd = torch.rsqrt((centred * centred).mean(dim=1, keepdim=True) + _EPS)
    xhat = centred * rstd
    out = {"y": (xhat * w + b).to(t)}
    if case["residual"]:
        out["sum"] = x.to(t)
    if case["train"]:
        dy = s["dy"].float()
        g = dy * w
        dx = rstd * (g - g.mean(dim=1, keepdim=True) - xhat * (g * xhat).mean(dim=1, keepdim=True))
        if case["residual"]:
            dx = dx + s["ds"].float()
        out["dx"], out["dweight"], out["dbias"] = dx.to(t), (dy * xhat).sum(dim=0).to(t), dy.sum(dim=0).to(t)
    return out


def _bias_own(case, s):
    from recboard_amd import ops
    bias = ops.relative_bias_fwd(s["table"], s["map"], case["queries"], case["keys"])
    return {"bias": bias, "dtable": ops.relative_bias_bwd(s["dbias"], s["map"], case["buckets"])}


def _bucket_ids(bucket_map, queries, keys, offset):
    """[..., queries, keys] buckets; offset: the position of the first query among the keys."""
    far = bucket_map.numel() // 2
    at = torch.arange(keys, device=bucket_map.device) - torch.arange(queries, device=bucket_map.device).unsqueeze(1)
    if torch.is_tensor(offset):
        at = at - offset.view(-1, 1, 1)
    else:
        at = at - offset
    return bucket_map[at.clamp(-far, far) + far].long()


def _sum_by_bucket(d, bucket_map, buckets, offset):
    """[buckets, heads] sums of d [heads, queries, keys]: along the diagonals first (a row is one longer than the row that it is read back
    in, so that row i moves i places), then the diagonals of a bucket."""
    heads, queries, keys = d.shape
    sheared = torch.nn.functional.pad(d.flip(1), (0, queries)).reshape(heads, -1)[:, :-queries].reshape(heads, queries, queries + keys - 1)
    along = sheared.sum(dim=1, dtype=torch.float64)                       # column c: key - query = c - (queries - 1)
    far = bucket_map.numel() // 2
    at = torch.arange(queries + keys - 1, device=d.device) - (queries - 1) - offset
    ids = bucket_map[at.clamp(-far, far) + far].long()
    member = (ids.unsqueeze(1) == torch.arange(buckets, device=d.device)).double()
    return torch.matmul(along, member).t()


def _bias_plain(case, s):
    queries, keys = case["queries"], case["keys"]
    ids = _bucket_ids(s["map"], queries, keys, keys - queries)
    t = s["table"].dtype
    bias = s["table"].t()[:, ids]
    return {"bias": bias, "dtable": _sum_by_bucket(s["dbias"].float(), s["map"], case["buckets"], keys - queries).to(t)}


def _attention_own(case, s):
    from recboard_amd import ops
    how = {"causal": case["causal"], "mask": s["mask"], "key_lengths": s["lengths"], "q_offset": s["offset"], "rel_table": s["table"],
           "bucket_map": s["map"]}
    out, lse = ops.attention_fwd(s["q"], s["k"], s["v"], **how)
    if not case["train"]:
        return {"out": out}
    dq, dk, dv, dtable = ops.attention_bwd(s["dout"], s["q"], s["k"], s["v"], out, lse, **how)
    r = {"out": out, "dq": dq, "dk": dk, "dv": dv}
    if case["buckets"]:
        r["dtable"] = dtable
    return r


def _visible(case, s):
    """Truth value for each (sequence, query, key), or None: the row may see the key."""
    queries, keys = case["queries"], case["keys"]
    dev = s["q"].device
    seen = None
    at = torch.arange(keys, device=dev)
    if case["causal"]:
        first = s["offset"].view(-1, 1, 1) if s["offset"] is not None else keys - queries
        seen = at <= first + torch.arange(queries, device=dev).unsqueeze(1)
        seen = seen if seen.dim() == 3 else seen.unsqueeze(0)
    if s["lengths"] is not None:
        there = (at < s["lengths"].unsqueeze(1)).unsqueeze(1)
        seen = there if seen is None else seen & there
    if s["mask"] is not None:
        seen = s["mask"][:, 0] if seen is None else seen & s["mask"][:, 0]
    return seen


def _attention_plain(case, s):
    t, scale = s["q"].dtype, 1.0 / math.sqrt(case["dim"])
    batch, heads, kv_heads, queries, keys, dim = (case[k] for k in ("batch", "heads", "kv_heads", "queries", "keys", "dim"))
    group = heads // kv_heads

    def folded(x):                      # [batch, kv_heads, group * queries, dim]: the heads that share keys in one product
        return x.float().reshape(batch, kv_heads, group * queries, dim)

    def rows(x):                        # ... and back, [batch, heads, queries, ...]
        return x.reshape(batch, heads, queries, -1)

    q, k, v = folded(s["q"]), s["k"].float().contiguous(), s["v"].float().contiguous()
    score = rows(torch.matmul(q, k.transpose(2, 3).contiguous()) * scale)
    ids = None
    if case["buckets"]:
        ids = _bucket_ids(s["map"], queries, keys, s["offset"] if s["offset"] is not None else keys - queries)
        bias = s["table"].float().t()[:, ids]
        score = score + (bias if ids.dim() == 2 else bias.transpose(0, 1))
    seen = _visible(case, s)
    if seen is not None:
        score = score.masked_fill(~seen.unsqueeze(1), -math.inf)
    top = score.amax(dim=3, keepdim=True).clamp_(min=-3.0e38)
    p = torch.exp(score - top)
    p = p / p.sum(dim=3, keepdim=True).clamp_(min=1e-30)
    out = rows(torch.matmul(p.reshape(batch, kv_heads, group * queries, keys), v))
    r = {"out": out.to(t)}
    if not case["train"]:
        return r
    dout = folded(s["dout"])
    dp = rows(torch.matmul(dout, v.transpose(2, 3).contiguous()))
    ds = p * (dp - (p * dp).sum(dim=3, keepdim=True))
    if case["buckets"]:
        r["dtable"] = _sum_by_bucket(ds.sum(dim=0), s["map"], case["buckets"], keys - queries).to(t)
    ds = ds.reshape(batch, kv_heads, group * queries, keys)
    r["dq"] = rows(torch.matmul(ds, k) * scale).to(t)
    r["dk"] = (torch.matmul(ds.transpose(2, 3).contiguous(), q) * scale).to(t)
    r["dv"] = torch.matmul(p.reshape(batch, kv_heads, group * queries, keys).transpose(2, 3).contiguous(), dout).to(t)
    return r


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def _pairs(case):
    """(query, key) pairs of one head that the triangle leaves."""
    queries, keys = case["queries"], case["keys"]
    return queries * keys - queries * (queries - 1) // 2 if case["causal"] else queries * keys


def work(case):
    size = _BYTES[case["type"]]
    if case["op"] == "layer_norm":
        rows, dim = case["rows"], case["dim"]
        tensors, ops_each = (4 if case["residual"] else 2), 8
        if case["train"]:
            tensors, ops_each = tensors + (3 if case["residual"] else 2), 22       # dy, (ds,) and dx
        return {"bytes": size * (tensors * rows * dim + (4 if case["train"] else 2) * dim), "flops": ops_each * rows * dim}
    if case["op"] == "relative_bias":
        n = case["heads"] * case["queries"] * case["keys"]
        return {"bytes": size * (2 * n + 2 * case["buckets"] * case["heads"]), "flops": n}
    queries_bytes = size * case["batch"] * case["heads"] * case["queries"] * case["dim"]
    keys_bytes = size * case["batch"] * case["kv_heads"] * case["keys"] * case["dim"]
    products = 7 if case["train"] else 2                     # the backward pass makes the scores once more
    return {"bytes": queries_bytes * (4 if case["train"] else 2) + keys_bytes * (4 if case["train"] else 2),
            "flops": 2 * products * case["batch"] * case["heads"] * case["dim"] * _pairs(case)}


# ------------------------------------------------------------------------------------------------ the definitions, in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "layer_norm":
        return _norm_exact(case, s)
    if case["op"] == "relative_bias":
        return _bias_exact(case, s)
    return _attention_exact(case, s)


def _norm_exact(case, s):
    leaf = {k: s[k].double().requires_grad_() for k in ("x", "weight", "bias")}
    total = leaf["x"] * 1.0 if s["residual"] is None else leaf["x"] + s["residual"].double()
    var, mean = torch.var_mean(total, dim=1, unbiased=False, keepdim=True)
    y = (total - mean) / torch.sqrt(var + _EPS) * leaf["weight"] + leaf["bias"]
    out = {"y": y.detach()}
    if case["residual"]:
        out["sum"] = total.detach()
    if case["train"]:
        loss = (y * s["dy"].double()).sum()
        if case["residual"]:
            loss = loss + (total * s["ds"].double()).sum()
        out["dx"], out["dweight"], out["dbias"] = torch.autograd.grad(loss, [leaf["x"], leaf["weight"], leaf["bias"]])
    return out


def _diagonal_buckets(case, low, high):
    """Buckets of the distances low .. high."""
    far = case["distance"]
    return torch.tensor([_bucket_of(max(-far, min(far, d)), case["buckets"], far, case["causal"]) for d in range(low, high + 1)], device="cuda")


def _bias_exact(case, s):
    heads, queries, keys = case["heads"], case["queries"], case["keys"]
    table, low = s["table"].double(), 1 - keys                      # distances run from 1 - keys to queries - 1 + (keys - queries)
    line = table[_diagonal_buckets(case, low, keys - 1)].t().contiguous()          # [heads, distances]
    bias = torch.stack([line[:, keys - 1 - (keys - queries + i):][:, :keys] for i in range(queries)], dim=1)
    along = torch.zeros(heads, 2 * keys - 1, dtype=torch.float64, device="cuda")   # the gradient summed along each diagonal
    for i in range(queries):
        first = keys - 1 - (keys - queries + i)
        along[:, first:first + keys] += s["dbias"][:, i].double()
    dtable = torch.zeros(case["buckets"], heads, dtype=torch.float64, device="cuda")
    where = _diagonal_buckets(case, low, keys - 1)
    for b in range(case["buckets"]):
        dtable[b] = along[:, where == b].sum(dim=1)
    return {"bias": bias, "dtable": dtable}


def _attention_exact(case, s):
    batch, heads, kv_heads, queries, keys, dim = (case[k] for k in ("batch", "heads", "kv_heads", "queries", "keys", "dim"))
    group, dev = heads // kv_heads, s["q"].device
    small = batch * heads if queries * keys <= 1 << 16 else 1          # short sequences: a whole sequence's heads at a time
    out = torch.zeros(batch, heads, queries, dim, dtype=torch.float64, device=dev)
    dq, dk, dv = out.clone(), torch.zeros(batch, kv_heads, keys, dim, dtype=torch.float64, device=dev), None
    dv = dk.clone()
    dtable = torch.zeros(case["buckets"], heads, dtype=torch.float64, device=dev)
    row, col = torch.arange(queries, device=dev).unsqueeze(1), torch.arange(keys, device=dev)
    if case["buckets"]:
        line = _diagonal_buckets(case, -keys - queries, keys + queries)
    for b in range(batch):
        first = int(s["offset"][b]) if s["offset"] is not None else keys - queries
        shut = torch.zeros(queries, keys, dtype=torch.bool, device=dev)
        if case["causal"]:
            shut |= col > row + first
        if s["lengths"] is not None:
            shut |= col >= s["lengths"][b]
        if s["mask"] is not None:
            shut |= ~s["mask"][b, 0]
        none = shut.all(dim=1, keepdim=True)
        for h0 in range(0, heads, heads if small > 1 else 1):
            hs = list(range(h0, h0 + (heads if small > 1 else 1)))
            kv = torch.tensor([h // group for h in hs], device=dev)
            q, k, v = s["q"][b, hs].double(), s["k"][b].index_select(0, kv).double(), s["v"][b].index_select(0, kv).double()
            score = torch.bmm(q, k.transpose(1, 2).contiguous()) / math.sqrt(dim)
            if case["buckets"]:
                ids = line[col - row - first + keys + queries]
                score += s["table"].double()[:, hs].t()[:, ids]
            score = score.masked_fill(shut, -math.inf).masked_fill(none, 0.0)
            p = torch.softmax(score, dim=2).masked_fill(none, 0.0)
            o = torch.bmm(p, v)
            out[b, hs] = o
            if not case["train"]:
                continue
            do = s["dout"][b, hs].double()
            ds = p * (torch.bmm(do, v.transpose(1, 2).contiguous()) - (do * o).sum(dim=2, keepdim=True))
            dq[b, hs] = torch.bmm(ds, k) / math.sqrt(dim)
            dk[b].index_add_(0, kv, torch.bmm(ds.transpose(1, 2).contiguous(), q) / math.sqrt(dim))
            dv[b].index_add_(0, kv, torch.bmm(p.transpose(1, 2).contiguous(), do))
            if case["buckets"]:
                for at, h in enumerate(hs):
                    dtable[:, h] += torch.bincount(ids.reshape(-1), weights=ds[at].reshape(-1), minlength=case["buckets"])
    r = {"out": out}
    if case["train"]:
        if case["buckets"]:
            r["dtable"] = dtable
        r.update(dq=dq, dk=dk, dv=dv)
    return r
