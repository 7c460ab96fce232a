"""The operators of a decoder layer outside its contractions: layer norm, rotary positions, attention.

Each comes in the directions that a program calls: forward for prompts and training, the gradients, and attention of
a few new tokens over a cache.  A pass is one call of a linked operator (`Context.layer_norm`, `layer_norm_grad`,
`rotary`, `attention`, `attention_grad` of `ocannl_b200.backend`) on nodes that stay on the GPU.

Definitions, for nodes in row-major order, statistics and sums in single precision or better:

  norm       h = x + r;  mean = sum(h) / n;  rstd = 1 / sqrt(sum((h - mean)^2) / n + eps)
             y = (h - mean) * rstd * gamma + beta                                  outputs y, h, mean, rstd
  norm grad  u = (h - mean) * rstd;  g = dy * gamma
             dx = rstd * (g - sum(g) / n - u * sum(g * u) / n) + dh;  dgamma = sum_rows(dy * u);  dbeta = sum_rows(dy)
  rotary     of a head's first 2 m elements, pairs (x_i, x_{i + m}) (half) or (x_2i, x_2i+1) (interleaved), i < m,
             turn by the angle position * f_i and are multiplied by a magnitude; the others are copied
  rotary grad  the same with the angle negated
  attention  x_rj = scale * <q_r, k_j>;  c = cap * tanh(x / cap) with a cap, x without;  s = c - slope_h * |pos_r - j|
             out_r = sum_j softmax_j(s_rj) v_j over the visible keys, lse_r = log sum_j exp(s_rj); no visible key: 0, -inf
             pos_r = len - queries + r; visible: j < len, j <= pos_r (causal) or j <= pos_r or j < prefix (prefix), and,
             with documents, the same document, not a negative one; len is the number of keys where no lengths are given
  attention grad  p = exp(s - lse);  dv_j = sum_r p_rj do_r;  ds_rj = p_rj (<do_r, v_j> - <do_r, out_r>)
             dx = ds * (1 - (c / cap)^2);  dq_r = scale * sum_j dx_rj k_j;  dk_j = scale * sum_r dx_rj q_r
             (a key head's gradients are sums over the query heads that share it)
"""
import math

import torch

own = False
EPS = 1e-5

_TORCH = {"single": torch.float32, "half": torch.float16, "bfloat16": torch.bfloat16}


def listed():
    return [
        # the norm of one new token: latency alone
        dict(name="norm_1x512_bf16", kind="norm", rows=1, n=512, prec="bfloat16", grad=False, stream=True),
        # the benchmark's transformer: 64 sequences of 256 positions, residual and norm
        dict(name="norm_16384x512_bf16", kind="norm", rows=16384, n=512, prec="bfloat16", grad=False, stream=True),
        # its gradients, with the sums over all rows for the scale and the shift
        dict(name="norm_grad_16384x512_bf16", kind="norm", rows=16384, n=512, prec="bfloat16", grad=True, stream=True),
        # widths and row counts that come from data, in default precision
        dict(name="norm_grad_1999x777_f32", kind="norm", rows=1999, n=777, prec="single", grad=True, stream=False),
        # queries and keys of the benchmark's transformer
        dict(name="rotary_64x256_bf16", kind="rotary", batch=64, seq=256, heads=8, kv_heads=8, d_head=64, turned=64, layout="half",
             scaling="none", far=0, prec="bfloat16", grad=False),
        # the gradient for a third of a head, at far positions of a stretched context, grouped heads
        dict(name="rotary_grad_4x1999_f16", kind="rotary", batch=4, seq=1999, heads=12, kv_heads=4, d_head=96, turned=32,
             layout="interleaved", scaling="yarn", far=1000000, prec="half", grad=True),
        # one layer's attention of the benchmark's transformer
        dict(name="attn_64x256_bf16", kind="attn", batch=64, queries=256, keys=256, heads=8, kv_heads=8, d_head=64, mask="causal",
             docs=False, lengths=False, cap=0.0, slopes=False, prec="bfloat16", grad=False),
        # long rows of packed documents, capped scores, grouped heads: evaluating a prompt
        dict(name="attn_2x4096_docs_cap_bf16", kind="attn", batch=2, queries=4096, keys=4096, heads=16, kv_heads=4, d_head=128,
             mask="causal", docs=True, lengths=False, cap=50.0, slopes=False, prec="bfloat16", grad=False),
        # a training step's gradients at the benchmark's sizes
        dict(name="attn_grad_64x256_bf16", kind="attn", batch=64, queries=256, keys=256, heads=8, kv_heads=8, d_head=64,
             mask="causal", docs=False, lengths=False, cap=0.0, slopes=False, prec="bfloat16", grad=True),
        # gradients over long rows, a prefix that all positions see, a bias by distance, grouped heads: the largest
        dict(name="attn_grad_2x4096_prefix_bf16", kind="attn", batch=2, queries=4096, keys=4096, heads=16, kv_heads=4, d_head=128,
             mask="prefix", docs=False, lengths=False, cap=0.0, slopes=True, prec="bfloat16", grad=True),
        # the next token of 16 sequences over caches of up to 8192 keys
        dict(name="attn_1_of_8192_bf16", kind="attn", batch=16, queries=1, keys=8192, heads=32, kv_heads=8, d_head=128,
             mask="causal", docs=False, lengths=True, cap=0.0, slopes=False, prec="bfloat16", grad=False),
        # default precision, odd lengths and head sizes, every term of the score
        dict(name="attn_grad_3x333_f32", kind="attn", batch=3, queries=333, keys=333, heads=5, kv_heads=5, d_head=40, mask="prefix",
             docs=True, lengths=False, cap=30.0, slopes=True, prec="single", grad=True),
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, spread evenly over the logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["norm", "norm", "rotary", "attn", "attn", "attn", "attn"])
    prec = rng.choice(["bfloat16", "bfloat16", "half", "single"])
    if kind == "norm":
        n = _log(rng, 16, 16384)
        return dict(kind=kind, rows=_log(rng, 1, (1 << 25) // n), n=n if rng.random() < 0.4 else max(16, n // 16 * 16), prec=prec,
                    grad=rng.random() < 0.5, stream=rng.random() < 0.5)
    if kind == "rotary":
        d = rng.choice([32, 64, 64, 80, 96, 128, 128])
        kv = _log(rng, 1, 8)
        seq = _log(rng, 1, 8192)
        return dict(kind=kind, batch=_log(rng, 1, max(1, 16384 // seq)), seq=seq, heads=kv * rng.choice([1, 1, 2, 4]), kv_heads=kv, d_head=d,
                    turned=rng.choice([d, d, d // 2]), layout=rng.choice(["half", "interleaved"]),
                    scaling=rng.choice(["none", "linear", "ntk", "yarn"]), far=rng.choice([0, 0, 100000, 1000000]), prec=prec,
                    grad=rng.random() < 0.4)
    d = rng.choice([32, 64, 64, 64, 72, 96, 128, 128])
    kv = _log(rng, 1, 8)
    heads = kv * rng.choice([1, 1, 2, 4])
    case = dict(kind=kind, heads=heads, kv_heads=kv, d_head=d, cap=rng.choice([0.0, 0.0, 20.0, 50.0]), slopes=rng.random() < 0.3)
    if rng.random() < 0.35:          # a few new tokens over a cache
        queries, keys = rng.choice([1, 1, 1, 2, 5]), _log(rng, 16, 16384)
        batch = _log(rng, 1, max(1, min(64, (1 << 18) // keys)))
        return dict(case, batch=batch, queries=queries, keys=keys, mask="causal", docs=False, lengths=True,
                    prec="bfloat16" if prec == "single" else prec, grad=False)
    seq = _log(rng, 16, 4096 if prec != "single" else 1024)
    # at most half the pairs of the largest listed case
    room = max(1, (1 << 28) // (seq * seq * heads))
    return dict(case, batch=_log(rng, 1, min(room, 128)), queries=seq, keys=seq, mask=rng.choice(["causal", "causal", "prefix", "none"]),
                docs=rng.random() < 0.4, lengths=rng.random() < 0.2, prec=prec, grad=rng.random() < 0.5)


# ------------------------------------------------------------------ inputs
def _frequencies(case):
    """Radians per position of each pair, in double precision, and the magnitude."""
    m, base, factor, original = case["turned"] // 2, 10000.0, 8.0, 4096.0
    f = [base ** (-i / m) for i in range(m)]
    if case["scaling"] == "linear":
        return [x / factor for x in f], 1.0
    if case["scaling"] == "ntk":
        longer = base * factor ** (m / max(1, m - 1))
        return [longer ** (-i / m) for i in range(m)], 1.0
    if case["scaling"] == "yarn":
        # pairs that turn often over the original context stay, those that turn less than once are stretched
        def at(turns):
            return m * math.log(original / (2.0 * math.pi * turns)) / math.log(base)
        low, high = max(0, math.floor(at(32.0))), min(m - 1, math.ceil(at(1.0)))
        ramp = [min(1.0, max(0.0, (i - low) / max(1e-3, high - low))) for i in range(m)]
        return [x * (1.0 - r) + x / factor * r for x, r in zip(f, ramp)], 0.1 * math.log(factor) + 1.0
    return f, 1.0


def _documents(gen, batch, seq):
    """Packed rows: documents of a few lengths one behind the other, the last positions of some rows padding."""
    starts = torch.rand((batch, seq), generator=gen, device="cuda") < 4.0 / seq
    ids = torch.cumsum(starts.int(), 1).int()
    tail = torch.randint(0, max(1, seq // 8), (batch, 1), generator=gen, device="cuda")
    keep = torch.arange(seq, device="cuda")[None, :] < seq - tail * (torch.rand((batch, 1), generator=gen, device="cuda") < 0.5)
    return torch.where(keep, ids, -1).int()


def _inputs(case, seed):
    """{node: values} of a case, on the GPU, from the seed alone."""
    gen = torch.Generator(device="cuda")
    gen.manual_seed(int(seed))
    t = _TORCH[case["prec"]]

    def normal(*shape, scale=1.0, shift=0.0):
        return torch.randn(shape, generator=gen, device="cuda") * scale + shift

    x = {}
    if case["kind"] == "norm":
        rows, n = case["rows"], case["n"]
        # activations with a mean of their own and rows of different size
        size = torch.exp(normal(rows, 1, scale=0.5))
        x["x"] = (normal(rows, n) * size + normal(rows, 1, scale=0.3)).to(t)
        x["gamma"] = normal(n, scale=0.2, shift=1.0)
        if not case["grad"]:
            x["beta"] = normal(n, scale=0.2)
            if case["stream"]:
                x["r"] = (normal(rows, n) * size).to(t)
        else:
            h = x["x"].float()
            mean = h.mean(1)
            x["mean"], x["rstd"] = mean, torch.rsqrt((h - mean[:, None]).square().mean(1) + EPS)
            x["dy"] = normal(rows, n, scale=0.1).to(t)
            if case["stream"]:
                x["dh"] = normal(rows, n, scale=0.1).to(t)
    elif case["kind"] == "rotary":
        b, s, d = case["batch"], case["seq"], case["d_head"]
        x["q"], x["k"] = normal(b, s, case["heads"], d).to(t), normal(b, s, case["kv_heads"], d).to(t)
        start = torch.randint(0, case["far"] + 1, (b, 1), generator=gen, device="cuda")
        x["positions"] = (start + torch.arange(s, device="cuda")[None, :]).int()
    else:
        b, s, n, d = case["batch"], case["queries"], case["keys"], case["d_head"]
        # with a cap, scores grow up to it
        spread = 2.0 if case["cap"] else 1.0
        x["q"] = normal(b, s, case["heads"], d, scale=spread).to(t)
        x["k"], x["v"] = normal(b, n, case["kv_heads"], d, scale=spread).to(t), normal(b, n, case["kv_heads"], d).to(t)
        if case["slopes"]:
            x["slopes"] = torch.exp2(-8.0 * torch.arange(1, case["heads"] + 1, device="cuda") / case["heads"]).float()
        if case["mask"] == "prefix":
            x["prefix"] = torch.randint(0, n // 2 + 1, (b,), generator=gen, device="cuda").int()
        if case["docs"]:
            x["docs"] = _documents(gen, b, n)
        if case["lengths"]:
            x["lengths"] = torch.randint(max(s, n // 2), n + 1, (b,), generator=gen, device="cuda").int()
        if case["grad"]:
            out, lse = _attention(case, x)
            x["out"], x["lse"] = out.to(t), lse
            x["d_out"] = normal(b, s, case["heads"], d, scale=0.1).to(t)
    return x


# ------------------------------------------------------------------ plain forms
def _norm(case, x):
    h = x["x"].float()
    if "r" in x:
        h = h + x["r"].float()
    mean = h.mean(1)
    centred = h - mean[:, None]
    rstd = 1.0 / torch.sqrt((centred * centred).mean(1) + EPS)
    y = centred * rstd[:, None] * x["gamma"] + x["beta"]
    t = x["x"].dtype
    out = {"y": y.to(t), "mean": mean, "rstd": rstd}
    if "r" in x:
        out["h"] = h.to(t)
    return out


def _norm_grad(case, x):
    dy = x["dy"].float()
    u = (x["x"].float() - x["mean"][:, None]) * x["rstd"][:, None]
    g = dy * x["gamma"]
    dx = x["rstd"][:, None] * (g - g.mean(1, keepdim=True) - u * (g * u).mean(1, keepdim=True))
    if "dh" in x:
        dx = dx + x["dh"].float()
    # sums over many rows: in 64 bits
    return {"dx": dx.to(x["x"].dtype), "dgamma": (dy * u).double().sum(0).float(), "dbeta": dy.double().sum(0).float()}


def _turn(case, x, cos, sin):
    m = case["turned"] // 2
    a = x.float()
    turned, rest = a[..., :2 * m], a[..., 2 * m:]
    if case["layout"] == "half":
        u, w = turned[..., :m], turned[..., m:]
        done = torch.cat((u * cos - w * sin, u * sin + w * cos), -1)
    else:
        u, w = turned[..., 0::2], turned[..., 1::2]
        done = torch.stack((u * cos - w * sin, u * sin + w * cos), -1).flatten(-2)
    return torch.cat((done, rest), -1).to(x.dtype)


def _rotary(case, x):
    f, magnitude = _frequencies(case)
    # far positions: angles in 64 bits
    angle = x["positions"].double()[:, :, None, None] * torch.tensor(f, dtype=torch.float64, device="cuda")
    if case["grad"]:
        angle = -angle
    cos, sin = (torch.cos(angle) * magnitude).float(), (torch.sin(angle) * magnitude).float()
    return {"q_out": _turn(case, x["q"], cos, sin), "k_out": _turn(case, x["k"], cos, sin)}


def _visible(case, x):
    """[batch, 1, queries, keys] of truth values, and |position - key| in the same shape."""
    b, s, n = case["batch"], case["queries"], case["keys"]
    length = x["lengths"].long() if case["lengths"] else torch.full((b,), n, device="cuda")
    pos = (length - s)[:, None] + torch.arange(s, device="cuda")
    j = torch.arange(n, device="cuda")
    seen = (j < length[:, None])[:, None, :].expand(b, s, n)
    if case["mask"] == "causal":
        seen = seen & (j <= pos[:, :, None])
    elif case["mask"] == "prefix":
        seen = seen & ((j <= pos[:, :, None]) | (j < x["prefix"][:, None, None]))
    if case["docs"]:
        theirs = x["docs"]
        mine = theirs[:, n - s:]
        seen = seen & (mine[:, :, None] == theirs[:, None, :]) & (mine[:, :, None] >= 0)
    return seen[:, None], (pos[:, :, None] - j).abs().float()[:, None]


def _scores(case, x):
    """Capped scores c and the scores s with the bias, [batch, heads, queries, keys]."""
    group = case["heads"] // case["kv_heads"]
    q = x["q"].float().transpose(1, 2)
    k = x["k"].float().transpose(1, 2).repeat_interleave(group, 1)
    c = torch.matmul(q, k.transpose(2, 3)) * (1.0 / math.sqrt(case["d_head"]))
    if case["cap"]:
        c = case["cap"] * torch.tanh(c / case["cap"])
    seen, far = _visible(case, x)
    s = c - x["slopes"][:, None, None] * far if case["slopes"] else c
    return q, k, c, torch.where(seen, s, -math.inf)


def _attention(case, x):
    group = case["heads"] // case["kv_heads"]
    _, _, _, s = _scores(case, x)
    top = s.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    e = torch.exp(s - top)
    total = e.sum(-1, keepdim=True)
    v = x["v"].float().transpose(1, 2).repeat_interleave(group, 1)
    out = torch.matmul(e, v) / torch.where(total == 0.0, 1.0, total)
    return out.transpose(1, 2), (top + torch.log(total))[..., 0]


def _attention_grad(case, x):
    b, n, h, hk, d, t = case["batch"], case["keys"], case["heads"], case["kv_heads"], case["d_head"], x["q"].dtype
    q, k, c, s = _scores(case, x)
    lse = torch.where(x["lse"] == -math.inf, 0.0, x["lse"])
    p = torch.exp(s - lse[..., None])
    do, out = x["d_out"].float().transpose(1, 2), x["out"].float().transpose(1, 2)
    v = x["v"].float().transpose(1, 2).repeat_interleave(h // hk, 1)
    ds = p * (torch.matmul(do, v.transpose(2, 3)) - (do * out).sum(-1, keepdim=True))
    if case["cap"]:
        ds = ds * (1.0 - (c / case["cap"]).square())
    ds = ds * (1.0 / math.sqrt(d))
    dq = torch.matmul(ds, k)
    dk = torch.matmul(ds.transpose(2, 3), q).reshape(b, hk, h // hk, n, d).sum(2)
    dv = torch.matmul(p.transpose(2, 3), do).reshape(b, hk, h // hk, n, d).sum(2)
    return {g: a.transpose(1, 2).to(t) for g, a in (("dq", dq), ("dk", dk), ("dv", dv))}


def _plain(case, x):
    if case["kind"] == "norm":
        return _norm_grad(case, x) if case["grad"] else _norm(case, x)
    if case["kind"] == "rotary":
        return _rotary(case, x)
    if case["grad"]:
        return _attention_grad(case, x)
    out, lse = _attention(case, x)
    return {"out": out.to(x["q"].dtype), "lse": lse}


# ------------------------------------------------------------------ the framework's operators
_device = None


def _results(case, x):
    """{node: (dims, type)} of what a case computes."""
    t = _TORCH[case["prec"]]
    if case["kind"] == "norm":
        rows, n = case["rows"], case["n"]
        if case["grad"]:
            return {"dx": ((rows, n), t), "dgamma": ((n,), torch.float32), "dbeta": ((n,), torch.float32)}
        r = {"y": ((rows, n), t), "mean": ((rows,), torch.float32), "rstd": ((rows,), torch.float32)}
        return dict(r, h=((rows, n), t)) if "r" in x else r
    if case["kind"] == "rotary":
        return {"q_out": (tuple(x["q"].shape), t), "k_out": (tuple(x["k"].shape), t)}
    if case["grad"]:
        return {"d" + g: (tuple(x[g].shape), t) for g in "qkv"}
    return {"out": (tuple(x["q"].shape), t), "lse": ((case["batch"], case["heads"], case["queries"]), torch.float32)}


class _Buffer:
    """A node's memory, for torch to look at."""


class _Program:
    """A context that holds a case's nodes and the operator linked to them; given back together, when nothing looks at a node
    any more (every view keeps its program)."""

    def __init__(self, case, x):
        global _device
        from ocannl_b200 import backend as bk
        from ocannl_b200.low_level import Tnode
        if _device is None:
            _device = bk.Device(0)
        self.context = self.operator = None
        kinds = {torch.float32: "single", torch.float16: "half", torch.bfloat16: "bfloat16", torch.int32: "int32"}
        nodes = [(n, tuple(v.shape), v.dtype) for n, v in x.items()] + [(n, d, t) for n, (d, t) in _results(case, x).items()]
        self.context = bk.Context(_device).allocate([Tnode(i + 1, n, kinds[t], d) for i, (n, d, t) in enumerate(nodes)])
        self.types = {n: t for n, _, t in nodes}
        _device.await_()
        for n, v in x.items():
            self.view(n).copy_(v)
        torch.cuda.synchronize()
        self.operator = self.link(case, self.context, x)

    def link(self, case, ctx, x):
        if case["kind"] == "norm":
            if case["grad"]:
                return ctx.layer_norm_grad("x", "dy", "dx", mean="mean", rstd="rstd", gamma="gamma", dgamma="dgamma", dbeta="dbeta",
                                           d_total="dh" if "dh" in x else None)
            more = dict(residual="r", total="h") if "r" in x else {}
            return ctx.layer_norm("x", "y", gamma="gamma", beta="beta", mean="mean", rstd="rstd", eps=EPS, **more)
        if case["kind"] == "rotary":
            f, magnitude = _frequencies(case)
            return ctx.rotary([("q", "q_out"), ("k", "k_out")], frequencies=f, magnitude=magnitude, positions="positions",
                              layout=case["layout"], inverse=case["grad"])
        documents = ("query_docs", "docs") if "query_docs" in x else "docs" if "docs" in x else None
        terms = dict(mask=case["mask"], prefix="prefix" if "prefix" in x else None, documents=documents,
                     lengths="lengths" if "lengths" in x else None, slopes="slopes" if "slopes" in x else None, cap=case["cap"])
        if case["grad"]:
            return ctx.attention_grad("q", "k", "v", "out", "lse", "d_out", "dq", "dk", "dv", **terms)
        return ctx.attention("q", "k", "v", "out", lse="lse", **terms)

    def view(self, ident):
        """A node's memory as a tensor; keeps the program that owns it."""
        pool, offset, t = self.context.arrays[ident]
        address, _ = _device.pool_address(pool)

        buffer = _Buffer()
        buffer.program = self
        buffer.__cuda_array_interface__ = {"shape": tuple(t.dims), "data": (address + offset, False), "version": 3, "strides": None,
                                           "typestr": {"single": "<f4", "half": "<f2", "bfloat16": "<i2", "int32": "<i4"}[t.prec]}
        return torch.as_tensor(buffer, device="cuda").view(self.types[ident])

    def __del__(self):
        if self.context is not None and getattr(self, "operator", None) is not None:
            _device.await_()
            self.operator.free()
            for pool in {p for p, _, _ in self.context.arrays.values()}:
                _device.free_pool(pool)
            self.context = None


class _State:
    pass


def prepare(case, seed):
    s = _State()
    s.case, s.x = case, _inputs(case, seed)
    if own:
        # the nodes lie in the context's pool, the operator is linked to them; with lengths the queries' documents, which are those of
        # the last entries and not of the queries' positions, are a node of their own
        if "docs" in s.x and "lengths" in s.x:
            s.x["query_docs"] = s.x["docs"][:, case["keys"] - case["queries"]:].contiguous()
        s.program = _Program(case, s.x)
        s.outputs = {n: s.program.view(n) for n in _results(case, s.x)}
        s.x = None
    return s


def run(s):
    if own:
        s.program.operator.run()
        return s.outputs
    return _plain(s.case, s.x)


# ------------------------------------------------------------------ work
def _pairs(case):
    """Pairs of a query and a key that a head looks at, as many as the distributions of the inputs give on average."""
    s, n = case["queries"], case["keys"]
    length = 0.75 * n if case["lengths"] else float(n)
    if s < n and case["lengths"] and s <= 16:
        seen = length
    elif case["mask"] == "causal":
        seen = length - s / 2.0 if length >= s else length / 2.0
    elif case["mask"] == "prefix":
        seen = length / 2.0 + n / 24.0      # a prefix of a random quarter: a twenty-fourth of the pairs behind the diagonal
    else:
        seen = length
    if case["docs"]:
        seen = min(seen, n / 4.0 if case["mask"] == "none" else n / 8.0 + (n / 24.0 if case["mask"] == "prefix" else 0.0))
    return s * max(1.0, seen)


def work(case):
    size = 4 if case["prec"] == "single" else 2
    if case["kind"] == "norm":
        rows, n = case["rows"], case["n"]
        planes = (3 + case["stream"]) if case["grad"] else (2 + 2 * case["stream"])
        return {"bytes": planes * rows * n * size + 8 * rows + (12 if case["grad"] else 8) * n, "flops": (14.0 if case["grad"] else 8.0) * rows * n}
    if case["kind"] == "rotary":
        tokens = case["batch"] * case["seq"]
        heads = case["heads"] + case["kv_heads"]
        return {"bytes": 2 * tokens * heads * case["d_head"] * size + 4 * tokens, "flops": 3.0 * tokens * heads * case["turned"]}
    b, s, n, d = case["batch"], case["queries"], case["keys"], case["d_head"]
    keys = 0.75 * n if case["lengths"] else n
    q, kv = b * s * case["heads"] * d * size, b * keys * case["kv_heads"] * d * size
    rows = b * s * case["heads"] * 4
    pairs = b * case["heads"] * _pairs(case)
    if case["grad"]:
        return {"bytes": 4 * q + 4 * kv + rows, "flops": 10.0 * pairs * d}
    return {"bytes": 2 * q + 2 * kv + rows, "flops": 4.0 * pairs * d}


# ------------------------------------------------------------------ the definitions in 64 bits
def _exact_attention(case, x):
    """A sequence and a key head at a time."""
    b, s, n, d, group = case["batch"], case["queries"], case["keys"], case["d_head"], case["heads"] // case["kv_heads"]
    res = {g: torch.zeros(x[g].shape, dtype=torch.float64, device="cuda") for g in "qkv"}
    out = torch.zeros(x["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.full((b, case["heads"], s), -math.inf, dtype=torch.float64, device="cuda")
    root = math.sqrt(d)
    for i in range(b):
        length = int(x["lengths"][i]) if case["lengths"] else n
        row = torch.arange(length - s, length, device="cuda")[:, None]
        col = torch.arange(length, device="cuda")[None, :]
        hidden = torch.zeros((s, length), dtype=torch.bool, device="cuda")
        if case["mask"] != "none":
            hidden |= col > row
        if case["mask"] == "prefix":
            hidden &= col >= int(x["prefix"][i])
        if case["docs"]:
            ids = x["docs"][i]
            hidden |= (ids[n - s:, None] != ids[None, :length]) | (ids[n - s:, None] < 0)
        empty = hidden.all(1)
        for g in range(case["kv_heads"]):
            k, v = x["k"][i, :length, g].double(), x["v"][i, :length, g].double()
            for h in range(g * group, (g + 1) * group):
                q = x["q"][i, :, h].double()
                raw = torch.einsum("rd,jd->rj", q, k) / root
                soft = case["cap"] * torch.tanh(raw / case["cap"]) if case["cap"] else raw
                z = soft - float(x["slopes"][h]) * (row - col).abs() if case["slopes"] else soft
                z = z.masked_fill(hidden, -math.inf)
                if not case["grad"]:
                    w = torch.softmax(z, 1).masked_fill(hidden | empty[:, None], 0.0)
                    out[i, :, h] = torch.einsum("rj,jd->rd", w, v)
                    lse[i, h] = torch.logsumexp(z, 1)
                    continue
                do = x["d_out"][i, :, h].double()
                w = torch.exp(z - x["lse"][i, h].double()[:, None]).masked_fill(hidden, 0.0)
                res["v"][i, :length, g] += torch.einsum("rj,rd->jd", w, do)
                dz = w * (torch.einsum("rd,jd->rj", do, v) - torch.einsum("rd,rd->r", do, x["out"][i, :, h].double())[:, None])
                if case["cap"]:
                    dz = dz / torch.cosh(raw / case["cap"]).square()
                res["q"][i, :, h] = torch.einsum("rj,jd->rd", dz, k) / root
                res["k"][i, :length, g] += torch.einsum("rj,rd->jd", dz, q) / root
    return {"d" + g: a for g, a in res.items()} if case["grad"] else {"out": out, "lse": lse}


def exact(case, seed):
    x = _inputs(case, seed)
    if case["kind"] == "attn":
        return _exact_attention(case, x)
    if case["kind"] == "rotary":
        f, magnitude = _frequencies(case)
        m, sign = case["turned"] // 2, -1.0 if case["grad"] else 1.0
        angle = torch.einsum("bs,i->bsi", x["positions"].double(), torch.tensor(f, dtype=torch.float64, device="cuda")) * sign
        turn = torch.polar(torch.full_like(angle, magnitude), angle)[:, :, None, :]
        res = {}
        for n in "qk":
            a = x[n].double()
            first, second = (slice(0, m), slice(m, 2 * m)) if case["layout"] == "half" else (slice(0, 2 * m, 2), slice(1, 2 * m, 2))
            z = torch.complex(a[..., first], a[..., second]) * turn
            y = a.clone()
            y[..., first], y[..., second] = z.real, z.imag
            res[n + "_out"] = y
        return res
    v = {n: a.double() for n, a in x.items()}
    if case["grad"]:
        unit = (v["x"] - v["mean"].unsqueeze(1)) * v["rstd"].unsqueeze(1)
        g = torch.einsum("rn,n->rn", v["dy"], v["gamma"])
        along = torch.einsum("rn,rn->r", g, unit) / case["n"]
        dx = (g - (g.sum(1) / case["n"]).unsqueeze(1) - unit * along.unsqueeze(1)) * v["rstd"].unsqueeze(1) + v.get("dh", 0.0)
        return {"dx": dx, "dgamma": torch.einsum("rn,rn->n", v["dy"], unit), "dbeta": v["dy"].sum(0)}
    h = v["x"] + v.get("r", 0.0)
    var, mean = torch.var_mean(h, 1, correction=0)
    rstd = (var + EPS).rsqrt()
    res = {"y": (h - mean.unsqueeze(1)) * rstd.unsqueeze(1) * v["gamma"] + v["beta"], "mean": mean, "rstd": rstd}
    return dict(res, h=h) if "r" in v else res
