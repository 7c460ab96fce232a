"""The operators that answer with the next tokens: appending to a paged cache, attention over it, choosing a token.

A pass is one call of a linked operator (`Context.cache_append`, `cache_attention`, `sample` of `ocannl_b200.backend`) on nodes that
stay on the GPU.

The cache of keys (and that of values) is [pages, kv_heads, page, d], in the nodes' type or in 8 bits (e4m3) with a scale for each page and
head.  `pages` [batch, max_pages] says which page holds a sequence's tokens 0 .. page - 1, page .. 2 page - 1, and so on (a number that is
no page's: there is none), `lengths` [batch] how many tokens a sequence has, the new ones included.  New tokens are rows: those of
sequence b are starts[b] .. starts[b + 1] - 1, or tokens / batch each; row i of n lies at position lengths[b] - n + i.  Rows of no
sequence are left as they were.

  append     (x_i, x_{i + m}) or (x_2i, x_2i+1) of a key (and a query) turn by the angle position * f_i; keys and values go to their slots.  8 bits:
             scale = 2^e, the least e >= -40 with |x| <= 448 scale for all values that the page has received, code = x / scale rounded to e4m3;
             codes that the page held are rounded again where its scale grows
  attention  x_rj = scale * <q_r, k_j>;  s = cap * tanh(x / cap) with a cap, x without;  out_r = sum_j softmax_j(s_rj) v_j over the keys
             j <= position_r with j > position_r - window or j < sinks (all without a window);  lse_r = log sum_j exp(s_rj)
  sample     w_i = exp((x_i - max x) / temperature); in the order of falling x (ties: of rising i) the first n are kept: n is the least of top_k, of
             the fewest whose sum is at least top_p times that of the first top_k, and of those with w >= min_p; the token is the first kept one, in the
             order of i, at which the running sum exceeds uniform * the kept sum; logprob = log(w_token / kept sum).  temperature 0: the
             first largest, 0
"""
import math
import random

import torch

own = False

_TORCH = {"single": torch.float32, "half": torch.float16, "bfloat16": torch.bfloat16}


def _append(name, **more):
    return dict(dict(name=name, kind="append", heads=32, kv_heads=8, d_head=128, turned=128, layout="half", prec="bfloat16"), **more)


def _attend(name, **more):
    return dict(dict(name=name, kind="attend", heads=32, kv_heads=8, d_head=128, window=0, sinks=0, cap=0.0, prec="bfloat16"), **more)


def listed():
    return [
        # the next token of four sequences, the heads of the benchmark's transformer: latency alone
        _append("append_4x1_bf16", batch=4, tokens=4, most=1, heads=8, kv_heads=8, d_head=64, turned=64, page=16, max_len=256, bits8=False),
        # a step of a busy server: 256 sequences, their last pages partly filled, 8 bits
        _append("append_256x1_e4m3", batch=256, tokens=256, most=1, page=64, max_len=1024, bits8=True),
        # prompts of different lengths that arrive together, some rows of the batch empty, 8 bits
        _append("append_prompts_8192_e4m3", batch=6, tokens=8192, most=2048, page=64, max_len=4096, bits8=True),
        # the next token of four sequences of up to 256: latency alone
        _attend("attn_4x1_of_256_bf16", batch=4, tokens=4, most=1, heads=8, kv_heads=8, d_head=64, page=16, max_len=256, bits8=False),
        # a step of a server over caches in 8 bits
        _attend("attn_64x1_of_8192_e4m3", batch=64, tokens=64, most=1, page=64, max_len=8192, bits8=True),
        # long contexts, small pages
        _attend("attn_16x1_of_32768_bf16", batch=16, tokens=16, most=1, page=16, max_len=32768, bits8=False),
        # far beyond a window: sinks and the last 1024 tokens, the pages between given back
        _attend("attn_32x1_window_e4m3", batch=32, tokens=32, most=1, page=64, max_len=16384, window=1024, sinks=4, bits8=True),
        # parts of prompts beside each other, over what is in the cache before them: the largest
        _attend("attn_prompts_4096_of_8192_e4m3", batch=4, tokens=4096, most=1500, page=64, max_len=8192, bits8=True),
        # evaluating prompts with a window and capped scores, 16-bit cache
        _attend("attn_prompts_window_f16", batch=3, tokens=3000, most=1500, heads=16, kv_heads=4, page=32, max_len=4096, window=700, sinks=4,
                cap=30.0, bits8=False, prec="half"),
        # a character of the benchmark's models (27 of them) for 32 sequences: latency alone
        dict(name="sample_32x27_f32", kind="sample", rows=32, vocab=27, prec="single", top_k=0, top_p=False, min_p=False),
        # a server's step: every row with settings of its own, an odd vocabulary
        dict(name="sample_64x50021_bf16", kind="sample", rows=64, vocab=50021, prec="bfloat16", top_k=50, top_p=True, min_p=False),
        # many rows of a large vocabulary, no bound on the number kept
        dict(name="sample_256x131072_f32", kind="sample", rows=256, vocab=131072, prec="single", top_k=0, top_p=True, min_p=True),
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, spread evenly over the logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["append", "append", "attend", "attend", "attend", "sample", "sample"])
    prec = rng.choice(["bfloat16", "bfloat16", "half", "single"])
    if kind == "sample":
        vocab = _log(rng, 16, 262144)
        return dict(kind=kind, rows=_log(rng, 1, max(1, min(1024, (1 << 25) // vocab))), vocab=vocab, prec=prec, top_k=rng.choice([0, 1, 20, 50, 1000]),
                    top_p=rng.random() < 0.6, min_p=rng.random() < 0.4)
    kv = _log(rng, 1, 8)
    case = dict(kind=kind, heads=kv * rng.choice([1, 2, 4, 8]), kv_heads=kv, d_head=rng.choice([32, 64, 64, 80, 96, 128, 128]), prec=prec,
                page=rng.choice([8, 16, 16, 32, 64, 64, 128]), bits8=rng.random() < 0.5)
    d = case["d_head"]
    if kind == "append":
        most = rng.choice([1, 1, 1, _log(rng, 2, 4096)])
        batch = _log(rng, 1, max(1, min(512, 8192 // most)))
        case.update(turned=rng.choice([d, d, d // 2]), layout=rng.choice(["half", "interleaved"]))
        return dict(case, batch=batch, tokens=batch * most, most=most, max_len=max(most, _log(rng, 16, (1 << 18) // batch)))
    case.update(cap=rng.choice([0.0, 0.0, 20.0, 50.0]))
    if rng.random() < 0.6:           # a few new tokens
        most = rng.choice([1, 1, 1, 2, 5])
        max_len = _log(rng, 16, 32768)
        batch = _log(rng, 1, max(1, min(256, (1 << 19) // max_len)))
    else:                            # parts of prompts
        most = _log(rng, 16, 2048 if prec != "single" else 256)
        max_len = max(most, _log(rng, 64, 8192 if prec != "single" else 2048))
        batch = _log(rng, 1, max(1, min(16, (1 << 29) // (most * max_len * case["heads"]))))
    window = rng.choice([0, 0, _log(rng, 8, 4096)])
    return dict(case, batch=batch, tokens=batch * most, most=most, max_len=max_len, window=window, sinks=rng.choice([0, 4, 16]) if window else 0)


# ------------------------------------------------------------------ inputs
def _counts(case, seed):
    """New tokens of each sequence: `most` each without starts, a quarter of it to all of it else, as far as the rows go."""
    if case["most"] == 1:
        return [1] * case["batch"]
    rng, left, counts = random.Random(seed), case["tokens"], []
    for i in range(case["batch"]):
        counts.append(min(rng.randint(max(1, case["most"] // 4), case["most"]), left - (case["batch"] - 1 - i)))
        left -= counts[-1]
    return counts


def _max_pages(case):
    return -(-case["max_len"] // case["page"])


def _frequencies(case):
    m = case["turned"] // 2
    return [10000.0 ** (-i / m) for i in range(m)]


def _quantized(values, alive):
    """Codes (as e4m3 tensors) and scales of [pages, heads, page, d], over the slots that hold something."""
    amax = (values.abs() * alive).amax((2, 3))
    scale = _pow2(amax)
    return (values / scale[:, :, None, None]).clamp(-448.0, 448.0).to(torch.float8_e4m3fn), scale


def _pow2(amax):
    """The least power of two, 2^-40 at least, that 448 of are no less than amax."""
    m, e = torch.frexp(amax)                       # amax = m 2^e, 1/2 <= m < 1; 448 = 7/8 2^9
    e = torch.where(m > 0.875, e - 8, e - 9)
    return torch.exp2(torch.where(amax == 0, -40, e.clamp(min=-40)).to(amax.dtype))


def _inputs(case, seed):
    """{node: values} of a case, on the GPU, from the seed alone."""
    gen = torch.Generator(device="cuda")
    gen.manual_seed(int(seed))
    t = _TORCH[case["prec"]]

    def normal(*shape, scale=1.0):
        return torch.randn(shape, generator=gen, device="cuda") * scale

    def uniform(*shape):
        return torch.rand(shape, generator=gen, device="cuda")

    def pick(rows, *choices):
        return torch.tensor(choices, device="cuda")[torch.randint(0, len(choices), (rows,), generator=gen, device="cuda")]

    x = {}
    if case["kind"] == "sample":
        rows, vocab = case["rows"], case["vocab"]
        # logits of a model: most tokens far below a few, rows more and less certain
        x["logits"] = (normal(rows, vocab) * torch.exp(0.4 * normal(rows, 1) + 0.9) + 4.0 * (uniform(rows, vocab) < 8.0 / vocab)).to(t)
        x["uniform"] = uniform(rows)
        # one row in ten takes the largest
        x["temperature"] = torch.where(uniform(rows) < 0.1, 0.0, 0.6 + 0.7 * uniform(rows))
        if case["top_k"]:
            x["top_k"] = pick(rows, 0, case["top_k"], max(1, case["top_k"] // 2)).int()
        if case["top_p"]:
            x["top_p"] = pick(rows, 1.0, 0.95, 0.9, 0.5)
        if case["min_p"]:
            x["min_p"] = pick(rows, 0.0, 0.001, 0.02, 0.1)
        return x
    b, n, page, hk, d, mp = case["batch"], case["tokens"], case["page"], case["kv_heads"], case["d_head"], _max_pages(case)
    counts, rng = _counts(case, seed), random.Random(seed + 1)
    # a sequence that is appended to may be new; attention has half the longest at least
    lengths = [c + rng.randint(0 if case["kind"] == "append" else max(0, case["max_len"] // 2 - c), case["max_len"] - c) for c in counts]
    x["lengths"] = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    if case["most"] > 1:
        x["starts"] = torch.tensor([sum(counts[:i]) for i in range(b + 1)], dtype=torch.int32, device="cuda")
    # pages are handed out in no order; those that a window has left behind, and the sinks' not among them, are given back
    live = torch.arange(mp, device="cuda")[None, :] * page < x["lengths"][:, None]
    if case.get("window"):
        first = x["lengths"] - torch.tensor(counts, device="cuda") - case["window"]
        at = torch.arange(mp, device="cuda")[None, :] * page
        live &= (at + page > first[:, None]) | (at < case["sinks"])
    pages = (min(mp, (case["window"] + case["sinks"] + case["most"]) // page + 4) if case.get("window") else mp) * b + 3
    order = torch.randperm(pages - 1, generator=gen, device="cuda") + 1       # (page 0 is nobody's)
    number = torch.cumsum(live.reshape(-1).long(), 0) - 1
    x["pages"] = torch.where(live, order[number.clamp(0, pages - 2)].view(b, mp), -1).int()
    # what lies in slots that hold nothing: something of earlier sequences
    size = torch.exp(normal(pages, hk, 1, 1, scale=0.5))
    for g in "kv":
        values = normal(pages, hk, page, d) * size
        if case["bits8"]:
            x[g + "_cache"], x[g + "_scale"] = _quantized(values, torch.ones((), device="cuda"))
        else:
            x[g + "_cache"] = values.to(t)
        del values
    x["q"] = normal(n, case["heads"], d).to(t)
    if case["kind"] == "append":
        x["k"], x["v"] = normal(n, hk, d).to(t), normal(n, hk, d).to(t)
    return x


# ------------------------------------------------------------------ plain forms
def _rows(case, x):
    """Of every row: its sequence, its number in it, its position, and whether it has one."""
    n, b = case["tokens"], case["batch"]
    row = torch.arange(n, device="cuda")
    if "starts" in x:
        starts = x["starts"].long()
        seq = torch.bucketize(row, starts[1:], right=True).clamp(max=b - 1)
        i, count = row - starts[seq], (starts[1:] - starts[:-1])[seq]
        there = row < starts[-1]
    else:
        seq, i = row // (n // b), row % (n // b)
        count, there = torch.full_like(row, n // b), torch.ones_like(row, dtype=torch.bool)
    return seq, i, x["lengths"].long()[seq] - count + i, there


def _turn(case, x, cos, sin):
    m = case["turned"] // 2
    turned, rest = x[..., :2 * m], x[..., 2 * m:]
    if case["layout"] == "half":
        u, w = turned[..., :m], turned[..., m:]
        return torch.cat((u * cos - w * sin, u * sin + w * cos, rest), -1)
    u, w = turned[..., 0::2], turned[..., 1::2]
    return torch.cat((torch.stack((u * cos - w * sin, u * sin + w * cos), -1).flatten(-2), rest), -1)


def _append_plain(case, x):
    seq, _, pos, there = _rows(case, x)
    t, page = x["q"].dtype, case["page"]
    # angles of far positions: in 64 bits
    angle = pos.double()[:, None, None] * torch.tensor(_frequencies(case), dtype=torch.float64, device="cuda")
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
    q = torch.where(there[:, None, None], _turn(case, x["q"].float(), cos, sin).to(t), x["q_out"])
    new = {"k": _turn(case, x["k"].float(), cos, sin), "v": x["v"].float()}
    # rows of no sequence go to slot 0 of page 0, which nobody has, and find there what they bring
    at = torch.where(there, x["pages"].long()[seq, (pos // page).clamp(0, _max_pages(case) - 1)], 0)
    slot = torch.where(there, pos % page, 0)
    out = {"q_out": q, "k_cache": x["k_cache"], "v_cache": x["v_cache"]}
    if not case["bits8"]:
        for g in "kv":
            x[g + "_cache"][at, :, slot] = torch.where(there[:, None, None], new[g].to(t), x[g + "_cache"][0, :, 0])
        return out
    # the pages that a sequence's new tokens touch, as many as the longest may
    counts = (x["starts"][1:] - x["starts"][:-1]).long() if "starts" in x else torch.full_like(x["lengths"], case["tokens"] // case["batch"]).long()
    first = x["lengths"].long() - counts
    index = first[:, None] // page + torch.arange((case["most"] + page - 2) // page + 1, device="cuda")
    touched = index * page < x["lengths"].long()[:, None]
    number = torch.where(touched, torch.gather(x["pages"].long(), 1, index.clamp(max=_max_pages(case) - 1)), 0)
    held = torch.where(touched, (first[:, None] - index * page).clamp(0, page), 0)       # tokens that a page had before
    for g in "kv":
        codes, scale = x[g + "_cache"], x[g + "_scale"]
        amax = torch.zeros_like(scale).index_reduce_(0, at, new[g].abs().amax(2) * there[:, None], "amax")
        need = _pow2(amax[number])
        before = scale[number]
        after = torch.where(touched[..., None], torch.where(held[..., None] > 0, torch.maximum(need, before), need), before)
        old = codes.view(torch.uint8)[number].view(torch.float8_e4m3fn)
        again = (old.float() * (before / after)[..., None, None]).to(torch.float8_e4m3fn)
        keep = torch.arange(page, device="cuda")[None, None, None, :, None] < held[:, :, None, None, None]
        codes.view(torch.uint8)[number] = torch.where(keep, again.view(torch.uint8), old.view(torch.uint8))
        scale[number] = after
        fresh = (new[g] / scale[at][:, :, None]).clamp(-448.0, 448.0).to(torch.float8_e4m3fn).view(torch.uint8)
        codes.view(torch.uint8)[at, :, slot] = torch.where(there[:, None, None], fresh, codes.view(torch.uint8)[0, :, 0])
        out[g + "_scale"] = scale
    return out


def _attend_plain(case, x):
    b, n, h, hk, d, page, t = case["batch"], case["tokens"], case["heads"], case["kv_heads"], case["d_head"], case["page"], x["q"].dtype
    group, most = h // hk, case["most"]
    seq, i, pos, there = _rows(case, x)
    table = x["pages"].long()
    exists = table >= 0
    number = torch.where(exists, table, 0)

    def dense(g):
        cache = x[g + "_cache"]
        if case["bits8"]:
            got = cache.view(torch.uint8)[number].view(torch.float8_e4m3fn).float() * x[g + "_scale"][number][..., None, None]
        else:
            got = cache[number].float()
        return got.transpose(1, 2).reshape(b, hk, -1, d)

    # queries side by side, [b, kv_heads, most * group, d]; rows of no sequence to a place behind the last one
    seq = torch.where(there, seq, b)
    i = torch.where(there, i, 0)
    q = torch.zeros((b + 1, most, h, d), device="cuda")
    q[seq, i] = x["q"].float()
    q = q[:b].view(b, most, hk, group, d).transpose(1, 2).reshape(b, hk, most * group, d)
    s = torch.matmul(q, dense("k").transpose(2, 3)).view(b, hk, most, group, -1) * (1.0 / math.sqrt(d))
    if case["cap"]:
        s = case["cap"] * torch.tanh(s / case["cap"])
    at = torch.full((b + 1, most), -1, device="cuda")
    at[seq, i] = pos
    at = at[:b, :, None]
    j = torch.arange(s.shape[-1], device="cuda")
    seen = (j <= at) & exists.repeat_interleave(page, 1)[:, None, :]
    if case["window"]:
        seen &= (j > at - case["window"]) | (j < case["sinks"])
    s = torch.where(seen[:, None, :, None, :], s, -math.inf)
    top = s.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    s = torch.exp(s - top)
    total = s.sum(-1, keepdim=True)
    out = torch.matmul(s.view(b, hk, most * group, -1), dense("v")).view(b, hk, most, group, d) / torch.where(total == 0.0, 1.0, total)
    lse = (top + torch.log(total))[..., 0]
    seq, there = seq.clamp(max=b - 1), there[:, None, None]
    return {"out": torch.where(there, out.transpose(1, 2).reshape(b, most, h, d)[seq, i].to(t), x["out"]),
            "lse": torch.where(there[..., 0], lse.transpose(1, 2).reshape(b, most, h)[seq, i], x["lse"])}


def _sample_plain(case, x):
    # sums and borders: in 64 bits
    logits = x["logits"].double()
    rows, vocab = logits.shape
    greedy = x["temperature"] == 0.0
    z, order = torch.sort(logits, dim=1, descending=True, stable=True)
    w = torch.exp((z - z[:, :1]) / torch.where(greedy, 1.0, x["temperature"]).double()[:, None])
    rank = torch.arange(vocab, device="cuda")
    keep = torch.ones_like(w, dtype=torch.bool)
    if "top_k" in x:
        keep &= (rank < x["top_k"][:, None]) | (x["top_k"][:, None] <= 0)
    running = torch.cumsum(w * keep, 1)
    if "top_p" in x:
        keep &= (running - w < x["top_p"].double()[:, None] * running[:, -1:]) | (rank == 0)
    if "min_p" in x:
        keep &= w >= x["min_p"].double()[:, None]
    # back to the order of the vocabulary
    w = torch.zeros_like(w).scatter_(1, order, w * keep)
    running = torch.cumsum(w, 1)
    total = running[:, -1:]
    token = (running <= x["uniform"].double()[:, None] * total).sum(1, keepdim=True)
    token = torch.where(greedy[:, None], order[:, :1], token)
    logprob = torch.where(greedy[:, None], 0.0, torch.log(w.gather(1, token.clamp(max=vocab - 1)) / total))
    return {"tokens": token[:, 0].int(), "logprob": logprob[:, 0].float()}


# ------------------------------------------------------------------ the framework's operators
_device = None


def _results(case):
    """{node: (dims, type)} of what a case computes beside the caches."""
    t = _TORCH[case["prec"]]
    if case["kind"] == "sample":
        return {"tokens": ((case["rows"],), torch.int32), "logprob": ((case["rows"],), torch.float32)}
    rows = (case["tokens"], case["heads"], case["d_head"])
    if case["kind"] == "append":
        return {"q_out": (rows, t)}
    return {"out": (rows, t), "lse": (rows[:2], torch.float32)}


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
        kinds = {torch.float32: "single", torch.float16: "half", torch.bfloat16: "bfloat16", torch.int32: "int32", torch.float8_e4m3fn: "byte"}
        nodes = [(n, tuple(v.shape), v.dtype) for n, v in x.items()] + [(n, d, t) for n, (d, t) in _results(case).items()]
        self.context = bk.Context(_device).allocate([Tnode(i + 1, n, kinds[t], d) for i, (n, d, t) in enumerate(nodes)])
        self.types = {n: t for n, _, t in nodes}
        _device.await_()
        for n, v in x.items():
            self.view(n).copy_(v)
        torch.cuda.synchronize()
        self.operator = self.link(case, self.context, x)

    def link(self, case, ctx, x):
        if case["kind"] == "sample":
            return ctx.sample("logits", "uniform", "tokens", logprob="logprob", **{n: n for n in ("temperature", "top_k", "top_p", "min_p") if n in x})
        cache = dict(pages="pages", lengths="lengths", starts="starts" if "starts" in x else None)
        if case["bits8"]:
            cache.update(k_scale="k_scale", v_scale="v_scale")
        if case["kind"] == "append":
            return ctx.cache_append("k", "v", "k_cache", "v_cache", q="q", q_out="q_out", frequencies=_frequencies(case), layout=case["layout"], **cache)
        return ctx.cache_attention("q", "k_cache", "v_cache", "out", lse="lse", window=case["window"], sinks=case["sinks"], cap=case["cap"], **cache)

    def view(self, ident):
        """A node's memory as a tensor; keeps the program that owns it."""
        pool, offset, t = self.context.arrays[ident]
        address, _ = _device.pool_address(pool)

        buffer = _Buffer()
        buffer.program = self
        buffer.__cuda_array_interface__ = {"shape": tuple(t.dims), "data": (address + offset, False), "version": 3, "strides": None,
                                           "typestr": {"single": "<f4", "half": "<f2", "bfloat16": "<i2", "int32": "<i4", "byte": "|u1"}[t.prec]}
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
        # the nodes lie in the context's pool, the operator is linked to them
        s.program = _Program(case, s.x)
        names = list(_results(case))
        if case["kind"] == "append":
            names += [n for n in ("k_cache", "v_cache", "k_scale", "v_scale") if n in s.x]
        s.outputs = {n: s.program.view(n) for n in names}
        s.x = None
    else:
        s.x.update({n: torch.zeros(d, dtype=t, device="cuda") for n, (d, t) in _results(case).items()})
    return s


def run(s):
    if own:
        s.program.operator.run()
        return s.outputs
    return {"append": _append_plain, "attend": _attend_plain, "sample": _sample_plain}[s.case["kind"]](s.case, s.x)


# ------------------------------------------------------------------ work
def work(case):
    size = 4 if case["prec"] == "single" else 2
    if case["kind"] == "sample":
        return {"bytes": case["rows"] * (case["vocab"] * size + 12), "flops": 4.0 * case["rows"] * case["vocab"]}
    rows = case["batch"] if case["most"] == 1 else min(case["tokens"], case["batch"] * case["most"] * 0.625)     # on average
    h, hk, d, of_cache = case["heads"], case["kv_heads"], case["d_head"], 1 if case["bits8"] else size
    if case["kind"] == "append":
        return {"bytes": rows * (2 * h * size + 2 * hk * (size + of_cache)) * d, "flops": 3.0 * rows * (h + hk) * case["turned"]}
    # tokens of a sequence, on average; what a row sees of them, and what all rows of a sequence do
    new = rows / case["batch"]
    length = min(case["max_len"], max(new, 0.75 * case["max_len"]))
    seen, touched = max(1.0, length - new / 2), length
    if case["window"]:
        seen, touched = min(seen, case["window"] + case["sinks"]), min(touched, case["window"] + new + case["sinks"])
    return {"bytes": 2 * rows * h * d * size + 4 * rows * h + case["batch"] * touched * 2 * hk * (d * of_cache + (4 / case["page"] if case["bits8"] else 0)),
            "flops": 4.0 * rows * h * d * seen}


# ------------------------------------------------------------------ the definitions in 64 bits
def _places(case, x):
    """(rows of the batch, position of the first, tokens) of every sequence, as numbers."""
    lengths = x["lengths"].tolist()
    starts = x["starts"].tolist() if "starts" in x else [i * (case["tokens"] // case["batch"]) for i in range(case["batch"] + 1)]
    return [(slice(starts[b], starts[b + 1]), lengths[b] - (starts[b + 1] - starts[b]), lengths[b]) for b in range(case["batch"])]


def _e4m3(v):
    """The nearest e4m3 number, ties to even: three bits behind the first, steps of 2^-9 at the least."""
    _, e = torch.frexp(v)
    step = torch.ldexp(torch.ones_like(v), (e - 4).clamp(min=-9))
    return torch.round(v / step) * step


def _exact_append(case, x):
    f = torch.tensor(_frequencies(case), dtype=torch.float64, device="cuda")
    m, page = case["turned"] // 2, case["page"]
    first, second = (slice(0, m), slice(m, 2 * m)) if case["layout"] == "half" else (slice(0, 2 * m, 2), slice(1, 2 * m, 2))
    res = {"q_out": torch.zeros(x["q"].shape, dtype=torch.float64, device="cuda")}
    for g in "kv":
        res[g + "_cache"] = x[g + "_cache"].double()
        if case["bits8"]:
            res[g + "_scale"] = x[g + "_scale"].double()
    for b, (rows, begin, end) in enumerate(_places(case, x)):
        turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), torch.outer(torch.arange(begin, end, dtype=torch.float64, device="cuda"), f))[:, None]
        new = {}
        for g in "qkv":
            y = x[g][rows].double()
            if g != "v":
                z = torch.complex(y[..., first], y[..., second]) * turn
                y[..., first], y[..., second] = z.real, z.imag
            new[g] = y
        res["q_out"][rows] = new["q"]
        for at in range(begin // page, -(-end // page)):
            number, lo, hi = int(x["pages"][b, at]), max(begin, at * page), min(end, (at + 1) * page)
            had = max(0, begin - at * page)
            for g in "kv":
                values = new[g][lo - begin:hi - begin].transpose(0, 1)
                cache = res[g + "_cache"][number]
                if case["bits8"]:
                    old = res[g + "_scale"][number]
                    bits = torch.ceil(torch.log2(values.abs().amax((1, 2)) / 448.0)).clamp(min=-40.0)
                    scale = torch.exp2(bits)
                    if had:
                        scale = torch.maximum(scale, old)
                        cache[:, :had] = _e4m3(cache[:, :had] * (old / scale)[:, None, None])
                    res[g + "_scale"][number] = scale
                    values = _e4m3(values / scale[:, None, None])
                cache[:, lo - at * page:hi - at * page] = values
    return res


def _exact_attend(case, x):
    group, page = case["heads"] // case["kv_heads"], case["page"]
    out = torch.zeros(x["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.zeros(x["q"].shape[:2], dtype=torch.float64, device="cuda")
    for b, (rows, begin, end) in enumerate(_places(case, x)):
        table = x["pages"][b, :-(-end // page)]
        pos = torch.arange(begin, end, device="cuda")[:, None]
        col = torch.arange(table.numel() * page, device="cuda")[None, :]
        hidden = (col > pos) | (table < 0).repeat_interleave(page)[None, :]
        if case["window"]:
            hidden |= (col <= pos - case["window"]) & (col >= case["sinks"])
        some = ~hidden.all(0)                       # keys that some row sees
        hidden = hidden[:, some]
        for g in range(case["kv_heads"]):
            kv = []
            for n in "kv":
                y = x[n + "_cache"].view(torch.uint8)[table.long().clamp(min=0), g].view(x[n + "_cache"].dtype).double() if case["bits8"] else \
                    x[n + "_cache"][table.long().clamp(min=0), g].double()
                if case["bits8"]:
                    y = y * x[n + "_scale"][table.long().clamp(min=0), g].double()[:, None, None]
                kv.append(y.reshape(-1, case["d_head"])[some])
            for h in range(g * group, (g + 1) * group):
                z = torch.einsum("rd,jd->rj", x["q"][rows, h].double(), kv[0]) / math.sqrt(case["d_head"])
                if case["cap"]:
                    z = case["cap"] * torch.tanh(z / case["cap"])
                z = z.masked_fill(hidden, -math.inf)
                out[rows, h] = torch.einsum("rj,jd->rd", torch.softmax(z, 1), kv[1])
                lse[rows, h] = torch.logsumexp(z, 1)
    return {"out": out, "lse": lse}


def _exact_sample(case, x):
    res = []
    for r in range(case["rows"]):
        t = float(x["temperature"][r])
        if t == 0.0:
            res.append(0.0)
            continue
        p = torch.softmax(x["logits"][r].double() / t, 0)
        # the smallest share that is kept: by number, by sum, by size
        falling, order = torch.sort(p, descending=True, stable=True)
        n = p.numel()
        if "top_k" in x and int(x["top_k"][r]) > 0:
            n = min(n, int(x["top_k"][r]))
        if "top_p" in x:
            sums = torch.cumsum(falling[:n], 0)
            n = min(n, int(torch.searchsorted(sums, float(x["top_p"][r]) * sums[-1])) + 1)
        if "min_p" in x:
            n = min(n, int((falling >= float(x["min_p"][r]) * falling[0]).sum()))
        kept = order[:n].sort()[0]
        sums = torch.cumsum(p[kept], 0)
        i = int(torch.searchsorted(sums, float(x["uniform"][r]) * sums[-1], right=True))
        res.append(float(torch.log(p[kept[min(i, n - 1)]] / sums[-1])))
    return {"tokens": None, "logprob": torch.tensor(res, dtype=torch.float64)}


def exact(case, seed):
    x = _inputs(case, seed)
    return {"append": _exact_append, "attend": _exact_attend, "sample": _exact_sample}[case["kind"]](case, x)
