"""The operators of the 4-bit K/V cache as cases that can be timed and compared.

`op` says which one a case runs:

  step     one new token of every sequence: its key and value join the cache, its query attends to all rows
  prompt   prompts of different lengths, packed one behind the other: appended and attended in one pass
  evict    the rows with the least accumulated attention weight leave, the others move together into a smaller cache

A cache row of `dim` values is held in blocks of 32: a bf16 scale, the largest magnitude times fp32(1/7), within 2^-17 … 2^13, and the codes
round(value / scale) of -7 … 7.  Rotation and quantization are fp32 operations, each rounded; they belong to the definition.
`ratio` query heads share a key/value head; `groups` counts the key/value heads.
"""
from __future__ import annotations

import math
import random

import torch

own = False

BLOCK = 32
SCALE_MIN, SCALE_MAX = 2.0 ** -17, 2.0 ** 13
MOST_STEP = 4 * 8 * 32700 * 128                 # cached values of the largest step
MOST_PROMPT = 32 * 128 * 6000 * 3000            # head values × (token, key) pairs of the largest prompt
MOST_EVICT = 16 * 32 * 4096 * 128               # cached values of the largest eviction
_next_id = [1 << 26]


# ───────────── cases ─────────────

def _step(batch, groups, ratio, dim, context, tracked, ragged, **more):
    return dict(op="step", batch=batch, groups=groups, ratio=ratio, dim=dim, context=context, tracked=tracked, ragged=ragged, **more)


def _prompt(batch, groups, ratio, dim, tokens, prefix, window, ragged, **more):
    return dict(op="prompt", batch=batch, groups=groups, ratio=ratio, dim=dim, tokens=tokens, prefix=prefix, window=window, ragged=ragged, **more)


def _evict(batch, groups, dim, context, budget, recent, ragged, **more):
    return dict(op="evict", batch=batch, groups=groups, dim=dim, context=context, budget=budget, recent=recent, ragged=ragged, **more)


def listed():
    return [
        # one conversation with a model of 16 heads × 128, early in it: latency is everything
        _step(1, 16, 1, 128, 300, False, False, name="step 1 of 16x128 at 300"),
        # the 7B-shaped model, one sequence, at the length its benchmark quotes
        _step(1, 32, 1, 128, 2048, False, False, name="step 1 of 32x128 at 2048"),
        # a server's batch of it: 16 sequences of different lengths, weights kept for eviction
        _step(16, 32, 1, 128, 2048, True, True, name="step 16 of 32x128 tracked"),
        # many short chats of a small model
        _step(64, 12, 1, 64, 200, False, True, name="step 64 of 12x64 at 200"),
        # long documents, four query heads to a key/value head
        _step(4, 8, 4, 128, 32700, True, True, name="step 4 of 32/8x128 at 32700"),
        # a few short prompts of a small model that arrived together
        _prompt(3, 25, 1, 64, 77, 0, 0, True, name="prompt 3 of 25x64 short"),
        # one prompt of the 7B-shaped model
        _prompt(1, 32, 1, 128, 2048, 0, 0, False, name="prompt 2048 of 32x128"),
        # a server's batch of prompts, grouped heads, weights kept for eviction
        _prompt(8, 8, 4, 128, 1500, 0, 32, True, name="prompt 8 of 32/8x128 packed"),
        # the next turn of a long conversation
        _prompt(1, 32, 1, 64, 300, 3001, 16, False, name="prompt 300 behind 3001"),
        # a long prompt
        _prompt(1, 8, 4, 128, 6000, 0, 0, False, name="prompt 6000 of 32/8x128"),
        # a full cache of one sequence of the 7B-shaped model is halved
        _evict(1, 32, 128, 2048, 1024, 128, False, name="evict 2048 to 1024"),
        # a batch of full caches shrinks to a quarter
        _evict(16, 32, 128, 4096, 1024, 256, True, name="evict 16 of 4096 to 1024"),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    dim = rng.choice((32, 64, 128, 128))
    groups, ratio = rng.choice((1, 2, 4, 5, 8, 12, 16, 25, 32)), rng.choice((1, 1, 1, 2, 3, 4, 7, 8))
    while groups * ratio > 64:
        ratio = max(1, ratio // 2)
    ragged = rng.random() < 0.7
    op = rng.choice(("step", "step", "prompt", "prompt", "evict"))
    batch = _log(rng, 1, 64)
    if op == "step":
        context = _log(rng, 1, 32700)
        while batch > 1 and batch * groups * context * dim > MOST_STEP:
            batch -= batch // 8 + 1
        context = min(context, MOST_STEP // (batch * groups * dim))
        return _step(batch, groups, ratio, dim, context, rng.random() < 0.5, ragged)
    if op == "prompt":
        batch = min(batch, 16)
        tokens, prefix = _log(rng, 1, 3000), rng.choice((0, 0, _log(rng, 1, 4000)))
        while batch > 1 and batch * groups * ratio * dim * tokens * (prefix + tokens) > MOST_PROMPT:
            batch -= 1
        while batch * groups * ratio * dim * tokens * (prefix + tokens) > MOST_PROMPT:
            tokens, prefix = tokens * 7 // 8 + 1, prefix * 7 // 8
        return _prompt(batch, groups, ratio, dim, tokens, prefix, rng.choice((0, 0, 1, 16, 32)), ragged)
    context = _log(rng, 2, 16000)
    while batch > 1 and batch * groups * context * dim > MOST_EVICT:
        batch -= batch // 8 + 1
    context = max(2, min(context, MOST_EVICT // (batch * groups * dim)))
    budget = max(1, int(context * rng.uniform(0.1, 0.9)))
    return _evict(batch, groups, dim, context, budget, int(budget * rng.uniform(0.0, 0.6)), ragged)


def _lengths(case):
    """Cached rows and new tokens of every sequence: they go with the case, not with the seed."""
    r = random.Random("%s %s %s" % (case["op"], case.get("context", case.get("tokens")), case["batch"]))
    n = case["batch"]
    spread = lambda most, low: [most] + [r.randint(max(low, most // 2), most) if case["ragged"] else most for _ in range(n - 1)]  # noqa: E731
    if case["op"] == "prompt":
        cached, new = spread(case["prefix"], 0), spread(case["tokens"], 1)
        if case["ragged"] and n >= 4:
            new[2] = 0                           # a sequence that has nothing to add
        return cached, new
    cached = spread(case["context"], 0)
    if case["op"] == "step" and case["ragged"] and n >= 8:
        cached[-1] = 0                           # a sequence that begins
    return cached, [1] * n


def work(case):
    cached, new = _lengths(case)
    groups, dim = case["groups"], case["dim"]
    row = 2 * (dim // 2 + dim // 16)             # bytes of a key and a value row
    if case["op"] == "evict":
        kept = sum(min(c, case["budget"]) for c in cached) * groups
        return {"bytes": 4 * groups * sum(cached) + kept * (2 * row + 4 * 2 + 8 * dim), "flops": groups * sum(cached)}
    heads = groups * case["ratio"]
    tokens = sum(new)
    rows = sum(c + t for c, t in zip(cached, new) if t > 0)
    pairs = sum(t * c + t * (t + 1) // 2 for c, t in zip(cached, new))
    byte = 4 * dim * tokens * (2 * heads + 2 * groups) + groups * (rows * row + 8 * dim * tokens)
    flops = 4 * heads * dim * pairs
    weights = case.get("tracked") or case.get("window", 0) > 0
    if weights:
        byte += 8 * groups * rows
    if case["op"] == "prompt":
        flops += 2 * heads * dim * sum(min(case["window"], t) * (c + t) for c, t in zip(cached, new))
    return {"bytes": byte, "flops": flops}


# ───────────── the cache format ─────────────

def _quantize(x):
    """Rows of values → (codes, scales), both fp32: one scale to 32 values."""
    x = torch.where(torch.isnan(x), torch.zeros_like(x), x).unflatten(-1, (-1, BLOCK))
    most = x.abs().amax(-1)
    scale = (most * torch.tensor(1.0 / 7.0, dtype=torch.float32, device=x.device)).to(torch.bfloat16).float().clamp(SCALE_MIN, SCALE_MAX)
    codes = (x / scale[..., None]).round().clamp(-7, 7)
    return codes.flatten(-2), torch.where(most > 0, scale, torch.zeros_like(scale))


def _values(codes, scales):
    return (codes.float().unflatten(-1, (-1, BLOCK)) * scales[..., None]).flatten(-2)


def _rotate(x, cos, sin):
    """Interleaved pairs (a, b) → (a·cos − b·sin, a·sin + b·cos)."""
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)


# ───────────── inputs ─────────────

def _rows(g, shape):
    """Keys or values as models make them: near normal, some channels several times the others."""
    gain = 1.0 + 3.0 * (torch.rand(shape[-1], generator=g, device="cuda") < 0.05)
    return torch.randn(shape, generator=g, device="cuda") * gain


def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(seed * 7919 + 17)
    cached, new = _lengths(case)
    batch, groups, dim = case["batch"], case["groups"], case["dim"]
    size = max(c + t for c, t in zip(cached, new))
    s = dict(case=case, size=size, len=torch.tensor(cached, dtype=torch.float32, device="cuda"), new=torch.tensor(new, device="cuda"))
    s["index"] = torch.arange(size, device="cuda")
    history = max(1, max(cached))
    k, v = _rows(g, (batch, groups, history, dim)), _rows(g, (batch, groups, history, dim))
    weights = torch.rand(batch, groups, size, generator=g, device="cuda").pow(6) * 8     # a few rows have most of the weight
    weights[torch.rand(batch, groups, size, generator=g, device="cuda") < 0.1] = 0.0     # and some were never looked at
    s["weights"] = weights
    full = lambda *n: torch.zeros(*n, device="cuda")  # noqa: E731
    if case["op"] == "evict":
        s["budget"] = case["budget"]
    else:
        ratio = case["ratio"]
        heads, tokens = groups * ratio, sum(new)
        qkv = torch.randn(tokens, (heads + 2 * groups) * dim, generator=g, device="cuda")
        qkv[:, heads * dim:] = _rows(g, (tokens, 2 * groups * dim))
        s["qkv"] = qkv
        gone = torch.randint(0, 500, (batch,), generator=g, device="cuda") if case.get("tracked") else torch.zeros(batch, device="cuda")
        s["pos"] = s["len"] + gone                                                       # rows evicted before count as positions
        top = size + 500
        angle = torch.arange(top, device="cuda", dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(dim // 2, device="cuda", dtype=torch.float64) * 2 / dim)
        s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
        starts = [0]
        for t in new:
            starts.append(starts[-1] + t)
        s["starts"] = torch.tensor(starts, dtype=torch.float32, device="cuda")
        s["seq"] = torch.repeat_interleave(torch.arange(batch, device="cuda"), s["new"])             # of every packed row: its sequence,
        s["token"] = torch.arange(tokens, device="cuda") - s["starts"].long()[s["seq"]]              # its token
        s["row"] = s["len"].long()[s["seq"]] + s["token"]                                            # and its place in the cache
    if own:
        s["handle"] = _Handle(s, k, v)
    else:
        for name, x in (("k", k), ("v", v)):
            codes, scales = _quantize(x)
            s[name] = torch.zeros(batch, groups, size, dim, dtype=torch.int8, device="cuda")
            s[name + "_scale"] = full(batch, groups, size, dim // BLOCK)
            s[name][:, :, :history], s[name + "_scale"][:, :, :history] = codes.to(torch.int8), scales
    return s


class _Owned:
    """A buffer that lives as long as somebody holds a view of it."""

    def __init__(self, rt, i):
        self.rt, self.id = rt, i

    def __del__(self):
        self.rt.release_buffers([self.id], 1)


class _Handle:
    """What a program built on the framework keeps: its device buffers, the cache object and the recorded streams."""

    def __init__(self, s, k, v):
        from deepj_b200 import _lib
        from deepj_b200 import compute_graph as cg
        self.rt = cg.CudaGpuRuntime()
        self.lib, self.ids, self.views = self.rt.lib, [], []
        case = s["case"]
        batch, groups, dim, size, history = case["batch"], case["groups"], case["dim"], s["size"], k.shape[2]
        kv = self._object()
        _lib.check(self.lib.deepj_cuda_kv_alloc_q4(kv, 1, batch, groups, size, dim))
        rows, view = self._buffer(batch * history, 2 * groups * dim)
        at, _ = self._buffer(batch)
        view.view(batch, history, 2, groups, dim).copy_(torch.stack((k, v), 2).permute(0, 3, 2, 1, 4))
        torch.cuda.synchronize()
        self._flush([cg.OP_KV_STORE_Q4, rows, 0, groups * dim, 2 * groups * dim, kv, 0, at, batch, history])
        self.views.pop(0)                        # the rows are in the cache: their buffer goes
        del view
        length, acc = self._given(s["len"]), self._given(s["weights"])
        if case["op"] == "evict":
            keep = case["budget"]
            small = self._object()
            _lib.check(self.lib.deepj_cuda_kv_alloc_q4(small, 1, batch, groups, keep, dim))
            acc_out, acc_view = self._buffer(batch, groups, keep)
            len_out, len_view = self._buffer(batch)
            kept, kept_view = self._buffer(batch, groups, keep)
            k_out, k_view = self._buffer(batch, groups, keep, dim)
            v_out, v_view = self._buffer(batch, groups, keep, dim)
            stream = [cg.OP_KV_EVICT_Q4, kv, small, 0, length, acc, case["budget"], case["recent"], batch, acc_out, len_out, kept,
                      cg.OP_KV_LOAD_Q4, small, 0, at, len_out, keep, k_out, v_out, batch]
            self.out = dict(k=k_view, v=v_view, weights=acc_view, len=len_view, kept=kept_view)
        else:
            heads, tokens, width = groups * case["ratio"], s["qkv"].shape[0], s["qkv"].shape[1]
            qkv, pos, cos, sin = self._given(s["qkv"]), self._given(s["pos"]), self._given(s["cos"]), self._given(s["sin"])
            out, out_view = self._buffer(tokens, heads * dim)
            tracked = case.get("tracked") or case.get("window", 0) > 0
            acc_out, acc_view = self._buffer(batch, groups, size) if tracked else (-1, None)
            most = int(s["new"].max())
            k_out, k_view = self._buffer(batch, groups, most, dim)
            v_out, v_view = self._buffer(batch, groups, most, dim)
            end = self._given(s["len"] + s["new"])
            place = [qkv, 0, heads * dim, (heads + groups) * dim, width, kv, 0]
            where = [length, pos, cos, sin, s["cos"].shape[0], out, 0, heads * dim, batch, heads]
            if case["op"] == "step":
                stream = [cg.OP_ATTN_DECODE_Q4] + place + where + [acc if tracked else -1, acc_out]
            else:
                starts = self._given(s["starts"])
                stream = [cg.OP_ATTN_PACKED_Q4] + place + [starts] + where + [tokens, acc if tracked else -1, acc_out, case["window"]]
            stream += [cg.OP_KV_LOAD_Q4, kv, 0, length, end, most, k_out, v_out, batch]
            self.out = dict(out=out_view, k=k_view, v=v_view)
            if tracked:
                self.out["weights"] = acc_view
        self.stream = cg.stream(stream)
        torch.cuda.synchronize()

    def _object(self):
        _next_id[0] += 1
        self.ids.append(_next_id[0])
        return _next_id[0]

    def _buffer(self, *shape):
        _next_id[0] += 1
        i = _next_id[0]
        self.rt.alloc_buffers([i], [math.prod(shape)], 1)
        self.rt.synchronize()                    # its zeros are written before torch's stream writes into it
        seen = self.rt.device_view(i, shape)
        seen.owner = _Owned(self.rt, i)          # the tensor keeps what it was made from, and that keeps the buffer
        self.views.append(torch.as_tensor(seen, device="cuda"))
        return i, self.views[-1]

    def _given(self, x):
        i, view = self._buffer(*x.shape)
        view.copy_(x)
        return i

    def _flush(self, words):
        from deepj_b200.compute_graph import stream
        words = stream(words)
        self.rt.flush_ops(words, words.size)

    def __del__(self):
        if self.ids:
            self.rt.release_buffers(self.ids, len(self.ids))


# ───────────── the operators ─────────────

def run(s):
    if own:
        h = s["handle"]
        h.rt.flush_ops_async(h.stream, h.stream.size)
        return h.out
    if s["case"]["op"] == "step":
        return _plain_step(s)
    return _plain_prompt(s) if s["case"]["op"] == "prompt" else _plain_evict(s)


def _append(s):
    """New rows into the cache → queries of the packed rows, the new rows' values."""
    case = s["case"]
    groups, dim = case["groups"], case["dim"]
    heads = groups * case["ratio"]
    where = s["pos"].long()[s["seq"]] + s["token"]
    cos, sin = s["cos"][where][:, None], s["sin"][where][:, None]
    q, k, v = s["qkv"].unflatten(1, (-1, dim)).split((heads, groups, groups), 1)
    kc, ks = _quantize(_rotate(k, cos, sin))
    vc, vs = _quantize(v)
    s["k"][s["seq"], :, s["row"]], s["k_scale"][s["seq"], :, s["row"]] = kc.to(torch.int8), ks
    s["v"][s["seq"], :, s["row"]], s["v_scale"][s["seq"], :, s["row"]] = vc.to(torch.int8), vs
    fresh = []
    for x in (_values(kc, ks), _values(vc, vs)):
        rows = torch.zeros(case["batch"], groups, case.get("tokens", 1), dim, device="cuda")
        rows[s["seq"], :, s["token"]] = x
        fresh.append(rows)
    return _rotate(q, cos, sin), fresh


def _weights_out(s, weights, rows):
    """Old weights of the rows that were there, plus the new ones; rows behind the last stay zero."""
    old = torch.where(s["index"] < s["len"][:, None, None], s["weights"], torch.zeros_like(s["weights"]))
    return torch.where(s["index"] < rows[:, None, None], old + weights, torch.zeros_like(old))


def _plain_step(s):
    case = s["case"]
    q, (k_new, v_new) = _append(s)
    q = q.unflatten(1, (case["groups"], case["ratio"]))
    k, v = _values(s["k"], s["k_scale"]), _values(s["v"], s["v_scale"])
    score = torch.matmul(q, k.transpose(-1, -2)) * (1.0 / math.sqrt(case["dim"]))
    score = score.masked_fill(s["index"] > s["len"][:, None, None, None], -math.inf)
    e = torch.exp(score - score.amax(-1, keepdim=True))
    p = e / e.sum(-1, keepdim=True)
    r = dict(out=torch.matmul(p, v).flatten(1), k=k_new, v=v_new)
    if case["tracked"]:
        r["weights"] = _weights_out(s, p.sum(2), s["len"] + 1)
    return r


def _plain_prompt(s):
    case = s["case"]
    batch, most = case["batch"], case["tokens"]
    q, (k_new, v_new) = _append(s)
    q = q.unflatten(1, (case["groups"], case["ratio"]))
    padded = torch.zeros(batch, most, *q.shape[1:], device="cuda")
    padded[s["seq"], s["token"]] = q
    k, v = _values(s["k"], s["k_scale"]), _values(s["v"], s["v_scale"])
    score = torch.matmul(padded.permute(0, 2, 3, 1, 4), k.transpose(-1, -2)[:, :, None])                   # [batch, groups, ratio, tokens, keys]
    score *= 1.0 / math.sqrt(case["dim"])
    last = s["len"][:, None] + torch.arange(most, device="cuda")
    score.masked_fill_((s["index"] > last[..., None])[:, None, None], -math.inf)
    score -= score.amax(-1, keepdim=True)
    p = score.exp_()
    p /= p.sum(-1, keepdim=True)
    o = torch.matmul(p, v[:, :, None]).permute(0, 3, 1, 2, 4)[s["seq"], s["token"]]
    r = dict(out=o.flatten(1), k=k_new, v=v_new)
    if case["window"]:
        place = s["new"][:, None] - 1 - torch.arange(min(case["window"], most), device="cuda")
        there = (place >= 0).float()
        seen = p.permute(0, 3, 1, 2, 4)[torch.arange(batch, device="cuda")[:, None], place.clamp(min=0)]     # [batch, window, groups, ratio, keys]
        r["weights"] = _weights_out(s, (seen * there[:, :, None, None, None]).sum((1, 3)), s["len"] + s["new"])
    return r


def _plain_evict(s):
    case = s["case"]
    budget, n = case["budget"], s["len"][:, None, None]
    rank = s["weights"].masked_fill(s["index"] >= n - case["recent"], math.inf).masked_fill(s["index"] >= n, -1.0)
    order = torch.sort(rank, dim=-1, descending=True, stable=True).indices[..., :budget]
    count = n.clamp(max=budget)
    there = torch.arange(budget, device="cuda") < count
    order = order.masked_fill(~there, s["size"]).sort(-1).values.clamp(max=s["size"] - 1)
    none = lambda x: torch.where(there[..., None] if x.dim() == 4 else there, x, torch.zeros_like(x))  # noqa: E731
    take = lambda x: x.gather(2, order[..., None].expand(-1, -1, -1, x.shape[-1]))  # noqa: E731
    moved = [take(s[name]) for name in ("k", "k_scale", "v", "v_scale")]
    return dict(k=none(_values(moved[0], moved[1])), v=none(_values(moved[2], moved[3])), weights=none(s["weights"].gather(2, order)),
                len=count[:, 0, 0], kept=none(order.float()))


# ───────────── the same from the definitions, in 64 bits ─────────────

def _stored(x):
    """What the cache gives back for fp32 rows x: the nearest of fifteen multiples of each block's scale."""
    out = torch.empty(x.shape, dtype=torch.float64, device=x.device)
    seventh = float(torch.tensor(1.0 / 7.0, dtype=torch.float32))
    for c in range(0, x.shape[-1], BLOCK):
        b = x[..., c:c + BLOCK].double()
        most = b.abs().max(-1, keepdim=True).values
        scale = (most * seventh).float().bfloat16().double()             # the product of two fp32 numbers is exact in 64 bits: one rounding to each
        scale = scale.clamp(SCALE_MIN, SCALE_MAX)
        code = (b / scale).float().round().clamp(-7, 7).double()
        out[..., c:c + BLOCK] = code * scale
    return out


def _turned(x, cos, sin):
    """Rotation in 64 bits of a pair by the tables' values."""
    y = torch.empty(x.shape, dtype=torch.float64, device=x.device)
    c, n = cos.double(), sin.double()
    y[..., ::2] = x[..., ::2].double() * c - x[..., 1::2].double() * n
    y[..., 1::2] = x[..., ::2].double() * n + x[..., 1::2].double() * c
    return y


def _turned32(x, cos, sin):
    """The keys' rotation as the cache's definition has it: products and sums rounded to fp32 one by one."""
    y = torch.empty_like(x)
    mul = lambda a, b: (a.double() * b.double()).float()  # noqa: E731
    y[..., ::2] = (mul(x[..., ::2], cos).double() - mul(x[..., 1::2], sin).double()).float()
    y[..., 1::2] = (mul(x[..., ::2], sin).double() + mul(x[..., 1::2], cos).double()).float()
    return y


def exact(case, seed):
    global own
    before, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = before
    cached, new = _lengths(case)
    batch, groups, dim = case["batch"], case["groups"], case["dim"]
    old = {n: (s[n].double().unflatten(-1, (-1, BLOCK)) * s[n + "_scale"].double()[..., None]).flatten(-2) for n in ("k", "v")}
    zeros = lambda *n: torch.zeros(*n, dtype=torch.float64, device="cuda")  # noqa: E731
    if case["op"] == "evict":
        keep = case["budget"]
        r = dict(k=zeros(batch, groups, keep, dim), v=zeros(batch, groups, keep, dim), weights=zeros(batch, groups, keep), len=zeros(batch), kept=zeros(batch, groups, keep))
        for b, n in enumerate(cached):
            m = min(n, keep)
            r["len"][b] = m
            recent = min(case["recent"], m)
            w = s["weights"][b, :, :n].double()
            place = torch.arange(n, device="cuda").expand(groups, n)
            # heavier first, then the lower index: a weight's rank among the rows that are not recent
            head = torch.argsort(w[:, :n - recent], dim=1, descending=True, stable=True)[:, :m - recent]
            chosen = torch.cat((head, place[:, n - recent:]), 1).sort(1).values
            for name in ("k", "v"):
                r[name][b, :, :m] = torch.take_along_dim(old[name][b], chosen[..., None], 1)
            r["weights"][b, :, :m], r["kept"][b, :, :m] = torch.take_along_dim(w, chosen, 1), chosen.double()
        return r
    heads = groups * case["ratio"]
    tracked = case.get("tracked") or case.get("window", 0) > 0
    most = max(new)
    r = dict(out=zeros(sum(new), heads * dim), k=zeros(batch, groups, most, dim), v=zeros(batch, groups, most, dim))
    if tracked:
        r["weights"] = zeros(batch, groups, s["size"])
    at = 0
    for b, (n, t) in enumerate(zip(cached, new)):
        p0 = int(s["pos"][b])
        cos, sin = s["cos"][p0:p0 + t, None], s["sin"][p0:p0 + t, None]
        x = s["qkv"][at:at + t].reshape(t, heads + 2 * groups, dim)
        q = _turned(x[:, :heads], cos, sin)
        r["k"][b, :, :t] = _stored(_turned32(x[:, heads:heads + groups], cos, sin)).transpose(0, 1)
        r["v"][b, :, :t] = _stored(x[:, heads + groups:]).transpose(0, 1)
        seen = torch.arange(n + t, device="cuda")[None] <= n + torch.arange(t, device="cuda")[:, None]
        total = zeros(groups, n + t)
        window = t if case["op"] == "step" else min(case["window"], t)
        for h in range(heads if t else 0):
            g = h // case["ratio"]
            k = torch.cat((old["k"][b, g, :n], r["k"][b, g, :t]))
            v = torch.cat((old["v"][b, g, :n], r["v"][b, g, :t]))
            p = torch.softmax((q[:, h] @ k.T / math.sqrt(dim)).masked_fill(~seen, -math.inf), 1)
            r["out"][at:at + t, h * dim:(h + 1) * dim] = p @ v
            total[g] += p[t - window:].sum(0)
        if tracked:
            r["weights"][b, :, :n] = s["weights"][b, :, :n].double()
            r["weights"][b, :, :n + t] += total
        at += t
    return r
