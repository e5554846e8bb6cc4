"""Workloads of the paged key/value history operators.

Three operators that serve transformer streams whose keys and values live in
pages of a shared pool:

  qk_norm   per-head RMS norm of queries and keys with the rotary embedding
            in the same pass (`fast_moss_b200.qk_norm_rope`)
  append    rotary embedding (optionally with those norms) of a ragged batch
            of new tokens, the rotated keys and the values written into their
            pages (`fast_moss_b200.rope_paged_kv`)
  attend    attention of a ragged batch of new tokens over their paged
            history, causal, optionally within a window of `context`
            positions (`fast_moss_b200.paged_attention`)

Layout: new tokens are packed [tokens, heads, head_dim], sequence s owning
rows q_start[s] .. q_start[s + 1] - 1; pages are [pages, kv_heads, page_size,
head_dim]; position p of sequence s lies in page page_table[s, p //
page_size], row p % page_size; kv_len[s] counts the positions that exist once
the new tokens are in, so the new tokens are the last ones.
"""

import math
import os
import random
import sys

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
_PERIOD = 10000.0
_EPS = 1e-6


# --------------------------------------------------------------------- cases
def listed():
    return [
        # -- qk_norm
        # one 80 ms chunk (4 tokens) of 64 audio streams in the codec's stack of 20 heads of 64
        dict(name="qk_norm 64 streams x 4", op="qk_norm", batch=64, tokens=4, heads=20, kv_heads=20, dim=64,
             type="bf16", interleaved=True, offset=3000000),
        # a full-precision pass over four sequences, 16 heads of 64
        dict(name="qk_norm 4 x 2048 f32", op="qk_norm", batch=4, tokens=2048, heads=16, kv_heads=16, dim=64,
             type="f32", interleaved=True, offset=100),
        # one long odd-sized prompt of a model with shared key heads, pairs half a head apart
        dict(name="qk_norm 1 x 16381 grouped", op="qk_norm", batch=1, tokens=16381, heads=32, kv_heads=8, dim=128,
             type="bf16", interleaved=False, offset=1000),
        # -- append
        # one token of one stream: the smallest call there is
        dict(name="append 1 x 1", op="append", sequences=1, singles=1, tokens_min=1, tokens_max=1, past_min=700,
             past_max=700, lengths=1, heads=20, kv_heads=20, dim=64, page=16, type="bf16", interleaved=True,
             norms=False),
        # one chunk of 64 audio streams that have run for up to a minute
        dict(name="append 64 streams x 4", op="append", sequences=64, singles=0, tokens_min=4, tokens_max=4,
             past_min=10, past_max=2990, lengths=2, heads=20, kv_heads=20, dim=64, page=16, type="bf16",
             interleaved=True, norms=False),
        # ragged prompts with normed queries and keys, shared key heads
        dict(name="append prompts normed", op="append", sequences=11, singles=3, tokens_min=300, tokens_max=4000,
             past_min=1, past_max=9000, lengths=3, heads=32, kv_heads=8, dim=128, page=64, type="bf16",
             interleaved=False, norms=True),
        # -- attend
        # one chunk of one audio stream after 40 s: latency counts
        dict(name="attend 1 stream x 4", op="attend", sequences=1, singles=0, tokens_min=4, tokens_max=4,
             past_min=2000, past_max=2000, lengths=4, heads=20, kv_heads=20, dim=64, page=16, context=0),
        # one chunk of 64 audio streams within the codec's window of 250 tokens
        dict(name="attend 64 streams window 250", op="attend", sequences=64, singles=0, tokens_min=4, tokens_max=4,
             past_min=10, past_max=2990, lengths=5, heads=20, kv_heads=20, dim=64, page=16, context=250),
        # single tokens of many sequences of very different lengths, shared key heads
        dict(name="attend 61 single tokens", op="attend", sequences=61, singles=61, tokens_min=1, tokens_max=1,
             past_min=20, past_max=8000, lengths=6, heads=32, kv_heads=8, dim=128, page=64, context=0),
        # a single token over one very long history: all the work is along the keys
        dict(name="attend 1 token over 131k", op="attend", sequences=1, singles=1, tokens_min=1, tokens_max=1,
             past_min=131000, past_max=131000, lengths=7, heads=32, kv_heads=8, dim=128, page=128, context=0),
        # prompts and single tokens in one batch
        dict(name="attend prompts and singles", op="attend", sequences=21, singles=16, tokens_min=400,
             tokens_max=1300, past_min=5, past_max=3000, lengths=8, heads=16, kv_heads=4, dim=128, page=32,
             context=0),
        # a chunk of a long recording over what came before: matrix work
        dict(name="attend 2048 over 14k", op="attend", sequences=1, singles=0, tokens_min=2048, tokens_max=2048,
             past_min=14300, past_max=14300, lengths=9, heads=20, kv_heads=20, dim=64, page=16, context=0),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    case = _draw(rng)
    # no dearer than the dearest listed case of its operator
    most = [work(c) for c in listed() if c["op"] == case["op"]]
    while any(work(case)[w] > max(m[w] for m in most) for w in ("bytes", "flops")):
        for size in ("tokens", "tokens_min", "tokens_max", "past_min", "past_max"):
            if size in case:
                case[size] = max(1, case[size] * 2 // 3)
    return case


def _draw(rng):
    op = rng.choice(["qk_norm", "append", "attend", "attend"])
    dim = rng.choice([64, 128])
    kv = rng.choice([1, 2, 4, 8, 10, 16, 20]) if dim == 64 else rng.choice([1, 2, 4, 8])
    group = min(rng.choice([1, 1, 2, 3, 4, 5, 8]), 40 // kv)
    heads = dict(heads=kv * group, kv_heads=kv, dim=dim)
    pairs = rng.random() < 0.5
    kind = rng.choice(["bf16", "bf16", "f32"])
    if op == "qk_norm":
        rows = _log(rng, 1, 16381)
        batch = min(rows, _log(rng, 1, 64))
        return dict(op=op, batch=batch, tokens=rows // batch, **heads, type=kind, interleaved=pairs,
                    offset=_log(rng, 1, 4000000))
    page = rng.choice([16, 32, 64, 128, 256])
    low = _log(rng, 1, 300)
    if op == "append":
        sequences = _log(rng, 1, 100)
        high = max(low, _log(rng, 1, max(2, 12000 // sequences)))
        return dict(op=op, sequences=sequences, singles=rng.randint(0, sequences) // 2, tokens_min=low,
                    tokens_max=high, past_min=1, past_max=_log(rng, 1, max(2, 60000 // sequences)),
                    lengths=rng.randint(1, 10 ** 6), **heads, page=page, type=kind, interleaved=pairs,
                    norms=rng.random() < 0.5)
    form = rng.choice(["single", "few", "chunk"])
    if form == "single":
        sequences = _log(rng, 1, 200)
        low = high = 1
        past = _log(rng, 200, 800000 // (sequences + 2))
    elif form == "few":
        sequences = _log(rng, 1, 64)
        low, high = 1, rng.randint(2, 33)
        past = _log(rng, 20, 200000 // (sequences + 2))
    else:
        sequences = rng.randint(1, 6)
        high = _log(rng, 40, 3000 // sequences)
        low = min(low, high)
        past = _log(rng, 20, 16000 // sequences)
    return dict(op=op, sequences=sequences, singles=0 if form != "chunk" else rng.randint(0, sequences - 1),
                tokens_min=low, tokens_max=high, past_min=1 + past // rng.choice([1, 3, 50]), past_max=1 + past,
                lengths=rng.randint(1, 10 ** 6), **heads, page=page,
                context=0 if rng.random() < 0.6 else _log(rng, 1, 4000))


def _lengths(case):
    """New tokens and earlier positions of every sequence, from the case alone."""
    rng = random.Random(case["lengths"])
    new, past = [], []
    for s in range(case["sequences"]):
        single = s < case["singles"]
        new.append(1 if single else _log(rng, case["tokens_min"], case["tokens_max"]))
        past.append(_log(rng, case["past_min"], case["past_max"]))
    order = list(range(case["sequences"]))
    rng.shuffle(order)
    return [new[i] for i in order], [past[i] for i in order]


# -------------------------------------------------------------------- inputs
def _heads(g, shape, kind):
    """Activations of a projection: channels of their own mean and spread."""
    d = shape[-1]
    spread = 0.5 + torch.rand(d, generator=g, device="cuda")
    mean = 0.4 * torch.randn(d, generator=g, device="cuda")
    x = torch.randn(shape, generator=g, device="cuda")
    return (x * spread + mean).to(kind)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    hq, hk, d = case["heads"], case["kv_heads"], case["dim"]
    state = dict(case)
    if case["op"] == "qk_norm":
        b, t = case["batch"], case["tokens"]
        # the projection's output [batch, tokens, all heads, dim]; q and k are views of it
        qkv = _heads(g, (b, t, hq + 2 * hk, d), _TYPES[case["type"]])
        state.update(q=qkv[:, :, :hq].transpose(1, 2), k=qkv[:, :, hq:hq + hk].transpose(1, 2),
                     offset=torch.randint(0, case["offset"] + 1, (b,), generator=g, device="cuda"))
    else:
        new, past = _lengths(case)
        page = case["page"]
        n = sum(new)
        length = [a + b for a, b in zip(new, past)]
        per = [-(-x // page) for x in length]
        width = max(per)
        pages = sum(per) + 3
        perm = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
        table = torch.full((len(new), width), -1, dtype=torch.int32)
        at = 0
        take = torch.arange(pages, dtype=torch.int32)
        for s, count in enumerate(per):
            table[s, :count] = take[at:at + count]
            at += count
        table = table.cuda()
        table = torch.where(table >= 0, perm[table.clamp(min=0).long()], table)
        start = torch.zeros(len(new) + 1, dtype=torch.int64)
        start[1:] = torch.tensor(new).cumsum(0)
        state.update(
            q_start=start.cuda(), kv_len=torch.tensor(length).cuda(), page_table=table, max_tokens=max(new),
            k_pages=_heads(g, (pages, hk, page, d), torch.bfloat16),
            v_pages=_heads(g, (pages, hk, page, d), torch.bfloat16))
        if case["op"] == "append":
            qkv = _heads(g, (n, hq + 2 * hk, d), _TYPES[case["type"]])
            state.update(q=qkv[:, :hq], k=qkv[:, hq:hq + hk], v=qkv[:, hq + hk:])
        else:
            state["q"] = torch.randn(n, hq, d, generator=g, device="cuda").to(torch.bfloat16)
    if case["op"] == "qk_norm" or case.get("norms"):
        state.update(q_weight=1 + 0.2 * torch.randn(d, generator=g, device="cuda"),
                     k_weight=1 + 0.2 * torch.randn(d, generator=g, device="cuda"))
    else:
        state.update(q_weight=None, k_weight=None)
    return state


# ---------------------------------------------------------------- plain form
def _tables(position, d):
    """cos, sin [..., d / 2] in 32 bits of angles formed in 64."""
    pair = torch.arange(d // 2, device=position.device, dtype=torch.float64)
    angle = position.double()[..., None] * torch.exp(pair * (-2 * math.log(_PERIOD) / d))
    return torch.cos(angle).float(), torch.sin(angle).float()


def _norm_rotate(x, weight, cos, sin, interleaved):
    """x [..., d] normed (where there is a weight) and rotated, in 32 bits."""
    x = x.float()
    d = x.shape[-1]
    if weight is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + _EPS) * weight
    if interleaved:
        a, b = x[..., 0::2], x[..., 1::2]
        return torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    a, b = x[..., :d // 2], x[..., d // 2:]
    return torch.cat([a * cos - b * sin, a * sin + b * cos], -1)


def _plain_qk_norm(s):
    position = s["offset"][:, None] + torch.arange(s["tokens"], device="cuda")
    cos, sin = _tables(position[:, None], s["dim"])
    out = s["q"].dtype
    return (_norm_rotate(s["q"], s["q_weight"], cos, sin, s["interleaved"]).to(out),
            _norm_rotate(s["k"], s["k_weight"], cos, sin, s["interleaved"]).to(out))


def _plain_append(s):
    row = torch.arange(s["q"].shape[0], device="cuda")
    seq = torch.searchsorted(s["q_start"], row, right=True) - 1
    position = s["kv_len"][seq] - (s["q_start"][seq + 1] - row)
    cos, sin = _tables(position[:, None], s["dim"])
    page = s["page_table"][seq, position // s["page"]].long()
    slot = position % s["page"]
    k = _norm_rotate(s["k"], s["k_weight"], cos, sin, s["interleaved"])
    s["k_pages"][page, :, slot] = k.to(torch.bfloat16)
    s["v_pages"][page, :, slot] = s["v"].to(torch.bfloat16)
    q = _norm_rotate(s["q"], s["q_weight"], cos, sin, s["interleaved"])
    return q.to(torch.bfloat16), s["k_pages"], s["v_pages"]


def _plain_attend(s):
    n, hq, d = s["q"].shape
    hk, t = s["kv_heads"], s["max_tokens"]
    count = s["q_start"].shape[0] - 1
    table = s["page_table"].clamp(min=0).long()
    k = s["k_pages"][table].permute(0, 2, 1, 3, 4).reshape(count, hk, -1, d).float()
    v = s["v_pages"][table].permute(0, 2, 1, 3, 4).reshape(count, hk, -1, d).float()
    new = s["q_start"][1:] - s["q_start"][:-1]
    step = torch.arange(t, device="cuda")
    there = step < new[:, None]
    row = torch.where(there, s["q_start"][:-1, None] + step, n)
    q = s["q"][row.clamp(max=n - 1)].float().view(count, t, hk, hq // hk, d)
    q = q.permute(0, 2, 3, 1, 4).reshape(count, hk, -1, d) / math.sqrt(d)
    position = (s["kv_len"] - new)[:, None] + step
    key = torch.arange(k.shape[2], device="cuda")
    seen = key <= position[..., None]
    if s["context"]:
        seen &= key > position[..., None] - s["context"]
    seen &= key < s["kv_len"][:, None, None]
    score = torch.matmul(q, k.transpose(2, 3)).view(count, hk, hq // hk, t, -1)
    score = score.masked_fill_(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True).clamp(min=-1e30)
    score = score.sub_(top).exp_()
    total = score.sum(-1, keepdim=True)
    out = torch.matmul(score.view(count, hk, -1, k.shape[2]), v).view(count, hk, hq // hk, t, d) / total
    out = out.permute(0, 3, 1, 2, 4).reshape(count, t, hq, d).to(torch.bfloat16)
    full = torch.empty(n + 1, hq, d, device="cuda", dtype=torch.bfloat16)
    full[row] = out
    return full[:n]


_PLAIN = {"qk_norm": _plain_qk_norm, "append": _plain_append, "attend": _plain_attend}


def _package():
    here = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "fast-moss-tokenizer_b200")
    if here not in sys.path:
        sys.path.insert(0, here)
    import fast_moss_b200

    return fast_moss_b200


def run(state):
    s = state
    if not own:
        return _PLAIN[s["op"]](s)
    fm = _package()
    if s["op"] == "qk_norm":
        return fm.qk_norm_rope(s["q"], s["k"], s["q_weight"], s["k_weight"], s["offset"], _PERIOD, eps=_EPS,
                               interleaved=s["interleaved"])
    if s["op"] == "append":
        q = fm.rope_paged_kv(s["q"], s["k"], s["v"], s["q_start"], s["kv_len"], s["page_table"], _PERIOD,
                             s["k_pages"], s["v_pages"], q_weight=s["q_weight"], k_weight=s["k_weight"], eps=_EPS,
                             interleaved=s["interleaved"])
        return q, s["k_pages"], s["v_pages"]
    return fm.paged_attention(s["q"], s["k_pages"], s["v_pages"], s["q_start"], s["kv_len"], s["page_table"],
                              context=s["context"] or None, max_tokens=s["max_tokens"])


# ---------------------------------------------------------------------- work
def work(case):
    hq, hk, d = case["heads"], case["kv_heads"], case["dim"]
    if case["op"] == "qk_norm":
        values = case["batch"] * case["tokens"] * (hq + hk) * d
        size = 2 if case["type"] == "bf16" else 4
        return {"bytes": 2 * size * values + 8 * case["batch"] + 8 * d, "flops": 7 * values}
    new, past = _lengths(case)
    n = sum(new)
    index = 16 * len(new) + 4 * sum(-(-(a + b) // case["page"]) for a, b in zip(new, past))
    if case["op"] == "append":
        size = 2 if case["type"] == "bf16" else 4
        values = n * (hq + 2 * hk) * d
        flops = n * (hq + hk) * d * (7 if case["norms"] else 3)
        return {"bytes": values * (size + 2) + 16 * len(new) + 4 * n, "flops": flops}
    keys = pairs = 0
    for a, b in zip(new, past):
        window = case["context"] or a + b
        keys += min(a + b, a + window - 1)
        # query i sees min(past + i + 1, window) positions
        full = max(0, min(a, a + b - window))
        short = a - full
        pairs += full * window + short * (b + 1) + short * (short - 1) // 2
    return {"bytes": 4 * n * hq * d + 4 * keys * hk * d + index, "flops": 4 * pairs * hq * d}


# --------------------------------------------------------------------- exact
def exact(case, seed):
    """From the definitions in 64 bits: complex rotations, one sequence and
    one key head at a time."""
    s = prepare(case, seed)
    d = s["dim"]
    rate = torch.tensor([_PERIOD ** (-2.0 * j / d) for j in range(d // 2)], dtype=torch.float64, device="cuda")

    def turned(x, weight, position):
        x = x.double()
        if weight is not None:
            x = x / torch.sqrt(x.square().sum(-1, keepdim=True) / d + _EPS) * weight.double()
        if s["interleaved"]:
            z = torch.view_as_complex(x.reshape(*x.shape[:-1], d // 2, 2).contiguous())
        else:
            z = torch.complex(x[..., :d // 2].contiguous(), x[..., d // 2:].contiguous())
        z = z * torch.polar(torch.ones_like(rate), position.double()[..., None] * rate)
        if s["interleaved"]:
            return torch.view_as_real(z).reshape(x.shape)
        return torch.cat([z.real, z.imag], -1)

    if case["op"] == "qk_norm":
        position = s["offset"].view(-1, 1, 1) + torch.arange(s["tokens"], device="cuda").view(1, 1, -1)
        return turned(s["q"], s["q_weight"], position), turned(s["k"], s["k_weight"], position)
    new, past = _lengths(case)
    start = 0
    if case["op"] == "append":
        k_pages, v_pages = s["k_pages"].double(), s["v_pages"].double()
        out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
        for i, (a, b) in enumerate(zip(new, past)):
            rows = slice(start, start + a)
            position = torch.arange(b, b + a, device="cuda")
            page, slot = s["page_table"][i].long()[position // s["page"]], position % s["page"]
            out[rows] = turned(s["q"][rows], s["q_weight"], position[:, None])
            k_pages[page, :, slot] = turned(s["k"][rows], s["k_weight"], position[:, None])
            v_pages[page, :, slot] = s["v"][rows].double()
            start += a
        return out, k_pages, v_pages
    group = s["heads"] // s["kv_heads"]
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    for i, (a, b) in enumerate(zip(new, past)):
        at = torch.arange(a + b, device="cuda")
        page, slot = s["page_table"][i].long()[at // s["page"]], at % s["page"]
        behind = torch.arange(b, b + a, device="cuda")[:, None] - at
        hidden = behind < 0
        if s["context"]:
            hidden |= behind >= s["context"]
        for h in range(s["kv_heads"]):
            k, v = s["k_pages"][page, h, slot].double(), s["v_pages"][page, h, slot].double()
            for j in range(h * group, (h + 1) * group):
                score = s["q"][start:start + a, j].double() @ k.T * d ** -0.5
                weight = torch.softmax(score.masked_fill(hidden, -math.inf), -1)
                out[start:start + a, j] = weight @ v
        start += a
    return out
