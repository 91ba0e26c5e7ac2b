"""Timed cases of the operators by which the tokens of a row see one another: rotary positions and attention.

A case is a dict; `op` names the call.  Tokens of all rows lie one after the other, as in the tokenizer's column, with int32 offsets.
`rows` rows have `tokens` tokens in all, of lengths that follow from the case: lognormal (sigma 0.6) as texts and prompts have.  A
token has `heads` heads of `width` values; keys and values have `kv_heads`, which is a divisor of that.  Queries, keys and values are
parts of one projection's result, as a model has them.

`earlier` more keys lie in front of the tokens of all rows together, in caches with room behind each row's keys (an eighth more): the next
tokens of texts that are under way, or their single next tokens where `tokens` equals `rows`.  `op` "attention" is what a model answers
with, "attention_step" what it learns with: attention and its gradient.
"""
import math

import numpy as np
import torch

own = False

DEVICE = "cuda"


def listed():
    return [
        # one token each of 32 texts under way, far in, with the frequencies of a lengthened context: query and key heads in one call
        dict(name="rotary_tokens", op="rotary", rows=32, tokens=32, start=131072, heads=40, width=128, rotated=128, layout="half", inverse=False, scaled=True, dtype="bfloat16"),
        # the query and key heads of a training batch
        dict(name="rotary_batch", op="rotary", rows=512, tokens=65536, start=0, heads=32, width=64, rotated=64, layout="half", inverse=False, scaled=False, dtype="bfloat16"),
        # the way back, with half of each head rotated in neighbouring pairs, in full precision
        dict(name="rotary_part", op="rotary", rows=77, tokens=20011, start=0, heads=24, width=80, rotated=40, layout="interleaved", inverse=True, scaled=False, dtype="float32"),
        # single next tokens of 24 texts under way
        dict(name="attend_tokens", op="attention", rows=24, tokens=24, earlier=36011, heads=32, kv_heads=8, width=128, causal=True, keep=False, dtype="bfloat16"),
        # the next token of one long text, where nothing but the cache's length is there to work on side by side
        dict(name="attend_token_far", op="attention", rows=1, tokens=1, earlier=131071, heads=32, kv_heads=8, width=128, causal=True, keep=False, dtype="bfloat16"),
        # a shard of a corpus of short texts, each token seeing all of its text
        dict(name="attend_texts", op="attention", rows=4001, tokens=512011, earlier=0, heads=16, kv_heads=16, width=64, causal=False, keep=False, dtype="float16"),
        # prompts of several thousand tokens
        dict(name="attend_prompts", op="attention", rows=6, tokens=32768, earlier=0, heads=32, kv_heads=8, width=128, causal=True, keep=False, dtype="bfloat16"),
        # further parts of prompts, with a width that no tile has and odd lengths
        dict(name="attend_chunks", op="attention", rows=5, tokens=1777, earlier=9001, heads=12, kv_heads=4, width=72, causal=True, keep=True, dtype="float16"),
        # texts in full precision
        dict(name="attend_f32", op="attention", rows=61, tokens=8191, earlier=0, heads=12, kv_heads=12, width=64, causal=False, keep=True, dtype="float32"),
        # a training step over short texts
        dict(name="step_texts", op="attention_step", rows=1024, tokens=131071, earlier=0, heads=12, kv_heads=12, width=64, causal=False, dtype="bfloat16"),
        # a training step over long ones
        dict(name="step_long", op="attention_step", rows=4, tokens=16384, earlier=0, heads=32, kv_heads=8, width=128, causal=True, dtype="bfloat16"),
        # a small batch of odd sizes
        dict(name="step_odd", op="attention_step", rows=37, tokens=5003, earlier=0, heads=10, kv_heads=2, width=80, causal=True, dtype="float16"),
    ]


def _log_between(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


_MOST_FLOPS = 1.5e12  # of a drawn case
_MOST_PAIRS = 2.0e10  # (of a query head's token and a key that it may see)


def draw(rng):
    op = rng.choice(["rotary", "attention", "attention", "attention", "attention_step", "attention_step"])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    width = rng.choice([32, 64, 64, 80, 96, 128, 128, 128, 256, 8 * rng.randint(1, 32), rng.randint(5, 256)])
    case = dict(op=op, dtype=dtype, width=width)
    if op == "rotary":
        heads = _log_between(rng, 1, 64)
        tokens = _log_between(rng, 1, max(2, 100_000_000 // (heads * width)))
        rows = max(1, tokens // _log_between(rng, 1, 2000))
        rotated = 2 * max(1, rng.choice([width, width, width // 2, rng.randint(2, width)]) // 2)
        case.update(rows=rows, tokens=tokens, start=rng.choice([0, 0, 4096, 131072]), heads=heads, rotated=rotated, layout=rng.choice(["half", "interleaved"]),
                    inverse=rng.choice([False, True]), scaled=rng.choice([False, True]))
        return case
    kv_heads = rng.choice([1, 2, 4, 8, 8, 12, 16])
    heads = kv_heads * rng.choice([1, 1, 2, 4, 5, 8] if kv_heads <= 8 else [1])
    kind = rng.choice(["texts", "prompts", "chunks", "single"]) if op == "attention" else rng.choice(["texts", "prompts"])
    case.update(heads=heads, kv_heads=kv_heads, causal=True if kind in ("chunks", "single") else rng.choice([False, True]))
    if op == "attention":
        case["keep"] = rng.choice([False, False, True])
    while True:
        rows = _log_between(rng, 1, dict(texts=4000, prompts=16, chunks=16, single=256)[kind])
        length = _log_between(rng, *dict(texts=(4, 512), prompts=(300, 16384), chunks=(2, 2048), single=(1, 1))[kind])
        earlier = rows * _log_between(rng, 1, 40_000) if kind in ("chunks", "single") else 0
        case.update(rows=rows, tokens=rows * length + (rng.randint(0, rows - 1) if kind != "single" else 0), earlier=earlier)
        pairs = heads * _pairs(case)
        bytes_of_cache = 4 * width * kv_heads * (earlier + case["tokens"])
        if pairs <= _MOST_PAIRS and work(case)["flops"] <= _MOST_FLOPS and bytes_of_cache <= 2_000_000_000 and case["tokens"] * heads * width <= 600_000_000:
            return case


# ------------------------------------------------------------------ inputs

def _split(total, rows, seed, least=0):
    """Lengths of `rows` rows, `total` in all, none below `least`."""
    weights = np.random.default_rng(seed).lognormal(0.0, 0.6, rows)
    ends = np.floor(np.cumsum(weights) * ((total - least * rows) / weights.sum()) + 1e-9)
    ends[-1] = total - least * rows
    return np.diff(np.concatenate([[0], ends])).astype(np.int64) + least


def _lengths(case):
    """(of each row its tokens, its keys): the same for every seed of a case, as its work is."""
    rows, tokens = case["rows"], case["tokens"]
    queries = _split(tokens, rows, tokens + 7 * rows, least=1 if tokens >= rows else 0)
    if not case.get("earlier"):
        return queries, queries
    return queries, queries + _split(case["earlier"], rows, case["earlier"] + 11 * rows)


def _pairs(case):
    queries, keys = (n.astype(np.float64) for n in _lengths(case))
    return float((queries * (keys - queries) + queries * (queries + 1) / 2).sum() if case["causal"] else (queries * keys).sum())


def _offsets(lengths):
    return np.concatenate([[0], np.cumsum(lengths)]).astype(np.int32)


def _on_device(a):
    return torch.from_numpy(a).to(DEVICE)


def _frequencies(case):
    """Radians a position, of each pair; scaled: a context of 8192 lengthened 32 times, frequencies that turn fewer than once in it
    divided by that, more than 4 times left as they are, in between by their turns."""
    n = case["rotated"] // 2
    f = (500000.0 if case["scaled"] else 10000.0) ** (-np.arange(n, dtype=np.float64) / n)
    if case["scaled"]:
        share = np.clip((f * 8192 / (2 * math.pi) - 1.0) / (4.0 - 1.0), 0.0, 1.0)
        f = f * share + f / 32.0 * (1.0 - share)
    return f


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(seed)
    dtype = getattr(torch, case["dtype"])
    heads, width = case["heads"], case["width"]

    def normal(*shape, scale=1.0):
        return (torch.randn(shape, generator=gen, device=DEVICE) * scale).to(dtype)

    queries, keys = _lengths(case)
    offsets = _offsets(queries)
    st = dict(case=case, offsets=_on_device(offsets))
    if case["op"] == "rotary":
        # (an eighth of the projection is not for this call: a model's values lie behind its queries and keys)
        more = max(1, heads // 8)
        st["x"] = normal(case["tokens"], heads + more, width)[:, :heads]
        st["frequencies"] = _on_device(_frequencies(case))
        st["magnitude"] = 0.1 * math.log(32.0) + 1.0 if case["scaled"] else 1.0
        starts = np.random.default_rng(seed).integers(0, case["start"] + 1, case["rows"]).astype(np.int32)
        st["starts"] = _on_device(starts) if case["start"] else None
        return st
    kv = case["kv_heads"]
    if case["earlier"]:
        room = keys + keys // 8 + 1
        key_offsets = _offsets(room)
        st["q"] = normal(case["tokens"], heads + 2 * kv, width, scale=2.0)[:, :heads]
        st["k"], st["v"] = normal(int(key_offsets[-1]), kv, width), normal(int(key_offsets[-1]), kv, width)
        st["key_offsets"], st["key_lengths"] = _on_device(key_offsets), _on_device(keys.astype(np.int32))
    else:
        key_offsets = offsets
        projection = normal(case["tokens"], heads + 2 * kv, width)
        projection[:, :heads] *= 2.0
        st["q"], st["k"], st["v"] = projection[:, :heads], projection[:, heads:heads + kv], projection[:, heads + kv:]
        st["key_offsets"] = st["key_lengths"] = None
    if case["op"] == "attention_step":
        st["grad"] = normal(case["tokens"], heads, width, scale=0.1)
    # (for the plain form: rows of like lengths go through its products together)
    st["groups"] = _groups(offsets, queries, key_offsets, keys, heads)
    return st


def _groups(offsets, queries, key_offsets, keys, heads):
    """[(tokens [rows, longest], their number in each row, keys [rows, longest], their number)], rows of a group within a quarter of
    one length, a token behind a row's last standing for one behind all."""
    order = np.argsort(-keys, kind="stable")
    order = order[queries[order] > 0]
    groups, at = [], 0
    while at < len(order):
        longest = int(keys[order[at]])
        most = max(1, 2**28 // max(1, heads * longest * int(queries[order[at:]].max())))
        end = at + 1
        while end < len(order) and end - at < most and keys[order[end]] * 5 >= longest * 4 - 40:
            end += 1
        rows = order[at:end]

        def index(first, count, behind):
            i = np.arange(max(1, int(count[rows].max())))[None, :]
            return _on_device(np.where(i < count[rows][:, None], first[rows][:, None] + i, behind).astype(np.int64))

        groups.append((index(offsets, queries, int(offsets[-1])), _on_device(queries[rows]), index(key_offsets, keys, int(key_offsets[-1])), _on_device(keys[rows])))
        at = end
    return groups


# ------------------------------------------------------------------ one pass

def run(st):
    return _call(st) if own else _PLAIN[st["case"]["op"]](st)


def _call(st):
    """The framework's operators, as a user's program calls them."""
    from cudf_amd import encoder
    case = st["case"]
    if case["op"] == "rotary":
        return encoder.rotary(st["x"], st["offsets"], st["frequencies"], st["starts"], case["layout"], case["inverse"], st["magnitude"])
    if case["op"] == "attention":
        result = encoder.attention(st["q"], st["k"], st["v"], st["offsets"], st["key_offsets"], st["key_lengths"], causal=case["causal"], keep=case["keep"])
        return (result[1].out, result[1].logsum) if case["keep"] else result
    out, saved = encoder.attention(st["q"], st["k"], st["v"], st["offsets"], causal=case["causal"], keep=True)
    return (out, saved.logsum) + encoder.attention_backward(st["grad"], st["q"], st["k"], st["v"], saved, st["offsets"], causal=case["causal"])


# ------------------------------------------------------------------ the plain forms

def _plain_rotary(st):
    case, x = st["case"], st["x"]
    tokens, n = case["tokens"], case["rotated"] // 2
    offsets = st["offsets"].long()
    t = torch.arange(tokens, device=DEVICE)
    row = torch.searchsorted(offsets, t, right=True) - 1
    at = t - offsets[row]
    if st["starts"] is not None:
        at = at + st["starts"].long()[row]
    # (angles in 64 bits: those of far positions have few bits left behind their turns)
    angle = at.double()[:, None] * st["frequencies"]
    cos, sin = (torch.cos(angle) * st["magnitude"]).float()[:, None], (torch.sin(angle) * st["magnitude"]).float()[:, None]
    if case["inverse"]:
        sin = -sin
    part = x[..., :2 * n].float()
    if case["layout"] == "half":
        a, b = part[..., :n], part[..., n:]
    else:
        a, b = part[..., 0::2], part[..., 1::2]
    first, second = a * cos - b * sin, a * sin + b * cos
    turned = torch.cat([first, second], -1) if case["layout"] == "half" else torch.stack([first, second], -1).flatten(-2)
    return torch.cat([turned.to(x.dtype), x[..., 2 * n:]], -1)


def _plain_attention(st, grad=None):
    """Group by group of rows, and of each the heads of one key head at a time where the scores of all would be large."""
    case, q, k, v = st["case"], st["q"], st["k"], st["v"]
    tokens, heads, width = q.shape
    kv = case["kv_heads"]
    each = heads // kv
    scale = width**-0.5

    def room(like, heads):  # one more token, which takes what is behind the rows
        return torch.zeros(like.shape[0] + 1, heads, width, device=DEVICE)

    out, logsum = room(q, heads), torch.full((tokens + 1, heads), -math.inf, device=DEVICE)
    if grad is not None:
        dq, dk, dv = room(q, heads), room(k, kv), room(v, kv)
    for at, count, key_at, key_count in st["groups"]:
        rows, longest, longest_keys = at.shape[0], at.shape[1], key_at.shape[1]
        i, j = torch.arange(longest, device=DEVICE)[:, None], torch.arange(longest_keys, device=DEVICE)[None, :]
        seen = (i < count[:, None, None]) & (j < key_count[:, None, None])
        if case["causal"]:
            seen = seen & (j <= i + (key_count - count)[:, None, None])
        seen = seen[:, None, None]
        safe, key_safe = at.clamp(max=tokens - 1), key_at.clamp(max=k.shape[0] - 1)
        step = kv if rows * heads * longest * longest_keys <= 2**28 else 1
        for g in range(0, kv, step):
            def of_queries(x):  # [rows, key heads, heads of each, tokens, width]
                return x[:, g * each:(g + step) * each][safe].float().view(rows, longest, step, each, -1).permute(0, 2, 3, 1, 4)

            def of_keys(x):
                return x[:, g:g + step][key_safe].float().permute(0, 2, 1, 3)[:, :, None]

            qs, ks, vs = of_queries(q), of_keys(k), of_keys(v)
            s = torch.where(seen, torch.matmul(qs, ks.transpose(-1, -2)) * scale, -math.inf)
            top = s.amax(-1, keepdim=True).clamp(min=-3e38)
            e = torch.exp(s - top)
            total = e.sum(-1, keepdim=True)
            p = e / total.clamp(min=1e-38)
            o = torch.matmul(p, vs)
            flat = at.flatten()

            def back(x):  # to rows of tokens
                return x.permute(0, 3, 1, 2, 4).reshape(rows * longest, step * each, -1)

            columns = slice(g * each, (g + step) * each)
            out[:, columns].index_copy_(0, flat, back(o))
            logsum[:, columns].index_copy_(0, flat, back(top + torch.log(total))[..., 0])
            if grad is None:
                continue
            gs = of_queries(grad)
            ds = p * (torch.matmul(gs, vs.transpose(-1, -2)) - (gs * o).sum(-1, keepdim=True)) * scale
            dq[:, columns].index_copy_(0, flat, back(torch.matmul(ds, ks)))

            def of_key_rows(x):
                return x.sum(2).permute(0, 2, 1, 3).reshape(rows * longest_keys, step, -1)

            dk[:, g:g + step].index_copy_(0, key_at.flatten(), of_key_rows(torch.matmul(ds.transpose(-1, -2), qs)))
            dv[:, g:g + step].index_copy_(0, key_at.flatten(), of_key_rows(torch.matmul(p.transpose(-1, -2), gs)))
    result = (out[:-1].to(q.dtype), logsum[:-1].t().contiguous())
    return result if grad is None else result + tuple(x[:-1].to(q.dtype) for x in (dq, dk, dv))


def _plain_attend(st):
    out, logsum = _plain_attention(st)
    return (out, logsum) if st["case"]["keep"] else out


_PLAIN = dict(rotary=_plain_rotary, attention=_plain_attend, attention_step=lambda st: _plain_attention(st, st["grad"]))


# ------------------------------------------------------------------ from the definitions, in 64 bits

def exact(case, seed):
    st = prepare(case, seed)
    queries, keys = _lengths(case)
    if case["op"] == "rotary":
        n = case["rotated"] // 2
        first = st["starts"].cpu().numpy().astype(np.int64) if st["starts"] is not None else np.zeros(case["rows"], np.int64)
        position = np.concatenate([np.arange(length) + begin for length, begin in zip(queries, first)])
        angle = torch.outer(_on_device(position).double(), _on_device(_frequencies(case)))
        turn = torch.polar(torch.full_like(angle, st["magnitude"]), -angle if case["inverse"] else angle)[:, None]
        x = st["x"].double()
        if case["layout"] == "half":
            z = torch.complex(x[..., :n].contiguous(), x[..., n:2 * n].contiguous()) * turn
            return torch.cat([z.real, z.imag, x[..., 2 * n:]], -1)
        z = torch.view_as_complex(x[..., :2 * n].reshape(*x.shape[:2], n, 2)) * turn
        return torch.cat([torch.view_as_real(z).flatten(-2), x[..., 2 * n:]], -1)
    kv, width = case["kv_heads"], case["width"]
    each = case["heads"] // kv
    step = case["op"] == "attention_step"
    key_first = st["key_offsets"].cpu().numpy() if case["earlier"] else _offsets(queries)
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device=DEVICE)
    logsum = torch.full((case["heads"], case["tokens"]), -math.inf, dtype=torch.float64, device=DEVICE)
    grads = [torch.zeros(st[x].shape, dtype=torch.float64, device=DEVICE) for x in ("q", "k", "v")] if step else []
    for first, length, key_at, key_length in zip(_offsets(queries), queries, key_first, keys):
        if length == 0:
            continue
        t, u = slice(int(first), int(first + length)), slice(int(key_at), int(key_at + key_length))
        hidden = torch.ones(length, key_length, dtype=torch.bool, device=DEVICE).triu(int(key_length - length) + 1) if case["causal"] else None
        at_once = kv if case["heads"] * length * key_length <= 2**27 else 1
        for g in range(0, kv, at_once):
            h, m = slice(g * each, (g + at_once) * each), slice(g, g + at_once)
            q = st["q"][t, h].double().transpose(0, 1).reshape(at_once, each * length, width).requires_grad_(step)
            k, v = (st[x][u, m].double().transpose(0, 1).contiguous().requires_grad_(step) for x in ("k", "v"))
            s = torch.bmm(q, k.mT.contiguous()).view(at_once, each, length, key_length) / math.sqrt(width)
            if hidden is not None:
                s = s.masked_fill(hidden, -math.inf)
            l = torch.logsumexp(s, -1)
            o = torch.bmm(torch.softmax(s, -1).view(at_once, each * length, key_length), v)
            out[t, h] = o.detach().view(at_once * each, length, width).transpose(0, 1)
            logsum[h, t] = l.detach().reshape(-1, length)
            if step:
                upper = st["grad"][t, h].double().transpose(0, 1).reshape(o.shape)
                dq, dk, dv = torch.autograd.grad(o, (q, k, v), upper)
                grads[0][t, h] = dq.view(at_once * each, length, width).transpose(0, 1)
                grads[1][u, m], grads[2][u, m] = dk.transpose(0, 1), dv.transpose(0, 1)
    if step:
        return (out, logsum, *grads)
    return (out, logsum) if case["keep"] else out


# ------------------------------------------------------------------ what a pass cannot do without

def work(case):
    b = 4 if case["dtype"] == "float32" else 2
    tokens, heads, width = case["tokens"], case["heads"], case["width"]
    if case["op"] == "rotary":
        columns = 4 * (case["rows"] + 1) + (4 * case["rows"] if case["start"] else 0) + 4 * case["rotated"]
        return {"bytes": 2 * b * tokens * heads * width + columns, "flops": 3 * tokens * heads * case["rotated"]}
    kv = case["kv_heads"]
    of_queries, of_keys = tokens * heads * width, (tokens + case["earlier"]) * kv * width
    columns = 4 * (case["rows"] + 1) * (3 if case["earlier"] else 1)
    pairs = heads * _pairs(case)
    if case["op"] == "attention":
        return {"bytes": b * 2 * (of_queries + of_keys) + columns + (4 * tokens * heads if case["keep"] else 0), "flops": int(4 * width * pairs)}
    # reads queries, keys, values and the gradient, writes the result and the gradients; two products forward, five back
    return {"bytes": b * (4 * of_queries + 4 * of_keys) + columns + 4 * tokens * heads, "flops": int(14 * width * pairs)}
