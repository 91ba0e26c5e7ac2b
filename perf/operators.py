"""Timed cases of the encoder operators: what stands between the tokenizer's column of ids and a model that learns from it.

A case is a dict; `op` names the call.  The column of an embedding has `rows` texts with `tokens` ids in all: lengths
lognormal (sigma 0.6) as the texts of a corpus have, ids drawn by Zipf's law (exponent 1.1) over a `vocabulary`, one in a
thousand the -1 that wordpiece_tokenize gives an unknown word where the vocabulary has no entry for those.  The other
operators see the tokens of a batch one after the other, packed, `rows` of them with `width` values each.  `linear` maps
`inputs` values a token to `outputs`.  `dtype` is the type of tensors and tables; `weights` that of a layer norm's weights.
"""
import math

import numpy as np
import torch

own = False

DEVICE = "cuda"

ACTIVATIONS = ["none", "relu", "gelu", "gelu_tanh", "silu"]


def listed():
    return [
        # a request to a serving process: 29 short texts against the table of a vocabulary of 30,522
        dict(name="embed_request", op="embedding", rows=29, tokens=1163, vocabulary=30522, positions=512, width=768, dtype="bfloat16"),
        # a shard of a corpus in several scripts, embedded over the vocabulary of 250,000
        dict(name="embed_corpus", op="embedding", rows=4001, tokens=512011, vocabulary=250000, positions=512, width=1024, dtype="float16"),
        # the gradients of both tables in a step of pre-training
        dict(name="embed_backward", op="embedding_backward", rows=2048, tokens=262139, vocabulary=30522, positions=512, width=768, dtype="bfloat16"),
        # activations of odd width in full precision, where the mask's cost has the least to hide behind
        dict(name="dropout_f32", op="dropout", rows=5001, width=1021, p=0.5, dtype="float32"),
        # the activations of a training batch
        dict(name="dropout_batch", op="dropout", rows=65536, width=1024, p=0.1, dtype="bfloat16"),
        # one token of one text, as a serving process normalizes it
        dict(name="norm_token", op="layer_norm", rows=1, width=1024, p=0.0, residual=True, weights="bfloat16", dtype="bfloat16"),
        # the end of a block in training: dropout, the residual and the norm, with what the gradient needs
        dict(name="norm_train", op="layer_norm", rows=32768, width=1024, p=0.1, residual=True, weights="float32", dtype="bfloat16"),
        # its gradient, half as wide again and an odd number of tokens
        dict(name="norm_backward", op="layer_norm_backward", rows=20011, width=1536, p=0.1, sum_grad=False, weights="float16", dtype="float16"),
        # one token through the first half of a feed-forward block
        dict(name="linear_token", op="linear", rows=1, inputs=1024, outputs=4096, activation="gelu", residual=False, keep=False, dtype="bfloat16"),
        # widths that no tile divides, the second half of a block with its residual
        dict(name="linear_odd", op="linear", rows=1777, inputs=2051, outputs=1003, activation="none", residual=True, keep=False, dtype="float16"),
        # the first half of a feed-forward block over a training batch, keeping what its gradient needs
        dict(name="linear_train", op="linear", rows=32768, inputs=1024, outputs=4096, activation="gelu", residual=False, keep=True, dtype="bfloat16"),
        # the gradients of the same half
        dict(name="linear_backward", op="linear_backward", rows=16384, inputs=1024, outputs=4096, activation="gelu", dtype="bfloat16"),
    ]


def _log_between(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """A width as models have them (a multiple of 64), or now and then any other."""
    w = _log_between(rng, lo, hi)
    kind = rng.choice(["model", "model", "model", "eight", "any"])
    w = max(64, w // 64 * 64) if kind == "model" else max(8, w // 8 * 8) if kind == "eight" else w
    return w if w != 3072 else 3136


def draw(rng):
    op = rng.choice(["embedding", "embedding_backward", "dropout", "layer_norm", "layer_norm_backward", "linear", "linear", "linear_backward"])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    case = dict(op=op, dtype=dtype)
    if op in ("embedding", "embedding_backward"):
        width = _width(rng, 64, 2048)
        most = 200_000_000 if op == "embedding" else 100_000_000
        tokens = _log_between(rng, 1, most // width)
        vocabulary = min(rng.choice([1000, 30522, 250000]), most // width)
        case.update(rows=max(1, tokens // _log_between(rng, 8, 400)), tokens=tokens, vocabulary=vocabulary, positions=rng.choice([0, 128, 512, 512]), width=width)
    elif op in ("dropout", "layer_norm", "layer_norm_backward"):
        width = _width(rng, 64, 8192)
        case.update(rows=_log_between(rng, 1, 30_000_000 // width), width=width)
        case["p"] = rng.choice([0.1, 0.1, 0.25, 0.5]) if op == "dropout" else rng.choice([0.0, 0.1, 0.3])
        if op != "dropout":
            case["weights"] = rng.choice([dtype, "float32"])
            case.update(residual=rng.choice([False, True, True])) if op == "layer_norm" else case.update(sum_grad=rng.choice([False, False, True]))
    else:
        case["dtype"] = rng.choice(["bfloat16", "bfloat16", "float16"])
        inputs, outputs = _width(rng, 64, 8192), _width(rng, 64, 8192)
        most = (130_000_000_000 if op == "linear" else 65_000_000_000) // (inputs * outputs)
        rows = _log_between(rng, 1, max(2, min(32768, most)))
        case.update(rows=rows, inputs=inputs, outputs=outputs, activation=rng.choice(ACTIVATIONS))
        if op == "linear":
            case.update(residual=rng.choice([False, True]), keep=rng.choice([False, False, True]))
    return case


# ------------------------------------------------------------------ inputs

def _zipf(vocabulary):
    p = 1.0 / np.arange(1, vocabulary + 1) ** 1.1
    return p / p.sum()


def _column(case, gen, seed):
    """The buffers of a LIST<INT32> column as the tokenizer returns it: bytes of int32 offsets and of int32 ids."""
    rows, tokens, vocabulary = case["rows"], case["tokens"], case["vocabulary"]
    lengths = np.random.default_rng(seed).lognormal(0.0, 0.6, rows)
    ends = np.minimum(np.floor(np.cumsum(lengths) * (tokens / lengths.sum())), tokens)
    offsets = np.concatenate([[0], ends]).astype(np.int32)
    offsets[-1] = tokens
    by_rank = torch.randperm(vocabulary, generator=gen, device=DEVICE)
    upto = torch.from_numpy(np.cumsum(_zipf(vocabulary))).to(DEVICE)
    rank = torch.searchsorted(upto, torch.rand(tokens, generator=gen, device=DEVICE, dtype=torch.float64)).clamp_(max=vocabulary - 1)
    unknown = torch.rand(tokens, generator=gen, device=DEVICE) < 0.001
    ids = torch.where(unknown, -1, by_rank[rank]).to(torch.int32)
    return torch.from_numpy(offsets).to(DEVICE).view(torch.uint8), ids.view(torch.uint8)


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(seed)
    dtype = getattr(torch, case["dtype"])

    def normal(*shape, scale=1.0, mean=0.0, dtype=dtype):
        return (torch.randn(shape, generator=gen, device=DEVICE) * scale + mean).to(dtype)

    st = dict(case=case, seed=(seed * 0x9E3779B97F4A7C15 + 12345) % 2**63, offset=seed % 1000)
    op = case["op"]
    if op in ("embedding", "embedding_backward"):
        st["offsets"], st["ids"] = _column(case, gen, seed)
        if op == "embedding":
            st["table"] = normal(case["vocabulary"], case["width"], scale=0.05)
            st["positions"] = normal(case["positions"], case["width"], scale=0.05) if case["positions"] else None
        else:
            st["grad"] = normal(case["tokens"], case["width"], scale=0.1)
    elif op == "dropout":
        st["x"] = normal(case["rows"], case["width"])
    elif op == "layer_norm":
        weights = getattr(torch, case["weights"])
        st["x"] = normal(case["rows"], case["width"], mean=0.1)
        st["residual"] = normal(case["rows"], case["width"]) if case["residual"] else None
        st["weight"] = normal(case["width"], scale=0.1, mean=1.0, dtype=weights)
        st["bias"] = normal(case["width"], scale=0.1, dtype=weights)
    elif op == "layer_norm_backward":
        st["grad"] = normal(case["rows"], case["width"], scale=0.1)
        st["sum"] = normal(case["rows"], case["width"], mean=0.1)
        st["mean"] = st["sum"].float().mean(1)
        st["rstd"] = torch.rsqrt((st["sum"].float() - st["mean"][:, None]).square().mean(1) + 1e-5)
        st["weight"] = normal(case["width"], scale=0.1, mean=1.0, dtype=getattr(torch, case["weights"]))
        st["sum_grad"] = normal(case["rows"], case["width"], scale=0.1) if case["sum_grad"] else None
    else:
        st["x"] = normal(case["rows"], case["inputs"])
        st["weight"] = normal(case["outputs"], case["inputs"], scale=case["inputs"] ** -0.5)
        if op == "linear":
            st["bias"] = normal(case["outputs"], scale=0.1)
            st["residual"] = normal(case["rows"], case["outputs"]) if case["residual"] else None
        else:
            st["grad"] = normal(case["rows"], case["outputs"], scale=0.1)
            st["preactivation"] = normal(case["rows"], case["outputs"]) if case["activation"] != "none" else None
    return st


# ------------------------------------------------------------------ one pass

def run(st):
    return _call(st) if own else _PLAIN[st["case"]["op"]](st)


def _call(st):
    """The framework's operators, as a user's program calls them."""
    from cudf_amd import encoder, nvtext
    case = st["case"]
    op = case["op"]
    if op == "embedding":
        tokens = nvtext.DeviceListColumn(st["offsets"], st["ids"], None, case["rows"], 0, np.dtype(np.int32), case["tokens"])
        return encoder.embedding(tokens, st["table"], st["positions"])
    if op == "embedding_backward":
        tokens = nvtext.DeviceListColumn(st["offsets"], st["ids"], None, case["rows"], 0, np.dtype(np.int32), case["tokens"])
        return encoder.embedding_backward(tokens, st["grad"], case["vocabulary"], case["positions"])
    if op == "dropout":
        return encoder.dropout(st["x"], case["p"], st["seed"], st["offset"])
    if op == "layer_norm":
        out, saved = encoder.layer_norm(st["x"], st["weight"], st["bias"], 1e-5, st["residual"], case["p"], st["seed"], st["offset"], keep=True)
        return out, saved.sum, saved.mean, saved.rstd
    if op == "layer_norm_backward":
        saved = encoder.LayerNormSaved(st["sum"], st["mean"], st["rstd"])
        return encoder.layer_norm_backward(st["grad"], saved, st["weight"], case["p"], st["seed"], st["offset"], st["sum_grad"])
    if op == "linear":
        return encoder.linear(st["x"], st["weight"], st["bias"], case["activation"], st["residual"], keep=case["keep"])
    return encoder.linear_backward(st["grad"], st["x"], st["weight"], case["activation"], st["preactivation"])


# ------------------------------------------------------------------ the plain forms

def _rows_of(st):
    """Of every token: its id or -1, and its position in its row."""
    offsets, ids = st["offsets"].view(torch.int32).long(), st["ids"].view(torch.int32).long()
    t = torch.arange(ids.numel(), device=ids.device)
    row = torch.searchsorted(offsets, t, right=True) - 1
    return ids, t - offsets[row]


def _plain_embedding(st):
    ids, at = _rows_of(st)
    table = st["table"]
    out = torch.where((ids >= 0)[:, None], table[ids.clamp(min=0)].float(), 0.0)
    if st["positions"] is not None:
        places = st["positions"]
        out = out + torch.where((at < places.shape[0])[:, None], places[at.clamp(max=places.shape[0] - 1)].float(), 0.0)
    return out.to(table.dtype)


def _plain_embedding_backward(st):
    ids, at = _rows_of(st)
    case, grad = st["case"], st["grad"].float()
    # (one row more takes what belongs to no entry)
    table = torch.zeros(case["vocabulary"] + 1, case["width"], device=grad.device).index_add_(0, torch.where(ids < 0, case["vocabulary"], ids), grad)
    positions = None
    if case["positions"]:
        positions = torch.zeros(case["positions"] + 1, case["width"], device=grad.device).index_add_(0, at.clamp(max=case["positions"]), grad)
        positions = positions[:-1].to(st["grad"].dtype)
    return table[:-1].to(st["grad"].dtype), positions


def _kept(rows, width, p, seed, offset):
    """Which values a dropout keeps, and what they are multiplied by: Philox4x32-10 (Salmon, Moraes, Dror and Shaw, 2011)
    of the counter {column / 8, row, row >> 32, offset} under the key `seed`, eight draws of 16 bits of it."""
    low = 0xFFFFFFFF
    blocks = -(-width // 8)
    i = torch.arange(rows, device=DEVICE)[:, None]
    c0 = torch.arange(blocks, device=DEVICE)[None, :].expand(rows, blocks)
    c1, c2 = (i & low).expand(rows, blocks), (i >> 32).expand(rows, blocks)
    c3 = torch.full((1, 1), offset, device=DEVICE).expand(rows, blocks)
    k0, k1 = seed & low, seed >> 32
    for _ in range(10):  # each round takes what the one before gives
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = ((b >> 32) & low) ^ c1 ^ k0, b & low, ((a >> 32) & low) ^ c3 ^ k1, a & low
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    draws = torch.stack([c0 & 0xFFFF, c0 >> 16, c1 & 0xFFFF, c1 >> 16, c2 & 0xFFFF, c2 >> 16, c3 & 0xFFFF, c3 >> 16], 2).reshape(rows, blocks * 8)[:, :width]
    dropped = round(p * 65536)
    return draws >= dropped, 65536 / (65536 - dropped)


def _plain_dropout(st):
    x, case = st["x"], st["case"]
    keep, scale = _kept(*x.shape, case["p"], st["seed"], st["offset"])
    return torch.where(keep, x.float() * scale, 0.0).to(x.dtype)


def _plain_layer_norm(st):
    x, case = st["x"], st["case"]
    s = x.float()
    if case["p"]:
        keep, scale = _kept(*x.shape, case["p"], st["seed"], st["offset"])
        s = torch.where(keep, s * scale, 0.0)
    if st["residual"] is not None:
        s = s + st["residual"].float()
    mean = s.mean(1, keepdim=True)
    rstd = 1 / torch.sqrt((s - mean).square().mean(1, keepdim=True) + 1e-5)
    out = (s - mean) * rstd * st["weight"].float() + st["bias"].float()
    return out.to(x.dtype), s.to(x.dtype), mean[:, 0], rstd[:, 0]


def _plain_layer_norm_backward(st):
    grad, case = st["grad"].float(), st["case"]
    dtype, weights = st["grad"].dtype, st["weight"].dtype
    xh = (st["sum"].float() - st["mean"][:, None]) * st["rstd"][:, None]
    a = grad * st["weight"].float()
    d = st["rstd"][:, None] * (a - a.mean(1, keepdim=True) - xh * (a * xh).mean(1, keepdim=True))
    if st["sum_grad"] is not None:
        d = d + st["sum_grad"].float()
    dx = d
    if case["p"]:
        keep, scale = _kept(*d.shape, case["p"], st["seed"], st["offset"])
        dx = torch.where(keep, d * scale, 0.0)
    return dx.to(dtype), d.to(dtype), (grad * xh).sum(0).to(weights), grad.sum(0).to(weights)


def _activate(z, name):
    if name == "relu":
        return torch.where(z > 0, z, 0.0)
    if name == "gelu":
        return z * (0.5 + 0.5 * torch.erf(z * 0.5**0.5))
    if name == "gelu_tanh":
        return z * (0.5 + 0.5 * torch.tanh((2 / math.pi) ** 0.5 * (z + 0.044715 * z * z * z)))
    if name == "silu":
        return z / (1 + torch.exp(-z))
    return z


def _slope(z, name):
    if name == "relu":
        return (z > 0).float()
    if name == "gelu":
        return 0.5 + 0.5 * torch.erf(z * 0.5**0.5) + z * torch.exp(-0.5 * z * z) * (2 * math.pi) ** -0.5
    if name == "gelu_tanh":
        t = torch.tanh((2 / math.pi) ** 0.5 * (z + 0.044715 * z * z * z))
        return 0.5 + 0.5 * t + 0.5 * z * (1 - t * t) * (2 / math.pi) ** 0.5 * (1 + 3 * 0.044715 * z * z)
    s = 1 / (1 + torch.exp(-z))
    return s * (1 + z * (1 - s))


def _plain_linear(st):
    x, case = st["x"], st["case"]
    z = x.float() @ st["weight"].float().t() + st["bias"].float()
    out = _activate(z, case["activation"])
    if st["residual"] is not None:
        out = out + st["residual"].float()
    return (out.to(x.dtype), z.to(x.dtype)) if case["keep"] else out.to(x.dtype)


def _plain_linear_backward(st):
    x, case, d = st["x"], st["case"], st["grad"].float()
    if case["activation"] != "none":
        d = d * _slope(st["preactivation"].float(), case["activation"])
    return (d @ st["weight"].float()).to(x.dtype), (d.t() @ x.float()).to(x.dtype), d.sum(0).to(x.dtype)


_PLAIN = dict(embedding=_plain_embedding, embedding_backward=_plain_embedding_backward, dropout=_plain_dropout, layer_norm=_plain_layer_norm,
              layer_norm_backward=_plain_layer_norm_backward, linear=_plain_linear, linear_backward=_plain_linear_backward)


# ------------------------------------------------------------------ from the definitions, in 64 bits

def _draws64(rows, width, seed, offset):
    """The 16-bit draws of a dropout, [rows, width], in whole numbers of numpy."""
    u, low = np.uint64, np.uint64(0xFFFFFFFF)
    block, row = np.meshgrid(np.arange(-(-width // 8), dtype=u), np.arange(rows, dtype=u))
    word = [block, row & low, row >> u(32), np.full_like(row, offset)]
    key = [seed % 2**32, seed >> 32]
    for _ in range(10):
        a, b = word[0] * u(0xD2511F53), word[2] * u(0xCD9E8D57)
        word = [(b >> u(32)) ^ word[1] ^ u(key[0]), b & low, (a >> u(32)) ^ word[3] ^ u(key[1]), a & low]
        key = [(key[0] + 0x9E3779B9) % 2**32, (key[1] + 0xBB67AE85) % 2**32]
    words = np.stack(word, axis=-1).astype("<u4")
    return words.reshape(rows, -1).view("<u2")[:, :width]


def _multipliers64(case, st):
    dropped = round(case["p"] * 65536)
    if dropped == 0:
        return 1.0
    kept = torch.from_numpy(_draws64(case["rows"], case["width"], st["seed"], st["offset"]).astype(np.int32) >= dropped).to(DEVICE)
    return kept.double() * 65536 / (65536 - dropped)


def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]
    wide = {k: v.double() for k, v in st.items() if isinstance(v, torch.Tensor) and v.is_floating_point()}
    if op in ("embedding", "embedding_backward"):
        offsets, ids = st["offsets"].cpu().numpy().view(np.int32), st["ids"].cpu().numpy().view(np.int32)
        lengths = np.diff(offsets)
        at = np.arange(case["tokens"]) - np.repeat(offsets[:-1], lengths)
        known, placed = np.flatnonzero(ids >= 0), np.flatnonzero(at < case["positions"])
        at, ids = torch.from_numpy(at[placed]).to(DEVICE), torch.from_numpy(ids[known].astype(np.int64)).to(DEVICE)
        known, placed = torch.from_numpy(known).to(DEVICE), torch.from_numpy(placed).to(DEVICE)

        def into(size, index, values):
            return torch.zeros(size, case["width"], dtype=torch.float64, device=DEVICE).index_add_(0, index, values)
        if op == "embedding":
            out = into(case["tokens"], known, wide["table"][ids])
            return out.index_add_(0, placed, wide["positions"][at]) if case["positions"] else out
        return into(case["vocabulary"], ids, wide["grad"][known]), into(case["positions"], at, wide["grad"][placed]) if case["positions"] else None
    if op == "dropout":
        return wide["x"] * _multipliers64(case, st)
    if op == "layer_norm":
        s = wide["x"] * _multipliers64(case, st) + wide.get("residual", 0.0)
        var, mean = torch.var_mean(s, dim=1, correction=0, keepdim=True)
        rstd = (var + 1e-5) ** -0.5
        return (s - mean) * rstd * wide["weight"] + wide["bias"], s, mean[:, 0], rstd[:, 0]
    if op == "layer_norm_backward":
        rstd, g, n = wide["rstd"][:, None], wide["grad"], case["width"]
        xh = wide["sum"] * rstd - wide["mean"][:, None] * rstd
        a = g * wide["weight"]
        d = (n * a - a.sum(1, keepdim=True) - xh * (a * xh).sum(1, keepdim=True)) * rstd / n + wide.get("sum_grad", 0.0)
        return d * _multipliers64(case, st), d, torch.linalg.vecdot(g, xh, dim=0), g.sum(0)
    act = {"none": lambda z: z, "relu": torch.relu, "gelu": torch.nn.functional.gelu, "silu": torch.nn.functional.silu,
           "gelu_tanh": lambda z: torch.nn.functional.gelu(z, approximate="tanh")}[case["activation"]]
    if op == "linear":
        z = torch.addmm(wide["bias"], wide["x"], wide["weight"].t())
        out = act(z) + wide.get("residual", 0.0)
        return (out, z) if case["keep"] else out
    d = wide["grad"]
    if case["activation"] != "none":
        z = wide["preactivation"].requires_grad_(True)
        d, = torch.autograd.grad(act(z), z, d)
    return d @ wide["weight"], d.t() @ wide["x"], d.sum(0)


# ------------------------------------------------------------------ what a pass cannot do without

def work(case):
    size = {"bfloat16": 2, "float16": 2, "float32": 4}
    b, op = size[case["dtype"]], case["op"]
    if op in ("embedding", "embedding_backward"):
        column = 4 * case["tokens"] + 4 * (case["rows"] + 1)
        values = case["tokens"] * case["width"]
        if op == "embedding":
            # of the table, the rows of the entries that occur
            distinct = float((1 - (1 - _zipf(case["vocabulary"])) ** case["tokens"]).sum())
            places = min(case["positions"], case["tokens"])
            return {"bytes": int(column + b * (values + (distinct + places) * case["width"])), "flops": values}
        return {"bytes": column + b * (values + (case["vocabulary"] + case["positions"]) * case["width"]), "flops": values * (2 if case["positions"] else 1)}
    if op in ("dropout", "layer_norm", "layer_norm_backward"):
        n = case["rows"] * case["width"]
        if op == "dropout":
            return {"bytes": 2 * b * n, "flops": n}
        weights = size[case["weights"]] * case["width"]
        if op == "layer_norm":
            read = 2 if case["residual"] else 1
            return {"bytes": b * n * (read + 2) + 8 * case["rows"] + 2 * weights, "flops": 8 * n}
        tensors = 3 + (1 if case["p"] else 0) + (1 if case["sum_grad"] else 0)
        return {"bytes": b * n * tensors + 8 * case["rows"] + 3 * weights, "flops": 14 * n}
    m, k, n = case["rows"], case["inputs"], case["outputs"]
    if op == "linear":
        return {"bytes": b * (m * k + n * k + n + m * n * (1 + case["residual"] + case["keep"])), "flops": 2 * m * n * k}
    return {"bytes": b * (2 * m * k + 2 * n * k + n + m * n * (1 if case["activation"] == "none" else 2)), "flops": 4 * m * n * k}
