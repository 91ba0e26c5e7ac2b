"""A text encoder, from strings to a training step, on one GPU:

    normalize_characters -> wordpiece_tokenize -> embedding -> layer_norm
        -> per layer: with heads, linear -> rotary positions of queries and keys -> attention -> linear -> layer_norm of residual + dropout;
                      linear with gelu -> linear -> layer_norm of residual + dropout
        -> linear

and the way back through the gradients of each.  The task is a small one that needs no labels: of every token, what stands next
to it in its text, as a row of a fixed random table of codes; the loss is the mean square of the differences.

    python -m cudf_amd.examples.text_encoder [--steps 100] [--rows 2000] [--width 256] [--layers 2] [--heads 0] [--dtype bfloat16]
"""
from __future__ import annotations

import argparse
import time
from typing import Dict, List, Tuple

import numpy as np
import torch

from cudf_amd import encoder, nvtext
from cudf_amd.arrow_host import HostStringsColumn


class TextEncoder:
    """The parameters by name, and the two directions through the layers.  Matrices are of `dtype`, what the layer norms scale
    by is float32.  With `heads`, which divide the width, every token sees those in front of it in its text; without, itself alone.
    `key_heads` of them, a divisor (as many as heads if not given), have keys and values."""

    def __init__(self, vocabulary_size: int, positions: int, width: int, layers: int, outputs: int, dtype: torch.dtype = torch.bfloat16, seed: int = 0, heads: int = 0,
                 key_heads: int = 0):
        self.layers, self.vocabulary_size, self.positions = layers, vocabulary_size, positions
        self.heads, self.key_heads = heads, key_heads or heads
        if heads and (width % heads or width // heads % 2 or heads % self.key_heads):
            raise ValueError("heads must divide the width into an even number of values each, and key_heads divide heads")
        gen = torch.Generator().manual_seed(seed)

        def random(*shape, scale):
            return (torch.randn(shape, generator=gen) * scale).to("cuda", dtype)

        self.parameters: Dict[str, torch.Tensor] = {
            "tokens": random(vocabulary_size, width, scale=1.0),
            "positions": random(positions, width, scale=0.1),
            "norm.weight": torch.ones(width, device="cuda"),
            "norm.bias": torch.zeros(width, device="cuda"),
            "out.weight": random(outputs, width, scale=width**-0.5),
            "out.bias": torch.zeros(outputs, device="cuda", dtype=dtype),
        }
        for i in range(layers):
            self.parameters.update({
                f"{i}.up.weight": random(4 * width, width, scale=width**-0.5),
                f"{i}.up.bias": torch.zeros(4 * width, device="cuda", dtype=dtype),
                f"{i}.down.weight": random(width, 4 * width, scale=0.5 * width**-0.5),
                f"{i}.down.bias": torch.zeros(width, device="cuda", dtype=dtype),
                f"{i}.norm.weight": torch.ones(width, device="cuda"),
                f"{i}.norm.bias": torch.zeros(width, device="cuda"),
            })
        if heads:
            of_head = width // heads
            self.frequencies = encoder.rotary_frequencies(of_head)
            for i in range(layers):
                self.parameters.update({
                    f"{i}.heads.weight": random((heads + 2 * self.key_heads) * of_head, width, scale=width**-0.5),
                    f"{i}.heads.bias": torch.zeros((heads + 2 * self.key_heads) * of_head, device="cuda", dtype=dtype),
                    f"{i}.mix.weight": random(width, width, scale=0.5 * width**-0.5),
                    f"{i}.mix.bias": torch.zeros(width, device="cuda", dtype=dtype),
                    f"{i}.mix_norm.weight": torch.ones(width, device="cuda"),
                    f"{i}.mix_norm.bias": torch.zeros(width, device="cuda"),
                })

    def _parts(self, x: torch.Tensor) -> Tuple[torch.Tensor, ...]:
        """(queries and keys, which are rotated; queries; keys; values) of a tensor of all heads side by side."""
        n, m = self.heads, self.key_heads
        x = x.unflatten(1, (n + 2 * m, -1))
        return x[:, : n + m], x[:, :n], x[:, n : n + m], x[:, n + m :]

    def _attend(self, i: int, h: torch.Tensor, tokens: nvtext.DeviceListColumn):
        """What every token takes from those up to it in its text, and what the way back needs."""
        q = self.parameters
        x = encoder.linear(h, q[f"{i}.heads.weight"], q[f"{i}.heads.bias"])
        turned, queries, keys, values = self._parts(x)
        encoder.rotary(turned, tokens, self.frequencies, out=turned)
        out, saved = encoder.attention(queries, keys, values, tokens, causal=True, keep=True)
        out = out.flatten(1)
        return encoder.linear(out, q[f"{i}.mix.weight"], q[f"{i}.mix.bias"]), (h, x, out, saved)

    def _attend_backward(self, i: int, g: torch.Tensor, kept: Tuple, tokens: nvtext.DeviceListColumn, grads: Dict[str, torch.Tensor]) -> torch.Tensor:
        q, (h, x, out, saved) = self.parameters, kept
        g, grads[f"{i}.mix.weight"], grads[f"{i}.mix.bias"] = encoder.linear_backward(g, out, q[f"{i}.mix.weight"])
        _, queries, keys, values = self._parts(x)
        x_grad = torch.empty_like(x)
        turned, *parts = self._parts(x_grad)
        encoder.attention_backward(g.view(queries.shape), queries, keys, values, saved, tokens, causal=True, out=tuple(parts))
        encoder.rotary(turned, tokens, self.frequencies, inverse=True, out=turned)
        g, grads[f"{i}.heads.weight"], grads[f"{i}.heads.bias"] = encoder.linear_backward(x_grad, h, q[f"{i}.heads.weight"])
        return g

    def forward(self, tokens: nvtext.DeviceListColumn, p: float = 0.0, seed: int = 0) -> Tuple[torch.Tensor, List]:
        """The outputs, a row a token, and what backward() needs.  Dropout call i draws under the number i of the seed, that behind
        the attention of layer i under the number of layers more."""
        q = self.parameters
        h, saved = encoder.layer_norm(encoder.embedding(tokens, q["tokens"], q["positions"]), q["norm.weight"], q["norm.bias"], keep=True)
        kept = [saved]
        for i in range(self.layers):
            mixed = None
            if self.heads:
                v, attended = self._attend(i, h, tokens)
                h, saved = encoder.layer_norm(v, q[f"{i}.mix_norm.weight"], q[f"{i}.mix_norm.bias"], residual=saved.sum, p=p, seed=seed, offset=self.layers + i, keep=True)
                mixed = (attended, saved)
            u, z = encoder.linear(h, q[f"{i}.up.weight"], q[f"{i}.up.bias"], "gelu", keep=True)
            v = encoder.linear(u, q[f"{i}.down.weight"], q[f"{i}.down.bias"])
            kept.append((h, z, u, mixed))
            h, saved = encoder.layer_norm(v, q[f"{i}.norm.weight"], q[f"{i}.norm.bias"], residual=saved.sum, p=p, seed=seed, offset=i, keep=True)
            kept.append(saved)
        kept.append(h)
        return encoder.linear(h, q["out.weight"], q["out.bias"]), kept

    def backward(self, grad: torch.Tensor, tokens: nvtext.DeviceListColumn, kept: List, p: float = 0.0, seed: int = 0) -> Dict[str, torch.Tensor]:
        """The gradients of all parameters, from that of forward()'s outputs."""
        q, grads = self.parameters, {}
        g, grads["out.weight"], grads["out.bias"] = encoder.linear_backward(grad, kept[-1], q["out.weight"])
        stream = None  # the gradient that comes back along the residual stream
        for i in reversed(range(self.layers)):
            h, z, u, mixed = kept[1 + 2 * i]
            g, stream, grads[f"{i}.norm.weight"], grads[f"{i}.norm.bias"] = encoder.layer_norm_backward(
                g, kept[2 + 2 * i], q[f"{i}.norm.weight"], p=p, seed=seed, offset=i, sum_grad=stream)
            g, grads[f"{i}.down.weight"], grads[f"{i}.down.bias"] = encoder.linear_backward(g, u, q[f"{i}.down.weight"])
            g, grads[f"{i}.up.weight"], grads[f"{i}.up.bias"] = encoder.linear_backward(g, h, q[f"{i}.up.weight"], "gelu", z)
            if mixed is not None:
                attended, saved = mixed
                g, stream, grads[f"{i}.mix_norm.weight"], grads[f"{i}.mix_norm.bias"] = encoder.layer_norm_backward(
                    g, saved, q[f"{i}.mix_norm.weight"], p=p, seed=seed, offset=self.layers + i, sum_grad=stream)
                g = self._attend_backward(i, g, attended, tokens, grads)
        g, _, grads["norm.weight"], grads["norm.bias"] = encoder.layer_norm_backward(g, kept[0], q["norm.weight"], sum_grad=stream)
        grads["tokens"], grads["positions"] = encoder.embedding_backward(tokens, g, self.vocabulary_size, self.positions)
        return grads

    def update(self, grads: Dict[str, torch.Tensor], rate: float, most: float = 0.1) -> None:
        """A step down the gradients, as if these were no longer than `most` together."""
        length = torch.stack([g.float().square().sum() for g in grads.values()]).sum().sqrt()
        scale = -rate * (most / length).clamp(max=1.0)
        for name, parameter in self.parameters.items():
            parameter.add_((grads[name].float() * scale).to(parameter.dtype))


def train_step(model: TextEncoder, tokens: nvtext.DeviceListColumn, target: torch.Tensor, rate: float, p: float, seed: int) -> torch.Tensor:
    """One step of gradient descent; the loss before it."""
    out, kept = model.forward(tokens, p, seed)
    difference = out.float() - target.float()
    grad = (difference * (2.0 / difference.numel())).to(out.dtype)
    model.update(model.backward(grad, tokens, kept, p, seed), rate)
    return difference.square().mean()


def synthetic_text(rows: int, seed: int = 0) -> Tuple[HostStringsColumn, HostStringsColumn]:
    """(texts with accents, capitals and punctuation, a vocabulary): words follow one another by a fixed order, now and then by
    chance."""
    rng = np.random.default_rng(seed)
    letters = list("abcdefghijklmnopqrstuvwxyz")
    stems = sorted({"".join(rng.choice(letters, int(rng.integers(2, 8)))) for _ in range(200)})
    vocabulary = ["[PAD]", "[UNK]"] + list(",.!") + stems
    follows = rng.permutation(len(stems))
    texts = []
    for _ in range(rows):
        word, words = int(rng.integers(0, len(stems))), []
        for _ in range(int(rng.integers(1, 40))):
            words.append(stems[word].capitalize() if rng.random() < 0.2 else stems[word])
            word = int(follows[word]) if rng.random() < 0.8 else int(rng.integers(0, len(stems)))
        texts.append(" ".join(words).replace("e", "é", 1) + str(rng.choice([",", ".", "!"])))
    return HostStringsColumn.from_pylist(texts), HostStringsColumn.from_pylist(vocabulary)


def tokenize(texts: HostStringsColumn, vocabulary: HostStringsColumn) -> nvtext.DeviceListColumn:
    normalizer = nvtext.CharacterNormalizer(True, nvtext.DeviceStringsColumn.from_host(HostStringsColumn.from_pylist([])))
    normalized = nvtext.normalize_characters(nvtext.DeviceStringsColumn.from_host(texts), normalizer)
    return nvtext.wordpiece_tokenize(normalized, nvtext.WordPieceVocabulary(nvtext.DeviceStringsColumn.from_host(vocabulary)))


def next_tokens(tokens: nvtext.DeviceListColumn) -> nvtext.DeviceListColumn:
    """The column in which every token is the one next to it; the last one of a row is -1, for which an embedding is zeros."""
    ids = tokens.child.view(torch.int32)[: tokens.child_size].roll(-1)
    ends = tokens.offsets.view(torch.int32)[1 : tokens.size + 1].long() - 1
    ids[ends[ends >= 0]] = -1  # (the last of an empty row is that of a row before it)
    return nvtext.DeviceListColumn(tokens.offsets, ids, None, tokens.size, 0, tokens.child_dtype, tokens.child_size)


def main(argv=None) -> None:
    parser = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    parser.add_argument("--steps", type=int, default=100)
    parser.add_argument("--rows", type=int, default=2000)
    parser.add_argument("--width", type=int, default=256)
    parser.add_argument("--layers", type=int, default=2)
    parser.add_argument("--heads", type=int, default=0, help="of attention; 0: every token by itself")
    parser.add_argument("--dtype", choices=["float32", "float16", "bfloat16"], default="bfloat16")
    parser.add_argument("--rate", type=float, default=4.0)
    args = parser.parse_args(argv)
    dtype = getattr(torch, args.dtype)
    texts, vocabulary = synthetic_text(args.rows)
    tokens = tokenize(texts, vocabulary)
    model = TextEncoder(vocabulary.size, positions=64, width=args.width, layers=args.layers, outputs=32, dtype=dtype, heads=args.heads)
    codes = torch.randn(vocabulary.size, 32, generator=torch.Generator().manual_seed(1)).to("cuda", dtype)
    target = encoder.embedding(next_tokens(tokens), codes)
    for step in range(args.steps):
        begin = time.perf_counter()
        loss = train_step(model, tokens, target, args.rate, p=0.1, seed=step).item()
        if step % 10 == 0 or step + 1 == args.steps:
            print(f"step {step}: loss {loss:.4f}, {tokens.child_size / (time.perf_counter() - begin) / 1e6:.2f} M tokens/s", flush=True)
    # what a service does: one text, no gradients
    one = tokenize(texts.slice(0, 1), vocabulary)
    out, _ = model.forward(one)
    nearest = torch.cdist(out.float(), codes.float()).argmin(1)
    words = [word.decode() for word in vocabulary.to_pylist()]
    print("first text:      ", " ".join(words[i] for i in one.to_host().to_pylist()[0]))
    print("what stands next:", " ".join(words[i] for i in nearest.tolist()))


if __name__ == "__main__":
    main()
