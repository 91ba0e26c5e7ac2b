"""The operators together where tokens see one another: the example's model with heads against the formulas in 64 bits, on another stream
and captured in a graph; and texts that go on token by token over caches of their keys."""
import os
import subprocess

import numpy as np
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

from cudf_amd import encoder  # noqa: E402
from cudf_amd.examples import text_encoder as te  # noqa: E402


@pytest.fixture(scope="module")
def data():
    texts, vocabulary = te.synthetic_text(40, seed=7)
    return te.tokenize(texts, vocabulary), vocabulary.size


def model_of(vocabulary_size, dtype, width=72, layers=2, outputs=17, heads=6, key_heads=3):
    return te.TextEncoder(vocabulary_size, positions=24, width=width, layers=layers, outputs=outputs, dtype=dtype, seed=5, heads=heads, key_heads=key_heads)


def offsets_of(tokens):
    return tokens.offsets.view(torch.int32)[: tokens.size + 1].cpu().numpy()


def turn(x, at, frequencies):
    """Rotary positions of [tokens, heads, values] in 64 bits, the halves of a head as its pairs."""
    angle = torch.outer(at.double(), frequencies.cpu())[:, None]
    a, b = x.chunk(2, -1)
    return torch.cat([a * angle.cos() - b * angle.sin(), a * angle.sin() + b * angle.cos()], -1)


def reference(model, tokens, masks, mix_masks):
    """forward() with torch's autograd in 64 bits on the host: (outputs, parameters)."""
    q = {k: v.detach().cpu().double().requires_grad_(True) for k, v in model.parameters.items()}
    ids = tokens.child.view(torch.int32)[: tokens.child_size].cpu().long()
    offsets = offsets_of(tokens)
    at = torch.from_numpy(np.concatenate([np.arange(b - a) for a, b in zip(offsets[:-1], offsets[1:])]).astype(np.int64))
    e = q["tokens"][ids] + torch.where((at < model.positions)[:, None], q["positions"][at.clamp(max=model.positions - 1)], 0.0)

    def norm(x, name):
        return torch.nn.functional.layer_norm(x, x.shape[-1:], q[name + ".weight"], q[name + ".bias"])

    stream, h = e, norm(e, "norm")
    n, m = model.heads, model.key_heads
    for i in range(model.layers):
        x = (h @ q[f"{i}.heads.weight"].T + q[f"{i}.heads.bias"]).unflatten(1, (n + 2 * m, -1))
        queries, keys, values = turn(x[:, :n], at, model.frequencies), turn(x[:, n:n + m], at, model.frequencies), x[:, n + m:]
        mixed = []
        for a, b in zip(offsets[:-1], offsets[1:]):
            k, v = (y[a:b].repeat_interleave(n // m, 1).transpose(0, 1) for y in (keys, values))
            s = queries[a:b].transpose(0, 1) @ k.transpose(1, 2) / k.shape[-1] ** 0.5
            s = s.masked_fill(torch.ones(s.shape[1:], dtype=torch.bool).triu(1), -float("inf"))
            mixed.append((s.softmax(-1) @ v).transpose(0, 1).flatten(1))
        stream = stream + (torch.cat(mixed) @ q[f"{i}.mix.weight"].T + q[f"{i}.mix.bias"]) * mix_masks[i]
        h = norm(stream, f"{i}.mix_norm")
        u = torch.nn.functional.gelu(h @ q[f"{i}.up.weight"].T + q[f"{i}.up.bias"])
        stream = stream + (u @ q[f"{i}.down.weight"].T + q[f"{i}.down.bias"]) * masks[i]
        h = norm(stream, f"{i}.norm")
    return h @ q["out.weight"].T + q["out.bias"], q


@pytest.mark.parametrize("p", [0.0, 0.25])
def test_gradients_of_the_whole(data, p):
    """As without heads: some thirty sums of up to 288 terms one after the other, each with an error of a few units of 2^-24 of its largest
    terms: 2^-24 * 30 * 16 = 3e-5 of the largest value, and twice that for the way back."""
    tokens, vocabulary_size = data
    model = model_of(vocabulary_size, torch.float32)
    out, kept = model.forward(tokens, p, seed=11)
    grad = torch.randn(out.shape, generator=torch.Generator().manual_seed(2)).cuda()
    grads = model.backward(grad, tokens, kept, p, seed=11)
    assert grads.keys() == model.parameters.keys()
    ones = torch.ones(tokens.child_size, 72, device="cuda")
    masks = [encoder.dropout(ones, p, 11, i).cpu().double() for i in range(2 * model.layers)]
    expected, q = reference(model, tokens, masks[: model.layers], masks[model.layers:])
    assert (out.cpu().double() - expected).abs().max() <= 3e-5 * expected.abs().max()
    expected.backward(grad.cpu().double())
    for name, parameter in q.items():
        error = (grads[name].cpu().double() - parameter.grad).abs().max()
        # (a bias of keys adds the same to all scores of a query: its gradient is what is left of sums that cancel)
        size = parameter.grad.abs().max() if not name.endswith("heads.bias") else max(parameter.grad.abs().max(), q[name.replace("bias", "weight")].grad.abs().max())
        assert error <= 6e-5 * size, (name, error, size)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_a_step_runs_and_is_finite(data, dtype):
    tokens, vocabulary_size = data
    model = model_of(vocabulary_size, dtype)
    codes = torch.randn(vocabulary_size, 17, generator=torch.Generator().manual_seed(1)).to("cuda", dtype)
    target = encoder.embedding(te.next_tokens(tokens), codes)
    for step in range(3):
        assert torch.isfinite(te.train_step(model, tokens, target, rate=1.0, p=0.1, seed=step))
    assert all(torch.isfinite(v).all() for v in model.parameters.values())


def test_another_stream(data):
    tokens, vocabulary_size = data
    model = model_of(vocabulary_size, torch.bfloat16)
    out, kept = model.forward(tokens, 0.1, 4)
    grads = model.backward(out, tokens, kept, 0.1, 4)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        out2, kept2 = model.forward(tokens, 0.1, 4)
        grads2 = model.backward(out2, tokens, kept2, 0.1, 4)
    torch.cuda.current_stream().wait_stream(stream)
    assert torch.equal(out, out2)
    for name in grads:
        assert torch.equal(grads[name], grads2[name]), name


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_captured_step(data, dtype):
    tokens, vocabulary_size = data
    model = model_of(vocabulary_size, dtype)

    def step():
        out, kept = model.forward(tokens, 0.1, 4)
        return out, model.backward(out, tokens, kept, 0.1, 4)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, grads = step()
    for replay in range(4):
        for parameter in model.parameters.values():
            parameter.mul_(0.9)
        graph.replay()
        torch.cuda.synchronize()
        got, got_grads = out.clone(), {name: g.clone() for name, g in grads.items()}
        expected, expected_grads = step()
        torch.cuda.synchronize()
        assert torch.equal(got, expected), replay
        for name in grads:
            assert torch.equal(got_grads[name], expected_grads[name]), (replay, name)


def test_one_text_alone_is_as_among_others(data):
    texts, vocabulary = te.synthetic_text(40, seed=7)
    tokens, vocabulary_size = data
    model = model_of(vocabulary_size, torch.float32)
    out, _ = model.forward(tokens)
    for row in (0, 11, 39):
        one = te.tokenize(texts.slice(row, row + 1), vocabulary)
        begin = int(offsets_of(tokens)[row])
        alone, _ = model.forward(one)
        assert (alone - out[begin : begin + one.child_size]).abs().max() <= 6e-5 * out.abs().max()


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_texts_that_go_on_token_by_token(dtype):
    """Keys and values written into places with room, one token of every text a step, its position and the number of its keys read on the
    device: what each token gets is what it gets when the whole texts are there, causal.  Both are off from it by as much as rounding allows:
    half a step of the result and of the exponentials of its type each, of sums of weights of 1 times values of up to 4."""
    heads, key_heads, width, room = 8, 2, 64, 700
    lengths = [3, 260, 650, 1, 90]
    steps = 12
    gen = torch.Generator(device="cuda").manual_seed(3)
    offsets = np.concatenate([[0], np.cumsum([n + steps for n in lengths])]).astype(np.int32)
    x = torch.randn(int(offsets[-1]), heads + 2 * key_heads, width, generator=gen, device="cuda").clamp(-4, 4).to(dtype)
    f = encoder.rotary_frequencies(width)
    rows = torch.from_numpy(offsets).cuda()
    turned = encoder.rotary(x[:, : heads + key_heads], rows, f)
    whole = encoder.attention(turned[:, :heads], turned[:, heads:], x[:, heads + key_heads:], rows, causal=True)

    texts = len(lengths)
    keys, values = (torch.full((texts * room, key_heads, width), float("nan"), dtype=dtype, device="cuda") for _ in range(2))
    key_rows = torch.arange(0, (texts + 1) * room, room, dtype=torch.int32, device="cuda")
    for r, n in enumerate(lengths):  # the prompts
        keys[r * room : r * room + n] = turned[offsets[r] : offsets[r] + n, heads:]
        values[r * room : r * room + n] = x[offsets[r] : offsets[r] + n, heads + key_heads:]
    count = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    single = torch.arange(texts + 1, dtype=torch.int32, device="cuda")
    unit = {torch.float32: 2.0**-24, torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}[dtype]
    most = 2 * (2 * unit * 4 + 800 * 2.0**-24 * 4 + 2.0**-18 * 8)
    for step in range(steps):
        at = torch.from_numpy(offsets[:-1]).cuda().long() + count
        token = x[at].contiguous()
        encoder.rotary(token[:, : heads + key_heads], single, f, starts=count, out=token[:, : heads + key_heads])
        place = key_rows[:-1].long() + count
        keys[place], values[place] = token[:, heads : heads + key_heads], token[:, heads + key_heads:]
        count = count + 1
        out = encoder.attention(token[:, :heads], keys, values, single, key_rows, count, causal=True)
        assert torch.equal(token[:, :heads], turned[at, :heads])
        assert (out.double() - whole[at].double()).abs().max() <= most, step


def test_refusals_of_heads():
    for heads, key_heads in ((5, 0), (24, 0), (6, 4)):
        with pytest.raises(ValueError, match="heads must divide"):
            model_of(10, torch.float32, heads=heads, key_heads=key_heads)


def test_cpp_api():
    exe = os.path.join(os.path.dirname(os.path.abspath(__file__)), "cpp", "attention_api_test")
    assert os.path.exists(exe), "build it with __graft_entry__.build() or make -C tests/cpp"
    run = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert run.returncode == 0 and "ALL PASSED" in run.stdout, run.stdout + run.stderr
