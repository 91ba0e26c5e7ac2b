"""The encoder's operators together: the example's model against the formulas in 64 bits, its training, on another stream, and
captured in a graph."""
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
    texts, vocabulary = te.synthetic_text(60, seed=3)
    return te.tokenize(texts, vocabulary), vocabulary.size


def model_of(vocabulary_size, dtype, width=72, layers=2, outputs=17):
    return te.TextEncoder(vocabulary_size, positions=24, width=width, layers=layers, outputs=outputs, dtype=dtype, seed=5)


def places(tokens):
    offsets = tokens.offsets.view(torch.int32)[: tokens.size + 1].cpu().numpy()
    return np.concatenate([np.arange(b - a) for a, b in zip(offsets[:-1], offsets[1:])]).astype(np.int64)


def reference(model, tokens, masks):
    """forward() with torch's autograd in 64 bits on the host: (outputs, parameters)."""
    q = {k: v.detach().cpu().double().requires_grad_(True) for k, v in model.parameters.items()}
    ids = tokens.child.view(torch.int32)[: tokens.child_size].cpu().long()
    at = torch.from_numpy(places(tokens))
    e = q["tokens"][ids] + torch.where((at < model.positions)[:, None], q["positions"][at.clamp(max=model.positions - 1)], 0.0)

    def norm(x, name):
        return torch.nn.functional.layer_norm(x, x.shape[-1:], q[name + ".weight"], q[name + ".bias"])

    stream, h = e, norm(e, "norm")
    for i in range(model.layers):
        u = torch.nn.functional.gelu(h @ q[f"{i}.up.weight"].T + q[f"{i}.up.bias"])
        v = u @ q[f"{i}.down.weight"].T + q[f"{i}.down.bias"]
        stream = stream + v * masks[i]
        h = norm(stream, f"{i}.norm")
    return h @ q["out.weight"].T + q["out.bias"], q


@pytest.mark.parametrize("p", [0.0, 0.25])
def test_gradients_of_the_whole(data, p):
    """Some twenty sums of up to 288 terms one after the other, each with an error of a few units of 2^-24 of its largest terms:
    2^-24 * 20 * 16 = 2e-5 of the largest value, and twice that for the way back."""
    tokens, vocabulary_size = data
    model = model_of(vocabulary_size, torch.float32)
    out, kept = model.forward(tokens, p, seed=11)
    grad = torch.randn(out.shape, generator=torch.Generator().manual_seed(2)).cuda()
    grads = model.backward(grad, tokens, kept, p, seed=11)
    ones = torch.ones(tokens.child_size, 72, device="cuda")
    masks = [encoder.dropout(ones, p, 11, i).cpu().double() for i in range(model.layers)]
    expected, q = reference(model, tokens, masks)
    assert (out.cpu().double() - expected).abs().max() <= 2e-5 * expected.abs().max()
    expected.backward(grad.cpu().double())
    for name, parameter in q.items():
        error = (grads[name].cpu().double() - parameter.grad).abs().max()
        assert error <= 4e-5 * parameter.grad.abs().max(), (name, error)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_training_lowers_the_loss(data, dtype):
    tokens, vocabulary_size = data
    model = model_of(vocabulary_size, dtype)
    codes = torch.randn(vocabulary_size, 17, generator=torch.Generator().manual_seed(1)).to("cuda", dtype)
    target = encoder.embedding(te.next_tokens(tokens), codes)
    losses = [te.train_step(model, tokens, target, rate=2.0, p=0.1, seed=step).item() for step in range(30)]
    assert all(np.isfinite(losses)) and losses[-1] < 0.8 * losses[0]


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
    """A graph of both directions, replayed with other parameters each time, gives what the calls give."""
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
    """The form for serving: what a text gives does not depend on the others, up to the order in which products are added."""
    texts, vocabulary = te.synthetic_text(60, seed=3)
    tokens, vocabulary_size = data
    model = model_of(vocabulary_size, torch.float32)
    out, _ = model.forward(tokens)
    for row in (0, 7, 59):
        one = te.tokenize(texts.slice(row, row + 1), vocabulary)
        begin = int(tokens.offsets.view(torch.int32)[row])
        alone, _ = model.forward(one)
        assert (alone - out[begin : begin + one.child_size]).abs().max() <= 4e-5 * out.abs().max()


def test_cpp_api():
    exe = os.path.join(os.path.dirname(os.path.abspath(__file__)), "cpp", "encoder_api_test")
    assert os.path.exists(exe), "build it with __graft_entry__.build() or make -C tests/cpp"
    run = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert run.returncode == 0 and "ALL PASSED" in run.stdout, run.stdout + run.stderr
