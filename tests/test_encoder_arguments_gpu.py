"""What the encoder's operators say to arguments that do not fit."""
import pytest
import torch

from cudf_amd import encoder

pytestmark = pytest.mark.gpu


def test_unevenly_spaced_rows_are_a_value_error():
    """As every other argument that does not fit; still what torch raises as well."""
    x = torch.randn(3, 4, 5, 16, device="cuda").transpose(0, 1)
    w = torch.randn(16, 16, device="cuda")
    b = torch.ones(16, device="cuda")
    for call in (lambda: encoder.dropout(x, 0.1, 1), lambda: encoder.linear(x, w), lambda: encoder.layer_norm(x, b, b),
                 lambda: encoder.layer_norm(x.contiguous(), b, b, residual=x), lambda: encoder.linear_backward(x, x.contiguous(), w)):
        with pytest.raises(ValueError, match="evenly spaced"):
            call()
        with pytest.raises(RuntimeError):
            call()


def test_as_many_rows_in_another_shape_are_refused():
    """[4, 3] rows beside [3, 4]: as many, but not the same."""
    x, other = torch.randn(3, 4, 16, device="cuda"), torch.randn(4, 3, 16, device="cuda")
    w, b = torch.randn(16, 16, device="cuda"), torch.ones(16, device="cuda")
    _, saved = encoder.layer_norm(x, b, b, keep=True)
    _, z = encoder.linear(x, w, keep=True)
    for call in (lambda r: encoder.layer_norm(x, b, b, residual=r), lambda r: encoder.linear(x, w, residual=r), lambda r: encoder.linear_backward(r, x, w, "relu", z),
                 lambda r: encoder.linear_backward(x, x, w, "relu", r), lambda r: encoder.layer_norm_backward(r, saved, b), lambda r: encoder.layer_norm_backward(x, saved, b, sum_grad=r),
                 lambda r: encoder.layer_norm_backward(x, saved._replace(sum=r), b)):
        with pytest.raises(ValueError, match="must be of shape"):
            call(other)
        with pytest.raises(ValueError):
            call(x[:, :3])
        call(x)
        call(x.view(12, 16))  # the rows alone


def test_rows_of_one_in_any_number_of_dimensions():
    x = torch.randn(1, 1, 16, device="cuda")
    w, b = torch.randn(16, 16, device="cuda"), torch.ones(16, device="cuda")
    want = encoder.linear(x, w, b, residual=x)
    assert torch.equal(encoder.linear(x, w, b, residual=x[0]), want) and torch.equal(encoder.linear(x, w, b, residual=x[0, 0]), want)
    assert torch.equal(encoder.linear(x[0, 0], w, b, residual=x), want[0, 0])
