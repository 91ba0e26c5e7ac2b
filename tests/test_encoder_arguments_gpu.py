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
