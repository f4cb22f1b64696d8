"""An eps below zero (or NaN) would divide by it where a second moment is small."""
import pytest
import torch

from llmt.ops import native

if not native.available():
    pytest.skip("extension not built", allow_module_level=True)
from llmt.optim.multi import MultiAdamW  # noqa: E402


@pytest.mark.parametrize("eps", [-1e-8, float("nan")])
def test_eps_below_zero_is_refused(eps):
    with pytest.raises(ValueError, match="eps must be"):
        MultiAdamW([torch.zeros(4)], eps=eps)
    MultiAdamW([torch.zeros(4)], eps=0.0)
