"""Tensors whose storage was freed (as wrappers that shard parameters do between steps) have no memory to step on."""
import pytest
import torch

from llmt.ops import native

if not native.available():
    pytest.skip("extension not built", allow_module_level=True)
from llmt.optim.multi import MultiAdamW  # noqa: E402


@pytest.mark.parametrize("which", ["parameter", "gradient", "bf16 copy"])
def test_a_freed_tensor_is_refused(which):
    p, s, g = [torch.zeros(8), torch.zeros(8)], [torch.zeros(8, dtype=torch.bfloat16) for _ in range(2)], [torch.ones(8), torch.ones(8)]
    opt = MultiAdamW(p, s)
    {"parameter": p, "gradient": g, "bf16 copy": s}[which][1].untyped_storage().resize_(0)
    with pytest.raises(RuntimeError, match="tensor 1 has no memory"):
        opt.step(g)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        opt.step([g[0], None])
