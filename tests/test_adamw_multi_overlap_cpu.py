"""Gradients of MultiAdamW that lie over the parameters or their bf16 copies: another warp would read what one has
already updated."""
import pytest
import torch

from llmt.ops import native

if not native.available():
    pytest.skip("extension not built", allow_module_level=True)
from llmt.optim.multi import MultiAdamW  # noqa: E402


def refusal(opt, grads):
    with pytest.raises(RuntimeError) as e:
        opt.step(grads)
    return str(e.value)


def test_gradients_over_parameters_and_copies():
    buf, half = torch.zeros(100), torch.zeros(100, dtype=torch.bfloat16)
    p = [buf[10:20], buf[40:60].view(4, 5), buf[30:35]]
    s = [half[10:20], half[40:60], half[30:35]]
    g = [torch.ones(10), torch.ones(20), torch.ones(5)]
    for opt in (MultiAdamW(p), MultiAdamW(p, s), MultiAdamW(p, s, zero_grad=True)):
        assert "CUDA tensor" in refusal(opt, g)
        assert "CUDA tensor" in refusal(opt, [buf[20:30], buf[60:80], buf[35:40]])  # side by side
        assert "gradient 0 overlaps" in refusal(opt, [buf[11:21], g[1], g[2]])
        assert "gradient 2 overlaps" in refusal(opt, [g[0], g[1], buf[36:41]])
        assert "gradient 2 overlaps" in refusal(opt, [None, None, buf[8:13]])
        assert "gradient 0 overlaps" in refusal(opt, [buf[40:50], None, None])  # another parameter's, from its first value
    opt = MultiAdamW(p, s)
    h = [x.bfloat16() for x in g]
    assert "CUDA tensor" in refusal(opt, h)
    assert "gradient 1 overlaps" in refusal(opt, [h[0], half[59:79], h[2]])


def test_a_parameter_as_its_own_gradient():
    """Each value is read and written by one thread; cleared after its update it would be lost."""
    p = [torch.zeros(10), torch.zeros(4)]
    assert "CUDA tensor" in refusal(MultiAdamW(p), p)
    assert "overlaps" in refusal(MultiAdamW(p, zero_grad=True), p)


def test_parameters_that_moved():
    """The addresses of the call count, also where their order changed since the optimizer was made."""
    a, b = torch.zeros(64), torch.zeros(64)
    opt = MultiAdamW([a, b])
    sa, sb = a.untyped_storage(), b.untyped_storage()
    first = [sa.data_ptr(), sb.data_ptr()]
    sa.resize_(0)
    sb.resize_(0)
    sb.resize_(256)
    sa.resize_(256)
    g = torch.ones(64)
    assert "CUDA tensor" in refusal(opt, [g, torch.ones(64)])
    assert "gradient 0 overlaps" in refusal(opt, [b, g]), first
    assert "gradient 1 overlaps" in refusal(opt, [g, a])
