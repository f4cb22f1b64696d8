"""Refusals of MultiAdamW (host checks)."""
import pytest
import torch

from llmt.ops import native

if not native.available():
    pytest.skip("extension not built", allow_module_level=True)
from llmt.optim.multi import MultiAdamW  # noqa: E402


def test_construction_refusals():
    p = [torch.zeros(10), torch.zeros(4, 4)]
    for params, kw, match in [
        ([], {}, "no tensors"), ([p[0].half()], {}, "dtype"), ([torch.zeros(4, 4).t()[:, :2]], {}, "contiguous"),
        ([torch.zeros(0)], {}, "empty"), (p, {"weight_decay": [0.1]}, "weight decay"), (p, {"shadows": [torch.zeros(10)]}, "bf16 copy"),
        (p, {"shadows": [torch.zeros(10), torch.zeros(4, 4)]}, "bf16 copy"),
        ([p[0], p[0]], {}, "share memory"), ([p[0][:6], p[0][5:]], {}, "share memory"),
    ]:
        with pytest.raises((RuntimeError, IndexError), match=match):
            MultiAdamW(params, **kw)
    for kw, match in [({"state_bits": 4}, "state_bits"), ({"betas": (0.9, 1.0)}, "betas")]:
        with pytest.raises(ValueError, match=match):
            MultiAdamW(p, **kw)


def test_step_refusals():
    p = [torch.zeros(10), torch.zeros(4, 4)]
    opt = MultiAdamW(p)
    with pytest.raises(ValueError, match="no gradients"):
        opt.step()
    for g, match in [
        ([p[0]], "1 gradients for 2"), ([p[0], 3.0], "not a tensor"), ([p[0].half(), p[1].half()], "dtype"),
        ([p[0], p[1].bfloat16()], "two dtypes"), ([p[0][:9], p[1]], "10 values"), ([p[0], p[1].repeat(1, 2)[:, ::2]], "contiguous"),
        ([p[0], p[1]], "CUDA tensor"),
    ]:
        with pytest.raises(RuntimeError, match=match):
            opt.step(g)
    same = [torch.ones(4), torch.ones(4)]
    with pytest.raises(RuntimeError, match="one gradient for two"):
        MultiAdamW(same, zero_grad=True).step([same[0], same[0]])
    with pytest.raises(ValueError, match="dtype must be"):
        opt.state_values(torch.float16)
    assert MultiAdamW(p, state_bits=32).state_values()[0].dtype == torch.float32  # not decoded


def test_gradients_that_overlap_in_part_are_not_cleared():
    p, g = [torch.zeros(4), torch.zeros(4)], torch.ones(9)
    with pytest.raises(RuntimeError, match="one gradient for two"):
        MultiAdamW(p, zero_grad=True).step([g[2:6], g[5:9]])
    with pytest.raises(RuntimeError, match="CUDA tensor"):  # side by side: refused for the device alone
        MultiAdamW(p, zero_grad=True).step([g[4:8], g[:4]])


def test_layout():
    opt = MultiAdamW([torch.zeros(1), torch.zeros(256), torch.zeros(257), torch.zeros(3)])
    assert opt.plan.blocks == 5 and list(opt.plan.first_block) == [0, 1, 2, 4]
    assert opt.exp_avg.dtype == torch.float8_e4m3fn and opt.exp_avg.numel() == 5 * 256 and opt.exp_avg_scale.numel() == 5
