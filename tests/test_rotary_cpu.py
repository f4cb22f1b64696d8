"""Rotary plans on the host: scalings against their definitions, and refusals."""
import math

import pytest
import torch

from llmt.ops import native
from llmt.ops.rotary import Rotary, frequencies


def test_frequencies():
    w, f = frequencies(128, 10000.0)
    assert f == 1.0 and w.dtype == torch.float64
    assert torch.allclose(w, torch.tensor([10000.0 ** (-j / 64) for j in range(64)], dtype=torch.float64), rtol=1e-14)
    assert torch.allclose(frequencies(128, 1e4, {"type": "linear", "factor": 4})[0], w / 4, rtol=1e-15)
    n = frequencies(128, 1e4, {"type": "ntk", "factor": 8.0})[0]
    assert n[0] == 1.0 and abs(n[-1] / w[-1] * 8 - 1) < 1e-12  # the fastest kept, the slowest stretched by 8
    L = {"type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0, "original_max_position": 8192}
    s = frequencies(128, 5e5, L)[0]
    w5 = frequencies(128, 5e5)[0]
    turns = 8192 * w5 / (2 * math.pi)
    assert torch.equal(s[turns > 4], w5[turns > 4]) and torch.allclose(s[turns < 1], w5[turns < 1] / 8, rtol=1e-15)
    mid = (turns > 1) & (turns < 4)
    t = (turns[mid] - 1) / 3
    assert mid.any() and torch.allclose(s[mid], w5[mid] * t + w5[mid] / 8 * (1 - t), rtol=1e-12)
    y, f = frequencies(128, 1e4, {"type": "yarn", "factor": 16.0, "original_max_position": 4096})
    assert abs(f - (0.1 * math.log(16) + 1)) < 1e-15
    assert y[0] == w[0] and torch.allclose(y[-1:], w[-1:] / 16, rtol=1e-15) and (y <= w).all() and (y >= w / 16 * (1 - 1e-12)).all()
    assert frequencies(64, 1e4, {"type": "yarn", "factor": 2.0, "original_max_position": 64, "attention_factor": 1.5})[1] == 1.5


def test_table_digits_make_every_position():
    """The product of the three digits' rotations is the position's, to the table's fp32."""
    rot = Rotary(64, rotary_dim=32, scaling={"type": "yarn", "factor": 4.0, "original_max_position": 2048}, device="cpu")
    t = torch.view_as_complex(rot.table.double())
    for p in (0, 1, 1023, 1024, 2 ** 20 - 1, 2 ** 20, 123456789, 2 ** 31 - 1):
        z = t[p & 1023] * t[1024 + (p >> 10 & 1023)] * t[2048 + (p >> 20)]
        a = rot.inv_freq * p
        want = torch.polar(torch.full_like(a, rot.factor), a)
        # three values of size up to 1.14, half a step of fp32 off in both parts, and on both sides angles
        # up to 2^31 in fp64 (2^-23 each)
        assert (z - want).abs().max() < 3 * 2.0 ** -23 + 2.0 ** -22
    cos, sin = rot.tables(50)
    assert cos.shape == (50, 32) and torch.equal(cos[:, :16], cos[:, 16:])
    assert torch.allclose(cos[7, :16].double(), (rot.inv_freq * 7).cos() * rot.factor, atol=1e-7)


@pytest.mark.parametrize("kw,match", [
    ({"head_dim": 64, "rotary_dim": 66}, "rotary_dim"), ({"head_dim": 64, "rotary_dim": 31}, "even"),
    ({"head_dim": 64, "rotary_dim": 0}, "rotary_dim"), ({"head_dim": 64, "base": 0.0}, "base"),
    ({"head_dim": 64, "scaling": {"type": "cubic"}}, "scaling type"), ({"head_dim": 64, "scaling": {"type": "linear"}}, "takes"),
    ({"head_dim": 64, "scaling": {"type": "linear", "factor": -1.0}}, "positive"),
    ({"head_dim": 64, "scaling": {"type": "ntk", "factor": 2.0, "more": 1}}, "takes"),
    ({"head_dim": 2, "scaling": {"type": "ntk", "factor": 2.0}}, "above 2"),
    ({"head_dim": 64, "scaling": {"type": "llama3", "factor": 8.0, "low_freq_factor": 4.0, "high_freq_factor": 1.0,
                                  "original_max_position": 8192}}, "below"),
])
def test_plan_refusals(kw, match):
    with pytest.raises(ValueError, match=match):
        Rotary(device="cpu", **kw)


@pytest.mark.skipif(not native.available(), reason="extension not built")
def test_call_refusals():
    rot = Rotary(64, device="cpu")
    q = torch.zeros(2, 3, 4, 64)
    pos = torch.zeros(2, 3, dtype=torch.long)
    with pytest.raises(ValueError, match="head_dim"):
        rot.rotate(torch.zeros(2, 3, 4, 32))
    for a, kw, match in [
        ((q[0],), {}, "q must be"), ((q.double(),), {}, "dtype"), ((q, q[:1]), {}, "k must be"), ((q, q.half()), {}, "share a dtype"),
        ((torch.zeros(2, 3, 4, 128)[..., ::2],), {}, "unit stride"),
        ((q, None, pos.float()), {}, "int32 or int64"), ((q, None, pos[:, :2]), {}, "positions must be"),
        ((q, None, pos[:, :1]), {}, "one position"), ((q, None, pos[None]), {}, "positions must be"),
        ((q, None, pos), {"k_out": q}, "k_out without k"),
        ((q, q.clone(), pos), {"q_out": None, "k_out": q}, "k_out is q"), ((q, None, pos), {}, "CUDA tensor"),
    ]:
        with pytest.raises(RuntimeError, match=match):
            rot.rotate(*a, **kw)
