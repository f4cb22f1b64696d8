"""Model options of the post-training operators on the CPU: the plain model's rotary layouts against the rotation
written out, tables, and refusals."""
import pytest
import torch

from llmt.config import get_config
from llmt.models.llama import build_model, make_batch, model_rope_tables, rope_tables, rotate_heads


def _by_hand(x, angle, rd, interleaved, factor=1.0):
    """Pair by pair, in fp64; x (..., T, hd), angle (T, rd / 2)."""
    y = x.double().clone()
    for j in range(rd // 2):
        a, b = (2 * j, 2 * j + 1) if interleaved else (j, j + rd // 2)
        c, s = angle[:, j].cos() * factor, angle[:, j].sin() * factor
        y[..., a] = x[..., a].double() * c - x[..., b].double() * s
        y[..., b] = x[..., b].double() * c + x[..., a].double() * s
    return y


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("rd", [None, 32, 10])
def test_rotate_heads(rd, interleaved):
    from llmt.ops.rotary import frequencies
    cfg = get_config("tiny256", rotary_dim=rd, rope_interleaved=interleaved, rope_scaling={"type": "linear", "factor": 2.0})
    cos, sin = model_rope_tables(cfg, 20, "cpu")
    x = torch.randn(2, 3, 20, cfg.hd)
    n = rd or cfg.hd
    w, _ = frequencies(n, cfg.rope_base, cfg.rope_scaling)
    want = _by_hand(x, torch.arange(20).double()[:, None] * w, n, interleaved)
    # a table value is half a step of fp32 off, the rotation three roundings of values below 6
    assert (rotate_heads(cfg, x, cos, sin).double() - want).abs().max() < 6 * 6 * 2.0 ** -24


def test_plain_models_are_unchanged():
    cfg = get_config("tiny256")
    for a, b in zip(model_rope_tables(cfg, 64, "cpu"), rope_tables(64, cfg.hd, cfg.rope_base, "cpu")):
        assert torch.equal(a, b)
    assert cfg.plain_rope and get_config("tiny256", rotary_dim=64).plain_rope
    assert not get_config("tiny256", rotary_dim=32).plain_rope and not get_config("tiny256", rope_interleaved=True).plain_rope


def test_scaled_model_trains_on_cpu():
    cfg = get_config("tiny256", vocab=128, L=1, rope_interleaved=True, rotary_dim=32,
                     rope_scaling={"type": "yarn", "factor": 4.0, "original_max_position": 16})
    m = build_model(cfg, 24)
    idx, tgt = make_batch(2, 24, cfg.vocab, "cpu")
    m(idx, tgt).backward()
    assert all(torch.isfinite(p.grad).all() for p in m.parameters())


def test_refusals():
    from llmt.parallel.pp import StageModel
    from llmt.parallel.tp import local_config
    from llmt.train import Trainer
    cfg = get_config("tiny256", rope_interleaved=True)
    with pytest.raises(ValueError, match="single-GPU"):
        local_config(cfg, 2)
    with pytest.raises(ValueError, match="single-GPU"):
        StageModel(cfg, 16, 0, 1, True, False)
    with pytest.raises(ValueError, match="adamw or adamw8"):
        Trainer(get_config("tiny256"), 2, 16, device="cpu", optimizer="sgd")
    with pytest.raises(ValueError, match="single-GPU"):
        Trainer(get_config("tiny256"), 2, 16, device="cpu", optimizer="adamw8", dp=object())
    with pytest.raises(ValueError, match="scaling type"):
        build_model(get_config("tiny256", vocab=64, L=1, rope_scaling={"type": "other"}), 16)
    # scaling alone goes through the tables of every layout
    assert local_config(get_config("tiny256", rope_scaling={"type": "linear", "factor": 2.0}), 2).rope_scaling["factor"] == 2.0
