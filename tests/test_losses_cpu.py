"""Refusals of the post-training operators: shapes, types and arguments are checked on the host before
anything is launched (and before the device is), so a wrong call is told apart from a tensor on the wrong device."""
import pytest
import torch

native = pytest.importorskip("llmt.ops.native")
if not native.available():
    pytest.skip("extension not built", allow_module_level=True)
from llmt.ops import losses  # noqa: E402


def args(B=2, T=3, V=8):
    return torch.zeros(B, T, V), torch.zeros(B, T, dtype=torch.long), torch.zeros(B, T), torch.zeros(B, T)


@pytest.mark.parametrize("change,match", [
    (lambda a: {"logits": a["logits"][0]}, "logits must be"),
    (lambda a: {"logits": a["logits"].double()}, "dtype"),
    (lambda a: {"logits": torch.zeros(2, 8, 3).transpose(1, 2)}, "unit stride"),
    (lambda a: {"logits": torch.zeros(2, 0, 8), "targets": torch.zeros(2, 0, dtype=torch.long)}, "empty batch"),
    (lambda a: {"targets": a["targets"].int()}, "dtype"),
    (lambda a: {"targets": a["targets"][:1]}, "targets must be"),
    (lambda a: {"old_logp": a["old_logp"].half()}, "dtype"),
    (lambda a: {"old_logp": torch.zeros(2, 4)}, "tokens"),
    (lambda a: {"old_logp": a["old_logp"].clone().requires_grad_()}, "detach"),
    (lambda a: {"advantages": torch.zeros(3, 1)}, "sequences"),
    (lambda a: {"ref_logp": torch.zeros(2, 3, 1)}, "ref_logp must be"),
    (lambda a: {"mask": torch.ones(2, 3)}, "dtype"),
    (lambda a: {"clip": (1.5, 0.2)}, "clip"),
    (lambda a: {"clip": (0.2, float("nan"))}, "clip"),
    (lambda a: {"out": torch.zeros(2, 3, 9)}, "out must match"),
    (lambda a: {"out": a["logits"], "grad": False}, "out without grad"),
    (lambda a: {"kl_coef": 0.1}, "kl_coef without"),
    (lambda a: {"out": torch.zeros(2, 3, 8, dtype=torch.half)}, "out must match"),
    (lambda a: {}, "CUDA tensor"),
])
def test_policy_refusals(change, match):
    z, y, old, adv = args()
    a = {"logits": z, "targets": y, "old_logp": old, "advantages": adv}
    a.update(change(a))
    with pytest.raises(RuntimeError, match=match):
        losses.policy_loss_rows(**a)


def test_preference_refusals():
    z, y, old, _ = args(B=3)
    with pytest.raises(RuntimeError, match="rejected"):
        losses.preference_loss_rows(z, y)
    z, y, old, _ = args()
    for kw, match in (({"beta": 0.0}, "beta"), ({"label_smoothing": 0.5}, "label_smoothing"),
                      ({"label_smoothing": 0.1, "kind": "ipo"}, "sigmoid"), ({"ref_logp": old.requires_grad_()}, "detach"),
                      ({}, "CUDA tensor")):
        with pytest.raises(RuntimeError, match=match):
            losses.preference_loss_rows(z, y, **kw)
    with pytest.raises(ValueError, match="kind must be one of"):
        losses.preference_loss_rows(z, y, kind="cube")
    with pytest.raises(ValueError, match="reduction must be one of"):
        losses.policy_loss_rows(z, y, None, old.detach(), reduction="mean")


def test_token_form_refusals():
    _, y, lp, adv = args()
    for bad, match in ((lp.half(), "dtype"), (lp[0], "logp must be"), (lp, "CUDA tensor")):
        with pytest.raises(RuntimeError, match=match):
            losses.policy_loss_tokens(bad, y, 8, None, adv)
        with pytest.raises(RuntimeError, match=match):
            losses.preference_loss_tokens(bad, y, 8)
