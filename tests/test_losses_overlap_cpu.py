"""An `out` of the losses over the ids, the mask or a token's numbers would be written while other rows still read them."""
import pytest
import torch

native = pytest.importorskip("llmt.ops.native")
if not native.available():
    pytest.skip("extension not built", allow_module_level=True)
from llmt.ops import losses  # noqa: E402


@pytest.mark.parametrize("name", ["targets", "mask", "old_logp", "advantages", "ref_logp"])
@pytest.mark.parametrize("loss", ["policy", "preference"])
def test_out_over_an_operand(loss, name):
    if loss == "preference" and name in ("old_logp", "advantages"):
        pytest.skip("not an operand of this loss")
    buf = torch.zeros(200)
    out = buf[:64].view(2, 4, 8)
    a = {"targets": torch.zeros(2, 4, dtype=torch.long), "mask": torch.ones(2, 4, dtype=torch.bool), "ref_logp": torch.zeros(2, 4)}
    if loss == "policy":
        a.update(old_logp=torch.zeros(2, 4), advantages=torch.zeros(2, 1))

    def at(k):  # the operand from the k-th float of the buffer on, transposed
        t = a[name]
        return buf.view(torch.uint8)[4 * k:].view(t.dtype)[:t.numel()].view(t.t().shape).t()
    call = losses.policy_loss_rows if loss == "policy" else losses.preference_loss_rows
    for k, match in ((62, f"out overlaps {name}"), (64, "CUDA tensor")):
        with pytest.raises(RuntimeError, match=match):
            call(torch.zeros(2, 4, 8), **{**a, name: at(k)}, out=out)


def test_operands_beside_rows_of_out():
    """Columns that the rows of out leave free may hold an operand."""
    wide = torch.zeros(2, 4, 12)
    for at, match in ((slice(8, 9), "CUDA tensor"), (slice(7, 8), "out overlaps advantages")):
        with pytest.raises(RuntimeError, match=match):
            losses.policy_loss_rows(torch.zeros(2, 4, 8), torch.zeros(2, 4, dtype=torch.long), None, wide[..., at][..., 0], out=wide[..., :8])
