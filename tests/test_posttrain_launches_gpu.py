"""The launch counter against the kernels that the profiler sees, for the post-training operators."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def launches(fn):
    """(kernels of this library on the device, kernels counted) of one call."""
    from torch.profiler import ProfilerActivity, profile
    from llmt.ops.native import LAUNCHES
    fn()
    torch.cuda.synchronize()
    before = LAUNCHES.count
    with profile(activities=[ProfilerActivity.CUDA], acc_events=True) as prof:
        fn()
        torch.cuda.synchronize()
    counted = LAUNCHES.count - before
    return sum(e.device_type == torch.autograd.DeviceType.CUDA and "llmt::" in e.name for e in prof.events()), counted


@pytest.mark.parametrize("T", [4, 300])
@pytest.mark.parametrize("grad", [False, True])
def test_losses(T, grad):
    from llmt.ops import losses as L
    z, y, adv = torch.randn(2, T, 100, device="cuda"), torch.randint(0, 100, (2, T), device="cuda"), torch.randn(2, T, device="cuda")
    lp = L.logprob_rows(z, y)
    calls = [lambda: L.logprob_rows(z, y), lambda: L.preference_loss_rows(z, y, grad=grad),
             lambda: L.policy_loss_tokens(lp, y, 100, None, adv), lambda: L.preference_loss_tokens(lp, y, 100)]
    calls += [lambda r=r: L.policy_loss_rows(z, y, None, adv, reduction=r, grad=grad) for r in L.REDUCTIONS]
    leaf = z.clone().requires_grad_()
    calls += [lambda: L.policy_loss(leaf, y, None, adv).loss.backward(), lambda: L.preference_loss(leaf, y).loss.backward()]
    for i, f in enumerate(calls):
        seen, counted = launches(f)
        assert seen == counted > 0, (i, seen, counted)


@pytest.mark.parametrize("n", [3, 641, 1500])
def test_adamw_over_many_tensors(n):
    from llmt.optim.multi import MultiAdamW
    p = list(torch.zeros(n, 10, device="cuda").unbind())
    opt = MultiAdamW(p)
    seen, counted = launches(lambda: opt.step([torch.ones_like(x) for x in p]))
    assert seen == counted > 0, (seen, counted)
    assert launches(lambda: opt.step([None] * n))[1] == 0


def test_rotary():
    from llmt.ops.rotary import Rotary
    rot = Rotary(64)
    q = torch.randn(2, 5, 4, 64, device="cuda")
    assert launches(lambda: rot.rotate(q, q[:, :, :2])) == (1, 1)
