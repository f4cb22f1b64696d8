"""The update of AdamW over many tensors where its factors lose digits: bias corrections of betas near 1, and second
moments below fp32's normal range."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("betas", [(0.9, 0.999), (0.95, 0.9999), (0.9999, 0.99999), (0.0, 0.0)])
def test_bias_corrections(betas, bits):
    """Updates from zero parameters against fp64: m and v are three fp32 roundings off, the corrections 1 - b^t three (b's
    logarithm and its multiple are fp64), square root, quotient and products six: under 2^-20 of an update. Steps
    start from the states the kernel holds, so that their rounding does not enter."""
    from llmt.optim.multi import MultiAdamW
    gen = torch.Generator(device="cuda").manual_seed(0)
    lr, eps = 0.5, 1e-12
    for first in (0, 1, 9, 999, 100000):
        p = [torch.zeros(700, device="cuda")]
        opt = MultiAdamW(p, lr=lr, betas=betas, eps=eps, weight_decay=0.0, state_bits=bits)
        opt.step_t.fill_(first)
        for t in (first + 1, first + 2):
            g = (torch.randn(700, device="cuda", generator=gen) + 3.0) * 1e-3
            m, v = (x.double() for x in opt.param_states()[0])
            p[0].zero_()
            opt.step([g])
            m = betas[0] * m + (1 - betas[0]) * g.double()
            v = betas[1] * v + (1 - betas[1]) * g.double() ** 2
            want = -lr / (1 - betas[0] ** t) * m / ((v / (1 - betas[1] ** t)).sqrt() + eps)
            assert ((p[0].double() - want).abs() <= 2.0 ** -20 * want.abs()).all(), ((p[0].double() / want - 1).abs().max().item(), t)


@pytest.mark.parametrize("bits", [8, 32])
def test_second_moments_below_the_normal_range(bits):
    """Gradients of 1e-20: v = 5e-42 is 3568 units of 2^-149, held to half a unit, its root to 7.1e-5 of itself. With eps far
    below the root the update is lr."""
    from llmt.optim.multi import MultiAdamW
    for n in (300, 256):  # a ragged block beside a whole one
        p = [torch.zeros(n, device="cuda")]
        opt = MultiAdamW(p, lr=0.5, eps=1e-30, weight_decay=0.0, state_bits=bits)
        opt.step([torch.full((n,), 1e-20, device="cuda")])
        assert ((p[0] + 0.5).abs() <= 0.5 * 1e-4).all(), p[0][:3]
