"""The losses over logits rows at values where digits are lost: NaN advantages, logits with a large common
offset, tokens that are almost certain, and the mean error of many log-probabilities."""
import pytest
import torch

from tests.test_losses_gpu import L, check_gradient, counted, make, oracle_logp, policy_oracle  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kl", [0.0, 0.1])
@pytest.mark.parametrize("form", ["rows", "tokens"])
def test_a_nan_advantage_has_a_nan_gradient_in_its_row_alone(L, form, kl):  # noqa: F811
    z, y, _, old, ref, adv = make(2, 5, 300, "fp32", mask=None)
    adv[1, 2] = float("nan")
    bad = adv.isnan()
    if form == "rows":
        r = L.policy_loss_rows(z, y, old, adv, ref_logp=ref, kl_coef=kl)
        loss, grad = r.loss, r.dlogits
    else:
        leaf = L.logprob_rows(z, y).requires_grad_()
        loss = L.policy_loss_tokens(leaf, y, 300, old, adv, ref_logp=ref, kl_coef=kl)
        loss.backward()
        grad = leaf.grad[..., None]
    assert loss.isnan() and grad[bad].isnan().all() and grad[~bad].isfinite().all()


@pytest.mark.parametrize("clip", [(0.2, 0.2), (0.2, float("inf"))])
def test_an_advantage_of_zero_takes_no_part(L, clip):  # noqa: F811
    """Whatever the ratio: here e^200, past fp32."""
    z, y, _, old, _, adv = make(1, 4, 300, "fp32", mask=None)
    adv[0, 1], old[0, 1] = 0.0, -200.0
    r = L.policy_loss_rows(z, y, old, adv, clip=clip, reduction="sum")
    assert r.loss.isfinite() and (r.dlogits[0, 1] == 0).all() and r.dlogits.isfinite().all()


@pytest.mark.parametrize("dtype,offset", [("bf16", 100.0), ("bf16", 1e3), ("bf16", 1e6), ("bf16", -1e30), ("fp16", 2e3),
                                          ("fp16", 6e4), ("fp32", 1e4)])
@pytest.mark.parametrize("V", [50, 40000])
def test_a_common_offset_leaves_the_gradient(L, dtype, offset, V):  # noqa: F811
    """softmax(z + a) = softmax(z): the exponents are differences of logits, as exact as those are (the other tests' bounds)."""
    z, y, m, _, _, adv = make(2, 3, V, dtype, seed=V)
    z = (z.float() + offset).to(z.dtype)
    c = counted(z, y, m)
    lp = oracle_logp(z, y, c)
    _, slope, terms = policy_oracle(lp, c, None, adv, None, (0.2, 0.2), 0.0, "sum")
    r = L.policy_loss_rows(z, y, None, adv, mask=m, reduction="sum")
    check_gradient(r.dlogits, z, y, c, slope, 2.0 ** -14 * terms)
    leaf = z.clone().requires_grad_()
    (L.policy_loss(leaf, y, None, adv, mask=m, reduction="sum").loss * 0.5).backward()
    check_gradient(leaf.grad, z, y, c, slope * 0.5, 2.0 ** -15 * terms)


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("drop", [18.0, 23.0])
def test_gradient_of_an_almost_certain_token(L, dtype, drop):  # noqa: F811
    """The target's own gradient c (1 - p) for 1 - p = 999 e^-drop (1.5e-5, 1e-7) and maxima of 8 to 120. The sum 1 + t of the
    row is at least 1 after any rounding, so the sign is c's or the value zero; it is off by at most 16
    additions' half steps of 2^-24 (a thread's, five steps of its warp, the warps' join) and c / s by one more."""
    T = 225
    top = 8.0 + 0.5 * torch.arange(T, device="cuda")
    z = (top - drop)[None, :, None].expand(1, T, 1000).contiguous().to({"bf16": torch.bfloat16, "fp16": torch.float16}.get(dtype, torch.float32))
    y = torch.arange(T, device="cuda")[None] * 4
    z.scatter_(-1, y[..., None], top.to(z.dtype)[None, :, None])
    adv = torch.ones(1, T, device="cuda")
    d = L.policy_loss_rows(z, y, None, adv, reduction="sum").dlogits
    got = -d.gather(-1, y[..., None]).double()
    want = 1 - torch.softmax(z.double(), -1).gather(-1, y[..., None])
    assert (got >= 0).all(), got.min().item()
    u = torch.finfo(z.dtype).eps / 2
    tiny = 2.0 ** -25 if dtype == "fp16" else 0.0
    assert ((got - want).abs() <= 17 * 2.0 ** -24 + u * want + tiny).all()


@pytest.mark.parametrize("V,dtype", [(2000, "fp32"), (2000, "bf16"), (40000, "bf16")])
def test_log_probabilities_have_no_common_error(L, V, dtype):  # noqa: F811
    """A sequence's reward adds up hundreds of log-probabilities, so an error of one sign counts. Each is rounded to fp32
    below 32 in size: half a step of 2^-20 at the most, 5.5e-7 in the standard deviation, so the mean of n has
    4.3e-9 (n = 16384) to 1.2e-8 (2048); six of those over the 5e-9 that the exponential's mean error is known to."""
    n = 16384 if V < 10000 else 2048
    z, y, _, _, _, _ = make(1, n, V, dtype, seed=1, mask=None)
    got = L.logprob_rows(z, y).double()
    want = torch.cat([torch.log_softmax(b.double(), -1).gather(-1, t[:, None])[:, 0] for b, t in zip(z[0].split(256), y[0].split(256))])
    assert abs((got[0] - want).mean().item()) <= 6 * 2.0 ** -20 / 12 ** 0.5 / n ** 0.5 + 5e-9
