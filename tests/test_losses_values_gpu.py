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
