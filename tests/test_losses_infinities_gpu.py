"""The losses where a token is impossible or an advantage infinite: limits where the formula has them, NaN or infinities in
the gradient wherever the loss has them."""
import pytest
import torch

from tests.test_losses_gpu import L, make  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("form", ["rows", "tokens"])
@pytest.mark.parametrize("kind,smoothing", [("sigmoid", 0.0), ("sigmoid", 0.1), ("hinge", 0.0)])
def test_an_impossible_token_of_a_rejected_sequence(L, form, kind, smoothing):  # noqa: F811
    """Its gain is -inf and D +inf: -log sigma(beta D) and the hinge are 0 there with slope 0; with smoothing the other
    term is infinite."""
    z, y, _, _, ref, _ = make(4, 3, 200, "fp32", mask=None)
    y[2:] += (y[2:] == 7)
    y[3, 1] = 7
    z[3, 1, 7] = float("-inf")
    if form == "rows":
        r = L.preference_loss_rows(z, y, ref_logp=ref, kind=kind, label_smoothing=smoothing)
        one = L.preference_loss_rows(z[[0, 2]], y[[0, 2]], ref_logp=ref[[0, 2]], kind=kind, label_smoothing=smoothing)
        grad = r.dlogits
    else:
        leaf = L.logprob_rows(z, y).requires_grad_()
        r = L.preference_loss_tokens(leaf, y, 200, ref_logp=ref, kind=kind, label_smoothing=smoothing)
        one = L.preference_loss_tokens(leaf.detach()[[0, 2]], y[[0, 2]], 200, ref_logp=ref[[0, 2]], kind=kind, label_smoothing=smoothing)
        r.loss.backward()
        grad = leaf.grad
    assert r.rewards[3] == float("-inf") and r.rewards[:3].isfinite().all()
    if smoothing:
        assert r.loss == float("inf")
    else:
        # the mean of the other pair's loss and 0, rounded once more
        assert abs(r.loss.item() - one.loss.item() / 2) <= 2.0 ** -23 * one.loss.item()
        assert (grad[[1, 3]] == 0).all()
    assert grad.isfinite().all() and (grad[[0, 2]] != 0).any()


def test_an_infinite_advantage_shows_in_the_gradient(L):  # noqa: F811
    """Also under a ratio that is zero in fp32, e^-200."""
    z, y, _, old, _, adv = make(1, 4, 300, "fp32", mask=None)
    adv[0, 1], adv[0, 2] = float("inf"), float("inf")
    old[0, 1] = 200.0
    r = L.policy_loss_rows(z, y, old, adv, reduction="sum")
    assert not r.loss.isfinite() and not r.dlogits[0, 1].isfinite().any() and not r.dlogits[0, 2].isfinite().any()
    assert r.dlogits[0, [0, 3]].isfinite().all()
