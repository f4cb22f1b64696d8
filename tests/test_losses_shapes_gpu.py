"""The losses over logits rows in the launch shapes of large batches: one CTA a row, each streaming several tiles
(on 148 SMs above 296 rows), against the definition in fp64. Tolerances are those of the smaller shapes."""
import pytest
import torch

from tests.test_losses_gpu import L, check_gradient, check_logp, counted, make, oracle_logp, policy_oracle  # noqa: F401

pytestmark = pytest.mark.gpu

ROWS = [  # B, T, V, dtype, mask: two tiles to five, whole and ragged rows, rows of 16-byte pieces and off them
    (300, 1, 24000, "bf16", "some"), (299, 1, 70001, "bf16", "some"), (3, 101, 40009, "fp32", None),
    (150, 2, 40960, "fp16", "some"), (1, 301, 32776, "bf16", "row"),
]


@pytest.mark.parametrize("B,T,V,dtype,mask", ROWS)
def test_logprob_rows_of_several_tiles(L, B, T, V, dtype, mask):  # noqa: F811
    z, y, m, _, _, _ = make(B, T, V, dtype, seed=V, mask=mask)
    check_logp(L.logprob_rows(z, y, m), oracle_logp(z, y, counted(z, y, m)))


@pytest.mark.parametrize("B,T,V,dtype,mask", ROWS)
@pytest.mark.parametrize("inplace", [False, True])
def test_policy_rows_of_several_tiles(L, B, T, V, dtype, mask, inplace):  # noqa: F811
    z, y, m, old, ref, adv = make(B, T, V, dtype, seed=V, mask=mask)
    c = counted(z, y, m)
    lp = oracle_logp(z, y, c)
    loss, slope, terms = policy_oracle(lp, c, old, adv, ref, (0.2, 0.3), 0.1, "token")
    work = z.clone()
    r = L.policy_loss_rows(work, y, old, adv, ref_logp=ref, mask=m, clip=(0.2, 0.3), kl_coef=0.1, out=work if inplace else None)
    assert (r.dlogits.data_ptr() == work.data_ptr()) == inplace
    check_logp(r.logp, lp)
    assert abs(r.loss.item() - loss.item()) <= 2.0 ** -14 * terms.sum().item()
    check_gradient(r.dlogits, z, y, c, slope, 2.0 ** -14 * terms)


@pytest.mark.parametrize("B,T,V,dtype", [(2, 300, 33000, "bf16"), (3, 201, 66, "fp32")])
@pytest.mark.parametrize("reduction", ["token", "sequence", "sum"])
def test_more_tokens_than_a_row_counts_itself(L, B, T, V, dtype, reduction):  # noqa: F811
    """Above 512 tokens a kernel of its own counts them."""
    z, y, m, old, ref, adv = make(B, T, V, dtype, seed=T)
    c = counted(z, y, m)
    lp = oracle_logp(z, y, c)
    loss, slope, terms = policy_oracle(lp, c, old, adv, ref, (0.2, 0.2), 0.1, reduction)
    r = L.policy_loss_rows(z, y, old, adv, ref_logp=ref, mask=m, kl_coef=0.1, reduction=reduction)
    assert abs(r.loss.item() - loss.item()) <= 2.0 ** -14 * terms.sum().item()
    check_gradient(r.dlogits, z, y, c, slope, 2.0 ** -14 * terms)


@pytest.mark.parametrize("kind", ["sigmoid", "ipo"])
@pytest.mark.parametrize("P,T,V,dtype,mask", [(150, 1, 70001, "bf16", "some"), (1, 151, 40009, "fp32", "some"), (2, 75, 40960, "fp16", "row")])
def test_preference_rows_of_several_tiles(L, P, T, V, dtype, mask, kind):  # noqa: F811
    from tests.test_losses_gpu import test_preference_rows
    test_preference_rows(L, P, T, V, dtype, mask, False, kind)


def test_autograd_of_rows_of_several_tiles(L):  # noqa: F811
    """The gradient computed again for an incoming gradient other than 1."""
    z, y, m, old, ref, adv = make(2, 150, 40001, "bf16", seed=4)
    c = counted(z, y, m)
    _, slope, terms = policy_oracle(oracle_logp(z, y, c), c, old, adv, ref, (0.2, 0.2), 0.1, "token")
    for scale in (1.0, 0.3):
        leaf = z.clone().requires_grad_()
        (L.policy_loss(leaf, y, old, adv, ref_logp=ref, mask=m, kl_coef=0.1).loss * scale).backward()
        check_gradient(leaf.grad, z, y, c, slope * scale, 2.0 ** -14 * terms * scale)
