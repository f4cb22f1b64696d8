"""Rotary positions, AdamW over many tensors and the losses on log-probabilities in launch shapes and values that the small
tests do not reach: several heads a thread, several blocks a warp, values past 2^31 elements, slopes of every kind."""
import pytest
import torch

from tests.test_losses_gpu import L, counted, make  # noqa: F401
from tests.test_rotary_gpu import DT, R, SCALINGS, check  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T", [901, 1101, 2203, 4099])  # whole heads of 128 on 148 SMs: one, two, four and eight heads a thread
@pytest.mark.parametrize("dtype,interleaved", [("bf16", False), ("fp16", True)])
@pytest.mark.parametrize("hd,rd", [(128, 128), (80, 80), (64, 32), (96, 40)])
def test_rotary_of_several_heads_a_thread(R, T, dtype, interleaved, hd, rd):  # noqa: F811
    g = torch.Generator(device="cuda").manual_seed(T)
    qkv = torch.randn(1, T, 47, hd, device="cuda", generator=g).to(DT[dtype])
    q, k = qkv[:, :, :32], qkv[:, :, 32:39]  # heads that do not fill the last group
    pos = torch.randint(0, 2 ** 21, (1, T), device="cuda", generator=g)
    rot = R.Rotary(hd, rotary_dim=rd, interleaved=interleaved, scaling=SCALINGS["yarn"])
    before = qkv.clone()
    qo, ko = rot.rotate(q, k, pos)
    check(qo, q, pos, rot.inv_freq, rot.factor, rd, interleaved, False)
    check(ko, k, pos, rot.inv_freq, rot.factor, rd, interleaved, False)
    rot.rotate(q, k, pos, q_out=q, k_out=k)
    assert torch.equal(q, qo) and torch.equal(k, ko) and torch.equal(qkv[:, :, 39:], before[:, :, 39:])


def test_rotary_past_2_31_elements(R):  # noqa: F811
    if torch.cuda.get_device_properties(0).total_memory < 60 << 30:
        pytest.skip("needs 20 GB")
    T = 2 ** 20 + 5
    x = torch.zeros(1, T, 17, 128, device="cuda", dtype=torch.bfloat16)
    rows = torch.tensor([0, 1, 986894, 986895, 986896, 1000000, T - 3, T - 2, T - 1], device="cuda")  # 986895 x 17 x 128 passes 2^31
    assert 986895 * 17 * 128 <= 2 ** 31 < 986896 * 17 * 128
    x[0, rows] = torch.randn(len(rows), 17, 128, device="cuda").bfloat16()
    some = x[:, rows].clone()
    rot = R.Rotary(128)
    y = rot.rotate(x, q_out=x)[0]
    check(y[:, rows], some, rows[None], rot.inv_freq, 1.0, 128, False, False)
    y[0, rows] = 0
    assert not y.any()


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("gdt,offset", [(torch.float32, 0), (torch.bfloat16, 0), (torch.bfloat16, 1)])
def test_adamw_of_several_blocks_a_warp(monkeypatch, bits, gdt, offset):
    """31500 blocks: seven a warp with 8-bit states, four in two waves with 32-bit ones; runs that pass from large tensors to
    many small ones and back, ragged and whole."""
    from llmt.optim import multi
    from tests import test_adamw_multi_gpu as one
    shapes = [(1000003,), (1, 1024), (2048, 1024)] + [(257 + 3 * i,) for i in range(100)] + [(700, 1001), (8,), (4096, 1024), (1024,), (511,)]
    monkeypatch.setattr(one, "SHAPES", shapes)
    one.test_steps(multi, bits, gdt, offset)


@pytest.mark.parametrize("kind", ["sigmoid", "hinge", "ipo"])
@pytest.mark.parametrize("average", [False, True])
@pytest.mark.parametrize("P,T", [(3, 9), (1, 1), (5, 700)])
def test_preference_slopes_of_log_probabilities(L, P, T, kind, average):  # noqa: F811
    """Gradients of logp against the loss's in fp64: gains are sums in fp64, rounded once with D; the slope's few fp32
    operations (three exponentials at most) are under 2^-20 of the largest slope, D's rounding 2^-23 of D times f'' at most 2."""
    z, y, m, _, ref, _ = make(2 * P, T, 50, "fp32", seed=P, mask="some")
    c = counted(z, y, m)
    leaf = L.logprob_rows(z, y, m).requires_grad_()
    beta, s = 0.3, (0.1 if kind == "sigmoid" else 0.0)
    out = L.preference_loss_tokens(leaf, y, 50, ref_logp=ref, mask=m, beta=beta, kind=kind, label_smoothing=s, average=average)
    (out.loss * 0.7).backward()
    lp = leaf.detach().double().requires_grad_()
    n = c.sum(1).clamp(min=1).double() if average else torch.ones(2 * P, dtype=torch.float64, device="cuda")
    gain = torch.where(c, lp - ref.double(), torch.zeros_like(lp)).sum(1) / n
    D = gain[:P] - gain[P:]
    sp = torch.nn.functional.softplus
    per = {"sigmoid": (1 - s) * sp(-beta * D) + s * sp(beta * D), "hinge": torch.relu(1 - beta * D), "ipo": (D - 0.5 / beta) ** 2}[kind]
    (want,) = torch.autograd.grad(0.7 * per.mean(), lp)
    size = torch.maximum(torch.full_like(D, beta), 2 * (D.abs() + 0.5 / beta)) if kind == "ipo" else torch.full_like(D, beta)
    # a log-probability less its reference is one fp32 rounding, 2^-24 of up to 2^5, so a gain T 2^-19 / n
    gain_err = torch.full_like(D, 2.0 ** -19 * (1 if average else T)) + 2.0 ** -23 * D.abs()
    bound = ((2.0 ** -20 * size + 2 * gain_err).repeat(2) / P / n)[:, None] * c
    assert ((leaf.grad.double() - want).abs() <= bound).all()
    assert want[c].abs().max() > 0 and (leaf.grad[~c] == 0).all()
    # kernels and definition agree to 1% of the slopes at least, so a wrong factor would show
    assert ((leaf.grad.double() - want).abs().max() <= 0.01 * want.abs().max())
