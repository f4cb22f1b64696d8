"""The post-training losses over logits rows against their definition in fp64 (autograd of the
formula), and against finite differences.

Tolerances, for half-step u = eps / 2 of the logits' type: exp(z - M) is off by the rounding of its
exponent (3 roundings of at most |z - M| < 60, 2^-24 each) and of the exponential (2^-22): under
2^-16; the sum of up to 2^17 such terms in a tree adds less; so logp is off by 2^-15 + 2^-22 |logp|, a
slope c = w (-rA + k (1 - e^d)) by its terms' sum times 2^-14, and a gradient value by u of itself
(fp16 results below its normal range: 2^-25) plus 2^-15 |c| plus the slope's own error."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


@pytest.fixture(scope="module")
def L():
    from llmt.ops import losses, native
    native.ext()
    return losses


def make(B, T, V, dtype, seed=0, mask="some", spread=3.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    z = (torch.randn(B, T, V, device="cuda", generator=g) * spread).to(DT[dtype])
    y = torch.randint(0, V, (B, T), device="cuda", generator=g)
    m = None
    if mask == "some":
        m = torch.rand(B, T, device="cuda", generator=g) < 0.6
        m[0, 0] = True
    elif mask == "row":  # a whole sequence without tokens
        m = torch.ones(B, T, dtype=torch.bool, device="cuda")
        m[-1] = False
    elif mask == "none":
        m = torch.zeros(B, T, dtype=torch.bool, device="cuda")
    lp = torch.log_softmax(z.double(), -1).gather(-1, y[..., None])[..., 0].float()
    n = torch.randn(3, B, T, device="cuda", generator=g)
    return z, y, m, lp + 0.2 * n[0], lp + 0.4 * n[1], n[2] + 0.3


def counted(z, y, m):
    c = (y >= 0) & (y < z.shape[-1])
    return c if m is None else c & m


def oracle_logp(z, y, c):
    """fp64 log-probabilities; rows that do not count are not looked at."""
    safe = torch.where(c[..., None], z.double(), torch.zeros((), dtype=torch.float64, device=z.device))
    return torch.log_softmax(safe, -1).gather(-1, torch.where(c, y, torch.zeros_like(y))[..., None])[..., 0] * c


def weights(c, reduction):
    n = c.sum(1).double()
    if reduction == "sum":
        return c.double()
    if reduction == "token":
        return c.double() / n.sum().clamp(min=1)
    return c.double() / (n[:, None].clamp(min=1) * (n > 0).sum().clamp(min=1))


def policy_oracle(lp, c, old, adv, ref, clip, k, reduction):
    """(loss, slope, bound of the slope's terms) from fp64 log-probabilities."""
    lp = lp.detach().requires_grad_()
    w = weights(c, reduction)
    r = (lp - (lp.detach() if old is None else old.double())).exp()
    A = adv.double().expand_as(lp)
    t = -torch.minimum(r * A, r.clamp(1 - clip[0], 1 + clip[1]) * A)
    terms = r.detach() * A.abs()
    if ref is not None:
        d = ref.double() - lp
        t = t + k * (d.exp() - 1 - d)
        terms = terms + k * (1 + d.detach().exp() + d.detach().abs())
    loss = (torch.where(c, t, torch.zeros_like(t)) * w).sum()
    (slope,) = torch.autograd.grad(loss, lp)
    return loss.detach(), torch.where(c, slope, torch.zeros_like(slope)), torch.where(c, terms * w, torch.zeros_like(w))


def check_gradient(got, z, y, c, slope, slope_err):
    soft = torch.softmax(torch.where(c[..., None], z.double(), torch.zeros((), dtype=torch.float64, device=z.device)), -1)
    hot = torch.zeros_like(soft).scatter_(-1, torch.where(c, y, torch.zeros_like(y))[..., None], 1.0)
    want = slope[..., None] * (hot - soft)
    u = torch.finfo(got.dtype).eps / 2
    tiny = 2.0 ** -25 if got.dtype == torch.float16 else 0.0
    bound = u * want.abs() + tiny + (2.0 ** -15 * slope.abs() + slope_err)[..., None] * (hot + soft)
    off = (got.double() - want).abs() - bound
    assert off.max().item() <= 0, (off.max().item(), (off > 0).sum().item())
    assert (got[~c] == 0).all()


def check_logp(got, want):
    assert ((got.double() - want).abs() <= 2.0 ** -15 + 2.0 ** -22 * want.abs()).all()


CASES = [  # B, T, V, dtype, mask: one id, rows off 16 bytes, whole pieces, many pieces, rows past every split
    (1, 1, 1, "fp32", None), (2, 3, 2, "bf16", "some"), (3, 5, 7, "fp16", "row"), (2, 4, 8, "bf16", "some"),
    (2, 3, 129, "fp32", "some"), (4, 9, 500, "bf16", "some"), (1, 33, 1000, "fp16", "none"), (2, 17, 4097, "bf16", "row"),
    (3, 2, 8192, "fp32", "some"), (2, 5, 32000, "bf16", "some"), (2, 5, 32003, "bf16", "some"), (1, 3, 32003, "fp32", "some"),
    (1, 2, 128256, "bf16", None), (2, 1, 128256, "fp32", "some"), (1, 2, 300007, "bf16", None), (1, 1, 300007, "fp32", None),
    (40, 8, 700, "bf16", "some"), (300, 1, 66, "fp32", "some"), (2, 100, 32000, "fp16", "some"),
]


@pytest.mark.parametrize("B,T,V,dtype,mask", CASES)
@pytest.mark.parametrize("reduction", ["token", "sequence"])
def test_policy_rows(L, B, T, V, dtype, mask, reduction):
    z, y, m, old, ref, adv = make(B, T, V, dtype, seed=B + T + V, mask=mask)
    c = counted(z, y, m)
    r = L.policy_loss_rows(z, y, old, adv, ref_logp=ref, mask=m, clip=(0.2, 0.3), kl_coef=0.1, reduction=reduction)
    lp = oracle_logp(z, y, c)
    loss, slope, terms = policy_oracle(lp, c, old, adv, ref, (0.2, 0.3), 0.1, reduction)
    check_logp(r.logp, lp)
    assert abs(r.loss.item() - loss.item()) <= 2.0 ** -14 * terms.sum().item() + 1e-30
    check_gradient(r.dlogits, z, y, c, slope, 2.0 ** -14 * terms)
    assert L.policy_loss_rows(z, y, old, adv, mask=m, grad=False).dlogits is None
    check_logp(L.logprob_rows(z, y, m), lp)


@pytest.mark.parametrize("kind", ["sigmoid", "hinge", "ipo"])
@pytest.mark.parametrize("average", [False, True])
@pytest.mark.parametrize("P,T,V,dtype,mask", [(1, 1, 5, "fp32", None), (2, 9, 500, "bf16", "some"), (3, 33, 4097, "fp16", "row"),
                                              (1, 300, 64, "fp32", "some"), (1, 7, 32003, "bf16", "some"),
                                              (2, 2, 128256, "bf16", "none"), (70, 3, 40, "bf16", "some")])
def test_preference_rows(L, P, T, V, dtype, mask, average, kind):
    z, y, m, _, ref, _ = make(2 * P, T, V, dtype, seed=P + T + V, mask=mask)
    c = counted(z, y, m)
    beta, s = 0.3, (0.1 if kind == "sigmoid" else 0.0)
    r = L.preference_loss_rows(z, y, ref_logp=ref, mask=m, beta=beta, kind=kind, label_smoothing=s, average=average)
    lp = oracle_logp(z, y, c)
    check_logp(r.logp, lp)
    lp.requires_grad_()
    n = c.sum(1).clamp(min=1).double() if average else torch.ones(2 * P, dtype=torch.float64, device="cuda")
    gain = torch.where(c, lp - ref.double(), torch.zeros_like(lp)).sum(1) / n
    D = gain[:P] - gain[P:]
    sp = torch.nn.functional.softplus
    per = {"sigmoid": (1 - s) * sp(-beta * D) + s * sp(beta * D), "hinge": torch.relu(1 - beta * D),
           "ipo": (D - 0.5 / beta) ** 2}[kind]
    (slope,) = torch.autograd.grad(per.mean(), lp)
    # a gain is off by its tokens' errors, a reward by beta times that, a slope by the change of f' (at most 2)
    err = (2.0 ** -15 + 2.0 ** -22 * (lp.detach().abs() + ref.abs())).mul(c).sum(1) / n
    assert ((r.rewards.double() - beta * gain.detach()).abs() <= beta * err + 2.0 ** -22 * (beta * gain).abs()).all()
    derr = err[:P] + err[P:] + 2.0 ** -22 * (gain[:P].abs() + gain[P:].abs())
    d1 = torch.maximum(torch.full_like(D, beta), 2 * (D - 0.5 / beta).abs()) if kind == "ipo" else torch.full_like(D, beta)
    assert abs(r.loss.item() - per.mean().item()) <= (d1 * derr + derr ** 2 + 2.0 ** -21 * per).mean().item()
    slope_err = (2 * derr + 2.0 ** -20 * d1).repeat(2)[:, None] / P / n[:, None] * c
    check_gradient(r.dlogits, z, y, c, slope.detach(), slope_err)


def test_rows_that_do_not_count_are_not_read(L):
    z, y, m, old, ref, adv = make(3, 6, 1000, "bf16", mask="some")
    y[~m] = -100
    want = L.policy_loss_rows(z, y, old, adv, ref_logp=ref, kl_coef=0.1)  # by the targets alone
    z2, old2 = z.clone(), old.clone()
    z2[~m] = float("nan")
    z2[0][~m[0]] = float("inf")
    old2[~m] = float("nan")
    got = L.policy_loss_rows(z2, torch.where(m, y, y.clamp(min=1000)), old2, adv, ref_logp=ref, mask=m, kl_coef=0.1)
    for a, b in zip(want, got):
        assert torch.equal(a, b)
    p = L.preference_loss_rows(z2[:2], y[:2], mask=m[:2])
    q = L.preference_loss_rows(z[:2], y[:2], mask=m[:2])
    for a, b in zip(p, q):
        assert torch.equal(a, b)


def test_no_token_counts(L):
    z, y, m, old, ref, adv = make(2, 3, 77, "fp32", mask="none")
    r = L.policy_loss_rows(torch.full_like(z, float("nan")), y, old, adv, mask=m)
    assert r.loss.item() == 0 and (r.dlogits == 0).all() and (r.logp == 0).all()
    r = L.preference_loss_rows(torch.full_like(z, float("nan")), y, mask=m)
    assert abs(r.loss.item() - 0.6931472) < 1e-6 and (r.dlogits == 0).all() and (r.rewards == 0).all()


def test_masked_ids_and_infinities(L):
    """-inf logits (ids that may not be chosen) are zero probabilities; the type's lowest value is one too;
    a row of nothing else, an infinite or a NaN logit gives NaN in that row and nowhere else."""
    z, y, _, old, ref, adv = make(1, 6, 3000, "bf16", mask=None)
    z[:, :, 100:2900] = float("-inf")
    z[:, 1, 2900:] = torch.finfo(torch.bfloat16).min
    y = y % 100
    c = torch.ones_like(y, dtype=torch.bool)
    r = L.policy_loss_rows(z, y, None, adv, reduction="sum")
    lp = oracle_logp(z, y, c)
    _, slope, terms = policy_oracle(lp, c, None, adv, None, (0.2, 0.2), 0.0, "sum")
    check_logp(r.logp, lp)
    check_gradient(r.dlogits, z, y, c, slope, 2.0 ** -14 * terms)
    z[0, 2, 5], z[0, 3, 7], z[0, 4] = float("inf"), float("nan"), float("-inf")
    r = L.policy_loss_rows(z, y, None, adv, reduction="sum")
    bad = torch.tensor([False, False, True, True, True, False], device="cuda")
    assert r.dlogits[0, bad].isnan().all() and not r.dlogits[0, ~bad].isnan().any()
    assert r.logp[0].isnan().equal(bad) and r.loss.isnan()


def test_strides_broadcasts_and_outputs(L):
    z, y, m, old, ref, adv = make(3, 5, 1001, "bf16", mask="some")
    c = counted(z, y, m)
    lp = oracle_logp(z, y, c)
    loss, slope, terms = policy_oracle(lp, c, old, adv[:, :1], ref, (0.2, 0.2), 0.1, "token")
    wide = torch.full((3, 5, 1040), -5.0, device="cuda", dtype=z.dtype)
    wide[:, :, 3:1004] = z
    turned = torch.empty(5, 3, 1001, device="cuda", dtype=z.dtype).transpose(0, 1)
    turned.copy_(z)
    for view in (wide[:, :, 3:1004], turned):
        got = L.policy_loss_rows(view, y.t().contiguous().t(), old.t().contiguous().t(), adv[:, :1], ref_logp=ref,
                                 mask=m.t().contiguous().t(), kl_coef=0.1)
        # a row's pieces begin at 16-byte borders, so another alignment adds its terms up in another
        # order: each result is held to the definition (two of them differ by up to twice that)
        check_logp(got.logp, lp)
        assert abs(got.loss.item() - loss.item()) <= 2.0 ** -14 * terms.sum().item()
        check_gradient(got.dlogits, z, y, c, slope, 2.0 ** -14 * terms)
    # in place, and into padded rows: the bytes around them stay
    inside = wide.clone()
    got = L.policy_loss_rows(inside[:, :, 3:1004], y, old, adv[:, :1], ref_logp=ref, mask=m, kl_coef=0.1,
                             out=inside[:, :, 3:1004])
    apart = torch.full_like(wide, 9.0)
    got2 = L.policy_loss_rows(wide[:, :, 3:1004], y, old, adv[:, :1], ref_logp=ref, mask=m, kl_coef=0.1,
                              out=apart[:, :, 4:1005])
    assert torch.equal(got.dlogits, got2.dlogits)
    assert (inside[:, :, :3] == -5).all() and (inside[:, :, 1004:] == -5).all()
    assert (apart[:, :, :4] == 9).all() and (apart[:, :, 1005:] == 9).all()


def test_equal_inputs_give_equal_bits(L):
    z, y, m, old, ref, adv = make(4, 64, 4096, "bf16")
    a = L.policy_loss_rows(z, y, old, adv, ref_logp=ref, mask=m, kl_coef=0.1)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        b = L.policy_loss_rows(z, y, old, adv, ref_logp=ref, mask=m, kl_coef=0.1)
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(u, v) for u, v in zip(a, b))


def test_two_graphs_replayed_together(L):
    z, y, m, old, ref, adv = make(4, 16, 4096, "bf16")
    z2, y2, m2, old2, ref2, _ = make(4, 16, 4096, "bf16", seed=9)
    want = [L.policy_loss_rows(z, y, old, adv, ref_logp=ref, mask=m, kl_coef=0.1), L.preference_loss_rows(z2, y2, ref2, m2)]
    torch.cuda.synchronize()
    g1, g2, s1, s2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph(), torch.cuda.Stream(), torch.cuda.Stream()
    with torch.cuda.graph(g1):
        r1 = L.policy_loss_rows(z, y, old, adv, ref_logp=ref, mask=m, kl_coef=0.1)
    with torch.cuda.graph(g2):
        r2 = L.preference_loss_rows(z2, y2, ref2, m2)
    for _ in range(5):
        with torch.cuda.stream(s1):
            g1.replay()
        with torch.cuda.stream(s2):
            g2.replay()
    torch.cuda.synchronize()
    for r, w in zip((r1, r2), want):
        assert all(torch.equal(a, b) for a, b in zip(r, w))


@pytest.mark.parametrize("scale", [1.0, 0.3])
def test_autograd(L, scale):
    """Once-rounded gradients for any incoming gradient, twice from one graph too."""
    z, y, m, old, ref, adv = make(2, 8, 3001, "bf16")
    c = counted(z, y, m)
    lp = oracle_logp(z, y, c)
    loss, slope, terms = policy_oracle(lp, c, old, adv, ref, (0.2, 0.2), 0.1, "token")
    leaf = z.clone().requires_grad_()
    out = L.policy_loss(leaf, y, old, adv, ref_logp=ref, mask=m, kl_coef=0.1)
    (out.loss * scale).backward(retain_graph=True)
    check_gradient(leaf.grad, z, y, c, slope * scale, 2.0 ** -14 * terms * scale)
    first, leaf.grad = leaf.grad, None
    (out.loss * 2.0).backward()
    check_gradient(leaf.grad, z, y, c, slope * 2, 2.0 ** -14 * terms * 2)
    check_gradient(first, z, y, c, slope * scale, 2.0 ** -14 * terms * scale)
    assert torch.equal(leaf.detach(), z)
    leaf.grad = None
    out = L.preference_loss(leaf, y, ref_logp=ref, mask=m)
    (out.loss * scale).backward()
    rows = L.preference_loss_rows(z, y, ref_logp=ref, mask=m)
    u = torch.finfo(z.dtype).eps / 2
    assert ((leaf.grad.double() - rows.dlogits.double() * scale).abs() <= 2.1 * u * rows.dlogits.double().abs() * scale).all()


def test_no_grad_writes_no_gradient(L):
    z, y, m, old, ref, adv = make(2, 64, 8192, "fp32")
    z.requires_grad_()
    want = L.policy_loss(z, y, old, adv, ref, m, kl_coef=0.1)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    with torch.no_grad():
        got = L.policy_loss(z, y, old, adv, ref, m, kl_coef=0.1)
    assert torch.cuda.max_memory_allocated() - before < z.numel()  # a gradient is 4 bytes a value
    assert not got.loss.requires_grad
    assert ((got.logp - want.logp).abs() <= 2 ** -14 + 2 ** -21 * want.logp.abs()).all()  # each is off by half of that


def test_token_forms_match_rows(L):
    z, y, m, old, ref, adv = make(4, 9, 2000, "fp32")
    leaf = L.logprob_rows(z, y, m).requires_grad_()
    rows = L.policy_loss_rows(z, y, old, adv, ref_logp=ref, mask=m, kl_coef=0.1, reduction="sequence")
    loss = L.policy_loss_tokens(leaf, y, 2000, old, adv, ref_logp=ref, mask=m, kl_coef=0.1, reduction="sequence")
    loss.backward()
    c = counted(z, y, m)
    _, slope, terms = policy_oracle(leaf.detach().double(), c, old, adv, ref, (0.2, 0.2), 0.1, "sequence")
    assert torch.equal(loss, rows.loss)
    assert ((leaf.grad.double() - slope).abs() <= 2.0 ** -18 * terms).all()
    leaf.grad = None
    rows = L.preference_loss_rows(z, y, ref_logp=ref, mask=m, kind="ipo", average=True)
    out = L.preference_loss_tokens(leaf, y, 2000, ref_logp=ref, mask=m, kind="ipo", average=True)
    assert torch.equal(out.loss, rows.loss) and torch.equal(out.rewards, rows.rewards)
    out.loss.backward()
    assert (leaf.grad[~c] == 0).all() and (leaf.grad[:2][c[:2]].sign() * leaf.grad[2:].sum().sign() <= 0).all()


def test_gradient_against_differences(L):
    """Central differences of the kernel's own fp32 loss, h = 2^-6: the loss (a sum of order 1) is
    computed to 2^-18, so a quotient to 2^-13, and the third derivative adds under 2^-12."""
    z, y, m, old, ref, adv = make(1, 3, 50, "fp32", spread=1.0)
    old = old + 0.0
    f = lambda x: L.policy_loss_rows(x, y, old, adv, ref_logp=ref, mask=m, clip=(0.9, 5.0), kl_coef=0.1, grad=False).loss.item()
    d = L.policy_loss_rows(z, y, old, adv, ref_logp=ref, mask=m, clip=(0.9, 5.0), kl_coef=0.1).dlogits
    h = 2.0 ** -6
    for t in range(3):
        for v in (0, 17, int(y[0, t]), 49):
            up, down = z.clone(), z.clone()
            up[0, t, v] += h
            down[0, t, v] -= h
            assert abs((f(up) - f(down)) / (2 * h) - d[0, t, v].item()) < 2.0 ** -11


def test_overlapping_outputs_are_refused(L):
    z, y, _, old, _, adv = make(2, 4, 64, "fp32", mask=None)
    buf = torch.zeros(2 * 4 * 64 + 64, device="cuda")
    a, b = buf[:512].view(2, 4, 64), buf[64:576].view(2, 4, 64)
    with pytest.raises(RuntimeError, match="overlap"):
        L.policy_loss_rows(a, y, old, adv, out=b)
    with pytest.raises(RuntimeError, match="overlap"):
        L.policy_loss_rows(z, y, old, adv, out=torch.zeros(1, 4, 64, device="cuda").expand(2, 4, 64))
