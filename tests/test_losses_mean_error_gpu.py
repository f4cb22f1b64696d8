"""Errors of one sign in the sums over a row: the factor that joins two warps' sums, and log-probabilities in the mean."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("k", [0, 1, 2, 5])
def test_the_factor_that_joins_two_sums(k):
    """Rows of two values, 0 and x in (-k - 1, -k), in two warps' parts: each sums to exactly 1 under its own maximum, so
    the row's sum is 1 + e^x with the joining factor alone. The sum's rounding is half a step of 2^-23, 3.4e-8 in the
    standard deviation, the factor's seven roundings and its last one under 2^-24: 4e-8 together at most, 1.6e-10 for the
    mean of 65536; six of those, and 1e-9 that the factor may be off in the mean."""
    from llmt.ops import native as N
    n, V = 65536, 512
    z = torch.full((1, n, V), float("-inf"), device="cuda")
    x = -k - torch.rand(n, device="cuda", generator=torch.Generator(device="cuda").manual_seed(k))
    z[0, :, 3], z[0, :, 200] = 0.0, x
    stats = N.ext().logprob_rows(z, torch.zeros(1, n, dtype=torch.long, device="cuda"), None)[1][0].double()
    assert (stats[:, 0] == 0).all()
    off = stats[:, 1] - (1 + x.double().exp())
    assert off.abs().max().item() <= 2.0 ** -24 + 2.0 ** -23 * x.max().exp().item()
    assert abs(off.mean().item()) <= 6 * 1.6e-10 + 1e-9


@pytest.mark.parametrize("V,dtype,n", [(200, torch.float32, 200000), (5110, torch.bfloat16, 40000), (128256, torch.bfloat16, 3000)])
def test_log_probabilities_in_the_mean(V, dtype, n):
    """Six standard errors of the n results' spread, over the 5e-9 to which the exponentials' mean error is known for normal
    logits of spread 2 (3.6e-8 to 4.5e-8, of which 4e-8 are taken back)."""
    from llmt.ops import losses as L
    off, part = [], max(1, 80_000_000 // V)
    for c, first in enumerate(range(0, n, part)):
        g = torch.Generator(device="cuda").manual_seed(c)
        rows = min(part, n - first)
        z = (torch.randn(1, rows, V, device="cuda", generator=g) * 2).to(dtype)
        y = torch.randint(0, V, (1, rows), device="cuda", generator=g)
        want = z.double().gather(-1, y[..., None])[..., 0] - torch.logsumexp(z.double(), -1)
        off.append((L.logprob_rows(z, y).double() - want)[0])
    off = torch.cat(off)
    assert abs(off.mean().item()) <= 6 * (off.std() / n ** 0.5).item() + 5e-9
