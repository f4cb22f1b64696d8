"""AdamW over many tensors against the update in fp64.

Tolerances: m and v are three fp32 roundings off (2^-22 of the sizes that go in), the step's quotient
a few more and the bias corrections' powers 2^-20: p is off by 2^-23 |p| + 2^-19 of its update's size.
An 8-bit state is one of the two values of its format around the fp64 one: the upper one where
the place between them passes 1 - u, u the value's 16 random bits (plus a half) / 2^16; where the fp32
value and the fp64 one may lie on two sides of that border (2^-18 of a step away) either is right."""
import pytest
import torch

pytestmark = pytest.mark.gpu
BLOCK = 256


@pytest.fixture(scope="module")
def M():
    from llmt.optim import multi
    from llmt.ops import native
    native.ext()
    return multi


def noise(n, step, seed):
    """The two 16-bit numbers of each place: the documented hash, in 64-bit integers."""
    low = 0xFFFFFFFF
    i = torch.arange(n, device="cuda")
    x = ((i & low) ^ ((i >> 32) * 0x6A09E667 & low)) * 0x9E3779B1 + step * 0xB7E15163 + seed * 0x3C6EF373 & low
    x = ((x ^ (x >> 16)) * 0xB7E15163) & low
    x = ((x ^ (x >> 15)) * 0x6A09E667) & low
    x = x ^ (x >> 16)
    return x >> 16, x & 0xFFFF


def quantized(x, r, low, top):
    """(value chosen, other value, whether the choice is clear) for blocks of x >= 0 in fp64: floats of 3
    mantissa bits, smallest normal 2^low, largest `top`, under the smallest fitting power of two."""
    b = x.view(-1, BLOCK)
    big = b.amax(1, keepdim=True)
    frac, e = torch.frexp(big / top)  # exact, where log2 of a power of two may fall short of it
    e = torch.where(big > 0, (e - (frac == 0.5).int()).double(), torch.full_like(big, -126.0))
    scale = torch.exp2(e.clamp(min=-126.0)).expand_as(b).reshape(-1)
    y = x / scale
    step = torch.exp2(torch.frexp(y.clamp(min=2.0 ** low))[1].double() - 4)
    place = y / step
    u = (r.double() * 16 + 8) / 2.0 ** 20
    at = place + u
    chosen = (torch.floor(at) * step).clamp(max=top)
    near = (at - at.round()).abs()
    other = (torch.where(at - at.floor() < 0.5, torch.floor(at) - 1, torch.floor(at) + 1) * step).clamp(max=top)
    # 2^-18 of a value in units of its step (at most 16 steps)
    return chosen * scale, other * scale, near > 16 * 2.0 ** -18, step * scale


def reference(p, g, m, v, wd, lr, b, eps, t):
    p, g, m, v = (x.double() for x in (p, g, m, v))
    m = b[0] * m + (1 - b[0]) * g
    v = b[1] * v + (1 - b[1]) * g * g
    up = lr / (1 - b[0] ** t) * m / ((v / (1 - b[1] ** t)).sqrt() + eps)
    return p * (1 - lr * wd) - up, m, v, up.abs()


SHAPES = [(1,), (255,), (256,), (257,), (3, 1001), (64, 64), (8,), (2048,), (511,), (4096, 33)]


def tensors(shapes, gdt, seed=0, offset=0):
    """Tensors of these shapes; `offset` elements into their allocations (off 32- and 16-byte borders)."""
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def one(s, scale, dt):
        n = int(torch.tensor(s).prod())
        buf = torch.zeros(n + offset + 7, device="cuda", dtype=dt)
        buf[offset:offset + n] = (torch.randn(n, device="cuda", generator=gen) * scale).to(dt)
        return buf[offset:offset + n].view(s)
    p = [one(s, 0.05, torch.float32) for s in shapes]
    g = [one(s, 1e-3, gdt) * torch.randint(0, 3, s, device="cuda", generator=gen) for s in shapes]
    if offset:
        g = [torch.cat([torch.zeros(offset, device="cuda", dtype=gdt), x.reshape(-1)])[offset:].view(s) for x, s in zip(g, shapes)]
    return p, g, [one(s, 0.0, torch.bfloat16) for s in shapes]


def per_tensor(opt):
    return opt.param_states()


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("gdt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("offset", [0, 1, 4])
def test_steps(M, bits, gdt, offset):
    p, g, s16 = tensors(SHAPES, gdt, offset=offset)
    wd = [0.1 if i % 2 else 0.0 for i in range(len(p))]
    b, eps, lr, seed = (0.9, 0.95), 1e-8, 1e-3, 5
    opt = M.MultiAdamW(p, s16, lr=lr, betas=b, eps=eps, weight_decay=wd, state_bits=bits, seed=seed)
    for t in range(1, 5):
        before = [(x.clone(), m, v) for x, (m, v) in zip(p, per_tensor(opt))]
        opt.step(g)
        assert opt.step_t.item() == t and opt.ticket.item() == 0
        n = opt.plan.blocks * BLOCK
        rm, rv = noise(n, t, seed)
        live = torch.zeros(n, dtype=torch.bool, device="cuda")
        m64, v64 = torch.zeros(n, dtype=torch.float64, device="cuda"), torch.zeros(n, dtype=torch.float64, device="cuda")
        for i, (x, m, v) in enumerate(before):
            want, wm, wv, up = reference(x, g[i].float(), m, v, wd[i], lr, b, eps, t)
            assert ((p[i].double() - want).abs() <= 2.0 ** -23 * (want.abs() + x.abs().double()) + 2.0 ** -19 * up + 1e-30).all(), i
            assert torch.equal(s16[i], p[i].bfloat16())
            o = opt.plan.first_block[i] * BLOCK
            at = slice(o, o + x.numel())
            m64[at], v64[at], live[at] = wm.reshape(-1), wv.reshape(-1), True
        m, v = opt.state_values(torch.float32)
        if bits == 32:
            assert ((m.double() - m64).abs() <= 2.0 ** -22 * (m64.abs() + 2e-3)).all() and ((v.double() - v64).abs() <= 2.0 ** -21 * v64).all()
        else:
            for got, want, r, low, top in ((m.abs(), m64.abs(), rm, -6, 448.0), (v, v64, rv, 3, 1.875 * 2.0 ** 33)):
                chosen, other, clear, _ = quantized(want, r, low, top)
                if low == 3:  # a non-zero second moment never becomes zero
                    unit = torch.exp2(opt.exp_avg_sq_scale.double() - 127)[:, None].expand(-1, BLOCK).reshape(-1)
                    chosen, other = (torch.where(want > 0, torch.maximum(c, unit), c) for c in (chosen, other))
                ok = (got.double() == chosen) | (~clear & (got.double() == other))
                assert ok.all(), ((~ok).sum().item(), got[~ok][:4], chosen[~ok][:4], want[~ok][:4])
                assert clear.double().mean() > 0.99
            assert (m.sign().double() * m64.sign() >= 0).all()
            m16, v16 = opt.state_values()
            assert torch.equal(m16.float(), m) and torch.equal(v16.float(), v)
        assert (m[~live] == 0).all() and (v[~live] == 0).all()


def test_more_tensors_than_one_launch_takes(M):
    """1500 tensors: three launches, one step counted; equal to the same tensors in lists of 100."""
    shapes = [(1 + 37 * i % 700,) for i in range(1500)]
    p, g, _ = tensors(shapes, torch.float32)
    q = [x.clone() for x in p]
    opt = M.MultiAdamW(p, state_bits=32, lr=1e-2)
    parts = [M.MultiAdamW(q[i:i + 100], state_bits=32, lr=1e-2) for i in range(0, 1500, 100)]
    for _ in range(2):
        opt.step(g)
        for k, o in enumerate(parts):
            o.step(g[100 * k:100 * k + 100])
    assert opt.step_t.item() == 2
    assert all(torch.equal(a, b) for a, b in zip(p, q))


def test_bits_are_repeated_and_seeded(M):
    shapes = [(1000,), (4096,)]
    runs = []
    for seed in (1, 1, 2):
        p, g, _ = tensors(shapes, torch.float32)
        opt = M.MultiAdamW(p, state_bits=8, seed=seed)
        for _ in range(3):
            opt.step(g)
        runs.append((p, opt.exp_avg.view(torch.uint8), opt.exp_avg_sq))
    assert all(torch.equal(a, b) for a, b in zip(runs[0][0], runs[1][0]))
    assert torch.equal(runs[0][1], runs[1][1]) and torch.equal(runs[0][2], runs[1][2])
    assert not torch.equal(runs[0][1], runs[2][1]) and not torch.equal(runs[0][2], runs[2][2])


def test_missing_gradients_clearing_and_scale(M):
    p, g, s16 = tensors([(300,), (700,), (50,)], torch.bfloat16)
    q, h, _ = tensors([(300,), (700,), (50,)], torch.bfloat16)
    a = M.MultiAdamW(p, s16, state_bits=8, zero_grad=True, grad_scale=0.5)
    scale = torch.tensor([0.5], device="cuda")
    b = M.MultiAdamW(q, state_bits=8, grad_scale=scale)
    keep = p[1].clone()
    a.step([g[0], None, g[2]])
    b.step([h[0], None, h[2]])
    assert torch.equal(p[1], keep) and (s16[1] == 0).all()
    o = a.plan.first_block[1]
    assert (a.exp_avg_scale[o:o + 3] == 1).all() and (a.exp_avg_sq[o * 256:(o + 3) * 256] == 0).all()
    assert (g[0] == 0).all() and (g[2] == 0).all() and (g[1] != 0).any() and (h[0] != 0).any()
    assert torch.equal(p[0], q[0]) and torch.equal(p[2], q[2]) and torch.equal(a.exp_avg_sq, b.exp_avg_sq)
    b.step([None, None, None])
    assert b.step_t.item() == 2 and torch.equal(p[0], q[0])
    scale.fill_(0.0)
    b.step(h)
    assert not torch.equal(p[0], q[0])


@pytest.mark.parametrize("bits", [8, 32])
def test_captured_steps_match_eager_ones(M, bits):
    runs = []
    for graph in (False, True):
        p, g, s16 = tensors([(5000,), (77, 3)], torch.float32)
        opt = M.MultiAdamW(p, s16, grads=g, state_bits=bits, lr=1e-2)
        step = opt.step
        if graph:
            gr = torch.cuda.CUDAGraph()
            with torch.cuda.graph(gr):
                opt.step()
            step = gr.replay
        for i in range(4):
            if i == 2:
                opt.set_lr(1e-3)
            for x in g:
                x.mul_(1.25)
            step()
        assert opt.step_t.item() == 4
        runs.append((p, s16, opt.state_values(torch.float32)))
    for a, b in zip(*runs):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_extreme_values(M):
    """Zero blocks, blocks across the whole range, values far below their block's largest, infinities and NaN."""
    p = [torch.ones(256 * 6, device="cuda")]
    g = torch.zeros(6, 256, device="cuda")
    g[1] = torch.logspace(-19, 0, 256, device="cuda")
    g[2, ::2], g[2, 1::2] = 1e-19, -1e-16
    g[3], g[3, 5] = 1e18, -1e-3
    g[4, 7], g[5, 9], g[5, 10] = float("nan"), float("inf"), 1.0
    opt = M.MultiAdamW(p, state_bits=8, lr=1e-3, weight_decay=0.0, betas=(0.9, 0.999))
    opt.step([g.view(-1)])
    m, v = (x.view(6, 256) for x in opt.state_values(torch.float32))
    new = p[0].view(6, 256)
    assert (new[0] == 1).all() and (m[0] == 0).all() and (v[0] == 0).all()
    for i in (1, 2, 3):
        assert new[i].isfinite().all() and (v[i][g[i] ** 2 * 0.001 > 0] > 0).all()
    top = g[1] > 1e-3
    assert (((m[1] - 0.1 * g[1]) / (0.1 * g[1]))[top].abs() <= 0.126).all()  # a step of 2^-3 at the most
    assert (((v[1] - 0.001 * g[1] ** 2) / (0.001 * g[1] ** 2))[top].abs() <= 0.126).all()
    assert new[4, 7].isnan() and m[4, 7].isnan() and new[4].isnan().sum() == 1 and m[4].isnan().sum() == 1
    assert new[5].isnan().sum() == 1 and new[5, 9].isnan()
    zeros = torch.zeros_like(g).view(-1)
    for _ in range(3):
        opt.step([zeros])
    good = torch.ones(6, 256, dtype=torch.bool, device="cuda")
    good[4, 7] = good[5, 9] = False
    assert p[0].view(6, 256)[good].isfinite().all()


def test_second_moment_follows_small_steps(M):
    """b2 = 0.999: a step moves v by 0.1 percent, far under its format's 12. Rounding to nearest would leave it
    where it started; the mean over 65536 values follows. The standard deviation of a value is under 0.5 of
    it (0.25 in equilibrium), of the mean under 0.002; six of those and the mean's own lag stay under 0.05."""
    n = 65536
    p = [torch.zeros(n, device="cuda")]
    opt = M.MultiAdamW(p, state_bits=8, lr=0.0, weight_decay=0.0, betas=(0.9, 0.999))
    g = [torch.full((n,), 1e-3, device="cuda")]
    for t in range(3000):
        opt.step(g)
    m, v = opt.state_values(torch.float32)
    want = 1e-6 * (1 - 0.999 ** 3000)
    assert abs(v[:n].double().mean().item() / want - 1) < 0.05
    assert abs(m[:n].double().mean().item() / 1e-3 - 1) < 0.01  # steps of 10 percent: spread 0.1 / 256 over the values


@pytest.mark.parametrize("bits", [8, 32])
def test_checkpoint_round_trip(M, bits):
    p, g, _ = tensors([(1000, 3), (77,)], torch.float32)
    opt = M.MultiAdamW(p, state_bits=bits, lr=1e-2, seed=3)
    for _ in range(3):
        opt.step(g)
    sd = opt.state_dict()
    q = [x.clone() for x in p]
    new = M.MultiAdamW(q, state_bits=bits, lr=1.0, seed=3)
    new.load_state_dict(sd)
    assert new.lr == opt.lr and new.step_t.item() == 3
    for a, b in zip(opt.state_values(torch.float32), new.state_values(torch.float32)):
        assert torch.equal(a, b)
    opt.step(g)
    new.step(g)
    assert all(torch.equal(a, b) for a, b in zip(p, q))


def test_matches_the_flat_optimizer(M):
    """32-bit states: the update of FusedAdamW, to the roundings of two orders of the same formula."""
    from llmt.optim.adamw import FusedAdamW
    n = 256 * 40
    gen = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(n, device="cuda", generator=gen) * 0.02
    g = torch.randn(n, device="cuda", generator=gen) * 1e-3
    a, sa = x.clone(), torch.empty(n, device="cuda", dtype=torch.bfloat16)
    flat = FusedAdamW(a, g, sa, lr=1e-3, zero_grad=False)
    b = [t.clone() for t in x.split(1000)]
    opt = M.MultiAdamW(b, lr=1e-3, state_bits=32)
    for _ in range(5):
        flat.step()
        opt.step(list(g.split(1000)))
    # five steps of at most 1e-3 / (1 - b1) times their relative error 2^-19, and the sums' own roundings
    assert (torch.cat(b) - a).abs().max().item() < 5 * (1e-2 * 2.0 ** -19 + 2.0 ** -23 * 0.2)
