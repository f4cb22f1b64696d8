"""Rotary positions against the rotation in fp64.

Tolerance: the table's values are off by 2^-25 of their size, each complex product adds 2^-23, so the
cosine and sine by under 2^-21.5 of the factor for two products; fp64 angles up to 2^31 are off by
2^-22; the rotation adds two roundings: an fp32 result is off by 2^-20 (|x1| + |x2|) times the
factor, and a rounding to u = eps / 2 comes on top (fp16 below its normal range: 2^-25)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SCALINGS = {
    "none": None, "linear": {"type": "linear", "factor": 4.0}, "ntk": {"type": "ntk", "factor": 8.0},
    "llama3": {"type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
               "original_max_position": 8192},
    "yarn": {"type": "yarn", "factor": 16.0, "original_max_position": 4096},
}


@pytest.fixture(scope="module")
def R():
    from llmt.ops import native, rotary
    native.ext()
    return rotary


def oracle(x, pos, w, factor, rd, interleaved, inverse):
    """(rotated x, sum of the sizes of each pair) in fp64; x (B, T, H, hd), pos (B, T)."""
    a = pos.double()[..., None] * w.to(x.device) * (-1.0 if inverse else 1.0)
    z = torch.polar(torch.full_like(a, factor), a)[:, :, None]
    xd = x.double()
    e, o = (xd[..., 0:rd:2], xd[..., 1:rd:2]) if interleaved else (xd[..., :rd // 2], xd[..., rd // 2:rd])
    y = torch.complex(e.contiguous(), o.contiguous()) * z
    size = (e.abs() + o.abs()) * factor
    out, mag = xd.clone(), torch.zeros_like(xd)
    if interleaved:
        out[..., 0:rd:2], out[..., 1:rd:2] = y.real, y.imag
        mag[..., 0:rd:2], mag[..., 1:rd:2] = size, size
    else:
        out[..., :rd // 2], out[..., rd // 2:rd] = y.real, y.imag
        mag[..., :rd // 2], mag[..., rd // 2:rd] = size, size
    return out, mag


def check(got, x, pos, w, factor, rd, interleaved, inverse):
    want, mag = oracle(x, pos, w, factor, rd, interleaved, inverse)
    u = torch.finfo(got.dtype).eps / 2
    tiny = 2.0 ** -25 if got.dtype == torch.float16 else 0.0
    assert ((got.double() - want).abs() <= u * want.abs() * 1.0001 + tiny + 2.0 ** -20 * mag).all()
    assert torch.equal(got[..., rd:], x[..., rd:])


CASES = [  # B, T, H, KV, hd, rd
    (1, 1, 1, 1, 2, 2), (2, 3, 2, 1, 64, 64), (1, 7, 5, 2, 80, 80), (3, 5, 4, 4, 96, 48), (2, 33, 8, 2, 128, 128),
    (64, 1, 32, 8, 128, 128), (1, 2, 3, 1, 66, 22), (2, 129, 16, 16, 64, 32), (1, 5, 71, 1, 64, 64), (1, 4, 2, 1, 256, 64),
    (1, 1000, 6, 2, 128, 128), (2, 3, 3, 3, 20, 10),
]


@pytest.mark.parametrize("B,T,H,KV,hd,rd", CASES)
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rotate(R, B, T, H, KV, hd, rd, dtype, interleaved):
    g = torch.Generator(device="cuda").manual_seed(hd + T)
    qkv = torch.randn(B, T, H + 2 * KV, hd, device="cuda", generator=g).to(DT[dtype])
    q, k = qkv[:, :, :H], qkv[:, :, H:H + KV]
    pos = torch.randint(0, 2 ** 20, (B, T), device="cuda", generator=g)
    pos[0, 0] = 2 ** 31 - 1
    pos[-1, -1] = -77777
    names = sorted(SCALINGS) if rd > 2 else ["none", "linear"]
    sc = SCALINGS[names[(B + T + hd) % len(names)]]
    rot = R.Rotary(hd, rotary_dim=rd, base=10000.0, interleaved=interleaved, scaling=sc)
    before = qkv.clone()
    for inverse in (False, True):
        for p in (pos, pos.int()):
            qo, ko = rot.rotate(q, k, p, inverse=inverse)
            check(qo, q, pos, rot.inv_freq, rot.factor, rd, interleaved, inverse)
            check(ko, k, pos, rot.inv_freq, rot.factor, rd, interleaved, inverse)
    assert torch.equal(qkv, before)
    # in place through the strided views: v and the other results stay
    rot.rotate(q, k, pos, inverse=True, q_out=q, k_out=k)
    assert torch.equal(qkv[:, :, :H], qo) and torch.equal(qkv[:, :, H:H + KV], ko)
    assert torch.equal(qkv[:, :, H + KV:], before[:, :, H + KV:])


def test_views_and_positions(R):
    rot = R.Rotary(64)
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(3, 6, 4, 64, device="cuda", generator=g)
    base = rot.rotate(x)[0]  # positions 0 .. 5
    check(base, x, torch.arange(6, device="cuda").expand(3, 6), rot.inv_freq, 1.0, 64, False, False)
    pos = torch.arange(6, device="cuda")
    for p in (pos, pos[None], pos.int().expand(3, 6), torch.stack([pos] * 6, 1)[:, 2][None]):
        assert torch.equal(rot.rotate(x, None, p)[0], base)
    # (B, H, T, hd) storage, a row pitch off 16 bytes, an odd start
    t = x.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3)
    assert torch.equal(rot.rotate(t)[0], base)
    for dt in (torch.float32, torch.bfloat16):
        wide = torch.full((3, 6, 4, 67), 7.0, device="cuda", dtype=dt)
        wide[..., 1:65] = x.to(dt)
        out = torch.full((3, 6, 4, 71), 5.0, device="cuda", dtype=dt)
        y = rot.rotate(wide[..., 1:65], q_out=out[..., 3:67])[0]
        assert torch.equal(y, rot.rotate(x.to(dt))[0])
        assert (out[..., :3] == 5).all() and (out[..., 67:] == 5).all() and (wide[..., 65:] == 7).all()
    assert torch.equal(rot.rotate(x[:, :, :1].expand(3, 6, 4, 64))[0], base[:, :, :1].expand(3, 6, 4, 64))
    far = rot.rotate(x[:1, :3], None, torch.tensor([[2 ** 31, -2 ** 31, -2 ** 63]], device="cuda"))[0]
    assert far.isnan().all()
    assert rot.rotate(x[:, :0])[0].shape == (3, 0, 4, 64)
    assert rot.rotate(x[:, :, :0], x, pos)[1].equal(base)


def test_inverse_and_gradient(R):
    rot = R.Rotary(128, rotary_dim=64, interleaved=True, scaling=SCALINGS["yarn"])
    g = torch.Generator(device="cuda").manual_seed(4)
    q = torch.randn(2, 9, 4, 128, device="cuda", generator=g)
    k = torch.randn(2, 9, 2, 128, device="cuda", generator=g)
    pos = torch.randint(0, 100000, (2, 9), device="cuda", generator=g)
    ql, kl = q.clone().requires_grad_(), k.clone().requires_grad_()
    y, z = rot.apply(ql, kl, pos)
    dy, dz = torch.randn_like(y).transpose(1, 2).contiguous().transpose(1, 2), torch.randn_like(z)
    torch.autograd.backward([y, z], [dy, dz])
    check(ql.grad, dy, pos, rot.inv_freq, rot.factor, 64, True, True)
    check(kl.grad, dz, pos, rot.inv_freq, rot.factor, 64, True, True)
    # <y, dy> = <x, dx>: the gradient is the transposed map; 2 * 9216 products of size about 2, each 2^-20 off
    assert abs((y.double() * dy.double()).sum() - (q.double() * ql.grad.double()).sum()) < 0.04
    one = q.clone().requires_grad_()
    out, none = rot.apply(one, None, pos)
    assert none is None and torch.equal(out, y)
    out.sum().backward()  # an expanded gradient (stride 0)
    check(one.grad, torch.ones_like(q), pos, rot.inv_freq, rot.factor, 64, True, True)


def test_graph_and_stream(R):
    rot = R.Rotary(64)
    q = torch.randn(2, 8, 4, 64, device="cuda").bfloat16()
    pos = torch.zeros(2, 8, dtype=torch.int32, device="cuda")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y, z = rot.rotate(q, q[:, :, :2], pos)
    s = torch.cuda.Stream()
    for start in (3, 70000):
        pos.copy_(start + torch.arange(16, device="cuda").view(2, 8))
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            g.replay()
            other = rot.rotate(q, None, pos)[0]
        torch.cuda.current_stream().wait_stream(s)
        check(y, q, pos, rot.inv_freq, 1.0, 64, False, False)
        assert torch.equal(other, y) and torch.equal(z, y[:, :, :2])


def test_tables_match_the_kernel(R):
    """The fused qkv path's tables turn whole heads as rotate() does."""
    from llmt.models.llama import rope
    rot = R.Rotary(64, base=500000.0, scaling=SCALINGS["llama3"])
    x = torch.randn(1, 200, 3, 64, device="cuda")
    cos, sin = rot.tables(200)
    want = rope(x.transpose(1, 2), cos, sin).transpose(1, 2)
    got = rot.rotate(x)[0]
    mag = oracle(x, torch.arange(200, device="cuda")[None], rot.inv_freq, 1.0, 64, False, False)[1]
    assert ((got - want).abs() <= 2.0 ** -19 * mag).all()


def test_large_rows(R):
    """Values past 2^31 elements of one tensor."""
    if torch.cuda.get_device_properties(0).total_memory < 60 << 30:
        pytest.skip("needs 20 GB")
    rot = R.Rotary(128)
    x = torch.zeros(1, 2 ** 20 + 5, 17, 128, device="cuda", dtype=torch.bfloat16)
    x[0, -3:] = torch.randn(3, 17, 128, device="cuda").bfloat16()
    y = rot.rotate(x, q_out=x)[0]
    assert y.data_ptr() == x.data_ptr() and (x[0, :-3] == 0).all() and math.isfinite(x[0, -3:].float().sum().item())
    assert (x[0, -3:] != 0).any()
