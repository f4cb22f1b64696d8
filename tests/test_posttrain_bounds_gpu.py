"""The post-training kernels in the bounds-checked build: ragged rows, odd alignments and strided heads leave
no record of an access outside its buffer, and give the release build's results. Run in a child process,
as the module is chosen when it is first imported."""
import json
import os
import subprocess
import sys

import pytest
import torch

pytestmark = pytest.mark.gpu


def run_ops():
    """Sums of every op's outputs on ragged shapes."""
    from llmt.ops import losses
    from llmt.ops.rotary import Rotary
    from llmt.optim.multi import MultiAdamW
    g = torch.Generator(device="cuda").manual_seed(0)
    res = {}
    for V, dt in ((7, torch.float32), (1001, torch.bfloat16), (40003, torch.float16), (140001, torch.float32)):
        for pad in (0, 3):
            buf = torch.randn(4, 3, V + 2 * pad, device="cuda", generator=g).to(dt)
            z = buf[:, :, pad:pad + V]
            y = torch.randint(0, V, (4, 3), device="cuda", generator=g)
            y[1, 1] = V  # does not count
            adv = torch.randn(4, 1, device="cuda", generator=g)
            r = losses.policy_loss_rows(z, y, None, adv, out=z if pad else None)
            res[f"policy {V} {pad}"] = [r.loss.item(), r.dlogits.double().abs().sum().item()]
            q = losses.preference_loss_rows(z.clone(), y, kind="ipo")
            res[f"preference {V} {pad}"] = [q.loss.item(), q.dlogits.double().abs().sum().item()]
    for off in (0, 1):
        p = [torch.randn(n + off, device="cuda", generator=g)[off:] for n in (1, 256, 1000, 70000)]
        grads = [torch.randn(n + off, device="cuda", generator=g)[off:] for n in (1, 256, 1000, 70000)]
        for bits in (8, 32):
            opt = MultiAdamW([x.clone() if not off else x for x in p], state_bits=bits)
            opt.step(grads)
            res[f"adamw {off} {bits}"] = [sum(x.double().sum().item() for x in opt.params)]
    for hd, rd, pad in ((64, 64, 0), (96, 48, 0), (66, 22, 1), (128, 128, 8)):
        x = torch.randn(2, 5, 7, hd + pad, device="cuda", generator=g).bfloat16()[..., :hd]
        rot = Rotary(hd, rotary_dim=rd, interleaved=pad > 0)
        a, b = rot.rotate(x[:, :, :5], x[:, :, 5:])
        rot.rotate(x[:, :, :5], x[:, :, 5:], q_out=x[:, :, :5], k_out=x[:, :, 5:])
        res[f"rotary {hd} {rd}"] = [a.double().sum().item(), b.double().sum().item(), x.double().sum().item()]
    torch.cuda.synchronize()
    return res


def test_bounds_checked_build_agrees():
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    env = dict(os.environ, LLMT_BOUNDS="1", PYTHONPATH=root)
    out = subprocess.run([sys.executable, "-m", "tests.test_posttrain_bounds_gpu"], cwd=root, env=env, capture_output=True,
                         text=True, timeout=600)
    assert out.returncode == 0, out.stdout[-2000:] + out.stderr[-2000:]
    got = json.loads(out.stdout.strip().splitlines()[-1])
    assert got["bounds_checking"] is True and got["record"] == 0, got
    want = run_ops()
    for k, v in want.items():  # the same arithmetic in another build
        assert all(abs(a - b) <= 1e-5 * (1 + abs(a)) for a, b in zip(v, got["ops"][k])), (k, v, got["ops"][k])


if __name__ == "__main__":
    from llmt.ops import native as N
    ops = run_ops()
    print(json.dumps({"bounds_checking": N.ext().bounds_checking(), "record": N.ext().bounds_error(True), "ops": ops}))
