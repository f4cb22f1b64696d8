"""The losses on rows of a few ids at every alignment in the bounds-checked build: no access outside a buffer is recorded,
also where a row has no whole 16-byte piece. In a child process, as the module is chosen when it is first imported."""
import json
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu


def run():
    import torch
    from llmt.ops import losses
    from llmt.ops import native as N
    records = {}
    for dt in (torch.float32, torch.bfloat16, torch.float16):
        for V in (1, 2, 3, 5, 7, 9, 17):
            for pad in range(9):
                z = torch.randn(2, 3, V + pad, device="cuda").to(dt)[:, :, pad:]
                y = torch.randint(0, V, (2, 3), device="cuda")
                y[0, 1] = -100
                losses.logprob_rows(z, y)
                losses.preference_loss_rows(z, y)
                losses.policy_loss_rows(z, y, None, torch.ones(2, 1, device="cuda"))
                losses.policy_loss_rows(z, y, None, torch.ones(2, 1, device="cuda"), out=z)
                r = N.ext().bounds_error(True)
                if r:
                    records[f"{dt} {V} {pad}"] = r >> 40 & 0x7FFFFF
    return {"checking": N.ext().bounds_checking(), "records": records}


def test_rows_of_a_few_ids():
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    out = subprocess.run([sys.executable, "-m", "tests.test_losses_bounds_gpu"], cwd=root, env=dict(os.environ, LLMT_BOUNDS="1", PYTHONPATH=root),
                         capture_output=True, text=True, timeout=300)
    assert out.returncode == 0, out.stdout[-2000:] + out.stderr[-2000:]
    got = json.loads(out.stdout.strip().splitlines()[-1])
    assert got == {"checking": True, "records": {}}


if __name__ == "__main__":
    print(json.dumps(run()))
