"""Rotary outputs that overlap an operand are refused, byte by byte: heads of packed rows that lie between one
another's are not."""
import itertools
import random

import pytest
import torch

from llmt.ops import native
from llmt.ops.rotary import Rotary

if not native.available():
    pytest.skip("extension not built", allow_module_level=True)


def refusal(q, k=None, positions=None, **kw):
    """What rotate() says on the CPU: an overlap, or at last that the tensors are not on a GPU."""
    with pytest.raises(RuntimeError) as e:
        Rotary(q.shape[-1], device="cpu").rotate(q, k, positions, **kw)
    return str(e.value)


def test_outputs_over_the_other_operand():
    rows = torch.zeros(2, 3, 12, 8)
    q, k = rows[:, :, :4], rows[:, :, 4:6]
    assert "CUDA tensor" in refusal(q, k, q_out=q, k_out=k)
    assert "CUDA tensor" in refusal(q, k, q_out=rows[:, :, 6:10], k_out=rows[:, :, 10:])
    assert "k_out overlaps q" in refusal(q, k, k_out=rows[:, :, 3:5])
    assert "q_out overlaps k" in refusal(q, k, q_out=rows[:, :, 5:9])
    assert "q_out overlaps k_out" in refusal(q, k, q_out=rows[:, :, 6:10], k_out=rows[:, :, 9:11])
    flat = torch.zeros(2 * 3 * 4 * 8 + 100)
    a = flat[100:].view(2, 3, 4, 8)
    assert "k_out overlaps q" in refusal(a, torch.zeros(2, 3, 2, 8), k_out=flat[4:4 + 96].view(2, 3, 2, 8).as_strided((2, 3, 2, 8), (48, 16, 8, 1), 5))
    assert "CUDA tensor" in refusal(a, torch.zeros(2, 3, 2, 8), k_out=flat[4:100].view(2, 3, 2, 8))


def test_outputs_over_positions():
    buf = torch.zeros(200)
    pos = buf.view(torch.int32)[90:96].view(2, 3)
    out = buf[:96].view(2, 3, 2, 8)
    assert "q_out overlaps positions" in refusal(torch.zeros(2, 3, 2, 8), None, pos, q_out=out)
    assert "CUDA tensor" in refusal(torch.zeros(2, 3, 2, 8), None, buf.view(torch.int32)[96:102].view(2, 3), q_out=out)


def test_against_enumeration():
    """Random layouts of k_out over one buffer with q against the sets of their elements."""
    rng = random.Random(0)
    seen = {True: 0, False: 0}
    for _ in range(400):
        buf = torch.zeros(4000)
        B, T, hd = rng.randint(1, 3), rng.randint(1, 4), rng.choice([2, 4, 6])

        def view():
            H = rng.randint(1, 4)
            order = rng.sample([0, 1, 2], 3)
            size, st, step = [B, T, H], [0, 0, 0], hd + rng.randint(0, 6)
            for d in order:
                st[d] = step
                step = step * size[d] + rng.randint(0, 9)
            return buf.as_strided((B, T, H, hd), (*st, 1), rng.randint(0, 300))
        q, out = view(), view()
        k = torch.zeros(out.shape)
        places = [{x.storage_offset() + sum(i * s for i, s in zip(ix, x.stride())) for ix in itertools.product(*map(range, x.shape))}
                  for x in (q, out)]
        share = bool(places[0] & places[1])
        said = refusal(q, k, k_out=out)
        assert ("k_out overlaps q" in said or "k_out is q" in said) == share, (q.shape, q.stride(), out.shape, out.stride(), said)
        seen[share] += 1
    assert min(seen.values()) > 50
