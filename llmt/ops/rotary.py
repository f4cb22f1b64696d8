"""Rotary positions as a plan: frequencies with a long-context scaling, and the kernel that applies
them to q and k at any positions.

    rot = Rotary(128, base=500000.0, scaling={"type": "llama3", "factor": 8.0, "low_freq_factor": 1.0,
                 "high_freq_factor": 4.0, "original_max_position": 8192})
    q, k = rot.rotate(q, k, positions)            # (B, T, heads, 128), strided views welcome
    q, k = rot.apply(q, k, positions)             # the same behind autograd
    cos, sin = rot.tables(T)                      # (T, rotary_dim) for the fused qkv path

Scalings (w = base^(-2j / rotary_dim), L = original_max_position):
  linear  w / factor
  ntk     base grown by factor^(rd / (rd - 2)): the slowest pair is stretched by factor, the fastest kept
  llama3  pairs with fewer than low_freq_factor turns in L stretched by factor, with more than
          high_freq_factor kept, between them blended by their turns
  yarn    pairs between those that turn beta_fast and beta_slow times in L blended by their index;
          rotated values times attention_factor (0.1 ln(factor) + 1 unless given)
"""
from __future__ import annotations

import math

import torch
from torch.autograd.function import once_differentiable

from llmt.ops import native as N

TABLE_ROWS = 4096  # 1024 low digits, 1024 middle digits, 2048 high digits of the position

_KEYS = {"linear": ({"factor"}, set()), "ntk": ({"factor"}, set()),
         "llama3": ({"factor", "low_freq_factor", "high_freq_factor", "original_max_position"}, set()),
         "yarn": ({"factor", "original_max_position"}, {"beta_fast", "beta_slow", "attention_factor"})}


def frequencies(rotary_dim, base=10000.0, scaling=None):
    """(angle per position of each pair, fp64 (rotary_dim / 2) on the CPU; factor on the values)."""
    if rotary_dim <= 0 or rotary_dim % 2:
        raise ValueError(f"rotary_dim must be even and positive, not {rotary_dim}")
    base = float(base)
    if not base > 0:
        raise ValueError("base must be positive")
    sc = dict(scaling) if scaling else {"type": "none"}
    kind = sc.pop("type", None)
    if kind == "none":
        sc.clear()
    elif kind not in _KEYS:
        raise ValueError(f"scaling type must be one of {', '.join(_KEYS)}, not {kind!r}")
    else:
        need, may = _KEYS[kind]
        if need - set(sc) or set(sc) - need - may:
            raise ValueError(f"{kind} scaling takes {sorted(need)}" + (f" and may take {sorted(may)}" if may else "")
                             + f", got {sorted(sc)}")
        for key, v in sc.items():
            if not float(v) > 0:
                raise ValueError(f"{key} must be positive, not {v}")
    f = float(sc.get("factor", 1.0))
    if kind == "ntk":
        if rotary_dim <= 2:
            raise ValueError("ntk scaling needs rotary_dim above 2")
        base *= f ** (rotary_dim / (rotary_dim - 2.0))
    j = torch.arange(rotary_dim // 2, dtype=torch.float64)
    w = torch.pow(torch.tensor(base, dtype=torch.float64), -2.0 * j / rotary_dim)
    if kind == "linear":
        return w / f, 1.0
    if kind == "llama3":
        lo, hi = float(sc["low_freq_factor"]), float(sc["high_freq_factor"])
        if not lo < hi:
            raise ValueError("low_freq_factor must be below high_freq_factor")
        kept = ((sc["original_max_position"] * w / (2 * math.pi) - lo) / (hi - lo)).clamp_(0.0, 1.0)
        return w * (kept + (1.0 - kept) / f), 1.0
    if kind == "yarn":
        fast, slow = float(sc.get("beta_fast", 32.0)), float(sc.get("beta_slow", 1.0))
        if not slow < fast:
            raise ValueError("beta_slow must be below beta_fast")

        def index(turns):  # of the pair that turns this often within the original context
            return rotary_dim * math.log(sc["original_max_position"] / (2 * math.pi * turns)) / (2 * math.log(base))
        lo, hi = max(math.floor(index(fast)), 0), min(math.ceil(index(slow)), rotary_dim - 1)
        stretched = ((j - lo) / max(hi - lo, 1e-3)).clamp_(0.0, 1.0)
        return w * (1.0 - stretched + stretched / f), float(sc.get("attention_factor", 0.1 * math.log(f) + 1.0))
    return w, 1.0


def position_tables(T, rotary_dim, base=10000.0, scaling=None, device="cpu"):
    """(cos, sin), each (T, rotary_dim) fp32 with both halves alike, for positions 0 .. T - 1; angles in fp64."""
    inv_freq, factor = frequencies(rotary_dim, base, scaling)
    angle = (torch.arange(T, dtype=torch.float64)[:, None] * inv_freq).repeat(1, 2)
    return (angle.cos() * factor).float().to(device), (angle.sin() * factor).float().to(device)


class Rotary:
    def __init__(self, head_dim, rotary_dim=None, base=10000.0, interleaved=False, scaling=None, device="cuda"):
        self.head_dim = int(head_dim)
        self.rotary_dim = int(rotary_dim) if rotary_dim is not None else self.head_dim
        if not 0 < self.rotary_dim <= self.head_dim:
            raise ValueError(f"rotary_dim must be in (0, head_dim = {self.head_dim}], not {self.rotary_dim}")
        self.interleaved, self.base, self.scaling = bool(interleaved), base, scaling
        self.inv_freq, self.factor = frequencies(self.rotary_dim, base, scaling)
        digit = torch.arange(TABLE_ROWS, device=device)  # made on the device: 0.1 ms in place of 2
        low, middle = digit < 1024, digit < 2048
        digit = torch.where(low, digit, torch.where(middle, (digit - 1024) << 10, (digit - 2048) << 20)).double()
        angle = digit[:, None] * self.inv_freq.to(device)
        size = (1.0 + low.double() * (self.factor - 1.0))[:, None]
        self.table = torch.stack([angle.cos() * size, angle.sin() * size], -1).float().contiguous()

    def tables(self, T, device=None):
        """(cos, sin), each (T, rotary_dim) fp32 with both halves alike, for positions 0 .. T - 1: the
        tables of the fused qkv path (which rotates half pairs of whole heads)."""
        return position_tables(T, self.rotary_dim, self.base, self.scaling, self.table.device if device is None else device)

    def rotate(self, q, k=None, positions=None, inverse=False, q_out=None, k_out=None):
        """(q, k) turned to their positions: q (B, T, H, head_dim), k (B, T, KV, head_dim) or None, bf16 /
        fp16 / fp32 with unit stride along head_dim. positions: int32 or int64, (B, T) or (T,), None
        for 0 .. T - 1; a position outside (-2^31, 2^31) gives NaN. inverse turns back (with the
        scaling's factor, it is the gradient of the rotation). q_out / k_out take the results; they may be q and
        k themselves, and otherwise overlap no other operand. Returns new contiguous tensors otherwise."""
        if q.shape[-1] != self.head_dim:
            raise ValueError(f"head_dim of q is {q.shape[-1]}, of the plan {self.head_dim}")
        y, z = N.ext().rotary(q, k, positions, self.table, self.rotary_dim, self.interleaved, bool(inverse), q_out, k_out)
        return y, (z if k is not None else None)

    def apply(self, q, k=None, positions=None):
        """rotate behind autograd; the backward is one inverse rotation of both gradients. Before it is
        captured into a CUDA graph, drop the results of eager calls on the same leaves."""
        if k is None:
            return _RotateOne.apply(q, positions, self), None
        return _RotateBoth.apply(q, k, positions, self)


def _rows(g):
    return g if g.stride(-1) == 1 else g.contiguous()


class _RotateBoth(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, positions, rot):
        ctx.rot = rot
        ctx.save_for_backward(positions)
        return rot.rotate(q.detach(), k.detach(), positions)

    @staticmethod
    @once_differentiable
    def backward(ctx, dq, dk):
        (positions,) = ctx.saved_tensors
        dq, dk = ctx.rot.rotate(_rows(dq), _rows(dk), positions, inverse=True)
        return dq, dk, None, None


class _RotateOne(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, positions, rot):
        ctx.rot = rot
        ctx.save_for_backward(positions)
        return rot.rotate(q.detach(), None, positions)[0]

    @staticmethod
    @once_differentiable
    def backward(ctx, dq):
        (positions,) = ctx.saved_tensors
        return ctx.rot.rotate(_rows(dq), None, positions, inverse=True)[0], None, None
