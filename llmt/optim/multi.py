"""AdamW over a list of tensors in one launch, with states in 8 bits or in 32.

The update is FusedAdamW's (torch.optim.AdamW's), for tensors that need not lie in one flat buffer,
each with its own weight decay. With state_bits=8 the two moments take 2 bytes and 2/256 per value
in place of 8: blocks of 256 values under a power-of-two scale, the first moment in e4m3, the second
in eight unsigned bits (csrc/adamw/adamw_multi.cu), rounded up or down with probabilities that keep their
mean. An update is computed from the moments before that rounding, with the approximate square root
and quotient (2^-22 of it; with 32-bit states both are correctly rounded). The random bits are a hash
of the value's place, the step count and the seed: the same run gives the same bits. A NaN gradient
makes its value and its first moment NaN, as in 32 bits.

lr and the step count live on the device, so `step()` can be captured in a CUDA graph and replayed.
"""
from __future__ import annotations

import torch

from llmt.ops import native as N

BLOCK = 256


class MultiAdamW:
    def __init__(self, params, shadows=None, grads=None, lr=3e-4, betas=(0.9, 0.95), eps=1e-8, weight_decay=0.1,
                 state_bits=8, seed=0, grad_scale=1.0, zero_grad=False):
        """params: fp32 tensors; shadows: a bf16 copy of each, written by every step, or None;
        grads: the gradient buffers step() reads when it is given none; weight_decay: one for all or one
        per tensor; grad_scale: multiplies the gradients, a number or a one-element device tensor;
        zero_grad: clear the gradients after reading them."""
        if state_bits not in (8, 32):
            raise ValueError(f"state_bits must be 8 or 32, not {state_bits}")
        b1, b2 = betas
        if not (0.0 <= b1 < 1.0 and 0.0 <= b2 < 1.0):
            raise ValueError(f"betas must be in [0, 1), not {betas}")
        if not eps >= 0.0:
            raise ValueError(f"eps must be at least 0, not {eps}")
        params = [p.detach() for p in params]
        wd = [float(w) for w in weight_decay] if isinstance(weight_decay, (list, tuple)) else [float(weight_decay)] * len(params)
        self.plan = N.ext().MultiPlan(params, [s.detach() for s in shadows] if shadows is not None else [], wd)
        self.params, self.grads = params, (list(grads) if grads is not None else None)
        self.state_bits, self.seed, self.zero_grad = int(state_bits), int(seed) & 0xFFFFFFFF, bool(zero_grad)
        self.betas, self.eps, self.weight_decay, self.grad_scale = (b1, b2), eps, weight_decay, grad_scale
        dev = params[0].device
        n = self.plan.blocks * BLOCK
        self.lr_t = torch.full((1,), float(lr), dtype=torch.float32, device=dev)
        self.step_t = torch.zeros(1, dtype=torch.int32, device=dev)
        self.ticket = torch.zeros(1, dtype=torch.int32, device=dev)
        self.exp_avg_scale = self.exp_avg_sq_scale = None
        if state_bits == 8:
            self.exp_avg = torch.zeros(n, dtype=torch.uint8, device=dev).view(torch.float8_e4m3fn)
            self.exp_avg_sq = torch.zeros(n, dtype=torch.uint8, device=dev)
            self.exp_avg_scale = torch.ones(self.plan.blocks, dtype=torch.uint8, device=dev)
            self.exp_avg_sq_scale = torch.ones(self.plan.blocks, dtype=torch.uint8, device=dev)
        else:
            self.exp_avg = torch.zeros(n, dtype=torch.float32, device=dev)
            self.exp_avg_sq = torch.zeros(n, dtype=torch.float32, device=dev)

    @property
    def lr(self):
        return float(self.lr_t.item())

    def set_lr(self, lr):
        self.lr_t.fill_(float(lr))

    @torch.no_grad()
    def step(self, grads=None):
        """One step on `grads` (one per tensor, all fp32 or all bf16; None leaves a tensor and its states
        as they are) or on the buffers given at construction. The step count, and with it the bias
        correction, is one for all tensors, those left out included. With zero_grad the gradients may not overlap."""
        grads = self.grads if grads is None else grads
        if grads is None:
            raise ValueError("no gradients: give them to step() or to MultiAdamW")
        scale, dev_scale = (1.0, self.grad_scale) if isinstance(self.grad_scale, torch.Tensor) else (float(self.grad_scale), None)
        N.LAUNCHES.count += self.plan.step(
            grads if isinstance(grads, list) else list(grads), self.state_bits, self.exp_avg, self.exp_avg_sq,
            self.exp_avg_scale, self.exp_avg_sq_scale, self.lr_t, self.step_t, self.ticket, self.betas[0], self.betas[1],
            self.eps, scale, dev_scale, self.seed, self.zero_grad)

    def state_values(self, dtype=torch.bfloat16):
        """The two moments of every tensor, flat in blocks of 256 (tensor i from plan.first_block[i] * 256
        on). 8-bit states are decoded, to bf16 (exact) or fp32; 32-bit states are returned as they are."""
        if self.state_bits == 32:
            return self.exp_avg, self.exp_avg_sq
        if dtype not in (torch.bfloat16, torch.float32):
            raise ValueError(f"dtype must be torch.bfloat16 or torch.float32, not {dtype}")
        return tuple(N.ext().adamw_state_values(self.exp_avg, self.exp_avg_scale, self.exp_avg_sq, self.exp_avg_sq_scale,
                                                dtype == torch.float32))

    # ------------------------------------------------------------------ checkpoints
    def tensor_state(self, i):
        """(exp_avg, exp_avg_sq) of tensor i, fp32 in its shape: decoded from its own blocks, with 32-bit
        states views of them."""
        p, b = self.params[i], self.plan.first_block[i]
        k = -(-p.numel() // BLOCK)
        at, n = slice(b * BLOCK, (b + k) * BLOCK), p.numel()
        m, v = self.exp_avg[at], self.exp_avg_sq[at]
        if self.state_bits == 8:
            m, v = N.ext().adamw_state_values(m, self.exp_avg_scale[b:b + k], v, self.exp_avg_sq_scale[b:b + k], True)
        return m[:n].view(p.shape), v[:n].view(p.shape)

    def load_tensor_state(self, i, exp_avg, exp_avg_sq):
        """Inverse of tensor_state, from any device. Values that came from 8-bit states are taken over exactly, others
        are rounded to the nearest."""
        p, b = self.params[i], self.plan.first_block[i]
        k = -(-p.numel() // BLOCK)
        at, n = slice(b * BLOCK, (b + k) * BLOCK), p.numel()
        m, v = self.exp_avg[at], self.exp_avg_sq[at]
        if self.state_bits == 32:
            m[:n].copy_(exp_avg.reshape(-1))
            v[:n].copy_(exp_avg_sq.reshape(-1))
            return
        full = torch.zeros((2, k * BLOCK), dtype=torch.float32, device=m.device)
        full[0, :n].copy_(exp_avg.reshape(-1))
        full[1, :n].copy_(exp_avg_sq.reshape(-1))
        N.ext().adamw_encode_states(full[0], full[1], m, self.exp_avg_scale[b:b + k], v, self.exp_avg_sq_scale[b:b + k])

    def param_states(self):
        """[(exp_avg, exp_avg_sq)] per tensor, fp32 in its shape (torch.optim.AdamW's layout), all at once: 8 bytes a value.
        A checkpoint of a model that fits only with 8-bit states takes tensor_state one by one."""
        return [tuple(x.clone() if self.state_bits == 32 else x for x in self.tensor_state(i)) for i in range(len(self.params))]

    def load_param_states(self, states):
        """Inverse of param_states, tensor by tensor; an entry None leaves that tensor's states."""
        for i, s in zip(range(len(self.params)), states):
            if s is not None:
                self.load_tensor_state(i, *s)

    def state_dict(self, flat=None):
        """torch.optim.AdamW-style state, the moments in fp32."""
        step = float(self.step_t.item())
        st = {i: {"step": torch.tensor(step), "exp_avg": m, "exp_avg_sq": v}
              for i, (m, v) in enumerate(self.param_states())}
        return {"state": st, "param_groups": [{"lr": self.lr, "betas": self.betas, "eps": self.eps,
                                               "weight_decay": self.weight_decay, "params": list(range(len(st)))}]}

    def load_state_dict(self, sd, flat=None):
        states = []
        for i in range(len(self.params)):
            s = sd["state"].get(i)
            states.append(None if s is None else (s["exp_avg"], s["exp_avg_sq"]))
            if s is not None:
                self.step_t.fill_(int(float(s["step"])))
        self.load_param_states(states)
        self.set_lr(sd["param_groups"][0]["lr"])
