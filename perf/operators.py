"""Measured cases of the operators behind a post-training step: the policy loss and the preference
loss over a batch of logits, AdamW over many tensors with 8-bit or 32-bit states, and rotary
positions in their layouts and long-context scalings.

`run` computes them in elementary fp32 torch operations (`own` false) or through llmt's kernels
(`own` true) on the same inputs; `exact` is their definition in 64 bits.
"""
import math

import torch

own = False

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}

# Clipped policy loss: the usual asymmetric clip range and a small KL weight.
CLIP_LOW, CLIP_HIGH, KL_COEF = 0.2, 0.28, 0.04
BETA = 0.1
# AdamW as this repository trains (lr 3e-4, betas 0.9 / 0.95, weight decay 0.1 on the matrices).
LR, B1, B2, EPS, WD, SEED = 3e-4, 0.9, 0.95, 1e-8, 0.1, 17
BLOCK = 256  # values that share one scale in an 8-bit state


def listed():
    return [
        # the last few answer tokens of two short rollouts: what counts is latency
        {"name": "policy_small", "op": "policy", "B": 2, "T": 40, "V": 32000, "dtype": "bf16", "reduction": "token"},
        # one micro-batch of rollouts on the medium model
        {"name": "policy_medium", "op": "policy", "B": 4, "T": 1024, "V": 32000, "dtype": "bf16", "reduction": "token"},
        # the same with logits kept in fp32 and a vocabulary grown by three added tokens (odd rows)
        {"name": "policy_fp32_odd", "op": "policy", "B": 3, "T": 701, "V": 32003, "dtype": "fp32",
         "reduction": "sequence"},
        # rollouts on the Llama-3 vocabulary
        {"name": "policy_llama3", "op": "policy", "B": 4, "T": 1024, "V": 128256, "dtype": "bf16",
         "reduction": "token"},
        # one pair of short answers, fp32 logits
        {"name": "preference_pair", "op": "preference", "P": 1, "T": 77, "V": 32000, "dtype": "fp32",
         "kind": "sigmoid", "average": False},
        # four pairs on the Llama-3 vocabulary: the largest loss
        {"name": "preference_llama3", "op": "preference", "P": 4, "T": 1024, "V": 128256, "dtype": "bf16",
         "kind": "sigmoid", "average": False},
        # low-rank adapters of the medium model: 336 small tensors
        {"name": "adamw8_adapters", "op": "adamw", "bits": 8, "d": 1024, "layers": 24, "ffn": 2816, "vocab": 0,
         "rank": 16, "grad": "bf16"},
        # every weight of the medium model, fp32 accumulated gradients
        {"name": "adamw8_medium", "op": "adamw", "bits": 8, "d": 1024, "layers": 24, "ffn": 2816, "vocab": 32000,
         "rank": 0, "grad": "fp32"},
        # every weight of the large model with fp32 states and bf16 gradients
        {"name": "adamw32_large", "op": "adamw", "bits": 32, "d": 2048, "layers": 16, "ffn": 5504, "vocab": 32000,
         "rank": 0, "grad": "bf16"},
        # one new token in each of 64 sequences, each at its own place in a long context
        {"name": "rope_tokens", "op": "rope", "B": 64, "T": 1, "H": 32, "KV": 8, "hd": 128, "rd": 128,
         "dtype": "bf16", "layout": "half", "scaling": "llama3", "far": 131072, "inverse": False},
        # the backward rotation of interleaved pairs in half of each head, an odd batch length
        {"name": "rope_partial_backward", "op": "rope", "B": 4, "T": 1023, "H": 16, "KV": 16, "hd": 64, "rd": 32,
         "dtype": "fp16", "layout": "interleaved", "scaling": "linear", "far": 4096, "inverse": True},
        # one whole long context of the 8B shape
        {"name": "rope_long", "op": "rope", "B": 1, "T": 131072, "H": 32, "KV": 8, "hd": 128, "rd": 128,
         "dtype": "bf16", "layout": "half", "scaling": "yarn", "far": 131072, "inverse": False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["policy", "preference", "adamw", "rope"])
    if op in ("policy", "preference"):
        V = rng.choice([32000, 128256, _log(rng, 500, 130000), _log(rng, 500, 130000)])
        c = {"op": op, "T": _log(rng, 5, 1024), "V": V, "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"])}
        if op == "policy":
            return {**c, "B": rng.randint(1, 4), "reduction": rng.choice(["token", "sequence"])}
        return {**c, "P": rng.randint(1, 2), "kind": rng.choice(["sigmoid", "hinge", "ipo"]),
                "average": rng.choice([False, True])}
    if op == "adamw":
        d = 2 * _log(rng, 64, 512) + rng.choice([0, 0, 1])
        return {"op": op, "bits": rng.choice([8, 8, 32]), "d": d, "layers": _log(rng, 2, 24), "ffn": 2 * d + rng.randint(0, 99),
                "vocab": rng.choice([0, _log(rng, 1000, 32000)]), "rank": rng.choice([0, 0, 8, 17]),
                "grad": rng.choice(["fp32", "bf16"])}
    hd = rng.choice([64, 128, 128, 80, 96])
    kv = rng.choice([1, 4, 8])
    T = rng.choice([1, _log(rng, 2, 16384)])
    return {"op": op, "B": _log(rng, 1, 256) if T == 1 else rng.randint(1, 4), "T": T, "H": kv * rng.randint(1, 4), "KV": kv,
            "hd": hd, "rd": rng.choice([hd, hd, hd // 2]), "dtype": rng.choice(["bf16", "fp16", "fp32"]),
            "layout": rng.choice(["half", "interleaved"]), "scaling": rng.choice(["none", "linear", "ntk", "llama3", "yarn"]),
            "far": max(T, _log(rng, 1000, 2000000)), "inverse": rng.choice([False, True])}


# ---------------------------------------------------------------- what a pass cannot do without
def _spans(rows, T):
    """[first, last) answer tokens of each sequence: a prompt in front, padding behind."""
    return [(T // 4 + (7 * b) % max(1, T // 8), T - (37 * b) % max(1, T // 4)) for b in range(rows)]


def work(case):
    op = case["op"]
    if op in ("policy", "preference"):
        rows = case["B"] if op == "policy" else 2 * case["P"]
        n, e = rows * case["T"], SIZE[case["dtype"]]
        valid = sum(b - a for a, b in _spans(rows, case["T"]))
        # logits of the answer tokens in, the whole gradient out; per token an id, a mask, 2 or 3 floats and logp
        per = 8 + 1 + 4 * (4 if op == "policy" else 2)
        return {"bytes": valid * case["V"] * e + n * case["V"] * e + n * per, "flops": 6 * valid * case["V"]}
    if op == "adamw":
        n = sum(a * b for a, b in _shapes(case))
        state = 2 * (2 if case["bits"] == 8 else 8) + (4 if case["bits"] == 8 else 0)  # 8 bits: the values too, in 16
        return {"bytes": n * (4 + 4 + 2 + (4 if case["grad"] == "fp32" else 2) + state), "flops": 20 * n}
    n = case["B"] * case["T"]
    vals = n * (case["H"] + case["KV"]) * case["hd"]
    return {"bytes": 2 * vals * SIZE[case["dtype"]] + 4 * n, "flops": 3 * vals}


# ---------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _token_batch(case, rows, g):
    """Logits of a trained model (most answer tokens likely, some not), ids and the answer mask."""
    T, V = case["T"], case["V"]
    mask = torch.zeros(rows, T, dtype=torch.bool)
    for b, (a, e) in enumerate(_spans(rows, T)):
        mask[b, a:e] = True
    mask = mask.cuda()
    y = torch.randint(0, V, (rows, T), device="cuda", generator=g)
    logits = torch.empty(rows, T, V, dtype=DT[case["dtype"]], device="cuda")
    lift = 2.0 + 10.0 * torch.rand(rows, T, 1, device="cuda", generator=g)
    logp = torch.empty(rows, T, device="cuda")
    for b in range(rows):
        z = torch.randn(T, V, device="cuda", generator=g) * 2.0
        z.scatter_add_(1, y[b, :, None], lift[b])
        logits[b] = z
        z = logits[b].float()
        logp[b] = z.gather(1, y[b, :, None])[:, 0] - torch.logsumexp(z, -1)
    return logits, torch.where(mask, y, torch.full_like(y, -100)), mask, logp


def _linear_shapes(d, ffn, rank):
    """Weights of one block; with a rank, the two low-rank factors of each instead."""
    full = [(3 * d, d), (d, d), (ffn, d), (ffn, d), (d, ffn)]
    if not rank:
        return full + [(1, d), (1, d)]
    return [s for o, i in ((d, d), (d, d), (d, d), (d, d), (ffn, d), (ffn, d), (d, ffn)) for s in ((rank, i), (o, rank))]


def _shapes(case):
    d = case["d"]
    s = _linear_shapes(d, case["ffn"], case["rank"]) * case["layers"]
    if case["vocab"]:
        s = s + [(case["vocab"], d), (1, d), (case["vocab"], d)]
    return s


def prepare(case, seed):
    g = _gen(seed)
    op = case["op"]
    if op == "policy":
        logits, y, mask, logp = _token_batch(case, case["B"], g)
        noise = torch.randn(2, *logp.shape, device="cuda", generator=g)
        adv = torch.randn(logp.shape, device="cuda", generator=g) + 0.5
        return {"case": case, "logits": logits, "targets": y, "mask": mask, "old": logp + 0.15 * noise[0],
                "ref": logp + 0.3 * noise[1], "adv": adv}
    if op == "preference":
        logits, y, mask, logp = _token_batch(case, 2 * case["P"], g)
        # the policy has moved towards the chosen answers (the first P) and away from the rejected ones
        moved = 1.5 / mask.sum(1, keepdim=True).clamp(min=1)
        moved[case["P"]:] *= -1.0
        ref = logp - moved + 0.02 * torch.randn(logp.shape, device="cuda", generator=g)
        return {"case": case, "logits": logits, "targets": y, "mask": mask, "ref": ref}
    if op == "adamw":
        return _prepare_adamw(case, g)
    n, H, KV, hd = case["B"] * case["T"], case["H"], case["KV"], case["hd"]
    # q and k as a packed projection leaves them: views of rows that hold the values too
    qkv = torch.randn(n, (H + 2 * KV) * hd, device="cuda", generator=g).to(DT[case["dtype"]])
    qkv = qkv.view(case["B"], case["T"], H + 2 * KV, hd)
    first = torch.randint(0, case["far"] - case["T"] + 1, (case["B"], 1), device="cuda", generator=g)
    pos = (first + torch.arange(case["T"], device="cuda")).int()
    s = {"case": case, "q": qkv[:, :, :H], "k": qkv[:, :, H:H + KV], "pos": pos}
    s["inv_freq"], s["factor"] = _frequencies(case)
    if own:
        from llmt.ops.rotary import Rotary
        s["rotary"] = Rotary(hd, rotary_dim=case["rd"], base=10000.0, interleaved=case["layout"] == "interleaved",
                             scaling=_scaling(case), device="cuda")
    return s


def _prepare_adamw(case, g):
    """Parameters, gradients and states of a run under way, each tensor starting at a block."""
    shapes = _shapes(case)
    blocks = [-(-(a * b) // BLOCK) for a, b in shapes]
    nb = sum(blocks)
    starts, at = [], 0
    for k in blocks:
        starts.append(at * BLOCK)
        at += k
    live = torch.zeros(nb * BLOCK, dtype=torch.bool, device="cuda")
    for (a, b), o in zip(shapes, starts):
        live[o:o + a * b] = True

    def normal(scale):
        return torch.randn(nb * BLOCK, device="cuda", generator=g).mul_(scale).mul_(live)

    s = {"case": case, "p": normal(0.02), "g": normal(1e-3).to(DT[case["grad"]])}
    m, v = normal(4e-4), normal(1e-3).square_()
    decay = [WD if a > 1 else 0.0 for a, b in shapes]
    s["p16"] = torch.empty(nb * BLOCK, dtype=torch.bfloat16, device="cuda")
    s["lr"], s["step"] = torch.full((1,), LR, device="cuda"), torch.full((1,), 100, dtype=torch.int32, device="cuda")
    if case["bits"] == 8:
        half = torch.full((nb, BLOCK), 1 << 19, dtype=torch.int32, device="cuda")
        s["m"], s["ms"] = _encode_m(m.view(nb, BLOCK), half)
        s["v"], s["vs"] = _encode_v(v.view(nb, BLOCK), half)
    else:
        s["m"], s["v"] = m, v
    s["wd"] = torch.tensor(decay, device="cuda")
    s["blocks"] = torch.tensor(blocks, device="cuda")
    if own:
        from llmt.optim.multi import MultiAdamW

        def views(flat):
            return [flat[o:o + a * b].view(a, b) for (a, b), o in zip(shapes, starts)]
        s["opt"] = MultiAdamW(views(s["p"]), views(s["p16"]), lr=LR, betas=(B1, B2), eps=EPS, weight_decay=decay,
                              state_bits=case["bits"], seed=SEED)
        s["grads"] = views(s["g"])
        s["opt"].step_t.copy_(s["step"])
        s["opt"].exp_avg.copy_(s["m"].view(s["opt"].exp_avg.dtype).view(-1))
        s["opt"].exp_avg_sq.copy_(s["v"].view(-1))
        if case["bits"] == 8:
            s["opt"].exp_avg_scale.copy_(s["ms"].view(-1))
            s["opt"].exp_avg_sq_scale.copy_(s["vs"].view(-1))
    return s


# ---------------------------------------------------------------- one pass
def run(s):
    return _run_own(s) if own else _run_plain(s)


def _run_own(s):
    c = s["case"]
    if c["op"] == "policy":
        from llmt.ops import losses
        r = losses.policy_loss_rows(s["logits"], s["targets"], s["old"], s["adv"], ref_logp=s["ref"], mask=s["mask"],
                                    clip=(CLIP_LOW, CLIP_HIGH), kl_coef=KL_COEF, reduction=c["reduction"])
        return {"loss": r.loss, "logp": r.logp, "dlogits": r.dlogits}
    if c["op"] == "preference":
        from llmt.ops import losses
        r = losses.preference_loss_rows(s["logits"], s["targets"], ref_logp=s["ref"], mask=s["mask"], beta=BETA,
                                        kind=c["kind"], average=c["average"])
        return {"loss": r.loss, "logp": r.logp, "rewards": r.rewards, "dlogits": r.dlogits}
    if c["op"] == "adamw":
        opt = s["opt"]
        opt.step(s["grads"])
        if c["bits"] == 32:
            return {"p": s["p"], "p16": s["p16"], "m": opt.exp_avg, "v": opt.exp_avg_sq}
        m, v = opt.state_values()
        return {"p": s["p"], "p16": s["p16"], "m": m, "v": v}
    q, k = s["rotary"].rotate(s["q"], s["k"], s["pos"], inverse=c["inverse"])
    return {"q": q, "k": k}


def _run_plain(s):
    c = s["case"]
    if c["op"] == "policy":
        return _plain_policy(s)
    if c["op"] == "preference":
        return _plain_preference(s)
    if c["op"] == "adamw":
        return _plain_adamw(s)
    return {"q": _plain_rope(s, s["q"]), "k": _plain_rope(s, s["k"])}


def _softmax_parts(s):
    """(softmax, logp, valid, target column) of the logits, in fp32."""
    z, y = s["logits"].float(), s["targets"]
    valid = s["mask"] & (y >= 0) & (y < z.shape[-1])
    y = torch.where(valid, y, torch.zeros_like(y))[..., None]
    top = z.amax(-1, keepdim=True)
    target = z.gather(-1, y) - top
    z = z.sub_(top).exp_() if z is not s["logits"] else torch.exp(z - top)
    total = z.sum(-1, keepdim=True)
    logp = (target - torch.log(total))[..., 0]
    return z.div_(total), torch.where(valid, logp, torch.zeros_like(logp)), valid, y


def _gradient(soft, coef, valid, y, dtype):
    """coef * (onehot - softmax) in the rows that count, zero in the others."""
    d = torch.where(valid[..., None], soft * -coef[..., None], torch.zeros((), device=soft.device))
    hit = d.gather(-1, y) + torch.where(valid, coef, torch.zeros_like(coef))[..., None]
    return d.scatter_(-1, y, hit).to(dtype)


def _plain_policy(s):
    soft, logp, valid, y = _softmax_parts(s)
    zero = torch.zeros_like(logp)
    per_seq = valid.sum(-1, keepdim=True)
    if s["case"]["reduction"] == "token":
        w = torch.where(valid, 1.0 / valid.sum(), zero)
    else:
        w = torch.where(valid, 1.0 / (per_seq * (per_seq > 0).sum()), zero)
    adv = s["adv"]
    ratio = torch.exp(logp - s["old"])
    clipped = ratio.clamp(1.0 - CLIP_LOW, 1.0 + CLIP_HIGH)
    free = ratio * adv <= clipped * adv  # the unclipped term is the smaller one
    d = s["ref"] - logp
    e = torch.exp(d)
    loss = -torch.minimum(ratio * adv, clipped * adv) + KL_COEF * (e - d - 1.0)
    slope = torch.where(free, -ratio * adv, zero) + KL_COEF * (1.0 - e)
    total = (torch.where(valid, loss, zero) * w).sum(dtype=torch.float64).float()
    return {"loss": total, "logp": logp, "dlogits": _gradient(soft, slope * w, valid, y, s["logits"].dtype)}


def _plain_preference(s):
    soft, logp, valid, y = _softmax_parts(s)
    P = s["case"]["P"]
    gain = torch.where(valid, (logp - s["ref"]).double(), torch.zeros((), dtype=torch.float64, device=logp.device)).sum(-1)
    share = 1.0 / valid.sum(-1).clamp(min=1) if s["case"]["average"] else torch.ones(2 * P, device=logp.device)
    gain = gain * share
    d = (gain[:P] - gain[P:]).float()
    kind = s["case"]["kind"]
    if kind == "sigmoid":
        x = BETA * d
        loss = torch.log1p(torch.exp(-x.abs())) + (-x).clamp(min=0.0)
        slope = -BETA / (1.0 + torch.exp(x))
    elif kind == "hinge":
        loss = (1.0 - BETA * d).clamp(min=0.0)
        slope = torch.where(BETA * d < 1.0, -BETA, 0.0)
    else:
        off = d - 1.0 / (2.0 * BETA)
        loss, slope = off * off, 2.0 * off
    coef = torch.cat([slope, -slope]) * share / P
    return {"loss": loss.mean(), "logp": logp, "rewards": (BETA * gain).float(),
            "dlogits": _gradient(soft, coef[:, None].expand_as(logp).float(), valid, y, s["logits"].dtype)}


# The 8-bit states hold blocks of 256 values under one power-of-two scale (an exponent byte e, 2^(e - 127)):
# the first moment in e4m3, the second in eight unsigned bits (5 of exponent, 3 of mantissa, unit 1).
# A value goes to one of its two neighbours with probabilities that keep its mean; the 16 random
# bits come from a hash of the value's place, the step and the seed, and are equal on both sides.
def _bits(x):
    return x.view(torch.int32)


def _power(e):
    """2^(e - 127) of exponent bytes."""
    return (e.int() << 23).view(torch.float32)


def _scale_of(top, places, limit):
    """Smallest exponent byte under which `top` is at most the format's largest value."""
    b = _bits(top)
    return ((b >> 23) - places + ((b & 0x7FFFFF) > limit).int()).clamp(1, 253)


def _encode_m(m, noise):
    e = _scale_of(m.abs().amax(1, keepdim=True), 8, 0x600000)
    y = m.abs() * _power(254 - e) * 2.0 ** -120
    code = ((_bits(y) + noise) >> 20).clamp(max=126) | torch.where(m < 0, 128, 0)
    return code.to(torch.uint8), e.to(torch.uint8)


def _encode_v(v, noise):
    e = _scale_of(v.amax(1, keepdim=True), 33, 0x700000)
    y = v * _power(254 - e) * 2.0 ** -129
    code = ((_bits(y) + noise) >> 20).clamp(max=255)
    return torch.where(v > 0, code.clamp(min=1), code).to(torch.uint8), e.to(torch.uint8)


def _decode_m(code, e):
    return code.view(torch.float8_e4m3fn).float() * _power(e)


def _decode_v(code, e):
    return (code.int() << 20).view(torch.float32) * 2.0 ** 64 * 2.0 ** 65 * _power(e)


def _hash(n, step, device):
    """32 mixed bits for each place 0..n-1 at this step."""
    i = torch.arange(n, device=device)
    low = 0xFFFFFFFF
    x = ((i & low) ^ ((i >> 32) * 0x6A09E667)) * 0x9E3779B1 + step.long() * 0xB7E15163 + SEED * 0x3C6EF373 & low
    x = ((x ^ (x >> 16)) * 0xB7E15163) & low
    x = ((x ^ (x >> 15)) * 0x6A09E667) & low
    return x ^ (x >> 16)


def _plain_adamw(s):
    c, n = s["case"], s["p"].numel()
    s["step"] += 1
    t = s["step"]
    g = s["g"].float()
    if c["bits"] == 8:
        m, v = _decode_m(s["m"], s["ms"]).view(-1), _decode_v(s["v"], s["vs"]).view(-1)
    else:
        m, v = s["m"], s["v"]
    m = m * B1 + g * (1.0 - B1)
    v = v * B2 + g * (1.0 - B2) * g
    bc1, bc2 = 1.0 - torch.pow(torch.tensor(B1, dtype=torch.float64, device="cuda"), t), 1.0 - torch.pow(
        torch.tensor(B2, dtype=torch.float64, device="cuda"), t)
    step_size, root = (s["lr"].double() / bc1).float(), (1.0 / torch.sqrt(bc2)).float()
    p = s["p"].view(-1, BLOCK)
    p *= (1.0 - s["lr"] * s["wd"].repeat_interleave(s["blocks"]))[:, None]
    p = s["p"]
    p -= step_size * (m / (torch.sqrt(v) * root + EPS))
    s["p16"].copy_(p)
    if c["bits"] == 32:
        s["m"].copy_(m)
        s["v"].copy_(v)
        return {"p": p, "p16": s["p16"], "m": s["m"], "v": s["v"]}
    h = _hash(n, t, p.device)
    s["m"], s["ms"] = _encode_m(m.view(-1, BLOCK), (((h >> 16) << 4) | 8).int().view(-1, BLOCK))
    s["v"], s["vs"] = _encode_v(v.view(-1, BLOCK), (((h & 0xFFFF) << 4) | 8).int().view(-1, BLOCK))
    return {"p": p, "p16": s["p16"], "m": _decode_m(s["m"], s["ms"]).view(-1).bfloat16(),
            "v": _decode_v(s["v"], s["vs"]).view(-1).bfloat16()}


def _scaling(case):
    return {"none": None, "linear": {"type": "linear", "factor": 4.0}, "ntk": {"type": "ntk", "factor": 8.0},
            "llama3": {"type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
                       "original_max_position": 8192},
            "yarn": {"type": "yarn", "factor": 16.0, "beta_fast": 32.0, "beta_slow": 1.0,
                     "original_max_position": 8192}}[case["scaling"]]


def _frequencies(case):
    """(angle per position of each pair, in 64 bits; factor on the rotated values)."""
    rd, sc, base = case["rd"], _scaling(case), 10000.0
    if sc and sc["type"] == "ntk":
        base = base * sc["factor"] ** (rd / (rd - 2.0))
    j = torch.arange(rd // 2, dtype=torch.float64, device="cuda")
    w = base ** (-2.0 * j / rd)
    if sc is None or sc["type"] == "ntk":
        return w, 1.0
    if sc["type"] == "linear":
        return w / sc["factor"], 1.0
    L = sc["original_max_position"]
    if sc["type"] == "llama3":
        # turns within the original context; few turns: stretched, many: kept, between: blended
        turns = L * w / (2.0 * math.pi)
        lo, hi = sc["low_freq_factor"], sc["high_freq_factor"]
        keep = ((turns - lo) / (hi - lo)).clamp(0.0, 1.0)
        return w * keep + (w / sc["factor"]) * (1.0 - keep), 1.0

    def pair_of(turns):  # the (fractional) pair that makes this many turns within the original context
        return rd * math.log(L / (turns * 2.0 * math.pi)) / (2.0 * math.log(base))
    lo, hi = max(math.floor(pair_of(sc["beta_fast"])), 0), min(math.ceil(pair_of(sc["beta_slow"])), rd - 1)
    keep = 1.0 - ((j - lo) / max(hi - lo, 0.001)).clamp(0.0, 1.0)
    return w * keep + (w / sc["factor"]) * (1.0 - keep), 0.1 * math.log(sc["factor"]) + 1.0


def _plain_rope(s, x):
    c = s["case"]
    angle = s["pos"].double()[..., None] * s["inv_freq"]
    cos, sin = (torch.cos(angle) * s["factor"]).float()[:, :, None], (torch.sin(angle) * s["factor"]).float()[:, :, None]
    if c["inverse"]:
        sin = -sin
    rd = c["rd"]
    turn, rest = x[..., :rd].float(), x[..., rd:]
    if c["layout"] == "half":
        a, b = turn[..., :rd // 2], turn[..., rd // 2:]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    else:
        a, b = turn[..., 0::2], turn[..., 1::2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    return torch.cat([turned.to(x.dtype), rest], -1)


# ---------------------------------------------------------------- the definition in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rope":
        return {"q": _exact_rope(s, s["q"]), "k": _exact_rope(s, s["k"])}
    return {"policy": _exact_policy, "preference": _exact_preference, "adamw": _exact_adamw}[case["op"]](s)


def _exact_tokens(s):
    """Per sequence: rows that count, their log-probabilities, and what builds their gradient."""
    for b in range(s["logits"].shape[0]):
        rows = torch.nonzero(s["mask"][b])[:, 0]
        z = torch.log_softmax(s["logits"][b, rows].double(), -1)
        yield b, rows, z, z[torch.arange(len(rows)), s["targets"][b, rows]]


def _exact_policy(s):
    n_seq, T, V = s["logits"].shape
    logp = torch.zeros(n_seq, T, dtype=torch.float64, device="cuda")
    grad = torch.zeros(n_seq, T, V, dtype=torch.float64, device="cuda")
    count = s["mask"].sum(1).double()
    loss = 0.0
    for b, rows, z, lp in _exact_tokens(s):
        if not len(rows):
            continue
        w = 1.0 / count.sum() if s["case"]["reduction"] == "token" else 1.0 / (count[b] * (count > 0).sum())
        lp = lp.detach().requires_grad_()
        A, old, ref = (s[k][b, rows].double() for k in ("adv", "old", "ref"))
        r = (lp - old).exp()
        gain = torch.where(A >= 0, A * r.clamp(max=1.0 + CLIP_HIGH), A * r.clamp(min=1.0 - CLIP_LOW))
        total = ((KL_COEF * (torch.expm1(ref - lp) - (ref - lp)) - gain) * w).sum()
        (slope,) = torch.autograd.grad(total, lp)
        loss = loss + total.detach()
        logp[b, rows] = lp.detach()
        d = z.exp_().mul_(-slope[:, None])
        d[torch.arange(len(rows)), s["targets"][b, rows]] += slope
        grad[b, rows] = d
    return {"loss": loss, "logp": logp, "dlogits": grad}


def _exact_preference(s):
    n_seq, T, V = s["logits"].shape
    P, c = n_seq // 2, s["case"]
    logp = torch.zeros(n_seq, T, dtype=torch.float64, device="cuda")
    for b, rows, z, lp in _exact_tokens(s):
        logp[b, rows] = lp
    lp = logp.clone().requires_grad_()
    score = ((lp - s["ref"].double()) * s["mask"]).sum(1)
    if c["average"]:
        score = score / s["mask"].sum(1).clamp(min=1)
    x = score[:P] - score[P:]
    if c["kind"] == "sigmoid":
        loss = torch.nn.functional.softplus(-BETA * x).mean()
    elif c["kind"] == "hinge":
        loss = torch.relu(1.0 - BETA * x).mean()
    else:
        loss = (x - 0.5 / BETA).square().mean()
    (slope,) = torch.autograd.grad(loss, lp)
    grad = torch.zeros(n_seq, T, V, dtype=torch.float64, device="cuda")
    for b, rows, z, _ in _exact_tokens(s):
        d = z.exp_().mul_(-slope[b, rows, None])
        d[torch.arange(len(rows)), s["targets"][b, rows]] += slope[b, rows]
        grad[b, rows] = d
    return {"loss": loss.detach(), "logp": logp, "rewards": BETA * score.detach(), "dlogits": grad}


def _exact_values(x, u, low, mantissa, top):
    """x (>= 0, scaled to the format's units) to a neighbour: up where the place between them passes 1 - u."""
    binade = torch.floor(torch.log2(x.clamp(min=2.0 ** low)))
    step = torch.exp2(binade - mantissa)
    return (torch.floor(x / step + u) * step).clamp(max=top)


def _exact_adamw(s):
    c, n, t = s["case"], s["p"].numel(), int(s["step"].item()) + 1
    p = torch.empty(n, dtype=torch.float64, device="cuda")
    m_out, v_out = torch.empty_like(p), torch.empty_like(p)
    wd = s["wd"].double().repeat_interleave(s["blocks"] * BLOCK)
    lr = s["lr"].double()
    h = _hash(n, torch.tensor([t], device="cuda"), "cuda") if c["bits"] == 8 else None
    for a in range(0, n, 1 << 26):
        b = min(n, a + (1 << 26))
        at = slice(a, b)
        if c["bits"] == 8:
            k = slice(a // BLOCK, b // BLOCK)
            m = s["m"][k].view(torch.float8_e4m3fn).double() * torch.exp2(s["ms"][k].double() - 127)
            code = s["v"][k].double()
            field = torch.floor(code / 8)
            v = torch.where(field > 0, (8 + code - 8 * field) * torch.exp2(field - 1), code) * torch.exp2(s["vs"][k].double() - 127)
            m, v = m.view(-1), v.view(-1)
        else:
            m, v = s["m"][at].double(), s["v"][at].double()
        g = s["g"][at].double()
        m = B1 * m + (1.0 - B1) * g
        v = B2 * v + (1.0 - B2) * g * g
        p[at] = s["p"][at].double() * (1.0 - lr * wd[at]) - lr * (m / (1.0 - B1 ** t)) / (torch.sqrt(v / (1.0 - B2 ** t)) + EPS)
        if c["bits"] == 8:
            def block(x, top):
                # smallest power of two that keeps the block's largest value within `top`
                big = x.abs().view(-1, BLOCK).amax(1, keepdim=True)
                e = torch.where(big > 0, torch.ceil(torch.log2(big.clamp(min=1e-300) / top)), torch.zeros_like(big))
                return torch.exp2(e.clamp(min=-126)).expand(-1, BLOCK).reshape(-1)
            scale = block(m, 448.0)
            u = ((h[at] >> 16) * 16 + 8).double() / 2.0 ** 20
            m = torch.sign(m) * _exact_values(m.abs() / scale, u, -6, 3, 448.0) * scale
            scale = block(v, 1.875 * 2.0 ** 33)
            u = ((h[at] & 0xFFFF) * 16 + 8).double() / 2.0 ** 20
            x = _exact_values(v / scale, u, 3, 3, 1.875 * 2.0 ** 33)
            v = torch.where(v > 0, x.clamp(min=1.0), x) * scale
        m_out[at], v_out[at] = m, v
    return {"p": p, "p16": p, "m": m_out, "v": v_out}


def _exact_rope(s, x):
    c, rd = s["case"], s["case"]["rd"]
    out = torch.empty(x.shape, dtype=torch.float64, device="cuda")
    for b in range(x.shape[0]):
        turn = torch.polar(torch.full_like(s["inv_freq"], s["factor"]).expand(x.shape[1], -1),
                           s["pos"][b].double()[:, None] * s["inv_freq"] * (-1.0 if c["inverse"] else 1.0))
        for h in range(x.shape[2]):
            head = x[b, :, h].double()
            even, odd = (head[:, :rd // 2], head[:, rd // 2:rd]) if c["layout"] == "half" else (head[:, :rd:2], head[:, 1:rd:2])
            z = torch.complex(even.contiguous(), odd.contiguous()) * turn
            out[b, :, h, rd:] = head[:, rd:]
            if c["layout"] == "half":
                out[b, :, h, :rd // 2], out[b, :, h, rd // 2:rd] = z.real, z.imag
            else:
                out[b, :, h, :rd:2], out[b, :, h, 1:rd:2] = z.real, z.imag
    return out
