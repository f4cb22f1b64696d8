"""The post-training operators together: models with their rotary layouts, losses from the native
model, 8-bit optimizer states in the trainer, and one whole post-training step of each kind.

Whole-model bounds are those of the native model's own tests (bf16 operands through four blocks): a loss
within 1e-2, a gradient within 5e-2 of fp32 PyTorch's in the 2-norm. A log-probability of these models
is off by its logit's and the others': operands of 2^-8 in about eight roundings on logits of standard deviation
0.32, four of them at the most: under 0.05."""
import pytest
import torch

from tests.helpers import rel_err

pytestmark = pytest.mark.gpu
LLAMA3 = {"type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0, "original_max_position": 64}
YARN = {"type": "yarn", "factor": 4.0, "original_max_position": 32}


def _pair(cfg, T, seed=0):
    from llmt.models.llama import build_model
    from llmt.models.native import NativeLlama
    return build_model(cfg, T, seed=seed, device="cuda"), NativeLlama(build_model(cfg, T, seed=seed, device="cuda"))


def _logits(ref, idx):
    """fp32 logits (B, T, V) of the plain model."""
    import torch.nn.functional as F
    from llmt.models.llama import rms_norm
    T = idx.shape[1]
    x = F.embedding(idx, ref.emb.weight)
    for blk in ref.blocks:
        x = blk(x, ref.rope_cos[:T], ref.rope_sin[:T])
    return F.linear(rms_norm(x, ref.norm_f.weight, ref.cfg.eps), ref.head.weight)


def _ref_logp(ref, idx, tgt):
    return torch.log_softmax(_logits(ref, idx), -1).gather(-1, tgt[..., None])[..., 0]


def _same_grads(ref, net):
    for (name, p_ref), p in zip(ref.named_parameters(), net.model.parameters()):
        assert p.grad is None
        assert rel_err(p.main_grad, p_ref.grad) < 5e-2, name


@pytest.mark.parametrize("rope", [
    {"rope_scaling": LLAMA3}, {"rope_interleaved": True}, {"rotary_dim": 32}, {"rope_scaling": YARN, "kv_heads": 2},
    {"rope_interleaved": True, "rotary_dim": 16, "rope_scaling": {"type": "linear", "factor": 2.0}, "kv_heads": 2},
    {"rotary_dim": 20, "rope_scaling": {"type": "ntk", "factor": 4.0}},
])
def test_models_with_other_rotary_positions(rope):
    from llmt.config import get_config
    from llmt.models.llama import make_batch
    cfg = get_config("tiny256", **rope)
    idx, tgt = make_batch(2, 128, cfg.vocab, "cuda")
    ref, net = _pair(cfg, 128)
    plain, _ = _pair(get_config("tiny256", kv_heads=rope.get("kv_heads")), 128)
    loss_ref = ref(idx, tgt)
    loss_ref.backward()
    assert plain(idx, tgt).item() != loss_ref.item()
    loss = net(idx, tgt)
    loss.backward()
    assert abs(loss.item() - loss_ref.item()) / loss_ref.item() < 1e-2
    _same_grads(ref, net)


def _answers(B, T, vocab, seed=0):
    from llmt.models.llama import make_batch
    idx, tgt = make_batch(B, T, vocab, "cuda", seed=seed)
    mask = torch.zeros(B, T, dtype=torch.bool, device="cuda")
    for b in range(B):
        mask[b, 10 + 3 * b:T - 7 * b] = True
    return idx, torch.where(mask, tgt, torch.full_like(tgt, -100)), mask


def test_token_logprobs():
    from llmt.config import get_config
    cfg = get_config("tiny256", vocab=1001 * 8)
    ref, net = _pair(cfg, 96)
    net.ce_chunk = 100  # chunks that end inside a sequence
    idx, tgt, mask = _answers(3, 96, cfg.vocab)
    want = _ref_logp(ref, idx, tgt.clamp(min=0))
    got = net.token_logprobs(idx, tgt)
    assert ((got - want).abs()[mask] < 0.05).all() and (got[~mask] == 0).all()
    g = torch.randn(3, 96, device="cuda")
    (got * g).sum().backward()
    (want * g * mask).sum().backward()
    _same_grads(ref, net)
    with torch.no_grad():
        assert torch.equal(net.token_logprobs(idx, tgt), got)


@pytest.mark.parametrize("kind", ["policy", "preference"])
def test_post_training_step(kind):
    """Old and reference log-probabilities without gradient, the loss, its gradient and an 8-bit AdamW step, on a
    model with scaled interleaved positions; gradients against fp32 PyTorch, a second step runs."""
    from llmt.config import get_config
    from llmt.optim.multi import MultiAdamW
    cfg = get_config("tiny256", rope_interleaved=True, rope_scaling=YARN)
    ref, net = _pair(cfg, 64)
    flat = net.flat
    opt = MultiAdamW(flat.params, [p.w16 for p in flat.params], [p.main_grad for p in flat.params], lr=1e-4,
                     weight_decay=[0.1 if p.dim() > 1 else 0.0 for p in flat.params], zero_grad=True)
    idx, tgt, mask = _answers(4, 64, cfg.vocab)
    g = torch.Generator(device="cuda").manual_seed(1)
    with torch.no_grad():
        base = net.token_logprobs(idx, tgt)
    ref_lp = base + 0.1 * torch.randn(4, 64, device="cuda", generator=g)
    adv = torch.randn(4, 1, device="cuda", generator=g)
    old = base + 0.1 * torch.randn(4, 64, device="cuda", generator=g)
    lp = _ref_logp(ref, idx, tgt.clamp(min=0))
    if kind == "policy":
        r = (lp - old).exp()
        d = ref_lp - lp
        per = -torch.minimum(r * adv, r.clamp(0.5, 2.0) * adv) + 0.05 * (d.exp() - 1 - d)
        want = (per * mask).sum() / mask.sum()

        def loss_of():
            return net.policy_loss(idx, tgt, old, adv, ref_logp=ref_lp, mask=mask, clip=(0.5, 1.0), kl_coef=0.05)
    else:
        gain = ((lp - ref_lp) * mask).sum(1)
        want = -torch.nn.functional.logsigmoid(0.1 * (gain[:2] - gain[2:])).mean()

        def loss_of():
            return net.preference_loss(idx, tgt, ref_logp=ref_lp, mask=mask, beta=0.1)
    want.backward()
    out = loss_of()
    out.loss.backward()
    assert abs(out.loss.item() - want.item()) < 2e-2 * max(1.0, abs(want.item()))
    _same_grads(ref, net)
    before = flat.master.clone()
    opt.step()
    moved = (flat.master - before).abs()
    assert (flat.grad == 0).all() and 0 < moved.max().item() < 1e-4 * 1.5
    assert torch.equal(flat.params[0].w16, flat.params[0].bfloat16())
    loss_of().loss.backward()
    opt.step()
    assert torch.isfinite(flat.master).all() and opt.step_t.item() == 2


def test_post_training_step_in_a_graph():
    """The whole step captured; replays equal eager steps bit for bit (the flat gradient's atomics aside)."""
    from llmt.config import get_config
    from llmt.optim.multi import MultiAdamW
    cfg = get_config("tiny256")
    idx, tgt, mask = _answers(2, 64, cfg.vocab)
    adv = torch.tensor([[1.0], [-0.5]], device="cuda")
    runs = []
    for graph in (False, True):
        _, net = _pair(cfg, 64)
        flat = net.flat
        opt = MultiAdamW(flat.params, [p.w16 for p in flat.params], [p.main_grad for p in flat.params], lr=1e-4, zero_grad=True)

        def step():
            loss = net.policy_loss(idx, tgt, None, adv, mask=mask).loss
            loss.backward()
            opt.step()
            return loss.detach()
        if graph:
            s = torch.cuda.Stream()
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                step()
            torch.cuda.current_stream().wait_stream(s)
            gr = torch.cuda.CUDAGraph()
            with torch.cuda.graph(gr):
                loss = step()
            for _ in range(2):
                gr.replay()
        else:
            for _ in range(3):
                loss = step()
        torch.cuda.synchronize()
        assert opt.step_t.item() == 3
        runs.append((loss.item(), flat.master.clone()))
        if graph:
            del gr
    # three steps of 1e-4; a gradient's sign may differ where it is near zero
    assert abs(runs[0][0] - runs[1][0]) < 1e-3 and (runs[0][1] - runs[1][1]).abs().max().item() < 6e-4
    assert rel_err(runs[1][1], runs[0][1]) < 1e-4


def test_trainer_with_8_bit_states(tmp_path):
    from llmt.ckpt import checkpoint
    from llmt.config import get_config
    from llmt.models.llama import make_batch
    from llmt.train import Trainer
    cfg = get_config("tiny256")
    idx, tgt = make_batch(2, 128, cfg.vocab, "cpu")
    eager = Trainer(cfg, 2, 128, cuda_graph=False, optimizer="adamw8")
    graph = Trainer(cfg, 2, 128, cuda_graph=True, optimizer="adamw8")
    full = Trainer(cfg, 2, 128, cuda_graph=False)
    le = [eager.train_step(idx, tgt) for _ in range(4)]
    lg = [graph.train_step(idx, tgt) for _ in range(4)]
    lf = [full.train_step(idx, tgt) for _ in range(4)]
    assert max(abs(a - b) / b for a, b in zip(lg, le)) < 2e-2 and graph.opt.step_t.item() == 4
    # one step is one update of the same size, so the losses stay near those of fp32 states
    assert max(abs(a - b) / b for a, b in zip(le, lf)) < 5e-2
    path = str(tmp_path / "ck.pt")
    checkpoint.save(path, eager.model, eager.opt, eager.net.flat)
    new = Trainer(cfg, 2, 128, cuda_graph=False, seed=0, optimizer="adamw8")
    new.train_step(idx, tgt)
    checkpoint.load(path, new.model, new.opt, new.net.flat)
    assert new.opt.step_t.item() == 4 and torch.equal(new.net.flat.master, eager.net.flat.master)
    assert torch.equal(new.net.flat.shadow, eager.net.flat.shadow)
    for a, b in zip(eager.opt.state_values(torch.float32), new.opt.state_values(torch.float32)):
        assert torch.equal(a, b)
    wide = Trainer(cfg, 2, 128, cuda_graph=False)
    checkpoint.load(path, wide.model, wide.opt, wide.net.flat)  # into fp32 states
    o, p = wide.net.flat.offsets[1], wide.net.flat.params[1]
    assert torch.equal(wide.opt.exp_avg[o:o + p.numel()].view(p.shape), eager.opt.param_states()[1][0])
    graph.release()
