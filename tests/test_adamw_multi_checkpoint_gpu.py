"""Checkpoints of 8-bit optimizer states go tensor by tensor: a model that fits the GPU only with them can be saved and
resumed there."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def peak(fn):
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    fn()
    torch.cuda.synchronize()
    return torch.cuda.max_memory_allocated() - before


def test_saving_and_loading_decode_one_tensor_at_a_time(tmp_path):
    from llmt.ckpt import checkpoint
    from llmt.config import get_config
    from llmt.models.llama import make_batch
    from llmt.train import Trainer
    cfg = get_config("tiny256", L=16, vocab=2048)
    t = Trainer(cfg, 2, 64, cuda_graph=False, optimizer="adamw8")
    t.train_step(*make_batch(2, 64, cfg.vocab, "cpu"))
    largest = max(p.numel() for p in t.net.flat.params)
    assert t.net.flat.numel > 16 * largest
    path = str(tmp_path / "ck.pt")
    limit = 2 * 8 * largest + (1 << 16)  # both moments in fp32, of one tensor and of the one before it, whose names are still held
    assert peak(lambda: checkpoint.save(path, t.model, t.opt, t.net.flat)) <= limit
    want = [x.clone() for x in (t.opt.exp_avg.view(torch.uint8), t.opt.exp_avg_sq, t.opt.exp_avg_scale, t.opt.exp_avg_sq_scale)]
    t.train_step(*make_batch(2, 64, cfg.vocab, "cpu", seed=1))
    assert peak(lambda: checkpoint.load(path, t.model, t.opt, t.net.flat)) <= limit
    got = (t.opt.exp_avg.view(torch.uint8), t.opt.exp_avg_sq, t.opt.exp_avg_scale, t.opt.exp_avg_sq_scale)
    m, v = t.opt.state_values(torch.float32)
    for x, y in zip(got, want):
        x.copy_(y)
    assert all(torch.equal(a, b) for a, b in zip((m, v), t.opt.state_values(torch.float32)))


@pytest.mark.parametrize("bits", [8, 32])
def test_a_tensor_without_saved_states_keeps_its_own(bits):
    from llmt.optim.multi import MultiAdamW
    g = torch.Generator(device="cuda").manual_seed(0)
    p = [torch.randn(n, device="cuda", generator=g) for n in (300, 256, 77)]
    opt = MultiAdamW(p, state_bits=bits)
    opt.step([torch.randn_like(x) for x in p])
    before = [(m.clone(), v.clone()) for m, v in opt.param_states()]
    new = [torch.full_like(x, 0.5) for x in p]
    opt.load_param_states([(new[0], new[0]), None, (new[2], new[2])])
    after = opt.param_states()
    assert all(torch.equal(a, b) for a, b in zip(after[1], before[1]))
    assert all((x == 0.5).all() for i in (0, 2) for x in after[i])
    again = opt.param_states()
    opt.step([torch.randn_like(x) for x in p])
    assert all(torch.equal(a, b) for s, t in zip(after, again) for a, b in zip(s, t))  # copies, not views of the states
