"""The expert layer's balance loss in a training step: what several ranks' steps return, and what a step refuses."""
import pytest
import torch

from megray_b200.models import MoEConfig
from megray_b200.models import moe as module

COEF, HIDDEN, EXPERTS, TOP = 0.3, 16, 4, 2


class Rank(module.MoELayer):
    """A layer on the CPU whose experts are the identity: one of ``n`` ranks with ``tokens`` tokens."""

    def __init__(self, n, tokens, coef=COEF):
        self.cfg = MoEConfig(experts=EXPERTS, hidden=HIDDEN, tokens=tokens, balance_coef=coef)
        self.n, self.balance_loss = n, None

    def forward(self, x, logits):
        return x

    def backward(self, dout):
        self.dout = dout
        if self.cfg.balance_coef:  # the loss over all ranks' tokens, the same on each
            self.balance_loss = torch.tensor([self.cfg.balance_coef])

    def optimizer_step(self):
        pass


@pytest.fixture
def squares(monkeypatch):
    """The squared error's definition for CPU tensors."""
    monkeypatch.setattr(module, "mse_loss_grad", lambda y, target, scale: ((y * y).sum().view(1) * scale, 2 * scale * y))


@pytest.mark.parametrize("coef", [COEF, 0.0])
@pytest.mark.parametrize("n", [1, 2, 4])
def test_returned_values_add_up_over_ranks_to_the_loss_that_is_differentiated(n, coef, squares):
    x = torch.randn(8 * n, HIDDEN, generator=torch.Generator().manual_seed(n))
    whole = Rank(1, 8 * n, coef)
    want = whole.train_step_device(x, None)
    ranks = [Rank(n, 8, coef) for _ in range(n)]
    got = [rank.train_step_device(part, None) for rank, part in zip(ranks, x.chunk(n))]
    torch.testing.assert_close(sum(got), want, rtol=1e-6, atol=0)
    torch.testing.assert_close(torch.cat([rank.dout for rank in ranks]), whole.dout, rtol=1e-6, atol=0)


@pytest.mark.gpu
def test_logits_may_be_overwritten_between_the_passes():
    cfg = MoEConfig(experts=8, hidden=256, ffn=128, tokens=300, capacity_factor=4.0, balance_coef=COEF)
    layer = module.MoELayer(cfg)
    x, dout = (torch.randn(300, 256, device="cuda").bfloat16() for _ in range(2))
    logits = torch.randn(300, 8, device="cuda")
    layer.forward(x, logits)
    want = [t.clone() for t in layer.backward(dout)] + [layer.balance_loss, layer.expert_counts]
    layer.forward(x, logits)
    logits.copy_(torch.randn(300, 8, device="cuda"))
    got = [*layer.backward(dout), layer.balance_loss, layer.expert_counts]
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_an_adamw_step_refuses_to_be_captured(monkeypatch):
    """Its number is counted on the host: every replay would take the first one's bias correction."""
    layer = Rank(1, 8)
    layer.adamw, layer.steps = object(), 3
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(RuntimeError):
        module.MoELayer.optimizer_step(layer)
    assert layer.steps == 3


@pytest.mark.gpu
@pytest.mark.parametrize("optimizer", ["sgd", "adamw"])
def test_steps_of_a_captured_layer(optimizer):
    cfg = MoEConfig(experts=4, hidden=256, ffn=128, tokens=200, capacity_factor=4.0, balance_coef=COEF, optimizer=optimizer, lr=10.0 if optimizer == "sgd" else 1e-3)
    layer = module.MoELayer(cfg)
    x, logits = torch.randn(200, 256, device="cuda").bfloat16(), torch.randn(200, 4, device="cuda")
    layer.train_step_device(x, logits)
    graph = torch.cuda.CUDAGraph()
    if optimizer == "adamw":
        with pytest.raises(RuntimeError), torch.cuda.graph(graph):
            layer.train_step_device(x, logits)
        assert layer.steps == 1
    else:
        before = layer.w_gu.clone()
        with torch.cuda.graph(graph):
            layer.train_step_device(x, logits)
        graph.replay()
        assert not torch.equal(layer.w_gu, before)
    assert bool(torch.isfinite(layer.train_step_device(x, logits)).all())
