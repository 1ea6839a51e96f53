"""The policy update's operators in a run, as a trainer uses them: LoRA layers with
counter-based dropout, a head, the old and the reference policy's log-probabilities, the
loss and its gradients, against the same update in float64.

Tolerance: a gradient passes at most 14 tensors rounded to bf16 (t, x W, u and y of two
layers, the logits, their gradient, and gi, grad_x and the adapters' of each), each off by at
most 2^-8 of its size: 14 * 2^-8 of the gradient's norm."""

from types import SimpleNamespace

import pytest
import torch

from oracle.policy_loss import dropout_factors

pytestmark = pytest.mark.gpu


def _model(dev, hidden, vocab, seed):
    from grpo_mi355x.core.lora import ManualLoRALayer
    from grpo_mi355x.core.nf4 import Linear4bitNF4

    g = torch.Generator().manual_seed(seed)
    layers = []
    for _ in range(2):
        base = Linear4bitNF4.from_weight(torch.randn(hidden, hidden, generator=g) * 0.1, None)
        layer = ManualLoRALayer(base, rank=8, alpha=16, dropout=0.1, counter_dropout=True)
        layer.lora_A.weight.data = torch.randn(8, hidden, generator=g) * 0.1
        layer.lora_B.weight.data = torch.randn(hidden, 8, generator=g) * 0.1
        layers.append(layer.to(dev).to(torch.bfloat16))
    head = (torch.randn(vocab, hidden, generator=g) * 0.2).bfloat16().to(dev)
    return layers, head


def test_one_update(dev):
    from grpo_mi355x import kernels
    from grpo_mi355x.kernels.dropout import CounterDropout

    b, s, hidden, vocab = 4, 30, 64, 1000
    layers, head = _model(dev, hidden, vocab, 1)
    g = torch.Generator().manual_seed(2)
    x = torch.randn(b, s, hidden, generator=g).bfloat16().to(dev)
    ids = torch.randint(0, vocab, (b, s), generator=g).to(dev)
    mask = (torch.arange(s)[None] < torch.tensor([30, 1, 17, 0])[:, None]).to(dev)
    adv = torch.tensor([1.0, -0.5, -1.5, 1.0], device=dev)

    def logits(h):
        for layer in layers:
            h = layer(h)
        return h.view(-1, hidden) @ head.t()

    for layer in layers:
        layer.eval()
    with torch.no_grad():  # the rollout's policy, and a reference near it
        old, ent = kernels.token_logprobs(logits(x).view(b, s, vocab), ids, mask,
                                          return_entropy=True)
        ref = old - 0.05
    assert (ent[mask] > 0).all() and not ent[~mask].any()
    for layer in layers:
        layer.train()
    torch.manual_seed(3)
    draws = [CounterDropout.draw(x.device) for _ in layers]
    torch.manual_seed(3)
    kw = dict(ref_logps=ref, beta=0.04, eps_high=100.0, eps_low=1.0, delta=None,
              normalizer="sequences")
    loss, logp, metrics = kernels.fused_grpo_loss(logits(x).view(b, s, vocab), ids, old, adv,
                                                  mask, **kw)
    loss.backward()

    # the same in float64, with the clip out of reach (no border to fall on either side of)
    h, params = x.double(), []
    for layer, rng in zip(layers, draws):
        f = torch.from_numpy(dropout_factors(x.numel(), 0.1, *rng.tolist())).view(x.shape).to(dev)
        w = layer.base_layer.dequantize().double()
        a, bb = (p.weight.detach().double().requires_grad_() for p in (layer.lora_A, layer.lora_B))
        params.append((a, bb))
        h = h @ w.t() + 2.0 * ((h * f) @ a.t()) @ bb.t()
    lp = torch.log_softmax(h @ head.double().t(), -1).gather(-1, ids[..., None])[..., 0]
    q = torch.where(mask, ref.double() - lp, 0.0)
    term = 0.04 * (q.exp() - q - 1) - (lp - old.double()).exp() * adv.double()[:, None]
    n = mask.sum(1, keepdim=True)
    want = (term * mask.double() / n.clamp(min=1) / 3).sum()
    want.backward()
    bound = 14 * 2.0 ** -8
    assert abs(float(loss.detach()) - float(want.detach())) <= bound * float(
        term.detach()[mask].abs().mean())
    assert not logp[~mask].any() and (metrics[0] > 0)
    for layer, (a, bb) in zip(layers, params):
        for p, d in ((layer.lora_A, a), (layer.lora_B, bb)):
            off = (p.weight.grad.double() - d.grad).norm() / d.grad.norm()
            print(f"grad off by {float(off):.2e}", flush=True)
            assert off <= bound


def test_where_another_device_is_current(dev, monkeypatch):
    """Every operator makes its tensors' device the current one for its launches."""
    from grpo_mi355x import kernels
    from grpo_mi355x.core.nf4 import quantize_nf4

    g = torch.Generator().manual_seed(1)
    rnd = lambda *s: torch.randn(*s, generator=g).bfloat16().to(dev)  # noqa: E731
    packed, state = quantize_nf4(rnd(64, 96).float(), 32)
    packed.quant_state = state
    base = SimpleNamespace(weight=packed, bias=None)
    x, a, b, logits = rnd(2, 5, 96), rnd(8, 96), rnd(64, 8), rnd(2, 5, 64)
    ids, adv = torch.arange(10, device=dev).view(2, 5), torch.tensor([1.0, -1.0], device=dev)
    rng = torch.tensor([3, 4], device=dev)

    def go():
        leaf = logits.clone().requires_grad_()
        logp = kernels.token_logprobs(leaf, ids)
        return [logp.detach(), kernels.grpo_policy_loss(logp, None, adv)[0].detach(),
                kernels.fused_grpo_loss(leaf, ids, None, adv)[0].detach(),
                kernels.counter_dropout(x, 0.3, rng),
                kernels.lora_fused_forward(x, base_layer=base, lora_A=a, lora_B=b, scaling=2.0,
                                           dropout=torch.nn.Dropout(0.3), dropout_rng=rng)]

    want, entered = go(), []

    class Entered(torch.cuda.device):
        def __init__(self, d):
            entered.append(d)
            super().__init__(d)

    monkeypatch.setattr(torch.cuda, "current_device", lambda: 1)
    monkeypatch.setattr(torch.cuda, "device", Entered)
    got = go()
    monkeypatch.undo()
    assert len(entered) == 5 and all(d.index == 0 for d in entered)
    for u, v in zip(got, want):
        assert torch.equal(u, v)
