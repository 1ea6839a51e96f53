"""Forward-mode derivatives of the policy update's operators: a dual tensor does not require
a gradient, so a call that looks at ``requires_grad`` alone would return its result without a
tangent, which forward mode reads as 0. Dropout has its tangent (it is linear: the tangent
under the same mask, bit for bit); the others raise."""

from types import SimpleNamespace

import pytest
import torch
import torch.autograd.forward_ad as fwAD

pytestmark = pytest.mark.gpu


def _inputs(dev):
    g = torch.Generator().manual_seed(3)
    logits, logps = torch.randn(2, 3, 40, generator=g), -torch.rand(2, 3, generator=g)
    ids = torch.randint(0, 40, (2, 3), generator=g)
    return logits.to(dev), logps.to(dev), ids.to(dev), torch.tensor([1.0, -1.0], device=dev)


@pytest.mark.parametrize("leaf", [False, True])
@pytest.mark.parametrize("grad", [False, True])
def test_losses_raise(dev, leaf, grad):
    from grpo_mi355x import kernels

    logits, logps, ids, adv = _inputs(dev)
    calls = [(logits, lambda x: kernels.token_logprobs(x, ids)),
             (logits, lambda x: kernels.token_logprobs(x, ids, return_entropy=True)),
             (logits, lambda x: kernels.fused_grpo_loss(x, ids, None, adv)),
             (logps, lambda x: kernels.grpo_policy_loss(x, None, adv))]
    for x, call in calls:
        x = x.clone().requires_grad_(leaf)
        with torch.set_grad_enabled(grad), fwAD.dual_level():
            with pytest.raises(RuntimeError, match="jvp"):
                call(fwAD.make_dual(x, torch.ones_like(x)))
            call(x)  # a level alone changes nothing


@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_dropout_has_a_tangent(dev, dtype, grad):
    from grpo_mi355x import kernels

    g = torch.Generator().manual_seed(4)
    x, t = (torch.randn(7, 33, generator=g).to(dtype).to(dev) for _ in range(2))
    rng = torch.tensor([5, 6], device=dev)
    with torch.set_grad_enabled(grad), fwAD.dual_level():
        y = fwAD.unpack_dual(kernels.counter_dropout(fwAD.make_dual(x, t), 0.4, rng))
        assert torch.equal(y.primal, kernels.counter_dropout(x, 0.4, rng))
        assert torch.equal(y.tangent, kernels.counter_dropout(t, 0.4, rng))


def test_dropout_tangent_is_differentiable(dev):
    from grpo_mi355x import kernels

    t = torch.randn(5, 9, generator=torch.Generator().manual_seed(5)).to(dev).requires_grad_()
    rng = torch.tensor([8, 1], device=dev)
    with fwAD.dual_level():
        dual = fwAD.make_dual(torch.ones_like(t).requires_grad_(), t)
        y = fwAD.unpack_dual(kernels.counter_dropout(dual, 0.5, rng)).tangent
        grad, = torch.autograd.grad(y.sum(), t)
    assert torch.equal(grad, kernels.counter_dropout(torch.ones_like(t), 0.5, rng))


@pytest.mark.parametrize("grad", [False, True])
def test_dropout_linear_raises(dev, grad):
    from grpo_mi355x.core.nf4 import quantize_nf4
    from grpo_mi355x.kernels import lora_fused_forward

    g = torch.Generator().manual_seed(6)
    packed, st = quantize_nf4((torch.randn(64, 64, generator=g) * 0.02).to(dev), 64)
    packed.quant_state = st
    a, b, x = (torch.randn(*s, generator=g).bfloat16().to(dev) for s in ((8, 64), (64, 8),
                                                                        (1, 5, 64)))
    kw = dict(base_layer=SimpleNamespace(weight=packed, bias=None), lora_A=a, lora_B=b,
              scaling=2.0, dropout=torch.nn.Dropout(0.3), dropout_rng=torch.tensor([1, 2], device=dev))
    with torch.set_grad_enabled(grad), fwAD.dual_level():
        with pytest.raises(RuntimeError, match="jvp"):
            lora_fused_forward(fwAD.make_dual(x, torch.ones_like(x)), **kw)


@pytest.mark.parametrize("use_triton", [True, False])
@pytest.mark.parametrize("grad", [False, True])
def test_layer_by_parts_has_the_whole_tangent(dev, grad, use_triton):
    """The layer runs by parts in forward mode and is linear in x: its tangent is the layer of
    the tangent by parts, operation for operation, at the same draw."""
    from grpo_mi355x.core.lora import ManualLoRALayer
    from grpo_mi355x.core.nf4 import Linear4bitNF4

    g = torch.Generator().manual_seed(7)
    base = Linear4bitNF4.from_weight(torch.randn(64, 64, generator=g) * 0.02, None)
    layer = ManualLoRALayer(base, rank=8, alpha=16, dropout=0.25, use_triton=use_triton,
                            counter_dropout=True).to(dev).to(torch.bfloat16)
    with torch.no_grad():
        layer.lora_B.weight.normal_(std=0.5)
    x, t = (torch.randn(1, 9, 64, generator=g).bfloat16().to(dev) for _ in range(2))
    with torch.set_grad_enabled(grad), fwAD.dual_level():
        torch.manual_seed(9)
        y = fwAD.unpack_dual(layer(fwAD.make_dual(x, t)))
    layer.use_triton = False
    torch.manual_seed(9)
    want = layer(t).double()
    base_only = base(t).double()
    assert (want - base_only).abs().max() > 0.1 * want.abs().max()  # the adapter counts
    # two roundings of the base product and of each adapter product, sums apart: 8 half steps
    off = (y.tangent.double() - want).abs().max() / want.abs().max()
    assert float(off.detach()) <= 8 * 2.0 ** -8


def test_transforms(dev):
    """A batched call's constants give what they give outside; a transform's own tensors raise."""
    from grpo_mi355x import kernels

    logits, logps, ids, adv = _inputs(dev)
    rng = torch.tensor([5, 6], device=dev)
    calls = [(logits, lambda x: kernels.token_logprobs(x, ids)),
             (logits, lambda x: kernels.fused_grpo_loss(x, ids, None, adv)[0]),
             (logps, lambda x: kernels.grpo_policy_loss(x, None, adv)[0]),
             (logits, lambda x: kernels.counter_dropout(x, 0.4, rng))]
    one = torch.ones(3, device=dev)
    for x, call in calls:
        want = call(x).sum()
        assert torch.equal(torch.vmap(lambda v: v * call(x).sum())(one), one * want)
        for transform in (lambda f: torch.vmap(f)(torch.stack([x, x])),
                          lambda f: torch.func.jvp(f, (x,), (x,)),
                          lambda f: torch.func.grad(lambda v: f(v).sum())(x)):
            with pytest.raises(RuntimeError):
                transform(call)
