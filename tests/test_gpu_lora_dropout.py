"""The NF4 + LoRA linear with counter-based dropout on the adapter's input.

The kernels against float64 torch on the same rounding points (x A^T and g B, scaled, in the
type; the base product and the LoRA term of y), the mask that of
``oracle.policy_loss.dropout_factors``. Tolerance: the result's rounding u, and an
intermediate of its size that falls to the other neighbour, 2 u: 3 u of max|result|."""

import math
from types import SimpleNamespace

import pytest
import torch

from oracle.policy_loss import dropout_factors

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
SEED, OFFSET = 2 ** 61 + 99, 2 ** 34 + 5


def _close(got, want, dt, what):
    scale = want.abs().max()
    err = float((got.double() - want).abs().max() / scale) if scale else float(got.abs().max())
    print(f"{what}: {err:.2e}", flush=True)
    assert err <= 3 * U[dt], what


def _state(dev, seed=SEED, offset=OFFSET):
    return torch.tensor([seed, offset], dtype=torch.int64, device=dev)


def _layer(dev, m, n, k, r, dt, seed):
    from grpo_mi355x.core.nf4 import quantize_nf4

    g = torch.Generator().manual_seed(seed)
    rnd = lambda *s, sd=1.0: (torch.randn(*s, generator=g) * sd).to(dt).to(dev)  # noqa: E731
    packed, st = quantize_nf4((torch.randn(n, k, generator=g) * 0.02).to(dev),
                              64 if k % 64 == 0 else 32)
    packed.quant_state = st
    bias = rnd(n)
    base = SimpleNamespace(weight=packed, bias=bias)
    return base, rnd(1, m, k), rnd(1, m, n, sd=0.1), rnd(r, k, sd=0.05), rnd(n, r, sd=0.05)


def _reference(base, x, g, a, b, s, factor, dt):
    from grpo_mi355x.kernels import ops

    st = base.weight.quant_state
    n, k = st.shape
    w = ops.nf4_dequant(base.weight.view(-1), st.absmax, st.code, n * k, st.blocksize,
                        dtype=dt).view(n, k).double()
    rt = lambda t: t.to(dt).double()  # noqa: E731
    x, g = x.reshape(-1, k), g.reshape(-1, n)
    keep = lambda t: torch.where(factor > 0, t.double(), 0.0)  # noqa: E731
    x, g, a, b, f = x.double(), g.double(), a.double(), b.double(), s * float(factor.max())
    gi, xa = rt(f * (g @ b)), rt(f * (keep(x) @ a.t()))
    y = rt(rt(x @ w.t()) + base.bias.double()) + rt(xa @ b.t())
    return y, g @ w + keep(gi @ a), gi.t() @ keep(x), g.t() @ xa


# one row to past each GEMM tile and row slice, remainders of every column tile, ranks
# below, at and past a tile of 16
SHAPES = [(1, 32, 32, 1), (16, 128, 64, 16), (33, 160, 544, 8), (127, 256, 1536, 17),
          (300, 1536, 96, 32), (1050, 288, 1024, 16), (1300, 4096, 512, 5),
          (8200, 512, 1536, 16), (1050, 1024, 288, 16), (2100, 160, 1536, 8)]


@pytest.mark.parametrize("m,n,k,r", SHAPES)
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("p", [0.1, 0.75])
def test_forward_and_gradients(dev, m, n, k, r, dt, p):
    from grpo_mi355x.kernels import lora_fused_forward

    base, x, g, a, b = _layer(dev, m, n, k, r, dt, m + n + k + r)
    leaves = [t.clone().requires_grad_() for t in (x, a, b)]
    y = lora_fused_forward(leaves[0], base_layer=base, lora_A=leaves[1], lora_B=leaves[2],
                           scaling=1.7, dropout=torch.nn.Dropout(p), dropout_rng=_state(dev))
    grads = torch.autograd.grad(y, leaves, g)
    factor = torch.from_numpy(dropout_factors(m * k, p, SEED, OFFSET)).float().view(m, k).to(dev)
    want = _reference(base, x, g, a, b, 1.7, factor, dt)
    for got, ref, what in zip((y.detach()[0], grads[0][0], *grads[1:]), want,
                              ("y", "grad_x", "grad_A", "grad_B")):
        assert got.dtype == dt
        _close(got, ref, dt, what)
    with torch.no_grad():
        again = lora_fused_forward(x, base_layer=base, lora_A=a, lora_B=b, scaling=1.7,
                                   dropout=torch.nn.Dropout(p), dropout_rng=_state(dev))
    assert torch.equal(again, y.detach())


def test_the_shapes_reach_every_tile():
    import ctypes

    from grpo_mi355x import _lib

    def tile(m, n):
        a, b = ctypes.c_int(0), ctypes.c_int(0)
        _lib.check(_lib.library().grpo_gemm16_tile(m, n, ctypes.byref(a), ctypes.byref(b)), "tile")
        return a.value, b.value

    # grad_x [M, K], whose epilogue makes the mask
    assert {tile(m, k) for m, _, k, _ in SHAPES} == {(256, 256), (128, 128), (64, 128), (64, 64)}


@pytest.mark.parametrize("which", ["x", "a", "b"])
def test_gradients_by_differences(dev, which):
    """y is linear in each of x, A and B for a given mask: <y(t + d) - y(t), g> is
    <grad_t, d>, up to the roundings of the two ys and of the gradient."""
    from grpo_mi355x.kernels import lora_fused_forward

    dt = torch.float16
    base, x, g, a, b = _layer(dev, 70, 96, 128, 8, dt, 5)
    t = dict(x=x, a=a, b=b)

    def y(**kw):
        v = {**t, **kw}
        return lora_fused_forward(v["x"], base_layer=base, lora_A=v["a"], lora_B=v["b"],
                                  scaling=2.0, dropout=torch.nn.Dropout(0.3),
                                  dropout_rng=_state(dev))

    leaf = t[which].clone().requires_grad_()
    grad, = torch.autograd.grad(y(**{which: leaf}), leaf, g)
    d = (torch.randn(leaf.shape, generator=torch.Generator().manual_seed(2)) * 0.5).to(dt).to(dev)
    moved = (t[which] + d).to(dt)
    d = moved.double() - t[which].double()
    with torch.no_grad():
        up, at = y(**{which: moved}).double(), y().double()
    got, want = float(((up - at) * g.double()).sum()), float((grad.double() * d).sum())
    # three roundings of each y and its parts, of the size of |y|; each gradient's 3 u
    tol = U[dt] * 3 * float(((up.abs() + at.abs() + 2 * base.bias.double().abs())
                             * g.double().abs()).sum())
    tol += 3 * U[dt] * float(grad.double().abs().max() * d.abs().sum())
    assert abs(got - want) <= tol
    assert abs(want) > 5 * tol / math.sqrt(g.numel())  # the bound is far below the value's size


def test_dropped_values_may_be_anything(dev):
    """An infinity in x reaches its row's base product; where its place is dropped it stays
    out of the adapter's gradient."""
    from grpo_mi355x.kernels import lora_fused_forward

    m, k = 40, 64
    base, x, g, a, b = _layer(dev, m, 64, k, 8, torch.bfloat16, 3)
    f = torch.from_numpy(dropout_factors(m * k, 0.5, SEED, OFFSET)).view(m, k)
    row, col = (int(v[0]) for v in torch.nonzero(f == 0, as_tuple=True))
    x[0, row, col] = math.inf
    av = a.clone().requires_grad_()
    y = lora_fused_forward(x, base_layer=base, lora_A=av, lora_B=b, scaling=1.0,
                           dropout=torch.nn.Dropout(0.5), dropout_rng=_state(dev))
    grad, = torch.autograd.grad(y, av, g)
    assert torch.isfinite(grad).all()


def test_what_the_linear_refuses_and_leaves_out(dev):
    from grpo_mi355x.kernels import lora_fused_forward

    base, x, g, a, b = _layer(dev, 8, 64, 64, 8, torch.bfloat16, 1)
    kw = dict(base_layer=base, lora_A=a, lora_B=b, scaling=1.0)
    with pytest.raises(ValueError, match="Dropout is not supported"):
        lora_fused_forward(x, dropout=torch.nn.Dropout(0.1), **kw)
    with pytest.raises(ValueError, match="two values"):
        lora_fused_forward(x, dropout=torch.nn.Dropout(0.1), dropout_rng=_state(dev)[:1], **kw)
    with pytest.raises(ValueError, match="dropout p"):
        lora_fused_forward(x, dropout=torch.nn.Dropout(1.0), dropout_rng=_state(dev), **kw)
    plain = lora_fused_forward(x, **kw)
    for dropout in (torch.nn.Dropout(0.5).eval(), torch.nn.Dropout(0.0), torch.nn.Identity(), None):
        assert torch.equal(lora_fused_forward(x, dropout=dropout, dropout_rng=_state(dev), **kw),
                           plain)
    odd, x2, _, a2, b2 = _layer(dev, 8, 48, 64, 8, torch.bfloat16, 1)
    with pytest.raises(ValueError, match="multiples of 32"):
        lora_fused_forward(x2, base_layer=odd, lora_A=a2, lora_B=b2, scaling=1.0,
                           dropout=torch.nn.Dropout(0.5), dropout_rng=_state(dev))
    none = lora_fused_forward(x[:, :0].clone().requires_grad_(), dropout=torch.nn.Dropout(0.5),
                              dropout_rng=_state(dev), **kw)
    assert none.shape == (1, 0, 64)
    none.sum().backward()
    # off the kernels' alignment: copied, not refused
    shifted = torch.cat([x.reshape(-1)[:1], x.reshape(-1)])[1:].view(x.shape)
    args = dict(dropout=torch.nn.Dropout(0.5), dropout_rng=_state(dev), **kw)
    assert torch.equal(lora_fused_forward(shifted, **args), lora_fused_forward(x, **args))


def test_adapter_branch(dev):
    """A base layer that is not quantized: the same mask on the adapter's input."""
    from grpo_mi355x.kernels import counter_dropout, lora_fused_forward

    lin = torch.nn.Linear(24, 40, device=dev, dtype=torch.bfloat16)
    g = torch.Generator().manual_seed(1)
    a, b, x = ((torch.randn(*s, generator=g) * 0.1).bfloat16().to(dev)
               for s in ((4, 24), (40, 4), (2, 5, 24)))
    got = lora_fused_forward(x, base_layer=lin, lora_A=a, lora_B=b, scaling=2.0,
                             dropout=torch.nn.Dropout(0.4), dropout_rng=_state(dev))
    xd = counter_dropout(x, 0.4, _state(dev)).double()
    want = lin(x).double() + 2.0 * (xd @ a.double().t()) @ b.double().t()
    # t, u, their product and the sum each rounded once to bf16
    off = (got.double() - want).detach().abs().max() / want.detach().abs().max()
    assert float(off) <= 4 * U[torch.bfloat16]


@pytest.mark.parametrize("n", [64, 48])
def test_layer_with_counter_dropout(dev, n):
    """``ManualLoRALayer(counter_dropout=True)``: fused where the shape allows, by parts
    otherwise; reproducible by torch's seed, a new mask each call, none in eval mode."""
    from grpo_mi355x.core.lora import ManualLoRALayer
    from grpo_mi355x.core.nf4 import Linear4bitNF4
    from grpo_mi355x.kernels.dropout import CounterDropout

    g = torch.Generator().manual_seed(4)
    base = Linear4bitNF4.from_weight(torch.randn(n, 64, generator=g) * 0.02, None)
    layer = ManualLoRALayer(base, rank=8, alpha=16, dropout=0.25,
                            counter_dropout=True).to(dev).to(torch.bfloat16)
    with torch.no_grad():
        layer.lora_B.weight.normal_(std=0.05)
    assert isinstance(layer.lora_dropout, CounterDropout)
    x = torch.randn(2, 9, 64, generator=g).bfloat16().to(dev)
    torch.manual_seed(7)
    one, two = layer(x), layer(x)
    torch.manual_seed(7)
    rng = CounterDropout.draw(torch.device(dev))
    torch.manual_seed(7)
    assert torch.equal(layer(x), one) and not torch.equal(one, two)
    f = torch.from_numpy(dropout_factors(x.numel(), 0.25, *rng.tolist())).view(x.shape).to(dev)
    a, b = layer.lora_A.weight.double(), layer.lora_B.weight.double()
    want = base(x).double() + 2.0 * ((x.double() * f) @ a.t()) @ b.t()
    # drop(x), t, u and y rounded once each
    off = (one.double() - want).detach().abs().max() / want.detach().abs().max()
    assert float(off) <= 4 * U[torch.bfloat16]
    (one.float() ** 2).sum().backward()
    assert layer.lora_A.weight.grad.abs().sum() > 0
    layer.eval()
    assert torch.equal(layer(x), layer(x))
    plain = ManualLoRALayer(base, rank=8, alpha=16, dropout=0.25).to(dev).to(torch.bfloat16)
    assert type(plain.lora_dropout) is torch.nn.Dropout  # the default is what it was


def test_captured_and_replayed(dev):
    """Forward and backward in one graph; the mask follows the state tensor."""
    from grpo_mi355x.kernels import lora_fused_forward

    base, x, g, a, b = _layer(dev, 65, 64, 96, 8, torch.bfloat16, 9)
    base.bias = None
    drop, rng = torch.nn.Dropout(0.3), _state(dev)

    def step(leaves, state):
        y = lora_fused_forward(leaves[0], base_layer=base, lora_A=leaves[1], lora_B=leaves[2],
                               scaling=2.0, dropout=drop, dropout_rng=state)
        return [y.detach(), *torch.autograd.grad(y, leaves, g)]

    fresh = lambda: [t.clone().requires_grad_() for t in (x, a, b)]  # noqa: E731
    held = fresh()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(held, rng)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(held, rng)
    for k in range(4):
        rng.copy_(_state(dev, SEED, k))
        graph.replay()
        torch.cuda.synchronize()
        for u, v in zip(out, step(fresh(), _state(dev, SEED, k))):
            assert torch.equal(u, v)
        torch.cuda.synchronize()


def test_checkpointed_layer(dev):
    """Activation checkpointing draws the mask again and gets the same one."""
    from torch.utils.checkpoint import checkpoint

    from grpo_mi355x.core.lora import ManualLoRALayer
    from grpo_mi355x.core.nf4 import Linear4bitNF4

    g = torch.Generator().manual_seed(4)
    base = Linear4bitNF4.from_weight(torch.randn(64, 64, generator=g) * 0.05, None)
    layer = ManualLoRALayer(base, rank=8, alpha=16, dropout=0.3,
                            counter_dropout=True).to(dev).to(torch.bfloat16)
    with torch.no_grad():
        layer.lora_B.weight.normal_(std=0.05)
    x = torch.randn(2, 9, 64, generator=g).bfloat16().to(dev)
    got = []
    for run in (lambda t: layer(layer(t)),
                lambda t: checkpoint(lambda u: layer(layer(u)), t, use_reentrant=False)):
        layer.zero_grad()
        torch.manual_seed(5)
        leaf = x.clone().requires_grad_()
        (run(leaf).float() ** 2).sum().backward()
        got.append((leaf.grad, layer.lora_A.weight.grad.clone(), layer.lora_B.weight.grad.clone()))
    for u, v in zip(*got):
        assert torch.equal(u, v)


@pytest.mark.parametrize("m,n,k,r", [(5, 64, 64, 4), (33, 160, 544, 8), (127, 256, 512, 17),
                                     (1050, 288, 1024, 16), (1300, 512, 96, 32)])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_results_are_rounded_once(dev, m, n, k, r, dt):
    """The definition in float64, without any rounding on the way. Each element: half a step of
    its own size, the float32 sums (e = 2^-24 a term of the sums of absolute terms, both
    stages), and what two 16-bit values leave of x A^T and g B (u^2 of them, and half of
    float16's least step where that is more) in the products that follow."""
    from grpo_mi355x.kernels import lora_fused_forward, ops

    base, x, g, a, b = _layer(dev, m, n, k, r, dt, seed=m + n)
    p, s = 0.25, 1.7
    leaves = [t.clone().requires_grad_() for t in (x, a, b)]
    y = lora_fused_forward(leaves[0], base_layer=base, lora_A=leaves[1], lora_B=leaves[2],
                           scaling=s, dropout=torch.nn.Dropout(p), dropout_rng=_state(dev))
    grads = torch.autograd.grad(y, leaves, g)
    st = base.weight.quant_state
    w = ops.nf4_dequant(base.weight.view(-1), st.absmax, st.code, n * k, st.blocksize,
                        dtype=dt).view(n, k).double().cpu()
    x, g, a, b, bias = (t.double().cpu() for t in (x[0], g[0], a, b, base.bias))
    on = torch.from_numpy(dropout_factors(m * k, p, SEED, OFFSET)).view(m, k) > 0
    f, xk = s / (1 - p), torch.where(on, x, 0.0)
    t, gi = f * xk @ a.t(), f * g @ b
    want = [x @ w.t() + bias + t @ b.t(), g @ w + torch.where(on, gi @ a, 0.0), gi.t() @ xk,
            g.t() @ t]
    absent = 2.0 ** -25 if dt == torch.float16 else 2.0 ** -134
    split = lambda v: U[dt] ** 2 * v.abs() + absent  # noqa: E731
    sums = lambda terms: (terms + 64) * 2.0 ** -24  # noqa: E731
    xk, x, g, a, b, w = (v.abs() for v in (xk, x, g, a, b, w))
    ta, ga = f * xk @ a.t(), f * g @ b  # of absolute terms
    t, gi = split(t) + sums(k) * ta, split(gi) + sums(n) * ga  # what they are off by
    slack = [sums(k) * (x @ w.t() + bias.abs()) + sums(r) * ta @ b.t() + t @ b.t(),
             sums(n) * g @ w + sums(r) * ga @ a + gi @ a,
             sums(m) * ga.t() @ xk + gi.t() @ xk, sums(m) * g.t() @ ta + g.t() @ t]
    for name, got, v, more in zip(("y", "grad_x", "grad_a", "grad_b"), (y[0], grads[0][0],
                                                                       *grads[1:]), want, slack):
        off = (got.detach().double().cpu() - v).abs() - more
        assert (off <= U[dt] * v.abs() + absent).all(), (name, float((off / v.abs()).max()) / U[dt])


@pytest.mark.parametrize("m", [1, 8, 64, 256])
@pytest.mark.parametrize("n, k", [(256, 512), (512, 256)])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_few_rows_beside_the_linear_without_dropout(dev, m, n, k, dt):
    """A share of 1/65536 and a draw that drops nothing: the linear without dropout, by its own
    route and rounding points (three of y and one of x A^T), 5 half steps of the largest."""
    from grpo_mi355x.kernels import lora_fused_forward

    base, x, _, a, b = _layer(dev, m, n, k, 16, dt, seed=m + n)
    p = 1 / 65536
    offset = next(o for o in range(1000) if dropout_factors(m * k, p, SEED, o).all())
    kw = dict(base_layer=base, lora_A=a, lora_B=b, scaling=2.0)
    y = lora_fused_forward(x, dropout=torch.nn.Dropout(p), dropout_rng=_state(dev, SEED, offset),
                           **kw)
    plain = lora_fused_forward(x, **kw).double()
    assert float((y.double() - plain).abs().max()) <= 5 * U[dt] * float(plain.abs().max())
