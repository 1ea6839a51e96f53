"""``counter_dropout`` against the mask of ``oracle.policy_loss.dropout_factors``: bit-exact,
as each value is one float32 product rounded once to its type."""

import math

import numpy as np
import pytest
import torch

from oracle.policy_loss import dropout_factors

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def drop(x, p, rng):
    from grpo_mi355x import kernels

    return kernels.counter_dropout(x, p, rng)


def state(dev, seed, offset):
    return torch.tensor([seed, offset], dtype=torch.int64, device=dev)


def want(x, p, seed, offset):
    f = dropout_factors(x.numel(), p, seed, offset).astype(np.float32)
    f = torch.from_numpy(f).view(x.shape)
    return torch.where(f > 0, x.float() * f, torch.zeros(())).to(x.dtype)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("shape", [(1,), (7,), (8,), (9,), (3, 5), (8, 1536), (33, 127), (5, 2049)])
@pytest.mark.parametrize("p", [0.0, 0.05, 0.5, 0.97])
def test_forward_and_backward(dev, dtype, shape, p):
    seed, offset = -(2 ** 62) + 12345, 2 ** 33 + 7  # every word of key and counter
    g = torch.Generator().manual_seed(3)
    x, up = (torch.randn(*shape, generator=g).to(DT[dtype]) for _ in range(2))
    leaf = x.to(dev).requires_grad_()
    y = drop(leaf, p, state(dev, seed, offset))
    assert torch.equal(y.detach().cpu(), want(x, p, seed, offset))
    grad, = torch.autograd.grad(y, leaf, up.to(dev))
    assert torch.equal(grad.cpu(), want(up, p, seed, offset))


def test_more_values_than_one_pass_of_the_grid(dev):
    """2^31 + 24 values: past the grid's first pass and past 32-bit indexes."""
    n = 2 ** 31 + 24
    x = torch.ones(n, dtype=torch.bfloat16, device=dev)
    y = drop(x, 0.5, state(dev, 5, 6))
    from oracle.policy_loss import philox

    at = n - 24
    i = np.arange(at // 8, n // 8, dtype=np.uint64)
    ctr = np.stack([i & np.uint64(0xFFFFFFFF), i >> np.uint64(32), np.full_like(i, 6),
                    np.zeros_like(i)], 1)
    w = philox(ctr, (5, 0))
    u = np.stack([w & 0xFFFF, w >> 16], 2).reshape(-1)
    assert torch.equal(y[at:].float().cpu(),
                       torch.from_numpy(np.where(u >= 32768, 2.0, 0.0)).float())


def test_not_finite_strided_and_unaligned(dev):
    x = torch.randn(64, 40, generator=torch.Generator().manual_seed(1)).bfloat16()
    x[::3] = math.nan
    x[1::3] = math.inf
    y = drop(x.to(dev), 0.5, state(dev, 1, 2)).cpu()
    assert torch.equal(torch.nan_to_num(y, 7.0, 9.0), torch.nan_to_num(want(x, 0.5, 1, 2), 7.0, 9.0))
    assert torch.isfinite(y[::3]).any()  # a dropped NaN is 0
    full = torch.randn(50, 41, generator=torch.Generator().manual_seed(2)).to(dev)
    for v in (full[:, 1:], full.t(), full[::2], full.view(-1)[3:].view(-1), full[:1].expand(9, 41)):
        assert torch.equal(drop(v, 0.3, state(dev, 4, 4)).cpu(), want(v.cpu(), 0.3, 4, 4))
    assert drop(full[:0], 0.3, state(dev, 4, 4)).shape == (0, 41)
    flat = torch.randn(5000, device=dev).bfloat16()
    for k in range(1, 8):  # every alignment of the first value
        assert torch.equal(drop(flat[k:], 0.2, state(dev, 1, 9)).cpu(), want(flat[k:].cpu(), 0.2, 1, 9))


def test_state_changed_before_the_backward_is_refused(dev):
    x = torch.randn(16, device=dev, requires_grad=True)
    rng = state(dev, 1, 1)
    y = drop(x, 0.5, rng)
    rng[1] += 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_refusals_on_the_device(dev):
    x, rng = torch.zeros(8, device=dev), state(dev, 0, 0)
    with pytest.raises(ValueError, match="bfloat16"):
        drop(x.double(), 0.1, rng)
    with pytest.raises(ValueError, match="must be on"):
        drop(x, 0.1, rng.cpu())
    with pytest.raises(ValueError, match="two values"):
        drop(x, 0.1, rng.int())


def test_captured_graph_draws_from_the_tensor(dev):
    x = torch.randn(300, 17, generator=torch.Generator().manual_seed(5))
    held, rng = x.to(dev), state(dev, 11, 0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        drop(held, 0.4, rng)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = drop(held, 0.4, rng)
    for k in range(4):
        rng.copy_(state(dev, 11, k))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y.cpu(), want(x, 0.4, 11, k))
        drop(held, 0.1, rng)
        torch.cuda.synchronize()


def test_differentiates_twice(dev):
    """Linear in x for a given mask: the second derivative's mask is the same one."""
    x = torch.randn(5, 9, dtype=torch.float32, device=dev, requires_grad=True)
    y = drop(x, 0.5, state(dev, 8, 1)) ** 2
    first, = torch.autograd.grad(y.sum(), x, create_graph=True)
    second, = torch.autograd.grad(first.sum(), x)
    f = torch.from_numpy(dropout_factors(45, 0.5, 8, 1)).view(5, 9).float().to(dev)
    assert torch.equal(second, 2 * f * f)  # powers of two: exact
