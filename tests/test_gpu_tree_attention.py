"""``paged_tree_attention`` where its weights are all there is to lose, against float64
(oracle/draft_tree.py)."""

import numpy as np
import pytest
import torch

from oracle import draft_tree as ref

pytestmark = pytest.mark.gpu

HALF = {"bf16": torch.bfloat16, "f16": torch.float16}


def f64(t):
    return t.detach().double().cpu().numpy()


def attend(dev, *args, **kw):
    from grpo_mi355x.kernels import paged_tree_attention

    return f64(paged_tree_attention(*(x if x is None else x.to(dev) for x in args), **kw))


def check(out, want, size, dtype, scores, adds, faint):
    """A weight in [1, 2) is two 16-bit values: in bf16 its rounding and the rest, at most 2^-8,
    whose own is 2^-17 off; in float16 what it is cut to and the rest, below 2^-10 and 2^-22 off
    (where it is subnormal 2^-25, the largest weight being 2^12 or more: 2^-37 of that, which
    `faint` sums over the tokens). It is of an exponential (2^-20) of a score of one product, which
    a few roundings of at most `scores` doublings move by 2^-22 of them. Twice that of the mean of
    |v|. A sum of `adds` float32 values one after another is off by 2^-24 of itself for each. One
    rounding of the result."""
    weight = {"bf16": 2.0 ** -17, "f16": 2.0 ** -22}[dtype] + 2.0 ** -20 + scores * 2.0 ** -22
    f = torch.finfo(HALF[dtype])
    bound = 2 * (weight + adds * 2.0 ** -24) * size + faint + f.eps / 2 * (np.abs(want) + f.tiny)
    worst = float((np.abs(out - want) / bound).max())
    assert worst <= 1, worst


@pytest.mark.parametrize("dtype", list(HALF))
@pytest.mark.parametrize("t,hq,hkv,d", [(8, 4, 2, 128), (40, 8, 2, 128), (1, 16, 4, 128),
                                        (6, 4, 2, 64), (20, 4, 1, 64), (40, 8, 2, 64),
                                        (3, 2, 1, 80)])
def test_weights_are_not_rounded_to_16_bits(dev, dtype, t, hq, hkv, d):
    """Means of values of both signs that almost cancel: their weights, of two sizes, would show
    in the result with 2^-9 (2^-12) of them lost."""
    g = torch.Generator().manual_seed(d + t)
    n, block, dt = 200, 16, HALF[dtype]
    nb = -(-(n + t) // block)
    kc, vc = (torch.zeros(nb, hkv, block, d, dtype=dt) for _ in range(2))
    faint = torch.rand(nb, hkv, block, generator=g) < 0.6
    kc[..., 0] = torch.where(faint, -1.0, 0.0).to(dt)
    vc[:] = (torch.randint(0, 2, vc.shape, generator=g) * 2 - 1).to(dt)
    q = torch.zeros(1, t, hq, d, dtype=dt)
    q[..., 0] = (torch.rand(1, t, hq, generator=g) * 3).to(dt)  # weights of 1 and exp(-0 .. -3)
    tables = torch.randperm(nb, generator=g).view(1, nb).int()
    lens = torch.tensor([n], dtype=torch.int32)
    out = attend(dev, q, kc, vc, tables, lens, scale=1.0)
    want, size = ref.tree_attention(f64(q), f64(kc), f64(vc), tables.numpy(), lens.numpy(),
                                    scale=1.0)
    # (a lane adds every fourth weight, with other dims than 64 and 128 a thread every one)
    check(out, want, size, dtype, 5, n + t if d == 80 else (n + t) / 4, (n + t) * 2.0 ** -37)


@pytest.mark.parametrize("dtype", list(HALF))
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("nats", [9.0, 17.0, 20.0])
def test_a_long_tail_beside_one_token_that_stands_out(dev, dtype, d, nats):
    """The first token has nearly all the mass and a value of 0; what the tail gives is its mass.
    One workgroup takes it all: there are more (sequence, head) pairs than parts."""
    b, n, block, dt = 130, 131071, 16, HALF[dtype]
    nb = -(-(n + 1) // block)
    kc, vc = (torch.zeros(nb, 1, block, d, dtype=dt) for _ in range(2))
    kc[..., 0] = -nats
    vc[:] = torch.linspace(-1, 1, d).to(dt)
    tables = torch.arange(nb).int()[None].repeat(b, 1)
    kc[0, :, 0] = 0
    vc[0, :, 0] = 0
    lens = torch.zeros(b, dtype=torch.int32)
    lens[77] = n
    q = torch.zeros(b, 1, 2, d, dtype=dt)
    q[..., 0] = 1
    q[..., 1, :] *= 0.5  # half the distance
    out = attend(dev, q, kc, vc, tables, lens, scale=1.0)[77:78]
    want, size = ref.tree_attention(f64(q[77:78]), f64(kc), f64(vc), tables[77:78].numpy(),
                                    lens[77:78].numpy(), scale=1.0)
    check(out, want, size, dtype, 1.5 * nats, (n + 1) / 4, (n + 1) * 2.0 ** -37)


@pytest.mark.parametrize("d", [64, 80, 128])
@pytest.mark.parametrize("parents", [None, [[-1, 0, 0]]])
def test_lengths_past_the_table(dev, d, parents):
    """A length past the block table is all of the table, and no node has a slot."""
    g = torch.Generator().manual_seed(d)
    kc, vc = (torch.randn(12, 2, 16, d, generator=g).bfloat16() for _ in range(2))
    q = torch.randn(3, 3, 4, d, generator=g).bfloat16()
    tables = torch.arange(12).view(3, 4).int()
    if parents is not None:
        parents = torch.tensor(parents, dtype=torch.int32).expand(3, 3)
    full = attend(dev, q, kc, vc, tables, torch.full((3,), 64, dtype=torch.int32), parents)
    want, _ = ref.tree_attention(f64(q), f64(kc), f64(vc), tables.numpy(), [64] * 3)
    assert np.abs(full - want).max() < 0.02
    for most in (65, 1 << 20, (1 << 31) - 3, (1 << 31) - 1):
        lens = torch.tensor([most, 64, most], dtype=torch.int32)
        assert (attend(dev, q, kc, vc, tables, lens, parents) == full).all(), most


def long_inputs(t, hq, hkv, d, block, dtype, contexts, rest, seed):
    """Sequences of the given contexts among others of up to `rest` tokens, so many that each
    (sequence, KV head) is one workgroup's; blocks in no order; the nodes' parents at random."""
    g = torch.Generator().manual_seed(seed)
    b, dt = -(-130 // hkv) + 1, HALF[dtype]
    lens = torch.randint(0, rest, (b,), generator=g).int()
    at = torch.randperm(b, generator=g)[:len(contexts)].tolist()
    lens[at] = torch.tensor(contexts, dtype=torch.int32)
    need = -(-(lens + t) // block)
    nb = int(need.sum()) + 3
    ids, used = torch.randperm(nb, generator=g).int(), 0
    tables = torch.full((b, int(need.max())), -1, dtype=torch.int32)
    for i, n in enumerate(need.tolist()):
        tables[i, :n] = ids[used:used + n]
        used += n
    kc, vc = (torch.randn(nb, hkv, block, d, generator=g).to(dt) for _ in range(2))
    q = (torch.randn(b, t, hq, d, generator=g) * 1.5).to(dt)
    parents = torch.full((b, t), -1, dtype=torch.int32)
    for i in range(1, t):
        parents[:, i] = torch.randint(0, i, (b,), generator=g)
    counts = torch.randint(t // 2 + 1, t + 1, (b,), generator=g).int()
    return [q, kc, vc, tables, lens, parents, counts], at


def check_some(out, args, some):
    """The sequences `some`, as test_gpu_draft_tree bounds them; nodes past the counts are 0."""
    from test_gpu_draft_tree import check_attention

    q, kc, vc, tables, lens, parents, counts = args
    assert np.isfinite(out).all()
    check_attention(torch.from_numpy(out[some]), q[some], kc, vc, tables[some], lens[some],
                    parents[some], counts[some])
    for i, n in enumerate(counts.tolist()):
        assert (out[i, n:] == 0).all()


WHOLE = [
    # t, hq, hkv, d, block: by rows of a KV head, 2 (64 dims), 4 and 8 waves side by side on them,
    # blocks that hold whole pieces of 1 KiB and others
    (8, 4, 2, 64, 16),
    (9, 7, 1, 64, 5),
    (20, 5, 1, 64, 16),
    (31, 4, 1, 64, 12),
    (33, 4, 1, 64, 64),
    (64, 7, 1, 64, 6),
    (9, 3, 1, 128, 16),
    (16, 14, 2, 128, 7),
    (40, 3, 1, 128, 12),
    (43, 3, 1, 128, 16),
    (64, 7, 1, 128, 10),
]


@pytest.mark.parametrize("dtype", list(HALF))
@pytest.mark.parametrize("case", WHOLE, ids=lambda c: "-".join(map(str, c)))
def test_long_sequences_of_one_workgroup_each(dev, dtype, case):
    """More steps than the ring of K and V holds, many times over, and more tokens than one window
    of cache rows (4096): contexts that end, and trees that lie, on both sides of its borders."""
    t = case[0]
    contexts = [1000, 4096 - t // 2, 4096, 4095, 8192 - t, 8192 + 77]
    args, at = long_inputs(*case, dtype, contexts, 200, seed=t)
    out = attend(dev, *args[:6], counts=args[6].to(dev))
    check_some(out, args, at + list(range(8)))


@pytest.mark.parametrize("case", WHOLE, ids=lambda c: "-".join(map(str, c)))
def test_long_sequences_of_one_workgroup_each_with_holes(dev, case):
    """The same with missing blocks in some windows and none in others, NaN where nothing is
    attended."""
    t, block = case[0], case[4]
    contexts = [1500, 4096 - t // 2, 8192 + 77]
    args, at = long_inputs(*case, "bf16", contexts, 100, seed=t + 1)
    q, kc, vc, tables, lens, parents, counts = args
    gone = torch.zeros(tables.shape, dtype=torch.bool)
    gone[at] = torch.rand(3, tables.shape[1], generator=torch.Generator().manual_seed(t)) < 0.02
    gone[at[2], 5000 // block:] = False  # the last of its windows is whole
    gone[at[1], 4000 // block:] = False
    gone &= tables >= 0
    for x in (kc, vc):
        x[tables[gone].long()] = float("nan")
        for i in range(len(lens)):  # behind the last node
            end = int(lens[i] + counts[i])
            if end % block:
                x[tables[i, end // block], :, end % block:] = float("nan")
    tables[gone] = -1
    out = attend(dev, *args[:6], counts=counts.to(dev))
    check_some(out, args, at + list(range(8)))


@pytest.mark.parametrize("dtype", list(HALF))
@pytest.mark.parametrize("many", [False, True])  # one workgroup for a whole sequence
@pytest.mark.parametrize("t,hq,hkv,d", [(4, 12, 2, 128), (20, 12, 2, 128), (64, 8, 1, 128),
                                        (7, 4, 2, 64), (20, 5, 1, 64), (40, 8, 2, 64),
                                        (5, 2, 1, 80)])
def test_infinite_values_of_cached_tokens(dev, dtype, many, t, hq, hkv, d):
    """An infinite value of a cached token makes that dim infinite, of its sign, for every node,
    however small its weight; two of opposite signs make it NaN; other dims stay as they are."""
    g, dt = torch.Generator().manual_seed(d + t), HALF[dtype]
    b, n, block = (140 if many else 2), 1000, 16
    nb = -(-(n + t) // block) + 1
    kc, vc = (torch.randn(nb, hkv, block, d, generator=g).to(dt) for _ in range(2))
    q = torch.randn(b, t, hq, d, generator=g).to(dt)
    lens = torch.full((b,), 100, dtype=torch.int32)
    lens[1] = n
    tables = torch.randperm(nb - 1, generator=g).int().expand(b, -1)
    first = attend(dev, q, kc, vc, tables, lens)

    def put(slot, dim, x):
        vc[tables[0, slot // block], :, slot % block, dim] = x

    put(200, 3, float("inf"))  # past the others' contexts and nodes
    put(500, 4, -float("inf"))
    put(333, 5, float("nan"))
    put(333, 6, float("inf"))
    put(900, 6, -float("inf"))
    put(701, 8, float("inf"))
    put(800, 8, float("inf"))
    out = attend(dev, q, kc, vc, tables, lens)
    inf = float("inf")
    assert (out[1][..., [3, 8]] == inf).all() and (out[1][..., 4] == -inf).all()
    assert np.isnan(out[1][..., [5, 6]]).all()
    same = [i for i in range(d) if i not in (3, 4, 5, 6, 8)]
    assert (out[..., same] == first[..., same]).all()
    others = [i for i in range(b) if i != 1]
    assert (out[others] == first[others]).all()
