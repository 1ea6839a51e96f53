"""The operators that check a tree of drafted tokens, against float64 (oracle/draft_tree.py)."""

import numpy as np
import pytest
import torch

from oracle import draft_tree as ref

pytestmark = pytest.mark.gpu

HALF = {"bf16": torch.bfloat16, "f16": torch.float16}


def rounding(dtype) -> float:
    """Largest relative error of one rounding."""
    return torch.finfo(dtype).eps / 2


def randn(g, *shape, dtype=torch.float32, std=1.0):
    return (torch.randn(*shape, generator=g) * std).to(dtype)


def f64(t):
    return t.detach().double().cpu().numpy()


def make_tables(g, b, width, spare=2):
    """(num_blocks, int32 [b, width]): distinct blocks in no order."""
    n = b * width + spare
    return n, torch.randperm(n, generator=g)[:b * width].view(b, width).int()


def rand_parents(g, b, t):
    up = torch.full((b, t), -1, dtype=torch.int32)
    for i in range(1, t):
        up[:, i] = torch.randint(-1 if i > 2 else 0, i, (b,), generator=g)
    return up


def tables_of_angles(d, most, dtype):
    a = torch.arange(most).double()[:, None] * 1e4 ** -(torch.arange(0, d, 2).double() / d)
    a = torch.cat([a, a], 1)
    # the halves differ, so that each is read from its own place
    return (a.cos() * torch.linspace(1, 1.25, d)).to(dtype), \
        (a.sin() * torch.linspace(0.75, 1, d)).to(dtype)


# ----------------------------------------------------------------- append --

APPEND = [
    # b, t, hq, hkv, d, block, dtype, table
    (1, 1, 1, 1, 16, 16, "bf16", "f32"),
    (3, 5, 12, 2, 128, 16, "bf16", "same"),
    (2, 61, 28, 4, 128, 16, "f16", "f32"),
    (4, 7, 14, 2, 64, 32, "f16", "same"),
    (2, 300, 4, 4, 32, 5, "bf16", "f32"),
    (3, 4, 3, 1, 10, 7, "bf16", "f32"),  # a head dim without 16-byte pieces
    (2, 3, 6, 3, 80, 16, "f16", "same"),
]


@pytest.mark.parametrize("b,t,hq,hkv,d,block,dtype,table", APPEND)
@pytest.mark.parametrize("given", [False, True])
def test_rope_append(dev, b, t, hq, hkv, d, block, dtype, table, given):
    from grpo_mi355x.kernels import paged_rope_append

    g = torch.Generator().manual_seed(b * 1000 + t)
    dt = HALF[dtype]
    width = -(-(40 + t) // block)
    nb, tables = make_tables(g, b, width)
    lens = torch.randint(0, 41, (b,), generator=g).int()
    qkv = randn(g, b, t, hq + 2 * hkv, d, dtype=dt)
    q, k, v = qkv.split((hq, hkv, hkv), 2)
    cos, sin = tables_of_angles(d, 64, dt if table == "same" else torch.float32)
    kc, vc = randn(g, nb, hkv, block, d, dtype=dt), randn(g, nb, hkv, block, d, dtype=dt)
    counts = positions = None
    if given:
        counts = torch.randint(0, t + 2, (b,), generator=g).int() - 1  # -1 and t among them
        positions = torch.randint(-2, 70, (b, t), generator=g).int()  # outside the table too
    want_q, want_k, want_v = ref.rope_append(f64(q), f64(k), f64(v), f64(cos), f64(sin), f64(kc),
                                             f64(vc), tables.numpy(), lens.numpy(),
                                             None if counts is None else counts.numpy(),
                                             None if positions is None else positions.numpy())
    at = lambda x: None if x is None else x.to(dev)  # noqa: E731
    kcd, vcd = kc.to(dev), vc.to(dev)
    qd, kd, vd = qkv.to(dev).split((hq, hkv, hkv), 2)
    out = paged_rope_append(qd, kd, vd, cos.to(dev), sin.to(dev), kcd, vcd, tables.to(dev),
                            lens.to(dev), counts=at(counts), positions=at(positions))
    # one rounding of the sum of two products, whose own roundings (float32, the second one
    # fused or not) are below 3 * 2^-24 of the larger of them, at most 1.25 * 6 here
    for got, want in ((out, want_q), (kcd, want_k)):
        err = np.abs(f64(got) - want)
        assert (err <= rounding(dt) * np.abs(want) + 3 * 2.0 ** -24 * 7.5 + 2.0 ** -25).all()
    assert torch.equal(vcd.cpu(), torch.from_numpy(want_v).to(dt))


def test_rope_append_leaves_the_rest_of_the_cache(dev):
    """Bad blocks, slots past the table, sequences without a context: nothing is written there."""
    from grpo_mi355x.kernels import paged_rope_append

    g = torch.Generator().manual_seed(5)
    b, t, hkv, d, block = 4, 6, 2, 64, 4
    tables = torch.tensor([[0, 1, 2], [3, -1, 4], [5, 6, 99], [7, 8, 9]], dtype=torch.int32)
    lens = torch.tensor([9, 2, 5, -1], dtype=torch.int32)
    qkv = randn(g, b, t, 4 + 2 * hkv, d, dtype=torch.bfloat16)
    cos, sin = tables_of_angles(d, 32, torch.float32)
    kc, vc = (randn(g, 12, hkv, block, d, dtype=torch.bfloat16) for _ in range(2))
    q, k, v = qkv.split((4, hkv, hkv), 2)
    _, want_k, want_v = ref.rope_append(f64(q), f64(k), f64(v), f64(cos), f64(sin), f64(kc),
                                        f64(vc), tables.numpy(), lens.numpy())
    kcd, vcd = kc.to(dev), vc.to(dev)
    q, k, v = qkv.to(dev).split((4, hkv, hkv), 2)
    out = paged_rope_append(q, k, v, cos.to(dev), sin.to(dev), kcd, vcd, tables.to(dev),
                            lens.to(dev))
    same = torch.from_numpy(want_v).to(torch.bfloat16) == vc
    assert torch.equal(vcd.cpu(), torch.from_numpy(want_v).to(torch.bfloat16))
    assert torch.equal((kcd.cpu() == kc) & same, (torch.from_numpy(want_k) == kc.double()) & same)
    assert (out[3] == 0).all()


# -------------------------------------------------------------- attention --

ATTEND = [
    # b, t, hq, hkv, d, block, dtype, contexts, tree, counts
    (1, 1, 1, 1, 128, 16, "bf16", [0], "chain", None),
    (2, 1, 12, 2, 128, 16, "bf16", [33, 0], "chain", None),
    (3, 4, 12, 2, 128, 16, "bf16", [700, 31, 1], "chain", None),
    (2, 16, 12, 2, 128, 16, "f16", [100, 257], "random", None),
    (3, 61, 28, 4, 128, 16, "bf16", [500, 0, 63], "random", [61, 30, 0]),
    (2, 64, 7, 1, 128, 16, "f16", [129, 1000], "random", [64, 63]),
    (2, 33, 8, 8, 64, 32, "bf16", [95, 320], "random", None),
    (2, 64, 16, 1, 64, 16, "bf16", [40, 15], "random", None),  # 1024 rows of one KV head
    (2, 9, 14, 2, 64, 64, "f16", [1, 130], "random", [9, 4]),
    (2, 20, 6, 2, 128, 7, "bf16", [50, 20], "random", None),  # a block size of no power of two
    (2, 5, 3, 1, 80, 16, "bf16", [77, 5], "random", None),
    (1, 3, 2, 2, 10, 3, "f16", [11], "random", None),
    (1, 2, 2, 1, 256, 16, "bf16", [300], "chain", None),
    (1, 8, 12, 2, 128, 16, "bf16", [9001], "random", None),
    (70, 3, 4, 2, 128, 16, "bf16", "many", "random", None),
]


def attend_inputs(b, t, hq, hkv, d, block, dtype, contexts, tree, counts, seed=0, fill=None):
    g = torch.Generator().manual_seed(seed + 17 * b + t)
    dt = HALF[dtype]
    if contexts == "many":
        contexts = torch.randint(0, 200, (b,), generator=g).tolist()
    lens = torch.tensor(contexts, dtype=torch.int32)
    nb, tables = make_tables(g, b, -(-(int(lens.max()) + t) // block))
    kc, vc = randn(g, nb, hkv, block, d, dtype=dt), randn(g, nb, hkv, block, d, dtype=dt)
    q = randn(g, b, t, hq, d, dtype=dt, std=1.5)
    parents = None if tree == "chain" else rand_parents(g, b, t)
    counts = None if counts is None else torch.tensor(counts, dtype=torch.int32)
    return q, kc, vc, tables, lens, parents, counts


def attend(dev, q, kc, vc, tables, lens, parents=None, counts=None, **kw):
    from grpo_mi355x.kernels import paged_tree_attention

    at = lambda x: None if x is None else x.to(dev)  # noqa: E731
    return paged_tree_attention(at(q), at(kc), at(vc), at(tables), at(lens), at(parents),
                                counts=at(counts), **kw)


def check_attention(out, q, kc, vc, tables, lens, parents, counts, scale=None):
    """Against float64. A weight is exp of a float32 score: its relative error is that of the
    score, d products of rounded sums (2^-24 of the sum of their magnitudes each, at most
    1.5 * 6 * 6 * d / sqrt(d)... bounded here by measuring |q||k|), plus a few 2^-23 of exp2, and
    one rounding of the weight to 16 bits where the products run on the matrix cores; numerator
    and denominator share it in the first order, twice that of the mean of |v|. The result is
    rounded once."""
    dt = q.dtype
    want, size = ref.tree_attention(f64(q), f64(kc), f64(vc), tables.numpy(), lens.numpy(),
                                    None if parents is None else parents.numpy(),
                                    None if counts is None else counts.numpy(), scale)
    d = q.shape[3]
    s = d ** -0.5 if scale is None else scale
    reach = abs(s) * float(q.double().norm(dim=-1).max()) * \
        float(torch.nan_to_num(kc.double(), 0.0, 0.0, 0.0).norm(dim=-1).max())
    weight = 2 * (rounding(dt) + (d + 8) * 2.0 ** -24 * reach + 2.0 ** -20)
    err = np.abs(f64(out) - want)
    bound = weight * size + rounding(dt) * np.abs(want) + 1e-7
    worst = float((err / bound).max())
    assert worst <= 1, worst
    # far below the bound on the whole: the roundings are independent
    if want.any():
        assert np.sqrt((err ** 2).sum() / (want ** 2).sum()) < 2 * rounding(dt)


@pytest.mark.parametrize("case", ATTEND, ids=lambda c: "-".join(map(str, c[:6])))
def test_tree_attention(dev, case):
    args = attend_inputs(*case)
    out = attend(dev, *args)
    check_attention(out, *args)
    if args[6] is not None:
        for b, n in enumerate(args[6].tolist()):
            assert (out[b, n:] == 0).all()


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("poison", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("t,hq,hkv,d", [(20, 12, 2, 128), (64, 8, 1, 128), (7, 4, 2, 64),
                                        (5, 2, 1, 80)])
def test_tree_attention_of_poisoned_slots(dev, dtype, poison, t, hq, hkv, d):
    """What no node of a sequence attends, and a drafted token that only its own descendants
    attend, do not reach the other nodes."""
    b, block = 3, 16
    q, kc, vc, tables, lens, parents, counts = attend_inputs(
        b, t, hq, hkv, d, block, dtype, [50, 0, 111], "random", [t, t - 1, t], seed=3)
    at = torch.zeros(kc.shape[0], block, dtype=torch.bool)
    for i in range(b):
        for s in range(int(lens[i]) + int(counts[i])):
            blk, off = ref.slot_of(tables[i].tolist(), s, block, kc.shape[0])
            at[blk, off] = True
    kc.permute(0, 2, 1, 3)[~at] = poison
    vc.permute(0, 2, 1, 3)[~at] = poison
    check_attention(attend(dev, q, kc, vc, tables, lens, parents, counts), q, kc, vc, tables, lens,
                    parents, counts)
    # node t // 2 of the last sequence
    node = t // 2
    blk, off = ref.slot_of(tables[2].tolist(), int(lens[2]) + node, block, kc.shape[0])
    kc[blk, :, off], vc[blk, :, off] = poison, poison
    out = attend(dev, q, kc, vc, tables, lens, parents, counts)
    hit = torch.from_numpy(ref.sees(parents[2].numpy(), t)[:, node])
    assert hit.any() and not hit.all()
    keep = torch.ones(b, t, dtype=torch.bool)
    keep[2, hit] = False
    assert torch.isfinite(out.cpu()[keep]).all()
    assert not torch.isfinite(out.cpu()[2, hit]).all(-1).any()
    kc[blk, :, off], vc[blk, :, off] = 0, 0  # not attended by the nodes that are compared
    want, _ = ref.tree_attention(f64(q), f64(kc), f64(vc), tables.numpy(), lens.numpy(),
                                 parents.numpy(), counts.numpy())
    keep = keep.numpy()
    err = np.abs(f64(out)[keep] - want[keep])
    assert np.sqrt((err ** 2).sum() / (want[keep] ** 2).sum()) < 2 * rounding(HALF[dtype])


def test_tree_attention_without_blocks(dev):
    """Missing blocks are not attended; a node that attends nothing gets 0."""
    q, kc, vc, tables, lens, parents, _ = attend_inputs(4, 8, 12, 2, 128, 16, "bf16",
                                                        [60, 40, 20, 300], "random", None)
    tables[0, 1] = -1
    tables[1] = 1 << 30
    tables[2, -1] = kc.shape[0]
    lens[2] = -1
    lens = lens.clone()
    lens[3] = tables.shape[1] * 16 - 3  # five nodes past the table
    parents[1] = -1
    args = (q, kc, vc, tables, lens, parents, None)
    out = attend(dev, *args)
    check_attention(out, *args)
    assert (out[1] == 0).all() and (out[2] == 0).all()


@pytest.mark.parametrize("t,hq,hkv,d", [(2, 12, 2, 128), (8, 12, 2, 128), (20, 12, 2, 128),
                                        (64, 7, 1, 128), (3, 4, 2, 64), (33, 14, 2, 64)])
@pytest.mark.parametrize("block", [16, 5])
def test_tree_attention_over_long_tables_with_holes(dev, t, hq, hkv, d, block):
    """Missing blocks in every part of a long table, and slots that hold NaN beside them."""
    args = attend_inputs(2, t, hq, hkv, d, block, "bf16", [9001, 4500], "random", None, seed=5)
    kc, vc, tables, lens = args[1:5]
    gone = torch.rand(tables.shape, generator=torch.Generator().manual_seed(t)) < 0.01
    gone[:, 3] = True
    gone[1, 4500 // block:] = False
    for x in (kc, vc):
        x[tables[gone].long()] = float("nan")
        blk = tables[1, (4500 + t) // block]  # what stands behind the last node
        x[blk, :, (4500 + t) % block:] = float("nan")
    tables[gone] = -1
    check_attention(attend(dev, *args), *args)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("t,hq,hkv,d", [(20, 12, 2, 128), (64, 8, 1, 128), (7, 4, 2, 64),
                                        (5, 2, 1, 80)])
def test_infinite_values_arrive_as_such(dev, dtype, t, hq, hkv, d):
    """An infinite value of an attended node makes that dim infinite, of its sign, and no other
    dim; two of opposite signs make it NaN."""
    q, kc, vc, tables, lens, parents, _ = attend_inputs(2, t, hq, hkv, d, 16, dtype, [50, 111],
                                                        "random", None, seed=6)
    parents[0, 3] = 1
    parents[0, 4] = 3

    def put(slot, dim, x):
        blk, off = ref.slot_of(tables[0].tolist(), slot, 16, kc.shape[0])
        vc[blk, :, off, dim] = x

    first = attend(dev, q, kc, vc, tables, lens, parents).cpu()
    put(50 + 1, 3, float("inf"))
    put(50 + 1, 4, -float("inf"))
    put(50 + 1, 5, float("nan"))
    put(50 + 1, 6, float("inf"))
    put(50 + 3, 6, -float("inf"))
    put(20, 9, float("inf"))
    out = attend(dev, q, kc, vc, tables, lens, parents).cpu()
    sees = torch.from_numpy(ref.sees(parents[0].numpy(), t))
    one, both = sees[:, 1], sees[:, 1] & sees[:, 3]
    assert one.any() and not one.all() and both.any()
    inf = float("inf")
    assert (out[0, one, :, 3] == inf).all() and (out[0, one, :, 4] == -inf).all()
    assert out[0, one, :, 5].isnan().all() and out[0, both, :, 6].isnan().all()
    assert (out[0, one & ~both, :, 6] == inf).all() and (out[0, :, :, 9] == inf).all()
    for dim in (3, 4, 5):
        assert torch.equal(out[0, ~one, :, dim], first[0, ~one, :, dim])
    same = [i for i in range(d) if i not in (3, 4, 5, 6, 9)]
    assert torch.equal(out[..., same], first[..., same])


def test_tree_attention_takes_odd_parents(dev):
    """A parent that is no earlier node is none; one tree may serve all sequences."""
    q, kc, vc, tables, lens, _, _ = attend_inputs(2, 6, 4, 2, 128, 16, "bf16", [40, 7], "chain",
                                                  None)
    parents = torch.tensor([[5, 1, 0, 99, 2, -7]], dtype=torch.int32).expand(2, 6)
    out = attend(dev, q, kc, vc, tables, lens, parents)
    check_attention(out, q, kc, vc, tables, lens, parents.contiguous(), None)
    from grpo_mi355x.kernels import paged_tree_attention

    shared = paged_tree_attention(q.to(dev), kc.to(dev), vc.to(dev), tables.to(dev), lens.to(dev),
                                  parents[:1].to(dev).expand(2, 6))
    assert torch.equal(shared, out)


def test_tree_attention_of_strided_queries(dev):
    q, kc, vc, tables, lens, parents, _ = attend_inputs(2, 12, 12, 2, 128, 16, "bf16", [90, 200],
                                                        "random", None)
    want = attend(dev, q, kc, vc, tables, lens, parents, scale=0.2)
    check_attention(want, q, kc, vc, tables, lens, parents, None, scale=0.2)
    for strided in (q.permute(2, 0, 1, 3).contiguous().permute(1, 2, 0, 3),
                    q.transpose(2, 3).contiguous().transpose(2, 3)):
        assert torch.equal(attend(dev, strided, kc, vc, tables, lens, parents, scale=0.2), want)
    odd = torch.empty(q.numel() + 1, dtype=q.dtype, device=dev)[1:].view(q.shape)
    odd.copy_(q)  # 2 bytes past a 16-byte boundary
    args = (q, kc, vc, tables, lens, parents, None)
    check_attention(attend(dev, odd, *args[1:], scale=0.2), *args, scale=0.2)


def test_large_scores_keep_their_order(dev):
    """Scores of hundreds: the running maximum carries them."""
    q, kc, vc, tables, lens, parents, _ = attend_inputs(2, 10, 8, 2, 128, 16, "bf16", [700, 64],
                                                        "random", None)
    q = q * 8
    out = attend(dev, q, kc, vc, tables, lens, parents)
    check_attention(out, q, kc, vc, tables, lens, parents, None)


@pytest.mark.parametrize("d,block,t", [(128, 16, 20), (64, 4, 33), (80, 16, 3)])
def test_blocks_past_32_bits(dev, d, block, t):
    """Blocks whose values stand 2^31 values and more into the cache: as in a small cache."""
    from grpo_mi355x import kernels

    q, kc, vc, tables, lens, parents, _ = attend_inputs(2, t, 6, 2, d, block, "bf16", [150, 33],
                                                        "random", None, seed=9)
    n, far = kc.shape[0], (1 << 31) // (2 * block * d) + 5
    small = [x[None].to(dev) for x in (kc, vc)]  # [1, blocks, ...]: one layer
    big = []
    for x in small:
        y = torch.empty(1, far + n, 2, block, d, dtype=x.dtype, device=dev)
        y[:, far:] = x
        big.append(y)
    g = torch.Generator().manual_seed(1)
    k = randn(g, 2, t, 2, d, dtype=torch.bfloat16).to(dev)
    cos, sin = (x.to(dev) for x in tables_of_angles(d, 256, torch.float32))
    drafted = torch.randint(0, 2, (2, t), generator=g).to(dev)
    drawn = torch.randint(0, 2, (2, t), generator=g).to(dev)
    q, tables, lens, parents = (x.to(dev) for x in (q, tables, lens, parents))
    out = []
    for (kk, vv), at in ((small, tables), (big, tables + far)):
        r = kernels.paged_rope_append(q, k, k, cos, sin, kk[0], vv[0], at, lens)
        out.append([r, kernels.paged_tree_attention(r, kk[0], vv[0], at, lens, parents),
                    *kernels.accept_draft_tree(drafted, parents, drawn, lens, kk, vv, at)])
        out[-1] += [x[:, -n:] for x in (kk, vv)]
    for x, y in zip(*out):
        assert torch.equal(x, y)
    assert (out[0][3] > 1).any()  # something moved


# ----------------------------------------------------------------- accept --

def accept_inputs(g, b, t, hkv, d, block, layers, vocab=3):
    lens = torch.randint(0, 40, (b,), generator=g).int()
    nb, tables = make_tables(g, b, -(-(40 + t) // block))
    kc, vc = (randn(g, layers, nb, hkv, block, d, dtype=torch.bfloat16) for _ in range(2))
    drafted = torch.randint(0, vocab, (b, t), generator=g)  # few ids: long paths, equal siblings
    sampled = torch.randint(0, vocab, (b, t), generator=g)
    return drafted, rand_parents(g, b, t), sampled, lens, kc, vc, tables


@pytest.mark.parametrize("b,t,hkv,d,block,layers", [
    (1, 1, 1, 16, 16, 1), (5, 8, 2, 128, 16, 3), (9, 64, 4, 128, 16, 2), (7, 61, 2, 64, 32, 28),
    (3, 20, 1, 10, 3, 2), (4, 33, 3, 24, 5, 1)])
@pytest.mark.parametrize("given", [False, True])
def test_accept_draft_tree(dev, b, t, hkv, d, block, layers, given):
    from grpo_mi355x.kernels import accept_draft_tree

    g = torch.Generator().manual_seed(t)
    drafted, parents, sampled, lens, kc, vc, tables = accept_inputs(g, b, t, hkv, d, block, layers)
    counts, kw, okw = None, {}, {}
    if given:
        counts = torch.randint(-1, t + 2, (b,), generator=g).int()
        sampled[0, 0] = -1
        lens[-1] = -1 if b > 1 else lens[-1]
        kw = dict(counts=counts.to(dev), eos_token_id=2, pad_token_id=-5)
        okw = dict(counts=counts.numpy(), eos=2, pad=-5)
    as_int = lambda x: x.view(torch.int16).numpy()  # noqa: E731
    want = ref.accept(drafted.numpy(), parents.numpy(), sampled.numpy(), lens.numpy(), as_int(kc),
                      as_int(vc), tables.numpy(), **okw)
    kcd, vcd = kc.to(dev), vc.to(dev)
    if layers == 1:
        kcd, vcd = kcd[0], vcd[0]
    got = accept_draft_tree(drafted.to(dev), parents.to(dev), sampled.to(dev), lens.to(dev), kcd,
                            vcd, tables.to(dev), **kw)
    for x, y in zip((*got, kcd.view(torch.int16), vcd.view(torch.int16)), want):
        assert np.array_equal(x.cpu().numpy().reshape(y.shape), y)


def test_accept_skips_missing_blocks(dev):
    from grpo_mi355x.kernels import accept_draft_tree

    drafted = torch.tensor([[0, 9, 1, 2]] * 3)
    sampled = torch.tensor([[1, 0, 2, 3]] * 3)
    parents = torch.tensor([[-1, 0, 0, 2]] * 3, dtype=torch.int32)
    tables = torch.tensor([[0, -1], [7, 1], [2, 3]], dtype=torch.int32)
    lens = torch.tensor([2, 1, 5], dtype=torch.int32)  # block size 4
    g = torch.Generator().manual_seed(1)
    kc, vc = (randn(g, 1, 4, 2, 4, 16, dtype=torch.bfloat16) for _ in range(2))
    as_int = lambda x: x.view(torch.int16).numpy()  # noqa: E731
    want = ref.accept(drafted.numpy(), parents.numpy(), sampled.numpy(), lens.numpy(), as_int(kc),
                      as_int(vc), tables.numpy())
    kcd, vcd = kc.to(dev), vc.to(dev)
    got = accept_draft_tree(drafted.to(dev), parents.to(dev), sampled.to(dev), lens.to(dev), kcd,
                            vcd, tables.to(dev))
    assert got[1].tolist() == [3, 3, 3]
    for x, y in zip((*got, kcd.view(torch.int16), vcd.view(torch.int16)), want):
        assert np.array_equal(x.cpu().numpy(), y)


# --------------------------------------------------------------- together --

class Toy:
    """Embedding, layers of rotated attention over a paged cache, tied head; bf16."""

    def __init__(self, dev, layers=2, hq=4, hkv=2, d=64, vocab=97):
        g = torch.Generator().manual_seed(11)
        w = hq * d
        self.hq, self.hkv, self.d, self.layers = hq, hkv, d, layers
        self.emb = randn(g, vocab, w, dtype=torch.bfloat16).to(dev)
        self.qkv = [randn(g, (hq + 2 * hkv) * d, w, std=w ** -0.5, dtype=torch.bfloat16).to(dev)
                    for _ in range(layers)]
        self.cos, self.sin = (x.to(dev) for x in tables_of_angles(d, 512, torch.float32))

    def step(self, tokens, kc, vc, tables, lens, parents, counts, positions):
        """Logits [B, T, V] of a tree of tokens."""
        from grpo_mi355x import kernels

        b, t = tokens.shape
        x = self.emb[tokens]
        for i in range(self.layers):
            y = (x @ self.qkv[i].T).view(b, t, -1, self.d)
            q, k, v = y.split((self.hq, self.hkv, self.hkv), 2)
            q = kernels.paged_rope_append(q, k, v, self.cos, self.sin, kc[i], vc[i], tables, lens,
                                          counts=counts, positions=positions)
            o = kernels.paged_tree_attention(q, kc[i], vc[i], tables, lens, parents, counts=counts)
            x = x + o.view(b, t, -1)
        return x.float() @ self.emb.float().T


def depth_of(parents):
    d = torch.zeros_like(parents)
    for i in range(1, parents.shape[1]):
        d[:, i] = torch.where(parents[:, i] >= 0,
                              d.gather(1, parents[:, i:i + 1].clamp(min=0).long())[:, 0] + 1, 0)
    return d


def test_speculative_decoding_gives_the_models_own_tokens(dev):
    """Trees of drafted tokens, some right, against one token at a time: the tokens are those
    that the model draws itself, and the cache ends up the same, with the same draws."""
    from grpo_mi355x import kernels

    g = torch.Generator().manual_seed(2)
    toy, b, new, block, width = Toy(dev), 3, 24, 16, 8
    nb, tables = make_tables(g, b, width)
    tables = tables.to(dev)
    shape = (toy.layers, nb, toy.hkv, block, toy.d)
    u = torch.rand(b, 64, generator=g, dtype=torch.float64).to(dev)
    prompt = torch.randint(0, 97, (b, 10), generator=g).to(dev)

    def pass_(tokens, kc, vc, lens, parents, counts):
        """The tokens drawn at each node, by the uniform number of its position."""
        depth = (torch.arange(tokens.shape[1], device=dev).int().expand(tokens.shape)
                 if parents is None else depth_of(parents))
        positions = (lens[:, None] + depth).int()
        logits = toy.step(tokens, kc, vc, tables, lens, parents, counts, positions)
        # sharp: a near tie would let a rounding decide
        return kernels.sample_tokens(logits, u.gather(1, positions.long()), temperature=0.05,
                                     top_k=5, top_p=0.95), logits

    def start():
        kc, vc = (torch.zeros(shape, dtype=torch.bfloat16, device=dev) for _ in range(2))
        lens = torch.zeros(b, dtype=torch.int32, device=dev)
        drawn, _ = pass_(prompt, kc, vc, lens, None, None)  # the prompt: one chain
        return kc, vc, lens + 10, drawn[:, -1:]

    kc, vc, lens, pending = start()
    plain = [pending]
    for _ in range(new):
        drawn, _ = pass_(plain[-1], kc, vc, lens, None, None)
        plain.append(drawn)
        lens = lens + 1
    plain = torch.cat(plain, 1)  # [b, new + 1]

    kc2, vc2, lens2, pending = start()
    made, t, steps = [[int(p)] for p in pending[:, 0]], 13, 0
    while min(map(len, made)) <= new:
        steps += 1
        parents = torch.tensor([-1] + [0, 1, 2, 3] + [0, 5, 6, 7] + [0, 9, 9, 11],
                               dtype=torch.int32).expand(b, t).contiguous()
        tokens = torch.randint(0, 97, (b, t), generator=g)
        for i in range(b):
            have = len(made[i])
            tokens[i, 0] = made[i][-1]
            first = (1, 5)[(steps + i) % 2]  # the right tokens, up to some depth
            for j in range((steps + 2 * i) % 5):
                if have + j <= new:
                    tokens[i, first + j] = plain[i, have + j]
        counts = torch.tensor([t if len(m) <= new else 0 for m in made], dtype=torch.int32)
        tokens, parents, counts = tokens.to(dev), parents.to(dev), counts.to(dev)
        drawn, _ = pass_(tokens, kc2, vc2, lens2, parents, counts)
        got, n, _ = kernels.accept_draft_tree(tokens, parents, drawn, lens2, kc2, vc2, tables,
                                              counts=counts)
        lens2 = lens2 + n
        for i in range(b):
            made[i] += got[i, :int(n[i])].tolist()
    assert steps < new  # several tokens were accepted at a time
    for i in range(b):
        assert made[i][:new + 1] == plain[i].tolist()
    # the cache of the accepted tokens
    for i in range(b):
        for s in range(10 + new):
            blk, off = int(tables[i, s // block]), s % block
            for x, y in ((kc, kc2), (vc, vc2)):
                diff = (x[:, blk, :, off].float() - y[:, blk, :, off].float()).abs()
                assert float(diff.max()) < 0.1, (i, s)
                # the first layer's do not depend on attention: the very same
                assert torch.equal(x[0, blk, :, off], y[0, blk, :, off])


# ------------------------------------------------- streams, graphs, other --

def test_a_captured_step_replays(dev):
    from grpo_mi355x import kernels

    q, kc, vc, tables, lens, parents, counts = (
        None if x is None else x.to(dev) for x in
        attend_inputs(3, 16, 12, 2, 128, 16, "bf16", [200, 40, 77], "random", [16, 9, 16]))
    g = torch.Generator().manual_seed(8)
    k = randn(g, 3, 16, 2, 128, dtype=torch.bfloat16).to(dev)
    cos, sin = (x.to(dev) for x in tables_of_angles(128, 512, torch.float32))
    head = randn(g, 1536, 500, std=0.05, dtype=torch.bfloat16).to(dev)
    draws = torch.rand(3, 16, generator=g).to(dev)
    drafted = torch.randint(0, 500, (3, 16), generator=g).to(dev)
    keep = [x.clone() for x in (kc, vc)]

    def step():
        r = kernels.paged_rope_append(q, k, k, cos, sin, kc, vc, tables, lens, counts=counts)
        o = kernels.paged_tree_attention(r, kc, vc, tables, lens, parents, counts=counts)
        drawn = kernels.sample_tokens(o.view(3, 16, -1) @ head, draws, temperature=0.7, top_p=0.9)
        return o, drawn, *kernels.accept_draft_tree(drafted, parents, drawn, lens, kc, vc, tables,
                                                    counts=counts)

    def eager():
        kc.copy_(keep[0])
        vc.copy_(keep[1])
        return [x.clone() for x in (*step(), kc, vc)]

    eager()
    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    with torch.cuda.graph(graph):
        held = step()
    for i in range(4):
        draws.copy_(torch.rand(3, 16, generator=g))
        q.mul_(-1)
        lens.copy_(torch.tensor([200 - 9 * i, 40, 60 + i], dtype=torch.int32))
        want = eager()
        torch.cuda.synchronize()
        kc.copy_(keep[0])
        vc.copy_(keep[1])
        graph.replay()
        torch.cuda.synchronize()
        for x, y in zip(want, (*held, kc, vc)):
            assert torch.equal(x, y)


def test_calls_on_two_streams_at_once(dev):
    """Each call's buffers are its own."""
    from grpo_mi355x import kernels

    sets = []
    for seed in (0, 1):
        args = [None if x is None else x.to(dev) for x in
                attend_inputs(4, 32, 12, 2, 128, 16, "bf16", [900, 400, 30, 2000], "random", None,
                              seed=seed)]
        logits = torch.randn(64, 50257, device=dev)
        draws = torch.rand(64, device=dev)
        sets.append((args, logits, draws, torch.cuda.Stream()))

    def both(s):
        args, logits, draws, _ = s
        return (kernels.paged_tree_attention(*args[:6]),
                kernels.sample_tokens(logits, draws, top_p=0.9))

    want = [both(s) for s in sets]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, s in enumerate(sets):
            with torch.cuda.stream(s[3]):
                got[i].append(both(s))
    torch.cuda.synchronize()
    for w, gs in zip(want, got):
        for x in gs:
            assert torch.equal(x[0], w[0]) and torch.equal(x[1], w[1])


def test_where_another_device_is_current(dev, monkeypatch):
    """Every operator makes its tensors' device the current one for its launch."""
    from grpo_mi355x import kernels

    q, kc, vc, tables, lens, parents, _ = (
        None if x is None else x.to(dev) for x in
        attend_inputs(2, 5, 4, 2, 64, 16, "bf16", [40, 9], "random", None))
    cos, sin = (x.to(dev) for x in tables_of_angles(64, 64, torch.float32))
    ids = torch.ones(2, 5, dtype=torch.int64, device=dev)
    logits, draws = torch.randn(5, 300, device=dev), torch.rand(5, device=dev)

    def go():
        k, v = kc.clone(), vc.clone()
        return [kernels.paged_rope_append(q, q[:, :, :2], q[:, :, 2:], cos, sin, k, v, tables, lens),
                kernels.paged_tree_attention(q, k, v, tables, lens, parents),
                kernels.sample_tokens(logits, draws, top_p=0.9),
                *kernels.accept_draft_tree(ids, parents, ids, lens, k, v, tables), k, v]

    want, entered = go(), []

    class Entered(torch.cuda.device):
        def __init__(self, d):
            entered.append(d)
            super().__init__(d)

    monkeypatch.setattr(torch.cuda, "current_device", lambda: 1)
    monkeypatch.setattr(torch.cuda, "device", Entered)
    got = go()
    monkeypatch.undo()
    assert len(entered) == 4 and all(d.index == 0 for d in entered)
    for x, y in zip(got, want):
        assert torch.equal(x, y)


# --------------------------------------------------------------- refusals --

def test_refusals(dev):
    from grpo_mi355x import kernels

    def inputs():
        q, kc, vc, tables, lens, parents, _ = attend_inputs(2, 4, 4, 2, 32, 16, "bf16", [20, 5],
                                                            "random", None)
        k = q[:, :, :2].contiguous()
        cos, sin = tables_of_angles(32, 64, torch.float32)
        ids = torch.zeros(2, 4, dtype=torch.int64)
        names = dict(q=q, k=k, v=k.clone(), cos=cos, sin=sin, k_cache=kc, v_cache=vc,
                     block_tables=tables, context_lens=lens, parents=parents, counts=lens.clone(),
                     positions=parents.clone(), draft_tokens=ids, sampled=ids.clone())
        return {n: x.to(dev) for n, x in names.items()}

    base = inputs()
    uses = {
        kernels.paged_rope_append: ("q k v cos sin k_cache v_cache block_tables context_lens",
                                    "counts positions"),
        kernels.paged_tree_attention: ("q k_cache v_cache block_tables context_lens parents",
                                       "counts"),
        kernels.accept_draft_tree: ("draft_tokens parents sampled context_lens k_cache v_cache "
                                    "block_tables", "counts"),
    }

    def call(fn, **change):
        args = {**base, **change}
        pos, kw = uses[fn]
        return fn(*(args[n] for n in pos.split()), **{n: args[n] for n in kw.split()})

    for fn, (pos, kw) in uses.items():
        call(fn)
        for n in (pos + " " + kw).split():
            x = base[n]
            bad = [x.cpu(), x[..., None], x.double() if x.is_floating_point() else x.bool()]
            if n not in ("cos", "sin"):
                bad.append(torch.cat([x, x], 0) if "cache" not in n else x[:, :1])
            for y in bad:
                with pytest.raises(ValueError):
                    call(fn, **{n: y})
        for n in ("k_cache", "v_cache"):
            with pytest.raises(ValueError):  # not contiguous
                call(fn, **{n: base[n].transpose(1, 2).contiguous().transpose(1, 2)})
    wide = torch.zeros(2, 65, 4, 32, dtype=torch.bfloat16, device=dev)
    with pytest.raises(ValueError, match="64 nodes"):
        kernels.paged_tree_attention(wide, *(base[n] for n in ("k_cache", "v_cache",
                                                               "block_tables", "context_lens")))
    with pytest.raises(ValueError, match="64 nodes"):
        ids = torch.zeros(2, 65, dtype=torch.int64, device=dev)
        call(kernels.accept_draft_tree, draft_tokens=ids, sampled=ids)
    with pytest.raises(ValueError, match="multiple"):
        call(kernels.paged_tree_attention, q=base["q"][:, :, :3])
    for scale in (float("nan"), float("inf")):
        with pytest.raises(ValueError, match="finite"):
            kernels.paged_tree_attention(*(base[n] for n in uses[kernels.paged_tree_attention][0]
                                           .split()), scale=scale)
    with pytest.raises(ValueError, match="512"):
        c = torch.zeros(2, 1, 16, 514, dtype=torch.bfloat16, device=dev)
        kernels.paged_tree_attention(torch.zeros(2, 4, 1, 514, dtype=c.dtype, device=dev), c, c,
                                     base["block_tables"], base["context_lens"])


def test_no_sequences_and_no_tokens(dev):
    from grpo_mi355x import kernels

    b = attend_inputs(2, 4, 4, 2, 32, 16, "bf16", [20, 5], "random", None)
    q, kc, vc, tables, lens, parents, _ = (None if x is None else x.to(dev) for x in b)
    none = (tables[:0], lens[:0], parents[:0])
    assert kernels.paged_tree_attention(q[:0], kc, vc, *none).shape == (0, 4, 4, 32)
    cos, sin = (x.to(dev) for x in tables_of_angles(32, 8, torch.float32))
    before = kc.clone()
    out = kernels.paged_rope_append(q[:, :0], q[:, :0, :2], q[:, :0, :2], cos, sin, kc, vc, tables,
                                    lens)
    assert out.shape == (2, 0, 4, 32) and torch.equal(kc, before)
    ids = torch.zeros(0, 4, dtype=torch.int64, device=dev)
    tokens, n, path = kernels.accept_draft_tree(ids, none[2], ids, none[1], kc, vc, none[0])
    assert tokens.shape == (0, 4) and n.shape == (0,) and path.shape == (0, 4)
