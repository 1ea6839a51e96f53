"""``sample_tokens`` against the float64 restatement (oracle/draft_tree.py): the same tokens and
the same numbers of kept tokens. Both sides' masses are within 2^-36 of each other (units of
2^-44 over 2^18 tokens at most, relative to a mass of 1 or more), so a draw or a border falls
between them once in many millions of rows; the seeds here are fixed."""

import numpy as np
import pytest
import torch

from oracle import draft_tree as ref

pytestmark = pytest.mark.gpu

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def check(dev, logits, u, **kw):
    """Tokens and kept counts of rows of logits [M, V]; a setting is a number or a list."""
    from grpo_mi355x.kernels import sample_tokens

    m = logits.shape[0]
    given = {k: torch.tensor(v, device=dev, dtype=torch.int32 if k == "top_k" else torch.float32)
             if isinstance(v, list) else v for k, v in kw.items()}
    tokens, kept = sample_tokens(logits.to(dev), u.to(dev), return_kept=True, **given)
    assert tokens.dtype == torch.int64 and kept.dtype == torch.int32
    x = logits.double().numpy()
    for i in range(m):
        # a row's float32 setting is the number that the kernel has
        at = {k: (float(np.float32(v[i])) if k != "top_k" else v[i]) if isinstance(v, list) else v
              for k, v in kw.items()}
        want = ref.sample(x[i], float(u[i]), **at)
        assert (int(tokens[i]), int(kept[i])) == want, (i, at)


def rows(seed, m, v, dtype, std=2.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(m, v, generator=g) * std).to(DTYPES[dtype]), \
        torch.rand(m, generator=g, dtype=torch.float64)


SETTINGS = [dict(), dict(temperature=0.7, top_p=0.9), dict(top_k=50), dict(min_p=0.02),
            dict(temperature=1.3, top_k=200, top_p=0.8, min_p=0.001), dict(top_k=1),
            dict(temperature=0.0), dict(top_p=0.0), dict(top_p=1e-30), dict(min_p=1.0),
            dict(min_p=1.5), dict(temperature=1e-3), dict(temperature=1e6, top_p=0.5),
            dict(top_k=10 ** 9, top_p=0.999999, min_p=1e-9)]


@pytest.mark.parametrize("kw", SETTINGS, ids=str)
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("v", [1, 2, 7, 63, 1000, 4097, 32003])
def test_sizes_and_settings(dev, kw, dtype, v):
    check(dev, *rows(v, 5, v, dtype), **kw)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("std", [0.0, 1e-38, 1e-6, 0.03, 2.0, 9.0])
def test_whole_vocabulary(dev, dtype, std):
    """From one value 151936 times (a tie of all) to a few that stand out."""
    x, u = rows(3, 4, 151936, dtype, std)
    for kw in (dict(temperature=0.7, top_p=0.9), dict(top_k=40), dict(min_p=0.1, top_p=0.99),
               dict()):
        check(dev, x, u, **kw)


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_ties_go_to_the_lowest_index(dev, dtype):
    g = torch.Generator().manual_seed(9)
    x = torch.randint(-3, 4, (6, 30011), generator=g).to(DTYPES[dtype])  # 0 of both signs
    x = torch.where((x == 0) & (torch.rand(x.shape, generator=g) < 0.5), -x, x)
    u = torch.rand(6, generator=g, dtype=torch.float64)
    for kw in (dict(top_k=100), dict(top_p=0.3), dict(top_k=20000, top_p=0.9), dict(min_p=0.5),
               dict(temperature=0.5), dict(temperature=0)):
        check(dev, x, u, **kw)


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_masked_rows(dev, dtype):
    """-inf, NaN, the type's lowest value and +inf."""
    x, u = rows(4, 12, 1003, dtype)
    lowest = torch.finfo(DTYPES[dtype]).min
    x[0] = -float("inf")
    x[1] = float("nan")
    x[2, 5:] = -float("inf")
    x[3, ::2] = float("nan")
    x[4, 1:] = lowest
    x[5] = lowest
    x[6, [3, 500, 700]] = float("inf")
    x[7, :-1] = -float("inf")
    x[8] = -float("inf")
    x[8, 77] = lowest
    x[9] *= 0
    x[10, :500] = -float("inf")
    x[11, 200] = torch.finfo(DTYPES[dtype]).max
    for kw in (dict(), dict(top_k=4), dict(top_p=0.9, temperature=0.6), dict(min_p=0.05),
               dict(temperature=0), dict(top_k=700, top_p=0.99, temperature=2.0)):
        check(dev, x, u, **kw)


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_settings_of_each_row(dev, dtype):
    x, u = rows(6, 9, 5000, dtype)
    check(dev, x, u, temperature=[0.0, 0.5, 1.0, 2.0, -1.0, 0.7, 1.0, 1e-4, 1.0],
          top_k=[0, 5, 5000, -1, 3, 0, 1, 100, 7000],
          top_p=[0.9, 1.0, 0.5, 0.99, 0.1, 0.95, 1.0, 0.9, 0.2],
          min_p=[0.0, 0.1, 0.0, 0.01, 0.5, 0.0, 0.2, 0.0, 1.0])


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("std", [0.3, 1.5])
def test_cuts_one_after_another(dev, dtype, std):
    """Few and many tokens before each cut and before the draw, few and many of one size."""
    x, u = rows(13, 12, 20011, dtype, std)
    x[:, ::7] = x[:, :1]  # 2859 of a value
    k = [3, 50, 900, 1023, 1024, 1025, 1100, 4096, 5000, 0, 700, 12000]
    for p in (0.05, 0.9, 0.999999):
        check(dev, x, u, top_k=k, top_p=p)
        check(dev, x, u, top_k=k, top_p=[p] * 6 + [1.0] * 6, min_p=0.2, temperature=1.1)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("v", [(1 << 18) - 1, 1 << 18, 1 << 20])
def test_the_largest_vocabularies(dev, dtype, v):
    x, u = rows(15, 2, v, dtype)
    for kw in (dict(), dict(temperature=0.8, top_k=5000, top_p=0.9), dict(top_p=0.99, min_p=1e-4)):
        check(dev, x, u, **kw)


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_more_rows_than_compute_units(dev, dtype):
    x, u = rows(14, 300, 1501, dtype)
    check(dev, x, u, temperature=0.9, top_k=300, top_p=0.95)


def test_ends_of_the_unit_interval(dev):
    x, _ = rows(7, 6, 1000, "f32")
    u = torch.tensor([0.0, 1 - 2.0 ** -53, 0.5, 2.0 ** -60, 1 - 2.0 ** -24, 0.25],
                     dtype=torch.float64)
    for kw in (dict(), dict(top_k=3), dict(top_p=0.5)):
        check(dev, x, u, **kw)
    from grpo_mi355x.kernels import sample_tokens

    flat = torch.zeros(6, 777, device=dev)  # the u-th index; draws outside [0, 1) are its ends
    at = torch.tensor([-1.0, 0.0, 0.5, 0.999999, 1.0, float("nan")], device=dev)
    assert sample_tokens(flat, at).tolist() == [0, 0, 388, 776, 776, 0]


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_strided_rows(dev, dtype):
    """Rows at odd addresses, an expanded row, rows inside a larger tensor."""
    from grpo_mi355x.kernels import sample_tokens

    x, u = rows(8, 6, 2999, dtype)
    kw = dict(temperature=0.8, top_p=0.9)
    want = sample_tokens(x.to(dev), u.to(dev), **kw)
    big = torch.full((6, 4001), 50.0, dtype=x.dtype, device=dev)
    for at in (0, 1, 3):
        view = big[:, at:at + 2999]
        view.copy_(x)
        assert torch.equal(sample_tokens(view, u.to(dev), **kw), want)
        big.fill_(50.0)
    turned = x.t().contiguous().t().to(dev)
    assert torch.equal(sample_tokens(turned, u.to(dev), **kw), want)
    one = x[2:3].to(dev).expand(6, 2999)
    assert torch.equal(sample_tokens(one, u.to(dev), **kw),
                       sample_tokens(one.contiguous(), u.to(dev), **kw))
    three = x.to(dev).view(2, 3, 2999)
    assert torch.equal(sample_tokens(three, u.to(dev).view(2, 3), **kw), want.view(2, 3))
    assert int(sample_tokens(x[1].to(dev), u[1].to(dev), **kw)) == int(want[1])


def test_draws_follow_the_distribution(dev):
    """20000 draws of one row against its probabilities: chi-squared over 12 tokens (top_k),
    below its 1 - 1e-6 quantile, 48.0 for 11 degrees of freedom."""
    from grpo_mi355x.kernels import sample_tokens

    x, _ = rows(12, 1, 300, "bf16")
    g = torch.Generator().manual_seed(1)
    n = 20000
    tokens = sample_tokens(x.to(dev).expand(n, 300), torch.rand(n, generator=g).to(dev), top_k=12)
    p, at = torch.topk(x[0].double(), 12)
    p = torch.softmax(p, 0).numpy() * n
    seen = np.array([(tokens == int(i)).sum().item() for i in at])
    assert seen.sum() == n
    assert float(((seen - p) ** 2 / p).sum()) < 48.0


def test_refusals(dev):
    from grpo_mi355x.kernels import sample_tokens

    x, u = rows(1, 4, 100, "bf16")
    x, u = x.to(dev), u.to(dev)
    sample_tokens(x, u)
    for args in ((x.cpu(), u), (x.double(), u), (x.long(), u), (x, u.cpu()), (x, u[:3]),
                 (x, u.bfloat16()), (x, u[:, None]), (x[:, :0], u)):
        with pytest.raises(ValueError):
            sample_tokens(*args)
    nan, inf = float("nan"), float("inf")
    for kw in (dict(temperature=nan), dict(temperature=inf), dict(top_p=nan), dict(min_p=inf),
               dict(top_k=u), dict(top_p=u[:2]), dict(temperature=u.cpu()),
               dict(min_p=u.to(torch.complex64))):
        with pytest.raises(ValueError):
            sample_tokens(x, u, **kw)
    assert sample_tokens(x[:0], u[:0]).shape == (0,)


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_values_of_every_size(dev, dtype):
    """Logits from the smallest to the largest of the type, zeros, and few of a size: the ways
    in which a row is counted, and their borders."""
    g = torch.Generator().manual_seed(21)
    n, dt = 3001, DTYPES[dtype]
    sign = torch.randint(0, 2, (n,), generator=g) * 2.0 - 1
    spread = sign * torch.exp2(torch.rand(n, generator=g) * 250 - 126)
    x = torch.stack([
        spread.clamp(-torch.finfo(dt).max, torch.finfo(dt).max),  # most far from each other
        (sign * 600 * torch.rand(n, generator=g)),  # around 512
        torch.where(torch.rand(n, generator=g) < 0.5, 0.0, sign * torch.rand(n, generator=g)),
        sign * torch.exp2(-29 - 2 * torch.rand(n, generator=g)),  # around 2^-30
        sign * 2.0 ** -35,
        -510 - 4 * torch.rand(n, generator=g),
        510 + 4 * torch.rand(n, generator=g),
        torch.full((n,), -512.0),
        torch.full((n,), 2.0 ** -30),
        -spread.abs().clamp(max=torch.finfo(dt).max)]).to(dt)
    u = torch.rand(len(x), generator=g, dtype=torch.float64)
    for kw in (dict(), dict(temperature=300.0, top_p=0.95), dict(top_k=1000), dict(min_p=0.3),
               dict(temperature=1e5, top_k=2500, top_p=0.99), dict(temperature=0.01)):
        check(dev, x, u, **kw)


@pytest.mark.filterwarnings("ignore:overflow")  # of the oracle's quotients: -inf, as meant
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("temperature", [5e-324, 2.2250738585072014e-308, 5e-307, 1e-300, 1e-250,
                                         1e-45])
def test_temperatures_next_to_zero(dev, dtype, temperature):
    """A draw among the maxima alone, down to the smallest number above 0; the filters count as
    ever."""
    x, u = rows(31, 7, 2003, dtype)
    x[1, 4::500] = x[1].max()  # five maxima
    x[2] = x[2, 0]  # nothing but maxima
    x[3] *= 300  # past 512, below it too
    x[4] = x[4] * 300 - 5000
    x[5, ::3] = -float("inf")
    x[6, 9] = float("inf")
    for kw in (dict(), dict(top_k=50), dict(top_p=0.9), dict(min_p=0.5),
               dict(top_k=900, top_p=0.99, min_p=1e-9)):
        check(dev, x, u, temperature=temperature, **kw)


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_more_rows_than_a_launch_takes(dev, dtype):
    """8 million draws from one expanded row, settings of each row's own: every thousandth as in a
    call of its own."""
    from grpo_mi355x.kernels import sample_tokens

    m, g = (1 << 23) + 1234, torch.Generator().manual_seed(41)
    x = (torch.randn(1, 5, generator=g) * 2).to(DTYPES[dtype]).to(dev).expand(m, 5)
    u = torch.rand(m, generator=g).to(dev)
    kw = dict(temperature=torch.rand(m, generator=g).to(dev) + 0.2,
              top_k=torch.randint(0, 6, (m,), generator=g).int().to(dev),
              top_p=1 - torch.rand(m, generator=g).to(dev) / 2,
              min_p=torch.rand(m, generator=g).to(dev) / 4)
    tokens, kept = sample_tokens(x, u, return_kept=True, **kw)
    some = slice(7, None, 1000)
    want = sample_tokens(x[some], u[some], return_kept=True, **{k: v[some] for k, v in kw.items()})
    assert torch.equal(tokens[some], want[0]) and torch.equal(kept[some], want[1])
    assert len(set(want[0].tolist())) > 2


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("v,apart", [(1 << 13, 1e-6), (50257, 1e-6), (151936, 3e-5),
                                     (1 << 18, 1e-4)])
def test_draws_next_to_a_border(dev, dtype, v, apart):
    """One token and v - 1 equal ones far below it, draws next to the border between two of these,
    by `apart` of one's weight. All of their weights are off by the same 2^-(71 - 2 bits of v) at
    most, and 1.3e-12, which moves a border by v - 1 times as much of one weight."""
    from grpo_mi355x.kernels import sample_tokens

    off = 2.0 ** -(71 - 2 * max(13, v.bit_length())) + 1.3e-12
    assert (v - 1) * off < 0.5 * apart
    x = torch.full((1, v), -13.828125, dtype=DTYPES[dtype])
    x[0, 0] = 0
    w = float(np.exp(np.longdouble(-13.828125)))
    total = 1 + (v - 1) * np.longdouble(w)
    rank = np.arange(1, 200)
    u = np.concatenate([(1 + np.longdouble(w) * (rank + s * np.longdouble(apart))) / total
                        for s in (-1, 1)]).astype(np.float64)
    tokens = sample_tokens(x.to(dev).expand(len(u), v), torch.from_numpy(u).to(dev)).cpu().numpy()
    assert (tokens[:199] == rank).all() and (tokens[199:] == rank + 1).all()


def test_top_p_keeps_the_token_that_passes_it(dev):
    """The shortest head that holds top_p of the mass; the sampled decode's rule cuts its last
    token."""
    from grpo_mi355x.kernels import sample_tokens
    from grpo_mi355x.kernels.paged_kv import _apply_top_p

    p = torch.tensor([0.15, 0.5, 0.05, 0.3], dtype=torch.float64)
    x = p.log().float()[None].to(dev).expand(4, 4)
    # the draws' places among .5, .3, .15
    u = torch.tensor([0.5, 0.55, 0.8, 0.86], dtype=torch.float64, device=dev)
    tokens, kept = sample_tokens(x, u, top_p=0.9, return_kept=True)
    assert kept.tolist() == [3] * 4 and tokens.tolist() == [1, 3, 3, 0]
    assert torch.isfinite(_apply_top_p(x, 0.9)).sum(1).tolist() == [2] * 4


def test_top_k_past_32_bits(dev):
    """More than the vocabulary is no bound, however large; below 0 is none either."""
    from grpo_mi355x.kernels import sample_tokens

    x, u = rows(51, 6, 900, "f32")
    x, u = x.to(dev), u.to(dev)
    want, kept = sample_tokens(x, u, return_kept=True)
    assert kept.tolist() == [900] * 6
    for k in (1 << 31, (1 << 32) + 3, (1 << 63) + 2, (1 << 64) + 3, -(1 << 64) + 3, 1e30):
        got = sample_tokens(x, u, top_k=k, return_kept=True)
        assert torch.equal(got[0], want) and torch.equal(got[1], kept), k
    at = torch.tensor([(1 << 31) + 1, (1 << 32) + 1, (1 << 62) + 1, -(1 << 62) + 1, 0, 901],
                      device=dev)
    got = sample_tokens(x, u, top_k=at, return_kept=True)
    assert torch.equal(got[0], want) and torch.equal(got[1], kept)
    for dtype in (torch.uint8, torch.int8, torch.int16, torch.int32, torch.int64):
        at = torch.arange(1, 7, device=dev).to(dtype)
        assert sample_tokens(x, u, top_k=at, return_kept=True)[1].tolist() == [1, 2, 3, 4, 5, 6]
    for k in (float("inf"), -float("inf"), float("nan")):
        with pytest.raises(ValueError):
            sample_tokens(x, u, top_k=k)


def test_rows_that_overlap(dev):
    from grpo_mi355x.kernels import sample_tokens

    x, u = rows(61, 1, 1500, "bf16")
    some = x[0].to(dev).unfold(0, 1000, 100)  # row m begins at 100 m
    u = torch.rand(len(some), generator=torch.Generator().manual_seed(2)).to(dev)
    for kw in (dict(), dict(top_k=30, temperature=0.8), dict(top_p=0.9)):
        assert torch.equal(sample_tokens(some, u, **kw), sample_tokens(some.contiguous(), u, **kw))
    one = torch.randn(9, 4).to(dev).t()  # tokens 4 apart, a row of one token
    assert sample_tokens(one[:, :1], u[:4]).tolist() == [0] * 4
