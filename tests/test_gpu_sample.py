"""lnsb_sample against the sampler's definition in 64 bits: the random number
is put in the middle of a kept token's share, so the token is certain."""
import math

import pytest
import torch

import serve_ref as ref

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def ks():
    import lnsb200
    return lnsb200.KernelSet(16, "base")


def _run(ks, x, u, t=None, k=None, p=None, m=None):
    n = x.shape[0]
    f = lambda v: None if v is None else torch.tensor(v, dtype=torch.float32, device="cuda")  # noqa: E731
    token = torch.full((n,), -9, dtype=torch.int32, device="cuda")
    prob = torch.full((n,), -9.0, device="cuda")
    ks.sample(x, f(u), token, prob, f(t), None if k is None else torch.tensor(k, dtype=torch.int32, device="cuda"), f(p), f(m))
    return token.cpu().tolist(), prob.cpu().double().tolist()


def _f32(v):
    return torch.tensor(v, dtype=torch.float32).double().item()


def _safe_p(x, t, k, p):
    """top_p moved off the places where 32-bit weights could disagree about the cut"""
    kept, w = ref.kept_tokens(x, t, k, 1.0, 0.0)
    run = w.cumsum(0) / w.sum()
    while float((run - _f32(p)).abs().min()) < 2e-6:
        p += 1e-5
    return p


def _case(x, t, k, p, m, g):
    """(u, token, prob) for a token of one row drawn by its weight"""
    kept, w = ref.kept_tokens(x, _f32(t), k, _f32(p), _f32(m))
    ok = w / w.sum() > 2e-6                                # wide enough to be hit with certainty
    i = torch.multinomial(w * ok, 1, generator=g).item()
    by = torch.argsort(kept)
    run = w[by].cumsum(0)
    j = (by == i).nonzero().item()
    return ((run[j] - w[i] / 2) / run[-1]).item(), kept[i].item(), (w[i] / run[-1]).item()


@pytest.mark.parametrize("type", sorted(TYPES))
@pytest.mark.parametrize("vocab", (1, 2, 31, 1000, 4097, 49152, 131071))
@pytest.mark.parametrize("spread", (0.05, 1.0, 4.0))
def test_sample(ks, type, vocab, spread):
    g = torch.Generator().manual_seed(int(vocab + 1000 * spread))
    pars = [(1.0, 0, 1.0, 0.0), (0.7, 40, 1.0, 0.0), (1.0, 0, 0.9, 0.0), (1.3, 0, 1.0, 0.05), (0.8, 40, 0.95, 0.05),
            (1.0, 1, 0.5, 0.0), (2.0, 5000, 0.3, 0.0), (0.25, 7, 0.999, 1e-6), (1.0, vocab, 1.0, 1.0), (1.0, 3, 0.0, 0.0)]
    x = (torch.randn((len(pars), vocab), generator=g) * spread).to(TYPES[type])
    rows = []
    for r, (t, k, p, m) in enumerate(pars):
        p = _safe_p(x[r], _f32(t), k, p) if 0 < p < 1 else p
        rows.append((t, k, p, m) + _case(x[r], t, k, p, m, g))
    t, k, p, m, u, want, prob = zip(*rows)
    got, gp = _run(ks, x.cuda(), u, t, k, p, m)
    assert got == list(want)
    # the kept sum in 32-bit weights: 2^-22 a weight, and the 2^-40 that each drops
    assert all(abs(a - b) <= (2.0 ** -21 + vocab * 2.0 ** -40) * b + 1e-12 for a, b in zip(gp, prob))


@pytest.mark.parametrize("type", sorted(TYPES))
@pytest.mark.parametrize("vocab,rows", ((300001, 2), (1 << 20, 1), (20000, 160)))
def test_long_rows_and_many(ks, type, vocab, rows):
    """the largest vocabularies, more rows than SMs, and cuts deep in the row"""
    g = torch.Generator().manual_seed(vocab)
    pars = [(1.0, vocab // 3, 1.0, 0.0), (0.9, vocab // 2, 0.9, 0.0), (1.0, 0, 0.97, 0.0), (1.5, 0, 0.5, 1e-4),
            (0.3, 0, 0.9, 0.0), (1.0, 4000, 0.99, 0.0), (1.0, 3000, 1.0, 0.01), (4.0, 0, 1.0, 0.6)]
    x = (torch.randn((len(pars), vocab), generator=g) * 2.0).to(TYPES[type])
    want = []
    for r, (t, k, p, m) in enumerate(pars):
        p = _safe_p(x[r], _f32(t), k, p) if 0 < p < 1 else p
        want.append((t, k, p, m) + _case(x[r], t, k, p, m, g))
    x = x.cuda()
    for r0 in range(0, len(pars), rows):
        part = [r % len(pars) for r in range(r0, r0 + rows)]
        t, k, p, m, u, token, prob = zip(*(want[r] for r in part))
        got, gp = _run(ks, x[part], u, t, k, p, m)
        assert got == list(token)
        assert all(abs(a - b) <= (2.0 ** -21 + vocab * 2.0 ** -40) * b + 1e-12 for a, b in zip(gp, prob))


@pytest.mark.parametrize("type", sorted(TYPES))
@pytest.mark.parametrize("rows", (1, 3, 200))
def test_equal_logits_go_by_index(ks, type, rows):
    """every cut falls inside a run of equal logits: the lowest indices stay"""
    vocab = 777
    x = torch.zeros((rows, vocab), dtype=TYPES[type], device="cuda")
    got, prob = _run(ks, x, [0.999] * rows, k=[10] * rows)
    assert got == [9] * rows and prob == pytest.approx([0.1] * rows, rel=1e-6)
    got, _ = _run(ks, x, [0.999] * rows, p=[0.5] * rows)
    assert got == [388] * rows                             # 388 < 0.5 * 777 <= 389: 389 tokens stay
    x[:, 100] = 1.0
    x[:, 300:] = -1.0
    got, _ = _run(ks, x, [0.9999] * rows, k=[50] * rows)
    assert got == [100] * rows                             # 0 .. 48 and 100: the last in order of index
    got, _ = _run(ks, x, [0.0] * rows, k=[50] * rows)
    assert got == [0] * rows


def test_ends_of_the_random_number(ks):
    x = torch.log(torch.tensor([[1.0, 2.0, 4.0, 1.0]])).cuda()
    for u, want in ((0.0, 0), (0.124, 0), (0.126, 1), (0.374, 1), (0.376, 2), (0.874, 2), (0.876, 3), (1 - 2.0 ** -24, 3),
                    (1.0, 3), (-1.0, 0), (float("nan"), 0)):
        assert _run(ks, x, [u])[0] == [want]


def test_greedy(ks):
    g = torch.Generator().manual_seed(5)
    x = torch.randn((6, 5000), generator=g).to(torch.bfloat16)
    x[1, 17] = x[1, 4000] = 9.0
    x[2, :] = -3.0
    got, prob = _run(ks, x.cuda(), [0.7] * 6, t=[0.0, -1.0, 0.0, float("nan"), 0.0, 0.0], k=[3] * 6, p=[0.1] * 6, m=[0.5] * 6)
    want = [int((row.float() == row.float().max()).nonzero()[0]) for row in x]
    assert got == want and prob == [1.0] * 6 and want[1] == 17 and want[2] == 0


def test_masked_and_broken_logits(ks):
    """-inf and NaN are never drawn, a row of nothing else gives -1, +inf takes it all"""
    inf, nan = math.inf, math.nan
    x = torch.full((6, 1001), -inf)
    x[0, 500], x[0, 700] = 2.0, 2.0
    x[1, :] = nan
    x[1, 3] = -1e30
    x[3, 10], x[3, 20], x[3, 30] = inf, 5.0, inf
    x[4, 5:9] = torch.tensor([nan, 1.0, nan, 1.0])
    x[5, :] = nan
    got, prob = _run(ks, x.cuda(), [0.75] * 6)
    assert got == [700, 3, -1, 30, 8, -1]
    assert prob == [0.5, 1.0, 0.0, 0.5, 0.5, 0.0]
    got, _ = _run(ks, x.cuda(), [0.2] * 6, t=[0.0] * 6)
    assert got == [500, 3, -1, 10, 6, -1]
    got, _ = _run(ks, x.cuda(), [0.2] * 6, k=[1] * 6, p=[0.5] * 6, m=[0.3] * 6)
    assert got == [500, 3, -1, 10, 6, -1]


def test_lowest_value_of_the_type(ks):
    """masks of the type's lowest value: the kept token is certain, the rest weigh nothing"""
    for type in TYPES.values():
        x = torch.full((2, 300), torch.finfo(type).min, dtype=type)
        x[0, 77] = 0.0
        got, prob = _run(ks, x.cuda(), [0.99, 0.5])
        assert got[0] == 77 and prob[0] == 1.0
        assert got[1] == 150 and prob[1] == pytest.approx(1 / 300, rel=1e-6)


def test_extreme_temperatures(ks):
    x = torch.tensor([[1.0, 3.0, 2.0, 3.0]] * 4).cuda()
    got, prob = _run(ks, x, [0.4, 0.6, 0.1, 0.9], t=[1e-30, 1e-42, 1e30, math.inf])
    assert got == [1, 3, 0, 3] and prob == pytest.approx([0.5, 0.5, 0.25, 0.25])


def test_row_stride_and_stream(ks):
    g = torch.Generator().manual_seed(6)
    wide = torch.randn((5, 3001), generator=g).cuda()
    x = wide[:, 1:2998]
    u = [0.1, 0.3, 0.5, 0.7, 0.9]
    plain = _run(ks, x.contiguous(), u, k=[30] * 5)
    assert _run(ks, x, u, k=[30] * 5) == plain
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        assert _run(ks, x, u, k=[30] * 5) == plain


def test_frequencies(ks):
    """numbers spread evenly over [0, 1) draw each token in proportion to its weight"""
    n = 4096
    w = torch.tensor([1.0, 3.0, 0.5, 2.0, 1.5])
    x = torch.log(w).repeat(n, 1).cuda()
    got, _ = _run(ks, x, [(i + 0.5) / n for i in range(n)])
    for i in range(5):
        assert abs(got.count(i) - n * float(w[i] / w.sum())) <= 1.0
