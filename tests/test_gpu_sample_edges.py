"""lnsb_sample where distances between logits, over the temperature, leave the ordinary range."""
import pytest
import torch

import serve_ref as ref

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
# top_k, top_p, min_p: each alone, in pairs, all, none
FILTERS = [(3, 1.0, 0.0), (0, 0.9, 0.0), (0, 1.0, 0.05), (3, 0.9, 0.0), (3, 1.0, 0.05), (0, 0.9, 0.05), (3, 0.9, 0.05),
           (0, 1.0, 0.0), (5000, 0.9, 0.0), (0, 0.9999, 0.0), (0, 1.0, 1e-6)]


@pytest.fixture(scope="module")
def ks():
    import lnsb200
    return lnsb200.KernelSet(16, "base")


def _run(ks, x, u, t, k, p, m):
    f = lambda v: torch.tensor(v, dtype=torch.float32, device="cuda")  # noqa: E731
    token = torch.full((x.shape[0],), -9, dtype=torch.int32, device="cuda")
    prob = torch.full((x.shape[0],), -9.0, device="cuda")
    ks.sample(x, f(u), token, prob, f(t), torch.tensor(k, dtype=torch.int32, device="cuda"), f(p), f(m))
    return token.cpu().tolist(), prob.cpu().double().tolist()


def _f32(v):
    return torch.tensor(v, dtype=torch.float32).double().item()


@pytest.mark.parametrize("type", sorted(TYPES))
@pytest.mark.parametrize("vocab,rows", ((4, 1), (5000, 2), (131071, 1), (3000, 160), (200001, 3)))
def test_tiny_temperatures(ks, type, vocab, rows):
    """only the largest logits weigh anything, whatever filter is on; two equal ones share"""
    g = torch.Generator().manual_seed(vocab)
    x = torch.randn((rows, vocab), generator=g).to(TYPES[type])
    first, second = vocab // 3, vocab - 1
    alone = x.clone()
    alone[:, first] = 9.0
    x[:, first] = x[:, second] = 9.0
    for t in (1e-36, 8e-37, 1e-37, float(torch.finfo(torch.float32).tiny), 1e-42):
        for k, p, m in FILTERS:
            par = [[v] * rows for v in (t, k, p, m)]
            assert _run(ks, alone.cuda(), [0.7] * rows, *par) == ([first] * rows, [1.0] * rows), (t, k, p, m)
            for u, want in ((0.3, first), (0.7, second)):
                assert _run(ks, x.cuda(), [u] * rows, *par) == ([want] * rows, [0.5] * rows), (t, k, p, m)


@pytest.mark.parametrize("type", ("f32", "bf16"))
@pytest.mark.parametrize("vocab,rows", ((1000, 1), (1000, 200), (9000, 1), (9000, 150)))
def test_logits_that_hardly_differ(ks, type, vocab, rows):
    """one logit above many equal ones by so little that every weight is 1: it comes first, then the lowest indices"""
    x = torch.zeros((rows, vocab), dtype=TYPES[type])
    at = vocab // 2 + 7
    for step in (1e-36, 1e-38):
        x[:, at] = step
        half = vocab // 2
        got = _run(ks, x.cuda(), [0.9999] * rows, [1.0] * rows, [0] * rows, [0.5] * rows, [0.0] * rows)
        assert got[0] == [at] * rows                       # at, and 0 .. half - 2
        assert got[1] == pytest.approx([1 / half] * rows, rel=1e-6)
        got = _run(ks, x.cuda(), [(half - 1.5) / half] * rows, [1.0] * rows, [0] * rows, [0.5] * rows, [0.0] * rows)
        assert got[0] == [half - 2] * rows
        got = _run(ks, x.cuda(), [0.5] * rows, [1.0] * rows, [2] * rows, [1.0] * rows, [0.0] * rows)
        assert got[0] == [at] * rows and got[1] == [0.5] * rows
        got = _run(ks, x.cuda(), [0.5] * rows, [1.0] * rows, [0] * rows, [1.0] * rows, [0.5] * rows)
        assert got[0] == [half] * rows


@pytest.mark.parametrize("vocab,rows", ((700, 1), (20000, 2), (20000, 150)))
@pytest.mark.parametrize("t", (3e-37, 2e-38, 5e-36))
def test_distances_of_the_temperatures_size(ks, vocab, rows, t):
    """logits and temperature both tiny: weights from 1 down to nothing, as at ordinary sizes"""
    g = torch.Generator().manual_seed(vocab)
    z = 40.0 * torch.rand((rows, vocab), generator=g) ** 2
    x = (-z * t).float()
    for k, p, m in ((40, 1.0, 0.0), (0, 0.9, 0.0), (0, 1.0, 0.05), (40, 0.95, 0.05), (vocab // 2, 1.0, 0.0), (0, 0.999, 0.0)):
        u, want, prob, ps = [], [], [], []
        for r in range(min(rows, 2)):
            # the cut by mass moved off the places where 32-bit weights could disagree: each weight is off by
            # 2 x 40 x 2^-24 (1 / t, the product) + 2^-22 (exp) < 2^-17 of itself, a prefix's share of all by twice
            # that of what lies behind it
            q = p
            if p < 1:
                kept, w = ref.kept_tokens(x[r], _f32(t), k, 1.0, 0.0)
                run = w.cumsum(0) / w.sum()
                while float((run - _f32(q)).abs().min()) < 2.0 ** -16 * (1 - q):
                    q += 0.01 * (1 - p)
                    assert q < 1
            _, w = ref.kept_tokens(x[r], _f32(t), k, _f32(q), 0.0)
            assert m == 0 or float((w - m).abs().min()) > 2.0 ** -17 * m
            kept, w = ref.kept_tokens(x[r], _f32(t), k, _f32(q), _f32(m))
            i = torch.multinomial(w * (w / w.sum() > 2.0 ** -15), 1, generator=g).item()
            by = torch.argsort(kept)
            run, j = w[by].cumsum(0), (by == i).nonzero().item()
            u.append(((run[j] - w[i] / 2) / run[-1]).item())
            want.append(kept[i].item())
            prob.append((w[i] / run[-1]).item())
            ps.append(q)
        if rows > 2:                                       # the same two rows again and again: more rows than SMs
            x2 = x[:2].repeat(rows // 2, 1)
            u, want, prob, ps = u * (rows // 2), want * (rows // 2), prob * (rows // 2), ps * (rows // 2)
        else:
            x2 = x
        n = len(u)
        got, gp = _run(ks, x2.cuda(), u, [t] * n, [k] * n, ps, [m] * n)
        assert got == want, (k, p, m)
        assert all(abs(a - b) <= 2.0 ** -16 * b for a, b in zip(gp, prob))
