"""lnsb_paged_attn at the ends of its arguments' ranges, against plain 64-bit forms."""
import pytest
import torch

import serve_ref as ref

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


@pytest.fixture(scope="module")
def ks():
    import lnsb200
    return lnsb200.KernelSet(16, "base")


@pytest.fixture(scope="module")
def work(ks):
    return ks.paged_attn_work()


def _q(P, heads, dim, dtype, seed, scale=1.5):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn((P.tokens, heads, dim), generator=g) * scale).to(dtype).cuda()


def _attn(ks, work, P, q, window=0, max_q=None, max_kv=None, scale=None):
    dst = torch.full_like(q, float("nan"))
    ks.paged_attn(q, P.k, P.v, P.table, P.q_start, P.kv_len, P.max_q if max_q is None else max_q,
                  P.max_kv if max_kv is None else max_kv, dst, work, window=window, scale=scale)
    return dst


def _check(P, q, got, window=0, scale=None):
    want, mag = ref.attention(P, q, q.shape[2] ** -0.5 if scale is None else scale, window)
    v_max = max([float(P.rows(P.v, s).abs().max()) for s in range(len(P.kv)) if P.kv[s]] + [0.0])
    bound = ref.attention_bound(q.dtype, want, mag, P.max_kv, v_max)
    bad = ~((got.double() - want).abs() <= bound)
    assert not bad.any(), "%d of %d values off, worst %g of the bound" % (
        int(bad.sum()), bad.numel(), float(((got.double() - want).abs() / bound).max()))


# ------------------------------------------------------------------- windows

@pytest.mark.parametrize("heads,kv_heads,dim", [(4, 2, 64), (4, 2, 128), (4, 2, 32)])
@pytest.mark.parametrize("lengths", [([200], [150]), ([200, 1, 40], [150, 70, 10]), ([300, 30], [1, 7]), ([1, 2], [90, 1])], ids=str)
def test_window_that_hides_nothing(ks, work, heads, kv_heads, dim, lengths):
    """a window of the longest sequence and any longer one, up to the type's end, gives the bits of none; also where a
    sequence has more new tokens than rows"""
    P = ref.Paged(*lengths, kv_heads, dim, 16, BF16, seed=40)
    q = _q(P, heads, dim, BF16, 41)
    plain = _attn(ks, work, P, q)
    _check(P, q, plain)
    for window in (P.max_kv, P.max_kv + 1, 1000, 2 ** 31 - 1, 2 ** 31, 2 ** 32, 2 ** 32 + 5, 2 ** 63 - 1):
        assert torch.equal(_attn(ks, work, P, q, window), plain), window
    assert ks.paged_errors() == (0, 0)


@pytest.mark.parametrize("heads,kv_heads,dim", [(4, 2, 64), (4, 2, 128), (4, 2, 32)])
@pytest.mark.parametrize("window", (1, 2, 33, 100, 149))
def test_window_with_rows_that_see_nothing(ks, work, heads, kv_heads, dim, window):
    """windows over sequences with more new tokens than rows"""
    P = ref.Paged([200, 1, 40, 3], [150, 70, 10, 0], kv_heads, dim, 16, BF16, seed=42)
    q = _q(P, heads, dim, BF16, 43)
    got = _attn(ks, work, P, q, window)
    _check(P, q, got, window)
    assert (got[:50] == 0).all() and (got[201:231] == 0).all() and (got[241:] == 0).all()
    assert ks.paged_errors() == (0, 0)


# -------------------------------------------------------------- large scores

@pytest.mark.parametrize("dtype,size", [(F16, 20000.0), (BF16, 1e6), (BF16, 1e15)])
@pytest.mark.parametrize("dim", (64, 128, 32))
@pytest.mark.parametrize("q", (1, 40, 300))
def test_scores_of_any_size(ks, work, dtype, size, dim, q):
    """scores far past 2^24, all apart by more than their rounding: each token takes the largest key it sees, whole;
    rising, falling, and all of them far below zero"""
    n, page = 700, 32
    for lo, hi in ((-1.0, 1.0), (1.0, -1.0), (-1.0, -0.25), (-0.25, -1.0)):
        P = ref.Paged([q], [n], 2, dim, page, dtype, seed=44)
        # 700 steps of the type's own grid would not fit bfloat16's: 100 levels, and within one the keys are equal
        level = torch.arange(n) // 7
        ramp = (lo + (hi - lo) * level / 99.0) * size
        for i in range(n):
            P.k[P.host_table[0, i // page], i % page] = ramp[i].to(dtype).cuda()
        qq = torch.full((q, 4, dim), size, dtype=dtype, device="cuda")
        got = _attn(ks, work, P, qq)
        _check(P, qq, got)
    assert ks.paged_errors() == (0, 0)


@pytest.mark.parametrize("dim", (64, 128, 32))
@pytest.mark.parametrize("q", (1, 300))
def test_large_scores_that_rise_slowly(ks, work, dim, q):
    """scores near 1.5 2^27, where floats are 16 apart, rise by 16 (base 2) every 128 keys: the weights stay below
    half's largest value"""
    n, page = 1500, 32
    P = ref.Paged([q], [n], 2, dim, page, F16, seed=45)
    k = torch.zeros((n, 2, dim))
    k[:, :, 0] = 12288.0
    k[:, :, 1] = (torch.arange(n) // 128).float()[:, None]
    for i in range(n):
        P.k[P.host_table[0, i // page], i % page] = k[i].half().cuda()
    qq = torch.zeros((q, 4, dim), dtype=F16, device="cuda")
    qq[..., 0], qq[..., 1] = 16384.0, 16.0
    scale = 0.6931471805599453                             # ln 2: the products are the scores to base 2
    _check(P, qq, _attn(ks, work, P, qq, scale=scale), scale=scale)


# -------------------------------------------------------- what is divided by

@pytest.mark.parametrize("dtype,value", [(F16, 1.9990234375), (BF16, 1.9921875)])
@pytest.mark.parametrize("heads,kv_heads,dim", [(4, 2, 64), (4, 2, 128), (4, 2, 32)])
@pytest.mark.parametrize("q", (1, 40, 300))
@pytest.mark.parametrize("spread", (0.3, 1.5, 6.0))
def test_equal_values_come_back(ks, work, dtype, value, heads, kv_heads, dim, q, spread):
    """where all values are one number, every output is that number: the weights as they meet the values are what the
    output is divided by, in chunks as for single tokens"""
    P = ref.Paged([q, 1], [900, 333], kv_heads, dim, 16, dtype, seed=46)
    for s in range(2):
        for i in range(P.kv[s]):
            P.v[P.host_table[s, i // 16], i % 16] = value
    qq = _q(P, heads, dim, dtype, 47, spread)
    assert (_attn(ks, work, P, qq) == value).all()


@pytest.mark.parametrize("dtype,value,over", [(F16, 1.9990234375, 0.00064), (BF16, 1.9921875, 0.00505)])
@pytest.mark.parametrize("dim", (64, 128, 32))
@pytest.mark.parametrize("q", (1, 40))
def test_one_heavy_weight_between_two_numbers(ks, work, dtype, value, over, dim, q):
    """the same where nearly all weight is one key's, which is 2^7 and almost half a place against the maximum of the
    tiles before it; enough sequences for several tiles to a CTA"""
    n, page, seqs = 1024, 128, 64
    P = ref.Paged([q] * seqs, [n] * seqs, 2, dim, page, dtype, seed=48)
    P.k[:], P.v[:] = 0.0, value
    P.k[..., 0] = -60.0
    P.k[P.host_table[:, 0].long(), 0] = 0.0
    P.k[P.host_table[:, 1].long(), 5, :, 0], P.k[P.host_table[:, 1].long(), 5, :, 1] = 7.0, over
    qq = torch.zeros((q * seqs, 4, dim), dtype=dtype, device="cuda")
    qq[..., :2] = 1.0
    assert (_attn(ks, work, P, qq, scale=0.6931471805599453) == value).all()   # ln 2: base 2


# ------------------------------------------------------------- light weights

@pytest.mark.parametrize("dim", (64, 128, 32))
@pytest.mark.parametrize("q", (1, 40, 300))
@pytest.mark.parametrize("lo,hi", [(26.0, 26.0), (18.0, 30.0)])
def test_many_light_weights_in_half(ks, work, dim, q, lo, hi):
    """one key outweighs each of 20,000 others by 2^18 to 2^30; its value is 0, theirs is 1.  Half's last place below its
    normal numbers is 2^-24, and the largest weight is 2^7 at least: a weight is off by 2^-32 of the largest, or by u.
    64 sequences share the pages, so that a CTA takes many tiles"""
    n, page, seqs = 20000, 1024, 64
    P = ref.Paged([q], [n], 1, dim, page, F16, seed=49, junk=0.0)
    g = torch.Generator().manual_seed(50)
    P.k[:], P.v[:] = 0.0, 1.0
    P.k[..., 0, 0] = -(lo + (hi - lo) * torch.rand(P.k.shape[:2], generator=g)).half().cuda()
    first = P.host_table[0, 0].item()
    P.k[first, 0], P.v[first, 0] = 0.0, 0.0
    qq = torch.zeros((q, 2, dim), dtype=F16, device="cuda")
    qq[..., 0] = 1.0
    scale = 0.6931471805599453                             # ln 2: base 2
    want, mag = ref.attention(P, qq, scale)
    u = ref.UNIT[F16]
    bound = (2 * u + 2.0 ** -12) * mag * 1.01 + u * want.abs() * 1.01 + n * 2.0 ** -32 + 2.0 ** -24
    P.table, P.kv_len = P.table.repeat(seqs, 1), P.kv_len.repeat(seqs)
    P.q_start = torch.arange(seqs + 1, dtype=torch.int32, device="cuda") * q
    got = _attn(ks, work, P, qq.repeat(seqs, 1, 1), scale=scale).view(seqs, q, 2, dim).double()
    assert float(want.min()) > 1e-4
    assert ((got - want).abs() <= bound).all(), float(((got - want).abs() / bound).max())


# ------------------------------------------------------------ many sequences

@pytest.mark.parametrize("seqs", (129, 300, 700))
@pytest.mark.parametrize("kind", ("tokens", "chunks", "mixed"))
@pytest.mark.parametrize("heads,kv_heads,dim", [(2, 1, 64), (4, 2, 128), (2, 2, 16)])
@pytest.mark.parametrize("window", (0, 40))
def test_many_sequences(ks, work, seqs, kind, heads, kv_heads, dim, window):
    """more sequences than one thread or lane looks at, idle ones first, last and in long runs"""
    g = torch.Generator().manual_seed(seqs)
    kv = torch.randint(0, 150, (seqs,), generator=g).tolist()
    most = {"tokens": 1, "chunks": 60, "mixed": 60}[kind]
    q = torch.randint(0 if kind == "tokens" else 2, most + 1, (seqs,), generator=g).tolist()
    if kind == "mixed":
        q = [n if i % 3 == 0 else n % 3 for i, n in enumerate(q)]
    for lo, hi in ((0, 5), (40, 75), (seqs - 9, seqs)):
        q[lo:hi] = [0] * (hi - lo)
    P = ref.Paged(q, kv, kv_heads, dim, 16, BF16, seed=51)
    x = _q(P, heads, dim, BF16, 52)
    _check(P, x, _attn(ks, work, P, x, window), window)
    assert ks.paged_errors() == (0, 0)


def test_one_sequence_among_thousands_of_idle_ones(ks, work):
    for seqs in (5000, 65536):
        for at in (0, seqs // 2 + 3, seqs - 1):
            q, kv = [0] * seqs, [0] * seqs
            q[at], kv[at] = 50, 333
            P = ref.Paged([50], [333], 2, 64, 16, BF16, seed=53)
            start = torch.zeros(seqs + 1, dtype=torch.int32, device="cuda")
            start[at + 1:] = 50
            lens, table = torch.zeros(seqs, dtype=torch.int32, device="cuda"), P.table.new_full((seqs, P.table.shape[1]), -1)
            lens[at], table[at] = 333, P.table[0]
            x = _q(P, 4, 64, BF16, 54)
            dst = torch.full_like(x, float("nan"))
            ks.paged_attn(x, P.k, P.v, table, start, lens, 50, 333, dst, work)
            _check(P, x, dst)


# ----------------------------------------------------------------- the bounds

@pytest.mark.parametrize("heads,kv_heads,dim", [(4, 2, 64), (8, 2, 128), (4, 2, 32)])
@pytest.mark.parametrize("lengths", [([1, 1, 0], [70, 500, 3]), ([40, 1, 130], [40, 700, 300]), ([90], [400])], ids=str)
def test_any_bound_on_the_new_tokens(ks, work, heads, kv_heads, dim, lengths):
    """max_q chooses the kernels and limits nothing, below the real one too"""
    P = ref.Paged(*lengths, kv_heads, dim, 16, BF16, seed=55)
    x = _q(P, heads, dim, BF16, 56)
    for max_q in (0, 1, 16, 1000, 2 ** 31 - 1, 2 ** 62, 2 ** 63 - 1):
        _check(P, x, _attn(ks, work, P, x, max_q=max_q))
    for max_kv in (P.max_kv + 1, P.table.shape[1] * 16):
        _check(P, x, _attn(ks, work, P, x, max_kv=max_kv))
    assert ks.paged_errors() == (0, 0)


@pytest.mark.parametrize("dim", (64, 32))
def test_a_bound_on_the_rows_below_the_real_one(ks, work, dim):
    """kv_len above max_kv is taken as max_kv"""
    P = ref.Paged([40, 1], [300, 90], 2, dim, 16, BF16, seed=57)
    x = _q(P, 4, dim, BF16, 58)
    got = _attn(ks, work, P, x, max_kv=200)
    P.kv = [200, 90]
    _check(P, x, got)
