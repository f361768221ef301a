"""The paged cache on the GPU: lnsb_paged_append and lnsb_paged_attn against
plain 64-bit forms, with junk (NaN) wherever a sequence owns nothing."""
import numpy as np
import pytest
import torch

import serve_ref as ref

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


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


def _attn(ks, work, P, q, window=0, scale=None, **kw):
    dst = torch.full_like(q, float("nan"))
    ks.paged_attn(q, P.k, P.v, P.table, P.q_start, P.kv_len, P.max_q, P.max_kv, dst, work, scale=scale, window=window, **kw)
    return dst


def _check(ks, work, P, q, window=0, scale=None):
    got = _attn(ks, work, P, q, window, scale).double()
    want, mag = ref.attention(P, q, q.shape[2] ** -0.5 if scale is None else scale, window)
    v_max = max([float(P.rows(P.v, s).abs().max()) for s in range(len(P.kv)) if P.kv[s]] + [0.0])
    bound = ref.attention_bound(q.dtype, want, mag, P.max_kv, v_max)
    bad = ~((got - want).abs() <= bound)
    assert not bad.any(), "%d of %d values off, worst %g of the bound" % (
        int(bad.sum()), bad.numel(), float(((got - want).abs() / bound).max()))
    assert ks.paged_errors() == (0, 0)
    return got


# one token, ragged; page edges inside a tile, one row, an idle slot, an empty cache
RAGGED = [1, 200, 64, 63, 65, 16, 15, 1000, 129, 7]


@pytest.mark.parametrize("dtype", (F16, BF16))
@pytest.mark.parametrize("heads,kv_heads,dim", [(9, 3, 64), (8, 2, 128), (4, 4, 16), (6, 2, 32), (4, 2, 256), (16, 1, 64),
                                                (5, 5, 128), (40, 2, 128)])
@pytest.mark.parametrize("page", (8, 64))
def test_one_token(ks, work, dtype, heads, kv_heads, dim, page):
    P = ref.Paged([1] * len(RAGGED), RAGGED, kv_heads, dim, page, dtype, seed=1)
    _check(ks, work, P, _q(P, heads, dim, dtype, 2))


@pytest.mark.parametrize("dtype", (F16, BF16))
@pytest.mark.parametrize("page", (8, 16, 32, 128, 256, 1024))
@pytest.mark.parametrize("window", (0, 1, 37, 300))
def test_chunks(ks, work, dtype, page, window):
    """prompt chunks beside single tokens and idle slots; a chunk longer than the cache has rows before it"""
    q_len = [5, 0, 130, 1, 64, 33, 1, 257]
    kv_len = [5, 70, 300, 900, 64, 500, 1, 300]
    P = ref.Paged(q_len, kv_len, 2, 64, page, dtype, seed=3)
    _check(ks, work, P, _q(P, 6, 64, dtype, 4), window)


@pytest.mark.parametrize("dtype", (F16, BF16))
@pytest.mark.parametrize("heads,kv_heads,dim", [(8, 2, 128), (3, 3, 128), (9, 3, 64), (2, 1, 256), (2, 2, 16), (32, 1, 64)])
@pytest.mark.parametrize("q,kv", [(2, 2), (17, 17), (128, 128), (129, 400), (300, 1100), (511, 2048)])
def test_one_chunk(ks, work, dtype, heads, kv_heads, dim, q, kv):
    P = ref.Paged([q], [kv], kv_heads, dim, 16, dtype, seed=5)
    _check(ks, work, P, _q(P, heads, dim, dtype, 6))


@pytest.mark.parametrize("dtype", (F16, BF16))
def test_rows_that_see_nothing(ks, work, dtype):
    """more new tokens than rows: the first ones have no row; no row at all"""
    P = ref.Paged([40, 3, 200, 1, 1], [10, 0, 150, 0, 33], 2, 64, 16, dtype, seed=7)
    got = _check(ks, work, P, _q(P, 4, 64, dtype, 8))
    assert (got[:30] == 0).all() and (got[40:43] == 0).all() and (got[43:93] == 0).all()


@pytest.mark.parametrize("dim", (64, 128))
@pytest.mark.parametrize("q", (1, 40, 300))
def test_scores_far_apart(ks, work, dim, q):
    """maxima that keep rising along the keys, by far more than exp's range, and that fall"""
    for sign in (1.0, -1.0):
        P = ref.Paged([q], [700], 2, dim, 32, BF16, seed=9)
        ramp = torch.linspace(-8, 8, 700) * sign
        for i in range(700):
            P.k[P.host_table[0, i // 32], i % 32] = ramp[i].to(BF16).cuda()
        qq = torch.full((q, 4, dim), 2.0, dtype=BF16, device="cuda")
        # equal dims: the score is 2 dim ramp scale, exact in 32 bits
        _check(ks, work, P, qq)


@pytest.mark.parametrize("q", (1, 200))
def test_strides(ks, work, q):
    """padded heads, head-major pages and query rows inside a wider row"""
    for head_major in (False, True):
        P = ref.Paged([q, q], [300, 210], 2, 64, 16, F16, seed=10, pad=8, head_major=head_major)
        wide = _q(P, 12, 64, F16, 11)
        out = torch.full((P.tokens, 10, 64), float("nan"), dtype=F16, device="cuda")
        qv, dv = wide[:, 3:9], out[:, 2:8]
        ks.paged_attn(qv, P.k, P.v, P.table, P.q_start, P.kv_len, P.max_q, P.max_kv, dv, work)
        want, mag = ref.attention(P, qv, 64 ** -0.5)
        assert ((dv.double() - want).abs() <= ref.attention_bound(F16, want, mag, 300, 6.0)).all()
        assert torch.isnan(out[:, :2]).all() and torch.isnan(out[:, 8:]).all()


def test_long_and_again(ks, work):
    """one token over a long cache is split over the whole device; twice the same bits, on another stream too,
    and the workspace serves other lengths in between"""
    P = ref.Paged([1, 1], [40000, 3], 2, 128, 64, BF16, seed=12)
    R = ref.Paged([300, 1], [900, 77], 2, 128, 64, BF16, seed=13)
    q, r = _q(P, 8, 128, BF16, 14), _q(R, 8, 128, BF16, 15)
    first = _check(ks, work, P, q)
    _check(ks, work, R, r)
    assert torch.equal(_attn(ks, work, P, q).double(), first)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    mine = ks.paged_attn_work()
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        got = _attn(ks, mine, P, q)
    s.synchronize()
    assert torch.equal(got.double(), first)


def test_graph_with_new_lengths(ks, work):
    """a captured call is replayed with other lengths in the same plan arrays"""
    P = ref.Paged([1, 1, 1], [500, 64, 900], 2, 64, 16, F16, seed=16)
    q, dst = _q(P, 6, 64, F16, 17), torch.zeros((3, 6, 64), dtype=F16, device="cuda")
    call = lambda: ks.paged_attn(q, P.k, P.v, P.table, P.q_start, P.kv_len, 1, 900, dst, work)  # noqa: E731
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    P.kv = [123, 1, 899]
    P.kv_len.copy_(torch.tensor(P.kv, dtype=torch.int32))
    graph.replay()
    torch.cuda.synchronize()
    want, mag = ref.attention(P, q, 64 ** -0.5)
    assert ((dst.double() - want).abs() <= ref.attention_bound(F16, want, mag, 900, 6.0)).all()


@pytest.mark.parametrize("q", (1, 150))
def test_page_outside_the_cache(ks, work, q):
    """a page id that points nowhere reads as zeros and is counted; nothing else changes"""
    P = ref.Paged([q, q], [256, 256], 2, 64, 32, F16, seed=18)
    good = P.host_table.clone()
    qq = _q(P, 4, 64, F16, 19)
    for bad in (-7, P.k.shape[0], 2 ** 31 - 1):
        P.table.copy_(good)
        P.table[0, 2] = bad
        got = _attn(ks, work, P, qq)
        assert ks.paged_errors()[0] > 0
        Z = ref.Paged([q, q], [256, 256], 2, 64, 32, F16, seed=18)
        for c in (Z.k, Z.v):
            c[good[0, 2]] = 0
        want, mag = ref.attention(Z, qq, 64 ** -0.5)
        assert ((got.double() - want).abs() <= ref.attention_bound(F16, want, mag, 256, 6.0)).all()


def test_offsets_past_32_bits(ks, work):
    """pages that lie more than 2^32 elements from the cache's start, for both calls"""
    page, heads, dim = 16, 1, 64
    gap = (1 << 32) + 4096
    base = torch.zeros(gap + 4 * page * dim, dtype=F16, device="cuda")
    k = base.as_strided((2, page, heads, dim), (gap, heads * dim, dim, 1))
    v = base.as_strided((2, page, heads, dim), (gap, heads * dim, dim, 1), page * dim)
    table = torch.tensor([[1, 0]], dtype=torch.int32, device="cuda")
    n = 20
    q_start = torch.tensor([0, n], dtype=torch.int32, device="cuda")
    kv_len = torch.tensor([n], dtype=torch.int32, device="cuda")
    g = torch.Generator().manual_seed(20)
    x = torch.randn((n, 3, dim), generator=g).half().cuda()
    ks.paged_append(x[:, 0:1], x[:, 1:2], k, v, table, q_start, kv_len, n)
    assert torch.equal(k[1, :, 0], x[:16, 0]) and torch.equal(v[1, :, 0], x[:16, 1])
    assert torch.equal(k[0, :4, 0], x[16:, 0]) and torch.equal(v[0, :4, 0], x[16:, 1])
    P = ref.Paged.__new__(ref.Paged)
    P.q_len, P.kv, P.page, P.k, P.v, P.host_table, P.start = [n], [n], page, k, v, table.cpu(), [0, n]
    P.table, P.q_start, P.kv_len, P.max_q, P.max_kv, P.tokens = table, q_start, kv_len, n, n, n
    _check(ks, work, P, x[:, 2:3].contiguous())


@pytest.mark.parametrize("dim", (64, 128, 32))
@pytest.mark.parametrize("q", (1, 150))
def test_visible_nan_stays(ks, work, dim, q):
    """a NaN in a query is that row's alone; one in a key or value that rows see is theirs, and no other sequence's"""
    P = ref.Paged([q, q], [400, 400], 2, dim, 16, BF16, seed=26)
    qq = _q(P, 4, dim, BF16, 27)
    clean = _attn(ks, work, P, qq)
    assert not torch.isnan(clean).any()
    bad = qq.clone()
    bad[q - 1, 1, 3] = float("nan")
    got = _attn(ks, work, P, bad)
    assert torch.isnan(got[q - 1, 1]).all()
    got[q - 1, 1] = clean[q - 1, 1]
    assert torch.equal(got, clean)
    for cache in (P.k, P.v):
        at = (P.host_table[0, 0].item(), 5)
        old = cache[at].clone()
        cache[at][0] = float("nan")
        got = _attn(ks, work, P, qq)
        cache[at] = old
        assert torch.isnan(got[:q, :2]).all()                # kv head 0 of the first sequence
        assert torch.equal(got[q:], clean[q:]) and torch.equal(got[:q, 2:], clean[:q, 2:])


# ------------------------------------------------------------------ append

def _cos_sin(rows, half, seed=0):
    a = torch.outer(torch.arange(rows).double(), 10000.0 ** (-torch.arange(half).double() / max(half, 1)))
    return torch.stack((a.cos(), a.sin()), -1).float().contiguous().cuda()


@pytest.mark.parametrize("src,dtype", [(F32, F16), (F32, BF16), (F16, F16), (BF16, BF16), (BF16, F16), (F16, BF16)])
@pytest.mark.parametrize("dim,rot,neox", [(64, 64, False), (64, 64, True), (128, 64, False), (128, 64, True), (128, 128, True),
                                          (16, 6, False), (16, 6, True), (32, 2, True), (256, 256, False), (64, 0, False)])
@pytest.mark.parametrize("with_q", (True, False))
def test_append(ks, src, dtype, dim, rot, neox, with_q):
    q_len, kv_len = [3, 1, 0, 40, 1, 18], [3, 77, 12, 200, 1, 10]       # the last: eight tokens without a row
    P = ref.Paged(q_len, kv_len, 2, dim, 16, dtype, seed=21, junk=3.0)
    before = [P.k.clone(), P.v.clone()]
    g = torch.Generator().manual_seed(22)
    x = torch.randn((P.tokens, 3 + 2 + 2, dim), generator=g).to(src).cuda()
    q, k, v = x.split((3, 2, 2), 1)
    cs = _cos_sin(P.max_kv, rot // 2) if rot else None
    q_out = torch.full((P.tokens, 3, dim), 5.0, dtype=dtype, device="cuda")
    ks.paged_append(k, v, P.k, P.v, P.table, P.q_start, P.kv_len, P.max_kv, q=q if with_q else None,
                    q_out=q_out if with_q else None, cos_sin=cs, neox=neox)
    u = ref.UNIT[dtype]

    def near(got, x, pos):
        if cs is None:
            want, mag = x.double(), torch.zeros_like(x, dtype=torch.float64)
        else:
            want, mag = ref.rotate(x, cs[pos], neox)
        # two products and a sum in 32 bits, then one rounding
        assert ((got.double() - want).abs() <= u * want.abs() * 1.001 + 3 * 2.0 ** -24 * mag * 1.001 + 2.0 ** -25).all()

    touched = torch.zeros(P.k.shape[:2], dtype=torch.bool)
    for s, n in enumerate(q_len):
        skip = max(0, n - kv_len[s])
        pos = torch.arange(kv_len[s] - n + skip, kv_len[s])
        a, b = P.start[s] + skip, P.start[s] + n
        ids, off = P.host_table[s].long()[pos // 16], pos % 16
        touched[ids, off] = True
        near(P.k[ids, off], k[a:b], pos)
        assert torch.equal(P.v[ids, off].double(), v[a:b].to(dtype).double())
        if with_q:
            near(q_out[a:b], q[a:b], pos)
            assert (q_out[a - skip:a] == 5.0).all()
    for now, old in zip((P.k, P.v), before):
        assert torch.equal(now[~touched], old[~touched])
    assert ks.paged_errors() == (0, 0)


def test_append_page_outside_the_cache(ks):
    P = ref.Paged([20], [20], 1, 64, 8, F16, seed=23, junk=3.0)
    good = P.host_table.clone()
    P.table[0, 1] = 99
    k, v = P.k.clone(), P.v.clone()
    x = torch.randn((20, 2, 64), device="cuda")
    ks.paged_append(x[:, :1], x[:, 1:], P.k, P.v, P.table, P.q_start, P.kv_len, 20)
    assert ks.paged_errors()[0] > 0
    changed = (P.k != k).flatten(1).any(1).cpu()
    assert changed[good[0, 0].long()] and changed[good[0, 2].long()] and int(changed.sum()) == 2


def test_append_then_attention_is_one_step(ks, work):
    """a prompt in one chunk and the same prompt in pieces give the same cache, and near outputs"""
    n, dim = 150, 64
    g = torch.Generator().manual_seed(24)
    x = torch.randn((n, 6, dim), generator=g).cuda()
    outs, caches = [], []
    for pieces in ([n], [1, 60, 1, 88]):
        P = ref.Paged([n], [n], 1, dim, 16, F16, seed=25, junk=0.0)
        cs = _cos_sin(n, dim // 2)
        out, at = [], 0
        for m in pieces:
            q, k, v = x[at:at + m].split((4, 1, 1), 1)
            q_start = torch.tensor([0, m], dtype=torch.int32, device="cuda")
            kv_len = torch.tensor([at + m], dtype=torch.int32, device="cuda")
            qo = torch.empty((m, 4, dim), dtype=F16, device="cuda")
            ks.paged_append(k, v, P.k, P.v, P.table, q_start, kv_len, n, q=q, q_out=qo, cos_sin=cs)
            dst = torch.empty_like(qo)
            ks.paged_attn(qo, P.k, P.v, P.table, q_start, kv_len, m, n, dst, work)
            out.append(dst)
            at += m
        outs.append(torch.cat(out).double())
        caches.append((P.k, P.v))
    assert torch.equal(caches[0][0], caches[1][0]) and torch.equal(caches[0][1], caches[1][1])
    # both within (3 u + 2^-12) max |v| of the exact value
    assert float((outs[0] - outs[1]).abs().max()) <= 2 * (3 * 2.0 ** -11 + 2.0 ** -12) * float(x.abs().max())
