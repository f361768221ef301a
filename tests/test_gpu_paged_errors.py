"""What lnsb_paged_errors counts."""
import threading

import pytest
import torch

import serve_ref as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ks():
    import lnsb200
    return lnsb200.KernelSet(16, "base")


@pytest.mark.parametrize("n_dims", (0, 64, 6))
@pytest.mark.parametrize("offset", (0, 1))
@pytest.mark.parametrize("with_q", (True, False))
def test_a_token_without_a_page_counts_once(ks, n_dims, offset, with_q):
    """whatever the alignment and the pairs, which choose the kernel"""
    P = ref.Paged([20, 30], [20, 40], 2, 64, 8, torch.float16, seed=60, junk=0.0)
    P.table[0, 1], P.table[1, 2] = 99, -5                  # rows 8 .. 15 of the first, 16 .. 23 of the second
    P.table[1, 0] = -1                                     # rows 0 .. 7, none of them new
    x = torch.randn(50 * 7 * 64 + 1, device="cuda")[offset:][:50 * 7 * 64].view(50, 7, 64)
    cs = torch.zeros(P.max_kv, n_dims // 2, 2, device="cuda") if n_dims else None
    ks.paged_errors()
    q, k, v = x.split((3, 2, 2), 1)
    ks.paged_append(k, v, P.k, P.v, P.table, P.q_start, P.kv_len, P.max_kv, q=q if with_q else None,
                    q_out=torch.zeros(50, 3, 64, dtype=torch.float16, device="cuda") if with_q else None, cos_sin=cs)
    assert ks.paged_errors() == (16, 0)
    assert ks.paged_errors() == (0, 0)


def test_no_count_is_lost(ks):
    """one thread launches, others read and clear all the while: what they were given adds up"""
    P = ref.Paged([20], [20], 1, 64, 8, torch.float16, seed=61, junk=0.0)
    P.table[0, 1] = 99
    x = torch.zeros((20, 2, 64), device="cuda")
    ks.paged_errors()
    steps, seen, done = 3000, [0, 0, 0], threading.Event()

    def launch():
        for _ in range(steps):
            ks.paged_append(x[:, :1], x[:, 1:], P.k, P.v, P.table, P.q_start, P.kv_len, 20)
        done.set()

    def read(i):
        while not done.is_set():
            seen[i] += ks.paged_errors()[0]

    threads = [threading.Thread(target=launch)] + [threading.Thread(target=read, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    seen[2] = ks.paged_errors()[0]
    assert sum(seen) == 8 * steps, seen


@pytest.mark.parametrize("dim", (64, 128))
def test_waits_that_run_out(ks, dim):
    """with a limit of nothing the first wait for memory gives up: the call ends, both counts say so, and with work
    zeroed and the limit back the next call is right"""
    import test_gpu_paged as paged
    P = ref.Paged([300, 40], [1100, 500], 2, dim, 16, torch.bfloat16, seed=62)
    q = paged._q(P, 8, dim, torch.bfloat16, 63)
    work, other = ks.paged_attn_work(), ks.paged_attn_work()
    paged._check(ks, work, P, q)
    ks.paged_attn_wait_limit(0)
    try:
        for i in range(3):
            paged._attn(ks, work, P, q)
            torch.cuda.synchronize()
            assert ks.paged_errors()[1] > 0 and ks.paged_attn_timeouts(work) > 0
    finally:
        ks.paged_attn_wait_limit(1 << 31)
    assert ks.paged_attn_timeouts(other) == 0
    paged._check(ks, other, P, q)
    work.zero_()
    paged._check(ks, work, P, q)
    assert ks.paged_attn_timeouts(work) == 0


def test_the_decoder_raises_and_goes_on(ks):
    from lnsb200 import model, serve
    cfg = dict(n_layer=1, n_embd=192, n_head=3, n_head_kv=1, head_dim=64, n_ff=256, vocab=320, rope_base=10000.0, eps=1e-5)
    ops = model.GpuOps(cfg, model.init_weights(cfg, seed=3), mode="base", n_ctx=128, fmt=32)
    prompt = model.prompt_ids(cfg, 50, seed=4)
    dec = serve.PagedDecoder(ops, n_pages=16)
    s = dec.open()
    want = dec.step([(s, prompt)], temperature=0.0)
    dec.close(s)
    s = dec.open()
    ops.ks.paged_attn_wait_limit(0)
    try:
        with pytest.raises(RuntimeError, match="ran out"):
            dec.step([(s, prompt)], temperature=0.0)
    finally:
        ops.ks.paged_attn_wait_limit(1 << 31)
    assert dec.pool.length[s] == 0
    assert dec.step([(s, prompt)], temperature=0.0) == want
    ops.ks.paged_errors()
