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
