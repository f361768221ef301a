"""Calls of the paged operators one behind the other, each reading what the one before it wrote."""
import pytest
import torch

import serve_ref as ref

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("heads,kv_heads,dim", [(9, 3, 64), (8, 2, 128), (4, 2, 32)])
@pytest.mark.parametrize("captured", (False, True))
def test_attention_sees_the_append_before_it(heads, kv_heads, dim, captured):
    """forty steps of append and attention on a batch of chunks and single tokens, with nothing between them, give the
    bits of the same steps with the device idle before every call"""
    import lnsb200
    ks = lnsb200.KernelSet(16, "base")
    work = ks.paged_attn_work()
    q_len, kv_len = [1, 70, 0, 33, 1, 150, 1, 2], [500, 300, 9, 33, 1, 700, 64, 90]
    P = ref.Paged(q_len, kv_len, kv_heads, dim, 16, torch.bfloat16, seed=30)
    g = torch.Generator().manual_seed(31)
    n = 40
    x = torch.randn((n, P.tokens, heads + 2 * kv_heads, dim), generator=g).to(torch.bfloat16).cuda()
    q_rot = torch.zeros((P.tokens, heads, dim), dtype=torch.bfloat16, device="cuda")
    out = [torch.zeros((n, P.tokens, heads, dim), dtype=torch.bfloat16, device="cuda") for _ in range(2)]

    def step(i, dst, wait):
        q, k, v = x[i].split((heads, kv_heads, kv_heads), 1)
        ks.paged_append(k, v, P.k, P.v, P.table, P.q_start, P.kv_len, P.max_kv, q=q, q_out=q_rot)
        wait()
        ks.paged_attn(q_rot, P.k, P.v, P.table, P.q_start, P.kv_len, P.max_q, P.max_kv, dst[i], work)
        wait()

    for i in range(n):
        step(i, out[0], torch.cuda.synchronize)
    steps = lambda: [step(i, out[1], lambda: None) for i in range(n)]  # noqa: E731
    if captured:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            steps()
        graph.replay()
    else:
        steps()
    torch.cuda.synchronize()
    assert torch.equal(out[0], out[1])
    assert not torch.equal(out[0][0], out[0][1])
    assert ks.paged_errors() == (0, 0)
