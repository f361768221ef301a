"""The paged decoder on the GPU: logits near those of the LNS graph with its own attention, whatever the batch and the
chunks, and sampled tokens."""
import pytest

pytestmark = pytest.mark.gpu

TINY = dict(n_layer=2, n_embd=64, n_head=4, n_head_kv=2, head_dim=16, n_ff=128, vocab=320, rope_base=10000.0, eps=1e-5)
WIDE = dict(n_layer=1, n_embd=192, n_head=3, n_head_kv=1, head_dim=64, n_ff=256, vocab=320, rope_base=10000.0, eps=1e-5)


def _ops(cfg):
    from lnsb200 import model
    return model.GpuOps(cfg, model.init_weights(cfg, seed=3), mode="sum32", n_ctx=128, fmt=32)


def _near(a, b):
    """xlns32's linears carry a difference along; the attention's own is 2^-11 for q, the weights and the output, which
    2^-7 of the largest logit covers over two layers"""
    return float((a - b).abs().max()) <= 2.0 ** -7 * float(b.abs().max())


@pytest.mark.parametrize("cfg", (TINY, WIDE), ids=("head 16", "head 64"))
def test_logits_of_the_graph(cfg):
    from lnsb200 import model, serve
    ops = _ops(cfg)
    prompts = [model.prompt_ids(cfg, n, seed=n) for n in (7, 1, 40)]
    want = [model.forward(ops, cfg, p, 0).view(1, -1).clone() for p in prompts]
    dec = serve.PagedDecoder(ops, n_pages=16)
    seqs = [dec.open() for _ in prompts]
    got = dec.forward(list(zip(seqs, prompts)))
    for g, w in zip(got, want):
        assert _near(g[None], w)
    # the same prompts in pieces, beside one another
    dec2 = serve.PagedDecoder(ops, n_pages=16)
    s0, s1, s2 = (dec2.open() for _ in prompts)
    dec2.forward([(s2, prompts[2][:17]), (s0, prompts[0][:6])])
    dec2.forward([(s0, prompts[0][6:]), (s2, prompts[2][17:39])])
    again = dec2.forward([(s1, prompts[1]), (s2, prompts[2][39:])])
    assert _near(again[0][None], want[1]) and _near(again[1][None], want[2])
    assert ops.ks.paged_errors() == (0, 0)


def test_steps_and_pages():
    from lnsb200 import model, serve
    ops = _ops(TINY)
    dec = serve.PagedDecoder(ops, n_pages=6)
    prompts = [model.prompt_ids(TINY, n, seed=n) for n in (20, 5)]
    seqs = [dec.open() for _ in prompts]
    logits = dec.forward(list(zip(seqs, prompts)))
    greedy, prob = dec.sample(logits, temperature=0.0)
    assert greedy.tolist() == [int(r.argmax()) for r in logits] and prob.tolist() == [1.0, 1.0]
    kept = logits.topk(5, 1).indices
    tokens, prob = dec.sample(logits, u=[0.1, 0.9], top_k=5)
    assert all(t in k for t, k in zip(tokens.tolist(), kept.tolist())) and ((prob > 0) & (prob <= 1)).all()
    for _ in range(8):
        out = dec.step([(s, [t]) for s, t in zip(seqs, tokens.tolist())], u=[0.3, 0.6], temperature=0.7, top_p=0.9)
        assert all(0 <= t < TINY["vocab"] for t in out)
    dec.close(seqs[0])
    other = dec.open()
    dec.forward([(other, prompts[0]), (seqs[1], [1])])
    with pytest.raises(MemoryError):
        dec.forward([(dec.open(), list(range(90)))])
    with pytest.raises(ValueError):
        dec.forward([(other, [])])
    with pytest.raises(ValueError):
        dec.forward([(other, [1] * 120)])
    assert ops.ks.paged_errors() == (0, 0)
