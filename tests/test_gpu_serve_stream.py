"""The paged decoder on a stream of the model's own."""
import pytest
import torch

pytestmark = pytest.mark.gpu

TINY = dict(n_layer=2, n_embd=64, n_head=4, n_head_kv=2, head_dim=16, n_ff=128, vocab=320, rope_base=10000.0, eps=1e-5)


def test_steps_on_another_stream_than_the_current():
    """with work ahead on either stream, the steps give what they give on the current stream"""
    from lnsb200 import model, serve
    weights = model.init_weights(TINY, seed=3)
    prompts = [model.prompt_ids(TINY, n, seed=n) for n in (20, 5, 40)]
    runs = []
    for stream in (None, torch.cuda.Stream()):
        ops = model.GpuOps(TINY, weights, mode="sum32", n_ctx=128, stream=stream, fmt=32)
        busy = torch.zeros(1 << 26, device="cuda")
        dec = serve.PagedDecoder(ops, n_pages=24)
        seqs = [dec.open() for _ in prompts]
        logits = dec.forward(list(zip(seqs, prompts)))
        seen = [logits.clone()]
        tokens = dec.sample(logits, u=[0.2, 0.5, 0.8], temperature=0.8, top_p=0.95)[0].tolist()
        out = [tokens]
        for i in range(6):
            for s in (torch.cuda.current_stream(), stream):
                if s is not None:
                    with torch.cuda.stream(s):              # some hundreds of microseconds, not a wait on anything
                        busy.add_(1.0).mul_(0.5)
            out.append(dec.step([(s, [t]) for s, t in zip(seqs, out[-1])], u=[0.3, 0.6, 0.9], temperature=0.7, top_p=0.9))
        seen.append(dec.forward([(s, [t]) for s, t in zip(seqs, out[-1])]).clone())
        runs.append((seen, out))
        assert ops.ks.paged_errors() == (0, 0)
    assert runs[0][1] == runs[1][1]
    assert all(torch.equal(a, b) for a, b in zip(runs[0][0], runs[1][0]))


@pytest.mark.parametrize("fused", (True, False))
def test_the_model_on_another_stream_than_the_current(fused):
    """the same of the graph with its own cache: a prompt, then steps, with work ahead on either stream"""
    from lnsb200 import model
    weights, runs = model.init_weights(TINY, seed=5), []
    for stream in (None, torch.cuda.Stream()):
        ops = model.GpuOps(TINY, weights, mode="sum32", n_ctx=64, stream=stream, fmt=32)
        ops.fused = fused
        busy = torch.zeros(1 << 26, device="cuda")
        ids, pos, out = model.prompt_ids(TINY, 9, seed=6), 0, []
        for i in range(6):
            for s in (torch.cuda.current_stream(), stream):
                if s is not None:
                    with torch.cuda.stream(s):
                        busy.add_(1.0).mul_(0.5)
            out.append(model.forward(ops, TINY, ids, pos).clone())
            pos, ids = pos + len(ids), [int(out[-1].argmax())]
        runs.append(out)
    assert all(torch.equal(a, b) for a, b in zip(*runs))
