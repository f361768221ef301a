"""The paged decoder's host side, on the CPU: a model's ops and kernels are stand-ins that write down what they are given
and on which stream."""
import contextlib

import pytest
import torch

from lnsb200.serve import PagedDecoder

CFG = dict(n_layer=2, n_embd=8, n_head=2, n_head_kv=1, head_dim=4, n_ff=8, vocab=11, eps=1e-5)


class Stream:
    def __init__(self, name, log):
        self.name, self.log = name, log

    def wait_stream(self, other):
        self.log.append(("wait", self.name, other.name))


class Cuda:
    """torch.cuda's part in it: which stream is current"""

    def __init__(self, log):
        self.now, self.log = Stream("current", log), log

    def current_stream(self, device=None):
        return self.now

    @contextlib.contextmanager
    def stream(self, s):
        before, self.now = self.now, s
        try:
            yield
        finally:
            self.now = before


class Torch:
    """torch, with each call that makes or moves device data written down with the stream it runs on"""

    def __init__(self, log):
        self.cuda, self.log = Cuda(log), log

    def __getattr__(self, name):
        v = getattr(torch, name)
        if name in ("tensor", "as_tensor", "empty", "empty_like", "zeros", "rand"):
            def call(*a, **kw):
                self.log.append((name, self.cuda.now.name))
                return v(*a, **kw)
            return call
        return v


class Kernels:
    def __init__(self, ops):
        self.ops, self.log = ops, ops.log

    def paged_attn_work(self, device=None):
        self.log.append(("work", self.ops.torch.cuda.now.name))
        return torch.zeros(64, dtype=torch.uint8)

    def paged_attn_timeouts(self, work):
        self.log.append(("timeouts", self.ops.torch.cuda.now.name))
        return work[-8:].view(torch.int64).item()

    def _call(self, name, stream):
        now = self.ops.torch.cuda.now
        self.log.append((name, (stream or now).name))
        assert stream in (None, now)
        if name == self.ops.fail:
            raise RuntimeError("out of memory")

    def paged_append(self, k, v, kc, vc, table, q_start, kv_len, max_kv, q=None, q_out=None, cos_sin=None, stream=None):
        self._call("append", stream)
        self.ops.plans.append((table.tolist(), q_start.tolist(), kv_len.tolist()))

    def paged_attn(self, q, kc, vc, table, q_start, kv_len, max_q, max_kv, dst, work, stream=None):
        self._call("attn", stream)
        dst.zero_()
        if self.ops.timeout:
            work[-8:].view(torch.int64).add_(1)
            work[0] = 1                                     # a counter left half way

    def f16_to_f32(self, src, dst, n, stream=None):
        self._call("to f32", stream)
        dst.copy_(src.view(dst.shape))

    def sample(self, logits, u, token, prob, t, k, p, m, stream=None):
        self._call("sample", stream)
        token.copy_(logits.argmax(1))
        prob.fill_(1.0)


class Ops:
    def __init__(self, stream=None, n_ctx=32):
        self.log, self.plans, self.fail, self.timeout = [], [], None, False
        self.torch, self.cfg, self.n_ctx, self.dev = Torch(self.log), CFG, n_ctx, torch.device("cpu")
        self.stream = Stream(stream, self.log) if stream else None
        self.rope_cs, self.ks = torch.zeros(n_ctx, 2, 2), Kernels(self)

    def _op(self, name, out):
        self.log.append((name, self.torch.cuda.now.name))
        if name == self.fail:
            raise RuntimeError("out of memory")
        return out

    def embed(self, ids):
        assert all(0 <= i < CFG["vocab"] for i in ids)
        return self._op("embed", torch.zeros(len(ids), CFG["n_embd"]))

    def w(self, il, name):
        return name

    def rms_norm(self, x, eps, name=None):
        return self._op("norm", x.clone())

    def mul(self, x, w):
        return self._op("mul", x.clone())

    def add(self, a, b):
        return self._op("add", a + b)

    def swiglu(self, gate, up):
        return self._op("swiglu", gate * up)

    def linear(self, w, x, name=None, src=None):
        out = torch.zeros(x.shape[0], CFG["vocab"] if w == "output" else CFG["n_embd"])
        out[:, 3] = 1.0
        return self._op("linear", out)

    def linears(self, il, ws, x, names=None, src=None):
        n = {"wq": 8, "wk": 4, "wv": 4, "w_up": 8, "w_gate": 8}
        return [self._op("linears", torch.zeros(x.shape[0], n[w])) for w in ws]


# -------------------------------------------------------------------- streams

def _ran(log):
    return {e[1] for e in log if e[0] != "wait"}


@pytest.mark.parametrize("u", (None, [0.5, 0.5]))
def test_everything_runs_on_the_models_stream(u):
    """kernels, copies, random numbers and allocations: a tensor made, read or freed on another stream would not be
    ordered with the kernels"""
    ops = Ops("side")
    dec = PagedDecoder(ops, n_pages=8, page_size=4)
    a, b = dec.open(), dec.open()
    assert dec.step([(a, [1, 2, 3]), (b, [4])], u=u, temperature=[0.5, 0.7], top_p=0.9) == [3, 3]
    assert _ran(ops.log) == {"side"}
    # the model's stream waits for the current one before the step's first work, and the current one for it behind the last
    work = [i for i, e in enumerate(ops.log) if e[0] != "wait"]
    first, last = ops.log.index(("embed", "side")), work[-1]
    assert ("wait", "side", "current") in ops.log[:first]
    assert ("wait", "current", "side") in ops.log[last:]
    assert ops.torch.cuda.now.name == "current"


def test_the_stream_is_left_after_an_error():
    ops = Ops("side")
    dec = PagedDecoder(ops, n_pages=8, page_size=4)
    a = dec.open()
    ops.fail = "attn"
    with pytest.raises(RuntimeError, match="out of memory"):
        dec.step([(a, [1, 2])])
    assert ops.torch.cuda.now.name == "current" and ops.log[-1] == ("wait", "current", "side")


def test_without_a_stream_the_current_one():
    ops = Ops()
    dec = PagedDecoder(ops, n_pages=8, page_size=4)
    a = dec.open()
    assert dec.step([(a, [1, 2, 3])]) == [3]
    assert _ran(ops.log) == {"current"} and not [e for e in ops.log if e[0] == "wait"]


# ------------------------------------------------------ a step that goes wrong

def _state(dec):
    p = dec.pool
    return dict(p.length), {s: list(v) for s, v in p.pages.items()}, list(p.free)


@pytest.mark.parametrize("fail", ("embed", "norm", "mul", "linears", "append", "attn", "to f32", "linear", "add", "swiglu", "sample"))
def test_a_failed_step_leaves_the_pool(fail):
    """whatever call raises: the sequences keep their rows and pages, and the step can be taken again, in smaller pieces"""
    ops = Ops()
    dec = PagedDecoder(ops, n_pages=8, page_size=4)
    a, b = dec.open(), dec.open()
    dec.step([(a, [1, 2, 3]), (b, [4])])
    before = _state(dec)
    ops.fail = fail
    with pytest.raises(RuntimeError, match="out of memory"):
        dec.step([(a, [5, 6, 7, 8, 9, 1]), (b, [2, 3, 4, 5])])
    assert _state(dec) == before
    ops.fail, ops.plans = None, []
    assert dec.step([(b, [2, 3])]) == [3]
    table, q_start, kv_len = ops.plans[0]
    assert q_start == [0, 2] and kv_len == [3] and table == [dec.pool.pages[b]]
    assert dec.pool.length == {a: 3, b: 3}


@pytest.mark.parametrize("bad", (dict(u=[0.1, 0.2]), dict(top_k="many"), dict(temperature=[1.0, 2.0, 3.0])), ids=str)
def test_parameters_that_do_not_fit_leave_the_pool(bad):
    dec = PagedDecoder(Ops(), n_pages=8, page_size=4)
    seqs = [dec.open(), dec.open(), dec.open(), dec.open()]
    before = _state(dec)
    with pytest.raises((RuntimeError, ValueError, TypeError)):
        dec.step([(s, [1, 2]) for s in seqs], **bad)
    assert _state(dec) == before


def test_forward_alone_too():
    ops = Ops()
    dec = PagedDecoder(ops, n_pages=8, page_size=4)
    a = dec.open()
    before = _state(dec)
    ops.fail = "attn"
    with pytest.raises(RuntimeError):
        dec.forward([(a, [1, 2, 3, 4, 5])])
    assert _state(dec) == before
    ops.fail = None
    assert dec.forward([(a, [1, 2, 3, 4, 5])]).shape == (1, CFG["vocab"])
    assert dec.pool.length == {a: 5}


# ------------------------------------------------------------------ token ids

@pytest.mark.parametrize("ids", ([-1], [1, CFG["vocab"]], [2 ** 40, 1], [3, -2 ** 31]), ids=str)
def test_tokens_outside_the_vocabulary(ids):
    """refused on the host before anything grows or runs: -1 is what a row without a finite logit samples"""
    ops = Ops()
    dec = PagedDecoder(ops, n_pages=8, page_size=4)
    a, b = dec.open(), dec.open()
    before, log = _state(dec), list(ops.log)
    for call in (dec.step, dec.forward):
        with pytest.raises(ValueError, match="vocab"):
            call([(b, [1]), (a, ids)])
    assert _state(dec) == before and ops.log == log


# ----------------------------------------------------------- waits that ran out

def test_an_attention_that_gave_up():
    """the step raises and takes its rows back, and the workspace is clean for the next"""
    ops = Ops()
    dec = PagedDecoder(ops, n_pages=8, page_size=4)
    a = dec.open()
    assert dec.step([(a, [1, 2, 3])]) == [3]
    before = _state(dec)
    ops.timeout = True
    with pytest.raises(RuntimeError, match="ran out"):
        dec.step([(a, [4, 5, 6])])
    assert _state(dec) == before and not dec.work.any()
    dec.forward([(a, [4])])
    with pytest.raises(RuntimeError, match="ran out"):
        dec.check()
    ops.timeout = False
    dec.check()
    assert dec.step([(a, [5])]) == [3]


def test_one_decoders_timeout_is_its_own():
    slow, fine = Ops(), Ops()
    a, b = PagedDecoder(slow, n_pages=8, page_size=4), PagedDecoder(fine, n_pages=8, page_size=4)
    slow.timeout = True
    sa, sb = a.open(), b.open()
    a.forward([(sa, [1])])
    assert b.step([(sb, [1, 2])]) == [3]
    with pytest.raises(RuntimeError, match="ran out"):
        a.check()
