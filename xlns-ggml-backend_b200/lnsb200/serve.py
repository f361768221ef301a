"""Decoding many sequences at once from a paged KV cache.

`PagedDecoder` runs the LLaMA graph of `model.forward` over a batch of prompt
chunks and single tokens: the matrix products, norms and activations go through
the LNS kernels as `model.GpuOps` runs them; the rotation, the cache, the
attention and the choice of the next token are ordinary floats (the ops that a
host takes out of LNS with LNS_DISABLE_OPS=rope,kq,kq_soft_max,kqv), through
`lnsb_paged_append`, `lnsb_paged_attn` and `lnsb_sample`.

    ops = model.GpuOps(cfg, weights, mode="sum32", n_ctx=2048)
    dec = serve.PagedDecoder(ops, n_pages=512)
    seqs = [dec.open() for _ in prompts]
    tokens = dec.step([(s, p) for s, p in zip(seqs, prompts)], temperature=0.8, top_p=0.95)
    tokens = dec.step([(s, [t]) for s, t in zip(seqs, tokens)], temperature=0.8, top_p=0.95)
"""
import contextlib

from .model import handed_over, on_stream

__all__ = ["PagePool", "PagedDecoder"]


class PagePool:
    """Which pages each open sequence holds (host side)."""

    def __init__(self, n_pages, page_size):
        self.page_size = page_size
        self.free = list(range(n_pages - 1, -1, -1))
        self.pages, self.length = {}, {}
        self.next_id = 0

    def open(self):
        s = self.next_id
        self.next_id += 1
        self.pages[s], self.length[s] = [], 0
        return s

    def grow(self, wanted):
        """room for n more rows of each (sequence, n) of `wanted`: for all of them, or MemoryError and nothing changes"""
        need = {}
        for s, n in wanted:
            if s not in self.pages:
                raise KeyError("sequence %r is not open" % (s,))
            if s in need:
                raise ValueError("sequence %r is given twice" % (s,))
            need[s] = max(0, -(-(self.length[s] + n) // self.page_size) - len(self.pages[s]))
        if sum(need.values()) > len(self.free):
            raise MemoryError("%d pages wanted, %d free" % (sum(need.values()), len(self.free)))
        for s, n in wanted:
            for _ in range(need[s]):
                self.pages[s].append(self.free.pop())
            self.length[s] += n

    def shrink(self, grown):
        """takes a grow back: the last n rows of each (sequence, n), and the pages that held nothing else"""
        for s, n in reversed(grown):
            self.length[s] -= n
            while len(self.pages[s]) > -(-self.length[s] // self.page_size):
                self.free.append(self.pages[s].pop())

    def close(self, s):
        self.free.extend(reversed(self.pages.pop(s)))
        del self.length[s]


class PagedDecoder:
    """One cache per layer and one pool of pages over a model's ops (`model.GpuOps`); the rotation's table bounds a
    sequence's length (ops.n_ctx).  All device work runs on the ops' stream, between what the caller's current stream
    was given before a call and what it is given after it; the ops without one use the current stream."""

    def __init__(self, ops, n_pages, page_size=16):
        torch, cfg = ops.torch, ops.cfg
        self.ops, self.cfg, self.ks, self.torch = ops, cfg, ops.ks, torch
        self.pool = PagePool(n_pages, page_size)
        shape = (n_pages, page_size, cfg["n_head_kv"], cfg["head_dim"])
        with on_stream(ops):
            # zeros: rows that no sequence has written are never seen, but a reader of the cache may look
            self.kc = [torch.zeros(shape, dtype=torch.float16, device=ops.dev) for _ in range(cfg["n_layer"])]
            self.vc = [torch.zeros(shape, dtype=torch.float16, device=ops.dev) for _ in range(cfg["n_layer"])]
            self.work = self.ks.paged_attn_work(ops.dev)

    def open(self):
        return self.pool.open()

    def close(self, seq):
        self.pool.close(seq)

    def _i32(self, v):
        return self.torch.tensor(v, dtype=self.torch.int32, device=self.ops.dev)

    def _grow(self, batch):
        """room in the pool for the new tokens of a batch"""
        if not batch or any(len(t) == 0 for _, t in batch):
            raise ValueError("every sequence of a batch needs a token")
        vocab = self.cfg["vocab"]
        if any(not 0 <= i < vocab for _, t in batch for i in t):     # -1: a row without a logit above -inf sampled it
            raise ValueError("a token is outside the vocabulary of %d" % vocab)
        if any(self.pool.length.get(s, 0) + len(t) > self.ops.n_ctx for s, t in batch):
            raise ValueError("a sequence would pass %d rows" % self.ops.n_ctx)
        grown = [(s, len(t)) for s, t in batch]
        self.pool.grow(grown)
        return grown

    @contextlib.contextmanager
    def _or_shrink(self, grown):
        """the rows of a step that raises are not the sequences': the next step writes them anew"""
        try:
            yield
        except BaseException:
            self.pool.shrink(grown)
            raise

    def forward(self, batch):
        """logits (F32, [len(batch)][vocab]) of the last of the new tokens of each (sequence, tokens) of `batch`; if it
        raises, the sequences are as they were.  The work is on its way when this returns: `check` says whether it went
        well"""
        with self._or_shrink(self._grow(batch)):
            return self._forward(batch)

    def _forward(self, batch):
        with on_stream(self.ops):
            logits = self._graph(batch)
        handed_over(self.ops, logits)
        return logits

    def _graph(self, batch):
        torch, ops, cfg, ks, stream = self.torch, self.ops, self.cfg, self.ks, self.ops.stream
        H, HKV, D = cfg["n_head"], cfg["n_head_kv"], cfg["head_dim"]
        pool = self.pool
        start = [0]
        for _, t in batch:
            start.append(start[-1] + len(t))
        T = start[-1]
        held = [pool.pages[s] for s, _ in batch]
        lengths = [pool.length[s] for s, _ in batch]
        wide = max(len(p) for p in held)
        plan = (self._i32([p + [-1] * (wide - len(p)) for p in held]), self._i32(start), self._i32(lengths))
        max_q, max_kv = max(len(t) for _, t in batch), max(lengths)
        x = ops.embed([i for _, t in batch for i in t])
        for il in range(cfg["n_layer"]):
            h = ops.mul(ops.rms_norm(x, cfg["eps"], "norm-%d" % il), ops.w(il, "attn_norm"))
            q, k, v = ops.linears(il, ("wq", "wk", "wv"), h, ("Qcur-%d" % il, "Kcur-%d" % il, "Vcur-%d" % il), "attn_norm-%d" % il)
            qh = torch.empty((T, H, D), dtype=torch.float16, device=ops.dev)
            ks.paged_append(k.view(T, HKV, D), v.view(T, HKV, D), self.kc[il], self.vc[il], *plan, max_kv,
                            q=q.view(T, H, D), q_out=qh, cos_sin=ops.rope_cs, stream=stream)
            oh = torch.empty_like(qh)
            ks.paged_attn(qh, self.kc[il], self.vc[il], *plan, max_q, max_kv, oh, self.work, stream=stream)
            a = torch.empty((T, H * D), dtype=torch.float32, device=ops.dev)
            ks.f16_to_f32(oh, a, a.numel(), stream=stream)
            x = ops.add(ops.linear(ops.w(il, "wo"), a, "attn_out-%d" % il, "kqv_out-%d" % il), x)
            h = ops.mul(ops.rms_norm(x, cfg["eps"], "norm-%d" % il), ops.w(il, "ffn_norm"))
            up, gate = ops.linears(il, ("w_up", "w_gate"), h, ("ffn_up-%d" % il, "ffn_gate-%d" % il), "ffn_norm-%d" % il)
            x = ops.add(ops.linear(ops.w(il, "w_down"), ops.swiglu(gate, up), "ffn_down-%d" % il, "ffn_swiglu-%d" % il), x)
        last = x[self._i32([n - 1 for n in start[1:]]).long()].contiguous()
        h = ops.mul(ops.rms_norm(last, cfg["eps"], "norm"), ops.w(None, "output_norm"))
        return ops.linear(ops.w(None, "output"), h, "result_output", "result_norm")

    def check(self):
        """raises RuntimeError if a wait inside the attention ran out since the last check: what came out of it and the
        rows written since are invalid (waits for the device)"""
        with on_stream(self.ops):
            n = self.ks.paged_attn_timeouts(self.work)
            if n:
                self.work.zero_()
        if n:
            raise RuntimeError("%d waits inside the attention ran out" % n)

    def sample(self, logits, u=None, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
        """next tokens (int32 on the device) and their probabilities; each parameter one number, or one for each row;
        u: the random numbers, or None to draw them"""
        torch, n = self.torch, logits.shape[0]
        each = lambda v, t: torch.as_tensor(v, dtype=t, device=self.ops.dev).expand(n).contiguous()  # noqa: E731
        with on_stream(self.ops):
            u = torch.rand(n, device=self.ops.dev) if u is None else each(u, torch.float32)
            token = torch.empty(n, dtype=torch.int32, device=self.ops.dev)
            prob = torch.empty(n, dtype=torch.float32, device=self.ops.dev)
            self.ks.sample(logits, u, token, prob, each(temperature, torch.float32), each(top_k, torch.int32),
                           each(top_p, torch.float32), each(min_p, torch.float32), stream=self.ops.stream)
        handed_over(self.ops, token, prob)
        return token, prob

    def step(self, batch, u=None, **sampling):
        """forward, then sample: the next token of each sequence of the batch, on the host; if it raises, the sequences
        are as they were"""
        with self._or_shrink(self._grow(batch)):
            tokens = self.sample(self._forward(batch), u, **sampling)[0].tolist()
            self.check()
            return tokens
