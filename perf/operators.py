"""What is measured of the paged serving operators: appending rotated keys and
values to a paged cache, attention of new tokens over that cache, and sampling
the next token.

Each operator has a plain form in elementary torch operations (32 bits, rounded
once at the end) and the framework's kernels; `own` picks which of the two `run`
computes.  `exact` computes the same outputs from the definitions in 64 bits.
"""
import math
import os
import random
import sys

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


# ---------------------------------------------------------------- the cases

def listed():
    return [
        # one user's next token, early in a chat, on the 9/3-head 64-wide decoder: latency
        dict(name="attn token short", op="attn", seqs=1, q_lo=1, q_hi=1, ones=0, kv_lo=200, kv_hi=200, lens=1, heads=9,
             kv_heads=3, dim=64, page=16, type="f16", window=0),
        # one decode step of a ragged batch of 64 requests
        dict(name="attn token batch", op="attn", seqs=64, q_lo=1, q_hi=1, ones=0, kv_lo=1, kv_hi=8192, lens=2, heads=32,
             kv_heads=8, dim=128, page=64, type="bf16", window=0),
        # one decode step over a very long document
        dict(name="attn token long", op="attn", seqs=1, q_lo=1, q_hi=1, ones=0, kv_lo=131072, kv_hi=131072, lens=3, heads=32,
             kv_heads=8, dim=128, page=128, type="bf16", window=0),
        # continuous batching: single tokens beside prompt chunks and idle slots, sliding window, 9/3 heads
        dict(name="attn mixed window", op="attn", seqs=16, q_lo=0, q_hi=512, ones=8, kv_lo=1, kv_hi=4096, lens=4, heads=9,
             kv_heads=3, dim=64, page=16, type="f16", window=1024),
        # one prompt chunk over what came before it
        dict(name="attn chunk", op="attn", seqs=1, q_lo=512, q_hi=512, ones=0, kv_lo=8192, kv_hi=8192, lens=5, heads=32,
             kv_heads=8, dim=128, page=16, type="bf16", window=0),
        # long prompts in large chunks: the largest
        dict(name="attn chunks long", op="attn", seqs=2, q_lo=1800, q_hi=2048, ones=0, kv_lo=12000, kv_hi=16384, lens=6,
             heads=32, kv_heads=8, dim=128, page=64, type="bf16", window=0),
        # one token's keys and values from the F32 projection rows: latency
        dict(name="append token", op="append", seqs=1, q_lo=1, q_hi=1, ones=0, kv_lo=200, kv_hi=200, lens=7, heads=9,
             kv_heads=3, dim=64, rot=64, neox=False, page=16, src="f32", type="f16"),
        # one decode step of a batch
        dict(name="append batch", op="append", seqs=256, q_lo=1, q_hi=1, ones=0, kv_lo=1, kv_hi=1024, lens=8, heads=32,
             kv_heads=8, dim=128, rot=128, neox=True, page=64, src="bf16", type="bf16"),
        # prompt chunks, ragged, half of each head rotated
        dict(name="append chunks", op="append", seqs=5, q_lo=1111, q_hi=2222, ones=0, kv_lo=2222, kv_hi=4096, lens=9, heads=32,
             kv_heads=8, dim=128, rot=64, neox=False, page=16, src="f32", type="bf16"),
        # one user's next token, every filter on: latency
        dict(name="sample row", op="sample", rows=1, vocab=49152, type="f32", filters="all", pars=10),
        # a batch of requests, each with its own filters
        dict(name="sample batch", op="sample", rows=48, vocab=49152, type="f32", filters="mixed", pars=11),
        # a large batch over a large odd vocabulary
        dict(name="sample wide", op="sample", rows=256, vocab=131071, type="bf16", filters="mixed", pars=12),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("attn", "attn", "append", "sample"))
    if op == "sample":
        vocab = _log(rng, 1000, 131072)
        return dict(op="sample", rows=_log(rng, 1, 256), vocab=vocab, type=rng.choice(("f32", "f16", "bf16")),
                    filters=rng.choice(("all", "mixed", "none")), pars=rng.randrange(1 << 20))
    heads, kv_heads, dim = rng.choice(((9, 3, 64), (32, 8, 128), (16, 16, 64), (12, 4, 128), (8, 1, 64), (20, 4, 128)))
    case = dict(op=op, heads=heads, kv_heads=kv_heads, dim=dim, page=rng.choice((16, 32, 64, 128)),
                type=rng.choice(("f16", "bf16")), lens=rng.randrange(1 << 20))
    if op == "append":
        seqs = _log(rng, 1, 256)
        q_hi = 1 if rng.random() < 0.4 else _log(rng, 2, max(2, 8192 // seqs))
        case.update(seqs=seqs, q_lo=max(1, q_hi // 2), q_hi=q_hi, ones=0, kv_lo=q_hi, kv_hi=q_hi + rng.randrange(1, 1025),
                    rot=rng.choice((dim, dim, dim // 2)), neox=rng.random() < 0.5, src=rng.choice(("f32", case["type"])))
        return case
    kind = rng.choice(("tokens", "tokens", "chunks", "mixed"))
    if kind == "tokens":                                    # decode: at most 131072 keys over the batch
        seqs = _log(rng, 1, 128)
        hi = _log(rng, 1, 131072 // seqs)
        case.update(seqs=seqs, q_lo=1, q_hi=1, ones=0, kv_lo=max(1, hi // 8), kv_hi=hi)
    elif kind == "chunks":
        seqs = _log(rng, 1, 8)
        hi = _log(rng, 64, 16384 // seqs)
        q = _log(rng, 2, min(hi, 2048))
        case.update(seqs=seqs, q_lo=max(2, q * 3 // 4), q_hi=q, ones=0, kv_lo=max(q, hi // 2), kv_hi=hi)
    else:
        seqs = _log(rng, 4, 24)
        hi = _log(rng, 64, 4096)
        case.update(seqs=seqs, q_lo=0, q_hi=_log(rng, 2, min(hi, 512)), ones=seqs // 2, kv_lo=1, kv_hi=hi)
    case["window"] = rng.choice((0, 0, _log(rng, 16, 4096)))
    return case


def _lengths(case):
    """new tokens and visible keys of every sequence (keys include the new tokens); `ones` of them get one token"""
    rng = random.Random(case["lens"])
    q, kv = [], []
    for s in range(case["seqs"]):
        n = 1 if s < case["ones"] else rng.randint(case["q_lo"], case["q_hi"])
        q.append(n)
        kv.append(max(n, rng.randint(case["kv_lo"], case["kv_hi"])))
    at = list(range(case["seqs"]))
    rng.shuffle(at)
    return [q[i] for i in at], [kv[i] for i in at]


# ------------------------------------------------------------------- inputs

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _randn(g, *shape, type=torch.float32, scale=1.0):
    return (torch.randn(shape, generator=g, device="cuda", dtype=torch.float32) * scale).to(type)


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    g = _gen(seed)
    if case["op"] == "sample":
        return _prepare_sample(case, g)
    q_len, kv_len = _lengths(case)
    page, dim, heads, kv_heads, type = case["page"], case["dim"], case["heads"], case["kv_heads"], TYPES[case["type"]]
    start = [0]
    for n in q_len:
        start.append(start[-1] + n)
    pages = [-(-n // page) for n in kv_len]
    n_pages = sum(pages) + 3
    # pages are handed out in the order in which requests grew, so a sequence's lie scattered
    ids = torch.randperm(n_pages, generator=g, device="cuda").to(torch.int32)
    owner = torch.repeat_interleave(torch.arange(len(pages), device="cuda"), torch.tensor(pages, device="cuda"))
    first = torch.tensor([sum(pages[:s]) for s in range(len(pages))], device="cuda")
    table = torch.full((len(pages), max(pages)), -1, dtype=torch.int32, device="cuda")
    table[owner, torch.arange(sum(pages), device="cuda") - first[owner]] = ids[: sum(pages)]
    state = dict(op=case["op"], q_start=_i32(start), kv_len=_i32(kv_len), table=table, max_q=max(max(q_len), 1),
                 max_kv=max(kv_len))
    tokens = start[-1]
    if case["op"] == "append":
        # the projection's output rows: q heads, k heads, v heads
        qkv = _randn(g, tokens, (heads + 2 * kv_heads) * dim, type=TYPES[case["src"]])
        q, k, v = qkv.view(tokens, heads + 2 * kv_heads, dim).split((heads, kv_heads, kv_heads), 1)
        half = case["rot"] // 2
        ang = torch.outer(torch.arange(state["max_kv"], device="cuda", dtype=torch.float64),
                          100000.0 ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half))
        state.update(q=q, k=k, v=v, cos_sin=torch.stack((ang.cos(), ang.sin()), -1).float().contiguous(), rot=case["rot"],
                     neox=case["neox"])
    else:
        # queries that look for something: scores spread over several units
        state.update(q=_randn(g, tokens, heads, dim, type=type, scale=2.0), window=case["window"], scale=dim ** -0.5)
    state["k_cache"] = _randn(g, n_pages, page, kv_heads, dim, type=type)
    state["v_cache"] = _randn(g, n_pages, page, kv_heads, dim, type=type)
    return state


def _prepare_sample(case, g):
    rows, vocab = case["rows"], case["vocab"]
    # logits as a decoder's last layer gives them: a wide bulk and a few tokens well above it
    x = _randn(g, rows, vocab, scale=2.0)
    near = torch.randint(0, vocab, (rows, 24), generator=g, device="cuda")
    x.scatter_add_(1, near, 3.0 + 2.0 * torch.randn((rows, 24), generator=g, device="cuda"))
    rng = random.Random(case["pars"])
    temperature, top_k, top_p, min_p = [], [], [], []
    for r in range(rows):
        on = [case["filters"] == "all" or (case["filters"] == "mixed" and rng.random() < 0.5) for _ in range(3)]
        greedy = case["filters"] == "mixed" and rng.random() < 0.1
        temperature.append(0.0 if greedy else round(rng.uniform(0.5, 1.3), 2))
        top_k.append(rng.choice((20, 40, 64, 200, 1000)) if on[0] else 0)
        top_p.append(rng.choice((0.8, 0.9, 0.95)) if on[1] else 1.0)
        min_p.append(rng.choice((0.02, 0.05, 0.1)) if on[2] else 0.0)
    f32 = lambda v: torch.tensor(v, dtype=torch.float32, device="cuda")  # noqa: E731
    return dict(op="sample", logits=x.to(TYPES[case["type"]]), u=torch.rand(rows, generator=g, device="cuda"),
                temperature=f32(temperature), top_k=_i32(top_k), top_p=f32(top_p), min_p=f32(min_p))


# --------------------------------------------------------------- plain forms

def run(state):
    if own:
        return OWN[state["op"]](state)
    return PLAIN[state["op"]](state)


def _places(state):
    """sequence, cache position and cache row (page, offset) of every new token"""
    q_start, kv_len = state["q_start"].long(), state["kv_len"].long()
    t = torch.arange(state["q"].shape[0], device="cuda")
    seq = torch.searchsorted(q_start, t, right=True) - 1
    pos = kv_len[seq] - q_start[seq + 1] + t
    page = state["k_cache"].shape[1]
    return pos, state["table"][seq, pos // page].long(), pos % page


def _rotate(x, cs, rot, neox):
    """x [tokens][heads][dim] in 32 bits, cs [tokens][rot / 2][2]"""
    c, s = cs[:, None, :, 0], cs[:, None, :, 1]
    half = rot // 2
    a, b = (x[..., :half], x[..., half:rot]) if neox else (x[..., 0:rot:2], x[..., 1:rot:2])
    u, w = a * c - b * s, a * s + b * c
    y = torch.cat((u, w), -1) if neox else torch.stack((u, w), -1).flatten(-2)
    return torch.cat((y, x[..., rot:]), -1)


def _plain_append(state):
    pos, page, off = _places(state)
    kc, vc = state["k_cache"], state["v_cache"]
    cs = state["cos_sin"][pos]
    q = _rotate(state["q"].float(), cs, state["rot"], state["neox"]).to(kc.dtype)
    kc[page, off] = _rotate(state["k"].float(), cs, state["rot"], state["neox"]).to(kc.dtype)
    vc[page, off] = state["v"].float().to(vc.dtype)
    return {"q": q, "k_cache": kc, "v_cache": vc}


def _plain_attn(state):
    q, kc, vc = state["q"], state["k_cache"], state["v_cache"]
    q_start, kv_len, table = state["q_start"].long(), state["kv_len"].long(), state["table"]
    tokens, heads, dim = q.shape
    page, kv_heads = kc.shape[1], kc.shape[2]
    seqs, nq, nk, group = table.shape[0], state["max_q"], state["max_kv"], heads // kv_heads
    q_len = q_start[1:] - q_start[:-1]
    t, j = torch.arange(nq, device="cuda"), torch.arange(nk, device="cuda")
    pos = kv_len[:, None] - q_len[:, None] + t                                        # [seq][t]
    row = (q_start[:-1, None] + t).clamp(max=tokens - 1)
    see = (t < q_len[:, None])[:, :, None] & (j <= pos[:, :, None])                   # [seq][t][key]
    if state["window"]:
        see &= j > pos[:, :, None] - state["window"]
    ids = table.long().clamp(min=0)[:, j // page]                                     # [seq][key]
    k, v = (c[ids, j % page].float().permute(0, 2, 1, 3) for c in (kc, vc))           # [seq][kv head][key][dim]
    v = torch.where((j < kv_len[:, None])[:, None, :, None], v, 0.0)
    qs = q[row].float().view(seqs, nq, kv_heads, group, dim).permute(0, 2, 3, 1, 4).reshape(seqs, kv_heads, group * nq, dim)
    s = torch.matmul(qs, k.transpose(2, 3)).view(seqs, kv_heads, group, nq, nk)
    s = torch.where(see[:, None, None], s * state["scale"], -math.inf)
    m = s.amax(-1, keepdim=True)
    s = torch.exp(s - torch.where(m == -math.inf, 0.0, m))
    total = s.sum(-1, keepdim=True)
    o = torch.matmul(s.view(seqs, kv_heads, group * nq, nk), v).view(seqs, kv_heads, group, nq, dim)
    o = torch.where(total > 0, o / total, 0.0).permute(0, 3, 1, 2, 4).reshape(seqs, nq, heads, dim)
    of = torch.arange(tokens, device="cuda")
    seq = torch.searchsorted(q_start, of, right=True) - 1
    return o[seq, of - q_start[seq]].to(q.dtype)


def _plain_sample(state):
    x, u, t = state["logits"].float(), state["u"], state["temperature"][:, None]
    vocab = x.shape[1]
    at = torch.arange(vocab, device="cuda")
    top = x.amax(1, keepdim=True)
    w = torch.where(x == top, 1.0, torch.exp((x - top) * (1.0 / t)))
    ranked, order = torch.sort(x, dim=1, descending=True, stable=True)                # ties: the lowest index first
    # masses in 64 bits: which token a number falls on must not hang on the order of the additions
    wr = w.gather(1, order).double()
    k = state["top_k"].long()[:, None]
    keep = at < torch.where((k <= 0) | (k > vocab), vocab, k)
    before = (wr * keep).cumsum(1) - wr
    whole = (wr * keep).sum(1, keepdim=True)
    top_p = state["top_p"][:, None]
    keep &= (top_p >= 1.0) | (before < top_p.double() * whole) | (at == 0)
    keep &= wr >= state["min_p"][:, None]
    kept = torch.zeros_like(keep).scatter_(1, order, keep)
    mass = (w.double() * kept).cumsum(1)
    total = mass[:, -1:]
    token = (mass <= u.double()[:, None] * total).sum(1)
    greedy = t[:, 0] <= 0.0
    token = torch.where(greedy, torch.where(x == top, at, vocab).amin(1), token)
    prob = w.gather(1, token[:, None])[:, 0].double() / total[:, 0]
    return {"token": token.int(), "prob": torch.where(greedy, 1.0, prob).float()}


PLAIN = {"append": _plain_append, "attn": _plain_attn, "sample": _plain_sample}


# ------------------------------------------------------ the framework's calls

_held = {}


def _kernels():
    """the kernel set and the attention workspace that a server holds for its lifetime"""
    if not _held:
        pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "xlns-ggml-backend_b200")
        if pkg not in sys.path:
            sys.path.insert(0, pkg)
        import lnsb200
        ks = lnsb200.KernelSet(lnsb200.XLNS16, "sum32")
        _held["ks"], _held["work"] = ks, ks.paged_attn_work()
    return _held["ks"], _held["work"]


def _own_append(state):
    ks, _ = _kernels()
    kc, vc, q = state["k_cache"], state["v_cache"], state["q"]
    q_out = torch.empty(q.shape, dtype=kc.dtype, device=kc.device)
    ks.paged_append(state["k"], state["v"], kc, vc, state["table"], state["q_start"], state["kv_len"], state["max_kv"],
                    q=q, q_out=q_out, cos_sin=state["cos_sin"], neox=state["neox"])
    return {"q": q_out, "k_cache": kc, "v_cache": vc}


def _own_attn(state):
    ks, work = _kernels()
    dst = torch.empty_like(state["q"])
    ks.paged_attn(state["q"], state["k_cache"], state["v_cache"], state["table"], state["q_start"], state["kv_len"],
                  state["max_q"], state["max_kv"], dst, work, scale=state["scale"], window=state["window"])
    return dst


def _own_sample(state):
    ks, _ = _kernels()
    x = state["logits"]
    token = torch.empty(x.shape[0], dtype=torch.int32, device=x.device)
    prob = torch.empty(x.shape[0], dtype=torch.float32, device=x.device)
    ks.sample(x, state["u"], token, prob=prob, temperature=state["temperature"], top_k=state["top_k"], top_p=state["top_p"],
              min_p=state["min_p"])
    return {"token": token, "prob": prob}


OWN = {"append": _own_append, "attn": _own_attn, "sample": _own_sample}


# ------------------------------------------------------------------- the work

def work(case):
    if case["op"] == "sample":
        n = case["rows"] * case["vocab"]
        size = TYPES[case["type"]].itemsize
        # one subtraction, one product, one exponential and one addition for each logit
        return {"bytes": n * size + case["rows"] * (5 * 4 + 2 * 4), "flops": 4 * n}
    q_len, kv_len = _lengths(case)
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    size, tokens = TYPES[case["type"]].itemsize, sum(q_len)
    plan = 4 * (2 * case["seqs"] + 1 + sum(-(-n // case["page"]) for n in kv_len))
    if case["op"] == "append":
        n = tokens * (heads + 2 * kv_heads) * dim
        return {"bytes": n * (TYPES[case["src"]].itemsize + size) + tokens * case["rot"] * 4 + plan,
                "flops": tokens * (heads + kv_heads) * case["rot"] * 3}
    pairs, keys = 0, 0
    for nq, nk in zip(q_len, kv_len):
        win = case["window"] or nk
        pairs += sum(min(nk - nq + t + 1, win) for t in range(nq))
        keys += min(nk, win + nq - 1) if nq else 0
    return {"bytes": 2 * tokens * heads * dim * size + 2 * keys * kv_heads * dim * size + plan, "flops": 4 * pairs * heads * dim}


# ------------------------------------------------------------- the exact form

def exact(case, seed):
    state = prepare(case, seed)
    return {"append": _exact_append, "attn": _exact_attn, "sample": _exact_sample}[case["op"]](case, state)


def _rows(cache, state, s, n):
    """the first n rows of sequence s in a cache, [n][kv head][dim]"""
    page = cache.shape[1]
    ids = state["table"][s, : -(-n // page)].long()
    return cache[ids].flatten(0, 1)[:n].double()


def _exact_append(case, state):
    q_len, kv_len = _lengths(case)
    kc, vc = state["k_cache"].double(), state["v_cache"].double()
    rot, half, page = case["rot"], case["rot"] // 2, case["page"]
    i = torch.arange(half, device="cuda")
    lo, hi = (i, i + half) if case["neox"] else (2 * i, 2 * i + 1)
    out, at = [], 0
    for s, n in enumerate(q_len):
        pos = torch.arange(kv_len[s] - n, kv_len[s], device="cuda")
        z = torch.view_as_complex(state["cos_sin"][pos].double().contiguous())[:, None]
        turned = []
        for x in (state["q"], state["k"]):
            y = x[at : at + n].double()
            r = torch.complex(y[..., lo], y[..., hi]) * z
            y[..., lo], y[..., hi] = r.real, r.imag
            turned.append(y)
        out.append(turned[0])
        ids = state["table"][s].long()[pos // page]
        kc[ids, pos % page], vc[ids, pos % page] = turned[1], state["v"][at : at + n].double()
        at += n
    return {"q": torch.cat(out), "k_cache": kc, "v_cache": vc}


def _exact_attn(case, state):
    q_len, kv_len = _lengths(case)
    out, at, group = torch.zeros(state["q"].shape, dtype=torch.float64, device="cuda"), 0, case["heads"] // case["kv_heads"]
    for s, n in enumerate(q_len):
        if n == 0:
            continue
        nk = kv_len[s]
        k, v = _rows(state["k_cache"], state, s, nk), _rows(state["v_cache"], state, s, nk)
        pos = torch.arange(nk - n, nk, device="cuda")[:, None]
        key = torch.arange(nk, device="cuda")[None]
        hidden = (key > pos) | ((key <= pos - case["window"]) if case["window"] else False)
        for h in range(case["heads"]):
            sc = state["q"][at : at + n, h].double() @ k[:, h // group].T / math.sqrt(case["dim"])
            out[at : at + n, h] = torch.softmax(sc.masked_fill(hidden, -math.inf), -1) @ v[:, h // group]
        at += n
    return out


def _exact_sample(case, state):
    prob = []
    for r in range(case["rows"]):
        t = state["temperature"][r].item()
        if t <= 0:
            prob.append(1.0)
            continue
        p = torch.softmax(state["logits"][r].double() / t, 0)
        best, idx = torch.sort(p, descending=True, stable=True)
        k = state["top_k"][r].item()
        n = k if 0 < k < case["vocab"] else case["vocab"]
        best = best[:n]
        if state["top_p"][r].item() < 1:
            n = int(((best.cumsum(0) - best) < state["top_p"][r].item() * best.sum()).sum())
        best = best[:n]
        n = int((best >= state["min_p"][r].item() * best[0]).sum())
        kept = idx[:n].sort().values
        mass = p[kept].cumsum(0)
        token = torch.searchsorted(mass, state["u"][r].double() * mass[-1], right=True)
        prob.append((p[kept[token]] / mass[-1]).item())
    return {"token": None, "prob": torch.tensor(prob, dtype=torch.float64, device="cuda")}
