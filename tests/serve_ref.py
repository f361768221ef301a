"""Plain 64-bit forms of the paged serving operators (torch, any device) and
the caches they are tried on."""
import math

import torch

# half the distance between neighbours, relative: the largest error of one rounding
UNIT = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


class Paged:
    """A paged cache with scattered pages: every row that no sequence owns, and every page that
    none uses, holds `junk`; table entries that no row needs are -1."""

    def __init__(self, q_len, kv_len, n_head_kv, head_dim, page_size, dtype, seed=0, junk=float("nan"), device="cuda",
                 pad=0, head_major=False):
        g = torch.Generator().manual_seed(seed)
        self.q_len, self.kv, self.page = q_len, kv_len, page_size
        pages = [-(-n // page_size) for n in kv_len]
        n_pages = sum(pages) + 2
        ids = torch.randperm(n_pages, generator=g)
        table = torch.full((len(kv_len), max(pages + [1]) + 1), -1, dtype=torch.int32)
        at = 0
        for s, n in enumerate(pages):
            table[s, :n] = ids[at:at + n].to(torch.int32)
            at += n
        shape = (n_pages, page_size, n_head_kv, head_dim + pad)
        if head_major:
            shape = (n_pages, n_head_kv, page_size, head_dim + pad)
        self.caches = []
        for _ in range(2):
            c = torch.randn(shape, generator=g)
            view = c.permute(0, 2, 1, 3) if head_major else c
            owned = torch.zeros(n_pages, page_size, dtype=torch.bool)
            for s, n in enumerate(kv_len):
                for i in range(n):
                    owned[table[s, i // page_size], i % page_size] = True
            view[~owned] = junk
            c = c.to(dtype).to(device)
            self.caches.append((c.permute(0, 2, 1, 3) if head_major else c)[..., :head_dim])
        self.k, self.v = self.caches
        self.host_table = table
        self.table = table.to(device)
        start = [0]
        for n in q_len:
            start.append(start[-1] + n)
        self.start = start
        self.q_start = torch.tensor(start, dtype=torch.int32, device=device)
        self.kv_len = torch.tensor(kv_len, dtype=torch.int32, device=device)
        self.max_q, self.max_kv = max(q_len + [1]), max(kv_len + [1])
        self.tokens = start[-1]

    def rows(self, cache, s):
        """the rows that sequence s owns, [kv_len][n_head_kv][head_dim], in 64 bits"""
        n = self.kv[s]
        i = torch.arange(n)
        ids = self.host_table[s].long()[i // self.page]
        return cache[ids.to(cache.device), (i % self.page).to(cache.device)].double()


def attention(P, q, scale, window=0):
    """(outputs, sum of p |v|, largest |v|) of every token in 64 bits, [tokens][heads][dim]"""
    group = q.shape[1] // P.k.shape[2]
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    mag = torch.zeros_like(out)
    for s, n in enumerate(P.q_len):
        kv, a = P.kv[s], P.start[s]
        if n == 0 or kv == 0:
            continue
        k, v = P.rows(P.k, s), P.rows(P.v, s)
        lo = max(0, kv - n - window + 1) if window else 0
        pos = torch.arange(kv - n, kv, device=q.device)[:, None]
        key = torch.arange(lo, kv, device=q.device)[None]
        see = key <= pos
        if window:
            see &= key > pos - window
        for h in range(q.shape[1]):
            x = q[a:a + n, h].double() @ k[lo:, h // group].T * scale
            x = torch.where(see, x, torch.full_like(x, -math.inf))
            m = x.amax(1, keepdim=True)
            p = torch.exp(x - torch.where(m == -math.inf, torch.zeros_like(m), m))
            total = p.sum(1, keepdim=True)
            total = torch.where(total > 0, total, torch.ones_like(total))
            out[a:a + n, h] = p @ v[lo:, h // group] / total
            mag[a:a + n, h] = p @ v[lo:, h // group].abs() / total
    return out, mag


def attention_bound(dtype, out, mag, n_keys, v_max):
    """The kernels round each weight p to the type (u, and in F16 2^-25 absolute where p is subnormal against a
    largest p of 1 at least), once in the numerator and once in the sum, and the output once (u); the score of
    32-bit products and exp2 moves p by less than 2^-12 relative at these sizes (|q.k| scale <= 2^6, 2^-24 a step,
    and 2^-22 for exp2)."""
    u = UNIT[dtype]
    sub = n_keys * 2.0 ** -25 * v_max if dtype == torch.float16 else 0.0
    return (2 * u + 2.0 ** -12) * mag * 1.01 + u * out.abs() * 1.01 + sub + 2.0 ** -24


def rotate(x, cs, neox):
    """(rotated, magnitude) of x [tokens][heads][dim] by cs [tokens][n_dims / 2][2], in 64 bits"""
    x, c, s = x.double(), cs[:, None, :, 0].double(), cs[:, None, :, 1].double()
    half = cs.shape[1]
    i = torch.arange(half, device=x.device)
    lo, hi = (i, i + half) if neox else (2 * i, 2 * i + 1)
    y, mag = x.clone(), torch.zeros_like(x)
    y[..., lo] = x[..., lo] * c - x[..., hi] * s
    y[..., hi] = x[..., lo] * s + x[..., hi] * c
    mag[..., lo] = (x[..., lo] * c).abs() + (x[..., hi] * s).abs()
    mag[..., hi] = (x[..., lo] * s).abs() + (x[..., hi] * c).abs()
    return y, mag


def kept_tokens(x, t, k, p, m):
    """(kept indices, their weights), both in falling order, of one row of logits in 64 bits"""
    x = torch.where(torch.isnan(x), torch.full_like(x, -math.inf), x).double().cpu()
    top = x.max()
    w = torch.where(x == top, torch.ones_like(x), torch.exp((x - top) / t))
    ws, order = torch.sort(x, descending=True, stable=True)
    ws = w[order]
    n = k if 0 < k < x.numel() else x.numel()
    ws, order = ws[:n], order[:n]
    if p < 1:
        before = ws.cumsum(0) - ws
        n = max(1, int((before < p * ws.sum()).sum()))
        ws, order = ws[:n], order[:n]
    ok = ws >= min(m, 1.0) if m > 0 else torch.ones_like(ws, dtype=torch.bool)
    return order[ok], ws[ok]
