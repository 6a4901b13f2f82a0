"""Plain forms of the 16-bit cache's operators for the tests, a sequence and a head
at a time: attention over pages and the gathered weights in 64 bits, eviction on whole
rows.  On the CPU or the GPU, without the library."""
import math

import torch

from tests._serve_bounds import U


def starts_of(lens):
    s = [0]
    for n in lens:
        s.append(s[-1] + n)
    return s


class Cache:
    """Pools with the pages of the sequences at random places, whose rows behind the keys, and
    pages that belong to nobody, hold NaN."""

    def __init__(self, keys, heads, D, dtype, page_size, seed=0, device="cuda", spare=3, wide=0):
        gen = torch.Generator(device=device).manual_seed(seed)
        need = [-(-n // page_size) for n in keys]
        pool = sum(need) + spare
        order = torch.randperm(pool, generator=torch.Generator().manual_seed(seed)).tolist()
        cols = max([1, *need]) + wide
        rows, at = [], 0
        for n in need:
            rows.append(order[at : at + n] + [order[-1]] * (cols - n))
            at += n
        self.keys, self.page_size, self.device = list(keys), page_size, device
        self.table = torch.tensor(rows, dtype=torch.int32, device=device)
        self.lens = torch.tensor(keys, dtype=torch.int32, device=device)
        shape = (pool, heads, page_size, D)
        self.K, self.V = (torch.full(shape, math.nan, dtype=dtype, device=device) for _ in range(2))
        self.weights = torch.rand(shape[:3], generator=gen, device=device)
        for b, n in enumerate(keys):
            page, row = self.slots(b, range(n))
            for x in (self.K, self.V):
                x[page, :, row] = torch.randn((n, heads, D), generator=gen, dtype=dtype, device=device)

    def slots(self, b, places):
        at = torch.tensor(list(places), dtype=torch.long, device=self.device)
        return self.table[b][at // self.page_size].long(), at % self.page_size

    def valid(self, b, n):
        page, _ = self.slots(b, range(n))
        return (page >= 0) & (page < self.K.shape[0])

    def rows(self, b, n, *pools):
        """[H, n, ...] of every pool, zeros on invalid pages."""
        page, row = self.slots(b, range(n))
        ok = self.valid(b, n)
        out = []
        for x in pools:
            y = x[torch.where(ok, page, 0), :, row].double().transpose(0, 1).contiguous()
            y[:, ~ok] = 0
            out.append(y)
        return out

    def clone(self):
        c = object.__new__(Cache)
        c.__dict__ = {k: v.clone() if isinstance(v, torch.Tensor) else v for k, v in self.__dict__.items()}
        return c


def seen_by(cache, b, q, n, causal):
    """[q, n]: whether query i sees the key at place j."""
    j = torch.arange(n, device=cache.device)
    i = torch.arange(q, device=cache.device)[:, None]
    seen = (j <= i + (n - q)) if causal else torch.ones((q, n), dtype=torch.bool, device=cache.device)
    return seen & cache.valid(b, n)


def attention(q, k, v, seen, dtype):
    """_serve_bounds.attention for any mask: O, LSE and the bound of O before its rounding."""
    H_q, n, D = q.shape
    m, ratio = k.shape[1], H_q // k.shape[0]
    out, lse, off = torch.zeros_like(q), q.new_full((H_q, n), -math.inf), torch.zeros_like(q)
    if m == 0 or n == 0:
        return out, lse, off
    half = torch.finfo(dtype).eps / 2
    some = seen.any(1)[:, None]
    for h in range(H_q):
        kh, vh = k[h // ratio], v[h // ratio]
        s = (q[h] @ kh.t().contiguous() / math.sqrt(D)).masked_fill(~seen, -math.inf)
        lse[h] = torch.logsumexp(s, 1)
        w = torch.exp(s - torch.where(some, lse[h][:, None], 0.0))
        out[h] = w @ vh
        size = q[h].norm(dim=1, keepdim=True) * kh.norm(dim=1).max() / math.sqrt(D)
        fp32 = 2 * U * ((D + 8) * size + 8) + U * (m / 16 + m / 32 + 64)
        off[h] = 8 * half * torch.sqrt((w * w) @ (vh * vh)) + fp32 * (w @ vh.abs())
        if dtype == torch.float16:
            off[h] += 8 * 2.0 ** -25 * torch.sqrt(seen.double() @ (vh * vh))
    return out, lse, off


def gathered(q, k, lse, seen):
    """Weights [H_kv, m] that keys k [H_kv, m, D] get from q [H_q, n, D], and how far 32 bits
    may be from them: a weight's exponent is a score (D products summed in 32 bits), its
    scale, and the difference to the log-sum-exp, each rounded relative to its size, u =
    2^-24; the exponential is off by 2 u; n H_q / H_kv terms are summed."""
    H_q, n, D = q.shape
    H, m = k.shape[:2]
    ratio = H_q // H
    sums, off = torch.zeros_like(k[..., 0]), torch.zeros_like(k[..., 0])
    for h in range(H_q):
        s = q[h] @ k[h // ratio].t().contiguous() / math.sqrt(D)
        e = torch.where(torch.isfinite(lse[h]), lse[h], 0.0)[:, None]
        some = seen & torch.isfinite(lse[h])[:, None]
        w = torch.exp(s - e).masked_fill(~some, 0.0)
        size = q[h].norm(dim=1, keepdim=True) * k[h // ratio].norm(dim=1) / math.sqrt(D)
        rel = U * ((D + 8) * size + 4 * s.abs() + 4 * e.abs() + 8)
        sums[h // ratio] += w.sum(0)
        off[h // ratio] += (w * rel).sum(0)
    return sums, off + U * (n * ratio + 8) * sums


def evict(cache, budgets, recent):
    """Moves the rows of `cache` itself; the new key counts."""
    kept = []
    for b, n in enumerate(cache.keys):
        m = min(n, max(0, budgets[b]))
        if m == n or not bool(cache.valid(b, n).all()):
            kept.append(n)
            continue
        kept.append(m)
        r = min(recent, m)
        k, old = m - r, n - r
        page, row = cache.slots(b, range(n))
        for h in range(cache.K.shape[1]):
            w = cache.weights[page[:old], h, row[:old]].cpu().tolist()
            best = sorted(range(old), key=lambda i: (0, 0.0, i) if math.isnan(w[i]) else (1, -w[i], i))[:k]
            free = sorted(set(range(k)) - set(best))
            to = free + list(range(k, m))
            at = sorted(i for i in best if i >= k) + list(range(old, n))
            assert len(to) == len(at)
            to, at = (torch.tensor(x, dtype=torch.long, device=cache.device) for x in (to, at))
            for x in (cache.K, cache.V, cache.weights):
                x[page[to], h, row[to]] = x[page[at], h, row[at]]
    return kept
