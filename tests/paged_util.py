"""A paged cache on the host, its oracle in float64, and what the operators on it may be off by."""
import math

import numpy as np
import torch

E4M3 = torch.float8_e4m3fn


def half_step(dtype) -> float:
    """A rounding's relative error at most."""
    return torch.finfo(dtype).eps / 2


def scale_byte(amax: float) -> int:
    """The least byte from 1 on with amax <= 448 * 2 ** (byte - 127)."""
    if amax == 0:
        return 1
    e = math.ceil(math.log2(amax / 448))
    while amax > 448 * 2.0 ** e:
        e += 1
    while amax <= 448 * 2.0 ** (e - 1):
        e -= 1
    return max(e + 127, 1)


def table_of(lengths, page, rng, width=None, spare=2):
    """(int32 table with pages in random order, pages): entries behind a sequence's last page are -1."""
    counts = [-(-n // page) for n in lengths]
    pages = sum(counts) + spare
    order = list(rng.permutation(pages))
    table = -np.ones((len(lengths), width or max(1, max(counts))), dtype=np.int32)
    for b, c in enumerate(counts):
        table[b, :c] = [order.pop() for _ in range(c)]
    return table, pages


class HostCache:
    """keys and values [pages, heads, page, D] as float32 that the stored type holds (8 bits: without the scale), scales as bytes."""

    def __init__(self, pages, heads, page, D, dtype, eight, fill=float("nan")):
        self.page, self.dtype, self.eight = page, dtype, eight
        self.x = [torch.full((pages, heads, page, D), fill) for _ in range(2)]
        self.scales = [torch.zeros(pages, heads, dtype=torch.uint8) for _ in range(2)] if eight else None

    def fill(self, table, lengths, rng, spread=1.0):
        """Random tokens for every sequence's keys; pages of unequal size where there are scales."""
        for which in range(2):
            for b, n in enumerate(lengths):
                for i in range(-(-n // self.page)):
                    p, m = table[b, i], min(self.page, n - i * self.page)
                    x = torch.from_numpy(rng.standard_normal((self.x[0].shape[1], m, self.x[0].shape[3])).astype(np.float32)) * spread
                    if self.eight:
                        x = x * 2.0 ** float(rng.integers(-2, 3))
                        for h in range(x.shape[0]):
                            s = scale_byte(float(x[h].abs().max()))
                            self.scales[which][p, h] = s
                            x[h] = (x[h] * 2.0 ** (127 - s)).to(E4M3).float()
                    else:
                        x = x.to(self.dtype).float()
                    self.x[which][p, :, :m] = x
        return self

    def to_device(self):
        from metalhlo_amd import kernels
        held = E4M3 if self.eight else self.dtype
        k, v = self.x
        v = v.view(v.shape[0], v.shape[1], self.page // 16, 16, v.shape[3]).transpose(3, 4)
        scales = [s.cuda() for s in self.scales] if self.eight else [None, None]
        return kernels.PagedCache(k.to(held).contiguous().cuda(), v.to(held).contiguous().cuda(), *scales)

    def dense(self, which, table, b, n):
        """float64 [heads, n, D] of sequence b; NaN where no page is."""
        heads, D = self.x[0].shape[1], self.x[0].shape[3]
        out = np.full((heads, n, D), np.nan)
        for i in range(-(-n // self.page)):
            p, m = int(table[b, i]), min(self.page, n - i * self.page)
            if not 0 <= p < self.x[0].shape[0]:
                continue
            x = self.x[which][p, :, :m].double().numpy()
            if self.eight:
                x = x * 2.0 ** (self.scales[which][p].numpy().astype(np.float64) - 127)[:, None, None]
            out[:, i * self.page:i * self.page + m] = x
        return out


def attention(q, cache, table, lengths, starts, scale=None, is_causal=True):
    """(result, bound) [T, H, D] in float64: softmax over each sequence's keys, and what a result in q's type may be off by.  One rounding of the result and one of every
    probability at half a step each; 2 ** -13 for fp32 scores and exponentials (a score is a sum of up to 128 products of unit size, off by 128 * 2 ** -24 of some tens, in the
    exponent); f16 probabilities and values below 2 ** -14 are off by 2 ** -25, which counts once a key."""
    u = half_step(q.dtype)
    qd = q.double().cpu().numpy()
    T, H, D = qd.shape
    KV = cache.x[0].shape[1]
    scale = D ** -0.5 if scale is None else scale
    out, bound = np.full((T, H, D), np.nan), np.zeros((T, H, D))
    for b, n in enumerate(lengths):
        k, v = (cache.dense(w, table, b, n) for w in range(2))
        m = starts[b + 1] - starts[b]
        for i in range(m):
            seen = max(0, n - m + i + 1) if is_causal else n
            there = ~np.isnan(k[0, :seen]).any(1)
            for h in range(H):
                kk, vv = k[h // (H // KV), :seen][there], v[h // (H // KV), :seen][there]
                row = starts[b] + i
                if not len(kk):
                    out[row, h] = 0
                    continue
                s = scale * (kk @ qd[row, h])
                p = np.exp(s - s.max())
                p /= p.sum()
                out[row, h] = p @ vv
                size = p @ np.abs(vv)
                bound[row, h] = 1.01 * (u * np.abs(out[row, h]) + (u + 2.0 ** -13) * size)
                if q.dtype == torch.float16:
                    bound[row, h] += 2.0 ** -25 * (1 + len(kk) * np.abs(vv).max()) + 2.0 ** -25
                bound[row, h] += 1e-30
    return out, bound


def assert_within(got, want, bound, what=""):
    g = got.detach().double().cpu().numpy()
    rows = ~np.isnan(want)
    off = np.abs(g - want)
    bad = rows & ~(off <= bound)
    if bad.any():
        i = np.unravel_index(np.argmax(np.where(bad, off / bound, 0)), g.shape)
        raise AssertionError(f"{what}: {bad.sum()} of {rows.sum()} too far off; worst at {i}: got {g[i]!r}, expected {want[i]!r}, bound {bound[i]:.3g}")


def attention_at_once(q, cache, table, lengths, starts, scale=None, is_causal=True):
    """What `attention` returns, a sequence's rows of a head at a time (every key on a page)."""
    u = half_step(q.dtype)
    qd = q.double().cpu().numpy()
    T, H, D = qd.shape
    KV = cache.x[0].shape[1]
    scale = D ** -0.5 if scale is None else scale
    out, bound = np.full((T, H, D), np.nan), np.zeros((T, H, D))
    for b, n in enumerate(lengths):
        k, v = (cache.dense(w, table, b, n) for w in range(2))
        m = starts[b + 1] - starts[b]
        rows = slice(starts[b], starts[b + 1])
        hidden = np.arange(n)[None] > (np.arange(n - m, n) if is_causal else np.full(m, n))[:, None]
        for h in range(H):
            s = np.where(hidden, -np.inf, scale * (qd[rows, h] @ k[h // (H // KV)].T))
            p = np.exp(s - s.max(1, keepdims=True))
            p /= p.sum(1, keepdims=True)
            vv = v[h // (H // KV)]
            out[rows, h] = p @ vv
            bound[rows, h] = 1.01 * (u * np.abs(out[rows, h]) + (u + 2.0 ** -13) * (p @ np.abs(vv))) + 1e-30
            if q.dtype == torch.float16:
                bound[rows, h] += 2.0 ** -25 * (2 + n * np.abs(vv).max())
    return out, bound
