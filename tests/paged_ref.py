"""The operators over many sequences in 64 bits, from their definitions, and the host images of
their inputs (numpy only): a paged cache with any strides, 16-bit types as bit patterns."""
import numpy as np

import mcpm

F32, F16, BF16 = mcpm.TYPE_F32, mcpm.TYPE_F16, mcpm.TYPE_BF16
NAME = {F32: "f32", F16: "f16", BF16: "bf16"}
# half a step of a rounding to the type, relative to the value
HALF = {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}


def store(x, t):
    """x rounded to type t, as the bytes that memory holds."""
    x = np.asarray(x, np.float32)
    if t == F32:
        return x.copy()
    if t == F16:
        return x.astype(np.float16)
    u = np.ascontiguousarray(x).view(np.uint32)
    r = ((u + 0x7fff + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7fc0), r)


def load(b, t):
    """The values, in 64 bits, of what memory holds."""
    if t == BF16:
        return (b.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    return b.astype(np.float64)


class Cache:
    """A pool of pages on the host: k, v as flat images under any strides, weight."""

    def __init__(self, t, n_pages, page, kvh, hd, order="phd", pad=0, weight=False, rng=None, fill=None):
        self.t, self.n_pages, self.page, self.kvh, self.hd = t, n_pages, page, kvh, hd
        step = 4 if t == F32 else 8
        row = hd + (step if pad else 0)
        if order == "phd":  # page, position, head
            self.strides = (page * kvh * row + pad * step, kvh * row, row)
        else:  # page, head, position
            self.strides = (page * kvh * row + pad * step, row, page * row)
        n = n_pages * self.strides[0]
        rng = rng or np.random.default_rng(0)
        if fill is None:
            self.k, self.v = (store(rng.standard_normal(n), t) for _ in range(2))
        else:
            self.k, self.v = (store(np.full(n, fill), t) for _ in range(2))
        self.weight = np.zeros((n_pages, kvh, page), np.float32) if weight else None

    def index(self, page, o, h):
        """Flat indexes of a row's elements."""
        return page * self.strides[0] + o * self.strides[1] + h * self.strides[2] + np.arange(self.hd)

    def rows(self, which, pages, n, h):
        """[n, hd] values of kv head h at positions 0..n-1; rows of pages outside the pool are NaN."""
        out = np.full((n, self.hd), np.nan)
        for j in range(n):
            p = pages[j // self.page]
            if 0 <= p < self.n_pages:
                out[j] = load(getattr(self, which)[self.index(p, j % self.page, h)], self.t)
        return out


def spans(lens, news):
    at = [0]
    for n in news:
        at.append(at[-1] + n)
    return at


def seen_mask(pos, n, b, rules, valid):
    """Which of positions 0..n-1 the row at pos sees."""
    j = np.arange(n)
    m = (j <= pos) | (j < (rules["prefix"][b] if rules.get("prefix") is not None else 0))
    if rules.get("window"):
        m &= pos - j < rules["window"]
    if rules.get("docs") is not None:
        d = rules["docs"][b]
        m &= (d[:n] == d[pos]) & (d[pos] >= 0)
    return m & valid


def attention(cache, tables, lens, news, q, io, H, rules, starts=None):
    """(out, bound, weight added): rows [n][H][hd] in 64 bits, how far an output may be off, and the shares
    per (page, kv head, position).

    The bound: a 32-bit sum of n products is off by at most n u sum |a b| in any order, with u = 2^-23 where an
    accumulator may cut instead of rounding.  So a score is off by at most
    e = (hd + 16) u scale sum|q k| + 8 u |s| (the cap's and bias's own steps), a share p by a factor
    exp(2 e) (1 + (n + 16) u), the output by that times sum p |v|, one rounding to its type more, and, where the
    rows are 16-bit, one rounding of each p to that type."""
    u = 2.0 ** -23
    hd, G = cache.hd, H // cache.kvh
    scale = rules.get("scale") or 1.0 / np.sqrt(hd)
    at = spans(lens, news) if starts is None else starts
    out = np.zeros((q.shape[0], H, hd))
    bound = np.zeros_like(out)
    weight = np.zeros((cache.n_pages, cache.kvh, cache.page))
    wbound = np.zeros_like(weight)
    qv = load(q, io).reshape(q.shape[0], H, hd)
    for b, (n, new) in enumerate(zip(lens, news)):
        pages = tables[b]
        valid = np.array([0 <= pages[j // cache.page] < cache.n_pages for j in range(n)], bool)
        for kh in range(cache.kvh):
            k, v = cache.rows("k", pages, n, kh), cache.rows("v", pages, n, kh)
            for t in range(new):
                pos, row = n - new + t, at[b] + t
                if pos < 0:
                    continue
                m = seen_mask(pos, n, b, rules, valid)
                idx = np.nonzero(m)[0]
                if idx.size == 0:
                    continue
                for h in range(kh * G, kh * G + G):
                    qr = qv[row, h]
                    s = k[idx] @ qr * scale
                    e = (hd + 16) * u * scale * (np.abs(k[idx]) @ np.abs(qr))
                    if rules.get("softcap"):
                        s = rules["softcap"] * np.tanh(s / rules["softcap"])
                    if rules.get("slopes") is not None:
                        s = s - float(rules["slopes"][h]) * np.abs(pos - idx)
                        e = e + 4 * u * float(rules["slopes"][h]) * np.abs(pos - idx)
                    e = (e + 8 * u * np.abs(s)).max()
                    p = np.exp(s - s.max())
                    p /= p.sum()
                    f = np.exp(2 * e) * (1 + (idx.size + 16) * u) - 1
                    o = p @ v[idx]
                    a = p @ np.abs(v[idx])
                    out[row, h] = o
                    # 2^-126: a share too small for a normal float may count as none
                    bound[row, h] = (f + (HALF[io] * 1.01 if io != F32 else 0)) * a + 1.01 * HALF[io] * (np.abs(o) + f * a) + 2.0 ** -24 * 1e-6
                    where = (np.asarray(pages)[idx // cache.page], kh, idx % cache.page)
                    np.add.at(weight, where, p)
                    np.add.at(wbound, where, p * (f + (G * new + 4) * u) + 1e-12)
    return out, bound, weight, wbound


def rope(x, pos, base):
    """x [heads, hd] rotated by pos in 64 bits."""
    hd = x.shape[-1]
    a = pos * float(base) ** (-np.arange(0, hd, 2) / hd)
    c, s = np.cos(a), np.sin(a)
    y = np.empty(x.shape)
    y[:, 0::2] = x[:, 0::2] * c - x[:, 1::2] * s
    y[:, 1::2] = x[:, 0::2] * s + x[:, 1::2] * c
    return y


def evict_kept(weight, n, budget, first, recent):
    """Positions kept of one head's n weights."""
    if n <= budget:
        return np.arange(n)
    mid = np.arange(first, n - recent)
    w = np.where(np.isnan(weight[mid]), -np.inf, weight[mid].astype(np.float64))
    nan = np.isnan(weight[mid])
    order = np.lexsort((mid, nan, -w))  # weight falling, NaN after -inf, position rising
    top = mid[order[:budget - first - recent]]
    return np.sort(np.concatenate([np.arange(first), top, np.arange(n - recent, n)]))


def logits(x, hist, rep, pres, freq, bias, allowed):
    """One row in 64 bits; hist: ids; bias: (id, value) pairs, the last of an id counts; allowed: bool or None."""
    y = x.astype(np.float64)
    n = y.size
    ids, cnt = np.unique([i for i in hist if 0 <= i < n], return_counts=True)
    ids = ids.astype(int)
    l = y[ids]
    with np.errstate(invalid="ignore"):
        y[ids] = np.where(l > 0, l / rep, l * rep) - (freq * cnt + pres)
    for i, v in {i: v for i, v in bias if 0 <= i < n}.items():
        y[i] += v
    if allowed is not None:
        y[~allowed] = -np.inf
    return y
