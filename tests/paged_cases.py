"""Pages with known values for the tests of the paged cache, and what the oracle says of them."""
import numpy as np
import torch

from oracle import paged as O

DEV = "cuda"


def kernels():
    from flashgrpo_amd import kernels

    return kernels


class Held:
    """Pages of random rows on the host (float64 values, codes, scales) and on the device."""

    def __init__(self, rows, width, size, heads, d, fmt, seed, spare=2, spread=1.0, device=DEV):
        rng = np.random.default_rng(seed)
        n = rows * width + spare
        self.size, self.heads, self.d, self.fmt, self.pages_n = size, heads, d, fmt, n
        self.table = rng.permutation(n)[:rows * width].reshape(rows, width).astype(np.int32)
        channel = np.exp(0.3 * rng.standard_normal((1, heads, 1, d)))
        draw = lambda c: torch.from_numpy(spread * rng.standard_normal((n, heads, size, d)) * c).to(torch.bfloat16)
        self.raw = [draw(channel), draw(1.0)]
        self.codes, self.scales, self.values = [None, None], [None, None], [None, None]
        for i in range(2):
            self.refresh(i)
        self.device = device
        self.upload()

    def refresh(self, i):
        x = self.raw[i].double().numpy()
        if self.fmt == "bf16":
            self.values[i] = x
        else:
            self.codes[i], self.scales[i] = O.quantize(x)
            self.values[i] = O.values(self.codes[i], self.scales[i])

    def set_rows(self, i, row, tokens, x):
        """Rows x [heads, tokens, d] (or a number) as tokens of a cache row, in K (i = 0) or V (1)."""
        for j, t in enumerate(tokens):
            p = O.page_of(self.table[row], t, self.size, self.pages_n)
            self.raw[i][p, :, t % self.size] = x if isinstance(x, float) else torch.as_tensor(x[:, j])
        self.refresh(i)

    def upload(self):
        dev = self.device
        if self.fmt == "bf16":
            self.k, self.v = (x.to(dev) for x in self.raw)
            self.ks = self.vs = None
        else:
            self.k, self.v = (torch.from_numpy(c).to(dev).view(torch.float8_e4m3fn) for c in self.codes)
            self.ks, self.vs = (torch.from_numpy(np.ascontiguousarray(s)).to(dev) for s in self.scales)
        self.device_table = torch.from_numpy(self.table).to(dev)
        return self

    def pages(self):
        return kernels().KVPages(self.k, self.v, self.ks, self.vs, self.device_table)

    def now(self, i):
        """The values that the device's pages hold, float64."""
        t = (self.k, self.v)[i]
        if self.fmt == "bf16":
            return t.double().cpu().numpy()
        return O.values(t.view(torch.uint8).cpu().numpy(), (self.ks, self.vs)[i].cpu().numpy())


def i32(x):
    return torch.as_tensor(np.asarray(x), dtype=torch.int32).to(DEV)


def masks(words):
    """Ancestor words (Python ints) as an int64 tensor."""
    a = np.array([[w & (2 ** 64 - 1) for w in row] for row in words], dtype=np.uint64).view(np.int64)
    return torch.from_numpy(a).to(DEV)


def tree_words(n, seed):
    rng = np.random.default_rng(seed)
    out = [1]
    for i in range(1, n):
        out.append(out[rng.integers(max(0, i - 6), i)] | 1 << i)
    return out


def queries(b, n, hq, d, seed):
    return torch.from_numpy(np.random.default_rng(seed).standard_normal((b, n, hq, d))).to(torch.bfloat16)


def attention_oracle(held, q, committed, fresh, words, scale, row=None, values=None):
    """Per sequence (out, bound) of the oracle; words: per sequence ancestor words, or None (chain)."""
    got = []
    for b in range(q.shape[0]):
        table = held.table[b if row is None else row[b]]
        tokens = np.arange(min(committed[b] + fresh[b], held.table.shape[1] * held.size))
        k, there = O.rows_at((values or held.values)[0], table, tokens)
        v, _ = O.rows_at((values or held.values)[1], table, tokens)
        new = len(tokens) - committed[b]
        o, e = O.attention(q[b].double().numpy(), k, v, there, committed[b], new, None if words is None else words[b], scale)
        got.append((o, e))
    return got


def close(out, want, fresh):
    """Asserts the first fresh[b] nodes of out [B, N, Hq, d] within the oracle's bound and half a bf16 step."""
    out = out.double().cpu().numpy()
    for b, (o, e) in enumerate(want):
        x = out[b, :fresh[b]]
        assert x.shape == o.shape
        assert (np.isnan(x) == np.isnan(o)).all(), f"sequence {b}: NaN elsewhere"
        whole = np.isfinite(o)
        assert (x[np.isinf(o)] == o[np.isinf(o)]).all()
        off, most = np.abs(x - o)[whole], (e + (np.abs(o) + e) * 2.0 ** -8 + 2.0 ** -120)[whole]
        assert (off <= most).all(), f"sequence {b}: {np.max(off / most)} of the bound"
