"""The paged operators as programs use them: one after the other over a growing cache, in captured graphs, on other streams, and
what their wrappers refuse."""
import numpy as np
import pytest
import torch

from oracle import paged as O
from paged_cases import DEV, Held, attention_oracle, close, i32, kernels, masks, queries, tree_words

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


def inv_freq(d):
    return (1.0 / 1.0e6 ** (torch.arange(0, d, 2).float() / d)).to(DEV)


def rows_of(n, width, seed):
    return torch.from_numpy(np.random.default_rng(seed).standard_normal((n, width))).to(torch.bfloat16)


class Round:
    """A verify round's calls over fixed buffers: write, attention, accepted path, read back."""

    def __init__(self, held, n, hq, depth, seed, chain=False):
        self.held, self.n, self.hq, self.depth = held, n, hq, depth
        b, h, d = held.table.shape[0], held.heads, held.d
        rng = np.random.default_rng(seed)
        self.words = None if chain else [tree_words(n, seed + i) for i in range(b)]
        self.nodes = np.stack([np.concatenate([[0], np.sort(rng.choice(np.arange(1, n), depth - 1, replace=False))]) for _ in range(b)])
        self.lens = rng.integers(1, depth + 1, b)
        self.qkv = rows_of(b * n, (hq + 2 * h) * d, seed)
        self.q = torch.zeros(b, n, hq, d, dtype=torch.bfloat16, device=DEV)
        self.dev = dict(qkv=self.qkv.to(DEV), off=i32(np.arange(n)), f=inv_freq(d), anc=None if chain else masks(self.words),
                        nodes=i32(self.nodes), lens=i32(self.lens), err=i32([0]))
        self.pages = held.pages()

    def __call__(self, seq):
        k, h, d, v = kernels(), self.held.heads, self.held.d, self.dev
        kw = dict(num_nodes=self.n, q_heads=self.hq, kv_heads=h, head_dim=d, seq_len=seq)
        k.rope_kv_write_paged(v["qkv"], self.pages, batch=seq.numel(), pos_offset=v["off"], inv_freq=v["f"], q_out=self.q,
                              err_flag=v["err"], **kw)
        out = k.paged_attention(self.q, self.pages, anc=v["anc"], **kw)
        k.kv_path_gather_paged(self.pages, seq_len=seq, acc_nodes=v["nodes"], acc_len=v["lens"], tree_nodes=self.n, err_flag=v["err"])
        return (out, *k.kv_read_paged(self.pages, start=seq, count=self.depth))

    def oracle(self, committed):
        """Updates held's values on the host; the attention's (out, bound) and the accepted rows."""
        x, b, h, d = self.held, len(committed), self.held.heads, self.held.d
        rows = self.qkv.double().numpy().reshape(b, self.n, self.hq + 2 * h, d)
        q = self.q.cpu()  # (tested by itself)
        for i in range(b):
            pos = committed[i] + np.arange(self.n)
            kr = O.rotate(rows[i, :, self.hq:self.hq + h], pos, inv_freq(d).cpu().numpy()).astype(np.float32)
            for w, y in enumerate((kr, rows[i, :, self.hq + h:])):
                vals = O.values(*O.quantize(y))
                for j in range(self.n):
                    t = committed[i] + j
                    x.values[w][O.page_of(x.table[i], t, x.size, x.pages_n), :, t % x.size] = vals[j]
        want = attention_oracle(x, q, committed, [self.n] * b, self.words, d ** -0.5)
        for i in range(b):
            for w in range(2):
                held, _ = O.rows_at(x.values[w], x.table[i], committed[i] + self.nodes[i])
                for j in range(self.lens[i]):
                    t = committed[i] + j
                    x.values[w][O.page_of(x.table[i], t, x.size, x.pages_n), :, t % x.size] = held[:, j]
        rows = [np.stack([O.rows_at(x.values[w], x.table[i], committed[i] + np.arange(self.depth))[0] for i in range(b)]) for w in range(2)]
        return want, rows


@pytest.mark.parametrize("size", [16, 64])
@pytest.mark.parametrize("hq,h,d,n", [(6, 2, 128, 13), (28, 4, 128, 29), (4, 2, 64, 7), (2, 1, 128, 3)])
def test_rounds_one_after_the_other(size, hq, h, d, n):
    """Three verify rounds, each with the accepted tokens of the one before, against the oracle."""
    b, depth = 3, min(4, n)
    held = Held(b, -(-220 // size), size, h, d, "e4m3", seed=n)
    committed = [0, 37, 150]
    for step in range(3):
        r = Round(held, n, hq, depth, 10 * n + step)
        out, k, v = r(i32(committed))
        want, rows = r.oracle(committed)
        close(out, want, [n] * b)
        assert (k.double().cpu().numpy() == rows[0]).all() and (v.double().cpu().numpy() == rows[1]).all()
        assert r.dev["err"].item() == 0
        committed = [c + int(l) for c, l in zip(committed, r.lens)]


@pytest.mark.parametrize("hq,n,width", [(2, 1, 60), (12, 13, 60), (28, 29, 10)])
def test_captured_and_replayed(hq, n, width):
    """Two graphs that both use workspaces, replayed in turn between eager calls: each replay gives the eager result."""
    held = [Held(2, width, 64, 2 if hq < 28 else 4, 128, "e4m3", seed=s) for s in (1, 2)]
    seqs = [i32([64 * width - 100, 200]), i32([64 * width - 300, 33])]
    rounds = [Round(h, n, hq, min(3, n), 5 + i) for i, h in enumerate(held)]
    eager = [[t.clone() for t in r(s)] for r, s in zip(rounds, seqs)]
    graphs, outs = [], []
    for r, s in zip(rounds, seqs):
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(r(s))
        graphs.append(g)
    other = torch.cuda.Stream()
    for turn in range(4):
        for o in outs:
            for t in o:
                t.fill_(float("nan"))
        if turn % 2:  # at once, on two streams
            other.wait_stream(torch.cuda.current_stream())
            graphs[0].replay()
            with torch.cuda.stream(other):
                graphs[1].replay()
            torch.cuda.current_stream().wait_stream(other)
        else:
            graphs[0].replay()
            rounds[1](seqs[1])
            graphs[1].replay()
        torch.cuda.synchronize()
        for want, got in zip(eager, outs):
            for a, b in zip(want, got):
                assert torch.equal(a, b)


def test_on_another_stream():
    held = Held(2, 50, 64, 2, 128, "e4m3", seed=3)
    r, seq = Round(held, 5, 4, 3, 1), i32([3000, 100])
    want = [t.clone() for t in r(seq)]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = r(seq)
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))


@pytest.mark.parametrize("hq,n", [(2, 1), (8, 4), (12, 13), (28, 29)])
def test_same_results_whatever_else_the_table_holds(hq, n):
    """A row's result depends on its tokens alone: other rows, other pages and repeated cache rows leave its bits."""
    held = Held(4, 8, 64, 2 if hq < 28 else 4, 128, "e4m3", seed=4)
    q = queries(2, n, hq, 128, 1).to(DEV)
    words = masks([tree_words(n, 1)] * 2)
    kw = dict(anc=words, num_nodes=n, q_heads=hq, kv_heads=held.heads, head_dim=128)
    a = kernels().paged_attention(q, held.pages(), seq_len=i32([333, 40]), row_map=i32([2, 1]), **kw)
    twice = kernels().paged_attention(q[:1].repeat(2, 1, 1, 1), held.pages(), seq_len=i32([333, 333]), row_map=i32([2, 2]), **kw)
    assert torch.equal(a[0], twice[0]) and torch.equal(a[0], twice[1])
    held.table[[0, 3]] = -1
    held.upload()
    b = kernels().paged_attention(q, held.pages(), seq_len=i32([333, 40]), row_map=i32([2, 1]), **kw)
    assert torch.equal(a, b)


def test_lengths_that_make_no_sense_see_nothing():
    held = Held(3, 2, 64, 2, 128, "e4m3", seed=5)
    q = queries(3, 2, 4, 128, 1).to(DEV)
    kw = dict(anc=None, num_nodes=2, q_heads=4, kv_heads=2, head_dim=128)
    out = kernels().paged_attention(q, held.pages(), seq_len=i32([-1, 50, 2 ** 31 - 1]), row_map=i32([0, 3, 1]), **kw)
    assert (out[:2] == 0).all() and torch.isfinite(out[2].float()).all()
    full = kernels().paged_attention(q, held.pages(), seq_len=i32([128, 128, 128]), row_map=i32([1, 1, 1]), **kw)
    assert torch.equal(full[2], out[2])  # what lies behind the table's pages is not there
    new = torch.full_like(q, 9.0)
    kernels().paged_attention(q, held.pages(), seq_len=i32([5, 5, 5]), out=new, new_len=i32([-3, 99, 1]), **kw)
    assert (new[0] == 9).all() and (new[1] != 9).any() and (new[2, 1] == 9).all()


def test_nothing_to_do():
    held = Held(1, 1, 16, 2, 64, "e4m3", seed=6)
    p, e = held.pages(), i32([])
    q = torch.empty(0, 3, 4, 64, dtype=torch.bfloat16, device=DEV)
    assert kernels().paged_attention(q, p, seq_len=e, anc=None, num_nodes=3, q_heads=4, kv_heads=2, head_dim=64).shape == q.shape
    kernels().rope_kv_write_paged(torch.empty(0, 8 * 64, dtype=torch.bfloat16, device=DEV), p, batch=0, num_nodes=3, q_heads=4, kv_heads=2,
                                  head_dim=64, seq_len=e, pos_offset=i32([0, 1, 2]), inv_freq=inv_freq(64), q_out=q)
    assert kernels().kv_read_paged(p, count=0)[0].shape == (1, 2, 0, 64) and kernels().kv_read_paged(p, start=e, count=4)[0].shape[0] == 0
    kernels().kv_path_gather_paged(p, seq_len=e, acc_nodes=torch.empty(0, 2, dtype=torch.int32, device=DEV), acc_len=e, tree_nodes=2)


def test_offsets_past_32_bits():
    """Pages whose codes and scales lie more than 2^32 bytes into a pool."""
    d, size, h = 128, 64, 2
    stride = 2 ** 30 + 2 ** 20
    raw = torch.empty(4 * stride + 2 * h * size * d, dtype=torch.uint8, device=DEV)
    scale_raw = torch.empty(4 * stride + 2 * h * size * 4, dtype=torch.uint8, device=DEV)
    k, v = (torch.as_strided(raw, (5, h, size, d), (stride, size * d, d, 1), i * h * size * d) for i in (0, 1))
    ks, vs = (torch.as_strided(scale_raw, (5, h, size, 4), (stride, size * 4, 4, 1), i * h * size * 4) for i in (0, 1))
    near = Held(1, 2, size, h, d, "e4m3", seed=7)
    for i in range(2):
        for dst, src in ((k, near.k), (v, near.v), (ks, near.ks), (vs, near.vs)):
            dst[4 - i].copy_((src.view(torch.uint8) if src.dtype != torch.uint8 else src)[near.table[0, i]])
    far = kernels().KVPages(k.view(torch.float8_e4m3fn), v.view(torch.float8_e4m3fn), ks, vs, i32([[4, 3]]))
    for n, hq in ((1, 4), (29, 12), (40, 12)):
        q = queries(1, n, hq, d, n).to(DEV)
        kw = dict(anc=None, num_nodes=n, q_heads=hq, kv_heads=h, head_dim=d, seq_len=i32([128 - n]))
        assert torch.equal(kernels().paged_attention(q, far, **kw), kernels().paged_attention(q, near.pages(), **kw))
    a, b = Round(near, 4, 2, 3, 3), Round(near, 4, 2, 3, 3)
    b.pages = far
    assert all(torch.equal(x, y) for x, y in zip(a(i32([62])), b(i32([62]))))


# ------------------------------------------------------------------ refusals
def test_wrappers_refuse():
    k, held = kernels(), Held(2, 3, 16, 2, 128, "e4m3", seed=8)
    p, i2, off = held.pages(), i32([1, 2]), i32([0, 1, 2])
    q = torch.zeros(2, 3, 4, 128, dtype=torch.bfloat16, device=DEV)
    sizes = dict(num_nodes=3, q_heads=4, kv_heads=2, head_dim=128)
    anc = torch.ones(2, 3, dtype=torch.int64, device=DEV)

    def attend(q=q, pages=p, seq=i2, anc=anc, **kw):
        return k.paged_attention(q, pages, seq_len=seq, anc=anc, **{**sizes, **kw})

    qkv = torch.zeros(6, 8 * 128, dtype=torch.bfloat16, device=DEV)

    def write(qkv=qkv, pages=p, seq=i2, off=off, f=inv_freq(128), q_out=q, **kw):
        k.rope_kv_write_paged(qkv, pages, batch=2, seq_len=seq, pos_offset=off, inv_freq=f, q_out=q_out, **{**sizes, **kw})

    def parts(x=torch.zeros(2, 6, 8 * 128, device=DEV), bias=None, **kw):
        k.rope_kv_write_paged_parts(x, bias, p, batch=2, seq_len=i2, pos_offset=off, inv_freq=inv_freq(128), q_out=q, **{**sizes, **kw})

    def path(nodes=i32([[0, 1], [0, 2]]), lens=i2, tree=3, **kw):
        k.kv_path_gather_paged(p, seq_len=i2, acc_nodes=nodes, acc_len=lens, tree_nodes=tree, **kw)

    attend(), write(), parts(), path(), attend(anc=None), attend(anc=anc[0])
    raw = torch.zeros(2 * 2 * q.numel(), dtype=torch.bfloat16, device=DEV)
    bad = [lambda: attend(q=q.float()), lambda: attend(q=q[:, :2]), lambda: attend(q=q.transpose(1, 2)), lambda: attend(pages=None),
           lambda: attend(seq=i2.long()), lambda: attend(seq=i2[:1]), lambda: attend(seq=i2.cpu()), lambda: attend(anc=anc.int()),
           lambda: attend(anc=anc[:1]), lambda: attend(anc=anc[:, :2]), lambda: attend(anc=anc.t().contiguous().t()), lambda: attend(out=q),
           lambda: attend(out=q.float()), lambda: attend(kv_heads=4), lambda: attend(head_dim=64), lambda: attend(new_len=i32([1])),
           lambda: attend(row_map=torch.zeros(4, dtype=torch.int32, device=DEV)[::2]), lambda: attend(q_heads=8),
           lambda: attend(q=raw[:q.numel()].view_as(q), out=raw[64:64 + q.numel()].view_as(q)), lambda: attend(q=raw[4:4 + q.numel()].view_as(q)),
           lambda: attend(q=torch.zeros(2, 65, 4, 128, dtype=torch.bfloat16, device=DEV), anc=torch.ones(65, dtype=torch.int64, device=DEV), num_nodes=65),
           lambda: attend(q=torch.zeros(2, 3, 3, 128, dtype=torch.bfloat16, device=DEV), q_heads=3),
           lambda: write(qkv=qkv.float()), lambda: write(qkv=qkv[:5]), lambda: write(qkv=qkv[:, :-1]), lambda: write(qkv=qkv.t().contiguous().t()),
           lambda: write(qkv=qkv.cpu()), lambda: write(off=off[:2]), lambda: write(off=off.long()), lambda: write(f=inv_freq(128)[:32]),
           lambda: write(f=inv_freq(128).double()), lambda: write(q_out=q.float()), lambda: write(q_out=q[:1]), lambda: write(q_out=qkv.view(-1)[:q.numel()]),
           lambda: write(err_flag=torch.zeros(1, device=DEV)), lambda: write(off=i32([[0, 1, 2]])), lambda: write(row_map=i32([0])),
           lambda: parts(x=torch.zeros(2, 5, 8 * 128, device=DEV)), lambda: parts(x=torch.zeros(6, 8 * 128, device=DEV)),
           lambda: parts(bias=torch.zeros(8 * 128, device=DEV)), lambda: parts(bias=torch.zeros(8, dtype=torch.bfloat16, device=DEV)),
           lambda: path(nodes=i32([0, 1])), lambda: path(nodes=i32(np.zeros((2, 33)))), lambda: path(nodes=i32(np.zeros((2, 4)))[:, ::2]),
           lambda: path(lens=i32([1])), lambda: path(tree=0), lambda: path(tree=49), lambda: path(layers=0),
           lambda: path(layers=2, layer_stride=2 * 16 * 128, scale_layer_stride=2 * 16 * 4), lambda: path(layers=2),
           lambda: k.kv_read_paged(p, count=-1), lambda: k.kv_read_paged(p, count=1, dtype=torch.float16), lambda: k.kv_read_paged(None, count=1),
           lambda: k.kv_read_paged(p, start=i32([1])[:, None].expand(1, 2), count=1, batch=2)]
    for n, call in enumerate(bad):
        with pytest.raises((ValueError, TypeError, RuntimeError)):
            call()
            pytest.fail(f"call {n} was taken")
    torch.cuda.synchronize()
