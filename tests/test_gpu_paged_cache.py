"""Writing K and V into pages, reading them back and moving an accepted path, on the GPU against the oracle, bit for bit."""
import numpy as np
import pytest
import torch

from oracle import paged as O
from paged_cases import DEV, Held, i32, kernels

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


def inv_freq(d, theta=1.0e6):
    return 1.0 / theta ** (torch.arange(0, d, 2).float() / d)


def rows_of(n, width, seed):
    rng = np.random.default_rng(seed)
    x = rng.standard_normal((n, width)) * np.exp(rng.standard_normal((n, width // 32))).repeat(32, 1)
    return torch.from_numpy(x).to(torch.bfloat16)


def write(held, qkv, committed, n, hq, *, offset=None, fresh=None, row=None, err=None, parts=None, bias=None, fill=3.0):
    b, d = len(committed), held.d
    q = torch.full((b, n, hq, d), fill, dtype=torch.bfloat16, device=DEV)
    kw = dict(batch=b, num_nodes=n, q_heads=hq, kv_heads=held.heads, head_dim=d, seq_len=i32(committed),
              pos_offset=i32(np.arange(n)) if offset is None else offset, inv_freq=inv_freq(d).to(DEV), q_out=q,
              new_len=None if fresh is None else i32(fresh), row_map=None if row is None else i32(row), err_flag=err)
    if parts is None:
        kernels().rope_kv_write_paged(qkv.to(DEV), held.pages(), **kw)
    else:
        kernels().rope_kv_write_paged_parts(parts, bias, held.pages(), **kw)
    return q


def oracle_write(held, qkv, committed, n, hq, *, offset=None, fresh=None, row=None):
    """(q float64 [b, n, hq, d], K and V codes and scales of every page) after the write."""
    b, d, h = len(committed), held.d, held.heads
    x = qkv.double().numpy().reshape(b, n, hq + 2 * h, d)
    offset = np.arange(n)[None].repeat(b, 0) if offset is None else offset
    qs = np.zeros((b, n, hq, d))
    codes, scales = [c.copy() for c in held.codes], [s.copy() for s in held.scales]
    for i in range(b):
        pos = committed[i] + offset[i]
        qs[i] = O.rotate(x[i, :, :hq], pos, inv_freq(d).numpy())
        k = O.rotate(x[i, :, hq:hq + h], pos, inv_freq(d).numpy()).astype(np.float32)
        for j in range(n if fresh is None else fresh[i]):
            t = committed[i] + j
            p = O.page_of(held.table[i if row is None else row[i]], t, held.size, held.pages_n)
            if p is None:
                continue
            for w, y in enumerate((k[j], x[i, j, hq + h:])):
                c, s = O.quantize(y)
                codes[w][p, :, t % held.size], scales[w][p, :, t % held.size] = c, s
    return qs, codes, scales


def same_pages(held, codes, scales):
    for t, c in ((held.k, codes[0]), (held.v, codes[1])):
        assert (t.view(torch.uint8).cpu().numpy() == c).all()
    for t, s in ((held.ks, scales[0]), (held.vs, scales[1])):
        assert (t.cpu().numpy() == s).all()


def near_q(q, want, fresh=None):
    """q within half a bf16 step and what fp32 leaves: two products and a sum, 3 roundings of 2^-24 of the larger operand."""
    x = q.double().cpu().numpy()
    big = np.abs(want).reshape(*want.shape[:-1], 2, -1)
    slack = 2.0 ** -22 * np.sqrt((big ** 2).sum(-2, keepdims=True)).repeat(2, -2).reshape(want.shape)
    for b in range(x.shape[0]):
        c = x.shape[1] if fresh is None else fresh[b]
        assert (np.abs(x[b, :c] - want[b, :c]) <= 2.0 ** -8 * np.abs(want[b, :c]) + 2 * slack[b, :c]).all()
        assert (x[b, c:] == 3.0).all()


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("size", [16, 64, 256])
@pytest.mark.parametrize("n", [1, 5, 29])
@pytest.mark.parametrize("heads", [(1, 1), (12, 2), (7, 7), (5, 1)])
def test_write_e4m3(d, size, n, heads):
    hq, h = heads
    committed = [0, 13, 250]
    held = Held(3, -(-290 // size), size, h, d, "e4m3", seed=n)
    qkv = rows_of(3 * n, (hq + 2 * h) * d, n)
    want = oracle_write(held, qkv, committed, n, hq)
    q = write(held, qkv, committed, n, hq)
    same_pages(held, *want[1:])
    near_q(q, want[0])


def test_write_far_positions_and_tree_offsets():
    """Positions about 10^5 and 2^30, and offsets per sequence: angles to 64 bits."""
    held = Held(2, 4, 64, 2, 128, "e4m3", seed=1)
    n, hq = 6, 4
    offset = np.array([[100000, 99999, 131071, 5, 0, 7], [2 ** 30, 2 ** 30 + 1, 12345678, 1, 2, 3]])
    qkv = rows_of(2 * n, (hq + 4) * 128, 2)
    want = oracle_write(held, qkv, [31, 100], n, hq, offset=offset)
    q = write(held, qkv, [31, 100], n, hq, offset=i32(offset))
    same_pages(held, *want[1:])
    near_q(q, want[0])


def test_write_padded_batch_row_map_and_missing_pages():
    held = Held(4, 5, 32, 2, 128, "e4m3", seed=3)
    held.table[2, 1] = -1
    held.upload()
    n, hq, fresh, row, committed = 11, 3, [11, 0, 4], [2, 0, 3], [28, 3, 150]
    qkv = rows_of(3 * n, (hq + 4) * 128, 4)
    want = oracle_write(held, qkv, committed, n, hq, fresh=fresh, row=row)
    err = i32([0])
    q = write(held, qkv, committed, n, hq, fresh=fresh, row=row, err=err)
    same_pages(held, *want[1:])
    near_q(q, want[0], fresh)
    assert err.item() == 8  # tokens 32 .. 38 of row 2 have no page
    err.zero_()
    write(held, qkv, [0, 3, 150], n, hq, fresh=fresh, row=row, err=err)
    assert err.item() == 0
    write(held, qkv, [0, 3, 157], n, hq, fresh=fresh, row=row, err=err)  # behind the table's last page
    assert err.item() == 8
    err.zero_()
    write(held, qkv, [0, 3, 150], n, hq, fresh=[1, 1, 1], row=[0, 1, 4], err=err)  # a cache row that is none
    assert err.item() == 8
    err.zero_()
    write(held, qkv, [-1, 3, 150], n, hq, fresh=[1, 1, 1], err=err)
    assert err.item() == 8


def test_write_infinities_and_nan():
    held = Held(1, 2, 64, 1, 128, "e4m3", seed=5)
    qkv = rows_of(4, 3 * 128, 6)
    qkv[0, 128 + 5], qkv[1, 256 + 70], qkv[2, 256 + 127] = float("inf"), float("nan"), float("-inf")
    write(held, qkv, [7], 4, 1)
    k, v = kernels().kv_read_paged(held.pages(), start=i32([7]), count=4)
    k, v = k[0, 0].float().cpu(), v[0, 0].float().cpu()
    bad_k, bad_v = torch.zeros(4, 128, dtype=torch.bool), torch.zeros(4, 128, dtype=torch.bool)
    bad_k[0, :32] = bad_k[0, 64:96] = True  # element 5 turns with element 69
    bad_v[1, 64:96] = bad_v[2, 96:] = True
    assert torch.equal(torch.isnan(k), bad_k) and torch.equal(torch.isnan(v), bad_v)


@pytest.mark.parametrize("d", [64, 128])
def test_bf16_pages_hold_what_the_contiguous_cache_does(d):
    hq, h, n, committed = 6, 2, 13, [0, 40, 99]
    held = Held(3, 4, 32, h, d, "bf16", seed=7)
    qkv = rows_of(3 * n, (hq + 2 * h) * d, 8)
    q = write(held, qkv, committed, n, hq)
    want_q = torch.empty_like(q)
    kc, vc = (torch.zeros(3, h, 128, d, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    kernels().rope_kv_write(qkv.to(DEV), batch=3, num_nodes=n, q_heads=hq, kv_heads=h, head_dim=d, seq_len=i32(committed),
                            pos_offset=i32(np.arange(n)), inv_freq=inv_freq(d).to(DEV), q_out=want_q, k_cache=kc, v_cache=vc)
    k, v = kernels().kv_read_paged(held.pages(), start=i32(committed), count=n)
    assert torch.equal(q, want_q)
    for b, c in enumerate(committed):
        assert torch.equal(k[b], kc[b, :, c:c + n]) and torch.equal(v[b], vc[b, :, c:c + n])


@pytest.mark.parametrize("fmt", ["e4m3", "bf16"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("splits,bias", [(1, False), (4, True)])
def test_parts(fmt, d, splits, bias):
    hq, h, n, committed = 3, 2, 5, [10, 60]
    a, b = (Held(2, 5, 16, h, d, fmt, seed=9) for _ in range(2))
    width = (hq + 2 * h) * d
    parts = torch.from_numpy(np.random.default_rng(1).standard_normal((splits, 2 * n, width))).float().to(DEV)
    bw = rows_of(1, width, 2)[0].to(DEV) if bias else None
    total = parts[0].clone()
    for s in range(1, splits):
        total += parts[s]
    qkv = (total + (bw.float() if bias else 0.0)).to(torch.bfloat16)
    q1 = write(a, qkv, committed, n, hq)
    q2 = write(b, None, committed, n, hq, parts=parts, bias=bw)
    assert torch.equal(q1, q2)
    for i in range(2):
        assert (a.now(i) == b.now(i)).all()


# ------------------------------------------------------------------ reading
@pytest.mark.parametrize("fmt", ["e4m3", "bf16"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_read(fmt, d, dtype):
    held = Held(3, 4, 16, 2, d, fmt, seed=10)
    held.table[1, 2] = -1
    held.upload()
    for start, row, count in (([0, 5, 60], None, 9), ([-3, 30, 63], None, 20), (None, [2, 2, 0, 1], 64), ([7], [1], 1)):
        k, v = kernels().kv_read_paged(held.pages(), start=None if start is None else i32(start), count=count,
                                       row_map=None if row is None else i32(row), dtype=dtype)
        for i, got in enumerate((k, v)):
            assert got.dtype == dtype
            for b in range(got.shape[0]):
                tokens = np.arange(count) + (0 if start is None else start[b])
                want, _ = O.rows_at(held.values[i], held.table[b if row is None else row[b]], tokens)
                assert (got[b].double().cpu().numpy() == want).all()


# ------------------------------------------------------------------ the accepted path
@pytest.mark.parametrize("fmt", ["e4m3", "bf16"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("size", [16, 64])
@pytest.mark.parametrize("stride", [1, 5, 17])
@pytest.mark.parametrize("layers", [1, 3])
def test_path_gather(fmt, d, size, stride, layers):
    """Paths of unequal length in every layer of a pool that holds a page's layers side by side."""
    rng, b, tree, h = np.random.default_rng(stride), 4, 40, 2
    committed = [0, 11, 100, 63]
    one = [Held(b, -(-150 // size), size, h, d, fmt, seed=20 + l) for l in range(layers)]
    table, n = one[0].table, one[0].pages_n
    as_bytes = lambda t: t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t
    pool = torch.stack([torch.stack([as_bytes(x.k), as_bytes(x.v)], 1) for x in one], 1)  # [pages, layers, 2, h, size, d]
    pool = pool.view(one[0].k.dtype) if fmt == "e4m3" else pool
    sc = torch.stack([torch.stack([x.ks, x.vs], 1) for x in one], 1) if fmt == "e4m3" else None
    pages = kernels().KVPages(pool[:, 0, 0], pool[:, 0, 1], None if sc is None else sc[:, 0, 0], None if sc is None else sc[:, 0, 1],
                              torch.from_numpy(table).to(DEV))
    nodes = np.stack([np.concatenate([[0], np.sort(rng.choice(np.arange(1, tree), stride - 1, replace=False))]) for _ in range(b)])
    lens, row, err = rng.integers(1, stride + 1, b), rng.permutation(b), i32([0])
    kernels().kv_path_gather_paged(pages, seq_len=i32(committed), acc_nodes=i32(nodes), acc_len=i32(lens), tree_nodes=tree,
                                   layers=layers, layer_stride=pool.stride(1), scale_layer_stride=0 if sc is None else sc.stride(1),
                                   row_map=i32(row), err_flag=err)
    assert err.item() == 0
    for l, x in enumerate(one):
        for i in range(2):
            raws = [as_bytes((x.k, x.v)[i]).cpu().float().numpy()] + ([] if sc is None else [(x.ks, x.vs)[i].cpu().numpy()])
            gots = [as_bytes(pool[:, l, i].contiguous()).cpu().float().numpy()] + ([] if sc is None else [sc[:, l, i].cpu().numpy()])
            for raw, got in zip(raws, gots):
                want = raw.copy()
                for j in range(b):
                    for m in range(lens[j]):
                        at = [(table[row[j]][t // size], t % size) for t in (committed[j] + nodes[j][m], committed[j] + m)]
                        want[at[1][0], :, at[1][1]] = raw[at[0][0], :, at[0][1]]
                assert (want == got).all()


def test_path_gather_reports_and_skips():
    held = Held(3, 4, 16, 1, 128, "e4m3", seed=30)
    held.table[2, 1] = -1
    held.upload()
    before = [held.now(i) for i in range(2)]
    call = lambda seq, nodes, lens, err, tree=20: kernels().kv_path_gather_paged(
        held.pages(), seq_len=i32(seq), acc_nodes=i32(nodes), acc_len=i32(lens), tree_nodes=tree, err_flag=err)
    for seq, nodes, lens in (([50, 0, 0], [[0, 5]] * 3, [2, 1, 1]),       # the tree reaches behind the row
                             ([0, 0, 0], [[0, 20], [0, 0], [0, 0]], [2, 1, 1]),  # a node outside the tree
                             ([0, 0, 0], [[0, -1], [0, 0], [0, 0]], [2, 1, 1]),
                             ([0, 0, 0], [[0, 1]] * 3, [3, 1, 1]),        # a path longer than its row
                             ([0, 0, 0], [[0, 1]] * 3, [0, 1, 1]),
                             ([0, 0, 10], [[0, 1], [0, 1], [0, 9]], [1, 1, 2])):  # a token without a page
        err = i32([0])
        call(seq, nodes, lens, err)
        assert err.item() == 1
        assert all((held.now(i) == before[i]).all() for i in range(2))
