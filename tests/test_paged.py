"""The paged cache without a GPU: the oracle, the host's page tables, and what the entry points refuse before they launch."""
import ctypes
import os

import numpy as np
import pytest
import torch

from flashgrpo_amd import kernels as K
from flashgrpo_amd.models import PagedKVCache, TargetConfig
from oracle import paged as O

CFG = TargetConfig(2, 64, 2, 2, 64, 128, 100)


def fill(cache, seed=0):
    g = torch.Generator().manual_seed(seed)
    cache.codes.view(torch.uint8).random_(0, 100, generator=g)
    if cache.scales is not None:
        cache.scales.random_(100, 130, generator=g)


def held(cache, row, tokens):
    """Codes and scales of a row's first tokens, from the device's table."""
    table = cache.table.numpy()[row]
    out = []
    for t in (cache.codes.view(torch.uint8) if cache.kv_format == "e4m3" else cache.codes, cache.scales):
        if t is not None:
            out.append(torch.stack([t[table[i // cache.page_size], :, :, :, i % cache.page_size] for i in range(tokens)]))
    return out


def same(a, b):
    return len(a) == len(b) and all(torch.equal(x, y) for x, y in zip(a, b))


def consistent(cache):
    """The host's table is the device's; use counts and the free list are what the table says."""
    assert (cache.table.numpy() == cache._rows).all()
    count = np.bincount(cache._rows[cache._rows >= 0], minlength=cache._uses.size)
    assert (count == cache._uses).all()
    assert sorted(cache._free) == np.nonzero(count == 0)[0].tolist()


# ------------------------------------------------------------------ the oracle
def test_oracle_attention_of_one_key_and_of_two():
    q = np.ones((1, 2, 4))
    k, v = np.zeros((1, 2, 4)), np.stack([[[1.0] * 4, [3.0] * 4]])
    out, bound = O.attention(q, k, v, np.ones(2, bool), 1, 1, None, 1.0)
    assert (out == 2.0).all() and (bound > 0).all()
    out, _ = O.attention(q, k, v, np.array([True, False]), 1, 1, None, 1.0)
    assert (out == 1.0).all()
    out, _ = O.attention(q, k, v, np.ones(2, bool), 1, 1, [0], 1.0)
    assert (out == 1.0).all()
    out, _ = O.attention(q, k[:, :1], v[:, :1], np.ones(1, bool), 0, 1, [0], 1.0)
    assert (out == 0.0).all()


def test_oracle_rotation_keeps_lengths_and_turns_by_the_position():
    x = np.random.default_rng(0).standard_normal((3, 2, 8))
    f = 1.0 / 100.0 ** (np.arange(4) / 4)
    y = O.rotate(x, [0, 1, 5], f)
    assert np.allclose(y[0], x[0]) and np.allclose((y ** 2).sum(-1), (x ** 2).sum(-1))
    assert np.allclose(O.rotate(y[1:2], [-1], f), x[1:2])


# ------------------------------------------------------------------ the host's tables
@pytest.mark.parametrize("fmt", ["bf16", "e4m3"])
def test_reserve_and_release(fmt):
    c = PagedKVCache(CFG, 3, 100, device="cpu", kv_format=fmt, page_size=16, pages=9)
    c.reserve([0, 16, 17])
    assert (c._rows >= 0).sum(1).tolist() == [0, 1, 2] and c.free_pages == 6
    c.reserve([0, 16, 17])
    assert c.free_pages == 6
    c.reserve(90, rows=[0], first=85)  # what lies before the first token too
    assert (c._rows[0] >= 0).sum() == 6 and c.free_pages == 0
    consistent(c)
    c.release([0, 2])
    assert c.free_pages == 8 and (c._rows[0] == -1).all()
    consistent(c)


def test_reserve_raises_and_changes_nothing_when_the_pool_is_empty():
    c = PagedKVCache(CFG, 2, 64, device="cpu", page_size=16, pages=5)
    c.reserve([48, 16])
    before = c._rows.copy()
    with pytest.raises(RuntimeError, match="1 of 5 free"):
        c.reserve([64, 64])
    assert (c._rows == before).all() and c.free_pages == 1
    consistent(c)
    with pytest.raises(ValueError, match="capacity"):
        c.reserve(65, rows=[1])
    c.release([0])
    assert c.free_pages == 4
    c.reserve([0, 64])
    consistent(c)


@pytest.mark.parametrize("fmt", ["bf16", "e4m3"])
def test_repeats_share_whole_pages_and_copy_the_last(fmt):
    c = PagedKVCache(CFG, 4, 80, device="cpu", kv_format=fmt, page_size=16)
    fill(c)
    c.reserve([40, 0, 32, 0], first=0)
    c.seq_len.copy_(torch.tensor([40, 0, 32, 0]))
    want = [held(c, 0, 40), None, held(c, 2, 32)]
    c.repeat_rows(torch.tensor([0, 2]), torch.tensor([1, 3]))
    consistent(c)
    assert c.seq_len.tolist() == [40, 40, 32, 32]
    assert (c._rows[0, :2] == c._rows[1, :2]).all() and c._rows[0, 2] != c._rows[1, 2]
    assert (c._rows[2] == c._rows[3]).all()
    assert same(held(c, 1, 40), want[0]) and same(held(c, 3, 32), want[2])
    free = c.free_pages
    c.reserve(48, first=[40, 40, 32, 32])  # new pages behind shared ones: nothing is copied
    assert c.free_pages == free - 2
    consistent(c)
    # a row that is about to write into a shared page gets a copy of it, the other keeps it
    old = c._rows[:, 1].copy()
    c.reserve(48, rows=[0], first=20)
    assert c._rows[0, 1] != old[0] and c._rows[1, 1] == old[1] and c._rows[0, 0] == c._rows[1, 0]
    assert same(held(c, 0, 40), want[0]) and same(held(c, 1, 40), want[0])
    consistent(c)
    # both at once: one of them keeps it
    c.reserve(48, rows=[2, 3], first=0)
    assert not set(c._rows[2, :3]) & set(c._rows[3, :3])
    assert same(held(c, 2, 32), want[2]) and same(held(c, 3, 32), want[2])
    consistent(c)


def test_rows_that_are_refused():
    """Rows that are not there, or twice, tokens before the first, lengths without pages: refused, with nothing changed."""
    c = PagedKVCache(CFG, 3, 64, device="cpu", page_size=16, pages=7)
    c.reserve([40, 16, 0])
    c.seq_len.copy_(torch.tensor([40, 16, 0]))
    before, free = c._rows.copy(), c.free_pages
    for call in (lambda: c.reserve(64, rows=[2, 2]), lambda: c.reserve(16, rows=[-1]), lambda: c.reserve(16, rows=[3]),
                 lambda: c.reserve([1, 2], rows=[0, 1, 2]), lambda: c.reserve(-1), lambda: c.reserve(16, first=-1),
                 lambda: c.release([3]), lambda: c.release([-1]), lambda: c.repeat_rows(torch.tensor([0]), torch.tensor([3])),
                 lambda: c.repeat_rows(torch.tensor([-3]), torch.tensor([1])), lambda: c.select_rows(torch.tensor([3])),
                 lambda: c.select_rows(torch.tensor([-1]))):
        with pytest.raises(ValueError):
            call()
        assert (c._rows == before).all() and c.free_pages == free
    c.seq_len[2] = 20  # committed tokens that were never written
    with pytest.raises(ValueError, match="no page"):
        c.repeat_rows(torch.tensor([2]), torch.tensor([1]))
    with pytest.raises(ValueError, match="no page"):
        c.select_rows(torch.tensor([2]))
    assert (c._rows == before).all() and c.free_pages == free
    consistent(c)


def test_repeat_rows_without_room_changes_nothing():
    c = PagedKVCache(CFG, 4, 64, device="cpu", page_size=16, pages=5)
    c.reserve([40, 0, 0, 16])
    c.seq_len.copy_(torch.tensor([40, 0, 0, 16]))
    before, lens = c._rows.copy(), c.seq_len.clone()
    with pytest.raises(RuntimeError, match="3 more pages needed, 2 of 5 free"):  # (row 3's page comes back)
        c.repeat_rows(torch.tensor([0, 0, 0]), torch.tensor([1, 2, 3]))
    assert (c._rows == before).all() and c.free_pages == 1 and torch.equal(c.seq_len, lens)
    consistent(c)
    c.repeat_rows(torch.tensor([0, 0]), torch.tensor([1, 3]))
    assert c.free_pages == 0
    consistent(c)


def test_repeat_rows_refusals():
    c = PagedKVCache(CFG, 3, 32, device="cpu", page_size=16)
    for src, dst in (([0, 1], [1, 2]), ([0, 0], [1, 1]), ([0], [1, 2])):
        with pytest.raises(ValueError, match="repeat_rows"):
            c.repeat_rows(torch.tensor(src), torch.tensor(dst))


@pytest.mark.parametrize("fmt", ["bf16", "e4m3"])
def test_select_rows_and_copies(fmt):
    c = PagedKVCache(CFG, 3, 64, device="cpu", kv_format=fmt, page_size=16)
    fill(c, 1)
    c.reserve([33, 0, 16], first=0)
    c.seq_len.copy_(torch.tensor([33, 0, 16]))
    want = [held(c, 0, 33), held(c, 2, 16)]
    s = c.select_rows(torch.tensor([2, 0, 2]), capacity=40)
    assert s.seq_len.tolist() == [16, 33, 16] and s.capacity == 40
    assert same(held(s, 0, 16), want[1]) and same(held(s, 1, 33), want[0]) and same(held(s, 2, 16), want[1])
    consistent(s)
    d, shared = c.deep_copy(), c.container_copy()
    consistent(d)
    fill(c, 2)
    assert same(held(d, 0, 33), want[0]) and not same(held(shared, 0, 33), want[0])
    shared.seq_len += 1
    assert c.seq_len.tolist() == [33, 0, 16]
    shared.reserve([34, 16, 16], first=[33, 0, 16])  # one pool, one table
    consistent(c)
    assert (c._rows == shared._rows).all()


def test_formats():
    with pytest.raises(ValueError, match="kv_format"):
        PagedKVCache(CFG, 1, 16, device="cpu", kv_format="int8")
    with pytest.raises(ValueError, match="head_dim"):
        PagedKVCache(TargetConfig(1, 64, 2, 2, 32, 128, 100), 1, 16, device="cpu")
    with pytest.raises(ValueError, match="page_size"):
        PagedKVCache(CFG, 1, 16, device="cpu", page_size=24)
    for size in (0, -16, 8):
        with pytest.raises(ValueError):
            PagedKVCache(CFG, 1, 16, device="cpu", page_size=size)


# ------------------------------------------------------------------ refusals
def pages(n=4, heads=2, size=16, d=64, fmt="e4m3", width=3, rows=2):
    if fmt == "bf16":
        k, v = (torch.zeros(n, heads, size, d, dtype=torch.bfloat16) for _ in range(2))
        ks = vs = None
    else:
        k, v = (torch.zeros(n, heads, size, d, dtype=torch.uint8).view(torch.float8_e4m3fn) for _ in range(2))
        ks, vs = (torch.ones(n, heads, size, d // 32, dtype=torch.uint8) for _ in range(2))
    return k, v, ks, vs, torch.zeros(rows, width, dtype=torch.int32)


def test_pages_that_are_refused():
    k, v, ks, vs, table = pages()
    p = K.KVPages(k, v, ks, vs, table)
    assert (p.format, p.pages, p.page_size, p.kv_heads, p.head_dim, p.capacity, p.device) == (0, 4, 16, 2, 64, 48, -1)
    kb, vb = pages(fmt="bf16")[:2]
    assert K.KVPages(kb, vb, None, None, table).format == 1
    bad = [((k.float(), v.float(), None, None, table), TypeError), ((k, vb, ks, vs, table), TypeError),
           ((k, v, None, None, table), ValueError), ((kb, vb, ks, vs, table), ValueError), ((k, v, ks, None, table), ValueError),
           ((k, v[:3], ks, vs, table), ValueError), ((k, v, ks[:3], vs, table), ValueError), ((k, v, ks, vs[..., :1], table), ValueError),
           ((k, v, ks, vs, table.long()), ValueError), ((k, v, ks, vs, table[0]), ValueError), ((k, v, ks, vs, table[:, :0]), ValueError),
           ((k, v, ks, vs, torch.zeros(3, 2, dtype=torch.int32).t()), ValueError),
           ((kb[..., :32], vb[..., :32], None, None, table), ValueError), ((kb[:, :, :12], vb[:, :, :12], None, None, table), ValueError),
           ((kb.transpose(1, 2), vb.transpose(1, 2), None, None, table), ValueError), ((kb[0], vb[0], None, None, table), ValueError),
           ((kb[:, :1], vb, None, None, table), ValueError), ((k, v, ks, vs, torch.zeros(1, 1, dtype=torch.int32).expand(2, 1)), ValueError)]
    for args, kind in bad:
        with pytest.raises(kind):
            K.KVPages(*args)
    raw = torch.zeros(4 * 2 * 16 * 64 + 8, dtype=torch.bfloat16)
    off = raw[4:4 + 4 * 2 * 16 * 64].view(4, 2, 16, 64)
    with pytest.raises(ValueError, match="aligned"):
        K.KVPages(off, off, None, None, table)


def test_calls_on_the_host_are_refused():
    p = K.KVPages(*pages())
    i = torch.zeros(2, dtype=torch.int32)
    q = torch.zeros(2, 1, 2, 64, dtype=torch.bfloat16)
    kw = dict(num_nodes=1, q_heads=2, kv_heads=2, head_dim=64)
    for call in (lambda: K.paged_attention(q, p, seq_len=i, anc=None, **kw),
                 lambda: K.rope_kv_write_paged(torch.zeros(2, 6 * 64, dtype=torch.bfloat16), p, batch=2, seq_len=i, pos_offset=i,
                                               inv_freq=torch.ones(32), q_out=q, **kw),
                 lambda: K.rope_kv_write_paged_parts(torch.zeros(1, 2, 6 * 64), None, p, batch=2, seq_len=i, pos_offset=i,
                                                     inv_freq=torch.ones(32), q_out=q, **kw),
                 lambda: K.kv_read_paged(p, start=i, count=1),
                 lambda: K.kv_path_gather_paged(p, seq_len=i, acc_nodes=i.view(2, 1), acc_len=i, tree_nodes=1)):
        with pytest.raises(ValueError, match="device tensors"):
            call()


def library():
    from flashgrpo_amd import _lib

    if not os.path.exists(_lib.library_path()):
        pytest.skip("native library not built")
    return _lib, _lib.load()


def struct(**changed):
    from flashgrpo_amd import _lib

    at = dict(k=4096, v=8192, k_scales=64, v_scales=128, table=256, page_stride=2 * 16 * 128, scale_stride=2 * 16 * 4, table_stride=3,
              format=0, pages=4, page_size=16, kv_heads=2, head_dim=128, table_rows=2, table_width=3)
    at.update(changed)
    return _lib.KvPages(*(at[n] for n, _ in _lib.KvPages._fields_))


@pytest.mark.parametrize("changed,message", [
    (dict(format=2), b"format"), (dict(k=None), b"null pointer"), (dict(v=None), b"null pointer"), (dict(table=None), b"null pointer"),
    (dict(k_scales=None), b"null pointer"), (dict(head_dim=96), b"head_dim"), (dict(page_size=24), b"power of two"),
    (dict(page_size=8), b"power of two"), (dict(page_size=0), b"power of two"), (dict(pages=0), b"bad sizes"),
    (dict(kv_heads=-1), b"bad sizes"), (dict(table_width=0), b"bad sizes"), (dict(table_rows=0), b"bad sizes"),
    (dict(table_width=2 ** 27, table_stride=2 ** 27), b"2^31 tokens"), (dict(page_stride=4095), b"overlap"), (dict(table_stride=2), b"overlap"),
    (dict(k=4100), b"16-byte"), (dict(page_stride=4104), b"16-byte"), (dict(k_scales=66), b"4-byte"), (dict(scale_stride=126), b"4-byte"),
    (dict(scale_stride=64), b"overlap"), (dict(page_size=2 ** 20, kv_heads=8, page_stride=2 ** 30, scale_stride=2 ** 25, table_width=1), b"2^30 elements"),
    (dict(page_stride=2 ** 31), b"2^31 elements"),
])
def test_descriptions_of_pages_that_every_entry_point_refuses(changed, message):
    _, lib = library()
    s = struct(**changed)
    p, x = ctypes.addressof(s), ctypes.c_void_p(1024)
    calls = [lambda: lib.fg_rope_kv_write_paged(x, 1024, 2, 1, 4, p, x, x, 0, x, None, None, x, None, None),
             lambda: lib.fg_rope_kv_write_paged_parts(x, 1, None, 2, 1, 4, p, x, x, 0, x, None, None, x, None, None),
             lambda: lib.fg_kv_read_paged(p, 2, None, 1, None, x, x, 1, None),
             lambda: lib.fg_paged_attention(x, x, p, 2, 1, 4, x, None, None, None, 0, 1.0, None, 0, None),
             lambda: lib.fg_kv_path_gather_paged(p, 1, 0, 0, 2, x, None, x, 1, x, 1, None, None)]
    for call in calls:
        assert call() != 0 and message in lib.fg_last_error(), lib.fg_last_error()


def test_calls_that_the_entry_points_refuse():
    _, lib = library()
    s = struct()
    p, x, y = ctypes.addressof(s), ctypes.c_void_p(1024), ctypes.c_void_p(1028)

    def write(qkv=x, ld=1024, b=2, n=1, hq=4, pages=p, seq=x, pos=x, f=x, q=x):
        return lib.fg_rope_kv_write_paged(qkv, ld, b, n, hq, pages, seq, pos, 0, f, None, None, q, None, None)

    def parts(part=x, splits=1, bias=None, pages=p):
        return lib.fg_rope_kv_write_paged_parts(part, splits, bias, 2, 1, 4, pages, x, x, 0, x, None, None, x, None, None)

    def read(b=2, n=1, k=x, v=x, dt=1, pages=p):
        return lib.fg_kv_read_paged(pages, b, None, n, None, k, v, dt, None)

    def attend(q=x, o=x, b=2, n=1, hq=4, seq=x, anc=None, pages=p):
        return lib.fg_paged_attention(q, o, pages, b, n, hq, seq, None, None, anc, 0, 1.0, None, 0, None)

    def path(layers=1, stride=0, sstride=0, b=2, seq=x, nodes=x, width=1, lens=x, tree=1, pages=p):
        return lib.fg_kv_path_gather_paged(pages, layers, stride, sstride, b, seq, None, nodes, width, lens, tree, None, None)

    for call, message in [
            (lambda: write(qkv=None), b"null pointer"), (lambda: write(seq=None), b"null pointer"), (lambda: write(q=None), b"null pointer"),
            (lambda: write(pages=None), b"null pointer"), (lambda: write(pos=None), b"null pointer"), (lambda: write(f=None), b"null pointer"),
            (lambda: write(ld=1020), b"stride"), (lambda: write(ld=1026), b"stride"), (lambda: write(b=0), b"bad shape"),
            (lambda: write(n=8193), b"bad shape"), (lambda: write(hq=0), b"bad shape"), (lambda: write(qkv=y), b"8-byte"),
            (lambda: write(q=y), b"8-byte"), (lambda: write(b=2 ** 30, n=2), b"bad shape"),
            (lambda: parts(part=None), b"null pointer"), (lambda: parts(pages=None), b"null pointer"), (lambda: parts(splits=0), b"splits"),
            (lambda: parts(part=y), b"aligned"), (lambda: parts(bias=y), b"aligned"),
            (lambda: read(k=None), b"null pointer"), (lambda: read(b=0), b"bad shape"), (lambda: read(n=0), b"bad shape"),
            (lambda: read(dt=2), b"dtype"), (lambda: read(v=y), b"aligned"), (lambda: read(b=2 ** 30, n=2 ** 30), b"too many rows"),
            (lambda: read(pages=None), b"null pointer"),
            (lambda: attend(q=None), b"null pointer"), (lambda: attend(seq=None), b"null pointer"), (lambda: attend(pages=None), b"null pointer"),
            (lambda: attend(n=65, anc=x), b"num_nodes"), (lambda: attend(n=8193), b"bad shape"), (lambda: attend(hq=5), b"bad shape"),
            (lambda: attend(b=0), b"bad shape"), (lambda: attend(q=y), b"aligned"), (lambda: attend(o=y), b"aligned"),
            (lambda: attend(b=2 ** 29, n=1), b"bad shape"),
            (lambda: path(seq=None), b"null pointer"), (lambda: path(nodes=None), b"null pointer"), (lambda: path(lens=None), b"null pointer"),
            (lambda: path(layers=0), b"bad shape"), (lambda: path(b=0), b"bad shape"), (lambda: path(width=33), b"acc_stride"),
            (lambda: path(width=0), b"acc_stride"), (lambda: path(tree=0), b"tree"), (lambda: path(tree=49), b"tree"),
            (lambda: path(layers=2, stride=8), b"16-byte"), (lambda: path(layers=2, stride=16, sstride=2), b"4-byte"),
            (lambda: path(layers=2 ** 20, stride=16, sstride=4, b=2 ** 20), b"too many rows")]:
        assert call() != 0 and message in lib.fg_last_error(), (message, lib.fg_last_error())


def test_workspace_only_where_parts_are_made():
    _, lib = library()
    w = lib.fg_paged_attention_workspace
    assert w(64, 29, 28, 4, 128, 4096) == 0 and w(64, 1, 32, 8, 128, 131072) == 0    # a workgroup per CU without it
    assert w(1, 1, 12, 2, 128, 256) == 0                                              # too short to cut
    few = w(2, 1, 32, 8, 128, 131072)
    assert few == 256 // 8 * 32 * (128 * 4 + 8) + 2 * 8                              # (O, m, l) of a row in 32 parts, each sequence's share
    assert w(0, 1, 32, 8, 128, 4096) == 0 and w(1, 1, 32, 8, 96, 4096) == 0 and w(1, 1, 5, 2, 128, 4096) == 0
