"""The paged attention with weights rounded to bf16, which callers (the target model among them) ask for, against the float64 oracle
(``oracle/paged.py``) within the bound of such weights."""
import ctypes
import os

import numpy as np
import pytest
import torch

from flashgrpo_amd import kernels as K
from flashgrpo_amd import models
from paged_cases import DEV, Held, attention_oracle, close, i32, masks, queries, tree_words

ROWS = [(2, 1), (4, 7), (4, 13), (4, 30), (5, 29), (7, 29), (2, 150)]  # 1 to 300 rows of a kv head: every row layout


def need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


def attend(held, q, committed, words, *, fresh=None, bf16_weights=True, **kw):
    b, n, hq, d = q.shape
    return K.paged_attention(q.to(DEV), held.pages(), seq_len=i32(committed), anc=None if words is None else masks(words), num_nodes=n, q_heads=hq,
                             kv_heads=held.heads, head_dim=d, new_len=None if fresh is None else i32(fresh), bf16_weights=bf16_weights, **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["e4m3", "bf16"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("group,n", ROWS)
def test_every_row_layout(fmt, d, group, n):
    need_gpu()
    committed, fresh = [330, 0, 21], [n, max(n - 3, 0), n // 2]
    held = Held(3, -(-(330 + n) // 32), 32, 2, d, fmt, seed=n)
    held.table[0, 2] = -1
    held.upload()
    words = None if n > 64 else [tree_words(n, i) for i in range(3)]
    q = queries(3, n, 2 * group, d, n)
    out = torch.full(q.shape, 7.5, dtype=torch.bfloat16, device=DEV)
    assert attend(held, q, committed, words, fresh=fresh, out=out) is out
    close(out, attention_oracle(held, q, committed, fresh, words, d ** -0.5), fresh)
    for b, c in enumerate(fresh):
        assert (out[b, c:] == 7.5).all()


@pytest.mark.gpu
@pytest.mark.parametrize("group,n", [(2, 1), (4, 29), (7, 29)])
def test_parts(group, n):
    need_gpu()
    committed = [2900, 700]
    held = Held(2, 46, 64, 1, 128, "e4m3", seed=3)
    q = queries(2, n, group, 128, n)
    close(attend(held, q, committed, None), attention_oracle(held, q, committed, [n, n], None, 128 ** -0.5), [n, n])


@pytest.mark.gpu
@pytest.mark.parametrize("group,n", ROWS)
def test_what_differs(group, n):
    """Up to 32 rows of a kv head the two are one; above, single weights differ by 2^-8 at most."""
    need_gpu()
    held = Held(2, 20, 32, 1, 128, "e4m3", seed=n)
    q = queries(2, n, group, 128, n)
    a, b = (attend(held, q, [400, 33], None, bf16_weights=w) for w in (True, False))
    assert torch.equal(a, b) == (group * n <= 32)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["e4m3", "bf16"])
@pytest.mark.parametrize("group,n", [r for r in ROWS if 1 < r[1] <= 64])
def test_values_that_are_not_finite(fmt, group, n):
    """V of new token 2: who sees it shows it in its dims, nobody else does."""
    need_gpu()
    held = Held(1, 5, 32, 1, 128, fmt, seed=n)
    p = held.table[0, 63 // 32]
    held.raw[1][p, 0, 63 % 32, 64], held.raw[1][p, 0, 63 % 32, 71] = float("inf"), float("nan")
    held.refresh(1)
    held.upload()
    words = [tree_words(n, 3)]
    q = queries(1, n, group, 128, n)
    out = attend(held, q, [61], words)
    with np.errstate(invalid="ignore"):
        close(out, attention_oracle(held, q, [61], [n], words, 128 ** -0.5), [n])


def test_the_entry_point_refuses_as_the_other():
    from flashgrpo_amd import _lib

    if not os.path.exists(_lib.library_path()):
        pytest.skip("native library not built")
    lib = _lib.load()
    s = _lib.KvPages(4096, 8192, 64, 128, 256, 2 * 16 * 128, 2 * 16 * 4, 3, 0, 4, 16, 2, 128, 2, 3)
    p, x, y = ctypes.addressof(s), ctypes.c_void_p(1024), ctypes.c_void_p(1028)

    def call(q=x, o=x, b=2, n=1, hq=4, seq=x, anc=None, pages=p, scale=1.0):
        return lib.fg_paged_attention_bf16_weights(q, o, pages, b, n, hq, seq, None, None, anc, 0, scale, None, 0, None)

    for kw, message in ((dict(q=None), b"null pointer"), (dict(seq=None), b"null pointer"), (dict(pages=None), b"null pointer"), (dict(scale=0.0), b"scale"),
                        (dict(n=65, anc=x), b"num_nodes"), (dict(n=8193), b"bad shape"), (dict(hq=5), b"bad shape"), (dict(b=0), b"bad shape"),
                        (dict(q=y), b"aligned"), (dict(o=y), b"aligned")):
        assert call(**kw) != 0 and message in lib.fg_last_error() and b"fg_paged_attention_bf16_weights" in lib.fg_last_error(), (kw, lib.fg_last_error())


@pytest.mark.gpu
def test_the_model_asks_for_it(monkeypatch):
    """Forwards on pages round the weights as those on the contiguous cache do."""
    need_gpu()
    model = models.TargetModel.random(models.TargetConfig(1, 256, 4, 2, 128, 512, 512), seed=1, std=0.05, device=DEV)
    asked, call = [], K.paged_attention
    monkeypatch.setattr(K, "paged_attention", lambda *a, **kw: asked.append(kw["bf16_weights"]) or call(*a, **kw))
    model.prefill(torch.arange(20)[None], model.new_cache(1, 40, kv_format="bf16"))
    assert asked == [True]
