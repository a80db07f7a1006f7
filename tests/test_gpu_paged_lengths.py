"""Batches of unlike lengths over a paged cache: how a sequence's keys are cut into parts, and which sequence goes first, changes
no row (float64 oracle, ``oracle/paged.py``)."""
import functools

import numpy as np
import pytest
import torch

from paged_cases import DEV, Held, attention_oracle, close, i32, kernels, masks, queries, tree_words

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


def check(held, n, hq, committed, *, trees=False, fresh=None, seed=0):
    b, d = len(committed), held.d
    q = queries(b, n, hq, d, seed)
    counts = [n] * b if fresh is None else fresh
    words = [tree_words(n, i) for i in range(b)] if trees else None
    out = torch.full(q.shape, 7.5, dtype=torch.bfloat16, device=DEV)
    for _ in range(2):  # (the second call finds the first's workspace)
        kernels().paged_attention(q.to(DEV), held.pages(), seq_len=i32(committed), anc=masks(words) if trees else None, out=out,
                                  num_nodes=n, q_heads=hq, kv_heads=held.heads, head_dim=d,
                                  new_len=None if fresh is None else i32(fresh))
    close(out, attention_oracle(held, q, committed, counts, words, d ** -0.5, None), counts)
    for i, c in enumerate(counts):
        assert (out[i, c:] == 7.5).all()


def lengths(kind, b, most, rng):
    if kind == "one long":
        return [most] + [int(x) for x in rng.integers(0, 40, b - 1)]
    if kind == "last long":
        return [int(x) for x in rng.integers(0, 40, b - 1)] + [most]
    if kind == "none":
        return [0] * b
    if kind == "equal":
        return [most // 2] * b
    return [int(x) for x in rng.integers(0, most + 1, b)]


@functools.lru_cache(2)
def held_rows(b, width, hkv, d):
    return Held(b, width, 32, hkv, d, "e4m3", seed=b)


@pytest.mark.parametrize("b,n,hq,d", [(b, *s) for b in (1, 7, 64, 65) for s in ((1, 2, 128), (9, 4, 64), (29, 7, 128)) if b < 64 or s[0] < 29])
@pytest.mark.parametrize("kind", ["one long", "last long", "none", "equal", "any"])
def test_parts(b, n, hq, d, kind):
    most = 2500 if b <= 7 else 1100
    committed = lengths(kind, b, most, np.random.default_rng([b, n]))
    check(held_rows(b, -(-(most + n) // 32), 1, d), n, hq, committed, trees=n > 1, seed=b)


@pytest.mark.parametrize("b", [3, 64])
def test_parts_of_a_padded_batch(b):
    rng = np.random.default_rng(b)
    committed, fresh = lengths("any", b, 700, rng), [int(x) for x in rng.integers(0, 14, b)]
    fresh[0], committed[0] = 0, 700   # the longest asks for nothing
    check(Held(b, 23, 32, 1, 128, "bf16", seed=1), 13, 5, committed, fresh=fresh)


@pytest.mark.parametrize("n,hq", [(1, 1), (11, 3)])
@pytest.mark.parametrize("b,hkv", [(257, 1), (129, 2), (512, 1), (513, 1), (33, 8)])
@pytest.mark.parametrize("kind", ["one long", "equal", "any"])
def test_longest_first(n, hq, b, hkv, kind):
    rng = np.random.default_rng([b, n])
    committed = lengths(kind, b, 120, rng)
    fresh = [int(x) for x in rng.integers(0, n + 1, b)] if kind == "any" else None
    check(held_rows(b, 5, hkv, 64), n, hq * hkv, committed, trees=n > 1 and kind == "equal", fresh=fresh)


@pytest.mark.parametrize("b,hkv,hq,n", [(1, 1, 64, 520), (9, 3, 12, 330), (9, 8, 8, 520)])
def test_row_tiles_in_order(b, hkv, hq, n):
    """Chains of more row tiles than CUs: the order in which they run has each of them once."""
    committed = lengths("any", b, 100, np.random.default_rng(hkv))
    fresh = None if b == 1 else [n - 30 * i for i in range(b)]
    check(Held(b, -(-(n + 100) // 64), 64, hkv, 64, "e4m3", seed=1), n, hq, committed, fresh=fresh)


@pytest.mark.parametrize("fmt", ["e4m3", "bf16"])
@pytest.mark.parametrize("hq", [4, 5, 6, 7, 9])
def test_pages_that_are_missing_whatever_the_rows(fmt, hq):
    n, committed = 29, [300, 127, 140]
    held = Held(3, 11, 32, 1, 128, fmt, seed=hq)
    held.table[0, 3], held.table[0, 0], held.table[1, 4] = -1, held.pages_n, 2 ** 31 - 1
    held.table[2] = -5
    held.upload()
    check(held, n, hq, committed, trees=True, seed=hq)
    check(held, n, hq, committed, seed=hq)


@pytest.mark.parametrize("fmt", ["e4m3", "bf16"])
@pytest.mark.parametrize("hq", [4, 5, 6, 7, 9])
@pytest.mark.parametrize("committed", [3, 40, 64, 95])
def test_values_that_are_not_finite_whatever_the_rows(fmt, hq, committed):
    """V of node 3, and of the slot behind the nodes, is NaN or infinite: who sees node 3 shows it, nobody else does."""
    n, d = 29, 128
    held = Held(1, 4, 32, 1, d, fmt, seed=hq)
    held.set_rows(1, 0, [committed + 3], float("inf"))
    if committed + n < 128:
        held.set_rows(1, 0, [committed + n], float("nan"))
    held.upload()
    words = [tree_words(n, committed)]
    q = queries(1, n, hq, d, 1)
    out = kernels().paged_attention(q.to(DEV), held.pages(), seq_len=i32([committed]), anc=masks(words), num_nodes=n, q_heads=hq,
                                    kv_heads=1, head_dim=d)
    sees = np.array([w >> 3 & 1 for w in words[0]], bool)
    assert sees.any() and not sees.all()
    x = out[0].double().cpu().numpy()
    assert (np.isnan(x[sees]) if fmt == "e4m3" else x[sees] == np.inf).all()
    keep = [i for i in range(n) if not sees[i]]
    want = attention_oracle(held, q, [committed], [n], words, d ** -0.5, None)
    close(out[:, keep], [(want[0][0][keep], want[0][1][keep])], [len(keep)])
