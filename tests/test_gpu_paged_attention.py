"""Attention over a paged cache on the GPU against the float64 oracle (``oracle/paged.py``), within its derived bound."""
import numpy as np
import pytest
import torch

from paged_cases import DEV, Held, attention_oracle, close, i32, kernels, masks, queries, tree_words

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


def run(held, q, committed, words, *, fresh=None, row=None, out=None, scale=None):
    b, n, hq, d = q.shape
    return kernels().paged_attention(
        q.to(DEV), held.pages(), seq_len=i32(committed), anc=None if words is None else masks(words), num_nodes=n, q_heads=hq,
        kv_heads=held.heads, head_dim=d, out=out, new_len=None if fresh is None else i32(fresh),
        row_map=None if row is None else i32(row), scale=scale)


def check(held, q, committed, words, *, fresh=None, row=None):
    n, d = q.shape[1], q.shape[3]
    counts = [n] * q.shape[0] if fresh is None else fresh
    want = attention_oracle(held, q, committed, counts, words, d ** -0.5, row)
    out = torch.full(q.shape, 7.5, dtype=torch.bfloat16, device=DEV)
    assert run(held, q, committed, words, fresh=fresh, row=row, out=out) is out
    close(out, want, counts)
    for b, c in enumerate(counts):  # rows behind the sequence's tokens
        assert (out[b, c:] == 7.5).all()
    return out


HEADS = [(1, 1), (4, 4), (12, 2), (14, 2), (5, 1), (8, 1), (33, 1)]


@pytest.mark.parametrize("fmt", ["e4m3", "bf16"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("n", [1, 2, 9, 29, 64])
@pytest.mark.parametrize("heads", HEADS)
def test_trees(fmt, d, n, heads):
    hq, hkv = heads
    committed = [0, 1, 61, 130]
    held = Held(4, 4, 64, hkv, d, fmt, seed=n)
    words = [tree_words(n, 100 * n + b) for b in range(4)]
    check(held, queries(4, n, hq, d, n), committed, words)


@pytest.mark.parametrize("fmt", ["e4m3", "bf16"])
@pytest.mark.parametrize("size", [16, 32, 128, 256])
@pytest.mark.parametrize("n", [1, 13])
def test_page_sizes_and_lengths_about_a_tile(fmt, size, n):
    committed = [0, 15, 16, 63, 64, 65, 127, 128, 129, 191, 192, 255, 256, 257]
    b = len(committed)
    held = Held(b, -(-300 // size), size, 2, 128, fmt, seed=size)
    check(held, queries(b, n, 8, 128, 1), committed, None)
    check(held, queries(b, n, 8, 128, 2), committed, [tree_words(n, b) for b in range(b)])


@pytest.mark.parametrize("fmt", ["e4m3", "bf16"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("n", [3, 65, 130, 300])
def test_chains(fmt, d, n):
    committed = [0, 77]
    held = Held(2, -(-(77 + n) // 32), 32, 2, d, fmt, seed=n)
    check(held, queries(2, n, 6, d, n), committed, None)


@pytest.mark.parametrize("n", [1, 5, 40])
@pytest.mark.parametrize("hq", [2, 14])
def test_long_rows_in_parts(n, hq):
    committed = [2900, 0, 700, 1]
    held = Held(4, 47, 64, 2, 128, "e4m3", seed=3)
    words = [tree_words(n, b) for b in range(4)]
    check(held, queries(4, n, hq, 128, n), committed, words)
    check(held, queries(4, n, hq, 128, n + 1), committed, None)


@pytest.mark.parametrize("fmt", ["e4m3", "bf16"])
@pytest.mark.parametrize("chain", [True, False])
def test_padded_batch(fmt, chain):
    """new_len: rows behind a sequence's tokens stay as they were, and nobody sees their tokens."""
    n, fresh, committed = 37, [37, 0, 1, 20], [100, 50, 0, 300]
    held = Held(4, 22, 16, 2, 128, fmt, seed=5)
    words = None if chain else [[(1 << n) - 1] * n for _ in range(4)]
    check(held, queries(4, n, 4, 128, 1), committed, words, fresh=fresh)


@pytest.mark.parametrize("n", [1, 29])
def test_row_map(n):
    held = Held(5, 5, 32, 2, 128, "e4m3", seed=6)
    row = [3, 0, 4]
    check(held, queries(3, n, 8, 128, 3), [40, 100, 3], [tree_words(n, b) for b in range(3)], row=row)


def test_one_mask_list_for_all():
    n, committed = 21, [64, 30]
    held = Held(2, 2, 64, 2, 128, "e4m3", seed=7)
    w, q = tree_words(n, 1), queries(2, n, 4, 128, 1)
    one = kernels().paged_attention(q.to(DEV), held.pages(), seq_len=i32(committed), anc=masks([w])[0], num_nodes=n, q_heads=4,
                                    kv_heads=2, head_dim=128)
    assert torch.equal(one, run(held, q, committed, [w, w]))


@pytest.mark.parametrize("fmt", ["e4m3", "bf16"])
@pytest.mark.parametrize("n", [1, 13, 50])
def test_rows_that_see_nothing_are_zero(fmt, n):
    committed = [0, 0, 70]
    held = Held(3, 3, 64, 2, 128, fmt, seed=8)
    words = [[0] * n, [0] * (n - 1) + [1 << (n - 1)], [0] * n]
    out = check(held, queries(3, n, 8, 128, 4), committed, words)
    assert (out[0] == 0).all()


@pytest.mark.parametrize("fmt", ["e4m3", "bf16"])
@pytest.mark.parametrize("n", [1, 20])
def test_tokens_without_a_page_are_not_seen(fmt, n):
    committed = [300, 300, 140]
    held = Held(3, 11, 32, 2, 128, fmt, seed=9)
    held.table[0, 3], held.table[0, 0], held.table[1, 9] = -1, held.pages_n, 2 ** 31 - 1
    held.table[2] = -5
    held.upload()
    check(held, queries(3, n, 8, 128, 5), committed, [tree_words(n, b) for b in range(3)])
    check(held, queries(3, n, 8, 128, 5), committed, None)


@pytest.mark.parametrize("fmt", ["e4m3", "bf16"])
@pytest.mark.parametrize("value", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("hq", [2, 16])
def test_masked_infinities_and_nan_reach_nobody(fmt, value, hq):
    """K and V rows of tree nodes, and of slots behind the tokens, that are not finite: only nodes that see them show it."""
    n, committed = 12, [45, 200]
    held = Held(2, 5, 64, 2, 128, fmt, seed=10)
    words = [[1 << i for i in range(n)], tree_words(n, 3)]
    held.set_rows(0, 0, [45 + 3, 45 + n, 45 + n + 30], value)   # K of node 3, and behind the tokens
    held.set_rows(1, 0, [45 + 3, 45 + 7, 45 + n], value)        # V of nodes 3 and 7, and behind
    held.set_rows(1, 1, [200 + n - 1, 200 + n], value)
    held.upload()
    q = queries(2, n, hq, 128, 6)
    want = attention_oracle(held, q, committed, [n, n], words, 128 ** -0.5)
    out = run(held, q, committed, words)
    x = out.double().cpu().numpy()
    for i in range(n):
        if i not in (3, 7):
            assert np.isfinite(x[0, i]).all()
        if i < n - 1:
            assert np.isfinite(x[1, i]).all()
    assert np.isnan(x[0, 3]).all()
    # a whole row of V that is the same infinity: that infinity (bf16), or NaN where the format has no infinity
    assert np.isnan(x[0, 7]).all() if fmt == "e4m3" or np.isnan(value) else (x[0, 7] == value).all()
    keep = [i for i in range(n) if i not in (3, 7)]
    close(out[:1, keep], [(want[0][0][keep], want[0][1][keep])], [len(keep)])
    close(out[1:, :n - 1], [(want[1][0][:n - 1], want[1][1][:n - 1])], [n - 1])


def test_one_block_of_v_that_is_not_finite():
    """A NaN block of 32 elements (e4m3) and one infinite element (bf16) leave the other elements of V's row as they are."""
    for fmt in ("e4m3", "bf16"):
        held = Held(1, 2, 64, 1, 128, fmt, seed=11)
        t = 30
        p = held.table[0, 0]
        held.raw[1][p, 0, t, 40] = float("inf")
        held.refresh(1)
        held.upload()
        q = queries(1, 3, 4, 128, 7)
        out = run(held, q, [70], [[0b001, 0b011, 0b101]]).double().cpu().numpy()
        bad = np.isnan(out) if fmt == "e4m3" else out == np.inf
        want = np.zeros(128, bool)
        want[32:64 if fmt == "e4m3" else 33] = fmt == "e4m3"
        if fmt == "bf16":
            want[40] = True
        assert (bad == want).all() and np.isfinite(out[..., ~want]).all()


def test_large_scores():
    """Scores of tens of thousands, all but one weight vanishing: no overflow, the largest key's value."""
    held = Held(1, 3, 64, 1, 128, "e4m3", seed=12, spread=40.0)
    q = (40 * queries(1, 5, 4, 128, 8).float()).to(torch.bfloat16)
    check(held, q, [150], None)
