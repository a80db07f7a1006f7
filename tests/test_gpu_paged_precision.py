"""How exact the attention over a paged cache is, whatever the number of rows: weights in two bf16 parts, so that what is left is the
output's own rounding. Against the float64 oracle (``oracle/paged.py``)."""
import numpy as np
import pytest
import torch

from oracle import paged as O
from paged_cases import DEV, Held, close, i32, kernels, masks, queries, tree_words

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


def exact_weights(held, q, committed, words, scale):
    """Per sequence the oracle's (out, bound) with the bound of weights in two bf16 parts. Each part is rounded to nearest, 2^-9 of
    it: together they are off by 2^-18 of the weight, and 2^-16 covers the quotient, where the oracle allows 2^-8 for one part.
    Twice as many products are added: (tokens + 8) 2^-23 more."""
    got = []
    for b, c in enumerate(committed):
        n = q.shape[1]
        tokens = np.arange(c + n)
        (k, there), (v, _) = (O.rows_at(held.values[i], held.table[b], tokens) for i in range(2))
        o, e = O.attention(q[b].double().numpy(), k, v, there, c, n, None if words is None else words[b], scale)
        size, _ = O.attention(q[b].double().numpy(), k, np.abs(v), there, c, n, None if words is None else words[b], scale)
        got.append((o, e + ((len(tokens) + 8) * 2.0 ** -23 + 2.0 ** -16 - 2.0 ** -8) * (size + np.abs(o))))
    return got


def attend(held, q, committed, words, **kw):
    b, n, hq, d = q.shape
    return kernels().paged_attention(q.to(DEV), held.pages(), seq_len=i32(committed), anc=None if words is None else masks(words), num_nodes=n,
                                     q_heads=hq, kv_heads=held.heads, head_dim=d, **kw)


ROWS = [(2, 1), (4, 7), (4, 13), (4, 30), (5, 29), (7, 29), (2, 150)]  # 1 to 203 rows of a kv head, and two tiles of them


@pytest.mark.parametrize("fmt", ["e4m3", "bf16"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("group,n", ROWS)
def test_weights_keep_their_bits(fmt, d, group, n):
    committed = [330, 21]
    held = Held(2, -(-(330 + n) // 32), 32, 2, d, fmt, seed=n)
    words = None if n > 64 else [tree_words(n, i) for i in range(2)]
    q = queries(2, n, 2 * group, d, n)
    close(attend(held, q, committed, words), exact_weights(held, q, committed, words, d ** -0.5), [n, n])


@pytest.mark.parametrize("group,n", [(2, 1), (4, 29), (7, 29)])
def test_weights_of_parts_keep_their_bits(group, n):
    """Keys cut into parts whose results are joined."""
    committed = [2900, 700]
    held = Held(2, 46, 64, 1, 128, "e4m3", seed=3)
    q = queries(2, n, group, 128, n)
    close(attend(held, q, committed, None), exact_weights(held, q, committed, None, 128 ** -0.5), [n, n])


def test_parts_that_the_slots_limit():
    """A fixed number of parts is shared by the sequences of a call in proportion to their keys: one of 3000 keys is cut into more
    beside a short sequence than beside one of 2500, which changes the order of its sums (not the bound)."""
    held = Held(2, 47, 64, 16, 64, "e4m3", seed=5)
    q = queries(2, 1, 32, 64, 1)
    for committed in ([3000, 2500], [3000, 10], [3000, 3000], [2990, 1]):
        close(attend(held, q, committed, None), exact_weights(held, q, committed, None, 64 ** -0.5), [1, 1])
