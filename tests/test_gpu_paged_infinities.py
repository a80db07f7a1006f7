"""Attention over bf16 pages whose V holds an infinity or a NaN in one element of a row: the row's other elements count as they are
(float64 oracle, ``oracle/paged.py``)."""
import numpy as np
import pytest
import torch

from oracle import paged as O
from paged_cases import Held, attention_oracle, close, i32, kernels, masks, queries, tree_words

pytestmark = pytest.mark.gpu
ROWS = [(2, 1), (4, 7), (4, 13), (4, 30), (5, 29), (7, 29), (2, 150)]  # 1 to 300 rows of a kv head: every row layout


@pytest.fixture(scope="module", autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


def put(held, token, d, value):
    held.raw[1][O.page_of(held.table[0], token, held.size, held.pages_n), 0, token % held.size, d] = value


def check(held, committed, group, n, words):
    q = queries(1, n, group, 128, n)
    out = kernels().paged_attention(q.cuda(), held.pages(), seq_len=i32([committed]), anc=None if words is None else masks([words]), num_nodes=n,
                                    q_heads=group, kv_heads=1, head_dim=128)
    with np.errstate(invalid="ignore"):
        close(out, attention_oracle(held, q, [committed], [n], None if words is None else [words], 128 ** -0.5), [n])
    return out[0].float().cpu()


@pytest.mark.parametrize("group,n", ROWS)
@pytest.mark.parametrize("committed", [130, 700])
def test_elements_that_every_row_sees(group, n, committed):
    """An infinity is that infinity in its dim of every row, a NaN a NaN, the other dims are those of the finite elements."""
    held = Held(1, -(-(committed + n) // 32), 32, 1, 128, "bf16", seed=n)
    for t, d, x in ((5, 40, np.inf), (committed - 1, 7, np.nan), (committed // 2, 99, -np.inf)):
        put(held, t, d, x)
    held.refresh(1)
    held.upload()
    x = check(held, committed, group, n, None if n > 64 else tree_words(n, 1))
    assert (x[..., 40] == np.inf).all() and (x[..., 99] == -np.inf).all() and torch.isnan(x[..., 7]).all()


@pytest.mark.parametrize("group,n", [r for r in ROWS if 1 < r[1] <= 64])
@pytest.mark.parametrize("committed", [0, 61])
def test_elements_that_some_rows_see(group, n, committed):
    """Of a new token: who sees it has the infinity in its dim and the token's finite elements in the others."""
    held = Held(1, 5, 32, 1, 128, "bf16", seed=n)
    put(held, committed + 2, 64, np.inf)
    put(held, committed + 2, 71, np.nan)
    held.refresh(1)
    held.upload()
    words = tree_words(n, 3)
    x = check(held, committed, group, n, words)
    sees = torch.tensor([bool(w >> 2 & 1) for w in words])
    assert sees.any() and not sees.all()
    assert torch.equal(x[..., 64].isinf(), sees[:, None].expand(n, group)) and torch.equal(x[..., 71].isnan(), sees[:, None].expand(n, group))
