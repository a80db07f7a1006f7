"""Verify rounds with compaction on bf16 pages beside the contiguous cache, with the same tokens on both: what the caches hold, and what
follows from it."""
import numpy as np
import pytest
import torch

from flashgrpo_amd.models import TargetConfig, TargetModel

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(scope="module", autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


@pytest.fixture(scope="module")
def model():
    m = TargetModel.random(TargetConfig(2, 256, 4, 2, 128, 512, 512), seed=1, std=0.05, device=DEV)
    m.split_k_linear = False  # one projection on both caches
    return m


def tree(n):
    anc, pos = [1], [0]
    for i in range(1, n):
        p = (i - 1) // 2
        anc.append(anc[p] | 1 << i)
        pos.append(pos[p] + 1)
    return torch.tensor(anc, dtype=torch.int64, device=DEV), torch.tensor(pos, dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("page", [16, 64])
def test_rounds_beside_the_contiguous_cache(model, page):
    """Layer 0's K and V follow from tokens and positions alone: the same bits after every round, through repeats of a prompt, writes and
    moves. The hidden states and logits are off by the rounding of each layer's two branches, in the round and in the rounds that wrote
    the cache: 8 roundings of 2^-8 in each of 2 layers, twice."""
    n, rng = 13, np.random.default_rng(3)
    prompt, lens = torch.from_numpy(rng.integers(0, 512, (2, 70))), [70, 33]
    first = torch.tensor([0, 2], dtype=torch.int32, device=DEV)
    caches = model.new_cache(4, 160), model.new_cache(4, 160, kv_format="bf16", page_size=page)
    for c in caches:
        model.prefill(prompt, c, lengths=lens, chunk=40, row_map=first)
        c.repeat_rows(torch.tensor([0, 2], device=DEV), torch.tensor([1, 3], device=DEV))
    anc, pos = tree(n)
    most, rel = 32 * 2.0 ** -8, lambda x, y: ((x.float() - y.float()).norm() / y.float().norm()).item()
    for step in range(5):
        tok = torch.from_numpy(rng.integers(0, 512, (4, n))).to(DEV, torch.int32)
        nodes = torch.from_numpy(np.stack([[0, a, 2 * a + 1 + b] for a, b in rng.integers(1, 3, (4, 2)) - [0, 1]])).to(DEV, torch.int32)
        taken = torch.from_numpy(rng.integers(1, 4, 4)).to(DEV, torch.int32)
        hidden = []
        for c in caches:
            at = c.seq_len.cpu().numpy()
            c.reserve(at + n, first=at)
            hidden.append(model.forward(tok, c, pos_offset=pos, anc=anc).clone())
            c.gather_path(c.seq_len, nodes, taken, n)
            c.seq_len += taken
        assert rel(hidden[1], hidden[0]) < most
        assert rel(model.logits(hidden[1].reshape(4 * n, -1)), model.logits(hidden[0].reshape(4 * n, -1)).clone()) < most
        assert torch.equal(caches[0].seq_len, caches[1].seq_len)
        for l in range(2):
            for a, b in ((caches[0].k(l), caches[1].k(l)), (caches[0].v(l), caches[1].v(l))):
                for r, m in enumerate(caches[0].seq_len.tolist()):
                    assert torch.equal(a[r, :, :m], b[r, :, :m]) if l == 0 else rel(b[r, :, :m], a[r, :, :m]) < most
    assert caches[0].seq_len.min() > 33 + 4
