"""Containers over one pool of pages (``container_copy``, ``clone_cache``): a row that one of them gives back, or makes a repeat of
another, has the length that its pages hold in all of them."""
import gc

import pytest
import torch

from flashgrpo_amd.models import PagedKVCache, TargetConfig
from flashgrpo_amd.models import qwen_flashgrpo_wrapper as W

CFG = TargetConfig(2, 64, 2, 2, 64, 128, 100)


def cache(lens, **kw):
    c = PagedKVCache(CFG, len(lens), 64, device="cpu", page_size=16, **kw)
    c.reserve(lens)
    c.seq_len.copy_(torch.tensor(lens))
    return c


def holds_its_tokens(c):
    """Every committed token has a page."""
    return all((c._rows[r, :-(-n // 16)] >= 0).all() for r, n in enumerate(c.seq_len.tolist()))


@pytest.mark.parametrize("other", [lambda c: W.clone_cache(c), lambda c: c.container_copy().container_copy()])
def test_release_by_one_of_them(other):
    c = cache([50, 20, 3])
    clone = other(c)
    clone.release([0])
    assert c.seq_len.tolist() == [0, 20, 3] == clone.seq_len.tolist() and holds_its_tokens(c) and holds_its_tokens(clone)
    clone.seq_len[1] = 25  # lengths are each container's own otherwise
    c.release([2, 2])
    assert c.seq_len.tolist() == [0, 20, 0] and clone.seq_len.tolist() == [0, 25, 0]
    assert c.free_pages == 10


def test_repeat_by_one_of_them():
    c = cache([50, 20, 3])
    clone = c.container_copy()
    clone.seq_len[1] = 5
    clone.repeat_rows(torch.tensor([1]), torch.tensor([0]))
    assert clone.seq_len.tolist() == [5, 5, 3] and c.seq_len.tolist() == [5, 20, 3]
    assert holds_its_tokens(c) and holds_its_tokens(clone)


def test_a_deep_copy_is_apart():
    c = cache([50, 20, 3])
    deep = W.clone_cache(c, clone_tensors=True)
    deep.release([0])
    deep.repeat_rows(torch.tensor([1]), torch.tensor([2]))
    assert c.seq_len.tolist() == [50, 20, 3] and deep.seq_len.tolist() == [0, 20, 20] and holds_its_tokens(c) and holds_its_tokens(deep)
    deep.container_copy().release([1])
    c.release([1])
    assert deep.seq_len.tolist() == [0, 0, 20] and c.seq_len.tolist() == [50, 0, 3]


def test_containers_are_not_kept():
    c = cache([50, 20, 3])
    clone = c.container_copy()
    del clone
    gc.collect()
    assert len(c._sharing) == 1
    c.release([0])
    assert c.seq_len.tolist() == [0, 20, 3]


def test_reserve_behind_committed_tokens_without_a_page():
    """Tokens that are committed but have no page are not given one, which would hold anything: refused, with nothing changed."""
    c = cache([20, 0, 40])
    c.seq_len[1] = 20              # never written
    c._drop(int(c._rows[2, 1]))    # tokens 16 .. 31 lost
    c._rows[2, 1] = -1
    before, free = c._rows.copy(), c.free_pages
    for call in (lambda: c.reserve(24, rows=[1], first=20), lambda: c.reserve([24, 24, 24], first=[20, 20, 40]), lambda: c.reserve(50, rows=[2], first=40),
                 lambda: c.reserve(50, rows=[2], first=17)):
        with pytest.raises(ValueError, match="committed tokens of row . have no page"):
            call()
        assert (c._rows == before).all() and c.free_pages == free
    c.reserve(50, rows=[2], first=16)  # what is about to be written needs no page yet
    c.reserve(24, rows=[1], first=0)
    c.reserve(30, rows=[0], first=25)  # a gap behind the committed tokens
    assert holds_its_tokens(c)


@pytest.mark.parametrize("fmt", ["bf16", "e4m3"])
def test_no_rows(fmt):
    """A cache of no rows, as the contiguous one has it: what is left when every sequence has ended."""
    c = cache([20, 0, 40], kv_format=fmt)
    none = W.select_cache_batch(c, torch.tensor([], dtype=torch.long))
    assert none.batch == 0 and none.seq_len.numel() == 0 and tuple(none.table.shape) == (0, 4)
    none.reserve(16)
    none.release([])
    none.repeat_rows(torch.tensor([], dtype=torch.long), torch.tensor([], dtype=torch.long))
    assert none.select_rows(torch.tensor([], dtype=torch.long)).batch == 0 and none.container_copy().deep_copy().batch == 0
