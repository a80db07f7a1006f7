"""KVPages are checked once: their attributes cannot be assigned, since what the kernels are given would not follow."""
import pytest
import torch

from flashgrpo_amd import kernels as K


def made(fmt="e4m3"):
    k, v = (torch.zeros(4, 2, 16, 64, dtype=torch.bfloat16) for _ in range(2))
    table = torch.zeros(2, 3, dtype=torch.int32)
    if fmt == "bf16":
        return K.KVPages(k, v, None, None, table), table
    k, v = (x.to(torch.float8_e4m3fn) for x in (k, v))
    return K.KVPages(k, v, *(torch.ones(4, 2, 16, 2, dtype=torch.uint8) for _ in range(2)), table), table


@pytest.mark.parametrize("fmt", ["e4m3", "bf16"])
def test_attributes_are_fixed(fmt):
    p, table = made(fmt)
    assert type(p) is K.KVPages and isinstance(p, K.KVPages) and p.table is table and "struct ``fg_kv_pages``" in K.KVPages.__doc__
    address = p.address
    for name in ("k", "v", "k_scales", "v_scales", "table", "format", "pages", "page_size", "kv_heads", "head_dim", "rows", "width", "device", "address",
                 "capacity", "another"):
        before = getattr(p, name, None)
        with pytest.raises(AttributeError, match="KVPages"):
            setattr(p, name, table.clone())
        with pytest.raises(AttributeError):
            delattr(p, name)
        assert getattr(p, name, None) is before or getattr(p, name, None) == before
    assert p.address == address
    table.fill_(3)  # the tensors' contents may change
    assert int(p.table[1, 2]) == 3
    assert {p: 1}[p] == 1 and p == p and p != made(fmt)[0]


def test_keywords_and_refusals_as_before():
    p, table = made()
    q = K.KVPages(k=p.k, v=p.v, k_scales=p.k_scales, v_scales=p.v_scales, table=table)
    assert (q.format, q.capacity) == (0, 48)
    with pytest.raises(ValueError):
        K.KVPages(p.k, p.v, None, None, table)
    with pytest.raises(TypeError):
        K.KVPages(p.k, p.v, table)


def test_copies_are_the_same():
    import copy

    p, _ = made()
    assert copy.copy(p) is p
