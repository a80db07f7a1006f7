"""The scale of the attention's scores: any positive finite one gives the formula's result, every other one is refused (masked
scores are minus infinity times it, and the running maximum is that of scaled scores)."""
import ctypes
import os

import pytest
import torch

from flashgrpo_amd import kernels as K

BAD = [0.0, -0.0, -1.0, -1e-30, float("nan"), float("inf"), -float("inf"), 3e38, 1e-50]  # (3e38: not finite times log2 e; 1e-50: 0 in fp32)


def test_the_entry_point_refuses():
    from flashgrpo_amd import _lib

    if not os.path.exists(_lib.library_path()):
        pytest.skip("native library not built")
    lib = _lib.load()
    s = _lib.KvPages(4096, 8192, 64, 128, 256, 2 * 16 * 128, 2 * 16 * 4, 3, 0, 4, 16, 2, 128, 2, 3)
    x = ctypes.c_void_p(1024)
    for scale in BAD:
        assert lib.fg_paged_attention(x, x, ctypes.addressof(s), 2, 1, 4, x, None, None, None, 0, scale, None, 0, None) != 0
        assert b"scale must be positive" in lib.fg_last_error(), (scale, lib.fg_last_error())


def need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


@pytest.mark.gpu
def test_the_wrapper_refuses():
    need_gpu()
    from paged_cases import Held, i32

    held = Held(1, 2, 32, 1, 128, "e4m3", seed=1)
    q = torch.zeros(1, 1, 2, 128, dtype=torch.bfloat16, device="cuda")
    out = torch.full_like(q, 7.0)
    for scale in BAD:
        with pytest.raises((ValueError, RuntimeError), match="scale must be positive"):
            K.paged_attention(q, held.pages(), seq_len=i32([20]), anc=None, num_nodes=1, q_heads=2, kv_heads=1, head_dim=128, out=out, scale=scale)
    torch.cuda.synchronize()
    assert (out == 7.0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["e4m3", "bf16"])
@pytest.mark.parametrize("scale", [1e-40, 1e-4, 0.3, 1.0, 5.0])
@pytest.mark.parametrize("group,n,committed", [(2, 1, [0, 200]), (4, 13, [0, 200]), (7, 29, [33, 200]), (2, 1, [3000, 70])])
def test_any_positive_scale(fmt, scale, group, n, committed):
    """Both kernels, keys whole and in parts, against the oracle."""
    need_gpu()
    from paged_cases import Held, attention_oracle, close, i32, masks, queries, tree_words

    held = Held(2, -(-(max(committed) + n) // 32), 32, 1, 128, fmt, seed=n)
    words = [tree_words(n, i) for i in range(2)]
    q = queries(2, n, group, 128, n)
    out = K.paged_attention(q.cuda(), held.pages(), seq_len=i32(committed), anc=masks(words), num_nodes=n, q_heads=group, kv_heads=1, head_dim=128,
                            scale=scale)
    close(out, attention_oracle(held, q, committed, [n, n], words, scale), [n, n])
