"""The scale of the bf16 tree attention's scores: positive and finite, every other one is refused (as in the paged attention: masked
scores are minus infinity times it). fp32 takes any."""
import ctypes
import os

import pytest
import torch

BAD = [0.0, -1.0, -1e-30, float("nan"), float("inf"), -float("inf"), 3e38, 1e-50]


def test_the_entry_point_refuses():
    from flashgrpo_amd import _lib

    if not os.path.exists(_lib.library_path()):
        pytest.skip("native library not built")
    lib = _lib.load()
    x = ctypes.c_void_p(1024)
    for scale in BAD:
        assert lib.fg_tree_attention(x, x, x, x, 1, 2, 1, 4, 2, 128, 64 * 128, 64 * 128, 64, x, None, None, 0, scale, None, 0, None) != 0
        assert b"scale must be positive" in lib.fg_last_error(), (scale, lib.fg_last_error())


def formula(q, k, v, committed, scale):
    """One sequence of one kv head: node n of a chain sees the committed tokens and new ones 0..n."""
    n = q.shape[1]
    s = torch.einsum("nhd,td->nht", q[0].double(), k[0, 0, :committed + n].double()) * scale
    sees = torch.arange(committed + n) <= committed + torch.arange(n)[:, None]
    return torch.softmax(s.masked_fill(~sees[:, None], -float("inf")), -1) @ v[0, 0, :committed + n].double()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,scales", [(torch.bfloat16, [1e-4, 0.3]), (torch.float32, [0.3, 0.0, -0.3])])
def test_what_is_taken(dtype, scales):
    """Of the largest |v|: bf16: 2^-8 for the weights, their sum and the output each. fp32: twice the error of the exponent, 136 roundings
    of 2^-24 of a score's sum of magnitudes (128 products of normal numbers: under 180)."""
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from flashgrpo_amd import kernels as K

    g = torch.Generator().manual_seed(1)
    q, k, v = (torch.randn(*s, generator=g).to(dtype) for s in ((1, 5, 4, 128), (1, 1, 128, 128), (1, 1, 128, 128)))
    for scale in scales:
        out = K.tree_attention(q.cuda(), k.cuda(), v.cuda(), seq_len=torch.tensor([70], dtype=torch.int32).cuda(), anc=None, num_nodes=5, q_heads=4,
                               kv_heads=1, head_dim=128, scale=scale)
        most = (2.0 ** -6 if dtype == torch.bfloat16 else 2 * 136 * 2.0 ** -24 * 0.3 * 180) * v.abs().max().item()
        assert ((out[0].cpu().double() - formula(q, k, v, 70, scale)).abs() <= most).all()


@pytest.mark.gpu
def test_the_wrapper_refuses():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from flashgrpo_amd import kernels as K

    q, c = torch.zeros(1, 1, 2, 128, dtype=torch.bfloat16, device="cuda"), torch.zeros(1, 1, 64, 128, dtype=torch.bfloat16, device="cuda")
    for scale in BAD:
        with pytest.raises((ValueError, RuntimeError), match="scale must be positive"):
            K.tree_attention(q, c, c, seq_len=torch.zeros(1, dtype=torch.int32, device="cuda"), anc=None, num_nodes=1, q_heads=2, kv_heads=1,
                             head_dim=128, scale=scale)
