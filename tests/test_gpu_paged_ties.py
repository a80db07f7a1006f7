"""The e4m3 codes of K next to ties: K is rotated in 64 bits, rounded to fp32 and quantised from there, so that a code is the 64-bit
definition's wherever the value is more than an fp32 rounding away from a tie, and follows the fp32 value there."""
import numpy as np
import pytest
import torch

from oracle import mx, paged as O
from paged_cases import DEV, Held, i32, kernels

pytestmark = pytest.mark.gpu
D, POSITIONS = 128, range(1, 13)


@pytest.fixture(scope="module", autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


def inv_freq():
    return 1.0 / 1.0e6 ** (torch.arange(0, D, 2).float() / D)


def near_ties(position):
    """Rows [tokens, D] of bf16 values whose rotation by ``position`` rounds in fp32 to a tie of e4m3 that it is not: y = x1 cos - x2 sin
    in [1, 2), where codes are 1/8 apart, in a block whose scale is 1 (element 31 is about 256)."""
    x1 = (128 + np.arange(128)) / 128.0
    x2 = np.concatenate([-x1, x1])
    rows = []
    for i in range(24):
        a = position * np.float64(inv_freq().numpy()[i])
        y = x1[:, None] * np.cos(a) - x2[None] * np.sin(a)
        f = y.astype(np.float32).astype(np.float64)
        for j, k in np.argwhere((f != y) & (np.abs(y) >= 1) & (np.abs(y) < 2) & (np.abs(f * 16) % 2 == 1)):
            row = np.zeros(D)
            row[i], row[i + 64], row[31] = x1[j], x2[k], 256.0
            rows.append(row)
    return np.array(rows).reshape(-1, D)


def test_codes_next_to_ties():
    rng = np.random.default_rng(0)
    found = 0
    for position in POSITIONS:
        rows = np.concatenate([near_ties(position), rng.standard_normal((40, D))])
        x = torch.from_numpy(rows).to(torch.bfloat16)
        n = len(rows)
        held = Held(n, 1, 16, 1, D, "e4m3", seed=position)
        qkv = torch.cat([x, x, x], 1).to(DEV)
        q = torch.empty(n, 1, 1, D, dtype=torch.bfloat16, device=DEV)
        kernels().rope_kv_write_paged(qkv, held.pages(), batch=n, num_nodes=1, q_heads=1, kv_heads=1, head_dim=D, seq_len=i32([position] * n),
                                      pos_offset=i32([0]), inv_freq=inv_freq().to(DEV), q_out=q)
        k = O.rotate(x.double().numpy()[:, None], [position] * n, inv_freq().numpy())[:, 0]
        page = held.table[:, 0]
        codes, scales = held.k.view(torch.uint8).cpu().numpy()[page, 0, position], held.ks.cpu().numpy()[page, 0, position]
        rounded, exact = O.quantize(k.astype(np.float32)), O.quantize(k)
        assert (codes == rounded[0]).all() and (scales == rounded[1]).all() and (scales == exact[1]).all()
        for r, c in np.argwhere(codes != exact[0]):
            f = np.exp2(float(scales[r, c // mx.BLOCK]) - 127)
            tie = O.values(np.array([[codes[r, c], exact[0][r, c]] + [0] * 30], np.uint8), np.array([[127]], np.uint8))[0, :2].mean()
            assert abs(k[r, c] / f - tie) <= 2.0 ** -24 * abs(k[r, c] / f)
            found += 1
    assert found
