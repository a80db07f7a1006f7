"""How precise the MX products are: what a worst-case bound over long sums is too wide to see.

mx_gate_up_swiglu sums whole products in fp32, whatever the kernel: its 8-bit codes are compared with those of the 64-bit
value, exactly where the sums are exact in fp32, and by count on random rows."""
import numpy as np
import pytest
import torch

from oracle import mx as O
from test_gpu_mx import DEV, K, device_mx, device_pair, held

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


def code_of(value, fmt):
    return int(np.flatnonzero(O.TABLE[fmt] == abs(value))[0]) + (O.SIGN[fmt] if value < 0 else 0)


# one token, few and many rows; whole and split reductions
SIZES = [(1, 64, 512), (16, 416, 9632), (17, 160, 544), (20, 288, 4128), (33, 18944, 1536), (64, 288, 1056), (65, 96, 256),
         (130, 352, 384), (300, 1056, 2080), (1000, 2080, 288), (1856, 1792, 2080), (2311, 768, 5120), (4096, 1280, 1376)]


@pytest.mark.parametrize("rows,inter,k", SIZES)
@pytest.mark.parametrize("fmt", ["e4m3", "e2m1"])
@pytest.mark.parametrize("where", [0.0, 0.6, 1.0])
def test_gate_up_sums_small_products_beside_large_ones(rows, inter, k, fmt, where):
    """Gates of 2688 and 2432 (with a scale of 8, ties between two codes) and 2^-4 more, as much less, or no change; up is 1.
    Both are sums of products of eight neighbours, 2^-4 is 2^-14 of the largest one's powers of two, and the matrix instruction
    keeps 13 bits of such a sum. All sums are exact in fp32 and SiLU of such a gate is the gate, so the codes are those of the
    definition."""
    # values of x (e2m1: two blocks with scales of 2^6 and 2^-2, so 384, 64, 128 and 0.125, 1)
    large = {0: 6.0, 1: 1.0, 2: 2.0} if fmt == "e2m1" else {0: 448.0, 1: 384.0, 2: 128.0}
    small, one, at_small, at_one, span = (0.5, 4.0, 32, 33, 64) if fmt == "e2m1" else (0.125, 1.0, 3, 8, 32)
    k0 = int(where * (k - span)) // 32 * 32  # whole blocks, so that a scale is one part's
    x = np.zeros((rows, k), np.uint8)
    w = np.zeros((2 * inter, k), np.uint8)
    sx = np.zeros((-(-k // 128), rows, 4), np.uint8)
    sw = np.zeros((-(-k // 128), 2 * inter, 4), np.uint8)
    for b in range(k // 32):
        sx[b // 4, :, b % 4] = 127
        sw[b // 4, :, b % 4] = 127
    for m, v in large.items():
        x[:, k0 + m] = code_of(v, fmt)
    if fmt == "e2m1":
        b0, b1 = k0 // 32, k0 // 32 + 1
        sx[b0 // 4, :, b0 % 4], sx[b1 // 4, :, b1 % 4] = 127 + 6, 127 - 2
    sign = np.arange(rows) % 3 - 1
    for s in (-1, 1):
        x[sign == s, k0 + at_small] = code_of(s * small, fmt)
    x[:, k0 + at_one] = code_of(one, fmt)
    even = np.arange(inter) % 2 == 0
    gate, up = w[:inter], w[inter:]
    if fmt == "e2m1":  # 384 * 6 + 64 * 6 = 2688; 384 * 6 + 128 * 1 = 2432
        gate[:, k0] = code_of(6.0, fmt)
        gate[even, k0 + 1] = code_of(6.0, fmt)
        gate[~even, k0 + 2] = code_of(1.0, fmt)
    else:  # 448 * 6 = 2688; 384 * 6 + 128 * 1 = 2432
        gate[even, k0] = code_of(6.0, "e2m1")
        gate[~even, k0 + 1] = code_of(6.0, "e2m1")
        gate[~even, k0 + 2] = code_of(1.0, "e2m1")
    gate[:, k0 + at_small] = code_of(0.5, "e2m1")
    up[:, k0 + at_one] = code_of(1.0, "e2m1")
    xv, wv = O.values(x, sx, fmt), O.values(w, sw, "e2m1")
    g, u = xv[:, k0:k0 + span] @ wv[:inter, k0:k0 + span].T, xv[:, k0:k0 + span] @ wv[inter:, k0:k0 + span].T
    assert (u == 1).all() and set(np.unique(g)) <= {c + d for c in (2688.0, 2432.0) for d in (-0.0625, 0.0, 0.0625)}
    codes, scales = held(K().mx_gate_up_swiglu(device_mx(x, sx, fmt), device_mx(w, sw, "e2m1")))
    want_c, want_s = O.quantize(g, "e4m3")
    assert np.array_equal(scales, want_s)
    assert np.array_equal(codes, want_c), f"{int((codes != want_c).sum())} of {codes.size} codes differ"


@pytest.mark.parametrize("rows,inter,k", [(8, 8960, 1536), (17, 4096, 1536), (64, 2048, 3584), (130, 1056, 3584), (416, 608, 512),
                                          (700, 544, 1568), (2311, 768, 1024)])
def test_gate_up_codes_on_random_rows(rows, inter, k):
    """A sum of K products in two parts is cut 2 K / 64 times by at most a last bit, 2^-23 of it, half of that in the mean; gate,
    up and the activation's few operations so put a value off by less than d = 2 (K / 32 + 8) 2^-24 of itself. A border between
    two codes is within that of a value for at most 2 d / 2^-4 of them (codes are 2^-4 of a value apart, or more)."""
    (x, xv), (w, wv) = device_pair(rows, k, "e4m3", rows, spread=0.5), device_pair(2 * inter, k, "e2m1", k, k ** -0.5, 0.5)
    y = xv.double() @ wv.double().t()
    v = O.silu_mul(y[:, :inter].cpu().numpy(), y[:, inter:].cpu().numpy())
    want_c, want_s = O.quantize(v, "e4m3")
    codes, scales = held(K().mx_gate_up_swiglu(x, w))
    d = 2 * (k / 32 + 8) * 2.0 ** -24
    share = float((codes != want_c).mean())
    assert share <= 2 * d / 2.0 ** -4, f"{share:.2e} of the codes differ"
    assert (scales != want_s).mean() <= 32 * 2 * d  # a block's scale by its largest value
