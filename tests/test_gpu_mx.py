"""Microscaled rows on the GPU against the float64 oracle (``oracle/mx.py``).

Quantisation, values and the norm are compared bit for bit. The products are held to a bound derived from what the
scaled matrix instruction does with its operands: products of two e2m1 codes are exact and summed with at least 24 bits;
with an e4m3 operand the products of 8 neighbouring elements are cut to multiples of 2^-13 of the power of two below the
largest of them. So a sum is off by at most 7 * 2^-13 of the largest product of each group of 8 (e4m3), plus 9 cuts of
2^-23 of the sum of magnitudes per 64 elements, plus the sum over splits; the bf16 result by half a step, 2^-8 of it.
"""
import numpy as np
import pytest
import torch

from oracle import mx as O

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(scope="module", autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


def K():
    from flashgrpo_amd import kernels

    return kernels


def rows_of(rows, cols, seed, dtype=torch.bfloat16, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, cols, generator=g) * torch.exp(spread * torch.randn(rows, cols // 32, generator=g)).repeat_interleave(32, 1)
    return x.to(dtype)


def random_mx(rows, cols, fmt, seed):
    """An MX pair of a spread of magnitudes, and its float64 values."""
    codes, scales = O.quantize(rows_of(rows, cols, seed).double().numpy(), fmt)
    return device_mx(codes, scales, fmt), O.values(codes, scales, fmt)


def device_mx(codes, scales, fmt):
    c = torch.from_numpy(np.ascontiguousarray(O.pack(codes, fmt))).to(DEV)
    return K().MX(c if fmt == "e2m1" else c.view(torch.float8_e4m3fn), torch.from_numpy(scales).to(DEV))


def held(q):
    """(codes one to an element, scales) of an MX pair on the host."""
    return O.unpack(q.codes.view(torch.uint8).cpu().numpy(), q.format), q.scales.cpu().numpy()


def host(q):
    return O.values(*held(q), q.format)


# ------------------------------------------------------------------ quantisation
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("fmt", ["e4m3", "e2m1"])
@pytest.mark.parametrize("rows,cols", [(1, 32), (1, 3584), (3, 96), (16, 512), (17, 544), (33, 160), (130, 1184)])
def test_quantize_is_the_oracle_bit_for_bit(rows, cols, fmt, dtype):
    x = rows_of(rows, cols, rows + cols, dtype, spread=3.0)
    codes, scales = held(K().mx_quantize(x.to(DEV), fmt))
    want_c, want_s = O.quantize(x.double().numpy(), fmt)
    assert np.array_equal(scales, want_s)
    assert np.array_equal(codes, want_c)


@pytest.mark.parametrize("fmt", ["e4m3", "e2m1"])
def test_quantize_borders(fmt):
    """Ties, block maxima at and next to a scale's border, zeros, subnormals, the ends of fp32's range."""
    big = O.LARGEST[fmt]
    rng = np.random.default_rng(0)
    blocks = [np.zeros(32), np.full(32, -0.0)]
    for n in (-130, -126, -20, 0, 7, 115):
        for edge in (1.0, 1 - 2.0 ** -23, 1 + 2.0 ** -22):
            b = rng.uniform(-1, 1, 32) * big * 2.0 ** n
            b[3] = big * edge * 2.0 ** n
            blocks.append(b)
        t = O.TABLE[fmt]
        mids = (t[1:] + t[:-1]) / 2 * 2.0 ** n
        for i in range(0, len(mids), 31):
            b = np.zeros(32)
            m = mids[i:i + 31]
            b[:len(m)] = m * np.where(np.arange(len(m)) % 2, -1, 1)
            b[31] = big * 2.0 ** n
            blocks.append(b)
    blocks.append(np.full(32, 3.4028234663852886e38))
    blocks.append(rng.uniform(-1, 1, 32) * 1e-44)
    x = torch.from_numpy(np.stack(blocks).astype(np.float32))
    codes, scales = held(K().mx_quantize(x.to(DEV), fmt))
    want_c, want_s = O.quantize(x.double().numpy(), fmt)
    assert np.array_equal(scales, want_s)
    assert np.array_equal(codes, want_c)


@pytest.mark.parametrize("fmt", ["e4m3", "e2m1"])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_a_block_with_a_non_finite_element_is_nan_and_no_other(fmt, bad):
    x = rows_of(5, 160, 3)
    x[2, 70] = bad
    q = K().mx_quantize(x.to(DEV), fmt)
    v, w = host(q), K().mx_dequantize(q, torch.float32).cpu().numpy()
    nan = np.zeros((5, 160), bool)
    nan[2, 64:96] = True
    assert np.array_equal(np.isnan(v), nan) and np.array_equal(np.isnan(w), nan)
    clean = x.clone()
    clean[2, 64:96] = 0
    assert np.array_equal(v[~nan], host(K().mx_quantize(clean.to(DEV), fmt))[~nan])


def test_quantize_strided_rows_and_in_place_pair():
    x = torch.randn(9, 320, device=DEV).to(torch.bfloat16)
    q = K().mx_quantize(x[:, 64:224], "e2m1")
    want = K().mx_quantize(x[:, 64:224].contiguous(), "e2m1")
    assert torch.equal(q.codes, want.codes) and torch.equal(q.scales, want.scales)
    again = K().mx_quantize(x[:, :160], "e2m1", out=q)
    assert again.codes.data_ptr() == q.codes.data_ptr()
    want = K().mx_quantize(x[:, :160].contiguous(), "e2m1")
    assert torch.equal(q.codes, want.codes) and torch.equal(q.scales, want.scales)


@pytest.mark.parametrize("fmt", ["e4m3", "e2m1"])
@pytest.mark.parametrize("rows,cols", [(1, 32), (19, 416), (64, 1024)])
def test_dequantize_every_code_and_scale(fmt, rows, cols):
    g = np.random.default_rng(rows)
    codes = g.integers(0, 2 * O.SIGN[fmt], (rows, cols)).astype(np.uint8)
    scales = g.integers(0, 256, (-(-cols // 128), rows, 4)).astype(np.uint8)
    v = O.values(codes, scales, fmt)
    q = device_mx(codes, scales, fmt)
    with np.errstate(over="ignore"):
        want = torch.from_numpy(v.astype(np.float32))
    got = K().mx_dequantize(q, torch.float32).cpu()
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(nan=1.0, posinf=9e9), want.nan_to_num(nan=1.0, posinf=9e9))
    got = K().mx_dequantize(q).cpu()
    want = want.to(torch.bfloat16)
    assert torch.equal(got.isnan(), want.isnan())
    assert torch.equal(got.nan_to_num(nan=1.0).view(torch.int16), want.nan_to_num(nan=1.0).view(torch.int16))


def test_no_rows():
    k = K()
    x = torch.empty(0, 64, dtype=torch.bfloat16, device=DEV)
    q = k.mx_quantize(x, "e4m3")
    w, _ = random_mx(64, 64, "e2m1", 0)
    assert q.codes.shape == (0, 64) and q.scales.shape == (1, 0, 4)
    assert k.mx_dequantize(q).shape == (0, 64)
    assert k.rmsnorm_mx(x, torch.ones(64, dtype=torch.bfloat16, device=DEV), 1e-6).codes.shape == (0, 64)
    assert k.mx_linear(q, w).shape == (0, 64) and k.mx_gate_up_swiglu(q, w).codes.shape == (0, 32)


# ------------------------------------------------------------------ norm
def norm_oracle(x, weight, eps, delta):
    s = x if delta is None else (x.float() + delta.float()).to(x.dtype)
    return s, O.quantize(O.rmsnorm(s.double().numpy(), weight.double().numpy(), eps), "e4m3")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("delta", [False, True])
@pytest.mark.parametrize("rows,cols", [(1, 32), (5, 160), (3, 1536), (2, 2080), (17, 3584), (4, 8192)])
def test_rmsnorm_codes_are_the_formulas(rows, cols, delta, dtype):
    x, d = rows_of(rows, cols, cols, dtype), rows_of(rows, cols, cols + 1, dtype)
    w = (1 + 0.2 * torch.randn(cols, generator=torch.Generator().manual_seed(cols))).to(dtype)
    eps = float(np.float32(1e-6))
    s, (want_c, want_s) = norm_oracle(x, w, eps, d if delta else None)
    xg = x.to(DEV)
    total = torch.full_like(xg, 7.0) if delta else None
    q = K().rmsnorm_mx(xg, w.to(DEV), 1e-6, delta=d.to(DEV) if delta else None, sum_out=total)
    codes, scales = held(q)
    assert np.array_equal(scales, want_s) and np.array_equal(codes, want_c)
    assert torch.equal(xg.cpu(), x)
    if delta:
        assert torch.equal(total.cpu(), s)
        q2 = K().rmsnorm_mx(xg, w.to(DEV), 1e-6, delta=d.to(DEV))  # into x itself
        assert torch.equal(xg.cpu(), s) and torch.equal(q2.scales, q.scales)
        assert torch.equal(q2.codes.view(torch.uint8), q.codes.view(torch.uint8))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("eps", [0.0, 1e-10, 3e-8])
def test_rmsnorm_next_to_ties(eps, dtype):
    """Rows of +-1 have a mean square of 1: the norm is the weight itself, an eighth of whose values are ties between
    two codes, or a part in 10^10 less, which 32 bits cannot hold and which takes a tie to the smaller magnitude."""
    g = torch.Generator().manual_seed(4)
    cols = 4096
    x = (torch.randint(0, 2, (9, cols), generator=g) * 2 - 1).to(dtype)
    w = torch.exp(torch.randn(cols, generator=g)).to(torch.bfloat16).to(dtype)
    want_c, want_s = O.quantize(O.rmsnorm(x.double().numpy(), w.double().numpy(), float(np.float32(eps))), "e4m3")
    codes, scales = held(K().rmsnorm_mx(x.to(DEV), w.to(DEV), eps))
    assert np.array_equal(scales, want_s) and np.array_equal(codes, want_c)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rmsnorm_codes_of_many_values(dtype):
    """Enough values for those that 32-bit arithmetic would round differently (one in a million) to be among them."""
    x = rows_of(1500, 4096, 11, dtype, spread=0.3)
    w = (1 + 0.2 * torch.randn(4096, generator=torch.Generator().manual_seed(1))).to(dtype)
    want_c, want_s = O.quantize(O.rmsnorm(x.double().numpy(), w.double().numpy(), float(np.float32(1e-6))), "e4m3")
    codes, scales = held(K().rmsnorm_mx(x.to(DEV), w.to(DEV), 1e-6))
    assert np.array_equal(scales, want_s) and np.array_equal(codes, want_c)


def test_rmsnorm_special_rows():
    """A row of zeros, one with an infinity, one with a NaN, tiny and huge rows; the others are as without them."""
    x = rows_of(7, 256, 5, torch.float32)
    x[1] = 0
    x[2, 40] = float("inf")
    x[3, 200] = float("nan")
    x[4] *= 1e-30
    x[5] *= 1e18
    w = torch.ones(256)
    q = K().rmsnorm_mx(x.to(DEV), w.to(DEV), 1e-6)
    v = host(q)
    assert (v[1] == 0).all() and np.isnan(v[3]).all()
    assert np.isnan(v[2, 32:64]).all() and (v[2, :32] == 0).all() and (v[2, 64:] == 0).all()
    fine = [0, 4, 5, 6]
    want_c, want_s = O.quantize(O.rmsnorm(x[fine].double().numpy(), w.double().numpy(), float(np.float32(1e-6))), "e4m3")
    codes, scales = held(q)
    assert np.array_equal(codes[fine], want_c) and np.array_equal(scales[:, fine], want_s)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("size", [2.0 ** -149, 2.0 ** -126, 1e-30, 1e-19, 1e19, 1e30, 2.0 ** 124])
def test_rmsnorm_near_the_ends_of_the_type(size, dtype):
    """Rows so small or large that the norm's factor (eps 0) or its rounding error has no place in 32 bits."""
    x = rows_of(40, 2080, 21, torch.float32, spread=0.2).clamp(-8, 8)
    x = (x.double() * size).to(dtype)
    x[:, 0] = size
    w = torch.exp(torch.randn(2080, generator=torch.Generator().manual_seed(2))).to(dtype)
    want_c, want_s = O.quantize(O.rmsnorm(x.double().numpy(), w.double().numpy(), 0.0), "e4m3")
    codes, scales = held(K().rmsnorm_mx(x.to(DEV), w.to(DEV), 0.0))
    assert np.array_equal(scales, want_s)  # (bf16 rows of 2^-149 are zeros: 0 / 0, NaN blocks, whose codes are free)
    assert np.array_equal(O.values(codes, scales, "e4m3"), O.values(want_c, want_s, "e4m3"), equal_nan=True)


# ------------------------------------------------------------------ products
def product_bound(xv, wv, fmt):
    """How far a product's fp32 sums may be off (see the head of this file), and the exact products."""
    k = xv.shape[1]
    x, w = torch.from_numpy(xv).to(DEV), torch.from_numpy(wv).to(DEV)
    exact, mags = x @ w.t(), x.abs() @ w.abs().t()
    err = (k / 64 + 1) * 9 * 2.0 ** -23 * mags + 256 * 2.0 ** -24 * mags
    if fmt == "e4m3":
        big = torch.zeros_like(exact)
        for g in range(0, k, 8):
            big += (x[:, None, g:g + 8] * w[None, :, g:g + 8]).abs().amax(-1)
        err += 7 * 2.0 ** -13 * big
    return exact, err


def check_linear(got, exact, err, bias=None, residual=None):
    ref = exact
    if bias is not None:
        ref = ref + bias.double()
        err = err + 2.0 ** -23 * (exact.abs() + bias.double().abs())
    if residual is not None:
        ref = ref + residual.double()
        err = err + 2.0 ** -23 * (exact.abs() + residual.double().abs() + (0 if bias is None else bias.double().abs()))
    far = (got.double() - ref).abs() - (2.0 ** -8 * ref.abs() + (1 + 2.0 ** -8) * err + 1e-38)
    assert not got.isnan().any()
    assert float(far.max()) <= 0, f"worst {float(far.max())} over the bound at {int(far.argmax())}"


SHAPES = [(1, 1, 32), (1, 2048, 1536), (2, 33, 96), (5, 77, 160), (15, 130, 512), (16, 64, 544), (17, 129, 640), (31, 256, 1184),
          (64, 200, 2048), (65, 384, 288), (129, 257, 416), (200, 513, 1056), (257, 300, 384), (300, 700, 128),
          # long reductions over few tiles (split over workgroups), and outputs of every tile size
          (8, 16400, 160), (9, 50, 8192), (40, 300, 9600), (130, 520, 6016), (400, 1031, 4448), (700, 2050, 1120),
          (1030, 4100, 576), (1900, 6000, 160)]


@pytest.mark.parametrize("fmt", ["e4m3", "e2m1"])
@pytest.mark.parametrize("rows,n,k", SHAPES)
def test_linear_matches_float64(rows, n, k, fmt):
    x, xv = random_mx(rows, k, fmt, rows + k)
    w, wv = random_mx(n, k, "e2m1", n + k + 1)
    exact, err = product_bound(xv, wv, fmt)
    check_linear(K().mx_linear(x, w), exact, err)


@pytest.mark.parametrize("rows,n,k", [(1, 40, 160), (3, 2048, 1536), (70, 129, 256), (130, 264, 1024)])
def test_linear_bias_residual_strides_and_in_place(rows, n, k):
    g = torch.Generator(device=DEV).manual_seed(rows)
    x, xv = random_mx(rows, k, "e4m3", rows)
    w, wv = random_mx(n, k, "e2m1", n)
    exact, err = product_bound(xv, wv, "e4m3")
    scale = float(exact.abs().mean())
    bias = (scale * torch.randn(n, device=DEV, generator=g)).to(torch.bfloat16)
    res = (scale * torch.randn(rows, n + 24, device=DEV, generator=g)).to(torch.bfloat16)
    check_linear(K().mx_linear(x, w, bias=bias), exact, err, bias)
    for off in (0, 3, 8):  # rows that start anywhere
        r = res[:, off:off + n]
        plain = K().mx_linear(x, w, bias=bias, residual=r)
        check_linear(plain, exact, err, bias, r)
        wide = torch.full((rows + 2, n + 24), 5.0, dtype=torch.bfloat16, device=DEV)
        wide[1:-1, off:off + n] = r
        view = wide[1:-1, off:off + n]
        assert K().mx_linear(x, w, bias=bias, residual=view, out=view) is view
        assert torch.equal(view, plain)
        assert (wide[0] == 5).all() and (wide[-1] == 5).all() and (wide[:, :off] == 5).all() and (wide[:, off + n:] == 5).all()


@pytest.mark.parametrize("rows,n,k", [(3, 50, 160), (140, 150, 288)])
@pytest.mark.parametrize("fmt", ["e4m3", "e2m1"])
def test_nan_blocks_reach_their_own_rows_and_columns_only(rows, n, k, fmt):
    """Also where K ends inside a step of 128: what lies behind a row's end, here a neighbour's NaN, is not read."""
    x, _ = random_mx(rows, k, fmt, 1)
    w, _ = random_mx(n, k, "e2m1", 2)
    clean = K().mx_linear(x, w)
    xs, ws = x.scales.clone(), w.scales.clone()
    xs[0, 1, 0] = 255   # row 1, first block: it follows row 0's end in memory
    ws[-1, n - 1, 0] = 255
    codes = x.codes.clone()
    if fmt == "e4m3":
        codes.view(torch.uint8)[2, :8] = 127  # e4m3 NaN codes at the start of row 2
    got = K().mx_linear(K().MX(codes, xs), K().MX(w.codes, ws))
    nan = torch.zeros(rows, n, dtype=torch.bool, device=DEV)
    nan[1] = True
    nan[:, n - 1] = True
    if fmt == "e4m3":
        nan[2] = True
    assert torch.equal(got.isnan(), nan)
    assert torch.equal(got[~nan], clean[~nan])


def check_gate_up(q, xv, wv, fmt, min_equal=0.97):
    n = wv.shape[0] // 2
    exact, err = product_bound(xv, wv, fmt)
    g, u, eg, eu = exact[:, :n], exact[:, n:], err[:, :n], err[:, n:]
    v = torch.from_numpy(O.silu_mul(g.cpu().numpy(), u.cpu().numpy())).to(DEV)
    # |SiLU'| <= 1.1; the fp32 exponential, reciprocal and products are within 8 * 2^-23 of the value
    d = 1.1 * eg * (u.abs() + eu) + g.abs() * eu + 8 * 2.0 ** -23 * v.abs()
    # a code is within half a step (2^-4 of the value, or of the least step, 2^-10 of the scale; the block's largest
    # value may move the scale up by one)
    step = torch.from_numpy(np.repeat(np.exp2(O.scale_exponents(v.cpu().numpy(), "e4m3") + 1.0), 32, 1)).to(DEV)
    got = torch.from_numpy(host(q)).to(DEV)
    far = (got - v).abs() - (d + 2.0 ** -4 * (v.abs() + d) + 2.0 ** -10 * step)
    assert float(far.max()) <= 0, f"worst {float(far.max())} over the bound"
    codes, scales = held(q)
    want_c, want_s = O.quantize(v.cpu().numpy(), "e4m3")
    last = scales[-1].copy()
    assert (last[:, (n // 32 - 1) % 4 + 1:] == 0).all()  # behind the last block
    assert (scales == want_s).mean() >= 0.99
    assert (codes == want_c).mean() >= min_equal


@pytest.mark.parametrize("fmt", ["e4m3", "e2m1"])
@pytest.mark.parametrize("rows,inter,k", [(1, 32, 32), (1, 480, 1536), (3, 64, 160), (16, 96, 512), (17, 160, 544), (64, 288, 1056),
                                          (65, 96, 256), (130, 352, 384), (260, 544, 128), (20, 288, 4128), (300, 1056, 2080),
                                          (1000, 2080, 288)])
def test_gate_up_matches_float64(rows, inter, k, fmt):
    # magnitudes as after a norm (the gate has to move through SiLU's bend)
    codes, scales = O.quantize(rows_of(rows, k, rows + k, spread=0.5).double().numpy(), fmt)
    x, xv = device_mx(codes, scales, fmt), O.values(codes, scales, fmt)
    codes, scales = O.quantize((rows_of(2 * inter, k, inter, spread=0.5) * k ** -0.5).double().numpy(), "e2m1")
    w, wv = device_mx(codes, scales, "e2m1"), O.values(codes, scales, "e2m1")
    check_gate_up(K().mx_gate_up_swiglu(x, w), xv, wv, fmt)


@pytest.mark.parametrize("rows,n,k", [(40, 300, 9600), (400, 1031, 4448)])
def test_without_workspace_a_split_product_runs_unsplit(rows, n, k):
    from flashgrpo_amd import _lib

    lib, kk = _lib.load(), K()
    x, xv = random_mx(rows, k, "e4m3", rows)
    w, wv = random_mx(n, k, "e2m1", n)
    need = lib.fg_mx_linear_workspace(rows, n, k, 0)
    assert need >= 2 * rows * n * 4
    exact, err = product_bound(xv, wv, "e4m3")
    for given in (0, need - 16, need):
        ws = torch.full((need + 64,), 255, dtype=torch.uint8, device=DEV)
        out = torch.empty(rows, n, dtype=torch.bfloat16, device=DEV)
        rc = lib.fg_mx_linear(x.codes.data_ptr(), x.scales.data_ptr(), 0, w.codes.data_ptr(), w.scales.data_ptr(), rows, n, k,
                              None, None, n, out.data_ptr(), n, ws.data_ptr() if given else None, given, kk._stream())
        assert rc == 0, lib.fg_last_error()
        check_linear(out, exact, err)
        assert (ws[need:] == 255).all() and ((ws == 255).all() or given == need)
    assert torch.equal(out, kk.mx_linear(x, w))


def strips(rows, n, at_once=32):
    """Rows and columns that meet every tile of an output: a pair of index lists, first and last ones included."""
    pick = lambda size: sorted({0, size - 1, *range(7, size, max(size // at_once, 1))})
    return torch.tensor(pick(rows), device=DEV), torch.tensor(pick(n), device=DEV)


def device_pair(rows, cols, fmt, seed, scale=1.0, spread=1.0):
    """An MX pair made on the device (bit for bit the oracle's, by the tests above) and its float64 values there."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(rows, cols, generator=g, device=DEV) * scale
    x *= torch.exp(spread * torch.randn(rows, cols // 32, generator=g, device=DEV)).repeat_interleave(32, 1)
    q = K().mx_quantize(x, fmt)
    return q, K().mx_dequantize(q, torch.float32)


# Sizes at which the choice takes each tile, whole and in parts; odd sizes where it allows them.
LARGE = [(777, 1280, 8960), (1408, 1533, 13824), (2311, 2048, 18944), (1856, 2045, 28672), (3500, 2047, 2048),
         (2311, 2559, 3584), (2311, 4607, 2080), (2311, 5119, 2080), (1856, 18943, 3584), (1194, 3584, 18944), (1194, 4608, 18944),
         (1856, 1536, 13824), (1856, 321, 5120), (1408, 1536, 2048), (2311, 897, 1536), (4096, 6145, 512), (777, 37888, 32), (2311, 2559, 28672),
         # a few rows beside streamed weights
         (1, 2047, 1536), (17, 33, 160), (30, 4090, 1376), (33, 1000, 416), (64, 3584, 3584), (16, 8190, 1056), (31, 7001, 416),
         (32, 8192, 2048), (3, 20000, 288), (12, 9001, 1376), (16, 151936, 128), (31, 37887, 1376)]


@pytest.mark.parametrize("fmt", ["e4m3", "e2m1"])
@pytest.mark.parametrize("rows,n,k", LARGE)
def test_linear_of_every_tile_with_bias_and_residual_in_place(rows, n, k, fmt):
    g = torch.Generator(device=DEV).manual_seed(n)
    (x, xv), (w, wv) = device_pair(rows, k, fmt, rows), device_pair(n, k, "e2m1", n)
    bias = torch.randn(n, device=DEV, generator=g).to(torch.bfloat16)
    res = (k ** 0.5 * torch.randn(rows, n, device=DEV, generator=g)).to(torch.bfloat16)
    out = res.clone()
    assert K().mx_linear(x, w, bias=bias, residual=out, out=out) is out
    rr, cc = strips(rows, n)
    for r, c in ((rr, slice(None)), (slice(None), cc)):
        exact, err = product_bound(xv[r].double().cpu().numpy(), wv[c].double().cpu().numpy(), fmt)
        check_linear(out[r][:, c], exact, err, bias[c], res[r][:, c])


@pytest.mark.parametrize("fmt", ["e4m3", "e2m1"])
@pytest.mark.parametrize("rows,inter,k", [(2311, 768, 5120), (1856, 1792, 2080), (4096, 1280, 1376), (2048, 4096, 1056),
                                          (500, 18944, 1536), (1408, 768, 13824), (777, 18944, 32), (3500, 768, 896),
                                          (2311, 2560, 512), (777, 1280, 896), (2311, 1792, 640), (16, 8960, 1536), (7, 416, 9632),
                                          (29, 18944, 3584)])
def test_gate_up_of_every_tile(rows, inter, k, fmt):
    (x, xv), (w, wv) = device_pair(rows, k, fmt, rows, spread=0.5), device_pair(2 * inter, k, "e2m1", k, k ** -0.5, 0.5)
    q = K().mx_gate_up_swiglu(x, w)
    rr = strips(rows, 1, 24)[0]
    cc = torch.tensor(sorted({0, inter // 32 - 1, *range(1, inter // 32, max(inter // 320, 1))}), device=DEV)  # whole blocks
    cols = (cc[:, None] * 32 + torch.arange(32, device=DEV)).flatten()
    every = torch.arange(rows, device=DEV)
    for r, b, c in ((rr, torch.arange(inter // 32, device=DEV), torch.arange(inter, device=DEV)), (every, cc, cols)):
        flat = torch.zeros(len(r), -(-len(b) // 4) * 4, dtype=torch.uint8, device=DEV)
        flat[:, :len(b)] = q.scales.transpose(0, 1).reshape(rows, -1)[r][:, b]
        part = K().MX(q.codes.view(torch.uint8)[r][:, c].contiguous().view(torch.float8_e4m3fn),
                      flat.view(len(r), -1, 4).transpose(0, 1).contiguous())
        check_gate_up(part, xv[r].double().cpu().numpy(), torch.cat([wv[c], wv[inter + c]]).double().cpu().numpy(), fmt)


# ------------------------------------------------------------------ together
def mlp(k, x, delta, norm, gate_up, down):
    q = k.rmsnorm_mx(x, norm, 1e-6, delta=delta)
    act = k.mx_gate_up_swiglu(q, gate_up)
    return q, act, k.mx_linear(act, down, residual=x, out=x)


def mlp_state(rows, hidden, inter, seed):
    k = K()
    x, d = rows_of(rows, hidden, seed).to(DEV), rows_of(rows, hidden, seed + 1, spread=0.1).to(DEV)
    norm = torch.ones(hidden, dtype=torch.bfloat16, device=DEV)
    gu = k.mx_quantize((rows_of(2 * inter, hidden, seed + 2, spread=0.2) * hidden ** -0.5).to(DEV), "e2m1")
    dn = k.mx_quantize((rows_of(hidden, inter, seed + 3, spread=0.2) * inter ** -0.5).to(DEV), "e2m1")
    return x, d, norm, gu, dn


@pytest.mark.parametrize("rows,hidden,inter", [(1, 256, 480), (29, 512, 1408), (416, 384, 608)])
def test_mlp_chain(rows, hidden, inter):
    """norm -> gate/up -> down + residual in place, each stage against the oracle on the stage's own inputs."""
    x, d, norm, gu, dn = mlp_state(rows, hidden, inter, rows)
    s, (want_c, want_s) = norm_oracle(x.cpu(), norm.cpu(), float(np.float32(1e-6)), d.cpu())
    q, act, y = mlp(K(), x, d, norm, gu, dn)
    codes, scales = held(q)
    assert np.array_equal(codes, want_c) and np.array_equal(scales, want_s)
    check_gate_up(act, host(q), host(gu), "e4m3")
    exact, err = product_bound(host(act), host(dn), "e4m3")
    assert y is x
    check_linear(y, exact, err, residual=s.to(DEV))


@pytest.mark.parametrize("rows", [1, 64, 150])
def test_chain_is_the_same_twice_captured_and_on_another_stream(rows):
    x, d, norm, gu, dn = mlp_state(rows, 512, 992, 3)
    first, k = x.clone(), K()
    want = mlp(k, x, d, norm, gu, dn)[2].clone()
    x.copy_(first)
    assert torch.equal(mlp(k, x, d, norm, gu, dn)[2], want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        x.copy_(first)
        got = mlp(k, x, d, norm, gu, dn)[2].clone()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    # two graphs of the same calls on rows of their own, replayed in turn with eager work between
    a, b = first.clone(), first.clone()
    graphs = []
    for t in (a, b):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            mlp(k, t, d, norm, gu, dn)
        graphs.append(g)
    for _ in range(3):
        for t in (a, b, x):
            t.copy_(first)
        graphs[0].replay()
        mlp(k, x, d, norm, gu, dn)
        graphs[1].replay()
        torch.cuda.synchronize()
        assert torch.equal(a, want) and torch.equal(b, want) and torch.equal(x, want)


def test_split_products_of_two_streams_at_once():
    """Two products whose sums go through workspaces, in flight together: each has its own."""
    k = K()
    pairs = [(random_mx(40, 9600, "e4m3", i)[0], random_mx(300, 9600, "e2m1", i + 5)[0]) for i in (1, 2)]
    want = [k.mx_linear(x, w) for x, w in pairs]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(k.mx_linear(*pairs[i]))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want[i]) for i in (0, 1) for o in got[i])


def test_calls_under_a_kernel_timer_are_timed_and_the_same():
    from flashgrpo_amd import timing

    k = K()
    x, d, norm, gu, dn = mlp_state(5, 256, 320, 9)
    first = x.clone()
    want = mlp(k, x, d, norm, gu, dn)[2].clone()
    x.copy_(first)
    t = timing.KernelTimer()
    with timing.active(t):
        assert torch.equal(mlp(k, x, d, norm, gu, dn)[2], want)
    torch.cuda.synchronize()
    assert {"fg_rmsnorm_mx", "fg_mx_gate_up_swiglu", "fg_mx_linear"} <= set(t.summary())


# ------------------------------------------------------------------ refusals
def test_refusals():
    k = K()
    x = torch.zeros(4, 128, dtype=torch.bfloat16, device=DEV)
    q, w = k.mx_quantize(x, "e4m3"), k.mx_quantize(x, "e2m1")
    one = torch.ones(128, dtype=torch.bfloat16, device=DEV)
    for call in (lambda: k.mx_quantize(x, "e5m2"), lambda: k.mx_quantize(x[:, :48]), lambda: k.mx_quantize(x[0]),
                 lambda: k.mx_quantize(x.t()), lambda: k.mx_quantize(x[:, 4:100]), lambda: k.mx_quantize(x, "e2m1", out=q),
                 lambda: k.mx_linear(q, k.mx_quantize(x[:, :64], "e2m1")), lambda: k.mx_linear(q, w, bias=one),
                 lambda: k.mx_linear(q, w, residual=x), lambda: k.mx_linear(q, w, out=x), lambda: k.mx_gate_up_swiglu(q, w),
                 lambda: k.rmsnorm_mx(x, one, 1e-6, sum_out=x), lambda: k.rmsnorm_mx(x, one, 1e-6, delta=x[:2]),
                 lambda: k.rmsnorm_mx(x[:, :64], one[:64], 1e-6), lambda: k.rmsnorm_mx(x, one[:64], 1e-6),
                 lambda: k.mx_linear(k.MX(q.codes, q.scales[:, :2]), w)):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: k.mx_linear(q, q), lambda: k.mx_quantize(x.half()), lambda: k.mx_dequantize(q, torch.float16),
                 lambda: k.mx_linear((x, q.scales), w), lambda: k.mx_gate_up_swiglu(w, q)):
        with pytest.raises(TypeError):
            call()
