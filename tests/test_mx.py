"""Microscaled rows without a GPU: the oracle's quantisation against values written out by hand, and what the
entry points refuse before they launch anything."""
import ctypes
import os

import numpy as np
import pytest
import torch

from oracle import mx as O


def _block(*v):
    x = np.zeros((1, 32))
    x[0, :len(v)] = v
    return x


def test_code_tables():
    assert O.TABLE["e2m1"].tolist() == [0, 0.5, 1, 1.5, 2, 3, 4, 6]
    t = O.TABLE["e4m3"]
    assert t[-1] == 448 and t[1] == 2.0 ** -9 and t[8] == 2.0 ** -6 and t[0x38] == 1.0
    for c in range(127):
        assert float(torch.tensor([c], dtype=torch.uint8).view(torch.float8_e4m3fn).float()) == t[c]


@pytest.mark.parametrize("fmt,largest", [("e4m3", 448.0), ("e2m1", 6.0)])
def test_scale_is_the_least_power_of_two_that_holds_the_block(fmt, largest):
    for n in (-20, -1, 0, 3):
        at = O.quantize(_block(largest * 2.0 ** n), fmt)[1][0, 0]
        above = O.quantize(_block(largest * 2.0 ** n * (1 + 2.0 ** -7)), fmt)[1][0, 0]
        assert at.tolist() == [127 + n, 0, 0, 0] and above.tolist() == [128 + n, 0, 0, 0]
    assert O.quantize(_block(), fmt)[1][0, 0, 0] == 1                 # nothing but zeros: the least scale
    assert O.quantize(_block(2.0 ** -140), fmt)[1][0, 0, 0] == 1
    assert O.quantize(_block(1.0, np.inf), fmt)[1][0, 0, 0] == 255 and O.quantize(_block(np.nan), fmt)[1][0, 0, 0] == 255


def test_ties_go_to_the_even_code():
    c, _ = O.quantize(_block(6, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5, -0.75, -0.25), "e2m1")
    assert c[0, :10].tolist() == [7, 0, 2, 2, 4, 4, 6, 6, 10, 8]
    c, _ = O.quantize(_block(448, 1.0625, 1.1875, 2.0 ** -10, 3 * 2.0 ** -10), "e4m3")
    assert c[0, :5].tolist() == [126, 0x38, 0x3a, 0, 2]


def test_oracle_round_trip_and_layout():
    x = np.random.default_rng(0).standard_normal((3, 160))
    for fmt, half in (("e4m3", 2.0 ** -4), ("e2m1", 2.0 ** -2)):
        codes, scales = O.quantize(x, fmt)
        assert scales.shape == (2, 3, 4) and (scales[1, :, 1:] == 0).all() and (scales[1, :, 0] > 0).all()
        v = O.values(O.unpack(O.pack(codes, fmt), fmt), scales, fmt)
        step = np.repeat(np.exp2(O.scale_exponents(x, fmt).astype(float)), 32, 1)
        assert (np.abs(v - x) <= np.maximum(half * np.abs(x), step * (2.0 ** -10 if fmt == "e4m3" else 0.25))).all()


# ------------------------------------------------------------------ refusals
def _lib():
    from flashgrpo_amd import _lib as L

    if not os.path.exists(L.library_path()):
        pytest.skip("native library not built")
    return L.load()


def test_entry_points_refuse_bad_arguments_on_the_host():
    lib = _lib()
    p, odd = ctypes.c_void_p(256), ctypes.c_void_p(264)

    def refused(rc, text):
        assert rc != 0 and text in lib.fg_last_error(), (rc, lib.fg_last_error())

    refused(lib.fg_mx_quantize(None, 1, 64, 1, 64, 0, p, p, None), b"null pointer")
    refused(lib.fg_mx_quantize(p, 2, 64, 1, 64, 0, p, p, None), b"dtype")
    refused(lib.fg_mx_quantize(p, 1, 64, 1, 64, 2, p, p, None), b"format")
    refused(lib.fg_mx_quantize(p, 1, 64, 0, 64, 0, p, p, None), b"shape")
    refused(lib.fg_mx_quantize(p, 1, 32, 1, 64, 0, p, p, None), b"shape")
    refused(lib.fg_mx_quantize(p, 1, 48, 1, 48, 0, p, p, None), b"multiple of 32")
    refused(lib.fg_mx_quantize(p, 1, 68, 1, 64, 0, p, p, None), b"aligned")
    refused(lib.fg_mx_quantize(odd, 1, 64, 1, 64, 0, p, p, None), b"aligned")
    refused(lib.fg_mx_dequantize(p, p, 0, 1, 48, p, 1, 48, None), b"multiple of 32")
    refused(lib.fg_mx_dequantize(p, None, 0, 1, 64, p, 1, 64, None), b"null pointer")
    refused(lib.fg_rmsnorm_mx(p, p, p, None, 1, 1, 64, 1e-6, p, p, None), b"null pointer")
    refused(lib.fg_rmsnorm_mx(p, None, p, None, 1, 1, 8224, 1e-6, p, p, None), b"8192")
    refused(lib.fg_rmsnorm_mx(p, None, p, None, 1, 1, 40, 1e-6, p, p, None), b"multiple of 32")
    refused(lib.fg_rmsnorm_mx(odd, None, p, None, 1, 1, 64, 1e-6, p, p, None), b"aligned")


def test_products_refuse_bad_arguments_on_the_host():
    lib = _lib()
    p, off8, off1, n = ctypes.c_void_p(256), ctypes.c_void_p(264), ctypes.c_void_p(257), None

    def refused(rc, text):
        assert rc != 0 and text in lib.fg_last_error(), (rc, lib.fg_last_error())

    def linear(xc=p, xs=p, f=0, wc=p, ws=p, rows=4, cols=64, hidden=64, bias=n, res=n, ldr=64, out=p, ldo=64, wksp=n, size=0):
        return lib.fg_mx_linear(xc, xs, f, wc, ws, rows, cols, hidden, bias, res, ldr, out, ldo, wksp, size, None)

    def gate_up(xc=p, xs=p, f=0, wc=p, ws=p, rows=4, inter=64, hidden=64, codes=p, scales=p, wksp=n, size=0):
        return lib.fg_mx_gate_up_swiglu(xc, xs, f, wc, ws, rows, inter, hidden, codes, scales, wksp, size, None)

    for call in (linear, gate_up):
        for name in ("xc", "xs", "wc", "ws"):
            refused(call(**{name: n}), b"null pointer")
        refused(call(f=2), b"format")
        refused(call(f=-1), b"format")
        refused(call(rows=0), b"shape")
        refused(call(rows=(1 << 22) + 1), b"shape")
        refused(call(hidden=0), b"shape")
        refused(call(hidden=48), b"multiple of 32")
        refused(call(xc=off8), b"aligned")
        refused(call(wc=off8), b"aligned")
        refused(call(xs=off1), b"aligned")
        refused(call(wksp=off8), b"workspace")
    refused(linear(cols=-1), b"shape")
    refused(linear(rows=1 << 22, cols=1 << 22, hidden=32, ldo=1 << 22), b"shape")  # more tiles than a launch takes
    refused(linear(cols=1 << 16, hidden=1 << 16, ldo=1 << 16), b"2 GiB")
    refused(linear(rows=1 << 22, hidden=1 << 16), b"2 GiB")   # the rows' scales
    refused(linear(out=n), b"null pointer")
    refused(linear(out=off1), b"aligned")
    refused(linear(bias=off1), b"aligned")
    refused(linear(ldo=63), b"strides")
    refused(linear(res=p, ldr=63), b"strides")
    refused(gate_up(codes=n), b"null pointer")
    refused(gate_up(scales=n), b"null pointer")
    refused(gate_up(inter=48), b"multiple of 32")
    refused(gate_up(inter=1 << 30), b"shape")
    refused(gate_up(codes=off8), b"aligned")
    refused(gate_up(scales=off1), b"aligned")


def test_more_rows_than_a_launch_takes_are_refused():
    lib = _lib()
    p = ctypes.c_void_p(256)
    most = 2 ** 31 - 1
    for rc in (lib.fg_mx_quantize(p, 1, 32, most, 32, 0, p, p, None), lib.fg_mx_dequantize(p, p, 1, most, 32, p, 1, 32, None),
               lib.fg_rmsnorm_mx(p, None, p, None, 1, 1 << 23, 32, 1e-6, p, p, None)):
        assert rc != 0 and b"too many rows" in lib.fg_last_error()


def test_workspace_sizes():
    """Sums of split products only; 0 for sizes that the calls refuse."""
    lib = _lib()
    assert lib.fg_mx_linear_workspace(1, 64, 64, 0) == 0
    need = lib.fg_mx_linear_workspace(40, 301, 9600, 0)
    assert need >= 2 * 40 * 304 * 4 and need % (40 * 304 * 4) == 0
    assert lib.fg_mx_gate_up_swiglu_workspace(20, 288, 4128, 0) % (20 * 576 * 4) == 0
    for bad in (0, -1, 2 ** 31 - 1):
        assert lib.fg_mx_linear_workspace(bad, 64, 64, 0) == lib.fg_mx_linear_workspace(64, bad, 64, 0) == 0
        assert lib.fg_mx_linear_workspace(64, 64, bad, 0) == lib.fg_mx_gate_up_swiglu_workspace(64, bad, 64, 0) == 0


def test_wrappers_take_device_tensors_only():
    from flashgrpo_amd import kernels as K

    x = torch.zeros(2, 64, dtype=torch.bfloat16)
    q = K.MX(torch.zeros(2, 32, dtype=torch.uint8), torch.zeros(1, 2, 4, dtype=torch.uint8))
    assert q.format == "e2m1" and q.shape == (2, 64)
    for call in (lambda: K.mx_quantize(x), lambda: K.mx_dequantize(q), lambda: K.rmsnorm_mx(x, x[0], 1e-6),
                 lambda: K.mx_linear(q, q), lambda: K.mx_gate_up_swiglu(q, q)):
        with pytest.raises(ValueError, match="device tensors"):
            call()


def test_mx_pairs_are_checked():
    from flashgrpo_amd import kernels as K

    codes, scales = torch.zeros(2, 96, dtype=torch.uint8), torch.zeros(2, 2, 4, dtype=torch.uint8)
    assert K._mx_of((codes, scales), "t")[2:] == (1, 2, 192, -1)
    for bad in ((codes.float(), scales), (codes, scales.float()), (codes[0], scales)):
        with pytest.raises(TypeError):
            K._mx_of(bad, "t")
    for bad in ((codes[:, :95], scales), (codes[:, :8], scales), (codes, scales[:1]), (codes, scales[:, :1]),
                (codes.t().contiguous().t(), scales), (codes[:0, :0], scales)):
        with pytest.raises(ValueError):
            K._mx_of(bad, "t")


def test_only_bf16_models_of_whole_blocks_are_quantised():
    from flashgrpo_amd.models.target import TargetConfig, TargetModel

    for hidden, inter, dtype in ((256, 512, torch.float32), (272, 512, torch.bfloat16), (256, 520, torch.bfloat16),
                                 (8224, 512, torch.bfloat16)):
        m = TargetModel(TargetConfig(1, hidden, 4, 2, 64, inter, 100), {"layers": []}, dtype=dtype, device="cpu")
        with pytest.raises(ValueError, match="multiples of 32"):
            m.quantize_mlp()
        assert m.quantize_mlp(False).mlp_mx is None


def test_residual_norm_of_parts_refuses_bad_arguments_on_the_host():
    lib = _lib()
    p, off8, off1, n = ctypes.c_void_p(256), ctypes.c_void_p(264), ctypes.c_void_p(257), None

    def refused(text, part=p, splits=2, rows=4, hidden=64, x=p, ldx=64, w=p, codes=p, scales=p):
        rc = lib.fg_residual_rmsnorm_mx_parts(part, splits, rows, hidden, x, ldx, w, 1e-6, codes, scales, None)
        assert rc != 0 and text in lib.fg_last_error(), (rc, lib.fg_last_error())

    for name in ("part", "x", "w", "codes", "scales"):
        refused(b"null pointer", **{name: n})
    for name in ("part", "x", "w", "codes"):
        refused(b"aligned", **{name: off8})
    refused(b"aligned", scales=off1)
    refused(b"shape", rows=0)
    refused(b"shape", splits=0)
    refused(b"multiple of 32", hidden=48, ldx=48)
    refused(b"8192", hidden=8224, ldx=8224)
    refused(b"stride", ldx=56)
    refused(b"stride", ldx=68)
    refused(b"too many rows", rows=1 << 23)


def test_pairs_of_more_than_an_int_counts_are_refused():
    """Sizes are C ints behind the wrappers: one over them would arrive as its last 32 bits."""
    from flashgrpo_amd import kernels as K

    big = 2 ** 32 + 4
    meta = lambda *shape: torch.empty(*shape, dtype=torch.uint8, device="meta")
    for codes, scales in ((meta(big, 16), meta(1, big, 4)), (meta(1, 2 ** 31), meta(2 ** 25, 1, 4)), (meta(2 ** 31, 16), meta(1, 2 ** 31, 4))):
        with pytest.raises(ValueError, match="2\\^31"):
            K._mx_of((codes, scales), "t")
    for rows, cols in ((big, 32), (1, 2 ** 32 + 64), (2 ** 31, 32)):
        with pytest.raises(ValueError, match="2\\^31"):
            K._mx_out(None, rows, cols, 0, torch.device("meta"), "t")
