"""Every kernel of the MX products, at sizes that are checked to take it (mx_sizes.py): bounds per element, precision over
whole outputs, NaN blocks."""
import numpy as np
import pytest
import torch

import mx_sizes as S
from oracle import mx as O
from test_gpu_mx import DEV, K, check_gate_up, check_linear, device_pair, held, product_bound, strips

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


@pytest.mark.parametrize("fmt,shape,detail,rows,n,k", S.every(S.linear))
def test_linear_of_every_kernel(fmt, shape, detail, rows, n, k):
    """With bias and residual in place: each element within its bound, over rows and columns that meet every tile; and
    without them, over the whole output, as precise as the 64-bit product rounded to bf16.

    The cut of e4m3 products is below 2^-13 of the largest of eight, which is at most sqrt(8) times their root mean square;
    random signs add to sqrt(8) 2^-13 of the sum's root mean square. fp32 sums of K / 64 instructions and at most 16 splits are
    below (K / 64 + 16) 2^-23 of it. Both are independent of the last rounding, so squares add."""
    assert S.is_plan(K().mx_plan(rows, n, k, fmt=fmt), shape, detail)
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
    exact = xv.double() @ wv.double().t()
    rms = lambda t: float(t.square().mean().sqrt())
    best = rms(exact.to(torch.bfloat16).double() - exact)
    sums = (8 ** 0.5 * 2.0 ** -13 if fmt == "e4m3" else 0.0) + (k / 64 + 16) * 2.0 ** -23
    got = rms(K().mx_linear(x, w).double() - exact)
    assert got <= (best ** 2 + (sums * rms(exact)) ** 2) ** 0.5, f"{got:.3e}, the rounding alone {best:.3e}"


@pytest.mark.parametrize("fmt,shape,detail,rows,inter,k", S.every(S.gate_up))
def test_gate_up_of_every_kernel(fmt, shape, detail, rows, inter, k):
    assert S.is_plan(K().mx_plan(rows, inter, k, fmt=fmt, gate_up=True), shape, detail)
    (x, xv), (w, wv) = device_pair(rows, k, fmt, rows, spread=0.5), device_pair(2 * inter, k, "e2m1", k, k ** -0.5, 0.5)
    q = K().mx_gate_up_swiglu(x, w)
    y = xv.double() @ wv.double().t()
    v = O.silu_mul(y[:, :inter].cpu().numpy(), y[:, inter:].cpu().numpy())
    want_c, want_s = O.quantize(v, "e4m3")
    codes, scales = held(q)
    # sums and activation within d of a value, half of the codes' least distance 2^-4 around each border (see
    # test_gpu_mx_precision.py)
    d = 2 * (k / 32 + 8) * 2.0 ** -24
    assert (codes != want_c).mean() <= 2 * d / 2.0 ** -4 + 1 / codes.size
    assert (scales != want_s).mean() <= 32 * 2 * d + 1 / scales.size
    assert (scales[-1][:, (inter // 32 - 1) % 4 + 1:] == 0).all()
    rr = strips(rows, 1, 24)[0]
    part = K().MX(q.codes.view(torch.uint8)[rr].contiguous().view(torch.float8_e4m3fn), q.scales[:, rr].contiguous())
    check_gate_up(part, xv[rr].double().cpu().numpy(), wv.double().cpu().numpy(), fmt)


@pytest.mark.parametrize("fmt,shape,detail,rows,inter,k", S.every(S.gate_up))
def test_nan_blocks_of_gate_up_reach_their_own_blocks_only(fmt, shape, detail, rows, inter, k):
    """A row's NaN block makes the row NaN; a gate row's, or an up row's, the blocks that hold its column. Others are as
    without."""
    (x, _), (w, _) = device_pair(rows, k, fmt, 1, spread=0.5), device_pair(2 * inter, k, "e2m1", 2, k ** -0.5, 0.5)
    clean = held(K().mx_gate_up_swiglu(x, w))
    xs, ws, codes = x.scales.clone(), w.scales.clone(), x.codes.clone()
    last = (k // 32 - 1) % 4
    nan = np.zeros((rows, inter // 32), bool)
    if rows > 1:
        xs[0, 1, 0] = 255
        nan[1] = True
    if rows > 4 and fmt == "e4m3":
        codes.view(torch.uint8)[4, -3:] = 127  # NaN codes at a row's end
        nan[4] = True
    ws[-1, inter - 1, last] = 255      # the last column's gate
    ws[0, inter + 33 % inter, 0] = 255  # a column's up
    nan[:, -1] = nan[:, 33 % inter // 32] = True
    got_c, got_s = held(K().mx_gate_up_swiglu(K().MX(codes, xs), K().MX(w.codes, ws)))
    by_block = got_s.transpose(1, 0, 2).reshape(rows, -1)[:, :inter // 32]
    assert np.array_equal(by_block == 255, nan)
    keep = ~np.repeat(nan, 32, 1)
    assert np.array_equal(got_c[keep], clean[0][keep])
    assert np.array_equal(by_block[~nan], clean[1].transpose(1, 0, 2).reshape(rows, -1)[:, :inter // 32][~nan])


SPLIT = [case for case in S.every(S.gate_up) if case[1][2] and case[2]]


@pytest.mark.parametrize("fmt,shape,detail,rows,inter,k", SPLIT)
def test_gate_up_without_workspace_and_in_two_graphs(fmt, shape, detail, rows, inter, k):
    """A split gate/up without its workspace, or with less, runs unsplit; two captured ones replayed in turn with eager calls
    between share nothing."""
    from flashgrpo_amd import _lib

    lib, kk = _lib.load(), K()
    (x, xv), (w, wv) = device_pair(rows, k, fmt, rows, spread=0.5), device_pair(2 * inter, k, "e2m1", k, k ** -0.5, 0.5)
    other = device_pair(rows, k, fmt, rows + 1, spread=0.5)[0]
    need = lib.fg_mx_gate_up_swiglu_workspace(rows, inter, k, kk.MX_FORMATS[fmt])
    assert need >= 2 * rows * 2 * inter * 4
    want = kk.mx_gate_up_swiglu(x, w)
    y = xv.double() @ wv.double().t()
    want_c = O.quantize(O.silu_mul(y[:, :inter].cpu().numpy(), y[:, inter:].cpu().numpy()), "e4m3")[0]
    d = 2 * (k / 32 + 8) * 2.0 ** -24
    for given in (0, need - 16, need):
        ws = torch.full((need + 64,), 255, dtype=torch.uint8, device=DEV)
        q = kk.MX(torch.zeros(rows, inter, dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn), torch.zeros_like(want.scales))
        rc = lib.fg_mx_gate_up_swiglu(x.codes.data_ptr(), x.scales.data_ptr(), kk.MX_FORMATS[fmt], w.codes.data_ptr(),
                                      w.scales.data_ptr(), rows, inter, k, q.codes.data_ptr(), q.scales.data_ptr(),
                                      ws.data_ptr() if given else None, given, kk._stream())
        assert rc == 0, lib.fg_last_error()
        assert (held(q)[0] != want_c).mean() <= 2 * d / 2.0 ** -4 + 1 / want_c.size
        assert (ws[need:] == 255).all() and ((ws == 255).all() or given == need)
    assert torch.equal(q.codes.view(torch.uint8), want.codes.view(torch.uint8)) and torch.equal(q.scales, want.scales)
    wanted, graphs = [want, kk.mx_gate_up_swiglu(other, w)], []
    for rows_in in (x, other):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = kk.mx_gate_up_swiglu(rows_in, w)
        graphs.append((g, out))
    for _ in range(3):
        for (g, out), ref in zip(graphs, wanted):
            out.codes.view(torch.uint8).zero_()
            g.replay()
            kk.mx_gate_up_swiglu(x, w)
        torch.cuda.synchronize()
        for (_, out), ref in zip(graphs, wanted):
            assert torch.equal(out.codes.view(torch.uint8), ref.codes.view(torch.uint8)) and torch.equal(out.scales, ref.scales)
