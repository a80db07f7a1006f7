"""Outputs of the MX wrappers that share memory with operands: the ones that the kernels allow, and the refusal of others."""
import pytest
import torch

from test_gpu_mx import DEV, K, device_pair, held, rows_of

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


def refused(call):
    with pytest.raises(ValueError, match="overlap"):
        call()


def shifted(q, rows, cols):
    """An e4m3 pair whose codes begin with the second row of q's."""
    return K().MX(q.codes.view(torch.uint8).flatten()[cols:cols + rows * cols].view(rows, cols).view(torch.float8_e4m3fn),
                  torch.empty((cols + 127) // 128, rows, 4, dtype=torch.uint8, device=DEV))


def test_gate_up_into_its_rows_is_refused():
    k = K()
    x, w = device_pair(40, 256, "e4m3", 1)[0], device_pair(512, 256, "e2m1", 2)[0]
    before = x.codes.view(torch.uint8).clone()
    refused(lambda: k.mx_gate_up_swiglu(x, w, out=x))
    refused(lambda: k.mx_gate_up_swiglu(k.MX(x.codes[:20], x.scales[:, :20].contiguous()), w, out=shifted(x, 20, 256)))
    fresh = device_pair(40, 256, "e4m3", 3)[0]
    refused(lambda: k.mx_gate_up_swiglu(x, w, out=k.MX(fresh.codes, x.scales)))
    assert torch.equal(x.codes.view(torch.uint8), before)
    assert k.mx_gate_up_swiglu(x, w, out=fresh).codes is fresh.codes
    want = k.mx_gate_up_swiglu(x, w)
    assert torch.equal(fresh.codes.view(torch.uint8), want.codes.view(torch.uint8)) and torch.equal(fresh.scales, want.scales)


def test_quantise_dequantise_and_norm_over_their_operands():
    k = K()
    x = rows_of(8, 128, 1).to(DEV)
    raw = x.view(torch.uint8).view(16, 128)
    scales = torch.empty(1, 8, 4, dtype=torch.uint8, device=DEV)
    refused(lambda: k.mx_quantize(x, "e4m3", out=k.MX(raw[:8].view(torch.float8_e4m3fn), scales)))
    refused(lambda: k.rmsnorm_mx(x, x[0].clone(), 1e-6, out=k.MX(raw[8:].view(torch.float8_e4m3fn), scales)))
    q = k.mx_quantize(x, "e4m3")
    buf = torch.empty(8 * 128 * 2, dtype=torch.uint8, device=DEV)
    held_q = k.MX(buf[:1024].view(8, 128).view(torch.float8_e4m3fn), q.scales)
    refused(lambda: k.mx_dequantize(held_q, out=buf.view(torch.bfloat16).view(8, 128)))
    w = torch.ones(128, dtype=torch.bfloat16, device=DEV)
    both = rows_of(9, 128, 2).to(DEV)
    refused(lambda: k.rmsnorm_mx(both[:8], w, 1e-6, delta=x, sum_out=both[1:]))
    refused(lambda: k.rmsnorm_mx(x, w, 1e-6, delta=both[:8], sum_out=both[1:]))
    parts = torch.zeros(1, 8, 128, device=DEV)
    refused(lambda: k.residual_rmsnorm_mx_parts(parts, x, w, 1e-6, out=k.MX(raw[:8].view(torch.float8_e4m3fn), scales)))
    refused(lambda: k.residual_rmsnorm_mx_parts(parts, parts.view(torch.bfloat16).view(16, 128)[:8], w, 1e-6))
    # the sum into x or into the addend
    d = rows_of(8, 128, 3).to(DEV)
    total = torch.empty_like(x)
    want = k.rmsnorm_mx(x, w, 1e-6, delta=d, sum_out=total)
    for into in ("delta", "x"):
        a, b = x.clone(), d.clone()
        got = k.rmsnorm_mx(a, w, 1e-6, delta=b, sum_out=b if into == "delta" else a)
        assert torch.equal(b if into == "delta" else a, total) and torch.equal(b, d) == (into == "x")
        assert (held(got)[0] == held(want)[0]).all() and (held(got)[1] == held(want)[1]).all()


@pytest.mark.parametrize("rows", [1, 6, 150])
def test_linear_beside_in_and_over_its_residual(rows):
    k, n = K(), 136
    x, w = device_pair(rows, 256, "e4m3", 1)[0], device_pair(n, 256, "e2m1", 2)[0]
    g = torch.Generator(device=DEV).manual_seed(1)
    fresh = lambda: torch.randn(rows + 2, 3 * n, device=DEV, generator=g).to(torch.bfloat16)
    buf = fresh()
    want = k.mx_linear(x, w, residual=buf[1:-1, :n].clone())
    for first in (n, n + 8, 2 * n):  # columns of one buffer beside each other
        b = buf.clone()
        assert torch.equal(k.mx_linear(x, w, residual=b[1:-1, :n], out=b[1:-1, first:first + n]), want)
        assert torch.equal(b[:, :n], buf[:, :n])
    b = buf.clone()
    assert torch.equal(k.mx_linear(x, w, residual=b[1:-1, :n], out=b[1:-1, :n]), want)
    for out in (b[1:-1, 8:8 + n], b[1:-1, 1:1 + n], *((b[2:, :n], b[:-2, :n]) if rows > 1 else ())):
        before = b.clone()
        refused(lambda: k.mx_linear(x, w, residual=b[1:-1, :n], out=out))
        assert torch.equal(b, before)
    flat = buf.flatten()
    if rows > 1:  # another row stride over the same memory
        refused(lambda: k.mx_linear(x, w, residual=flat[:rows * n].view(rows, n), out=flat[:rows * (n + 8)].view(rows, n + 8)[:, :n]))
    shared = torch.zeros(max(rows * n * 2, n * 128), dtype=torch.uint8, device=DEV)
    held_w = k.MX(shared[:n * 128].view(n, 128), w.scales)
    refused(lambda: k.mx_linear(x, held_w, out=shared[:rows * n * 2].view(torch.bfloat16).view(rows, n)))
    o = torch.zeros(rows + 1, n, dtype=torch.bfloat16, device=DEV)
    refused(lambda: k.mx_linear(x, w, bias=o[0], out=o[:rows]))
    k.mx_linear(x, w, bias=o[rows], out=o[:rows])
