"""The attention output projection of a quantised layer: split-K parts to the residual stream and MX rows
(``fg_residual_rmsnorm_mx_parts``), and the forward that takes it wherever the layer's bf16 form takes split-K."""
import numpy as np
import pytest
import torch

from oracle import mx as O
from test_gpu_mx import DEV, K, held, norm_oracle, rows_of
from test_gpu_mx_model import build, run, same

pytestmark = pytest.mark.gpu
EPS = float(np.float32(1e-6))


@pytest.fixture(scope="module", autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


def check_codes(q, x, w):
    """q holds the codes of RMSNorm(x) * w by the formula in 64 bits."""
    codes, scales = held(q)
    want_c, want_s = norm_oracle(x.cpu(), w.cpu(), EPS, None)[1]
    assert np.array_equal(codes, want_c) and np.array_equal(scales, want_s)


@pytest.mark.parametrize("splits,rows,cols", [(1, 1, 32), (2, 5, 160), (3, 3, 1536), (9, 2, 2080), (6, 17, 3584), (4, 4, 8192),
                                              (2, 300, 512)])
def test_parts_to_residual_and_codes(splits, rows, cols):
    g = torch.Generator(device=DEV).manual_seed(cols)
    parts = torch.randn(splits, rows, cols, device=DEV, generator=g)
    w = (1 + 0.2 * torch.randn(cols, device=DEV, generator=g)).to(torch.bfloat16)
    x = rows_of(rows, cols, cols).to(DEV)
    total = parts[0].clone()
    for s in range(1, splits):
        total += parts[s]
    want = (x.float() + total.to(torch.bfloat16).float()).to(torch.bfloat16)
    plain = x.clone()
    K().residual_rmsnorm_parts(parts, plain, w, 1e-6)
    assert torch.equal(plain, want)
    wide = torch.full((rows + 2, cols + 16), 3.0, dtype=torch.bfloat16, device=DEV)
    view = wide[1:-1, 8:8 + cols]
    view.copy_(x)
    for t in (x, view):  # contiguous rows and a view's
        q = K().residual_rmsnorm_mx_parts(parts, t, w, 1e-6)
        assert torch.equal(t, want)
        check_codes(q, t, w)
    assert (wide[0] == 3).all() and (wide[-1] == 3).all() and (wide[:, :8] == 3).all() and (wide[:, 8 + cols:] == 3).all()


def test_special_parts():
    """An infinity or a NaN in the parts stays in its row; rows of zeros are zeros."""
    parts = torch.randn(3, 5, 256, device=DEV)
    x = torch.randn(5, 256, device=DEV).to(torch.bfloat16)
    parts[1, 1, 40], parts[2, 3, 7] = float("inf"), float("nan")
    parts[:, 4], x[4] = 0, 0
    first, w = x.clone(), torch.ones(256, dtype=torch.bfloat16, device=DEV)
    q = K().residual_rmsnorm_mx_parts(parts, x, w, 1e-6)
    v = O.values(*held(q), "e4m3")
    assert np.isnan(v[1, 32:64]).all() and (v[1, :32] == 0).all() and (v[1, 64:] == 0).all() and np.isnan(v[3]).all()
    assert (v[4] == 0).all()
    clean = first[[0, 2]].contiguous()
    again = K().residual_rmsnorm_mx_parts(parts[:, [0, 2]].contiguous(), clean, w, 1e-6)
    assert np.array_equal(held(again)[0], held(q)[0][[0, 2]]) and torch.equal(clean, x[[0, 2]])


def test_no_rows_and_refusals():
    k = K()
    w = torch.ones(64, dtype=torch.bfloat16, device=DEV)
    x, parts = torch.zeros(4, 64, dtype=torch.bfloat16, device=DEV), torch.zeros(2, 4, 64, device=DEV)
    assert k.residual_rmsnorm_mx_parts(parts[:, :0], x[:0], w, 1e-6).codes.shape == (0, 64)
    odd = torch.zeros(4, 72, dtype=torch.bfloat16, device=DEV)
    for call in (lambda: k.residual_rmsnorm_mx_parts(parts[:, :, ::2], x, w, 1e-6), lambda: k.residual_rmsnorm_mx_parts(parts[0], x, w, 1e-6),
                 lambda: k.residual_rmsnorm_mx_parts(parts.double(), x, w, 1e-6), lambda: k.residual_rmsnorm_mx_parts(parts, x[:3], w, 1e-6),
                 lambda: k.residual_rmsnorm_mx_parts(parts, x.float(), w, 1e-6), lambda: k.residual_rmsnorm_mx_parts(parts, odd[:, 4:68], w, 1e-6),
                 lambda: k.residual_rmsnorm_mx_parts(parts, x[:1].expand(4, 64), w, 1e-6),
                 lambda: k.residual_rmsnorm_mx_parts(parts, x, w.float(), 1e-6), lambda: k.residual_rmsnorm_mx_parts(parts, x, w[:32], 1e-6),
                 lambda: k.residual_rmsnorm_mx_parts(parts[:0], x, w, 1e-6),
                 lambda: k.residual_rmsnorm_mx_parts(parts, x, w, 1e-6, out=k.mx_quantize(x, "e2m1")),
                 lambda: k.residual_rmsnorm_mx_parts(torch.zeros(1, 4, 8224, device=DEV), torch.zeros(4, 8224, dtype=torch.bfloat16, device=DEV),
                                                     torch.ones(8224, dtype=torch.bfloat16, device=DEV), 1e-6)):
        with pytest.raises(ValueError):
            call()


class Counted:
    """The kernels module, the norms in front of a quantised MLP checked on their own inputs and listed."""

    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        return getattr(K(), name)

    def rmsnorm_mx(self, x, w, eps, *, out):
        q = K().rmsnorm_mx(x, w, eps, out=out)
        check_codes(q, x, w)
        self.calls.append("addmm")
        return q

    def residual_rmsnorm_mx_parts(self, parts, x, w, eps, *, out):
        total, first = parts[0].clone(), x.clone()
        for p in parts[1:]:
            total += p
        q = K().residual_rmsnorm_mx_parts(parts, x, w, eps, out=out)
        assert torch.equal(x, (first.float() + total.to(torch.bfloat16).float()).to(torch.bfloat16))
        check_codes(q, x, w)
        self.calls.append("parts")
        return q


@pytest.mark.parametrize("split_k,expected", [(True, "parts"), (False, "addmm"), (None, "addmm")])
def test_split_k_linear_holds_in_a_quantised_model(monkeypatch, split_k, expected):
    from flashgrpo_amd.models import target

    m = build()
    m.split_k_linear = split_k
    m.quantize_mlp()
    eager = run(m)
    counted = Counted()
    monkeypatch.setattr(target, "K", counted)
    assert same(run(m), eager)
    monkeypatch.undo()
    assert counted.calls == [expected] * (2 * m.cfg.num_layers)  # a prefill and a tree forward (of a size no table covers)
    assert same(run(m, graph=True, calls=5), eager)
    assert m._graphs and all(g is not None for g in m._graphs.values())


def test_measured_sizes_take_their_measured_path(monkeypatch):
    """Rows and sizes for which the table has the output projection fastest as split-K."""
    from flashgrpo_amd.decoding.medusa_tree import TreeTopology
    from flashgrpo_amd.models import target
    from flashgrpo_amd.models.target import TargetConfig, TargetModel

    m = TargetModel.random(TargetConfig(1, 3584, 28, 4, 128, 512, 100)).quantize_mlp()
    topo = TreeTopology([2, 1], 4)
    d = topo.device(DEV)
    n = topo.num_nodes
    batch = 128 // n
    assert target.linear_path("o", batch * n, 3584, 3584) is not None
    counted = Counted()
    monkeypatch.setattr(target, "K", counted)
    m.forward(torch.zeros(batch, n, dtype=torch.int32, device=DEV), m.new_cache(batch, 64), pos_offset=d["pos_offset"],
              anc=d["anc"])
    assert counted.calls == ["parts"]
