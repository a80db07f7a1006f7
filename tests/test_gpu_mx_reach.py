"""``quantize_mlp`` for users of a transformers model, and MX operands whose offsets pass 32 bits."""
import numpy as np
import pytest
import torch

from test_gpu_mx import DEV, K, check_linear, device_pair, held, product_bound

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


def hf_model():
    transformers = pytest.importorskip("transformers")
    hc = transformers.Qwen2Config(vocab_size=97, hidden_size=256, intermediate_size=512, num_hidden_layers=2,
                                  num_attention_heads=2, num_key_value_heads=1, max_position_embeddings=512)
    torch.manual_seed(0)
    return transformers.Qwen2ForCausalLM(hc).to(DEV).to(torch.bfloat16).eval()


class Tok:
    pad_token_id, eos_token_id = 0, -1


def test_decoder_of_a_transformers_model(monkeypatch):
    from flashgrpo_amd.decoding import FlashMedusaConfig, FlashMedusaDecoder
    from flashgrpo_amd.models import MedusaHeads, target

    hf = hf_model()
    dec = FlashMedusaDecoder(hf, MedusaHeads(256, 97, 2).to(DEV), Tok(),
                             FlashMedusaConfig(num_medusa_heads=2, tree_mode="fixed", max_tree_nodes_per_seq=8, max_tree_depth=3,
                                               fixed_tree_topk_by_depth=(3, 1), do_sample=False))
    dec.model.quantize_mlp()
    ids = torch.randint(1, 97, (2, 19))
    calls = []

    class Counted:
        def __getattr__(self, name):
            if name == "mx_linear":
                calls.append(name)
            return getattr(K(), name)

    monkeypatch.setattr(target, "K", Counted())
    out = dec.generate(ids, torch.ones_like(ids), max_length=30)
    assert all(len(g) == 11 for g in out["generated_token_ids"]) and calls
    old = dec.model.mlp_mx[0][0].codes.clone()
    with torch.no_grad():
        hf.model.layers[0].mlp.gate_proj.weight.mul_(-1.5)
    dec.generate(ids, torch.ones_like(ids), max_length=24)  # the rollout starts with the new weights
    fresh = K().mx_quantize(dec.model.w["layers"][0]["gate_up_w"], "e2m1")
    assert not torch.equal(dec.model.mlp_mx[0][0].codes, old) and torch.equal(dec.model.mlp_mx[0][0].codes, fresh.codes)


def test_wrapper_functions_of_a_transformers_model():
    from flashgrpo_amd.models.qwen_flashgrpo_wrapper import as_target_model, prefill

    hf = hf_model()
    ids = torch.randint(1, 97, (2, 19), device=DEV)
    mask = torch.ones_like(ids)
    with torch.inference_mode():
        full = prefill(hf, ids, mask)
        as_target_model(hf).quantize_mlp()
        quantised = prefill(hf, ids, mask)
        assert as_target_model(hf).mlp_mx is not None
        as_target_model(hf).quantize_mlp(False)
        again = prefill(hf, ids, mask)
    a, b, c = ([v for v in p.values() if torch.is_tensor(v) and v.is_floating_point()] for p in (full, quantised, again))
    assert a and all(torch.equal(x, y) for x, y in zip(a, c)) and not all(torch.equal(x, y) for x, y in zip(a, b))


def test_rows_past_32_bits():
    """Quantisation, values and norm of 5 x 2^30 elements (10 GB): chunks are what their rows alone give."""
    k, rows, cols = K(), 655363, 8192
    x = torch.empty(rows, cols, dtype=torch.bfloat16, device=DEV)
    for r in range(0, rows, 65536):
        g = torch.Generator(device=DEV).manual_seed(r)
        x[r:r + 65536].normal_(generator=g)
    w = torch.ones(cols, dtype=torch.bfloat16, device=DEV)
    at = torch.tensor([0, 1, 262143, 262144, 300001, 524287, 524288, rows - 1], device=DEV)
    some = x[at]
    for fmt in ("e4m3", "e2m1"):
        q, part = k.mx_quantize(x, fmt), k.mx_quantize(some, fmt)
        assert torch.equal(q.codes.view(torch.uint8)[at], part.codes.view(torch.uint8)) and torch.equal(q.scales[:, at], part.scales)
        y = k.mx_dequantize(q)
        assert torch.equal(y[at], k.mx_dequantize(part))
        del y, q
    n, part = k.rmsnorm_mx(x, w, 1e-6), k.rmsnorm_mx(some, w, 1e-6)
    assert torch.equal(n.codes.view(torch.uint8)[at], part.codes.view(torch.uint8)) and torch.equal(n.scales[:, at], part.scales)


@pytest.mark.parametrize("fmt", ["e4m3", "e2m1"])
@pytest.mark.parametrize("rows,n,k", [(655363, 40, 8192), (40003, 65544, 32), (1300003, 33, 32)])
def test_products_past_32_bits(fmt, rows, n, k):
    """Rows of 5 GB of codes, and an output of 5 GB: rows at the start, the borders of 2^31 and 2^32 bytes and the end."""
    (x, xv), (w, wv) = device_pair(rows, k, fmt, 1), device_pair(n, k, "e2m1", 2)
    out = K().mx_linear(x, w)
    borders = [0, 2 ** 31 // k, 2 ** 32 // k, 2 ** 31 // (2 * n), 2 ** 32 // (2 * n), rows - 1]
    at = torch.tensor(sorted({min(max(b + d, 0), rows - 1) for b in borders for d in (-1, 0, 1)}), device=DEV)
    exact, err = product_bound(xv[at].double().cpu().numpy(), wv.double().cpu().numpy(), fmt)
    check_linear(out[at], exact, err)


def test_gate_up_past_32_bits():
    k = K()
    rows, inter = 240007, 18944
    (x, _), (w, _) = device_pair(rows, 32, "e4m3", 1, spread=0.5), device_pair(2 * inter, 32, "e2m1", 2, 0.18, 0.5)
    q = k.mx_gate_up_swiglu(x, w)
    at = torch.tensor([0, 2 ** 31 // inter, 2 ** 31 // inter + 1, 2 ** 32 // inter, 2 ** 32 // inter + 1, rows - 1], device=DEV)
    some = k.MX(x.codes.view(torch.uint8)[at].contiguous().view(torch.float8_e4m3fn), x.scales[:, at].contiguous())
    part = k.mx_gate_up_swiglu(some, w)
    a, b = q.codes.view(torch.uint8)[at], part.codes.view(torch.uint8)
    # another kernel for so few rows: values within d of one another (test_gpu_mx_precision.py), codes 2^-4 apart or more
    d = 2 * (1 + 8) * 2.0 ** -24
    assert float((a != b).float().mean()) <= 2 * 2 * d / 2.0 ** -4
    assert float((q.scales[:, at] != part.scales).float().mean()) <= 32 * 4 * d
