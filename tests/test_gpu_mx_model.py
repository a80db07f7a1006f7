"""``TargetModel.quantize_mlp``: the decoder layers' MLPs on 4-bit weights and 8-bit rows.

Every MX call that a forward makes is compared with the float64 oracle on the call's own inputs (bounds as in
test_gpu_mx.py), and the forward eager with captured, quantised with not quantised again, and before with after a
weight update.
"""
import numpy as np
import pytest
import torch

from oracle import model as OM
from test_gpu_mx import check_gate_up, check_linear, held, host, norm_oracle, product_bound

pytestmark = pytest.mark.gpu
DEV = "cuda"
CFG = OM.ModelConfig(num_layers=2, hidden=512, q_heads=8, kv_heads=2, head_dim=128, intermediate=768, vocab=1000)


@pytest.fixture(scope="module", autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


def build(seed=3):
    from flashgrpo_amd.models.target import TargetConfig, TargetModel

    c = CFG
    t = TargetConfig(c.num_layers, c.hidden, c.q_heads, c.kv_heads, c.head_dim, c.intermediate, c.vocab, c.rope_theta,
                     c.rms_eps, c.qkv_bias, c.tie_word_embeddings)
    return TargetModel.from_numpy(t, OM.random_weights(c, seed=seed, std=0.05), dtype=torch.bfloat16, device=DEV)


def run(m, *, graph=False, calls=1):
    """Hidden states of a prefill of 3 prompts and a tree of 10 nodes after it, and the cache."""
    from flashgrpo_amd.decoding.medusa_tree import TreeTopology

    rng = np.random.default_rng(6)
    prompts = torch.from_numpy(rng.integers(0, CFG.vocab, (3, 41))).to(DEV)
    topo = TreeTopology([3, 2, 1], 12)
    d = topo.device(DEV)
    toks = torch.from_numpy(rng.integers(0, CFG.vocab, (3, topo.num_nodes))).to(DEV).to(torch.int32)
    cache = m.new_cache(3, 128)
    last = m.prefill(prompts, cache).clone()
    for _ in range(calls):
        tree = m.forward(toks, cache, pos_offset=d["pos_offset"], anc=d["anc"], graph=graph).clone()
    return last, tree, cache.kv.clone()


def same(a, b):
    return all(torch.equal(x, y) for x, y in zip(a, b))


def test_forward_runs_the_operators_and_switches_back(monkeypatch):
    from flashgrpo_amd import kernels as K
    from flashgrpo_amd.models import target

    m = build()
    before = run(m)
    assert m.quantize_mlp() is m and len(m.mlp_mx) == 2
    got = run(m)
    assert not same(got, before)
    calls = []

    class Checked:
        """The kernels module, the MLP's three operators checked against the oracle call by call."""

        def __getattr__(self, name):
            return getattr(K, name)

        def rmsnorm_mx(self, x, w, eps, *, out):
            q = K.rmsnorm_mx(x, w, eps, out=out)
            codes, scales = held(q)
            want_c, want_s = norm_oracle(x.cpu(), w.cpu(), float(np.float32(eps)), None)[1]
            assert np.array_equal(codes, want_c) and np.array_equal(scales, want_s)
            calls.append("norm")
            return q

        def mx_gate_up_swiglu(self, x, w, *, out):
            q = K.mx_gate_up_swiglu(x, w, out=out)
            check_gate_up(q, host(x), host(w), "e4m3")
            calls.append("gate_up")
            return q

        def mx_linear(self, x, w, *, residual, out):
            assert residual is out
            exact, err = product_bound(host(x), host(w), "e4m3")
            r = residual.clone()
            K.mx_linear(x, w, residual=residual, out=out)
            check_linear(out, exact, err, residual=r)
            calls.append("linear")
            return out

    monkeypatch.setattr(target, "K", Checked())
    assert same(run(m), got)
    monkeypatch.undo()
    assert calls == ["norm", "gate_up", "linear"] * (2 * CFG.num_layers)  # a prefill and a tree forward
    m.quantize_mlp(False)
    assert m.mlp_mx is None and same(run(m), before)


def test_captured_forward_is_the_eager_one():
    m = build().quantize_mlp()
    eager = run(m)
    captured = run(m, graph=True, calls=5)
    assert m._graphs and all(g is not None for g in m._graphs.values())
    assert same(eager, captured)


def test_copies_follow_the_weights():
    transformers = pytest.importorskip("transformers")
    from flashgrpo_amd import kernels as K
    from flashgrpo_amd.models import TargetModel

    hc = transformers.Qwen2Config(vocab_size=64, hidden_size=256, intermediate_size=512, num_hidden_layers=2,
                                  num_attention_heads=2, num_key_value_heads=1, max_position_embeddings=512)
    torch.manual_seed(0)
    hf = transformers.Qwen2ForCausalLM(hc).to(DEV).to(torch.bfloat16).eval()
    m = TargetModel.from_hf(hf).quantize_mlp()
    held = [t.data_ptr() for pair in m.mlp_mx for q in pair for t in q]
    old = m.mlp_mx[1][1].codes.clone()
    with torch.no_grad():
        hf.model.layers[1].mlp.down_proj.weight.add_(0.05 * torch.randn_like(hf.model.layers[1].mlp.down_proj.weight))
        hf.model.layers[0].mlp.up_proj.weight.mul_(3.0)
    assert m.sync_from_hf() and not torch.equal(m.mlp_mx[1][1].codes, old)
    assert [t.data_ptr() for pair in m.mlp_mx for q in pair for t in q] == held
    for lw, (gate_up, down) in zip(m.w["layers"], m.mlp_mx):
        for w, q in ((lw["gate_up_w"], gate_up), (lw["down_w"], down)):
            fresh = K.mx_quantize(w, "e2m1")
            assert torch.equal(fresh.codes, q.codes) and torch.equal(fresh.scales, q.scales)


def test_rollout_on_a_quantised_target():
    """A greedy rollout samples the quantised model: its first hidden states are the quantised prefill's, every root and
    accepted token is the argmax of the round's own logits, and captured and eager rollouts emit the same tokens."""
    from flashgrpo_amd.decoding import FlashMedusaConfig, FlashMedusaDecoder
    from flashgrpo_amd.models import MedusaHeads

    class Tok:
        pad_token_id, eos_token_id = 0, -1

    m = build(seed=5)
    prompts = torch.from_numpy(np.random.default_rng(1).integers(0, CFG.vocab, (2, 21)))
    full = m.prefill(prompts.to(DEV), m.new_cache(2, 64)).clone()
    m.quantize_mlp()
    hidden = m.prefill(prompts.to(DEV), m.new_cache(2, 64)).float().cpu().numpy()
    heads = MedusaHeads(CFG.hidden, CFG.vocab, 3).to(DEV)
    kw = dict(num_medusa_heads=3, tree_mode="fixed", max_tree_nodes_per_seq=16, max_tree_depth=4,
              fixed_tree_topk_by_depth=(4, 2, 1), do_sample=False, noise_seed=1)
    outs, trace = [], []
    for graph, tr in ((False, trace), (False, None), (True, None)):
        dec = FlashMedusaDecoder(m, heads, Tok(), FlashMedusaConfig(graph_verify_forward=graph, **kw))
        outs.append(dec.generate(prompts, torch.ones(2, 21, dtype=torch.long), max_length=21 + 16, trace=tr))
    assert outs[0]["generated_token_ids"] == outs[1]["generated_token_ids"] == outs[2]["generated_token_ids"]
    assert all(len(g) == 16 for g in outs[0]["generated_token_ids"])
    assert np.array_equal(trace[0]["hidden_in"], hidden) and not np.array_equal(full.float().cpu().numpy(), hidden)
    for rec in trace:
        assert rec["roots"].tolist() == rec["logits_in"].argmax(-1).tolist()
        for i in range(len(rec["active"])):
            for t in range(int(rec["acc_len"][i]) - 1):
                assert int(rec["acc_tokens"][i, t + 1]) == int(rec["walk_logits"][t, i].argmax())
