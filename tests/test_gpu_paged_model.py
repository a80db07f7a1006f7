"""The paged cache through the target model, the wrapper's functions and the decoder."""
import numpy as np
import pytest
import torch

from flashgrpo_amd.decoding import FlashMedusaConfig, FlashMedusaDecoder, extract_accepted_path_kv
from flashgrpo_amd.models import MedusaHeads, PagedKVCache, TargetConfig, TargetModel
from flashgrpo_amd.models import qwen_flashgrpo_wrapper as W

pytestmark = pytest.mark.gpu
DEV = "cuda"
FORMATS = ["bf16", "e4m3"]


@pytest.fixture(scope="module", autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


@pytest.fixture(scope="module")
def model():
    return TargetModel.random(TargetConfig(2, 256, 4, 2, 128, 512, 512), seed=1, std=0.05, device=DEV)


@pytest.fixture(scope="module")
def heads(model):
    h = MedusaHeads(256, 512, 3).to(DEV, torch.bfloat16)
    g = torch.Generator().manual_seed(0)
    with torch.no_grad():
        for x in h.heads:
            x.fc.weight.copy_(0.02 * torch.randn(256, 256, generator=g))
    return h


class Tok:
    pad_token_id, eos_token_id = 0, -1


def decoder(model, heads, **kw):
    return FlashMedusaDecoder(model, heads, Tok(), FlashMedusaConfig(
        tree_mode="fixed", max_tree_nodes_per_seq=16, fixed_tree_topk_by_depth=(4, 2, 1), num_medusa_heads=3, top_p=1.0, noise_seed=5, **kw))


def prompts(n, length, seed=2):
    return torch.from_numpy(np.random.default_rng(seed).integers(0, 512, (n, length)))


def tree(n):
    anc, pos = [1], [0]
    for i in range(1, n):
        p = (i - 1) // 2
        anc.append(anc[p] | 1 << i)
        pos.append(pos[p] + 1)
    return torch.tensor(anc, dtype=torch.int64, device=DEV), torch.tensor(pos, dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("fmt", FORMATS)
def test_forward_next_to_the_contiguous_cache(model, fmt):
    """Prefill of ragged prompts and a tree on both caches. Each layer's two branches are off by a few bf16 roundings (2^-8 of
    what they add), on 8-bit pages by the rounding of K and V too (2^-4 of each element at most, random, in a softmax's mean of
    them): 8 roundings of 2^-8 in each of 2 layers, or 2^-3 of the whole."""
    ids, lens = prompts(3, 90), [90, 17, 64]
    want_cache, cache = model.new_cache(3, 160), model.new_cache(3, 160, kv_format=fmt, page_size=16)
    a = model.prefill(ids, want_cache, lengths=lens, chunk=40)
    b = model.prefill(ids, cache, lengths=lens, chunk=40)
    assert cache.seq_len.tolist() == lens
    most = 16 * 2.0 ** -8 if fmt == "bf16" else 2.0 ** -3
    rel = lambda x, y: ((x.float() - y.float()).norm() / y.float().norm()).item()
    assert rel(b, a) < most
    anc, pos = tree(13)
    tok = prompts(3, 13, 3).to(DEV, torch.int32)
    cache.reserve(np.array(lens) + 13, first=lens)
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    x = model.forward(tok, want_cache, pos_offset=pos, anc=anc)
    y = model.forward(tok, cache, pos_offset=pos, anc=anc, err_flag=err)
    assert err.item() == 0 and rel(y, x) < most
    # layer 0's K and V follow from the tokens alone: those of the contiguous cache, or their 8-bit forms
    for i, (p, c) in enumerate(((cache.k(0), want_cache.k(0)), (cache.v(0), want_cache.v(0)))):
        for r, n in enumerate(lens):
            u, v = p[r, :, :n].float(), c[r, :, :n].float()
            if fmt == "bf16" and i == 1:
                assert torch.equal(u, v)
            else:  # 2^-4 of a value and half a step of 2^-9 of its block's scale (at most 2^-8 of its largest); K: HF's roundings
                top = v.unflatten(-1, (-1, 32)).abs().amax(-1, keepdim=True).expand(*v.shape[:-1], 4, 32).flatten(-2)
                turn = 0.0 if i else 8 * 2.0 ** -8 * (v.abs() + v.roll(64, -1).abs())
                assert ((u - v).abs() <= (0 if fmt == "bf16" else 2.0 ** -4) * (v.abs() + turn) + 2.0 ** -17 * top + turn).all()
    # slots without a page are reported
    model.forward(tok, cache, pos_offset=pos, anc=anc, seq_len=cache.seq_len + 60, err_flag=err)
    assert err.item() & 8


@pytest.mark.parametrize("fmt", FORMATS)
def test_shared_prompts_give_what_copies_give(model, fmt):
    """Repeats that share a prompt's pages against a cache in which every row has pages of its own, bit for bit, over rounds."""
    ids, lens = prompts(2, 50), [50, 33]
    first = model.new_cache(6, 120, kv_format=fmt, page_size=16)
    model.prefill(ids, first, lengths=lens, row_map=torch.tensor([0, 3], dtype=torch.int32, device=DEV))
    first.repeat_rows(torch.tensor([0, 0, 3, 3]), torch.tensor([1, 2, 4, 5]))
    own = first.select_rows(torch.arange(6))
    assert first._uses.max() == 3 and own._uses.max() == 1
    anc, pos = tree(10)
    g = np.random.default_rng(4)
    for step in range(3):
        tok = torch.from_numpy(g.integers(0, 512, (6, 10))).to(DEV, torch.int32)
        nodes = torch.tensor([[0, 1, 4], [0, 2, 5], [0, 2, 6], [0, 1, 3], [0, 0, 0], [0, 2, 5]], dtype=torch.int32, device=DEV)
        lens_d = torch.tensor([3, 2, 3, 1, 1, 3], dtype=torch.int32, device=DEV)
        got = []
        for c in (first, own):
            at = c.seq_len.cpu().numpy()
            c.reserve(at + 10, first=at)
            got.append(model.forward(tok, c, pos_offset=pos, anc=anc).clone())
            c.gather_path(c.seq_len, nodes, lens_d, 10)
            c.seq_len += lens_d
        assert torch.equal(*got)
    for l in range(2):
        for r in range(6):
            n = int(first.seq_len[r])
            assert torch.equal(first.k(l)[r, :, :n], own.k(l)[r, :, :n]) and torch.equal(first.v(l)[r, :, :n], own.v(l)[r, :, :n])


@pytest.mark.parametrize("fmt", FORMATS)
def test_graph_of_the_forward(model, fmt):
    cache = model.new_cache(4, 100, kv_format=fmt)
    model.prefill(prompts(4, 30), cache)
    cache.reserve(60)
    anc, pos = tree(7)
    for step in range(4):
        tok = prompts(4, 7, step).to(DEV, torch.int32)
        seq = cache.seq_len + step
        want = model.forward(tok, cache, pos_offset=pos, anc=anc, seq_len=seq).clone()
        assert torch.equal(model.forward(tok, cache, pos_offset=pos, anc=anc, seq_len=seq, graph=True), want)
    assert any(g for g in model._graphs.values())
    model.drop_graphs(cache)
    assert not model._graphs


@pytest.mark.parametrize("kind", ["paged", "paged_e4m3"])
@pytest.mark.parametrize("mode", ["extract_path", "recompute_accepted"])
def test_rollout(model, heads, kind, mode):
    """A whole rollout with repeats: the same with and without graphs, and whatever the page size, of the right lengths."""
    ids, mask = prompts(2, 20), torch.ones(2, 20, dtype=torch.long)
    mask[1, :6] = 0
    outs = [decoder(model, heads, kv_cache=kind, cache_update_mode=mode, graph_verify_forward=g, kv_page_size=p).generate(
        ids, mask, repeated_generate_nums=3, max_length=48)["generated_token_ids"] for g, p in ((True, 16), (False, 16), (True, 64))]
    assert outs[0] == outs[1] == outs[2]
    assert [len(x) for x in outs[0]] == [28] * 3 + [34] * 3 and all(0 <= t < 512 for x in outs[0] for t in x)
    assert len({tuple(x) for x in outs[0]}) == 6


def test_rollout_on_bf16_pages_follows_the_contiguous_one(model, heads):
    """The first token of each sequence is drawn from logits that the cache has no part in but through rounding."""
    ids, mask = prompts(4, 24, 5), torch.ones(4, 24, dtype=torch.long)
    a, b = (decoder(model, heads, kv_cache=k).generate(ids, mask, max_length=30)["generated_token_ids"] for k in ("contiguous", "paged"))
    assert [len(x) for x in a] == [len(x) for x in b]


def test_config_and_models_that_are_refused(model, heads):
    with pytest.raises(ValueError, match="kv_cache"):
        decoder(model, heads, kv_cache="pages")
    f32 = TargetModel.random(TargetConfig(1, 64, 1, 1, 64, 64, 64), dtype=torch.float32, device=DEV)
    with pytest.raises(ValueError, match="bf16"):
        f32.new_cache(1, 16, kv_format="e4m3")
    with pytest.raises(ValueError, match="new_len"):
        c = model.new_cache(1, 16)
        model.forward(torch.zeros(1, 1, dtype=torch.int32, device=DEV), c, pos_offset=torch.zeros(1, dtype=torch.int32, device=DEV), anc=None,
                      new_len=torch.ones(1, dtype=torch.int32, device=DEV))


@pytest.mark.parametrize("fmt", FORMATS)
def test_wrapper_functions(model, fmt):
    """prefill, forward_tokens, forward_tree and the accepted path's extraction of the wrapper over a paged cache."""
    ids, mask = prompts(2, 12), torch.ones(2, 12, dtype=torch.long)
    mask[0, :3] = 0
    out = W.prefill(model, ids, mask, capacity=64, kv_format=fmt)
    cache = out["past_key_values"]
    assert isinstance(cache, PagedKVCache) and W.cache_seq_length(cache) == 12
    rep = W.repeat_interleave_cache(cache, 2)
    assert isinstance(rep, PagedKVCache) and rep.seq_len.tolist() == [9, 9, 12, 12]
    new = prompts(2, 3, 7)
    full = torch.cat([torch.ones(2, 12, dtype=torch.long).masked_fill(mask == 0, 0), torch.ones(2, 3, dtype=torch.long)], 1)
    pos = mask.sum(1, keepdim=True) + torch.arange(3)
    a = W.forward_tokens(model, new, full, W.clone_cache(cache, clone_tensors=True), pos)
    b = W.forward_tokens(model, new, full, cache, pos)
    assert torch.equal(a["hidden_states"], b["hidden_states"]) and cache.seq_len.tolist() == [12, 15]
    N = 4
    P = 15
    m4 = torch.full((2, 1, N, P + N), torch.finfo(torch.float32).min, device=DEV)
    for r, n in enumerate((12, 15)):
        m4[r, :, :, :n] = 0
    sees = torch.tensor([[1, 0, 0, 0], [1, 1, 0, 0], [1, 0, 1, 0], [1, 1, 0, 1]], dtype=torch.bool, device=DEV)
    m4[:, 0, :, P:].masked_fill_(sees, 0)
    depth = torch.tensor([0, 1, 1, 2], device=DEV)
    t = W.forward_tree(model, prompts(2, N, 8), m4, cache, cache.seq_len.long()[:, None] + depth)
    assert t["logits"].shape == (2, N, 512) and torch.isfinite(t["logits"].float()).all()
    tree_cache = t["past_key_values"]
    want = [tree_cache.k(1)[0, :, 12 + i].clone() for i in (0, 1, 3)]
    got = extract_accepted_path_kv(cache, tree_cache, [[0, 1, 3], [0]]).past_key_values
    assert got.seq_len.tolist() == [15, 16] and cache.seq_len.tolist() == [12, 15]
    assert all(torch.equal(got.k(1)[0, :, 12 + j], w) for j, w in enumerate(want))


@pytest.mark.parametrize("fmt", FORMATS)
def test_a_captured_forward_belongs_to_one_table(model, fmt):
    """A second cache over the same pool, with a table (and scales) of its own, does not replay the first one's graph."""
    ids, lens = prompts(2, 40), [40, 23]
    first = model.new_cache(2, 80, kv_format=fmt, page_size=16, pages=20)
    model.prefill(ids, first, lengths=lens)
    first.reserve(np.array(lens) + 8, first=lens)
    anc, pos = tree(8)
    tok = prompts(2, 8, 9).to(DEV, torch.int32)
    want = model.forward(tok, first, pos_offset=pos, anc=anc).clone()
    for _ in range(3):
        assert torch.equal(model.forward(tok, first, pos_offset=pos, anc=anc, graph=True), want)
    second = first.container_copy()  # its rows in the other order
    second.table = first.table.flip(0).contiguous()
    second.scales = None if first.scales is None else first.scales.clone()
    second.seq_len = first.seq_len.flip(0).contiguous()
    second._make_views()
    for _ in range(3):
        assert torch.equal(model.forward(tok.flip(0), second, pos_offset=pos, anc=anc, graph=True), want.flip(0))
    model.drop_graphs(first)
