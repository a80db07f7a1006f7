"""Torch-facing wrappers over the C ABI (one function per entry point).

Each wrapper checks devices, dtypes and shapes on the host, passes raw
pointers plus torch's current HIP stream, and raises on any error code. All
device work happens in the HIP kernels of ``ss-grpo_amd/csrc``.
"""
from __future__ import annotations

import ctypes as C
import functools
import math
from typing import NamedTuple

import torch

from . import _lib, timing

F32, BF16 = 0, 1


def _call(name: str, *args) -> None:
    if timing.idle():  # no timer installed: launch directly (the context manager costs ~3 us)
        _lib.call(name, *args)
        return
    with timing.launch(name):
        _lib.call(name, *args)
_DT = {torch.float32: F32, torch.bfloat16: BF16}


def dtype_code(t: torch.Tensor) -> int:
    try:
        return _DT[t.dtype]
    except KeyError:
        raise TypeError(f"unsupported dtype {t.dtype}; expected float32 or bfloat16") from None


def _ptr(t):
    return None if t is None else t.data_ptr()


_raw_stream = torch._C._cuda_getCurrentRawStream
_cur_device = torch._C._cuda_getDevice


def _stream() -> int:
    """hipStream_t of torch's current stream on the current device (the two direct
    C calls cost ~1 us; torch.cuda.current_stream() costs ~9 us per launch)."""
    return _raw_stream(_cur_device())


_SCRATCH = {}
_SCRATCH_RETIRED = []


def _scratch(name: str, nbytes: int, device) -> torch.Tensor:
    """A cached uint8 device buffer of at least nbytes for one kind of workspace.
    Launches are ordered on the current stream, so successive calls may share it.
    A buffer outgrown is kept alive: a captured graph may still address it."""
    key = (name, str(device))
    buf = _SCRATCH.get(key)
    if buf is None or buf.numel() < nbytes:
        if buf is not None:
            _SCRATCH_RETIRED.append(buf)
        buf = torch.empty(int(nbytes), dtype=torch.uint8, device=device)
        _SCRATCH[key] = buf
    return buf


def _dev(*ts):
    for t in ts:
        if t is not None and not t.is_cuda:
            raise ValueError("flashgrpo_amd kernels take device tensors (got a CPU tensor)")


def _i32(t, name):
    if t is not None and t.dtype != torch.int32:
        raise TypeError(f"{name} must be int32")


def aligned_rows(x: torch.Tensor) -> torch.Tensor:
    """x itself when its rows start 32-byte aligned with a stride that is a
    multiple of 8 elements (what the row kernels load with 16-byte vectors),
    otherwise a padded copy viewed back to x's shape."""
    x2 = x.reshape(-1, x.shape[-1]) if x.dim() != 2 else x
    if x2.stride(-1) == 1 and x2.stride(0) % 8 == 0 and x2.data_ptr() % 32 == 0:
        return x2
    V = x2.shape[-1]
    pad = torch.empty(x2.shape[0], (V + 7) // 8 * 8, dtype=x2.dtype, device=x2.device)
    pad[:, :V].copy_(x2)
    return pad[:, :V]


def top_p_fixed(top_p) -> int:
    """floor(top_p * 2^32) for 0 < top_p < 1, else 0 (no nucleus cut)."""
    if top_p is None or not (0.0 < float(top_p) < 1.0):
        return 0
    return int(float(top_p) * 4294967296.0)


# ------------------------------------------------------------------ contractions
def medusa_heads(hidden, ln_w, ln_b, fc_w, fc_b, *, eps=1e-5, out=None, out_dtype=None, workspace=None):
    """[heads*B, H] = hidden + SiLU(fc(LayerNorm(hidden))) per head (heads stacked)."""
    _dev(hidden, ln_w, ln_b, fc_w, fc_b)
    B, H = hidden.shape
    heads = fc_w.shape[0]
    if hidden.stride(1) != 1 or fc_w.shape[1:] != (H, H) or not fc_w.is_contiguous() or not fc_b.is_contiguous():
        raise ValueError("medusa_heads: expected hidden [B,H] row-major, fc_w [heads,H,H], fc_b [heads,H]")
    if fc_w.dtype != hidden.dtype or fc_b.dtype != hidden.dtype:
        raise TypeError("medusa_heads: fc weights must share the hidden dtype")
    ln_w = ln_w.float().contiguous()
    ln_b = ln_b.float().contiguous()
    od = out_dtype or hidden.dtype
    if out is None:
        out = torch.empty(heads * B, H, dtype=od, device=hidden.device)
    need = _lib.load().fg_medusa_heads_workspace(B, H, heads, dtype_code(hidden))
    if workspace is None or workspace.numel() * workspace.element_size() < need:
        workspace = torch.empty(need, dtype=torch.uint8, device=hidden.device)
    _call("fg_medusa_heads", _ptr(hidden), dtype_code(hidden), B, H, hidden.stride(0), heads, _ptr(ln_w),
              _ptr(ln_b), float(eps), _ptr(fc_w), _ptr(fc_b), _ptr(out), dtype_code(out), _ptr(workspace),
              workspace.numel() * workspace.element_size(), _stream())
    return out


def lm_head(x, weight, *, row_index=None, row_active=None, out=None, out_dtype=None):
    """out[m] = x[row_index[m] if row_index is given else m] @ weight.T

    row_active (int32 [M], optional): output tiles whose rows are all 0 are skipped."""
    _dev(x, weight, row_index, row_active)
    _i32(row_index, "row_index")
    _i32(row_active, "row_active")
    K = x.shape[-1]
    x2 = x.reshape(-1, K)
    if x2.stride(1) != 1 or weight.stride(1) != 1 or weight.shape[1] != K:
        raise ValueError("lm_head: operands must be K-contiguous with matching K")
    if x.dtype != weight.dtype:
        raise TypeError("lm_head: x and weight dtypes differ")
    M = row_index.numel() if row_index is not None else x2.shape[0]
    N = weight.shape[0]
    od = out_dtype or x.dtype
    if out is None:
        out = torch.empty(M, N, dtype=od, device=x.device)
    if M == 0:
        return out
    _call("fg_lm_head", _ptr(x2), dtype_code(x), M, K, x2.stride(0), _ptr(row_index), _ptr(row_active),
          _ptr(weight), weight.stride(0), N, _ptr(out), dtype_code(out), out.stride(0), _stream())
    return out


def lm_head_parts(vocab):
    """Row maxima parts per row that ``lm_head_topk(..., parts=...)`` writes."""
    return int(_lib.load().fg_lm_head_topk_parts(int(vocab)))


def lm_head_topk(x, weight, kmax=0, *, row_index=None, row_active=None, out=None, out_dtype=None,
                 logits=True, stats=False, sanitize=False, workspace=None, parts=None):
    """Tied LM head over <= 256 rows (bf16) on the weight-streaming kernel, with the
    per-row top-kmax candidates fused (``fg_lm_head_topk``).

    Returns (logits [M, N] or None, tokens int32 [M, kmax] or None, scores fp32 [M, kmax]
    or None, stats fp32 [M, 2] or None); the candidates and stats equal
    ``medusa_topk(logits, kmax, stats=..., sanitize=...)`` on the bf16 logits.
    ``parts`` (kmax 0): a (part_max fp32, part_key int64) pair of [M, lm_head_parts(N)]
    tensors that receive each row's per-workgroup maxima (for ``walk_step``).
    """
    _dev(x, weight, row_index, row_active)
    _i32(row_index, "row_index")
    _i32(row_active, "row_active")
    K = x.shape[-1]
    x2 = x.reshape(-1, K)
    if x2.dtype != torch.bfloat16 or weight.dtype != torch.bfloat16:
        raise TypeError("lm_head_topk: x and weight must be bf16")
    if x2.stride(1) != 1 or weight.stride(1) != 1 or weight.shape[1] != K:
        raise ValueError("lm_head_topk: operands must be K-contiguous with matching K")
    if (x2.numel() + x2.storage_offset()) * 2 >= 1 << 32:
        raise ValueError("lm_head_topk: x must span less than 4 GiB")
    M = row_index.numel() if row_index is not None else x2.shape[0]
    N = weight.shape[0]
    dev = x.device
    if logits and out is None:
        out = torch.empty(M, N, dtype=out_dtype or torch.bfloat16, device=dev)
    elif not logits:
        out = None
    elif out is not None:
        _dev(out)
        if out.dtype not in (torch.bfloat16, torch.float32) or (out_dtype is not None and out.dtype != out_dtype):
            raise TypeError("lm_head_topk: out must be bf16 or fp32 (and match out_dtype)")
        if out.dim() != 2 or tuple(out.shape) != (M, N) or out.stride(1) != 1 or out.stride(0) < N:
            raise ValueError(f"lm_head_topk: out must be a [{M}, {N}] view with unit column stride")
        if out.stride(0) % 4 == 0 and out.data_ptr() % (4 * out.element_size()):
            raise ValueError("lm_head_topk: out rows with a stride of 4k elements need a base aligned to 4 columns")
    tok = torch.empty(M, kmax, dtype=torch.int32, device=dev) if kmax else None
    sc = torch.empty(M, kmax, dtype=torch.float32, device=dev) if kmax else None
    st = torch.empty(M, 2, dtype=torch.float32, device=dev) if kmax and stats else None
    if M == 0:
        return out, tok, sc, st
    ws_bytes = 0
    if kmax:
        need = _lib.load().fg_lm_head_topk_workspace(M, N, kmax)
        if workspace is None or workspace.numel() * workspace.element_size() < need:
            workspace = torch.empty(need, dtype=torch.uint8, device=dev)
        ws_bytes = workspace.numel() * workspace.element_size()
    else:
        workspace = None
    pmax = pkey = None
    if parts is not None:
        pmax, pkey = parts
        P = lm_head_parts(N)
        if (kmax or pmax.dtype != torch.float32 or pkey.dtype != torch.int64 or tuple(pmax.shape) != (M, P)
                or tuple(pkey.shape) != (M, P) or not pmax.is_contiguous() or not pkey.is_contiguous()):
            raise ValueError(f"lm_head_topk: parts must be contiguous fp32 / int64 [{M}, {P}] with kmax 0")
    _call("fg_lm_head_topk", _ptr(x2), M, K, x2.stride(0), _ptr(row_index), _ptr(row_active), _ptr(weight),
          weight.stride(0), N, _ptr(out), dtype_code(out) if out is not None else 1,
          out.stride(0) if out is not None else N, int(kmax), int(bool(sanitize)), _ptr(tok), _ptr(sc), _ptr(st),
          _ptr(pmax), _ptr(pkey), _ptr(workspace), ws_bytes, _stream())
    return out, tok, sc, st


# ------------------------------------------------------------------ tree construction
def medusa_topk(logits, kmax, *, stats=False, sanitize=False, workspace=None):
    """Top-kmax candidates per row ranked (value desc, index asc).

    Returns (tokens int32 [R, kmax], scores fp32 [R, kmax], stats fp32 [R, 2] or None)
    where stats holds (row max, row logsumexp). ``sanitize`` ranks
    nan_to_num(logits, nan=-1e9, posinf=1e9, neginf=-1e9) (chain proposals).
    """
    _dev(logits)
    logits = aligned_rows(logits)
    R, V = logits.shape
    tok = torch.empty(R, kmax, dtype=torch.int32, device=logits.device)
    sc = torch.empty(R, kmax, dtype=torch.float32, device=logits.device)
    st = torch.empty(R, 2, dtype=torch.float32, device=logits.device) if stats else None
    need = _lib.load().fg_medusa_topk_workspace(R, V, kmax)
    if workspace is None or workspace.numel() * workspace.element_size() < need:
        workspace = torch.empty(need, dtype=torch.uint8, device=logits.device)
    _call("fg_medusa_topk", _ptr(logits), dtype_code(logits), logits.stride(0), R, V, kmax, int(bool(sanitize)),
          _ptr(tok), _ptr(sc), _ptr(st), _ptr(workspace), workspace.numel() * workspace.element_size(), _stream())
    return tok, sc, st


def tree_layout(cand_tokens, cand_scores, batch, roots, node_depth, node_rank, num_nodes, *, out_tokens=None,
                out_scores=None):
    _dev(cand_tokens, cand_scores, roots, node_depth, node_rank)
    for t, n in ((cand_tokens, "cand_tokens"), (roots, "roots"), (node_depth, "node_depth"), (node_rank, "node_rank")):
        _i32(t, n)
    dev = roots.device
    if out_tokens is None:
        out_tokens = torch.empty(batch, num_nodes, dtype=torch.int32, device=dev)
    if out_scores is None:
        out_scores = torch.empty(batch, num_nodes, dtype=torch.float32, device=dev)
    kstride = cand_tokens.shape[-1] if cand_tokens is not None else 0
    _call("fg_tree_layout", _ptr(cand_tokens), _ptr(cand_scores), kstride, batch, _ptr(roots), _ptr(node_depth),
              _ptr(node_rank), num_nodes, _ptr(out_tokens), _ptr(out_scores), out_tokens.stride(0), _stream())
    return out_tokens, out_scores


def sparse_tree_layout(cand_tokens, cand_scores, batch, roots, nodes_by_head, *, vocab, budget, num_nodes,
                       temperature=1.0, diversity_penalty=0.0, head3_gate=None, scores=False):
    """Sparse asymmetric trees on the device (``fg_sparse_tree_layout``).

    cand_tokens/cand_scores: [heads*batch, kstride] top-k lists (head-major rows).
    Returns a dict of [batch, num_nodes] int32 ``tokens``, ``parents``, ``depth``,
    ``pos_offset``, ``n_children``, int64 ``anc`` bit masks, ``n_nodes`` [batch], and
    with ``scores`` the fp64 path scores [batch, num_nodes].
    """
    _dev(cand_tokens, cand_scores, roots, head3_gate)
    _i32(cand_tokens, "cand_tokens")
    _i32(roots, "roots")
    nodes = [int(n) for n in nodes_by_head]
    if not nodes:
        raise ValueError("sparse_tree_layout: no heads")
    if cand_tokens.shape[0] < min(len(nodes), 3) * batch or cand_scores.shape != cand_tokens.shape:
        raise ValueError("sparse_tree_layout: candidate rows missing")
    if not (cand_tokens.is_contiguous() and cand_scores.is_contiguous() and cand_scores.dtype == torch.float32):
        raise ValueError("sparse_tree_layout: contiguous int32 tokens and fp32 scores required")
    if head3_gate is not None:
        if head3_gate.dtype not in (torch.bool, torch.uint8) or head3_gate.numel() != batch:
            raise ValueError("sparse_tree_layout: head3_gate must be bool/uint8 [batch]")
        head3_gate = head3_gate.contiguous().view(torch.uint8)
    dev = roots.device
    i32 = dict(dtype=torch.int32, device=dev)
    out = dict(tokens=torch.empty(batch, num_nodes, **i32), parents=torch.empty(batch, num_nodes, **i32),
               depth=torch.empty(batch, num_nodes, **i32), pos_offset=torch.empty(batch, num_nodes, **i32),
               anc=torch.empty(batch, num_nodes, dtype=torch.int64, device=dev),
               n_children=torch.empty(batch, num_nodes, **i32), n_nodes=torch.empty(batch, **i32),
               scores=torch.empty(batch, num_nodes, dtype=torch.float64, device=dev) if scores else None)
    nodes_arr = (C.c_int32 * len(nodes))(*nodes)
    _call("fg_sparse_tree_layout", _ptr(cand_tokens), _ptr(cand_scores), cand_tokens.shape[1], batch, int(vocab),
          _ptr(roots), _ptr(head3_gate), C.cast(nodes_arr, C.c_void_p), len(nodes), int(budget), float(temperature),
          float(diversity_penalty), num_nodes, _ptr(out["tokens"]), _ptr(out["parents"]), _ptr(out["depth"]),
          _ptr(out["pos_offset"]), _ptr(out["anc"]), _ptr(out["n_children"]), _ptr(out["n_nodes"]),
          _ptr(out["scores"]), _stream())
    return out


# ------------------------------------------------------------------ verify forward pieces
def rope_kv_write(qkv, *, batch, num_nodes, q_heads, kv_heads, head_dim, seq_len, pos_offset, inv_freq, q_out,
                  k_cache, v_cache, row_map=None, err_flag=None):
    _dev(qkv, seq_len, pos_offset, inv_freq, q_out, k_cache, v_cache, row_map)
    _i32(seq_len, "seq_len")
    _i32(pos_offset, "pos_offset")
    _i32(row_map, "row_map")
    if k_cache.stride(-1) != 1 or k_cache.stride(-2) != head_dim:
        raise ValueError("rope_kv_write: cache rows must be contiguous [.., capacity, d]")
    if v_cache.stride() != k_cache.stride() or v_cache.shape != k_cache.shape or v_cache.dtype != k_cache.dtype:
        raise ValueError("rope_kv_write: v_cache must have k_cache's shape, strides and dtype")
    width = (q_heads + 2 * kv_heads) * head_dim
    if qkv.dtype != k_cache.dtype or qkv.stride(-1) != 1 or qkv.shape[-1] < width or \
            qkv.numel() // qkv.shape[-1] != batch * num_nodes:
        raise ValueError(f"rope_kv_write: qkv must hold {batch * num_nodes} rows of >= {width} unit-stride values "
                         "in the cache dtype")
    if not q_out.is_contiguous() or q_out.numel() != batch * num_nodes * q_heads * head_dim or \
            q_out.dtype != k_cache.dtype:
        raise ValueError("rope_kv_write: q_out must be a contiguous [batch * num_nodes, q_heads, d] tensor")
    if pos_offset.dim() == 2:
        if tuple(pos_offset.shape) != (batch, num_nodes) or not pos_offset.is_contiguous():
            raise ValueError("rope_kv_write: per-sequence pos_offset must be contiguous [batch, num_nodes]")
        pos_stride = num_nodes
    else:
        if pos_offset.numel() < num_nodes:
            raise ValueError("rope_kv_write: pos_offset shorter than num_nodes")
        pos_stride = 0
    _call("fg_rope_kv_write", _ptr(qkv), dtype_code(qkv), qkv.stride(0), batch, num_nodes, q_heads, kv_heads,
              head_dim, _ptr(seq_len), _ptr(pos_offset), pos_stride, _ptr(inv_freq), _ptr(q_out), _ptr(k_cache),
              _ptr(v_cache),
              k_cache.stride(0), k_cache.stride(1), k_cache.shape[-2], _ptr(row_map), _ptr(err_flag), _stream())


def tree_attention(q, k_cache, v_cache, *, seq_len, anc, num_nodes, q_heads, kv_heads, head_dim, out=None,
                   row_map=None, scale=None):
    """q [B, N, Hq, d]; caches [Bc, Hkv, S, d]; anc uint64 as int64 [B, N] or [N], or None for a
    causal chain of new keys (node n sees new keys 0..n). scale: of the scores (None: d^-0.5),
    positive and finite where q is bf16."""
    _dev(q, k_cache, v_cache, seq_len, anc, row_map)
    _i32(seq_len, "seq_len")
    if anc is not None and anc.dtype != torch.int64:
        raise TypeError("anc must be int64 (bit pattern of the uint64 masks)")
    B = q.shape[0]
    if out is None:
        out = torch.empty_like(q)
    anc_stride = 0 if anc is None or anc.dim() == 1 else anc.stride(0)
    scale = 1.0 / math.sqrt(head_dim) if scale is None else scale
    capacity = k_cache.shape[2]
    ws, ws_bytes = None, 0
    if q.dtype == torch.bfloat16:
        need = _lib.load().fg_tree_attention_workspace(B, num_nodes, q_heads, kv_heads, head_dim, capacity)
        if need:
            ws = _scratch("tree_attention", need, q.device)
            ws_bytes = ws.numel()
    _call("fg_tree_attention", _ptr(q), _ptr(out), _ptr(k_cache), _ptr(v_cache), dtype_code(q), B, num_nodes,
          q_heads, kv_heads, head_dim, k_cache.stride(0), k_cache.stride(1), capacity, _ptr(seq_len),
          _ptr(row_map), _ptr(anc), anc_stride, float(scale), _ptr(ws), ws_bytes, _stream())
    return out


def rmsnorm(x, weight, eps, *, delta=None, out=None):
    """RMSNorm(x [+ delta]) * weight over the last dimension (``fg_rmsnorm``); with delta the
    sum is written back to x first. x, delta and out contiguous, one dtype, one shape."""
    _dev(x, weight, delta)
    H = x.shape[-1]
    rows = x.numel() // H
    if not x.is_contiguous() or weight.numel() != H or weight.dtype != x.dtype or not weight.is_contiguous():
        raise ValueError("rmsnorm: x must be contiguous and weight a contiguous [H] tensor of its dtype")
    if delta is not None and (delta.shape != x.shape or delta.dtype != x.dtype or not delta.is_contiguous()):
        raise ValueError("rmsnorm: delta must be a contiguous tensor of x's shape and dtype")
    if out is None:
        out = torch.empty_like(x)
    elif out.shape != x.shape or out.dtype != x.dtype or not out.is_contiguous():
        raise ValueError("rmsnorm: out must be a contiguous tensor of x's shape and dtype")
    if rows == 0:
        return out
    _call("fg_rmsnorm", _ptr(x), _ptr(delta), _ptr(weight), _ptr(out), dtype_code(x), rows, H, float(eps),
              _stream())
    return out


def swiglu(gate_up, *, out=None):
    """SiLU(gate_up[:, :F]) * gate_up[:, F:] (``fg_swiglu``): gate_up a contiguous [rows, 2F]
    tensor (F a multiple of 8), out a contiguous [rows, F] tensor of the same dtype."""
    _dev(gate_up)
    if gate_up.dim() != 2 or gate_up.shape[1] % 16 or not gate_up.is_contiguous():
        raise ValueError("swiglu: gate_up must be a contiguous [rows, 2F] tensor with F a multiple of 8")
    rows, two_f = gate_up.shape
    F = two_f // 2
    if out is None:
        out = torch.empty(rows, F, dtype=gate_up.dtype, device=gate_up.device)
    elif tuple(out.shape) != (rows, F) or out.dtype != gate_up.dtype or not out.is_contiguous():
        raise ValueError(f"swiglu: out must be a contiguous [{rows}, {F}] tensor of the input dtype")
    if rows == 0:
        return out
    _call("fg_swiglu", _ptr(gate_up), _ptr(out), dtype_code(gate_up), rows, F, _stream())
    return out


class ArrayCopies:
    """Copies into a fixed set of at most 8 small device tensors (``fg_copy_arrays``): calling it with
    one source per destination copies all of them in one launch on the current stream. A source
    that is not a contiguous tensor of its destination's dtype and device is copied by torch."""

    def __init__(self, dsts):
        self.dsts = list(dsts)
        n = len(self.dsts)
        if not 0 < n <= 8 or any(not d.is_contiguous() or d.numel() == 0 for d in self.dsts):
            raise ValueError("ArrayCopies: 1 to 8 contiguous non-empty tensors")
        self.n = n
        self._all = [(d.dtype, d.shape, d.device, d.numel() * d.element_size()) for d in self.dsts]

    def __call__(self, srcs):
        fast = []
        for d, s, (dt, shape, dev, nbytes) in zip(self.dsts, srcs, self._all):
            if (s.dtype == dt and s.shape == shape and s.device == dev and s.is_contiguous() and dev.type == "cuda"
                    and nbytes % 4 == 0 and s.data_ptr() % 4 == 0):
                if s.data_ptr() != d.data_ptr():
                    fast.append((s.data_ptr(), d.data_ptr(), nbytes))
            else:
                d.copy_(s)
        if not fast:
            return
        n = len(fast)
        a, b, c = zip(*fast)
        _call("fg_copy_arrays", (C.c_void_p * n)(*a), (C.c_void_p * n)(*b), (C.c_int64 * n)(*c), n, _stream())


def chain_cell_norm(state, token, state_w, state_b, token_w, token_b, eps, *, out=None):
    """[rows, 2H] = [LayerNorm(state) * state_w + state_b, LayerNorm(token) * token_w + token_b]
    (``fg_chain_cell_norm``): the ChainDraftCell's two normalised inputs side by side. state and
    token [rows, H] in one dtype (unit column stride), the affine weights [H] in that dtype."""
    _dev(state, token, state_w, state_b, token_w, token_b)
    rows, H = state.shape
    if tuple(token.shape) != (rows, H) or token.dtype != state.dtype or state.stride(1) != 1 or token.stride(1) != 1:
        raise ValueError("chain_cell_norm: state and token must be [rows, H] of one dtype with unit column stride")
    ws = [t.contiguous() for t in (state_w, state_b, token_w, token_b)]
    if any(t.dtype != state.dtype or t.numel() != H for t in ws):
        raise ValueError("chain_cell_norm: affine weights must be [H] in the row dtype")
    if out is None:
        out = torch.empty(rows, 2 * H, dtype=state.dtype, device=state.device)
    elif tuple(out.shape) != (rows, 2 * H) or not out.is_contiguous() or out.dtype != state.dtype:
        raise ValueError("chain_cell_norm: out must be a contiguous [rows, 2H] tensor of the row dtype")
    _call("fg_chain_cell_norm", _ptr(state), state.stride(0), _ptr(token), token.stride(0), dtype_code(state), rows, H,
          *[_ptr(t) for t in ws], float(eps), _ptr(out), _stream())
    return out


def chain_cell_step_ok(state, token, weights) -> bool:
    """Whether fg_chain_cell_step takes this cell: everything fp32 on the GPU (the token rows bf16 too),
    hidden a multiple of 8 up to 8192, the bottleneck a multiple of 4, whole rows, 16-byte aligned. ``weights`` are the eight
    tensors after (state, token) of :func:`chain_cell_step`, the gate aside."""
    out_w = weights[6]
    H, bott = out_w.shape
    shapes = [(H,)] * 4 + [(bott, H)] * 2 + [(H, bott), (H,)]
    rows = lambda t: t.shape[-1] == H and t.numel() > 0 and t.is_contiguous()
    return (H % 8 == 0 and 0 < H <= 8192 and bott % 4 == 0 and bott > 0 and state.shape == token.shape
            and rows(state) and rows(token) and all(tuple(w.shape) == s for w, s in zip(weights, shapes))
            and token.dtype in (torch.float32, torch.bfloat16) and token.is_cuda and token.data_ptr() % 16 == 0
            and all(t.is_cuda and t.dtype == torch.float32 and t.is_contiguous() and t.data_ptr() % 16 == 0
                    for t in (state, *weights)))


def chain_cell_step(state, token, state_w, state_b, token_w, token_b, state_proj_w, token_proj_w, out_w, out_b, gate,
                    eps):
    """One fp32 ChainDraftCell step (``fg_chain_cell_step``): state and token [rows, H] contiguous
    (token fp32 or bf16), the projections [bottleneck, H], gate the sigmoid of the cell's gate (one element). Returns the
    new states [rows, H]."""
    weights = (state_w, state_b, token_w, token_b, state_proj_w, token_proj_w, out_w, out_b)
    _dev(state, token, *weights, gate)
    if state.ndim != 2 or not chain_cell_step_ok(state, token, weights) or gate.dtype != torch.float32 \
            or gate.numel() != 1:
        raise ValueError("chain_cell_step: needs contiguous fp32 state and fp32 or bf16 token [rows, H], projections [bottleneck, H], "
                         "out_w [H, bottleneck] with H % 8 == 0, bottleneck % 4 == 0, 16-byte aligned, and an fp32 gate")
    rows, H = state.shape
    bott = out_w.shape[1]
    out = torch.empty(rows, H, dtype=torch.float32, device=state.device)
    ws = torch.empty(_lib.load().fg_chain_cell_step_workspace(rows, H, bott), dtype=torch.uint8, device=state.device)
    _call("fg_chain_cell_step", _ptr(state), H, _ptr(token), H, dtype_code(token), rows, H, bott, *[_ptr(t) for t in weights[:4]],
          float(eps), *[_ptr(t) for t in weights[4:]], _ptr(gate), _ptr(out), _ptr(ws), ws.numel(), _stream())
    return out


def gate_up_swiglu_ok(x, w) -> bool:
    """Whether fg_gate_up_swiglu takes x [rows, hidden] and w [2*inter, hidden] as they are:
    bf16 on the GPU, hidden a multiple of 64, inter a multiple of 4, unit column strides and
    16-byte aligned rows."""
    if not (x.is_cuda and x.dtype == torch.bfloat16 and w.dtype == torch.bfloat16 and x.dim() == 2 and w.dim() == 2):
        return False
    H = x.shape[1]
    if H == 0 or H % 64 or w.shape[1] != H or w.shape[0] % 8 or x.shape[0] == 0:
        return False
    if x.stride(1) != 1 or w.stride(1) != 1 or x.stride(0) % 8 or w.stride(0) % 8:
        return False
    return x.data_ptr() % 16 == 0 and w.data_ptr() % 16 == 0


def gate_up_swiglu(x, w, *, out=None, tile_rows=0):
    """SiLU(x . w[:I]^T) * (x . w[I:]^T) with both projections rounded to bf16 first, as one GEMM
    (``fg_gate_up_swiglu``): x [rows, H] bf16, w [2I, H] bf16 (gate rows, then up rows) ->
    [rows, I] bf16. tile_rows: 0 (the kernel's choice of 192 / 256), 64, 128, 192 or 256."""
    _dev(x, w)
    if not gate_up_swiglu_ok(x, w):
        raise ValueError("gate_up_swiglu: needs bf16 x [rows, H] and w [2I, H] with H % 64 == 0, I % 4 == 0, "
                         "unit column strides and 16-byte aligned rows")
    rows, H = x.shape
    inter = w.shape[0] // 2
    if out is None:
        out = torch.empty(rows, inter, dtype=torch.bfloat16, device=x.device)
    elif out.dtype != torch.bfloat16 or tuple(out.shape) != (rows, inter) or out.stride(1) != 1:
        raise ValueError(f"gate_up_swiglu: out must be bf16 [{rows}, {inter}] with unit column stride")
    _call("fg_gate_up_swiglu", _ptr(x), x.stride(0), _ptr(w), w.stride(0), _ptr(out), out.stride(0), rows, inter, H,
          int(tile_rows), _stream())
    return out


LINEAR_TILES = (64, 128)


def linear_splits(hidden: int, splits: int) -> int:
    """The largest split count <= ``splits`` that gives every split of ``hidden / 64``
    k-steps at least one (the rule fg_linear_parts checks)."""
    nk = hidden // 64
    s = max(1, min(int(splits), nk))
    while s > 1 and -(-nk // -(-nk // s)) != s:
        s -= 1
    return s


def linear_ok(x, w) -> bool:
    """Whether fg_linear_parts takes x [rows, K] and w [N, K] as they are: bf16 on the GPU,
    K a multiple of 64, N a multiple of 4, unit column strides and 16-byte aligned rows."""
    if not (x.is_cuda and x.dtype == torch.bfloat16 and w.dtype == torch.bfloat16 and x.dim() == 2 and w.dim() == 2):
        return False
    K_ = x.shape[1]
    if K_ == 0 or K_ % 64 or w.shape[1] != K_ or w.shape[0] % 4 or x.shape[0] == 0:
        return False
    if x.stride(1) != 1 or w.stride(1) != 1 or x.stride(0) % 8 or w.stride(0) % 8:
        return False
    return x.data_ptr() % 16 == 0 and w.data_ptr() % 16 == 0 and x.stride(0) < (1 << 22) and w.stride(0) < (1 << 22)


def linear_parts(x, w, *, splits=1, tile=(128, 128), stages=0, out=None):
    """Split-K partial products of x [rows, K] . w [N, K]^T (``fg_linear_parts``): fp32
    [splits, rows, N] whose sum over the first dimension (in order) is the projection.
    ``splits`` must satisfy the kernel's rule (see ``linear_splits``); ``stages``: k-steps in
    the kernel's LDS ring (2-4, 0 for 4)."""
    _dev(x, w)
    if not linear_ok(x, w):
        raise ValueError("linear_parts: needs bf16 x [rows, K] and w [N, K] with K % 64 == 0, N % 4 == 0, "
                         "unit column strides and 16-byte aligned rows")
    rows, K_ = x.shape
    N = w.shape[0]
    tm, tn = (int(t) for t in tile)
    if tm not in LINEAR_TILES or tn not in LINEAR_TILES:
        raise ValueError(f"linear_parts: tile sizes must be in {LINEAR_TILES}")
    if int(stages) not in (0, 2, 3, 4):
        raise ValueError("linear_parts: stages must be 0, 2, 3 or 4")
    if linear_splits(K_, splits) != int(splits):
        raise ValueError(f"linear_parts: {splits} splits leave a split of {K_ // 64} k-steps empty")
    shape = (int(splits), rows, N)
    if out is None:
        out = torch.empty(shape, dtype=torch.float32, device=x.device)
    elif out.dtype != torch.float32 or tuple(out.shape) != shape or not out.is_contiguous() or out.data_ptr() % 16:
        raise ValueError(f"linear_parts: out must be a contiguous 16-byte aligned fp32 {list(shape)} tensor")
    _call("fg_linear_parts", _ptr(x), x.stride(0), _ptr(w), w.stride(0), _ptr(out), rows, N, K_, int(splits), tm, tn,
          int(stages), _stream())
    return out


def residual_rmsnorm_parts(parts, x, weight, eps, *, out=None):
    """x <- bf16(x + bf16(parts.sum(0))) in place, then RMSNorm(x) * weight
    (``fg_residual_rmsnorm_parts``): parts fp32 [S, rows, H], x bf16 [rows, H]."""
    _dev(parts, x, weight)
    S, rows, H = parts.shape
    if parts.dtype != torch.float32 or not parts.is_contiguous():
        raise ValueError("residual_rmsnorm_parts: parts must be contiguous fp32 [S, rows, H]")
    if x.dtype != torch.bfloat16 or tuple(x.shape) != (rows, H) or x.stride(1) != 1:
        raise ValueError(f"residual_rmsnorm_parts: x must be bf16 [{rows}, {H}] with unit column stride")
    if weight.dtype != torch.bfloat16 or weight.numel() != H or not weight.is_contiguous():
        raise ValueError("residual_rmsnorm_parts: weight must be a contiguous bf16 [H] tensor")
    if out is None:
        out = torch.empty(rows, H, dtype=torch.bfloat16, device=x.device)
    elif out.dtype != torch.bfloat16 or tuple(out.shape) != (rows, H) or out.stride(1) != 1:
        raise ValueError(f"residual_rmsnorm_parts: out must be bf16 [{rows}, {H}] with unit column stride")
    _call("fg_residual_rmsnorm_parts", _ptr(parts), S, rows, H, _ptr(x), x.stride(0), _ptr(weight), float(eps),
          _ptr(out), out.stride(0), _stream())
    return out


def rope_kv_write_parts(parts, bias, *, batch, num_nodes, q_heads, kv_heads, head_dim, seq_len, pos_offset,
                        inv_freq, q_out, k_cache, v_cache, row_map=None, err_flag=None):
    """``rope_kv_write`` with the qkv rows given as split-K parts fp32 [S, batch*num_nodes,
    (q_heads + 2 kv_heads) * head_dim] plus the projection's bias (or None), each value
    rounded to the cache dtype after the sum (``fg_rope_kv_write_parts``)."""
    _dev(parts, bias, seq_len, pos_offset, inv_freq, q_out, k_cache, v_cache, row_map)
    _i32(seq_len, "seq_len")
    _i32(pos_offset, "pos_offset")
    _i32(row_map, "row_map")
    width = (q_heads + 2 * kv_heads) * head_dim
    if parts.dtype != torch.float32 or not parts.is_contiguous() or tuple(parts.shape[1:]) != (batch * num_nodes,
                                                                                                width):
        raise ValueError(f"rope_kv_write_parts: parts must be contiguous fp32 [S, {batch * num_nodes}, {width}]")
    if bias is not None and (bias.dtype != k_cache.dtype or bias.numel() != width or not bias.is_contiguous()):
        raise ValueError("rope_kv_write_parts: bias must be a contiguous [width] tensor of the cache dtype")
    if k_cache.stride(-1) != 1 or k_cache.stride(-2) != head_dim:
        raise ValueError("rope_kv_write_parts: cache rows must be contiguous [.., capacity, d]")
    if pos_offset.dim() == 2:
        if tuple(pos_offset.shape) != (batch, num_nodes) or not pos_offset.is_contiguous():
            raise ValueError("rope_kv_write_parts: per-sequence pos_offset must be contiguous [batch, num_nodes]")
        pos_stride = num_nodes
    else:
        if pos_offset.numel() < num_nodes:
            raise ValueError("rope_kv_write_parts: pos_offset shorter than num_nodes")
        pos_stride = 0
    _call("fg_rope_kv_write_parts", _ptr(parts), parts.shape[0], _ptr(bias), dtype_code(k_cache), batch, num_nodes,
          q_heads, kv_heads, head_dim, _ptr(seq_len), _ptr(pos_offset), pos_stride, _ptr(inv_freq), _ptr(q_out),
          _ptr(k_cache), _ptr(v_cache), k_cache.stride(0), k_cache.stride(1), k_cache.shape[-2], _ptr(row_map),
          _ptr(err_flag), _stream())


def rope_pair_rows(t, q_heads, kv_heads, head_dim):
    """The rows (dim 0) of a q/k/v projection weight [width, K] or bias [width] in the order
    ``fg_linear_rope_kv_write`` takes: each q and k head's rows pair-interleaved (row 2j holds the
    head's row j, row 2j + 1 its row j + head_dim/2), the v heads' rows in order. A new tensor."""
    d, h = int(head_dim), int(q_heads) + int(kv_heads)
    if d % 2 or t.shape[0] != (h + int(kv_heads)) * d:
        raise ValueError("rope_pair_rows: rows must be (q_heads + 2 kv_heads) * head_dim with an even head_dim")
    qk = t[:h * d].reshape(h, 2, d // 2, *t.shape[1:]).transpose(1, 2).reshape(h * d, *t.shape[1:])
    return torch.cat([qk, t[h * d:]]).contiguous()


def rope_cos_sin(*, batch, num_nodes, head_dim, seq_len, pos_offset, inv_freq, out=None):
    """fp32 [batch*num_nodes, head_dim/2, 2]: (cos, sin) of each row's rotary angles rounded to bf16
    (``fg_rope_cos_sin``), the table ``linear_rope_kv_write`` reads."""
    _dev(seq_len, pos_offset, inv_freq, out)
    _i32(seq_len, "seq_len")
    _i32(pos_offset, "pos_offset")
    pos_stride = _pos_stride(pos_offset, batch, num_nodes, "rope_cos_sin")
    shape = (batch * num_nodes, head_dim // 2, 2)
    if out is None:
        out = torch.empty(shape, dtype=torch.float32, device=seq_len.device)
    elif out.dtype != torch.float32 or tuple(out.shape) != shape or not out.is_contiguous():
        raise ValueError(f"rope_cos_sin: out must be a contiguous fp32 {list(shape)} tensor")
    _call("fg_rope_cos_sin", _ptr(seq_len), _ptr(pos_offset), pos_stride, _ptr(inv_freq), batch, num_nodes, head_dim,
          _ptr(out), _stream())
    return out


def _pos_stride(pos_offset, batch, num_nodes, what):
    if pos_offset.dim() == 2:
        if tuple(pos_offset.shape) != (batch, num_nodes) or not pos_offset.is_contiguous():
            raise ValueError(f"{what}: per-sequence pos_offset must be contiguous [batch, num_nodes]")
        return num_nodes
    if pos_offset.numel() < num_nodes:
        raise ValueError(f"{what}: pos_offset shorter than num_nodes")
    return 0


def linear_rope_kv_write(x, w_pairs, bias_pairs, *, tile=(64, 64), stages=0, batch, num_nodes, q_heads, kv_heads,
                         head_dim, seq_len, q_out, k_cache, v_cache, cos_sin=None, pos_offset=None, inv_freq=None,
                         row_map=None, err_flag=None):
    """The q/k/v projection x [batch*num_nodes, K] . w^T with the bias, rotary embedding and KV-slot
    write in the GEMM epilogue (``fg_linear_rope_kv_write``): the weight and bias given in
    ``rope_pair_rows`` order, the rows' rotary table ``cos_sin`` (``rope_cos_sin``; made here from
    pos_offset and inv_freq when not given); q rows to q_out [batch*num_nodes, q_heads, d], k / v
    rows to their cache slots, bit for bit as ``linear_parts`` (one split) + ``rope_kv_write_parts``."""
    _dev(x, w_pairs, bias_pairs, seq_len, cos_sin, q_out, k_cache, v_cache, row_map)
    _i32(seq_len, "seq_len")
    _i32(row_map, "row_map")
    width = (q_heads + 2 * kv_heads) * head_dim
    if not linear_ok(x, w_pairs) or w_pairs.shape[0] != width or x.shape[0] != batch * num_nodes:
        raise ValueError(f"linear_rope_kv_write: needs bf16 x [{batch * num_nodes}, K] and w [{width}, K] with "
                         "K % 64 == 0, unit column strides and 16-byte aligned rows")
    if bias_pairs is not None and (bias_pairs.dtype != torch.bfloat16 or bias_pairs.numel() != width or
                                   not bias_pairs.is_contiguous()):
        raise ValueError("linear_rope_kv_write: bias must be a contiguous bf16 [width] tensor")
    tm, tn = (int(t) for t in tile)
    if tm not in LINEAR_TILES or tn not in LINEAR_TILES or int(stages) not in (0, 2, 3, 4):
        raise ValueError(f"linear_rope_kv_write: tiles in {LINEAR_TILES}, stages 0, 2, 3 or 4")
    if k_cache.dtype != torch.bfloat16 or k_cache.stride(-1) != 1 or k_cache.stride(-2) != head_dim:
        raise ValueError("linear_rope_kv_write: cache rows must be contiguous bf16 [.., capacity, d]")
    if v_cache.stride() != k_cache.stride() or v_cache.shape != k_cache.shape or v_cache.dtype != k_cache.dtype:
        raise ValueError("linear_rope_kv_write: v_cache must have k_cache's shape, strides and dtype")
    if not q_out.is_contiguous() or q_out.numel() != batch * num_nodes * q_heads * head_dim or \
            q_out.dtype != torch.bfloat16:
        raise ValueError("linear_rope_kv_write: q_out must be a contiguous bf16 [batch * num_nodes, q_heads, d] tensor")
    if cos_sin is None:
        cos_sin = rope_cos_sin(batch=batch, num_nodes=num_nodes, head_dim=head_dim, seq_len=seq_len,
                               pos_offset=pos_offset, inv_freq=inv_freq)
    elif cos_sin.dtype != torch.float32 or cos_sin.numel() != batch * num_nodes * head_dim or \
            not cos_sin.is_contiguous():
        raise ValueError("linear_rope_kv_write: cos_sin must be rope_cos_sin's table of these rows")
    _call("fg_linear_rope_kv_write", _ptr(x), x.stride(0), _ptr(w_pairs), w_pairs.stride(0), _ptr(bias_pairs),
          x.shape[0], x.shape[1], tm, tn, int(stages), batch, num_nodes, q_heads, kv_heads, head_dim, _ptr(seq_len),
          _ptr(cos_sin), _ptr(q_out), _ptr(k_cache), _ptr(v_cache), k_cache.stride(0), k_cache.stride(1),
          k_cache.shape[-2], _ptr(row_map), _ptr(err_flag), _stream())


# ------------------------------------------------------------------ microscaled (MX) rows
MX_BLOCK = 32                         # elements per scale
MX_FORMATS = {"e4m3": 0, "e2m1": 1}   # fg_mx_quantize's format codes
_U8, _FP8, _BF16, _I32 = torch.uint8, torch.float8_e4m3fn, torch.bfloat16, torch.int32


class MX(NamedTuple):
    """Microscaled rows [rows, cols] (``mx_quantize``). ``codes``: float8_e4m3fn [rows, cols], or uint8
    [rows, cols / 2] holding two e2m1 codes to a byte (the earlier element in the low half). ``scales``: uint8
    [ceil(cols / 128), rows, 4], byte s of the block of 32 elements standing for the factor 2^(s - 127) (255: the
    block is NaN; bytes behind the last block 0)."""
    codes: torch.Tensor
    scales: torch.Tensor

    @property
    def format(self) -> str:
        return "e2m1" if self.codes.dtype == torch.uint8 else "e4m3"

    @property
    def shape(self) -> tuple:
        return self.codes.shape[0], self.codes.shape[1] * (2 if self.codes.dtype == torch.uint8 else 1)


# The calls below serve single tokens, where a launch costs 3.5 us of host time and every check counts: devices are
# compared as indices and shapes in one expression each, and what is wrong is worked out after a check has failed.
def _same_device(what, dev, *ts) -> None:
    """Raises unless every given tensor (None aside) is on GPU ``dev`` (a device index, -1 for the CPU)."""
    if dev < 0:
        raise ValueError("flashgrpo_amd kernels take device tensors (got a CPU tensor)")
    for t in ts:
        if t is not None and t.get_device() != dev:
            raise ValueError(f"{what}: tensors on different devices")


def _call_on(dev, name, *args):
    """The call on GPU ``dev``'s current stream, whichever device is the current one."""
    if dev == _cur_device():
        if timing.idle():
            if getattr(_lib.load(), name)(*args, _raw_stream(dev)):
                _lib.raise_last_error()
        else:
            _call(name, *args, _raw_stream(dev))
    else:
        with torch.cuda.device(dev):
            _call(name, *args, _raw_stream(dev))


def _apart(what, outs, ins) -> None:
    """Raises where the memory of an output that the caller gave meets an operand's, each as (address, bytes)."""
    for a, n in outs:
        for b, m in ins:
            if b < a + n and a < b + m:
                raise ValueError(f"{what}: an output overlaps an operand")


def _mx_spans(c, s, fmt, rows, cols):
    """(address, bytes) of an MX pair's codes and scales."""
    return (c, rows * cols >> fmt), (s, (cols + 127 >> 7) * rows * 4)


def _too_large(what):
    raise ValueError(f"{what}: rows and columns must be less than 2^31")


def _mx_bad(codes, scales, what):
    if codes.dtype not in (_U8, _FP8) or scales.dtype != _U8 or codes.dim() != 2:
        raise TypeError(f"{what}: MX codes must be float8_e4m3fn or uint8 [rows, ..] with uint8 scales")
    rows, k = MX(codes, scales).shape
    if k == 0 or k % MX_BLOCK:
        raise ValueError(f"{what}: MX rows of {k} elements; expected a multiple of 32")
    if (rows | k) >> 31:
        _too_large(what)
    if tuple(scales.shape) != (-(-k // 128), rows, 4):
        raise ValueError(f"{what}: MX scales must be [{-(-k // 128)}, {rows}, 4], got {list(scales.shape)}")
    raise ValueError(f"{what}: MX codes and scales must be contiguous, 16- and 4-byte aligned, on one device")


def _mx_of(q, what):
    """(codes' address, scales' address, format code, rows, cols, device index) of an MX pair that the kernels take."""
    codes, scales = q
    dt, shape = codes.dtype, codes.shape
    if (dt is not _U8 and dt is not _FP8) or len(shape) != 2:
        _mx_bad(codes, scales, what)
    rows, k = shape
    fmt = 0
    if dt is _U8:
        fmt, k = 1, 2 * k
    dev = codes.get_device()
    c, s = codes.data_ptr(), scales.data_ptr()
    if (k % 32 or k == 0 or (rows | k) >> 31 or c % 16 or s % 4 or scales.dtype is not _U8
            or scales.shape != ((k + 127) // 128, rows, 4) or not codes.is_contiguous() or not scales.is_contiguous()
            or scales.get_device() != dev):
        _mx_bad(codes, scales, what)
    return c, s, fmt, rows, k, dev


def _mx_out(out, rows, cols, fmt, device, what, operands=()) -> MX:
    """out, checked against what it has to be and (address, bytes) of the operands, or a new pair."""
    if (rows | cols) >> 31:
        _too_large(what)
    if out is None:
        return MX(torch.empty(rows, cols // 2 if fmt else cols, dtype=_U8 if fmt else _FP8, device=device),
                  torch.empty((cols + 127) // 128, rows, 4, dtype=_U8, device=device))
    held = _mx_of(out, what)
    if held[2:] != (fmt, rows, cols, device.index):
        raise ValueError(f"{what}: out must be an {'e2m1' if fmt else 'e4m3'} MX pair of [{rows}, {cols}] on {device}")
    _apart(what, _mx_spans(*held[:5]), operands)
    return MX(*out)


def mx_quantize(x, fmt="e2m1", *, out=None) -> MX:
    """The MX form of x [rows, cols] (``fg_mx_quantize``), cols a multiple of 32: fmt "e4m3" (8 bits) or "e2m1"
    (4 bits). Each block of 32 elements gets the smallest power-of-two scale >= 2^-126 that holds it without
    saturation; a block that holds an infinity or a NaN becomes NaN. x bf16 or fp32 with unit column stride and
    16-byte aligned rows. ``out``: an MX pair to overwrite (a weight that is quantised again), apart from x."""
    dev = x.get_device()
    _same_device("mx_quantize", dev)
    f = MX_FORMATS.get(fmt)
    if f is None:
        raise ValueError(f"mx_quantize: fmt must be one of {tuple(MX_FORMATS)}")
    dt = dtype_code(x)
    shape = x.shape
    if len(shape) != 2 or shape[1] == 0 or shape[1] % MX_BLOCK:
        raise ValueError("mx_quantize: x must be [rows, cols] with cols a multiple of 32")
    rows, cols = shape
    ldx = cols
    if not x.is_contiguous():
        ldx = x.stride(0) if rows > 1 else cols
        if x.stride(1) != 1 or ldx < cols:
            raise ValueError("mx_quantize: x rows must have unit column stride")
    q = _mx_out(out, rows, cols, f, x.device, "mx_quantize", () if out is None else
                ((x.data_ptr(), ((rows - 1) * ldx + cols) * x.element_size()),))
    if rows == 0:
        return q
    if ldx % 8 or x.data_ptr() % 16:
        raise ValueError("mx_quantize: x rows must start 16-byte aligned")
    _call_on(dev, "fg_mx_quantize", x.data_ptr(), dt, ldx, rows, cols, f, q[0].data_ptr(), q[1].data_ptr())
    return q


def mx_dequantize(q, dtype=torch.bfloat16, *, out=None):
    """The values that an MX pair stands for, [rows, cols] in bf16 (exact but under 2^-126) or fp32
    (``fg_mx_dequantize``)."""
    codes, scales, f, rows, cols, dev = _mx_of(q, "mx_dequantize")
    _same_device("mx_dequantize", dev, out)
    if out is None:
        if dtype not in _DT:
            raise TypeError("mx_dequantize: dtype must be bfloat16 or float32")
        out = torch.empty(rows, cols, dtype=dtype, device=q[0].device)
    elif tuple(out.shape) != (rows, cols) or out.dtype not in _DT or not out.is_contiguous() or out.data_ptr() % 16:
        raise ValueError(f"mx_dequantize: out must be a contiguous 16-byte aligned bf16 or fp32 [{rows}, {cols}] tensor")
    else:
        _apart("mx_dequantize", ((out.data_ptr(), rows * cols * out.element_size()),),
               _mx_spans(codes, scales, f, rows, cols))
    if rows:
        _call_on(dev, "fg_mx_dequantize", codes, scales, f, rows, cols, out.data_ptr(), dtype_code(out), cols)
    return out


def rmsnorm_mx(x, weight, eps, *, delta=None, sum_out=None, out=None) -> MX:
    """``rmsnorm`` with an 8-bit output (``fg_rmsnorm_mx``): MX e4m3 of RMSNorm(x [+ delta]) * weight over the last
    dimension of x [rows, H], H a multiple of 32 up to 8192. With delta the sum, rounded to x's dtype, is written to
    ``sum_out`` (x itself when not given; x, delta, or apart from both). x, delta, weight and sum_out contiguous, one
    dtype (bf16 or fp32). The norm is not rounded between its steps: the codes are those of the formula in 64 bits."""
    dev = x.get_device()
    _same_device("rmsnorm_mx", dev, weight, delta, sum_out)
    dt = dtype_code(x)
    shape, dtype = x.shape, x.dtype
    if len(shape) != 2:
        raise ValueError("rmsnorm_mx: x must be [rows, H]")
    rows, H = shape
    if H == 0 or H % MX_BLOCK or H > 8192:
        raise ValueError("rmsnorm_mx: H must be a multiple of 32, at most 8192")
    if weight.numel() != H or weight.dtype is not dtype or not weight.is_contiguous() or weight.data_ptr() % 16:
        raise ValueError("rmsnorm_mx: weight must be a contiguous 16-byte aligned [H] tensor of x's dtype")
    if delta is None:
        if sum_out is not None:
            raise ValueError("rmsnorm_mx: sum_out without delta")
        rest = (x,)
    elif sum_out is None:
        sum_out = x
        rest = (x, delta)
    else:
        rest = (x, delta, sum_out)
    at = []
    for t in rest:
        p = t.data_ptr()
        if not t.is_contiguous() or p % 16 or (t is not x and (t.shape != shape or t.dtype is not dtype)):
            raise ValueError("rmsnorm_mx: x, delta and sum_out must be contiguous, 16-byte aligned and of one shape and "
                             "dtype")
        at.append(p)
    row = H * (2 if dt else 4)
    size, w, total = rows * row, weight.data_ptr(), None
    if delta is not None:
        total = at[0] if sum_out is x else at[2]
        for p in at:
            if -size < p - total < size and p != total:
                raise ValueError("rmsnorm_mx: sum_out overlaps x or delta without being it")
        if w < total + size and total < w + row:
            raise ValueError("rmsnorm_mx: sum_out overlaps the weight")
    q = _mx_out(out, rows, H, 0, x.device, "rmsnorm_mx", () if out is None else ((w, row), *((p, size) for p in at)))
    if rows:
        _call_on(dev, "fg_rmsnorm_mx", at[0], None if delta is None else at[1], w, total, dt, rows, H, float(eps),
                 q[0].data_ptr(), q[1].data_ptr())
    return q


def residual_rmsnorm_mx_parts(parts, x, weight, eps, *, out=None) -> MX:
    """``residual_rmsnorm_parts`` with an 8-bit output (``fg_residual_rmsnorm_mx_parts``): x <- bf16(x +
    bf16(parts.sum(0))) in place, then MX e4m3 of RMSNorm(x) * weight as ``rmsnorm_mx`` makes it. parts fp32
    [S, rows, H], H a multiple of 32 up to 8192, x bf16 [rows, H] with unit column stride and 16-byte aligned rows."""
    dev = x.get_device()
    _same_device("residual_rmsnorm_mx_parts", dev, parts, weight)
    if parts.dim() != 3 or parts.dtype != torch.float32 or not parts.is_contiguous() or parts.shape[0] == 0:
        raise ValueError("residual_rmsnorm_mx_parts: parts must be contiguous fp32 [S, rows, H]")
    S, rows, H = parts.shape
    if H == 0 or H % MX_BLOCK or H > 8192:
        raise ValueError("residual_rmsnorm_mx_parts: H must be a multiple of 32, at most 8192")
    if x.dtype is not _BF16 or x.shape != (rows, H) or x.stride(1) != 1:
        raise ValueError(f"residual_rmsnorm_mx_parts: x must be bf16 [{rows}, {H}] with unit column stride")
    ldx = x.stride(0) if rows > 1 else H
    if ldx < H or ldx % 8 or x.data_ptr() % 16 or parts.data_ptr() % 16:
        raise ValueError("residual_rmsnorm_mx_parts: rows must be apart and start 16-byte aligned")
    if weight.dtype is not _BF16 or weight.numel() != H or not weight.is_contiguous() or weight.data_ptr() % 16:
        raise ValueError("residual_rmsnorm_mx_parts: weight must be a contiguous 16-byte aligned bf16 [H] tensor")
    into = (x.data_ptr(), ((rows - 1) * ldx + H) * 2)
    read = (parts.data_ptr(), S * rows * H * 4), (weight.data_ptr(), H * 2)
    _apart("residual_rmsnorm_mx_parts", (into,), read)
    q = _mx_out(out, rows, H, 0, x.device, "residual_rmsnorm_mx_parts", (into, *read))
    if rows:
        _call_on(dev, "fg_residual_rmsnorm_mx_parts", parts.data_ptr(), S, rows, H, x.data_ptr(), ldx, weight.data_ptr(),
                 float(eps), q[0].data_ptr(), q[1].data_ptr())
    return q


def _mx_operands(x, w, what):
    """Both operands of a product as addresses and sizes: x's and w's pointers and x's format in the entry points'
    order, then rows, weight rows, K and the device index."""
    xc, xs, f, rows, k, dev = _mx_of(x, what)
    wc, ws, wf, n, kw, wdev = _mx_of(w, what)
    if dev != wdev or dev < 0:
        _same_device(what, dev, w[0])
    if kw != k:
        raise ValueError(f"{what}: x has {k} columns and the weight {kw}")
    if wf != 1:
        raise TypeError(f"{what}: the weight must be in e2m1 (4 bits)")
    return (xc, xs, f, wc, ws), rows, n, k, dev


@functools.lru_cache(maxsize=4096)
def _mx_workspace_bytes(name, rows, cols, k, fmt):
    return getattr(_lib.load(), name)(rows, cols, k, fmt)


def _mx_workspace(name, rows, cols, k, fmt, device):
    """(tensor, address, bytes) for a split product's sums: a buffer of the call's own, so that calls on two streams, or
    two captured graphs, share none (torch's allocator keeps it until the stream, or the graph, is done with it)."""
    n = _mx_workspace_bytes(name, rows, cols, k, fmt)
    if n == 0:
        return None, None, 0
    ws = torch.empty(n, dtype=_U8, device=device)
    return ws, ws.data_ptr(), n


def mx_linear(x, w, *, bias=None, residual=None, out=None):
    """bf16 [rows, N] = x . w^T (+ bias) (+ residual) of MX rows x [rows, K] (e4m3 or e2m1) and a 4-bit MX weight w
    [N, K] (``fg_mx_linear``), summed in fp32 and rounded once (of e4m3 rows' products, the bits below 2^-13 of the
    largest of eight neighbours are lost: 1e-5 of the sum of magnitudes). bias bf16 [N]; residual bf16 [rows, N] with unit
    column stride; ``out`` bf16 with unit column stride, which may be the residual (an update in place) and must not overlap
    an operand otherwise."""
    operands, rows, N, k, dev = _mx_operands(x, w, "mx_linear")
    _same_device("mx_linear", dev, bias, residual, out)
    if bias is not None and (bias.dtype is not _BF16 or bias.numel() != N or not bias.is_contiguous()):
        raise ValueError(f"mx_linear: bias must be a contiguous bf16 [{N}] tensor")
    device = w[0].device
    given = out is not None
    if not given:
        out = torch.empty(rows, N, dtype=_BF16, device=device)
        ldo = N
    else:
        ldo = _mx_rows(out, rows, N, "out")
    ldr = N if residual is None else _mx_rows(residual, rows, N, "residual")
    if rows == 0 or N == 0:
        return out
    if given:
        xc, xs, f, wc, ws = operands
        _apart("mx_linear", ((out.data_ptr(), 2 * ((rows - 1) * ldo + N)),),
               (*_mx_spans(xc, xs, f, rows, k), *_mx_spans(wc, ws, 1, N, k),
                (0, 0) if bias is None else (bias.data_ptr(), 2 * N)))
        if residual is not None and _rows_meet(out.data_ptr() // 2, ldo, residual.data_ptr() // 2, ldr, rows, N):
            raise ValueError("mx_linear: out overlaps the residual without being it")
    ws, ws_ptr, ws_bytes = _mx_workspace("fg_mx_linear_workspace", rows, N, k, operands[2], device)
    _call_on(dev, "fg_mx_linear", *operands, rows, N, k, _ptr(bias), _ptr(residual), ldr, out.data_ptr(), ldo, ws_ptr,
             ws_bytes)
    return out


def _mx_rows(t, rows, n, what):
    """The row stride of a bf16 [rows, n] tensor with unit column stride."""
    if t.dtype is not _BF16 or t.shape != (rows, n):
        raise ValueError(f"mx_linear: {what} must be bf16 [{rows}, {n}]")
    if t.is_contiguous() or rows == 1 and (n == 1 or t.stride(1) == 1):
        return n
    if (n > 1 and t.stride(1) != 1) or t.stride(0) < n:
        raise ValueError(f"mx_linear: {what} must have unit column stride and rows apart")
    return t.stride(0)


def _rows_meet(a, lda, b, ldb, rows, n) -> bool:
    """Whether rows x n elements at a (row stride lda >= n) and at b (ldb) share any without being the same."""
    if a == b and lda == ldb or a + (rows - 1) * lda + n <= b or b + (rows - 1) * ldb + n <= a:
        return False
    d = (b - a) % lda
    return lda != ldb or not n <= d <= lda - n  # of one buffer's columns beside each other, none


def mx_gate_up_swiglu(x, w, *, out=None) -> MX:
    """MX e4m3 [rows, I] of SiLU(x . w[:I]^T) * (x . w[I:]^T) (``fg_mx_gate_up_swiglu``): MX rows x [rows, K] (e4m3
    or e2m1), a 4-bit MX weight w [2I, K] (gate rows, then up rows), I a multiple of 32. Sums (of whole products, where
    ``mx_linear`` cuts those of e4m3 rows) and the activation in fp32, rounded once, to the 8-bit codes."""
    operands, rows, n2, k, dev = _mx_operands(x, w, "mx_gate_up_swiglu")
    if n2 == 0 or n2 % (2 * MX_BLOCK):
        raise ValueError("mx_gate_up_swiglu: the weight must have 2 I rows, I a multiple of 32")
    device = w[0].device
    inter = n2 // 2
    xc, xs, f, wc, ws = operands
    q = _mx_out(out, rows, inter, 0, device, "mx_gate_up_swiglu", () if out is None else
                (*_mx_spans(xc, xs, f, rows, k), *_mx_spans(wc, ws, 1, n2, k)))
    if rows:
        ws, ws_ptr, ws_bytes = _mx_workspace("fg_mx_gate_up_swiglu_workspace", rows, inter, k, operands[2], device)
        _call_on(dev, "fg_mx_gate_up_swiglu", *operands, rows, inter, k, q[0].data_ptr(), q[1].data_ptr(), ws_ptr,
                 ws_bytes)
    return q


class MXPlan(NamedTuple):
    """The kernel of an MX product (``mx_plan``): rows and weight rows of a workgroup; steps in its LDS ring and splits of
    the reduction, or, with 0 stages, the stream of the weights and its waves per workgroup."""
    rows: int
    cols: int
    stages: int
    splits_or_waves: int


def mx_plan(rows, cols, k, *, fmt="e4m3", gate_up=False) -> MXPlan:
    """Which kernel ``mx_linear`` (or ``mx_gate_up_swiglu``, cols its I) runs for x [rows, k] of a format
    (``fg_mx_plan``); for profiles and tests. Needs no GPU."""
    if fmt not in MX_FORMATS:
        raise ValueError(f"mx_plan: fmt must be one of {tuple(MX_FORMATS)}")
    if max(rows, cols, k) >> 31:
        _too_large("mx_plan")
    p = (C.c_int * 4)()
    _lib.call("fg_mx_plan", int(gate_up), rows, cols, k, MX_FORMATS[fmt], p)
    return MXPlan(*p)


# ------------------------------------------------------------------ a KV cache in pages
PAGE_FORMATS = {torch.float8_e4m3fn: 0, torch.bfloat16: 1}  # struct fg_kv_pages' format


class _Pages:
    """``KVPages`` until they are filled."""

    __slots__ = ("k", "v", "k_scales", "v_scales", "table", "format", "pages", "page_size", "kv_heads", "head_dim", "rows",
                 "width", "device", "address", "_spans", "_table", "_c")

    def _fill(self, k, v, k_scales, v_scales, table):
        fmt = PAGE_FORMATS.get(k.dtype)
        shape, stride, dev = k.shape, k.stride(), k.get_device()  # (-1: on the host, which no call takes)
        if fmt is None or v.dtype is not k.dtype or table.dtype is not _I32 or len(shape) != 4 or table.dim() != 2:
            self._refuse(k, v, k_scales, v_scales, table)
        n, heads, size, d = shape
        (rows, width), (row, unit) = table.shape, table.stride()
        at, at_v, page = k.data_ptr(), v.data_ptr(), heads * size * d
        first = stride[0] if n > 1 else page
        ok = (v.shape == shape and (d == 64 or d == 128) and size >= 16 and not size & (size - 1) and n and heads and rows and width
              and stride[3] == 1 and stride[2] == d and (heads == 1 or stride[1] == size * d) and first >= page
              and v.stride() == stride and (width == 1 or unit == 1) and (rows == 1 or row >= width)
              and width * size < (1 << 31) - 65536 and page < 1 << 30 and not (n | rows) >> 31
              and first < 1 << 31 and not (at | at_v | first * (1 + fmt)) & 15 and v.get_device() == dev == table.get_device())
        at_ks = at_vs = scale_first = None
        if ok and fmt == 0:
            ok = k_scales is not None and v_scales is not None
            if ok:
                blocks = d >> 5
                page >>= 5
                s = k_scales.stride()
                scale_first = s[0] if n > 1 else page
                at_ks, at_vs = k_scales.data_ptr(), v_scales.data_ptr()
                ok = (k_scales.shape == (n, heads, size, blocks) == v_scales.shape and k_scales.dtype is _U8 is v_scales.dtype
                      and s[3] == 1 and s[2] == blocks and (heads == 1 or s[1] == size * blocks) and scale_first >= page
                      and v_scales.stride() == s and scale_first < 1 << 32 and not (at_ks | at_vs | scale_first) & 3
                      and k_scales.get_device() == dev == v_scales.get_device())
        elif ok:
            ok = k_scales is None is v_scales
        if not ok:
            self._refuse(k, v, k_scales, v_scales, table)
        self.k, self.v, self.k_scales, self.v_scales, self.table = k, v, k_scales, v_scales, table
        self.format, self.pages, self.page_size, self.kv_heads, self.head_dim = fmt, n, size, heads, d
        self.rows, self.width, self.device = rows, width, dev
        held = ((n - 1) * first + heads * size * d) * (1 + fmt)
        self._spans = (at, held), (at_v, held)  # (address, bytes) from the first page to the end of the last
        if fmt == 0:
            held = (n - 1) * scale_first + page
            self._spans += (at_ks, held), (at_vs, held)
        at_table = table.data_ptr()
        self._table = at_table, 4 * ((rows - 1) * row + width)
        self._c = _lib.KvPages(at, at_v, at_ks, at_vs, at_table, first, scale_first or 0, row if rows > 1 else width, fmt, n, size,
                               heads, d, rows, width)
        self.address = C.addressof(self._c)

    @staticmethod
    def _refuse(k, v, k_scales, v_scales, table):
        fmt = PAGE_FORMATS.get(k.dtype)
        if fmt is None or v.dtype is not k.dtype:
            raise TypeError("KVPages: k and v must be bfloat16 or float8_e4m3fn")
        if table.dtype is not _I32 or table.dim() != 2 or 0 in table.shape:
            raise ValueError("KVPages: table must be a non-empty int32 [rows, width] tensor")
        dev = k.get_device()
        if any(t is not None and t.get_device() != dev for t in (v, table, k_scales, v_scales)):
            raise ValueError("KVPages: tensors on different devices")
        stride, scale_stride = _page_stride(k, "k"), 0
        n, heads, size, d = k.shape
        if v.shape != k.shape or _page_stride(v, "v") != stride:
            raise ValueError("KVPages: k and v must have one shape and one page stride")
        if d not in (64, 128) or size < 16 or size & (size - 1):
            raise ValueError("KVPages: head_dim must be 64 or 128 and page_size a power of two from 16 on")
        if (fmt == 0) != (k_scales is not None) or (k_scales is None) != (v_scales is None):
            raise ValueError("KVPages: float8_e4m3fn pages need scales, bfloat16 pages have none")
        if fmt == 0:
            shape = (n, heads, size, d // MX_BLOCK)
            if k_scales.shape != shape or v_scales.shape != shape or k_scales.dtype is not _U8 or v_scales.dtype is not _U8:
                raise ValueError(f"KVPages: scales must be uint8 {list(shape)}")
            scale_stride = _page_stride(k_scales, "k_scales")
            if _page_stride(v_scales, "v_scales") != scale_stride:
                raise ValueError("KVPages: k_scales and v_scales must have one page stride")
        rows, width = table.shape
        if (width > 1 and table.stride(1) != 1) or (rows > 1 and table.stride(0) < width):
            raise ValueError("KVPages: table rows must have unit stride and be apart")
        if width * size >= (1 << 31) - 65536 or heads * size * d >= 1 << 30 or (n | rows) >> 31 or stride >> 31 or scale_stride >> 32:
            raise ValueError("KVPages: rows must hold less than 2^31 - 65536 tokens, pages less than 2^30 elements and lie less than "
                             "2^31 elements apart")
        raise ValueError("KVPages: pages must start 16-byte aligned and scales 4-byte aligned")

    @property
    def capacity(self) -> int:
        """Tokens that a cache row's table has entries for."""
        return self.width * self.page_size


class KVPages(_Pages):
    """One layer's K and V in pages (struct ``fg_kv_pages``), checked once: token t of cache row r lies in page
    ``table[r, t // page_size]``, slot ``t % page_size`` (a page number outside [0, pages): no page).

    ``k``, ``v``: bf16 or float8_e4m3fn [pages, kv_heads, page_size, head_dim] views of the same strides, each page
    contiguous and 16-byte aligned (a pool may hold a page's layers side by side), head_dim 64 or 128, page_size a power of
    two from 16 on. float8_e4m3fn pages hold MX rows: ``k_scales``, ``v_scales`` uint8 [pages, kv_heads, page_size, head_dim /
    32], as ``mx_quantize`` makes them but a row's scales side by side (codes 0x7f and 0xff must not occur; a scale of 255
    makes its block NaN). ``table``: int32 [rows, width]. The tensors are kept and their contents may change; the attributes may
    not."""

    __slots__ = ()

    def __new__(cls, k, v, k_scales, v_scales, table):
        self = object.__new__(_Pages)
        self._fill(k, v, k_scales, v_scales, table)
        self.__class__ = cls  # (from here on its attributes are fixed)
        return self

    def __setattr__(self, name, value):
        raise AttributeError(f"KVPages are checked once, {name} is fixed: make new ones")

    def __delattr__(self, name):
        self.__setattr__(name, None)

    def __copy__(self):
        return self


def _page_stride(t, what):
    """Elements between pages of a [pages, heads, size, n] view whose pages are contiguous."""
    if t.dim() != 4 or 0 in t.shape:
        raise ValueError(f"KVPages: {what} must be a non-empty [pages, kv_heads, page_size, n] tensor")
    n, heads, size, d = t.shape
    a, b, c, e = t.stride()
    if e != 1 or c != d or (heads > 1 and b != size * d) or (n > 1 and a < heads * size * d):
        raise ValueError(f"KVPages: {what} must have contiguous pages that are apart")
    return a if n > 1 else heads * size * d


def _held(t, dev, rows) -> bool:
    """Whether t is a contiguous int32 tensor of at least ``rows`` entries on GPU ``dev``."""
    return t.dtype is _I32 and t.numel() >= rows and t.is_contiguous() and t.get_device() == dev


def _index(what, dev, rows, *named):
    for name, t in named:
        if t is not None and not _held(t, dev, rows):
            raise ValueError(f"{what}: {name} must be a contiguous int32 tensor of {rows} entries on the pages' device")


def _paged_sizes(what, pages, kv_heads, head_dim):
    if type(pages) is not KVPages:
        raise TypeError(f"{what}: pages must be KVPages")
    if pages.device < 0:
        raise ValueError("flashgrpo_amd kernels take device tensors (got a CPU tensor)")
    if kv_heads != pages.kv_heads or head_dim != pages.head_dim:
        raise ValueError(f"{what}: the pages hold {pages.kv_heads} kv heads of {pages.head_dim}")


def _write_paged(name, lead, pages, batch, num_nodes, q_heads, head_dim, seq_len, pos_offset, inv_freq, q_out, new_len, row_map, err_flag,
                 read):
    dev, size, at = pages.device, batch * num_nodes * q_heads * head_dim, q_out.data_ptr()
    pos_stride = num_nodes if pos_offset.dim() == 2 else 0
    if not (_held(seq_len, dev, batch) and _held(pos_offset, dev, num_nodes)
            and (pos_stride == 0 or pos_offset.shape == (batch, num_nodes)) and inv_freq.dtype is torch.float32
            and inv_freq.numel() >= head_dim >> 1 and inv_freq.is_contiguous() and inv_freq.get_device() == dev
            and q_out.dtype is _BF16 and q_out.numel() == size and q_out.is_contiguous() and q_out.get_device() == dev and not at & 7
            and (new_len is None or _held(new_len, dev, batch)) and (row_map is None or _held(row_map, dev, batch))
            and (err_flag is None or _held(err_flag, dev, 1))):
        what = name[3:]
        _index(what, dev, batch, ("seq_len", seq_len), ("new_len", new_len), ("row_map", row_map))
        _index(what, dev, num_nodes, ("pos_offset", pos_offset))
        _index(what, dev, 1, ("err_flag", err_flag))
        _pos_stride(pos_offset, batch, num_nodes, what)
        if inv_freq.dtype is not torch.float32 or inv_freq.numel() < head_dim >> 1 or not inv_freq.is_contiguous() or inv_freq.get_device() != dev:
            raise ValueError(f"{what}: inv_freq must be a contiguous fp32 tensor of {head_dim // 2} entries on the pages' device")
        raise ValueError(f"{what}: q_out must be a contiguous 8-byte aligned bf16 [batch * num_nodes, q_heads, d] tensor on the pages' device")
    if size:
        lens, pos, freq, few = seq_len.data_ptr(), pos_offset.data_ptr(), inv_freq.data_ptr(), 4 * batch
        new, rows = None if new_len is None else new_len.data_ptr(), None if row_map is None else row_map.data_ptr()
        what, out = name[3:], (at, 2 * size)
        _apart(what, (out, *pages._spans), read)
        _apart(what, (out,), (*pages._spans, pages._table, (lens, few), (pos, 4 * (batch * pos_stride or num_nodes)), (freq, 2 * head_dim),
                              (new or 0, few), (rows or 0, few)))
        _call_on(dev, name, *lead, batch, num_nodes, q_heads, pages.address, lens, pos, pos_stride, freq, new, rows, at,
                 None if err_flag is None else err_flag.data_ptr())


def rope_kv_write_paged(qkv, pages, *, batch, num_nodes, q_heads, kv_heads, head_dim, seq_len, pos_offset, inv_freq, q_out,
                        new_len=None, row_map=None, err_flag=None):
    """``rope_kv_write`` into pages (``fg_rope_kv_write_paged``): bf16 qkv rows; K and V go to slots seq_len[b] + n of cache
    row row_map[b], in the pages' format. e4m3 pages: q is rotated in fp32 and rounded once, K in 64 bits (angles too) and rounded
    to fp32, from which it is quantised; bf16 pages and their q: ``rope_kv_write``'s values. ``new_len`` int32 [batch]:
    tokens from new_len[b] on are left out (their q_out rows and slots stay as they were). A slot without a page sets
    err_flag bit 8. Cache rows that share a page must not both write to it."""
    _paged_sizes("rope_kv_write_paged", pages, kv_heads, head_dim)
    width, rows, shape, at = (q_heads + 2 * kv_heads) * head_dim, batch * num_nodes, qkv.shape, qkv.data_ptr()
    last, ld = shape[-1], qkv.stride(0) if len(shape) == 2 and rows > 1 else shape[-1]
    if qkv.dtype is not _BF16 or len(shape) < 2 or last < width or qkv.numel() != rows * last or qkv.get_device() != pages.device \
            or not (qkv.is_contiguous() or len(shape) == 2 and qkv.stride(1) == 1) or at & 7 or ld & 3 or ld < width:
        raise ValueError(f"rope_kv_write_paged: qkv must hold {rows} rows of >= {width} unit-stride bf16 values on the pages' device, apart "
                         "and 8-byte aligned")
    _write_paged("fg_rope_kv_write_paged", (at, ld), pages, batch, num_nodes, q_heads, head_dim, seq_len, pos_offset, inv_freq, q_out,
                 new_len, row_map, err_flag, ((at, 2 * ((rows - 1) * ld + width)),))


def rope_kv_write_paged_parts(parts, bias, pages, *, batch, num_nodes, q_heads, kv_heads, head_dim, seq_len, pos_offset, inv_freq,
                              q_out, new_len=None, row_map=None, err_flag=None):
    """``rope_kv_write_parts`` into pages (``fg_rope_kv_write_paged_parts``): the qkv rows are bf16(parts.sum(0) + bias), parts fp32
    [S, batch * num_nodes, (q_heads + 2 kv_heads) * head_dim], then written as ``rope_kv_write_paged`` does."""
    what = "rope_kv_write_paged_parts"
    _paged_sizes(what, pages, kv_heads, head_dim)
    width, rows = (q_heads + 2 * kv_heads) * head_dim, batch * num_nodes
    if parts.dtype is not torch.float32 or parts.dim() != 3 or tuple(parts.shape[1:]) != (rows, width) or not parts.is_contiguous() \
            or parts.shape[0] == 0 or parts.data_ptr() % 16 or parts.get_device() != pages.device:
        raise ValueError(f"{what}: parts must be contiguous 16-byte aligned fp32 [S, {rows}, {width}] on the pages' device")
    read = [(parts.data_ptr(), parts.numel() * 4)]
    if bias is not None:
        if bias.dtype is not _BF16 or bias.numel() != width or not bias.is_contiguous() or bias.data_ptr() % 8 \
                or bias.get_device() != pages.device:
            raise ValueError(f"{what}: bias must be a contiguous 8-byte aligned bf16 [{width}] tensor")
        read.append((bias.data_ptr(), 2 * width))
    _write_paged("fg_rope_kv_write_paged_parts", (parts.data_ptr(), parts.shape[0], _ptr(bias)), pages, batch, num_nodes, q_heads,
                 head_dim, seq_len, pos_offset, inv_freq, q_out, new_len, row_map, err_flag, read)


def kv_read_paged(pages, *, count, start=None, row_map=None, batch=None, dtype=torch.bfloat16):
    """(k, v), each [batch, kv_heads, count, head_dim] in bf16 (exact but under 2^-126) or fp32: the values of tokens start[b] ..
    start[b] + count - 1 (start None: 0) of cache row row_map[b] (None: b); tokens without a page are 0 (``fg_kv_read_paged``).
    batch: that of start or row_map, or every row of the table."""
    if type(pages) is not KVPages:
        raise TypeError("kv_read_paged: pages must be KVPages")
    dev = pages.device
    if batch is None:
        batch = start.numel() if start is not None else row_map.numel() if row_map is not None else pages.rows
    if dev < 0:
        _same_device("kv_read_paged", dev)
    if dtype not in _DT:
        raise TypeError("kv_read_paged: dtype must be bfloat16 or float32")
    if batch < 0 or count < 0:
        raise ValueError("kv_read_paged: batch and count must not be negative")
    if not ((start is None or _held(start, dev, batch)) and (row_map is None or _held(row_map, dev, batch))):
        _index("kv_read_paged", dev, batch, ("start", start), ("row_map", row_map))
    k = torch.empty((batch, pages.kv_heads, count, pages.head_dim), dtype=dtype, device=pages.k.device)
    v = torch.empty_like(k)
    if batch and count:
        _call_on(dev, "fg_kv_read_paged", pages.address, batch, None if start is None else start.data_ptr(), count,
                 None if row_map is None else row_map.data_ptr(), k.data_ptr(), v.data_ptr(), _DT[dtype])
    return k, v


@functools.lru_cache(maxsize=4096)
def _paged_workspace_bytes(batch, num_nodes, q_heads, kv_heads, head_dim, capacity):
    return _lib.load().fg_paged_attention_workspace(batch, num_nodes, q_heads, kv_heads, head_dim, capacity)


def paged_attention(q, pages, *, seq_len, anc, num_nodes, q_heads, kv_heads, head_dim, out=None, new_len=None, row_map=None, scale=None,
                    bf16_weights=False):
    """``tree_attention`` over pages (``fg_paged_attention``): q bf16 [B, N, Hq, d] contiguous; anc int64 [B, N] or [N] (bits of
    the new tokens that a node sees), or None for a causal chain. ``new_len`` int32 [B]: the rows of nodes from new_len[b] on
    stay as they were in ``out`` (bf16, q's shape, apart from what is read), and nobody sees their tokens. A row that sees no token is 0, and
    infinities and NaN of tokens that it does not see do not reach it. ``scale``: positive and finite (None: head_dim^-0.5).
    ``bf16_weights``: the softmax's weights may be rounded to bf16, as ``tree_attention`` rounds them
    (``fg_paged_attention_bf16_weights``: faster where more than 32 rows share a kv head); otherwise they keep 17 bits."""
    _paged_sizes("paged_attention", pages, kv_heads, head_dim)
    dev, shape, at = pages.device, q.shape, q.data_ptr()
    given = out is not None
    if len(shape) != 4:
        raise ValueError(f"paged_attention: q must be contiguous bf16 [B, {num_nodes}, {q_heads}, {head_dim}]")
    B = shape[0]
    if not given:
        out = torch.empty_like(q)
    into, anc_stride, size = out.data_ptr(), 0, B * num_nodes * q_heads * head_dim
    ok = (q.dtype is _BF16 is out.dtype and shape == (B, num_nodes, q_heads, head_dim) == out.shape and q.is_contiguous()
          and out.is_contiguous() and q.get_device() == dev == out.get_device() and not at & 15 and not into & 7
          and _held(seq_len, dev, B) and (new_len is None or _held(new_len, dev, B)) and (row_map is None or _held(row_map, dev, B))
          and (scale is None or 0.0 < scale < math.inf))
    if ok and anc is not None:
        if anc.dtype is not torch.int64:
            raise TypeError("anc must be int64 (bit pattern of the uint64 masks)")
        two = anc.dim() == 2
        ok = anc.shape == ((B, num_nodes) if two else (num_nodes,)) and (num_nodes == 1 or anc.stride(-1) == 1) and anc.get_device() == dev
        anc_stride = anc.stride(0) if two else 0
    if not ok:
        what = "paged_attention"
        _index(what, dev, B, ("seq_len", seq_len), ("new_len", new_len), ("row_map", row_map))
        if anc is not None and (anc.get_device() != dev or tuple(anc.shape) not in ((B, num_nodes), (num_nodes,)) or (num_nodes > 1 and anc.stride(-1) != 1)):
            raise ValueError(f"{what}: anc must be [{B}, {num_nodes}] or [{num_nodes}] with unit stride on the pages' device")
        if q.dtype is not _BF16 or shape != (B, num_nodes, q_heads, head_dim) or not q.is_contiguous() or at & 15 or q.get_device() != dev:
            raise ValueError(f"{what}: q must be contiguous 16-byte aligned bf16 [B, {num_nodes}, {q_heads}, {head_dim}] on the pages' device")
        if not (scale is None or 0.0 < scale < math.inf):
            raise ValueError(f"{what}: scale must be positive and finite")
        raise ValueError(f"{what}: out must be a contiguous 8-byte aligned bf16 tensor of q's shape")
    if size == 0:
        return out
    lens, few = seq_len.data_ptr(), 4 * B
    new, rows = None if new_len is None else new_len.data_ptr(), None if row_map is None else row_map.data_ptr()
    masks = None if anc is None else anc.data_ptr()
    if given:
        _apart("paged_attention", ((into, 2 * size),), (*pages._spans, pages._table, (at, 2 * size), (lens, few), (new or 0, few), (rows or 0, few),
                                                        (masks or 0, 8 * ((B - 1) * anc_stride + num_nodes))))
    n = _paged_workspace_bytes(B, num_nodes, q_heads, kv_heads, head_dim, pages.width * pages.page_size)
    ws = torch.empty(n, dtype=_U8, device=q.device) if n else None  # the call's own, as in _mx_workspace
    _call_on(dev, "fg_paged_attention_bf16_weights" if bf16_weights else "fg_paged_attention", at, into, pages.address, B, num_nodes, q_heads,
             lens, new, rows, masks, anc_stride, head_dim ** -0.5 if scale is None else scale, None if ws is None else ws.data_ptr(), n)
    return out


def kv_path_gather_paged(pages, *, seq_len, acc_nodes, acc_len, tree_nodes, layers=1, layer_stride=0, scale_layer_stride=0,
                         row_map=None, err_flag=None):
    """``kv_path_gather`` over pages (``fg_kv_path_gather_paged``): tokens seq_len[b] + acc_nodes[b, j] move to seq_len[b] + j for
    j < acc_len[b], in ``layers`` layers whose pages lie ``layer_stride`` elements (their scales ``scale_layer_stride`` bytes)
    behind each other in the same pool. acc_nodes int32 [B, up to 32] contiguous."""
    what = "kv_path_gather_paged"
    if not isinstance(pages, KVPages):
        raise TypeError(f"{what}: pages must be KVPages")
    dev, B = pages.device, seq_len.numel()
    if dev < 0:
        _same_device(what, dev)
    if not (_held(seq_len, dev, B) and _held(acc_len, dev, B) and _held(acc_nodes, dev, B) and (row_map is None or _held(row_map, dev, B))
            and (err_flag is None or _held(err_flag, dev, 1))):
        _index(what, dev, B, ("seq_len", seq_len), ("acc_len", acc_len), ("acc_nodes", acc_nodes), ("row_map", row_map))
        _index(what, dev, 1, ("err_flag", err_flag))
    if acc_nodes.dim() != 2 or acc_nodes.shape[0] != B or not 1 <= acc_nodes.shape[1] <= 32:
        raise ValueError(f"{what}: acc_nodes must be [{B}, 1 to 32]")
    if layers < 1 or not 1 <= tree_nodes <= pages.capacity:
        raise ValueError(f"{what}: layers must be positive and the tree fit a cache row")
    if layers > 1:
        for t, s in ((pages.k, layer_stride), (pages.v, layer_stride), (pages.k_scales, scale_layer_stride),
                     (pages.v_scales, scale_layer_stride)):
            if t is not None:
                size = t.shape[1] * t.shape[2] * t.shape[3]
                last = t.storage_offset() + (pages.pages - 1) * t.stride(0) + (layers - 1) * s + size
                if s < size or last * t.element_size() > t.untyped_storage().nbytes():
                    raise ValueError(f"{what}: {layers} layers that far apart reach behind the pool")
    if B:
        _call_on(dev, "fg_kv_path_gather_paged", pages.address, layers, layer_stride, scale_layer_stride, B, seq_len.data_ptr(),
                 _ptr(row_map), acc_nodes.data_ptr(), acc_nodes.shape[1], acc_len.data_ptr(), tree_nodes, _ptr(err_flag))


# ------------------------------------------------------------------ sampling / acceptance
def sample_workspace(rows, device):
    """Scratch that lets draws of long rows run split over several workgroups per row."""
    n = _lib.load().fg_sample_workspace(int(rows))
    return torch.empty(n, dtype=torch.uint8, device=device)


def sample_tokens(logits, *, noise=None, noise_col=0, seed=0, step=0, seq_ids=None, draw=0, row_index=None,
                  forced=None, temperature=1.0, greedy=False, top_k=None, top_p=1.0, out=None, split=True):
    """One token per row (see the rule in csrc/sample.hip). noise: uint32 bits as int32 [R, C].
    split=False keeps every row in one workgroup (same tokens; used to cross-check)."""
    _dev(logits, noise, seq_ids, row_index, forced)
    for t, n in ((seq_ids, "seq_ids"), (row_index, "row_index"), (forced, "forced")):
        _i32(t, n)
    if noise is not None and noise.dtype != torch.int32:
        raise TypeError("noise must be int32 holding uint32 bit patterns")
    logits = aligned_rows(logits)
    V = logits.shape[-1]
    rows = row_index.numel() if row_index is not None else logits.shape[0]
    if out is None:
        out = torch.empty(rows, dtype=torch.int32, device=logits.device)
    T = 0.0 if temperature is None else float(temperature)
    use_T = T if T > 0 else (-1.0 if T < 0 or temperature is None else 0.0)
    g = bool(greedy) or (temperature is not None and T == 0.0)
    ws = sample_workspace(rows, logits.device) if split else None
    _call("fg_sample_tokens", _ptr(logits), dtype_code(logits), logits.stride(0), rows,
              V, _ptr(row_index), _ptr(forced), _ptr(noise), noise.stride(0) if noise is not None else 0,
              int(noise_col), int(seed) & (2 ** 64 - 1), int(step), _ptr(seq_ids), int(draw), use_T, int(g),
              int(top_k or 0), top_p_fixed(top_p), _ptr(out), _ptr(ws), 0 if ws is None else ws.numel(), _stream())
    return out


def accept_walk(tree_logits, tree_tokens, parents, n_nodes, *, max_walk_steps, slot_map=None, noise=None,
                noise_col0=0, seed=0, step=0, seq_ids=None, draw0=1, temperature=1.0, greedy=False, top_k=None,
                top_p=1.0, acc_stride=None, err_flag=None, out=None):
    """exact_target walk. Returns dict of int32 device tensors (acc_tokens, acc_nodes, acc_len, last_node, correction)."""
    _dev(tree_logits, tree_tokens, parents, n_nodes, slot_map, noise, seq_ids)
    for t, n in ((tree_tokens, "tree_tokens"), (parents, "parents"), (n_nodes, "n_nodes"), (slot_map, "slot_map"),
                 (seq_ids, "seq_ids")):
        _i32(t, n)
    B, nmax = tree_tokens.shape
    V = tree_logits.shape[-1]
    dev = tree_tokens.device
    acc_stride = acc_stride or (max_walk_steps + 1)
    if out is None:
        out = dict(acc_tokens=torch.zeros(B, acc_stride, dtype=torch.int32, device=dev),
                   acc_nodes=torch.zeros(B, acc_stride, dtype=torch.int32, device=dev),
                   acc_len=torch.empty(B, dtype=torch.int32, device=dev),
                   last_node=torch.empty(B, dtype=torch.int32, device=dev),
                   correction=torch.empty(B, dtype=torch.int32, device=dev),
                   state=torch.empty(3 * B, dtype=torch.int32, device=dev))
    T = 0.0 if temperature is None else float(temperature)
    use_T = T if T > 0 else (-1.0 if T < 0 or temperature is None else 0.0)
    g = bool(greedy) or (temperature is not None and T == 0.0)
    lg = aligned_rows(tree_logits.reshape(-1, V))
    _call("fg_accept_walk", _ptr(lg), dtype_code(lg), lg.stride(0), V, _ptr(slot_map), _ptr(tree_tokens),
              _ptr(parents), _ptr(n_nodes), nmax, B, int(max_walk_steps), _ptr(noise),
              noise.stride(0) if noise is not None else 0, int(noise_col0), int(seed) & (2 ** 64 - 1), int(step),
              _ptr(seq_ids), int(draw0), use_T, int(g), int(top_k or 0), top_p_fixed(top_p), _ptr(out["acc_tokens"]),
              _ptr(out["acc_nodes"]), acc_stride, _ptr(out["acc_len"]), _ptr(out["last_node"]),
              _ptr(out["correction"]), _ptr(out["state"]), _ptr(err_flag), _stream())
    return out


def walk_begin(tree_tokens, parents, n_nodes, *, acc_stride):
    """Initialise a step-at-a-time walk; returns the walk dict (outputs + state)."""
    _dev(tree_tokens, parents, n_nodes)
    B, nmax = tree_tokens.shape
    dev = tree_tokens.device
    w = dict(acc_tokens=torch.empty(B, acc_stride, dtype=torch.int32, device=dev),  # zeroed by fg_walk_begin
             acc_nodes=torch.empty(B, acc_stride, dtype=torch.int32, device=dev),
             acc_len=torch.empty(B, dtype=torch.int32, device=dev),
             last_node=torch.empty(B, dtype=torch.int32, device=dev),
             correction=torch.empty(B, dtype=torch.int32, device=dev),
             state=torch.empty(3 * B, dtype=torch.int32, device=dev),
             row_index=torch.empty(B, dtype=torch.int32, device=dev),
             row_active=torch.empty(B, dtype=torch.int32, device=dev),
             workspace=sample_workspace(B, dev))
    _call("fg_walk_begin", _ptr(tree_tokens), _ptr(parents), _ptr(n_nodes), nmax, B, _ptr(w["acc_tokens"]),
          _ptr(w["acc_nodes"]), acc_stride, _ptr(w["acc_len"]), _ptr(w["last_node"]), _ptr(w["correction"]),
          _ptr(w["state"]), _stream())
    return w


def walk_rows(walk, nmax):
    """Fill walk['row_index'] (b*nmax + parent) and walk['row_active'] for the next step."""
    B = walk["acc_len"].numel()
    _call("fg_walk_rows", _ptr(walk["state"]), B, nmax, _ptr(walk["row_index"]), _ptr(walk["row_active"]), _stream())


def walk_step(walk, step_logits, tree_tokens, parents, n_nodes, *, walk_step, noise=None, noise_col0=0, seed=0,
              step=0, seq_ids=None, draw0=1, temperature=1.0, greedy=False, top_k=None, top_p=1.0, err_flag=None,
              split=True, parts=None, next_rows=False):
    """One walk step: active row b draws from row b of step_logits.

    ``parts``: the (part_max, part_key) row maxima that ``lm_head_topk`` wrote with
    step_logits (a step that splits its rows then needs no chunk-maxima launch). ``next_rows``: also
    fill walk['row_index'] / walk['row_active'] for the next step (as ``walk_rows``)."""
    _dev(step_logits, tree_tokens, parents, n_nodes, noise, seq_ids)
    if parts is not None:
        _dev(*parts)
        pm, pk = parts
        if (pm.dtype != torch.float32 or pk.dtype != torch.int64 or pm.dim() != 2 or pm.shape != pk.shape
                or pm.shape[0] != tree_tokens.shape[0] or not pm.is_contiguous() or not pk.is_contiguous()):
            raise ValueError("walk_step: parts must be contiguous fp32 / int64 [batch, P] pairs")
    B, nmax = tree_tokens.shape
    lg = aligned_rows(step_logits)
    V = lg.shape[-1]
    T = 0.0 if temperature is None else float(temperature)
    use_T = T if T > 0 else (-1.0 if T < 0 or temperature is None else 0.0)
    g = bool(greedy) or (temperature is not None and T == 0.0)
    _call("fg_walk_step", _ptr(lg), dtype_code(lg), lg.stride(0), V, _ptr(tree_tokens), _ptr(parents), _ptr(n_nodes),
          nmax, B, int(walk_step), _ptr(noise), noise.stride(0) if noise is not None else 0, int(noise_col0),
          int(seed) & (2 ** 64 - 1), int(step), _ptr(seq_ids), int(draw0), use_T, int(g), int(top_k or 0),
          top_p_fixed(top_p), _ptr(walk["acc_tokens"]), _ptr(walk["acc_nodes"]), walk["acc_tokens"].stride(0),
          _ptr(walk["acc_len"]), _ptr(walk["last_node"]), _ptr(walk["correction"]), _ptr(walk["state"]),
          _ptr(err_flag), _ptr(parts[0]) if parts is not None else None, _ptr(parts[1]) if parts is not None else None,
          parts[0].shape[1] if parts is not None else 0, _ptr(walk["row_index"]) if next_rows else None,
          _ptr(walk["row_active"]) if next_rows else None, _ptr(walk["workspace"]) if split else None,
          walk["workspace"].numel() if split else 0, _stream())


def accept_finalize(walk, old_len, *, max_length, eos_token_id, finished=None, pending_root=None):
    _dev(old_len)
    _i32(old_len, "old_len")
    B = walk["acc_len"].numel()
    if finished is None:
        finished = torch.empty(B, dtype=torch.int32, device=old_len.device)
    _call("fg_accept_finalize", _ptr(walk["acc_tokens"]), _ptr(walk["acc_nodes"]), walk["acc_tokens"].stride(0),
              _ptr(walk["acc_len"]), _ptr(walk["last_node"]), _ptr(walk["correction"]), _ptr(old_len),
              int(max_length), -1 if eos_token_id is None else int(eos_token_id), _ptr(finished),
              _ptr(pending_root), B, _stream())
    return finished


def kv_path_gather(tensor_ptrs, *, batch, kv_heads, head_dim, elem_bytes, strides, capacity, seq_len, acc_nodes,
                   acc_len, tree_nodes, row_map=None, err_flag=None):
    """tensor_ptrs: int64 device tensor of cache base addresses (K0, V0, K1, V1, ...)."""
    _dev(tensor_ptrs, seq_len, acc_nodes, acc_len, row_map, err_flag)
    for t, n in ((seq_len, "seq_len"), (acc_nodes, "acc_nodes"), (acc_len, "acc_len"), (row_map, "row_map")):
        _i32(t, n)
    bs, hs, rs = strides
    _call("fg_kv_path_gather", _ptr(tensor_ptrs), tensor_ptrs.numel(), batch, kv_heads, head_dim, elem_bytes, bs,
              hs, rs, capacity, _ptr(seq_len), _ptr(row_map), _ptr(acc_nodes), acc_nodes.stride(0), _ptr(acc_len),
              int(tree_nodes), _ptr(err_flag), _stream())
