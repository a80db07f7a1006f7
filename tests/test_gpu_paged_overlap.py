"""Outputs that lie in what a paged operator reads, or in the pages, and projected rows that lie in the pages they are written to:
refused before anything is launched. What lies next to them is taken."""
import pytest
import torch

from paged_cases import DEV, i32, kernels

pytestmark = pytest.mark.gpu
B, N, HQ, H, D, SIZE = 2, 2, 4, 2, 128, 16
PAGE = H * SIZE * D


@pytest.fixture(scope="module", autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


class Arena:
    """One allocation that holds everything: pages of K and V side by side, their scales, and room around them."""

    def __init__(self, fmt):
        self.raw = torch.zeros(1 << 20, dtype=torch.uint8, device=DEV)
        es, n = (2, 4) if fmt == "bf16" else (1, 4)
        self.es, self.pool = es, (1 << 16, n * 2 * PAGE * es)
        codes = self.take(1 << 16, n * 2 * PAGE * es, torch.bfloat16 if fmt == "bf16" else torch.float8_e4m3fn).view(n, 2, H, SIZE, D)
        ks = vs = None
        self.scales = (1 << 19, n * 2 * H * SIZE * 4)
        if fmt != "bf16":
            s = self.take(*self.scales, torch.uint8).view(n, 2, H, SIZE, 4)
            s.fill_(127)
            ks, vs = s[:, 0], s[:, 1]
        self.table = i32([[0, 1], [2, 3]])
        self.pages = kernels().KVPages(codes[:, 0], codes[:, 1], ks, vs, self.table)

    def take(self, at, n, dtype):
        return self.raw[at:at + n].view(dtype)

    def rows(self, at):
        return self.take(at, B * N * HQ * D * 2, torch.bfloat16).view(B, N, HQ, D)

    def inside(self):
        """Byte offsets at which q-shaped rows meet the pages or the scales, and such at which they do not."""
        (p, n), (s, m), size = self.pool, self.scales, B * N * HQ * D * 2
        last = [s, s + m - 16, s - size + 16] if self.es == 1 else []
        return [p, p + PAGE * self.es, p + n - 16, p - size + 16, *last], [p - size, p + n, s - size, s + m]


@pytest.mark.parametrize("fmt", ["e4m3", "bf16"])
def test_outputs_and_rows_in_the_pages(fmt):
    k, a = kernels(), Arena(fmt)
    seq, off, f = i32([3, 5]), i32([0, 1]), torch.ones(D // 2, device=DEV)
    sizes = dict(num_nodes=N, q_heads=HQ, kv_heads=H, head_dim=D)
    q = torch.zeros(B, N, HQ, D, dtype=torch.bfloat16, device=DEV)
    qkv = torch.zeros(B * N, (HQ + 2 * H) * D, dtype=torch.bfloat16, device=DEV)
    calls = {"attend": lambda at: k.paged_attention(q, a.pages, seq_len=seq, anc=None, out=a.rows(at), **sizes),
             "write": lambda at: k.rope_kv_write_paged(qkv, a.pages, batch=B, seq_len=seq, pos_offset=off, inv_freq=f, q_out=a.rows(at), **sizes)}
    bad, good = a.inside()
    for what, call in calls.items():
        for at in bad:
            with pytest.raises(ValueError, match="overlap"):
                call(at)
                pytest.fail(f"{what} {at}")
        for at in good:
            call(at)
    width = qkv.numel() * 2
    rows = lambda at: a.take(at, width, torch.bfloat16).view(B * N, -1)
    write = lambda x: k.rope_kv_write_paged(x, a.pages, batch=B, seq_len=seq, pos_offset=off, inv_freq=f, q_out=q, **sizes)
    p, n = a.pool
    for at in (p, p + n - 16, p - width + 16):
        with pytest.raises(ValueError, match="overlap"):
            write(rows(at))
    write(rows(p - width)), write(rows(p + n))
    parts = a.take(p, width * 2, torch.float32).view(1, B * N, -1)
    with pytest.raises(ValueError, match="overlap"):
        k.rope_kv_write_paged_parts(parts, None, a.pages, batch=B, seq_len=seq, pos_offset=off, inv_freq=f, q_out=q, **sizes)
    torch.cuda.synchronize()


def test_outputs_in_the_small_operands():
    k, a = kernels(), Arena("e4m3")
    out = torch.zeros(B, N, HQ, D, dtype=torch.bfloat16, device=DEV)
    ints = out.view(torch.int32).view(-1)
    seq, off, f = i32([3, 5]), i32([0, 1]), torch.ones(D // 2, device=DEV)
    sizes = dict(num_nodes=N, q_heads=HQ, kv_heads=H, head_dim=D)
    q = torch.zeros_like(out)
    qkv = torch.zeros(B * N, (HQ + 2 * H) * D, dtype=torch.bfloat16, device=DEV)
    anc = out.view(torch.int64).view(-1)[:B * N].view(B, N)
    over = kernels().KVPages(a.pages.k, a.pages.v, a.pages.k_scales, a.pages.v_scales, ints[:4].view(2, 2))

    def attend(pages=a.pages, seq=seq, **kw):
        k.paged_attention(q, pages, seq_len=seq, out=out, **{**dict(anc=None), **sizes, **kw})

    def write(pages=a.pages, seq=seq, off=off, f=f, **kw):
        k.rope_kv_write_paged(qkv, pages, batch=B, seq_len=seq, pos_offset=off, inv_freq=f, q_out=out, **sizes, **kw)

    attend(), write()
    two = ints[:2]
    for call in [lambda: attend(seq=two), lambda: attend(new_len=two), lambda: attend(row_map=two), lambda: attend(anc=anc), lambda: attend(pages=over),
                 lambda: write(seq=two), lambda: write(off=two), lambda: write(f=out.view(torch.float32).view(-1)[:D // 2]), lambda: write(new_len=two),
                 lambda: write(row_map=two), lambda: write(pages=over)]:
        with pytest.raises(ValueError, match="overlap"):
            call()
    torch.cuda.synchronize()
