"""Which kernel an MX product takes (``kernels.mx_plan``): the sizes of the GPU tests meet every one."""
import os

import pytest

import mx_sizes as S


@pytest.fixture(scope="module", autouse=True)
def _need_library():
    from flashgrpo_amd import _lib

    if not os.path.exists(_lib.library_path()):
        pytest.skip("native library not built")


@pytest.mark.parametrize("kind", [S.linear, S.gate_up])
@pytest.mark.parametrize("fmt", ["e4m3", "e2m1"])
def test_sizes_meet_the_kernels_they_are_listed_for(kind, fmt):
    from flashgrpo_amd import kernels as K

    for shape, detail, rows, cols, k in kind(fmt):
        plan = K.mx_plan(rows, cols, k, fmt=fmt, gate_up=kind is S.gate_up)
        assert S.is_plan(plan, shape, detail), (rows, cols, k, plan, shape, detail)


@pytest.mark.parametrize("fmt", ["e4m3", "e2m1"])
def test_every_kernel_has_a_size(fmt):
    whole = {(shape, cols % 8 == 0) for shape, detail, _, cols, _ in S.linear(fmt) if shape[2] and not detail}
    assert whole == {(t, wide) for t in S.TILES for wide in (True, False)}
    assert {shape for shape, detail, *_ in S.linear(fmt) if shape[2] and detail} == set(S.SPLIT_TILES)
    streams = {(shape[:2], detail == 12) for shape, detail, *_ in S.linear(fmt) if shape[2] == 0}
    held = {(16, 16), (16, 32), (16, 64), (32, 16), (32, 32), (64, 16)}
    assert {s for s, _ in streams} == held and ((16, 16), True) in streams
    whole = {shape for shape, detail, *_ in S.gate_up(fmt) if shape[2] and not detail}
    assert whole == set(S.TILES) - (set(S.TILES[1:3]) if fmt == "e4m3" else set())
    assert {shape for shape, detail, *_ in S.gate_up(fmt) if shape[2] and detail} == set(S.SPLIT_TILES)
    assert any(shape[2] == 0 for shape, *_ in S.gate_up(fmt))


def test_plans_agree_with_workspaces_and_refuse():
    from flashgrpo_amd import _lib
    from flashgrpo_amd import kernels as K

    lib = _lib.load()
    for fmt, shape, detail, rows, cols, k in S.every(S.linear):
        need = lib.fg_mx_linear_workspace(rows, cols, k, K.MX_FORMATS[fmt])
        plan = K.mx_plan(rows, cols, k, fmt=fmt)
        assert need == (plan.splits_or_waves * rows * ((cols + 3) // 4 * 4) * 4 if plan.stages and plan.splits_or_waves > 1 else 0)
    for bad in (dict(rows=0), dict(cols=0), dict(k=48), dict(k=0), dict(rows=(1 << 22) + 1), dict(fmt="e5m2"),
                dict(rows=2 ** 32 + 4), dict(cols=2 ** 32 + 64), dict(k=2 ** 32 + 64), dict(cols=1 << 30, gate_up=True)):
        with pytest.raises(ValueError):
            K.mx_plan(**{**dict(rows=4, cols=64, k=64), **bad})
