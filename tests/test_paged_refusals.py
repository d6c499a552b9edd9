"""What the paged cache refuses on the host, and its bookkeeping of pages (no GPU needed)."""
import ctypes

import pytest
import torch

from world_engine_b200 import PagedSlab, _lib, ops
from world_engine_b200._lib import PagedAppendArgs, PagedAttnArgs, PagedGeom
from world_engine_b200.csrc import build as csrc_build

FAKE = 0x10000  # a 16-byte aligned, never dereferenced "device pointer"


@pytest.fixture(scope="module")
def lib():
    csrc_build.build()
    return _lib.load()


def geom(**kw):
    g = PagedGeom(3, 4, 128, 32, 50, 10, _lib.BF16, 0, 50 * 4 * 32 * 128, 4 * 32 * 128, 32 * 128, 128, 10)
    for k, v in kw.items():
        setattr(g, k, v)
    return g


def append_args(g=None, **kw):
    a = PagedAppendArgs(g or geom(), FAKE, FAKE, (4 * 8 * 128, 8 * 128, 128), (4 * 8 * 128, 8 * 128, 128), FAKE, FAKE, FAKE,
                        FAKE, FAKE, FAKE, FAKE, FAKE, None, None, (0, 0, 0), FAKE, 1 << 40, 8, 100, 4, 16)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def attn_args(g=None, **kw):
    a = PagedAttnArgs(g or geom(), FAKE, FAKE, (8 * 128, 128), (8 * 128, 128), FAKE, FAKE, FAKE, None, None, FAKE, 1 << 40, 8, 0.0)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


BAD_GEOMETRY = [(dict(S=0), -3), (dict(Hkv=0), -3), (dict(n_pages=0), -3), (dict(max_pages=0), -3), (dict(page=8), -3),
                (dict(page=48), -3), (dict(page=512), -3), (dict(Dh=96), -4), (dict(Dh=256), -4), (dict(dtype=_lib.F32), -4),
                (dict(token_stride=64), -3), (dict(token_stride=132), -2), (dict(head_stride=4), -2), (dict(page_stride=-8), -3),
                (dict(plane_stride=1), -2), (dict(table_stride=-1), -3), (dict(max_pages=1 << 26), -7), (dict(S=1 << 20), -7)]


@pytest.mark.parametrize("change,code", BAD_GEOMETRY)
def test_bad_geometry(lib, change, code):
    g = geom(**change)
    assert lib.we_b200_paged_append(ctypes.byref(append_args(g)), None, None) == code
    assert lib.we_b200_paged_append_evict(ctypes.byref(append_args(g)), None, None) == code
    assert lib.we_b200_paged_attn(ctypes.byref(attn_args(g)), None, None) == code
    assert lib.we_b200_paged_evict_workspace_bytes(ctypes.byref(g), 1, 10) == 0
    assert lib.we_b200_paged_attn_workspace_bytes(ctypes.byref(g), 8, 1) == 0


@pytest.mark.parametrize("change,code", [
    (dict(k_new=None), -1), (dict(v_new=None), -1), (dict(kv=None), -1), (dict(table=None), -1), (dict(lens=None), -1),
    (dict(next_pos=None), -1), (dict(lens_out=None), -1), (dict(next_pos_out=None), -1), (dict(weights=None, w_new=FAKE), -1),
    (dict(T=-1), -3), (dict(T=1 << 27), -7), (dict(k_new=FAKE + 2), -2), (dict(kv=FAKE + 8), -2),
    (dict(k_strides=(8, 8, 4)), -2), (dict(v_strides=(8, -8, 8)), -3), (dict(w_new=FAKE, w_strides=(1, -1, 1)), -3)])
def test_bad_appends(lib, change, code):
    assert lib.we_b200_paged_append(ctypes.byref(append_args(**change)), None, None) == code
    assert lib.we_b200_paged_append_evict(ctypes.byref(append_args(**change)), None, None) == code


@pytest.mark.parametrize("change,code", [
    (dict(weights=None), -1), (dict(positions=None), -1), (dict(keep=0), -3), (dict(sink=-1), -3), (dict(recent=-1), -3),
    (dict(sink=90, recent=11), -3), (dict(sink=2 ** 31 - 1, recent=2 ** 31 - 1), -3), (dict(keep=321), -3),
    (dict(workspace=FAKE + 1), -2), (dict(weights=FAKE + 4), -2), (dict(positions=FAKE + 8), -2)])
def test_bad_budgets(lib, change, code):
    assert lib.we_b200_paged_append_evict(ctypes.byref(append_args(**change)), None, None) == code


def test_a_table_too_wide_for_a_budget(lib):
    g = geom(max_pages=1 << 16, table_stride=1 << 16)
    assert lib.we_b200_paged_append_evict(ctypes.byref(append_args(g)), None, None) == -7


def test_workspaces(lib):
    # a table much wider than the budget: the lists of a session that holds that much need room
    g = geom(max_pages=4096, table_stride=4096)
    need = lib.we_b200_paged_evict_workspace_bytes(ctypes.byref(g), 8, 100)
    assert need > 0
    for change in (dict(workspace=None), dict(workspace_bytes=need - 1)):
        assert lib.we_b200_paged_append_evict(ctypes.byref(append_args(g, **change)), None, None) == -5
    need = lib.we_b200_paged_attn_workspace_bytes(ctypes.byref(g), 8, 0)
    more = lib.we_b200_paged_attn_workspace_bytes(ctypes.byref(g), 8, 1)
    assert 0 < need < more
    for change in (dict(workspace=None), dict(workspace_bytes=need - 1), dict(weights=FAKE, workspace_bytes=more - 1)):
        assert lib.we_b200_paged_attn(ctypes.byref(attn_args(g, **change)), None, None) == -5
    assert lib.we_b200_paged_attn(ctypes.byref(attn_args(g, workspace=FAKE + 4)), None, None) == -2


@pytest.mark.parametrize("change,code", [
    (dict(q=None), -1), (dict(out=None), -1), (dict(kv=None), -1), (dict(table=None), -1), (dict(lens=None), -1),
    (dict(Hq=0), -3), (dict(Hq=6), -3), (dict(Hq=65536), -7), (dict(q=FAKE + 8), -2), (dict(q_strides=(4, 8)), -2),
    (dict(out_strides=(8, -8)), -3), (dict(weights=FAKE + 4), -2)])
def test_bad_attention(lib, change, code):
    assert lib.we_b200_paged_attn(ctypes.byref(attn_args(**change)), None, None) == code


def test_null_arguments(lib):
    assert lib.we_b200_paged_append(None, None, None) == -1
    assert lib.we_b200_paged_append_evict(None, None, None) == -1
    assert lib.we_b200_paged_attn(None, None, None) == -1
    assert lib.we_b200_paged_evict_workspace_bytes(None, 1, 1) == 0
    assert lib.we_b200_paged_attn_workspace_bytes(None, 1, 0) == 0


def test_ops_refuse_cpu_tensors():
    slab = PagedSlab(2, 2, 64, torch.bfloat16, 16, 4, 32, device="cpu")
    x = torch.zeros(2, 2, 1, 64, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="no CPU path"):
        slab.append(x, x)
    with pytest.raises(RuntimeError, match="no CPU path"):
        slab.attend(x)


def test_pages_are_handed_out_once_and_come_back():
    slab = PagedSlab(3, 2, 64, torch.bfloat16, 16, 6, 64, device="cpu")
    slab.reserve(0, 17)
    slab.reserve(2, 64)
    assert slab.free_pages == 0 and (slab.room(0), slab.room(1), slab.room(2)) == (32, 0, 64)
    used = slab.table[slab.table >= 0].tolist()
    assert sorted(used) == list(range(6)) and torch.all(slab.table[1] == -1)
    with pytest.raises(RuntimeError, match="free pages"):
        slab.reserve(1, 1)
    slab.reserve(0, 5)                                        # has them already
    with pytest.raises(ValueError, match="at most"):
        slab.reserve(0, 65)
    slab.release(2)
    assert slab.free_pages == 4 and torch.all(slab.table[2] == -1)
    slab.reserve(1, 40)
    assert slab.free_pages == 1


@pytest.mark.parametrize("kw", [dict(page=24), dict(n_pages=0), dict(max_tokens=0), dict(keep=0), dict(keep=65),
                                dict(keep=10, sink=6, recent=5), dict(keep=10, sink=-1)])
def test_slab_refuses(kw):
    args = dict(n_sessions=2, H=2, Dh=64, dtype=torch.bfloat16, page=16, n_pages=8, max_tokens=64, device="cpu")
    args.update(kw)
    with pytest.raises(ValueError):
        PagedSlab(**args)
