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


def test_ops_refuse_what_has_a_gradient():
    slab = PagedSlab(2, 2, 64, torch.bfloat16, 16, 4, 32, device="cpu")
    x = torch.zeros(2, 2, 1, 64, dtype=torch.bfloat16, requires_grad=True)
    for call in (lambda: slab.append(x, x), lambda: slab.attend(x)):
        with pytest.raises(RuntimeError, match="no backward"):
            call()
        with torch.no_grad(), pytest.raises(RuntimeError, match="no CPU path"):
            call()


def meta(shape, dtype=torch.bfloat16, stride=None, device=0):
    t = torch.empty(shape, dtype=dtype, device="meta")
    return t.shape, t.stride() if stride is None else stride, dtype, device


def attn_metas(**kw):
    m = dict(q=meta((3, 8, 1, 128)), kv=meta((2, 50, 4, 32, 128)), table=meta((3, 10), torch.int32),
             lens=meta((3, 4), torch.int32), weights=meta((50, 4, 32), torch.float32), out=ops._NONE, lse=ops._NONE)
    m.update(kw)
    return m


def test_shapes_types_and_devices_of_attention(lib):
    geom, shape, need = ops._attn_plan(**attn_metas())
    assert shape == (3, 8, 1, 128) and need > 0 and geom[:6] == (3, 4, 128, 32, 50, 10)
    for change in (dict(q=meta((3, 8, 2, 128))), dict(q=meta((2, 8, 1, 128))), dict(q=meta((3, 8, 1, 128), torch.float16)),
                   dict(q=meta((3, 8, 1, 128), stride=(1, 3, 1, 24))), dict(q=meta((3, 8, 128))),
                   dict(kv=meta((2, 50, 4, 32, 128), stride=(1, 2, 3, 4, 5))), dict(kv=meta((1, 50, 4, 32, 128))),
                   dict(kv=meta((50, 4, 32, 128))), dict(table=meta((3, 10), torch.int64)), dict(table=meta((10,), torch.int32)),
                   dict(lens=meta((3,), torch.int32)), dict(lens=meta((3, 4), torch.int64)),
                   dict(lens=meta((3, 4), torch.int32, stride=(1, 3))), dict(weights=meta((50, 4, 32), torch.float16)),
                   dict(weights=meta((50, 4, 16), torch.float32)), dict(out=meta((3, 8, 128))),
                   dict(out=meta((3, 8, 1, 128), torch.float32)), dict(lse=meta((3, 4), torch.float32)),
                   dict(lens=meta((3, 4), torch.int32, device=1)), dict(q=meta((3, 8, 1, 128), device=1))):
        with pytest.raises(ValueError):
            ops._attn_plan(**attn_metas(**change))
    with pytest.raises(TypeError):
        ops._attn_plan(**attn_metas(kv=meta((2, 50, 4, 32, 128), torch.float64)))
    with pytest.raises(RuntimeError, match="no CPU path"):
        ops._attn_plan(**attn_metas(lens=meta((3, 4), torch.int32, device=-1)))


def append_metas(**kw):
    counts = meta((3, 4), torch.int32)
    m = dict(kv=meta((2, 50, 4, 32, 128)), table=meta((3, 10), torch.int32), lens=counts, next_pos=counts, lens_out=counts,
             next_pos_out=counts, k_new=meta((3, 4, 7, 128)), v_new=meta((3, 4, 7, 128)), n_new=meta((3,), torch.int32),
             weights=meta((50, 4, 32), torch.float32), positions=meta((50, 4, 32), torch.int32),
             w_new=meta((3, 4, 7), torch.float32))
    m.update(kw)
    return m


def test_shapes_and_types_of_appends(lib):
    geom, strides, w_strides, T, need = ops._append_plan(**append_metas())
    assert T == 7 and need == 0 and strides == (4 * 7 * 128, 7 * 128, 128) * 2 and w_strides == (28, 7, 1)
    for change in (dict(k_new=meta((3, 4, 6, 128))), dict(v_new=meta((3, 4, 7, 64))), dict(k_new=meta((3, 7, 4, 128))),
                   dict(v_new=meta((3, 4, 7, 128), torch.float16)), dict(k_new=meta((3, 4, 7, 128), stride=(1, 1, 1, 2))),
                   dict(n_new=meta((3,), torch.int64)), dict(n_new=meta((4,), torch.int32)), dict(w_new=meta((3, 4, 6), torch.float32)),
                   dict(w_new=meta((3, 4, 7), torch.bfloat16)), dict(positions=meta((50, 4, 32), torch.int64)),
                   dict(next_pos=meta((4, 3), torch.int32)), dict(lens_out=meta((3, 4), torch.float32))):
        with pytest.raises(ValueError):
            ops._append_plan(**append_metas(**change))


@pytest.mark.parametrize("budget", [(0, 0, 0), (-5, 0, 0), (2 ** 31, 0, 0), (10, -1, 0), (10, 0, -1), (10, 6, 5)])
def test_budgets_that_make_no_sense(budget):
    slab = PagedSlab(2, 2, 64, torch.bfloat16, 16, 4, 32, device="cpu")
    x = torch.zeros(2, 2, 1, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        ops.paged_append_evict_(slab.kv, slab.table, slab.lens, slab.next_pos, x, x, slab.weights, slab.positions, *budget)


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
