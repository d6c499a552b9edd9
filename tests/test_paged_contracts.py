"""What the paged cache promises where no GPU is needed: refusals, sizes of workspaces, layouts under tracing."""
import ctypes

import pytest
import torch
import torch.autograd.forward_ad as forward_ad
from torch._subclasses.fake_tensor import FakeTensorMode

from tests.test_paged_refusals import FAKE, attn_args, attn_metas, geom, meta
from world_engine_b200 import PagedSlab, _lib, ops
from world_engine_b200._lib import PagedGeom
from world_engine_b200.csrc import build as csrc_build


@pytest.fixture(scope="module")
def lib():
    csrc_build.build()
    return _lib.load()


def test_who_sits_out_is_checked(lib):
    good = meta((3,), torch.int32)
    plain, padded = ops._attn_plan(**attn_metas()), ops._attn_plan(**attn_metas(), n_new=good)
    assert padded[:2] == plain[:2] and padded[2] == plain[2] + 3 * 4 * 4
    for bad in (meta((3,), torch.int64), meta((4,), torch.int32), meta((3, 1), torch.int32), meta((3,), torch.int32, stride=(2,)),
                meta((3,), torch.int32, device=1)):
        with pytest.raises(ValueError):
            ops._attn_plan(**attn_metas(), n_new=bad)
    with pytest.raises(RuntimeError, match="no CPU path"):
        ops._attn_plan(**attn_metas(), n_new=meta((3,), torch.int32, device=-1))


@pytest.mark.parametrize("max_pages", [4, 400])
@pytest.mark.parametrize("weights", [0, 1])
def test_sitting_out_needs_a_workspace(lib, max_pages, weights):
    g = geom(max_pages=max_pages, table_stride=max_pages)
    need = lib.we_b200_paged_attn_workspace_bytes(ctypes.byref(g), 8, weights)
    more = lib.we_b200_paged_attn_workspace_bytes(ctypes.byref(g), 8, weights + 2)
    assert more == need + 3 * 4 * 4 and (need == 0) == (max_pages == 4 and not weights)
    a = attn_args(g, n_new=FAKE, weights=FAKE if weights else None, workspace_bytes=more - 1)
    assert lib.we_b200_paged_attn(ctypes.byref(a), None, None) == -5


@pytest.mark.parametrize("order", [(0, 1, 2, 3), (1, 0, 2, 3), (2, 1, 0, 3), (1, 2, 0, 3)])
def test_a_traced_output_has_the_strides_of_the_real_one(order):
    shape = (4, 8, 1, 64)
    with FakeTensorMode():
        q = torch.empty([shape[i] for i in order], dtype=torch.bfloat16).permute([order.index(i) for i in range(4)])
        assert q.shape == shape
        kv = torch.empty(2, 9, 2, 16, 64, dtype=torch.bfloat16)
        table, lens = torch.empty(4, 2, dtype=torch.int32), torch.empty(4, 2, dtype=torch.int32)
        out = ops.paged_attn_op(q, kv, table, lens, 0.0, None)
        assert out.shape == shape and out.stride() == torch.empty_like(q).stride()


def test_ops_refuse_what_has_a_tangent():
    slab = PagedSlab(2, 2, 64, torch.bfloat16, 16, 4, 32, keep=20, device="cpu")
    x = torch.zeros(2, 2, 1, 64, dtype=torch.bfloat16)
    w = torch.zeros(2, 2, 1)
    with forward_ad.dual_level():
        d, dw = forward_ad.make_dual(x, torch.ones_like(x)), forward_ad.make_dual(w, torch.ones_like(w))
        for call in (lambda: slab.append(d, x), lambda: slab.append(x, d), lambda: slab.append(x, x, w_new=dw), lambda: slab.attend(d)):
            with pytest.raises(RuntimeError, match="derivative"):
                call()
            with torch.no_grad(), pytest.raises(RuntimeError, match="derivative"):
                call()
        with pytest.raises(RuntimeError, match="no CPU path"):
            slab.append(x, x)


def test_a_budgeted_slab_costs_what_its_budget_needs(lib):
    slab = PagedSlab(2, 2, 64, torch.bfloat16, 16, 40, 4096, keep=100, sink=2, recent=8, device="cpu")
    assert slab.table.shape[1] == slab.max_pages == 7
    g = PagedGeom(2, 2, 64, 16, 40, slab.max_pages, _lib.BF16, 0, *slab.kv.stride()[:4], slab.table.stride(0))
    assert lib.we_b200_paged_evict_workspace_bytes(ctypes.byref(g), 1, 100) == 0
    slab.reserve(0, 4096)                        # as before, but a session under a budget gets no more than that needs
    assert slab.room(0) == 112 and slab.free_pages == 33
    slab.reserve(0, 100)
    assert slab.free_pages == 33
    with pytest.raises(ValueError, match="at most"):
        slab.reserve(1, 4097)
