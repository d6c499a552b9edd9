"""Tensor-level entry points over the C ABI, plus their `torch.library` custom
ops so that the calls survive `torch.compile(fullgraph=True)` -- the way the
reference wraps its own native kernel (src/quantize.py:17-42).

Every function here enqueues on the caller's current CUDA stream, performs no
host synchronisation and allocates nothing except (once per device) the
split-KV workspace and the status word.
"""
from __future__ import annotations

import ctypes
from typing import Optional, Tuple

import torch
import torch.autograd.forward_ad as _forward_ad

from . import _lib
from ._lib import CacheGeom, PagedGeom, PrologueArgs, Strides3

_DTYPE_CODE = {torch.bfloat16: _lib.BF16, torch.float16: _lib.F16, torch.float32: _lib.F32}


def dtype_code(dtype: torch.dtype) -> int:
    try:
        return _DTYPE_CODE[dtype]
    except KeyError:
        raise TypeError(f"world_engine_b200: unsupported cache dtype {dtype}") from None


def _require_cuda(*tensors: torch.Tensor) -> None:
    for t in tensors:
        if t is not None and not t.is_cuda:
            raise RuntimeError(
                "world_engine_b200 runs on CUDA tensors only (sm_100a); there is no CPU path")


def _strides3(t: torch.Tensor) -> Strides3:
    if t.dim() != 4 or t.stride(3) != 1:
        raise ValueError("expected a [B, H, T, Dh] tensor whose last axis is contiguous")
    return Strides3(t.stride(0), t.stride(1), t.stride(2))


def _stream_ptr(device: torch.device) -> int:
    return torch.cuda.current_stream(device).cuda_stream


def make_geom(kv: torch.Tensor, written: torch.Tensor, tokens_per_frame: int, dilation: int,
              frame_t_stride: int = 0) -> CacheGeom:
    """Geometry of a reference-layout cache tensor kv[2, B, H, L+T, Dh]
    (src/model/kv_cache.py:81-84)."""
    if kv.dim() != 5 or kv.size(0) != 2:
        raise ValueError("kv must be [2, B, H, L + tokens_per_frame, Dh]")
    if kv.stride(4) != 1 or kv.stride(3) != kv.size(4) or kv.stride(2) != kv.size(3) * kv.size(4):
        raise ValueError("kv must be contiguous over (head, token, head_dim)")
    _, B, H, C, Dh = kv.shape
    g = CacheGeom()
    g.B, g.Hkv, g.T, g.Dh = B, H, tokens_per_frame, Dh
    g.L = C - tokens_per_frame
    g.dilation = dilation
    g.dtype = dtype_code(kv.dtype)
    g.kv_plane_stride = kv.stride(0)
    g.kv_batch_stride = kv.stride(1)
    g.written_batch_stride = written.stride(0) if written.dim() == 2 else 0
    g.frame_t_stride = frame_t_stride
    return g


# ------------------------------------------------------------------ workspace
_workspaces = {}
_status_words = {}


def workspace_for(device: torch.device, nbytes: int) -> torch.Tensor:
    """Zero-initialised split-KV workspace of the device (grown on demand).
    Calls that share it must be ordered on one stream."""
    key = (device.type, device.index if device.index is not None else torch.cuda.current_device())
    ws = _workspaces.get(key)
    if ws is None or ws.numel() < nbytes:
        ws = torch.zeros(max(nbytes, 1 << 20), dtype=torch.uint8, device=device)
        _workspaces[key] = ws
    return ws


def status_word(device: torch.device) -> torch.Tensor:
    key = (device.type, device.index if device.index is not None else torch.cuda.current_device())
    st = _status_words.get(key)
    if st is None:
        st = torch.zeros(1, dtype=torch.int32, device=device)
        _status_words[key] = st
    return st


def check_status(device: torch.device) -> None:
    """Synchronising health check: raises if a kernel on `device` reported a device-side anomaly."""
    st = int(status_word(device).item())
    if st != 0:
        status_word(device).zero_()
        what = {1: "a bounded wait of the attention kernel expired; the output of that call is invalid",
                2: "a token position points outside the RoPE table (IndexError in the reference)",
                3: "a page index or a token count of a paged cache is out of range"}.get(st & 0xFF, "unknown")
        where = f" (debug build: wait at source line {st >> 8})" if st >> 8 else ""
        raise RuntimeError(f"world_engine_b200: device status {st & 0xFF}: {what}{where}")


def kv_append_(kv: torch.Tensor, written: torch.Tensor, k_new: torch.Tensor, v_new: torch.Tensor,
               frame_t: torch.Tensor, tokens_per_frame: int, dilation: int, is_frozen: bool,
               mask_written: Optional[torch.Tensor] = None, frame_t_stride: int = 0) -> None:
    """In-place append of one frame (we_b200_kv_append)."""
    _require_cuda(kv, written, k_new, v_new, frame_t, mask_written)
    g = make_geom(kv, written, tokens_per_frame, dilation, frame_t_stride)
    lib = _lib.load()
    with torch.cuda.device(kv.device):
        rc = lib.we_b200_kv_append(
            k_new.data_ptr(), _strides3(k_new), v_new.data_ptr(), _strides3(v_new),
            kv.data_ptr(), written.data_ptr(),
            mask_written.data_ptr() if mask_written is not None else None,
            frame_t.data_ptr(), ctypes.byref(g), int(bool(is_frozen)), _stream_ptr(kv.device))
    _lib.check(rc, "we_b200_kv_append")


def frame_attn(q: torch.Tensor, kv: torch.Tensor, written: torch.Tensor, frame_t: torch.Tensor,
               tokens_per_frame: int, dilation: int, scale: float = 0.0,
               out: Optional[torch.Tensor] = None, frame_t_stride: int = 0) -> torch.Tensor:
    """Attention of the new frame's queries over the cache (we_b200_frame_attn).
    The output has q's shape and strides, like flex_attention's."""
    _require_cuda(q, kv, written, frame_t)
    g = make_geom(kv, written, tokens_per_frame, dilation, frame_t_stride)
    if out is None:
        out = torch.empty_like(q)
    lib = _lib.load()
    B, Hq, T, Dh = q.shape
    with torch.cuda.device(q.device):
        need = lib.we_b200_attn_workspace_bytes(B, Hq, T, Dh, g.L)
        ws = workspace_for(q.device, need)
        rc = lib.we_b200_frame_attn(
            q.data_ptr(), _strides3(q), out.data_ptr(), _strides3(out), Hq,
            kv.data_ptr(), written.data_ptr(), frame_t.data_ptr(), ctypes.byref(g), float(scale),
            ws.data_ptr(), ws.numel(), status_word(q.device).data_ptr(), _stream_ptr(q.device))
    _lib.check(rc, "we_b200_frame_attn")
    return out


def frame_attn_no_alloc(q: torch.Tensor, out: torch.Tensor, status: torch.Tensor, kv: torch.Tensor,
                        written: torch.Tensor, frame_t: torch.Tensor, tokens_per_frame: int, dilation: int,
                        scale: float = 0.0, frame_t_stride: int = 0) -> torch.Tensor:
    """`frame_attn` for hosts that must not allocate device memory while running (an engine that gave
    the whole GPU to its own arena, a plug-in limited to the buffers it receives): binds
    we_b200_frame_attn_static, whose split-KV scratch is a fixed 12 MiB array inside the library.
    Nothing is allocated here either, so `out` (q's shape) and `status` (one int32) are the caller's.
    Raises WeB200Error (code -8) for shapes that need more scratch.  Calls share that one array:
    keep them on one stream per device, and make the first call on a device outside stream capture."""
    _require_cuda(q, out, status, kv, written, frame_t)
    g = make_geom(kv, written, tokens_per_frame, dilation, frame_t_stride)
    lib = _lib.load()
    with torch.cuda.device(q.device):
        rc = lib.we_b200_frame_attn_static(
            q.data_ptr(), _strides3(q), out.data_ptr(), _strides3(out), q.size(1),
            kv.data_ptr(), written.data_ptr(), frame_t.data_ptr(), ctypes.byref(g), float(scale),
            status.data_ptr(), _stream_ptr(q.device))
    _lib.check(rc, "we_b200_frame_attn_static")
    return out


def append_attend(q: torch.Tensor, k_new: torch.Tensor, v_new: torch.Tensor, kv: torch.Tensor,
                  written: torch.Tensor, frame_t: torch.Tensor, tokens_per_frame: int, dilation: int,
                  is_frozen: bool, scale: float = 0.0, out: Optional[torch.Tensor] = None,
                  mask_written: Optional[torch.Tensor] = None, frame_t_stride: int = 0,
                  gate: Optional[torch.Tensor] = None, gate_is_logits: bool = False) -> torch.Tensor:
    """One layer-step: append the frame, then attend (we_b200_append_attend).  With `gate` (a `[B,Hq,T]` view of
    q's dtype) the output rows are multiplied by it, or by its sigmoid when `gate_is_logits`, on their way out
    (we_b200_append_attend_gated; src/model/attn.py:117-119)."""
    _require_cuda(q, k_new, v_new, kv, written, frame_t, mask_written, gate)
    g = make_geom(kv, written, tokens_per_frame, dilation, frame_t_stride)
    if out is None:
        out = torch.empty_like(q)
    lib = _lib.load()
    B, Hq, T, Dh = q.shape
    if gate is not None and (gate.shape != (B, Hq, T) or gate.dtype != q.dtype):
        raise ValueError("gate must be a [B, Hq, T] view of q's dtype")
    with torch.cuda.device(q.device):
        need = lib.we_b200_attn_workspace_bytes(B, Hq, T, Dh, g.L)
        ws = workspace_for(q.device, need)
        head = (q.data_ptr(), _strides3(q), out.data_ptr(), _strides3(out), Hq,
                k_new.data_ptr(), _strides3(k_new), v_new.data_ptr(), _strides3(v_new),
                kv.data_ptr(), written.data_ptr(),
                mask_written.data_ptr() if mask_written is not None else None,
                frame_t.data_ptr(), ctypes.byref(g), int(bool(is_frozen)), float(scale))
        tail = (ws.data_ptr(), ws.numel(), status_word(q.device).data_ptr(), _stream_ptr(q.device))
        if gate is None:
            rc = lib.we_b200_append_attend(*head, *tail)
        else:
            rc = lib.we_b200_append_attend_gated(*head, gate.data_ptr(), Strides3(*gate.stride()),
                                                 int(bool(gate_is_logits)), *tail)
    _lib.check(rc, "we_b200_append_attend")
    return out


def qkv_prologue(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, v1: Optional[torch.Tensor],
                 v_lamb: Optional[torch.Tensor], cos_table: torch.Tensor, sin_table: torch.Tensor,
                 t_pos: torch.Tensor, y_pos: torch.Tensor, x_pos: torch.Tensor, height: int, width: int,
                 eps: Optional[float] = None) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """q, k, v `[B,H,T,Dh]` views (any strides, head dim contiguous) -> (q', k', v') as the attention and the
    cache receive them: value residual, weightless RMS norm and RoPE in one pass (we_b200_qkv_prologue;
    src/model/attn.py:105-110).  `v1=None` skips the residual.  Outputs are fresh `[B,T,H,Dh]`-ordered
    buffers viewed as `[B,H,T,Dh]`, the layout the merged-QKV slices have."""
    _require_cuda(q, k, v, v1, v_lamb, cos_table, sin_table, t_pos, y_pos, x_pos)
    B, Hq, T, Dh = q.shape
    Hkv = k.shape[1]
    if cos_table.dtype != torch.float32 or sin_table.dtype != torch.float32 or not cos_table.is_contiguous() \
            or not sin_table.is_contiguous() or cos_table.shape != sin_table.shape or cos_table.shape[-1] != Dh // 2:
        raise ValueError("cos / sin tables must be contiguous float32 [rows, Dh/2]")
    for name, t in (("t_pos", t_pos), ("y_pos", y_pos), ("x_pos", x_pos)):
        if t.dtype != torch.int64 or t.shape != (B, T) or t.stride() != t_pos.stride() or t.stride(1) != 1:
            raise ValueError(f"{name} must be int64 [B, T] with contiguous rows")
    q_out = torch.empty((B, T, Hq, Dh), dtype=q.dtype, device=q.device).transpose(1, 2)
    k_out = torch.empty((B, T, Hkv, Dh), dtype=k.dtype, device=k.device).transpose(1, 2)
    v_out = torch.empty((B, T, Hkv, Dh), dtype=v.dtype, device=v.device).transpose(1, 2)
    a = PrologueArgs()
    a.q_in, a.k_in, a.v_in = q.data_ptr(), k.data_ptr(), v.data_ptr()
    a.v1 = v1.data_ptr() if v1 is not None else None
    a.q_out, a.k_out, a.v_out = q_out.data_ptr(), k_out.data_ptr(), v_out.data_ptr()
    a.q_in_strides, a.k_in_strides, a.v_in_strides = _strides3(q), _strides3(k), _strides3(v)
    a.v1_strides = _strides3(v1) if v1 is not None else Strides3(0, 0, 0)
    a.q_out_strides, a.k_out_strides, a.v_out_strides = _strides3(q_out), _strides3(k_out), _strides3(v_out)
    if v1 is not None:
        if v_lamb is None or v_lamb.numel() != 1:
            raise ValueError("v_lamb must be a one-element tensor when v1 is given")
        a.v_lamb, a.v_lamb_dtype = v_lamb.data_ptr(), dtype_code(v_lamb.dtype)
    a.cos_table, a.sin_table, a.table_rows = cos_table.data_ptr(), sin_table.data_ptr(), cos_table.shape[0]
    a.t_pos, a.y_pos, a.x_pos = t_pos.data_ptr(), y_pos.data_ptr(), x_pos.data_ptr()
    a.pos_batch_stride = t_pos.stride(0)
    a.height, a.width = int(height), int(width)
    a.B, a.T, a.Hq, a.Hkv, a.Dh = B, T, Hq, Hkv, Dh
    a.dtype = dtype_code(q.dtype)
    a.eps = float(torch.finfo(torch.float32).eps if eps is None else eps)
    lib = _lib.load()
    with torch.cuda.device(q.device):
        rc = lib.we_b200_qkv_prologue(ctypes.byref(a), status_word(q.device).data_ptr(), _stream_ptr(q.device))
    _lib.check(rc, "we_b200_qkv_prologue")
    return q_out, k_out, v_out


def block_mask_tables(mask_written: torch.Tensor, tokens_per_frame: int
                      ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """int32 tables of the flex BlockMask for a visibility vector (we_b200_block_mask)."""
    _require_cuda(mask_written)
    C = mask_written.numel()
    qb = (tokens_per_frame + 127) // 128
    kb = (C + 127) // 128
    dev = mask_written.device
    kv_num = torch.empty((1, 1, qb), dtype=torch.int32, device=dev)
    kv_idx = torch.empty((1, 1, qb, kb), dtype=torch.int32, device=dev)
    full_num = torch.empty((1, 1, qb), dtype=torch.int32, device=dev)
    full_idx = torch.empty((1, 1, qb, kb), dtype=torch.int32, device=dev)
    lib = _lib.load()
    with torch.cuda.device(dev):
        rc = lib.we_b200_block_mask(mask_written.data_ptr(), C, tokens_per_frame, kv_num.data_ptr(),
                                    kv_idx.data_ptr(), full_num.data_ptr(), full_idx.data_ptr(),
                                    _stream_ptr(dev))
    _lib.check(rc, "we_b200_block_mask")
    return kv_num, kv_idx, full_num, full_idx


# ---------------------------------------------------------------- paged cache
# A decoding step makes these calls for every layer, so their cost on the host counts: all checks of shapes, types,
# strides and devices are one look-up of the values they depend on, and the arguments are packed in one go.
_status_ptrs = {}
_append_plans = {}
_attn_plans = {}
_MAX_PLANS = 4096
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or \
    (lambda index: torch.cuda.current_stream(index).cuda_stream)
_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device
_NONE = (None, None, None, None)


def _refuse_grad(*tensors) -> None:
    for t in tensors:
        if t is not None and t.requires_grad:
            raise RuntimeError("the paged cache operators have no backward pass; call them under torch.no_grad()")


def _refuse_tangents(*tensors) -> None:
    """Within forward_ad.dual_level() (which torch.no_grad() does not end)."""
    for t in tensors:
        if t is not None and _forward_ad.unpack_dual(t).tangent is not None:
            raise RuntimeError("the paged cache operators have no forward derivative; give them the primals")


def _check_paged(kv, table, counts, per_slot, others) -> Tuple[int, ...]:
    """What every paged entry point checks; the geometry's fields.  A tensor is given as its (shape, strides, type,
    device index), one that is left out as `_NONE`."""
    for meta in (kv, table, *counts, *per_slot, *others):
        if meta == _NONE:
            continue
        if meta[3] < 0:
            raise RuntimeError("world_engine_b200 runs on CUDA tensors only (sm_100a); there is no CPU path")
        if meta[3] != kv[3]:
            raise ValueError("all tensors of a paged cache call must be on the device of kv")
    shape, stride, dtype, _ = kv
    if len(shape) != 5 or shape[0] != 2 or stride[4] != 1:
        raise ValueError("kv must be [2, pages, Hkv, page, Dh] with a contiguous last axis")
    _, P, Hkv, page, Dh = shape
    if len(table[0]) != 2 or table[1][1] != 1 or table[2] != torch.int32:
        raise ValueError("table must be int32 [S, max_pages] with contiguous rows")
    S, M = table[0]
    for meta in counts:
        if meta == _NONE:
            continue
        if meta[2] != torch.int32 or meta[0] != (S, Hkv) or not _dense(meta):
            raise ValueError("token counts and positions must be contiguous int32 [S, Hkv]")
    for meta, want in zip(per_slot, (torch.float32, torch.int32)):
        if meta != _NONE and (meta[2] != want or meta[0] != (P, Hkv, page) or not _dense(meta)):
            raise ValueError("weights (float32) and positions (int32) must be contiguous [pages, Hkv, page]")
    return (S, Hkv, Dh, page, P, M, dtype_code(dtype), 0, stride[0], stride[1], stride[2], stride[3], table[1][0])


def _check_n_new(meta, S: int) -> None:
    if meta != _NONE and (meta[2] != torch.int32 or meta[0] != (S,) or not _dense(meta)):
        raise ValueError("n_new must be contiguous int32 [S]")


def _dense(meta) -> bool:
    want = 1
    for n, s in zip(reversed(meta[0]), reversed(meta[1])):
        if n != 1 and s != want:
            return False
        want *= n
    return True


def _call_paged(fn, args: bytes, index: int, where: str) -> None:
    """One library call on the device of the tensors and its current stream."""
    status = _status_ptrs.get(index)
    if status is None:
        status = _status_ptrs[index] = status_word(torch.device("cuda", index)).data_ptr()
    if index == _current_device():
        rc = fn(args, status, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(args, status, _raw_stream(index))
    if rc:
        _lib.check(rc, where)


def _plan(plans, make, key):
    """The plan of a call nobody made before (a plan depends on nothing but the values in its key)."""
    if len(plans) >= _MAX_PLANS:
        plans.clear()
    args = (*(key[i:i + 4] for i in range(0, len(key) // 4 * 4, 4)), *key[len(key) // 4 * 4:])
    if key[3] < 0:                       # not on a GPU: refused in there
        return make(*args)
    with torch.cuda.device(key[3]):      # (a workspace's size depends on the device's SMs)
        plans[key] = plan = make(*args)
    return plan


def _append_plan(kv, table, lens, next_pos, lens_out, next_pos_out, k_new, v_new, n_new, weights, positions, w_new,
                 keep=0):
    """Checks of an append; (geometry, strides of k_new and v_new, strides of w_new, T, workspace bytes)."""
    geom = _check_paged(kv, table, (lens, next_pos, lens_out, next_pos_out), (weights, positions),
                        (k_new, v_new, n_new, w_new))
    S, Hkv, Dh = geom[:3]
    shape = k_new[0]
    if len(shape) != 4 or (shape[0], shape[1], shape[3]) != (S, Hkv, Dh) or v_new[0] != shape \
            or k_new[2] != kv[2] or v_new[2] != kv[2] or k_new[1][3] != 1 or v_new[1][3] != 1:
        raise ValueError("k_new and v_new must be [S, Hkv, T, Dh] of the cache's type with a contiguous last axis")
    _check_n_new(n_new, S)
    if w_new != _NONE and (w_new[2] != torch.float32 or w_new[0] != shape[:3]):
        raise ValueError("w_new must be float32 [S, Hkv, T]")
    need = 0
    if keep > 0:
        need = _lib.load().we_b200_paged_evict_workspace_bytes(ctypes.byref(PagedGeom(*geom)), shape[2], keep)
    return geom, (*k_new[1][:3], *v_new[1][:3]), w_new[1] if w_new != _NONE else (0, 0, 0), shape[2], need


def _append(fn, where, kv, table, lens, next_pos, k_new, v_new, n_new, weights, positions, w_new, lens_out,
            next_pos_out, keep, sink, recent) -> None:
    if torch.is_grad_enabled():
        _refuse_grad(kv, k_new, v_new, weights, w_new)
    if getattr(_forward_ad, "_current_level", 0) >= 0:         # (-1: nobody is taking forward derivatives)
        _refuse_tangents(kv, k_new, v_new, weights, w_new)
    index = kv.get_device()
    key = (kv.shape, kv.stride(), kv.dtype, index,
           table.shape, table.stride(), table.dtype, table.get_device(),
           lens.shape, lens.stride(), lens.dtype, lens.get_device(),
           next_pos.shape, next_pos.stride(), next_pos.dtype, next_pos.get_device(),
           *(_NONE if lens_out is None else (lens_out.shape, lens_out.stride(), lens_out.dtype, lens_out.get_device())),
           *(_NONE if next_pos_out is None else
             (next_pos_out.shape, next_pos_out.stride(), next_pos_out.dtype, next_pos_out.get_device())),
           k_new.shape, k_new.stride(), k_new.dtype, k_new.get_device(),
           v_new.shape, v_new.stride(), v_new.dtype, v_new.get_device(),
           *(_NONE if n_new is None else (n_new.shape, n_new.stride(), n_new.dtype, n_new.get_device())),
           *(_NONE if weights is None else (weights.shape, weights.stride(), weights.dtype, weights.get_device())),
           *(_NONE if positions is None else
             (positions.shape, positions.stride(), positions.dtype, positions.get_device())),
           *(_NONE if w_new is None else (w_new.shape, w_new.stride(), w_new.dtype, w_new.get_device())), keep)
    geom, strides, w_strides, T, need = _append_plans.get(key) or _plan(_append_plans, _append_plan, key)
    ws = kv.new_empty((need + 1) // 2) if need else None          # (in 16-bit values: cheaper to ask for than bytes)
    _call_paged(fn, _lib.PAGED_APPEND_PACK.pack(
        *geom, k_new.data_ptr(), v_new.data_ptr(), *strides, kv.data_ptr(),
        0 if weights is None else weights.data_ptr(), 0 if positions is None else positions.data_ptr(),
        table.data_ptr(), lens.data_ptr(), next_pos.data_ptr(), (lens if lens_out is None else lens_out).data_ptr(),
        (next_pos if next_pos_out is None else next_pos_out).data_ptr(),
        0 if n_new is None else n_new.data_ptr(), 0 if w_new is None else w_new.data_ptr(), *w_strides,
        0 if ws is None else ws.data_ptr(), need, T, keep, sink, recent), index, where)


def paged_append_(kv: torch.Tensor, table: torch.Tensor, lens: torch.Tensor, next_pos: torch.Tensor,
                  k_new: torch.Tensor, v_new: torch.Tensor, n_new: Optional[torch.Tensor] = None,
                  weights: Optional[torch.Tensor] = None, positions: Optional[torch.Tensor] = None,
                  w_new: Optional[torch.Tensor] = None, lens_out: Optional[torch.Tensor] = None,
                  next_pos_out: Optional[torch.Tensor] = None) -> None:
    """In-place append to a paged cache (we_b200_paged_append).  `kv [2, P, Hkv, page, Dh]` is the pool, row s of
    `table [S, M]` the pages of session s, `lens` / `next_pos` `[S, Hkv]` the tokens a kv head holds and was ever
    given.  `k_new` / `v_new` are `[S, Hkv, T, Dh]` views (any strides, head dim contiguous); of a padded batch only
    the first `n_new[s]` tokens count.  The counts are updated in place unless `lens_out` / `next_pos_out` are
    given.  The first token for which a session has no page is dropped with all behind it and reported by
    `check_status`: `lens` counts what is held, `next_pos` what was given."""
    _append(_lib.load().we_b200_paged_append, "we_b200_paged_append", kv, table, lens, next_pos, k_new, v_new, n_new,
            weights, positions, w_new, lens_out, next_pos_out, 0, 0, 0)


def paged_append_evict_(kv: torch.Tensor, table: torch.Tensor, lens: torch.Tensor, next_pos: torch.Tensor,
                        k_new: torch.Tensor, v_new: torch.Tensor, weights: torch.Tensor, positions: torch.Tensor,
                        keep: int, sink: int = 0, recent: int = 0, n_new: Optional[torch.Tensor] = None,
                        w_new: Optional[torch.Tensor] = None, lens_out: Optional[torch.Tensor] = None,
                        next_pos_out: Optional[torch.Tensor] = None) -> None:
    """`paged_append_` under a budget (we_b200_paged_append_evict): afterwards no kv head holds more than `keep`
    tokens.  Kept are the positions below `sink`, the last `recent` positions, and of the rest those with the
    largest accumulated weight (of equal ones the lower index); tokens move only into the slots that evicted ones
    left, so the order of a session's tokens is not kept (`positions` tells which is which)."""
    if weights is None or positions is None:
        raise ValueError("eviction needs weights and positions")
    if not (0 < keep < 2 ** 31 and 0 <= sink and 0 <= recent and sink + recent <= keep):
        raise ValueError("a budget needs 0 <= sink + recent <= keep and at least one token")
    _append(_lib.load().we_b200_paged_append_evict, "we_b200_paged_append_evict", kv, table, lens, next_pos, k_new,
            v_new, n_new, weights, positions, w_new, lens_out, next_pos_out, keep, sink, recent)


def _attn_plan(q, kv, table, lens, weights, out, lse, n_new=_NONE):
    """Checks of an attention call; (geometry, shape, workspace bytes)."""
    geom = _check_paged(kv, table, (lens,), (weights,), (q, out, lse, n_new))
    S, _, Dh = geom[:3]
    shape = q[0]
    if len(shape) != 4 or (shape[0], shape[2], shape[3]) != (S, 1, Dh) or q[2] != kv[2] or q[1][3] != 1:
        raise ValueError("q must be [S, Hq, 1, Dh] of the cache's type with a contiguous last axis")
    if out != _NONE and (out[0] != shape or out[2] != q[2] or out[1][3] != 1):
        raise ValueError("out must have q's shape and type and a contiguous last axis")
    if lse != _NONE and (lse[2] != torch.float32 or lse[0] != shape[:2] or not _dense(lse)):
        raise ValueError("lse must be contiguous float32 [S, Hq]")
    _check_n_new(n_new, S)
    need = _lib.load().we_b200_paged_attn_workspace_bytes(
        ctypes.byref(PagedGeom(*geom)), shape[1], (weights != _NONE) + 2 * (n_new != _NONE))
    return geom, (S, shape[1], 1, Dh), need


def paged_attn(q: torch.Tensor, kv: torch.Tensor, table: torch.Tensor, lens: torch.Tensor, scale: float = 0.0,
               weights: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
               lse: Optional[torch.Tensor] = None, n_new: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of one new token per session over its paged cache (we_b200_paged_attn).  `q` is a
    `[S, Hq, 1, Dh]` view; the output has its shape.  With `weights` the softmax weight every held token is given
    (summed over the query heads of its kv head) is added to it in place; `lse` (float32 `[S, Hq]`, contiguous)
    receives the logarithm of the softmax sum.  A kv head that holds nothing gives 0 and -inf.  So does a
    session that sits out (`n_new[s] < 1`, int32 `[S]`, as in a padded append): its weights stay as they are, and
    neither its cache nor its row of `q` is read.  `out` must not overlap `q`.  Results repeat bit for bit (but for the
    weights of pages that several sessions share)."""
    if torch.is_grad_enabled():
        _refuse_grad(q, kv, weights, out, lse)
    if getattr(_forward_ad, "_current_level", 0) >= 0:         # (-1: nobody is taking forward derivatives)
        _refuse_tangents(q, kv, weights, out, lse)
    index, qs = q.get_device(), q.stride()
    key = (q.shape, qs, q.dtype, index,
           kv.shape, kv.stride(), kv.dtype, kv.get_device(),
           table.shape, table.stride(), table.dtype, table.get_device(),
           lens.shape, lens.stride(), lens.dtype, lens.get_device(),
           *(_NONE if weights is None else (weights.shape, weights.stride(), weights.dtype, weights.get_device())),
           *(_NONE if out is None else (out.shape, out.stride(), out.dtype, out.get_device())),
           *(_NONE if lse is None else (lse.shape, lse.stride(), lse.dtype, lse.get_device())),
           *(_NONE if n_new is None else (n_new.shape, n_new.stride(), n_new.dtype, n_new.get_device())))
    geom, shape, need = _attn_plans.get(key) or _plan(_attn_plans, _attn_plan, key)
    if out is None:
        out = torch.empty_like(q)
    elif out.data_ptr() == q.data_ptr():
        raise ValueError("out must not be q itself: a head's query is read by several CTAs, not all at the same time")
    ws = q.new_empty((need + 1) // 2) if need else None            # (in 16-bit values: cheaper to ask for than bytes)
    os_ = out.stride()
    _call_paged(_lib.load().we_b200_paged_attn, _lib.PAGED_ATTN_PACK.pack(
        *geom, q.data_ptr(), out.data_ptr(), qs[0], qs[1], os_[0], os_[1], kv.data_ptr(), table.data_ptr(),
        lens.data_ptr(), 0 if weights is None else weights.data_ptr(), 0 if lse is None else lse.data_ptr(),
        0 if ws is None else ws.data_ptr(), need, shape[1], scale, 0 if n_new is None else n_new.data_ptr()),
        index, "we_b200_paged_attn")
    return out


# ----------------------------------------------------------------- custom ops
# Registered under the reference's own namespace style ("world_engine::...").
@torch.library.custom_op("world_engine_b200::append_attend", mutates_args=("kv", "written"))
def append_attend_op(q: torch.Tensor, k_new: torch.Tensor, v_new: torch.Tensor, kv: torch.Tensor,
                     written: torch.Tensor, frame_t: torch.Tensor, tokens_per_frame: int,
                     dilation: int, is_frozen: bool, scale: float) -> torch.Tensor:
    return append_attend(q, k_new, v_new, kv, written, frame_t, tokens_per_frame, dilation,
                         is_frozen, scale)


@append_attend_op.register_fake
def _append_attend_fake(q, k_new, v_new, kv, written, frame_t, tokens_per_frame, dilation,
                        is_frozen, scale):
    return torch.empty_like(q)


@torch.library.custom_op("world_engine_b200::kv_append", mutates_args=("kv", "written", "mask_written"))
def kv_append_op(kv: torch.Tensor, written: torch.Tensor, mask_written: torch.Tensor,
                 k_new: torch.Tensor, v_new: torch.Tensor, frame_t: torch.Tensor,
                 tokens_per_frame: int, dilation: int, is_frozen: bool) -> None:
    kv_append_(kv, written, k_new, v_new, frame_t, tokens_per_frame, dilation, is_frozen,
               mask_written=mask_written)


@kv_append_op.register_fake
def _kv_append_fake(kv, written, mask_written, k_new, v_new, frame_t, tokens_per_frame, dilation,
                    is_frozen):
    return None


@torch.library.custom_op("world_engine_b200::frame_attn", mutates_args=())
def frame_attn_op(q: torch.Tensor, kv: torch.Tensor, written: torch.Tensor, frame_t: torch.Tensor,
                  tokens_per_frame: int, dilation: int, scale: float) -> torch.Tensor:
    return frame_attn(q, kv, written, frame_t, tokens_per_frame, dilation, scale)


@frame_attn_op.register_fake
def _frame_attn_fake(q, kv, written, frame_t, tokens_per_frame, dilation, scale):
    return torch.empty_like(q)


@torch.library.custom_op("world_engine_b200::qkv_prologue", mutates_args=())
def qkv_prologue_op(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, v1: Optional[torch.Tensor],
                    v_lamb: Optional[torch.Tensor], cos_table: torch.Tensor, sin_table: torch.Tensor,
                    t_pos: torch.Tensor, y_pos: torch.Tensor, x_pos: torch.Tensor, height: int,
                    width: int) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    return qkv_prologue(q, k, v, v1, v_lamb, cos_table, sin_table, t_pos, y_pos, x_pos, height, width)


@qkv_prologue_op.register_fake
def _qkv_prologue_fake(q, k, v, v1, v_lamb, cos_table, sin_table, t_pos, y_pos, x_pos, height, width):
    def like(t):
        B, H, T, Dh = t.shape
        return torch.empty((B, T, H, Dh), dtype=t.dtype, device=t.device).transpose(1, 2)
    return like(q), like(k), like(v)


@torch.library.custom_op("world_engine_b200::append_attend_gated", mutates_args=("kv", "written"))
def append_attend_gated_op(q: torch.Tensor, k_new: torch.Tensor, v_new: torch.Tensor, kv: torch.Tensor,
                           written: torch.Tensor, frame_t: torch.Tensor, gate: torch.Tensor,
                           tokens_per_frame: int, dilation: int, is_frozen: bool, scale: float,
                           gate_is_logits: bool) -> torch.Tensor:
    return append_attend(q, k_new, v_new, kv, written, frame_t, tokens_per_frame, dilation, is_frozen, scale,
                         gate=gate, gate_is_logits=gate_is_logits)


@append_attend_gated_op.register_fake
def _append_attend_gated_fake(q, k_new, v_new, kv, written, frame_t, gate, tokens_per_frame, dilation, is_frozen,
                              scale, gate_is_logits):
    return torch.empty_like(q)


@torch.library.custom_op("world_engine_b200::paged_append",
                         mutates_args=("kv", "lens", "next_pos", "weights", "positions"))
def paged_append_op(kv: torch.Tensor, table: torch.Tensor, lens: torch.Tensor, next_pos: torch.Tensor,
                    k_new: torch.Tensor, v_new: torch.Tensor, n_new: Optional[torch.Tensor], weights: torch.Tensor,
                    positions: torch.Tensor, w_new: Optional[torch.Tensor]) -> None:
    paged_append_(kv, table, lens, next_pos, k_new, v_new, n_new, weights, positions, w_new)


@paged_append_op.register_fake
def _paged_append_fake(kv, table, lens, next_pos, k_new, v_new, n_new, weights, positions, w_new):
    return None


@torch.library.custom_op("world_engine_b200::paged_append_evict",
                         mutates_args=("kv", "lens", "next_pos", "weights", "positions"))
def paged_append_evict_op(kv: torch.Tensor, table: torch.Tensor, lens: torch.Tensor, next_pos: torch.Tensor,
                          k_new: torch.Tensor, v_new: torch.Tensor, weights: torch.Tensor, positions: torch.Tensor,
                          keep: int, sink: int, recent: int, n_new: Optional[torch.Tensor],
                          w_new: Optional[torch.Tensor]) -> None:
    paged_append_evict_(kv, table, lens, next_pos, k_new, v_new, weights, positions, keep, sink, recent, n_new, w_new)


@paged_append_evict_op.register_fake
def _paged_append_evict_fake(kv, table, lens, next_pos, k_new, v_new, weights, positions, keep, sink, recent, n_new,
                             w_new):
    return None


@torch.library.custom_op("world_engine_b200::paged_attn", mutates_args=("weights",))
def paged_attn_op(q: torch.Tensor, kv: torch.Tensor, table: torch.Tensor, lens: torch.Tensor, scale: float,
                  weights: Optional[torch.Tensor], n_new: Optional[torch.Tensor] = None) -> torch.Tensor:
    return paged_attn(q, kv, table, lens, scale, weights, n_new=n_new)


@paged_attn_op.register_fake
def _paged_attn_fake(q, kv, table, lens, scale, weights, n_new=None):
    return torch.empty_like(q)
