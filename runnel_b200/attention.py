"""Attention over a paged key-value cache: the other half of a full-attention
decoder layer around the MoE block, for serving.

Functional layer over the C ABI (``rnb_kv_*``, ``rnb_rope_append``,
``rnb_paged_attention``), in the order of a step:

* :func:`kv_plan` gives a step's new tokens their pages, slots and positions;
* :func:`rope_append` norms and rotates queries and keys and writes keys and
  values to the cache (:func:`rope`: queries alone, without a cache);
* :func:`paged_attention` attends to it: one new token for each request, a few,
  or whole prompts, in any mix;
* :func:`kv_release` gives the pages of finished requests back;
* :func:`status` reads and clears the device's status bits.

A layer's cache is two tensors ``[num_pages, n_kv_heads, page_size, head_dim]``
(bf16 or fp16; page and head strides are free).  Lengths, tables, slots and
positions are int32 CUDA tensors and stay on the device.  Calls are
asynchronous on the current stream of their tensors' device and can be captured
in a CUDA graph; each takes its scratch from torch's allocator unless it is
given one.  Nothing falls back to another implementation.
"""
from __future__ import annotations

import ctypes
from typing import NamedTuple

import torch

from . import _lib

_DTYPES = {torch.bfloat16: 0, torch.float16: 1}
_i32 = torch.int32


class KVPlan(NamedTuple):
    """What :func:`kv_plan` says of a step (views of one buffer, int32)."""

    seq_lens: torch.Tensor  # [B] cached plus new tokens
    cu_q: torch.Tensor  # [B + 1] first new-token row of each request, then their number
    positions: torch.Tensor  # [max_tokens]
    slots: torch.Tensor  # [max_tokens], -1 behind the last request's rows
    free_count: torch.Tensor  # [1] pages left on the free list


def _ints(t: torch.Tensor, name: str, device: torch.device, shape: tuple | None = None) -> int:
    """data_ptr of a contiguous int32 tensor on ``device``."""
    if t.dtype is not _i32 or t.device != device or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int32 tensor on {device}")
    if shape is not None and t.shape != shape:
        raise ValueError(f"{name} must have shape {list(shape)}, not {list(t.shape)}")
    return t.data_ptr()


def _cuda(t: torch.Tensor, name: str) -> torch.device:
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor: the kernels have no other implementation")
    return t.device


_fns: dict = {}  # bound C functions by name
_raw_stream = torch._C._cuda_getCurrentRawStream  # what current_stream(device).cuda_stream gives, 2 us sooner
_current_device = torch._C._cuda_getDevice


def _call(fn: str, device: torch.device, *args) -> None:
    """One C call on the current stream of ``device``."""
    f = _fns.get(fn)
    if f is None:
        f = _fns[fn] = getattr(_lib.load(), fn)
    i = device.index
    if i == _current_device():
        rc = f(*args, _raw_stream(i))
    else:
        with torch.cuda.device(device):
            rc = f(*args, _raw_stream(i))
    if rc:
        _lib.check(fn, rc)


def kv_plan(table: torch.Tensor, ctx_lens: torch.Tensor, new_lens: torch.Tensor, free_pages: torch.Tensor,
            free_count: torch.Tensor, *, page_size: int, num_pages: int, max_tokens: int) -> KVPlan:
    """Pages, slots and positions of one step.

    Request ``b`` holds ``ctx_lens[b]`` cached tokens in its row of ``table``
    ``[B, cols]`` and gets ``new_lens[b]`` more (0: idle).  The pages it lacks
    come from the end of ``free_pages[:free_count]`` (``free_count``: one
    element) and are written into ``table``, in place; the inputs are otherwise
    left as they are, so the same call gives the same answer again until
    ``plan.free_count`` and ``plan.seq_lens`` are taken over.  ``max_tokens``
    bounds the step's new tokens; rows behind the last one get slot -1, which
    the other calls skip.

    All or nothing: where pages, table columns or ``max_tokens`` do not
    suffice, or a length is negative, the plan is void (``cu_q`` 0, slots -1,
    ``seq_lens`` = ``ctx_lens``, nothing taken) and :func:`status` has
    ``STATUS_NO_PAGES``.
    """
    dev = _cuda(table, "table")
    if table.dim() != 2:
        raise ValueError("table must be [requests, columns]")
    B, cols = table.shape
    if max_tokens < 0:
        raise ValueError("max_tokens must be >= 0")
    args = (_ints(table, "table", dev), _ints(ctx_lens, "ctx_lens", dev, (B,)), _ints(new_lens, "new_lens", dev, (B,)),
            _ints(free_pages, "free_pages", dev), free_pages.numel(), _ints(free_count, "free_count", dev, (1,)))
    buf = torch.empty(2 * B + 2 + 2 * max_tokens, dtype=_i32, device=dev)
    p = buf.data_ptr()
    cu, pos = p + 4 * B, p + 8 * B + 4
    slots = pos + 4 * max_tokens
    _call("rnb_kv_plan", dev, B, cols, page_size, num_pages, max_tokens, *args, p, cu, pos, slots,
          slots + 4 * max_tokens)
    return KVPlan(*buf.split_with_sizes((B, B + 1, max_tokens, max_tokens, 1)))


def kv_release(table: torch.Tensor, lens: torch.Tensor, finished: torch.Tensor, free_pages: torch.Tensor,
               free_count: torch.Tensor, *, page_size: int) -> tuple[torch.Tensor, torch.Tensor]:
    """Append the pages of requests with ``finished[b] != 0`` (int32) to
    ``free_pages[:free_count]``, in place; returns (lengths with theirs 0, the
    new count).  Does nothing, with ``STATUS_NO_PAGES``, if they do not fit."""
    dev = _cuda(table, "table")
    if table.dim() != 2:
        raise ValueError("table must be [requests, columns]")
    B, cols = table.shape
    args = (_ints(table, "table", dev), _ints(lens, "lens", dev, (B,)), _ints(finished, "finished", dev, (B,)),
            _ints(free_pages, "free_pages", dev), free_pages.numel(), _ints(free_count, "free_count", dev, (1,)))
    out = torch.empty(B + 1, dtype=_i32, device=dev)
    _call("rnb_kv_release", dev, B, cols, page_size, *args, out.data_ptr(), out.data_ptr() + 4 * B)
    return out[:B], out[B:]


def status(device=None) -> int:
    """Status bits (``_lib.STATUS_*``) of this module's calls on a device since
    the last read; clears them and synchronises the current stream."""
    dev = torch.device("cuda" if device is None else device)
    if dev.type != "cuda":
        raise ValueError("status is kept for CUDA devices")
    if dev.index is None:
        dev = torch.device("cuda", torch.cuda.current_device())
    out = ctypes.c_uint32()
    _call("rnb_kv_status", dev, ctypes.byref(out))
    return out.value


# ------------------------------------------------------------- tensors

def _rows(t: torch.Tensor, name: str, dtype: torch.dtype, device: torch.device, shape: tuple) -> torch.Tensor:
    """``t`` itself if the kernels take its strides, else a packed copy."""
    if t.dtype is not dtype or t.device != device:
        raise ValueError(f"{name} must be a {dtype} tensor on {device}")
    if t.shape != shape:
        raise ValueError(f"{name} must have shape {list(shape)}, not {list(t.shape)}")
    st = t.stride()
    if st[2] == 1 and not (st[0] | st[1]) & 7 and not t.data_ptr() & 15:
        return t
    return torch.empty(shape, dtype=dtype, device=device).copy_(t)


def _cache(k: torch.Tensor, v: torch.Tensor) -> _lib.RnbKvCache:
    code = _DTYPES.get(k.dtype)
    if code is None or v.dtype is not k.dtype:
        raise ValueError("k_cache and v_cache must be bfloat16 or float16, both of one type")
    if k.dim() != 4 or v.shape != k.shape or v.device != k.device:
        raise ValueError("k_cache and v_cache must be [num_pages, n_kv_heads, page_size, head_dim] on one device")
    N, H, P, D = k.shape
    ks, vs = k.stride(), v.stride()
    if ks[3] != 1 or ks[2] != D or vs[3] != 1 or vs[2] != D:
        raise ValueError("a head's page must be contiguous in k_cache and v_cache")
    return _lib.RnbKvCache(code, N, P, H, D, 0, k.data_ptr(), v.data_ptr(), ks[0], ks[1], vs[0], vs[1])


def _out(out: torch.Tensor | None, like: torch.Tensor, shape: tuple, name: str = "out") -> torch.Tensor:
    if out is None:
        return torch.empty(shape, dtype=like.dtype, device=like.device)
    if out.dtype is not like.dtype or out.device != like.device or out.shape != shape or not out.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {like.dtype} tensor of shape {list(shape)} on {like.device}")
    return out


# -------------------------------------------------------------- rotary

def _rope(q, k, v, positions, inv_freq, slots, k_cache, v_cache, sections, interleaved, q_norm, k_norm, eps, out):
    dev = _cuda(q, "q")
    if q.dim() != 3:
        raise ValueError("q must be [tokens, heads, head_dim]")
    T, Hq, D = q.shape
    dt = q.dtype
    code = _DTYPES.get(dt)
    if code is None:
        raise ValueError("q must be bfloat16 or float16")
    half = inv_freq.numel()
    if inv_freq.dtype is not torch.float32 or inv_freq.device != dev or not inv_freq.is_contiguous():
        raise ValueError(f"inv_freq must be a contiguous float32 tensor on {dev}")
    sections = (half,) if sections is None else tuple(sections)
    axes = len(sections)
    if not 1 <= axes <= 4:
        raise ValueError("sections must name one to four axes")
    if positions.dtype is torch.int64:
        positions = positions.to(_i32)
    if positions.shape != (axes, T) and not (axes == 1 and positions.shape == (T,)):
        if positions.shape != (T,):
            raise ValueError(f"positions must have shape {[axes, T]} or {[T]}, not {list(positions.shape)}")
        positions = positions.expand(axes, T).contiguous()  # text: every axis at the token's position
    pos = _ints(positions, "positions", dev)
    for w, name in ((q_norm, "q_norm"), (k_norm, "k_norm")):
        if w is not None and (w.dtype is not dt or w.device != dev or w.shape != (D,) or not w.is_contiguous()):
            raise ValueError(f"{name} must be a contiguous {dt} tensor of {D} elements on {dev}")
    Hkv = 0
    ks = vs = (0, 0, 1)
    cache = kp = vp = sp = None
    if k_cache is not None:
        _cuda(k_cache, "k_cache")
        if k_cache.device != dev or k_cache.dtype is not dt:
            raise ValueError(f"k_cache and v_cache must be {dt} tensors on {dev}, like q")
        cache = _cache(k_cache, v_cache)
        Hkv = cache.n_kv_heads
        if cache.head_dim != D:
            raise ValueError("q and the cache must have one head_dim")
        k = _rows(k, "k", dt, dev, (T, Hkv, D))
        v = _rows(v, "v", dt, dev, (T, Hkv, D))
        ks, vs, kp, vp = k.stride(), v.stride(), k.data_ptr(), v.data_ptr()
        sp = _ints(slots, "slots", dev, (T,))
    qr = _rows(q, "q", dt, dev, (T, Hq, D))
    if out is None:
        out = torch.empty((T, Hq, D), dtype=dt, device=dev)
    else:
        _out(out, q, (T, Hq, D))
    if T == 0:
        return out
    qs = qr.stride()
    d = _lib.RnbRopeDesc(code, T, Hq, Hkv, D, 2 * half, axes, 1 if interleaved else 0, sections + (0,) * (4 - axes), eps, 0,
                         qs[0], qs[1], ks[0], ks[1], vs[0], vs[1])
    _call("rnb_rope_append", dev, ctypes.byref(d), qr.data_ptr(), kp, vp,
          None if q_norm is None else q_norm.data_ptr(), None if k_norm is None else k_norm.data_ptr(), pos,
          inv_freq.data_ptr(), sp, None if cache is None else ctypes.byref(cache), out.data_ptr())
    return out


def rope_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, positions: torch.Tensor, inv_freq: torch.Tensor,
                slots: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, *, sections=None,
                interleaved: bool = False, q_norm: torch.Tensor | None = None, k_norm: torch.Tensor | None = None,
                eps: float = 1e-6, out: torch.Tensor | None = None) -> torch.Tensor:
    """Norm, rotate, append: the rotated queries ``[T, Hq, D]``; rotated keys and
    the values go to the cache rows of ``slots`` ``[T]``, in place.

    ``q``, ``k``, ``v`` are ``[tokens, heads, head_dim]`` and may be views of one
    joint projection.  With ``q_norm`` / ``k_norm`` (``[head_dim]``) each head is
    RMS-normed first.  ``inv_freq`` (fp32, ``rot / 2``) turns the first ``rot``
    elements of a head in halves: element ``i`` with ``i + rot / 2``.
    ``positions`` is ``[axes, T]`` (or ``[T]``: all axes alike); ``sections`` says how many
    frequencies each axis (for images: time, height, width) turns, one section
    after the other, or in turns with ``interleaved``.  Rows with slot -1 are
    left alone, in ``out`` too.  ``out`` may be ``q`` if that is contiguous.
    """
    if k_cache is None or slots is None:
        raise ValueError("rope_append needs a cache and slots; rope() turns queries without them")
    return _rope(q, k, v, positions, inv_freq, slots, k_cache, v_cache, sections, interleaved, q_norm, k_norm, eps, out)


def rope(q: torch.Tensor, positions: torch.Tensor, inv_freq: torch.Tensor, *, sections=None, interleaved: bool = False,
         norm: torch.Tensor | None = None, eps: float = 1e-6, out: torch.Tensor | None = None) -> torch.Tensor:
    """:func:`rope_append`'s norm and rotation of one tensor ``[T, heads, head_dim]``, without a cache."""
    return _rope(q, None, None, positions, inv_freq, None, None, None, sections, interleaved, norm, None, eps, out)


# ----------------------------------------------------------- attention

_ws_bytes: dict[tuple, int] = {}  # workspace bytes by what they depend on (shapes and device)


def paged_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, table: torch.Tensor,
                    seq_lens: torch.Tensor, *, cu_q: torch.Tensor | None = None, max_q: int | None = None,
                    scale: float | None = None, window: int = 0, gate: torch.Tensor | None = None,
                    out: torch.Tensor | None = None, return_lse: bool = False):
    """Causal attention of ``q`` ``[T, Hq, D]`` over the paged cache: ``[T, Hq, D]``, or
    (that, lse ``[T, Hq]`` fp32).

    Request ``b`` has query rows ``cu_q[b]:cu_q[b + 1]`` (``cu_q`` None: one row each), the last
    of its ``seq_lens[b]`` cached positions, and sees itself and what lies before
    it (``window`` > 0: its last ``window`` positions only).  ``scale`` defaults to
    ``head_dim ** -0.5``; with ``gate`` ``[T, Hq, D]`` the output is multiplied by its
    sigmoid.  A row that sees nothing gives zeros and lse -inf.  Rows of ``out``
    behind ``cu_q[-1]`` are left as they were.  ``max_q``, a bound on the rows of one
    request, picks the kernels and is worth giving.
    """
    dev = _cuda(q, "q")
    if q.dim() != 3:
        raise ValueError("q must be [tokens, heads, head_dim]")
    T, Hq, D = q.shape
    dt = q.dtype
    if k_cache.device != dev or k_cache.dtype is not dt:
        raise ValueError(f"k_cache and v_cache must be {dt} tensors on {dev}, like q")
    cache = _cache(k_cache, v_cache)
    if cache.head_dim != D:
        raise ValueError("q and the cache must have one head_dim")
    if table.dim() != 2:
        raise ValueError("table must be [requests, columns]")
    B, cols = table.shape
    tp, sl = _ints(table, "table", dev), _ints(seq_lens, "seq_lens", dev, (B,))
    cu = None
    if cu_q is not None:
        cu = _ints(cu_q, "cu_q", dev, (B + 1,))
    elif T != B:
        raise ValueError("without cu_q every request has one query row: q must have as many as table")
    qr = _rows(q, "q", dt, dev, (T, Hq, D))
    gp, gs = None, (0, 0, 1)
    if gate is not None:
        gr = _rows(gate, "gate", dt, dev, (T, Hq, D))
        gp, gs = gr.data_ptr(), gr.stride()
    if out is None:
        out = torch.empty((T, Hq, D), dtype=dt, device=dev)
    else:
        _out(out, q, (T, Hq, D))
    lse = torch.empty((T, Hq), dtype=torch.float32, device=dev) if return_lse else None
    qs = qr.stride()
    most = 0 if max_q is None else int(max_q)
    if most < 0:
        raise ValueError("max_q must be >= 0")
    if cu is None:
        most = 1
    d = _lib.RnbAttnDesc(B, T, Hq, cols, most, window, D ** -0.5 if scale is None else scale, 0, qs[0], qs[1], gs[0], gs[1])
    key = (dev.index, B, T, Hq, cache.n_kv_heads, D, most)
    need = _ws_bytes.get(key)
    if need is None:
        n = ctypes.c_size_t()
        with torch.cuda.device(dev):
            _lib.call("rnb_paged_attention_workspace_size", ctypes.byref(d), ctypes.byref(cache), ctypes.byref(n))
        if len(_ws_bytes) > 4096:
            _ws_bytes.clear()
        need = _ws_bytes[key] = n.value
    ws = torch.empty(need, dtype=torch.uint8, device=dev)
    _call("rnb_paged_attention", dev, ctypes.byref(d), ctypes.byref(cache), qr.data_ptr(), gp, tp, sl, cu,
          out.data_ptr(), None if lse is None else lse.data_ptr(), ws.data_ptr(), need)
    return (out, lse) if return_lse else out
