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
in a CUDA graph; each takes its scratch from torch's allocator.  Nothing falls
back to another implementation.

What goes wrong on the device (plans that do not fit, ids and lengths out of
range, a wait that gave up) shows in :func:`status` alone, so a server reads it every
so many steps.
"""
from __future__ import annotations

import ctypes
from typing import NamedTuple

import torch

from . import _lib

_calls = None  # the extension module (csrc/rnb_torch.cpp), bound to the loaded library


def _native():
    """The calls on torch tensors, bound once to the C functions of ``librnb_moe.so``."""
    global _calls
    if _calls is None:
        lib = _lib.load()
        try:
            from . import _torch_calls
        except ImportError as e:
            raise RuntimeError("runnel_b200/_torch_calls.so is missing or does not load: build it first (python -c "
                               "'import __graft_entry__ as g; g.build()' or make -C runnel_b200/csrc)") from e
        names = ("rnb_kv_plan", "rnb_kv_release_bounded", "rnb_rope_append", "rnb_paged_attention_workspace_size",
                 "rnb_paged_attention")
        _torch_calls.bind({n: ctypes.cast(getattr(lib, n), ctypes.c_void_p).value for n in names})
        _calls = _torch_calls
    return _calls


class KVPlan(NamedTuple):
    """What :func:`kv_plan` says of a step (parts of one int32 buffer)."""

    seq_lens: torch.Tensor  # [B] cached plus new tokens
    cu_q: torch.Tensor  # [B + 1] first new-token row of each request, then their number
    positions: torch.Tensor  # [max_tokens]
    slots: torch.Tensor  # [max_tokens], -1 behind the last request's rows
    free_count: torch.Tensor  # [1] pages left on the free list


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
    ``STATUS_NO_PAGES``; so it is where the free list's ids that it would take are
    not all in ``[0, num_pages)``, with ``STATUS_BAD_INDEX`` too.
    """
    return KVPlan(*(_calls or _native()).kv_plan(table, ctx_lens, new_lens, free_pages, free_count, page_size, num_pages,
                                                 max_tokens))


def kv_release(table: torch.Tensor, lens: torch.Tensor, finished: torch.Tensor, free_pages: torch.Tensor,
               free_count: torch.Tensor, *, page_size: int, num_pages: int | None = None
               ) -> tuple[torch.Tensor, torch.Tensor]:
    """Append the pages of requests with ``finished[b] != 0`` (int32) to
    ``free_pages[:free_count]``, in place; returns (lengths with theirs 0, the
    new count).  Does nothing, with ``STATUS_NO_PAGES``, if they do not fit.

    Negative table entries hold no page and are passed over: an entry before a
    request's window whose page was given away has to be negative by now.  Ids from
    ``num_pages`` on (None: any is a page) are left out too, with ``STATUS_BAD_INDEX``.
    """
    return (_calls or _native()).kv_release(table, lens, finished, free_pages, free_count, page_size, num_pages)


def status(device=None) -> int:
    """Status bits (``_lib.STATUS_*``) of this module's calls on a device, on any
    stream, since the last read; clears them and synchronises the current stream.
    One reader a device: it takes the bits of all callers."""
    dev = torch.device("cuda" if device is None else device)
    if dev.type != "cuda":
        raise ValueError("status is kept for CUDA devices")
    if dev.index is None:
        dev = torch.device("cuda", torch.cuda.current_device())
    out = ctypes.c_uint32()
    with torch.cuda.device(dev):
        _lib.call("rnb_kv_status", ctypes.byref(out), torch.cuda.current_stream(dev).cuda_stream)
    return out.value


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
    left alone, in ``out`` too; the other slots are distinct (of two tokens in one,
    either may stay).  ``out`` may be ``q`` if that is contiguous, but not share memory
    with ``q``, ``k`` or ``v`` otherwise.
    """
    if k_cache is None or slots is None:
        raise ValueError("rope_append needs a cache and slots; rope() turns queries without them")
    return (_calls or _native()).rope(q, k, v, positions, inv_freq, slots, k_cache, v_cache, sections, interleaved, q_norm,
                                      k_norm, eps, out)


def rope(q: torch.Tensor, positions: torch.Tensor, inv_freq: torch.Tensor, *, sections=None, interleaved: bool = False,
         norm: torch.Tensor | None = None, eps: float = 1e-6, out: torch.Tensor | None = None) -> torch.Tensor:
    """:func:`rope_append`'s norm and rotation of one tensor ``[T, heads, head_dim]``, without a cache."""
    return (_calls or _native()).rope(q, None, None, positions, inv_freq, None, None, None, sections, interleaved, norm,
                                      None, eps, out)


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
    behind ``cu_q[-1]`` are left as they were.  ``out`` may be ``q`` if that is contiguous,
    but not share memory with it otherwise, nor with ``gate``.  ``max_q``, a bound on the rows of one
    request, picks the kernels and is worth giving.

    Device waits are bounded: after one that gave up (a second), :func:`status` has
    ``STATUS_TIMEOUT`` and that call's outputs are void: the rest of its many-row requests
    are left unwritten (without ``out``, memory as it was allocated), and so they are
    where a graph replays the call, until the status is read.
    """
    return (_calls or _native()).paged_attention(q, k_cache, v_cache, table, seq_lens, cu_q, max_q, scale, window, gate, out,
                                                 return_lse)
