"""Refusals of the attention-side calls: what needs no GPU.  Shapes, strides,
alignment and aliasing are checked on the host before any device work, so the
pointers here are never used."""
import ctypes
import os
import subprocess
import sys

import pytest
import torch

from runnel_b200 import _lib, attention

F = 1 << 20  # a 16-byte aligned address that is never used


def _err():
    return _lib.load().rnb_last_error().decode()


def _plan(**kw):
    a = dict(B=4, cols=8, page=16, pages=32, tokens=10, table=F, ctx=F + 64, new=F + 128, free=F + 192, cap=8,
             count=F + 256, seq=F + 320, cu=F + 384, pos=F + 448, slots=F + 512, out=F + 576)
    a.update(kw)
    return _lib.load().rnb_kv_plan(a["B"], a["cols"], a["page"], a["pages"], a["tokens"], a["table"], a["ctx"],
                                   a["new"], a["free"], a["cap"], a["count"], a["seq"], a["cu"], a["pos"], a["slots"],
                                   a["out"], None)


@pytest.mark.parametrize("kw,msg", [
    (dict(B=-1), "B must"), (dict(B=16385), "B must"), (dict(cols=0), "table_cols"), (dict(page=8), "page_size"),
    (dict(page=48), "page_size"), (dict(page=512), "page_size"), (dict(pages=0), "num_pages"),
    (dict(pages=1 << 27), "num_pages"), (dict(tokens=-1), "max_tokens"), (dict(cap=-1), "free_capacity"),
    (dict(table=None), "non-NULL"), (dict(slots=None), "non-NULL"), (dict(free=None), "non-NULL"),
    (dict(out=F + 256), "free_count_out"), (dict(seq=F + 64), "seq_lens"), (dict(seq=F + 128), "seq_lens"),
])
def test_plan_refuses(kw, msg):
    assert _plan(**kw) == -1 and msg in _err()


@pytest.mark.parametrize("kw,msg", [
    (dict(B=16385), "B must"), (dict(page=17), "page_size"), (dict(cap=-1), "free_capacity"),
    (dict(lens=None), "non-NULL"), (dict(out=F + 256), "free_count_out"),
])
def test_release_refuses(kw, msg):
    a = dict(B=4, cols=8, page=16, table=F, lens=F + 64, fin=F + 128, free=F + 192, cap=8, count=F + 256,
             lens_out=F + 64, out=F + 320)
    a.update(kw)
    rc = _lib.load().rnb_kv_release(a["B"], a["cols"], a["page"], a["table"], a["lens"], a["fin"], a["free"], a["cap"],
                                    a["count"], a["lens_out"], a["out"], None)
    assert rc == -1 and msg in _err()


def test_bounded_release_refuses():
    def call(cols=8, pages=32, fin=F + 128):
        return _lib.load().rnb_kv_release_bounded(4, cols, 16, pages, F, F + 64, fin, F + 192, 8, F + 256, F + 64, F + 320,
                                                  None)
    for kw, msg in ((dict(pages=0), "num_pages"), (dict(cols=0), "table_cols"), (dict(fin=None), "non-NULL")):
        assert call(**kw) == -1 and msg in _err()


def _kv(**kw):
    c = _lib.RnbKvCache(dtype=0, num_pages=16, page_size=16, n_kv_heads=2, head_dim=128, k=F, v=F,
                        k_page_stride=2 * 16 * 128, k_head_stride=16 * 128, v_page_stride=2 * 16 * 128,
                        v_head_stride=16 * 128)
    for k, v in kw.items():
        setattr(c, k, v)
    return c


BAD_CACHES = [
    (dict(dtype=2), -1, "dtype"), (dict(head_dim=96), -1, "head_dim"), (dict(page_size=12), -1, "page_size"),
    (dict(num_pages=0), -1, "num_pages"), (dict(num_pages=1 << 27), -1, "num_pages"), (dict(n_kv_heads=0), -1, "n_kv"),
    (dict(k=None), -1, "non-NULL"), (dict(v=F + 8), -2, "aligned"), (dict(k_head_stride=2044), -1, "strides"),
    (dict(v_page_stride=-8), -1, "strides"),
]


def _attn(cache=None, q=F, gate=None, table=F, seq=F, cu=None, out=F, ws=F, nbytes=1 << 30, **kw):
    d = _lib.RnbAttnDesc(B=4, T=4, n_q_heads=8, table_cols=8, max_q=1, window=0, scale=0.1, q_token_stride=8 * 128,
                         q_head_stride=128)
    for k, v in kw.items():
        setattr(d, k, v)
    cache = _kv() if cache is None else cache
    return _lib.load().rnb_paged_attention(ctypes.byref(d), ctypes.byref(cache), q, gate, table, seq, cu, out, None, ws,
                                           nbytes, None)


@pytest.mark.parametrize("kw,code,msg", BAD_CACHES)
def test_attention_refuses_caches(kw, code, msg):
    assert _attn(cache=_kv(**kw)) == code and msg in _err()


@pytest.mark.parametrize("kw,code,msg", [
    (dict(B=-1), -1, "B and T"), (dict(n_q_heads=7), -1, "n_q_heads"), (dict(n_q_heads=0), -1, "n_q_heads"),
    (dict(T=5), -1, "T == B"), (dict(table_cols=0), -1, "table_cols"), (dict(max_q=-1), -1, "max_q"),
    (dict(window=-1), -1, "window"), (dict(scale=0.0), -1, "scale"), (dict(scale=float("nan")), -1, "scale"),
    (dict(scale=float("inf")), -1, "scale"), (dict(q_head_stride=4), -1, "strides"),
    (dict(gate_token_stride=-8), -1, "strides"), (dict(B=1 << 29, T=1 << 29), -1, "2^31"), (dict(q=None), -1, "non-NULL"),
    (dict(seq=None), -1, "non-NULL"), (dict(q=F + 2), -2, "aligned"), (dict(gate=F + 8), -2, "aligned"),
])
def test_attention_refuses(kw, code, msg):
    assert _attn(**kw) == code and msg in _err()


@pytest.mark.parametrize("kw,msg", [
    (dict(q_token_stride=2048, q_head_stride=256), "packed"),  # out at the head of interleaved queries
    (dict(out=F + 4 * 2048 - 16), "packed"), (dict(out=F + 64), "packed"), (dict(q=F + 4 * 2048 - 16), "packed"),
    (dict(gate=F, q=F + 8192, gate_token_stride=1024, gate_head_stride=128), "gate"),
    (dict(gate=F + 8192 - 256, q=F + 32768, gate_token_stride=2048, gate_head_stride=128), "gate"),
])
def test_attention_refuses_outputs_over_its_inputs(kw, msg):
    assert _attn(**kw) == -1 and msg in _err()


@pytest.mark.skipif(torch.cuda.is_available(), reason="a CUDA device is present")
@pytest.mark.parametrize("kw", [
    dict(), dict(q=F + 8192), dict(out=F + 8192), dict(q_token_stride=2048, out=F + 16384),
    dict(T=1, B=1, q_token_stride=8),  # a stride over one token is never used
    dict(gate=F + 8192, gate_token_stride=1024, gate_head_stride=128),
    dict(q=F + 8192, q_token_stride=8192, T=1, B=1),
    dict(T=2, B=2, q=F + 1024, out=F + 4096, n_q_heads=4, q_token_stride=8192, q_head_stride=128),  # between two tokens
])
def test_attention_takes_outputs_beside_its_inputs(kw):
    """(what is refused here is the missing device)"""
    assert _attn(**kw) == -5


def test_attention_of_nothing_is_ok():
    assert _attn(B=0, T=0, q=None, out=None, table=None, seq=None, ws=None, nbytes=0) == 0


def test_attention_workspace_size():
    d = _lib.RnbAttnDesc(B=4, T=4, n_q_heads=8, table_cols=8, max_q=1, scale=0.1, q_token_stride=8 * 128,
                         q_head_stride=128)
    n = ctypes.c_size_t()
    lib = _lib.load()
    assert lib.rnb_paged_attention_workspace_size(ctypes.byref(d), ctypes.byref(_kv()), ctypes.byref(n)) == 0
    assert 0 < n.value < 64 << 20
    assert lib.rnb_paged_attention_workspace_size(ctypes.byref(d), ctypes.byref(_kv()), None) == -1


def _rope(cache=False, k=None, v=None, slots=None, q=F, out=F + 4096, pos=F, inv=F, qw=None, **kw):
    d = _lib.RnbRopeDesc(dtype=0, T=4, n_q_heads=8, n_kv_heads=2 if cache else 0, head_dim=128, rot=64, n_axes=1,
                         interleaved=0, eps=1e-6, q_token_stride=8 * 128, q_head_stride=128)
    sections = kw.pop("sections", (32,))
    for i, s in enumerate(sections):
        d.sections[i] = s
    for n, x in kw.items():
        setattr(d, n, x)
    c = None
    if cache is True:
        c = ctypes.byref(_kv())
    elif cache:
        c = ctypes.byref(cache)
    return _lib.load().rnb_rope_append(ctypes.byref(d), q, k, v, qw, None, pos, inv, slots, c, out, None)


@pytest.mark.parametrize("kw,code,msg", [
    (dict(dtype=3), -1, "dtype"), (dict(T=-1), -1, "T must"), (dict(head_dim=80), -1, "head_dim"),
    (dict(rot=24), -1, "rot"), (dict(rot=144), -1, "rot"), (dict(rot=0), -1, "rot"), (dict(n_axes=0), -1, "n_axes"),
    (dict(n_axes=5), -1, "n_axes"), (dict(sections=(31,)), -1, "sum"), (dict(n_axes=2, sections=(33, -1)), -1, ">= 0"),
    (dict(n_axes=3, sections=(10, 11, 11), interleaved=1), -1, "interleaved"), (dict(n_q_heads=0), -1, "n_q_heads"),
    (dict(q_token_stride=1020), -1, "strides"), (dict(k=F), -1, "together"), (dict(n_kv_heads=2), -1, "n_kv_heads"),
    (dict(cache=True, k=F, v=F, slots=F, n_kv_heads=4), -1, "match"),
    (dict(cache=True, k=F, v=F, slots=F, dtype=1), -1, "match"),
    (dict(cache=True, k=F + 8, v=F, slots=F), -2, "aligned"), (dict(q=None), -1, "non-NULL"),
    (dict(pos=None), -1, "non-NULL"), (dict(qw=F + 2), -2, "aligned"),
    (dict(out=F, q_token_stride=2048), -1, "packed"),
])
def test_rope_refuses(kw, code, msg):
    assert _rope(**kw) == code and msg in _err()


@pytest.mark.parametrize("kw,code,msg", BAD_CACHES)
def test_rope_refuses_caches(kw, code, msg):
    assert _rope(cache=_kv(**kw), k=F, v=F, slots=F) == code and msg in _err()


def test_status_refuses_null():
    assert _lib.load().rnb_kv_status(None, None) == -1


@pytest.mark.skipif(torch.cuda.is_available(), reason="a CUDA device is present")
def test_calls_without_device_fail_loudly():
    assert _plan() == -5
    assert _attn() != 0
    assert _rope() == -5


def test_python_refuses_cpu_tensors():
    i = torch.zeros(2, dtype=torch.int32)
    q = torch.zeros(2, 4, 64, dtype=torch.bfloat16)
    kc = torch.zeros(3, 2, 16, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        attention.kv_plan(i.view(2, 1), i, i, i, i[:1], page_size=16, num_pages=3, max_tokens=2)
    with pytest.raises(ValueError, match="CUDA"):
        attention.kv_release(i.view(2, 1), i, i, i, i[:1], page_size=16)
    with pytest.raises(ValueError, match="CUDA"):
        attention.paged_attention(q, kc, kc, i.view(2, 1), i)
    with pytest.raises(ValueError, match="CUDA"):
        attention.rope(q, i, torch.zeros(16))
    with pytest.raises(ValueError, match="slots"):
        attention.rope_append(q, q, q, i, torch.zeros(16), None, kc, kc)
    with pytest.raises(ValueError, match="CUDA"):
        attention.status("cpu")


def test_extension_module_is_rebuilt_for_another_torch():
    """It holds torch's inline code: a torch installed later makes it out of date."""
    here = os.path.dirname(os.path.abspath(_lib.__file__))
    version = os.path.join(os.path.dirname(torch.__file__), "version.py")
    cmd = ["make", "-n", "-C", os.path.join(here, "csrc"), f"PYTHON={sys.executable}", os.path.join(here, "_torch_calls.so")]
    assert "rnb_torch.cpp" in subprocess.run(cmd + ["-W", version], capture_output=True, text=True, check=True).stdout
