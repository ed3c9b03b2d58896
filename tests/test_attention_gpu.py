"""The attention-side operators on a B200 against 64-bit definitions: pages and
slots of a step, rotary append, paged attention, and a run of them together."""
import itertools
import random

import pytest
import torch

from runnel_b200 import _lib, attention
from tests import _attn_ref as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, FP16 = torch.bfloat16, torch.float16


def _i(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _rand(g, dtype, *shape, scale=1.0):
    return (torch.randn(shape, generator=g, device=DEV) * scale).to(dtype)


@pytest.fixture(autouse=True)
def _clean_status():
    attention.status()
    yield


# ------------------------------------------------------------------ plan

def _plan_ref(table, ctx, new, free, fc, P, max_tokens):
    """The plan by Python integers: (table, seq, cu, positions, slots, free count, ok)."""
    B, W = len(table), len(table[0]) if table else 0
    need = [-(-(c + n) // P) - -(-c // P) for c, n in zip(ctx, new)]
    ok = (min(ctx + new, default=0) >= 0 and sum(need) <= fc and sum(new) <= max_tokens
          and all(-(-(c + n) // P) <= W for c, n in zip(ctx, new)))
    table = [list(r) for r in table]
    if not ok:
        return table, list(ctx), [0] * (B + 1), [0] * max_tokens, [-1] * max_tokens, fc, False
    pos, slots, left = [], [], fc
    for b in range(B):
        for j in range(need[b]):
            left -= 1
            table[b][-(-ctx[b] // P) + j] = free[left]
        for p in range(ctx[b], ctx[b] + new[b]):
            pos.append(p)
            slots.append(table[b][p // P] * P + p % P)
    pad = max_tokens - len(pos)
    return (table, [c + n for c, n in zip(ctx, new)], [0, *itertools.accumulate(new)], pos + [0] * pad,
            slots + [-1] * pad, left, True)


def _check_plan(ctx, new, P, W, max_tokens, spare=3, short=0, seed=0):
    r = random.Random(seed)
    B = len(ctx)
    held = [-(-max(c, 0) // P) for c in ctx]
    need = sum(max(0, -(-(c + n) // P) - -(-c // P)) for c, n in zip(ctx, new))
    total = sum(held) + need + spare
    ids = list(range(total))
    r.shuffle(ids)
    table = [[-7] * W for _ in range(B)]
    for b in range(B):
        for j in range(min(held[b], W)):
            table[b][j] = ids.pop()
    free = list(ids)
    fc = need - short if short else len(free) - 1
    tt = _i(table).view(B, W)
    args = (tt, _i(ctx), _i(new), _i(free), _i([fc]))
    want = _plan_ref(table, ctx, new, free, fc, P, max_tokens)
    for _ in range(2):  # the same call gives the same answer again
        p = attention.kv_plan(*args, page_size=P, num_pages=max(total, 1), max_tokens=max_tokens)
        got = (tt.tolist(), p.seq_lens.tolist(), p.cu_q.tolist(), p.positions.tolist(), p.slots.tolist(),
               p.free_count.item())
        assert got == want[:6]
    assert args[4].item() == fc and args[3].tolist() == free
    assert attention.status() == (0 if want[6] else _lib.STATUS_NO_PAGES)
    assert attention.status() == 0


@pytest.mark.parametrize("ctx,new,P,W,cap", [
    ([0], [1], 16, 1, 1), ([0], [0], 16, 1, 0), ([15], [1], 16, 1, 4), ([16], [1], 16, 2, 1), ([0], [16], 16, 1, 16),
    ([0], [17], 16, 3, 20), ([5, 0, 31, 32], [0, 0, 0, 0], 32, 4, 3), ([5, 0, 31, 32], [1, 0, 1, 1], 32, 4, 3),
    ([0, 0, 300], [700, 0, 5], 256, 4, 900), ([7] * 257, [1] * 257, 64, 2, 300),
])
def test_plan_small(ctx, new, P, W, cap):
    _check_plan(ctx, new, P, W, cap)


@pytest.mark.parametrize("B,P,most_ctx,most_new", [(1, 16, 100000, 70000), (255, 16, 900, 40), (256, 128, 5000, 1),
                                                   (1000, 32, 2000, 90), (16384, 64, 100, 3)])
def test_plan_ragged(B, P, most_ctx, most_new):
    r = random.Random(B)
    ctx = [r.randint(0, most_ctx) for _ in range(B)]
    new = [r.randint(0, most_new) if r.random() < 0.8 else 0 for _ in range(B)]
    W = max(-(-(c + n) // P) for c, n in zip(ctx, new)) + 1
    _check_plan(ctx, new, P, W, sum(new) + 5, seed=B)


@pytest.mark.parametrize("B", [6000, 6016, 6017, 6126, 6127, 6144, 6145, 16384])
def test_plan_and_release_of_any_batch(B):
    """Batches around the border of the shared memory that a kernel has unasked."""
    r = random.Random(B)
    ctx, new = [r.randint(0, 40) for _ in range(B)], [r.randint(0, 2) for _ in range(B)]
    _check_plan(ctx, new, 16, 3, sum(new) + 1, seed=B)
    lens, fin = [r.randint(0, 32) for _ in range(B)], [int(r.random() < 0.3) for _ in range(B)]
    table = torch.arange(2 * B, dtype=torch.int32, device=DEV).view(B, 2)
    free = torch.full((2 * B,), -5, dtype=torch.int32, device=DEV)
    out, n = attention.kv_release(table, _i(lens), _i(fin), free, _i([0]), page_size=16)
    want = [2 * b + j for b in range(B) if fin[b] for j in range(-(-lens[b] // 16))]
    assert free.tolist() == want + [-5] * (2 * B - len(want)) and n.item() == len(want)
    assert out.tolist() == [0 if f else x for x, f in zip(lens, fin)]
    assert attention.status() == 0


@pytest.mark.parametrize("ctx,new,W,cap,short", [
    ([10, 0], [10, 40], 4, 50, 1),  # a page too few
    ([10, 0], [10, 40], 4, 49, 0),  # a token row too few
    ([10, 0], [10, 40], 2, 50, 0),  # a table column too few
    ([-1, 0], [10, 40], 4, 50, 0), ([10, 0], [-10, 40], 4, 50, 0),
])
def test_plan_is_all_or_nothing(ctx, new, W, cap, short):
    _check_plan(ctx, new, 16, W, cap, short=short)


def test_plan_of_huge_lengths_is_void():
    big = 2 ** 31 - 1
    t = torch.zeros(3, 2, dtype=torch.int32, device=DEV)
    p = attention.kv_plan(t, _i([big, 0, 5]), _i([1, big, 1]), _i([0, 1]), _i([2]), page_size=16, num_pages=4,
                          max_tokens=8)
    assert p.cu_q.tolist() == [0] * 4 and p.slots.tolist() == [-1] * 8 and p.free_count.item() == 2
    assert p.seq_lens.tolist() == [big, 0, 5]
    assert attention.status() == _lib.STATUS_NO_PAGES


def test_plan_refuses_a_bad_free_count_and_marks_bad_pages():
    t = _i([[99, 0]])
    for fc in (-1, 3):
        p = attention.kv_plan(t, _i([16]), _i([1]), _i([0, 1]), _i([fc]), page_size=16, num_pages=4, max_tokens=1)
        assert p.slots.tolist() == [-1] and attention.status() == _lib.STATUS_NO_PAGES
    p = attention.kv_plan(t, _i([3]), _i([1]), _i([0, 1]), _i([2]), page_size=16, num_pages=4, max_tokens=1)
    assert p.slots.tolist() == [-1] and p.positions.tolist() == [3]
    assert attention.status() == _lib.STATUS_BAD_INDEX


@pytest.mark.parametrize("need,at", [(2, 0), (2, 1), (700, 3), (700, 300), (700, 699), (5000, 4400), (5000, 4999)])
@pytest.mark.parametrize("bad", [-1, 5010])
def test_plan_that_would_take_a_bad_id_is_void(need, at, bad):
    """A free id that is no page voids the plan; behind what the step takes it does not matter."""
    free = list(range(need + 1))
    free[need - at] = bad
    t = torch.full((2, need + 2), 7, dtype=torch.int32, device=DEV)
    args = (_i([16, 5]), _i([16 * need, 1]), _i(free), _i([need + 1]))
    p = attention.kv_plan(t, *args, page_size=16, num_pages=5010, max_tokens=16 * need + 4)
    assert p.cu_q.tolist() == [0, 0, 0] and p.seq_lens.tolist() == [16, 5] and p.free_count.item() == need + 1
    assert (p.slots == -1).all() and (p.positions == 0).all() and (t == 7).all()
    assert attention.status() == _lib.STATUS_NO_PAGES | _lib.STATUS_BAD_INDEX
    free[need - at], free[0] = need - at, bad
    p = attention.kv_plan(t, args[0], args[1], _i(free), args[3], page_size=16, num_pages=5010, max_tokens=16 * need + 4)
    assert p.free_count.item() == 1 and t[0, 1:need + 1].tolist() == free[:0:-1]
    assert attention.status() == 0


def test_plan_of_almost_2_to_31_rows():
    """The rows behind the last request are filled to the end, and nothing else is."""
    n = 2 ** 31 - 1
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 17 GB for positions and slots")
    t = torch.zeros(2, 3, dtype=torch.int32, device=DEV)
    p = attention.kv_plan(t, _i([0, 5]), _i([17, 1]), _i([4, 3, 2]), _i([3]), page_size=16, num_pages=8, max_tokens=n)
    assert p.slots[:20].tolist() == [*range(32, 48), 48, 5, -1, -1] and p.slots.numel() == n
    assert p.positions[:20].tolist() == [*range(17), 5, 0, 0]
    for i in range(18, n, 1 << 28):
        assert (p.slots[i:i + (1 << 28)] == -1).all() and not p.positions[i:i + (1 << 28)].any()
    assert p.cu_q.tolist() == [0, 17, 18] and p.free_count.item() == 1 and attention.status() == 0


def test_plan_of_no_requests():
    e = torch.zeros(0, dtype=torch.int32, device=DEV)
    p = attention.kv_plan(e.view(0, 3), e, e, _i([4, 5]), _i([2]), page_size=16, num_pages=6, max_tokens=3)
    assert p.cu_q.tolist() == [0] and p.slots.tolist() == [-1] * 3 and p.free_count.item() == 2
    assert attention.status() == 0


def test_release_returns_pages_in_order():
    P, table = 16, [[3, 4, 5], [6, 7, -1], [8, -1, -1], [-9, -9, -9]]
    free = _i([0, 1, 2, -1, -1, -1, -1, -1])
    lens, n = attention.kv_release(_i(table), _i([33, 32, 1, 0]), _i([1, 0, 1, 1]), free, _i([3]), page_size=P)
    assert lens.tolist() == [0, 32, 0, 0] and n.item() == 7
    assert free.tolist() == [0, 1, 2, 3, 4, 5, 8, -1]
    free = _i([0, 1, 2, -1])
    lens, n = attention.kv_release(_i(table), _i([33, 32, 1, 0]), _i([1, 0, 1, 1]), free, _i([3]), page_size=P)
    assert lens.tolist() == [33, 32, 1, 0] and n.item() == 3 and free.tolist() == [0, 1, 2, -1]
    assert attention.status() == _lib.STATUS_NO_PAGES


def test_release_passes_over_entries_without_a_page():
    """Entries given away before a window, and ids beyond the cache, do not come back as free pages."""
    table, lens, fin = _i([[-1, -1, 3], [6, 7, 8], [4, 12, 5]]), _i([48, 33, 40]), _i([1, 0, 1])
    free = _i([9, -1, -1, -1, -1])
    out, n = attention.kv_release(table, lens, fin, free, _i([1]), page_size=16, num_pages=12)
    assert free.tolist() == [9, 3, 4, 5, -1] and n.item() == 4 and out.tolist() == [0, 33, 0]
    assert attention.status() == _lib.STATUS_BAD_INDEX
    p = attention.kv_plan(table, out, _i([20, 0, 17]), free, n, page_size=16, num_pages=12, max_tokens=37)
    assert table.tolist() == [[5, 4, 3], [6, 7, 8], [3, 9, 5]] and p.free_count.item() == 0
    assert attention.status() == 0
    # without num_pages every id from 0 on is a page
    free = _i([9, -1, -1, -1, -1])
    attention.kv_release(_i([[-1, 12, -2 ** 31]]), _i([48]), _i([1]), free, _i([1]), page_size=16)
    assert free.tolist() == [9, 12, -1, -1, -1] and attention.status() == 0


@pytest.mark.parametrize("B,W", [(1, 1), (1, 300), (7, 100), (300, 9), (2, 5000)])
@pytest.mark.parametrize("gone", [0.0, 0.3, 1.0])
def test_release_of_any_length(B, W, gone):
    """The free list is just long enough, and one too short."""
    r = random.Random(B * W)
    lens = [r.choice([0, 1, 16 * W, r.randint(0, 16 * W)]) for _ in range(B)]
    lens[0], fin = 16 * W, [1] + [int(r.random() < 0.7) for _ in range(B - 1)]
    table = [[r.choice([-1, -9]) if r.random() < gone else b * W + j for j in range(W)] for b in range(B)]
    back = [e for b in range(B) if fin[b] for e in table[b][:-(-lens[b] // 16)] if e >= 0]
    t, ln, fn = _i(table).view(B, W), _i(lens), _i(fin)
    free = torch.full((2 + len(back),), -7, dtype=torch.int32, device=DEV)
    out, n = attention.kv_release(t, ln, fn, free, _i([2]), page_size=16, num_pages=B * W)
    assert free.tolist() == [-7, -7] + back and n.item() == 2 + len(back)
    assert out.tolist() == [0 if f else x for x, f in zip(lens, fin)] and attention.status() == 0
    if back:
        free = torch.full((1 + len(back),), -7, dtype=torch.int32, device=DEV)
        out, n = attention.kv_release(t, ln, fn, free, _i([2]), page_size=16, num_pages=B * W)
        assert (free == -7).all() and n.item() == 2 and torch.equal(out, ln)
        assert attention.status() == _lib.STATUS_NO_PAGES


# ------------------------------------------------------------------ rotary

def _sections(n, axes):
    w = n // axes
    rest = [w] * (axes - 1)
    return (n - sum(rest), *rest)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("T,Hq,Hkv,D,rot,axes,inter,norm,P", [
    (1, 16, 2, 256, 64, 3, True, True, 64), (3, 1, 1, 64, 64, 1, False, False, 16),
    (37, 5, 5, 64, 32, 3, True, True, 32), (8, 16, 2, 256, 256, 3, False, True, 128),
    (129, 28, 4, 128, 128, 3, True, False, 16), (1000, 12, 1, 128, 96, 2, True, True, 256),
    (2311, 8, 2, 256, 16, 4, True, False, 16), (65, 7, 1, 64, 48, 4, False, True, 64),
    (5000, 16, 2, 256, 64, 3, True, True, 64),
])
def test_rope_append(dtype, T, Hq, Hkv, D, rot, axes, inter, norm, P):
    g = _gen(T + D)
    qkv = _rand(g, dtype, T, Hq + 2 * Hkv, D)
    q, k, v = qkv.split([Hq, Hkv, Hkv], 1)
    n = rot // 2
    inv = (1e6 ** (-torch.arange(n, device=DEV, dtype=torch.float64) / n)).float()
    pos = torch.randint(0, 2 ** 20, (axes, T), generator=g, device=DEV).to(torch.int32)
    N = -(-T // P) + 2
    kc, vc = _rand(g, dtype, N, Hkv, P, D), _rand(g, dtype, N, Hkv, P, D)
    k0, v0 = kc.clone(), vc.clone()
    slots = torch.randperm(N * P, generator=g, device=DEV)[:T].to(torch.int32)
    if T > 2:
        slots[1] = -1  # a row that is left alone
    qw, kw = (1 + _rand(g, dtype, D, scale=0.2), 1 + _rand(g, dtype, D, scale=0.2)) if norm else (None, None)
    sec = _sections(n, axes)
    out = _rand(g, dtype, T, Hq, D)
    out0 = out.clone()
    attention.rope_append(q, k, v, pos, inv, slots, kc, vc, sections=sec, interleaved=inter, q_norm=qw, k_norm=kw,
                          out=out)
    live = slots >= 0
    want, tol = ref.rope(q, pos, inv, sec, inter, qw)
    ref.close(out[live], want[live], tol[live], "q")
    assert torch.equal(out[~live], out0[~live])
    s = slots[live].long()
    want, tol = ref.rope(k, pos, inv, sec, inter, kw)
    flat = kc.transpose(1, 2).reshape(N * P, Hkv, D)
    ref.close(flat[s], want[live], tol[live], "k")
    assert torch.equal(vc.transpose(1, 2).reshape(N * P, Hkv, D)[s], v[live])
    others = torch.ones(N * P, dtype=torch.bool, device=DEV)
    others[s] = False
    assert torch.equal(flat[others], k0.transpose(1, 2).reshape(N * P, Hkv, D)[others])
    assert torch.equal(vc.transpose(1, 2).reshape(N * P, Hkv, D)[others], v0.transpose(1, 2).reshape(N * P, Hkv, D)[others])
    assert attention.status() == 0


def test_rope_of_text_positions_and_in_place():
    g = _gen(3)
    x = _rand(g, BF16, 50, 6, 128)
    inv = torch.rand(32, generator=g, device=DEV) + 0.01
    pos = torch.arange(50, device=DEV) + 777  # int64 is taken too
    a = attention.rope(x, pos, inv)
    b = attention.rope(x, pos.to(torch.int32), inv, sections=(12, 10, 10), interleaved=True)
    assert torch.equal(a, b)
    want, tol = ref.rope(x, pos[None], inv, (32,), False)
    ref.close(a, want, tol)
    assert torch.equal(attention.rope(x, pos, inv, out=x), a) and torch.equal(x, a)
    assert attention.rope(x[:0], pos[:0], inv).shape == (0, 6, 128)


def test_rope_outputs_over_inputs_are_refused():
    g = _gen(34)
    T, D = 4, 64
    buf = _rand(g, BF16, 2 * T * 16 * D)
    joint = buf[:T * 12 * D].view(T, 12, D)  # eight query heads, two key, two value heads
    q, k, v = joint.split([8, 2, 2], 1)
    kc, vc = _rand(g, BF16, 2, 2, 16, D), _rand(g, BF16, 2, 2, 16, D)
    inv, pos, slots = torch.rand(32, generator=g, device=DEV), _i([0, 1, 2, 3]), _i([3, 20, 1, 0])
    n, packed = T * 8 * D, _rand(g, BF16, T, 8, D)
    was = buf.clone(), kc.clone(), vc.clone()
    apart = [x.contiguous() for x in (q, k, v)]
    over = lambda at: buf[at:at + n].view(T, 8, D)  # noqa: E731
    for qq, kk, vv, out in ((q, apart[1], apart[2], over(0)), (packed, k, apart[2], over(8 * D + 64)),
                            (packed, apart[1], v, over(T * 12 * D - 64)), (buf[64:64 + n].view(T, 8, D), *apart[1:], over(0))):
        with pytest.raises(_lib.RnbError, match="share memory|packed"):
            attention.rope_append(qq, kk, vv, pos, inv, slots, kc, vc, out=out)
    with pytest.raises(_lib.RnbError, match="share memory|packed"):
        attention.rope(q, pos, inv, out=over(0))
    assert all(torch.equal(a, b) for a, b in zip((buf, kc, vc), was))
    want = attention.rope_append(*apart, pos, inv, slots, kc, vc)
    assert torch.equal(attention.rope_append(q, k, v, pos, inv, slots, kc, vc, out=over(T * 12 * D)), want)
    # two tokens of heads 0-7, and their outputs between the joint rows of a wider buffer
    wide = _rand(g, BF16, 2, 3 * 8 * D)
    qw = wide[:, :8 * D].view(2, 8, D)
    want = attention.rope(qw.contiguous(), pos[:2], inv)
    out = wide.view(-1)[8 * D:24 * D].view(2, 8, D)
    assert torch.equal(attention.rope(qw, pos[:2], inv, out=out), want)


def test_rope_slot_beyond_the_cache_and_negative_positions():
    g = _gen(4)
    q, k, v = (_rand(g, FP16, 3, 2, 64) for _ in range(3))
    kc, vc = _rand(g, FP16, 2, 2, 16, 64), _rand(g, FP16, 2, 2, 16, 64)
    k0 = kc.clone()
    inv = torch.rand(32, generator=g, device=DEV)
    pos = _i([-5, 2 ** 31 - 1, -2 ** 31])
    out = attention.rope_append(q, k, v, pos, inv, _i([32, 2 ** 31 - 1, 31]), kc, vc)
    want, tol = ref.rope(q, pos[None], inv, (32,), False)
    ref.close(out, want, tol)
    k0[1, :, 15] = kc[1, :, 15]
    assert torch.equal(kc, k0)
    assert attention.status() == _lib.STATUS_BAD_INDEX


def test_rope_far_cache_offsets():
    """Pages whose element offsets pass 2^31 (a cache of 4.5 GB a tensor)."""
    g = _gen(5)
    N, H, P, D = 17200, 8, 64, 256
    kc, vc = torch.empty(N, H, P, D, dtype=BF16, device=DEV), torch.empty(N, H, P, D, dtype=BF16, device=DEV)
    q, k, v = (_rand(g, BF16, 4, 8, D) for _ in range(3))
    slots = _i([N * P - 1, (N - 1) * P, 17000 * P + 5, 3])
    inv = torch.rand(32, generator=g, device=DEV)
    attention.rope_append(q, k, v, _i([1, 2, 3, 4]), inv, slots, kc, vc)
    want, tol = ref.rope(k, _i([[1, 2, 3, 4]]), inv, (32,), False)
    for t, s in enumerate(slots.tolist()):
        ref.close(kc[s // P, :, s % P], want[t], tol[t])
        assert torch.equal(vc[s // P, :, s % P], v[t])
    # and attention reads them
    table = _i([[N - 1], [17000]])
    kc[[N - 1, 17000]] = _rand(g, BF16, 2, H, P, D)
    vc[[N - 1, 17000]] = _rand(g, BF16, 2, H, P, D)
    _check_attention(q[:2], kc, vc, table, [64, 6], [1, 1])


# ------------------------------------------------------------------ attention

def _cache_of(g, dtype, lens, Hkv, D, P, extra_cols=1, combined=False):
    """A cache of scattered pages for these lengths; NaN everywhere behind a
    length, in unused pages too, and ids far out of range in unused columns."""
    held = [-(-n // P) for n in lens]
    N = sum(held) + 3
    if combined:  # keys and values of a page side by side: page strides of both
        both = _rand(g, dtype, N, 2, Hkv, P, D)
        kc, vc = both[:, 0], both[:, 1]
    else:
        kc, vc = _rand(g, dtype, N, Hkv, P, D), _rand(g, dtype, N, Hkv, P, D)
    ids = torch.randperm(N, generator=g, device=DEV).tolist()
    W = max(held, default=0) + extra_cols
    table = [[2 ** 30] * W for _ in lens]
    for b, n in enumerate(lens):
        for j in range(held[b]):
            table[b][j] = ids.pop()
        if n % P:
            for c in (kc, vc):
                c[table[b][held[b] - 1], :, n % P:] = float("nan")
    for i in ids:
        kc[i] = float("nan")
        vc[i] = float("inf")
    return kc, vc, _i(table).view(len(lens), W)


def _check_attention(q, kc, vc, table, lens, rows, max_q=None, cu=None, gate=None, keep=None, **kw):
    want, wlse, tol, ltol = ref.attention(q, kc, vc, table, lens, rows, gate=gate, keep=keep, **kw)
    if cu is None and any(r != 1 for r in rows):
        cu = _i([0, *itertools.accumulate(rows)])
    first = None
    for _ in range(2):  # equal inputs, equal bits
        out, lse = attention.paged_attention(q, kc, vc, table, _i(lens), cu_q=cu, max_q=max_q, gate=gate,
                                             return_lse=True, **kw)
        if first is not None:
            assert torch.equal(out, first[0]) and torch.equal(lse, first[1])
        first = (out, lse)
    n = sum(rows)
    ref.close(out[:n], want[:n], tol[:n], "out")
    ref.close(lse[:n], wlse[:n], ltol[:n], "lse")
    return out, lse


HEADS = [(16, 2, 256), (1, 1, 256), (24, 2, 256), (32, 8, 128), (28, 4, 128), (12, 1, 128), (40, 2, 128), (8, 8, 64),
         (14, 2, 64), (64, 2, 64)]


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("Hq,Hkv,D", HEADS)
def test_one_token_each(dtype, Hq, Hkv, D):
    """Lengths around every boundary: none, one, subtile, page, unit, split."""
    g = _gen(Hq * D)
    for P, lens in ((16, [0, 1, 15, 16, 17, 63, 64, 65, 127, 130, 1000]), (64, [64, 0, 63, 700, 1]), (256, [513]),
                    (32, [4099, 31])):
        kc, vc, table = _cache_of(g, dtype, lens, Hkv, D, P)
        q = _rand(g, dtype, len(lens), Hq, D, scale=1.5)
        out, lse = _check_attention(q, kc, vc, table, lens, [1] * len(lens))
        for b, n in enumerate(lens):
            if n == 0:
                assert not out[b].any() and torch.isneginf(lse[b]).all()
    assert attention.status() == 0


@pytest.mark.parametrize("Hq,Hkv,D", HEADS)
@pytest.mark.parametrize("B", [1, 7, 700])
def test_one_token_each_over_short_tables(Hq, Hkv, D, B):
    """Tables short enough that whole tiles are dealt by number, up to more tiles than CTAs."""
    g = _gen(B + D)
    r = random.Random(B)
    lens = [r.choice([0, 1, 16, 17, 63, 64, 100, 127]) for _ in range(B)]
    lens[0] = 127
    kc, vc, table = _cache_of(g, BF16, lens, Hkv, D, 16)
    q = _rand(g, BF16, B, Hq, D, scale=1.5)
    gate = _rand(g, BF16, B, Hq, D)
    few = min(B, 40)  # the rows that are checked
    want, wlse, tol, ltol = ref.attention(q[-few:], kc, vc, table[-few:], lens[-few:], [1] * few, gate=gate[-few:], window=70)
    out, lse = attention.paged_attention(q, kc, vc, table, _i(lens), gate=gate, window=70, return_lse=True)
    ref.close(out[-few:], want, tol, "out")
    ref.close(lse[-few:], wlse, ltol, "lse")
    long = torch.cat([table, torch.full((B, 64), 2 ** 30, dtype=torch.int32, device=DEV)], 1)
    alike, _ = attention.paged_attention(q, kc, vc, long, _i(lens), gate=gate, window=70, return_lse=True)
    ref.close(alike[-few:], want, tol, "the same over a long table")
    assert attention.status() == 0


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("Hq,Hkv,D", HEADS)
@pytest.mark.parametrize("max_q", [None, 5])
def test_few_tokens_each(dtype, Hq, Hkv, D, max_q):
    g = _gen(Hq + D)
    lens, rows = [5, 0, 64, 3, 700, 2, 130, 1], [5, 0, 4, 1, 3, 5, 0, 1]  # a request with more rows than positions
    kc, vc, table = _cache_of(g, dtype, lens, Hkv, D, 16)
    q = _rand(g, dtype, sum(rows), Hq, D)
    gate = _rand(g, dtype, sum(rows), Hq, D, scale=3.0)
    _check_attention(q, kc, vc, table, lens, rows, max_q=max_q, gate=gate)


@pytest.mark.parametrize("Hq,Hkv,D", [(16, 2, 256), (32, 8, 128), (14, 2, 64), (6, 6, 128)])
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_prompts(Hq, Hkv, D, dtype):
    g = _gen(D)
    lens, rows = [300, 129, 1, 513, 40, 260], [300, 65, 1, 200, 0, 1]
    kc, vc, table = _cache_of(g, dtype, lens, Hkv, D, 16 if D == 128 else 64)
    q = _rand(g, dtype, sum(rows), Hq, D)
    gate = _rand(g, dtype, sum(rows), Hq, D)
    _check_attention(q, kc, vc, table, lens, rows, max_q=300)
    _check_attention(q, kc, vc, table, lens, rows, gate=gate)


@pytest.mark.parametrize("B,active", [(33, 2), (300, 3), (3000, 5), (3000, 900)])
@pytest.mark.parametrize("max_q", [1, 3])
def test_idle_places_between_requests(B, active, max_q):
    """A large batch with few requests at work, anywhere in it; the others have lengths but no rows, or nothing."""
    g, r = _gen(B + active), random.Random(B * active)
    rows, lens = [0] * B, [r.choice([0, 0, 40]) for _ in range(B)]
    for b in [0, B - 1] + r.sample(range(1, B - 1), active - 2):
        rows[b], lens[b] = r.randint(1, max_q), r.choice([1, 65, 300, 900])
    kc, vc, table = _cache_of(g, BF16, lens, 2, 64, 16)
    T = sum(rows)
    q = _rand(g, BF16, T, 14, 64)
    cu = _i([0, *itertools.accumulate(rows)])
    out, lse = attention.paged_attention(q, kc, vc, table, _i(lens), cu_q=cu, max_q=max_q, return_lse=True)
    few = [b for b in range(B) if rows[b]][:40]
    n = sum(rows[b] for b in few)
    want, wlse, tol, ltol = ref.attention(q[:n], kc, vc, table[few], [lens[b] for b in few], [rows[b] for b in few])
    ref.close(out[:n], want, tol, "out")
    ref.close(lse[:n], wlse, ltol, "lse")
    last = [b for b in range(B) if rows[b]][-5:]
    m = sum(rows[b] for b in last)
    want, _, tol, _ = ref.attention(q[T - m:], kc, vc, table[last], [lens[b] for b in last], [rows[b] for b in last])
    ref.close(out[T - m:], want, tol, "the last requests")
    assert attention.status() == 0


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("Hq,Hkv,D,lens,rows", [
    (12, 1, 128, [9000, 300, 4097, 1], [7, 7, 6, 1]), (16, 2, 256, [5000], [40]), (40, 2, 64, [3001, 2500], [9, 200]),
    (12, 1, 256, [2000, 0, 1500], [20, 0, 7]), (100, 1, 128, [1300, 700], [1, 3]),
])
def test_few_tiles_over_long_caches(dtype, Hq, Hkv, D, lens, rows):
    """Tiles whose positions are split over CTAs and joined, single rows among them, windows and gates too."""
    g = _gen(sum(lens))
    kc, vc, table = _cache_of(g, dtype, lens, Hkv, D, 16 if D == 64 else 64)
    q = _rand(g, dtype, sum(rows), Hq, D, scale=1.5)
    gate = _rand(g, dtype, sum(rows), Hq, D)
    _check_attention(q, kc, vc, table, lens, rows, max_q=max(rows), cu=_i([0, *itertools.accumulate(rows)]))
    _check_attention(q, kc, vc, table, lens, rows, cu=_i([0, *itertools.accumulate(rows)]), gate=gate)
    _check_attention(q, kc, vc, table, lens, rows, cu=_i([0, *itertools.accumulate(rows)]), gate=gate, window=1000)
    assert attention.status() == 0


@pytest.mark.parametrize("n,r", [(1, 1), (70, 1), (300, 3), (40, 64), (257, 200), (0, 5), (130, 0)])
@pytest.mark.parametrize("Hq,Hkv,D", [(16, 2, 256), (7, 1, 128), (64, 1, 64), (200, 1, 64)])
def test_a_single_request_of_any_rows(n, r, Hq, Hkv, D):
    """One request, its rows known to the device alone; padding behind them stays."""
    g = _gen(n + r)
    kc, vc, table = _cache_of(g, BF16, [n], Hkv, D, 16)
    q = _rand(g, BF16, r + 70, Hq, D)
    gate = _rand(g, BF16, r + 70, Hq, D)
    for window in (0, 33):
        out = torch.full_like(q, 9.0)
        got, lse = attention.paged_attention(q, kc, vc, table, _i([n]), cu_q=_i([0, r]), gate=gate, window=window,
                                             out=out, return_lse=True)
        want, wlse, tol, ltol = ref.attention(q[:r], kc, vc, table, [n], [r], gate=gate[:r], window=window)
        ref.close(out[:r], want, tol, "out")
        ref.close(lse[:r], wlse, ltol, "lse")
        assert got is out and (out[r:] == 9).all()
    assert attention.status() == 0


@pytest.mark.parametrize("window", [1, 7, 16, 64, 100, 1000])
@pytest.mark.parametrize("rows", [[1, 1, 1, 1], [3, 1, 150, 70]])
def test_windows(window, rows):
    g = _gen(window)
    lens = [700, 5, 600, 70]
    for Hq, Hkv, D in ((16, 2, 256), (8, 8, 64), (32, 8, 128)):
        kc, vc, table = _cache_of(g, BF16, lens, Hkv, D, 32)
        q = _rand(g, BF16, sum(rows), Hq, D)
        _check_attention(q, kc, vc, table, lens, rows, window=window)


def test_single_rows_ignore_any_bits_before_their_window():
    g = _gen(8)
    kc, vc, table = _cache_of(g, FP16, [300], 2, 64, 16)
    q = _rand(g, FP16, 1, 4, 64)
    want = attention.paged_attention(q, kc, vc, table, _i([300]), window=37)
    for j in range(300 - 37):
        kc[table[0, j // 16], :, j % 16] = float("nan")
        vc[table[0, j // 16], :, j % 16] = float("inf")
    assert torch.equal(attention.paged_attention(q, kc, vc, table, _i([300]), window=37), want)


@pytest.mark.parametrize("lens,rows", [([300, 70, 9000], [1, 1, 1]), ([300, 70, 9000], [3, 2, 4]),
                                       ([300, 150, 700], [1, 150, 130]), ([5000], [70])])
@pytest.mark.parametrize("Hq,Hkv,D", [(16, 2, 256), (28, 4, 128), (4, 4, 64)])
def test_outputs_in_place(lens, rows, Hq, Hkv, D):
    g = _gen(31)
    kc, vc, table = _cache_of(g, BF16, lens, Hkv, D, 16)
    q, gate = _rand(g, BF16, sum(rows), Hq, D), _rand(g, BF16, sum(rows), Hq, D)
    cu = None if rows == [1] * len(rows) else _i([0, *itertools.accumulate(rows)])
    for gt in (None, gate):
        args = dict(cu_q=cu, max_q=max(rows))
        want = attention.paged_attention(q, kc, vc, table, _i(lens), gate=gt, **args)
        for _ in range(5):
            x = q.clone()
            assert attention.paged_attention(x, kc, vc, table, _i(lens), gate=gt, out=x, **args) is x
            assert torch.equal(x, want)
    assert attention.status() == 0


@pytest.mark.parametrize("rows", [1, 3, 80])
@pytest.mark.parametrize("D,Hq,Hkv,P", [(256, 16, 2, 16), (128, 32, 8, 64), (64, 4, 4, 32), (128, 4, 4, 256)])
@pytest.mark.parametrize("window", [1, 37, 200])
def test_positions_before_every_window_hold_any_bits(rows, D, Hq, Hkv, P, window):
    """What no row of a request sees never counts, and its pages may be another's, or gone."""
    g, n = _gen(8), 700
    kc, vc, table = _cache_of(g, BF16, [n, 20], Hkv, D, P)
    q = _rand(g, BF16, rows + 1, Hq, D)
    args = dict(cu_q=_i([0, rows, rows + 1]), max_q=rows, window=window, return_lse=True)
    want = attention.paged_attention(q, kc, vc, table, _i([n, 20]), **args)
    before = n - rows - window + 1
    for j in range(before):
        kc[table[0, j // P], :, j % P] = float("nan")
        vc[table[0, j // P], :, j % P] = float("inf")
    table[0, : before // P] = -1
    assert attention.status() == 0
    got = attention.paged_attention(q, kc, vc, table, _i([n, 20]), **args)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert attention.status() == 0


@pytest.mark.parametrize("D,Hq,Hkv", [(256, 16, 2), (128, 32, 8), (64, 4, 4)])
def test_large_scores_and_scales(D, Hq, Hkv):
    """Peaked softmax, its maximum late, and a scale that is not the default."""
    g = _gen(9)
    lens, rows = [900, 333, 70], [1, 90, 2]
    kc, vc, table = _cache_of(g, BF16, lens, Hkv, D, 64)
    q = _rand(g, BF16, sum(rows), Hq, D, scale=8.0)
    _check_attention(q, kc, vc, table, lens, rows, scale=0.5)
    _check_attention(q, kc, vc, table, lens, rows, scale=1e-3)


def test_strided_queries_gates_and_caches():
    """q and gate interleaved per head as one projection gives them; keys and values of a page side by side."""
    g = _gen(10)
    lens, rows = [200, 64, 500], [70, 1, 2]
    for dtype, Hq, Hkv, D in ((BF16, 16, 2, 256), (FP16, 8, 2, 128), (BF16, 4, 1, 64)):
        kc, vc, table = _cache_of(g, dtype, lens, Hkv, D, 32, combined=True)
        qg = _rand(g, dtype, sum(rows), Hq, 2 * D)
        q, gate = qg[..., :D], qg[..., D:]
        a, _ = _check_attention(q, kc, vc, table, lens, rows, gate=gate)
        b = attention.paged_attention(q.contiguous(), kc.contiguous(), vc.contiguous(), table, _i(lens),
                                      cu_q=_i([0, 70, 71, 73]), gate=gate.contiguous())
        assert torch.equal(a, b)
        odd = torch.zeros(sum(rows), Hq, D + 1, dtype=dtype, device=DEV)[..., 1:]  # not 16-byte aligned: copied
        odd.copy_(q)
        assert torch.equal(attention.paged_attention(odd, kc, vc, table, _i(lens), cu_q=_i([0, 70, 71, 73]),
                                                     gate=gate), a)


def test_outputs_over_strided_queries_are_refused():
    """The query part of a joint projection is not packed: out may not lie there."""
    g = _gen(33)
    kc, vc, table = _cache_of(g, BF16, [50, 60, 70], 2, 64, 16)
    buf = _rand(g, BF16, 3 * 8 * 64 * 3)
    joint = buf[:3 * 8 * 128].view(3, 8, 128)
    was, sl = buf.clone(), _i([50, 60, 70])
    out = buf[:3 * 8 * 64].view(3, 8, 64)
    with pytest.raises(_lib.RnbError, match="packed"):
        attention.paged_attention(joint[..., :64], kc, vc, table, sl, out=out)
    with pytest.raises(_lib.RnbError, match="gate"):
        attention.paged_attention(joint[..., :64].contiguous(), kc, vc, table, sl, gate=joint[..., 64:], out=out)
    assert torch.equal(buf, was)
    behind = buf[3 * 8 * 128:].view(3, 8, 64)
    want = attention.paged_attention(joint[..., :64], kc, vc, table, sl, gate=joint[..., 64:])
    assert torch.equal(attention.paged_attention(joint[..., :64], kc, vc, table, sl, gate=joint[..., 64:], out=behind), want)
    assert attention.status() == 0


def test_rows_behind_the_last_request_stay():
    g = _gen(11)
    lens, rows = [100, 200], [3, 80]
    kc, vc, table = _cache_of(g, BF16, lens, 2, 128, 16)
    q = _rand(g, BF16, 120, 8, 128)
    q[83:] = float("nan")
    out = _rand(g, BF16, 120, 8, 128)
    was = out.clone()
    got = attention.paged_attention(q, kc, vc, table, _i(lens), cu_q=_i([0, 3, 83]), max_q=80, out=out)
    assert got is out and torch.equal(out[83:], was[83:]) and not torch.equal(out[:83], was[:83])


def test_bad_pages_and_lengths_are_left_out_and_told():
    g = _gen(12)
    for rows in ([1, 1], [70, 2]):
        lens = [200, 90]
        kc, vc, table = _cache_of(g, BF16, lens, 2, 128, 16, extra_cols=0)
        cu = None if rows == [1, 1] else _i([0, 70, 72])
        q = _rand(g, BF16, sum(rows), 8, 128)
        bad = table.clone()
        bad[0, 3], bad[0, 7], bad[1, 0] = -1, kc.shape[0], 2 ** 31 - 1
        keep = {0: torch.ones(200, dtype=torch.bool, device=DEV), 1: torch.ones(90, dtype=torch.bool, device=DEV)}
        keep[0][48:64] = False
        keep[0][112:128] = False
        keep[1][:16] = False
        want, wlse, tol, ltol = ref.attention(q, kc, vc, table, lens, rows, keep=keep.get)
        out, lse = attention.paged_attention(q, kc, vc, bad, _i(lens), cu_q=cu, return_lse=True)
        ref.close(out, want, tol)
        ref.close(lse, wlse, ltol)
        assert attention.status() == _lib.STATUS_BAD_INDEX
        # a length beyond the table is cut to it; a negative one is none
        W = table.shape[1] * 16
        full = torch.zeros_like(table)
        out = attention.paged_attention(q, kc[:1].nan_to_num(0.5), vc[:1].nan_to_num(0.5), full, _i([W + 1, -3]), cu_q=cu)
        ok = attention.paged_attention(q, kc[:1].nan_to_num(0.5), vc[:1].nan_to_num(0.5), full, _i([W, 0]), cu_q=cu)
        assert torch.equal(out, ok) and attention.status() == _lib.STATUS_BAD_INDEX


def test_bad_row_bounds_stay_inside():
    g = _gen(13)
    kc, vc, table = _cache_of(g, BF16, [50, 60], 2, 64, 16)
    q = _rand(g, BF16, 6, 4, 64)
    out = attention.paged_attention(q, kc, vc, table, _i([50, 60]), cu_q=_i([-5, 4, 100]))
    want, _, tol, _ = ref.attention(q, kc, vc, table, [50, 60], [4, 2])
    ref.close(out, want, tol)
    out = torch.zeros_like(q)
    attention.paged_attention(q, kc, vc, table, _i([50, 60]), cu_q=_i([6, 2, 1]), out=out)
    assert not out.any()


def test_other_streams_and_overlapping_calls():
    g = _gen(14)
    lens = [5000, 300, 2000]
    kc, vc, table = _cache_of(g, BF16, lens, 2, 256, 64)
    qs = [_rand(g, BF16, 3, 16, 256) for _ in range(4)]
    sl = _i(lens)
    want = [attention.paged_attention(q, kc, vc, table, sl) for q in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in qs]
    got = [[] for _ in qs]
    for _ in range(20):
        for i, (q, s) in enumerate(zip(qs, streams)):
            with torch.cuda.stream(s):
                got[i].append(attention.paged_attention(q, kc, vc, table, sl))
    torch.cuda.synchronize()
    for i in range(len(qs)):
        assert all(torch.equal(o, want[i]) for o in got[i])


@pytest.mark.parametrize("max_q", [None, 3])
@pytest.mark.parametrize("D,Hq,Hkv", [(64, 4, 2), (256, 16, 2), (128, 32, 1)])
def test_bad_row_bounds_are_told(D, Hq, Hkv, max_q):
    """Row bounds outside the tensors or descending set a bit, whichever kernel has the requests; others do not."""
    g, lens = _gen(13), [50, 60]
    kc, vc, table = _cache_of(g, BF16, lens, Hkv, D, 16)
    q = _rand(g, BF16, 6, Hq, D)
    for cu in ([-1, 2, 6], [0, 2, 7], [0, 4, 3], [0, 7], [-2, 6], [3, 1], [7, 7]):
        attention.paged_attention(q, kc, vc, table[:len(cu) - 1], _i(lens[:len(cu) - 1]), cu_q=_i(cu), max_q=max_q)
        assert attention.status() == _lib.STATUS_BAD_INDEX, cu
    for cu in ([0, 2, 6], [1, 2, 4], [3, 3, 3], [0, 6], [6, 6], [2, 3]):
        attention.paged_attention(q, kc, vc, table[:len(cu) - 1], _i(lens[:len(cu) - 1]), cu_q=_i(cu), max_q=max_q)
        assert attention.status() == 0, cu


def test_status_reads_lose_no_bit_of_another_stream():
    """A void plan on a side stream, at any moment of a read: its bit is in that read or in a later one."""
    r, side = random.Random(1), torch.cuda.Stream()
    t, one, none = _i([[0]]), _i([1]), _i([0])
    for _ in range(400):
        done = torch.cuda.Event()
        with torch.cuda.stream(side):
            torch.cuda._sleep(r.randint(100_000, 500_000))
            attention.kv_plan(t, none, one, none, none, page_size=16, num_pages=1, max_tokens=1)
            done.record()
        seen = 0
        while not done.query():
            seen |= attention.status()
        assert seen | attention.status() == _lib.STATUS_NO_PAGES


@pytest.mark.parametrize("Hq,Hkv,D,lens,rows", [
    (16, 2, 256, [2000, 300], [200, 90]),  # many rows, whole tiles
    (16, 2, 256, [5000], [40]), (12, 1, 128, [9000, 300], [7, 7]),  # split and joined
    (32, 8, 128, [700, 90, 3000], [300, 1, 4]),  # both kernels
])
def test_many_rows_on_several_streams(Hq, Hkv, D, lens, rows):
    """Overlapping calls of the many-row kernel, and a status read beside them, as if each were alone."""
    g = _gen(sum(lens) + D)
    kc, vc, table = _cache_of(g, BF16, lens, Hkv, D, 64)
    sl, cu = _i(lens), _i([0, *itertools.accumulate(rows)])
    qs = [_rand(g, BF16, sum(rows), Hq, D) for _ in range(4)]
    call = lambda q: attention.paged_attention(q, kc, vc, table, sl, cu_q=cu, max_q=max(rows), return_lse=True)  # noqa: E731
    want = [call(q) for q in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in qs]
    got = [[] for _ in qs]
    for n in range(20):
        for i, (q, s) in enumerate(zip(qs, streams)):
            with torch.cuda.stream(s):
                got[i].append(call(q))
        if n % 7 == 3:
            assert attention.status() == 0
    torch.cuda.synchronize()
    for w, outs in zip(want, got):
        assert all(torch.equal(o, w[0]) and torch.equal(e, w[1]) for o, e in outs)
    assert attention.status() == 0


def test_refusals_on_the_device():
    g = _gen(15)
    kc, vc, table = _cache_of(g, BF16, [20, 20], 2, 64, 16)
    q, sl = _rand(g, BF16, 2, 4, 64), _i([20, 20])
    for bad in (dict(q=q.half()), dict(q=q[:, :3]), dict(q=q[..., :32]), dict(seq_lens=sl.long()), dict(seq_lens=sl[:1]),
                dict(table=table.long()), dict(q=q[:1]), dict(cu_q=_i([0, 1])), dict(gate=q[:1]), dict(out=q[:1]),
                dict(v_cache=vc.half()), dict(k_cache=kc.transpose(2, 3)), dict(scale=-1.0), dict(window=-1),
                dict(max_q=-2), dict(seq_lens=sl.cpu())):
        a = dict(q=q, k_cache=kc, v_cache=vc, table=table, seq_lens=sl)
        a.update(bad)
        with pytest.raises((ValueError, _lib.RnbError)):
            attention.paged_attention(**a)
    inv, pos = torch.rand(32, device=DEV), _i([0, 1])
    for bad in (dict(inv_freq=inv.double()), dict(positions=pos[:1]), dict(sections=(16, 15)), dict(sections=()),
                dict(slots=_i([0])), dict(k=q[:1]), dict(k_cache=kc[..., :32]), dict(q_norm=q[0, 0, :32]),
                dict(positions=pos.float()), dict(out=q[:1])):
        a = dict(q=q, k=q[:, :2], v=q[:, :2], positions=pos, inv_freq=inv, slots=_i([0, 1]), k_cache=kc, v_cache=vc)
        a.update(bad)
        with pytest.raises((ValueError, _lib.RnbError)):
            attention.rope_append(**a)
    with pytest.raises(ValueError):
        attention.kv_plan(table, sl, sl[:1], sl, sl[:1], page_size=16, num_pages=4, max_tokens=4)
    with pytest.raises(_lib.RnbError):
        attention.kv_plan(table, sl, sl, sl, sl[:1], page_size=24, num_pages=4, max_tokens=4)


# ------------------------------------------------------------------ together

def test_steps_together_and_in_a_graph():
    """Prompt, decode and mixed steps through plan, rope_append and attention,
    each step's queries, pages and rows against 64 bits over the whole history;
    all once eagerly and once as one captured graph, with equal bits."""
    g = _gen(16)
    B, Hq, Hkv, D, P, N, W = 3, 16, 2, 256, 16, 64, 20
    sec, cap = (11, 11, 10), 160
    inv = (1e6 ** (-torch.arange(32, device=DEV, dtype=torch.float64) / 32)).float()
    steps = [[100, 0, 37], [1, 20, 1], [1, 1, 1], [1, 1, 1], [3, 1, 1], [1, 1, 1]]
    data = [[_rand(g, BF16, cap, h, D) for h in (Hq, Hkv, Hkv)] for _ in steps]
    order = torch.randperm(N, generator=g, device=DEV).to(torch.int32)

    def fresh():
        return dict(table=torch.full((B, W), -1, dtype=torch.int32, device=DEV), lens=_i([0] * B), count=_i([N]),
                    kc=torch.full((N, Hkv, P, D), float("nan"), dtype=BF16, device=DEV),
                    vc=torch.full((N, Hkv, P, D), float("nan"), dtype=BF16, device=DEV))

    def step(s, new, q, k, v, out):
        p = attention.kv_plan(s["table"], s["lens"], new, order, s["count"], page_size=P, num_pages=N, max_tokens=cap)
        qr = attention.rope_append(q, k, v, p.positions, inv, p.slots, s["kc"], s["vc"], sections=sec, interleaved=True)
        attention.paged_attention(qr, s["kc"], s["vc"], s["table"], p.seq_lens, cu_q=p.cu_q, out=out)
        s["lens"].copy_(p.seq_lens)
        s["count"].copy_(p.free_count)
        return qr

    s = fresh()
    hist = [[torch.zeros(0, Hkv, D, dtype=BF16, device=DEV) for _ in range(2)] for _ in range(B)]
    outs = []
    for new, (q, k, v) in zip(steps, data):
        out = torch.zeros(cap, Hq, D, dtype=BF16, device=DEV)
        qr = step(s, _i(new), q, k, v, out)
        outs.append(out)
        t, lens = 0, s["lens"].tolist()
        for b, n in enumerate(new):
            at = lens[b] - n
            pos = torch.arange(at, lens[b], device=DEV)[None].expand(3, n)
            want, tol = ref.rope(q[t:t + n], pos, inv, sec, True)
            ref.close(qr[t:t + n], want, tol, f"step {new} request {b} q")
            # the whole history is in the request's pages, old pages untouched
            hist[b] = [torch.cat([hist[b][0], k[t:t + n]]), torch.cat([hist[b][1], v[t:t + n]])]
            want, tol = ref.rope(hist[b][0], torch.arange(lens[b], device=DEV)[None].expand(3, -1), inv, sec, True)
            ref.close(ref.gather(s["kc"], s["table"][b], lens[b], P), want, tol, f"step {new} request {b} k")
            assert torch.equal(ref.gather(s["vc"], s["table"][b], lens[b], P), hist[b][1].double())
            t += n
        want, _, tol, _ = ref.attention(qr, s["kc"], s["vc"], s["table"], lens, new)
        ref.close(out[:t], want[:t], tol[:t], f"step {new}")
        assert not out[t:].any()
    assert s["lens"].tolist() == [sum(x) for x in zip(*steps)]
    assert attention.status() == 0

    # the same steps from one graph: lengths, pages and rows come from the device
    r = fresh()
    new, q, k, v = _i(steps[0]), *(x.clone() for x in data[0])
    out = torch.zeros(cap, Hq, D, dtype=BF16, device=DEV)
    keep = {n: x.clone() for n, x in r.items()}
    step(r, new, q, k, v, out)  # load the kernels outside the capture
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(r, new, q, k, v, out)
    for n, x in keep.items():
        r[n].copy_(x)
    for n, d, want in zip(steps, data, outs):
        new.copy_(_i(n))
        for to, x in zip((q, k, v), d):
            to.copy_(x)
        out.zero_()
        graph.replay()
        assert torch.equal(out, want)
    assert torch.equal(r["table"], s["table"]) and torch.equal(r["count"], s["count"])


def test_a_void_plan_leaves_the_step_without_effect():
    g = _gen(17)
    kc, vc, table = _cache_of(g, BF16, [16, 16], 2, 64, 16)
    k0, lens = kc.nan_to_num(7.0), _i([16, 16])
    q, k, v = _rand(g, BF16, 8, 4, 64), _rand(g, BF16, 8, 2, 64), _rand(g, BF16, 8, 2, 64)
    p = attention.kv_plan(table, lens, _i([1, 1]), _i([0]), _i([1]), page_size=16, num_pages=kc.shape[0], max_tokens=8)
    out = torch.full_like(q, 3.0)
    attention.rope_append(q, k, v, p.positions, torch.rand(32, device=DEV), p.slots, kc, vc, out=out)
    got = torch.full_like(q, 5.0)
    attention.paged_attention(out, kc, vc, table, p.seq_lens, cu_q=p.cu_q, out=got)
    assert (out == 3).all() and (got == 5).all() and torch.equal(kc.nan_to_num(7.0), k0)
    assert attention.status() == _lib.STATUS_NO_PAGES
