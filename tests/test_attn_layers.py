"""The full-attention layer: loaded from a checkpoint (CPU), and on the GPU each
of its stages against 64 bits, and a stack with attention over a paged cache
against the calls it is made of, eagerly and from a graph."""
import numpy as np
import pytest
import torch

from runnel_b200 import _lib, attention, attn_layers, checkpoint, ops, probes, quant, stack
from runnel_b200.switch_layers import QuantizedLinear
from tests import _attn_ref as ref

DEV = "cuda"


def _linear_arrays(rng, rows, K, bits):
    w = rng.integers(0, 2 ** 32, (rows, K * bits // 32), dtype=np.uint64).astype(np.uint32)
    s = quant.f32_to_bf16_bits(rng.uniform(0.001, 0.01, (rows, K // 64)) * (1 if bits == 4 else 1 / 16))
    b = quant.f32_to_bf16_bits(rng.standard_normal((rows, K // 64)) * 0.01 - 7.5 * 0.0055)
    return w, s, b


def _write(path, rng, H, Hq, Hkv, D, bits=(4, 4, 4, 8), gated=True, layer=3):
    p = f"language_model.model.layers.{layer}"
    t = {f"{p}.input_layernorm.weight": (quant.f32_to_bf16_bits(1 + 0.02 * rng.standard_normal(H)), "BF16")}
    for n in ("q_norm", "k_norm"):
        t[f"{p}.self_attn.{n}.weight"] = (quant.f32_to_bf16_bits(1 + 0.1 * rng.standard_normal(D)), "BF16")
    shapes = {"q": (Hq * D * (2 if gated else 1), H), "k": (Hkv * D, H), "v": (Hkv * D, H), "o": (H, Hq * D)}
    for (proj, (rows, K)), b in zip(shapes.items(), bits):
        for n, a in zip(("weight", "scales", "biases"), _linear_arrays(rng, rows, K, b)):
            t[f"{p}.self_attn.{proj}_proj.{n}"] = (a, "U32" if n == "weight" else "BF16")
    checkpoint.write_safetensors(str(path / "model.safetensors"), t)
    return checkpoint.TensorStore(str(path))


@pytest.mark.parametrize("gated", [True, False])
def test_checkpoint_attention_arrays(tmp_path, gated):
    st = _write(tmp_path, np.random.default_rng(0), 512, 8, 2, 64, gated=gated)
    a = checkpoint.load_attention_arrays(st, 3)
    assert (a["head_dim"], a["n_heads"], a["n_kv_heads"], a["gated"]) == (64, 8, 2, gated)
    assert a["bits"] == {"q": 4, "k": 4, "v": 4, "o": 8}
    assert a["q"][0].shape == (512 * (2 if gated else 1), 64) and a["o"][0].shape == (512, 128)
    with pytest.raises(ValueError, match="no full attention"):
        checkpoint.load_attention_arrays(st, 0)


def test_checkpoint_attention_refuses_other_types_and_biases(tmp_path):
    """Scales, biases and norms are taken as bf16 bits and codes as 32-bit words; a projection's own bias has no place."""
    p = "language_model.model.layers.3"
    odd = {f"{p}.input_layernorm.weight": "F16", f"{p}.self_attn.q_norm.weight": "F16",
           f"{p}.self_attn.k_norm.weight": "F32", f"{p}.self_attn.v_proj.scales": "F16",
           f"{p}.self_attn.o_proj.biases": "F16", f"{p}.self_attn.k_proj.weight": "I32",
           f"{p}.self_attn.q_proj.bias": "BF16", f"{p}.self_attn.o_proj.bias": "BF16"}
    st = _write(tmp_path, np.random.default_rng(5), 512, 8, 2, 64)
    good = {n: (st.read(n)[0], e[3]) for n, e in st.entries.items()}
    for name, dtype in odd.items():
        arr = good[name][0] if name in good else np.zeros(512, np.uint16)
        checkpoint.write_safetensors(str(tmp_path / "model.safetensors"), {**good, name: (arr, dtype)})
        with pytest.raises(ValueError, match=name):
            checkpoint.load_attention_arrays(checkpoint.TensorStore(str(tmp_path)), 3)
    checkpoint.write_safetensors(str(tmp_path / "model.safetensors"), good)
    assert checkpoint.load_attention_arrays(checkpoint.TensorStore(str(tmp_path)), 3)["n_heads"] == 8


def test_attention_layer_on_cpu_refuses_mixed_formats(tmp_path):
    st = _write(tmp_path, np.random.default_rng(1), 512, 8, 2, 64, bits=(4, 8, 4, 8))
    with pytest.raises(ValueError, match="one quantization format"):
        checkpoint.load_attention(st, 3, attn_layers.RotarySpec(rot=32), device="cpu")
    st = _write(tmp_path, np.random.default_rng(1), 512, 8, 2, 64)
    layer, norm = checkpoint.load_attention(st, 3, attn_layers.RotarySpec(rot=32), device="cpu")
    assert layer.weight.shape == (2 * 512 + 256, 64) and norm.shape == (512,) and layer.inv_freq.shape == (16,)
    bad = QuantizedLinear(layer.weight[:64], layer.scales[:64], layer.biases[:64], bits=4)
    kv = QuantizedLinear(layer.weight[:128], layer.scales[:128], layer.biases[:128], bits=4)
    with pytest.raises(ValueError, match="rows"):
        attn_layers.GatedAttention(bad, kv, kv, layer.o_proj, layer.q_norm, layer.k_norm, 64, layer.rotary)


@pytest.mark.parametrize("proj", ["q_proj", "k_proj", "v_proj", "o_proj"])
def test_attention_layer_refuses_what_its_products_would_leave_out(proj):
    """Module biases and projections without affine biases, in each of the four."""
    rng = np.random.default_rng(4)

    def linear(rows, K, affine=True):
        w, s, b = (torch.from_numpy(a.view(np.int32 if a.dtype == np.uint32 else np.int16))
                   for a in _linear_arrays(rng, rows, K, 4))
        return QuantizedLinear(w.view(torch.uint32), s.view(torch.bfloat16), b.view(torch.bfloat16) if affine else None)

    def layer(**other):
        lin = dict(q_proj=linear(1024, 512), k_proj=linear(128, 512), v_proj=linear(128, 512), o_proj=linear(512, 512))
        lin.update(other)
        return attn_layers.GatedAttention(**lin, q_norm=None, k_norm=None, head_dim=64, rotary=attn_layers.RotarySpec(32))

    assert layer().n_kv_heads == 2
    rows = {"q_proj": 1024, "o_proj": 512}.get(proj, 128)
    biased = linear(rows, 512)
    biased.register_buffer("bias", torch.zeros(rows))
    for bad in (biased, linear(rows, 512, affine=False)):
        with pytest.raises(ValueError, match="affine|format"):
            layer(**{proj: bad})


def test_a_release_makes_plans_stale(monkeypatch):
    """(the calls are stood in for: what is tested is the order)"""
    cache = _cache(1, 2, 64, 3, device="cpu")
    plan = attention.KVPlan(cache.lens + 1, None, None, None, cache.free_count - 1)
    monkeypatch.setattr(attention, "kv_plan", lambda *a, **k: plan)
    monkeypatch.setattr(attention, "kv_release", lambda *a, **k: (cache.lens * 0, cache.free_count + 3))
    cache.commit(cache.plan(None, 3))
    assert cache.lens.tolist() == [1, 1, 1] and cache.free_count.item() == 39
    cache.plan(None, 3)
    cache.release(None)
    with pytest.raises(RuntimeError, match="plan again"):
        cache.commit(plan)
    assert cache.lens.tolist() == [0, 0, 0] and cache.free_count.item() == 42
    cache.commit(cache.plan(None, 3))
    assert cache.lens.tolist() == [1, 1, 1]


def _cpu_linears(rng, H=512, Hq=8, Hkv=2, D=64):
    def linear(rows, K):
        w, s, b = (torch.from_numpy(a.view(np.int32 if a.dtype == np.uint32 else np.int16))
                   for a in _linear_arrays(rng, rows, K, 4))
        return [w.view(torch.uint32), s.view(torch.bfloat16), b.view(torch.bfloat16)]
    return {"q_proj": linear(2 * Hq * D, H), "k_proj": linear(Hkv * D, H), "v_proj": linear(Hkv * D, H),
            "o_proj": linear(H, Hq * D)}


def test_attention_layer_refuses_shapes_that_do_not_fit():
    """The products read what the codes' shape says: scales, biases and sizes have to agree with it."""
    def layer(lin, D=64, norm=None):
        return attn_layers.GatedAttention(**{n: QuantizedLinear(*t) for n, t in lin.items()}, q_norm=norm, k_norm=None,
                                          head_dim=D, rotary=attn_layers.RotarySpec(32))

    new = lambda: _cpu_linears(np.random.default_rng(6))  # noqa: E731
    assert layer(new()).n_heads == 8
    for proj in ("q_proj", "k_proj", "v_proj", "o_proj"):
        for part, cut in ((1, lambda t: t[:-1]), (2, lambda t: t[:-1]), (1, lambda t: t[:, :-1]), (2, lambda t: t[:, :-1]),
                          (1, lambda t: t.half()), (2, lambda t: t.float()), (0, lambda t: t.view(torch.int32).long())):
            lin = new()
            lin[proj][part] = cut(lin[proj][part])
            with pytest.raises(ValueError, match=proj):
                layer(lin)
    lin = new()
    lin["v_proj"] = [t[:, :t.shape[1] // 2] for t in lin["v_proj"]]  # another hidden size
    with pytest.raises(ValueError, match="hidden"):
        layer(lin)
    lin = new()
    lin["o_proj"] = [t[:256] for t in lin["o_proj"]]
    with pytest.raises(ValueError, match="hidden"):
        layer(lin)
    lin = new()
    for proj in ("k_proj", "v_proj"):
        lin[proj] = [t[:100] for t in lin[proj]]  # not whole heads
    with pytest.raises(ValueError, match="heads"):
        layer(lin)
    lin = _cpu_linears(np.random.default_rng(7), Hkv=3)
    with pytest.raises(ValueError, match="heads"):
        layer(lin)
    for norm in (torch.ones(63, dtype=torch.bfloat16), torch.ones(64), torch.ones(1, 64, dtype=torch.bfloat16)):
        with pytest.raises(ValueError, match="q_norm"):
            layer(new(), norm=norm)


def test_attention_layers_refuse_tokens_that_are_not_bf16_rows():
    a = attn_layers.GatedAttention(**{n: QuantizedLinear(*t) for n, t in _cpu_linears(np.random.default_rng(8)).items()},
                                   q_norm=None, k_norm=None, head_dim=64, rotary=attn_layers.RotarySpec(32))
    for x in (torch.zeros(3, 512), torch.zeros(3, 512, dtype=torch.float16), torch.zeros(3, 256, dtype=torch.bfloat16),
              torch.zeros(1, 3, 512, dtype=torch.bfloat16), torch.zeros(512, dtype=torch.bfloat16)):
        with pytest.raises(ValueError, match="bf16"):
            a(x, None, 0, None)
    x = torch.zeros(3, 512, dtype=torch.bfloat16)
    for norm in (torch.ones(511, dtype=torch.bfloat16), torch.ones(512)):
        s = stack.LayerStack([object()], [object()], attn=[a], attn_norm_w=[norm])
        with pytest.raises(ValueError, match="attn_norm_w"):
            s.forward(x, cache=object(), plan=object())


def test_layers_run_on_the_device_of_their_tokens(monkeypatch):
    """The products launch on the current device: the layer and the stack make it that of their tokens."""
    at, current = [], [0]

    class DeviceOf:
        def __init__(self, t):
            self.index = int(t[0, 0])  # (stands in for the tensor's device)

        def __enter__(self):
            self.was, current[0] = current[0], self.index

        def __exit__(self, *exc):
            current[0] = self.was

    class Stop(Exception):
        pass

    def first_call(*a, **k):
        at.append(current[0])
        raise Stop

    monkeypatch.setattr(torch.cuda, "device_of", DeviceOf)
    monkeypatch.setattr(attn_layers.probes, "qmm", first_call)
    monkeypatch.setattr(stack, "add_rmsnorm", first_call)
    x = torch.full((1, 512), 3.0, dtype=torch.bfloat16)
    layer = attn_layers.GatedAttention(**{n: QuantizedLinear(*t) for n, t in _cpu_linears(np.random.default_rng(9)).items()},
                                       q_norm=None, k_norm=None, head_dim=64, rotary=attn_layers.RotarySpec(32))
    s = stack.LayerStack([object()], [object()], attn=[layer], attn_norm_w=[torch.ones(512, dtype=torch.bfloat16)])
    with pytest.raises(Stop):
        layer.forward(x, None, 0, None)
    with pytest.raises(Stop):
        s.forward(x, cache=object(), plan=object())
    assert at == [3, 3] and current == [0]


def test_stack_checks_its_attention_layers():
    with pytest.raises(ValueError, match="attn_norm_w"):
        stack.LayerStack([object()], [object()], attn=[object()])


def _cache(n_layers, Hkv, D, B, device=DEV):
    return attn_layers.PagedKVCache(n_layers, 40, Hkv, D, B, 400, page_size=32, device=device)


@pytest.mark.gpu
@pytest.mark.parametrize("gated,sections", [(True, (6, 5, 5)), (False, None)])
def test_layer_stages_against_64_bits(tmp_path, gated, sections):
    H, Hq, Hkv, D = 512, 8, 2, 64
    st = _write(tmp_path, np.random.default_rng(2), H, Hq, Hkv, D, gated=gated)
    spec = attn_layers.RotarySpec(rot=32, theta=1e6, sections=sections)
    layer, _ = checkpoint.load_attention(st, 3, spec, device=DEV)
    cache = _cache(1, Hkv, D, 3)
    g = torch.Generator(device=DEV).manual_seed(3)
    sec = sections or (16,)
    lens = [0, 0, 0]
    for new in ([90, 0, 33], [1, 4, 1], [1, 1, 70]):
        cap = sum(new) + 3
        plan = cache.plan(torch.tensor(new, dtype=torch.int32, device=DEV), cap)
        x = torch.randn(cap, H, generator=g, device=DEV).to(torch.bfloat16)
        rec = {}
        out = layer(x, cache, 0, plan, max(new), record=rec)
        cache.commit(plan)
        n = sum(new)
        lens = [a + b for a, b in zip(lens, new)]
        assert cache.lens.tolist() == lens
        axes = plan.positions[None].expand(len(sec), -1)
        want, tol = ref.rope(rec["q"], axes, layer.inv_freq, sec, True, layer.q_norm)
        ref.close(rec["q_rot"][:n], want[:n], tol[:n], "q")
        want, tol = ref.rope(rec["k"], axes, layer.inv_freq, sec, True, layer.k_norm)
        t = 0
        for b, m in enumerate(new):
            got = ref.gather(cache.k[0], cache.table[b], lens[b], 32)[lens[b] - m:]
            ref.close(got, want[t:t + m], tol[t:t + m], "k")
            assert torch.equal(ref.gather(cache.v[0], cache.table[b], lens[b], 32)[lens[b] - m:], rec["v"][t:t + m].double())
            t += m
        want, _, tol, _ = ref.attention(rec["q_rot"][:n], cache.k[0], cache.v[0], cache.table, lens, new,
                                        gate=rec["gate"][:n] if gated else None)
        ref.close(rec["attn"][:n], want, tol, "attention")
        # the two products: bf16 inputs, exact weights s q + b rounded once to fp16 by the product's
        # converters (2^-11), fp32 sums over K, rounded once to bf16 (2^-8)
        for y, xin, w in ((rec["qkv"], x, (layer.bits, layer.weight, layer.scales, layer.biases)),
                          (out, rec["attn"].reshape(cap, -1),
                           (layer.o_bits, layer.o_proj.weight, layer.o_proj.scales, layer.o_proj.biases))):
            W = probes.dequant_reference(*w)
            z, mag = xin.double() @ W.T, xin.double().abs() @ W.abs().T
            ref.close(y, z, 1.05 * (2.0 ** -8 * z.abs() + (2.0 ** -10 + W.shape[1] * 2.0 ** -24) * mag) + 1e-30, "product")
        assert torch.isfinite(out).all()
    assert attention.status() == 0


@pytest.mark.gpu
def test_layer_of_no_tokens(tmp_path):
    st = _write(tmp_path, np.random.default_rng(20), 512, 8, 2, 64)
    layer, _ = checkpoint.load_attention(st, 3, attn_layers.RotarySpec(rot=32), device=DEV)
    cache = _cache(1, 2, 64, 3)
    plan = cache.plan(torch.zeros(3, dtype=torch.int32, device=DEV), 0)
    assert layer(torch.zeros(0, 512, dtype=torch.bfloat16, device=DEV), cache, 0, plan).shape == (0, 512)
    cache.commit(plan)
    assert cache.lens.tolist() == [0, 0, 0] and attention.status() == 0


@pytest.mark.gpu
def test_release_lets_pages_serve_again():
    cache = attn_layers.PagedKVCache(1, 4, 1, 64, 2, 128, page_size=32)
    new = torch.tensor([100, 28], dtype=torch.int32, device=DEV)
    plan = cache.plan(new, 128)
    cache.commit(plan)
    # four pages hold 128 tokens; 100 and 28 need five: the plan was void
    assert attention.status() == _lib.STATUS_NO_PAGES and cache.lens.tolist() == [0, 0]
    plan = cache.plan(torch.tensor([96, 28], dtype=torch.int32, device=DEV), 128)
    cache.commit(plan)
    assert cache.lens.tolist() == [96, 28] and cache.free_count.item() == 0
    first = sorted(cache.table[0, :3].tolist())
    cache.release(torch.tensor([1, 0], dtype=torch.int32, device=DEV))
    assert cache.lens.tolist() == [0, 28] and cache.free_count.item() == 3
    plan = cache.plan(torch.tensor([0, 90], dtype=torch.int32, device=DEV), 128)
    cache.commit(plan)
    assert cache.lens.tolist() == [0, 118] and cache.free_count.item() == 0
    assert sorted(cache.table[1, 1:4].tolist()) == first
    assert attention.status() == 0


@pytest.mark.gpu
def test_a_plan_from_before_a_release_is_refused():
    """Its lengths and free count would undo the release."""
    cache = attn_layers.PagedKVCache(1, 6, 1, 64, 2, 128, page_size=32)
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    cache.commit(cache.plan(ints([40, 40]), 80))
    plan = cache.plan(ints([1, 0]), 1)
    cache.release(ints([0, 1]))
    with pytest.raises(RuntimeError, match="plan again"):
        cache.commit(plan)
    assert cache.lens.tolist() == [40, 0] and cache.free_count.item() == 4
    plan = cache.plan(ints([1, 90]), 91)
    cache.commit(plan)
    assert cache.lens.tolist() == [41, 90] and cache.free_count.item() == 1
    assert len({*cache.table[0, :2].tolist(), *cache.table[1, :3].tolist()}) == 5
    cache.commit(plan)  # twice is once
    assert cache.lens.tolist() == [41, 90] and attention.status() == 0

    # a plan in a graph is made anew by every replay
    new = ints([0, 1])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        plan = cache.plan(new, 1)
    cache.release(ints([1, 0]))
    graph.replay()
    cache.commit(plan)
    assert cache.lens.tolist() == [0, 91] and cache.free_count.item() == 3 and attention.status() == 0


def _stack(tmp_path, seed):
    """Two MoE layers, the second with attention before it."""
    layers, norms = stack.synthetic_layers(2, 4, seed=seed, device=DEV, H=2048, I=512, E=16)
    st = _write(tmp_path, np.random.default_rng(seed), 2048, 16, 2, 128)
    a, an = checkpoint.load_attention(st, 3, attn_layers.RotarySpec(rot=64, sections=(12, 10, 10)), device=DEV)
    return stack.LayerStack(layers, norms, ws=ops.Workspace(DEV), attn=[None, a], attn_norm_w=[None, an])


@pytest.mark.gpu
def test_stack_with_attention_steps_and_graph(tmp_path):
    s = _stack(tmp_path, 11)
    steps = [[40, 0, 3], [1, 30, 1], [1, 1, 1], [1, 1, 1]]
    cap = 64
    g = torch.Generator(device=DEV).manual_seed(12)
    xs = [torch.randn(cap, 2048, generator=g, device=DEV).to(torch.bfloat16) for _ in steps]
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731

    cache = _cache(1, 2, 128, 3)
    outs = []
    for new, x in zip(steps, xs):
        plan = cache.plan(ints(new), cap)
        outs.append(s.forward(x, cache=cache, plan=plan))
        cache.commit(plan)

    # the calls it is made of
    cache = _cache(1, 2, 128, 3)
    a, an = s.attn[1], s.attn_norm_w[1]
    for new, x, want in zip(steps, xs, outs):
        plan = cache.plan(ints(new), cap)
        r, xn = torch.empty_like(x), torch.empty_like(x)
        stack.add_rmsnorm(x, None, s.norm_w[0], r, xn)
        y = ops.moe_block(s.layers[0], xn)
        stack.add_rmsnorm(r, y, an, r, xn)
        y = a(xn, cache, 0, plan)
        stack.add_rmsnorm(r, y, s.norm_w[1], r, xn)
        y = ops.moe_block(s.layers[1], xn)
        stack.add_rmsnorm(r, y, s.norm_w[1], r, xn)
        cache.commit(plan)
        assert torch.equal(r[:sum(new)], want[:sum(new)])

    # one captured step for all of them
    cache = _cache(1, 2, 128, 3)
    new, x, out = ints(steps[0]), xs[0].clone(), torch.empty_like(xs[0])

    def step():
        plan = cache.plan(new, cap)
        s.forward(x, out=out, cache=cache, plan=plan)
        cache.commit(plan)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    cache.lens.zero_()
    cache.free_count.fill_(40)
    for n, xx, want in zip(steps, xs, outs):
        new.copy_(ints(n))
        x.copy_(xx)
        graph.replay()
        assert torch.equal(out[:sum(n)], want[:sum(n)])
    assert cache.lens.tolist() == [sum(v) for v in zip(*steps)]
    assert attention.status() == 0


@pytest.mark.gpu
def test_stack_hands_windows_to_its_attention_layers(tmp_path):
    """One window for all of them, or one each: the two layers of a stack against the calls it is made of."""
    one = _stack(tmp_path, 14)
    a, an = one.attn[1], one.attn_norm_w[1]
    s = stack.LayerStack(one.layers, one.norm_w, ws=one.ws, attn=[a, a], attn_norm_w=[an, an])
    g = torch.Generator(device=DEV).manual_seed(15)
    x = torch.randn(90, 2048, generator=g, device=DEV).to(torch.bfloat16)
    new = torch.tensor([60, 0, 30], dtype=torch.int32, device=DEV)
    got = {}
    for window in (0, 7, (0, 7), (7, 0)):
        cache = _cache(2, 2, 128, 3)
        plan = cache.plan(new, 90)
        got[window] = s.forward(x, cache=cache, plan=plan, window=window)
        each = (window, window) if isinstance(window, int) else window
        r, xn, y = torch.empty_like(x), torch.empty_like(x), None
        for i, w in enumerate(each):
            stack.add_rmsnorm(r if i else x, y, an, r, xn)
            y = a(xn, cache, i, plan, window=w)
            stack.add_rmsnorm(r, y, s.norm_w[i], r, xn)
            y = ops.moe_block(s.layers[i], xn)
        stack.add_rmsnorm(r, y, s.norm_w[1], r, xn)
        assert torch.equal(r, got[window])
    assert not any(torch.equal(got[u], got[v]) for u, v in ((0, 7), ((0, 7), (7, 0)), (0, (0, 7)), (7, (7, 0))))
    for window in ((), (1,), (1, 2, 3)):
        with pytest.raises(ValueError, match="window"):
            s.forward(x, cache=cache, plan=plan, window=window)
    assert attention.status() == 0


@pytest.mark.gpu
def test_stack_refuses_attention_without_a_cache(tmp_path):
    s = _stack(tmp_path, 13)
    with pytest.raises(ValueError, match="cache and a plan"):
        s.forward(torch.zeros(1, 2048, dtype=torch.bfloat16, device=DEV))
