"""Cases, plain forms and 64-bit definitions of the attention-side operators.

Three operators of a paged key-value cache, in the order in which a serving step uses them:

* ``plan``       block tables, slots and positions of a step from the requests' lengths
                 (``runnel_b200.attention.kv_plan``);
* ``rope``       per-head RMS norm, rotary positions with one to three axes, and the append of
                 the step's keys and values to the cache (``rope_append``);
* ``attention``  attention of the step's queries over the paged cache (``paged_attention``):
                 one new token for each request (``q`` 1), a few (``q`` up to 8), and prompts.

A case is a dict of plain values.  Lengths of ragged batches are a function of the case, the
tensors' values one of the seed.
"""
import itertools
import math
import random

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
_THETA = 1.0e6


# ------------------------------------------------------------------ cases

def _attention(name, dtype, B, Hq, Hkv, D, page, prior, q, ragged=False, window=0, gate=False, lse=False):
    return {"name": name, "op": "attention", "dtype": dtype, "B": B, "Hq": Hq, "Hkv": Hkv, "D": D, "page": page,
            "prior": prior, "q": q, "ragged": ragged, "window": window, "gate": gate, "lse": lse}


def _rope(name, dtype, T, Hq, Hkv, D, rot, axes, interleaved, norm, page):
    return {"name": name, "op": "rope", "dtype": dtype, "T": T, "Hq": Hq, "Hkv": Hkv, "D": D, "rot": rot,
            "axes": axes, "interleaved": interleaved, "norm": norm, "page": page}


def _plan(name, B, page, prior, q, ragged):
    return {"name": name, "op": "plan", "B": B, "page": page, "prior": prior, "q": q, "ragged": ragged}


def listed():
    return [
        # a decode step of a few requests: one launch's latency
        _plan("plan-decode-8", 8, 16, 1000, 1, True),
        # a large scheduler step: many requests, prompts among them, small pages
        _plan("plan-mixed-2048", 2048, 16, 8000, 60, True),
        # one decode step of 8 requests, partial rotation with three interleaved axes, normed heads
        _rope("rope-decode-8", "bf16", 8, 16, 2, 256, 64, 3, True, True, 64),
        # a prompt chunk of the prefill benchmark's token count
        _rope("rope-prompt-16384", "bf16", 16384, 16, 2, 256, 64, 3, True, True, 64),
        # an odd chunk, whole heads rotated, axes in sections, no norm
        _rope("rope-odd-4097-fp16", "fp16", 4097, 32, 8, 128, 128, 3, False, False, 16),
        # chat with one user and a short context: latency
        _attention("decode-1-short", "bf16", 1, 16, 2, 256, 64, 300, 1),
        # a serving batch of uneven contexts, gated output
        _attention("decode-64-ragged", "bf16", 64, 16, 2, 256, 64, 8191, 1, ragged=True, gate=True),
        # few requests with long contexts: the cache's length is split
        _attention("decode-2-long-fp16", "fp16", 2, 32, 8, 128, 16, 131071, 1, lse=True),
        # a wide batch of a model with as many key as query heads and a sliding window
        _attention("decode-192-window", "bf16", 192, 16, 16, 64, 32, 5000, 1, ragged=True, window=1024),
        # checking four drafted tokens for each request
        _attention("verify-32x4", "bf16", 32, 32, 8, 128, 16, 2047, 4, ragged=True),
        # one long prompt
        _attention("prompt-8192", "bf16", 1, 16, 2, 256, 64, 0, 8192, gate=True),
        # prompts of uneven length, some with a cached beginning
        _attention("prompt-ragged-12", "bf16", 12, 32, 8, 128, 16, 1000, 1500, ragged=True, lse=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["plan", "rope", "decode", "decode", "prompt", "verify"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    Hq, Hkv, D = rng.choice([(16, 2, 256), (8, 1, 256), (32, 8, 128), (28, 4, 128), (40, 8, 128), (16, 16, 64),
                             (14, 2, 64), (24, 8, 64), (12, 1, 128)])
    page = rng.choice([16, 32, 64, 128])
    if op == "plan":
        B = _log(rng, 1, 2048)
        c = _plan("", B, page, _log(rng, 1, 8000), rng.choice([1, 1, _log(rng, 1, max(1, 60000 // B))]),
                  rng.random() < 0.8)
    elif op == "rope":
        c = _rope("", dtype, _log(rng, 1, 16384 if Hq * D <= 4096 else 12000), Hq, Hkv, D,
                  rng.choice([D, D // 2, D // 4]), rng.choice([1, 3, 3]), rng.random() < 0.5, rng.random() < 0.5, page)
    elif op == "prompt":
        B = _log(rng, 1, 8)
        q = _log(rng, 24, 6000 // B)
        c = _attention("", dtype, B, Hq, Hkv, D, page, rng.choice([0, _log(rng, 1, 2000)]), q, rng.random() < 0.7,
                       rng.choice([0, 0, _log(rng, 16, 2048)]), rng.random() < 0.3, rng.random() < 0.3)
    else:
        B = _log(rng, 1, 192)
        most = min(131000, 250_000_000 // (B * Hkv * D))
        c = _attention("", dtype, B, Hq, Hkv, D, page, _log(rng, 1, most), 1 if op == "decode" else rng.randint(2, 8),
                       rng.random() < 0.7, rng.choice([0, 0, _log(rng, 16, 4096)]), rng.random() < 0.3,
                       rng.random() < 0.3)
    del c["name"]
    return c


# ------------------------------------------------------------------ inputs

def _lens(case):
    """[(cached tokens, new tokens)] of the requests; the last of a ragged batch of four or more is idle."""
    B, prior, q = case["B"], case["prior"], case["q"]
    if not case["ragged"]:
        return [(prior, q)] * B
    r = random.Random("%d %d %d" % (B, prior, q))
    out = [(prior, q)]
    for _ in range(B - 1):
        out.append((int((prior + 1) ** r.random()) if r.random() < 0.3 else int(prior * r.random()),
                    max(1, int(q * r.random() ** 1.5 + 0.5))))
    if B >= 4:
        out[-1] = (0, 0)
    return out


def _kv_q(case):
    """Key lengths and query rows of an attention case; with one token each every request has a row."""
    lens = _lens(case)
    kv = [p + n for p, n in lens]
    return kv, [1 if case["q"] == 1 else n for _, n in lens]


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _sections(case):
    """How many of the rot / 2 frequencies each axis (time, height, width) turns."""
    n = case["rot"] // 2
    if case["axes"] == 1:
        return (n,)
    w = n // 3
    h = (n - w) // 2
    return (n - w - h, h, w)


def _tables(lens, page, extra, g):
    """A block table of scattered pages for these lengths, [B, most + extra], and the number of pages."""
    held = [-(-n // page) for n in lens]
    W, N = max(max(held), 1) + extra, sum(held) + 3
    order = torch.randperm(N, generator=g, device="cuda").to(torch.int32)
    start = torch.tensor([0, *itertools.accumulate(held)][:-1], device="cuda")
    cols = torch.arange(W, device="cuda")
    inside = cols[None] < torch.tensor(held, device="cuda")[:, None]
    table = torch.where(inside, order[(start[:, None] + cols[None]).clamp(max=N - 1)], torch.zeros_like(order[:1]))
    return table.contiguous(), N


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, scale=1.0):
        return (torch.randn(shape, generator=g, device="cuda") * scale).to(_TYPES[case["dtype"]])

    s = {"case": dict(case)}
    if case["op"] == "plan":
        lens, P = _lens(case), case["page"]
        ctx, new = [c for c, _ in lens], [n for _, n in lens]
        turn = torch.randperm(len(lens), generator=g, device="cuda")  # which request has which lengths
        need = sum(-(-(c + n) // P) - -(-c // P) for c, n in lens)
        s["ctx"], s["new"] = _ints(ctx)[turn], _ints(new)[turn]
        held, N = _tables(ctx, P, -(-max(new) // P) + 2, g)
        total = N + need + 5
        s["table"], s["num_pages"] = held[turn].contiguous(), total
        s["free_pages"] = (torch.randperm(total - N, generator=g, device="cuda") + N).to(torch.int32)
        s["free_count"] = _ints([total - N - 2])
        s["max_tokens"] = sum(new) + max(1, sum(new) // 8)
        return s
    D, Hq, Hkv, P = case["D"], case["Hq"], case["Hkv"], case["page"]
    if case["op"] == "rope":
        T, n = case["T"], case["rot"] // 2
        both = normal(T, (Hq + 2 * Hkv) * D)  # what the joint projection gives
        q, k, v = both.split([Hq * D, Hkv * D, Hkv * D], dim=1)
        s["q"], s["k"], s["v"] = q.view(T, Hq, D), k.view(T, Hkv, D), v.view(T, Hkv, D)
        s["inv_freq"] = (_THETA ** (-torch.arange(n, device="cuda", dtype=torch.float64) / n)).float()
        # text and images far into a conversation: each axis moves by itself
        base = int(torch.randint(0, 100000, (1,), generator=g, device="cuda").item())
        t = torch.arange(T, device="cuda", dtype=torch.int32)
        s["positions"] = (t + base)[None].repeat(case["axes"], 1)
        s["positions"][1:] += torch.randint(0, 64, (case["axes"] - 1, T), generator=g, device="cuda").to(torch.int32)
        N = -(-T // P) + 2
        s["k_cache"], s["v_cache"] = normal(N, Hkv, P, D), normal(N, Hkv, P, D)
        s["slots"] = torch.randperm(N * P, generator=g, device="cuda")[:T].to(torch.int32)
        s["q_norm"] = s["k_norm"] = None
        if case["norm"]:
            s["q_norm"], s["k_norm"] = 1 + normal(D, scale=0.1), 1 + normal(D, scale=0.1)
        return s
    kv, rows = _kv_q(case)
    T = sum(rows)
    s["table"], N = _tables(kv, P, 1, g)
    s["q"] = normal(T, Hq, D, scale=1.5)
    s["k_cache"], s["v_cache"] = normal(N, Hkv, P, D), normal(N, Hkv, P, D)
    s["gate"] = normal(T, Hq, D) if case["gate"] else None
    s["seq_lens"] = _ints(kv)
    s["cu_q"] = None if case["q"] == 1 else _ints([0, *itertools.accumulate(rows)])
    s["max_q"] = max(rows)
    return s


# ------------------------------------------------------------------ plain forms

def _plain_plan(s):
    ctx, new, table, P, fc = s["ctx"], s["new"], s["table"], s["case"]["page"], s["free_count"]
    B, W = table.shape
    held = (ctx + P - 1) // P
    need = (ctx + new + P - 1) // P - held
    taken = need.cumsum(0, dtype=torch.int32)
    ends = new.cumsum(0, dtype=torch.int32)
    fits = (taken[-1:] <= fc) & (ends[-1:] <= s["max_tokens"]) & ((held + need).amax(0, keepdim=True) <= W)
    off = torch.arange(W, device="cuda")[None] - held[:, None]
    fresh = (off >= 0) & (off < need[:, None]) & fits
    at = (fc - 1 - ((taken - need)[:, None] + off)).clamp(0, s["free_pages"].numel() - 1)
    table = torch.where(fresh, s["free_pages"][at], table)
    zero = torch.zeros_like(ends[:1])
    cu = torch.cat([zero, ends]) * fits
    t = torch.arange(s["max_tokens"], device="cuda", dtype=torch.int32)
    b = torch.searchsorted(cu[1:].contiguous(), t, right=True).clamp(max=B - 1)
    live = t < cu[-1:]
    pos = torch.where(live, ctx[b] + t - cu[b], zero)
    slots = torch.where(live, table[b, pos // P] * P + pos % P, zero - 1)
    return {"table": table, "seq_lens": ctx + new * fits, "cu_q": cu.to(torch.int32), "positions": pos.to(torch.int32),
            "slots": slots.to(torch.int32), "free_count": (fc - taken[-1:] * fits).to(torch.int32)}


def _axis_of(case):
    """The axis that turns each frequency: sections one after the other, or taken in turns."""
    n, sec = case["rot"] // 2, _sections(case)
    i = torch.arange(n, device="cuda")
    if len(sec) == 1:
        return i * 0
    if case["interleaved"]:
        return torch.where((i % 3 == 1) & (i < 3 * sec[1]), 1, torch.where((i % 3 == 2) & (i < 3 * sec[2]), 2, 0))
    return (i >= sec[0]).long() + (i >= sec[0] + sec[1]).long()


def _plain_rope(s):
    case = s["case"]
    n, P = case["rot"] // 2, case["page"]
    angle = s["positions"].double()[_axis_of(case)].T * s["inv_freq"].double()[None]  # [T, n]
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]

    def turned(x, w):
        x = x.float()
        if w is not None:
            x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * w.float()
        a, b = x[..., :n], x[..., n:2 * n]
        return torch.cat([a * cos - b * sin, b * cos + a * sin, x[..., 2 * n:]], -1).to(s["q"].dtype)

    page, off = s["slots"].long() // P, s["slots"].long() % P
    s["k_cache"][page, :, off] = turned(s["k"], s["k_norm"])
    s["v_cache"][page, :, off] = s["v"]
    return {"q": turned(s["q"], s["q_norm"]), "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _plain_attention(s):
    case, q, table = s["case"], s["q"], s["table"]
    T, Hq, D = q.shape
    Hkv, P, B = case["Hkv"], case["page"], case["B"]
    G, Q, S = Hq // Hkv, s["max_q"], table.shape[1] * P
    seq = s["seq_lens"].long()
    cu = torch.arange(B + 1, device="cuda") if s["cu_q"] is None else s["cu_q"].long()
    rows = cu[1:] - cu[:-1]
    i = torch.arange(Q, device="cuda")
    qp = q[(cu[:-1, None] + i[None]).clamp(max=T - 1)].float()  # [B, Q, Hq, D]
    qp = qp.view(B, Q, Hkv, G, D).permute(0, 2, 3, 1, 4).reshape(B, Hkv, G * Q, D)
    j = torch.arange(S, device="cuda")
    keys = s["k_cache"][table.long()].transpose(1, 2).reshape(B, Hkv, S, D).float()
    score = (qp @ keys.transpose(2, 3)).view(B, Hkv, G, Q, S)
    del keys
    at = seq[:, None] - rows[:, None] + i[None]  # each row's own position, [B, Q]
    seen = j <= at[..., None]
    if case["window"]:
        seen = seen & (j > at[..., None] - case["window"])
    score = torch.where(seen[:, None, None], score * D ** -0.5, -math.inf)
    top = score.amax(-1, keepdim=True)
    prob = torch.exp(score - torch.where(top == -math.inf, 0.0, top))
    del score
    mass = prob.sum(-1, keepdim=True)
    values = s["v_cache"][table.long()].transpose(1, 2).reshape(B, Hkv, S, D).float()
    values = torch.where((j[None] < seq[:, None])[:, None, :, None], values, 0.0)
    out = (prob.view(B, Hkv, G * Q, S) @ values).view(B, Hkv, G, Q, D) / torch.where(mass == 0, 1.0, mass)
    del prob, values
    t = torch.arange(T, device="cuda")
    b = torch.searchsorted(cu[1:].contiguous(), t, right=True)
    out = out[b, :, :, t - cu[b]].reshape(T, Hq, D)
    if s["gate"] is not None:
        out = out / (1 + torch.exp(-s["gate"].float()))
    got = {"out": out.to(q.dtype)}
    if case["lse"]:
        got["lse"] = (top + torch.log(mass))[b, :, :, t - cu[b], 0].reshape(T, Hq)
    return got


# ------------------------------------------------------------------ the framework's calls

def _own_plan(s):
    from runnel_b200 import attention

    p = attention.kv_plan(s["table"], s["ctx"], s["new"], s["free_pages"], s["free_count"], page_size=s["case"]["page"],
                          num_pages=s["num_pages"], max_tokens=s["max_tokens"])
    return {"table": s["table"], "seq_lens": p.seq_lens, "cu_q": p.cu_q, "positions": p.positions, "slots": p.slots,
            "free_count": p.free_count}


def _own_rope(s):
    from runnel_b200 import attention

    case = s["case"]
    q = attention.rope_append(s["q"], s["k"], s["v"], s["positions"], s["inv_freq"], s["slots"], s["k_cache"],
                              s["v_cache"], sections=_sections(case), interleaved=case["interleaved"],
                              q_norm=s["q_norm"], k_norm=s["k_norm"], eps=1e-6)
    return {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _own_attention(s):
    from runnel_b200 import attention

    case = s["case"]
    got = attention.paged_attention(s["q"], s["k_cache"], s["v_cache"], s["table"], s["seq_lens"], cu_q=s["cu_q"],
                                    max_q=s["max_q"], window=case["window"], gate=s["gate"], return_lse=case["lse"])
    return {"out": got[0], "lse": got[1]} if case["lse"] else {"out": got}


def run(state):
    op = state["case"]["op"]
    if own:
        return {"plan": _own_plan, "rope": _own_rope, "attention": _own_attention}[op](state)
    return {"plan": _plain_plan, "rope": _plain_rope, "attention": _plain_attention}[op](state)


# ------------------------------------------------------------------ work

def work(case):
    if case["op"] == "plan":
        lens, P = _lens(case), case["page"]
        T, B = sum(n for _, n in lens), len(lens)
        fresh = sum(-(-(c + n) // P) - -(-c // P) for c, n in lens)
        begun = sum(1 for c, n in lens if n and c % P)  # pages half full: their table entries are read
        return {"bytes": 4 * (4 * B + 2 * fresh + begun + 2 * (T + max(1, T // 8)) + 3), "flops": 0}
    D, Hq, Hkv = case["D"], case["Hq"], case["Hkv"]
    if case["op"] == "rope":
        T, rot = case["T"], case["rot"]
        return {"bytes": T * (4 * (Hq + 2 * Hkv) * D + 4 * case["axes"] + 4) + 2 * rot + (4 * D if case["norm"] else 0),
                "flops": T * (Hq + Hkv) * (3 * rot + (4 * D if case["norm"] else 0))}
    kv, rows = _kv_q(case)
    T, w = sum(rows), case["window"]
    read = pairs = 0
    for n, r in zip(kv, rows):
        if r:
            read += min(n, w + r - 1) if w else n
            pairs += _seen(n, w) - _seen(n - r, w)
    return {"bytes": 4 * read * Hkv * D + T * Hq * (D * (6 if case["gate"] else 4) + (4 if case["lse"] else 0)),
            "flops": 4 * pairs * Hq * D}


def _seen(n, w):
    """How many (row, key) pairs the first n rows of a causal mask have, each row seeing its last w keys."""
    n = max(n, 0)
    return n * (n + 1) // 2 if not w or n <= w else w * (w + 1) // 2 + (n - w) * w


# ------------------------------------------------------------------ definitions in 64 bits

def _exact_rope(s, case):
    n, P = case["rot"] // 2, case["page"]
    sec = _sections(case)
    axis = [0] * n
    for a in range(1, len(sec)):
        for m in range(sec[a]):
            axis[a + 3 * m if case["interleaved"] else sum(sec[:a]) + m] = a
    turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"),
                       torch.stack([s["positions"][a].double() * float(s["inv_freq"][f])
                                    for f, a in enumerate(axis)], 1))

    def turned(x, w):
        x = x.double()
        if w is not None:
            x = x / (x.square().sum(-1, keepdim=True) / x.shape[-1] + 1e-6).sqrt() * w.double()
        z = torch.complex(x[..., :n], x[..., n:2 * n]) * turn[:, None]
        return torch.cat([z.real, z.imag, x[..., 2 * n:]], -1)

    k, v = s["k_cache"].double(), s["v_cache"].double()
    flat_k, flat_v = k.transpose(1, 2).reshape(-1, *s["k"].shape[1:]), v.transpose(1, 2).reshape(-1, *s["v"].shape[1:])
    flat_k[s["slots"].long()], flat_v[s["slots"].long()] = turned(s["k"], s["k_norm"]), s["v"].double()
    back = lambda f: f.view(-1, P, *f.shape[1:]).transpose(1, 2).contiguous()  # noqa: E731
    return {"q": turned(s["q"], s["q_norm"]), "k_cache": back(flat_k), "v_cache": back(flat_v)}


def _exact_attention(s, case):
    q = s["q"]
    T, Hq, D = q.shape
    G, w = Hq // case["Hkv"], case["window"]
    kv, rows = _kv_q(case)
    out = torch.zeros(T, Hq, D, dtype=torch.float64, device="cuda")
    lse = torch.full((T, Hq), -math.inf, dtype=torch.float64, device="cuda")
    first = 0
    for b, (n, r) in enumerate(zip(kv, rows)):
        if n and r:
            pages = s["table"][b, :-(-n // case["page"])].long()
            k = s["k_cache"][pages].transpose(1, 2).reshape(-1, case["Hkv"], D)[:n].double()
            v = s["v_cache"][pages].transpose(1, 2).reshape(-1, case["Hkv"], D)[:n].double()
            for h in range(Hq):
                for lo in range(0, r, 2048):
                    m = min(2048, r - lo)
                    a = q[first + lo:first + lo + m, h].double() @ k[:, h // G].T / math.sqrt(D)
                    p = torch.arange(n - r + lo, n - r + lo + m, device="cuda")[:, None] - torch.arange(n, device="cuda")
                    a.masked_fill_((p < 0) | (p >= w) if w else p < 0, -math.inf)
                    z = torch.logsumexp(a, -1)
                    lse[first + lo:first + lo + m, h] = z
                    out[first + lo:first + lo + m, h] = torch.exp(a - z[:, None]) @ v[:, h // G]
        first += r
    if s["gate"] is not None:
        out = out * torch.sigmoid(s["gate"].double())
    return {"out": out, "lse": lse} if case["lse"] else {"out": out}


def exact(case, seed):
    if case["op"] == "plan":
        return None
    s = prepare(case, seed)
    return _exact_rope(s, case) if case["op"] == "rope" else _exact_attention(s, case)
