"""The operators beside the attention layer that are measured: rotary positions over several axes (fused into the
qk-norm + pack, and alone), attention with a sliding window and always-visible first tokens, and low-rank adapters of
many requests beside a shared projection.

`run` computes them in plain torch operations (own = False) or through the framework's entry points (own = True)."""
import math
import os
import sys

import torch

own = False

D = 128
EPS = 1e-6


def _ops():
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "minimaxh3-on-a100-x4_b200")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import h3attn
    return h3attn


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one rank's token shard of an 8-way 42000-token video: norm + (t, h, w) rotary + send buffer
        {"name": "pack rank of 8", "op": "pack", "s": 5250, "heads": 56, "world": 8, "axes": 3, "mixed": False,
         "real": False},
        # the whole packed sequence on one GPU, fractional positions, axes interleaved over the pairs
        {"name": "pack 42000", "op": "pack", "s": 42000, "heads": 56, "world": 1, "axes": 3, "mixed": True,
         "real": True},
        # a short text-to-image call: latency
        {"name": "pack short", "op": "pack", "s": 77, "heads": 56, "world": 2, "axes": 3, "mixed": False,
         "real": False},
        # one new token's keys rotated on their way into a cache: latency
        {"name": "rope one token", "op": "rope", "s": 1, "heads": 56, "axes": 3, "mixed": False, "real": False,
         "inverse": False},
        # the gradient of the rotation over a rank's query heads of a long video
        {"name": "rope inverse 40868", "op": "rope", "s": 40868, "heads": 28, "axes": 3, "mixed": False,
         "real": True, "inverse": True},
        # one token over a windowed cache, the prompt staying visible: latency
        {"name": "window one token", "op": "window", "s_q": 1, "s_kv": 42000, "heads": 56, "kv_heads": 56,
         "left": 1023, "right": 0, "sinks": 512, "causal": True, "token_major": False},
        # a few tokens over a long cache with shared key heads and no left bound: the cache's bandwidth counts
        {"name": "window cache stream", "op": "window", "s_q": 5, "s_kv": 168000, "heads": 56, "kv_heads": 8,
         "left": -1, "right": 0, "sinks": 0, "causal": True, "token_major": False},
        # a medium clip, narrow two-sided window
        {"name": "window 4096", "op": "window", "s_q": 4096, "s_kv": 4096, "heads": 28, "kv_heads": 28,
         "left": 511, "right": 512, "sinks": 64, "causal": False, "token_major": True},
        # one rank of a 4-way 42000-token video, text prefix visible to every token
        {"name": "window 42000", "op": "window", "s_q": 42000, "s_kv": 42000, "heads": 14, "kv_heads": 14,
         "left": 2048, "right": 2048, "sinks": 512, "causal": False, "token_major": False},
        # the modulation rows of a step (a few rows, short inner size, wide output): latency
        {"name": "adapters modulation", "op": "lora", "m": 4, "k": 256, "n": 32256, "rank": 16, "adapters": 2,
         "scattered": False},
        # single tokens of many requests, each with its own adapter, beside the qkv projection
        {"name": "adapters many requests", "op": "lora", "m": 37, "k": 5376, "n": 21504, "rank": 16, "adapters": 24,
         "scattered": True},
        # a whole sequence through the output projection, one adapter per segment
        {"name": "adapters 42000", "op": "lora", "m": 42000, "k": 7168, "n": 5376, "rank": 32, "adapters": 4,
         "scattered": False},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["pack", "rope", "window", "window", "lora", "lora"])
    if op in ("pack", "rope"):
        c = {"op": op, "s": _log(rng, 1, 42000), "axes": rng.choice([1, 2, 3, 3, 4]), "mixed": rng.random() < 0.5,
             "real": rng.random() < 0.5}
        if op == "pack":
            world = rng.choice([1, 2, 4])
            return dict(c, heads=world * rng.randint(1, 56 // world), world=world)
        return dict(c, heads=rng.randint(1, 56), inverse=rng.random() < 0.5)
    if op == "window":
        group = rng.choice([1, 1, 2, 5, 7, 8])
        kv_heads = rng.randint(1, max(1, 28 // group))
        c = {"op": op, "kv_heads": kv_heads, "heads": kv_heads * group, "sinks": rng.choice([0, rng.randint(1, 700)]),
             "causal": rng.random() < 0.5, "token_major": rng.random() < 0.5}
        if rng.random() < 0.5:  # new tokens over a cache
            s_q = _log(rng, 1, 64)
            s_kv = s_q + _log(rng, 1, 100000)
            return dict(c, s_q=s_q, s_kv=s_kv, left=rng.choice([-1, _log(rng, 1, 16000)]), right=0)
        s = _log(rng, 65, 12000)
        return dict(c, s_q=s, s_kv=s, left=_log(rng, 1, 4000), right=rng.choice([0, _log(rng, 1, 2000)]))
    return {"op": op, "m": _log(rng, 1, 20000), "k": 8 * _log(rng, 8, 896), "n": 8 * _log(rng, 16, 1000),
            "rank": rng.choice([8, 16, 32, 64, 128]), "adapters": _log(rng, 1, 32), "scattered": rng.random() < 0.5}


# ------------------------------------------------------------------------------------------------ inputs
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _randn(g, *shape, std=1.0):
    return (torch.randn(*shape, generator=g, device="cuda") * std).to(torch.bfloat16)


def _positions(case, g):
    """Token positions [s, axes]: raster order over a (.., time, height, width) grid from a random origin; real:
    the first axis in fractions of a frame, as audio and video of different rates share it."""
    s, axes = case["s"], case["axes"]
    i = torch.arange(s, device="cuda")
    w, h = 60, 34
    cols = [i // (w * h), (i // w) % h, i % w, i % 7][:axes] if axes > 1 else [i]
    pos = torch.stack(cols, 1) + torch.randint(0, 5000, (axes,), generator=g, device="cuda")
    if case["real"]:
        pos = pos.to(torch.float32)
        pos[:, 0] *= 0.3125 + float(torch.rand((), generator=g, device="cuda"))
        return pos.contiguous()
    return pos.to(torch.int32).contiguous()


def _frequencies(case):
    """(inv_freq [64] fp64, axis [64] int32): each axis turns its own pairs with its own geometric series; mixed:
    pair by pair in turn, else one run of pairs per axis. The last pairs of a 4-axis plan do not turn (axis -1)."""
    axes = case["axes"]
    sizes = {1: [64], 2: [32, 32], 3: [16, 24, 24], 4: [12, 20, 20, 8]}[axes]
    pairs = [(j, a) for a in range(axes) for j in range(sizes[a])]
    pairs = sorted(pairs) if case["mixed"] else pairs
    axis = [a for _, a in pairs]
    inv = [10000.0 ** (-j / sizes[a]) for j, a in pairs]
    rest = 64 - len(axis)
    return (torch.tensor(inv + [0.0] * rest, dtype=torch.float64, device="cuda"),
            torch.tensor(axis + [-1] * rest, dtype=torch.int32, device="cuda"))


def prepare(case, seed):
    g = _gen(seed)
    op = case["op"]
    st = {"case": case}
    if op in ("pack", "rope"):
        st["pos"] = _positions(case, g)
        st["inv_freq"], st["axis"] = _frequencies(case)
        s, h = case["s"], case["heads"]
        if op == "pack":  # q, k, v are column blocks of the fused projection's output
            st["q"], st["k"], st["v"] = _randn(g, s, 3 * h * D).split(h * D, dim=-1)
            st["qw"], st["kw"] = _randn(g, D, std=0.1) + 1, _randn(g, D, std=0.1) + 1
        else:
            st["x"] = _randn(g, s, h, D)
    elif op == "window":
        h, hk, s_q, s_kv = case["heads"], case["kv_heads"], case["s_q"], case["s_kv"]
        if case["token_major"]:
            st["q"] = _randn(g, s_q, h, D).transpose(0, 1)
            st["k"], st["v"] = (_randn(g, s_kv, hk, D).transpose(0, 1) for _ in range(2))
        else:  # head-major; the cache has room for more keys than it holds
            st["q"] = _randn(g, h, s_q, D)
            st["k"], st["v"] = (_randn(g, hk, s_kv + 256, D)[:, :s_kv] for _ in range(2))
    else:
        m, k, n, r, na = case["m"], case["k"], case["n"], case["rank"], case["adapters"]
        st["x"] = _randn(g, m, k)
        st["w"] = _randn(g, n, k, std=0.02)
        st["a"] = _randn(g, na * r, k, std=k ** -0.5)
        st["b"] = _randn(g, n, na * r, std=0.05)
        st["scale"] = 0.5 + torch.rand(na, generator=g, device="cuda")
        if case["scattered"]:  # every row its own request; some without an adapter
            st["rows"] = torch.randint(-1, na, (m,), generator=g, device="cuda").to(torch.int32)
        else:                  # one segment per request, the last one without an adapter
            st["rows"] = (torch.arange(m, device="cuda") * (na + 1) // m).to(torch.int32)
            st["rows"][st["rows"] == na] = -1
    return st


# ------------------------------------------------------------------------------------------------ plain forms
def _turn(x, pos, inv_freq, axis, inverse):
    """Pairs (i, i + 64) of x [s, heads, 128] (fp32) turned by pos[:, axis_i] * inv_freq_i."""
    along = pos.double()[:, axis.clamp_min(0).long()] * (axis >= 0)
    ang = (along * inv_freq)[:, None]
    c, s = ang.cos().float(), ang.sin().float()
    s = -s if inverse else s
    a, b = x[..., :64], x[..., 64:]
    return torch.cat([a * c - b * s, a * s + b * c], -1)


def _plain_pack(st):
    c = st["case"]
    s, h, w = c["s"], c["heads"], c["world"]
    q, k, v = (st[n].float().view(s, h, D) for n in "qkv")

    def one(x, weight):
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * weight.float()
        return _turn(x, st["pos"], st["inv_freq"], st["axis"], False)

    out = torch.stack([one(q, st["qw"]), one(k, st["kw"]), v])  # [3, s, h, D]
    return out.view(3, s, w, h // w, D).permute(2, 0, 3, 1, 4).to(torch.bfloat16).contiguous()


def _sides(case):
    left = case["s_kv"] if case["left"] < 0 else min(case["left"], case["s_kv"])
    return left, 0 if case["causal"] else case["right"]


def _plain_window(st):
    """Blocks of queries against the run of keys that one of them can see, plus the first tokens."""
    c = st["case"]
    h, hk, s_q, s_kv, sinks = c["heads"], c["kv_heads"], c["s_q"], c["s_kv"], min(c["sinks"], c["s_kv"])
    left, right = _sides(c)
    dev = st["q"].device
    blk = min(512, s_q)
    nb = -(-s_q // blk)
    q = st["q"].float() * D ** -0.5
    q = torch.cat([q, q.new_zeros(h, nb * blk - s_q, D)], 1).view(hk, h // hk, nb, blk, D).transpose(1, 2)
    q = q.reshape(hk, nb, h // hk * blk, D)
    p = s_kv - s_q + torch.arange(nb * blk, device=dev).view(nb, blk)
    j = p[:, :1] - left + torch.arange(left + right + blk, device=dev)  # [nb, keys]
    at = j.clamp(0, s_kv - 1)
    near, first_k, first_v = (t.float() for t in (st["k"][:, at], st["k"][:, :sinks], st["v"][:, :sinks]))
    far = (j < sinks) | (j < 0) | (j >= s_kv)
    hidden = far[:, None] | (j[:, None] < p[..., None] - left) | (j[:, None] > p[..., None] + right)
    sc = torch.matmul(q, near.transpose(-1, -2))                        # [hk, nb, g * blk, keys]
    sc.view(hk, nb, h // hk, blk, -1).masked_fill_(hidden[:, None], -math.inf)
    first = torch.matmul(q.view(hk, -1, D), first_k.transpose(-1, -2)).view(hk, nb, h // hk, blk, sinks)
    if c["causal"]:
        first.masked_fill_((torch.arange(sinks, device=dev) > p[..., None])[:, None], -math.inf)
    first = first.view(hk, nb, h // hk * blk, sinks)
    top = sc.amax(-1, keepdim=True)
    top = torch.maximum(top, first.amax(-1, keepdim=True)) if sinks else top
    top = top.clamp_min(torch.finfo(torch.float32).min)
    sc, first = sc.sub_(top).exp_(), first.sub_(top).exp_()
    o = torch.matmul(sc, st["v"][:, at].float())
    o += torch.matmul(first.view(hk, nb * h // hk * blk, sinks), first_v).view_as(o)
    o = o / (sc.sum(-1, keepdim=True) + first.sum(-1, keepdim=True)).clamp_min(1e-30)
    o = o.view(hk, nb, h // hk, blk, D).transpose(1, 2).reshape(h, nb * blk, D)
    return o[:, :s_q].to(torch.bfloat16).contiguous()


def _plain_lora(st):
    r, rows = st["case"]["rank"], st["rows"]
    x = st["x"].float()
    t = x @ st["a"].float().T                                          # every adapter's columns
    mine = rows[:, None] == (torch.arange(t.shape[1], device=t.device) // r)
    t = t * mine * st["scale"].repeat_interleave(r)
    y = x @ st["w"].float().T
    return y.addmm_(t, st["b"].float().T).to(torch.bfloat16)


def run(state):
    c = state["case"]
    op = c["op"]
    if not own:
        if op == "pack":
            return _plain_pack(state)
        if op == "rope":
            return _turn(state["x"].float(), state["pos"], state["inv_freq"], state["axis"],
                         c["inverse"]).to(torch.bfloat16)
        return _plain_window(state) if op == "window" else _plain_lora(state)
    O = _ops()
    if op == "pack":
        rope = O.RopePositions(state["pos"], state["inv_freq"], state["axis"])
        return O.qknorm_rope_pack(state["q"], state["k"], state["v"], rope, state["qw"], state["kw"], EPS, c["world"])
    if op == "rope":
        rope = O.RopePositions(state["pos"], state["inv_freq"], state["axis"])
        return O.rope_axes(state["x"], rope, inverse=c["inverse"])
    if op == "window":
        return O.window_attention(state["q"], state["k"], state["v"], left=None if c["left"] < 0 else c["left"],
                                  right=c["right"], sinks=c["sinks"], causal=c["causal"])
    return O.linear_lora(state["x"], state["w"], state["a"], state["b"], state["scale"], state["rows"])


# ------------------------------------------------------------------------------------------------ work
def _visible(case):
    """(query, key) pairs of one head that see each other, and the keys that some query sees."""
    s_q, s_kv, sinks = case["s_q"], case["s_kv"], min(case["sinks"], case["s_kv"])
    left, right = _sides(case)
    p = s_kv - s_q + torch.arange(s_q)
    lo, hi = (p - left).clamp_min(0), (p + right).clamp_max(s_kv - 1)
    first = torch.minimum(p + 1, torch.tensor(sinks)) if case["causal"] else torch.full_like(p, sinks)
    pairs = (hi - torch.maximum(lo, first) + 1).clamp_min(0) + first
    keys = int(hi.max()) + 1 - max(int(lo.min()), sinks)
    return int(pairs.sum()), max(keys, 0) + sinks


def work(case):
    op = case["op"]
    if op in ("pack", "rope"):
        tensors = 3 if op == "pack" else 1
        n = case["s"] * case["heads"] * D
        turned = n * (2 if op == "pack" else 1)
        return {"bytes": 2 * 2 * tensors * n + 4 * case["s"] * case["axes"],
                "flops": turned * (7 if op == "pack" else 3)}
    if op == "window":
        pairs, keys = _visible(case)
        return {"bytes": 2 * D * (2 * case["heads"] * case["s_q"] + 2 * case["kv_heads"] * keys),
                "flops": 4 * D * case["heads"] * pairs}
    m, k, n, r = case["m"], case["k"], case["n"], case["rank"]
    used = min(case["adapters"], m)
    return {"bytes": 2 * (m * k + n * k + m * n + used * r * (k + n)) + 4 * m,
            "flops": 2 * m * k * n + 2 * m * r * (k + n)}


# ------------------------------------------------------------------------------------------------ 64 bits
def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]
    if op in ("pack", "rope"):
        axis = st["axis"].long()
        still = axis < 0
        angle = torch.gather(st["pos"].double(), 1, axis.masked_fill(still, 0).expand(case["s"], 64))
        angle = (angle * st["inv_freq"]).masked_fill(still, 0.0)
        turn = torch.polar(torch.ones_like(angle), -angle if case.get("inverse") else angle)[:, None]

        def rotate(x):
            z = torch.complex(x[..., :64].contiguous(), x[..., 64:].contiguous()) * turn
            return torch.cat([z.real, z.imag], -1)

        if op == "rope":
            return rotate(st["x"].double())
        s, h, w = case["s"], case["heads"], case["world"]
        out = torch.empty(w, 3, h // w, s, D, dtype=torch.float64, device="cuda")
        for i, name in enumerate("qkv"):
            x = st[name].double().reshape(s, h, D)
            if name != "v":
                x = rotate(x / (x.pow(2).sum(-1, keepdim=True) / D + EPS).sqrt() * st[name + "w"].double())
            out[:, i] = x.reshape(s, w, h // w, D).permute(1, 2, 0, 3)
        return out
    if op == "lora":
        x, y = st["x"].double(), torch.empty(case["m"], case["n"], dtype=torch.float64, device="cuda")
        for c in range(0, case["n"], 8192):
            y[:, c:c + 8192] = x @ st["w"][c:c + 8192].double().T
        r = case["rank"]
        for i in range(case["adapters"]):
            at = (st["rows"] == i).nonzero()[:, 0]
            low = (x[at] @ st["a"][i * r:(i + 1) * r].double().T) * st["scale"][i].double()
            y[at] += low @ st["b"][:, i * r:(i + 1) * r].double().T
        return y
    h, hk, s_q, s_kv, sinks = case["heads"], case["kv_heads"], case["s_q"], case["s_kv"], case["sinks"]
    left = case["left"] if case["left"] >= 0 else s_kv + s_q
    right = case["right"]
    o = torch.zeros(h, s_q, D, dtype=torch.float64, device="cuda")
    for i0 in range(0, s_q, 2048):
        i1 = min(i0 + 2048, s_q)
        p = torch.arange(i0, i1, device="cuda") + (s_kv - s_q)
        lo, hi = max(int(p[0]) - left, 0), min(int(p[-1]) + right, s_kv - 1)
        near = torch.arange(s_kv, device="cuda")
        near = near[(near < sinks) | ((near >= lo) & (near <= hi))]
        see = (near < sinks) | ((near >= p[:, None] - left) & (near <= p[:, None] + right))
        if case["causal"]:
            see &= near <= p[:, None]
        for head in range(h):
            kv = head * hk // h
            sc = (st["q"][head, i0:i1].double() @ st["k"][kv, near].double().T) / math.sqrt(D)
            wt = torch.exp(sc - sc.masked_fill(~see, -math.inf).amax(-1, keepdim=True).clamp_min(-1e300)) * see
            o[head, i0:i1] = (wt @ st["v"][kv, near].double()) / wt.sum(-1, keepdim=True).clamp_min(1e-300)
    return o
