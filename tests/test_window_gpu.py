"""Windowed attention with first tokens that stay visible, against the definition in 64 bits.

Tolerance, element by element. The weights p_j are rounded to bf16 for the second product (2^-8 p_j each) and the
output once (2^-8 |o|). fp32 sums of 128 products in a score of size up to ~8 and of the weights, the exponential
(2^-22) and the fp32 accumulation of O stay below 2^-12 of sum_j p_j |v_j|. So
|o - ref| <= 2^-8 |ref| + (2^-8 + 2^-12) sum_j p_j |v_j|."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
D = 128


def _rand(shape, seed, dev):
    g = torch.Generator(device="cpu").manual_seed(seed)
    return torch.randn(shape, generator=g).to(torch.bfloat16).to(dev)


def _reference(q, k, v, left, right, sinks, causal, q_start, s_kv, scale=D ** -0.5):
    """(o, sum p |v|) in fp64; zeros where a query sees no key."""
    H, sq, _ = q.shape
    k, v = (t[:, :s_kv].double().repeat_interleave(H // k.shape[0], 0) for t in (k, v))
    p = q_start + torch.arange(sq, device=q.device)[:, None]
    j = torch.arange(s_kv, device=q.device)[None]
    near = torch.ones_like(p + j, dtype=torch.bool)
    if left is not None:
        near &= j >= p - left
    if right is not None:
        near &= j <= p + right
    see = near | (j < sinks)
    if causal:
        see &= j <= p
    s = (q.double() @ k.transpose(1, 2) * scale).masked_fill(~see, -math.inf)
    m = s.amax(-1, keepdim=True)
    w = torch.exp(s - torch.where(m == -math.inf, torch.zeros_like(m), m))
    w = w / w.sum(-1, keepdim=True).clamp_min(1e-300)
    v = torch.where((see.any(0) if see.dim() == 2 else see)[None, :, None], v, torch.zeros_like(v))
    return w @ v, w @ v.abs()


def _check(got, ref, mag):
    err = (got.double() - ref).abs()
    bound = 2 ** -8 * ref.abs() + (2 ** -8 + 2 ** -12) * mag
    assert bool((err <= bound).all()), ((err - bound).max().item(), err.max().item())


def _run(O, q, k, v, left, right, sinks=0, causal=False, q_start=None, s_kv=None, **kw):
    o = O.window_attention(q, k, v, left, right, sinks=sinks, causal=causal, q_start=q_start, s_kv=s_kv, **kw)
    O.check_status()
    s_kv = k.shape[1] if s_kv is None else s_kv
    q_start = max(s_kv - q.shape[1], 0) if q_start is None else q_start
    return o, _reference(q, k, v, left, right, sinks, causal, q_start, s_kv)


# (heads, key heads, queries, keys, left, right, sinks, causal)
CASES = [
    (1, 1, 1, 1, 0, 0, 0, False), (2, 1, 1, 2, 0, 0, 1, True), (3, 3, 127, 127, 5, 5, 0, False),
    (2, 2, 128, 128, 0, 0, 0, False), (2, 2, 129, 129, 0, 0, 0, True), (2, 2, 255, 255, 1, 0, 4, True),
    (2, 2, 300, 300, None, None, 0, False), (2, 2, 300, 300, None, 0, 0, True), (2, 1, 513, 513, 100, 27, 64, False),
    (4, 2, 700, 700, 128, 128, 130, False), (7, 1, 333, 333, 31, 0, 3, True), (10, 2, 260, 260, 64, 1, 128, False),
    (8, 1, 1000, 1000, 200, 50, 700, False), (3, 3, 1500, 1500, 300, 0, 512, True), (2, 2, 900, 900, 0, 511, 0, False),
    (16, 16, 1, 4000, 500, 0, 100, True), (56, 8, 1, 3001, None, 0, 0, True), (56, 8, 5, 2777, 1023, 0, 17, True),
    (128, 1, 3, 1111, 400, 0, 9, False), (129, 3, 2, 600, 100, 0, 9, False), (6, 2, 64, 5000, 2000, 0, 256, True),
    (1, 1, 64, 9000, None, None, 0, False), (1, 1, 200, 20000, 9000, 0, 1, True),
]


@pytest.mark.parametrize("case", CASES, ids=str)
def test_against_the_definition(cuda_dev, case):
    import h3attn as O
    H, hk, sq, skv, left, right, sinks, causal = case
    q, k, v = _rand((H, sq, D), 1, cuda_dev), _rand((hk, skv, D), 2, cuda_dev), _rand((hk, skv, D), 3, cuda_dev)
    o, (ref, mag) = _run(O, q, k, v, left, right, sinks, causal)
    _check(o, ref, mag)


# more blocks of queries than the GPU holds CTAs: (heads, key heads, queries, keys, left, right, sinks, causal, q_start)
MANY = [(40, 40, 1500, 1500, 70, 30, 20, False, 0), (48, 24, 1000, 1000, None, 0, 0, True, 0),
        (300, 300, 130, 600, 100, 0, 200, True, 470), (64, 64, 900, 400, 10, 10, 0, False, -450),
        (64, 64, 900, 300, 40, 0, 7, True, 0), (400, 400, 20, 500, 120, 5, 30, False, 200),
        (600, 300, 50, 350, 3, 0, 0, True, 320), (350, 350, 9, 200, 1, 1, 0, False, 150)]


@pytest.mark.parametrize("case", MANY, ids=str)
@pytest.mark.parametrize("splits", [None, 1])
def test_more_blocks_than_ctas(cuda_dev, case, splits):
    import h3attn as O
    H, hk, sq, skv, left, right, sinks, causal, q_start = case
    q, k, v = _rand((H, sq, D), 1, cuda_dev), _rand((hk, skv, D), 2, cuda_dev), _rand((hk, skv, D), 3, cuda_dev)
    out = torch.full((H, sq, D), 9.0, dtype=torch.bfloat16, device=cuda_dev)
    o, (ref, mag) = _run(O, q, k, v, left, right, sinks, causal, q_start, out=out, splits=splits)
    _check(o, ref, mag)
    assert torch.equal(o, O.window_attention(q, k, v, left, right, sinks=sinks, causal=causal, q_start=q_start,
                                             splits=splits))


@pytest.mark.parametrize("H,hk", [(1, 1), (20, 20), (40, 20), (57, 19), (80, 20), (100, 20), (60, 60), (240, 60)])
@pytest.mark.parametrize("skv,left,right,sinks,q_start", [
    (1, 0, 0, 0, 0), (2, 0, 0, 1, 1), (63, None, 0, 0, 62), (64, 10, 0, 5, 63), (129, None, None, 0, 60),
    (1000, 300, 0, 100, 999), (1000, 300, 20, 700, 800), (5000, 4097, 0, 3, 4999), (777, 5, 5, 0, 5000),
    (777, 5, 5, 9, 5000), (777, 40, 0, 0, -3)])
def test_single_tokens(cuda_dev, H, hk, skv, left, right, sinks, q_start):
    """One query position over a cache: groups of 1 to 4 query heads to a key head have a kernel of their own, 5 go
    through the tiles; one, two or no runs of keys, and NaN wherever the token does not look."""
    import h3attn as O
    q, k, v = _rand((H, 1, D), 1, cuda_dev), _rand((hk, skv + 9, D), 2, cuda_dev), _rand((hk, skv + 9, D), 3, cuda_dev)
    j = torch.arange(skv + 9, device=cuda_dev)
    seen = (j < sinks) | ((j >= q_start - (left if left is not None else 10 ** 6)) &
                          (j <= q_start + (right if right is not None else 10 ** 6)))
    k[:, ~seen | (j >= skv)] = float("nan")
    v[:, ~seen | (j >= skv)] = float("inf")
    out = torch.full((H, 1, D), 5.0, dtype=torch.bfloat16, device=cuda_dev)
    o = O.window_attention(q, k, v, left, right, sinks=sinks, q_start=q_start, s_kv=skv, out=out)
    O.check_status()
    k, v = (torch.where(seen[None, :, None], t, torch.zeros_like(t)) for t in (k, v))
    ref, mag = _reference(q, k, v, left, right, sinks, False, q_start, skv)
    _check(o, ref, mag)
    token = O.window_attention(q, k, v, left, right, sinks=sinks, q_start=q_start, s_kv=skv, layout="token")
    assert torch.equal(token.view(H, 1, D), o)


@pytest.mark.parametrize("splits", [1, 2, 3, 7, 64])
def test_any_number_of_splits(cuda_dev, splits):
    import h3attn as O
    q, k, v = _rand((4, 70, D), 4, cuda_dev), _rand((2, 1200, D), 5, cuda_dev), _rand((2, 1200, D), 6, cuda_dev)
    o, (ref, mag) = _run(O, q, k, v, 600, 0, 40, True, splits=splits)
    _check(o, ref, mag)
    assert torch.equal(o, O.window_attention(q, k, v, 600, 0, sinks=40, causal=True, splits=splits))


@pytest.mark.parametrize("q_start", [-500, -100, -1, 0, 50, 399, 400, 700])
@pytest.mark.parametrize("causal,sinks", [(False, 0), (True, 0), (True, 20), (False, 20)])
@pytest.mark.parametrize("splits", [1, 3])
def test_queries_that_see_nothing_get_zeros(cuda_dev, q_start, causal, sinks, splits):
    import h3attn as O
    q, k, v = _rand((2, 300, D), 7, cuda_dev), _rand((2, 400, D), 8, cuda_dev), _rand((2, 400, D), 9, cuda_dev)
    out = torch.full((2, 300, D), 7.0, dtype=torch.bfloat16, device=cuda_dev)
    o, (ref, mag) = _run(O, q, k, v, 60, 10, sinks, causal, q_start=q_start, out=out, splits=splits)
    _check(o, ref, mag)
    assert bool((o[ref == 0] == 0).all())


def test_unseen_keys_may_hold_anything(cuda_dev):
    """NaN and infinities in K and V at keys that no query sees, between and behind the visible runs, and past s_kv."""
    import h3attn as O
    q, k, v = _rand((2, 20, D), 10, cuda_dev), _rand((2, 1000, D), 11, cuda_dev), _rand((2, 1000, D), 12, cuda_dev)
    for splits in (1, 3):
        clean = O.window_attention(q, k, v, 90, 0, sinks=70, causal=True, s_kv=900, q_start=640, splits=splits)
        dirty_k, dirty_v = k.clone(), v.clone()
        for t in (dirty_k, dirty_v):  # seen: [0, 70) and [550, 660)
            t[:, 70:550] = float("nan")
            t[:, 660:] = float("inf")
            t[:, 880:] = torch.finfo(torch.bfloat16).min
        dirty = O.window_attention(q, dirty_k, dirty_v, 90, 0, sinks=70, causal=True, s_kv=900, q_start=640,
                                   splits=splits)
        assert torch.equal(clean, dirty)
    # K alone may be anything for the rows that do not see it
    q1, k1 = _rand((1, 300, D), 13, cuda_dev), _rand((1, 300, D), 14, cuda_dev)
    k1[0, 150] = float("nan")
    o = O.window_attention(q1, k1, v[:1, :300], 3, 0, causal=True, q_start=0)
    bad = torch.isnan(o).any(-1)[0].nonzero()[:, 0].tolist()
    assert bad == [150, 151, 152, 153]


def test_large_scores_and_growing_maxima(cuda_dev):
    """Score maxima that grow along the walk (the accumulator is rescaled) and weights that underflow."""
    import h3attn as O
    q, k, v = _rand((2, 200, D), 15, cuda_dev), _rand((2, 1300, D), 16, cuda_dev), _rand((2, 1300, D), 17, cuda_dev)
    k *= torch.linspace(0.1, 4, 1300, device=cuda_dev)[None, :, None].to(torch.bfloat16)
    for flip in (k, k.flip(1).contiguous()):
        o = O.window_attention(q, flip, v, 700, 600, sinks=30, q_start=500)
        ref, mag = _reference(q, flip, v, 700, 600, 30, False, 500, 1300)
        # scores reach ~45: their fp32 sums carry 2^-18 each, a weight 2^-17 of itself more
        _check(o, ref, mag)


def test_strides_layouts_and_neighbours(cuda_dev):
    import h3attn as O
    H, hk, s = 4, 2, 390
    qkv = _rand((s, (H + 2 * hk) * D), 18, cuda_dev)
    q = qkv[:, :H * D].view(s, H, D).transpose(0, 1)
    k = qkv[:, H * D:(H + hk) * D].view(s, hk, D).transpose(0, 1)
    v = qkv[:, (H + hk) * D:].view(s, hk, D).transpose(0, 1)
    want = O.window_attention(q.contiguous(), k.contiguous(), v.contiguous(), 50, 20, sinks=10)
    assert torch.equal(O.window_attention(q, k, v, 50, 20, sinks=10), want)
    token = O.window_attention(q, k, v, 50, 20, sinks=10, layout="token")
    assert torch.equal(token.view(s, H, D).transpose(0, 1), want)
    send = O.window_attention(q, k, v, 50, 20, sinks=10, layout="send", world=3)  # [3, H, 130, D]
    assert torch.equal(send.permute(1, 0, 2, 3).reshape(H, s, D), want)
    cache_k, cache_v = (torch.full((hk, 600, D), float("nan"), dtype=torch.bfloat16, device=cuda_dev) for _ in "kv")
    cache_k[:, :s], cache_v[:, :s] = k, v
    assert torch.equal(O.window_attention(q, cache_k, cache_v, 50, 20, sinks=10, s_kv=s), want)
    assert torch.equal(O.window_attention(q, cache_k[:, :s], cache_v[:, :s], 50, 20, sinks=10), want)
    few = O.window_attention(q[:, -3:], cache_k, cache_v, 50, 20, sinks=10, s_kv=s, layout="token")
    assert few.shape == (3, H * D)


def test_full_window_equals_attention(cuda_dev):
    """No bounds: the dense attention operator's value, to both operators' tolerance."""
    import h3attn as O
    q, k, v = (_rand((3, 700, D), 19 + i, cuda_dev) for i in range(3))
    a, b = O.attention(q, k, v, s_kv=650), O.window_attention(q, k, v, None, None, s_kv=650)
    ref, mag = _reference(q, k, v, None, None, 0, False, 0, 650)
    for o in (a, b):
        _check(o, ref, mag)


def test_one_split_rows_do_not_depend_on_the_heads_of_the_call(cuda_dev):
    import h3attn as O
    q, k, v = (_rand((6, 640, D), 22 + i, cuda_dev) for i in range(3))
    whole = O.window_attention(q, k, v, 128, 64, sinks=32, splits=1)
    part = O.window_attention(q[2:4], k[2:4], v[2:4], 128, 64, sinks=32, splits=1)
    assert torch.equal(part, whole[2:4])


def test_streams_graphs_and_two_calls_at_once(cuda_dev):
    import h3attn as O
    q, k, v = _rand((8, 2, D), 25, cuda_dev), _rand((8, 3000, D), 26, cuda_dev), _rand((8, 3000, D), 27, cuda_dev)
    args = dict(left=2000, right=0, sinks=5, causal=True)
    want = O.window_attention(q, k, v, **args)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs = []
    for st in streams:
        with torch.cuda.stream(st):
            outs.append([O.window_attention(q, k, v, **args) for _ in range(4)])
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for some in outs for o in some)
    graphs, got = [], []
    for _ in range(2):  # two graphs, replayed at once on two streams
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            got.append(O.window_attention(q, k, v, **args))
        graphs.append(g)
    q.copy_(_rand((8, 2, D), 28, cuda_dev))
    torch.cuda.synchronize()
    for g, st in zip(graphs, streams):
        with torch.cuda.stream(st):
            g.replay()
    torch.cuda.synchronize()
    want = O.window_attention(q, k, v, **args)
    assert all(torch.equal(o, want) for o in got)
    O.check_status()


def test_refusals(cuda_dev):
    import h3attn as O
    q, k, v = (_rand((4, 64, D), 30 + i, cuda_dev) for i in range(3))
    bad = [lambda: O.window_attention(q.half(), k, v, 1, 1), lambda: O.window_attention(q[:, :, :64], k, v, 1, 1),
           lambda: O.window_attention(q, k[:3], v[:3], 1, 1), lambda: O.window_attention(q, k, v[:, :32], 1, 1),
           lambda: O.window_attention(q, k, v, -1, 1), lambda: O.window_attention(q, k, v, 1, -2),
           lambda: O.window_attention(q, k, v, 1, 1, sinks=-1), lambda: O.window_attention(q, k, v, 1, 1, s_kv=65),
           lambda: O.window_attention(q, k, v, 1, 1, s_kv=0), lambda: O.window_attention(q[:, :0], k, v, 1, 1),
           lambda: O.window_attention(q, k, v, 1, 1, splits=65), lambda: O.window_attention(q, k, v, 1, 1, splits=0),
           lambda: O.window_attention(q, k, v, 1, 1, layout="rows"),
           lambda: O.window_attention(q, k, v, 1, 1, layout="send", world=5),
           lambda: O.window_attention(q, k, v, 1, 1, out=q[:2]), lambda: O.window_attention(q, k, v, 1, 1, scale=0.0),
           lambda: O.window_attention(q, k, v, 1, 1, q_start=1 << 30),
           lambda: O.window_attention(q, k.transpose(0, 1).contiguous().transpose(0, 1), v, 1, 1)]
    for f in bad:
        with pytest.raises(O.H3Error):
            f()


def test_status_word_is_not_made_inside_a_capture(cuda_dev, monkeypatch):
    import h3attn as O
    monkeypatch.setattr(O, "_status", {})
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    q = _rand((2, 3, D), 40, cuda_dev)
    with pytest.raises(O.H3Error):
        O.window_attention(q, q, q, 1, 1)


FAR = 1 << 29  # the farthest position


@pytest.mark.parametrize("s_q", [1, 3, 140, 300])
@pytest.mark.parametrize("q_start,left,right,sinks,causal", [
    (-FAR, None, None, 0, False), (-FAR, 7, None, 5, False), (-FAR, None, FAR, 0, False), (-FAR, None, 2 * FAR, 0, False),
    (FAR, None, None, 0, False), (FAR, None, 0, 0, True), (FAR, FAR, 0, 9, True), (FAR, FAR - 40, 3, 0, False),
    (FAR, 2 * FAR, 0, 0, True), (FAR, 100, 100, 0, False), (-FAR, 100, 100, 30, True)])
def test_far_positions(cuda_dev, s_q, q_start, left, right, sinks, causal):
    """Sides without a bound have none at the ends of the range of positions either, and bounds of 2^29 are exact."""
    import h3attn as O
    q, k, v = _rand((4, s_q, D), 50, cuda_dev), _rand((2, 1000, D), 51, cuda_dev), _rand((2, 1000, D), 52, cuda_dev)
    for splits in (None, 1, 3):
        o, (ref, mag) = _run(O, q, k, v, left, right, sinks, causal, q_start, splits=splits)
        _check(o, ref, mag)


def test_far_sides_through_the_c_entry(cuda_dev):
    """The C call's own -1 and sides past 2^29, which the Python entry clips before."""
    import h3attn as O
    q, k, v = _rand((2, 40, D), 53, cuda_dev), _rand((2, 600, D), 54, cuda_dev), _rand((2, 600, D), 55, cuda_dev)
    out = torch.empty_like(q)
    st = O.status_word(cuda_dev)
    for q_start, left, right, want in ((-FAR, -1, -1, (None, None)), (FAR, -1, 0, (None, 0)), (FAR, FAR + 20, 0, (FAR + 20, 0)),
                                       (FAR, 1 << 62, 1 << 62, (None, None)), (-FAR, 0, FAR + 20, (0, FAR + 20))):
        rc = O.lib().h3_window_attn(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), 2, 2, 40, 600, 40 * D, D,
                                    600 * D, D, 40, 0, 40 * D, D, D ** -0.5, left, right, 0, 0, q_start, 1, None, 0,
                                    st.data_ptr(), torch.cuda.current_stream().cuda_stream)
        assert rc == 0
        O.check_status()
        _check(out, *_reference(q, k, v, *want, 0, False, q_start, 600))


@pytest.mark.parametrize("group", [2, 5])
def test_one_split_rows_do_not_depend_on_the_key_heads_of_the_call(cuda_dev, group):
    """Query heads of any key heads of the call, with the same number of them to a key head."""
    import h3attn as O
    q = _rand((4 * group, 500, D), 56, cuda_dev)
    k, v = (_rand((4, 500, D), 57 + i, cuda_dev) for i in range(2))
    whole = O.window_attention(q, k, v, 100, 30, sinks=20, splits=1)
    part = O.window_attention(q[group:3 * group], k[1:3], v[1:3], 100, 30, sinks=20, splits=1)
    assert torch.equal(part, whole[group:3 * group])
