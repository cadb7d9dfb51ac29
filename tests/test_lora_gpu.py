"""Projections with low-rank adapters per row, against the definition in 64 bits.

Tolerance, element by element. The tensor cores add 16 products at a time to an fp32 sum, so a sum over k products is off
by at most (k / 16 + 4) 2^-23 of the sum of their magnitudes (one step of the running sum each); T = s A x is rounded to
bf16 (2^-8 |T_j| for each j); y is rounded once (2^-8 |y|). So
|y - ref| <= 2^-8 |ref| + 2^-8 sum_j |T_j B_j| + (k / 16 + 4) 2^-23 (sum |x w| + sum_j |B_j| s sum |x A_j|)
and the r products of B T add (r + 4) 2^-23 sum_j |T_j B_j|."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _rand(shape, seed, dev, std=1.0):
    g = torch.Generator(device="cpu").manual_seed(seed)
    return (torch.randn(shape, generator=g) * std).to(torch.bfloat16).to(dev)


def _case(dev, m, k, n, rank, na, seed, how="scattered"):
    x, w = _rand((m, k), seed, dev), _rand((n, k), seed + 1, dev, k ** -0.5)
    a, b = _rand((na * rank, k), seed + 2, dev, k ** -0.5), _rand((n, na * rank), seed + 3, dev, rank ** -0.5)
    g = torch.Generator(device="cpu").manual_seed(seed + 4)
    scale = (torch.rand(na, generator=g) * 2 - 0.5).to(dev)
    if how == "scattered":
        rows = torch.randint(-1, na, (m,), generator=g)
    elif how == "segments":
        rows = torch.arange(m) * (na + 1) // m
        rows[rows == na] = -1
    elif how == "none":
        rows = torch.full((m,), -1)
    else:
        rows = torch.full((m,), na - 1)
    return x, w, a, b, scale, rows.int().to(dev)


def _reference(x, w, a, b, scale, rows):
    """(y, bound) in fp64."""
    m, k = x.shape
    na = scale.shape[0]
    r = a.shape[0] // na
    x, w, a, b = (t.double() for t in (x, w, a, b))
    ok = (rows >= 0) & (rows < na)
    mine = (rows.clamp(0, na - 1)[:, None] == torch.arange(na * r, device=x.device)[None] // r) & ok[:, None]
    s = scale.double().repeat_interleave(r) * mine
    t, t_mag = (x @ a.T) * s, (x.abs() @ a.abs().T) * s.abs()
    y = x @ w.T + t @ b.T
    steps = (k / 16 + 4) * 2 ** -23
    low = t.abs() @ b.abs().T
    bound = 2 ** -8 * y.abs() + 2 ** -8 * low + (r + 4) * 2 ** -23 * low
    return y, bound + steps * (x.abs() @ w.abs().T + t_mag @ b.abs().T)


def _check(O, c, **kw):
    y = O.linear_lora(*c, **kw)
    O.check_status()
    ref, bound = _reference(*c)
    err = (y.double() - ref).abs()
    assert bool((err <= bound).all()), ((err - bound).max().item(), err.max().item())
    return y


@pytest.mark.parametrize("m,k,n", [(1, 64, 8), (1, 5376, 264), (4, 256, 2048), (16, 200, 520), (17, 1024, 128),
                                   (33, 8, 1000), (48, 712, 384), (64, 2048, 776)])
@pytest.mark.parametrize("rank,na", [(8, 1), (16, 24), (32, 3), (64, 5), (128, 2), (192, 3), (256, 1)])
def test_few_rows(cuda_dev, m, k, n, rank, na):
    import h3attn as O
    _check(O, _case(cuda_dev, m, k, n, rank, na, 10 * rank + m))


@pytest.mark.parametrize("m,k,n,how", [(65, 64, 8, "scattered"), (127, 200, 264, "segments"), (128, 1024, 256, "last"),
                                       (129, 8, 1000, "scattered"), (257, 576, 512, "segments"),
                                       (513, 3584, 328, "scattered"), (1300, 256, 2304, "segments"),
                                       (2900, 128, 136, "segments")])
@pytest.mark.parametrize("rank,na", [(8, 1), (8, 32), (16, 24), (32, 3), (64, 5), (128, 2), (192, 3), (256, 1)])
def test_many_rows(cuda_dev, m, k, n, how, rank, na):
    import h3attn as O
    _check(O, _case(cuda_dev, m, k, n, rank, na, 20 * rank + m, how))


@pytest.mark.parametrize("m", [1, 40, 64, 300, 1030])
def test_rows_without_an_adapter_are_the_projection(cuda_dev, m):
    """Adapters outside [0, n) leave W x: the definition's value, and above 64 rows the projection's own bits."""
    import h3attn as O
    x, w, a, b, scale, rows = _case(cuda_dev, m, 640, 520, 16, 4, 30, "none")
    rows[::3] = 4
    rows[::5] = -7
    rows[::7] = 2 ** 31 - 1
    _check(O, (x, w, a, b, scale, rows))
    if m > 64:
        rows[0] = 1
        y, base = O.linear_lora(x, w, a, b, scale, rows), O.linear(x, w)
        assert torch.equal(y[1:], base[1:])
        assert not torch.equal(y[0], base[0])


@pytest.mark.parametrize("m", [50, 900])
def test_a_row_does_not_depend_on_the_others(cuda_dev, m):
    """Up to 64 rows: while the call uses the same adapters (each part here uses all of them)."""
    import h3attn as O
    x, w, a, b, scale, rows = _case(cuda_dev, m, 1088, 520, 32, 6, 40)
    y = O.linear_lora(x, w, a, b, scale, rows)
    parts = [(0, m), (3, 37), (m - 20, m)] if m <= 64 else [(0, 70), (129, 640), (m - 65, m)]
    for lo, hi in parts:
        assert torch.equal(O.linear_lora(x[lo:hi], w, a, b, scale, rows[lo:hi].contiguous()), y[lo:hi])
    others = rows.clone()
    others[1:] = (others[1:] + 2) % 6
    assert torch.equal(O.linear_lora(x, w, a, b, scale, others)[0], y[0])


def test_a_row_does_not_depend_on_the_calls_length(cuda_dev):
    """Thousands of rows make T in one CTA a tile, hundreds in a cluster: the same bits."""
    import h3attn as O
    for k in (64, 136, 1088):
        x, w, a, b, scale, rows = _case(cuda_dev, 5000, k, 136, 16, 9, 45, "scattered")
        y = _check(O, (x, w, a, b, scale, rows))
        for lo, hi in ((0, 100), (1000, 1700), (4935, 5000)):
            assert torch.equal(O.linear_lora(x[lo:hi], w, a, b, scale, rows[lo:hi].contiguous()), y[lo:hi])


@pytest.mark.parametrize("m", [30, 300])
def test_adapters_that_no_row_uses_may_hold_anything(cuda_dev, m):
    """Whole groups of 64 stacked columns out of use, and A of any adapter that a row does not use itself."""
    import h3attn as O
    x, w, a, b, scale, rows = _case(cuda_dev, m, 512, 264, 16, 20, 50)
    rows.clamp_(max=7)
    want = O.linear_lora(x, w, a, b, scale, rows)
    a[8 * 16:], b[:, 8 * 16:], scale[8:] = float("nan"), float("inf"), float("nan")
    assert torch.equal(O.linear_lora(x, w, a, b, scale, rows), want)
    a[3 * 16:4 * 16] = float("nan")
    y = O.linear_lora(x, w, a, b, scale, rows)
    hit = rows == 3
    assert torch.equal(y[~hit], want[~hit]) and bool(torch.isnan(y[hit]).all())


@pytest.mark.parametrize("m", [40, 700])
def test_head_major_and_strides(cuda_dev, m):
    import h3attn as O
    H, n = 6, 264
    heads = _rand((H, m, 128), 60, cuda_dev)
    flat = heads.transpose(0, 1).reshape(m, H * 128).contiguous()
    _, w, a, b, scale, rows = _case(cuda_dev, m, H * 128, n, 16, 5, 61)
    want = O.linear_lora(flat, w, a, b, scale, rows)
    assert torch.equal(O.linear_lora(heads, w, a, b, scale, rows), want)
    wide_x, wide_w = _rand((m, H * 128 + 64), 62, cuda_dev), _rand((n, H * 128 + 8), 63, cuda_dev)
    wide_a, wide_b = _rand((80, H * 128 + 16), 64, cuda_dev), _rand((n, 80 + 40), 65, cuda_dev)
    wide_x[:, 32:32 + H * 128], wide_w[:, :H * 128], wide_a[:, 8:8 + H * 128], wide_b[:, 16:96] = flat, w, a, b
    out = torch.full((m, n + 24), 3.0, dtype=torch.bfloat16, device=cuda_dev)
    y = O.linear_lora(wide_x[:, 32:32 + H * 128], wide_w[:, :H * 128], wide_a[:, 8:8 + H * 128], wide_b[:, 16:96],
                      scale, rows, out=out[:, 8:8 + n])
    assert torch.equal(y, want)
    assert bool((out[:, :8] == 3).all()) and bool((out[:, 8 + n:] == 3).all())


@pytest.mark.parametrize("m", [5, 64, 400])
def test_swiglu(cuda_dev, m):
    """The epilogue on top of the adapters' own sums: silu(g) * u with the roundings of linear()'s."""
    import h3attn as O
    f = 256
    c = _case(cuda_dev, m, 640, 2 * f, 32, 3, 70)
    y = O.linear_lora(*c, epilogue="swiglu")
    O.check_status()
    plain = O.linear_lora(*c)  # the same sums, rounded: what the epilogue starts from
    g, u = plain.float().chunk(2, dim=-1)
    s = (g * torch.sigmoid(g)).to(torch.bfloat16).float()
    ref = s * u
    # silu rounds to bf16 from an fp32 value that may sit on a border: one step (2^-7) of it, and the product's half step
    assert bool(((y.float() - ref).abs() <= (2 ** -7 + 2 ** -8) * ref.abs() + 1e-6).all())
    if m > 64:
        assert torch.equal(O.linear_lora(c[0], c[1], c[2], c[3], c[4], torch.full_like(c[5], -1), epilogue="swiglu"),
                           O.linear(c[0], c[1], epilogue="swiglu"))


def test_stacked_adapters_of_mixed_ranks(cuda_dev):
    import h3attn as O
    k, n, m = 320, 136, 100
    pairs = [(_rand((r, k), 80 + r, cuda_dev, k ** -0.5), _rand((n, r), 90 + r, cuda_dev, 0.3)) for r in (4, 24, 1)]
    a, b, scale = O.stack_adapters(pairs, [0.5, 2.0, -1.0])
    assert a.shape == (96, k) and b.shape == (n, 96)
    x, w = _rand((m, k), 81, cuda_dev), _rand((n, k), 82, cuda_dev, 0.05)
    rows = (torch.arange(m, device=cuda_dev) % 4 - 1).int()
    y = _check(O, (x, w, a, b, scale, rows))
    for i, (A, B) in enumerate(pairs):
        at = rows == i
        ref = x[at].double() @ w.double().T + float(scale[i]) * (x[at].double() @ A.double().T) @ B.double().T
        assert (y[at].double() - ref).abs().max() < 0.02 * ref.abs().max()


@pytest.mark.parametrize("m", [20, 600])
def test_streams_graphs_and_two_calls_at_once(cuda_dev, m):
    import h3attn as O
    c = _case(cuda_dev, m, 1024, 1032, 16, 6, 100)
    want = O.linear_lora(*c)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs = []
    for st in streams:
        with torch.cuda.stream(st):
            outs += [O.linear_lora(*c) for _ in range(5)]
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)
    graphs, got = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            got.append(O.linear_lora(*c))
        graphs.append(g)
    c[0].copy_(_rand(c[0].shape, 110, cuda_dev))
    c[5].copy_((c[5] + 1) % 6)
    torch.cuda.synchronize()
    for _ in range(3):
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    want = O.linear_lora(*c)
    assert all(torch.equal(o, want) for o in got)
    O.check_status()


def test_refusals(cuda_dev):
    import h3attn as O
    x, w, a, b, scale, rows = _case(cuda_dev, 20, 128, 64, 16, 3, 120)
    bad = [(x.float(), w, a, b, scale, rows), (x[:, :120], w, a, b, scale, rows), (x, w, a[:47], b, scale, rows),
           (x, w, a[:40], b[:, :40], scale, rows), (x, w, a, b[:, :40], scale, rows), (x, w, a, b, scale.half(), rows),
           (x, w, a, b, scale[:0], rows), (x, w, a, b, scale, rows.long()), (x, w, a, b, scale, rows[:19]),
           (x, w, a, b, scale, rows.cpu()), (x[:0], w, a, b, scale, rows[:0]), (x, w[:60], a, b[:60], scale, rows),
           (x, w, a[:, :64], b, scale, rows), (x, w, a[:36], b[:, :36], scale, rows)]
    for c in bad:
        with pytest.raises(O.H3Error):
            O.linear_lora(*c)
    with pytest.raises(O.H3Error):
        O.linear_lora(x, w, a, b, scale, rows, epilogue="gelu")
    with pytest.raises(O.H3Error):
        O.linear_lora(x, w, a, b, scale, rows, epilogue="swiglu")  # 32 columns, not a multiple of 128


@pytest.mark.parametrize("m", [1, 3, 7, 13, 21, 35, 51, 63])
@pytest.mark.parametrize("rank,na", [(8, 3), (16, 9), (64, 2)])
def test_odd_row_counts(cuda_dev, m, rank, na):
    """Odd counts end the loop over a cluster's sums in the middle of a warp, in front of the cluster barrier."""
    import h3attn as O
    for k, n in ((8, 264), (1096, 136)):
        _check(O, _case(cuda_dev, m, k, n, rank, na, 130 + m))


@pytest.mark.parametrize("m", [65, 131, 259, 601])
def test_scattered_rows_of_few_columns(cuda_dev, m):
    """Neighbouring rows of other adapters part the lanes of a warp at every piece of T, with clusters and without."""
    import h3attn as O
    for rank, na in ((8, 40), (16, 24), (128, 5)):
        _check(O, _case(cuda_dev, m, 328, 136, rank, na, 140 + m))


@pytest.mark.parametrize("rank,na", [(8, 5), (16, 24), (128, 3)])
def test_row_independent_calls_of_any_length(cuda_dev, rank, na):
    """Shards of a sequence have the bits of the whole, however short: 1000 rows in pieces of 1 to 64, both epilogues,
    head-major input; rows without an adapter have the projection's own."""
    import h3attn as O
    x, w, a, b, scale, rows = _case(cuda_dev, 1000, 640, 512, rank, na, 150 + rank)
    heads = x.view(1000, 5, 128).transpose(0, 1).contiguous()
    for ep in ("none", "swiglu"):
        whole, base = O.linear_lora(x, w, a, b, scale, rows, epilogue=ep), O.linear(x, w, epilogue=ep)
        bare = rows < 0
        for lo, n in ((0, 1), (5, 50), (500, 64), (936, 64), (983, 17)):
            r = rows[lo:lo + n].contiguous()
            y = O.linear_lora(x[lo:lo + n], w, a, b, scale, r, epilogue=ep, row_independent=True)
            assert torch.equal(y, whole[lo:lo + n]), (ep, lo, n)
            at = bare[lo:lo + n]
            assert torch.equal(y[at], base[lo:lo + n][at])
            part = heads[:, lo:lo + n].contiguous()
            assert torch.equal(O.linear_lora(part, w, a, b, scale, r, epilogue=ep, row_independent=True), y)
        assert torch.equal(O.linear_lora(x, w, a, b, scale, rows, epilogue=ep, row_independent=True), whole)
    O.check_status()
    _check(O, (x[:33], w, a, b, scale, rows[:33].contiguous()), row_independent=True)
