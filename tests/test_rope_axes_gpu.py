"""Rotary positions over several axes against the definition in 64 bits.

Tolerance. The rotated value is y = c a - s b in fp32, rounded once to bf16 (half a step: 2^-8 |y|). c and s carry
the rounding of the reduced angle (at most half a turn, 2^-25 of it, times 2 pi: 2^-23 rad) and 2 ulp of the
sine/cosine (2^-23); two products and a sum add 3 * 2^-24: below 2^-20 (|a| + |b|) together. The pack's norm adds a sum
of 128 squares, a square root, a divide and two products: below 24 * 2^-24 of the value, so 2^-18 (|a| + |b|) there."""
import pytest
import torch

pytestmark = pytest.mark.gpu
D = 128


def _rand(shape, seed, dev):
    g = torch.Generator(device="cpu").manual_seed(seed)
    return torch.randn(shape, generator=g).to(torch.bfloat16).to(dev)


def _plan(O, dev, axes, tokens, seed, real=False, mixed=False, far=5000):
    sections = {1: [64], 2: [32, 32], 3: [16, 24, 24], 4: [12, 20, 20, 8]}[axes]
    g = torch.Generator(device="cpu").manual_seed(seed)
    pos = torch.randint(0, far, (tokens, axes), generator=g)
    pos = pos.float() + torch.rand(tokens, axes, generator=g) if real else pos.int()
    f, a = O.rope_axes_freqs(sections, interleaved=mixed, device=dev)
    return O.RopePositions(pos.to(dev), f, a)


def _turn64(x, rp, inverse=False):
    """x [tokens, heads, 128] fp64 -> (rotated, |a| + |b| of each element's pair)."""
    axis = rp.axis.long()
    ang = rp.pos.double()[:, axis.clamp_min(0)] * rp.inv_freq
    ang = torch.where(axis >= 0, ang, torch.zeros_like(ang))[:, None] * (-1 if inverse else 1)
    a, b = x[..., :64], x[..., 64:]
    y = torch.cat([a * ang.cos() - b * ang.sin(), a * ang.sin() + b * ang.cos()], -1)
    mag = (a.abs() + b.abs()).repeat(1, 1, 2)
    return y, mag


def _assert_close(got, ref, mag, slack):
    err = (got.double() - ref).abs()
    bound = 2 ** -8 * ref.abs() + slack * mag
    assert bool((err <= bound).all()), (err - bound).max().item()


@pytest.mark.parametrize("tokens,heads", [(1, 1), (1, 56), (3, 5), (77, 28), (1000, 7), (2500, 3)])
@pytest.mark.parametrize("axes,real,mixed", [(1, False, False), (3, False, True), (3, True, False), (4, True, True)])
def test_rope_axes(cuda_dev, tokens, heads, axes, real, mixed):
    import h3attn as O
    x = _rand((tokens, heads, D), 1, cuda_dev)
    rp = _plan(O, cuda_dev, axes, tokens, 2, real, mixed)
    for inverse in (False, True):
        y = O.rope_axes(x, rp, inverse=inverse)
        ref, mag = _turn64(x.double(), rp, inverse)
        _assert_close(y, ref, mag, 2 ** -20)


def test_far_positions_keep_their_angles(cuda_dev):
    """Integer positions up to 2^31 - 1 and fp32 positions up to 2^24: the angle is formed in fp64."""
    import h3attn as O
    f, a = O.rope_axes_freqs([32, 32], device=cuda_dev)
    pos = torch.tensor([[2 ** 31 - 1, -2 ** 31], [1000003, -168001], [0, 1]], dtype=torch.int32, device=cuda_dev)
    x = _rand((3, 2, D), 3, cuda_dev)
    for p in (pos, torch.tensor([[2.0 ** 24, -123456.75], [0.125, 1e7], [3e5, -0.0]], device=cuda_dev)):
        rp = O.RopePositions(p, f, a)
        ref, mag = _turn64(x.double(), rp)
        _assert_close(O.rope_axes(x, rp), ref, mag, 2 ** -20)


def test_strides_in_place_and_neighbours(cuda_dev):
    import h3attn as O
    big = _rand((50, 6, 160), 4, cuda_dev)
    before = big.clone()
    x = big[:, 1:5, 16:144]
    rp = _plan(O, cuda_dev, 3, 50, 5)
    want = O.rope_axes(x.contiguous(), rp)
    assert torch.equal(O.rope_axes(x, rp), want)
    hm = x.transpose(0, 1).contiguous().transpose(0, 1)  # head-major memory
    assert torch.equal(O.rope_axes(hm, rp), want)
    O.rope_axes(x, rp, out=x)
    assert torch.equal(x, want)
    big[:, 1:5, 16:144] = before[:, 1:5, 16:144]
    assert torch.equal(big, before)  # nothing beside x was written
    one = _rand((1, 4, D), 6, cuda_dev).expand(50, 4, D)  # one row shared by all tokens
    assert torch.equal(O.rope_axes(one, rp), O.rope_axes(one.contiguous(), rp))


def test_pairs_without_an_axis_are_copied(cuda_dev):
    import h3attn as O
    x = _rand((20, 3, D), 7, cuda_dev)
    f, a = O.rope_axes_freqs([5, 0, 7], device=cuda_dev)
    rp = O.RopePositions(torch.full((20, 3), 11, dtype=torch.int32, device=cuda_dev), f, a)
    y = O.rope_axes(x, rp)
    assert torch.equal(y[..., 12:64], x[..., 12:64]) and torch.equal(y[..., 76:], x[..., 76:])
    assert not torch.equal(y[..., :12], x[..., :12])
    wild = a.clone()
    wild[3] = 1000  # an axis that pos does not have: not turned, not read
    ref, mag = _turn64(x.double(), O.RopePositions(rp.pos, f, torch.where(wild > 2, -1, wild)))
    _assert_close(O.rope_axes(x, O.RopePositions(rp.pos, f, wild)), ref, mag, 2 ** -20)


def test_gradient_is_the_inverse(cuda_dev):
    """<R x, g> = <x, R^T g> for the definition's R, and R^T from the kernel matches finite differences of <R x, g>
    in 64 bits (the map is linear: a step of 1 along each coordinate is exact)."""
    import h3attn as O
    rp = _plan(O, cuda_dev, 3, 2, 8, real=True)
    g = _rand((2, 1, D), 9, cuda_dev)
    grad = O.rope_axes(g, rp, inverse=True)
    eye = torch.eye(D, device=cuda_dev, dtype=torch.float64)
    for t in range(2):
        one = O.RopePositions(rp.pos[t:t + 1].expand(D, 3).contiguous(), rp.inv_freq, rp.axis)
        cols, _ = _turn64(eye[:, None], one)                      # R e_j for every j
        diff = (cols[:, 0] * g[t, 0].double()).sum(-1)
        _, mag = _turn64(g[t:t + 1].double(), O.RopePositions(rp.pos[t:t + 1], rp.inv_freq, rp.axis))
        _assert_close(grad[t, 0], diff, mag[0, 0], 2 ** -20)


def _pack64(x, w, rp, eps, s, H, turned=True):
    x = x.double().reshape(s, H, D)
    y = x / (x.pow(2).mean(-1, keepdim=True) + eps).sqrt()
    y = y * w.double() if w is not None else y
    return _turn64(y, rp)


@pytest.mark.parametrize("s,H,world,axes,real", [(1, 1, 1, 1, False), (1, 56, 2, 3, False), (67, 8, 4, 3, True),
                                                 (333, 56, 8, 4, False), (2600, 7, 1, 2, True), (40, 8, 8, 3, False),
                                                 (20, 21, 7, 3, False), (9, 300, 4, 1, False)])
def test_pack_with_positions(cuda_dev, s, H, world, axes, real):
    import h3attn as O
    q, k, v = _rand((s, 3 * H * D), 10, cuda_dev).split(H * D, -1)
    qw, kw = _rand((D,), 11, cuda_dev), None
    rp = _plan(O, cuda_dev, axes, s, 12, real)
    send = O.qknorm_rope_pack(q, k, v, rp, qw, kw, 1e-6, world)
    assert send.shape == (world, 3, H // world, s, D)
    got = send.permute(1, 3, 0, 2, 4).reshape(3, s, H, D)
    for i, (x, w) in enumerate(((q, qw), (k, kw))):
        ref, mag = _pack64(x, w, rp, 1e-6, s, H)
        _assert_close(got[i], ref, mag, 2 ** -18)
    assert torch.equal(got[2], v.reshape(s, H, D))
    hm = O.qknorm_rope_pack(q, k, v, rp, qw, kw, 1e-6, world, head_major=True)  # [H/W, W, 3, s, D]
    assert torch.equal(hm.permute(1, 2, 0, 3, 4), send)
    one = O.qknorm_rope_pack(q[s // 2:], k[s // 2:], v[s // 2:], rp.rows(s // 2, s), qw, kw, 1e-6, world)
    assert torch.equal(one, send[:, :, :, s // 2:])  # a token's rows do not depend on its neighbours


def test_pack_peer_form_writes_the_same_rows(cuda_dev):
    """The form that stores into per-rank buffers (here all on this GPU) against the local one."""
    import h3attn as O
    s, H, W = 40, 8, 2
    q, k, v = _rand((s, 3 * H * D), 13, cuda_dev).split(H * D, -1)
    rp = _plan(O, cuda_dev, 3, s, 14)
    send = O.qknorm_rope_pack(q, k, v, rp, None, None, 1e-6, W)
    bufs = [torch.zeros(3, H // W, 2 * s, D, dtype=torch.bfloat16, device=cuda_dev) for _ in range(W)]
    base = torch.tensor([b.data_ptr() for b in bufs], dtype=torch.int64, device=cuda_dev)
    O.qknorm_rope_pack_peer(q, k, v, rp, None, None, 1e-6, W, base, H // W * 2 * s * D, 2 * s * D, s)
    torch.cuda.synchronize()
    for r in range(W):
        assert torch.equal(bufs[r][:, :, s:], send[r]) and not bool(bufs[r][:, :, :s].any())


def test_other_stream_and_graph(cuda_dev):
    import h3attn as O
    x = _rand((300, 28, D), 15, cuda_dev)
    rp = _plan(O, cuda_dev, 3, 300, 16)
    want = O.rope_axes(x, rp)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = O.rope_axes(x, rp)
    side.synchronize()
    assert torch.equal(y, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        z = O.rope_axes(x, rp)
    x.copy_(_rand((300, 28, D), 17, cuda_dev))
    rp.pos.add_(3)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(z, O.rope_axes(x, rp))


def test_refusals(cuda_dev):
    import h3attn as O
    x = _rand((8, 2, D), 18, cuda_dev)
    rp = _plan(O, cuda_dev, 3, 8, 19)
    bad = [lambda: O.rope_axes(x.float(), rp), lambda: O.rope_axes(x[:, :, :64], rp), lambda: O.rope_axes(x[:7], rp),
           lambda: O.rope_axes(x, O.RopePositions(rp.pos.long(), rp.inv_freq, rp.axis)),
           lambda: O.rope_axes(x, O.RopePositions(rp.pos, rp.inv_freq.float(), rp.axis)),
           lambda: O.rope_axes(x, O.RopePositions(rp.pos, rp.inv_freq[:32], rp.axis)),
           lambda: O.rope_axes(x, O.RopePositions(rp.pos, rp.inv_freq, rp.axis.cpu())),
           lambda: O.rope_axes(x, O.RopePositions(rp.pos.t(), rp.inv_freq, rp.axis)),
           lambda: O.rope_axes(x, rp, out=x[:, :1]), lambda: O.rope_axes(x[:0], rp.rows(0, 0)),
           lambda: O.qknorm_rope_pack(x.view(8, -1), x.view(8, -1), x.view(8, -1), rp.rows(0, 7), None, None, 1e-6, 1)]
    for f in bad:
        with pytest.raises(O.H3Error):
            f()
