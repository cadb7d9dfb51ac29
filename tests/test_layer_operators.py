"""The runtime's options (rotary positions, window, adapters) on CPU gloo ranks: sharding of positions and adapter
segments, the pad path, and the options' host logic, with oracle/cpu_ops in place of the kernels."""
import pytest
import torch

import layer_operators as T


@pytest.mark.parametrize("world", [1, 2])
def test_run_blocks_with_every_option(world, tmp_path):
    S = 203  # odd: the last rank has a pad row
    one = T.run(1, S, tmp_path)
    ref = torch.load(tmp_path / "plain.pt")
    got = one if world == 1 else T.run(world, S, tmp_path)
    assert T.near(got["out"], ref["out"]) and T.near(got["dense"], ref["dense"])
    assert torch.equal(got["bare"], got["unnamed"]) and torch.equal(got["bare"], got["off"])
    for other in ("bare", "dense"):  # the options do something: far beyond the tolerance
        assert (got["out"] - got[other]).abs().mean() > 0.1 * ref["out"].abs().mean()


def test_option_checks(monkeypatch):
    import sp_runtime
    assert sp_runtime._window({}) is None and sp_runtime._window(None) is None
    assert sp_runtime._window({"h3_window": {"left": 3}}) == (3, None, 0)
    with pytest.raises(ValueError):
        sp_runtime._window({"h3_window": {"lft": 3}})
    lin = torch.nn.Linear(8, 8, bias=True, dtype=torch.bfloat16)
    sp_runtime.set_adapters(lin, (torch.zeros(8, 8), torch.zeros(8, 8), torch.ones(1)))
    x = torch.zeros(2, 8, dtype=torch.bfloat16)
    assert sp_runtime._gemm_weight(lin, x) is None
    monkeypatch.setattr(sp_runtime, "_ADAPTER_ROWS", torch.zeros(2, dtype=torch.int32))
    with pytest.raises(RuntimeError):  # adapters cannot be dropped silently
        sp_runtime._gemm_weight(lin, x)
    sp_runtime.set_adapters(lin, None)
    assert sp_runtime._gemm_weight(lin, x) is None
    monkeypatch.setattr(sp_runtime, "_SP_ACTIVE", True)
    monkeypatch.setattr(sp_runtime, "WORLD", 2)
    with pytest.raises(NotImplementedError):
        sp_runtime._sp_attn_forward_peer(None, x, None, {"h3_window": {"left": 1}})


def _one_block(S, monkeypatch, positions):
    """run_blocks of a one-block model on host tensors, with positions for `positions` tokens."""
    import h3_model as M
    import h3attn as O
    import sp_runtime
    from oracle import cpu_ops
    monkeypatch.setattr(sp_runtime, "_ops", cpu_ops)
    model = M.MiniMaxH3Model(1, hidden=64, heads=2, ffn=128, t_dim=16, dtype=torch.bfloat16)
    M.init_weights(model, 3, std=0.1)
    model.blocks[0].adaln_proj.lin.bias.data.fill_(0.5)
    h = torch.randn(S, 64, generator=torch.Generator().manual_seed(4)).bfloat16()
    pos = (torch.arange(positions, dtype=torch.int32) + 3)[:, None]
    rope = O.RopePositions(pos, *O.rope_axes_freqs([64]))
    with torch.no_grad():
        return M, model, lambda: sp_runtime._sp_run_blocks(model, h, torch.ones(1, 16).bfloat16(), [(0, S, 0)], rope)


def test_positions_of_every_token(monkeypatch):
    """A token without a position is an error, as a short table is; positions behind the last token are not looked at,
    by the padding either."""
    import sp_runtime
    S = 13
    runs = {}
    for n in (S - 1, S, S + 1):
        M, _, run = _one_block(S, monkeypatch, n)
        sp_runtime.install(M)
        try:
            with torch.no_grad():
                if n < S:
                    with pytest.raises(ValueError, match="positions of 12 tokens"):
                        run()
                    assert not sp_runtime._SP_ACTIVE
                else:
                    runs[n] = run()
        finally:
            sp_runtime.uninstall()
    assert torch.equal(runs[S], runs[S + 1])


def test_rows_of_positions():
    import h3attn as O
    rp = O.RopePositions(torch.arange(5, dtype=torch.int32)[:, None] + 1, *O.rope_axes_freqs([64]))
    assert rp.rows(2, 6, 4).pos[:, 0].tolist() == [3, 4, 0, 0]  # token 4 is behind the sequence: padding
    assert rp.rows(2, 6).pos[:, 0].tolist() == [3, 4, 5, 0]
    assert rp.rows(4, 6, 4).pos[:, 0].tolist() == [0, 0]
    with pytest.raises(O.H3Error):
        rp.rows(0, 6, 6)


def _adapters(lin, count):
    import h3attn as O
    n, k = lin.weight.shape
    g = torch.Generator().manual_seed(n + k)
    pairs = [(torch.randn(8, k, generator=g) * k ** -0.5, torch.randn(n, 8, generator=g)) for _ in range(count)]
    return O.stack_adapters(pairs, [1.0] * count)


def _run_adapted(M, model, S, segments):
    import sp_runtime
    h = torch.randn(S, 64, generator=torch.Generator().manual_seed(4)).bfloat16()
    with torch.no_grad():
        return sp_runtime._sp_run_blocks(model, h, torch.ones(1, 16).bfloat16(), [(0, S, 0)], None,
                                         {"h3_adapter_segments": segments})


@pytest.mark.parametrize("where", ["adaln", "unpatched mlp", "fc2 with a bias", "3-D input"])
def test_adapters_that_could_not_act_are_an_error(monkeypatch, where):
    import sp_runtime
    S = 6
    M, model, _ = _one_block(S, monkeypatch, S)
    blk = model.blocks[0]
    lin = blk.adaln_proj.lin if where == "adaln" else blk.mlp.fc1
    sp_runtime.set_adapters(lin, _adapters(lin, 2))
    if where == "fc2 with a bias":  # fc1's adapters must not go with fc2's fall back to the host's MLP
        blk.mlp.fc2.bias = torch.nn.Parameter(torch.zeros(64, dtype=torch.bfloat16))
    elif where == "3-D input":
        blk.mlp.register_forward_pre_hook(lambda m, x: (x[0][None],))
    elif where == "unpatched mlp":
        monkeypatch.setattr(M, "MLP", torch.nn.Identity)  # not the class of the block's MLP
    sp_runtime.install(M)
    try:
        _run_adapted(M, model, S, [])  # no segments: the bare model
        with pytest.raises(RuntimeError, match="adapters"):
            _run_adapted(M, model, S, [(0, S, 0)])
        assert sp_runtime._ADAPTER_ROWS is None and not sp_runtime._SP_ACTIVE
    finally:
        sp_runtime.uninstall()


def test_adapter_numbers_of_segments(monkeypatch):
    """A number that no projection's stack reaches is an error; one that some stack has acts there and there alone."""
    import sp_runtime
    S = 6
    M, model, _ = _one_block(S, monkeypatch, S)
    blk = model.blocks[0]
    blk.adaln_proj.lin.bias.data.fill_(1.0)
    sp_runtime.install(M)
    try:
        bare = _run_adapted(M, model, S, [(0, S, 5)])  # nothing attached: nothing to reach
        sp_runtime.set_adapters(blk.attn.qkv_proj, _adapters(blk.attn.qkv_proj, 3))
        for bad in ([(0, 2, 0), (2, S, 3)], [(0, S, -2)]):
            with pytest.raises(ValueError, match="h3_adapter_segments"):
                _run_adapted(M, model, S, bad)
        assert torch.equal(_run_adapted(M, model, S, [(0, S, -1), (S, S + 4, 9), (3, 3, 9)]), bare)
        last = _run_adapted(M, model, S, [(0, S, 2)])
        assert not torch.equal(last, bare)
        sp_runtime.set_adapters(blk.mlp.fc2, _adapters(blk.mlp.fc2, 2))
        assert torch.equal(_run_adapted(M, model, S, [(0, S, 2)]), last)
        assert not torch.equal(_run_adapted(M, model, S, [(0, S, 1)]), last)
    finally:
        sp_runtime.uninstall()


def test_projections_with_adapters_do_not_depend_on_the_shard(monkeypatch):
    """The runtime asks for kernels whose rows have the same bits in a shard of any length."""
    import sp_runtime
    S = 6
    M, model, _ = _one_block(S, monkeypatch, S)
    blk, asked = model.blocks[0], []
    for lin in (blk.attn.qkv_proj, blk.attn.out_proj, blk.mlp.fc1, blk.mlp.fc2):
        sp_runtime.set_adapters(lin, _adapters(lin, 1))
    plain = sp_runtime.ops().linear_lora
    monkeypatch.setattr(sp_runtime.ops(), "linear_lora",
                        lambda *a, **k: asked.append(k.get("row_independent")) or plain(*a, **k))
    sp_runtime.install(M)
    try:
        _run_adapted(M, model, S, [(0, 3, 0)])
    finally:
        sp_runtime.uninstall()
    assert asked == [True] * 4


@pytest.mark.parametrize("world", [1, 2, 4])
def test_every_row_of_run_blocks(world, tmp_path):
    """Row by row, so that one token with a neighbour's adapter, or a window one key off, shows -- which it does when
    the mistake is made in the model that the run is compared with."""
    S = 203
    if world > 1:
        T.run(1, S, tmp_path)  # leaves the fp32 model's output
    got, ref = T.run(world, S, tmp_path), torch.load(tmp_path / "plain.pt")
    for k in ("out", "dense"):
        assert T.row_errors(got[k], ref[k]).max() < T.ROW_BOUND, k
    if world == 1:
        for change, wrong in T.mistakes(S):
            assert T.row_errors(got["out"], wrong).max() > T.ROW_BOUND, change


def test_adapters_through_wrappers(monkeypatch):
    """A forward that wraps the patched one, on the instance or in a subclass, still applies its adapters; segments may
    be any iterable."""
    import sp_runtime
    S = 6
    M, model, _ = _one_block(S, monkeypatch, S)
    blk = model.blocks[0]
    sp_runtime.set_adapters(blk.attn.qkv_proj, _adapters(blk.attn.qkv_proj, 2))
    sp_runtime.set_adapters(blk.mlp.fc1, _adapters(blk.mlp.fc1, 2))
    sp_runtime.install(M)
    try:
        bare, want = _run_adapted(M, model, S, []), _run_adapted(M, model, S, [(0, S, 1)])
        assert not torch.equal(bare, want)
        assert torch.equal(_run_adapted(M, model, S, iter([(0, S, 1)])), want)
        inner = blk.attn.forward
        blk.attn.forward = lambda *a, **k: inner(*a, **k)
        blk.mlp.__class__ = type("Wrapped", (M.MLP,), {"forward": lambda self, x: M.MLP.forward(self, x)})
        assert torch.equal(_run_adapted(M, model, S, [(0, S, 1)]), want)
    finally:
        sp_runtime.uninstall()
