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
