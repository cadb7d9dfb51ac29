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
