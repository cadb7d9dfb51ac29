"""The layer's operators together, as the runtime runs them: projections with adapters, rotary positions inside the
pack, windowed attention -- over a two-block model against plain torch, and across GPUs bit for bit."""
import pytest
import torch

import layer_operators as T

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("S", [203, 1001])
def test_run_blocks_with_every_option(S, tmp_path):
    got = T.run(1, S, tmp_path, on_gpu=True)
    ref = torch.load(tmp_path / "plain.pt")
    assert T.near(got["out"], ref["out"]) and T.near(got["dense"], ref["dense"])
    assert torch.equal(got["bare"], got["unnamed"]) and torch.equal(got["bare"], got["off"])
    for other in ("bare", "dense"):
        assert (got["out"] - got[other]).abs().mean() > 0.1 * ref["out"].abs().mean()


@pytest.mark.parametrize("world,overlap", [(2, None), (2, "heads"), (2, "ce"), (2, "1"), (4, None)])
def test_across_gpus(world, overlap, tmp_path):
    if torch.cuda.device_count() < world:
        pytest.skip(f"needs {world} GPUs")
    S = 1001
    one, many = T.run(1, S, tmp_path, on_gpu=True), T.run(world, S, tmp_path, overlap, on_gpu=True)
    for k in one:
        # token pieces start the window's key walk at other rows: equal values, not equal bits
        assert T.near(many[k], one[k]) if overlap == "1" else torch.equal(many[k], one[k])


@pytest.mark.parametrize("world", [2, 4])
def test_short_shards_with_adapters_across_gpus(world, tmp_path):
    """Shards of 64 rows and fewer, where one GPU has more: the same bits."""
    if torch.cuda.device_count() < world:
        pytest.skip(f"needs {world} GPUs")
    for S in (101, 203):
        one, many = T.run(1, S, tmp_path, on_gpu=True), T.run(world, S, tmp_path, on_gpu=True)
        for k in ("dense", "out"):
            assert torch.equal(many[k], one[k]), (S, k)


@pytest.mark.parametrize("S", [203, 1001])
def test_every_row_of_run_blocks(S, tmp_path):
    got = T.run(1, S, tmp_path, on_gpu=True)
    ref = torch.load(tmp_path / "plain.pt")
    for k in ("out", "dense"):
        assert T.row_errors(got[k], ref[k]).max() < T.ROW_BOUND, k
