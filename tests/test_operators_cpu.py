"""Entry points of the rotary, window and adapter operators on the CPU: plans, and arguments that are rejected before
any CUDA work."""
import ctypes
import os

import pytest
import torch


@pytest.fixture(scope="module")
def L():
    import h3attn
    if not os.path.exists(h3attn.LIB_PATH):
        from build import build
        build()
    return h3attn.lib()


def test_rope_plan():
    import h3attn as O
    f, a = O.rope_axes_freqs([2, 0, 3], theta=100.0)
    assert a.tolist() == [0, 0, 2, 2, 2] + [-1] * 59 and f.dtype == torch.float64
    assert torch.allclose(f[:5], torch.tensor([1, 100 ** -0.5, 1, 100 ** (-1 / 3), 100 ** (-2 / 3)],
                                              dtype=torch.float64), rtol=1e-15, atol=0)
    f, a = O.rope_axes_freqs([2, 1, 3], interleaved=True)
    assert a[:6].tolist() == [0, 1, 2, 0, 2, 2]
    for bad in ([65], [], [-1], [32, 33]):
        with pytest.raises(O.H3Error):
            O.rope_axes_freqs(bad)
    rp = O.RopePositions(torch.arange(10, dtype=torch.int32)[:, None], f, a)
    assert rp.rows(8, 12).pos[:, 0].tolist() == [8, 9, 0, 0] and rp.rows(12, 14).pos[:, 0].tolist() == [0, 0]


def test_rope_rejects_bad_arguments_before_launch(L):
    p = ctypes.c_void_p(0x1000)
    ok = [p, 256, 128, p, 0, 3, p, p, 0, p, 256, 128, 10, 2, None]
    for at, value, code in ((0, None, -1), (3, None, -1), (6, None, -1), (9, None, -1), (0, ctypes.c_void_p(0x1008), -2),
                            (6, ctypes.c_void_p(0x1004), -2), (4, 7, -3), (5, 0, -3), (5, 65, -3), (12, 0, -3),
                            (13, 0, -3), (12, 1 << 40, -3), (1, 257, -4), (10, 100, -4), (11, 64, -4), (2, -8, -4)):
        bad = list(ok)
        bad[at] = value
        assert L.h3_rope_axes(*bad) == code, (at, value)
    ok = [p, p, p, 3 * 4 * 128, p, 1, 2, p, p, None, None, ctypes.c_float(1e-6), p, p, p, 10, 4, 2, 4 * 10 * 128,
          10 * 128, None]
    for at, value, code in ((0, None, -1), (14, None, -1), (4, None, -1), (17, 3, -3), (5, 2, -3), (3, 4 * 128 - 8, -4),
                            (15, 0, -3), (18, 4, -4), (11, ctypes.c_float(-1.0), -3), (12, ctypes.c_void_p(0x1008), -2)):
        bad = list(ok)
        bad[at] = value
        assert L.h3_qknorm_rope_pack_axes(*bad) == code, (at, value)
    ok = [p, p, p, 4 * 128, p, 0, 1, p, p, None, None, ctypes.c_float(1e-6), p, 2, 20 * 128, 10 * 128, 0, 10, 4, 2,
          None]
    for at, value, code in ((12, None, -1), (12, ctypes.c_void_p(0x1004), -2), (13, 1, -3), (16, -1, -3), (19, 3, -3),
                            (14, 4, -4)):
        bad = list(ok)
        bad[at] = value
        assert L.h3_qknorm_rope_pack_axes_peer(*bad) == code, (at, value)


def test_rope_has_no_cpu_path():
    import h3attn as O
    f, a = O.rope_axes_freqs([64])
    rp = O.RopePositions(torch.zeros(4, 1, dtype=torch.int32), f, a)
    with pytest.raises(O.H3Error):
        O.rope_axes(torch.zeros(4, 1, 128, dtype=torch.bfloat16), rp)
