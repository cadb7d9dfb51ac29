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


def test_window_rejects_bad_arguments_before_launch(L):
    p, st = ctypes.c_void_p(0x1000), ctypes.c_void_p(0x2000)
    #     q  k  v  o  H  Hk sq  skv  q strides    kv strides   rows rank head     row  scale
    ok = [p, p, p, p, 8, 2, 64, 500, 64 * 128, 128, 500 * 128, 128, 64, 0, 64 * 128, 128, ctypes.c_float(0.09),
          100, 0, 4, 1, 436, 1, None, 0, st, None]  # left right sinks causal q_start splits ws bytes status stream
    for at, value, code in ((0, None, -1), (25, None, -1), (3, ctypes.c_void_p(0x1008), -2), (4, 9, -3), (5, 0, -3),
                            (6, 0, -3), (7, 0, -3), (7, (1 << 29) + 1, -3), (19, -1, -3), (21, 1 << 30, -3),
                            (22, -1, -3), (22, 65, -3), (12, 0, -3), (16, ctypes.c_float(0.0), -3),
                            (16, ctypes.c_float(float("nan")), -3), (9, 100, -4), (9, 120, -4), (11, 64, -4),
                            (8, 0, -4), (10, 0, -4), (15, 64, -4), (14, -8, -4)):
        bad = list(ok)
        bad[at] = value
        assert L.h3_window_attn(*bad) == code, (at, value)
    bad = list(ok)
    bad[4], bad[5] = 258, 2  # more than 128 query heads to a key head
    assert L.h3_window_attn(*bad) == -3
    assert L.h3_window_attn_workspace(8, 3, 64, 500, 100, 0, 4, 1, 436, 0) == -3
    assert L.h3_window_attn_workspace(8, 2, 64, 500, 100, 0, 4, 1, 436, 65) == -3


def _walk(left, right, sinks, causal, s_kv, p_first, p_last, tile=128):
    """The key tiles of a CTA whose rows sit at positions p_first .. p_last: (first key, end of its run)."""
    lo, hi = max(0, p_first - left), min(s_kv - 1, p_last + right)
    ns = max(0, min(sinks, p_last + 1)) if causal else sinks
    window = lo <= hi
    joined = window and lo <= ns
    out = [] if joined else [(b, ns) for b in range(0, ns, tile)]
    if window:
        start, end = (0, max(hi + 1, ns)) if joined else (lo, hi + 1)
        out += [(b, end) for b in range(start, end, tile)]
    return out


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("left,right,sinks", [(0, 0, 0), (5, 3, 0), (5, 0, 7), (200, 40, 150), (1000, 1000, 300)])
def test_window_walk_covers_each_visible_key_once(left, right, sinks, causal):
    """The walk the kernel takes, restated: every key that a row sees lies in exactly one tile in which the row's mask
    lets it through, tiles start inside the keys, and no key of a run is one that no row sees."""
    s_kv, right = 700, 0 if causal else right
    for p_first, p_last in ((0, 0), (0, 255), (100, 227), (600, 699), (690, 800), (-40, 20), (-300, -100), (900, 950)):
        tiles = _walk(left, right, min(sinks, s_kv), causal, s_kv, p_first, p_last)
        ns_all = max(0, min(sinks, p_last + 1)) if causal else sinks
        first_run = [t for t in tiles if t[1] == ns_all and t[0] % 128 == 0 and t[0] < ns_all]
        assert all(0 <= b < s_kv for b, _ in tiles)
        seen_any = set()
        for p in {p_first, (p_first + p_last) // 2, p_last}:
            see = {j for j in range(s_kv) if (j < sinks or p - left <= j <= p + right) and (not causal or j <= p)}
            seen_any |= see
            got = []
            for b, end in tiles:
                separate = (b, end) in first_run and len(tiles) > 0 and end == ns_all and max(0, p_first - left) > ns_all
                for j in range(b, min(b + 128, s_kv)):
                    ns = min(sinks, p + 1) if causal else sinks
                    in_window = (not separate) and max(0, p - left) <= j <= min(s_kv - 1, p + right)
                    if in_window or j < ns:
                        assert j < end
                        got.append(j)
            assert sorted(got) == sorted(see), (p_first, p_last, p)


def test_adapters_reject_bad_arguments_before_launch(L):
    p, st = ctypes.c_void_p(0x1000), ctypes.c_void_p(0x2000)
    #     a  m  chunks cols cstride row  w  n    wrow A  Arow B  Brow rank na scale rows c  crow ep ws bytes status stream
    ok = [p, 300, 1, 512, 0, 512, p, 256, 512, p, 512, p, 64, 16, 4, p, p, p, 256, 0, p, 0, st, None]
    for at, value, code in ((0, None, -1), (9, None, -1), (11, None, -1), (15, None, -1), (16, None, -1), (20, None, -1),
                            (9, ctypes.c_void_p(0x1008), -2), (20, ctypes.c_void_p(0x1008), -2),
                            (16, ctypes.c_void_p(0x1002), -2), (13, 12, -3), (13, 4, -3), (13, 96, -3), (13, 320, -3),
                            (14, 0, -3), (14, 4097, -3), (7, 100, -3), (19, 2, -3), (10, 504, -4), (12, 56, -4),
                            (12, 68, -4), (18, 128, -4), (8, 256, -4)):
        bad = list(ok)
        bad[at] = value
        assert L.h3_gemm_adapters(*bad) == code, (at, value)
    assert L.h3_gemm_adapters(*ok) == -12  # no workspace bytes
    need = L.h3_gemm_adapters_workspace(300, 1, 512, 256, 0, 16, 4)
    assert need >= 300 * 16 * 2
    assert L.h3_gemm_adapters_workspace(0, 1, 512, 256, 0, 16, 4) == -3
    assert L.h3_gemm_adapters_workspace(300, 1, 512, 256, 0, 24, 4) == -3
    assert L.h3_gemm_adapters_workspace(300, 1, 1 << 24, 1 << 30, 1, 16, 4) == -3


def test_stack_adapters():
    import h3attn as O
    A = [torch.randn(r, 40) for r in (3, 20)]
    B = [torch.randn(16, r) for r in (3, 20)]
    a, b, s = O.stack_adapters(zip(A, B), [1, 0.5])
    assert a.shape == (64, 40) and b.shape == (16, 64) and s.tolist() == [1.0, 0.5]
    assert torch.equal(a[:3], A[0].bfloat16()) and not a[3:32].any() and torch.equal(a[32:52], A[1].bfloat16())
    assert torch.equal(b[:, 32:52], B[1].bfloat16()) and not b[:, 52:].any()
    for bad in (([], []), ([(A[0], B[0])], [1, 2]), ([(A[0], B[1])], [1]), ([(torch.zeros(300, 8), torch.zeros(8, 300))], [1]),
                ([(A[0], B[0] * float("nan"))], [1])):
        with pytest.raises(O.H3Error):
            O.stack_adapters(*bad)


@pytest.mark.parametrize("tiles,n_kb,chunks,sms", [(1, 1, 0, 148), (168, 84, 6, 148), (42, 112, 1, 148),
                                                   (252, 4, 256, 148), (9, 3, 2, 4), (2, 1000, 0, 3), (7, 30, 40, 148)])
def test_streamed_blocks_are_dealt_once(tiles, n_kb, chunks, sms):
    """The row path's split of (tile, k-block) over CTAs, restated: every block in one CTA, a tile's pieces numbered
    from 0 without gaps, and never more of them than the workspace holds, whatever the chunks in use add."""
    ctas = max(1, min(2 * sms, tiles * n_kb // 4))
    most = -(-ctas // tiles) + 2
    per_tile = n_kb + chunks
    total = tiles * per_tile
    per = -(-total // ctas)
    seen = set()
    for cta in range(ctas):
        g, end = min(total, cta * per), min(total, cta * per + per)
        while g < end:
            tile, kb0 = divmod(g, per_tile)
            kb1 = min(per_tile, kb0 + end - g)
            first, last = tile * per_tile // per, ((tile + 1) * per_tile - 1) // per
            assert 0 <= cta - first <= last - first < most
            for kb in range(kb0, kb1):
                assert (tile, kb) not in seen
                seen.add((tile, kb))
            g += kb1 - kb0
    assert len(seen) == total


def test_launch_order_of_query_blocks():
    """The window kernel's launch order, restated: every (block, head) once; the middle first, then the ends from the
    middle outwards, where walks get shorter."""
    import itertools

    def block_of(w, blocks, first, mid, heads, turn):
        if w < mid * heads:
            return first + w % mid, w // mid
        ends, u = blocks - mid, w - mid * heads
        kvh, k = (u % heads, u // heads) if turn else (u // ends, u % ends)
        before, behind = first, ends - first
        both = 2 * min(before, behind)
        i = k >> 1 if k < both else k - (both >> 1)
        front = k % 2 == 0 if k < both else before > behind
        return (before - 1 - i if front else first + mid + i), kvh

    for blocks in range(1, 9):
        for first in range(blocks + 1):
            for mid in range(blocks - first + 1):
                for heads, turn in itertools.product((1, 3), (False, True)):
                    got = [block_of(w, blocks, first, mid, heads, turn) for w in range(blocks * heads)]
                    assert sorted(got) == sorted(itertools.product(range(blocks), range(heads)))
                    for h in range(heads):
                        far = [max(first - b, b - first - mid + 1, 0) for b, kvh in got if kvh == h]
                        assert far == sorted(far)


def test_rank_of_a_head_by_multiplication():
    """h // heads_per_rank as the pack computes it (2 heads a rank and more), for every head it takes."""
    for per in list(range(2, 300)) + [1000, 4095, 32768, 65535]:
        magic = (2 ** 32 + per - 1) // per
        assert magic < 2 ** 32
        for h in {0, 1, per - 1, per, min(per + 1, 65535), min(2 * per - 1, 65535), 65534, 65535 - 65535 % per, 65535}:
            assert h * magic >> 32 == h // per


def test_whole_warps_at_cluster_barriers_and_tensor_memory():
    """Cluster barriers and the release of tensor memory take whole warps (.aligned): their wrappers bring the warp
    together themselves, whatever the code before them left."""
    import re
    here = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    src = open(os.path.join(here, "minimaxh3-on-a100-x4_b200", "csrc", "h3_ptx.cuh")).read()
    for name in ("cluster_sync_all", "tmem_dealloc", "tmem_dealloc_pair"):
        body = re.search(r"void %s\([^)]*\) \{\n(.*?)\n\}" % name, src, re.S).group(1)
        assert body.lstrip().startswith("__syncwarp();"), name


def test_row_independent_adapters_take_the_tiles(L):
    """The flag asks for the launch whose rows do not depend on the call's length: its workspace grows with the rows
    and the chunk lists alone, also below 65 rows, and needs no device to size."""
    flag = 0x100
    tiles = lambda m: (m * 16 * 2 + 255) // 256 * 256 + (m + 255) // 256 * (1 + 1) * 4  # noqa: E731
    for m in (1, 40, 64, 65, 300):
        assert L.h3_gemm_adapters_workspace(m, 1, 512, 256, flag, 16, 4) == tiles(m)
        assert L.h3_gemm_adapters_workspace(m, 1, 512, 256, flag | 1, 16, 4) == tiles(m)
    assert L.h3_gemm_adapters_workspace(300, 1, 512, 256, 0, 16, 4) == tiles(300)
    assert L.h3_gemm_adapters_workspace(300, 1, 512, 256, flag | 2, 16, 4) == -3
    assert L.h3_gemm_adapters_workspace(300, 1, 512, 256, 2 * flag, 16, 4) == -3
    p, st = ctypes.c_void_p(0x1000), ctypes.c_void_p(0x2000)
    ok = [p, 20, 1, 512, 0, 512, p, 256, 512, p, 512, p, 64, 16, 4, p, p, p, 256, flag, p, 0, st, None]
    assert L.h3_gemm_adapters(*ok) == -12
    assert L.h3_gemm_adapters(*(ok[:19] + [flag | 2] + ok[20:])) == -3


def test_status_is_read_on_its_devices_stream(monkeypatch):
    """check_status(device) waits for the stream of that device, not of the current one (faked: no GPU)."""
    import contextlib

    import h3attn as O
    current, read = [0], []

    class Word:
        get_device = staticmethod(lambda: 3)
        data_ptr = staticmethod(lambda: 0x1000)

    class Lib:
        @staticmethod
        def h3_status_read(status, stream):
            read.append((status.value, stream.value))
            return 0

    @contextlib.contextmanager
    def device(index):
        before, current[0] = current[0], index
        yield
        current[0] = before

    monkeypatch.setattr(O, "lib", Lib)
    monkeypatch.setattr(O, "status_word", lambda device=None: Word)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: current[0])
    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(O, "_stream", lambda: 0x100 + current[0])
    O.check_status(torch.device("cuda", 3))
    assert read == [(0x1000, 0x103)] and current == [0]
