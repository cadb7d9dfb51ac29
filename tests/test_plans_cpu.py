"""The plans of the window, adapter and pack kernels, computed on the host by the kernels' own functions
(h3_*_kat entry points): every key, k-block and head once, masks equal to the definition. No GPU."""
import ctypes
import os

import numpy as np
import pytest


@pytest.fixture(scope="module")
def L():
    import h3attn
    if not os.path.exists(h3attn.LIB_PATH):
        from build import build
        build()
    return h3attn.lib()


def _ints(n, dtype=np.int32):
    a = np.zeros(n, dtype=dtype)
    return a, a.ctypes.data_as(ctypes.c_void_p)


def _plan(L, *shape, most=200000):
    out, p = _ints((most, 8))
    n = L.h3_window_plan_kat(*shape, p, most)
    assert n >= 0, n
    return out[:n]


def _seen(p, left, right, sinks, causal, s_kv):
    """Keys that position p sees: the definition."""
    j = np.arange(s_kv)
    near = np.ones(s_kv, bool)
    if left >= 0:
        near &= j >= p - left
    if not causal and right >= 0:
        near &= j <= p + right
    see = near | (j < sinks)
    return see & (j <= p) if causal else see


# heads, key heads, queries, keys, left, right, sinks, causal, q_start, splits, SMs
WINDOWS = [
    (1, 1, 1, 1, 0, 0, 0, 0, 0, 1, 148), (2, 2, 300, 300, 5, 3, 0, 0, 0, 1, 148), (2, 1, 700, 700, 200, 150, 150, 0, 0, 1, 4),
    (3, 3, 600, 900, 40, 0, 17, 1, 300, 1, 4), (4, 2, 513, 700, -1, 0, 0, 1, 187, 1, 148), (7, 1, 90, 400, 31, 0, 3, 1, 310, 2, 148),
    (10, 2, 64, 1500, 1000, 0, 300, 1, 1436, 7, 148), (2, 2, 500, 400, 60, 10, 20, 0, -200, 1, 3), (2, 2, 500, 400, 60, 10, 0, 1, -200, 3, 3),
    (2, 2, 300, 400, 60, 10, 20, 0, 700, 2, 148), (128, 1, 9, 333, 50, 0, 9, 1, 324, 1, 148), (5, 5, 1, 777, 100, 0, 64, 0, 600, 64, 148),
    (2, 2, 300, 500, -1, -1, 0, 0, -(1 << 29), 1, 148), (2, 2, 300, 500, -1, 0, 0, 1, 1 << 29, 2, 148),
    (2, 2, 300, 500, 1 << 29, 5, 3, 0, 1 << 29, 1, 148), (1, 1, 200, 500, 0, 1 << 62, 0, 0, -(1 << 29), 1, 148),
    (1, 1, 260, 500, 128, 128, 128, 0, 0, 1, 148), (1, 1, 260, 500, 0, 0, 129, 0, 240, 1, 148), (40, 40, 400, 400, 10, 10, 5, 0, 0, 0, 6),
    (6, 2, 900, 300, 20, 0, 0, 0, -100, 0, 5),
]


@pytest.mark.parametrize("case", WINDOWS, ids=str)
def test_window_plan_shows_each_row_its_keys_once(L, case):
    H, hk, s_q, s_kv, left, right, sinks, causal, q_start, splits, sms = case
    rows = _plan(L, *case)
    group = H // hk
    tile_pos = 128 // group
    tiles = 1 if s_q <= tile_pos else 2
    per_item = tiles * tile_pos
    # every (key head, block, part) is one item, and a CTA has at most one a round
    items = {}
    for r in rows.tolist():
        items.setdefault((r[2], r[3], r[4]), []).append(r)
    parts = max(splits, 1) if splits else max(k[2] for k in items) + 1
    assert set(items) == {(h, i0, z) for h in range(hk) for i0 in range(0, s_q, per_item) for z in range(parts)}
    places = {}
    for key, group_rows in items.items():
        assert len({(r[0], r[1]) for r in group_rows}) == 1
        places.setdefault((group_rows[0][0], group_rows[0][1]), []).append(key)
    assert all(len(v) == 1 for v in places.values())
    if tiles == 2:
        assert max(c for c, _ in places) < sms

    bits, bits_p = _ints(4, np.uint32)
    for i0 in range(0, s_q, per_item):
        walks = [[(r[5], r[6], r[7]) for z in range(parts) for r in items[h, i0, z] if r[5] >= 0] for h in range(hk)]
        assert all(w == walks[0] for w in walks)
        queries = range(i0, min(i0 + per_item, s_q))
        defined = np.stack([_seen(q_start + i, left, right, sinks, causal, s_kv) for i in queries])
        some = set(np.flatnonzero(defined.any(0)).tolist())
        loaded = [j for key, end, _ in walks[0] for j in range(key, min(key + 128, end))]
        assert len(loaded) == len(set(loaded)) and set(loaded) == some, i0  # no key that no row sees, each once
        for n, i in enumerate(queries):
            if n not in (0, 1, tile_pos - 1, tile_pos, len(queries) - 1, len(queries) // 3):
                continue
            got = []
            for key, end, flags in walks[0]:
                assert 0 <= key < s_kv
                if flags >> (1 + n // tile_pos) & 1:
                    assert L.h3_window_mask_kat(s_kv, left, right, sinks, causal, s_q, q_start, i, key, flags & 1, bits_p) == 0
                    mine = [key + e for e in range(128) if bits[e // 32] >> (e % 32) & 1]
                    assert all(j < end for j in mine)
                    got += mine
                else:
                    got += list(range(key, key + 128))
            assert sorted(got) == np.flatnonzero(defined[n]).tolist(), (i0, i)


def test_window_launch_order(L):
    """Blocks with whole windows first, head by head; then those at the two ends of the sequence, each side from its longest
    walk down."""
    for causal, left, right in ((0, 511, 512), (1, -1, 0), (1, 1000, 0)):
        rows = _plan(L, 7, 7, 6000, 6000, left, right, 64, causal, 0, 1, 20)
        length, order = {}, {}
        for c, r, h, i0, _, _, _, _ in rows.tolist():
            length[h, i0] = length.get((h, i0), 0) + 1
            order[r * 20 + (19 - c if r & 1 else c)] = (h, i0)
        assert sorted(order) == list(range(len(order)))
        walk = [order[w] for w in sorted(order)]
        top = max(length.values())
        last_whole = max(n for n, item in enumerate(walk) if length[item] == top)
        assert min(length[item] for item in walk[:last_whole + 1]) >= top - 1  # the sequence's last tile may be short
        ends = walk[last_whole + 1:]
        for h in range(7):
            for front in (True, False):
                side = [length[item] for item in ends if item[0] == h and (item[1] < 3000) == front]
                assert side == sorted(side, reverse=True)


def test_window_plan_refusals(L):
    out, p = _ints((10, 8))
    ok = [2, 2, 300, 300, 5, 3, 0, 0, 0, 1, 148]
    assert L.h3_window_plan_kat(*ok, None, 10) == -1
    assert L.h3_window_plan_kat(*ok, p, 3) == -12 and not out[3:].any()
    assert L.h3_window_plan_kat(*(ok[:10] + [0]), p, 10) == -3 and L.h3_window_plan_kat(*(ok[:1] + [3] + ok[2:]), p, 10) == -3
    assert L.h3_window_plan_kat(8, 8, 1, 500, -1, 0, 0, 1, 499, 0, 148, p, 10) == -8  # the single-token kernel
    bits, bp = _ints(4, np.uint32)
    for query, key in ((-1, 0), (300, 0), (0, -1), (0, 300)):
        assert L.h3_window_mask_kat(300, 5, 3, 0, 0, 300, 0, query, key, 0, bp) == -3
    assert L.h3_window_mask_kat(300, 5, 3, 0, 0, 300, 0, 0, 0, 0, None) == -1


@pytest.mark.parametrize("w_rows,n_kb,chunks,sms", [(128, 1, 0, 148), (21504, 84, 6, 148), (5376, 112, 1, 148),
                                                    (32256, 4, 256, 148), (1150, 3, 2, 4), (200, 1000, 0, 3), (896, 30, 40, 148),
                                                    (8, 1, 1, 148), (32256, 4, 1, 148)])
def test_streamed_blocks_are_dealt_once(L, w_rows, n_kb, chunks, sms):
    """Every k-block of every tile in one piece of one CTA, a tile's pieces numbered from 0 without gaps in the order of
    their k-blocks, and never more of them than the workspace holds."""
    out, p = _ints((500000, 6))
    most = ctypes.c_int64()
    n = L.h3_adapters_deal_kat(w_rows, n_kb, chunks, sms, p, len(out), ctypes.byref(most))
    assert n > 0
    tiles, ctas = -(-w_rows // 128), set()
    covered = {}
    for cta, tile, kb0, kb1, piece, pieces in out[:n].tolist():
        assert 0 <= tile < tiles and 0 <= kb0 < kb1 <= n_kb + chunks and 0 <= piece < pieces <= most.value
        covered.setdefault(tile, []).append((piece, kb0, kb1, pieces))
        ctas.add(cta)
    assert set(covered) == set(range(tiles)) and max(ctas) < 2 * sms
    for parts in covered.values():
        parts.sort()
        assert [q[0] for q in parts] == list(range(parts[0][3]))
        assert [q[1] for q in parts] == [0] + [q[2] for q in parts[:-1]] and parts[-1][2] == n_kb + chunks


def test_deal_refusals(L):
    out, p = _ints((4, 6))
    most = ctypes.c_int64()
    assert L.h3_adapters_deal_kat(1024, 84, 2, 148, p, 3, ctypes.byref(most)) == -12
    assert L.h3_adapters_deal_kat(1024, 84, 2, 148, None, 3, ctypes.byref(most)) == -1
    for bad in ((0, 84, 2, 148), (1024, 0, 2, 148), (1024, 84, -1, 148), (1024, 84, 257, 148), (1024, 84, 2, 0)):
        assert L.h3_adapters_deal_kat(*bad, p, 4, ctypes.byref(most)) == -3


def test_rank_of_every_head(L):
    for n, per in [(56, d) for d in (1, 2, 4, 7, 8, 14, 28, 56)] + [(65535, d) for d in (1, 2, 3, 255, 4369, 21845, 65535)]:
        out, p = _ints(n)
        assert L.h3_pack_ranks_kat(n, per, p) == 0
        assert np.array_equal(out, np.arange(n) // per)
    for n in (977, 4096, 65000):
        for per in list(range(1, 60)) + [n - 1, n]:
            out, p = _ints(n)
            assert L.h3_pack_ranks_kat(n, per, p) == 0 and np.array_equal(out, np.arange(n) // per)
    assert L.h3_pack_ranks_kat(8, 2, None) == -1 and L.h3_pack_ranks_kat(0, 1, p) == -3 and L.h3_pack_ranks_kat(8, 9, p) == -3


@pytest.mark.parametrize("group,kv_heads,keys,token", [
    (1, 56, 8000, True), (1, 56, 8300, False), (1, 28, 2000, True), (1, 28, 2200, False), (1, 200, 2000, True),
    (2, 28, 2000, True), (2, 32, 1000, True), (2, 37, 1000, False), (2, 56, 500, True), (2, 56, 1000, False), (2, 56, 8000, False),
    (3, 8, 2000, True), (3, 40, 700, True), (3, 60, 700, False), (4, 20, 1500, True), (4, 20, 1600, False), (4, 100, 250, True),
    (4, 100, 500, False), (4, 56, 4000, False), (5, 4, 100, False)])
def test_which_single_tokens_leave_the_tiles(L, group, kv_heads, keys, token):
    """Both sides of the rule, on 148 SMs."""
    out, p = _ints((400000, 8))
    n = L.h3_window_plan_kat(group * kv_heads, kv_heads, 1, keys, -1, 0, 0, 1, keys - 1, 0, 148, p, len(out))
    assert (n == -8) == token
    assert L.h3_window_plan_kat(group * kv_heads, kv_heads, 1, keys, -1, 0, 0, 1, keys - 1, 1, 148, p, len(out)) > 0
