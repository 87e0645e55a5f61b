"""The work plan of the shared-prefix decode (flydsl_amd/csrc/sp_plan.h) on
the host: every tile of every item is worked exactly once, pieces have slots
of their own inside the workspace, and a piece of an item belongs to each
worker between its first and its last."""

from __future__ import annotations

import numpy as np
import pytest

from flydsl_amd import _lib

TILE = 64


def rows_of(eq, d):
    """Rows of an item."""
    most = 2 if d <= 128 else 1
    if eq <= 16 and d <= 128:
        return 16
    return 32 if eq <= 32 else 64 if eq <= 64 else 64 * most


def check(ctx, indptr, prefix, hkv, ql, gqa, d, capacity, workers):
    pieces = _lib.plan_shared_prefix(ctx, indptr, prefix, hkv, ql, gqa, d, capacity, workers)
    B, G, eq = len(ctx), len(prefix), ql * gqa
    first = np.maximum.accumulate(np.clip(indptr, 0, B)) if G else np.zeros(1, int)
    own = [0] * B
    want = {}  # (prefix, item) -> (of, head, first tile, end tile)
    p_rows, s_rows = rows_of(max(-(-B * eq // max(G, 1)), eq), d), rows_of(eq, d)
    most = [workers * (4 if r == 16 else 1) for r in (s_rows, p_rows)]  # a wave alone, or a workgroup
    item = 0
    for g in range(G):
        rows = (first[g + 1] - first[g]) * eq
        p = min(max(prefix[g], 0), capacity) if rows else 0
        for b in range(first[g], first[g + 1]):
            own[b] = p
        tiles = -(-rows // p_rows) if p else 0
        for h in range(hkv):
            for _ in range(tiles):
                want[1, item] = (g, h, 0, -(-p // TILE))
                item += 1
    bound = (B * eq // p_rows + min(G, B)) * hkv if G else 0
    assert item <= bound
    ct = -(-eq // s_rows)
    for b in range(B):
        n = min(max(ctx[b], 0), capacity)
        if n > own[b]:
            for i in range(hkv * ct):
                want[0, b * hkv * ct + i] = (b, i // ct, own[b] // TILE, -(-n // TILE))
    got, slots = {}, set()
    for is_p, it, w, slot, of, h, t0, t1 in pieces.tolist():
        assert t1 > t0 and 0 <= w < most[is_p]
        assert (is_p, slot) not in slots and 0 <= slot < (bound if is_p else B * hkv * ct) + most[is_p]
        slots.add((is_p, slot))
        got.setdefault((is_p, it), []).append((of, h, t0, t1, w, slot))
    assert got.keys() == want.keys()
    for key, (of, h, t0, t1) in want.items():
        ps = got[key]
        assert ps[0][2] == t0 and ps[-1][3] == t1
        assert all(p[:2] == (of, h) for p in ps)
        for a, b in zip(ps, ps[1:]):
            assert b[2] == a[3] and b[4] == a[4] + 1 and b[5] == a[5] + 1
    return pieces


CASES = [
    # ctx, indptr, prefix, hkv, ql, gqa, d
    ([500 + i for i in range(4)], [0, 4], [500], 2, 1, 4, 128),
    ([1], [0, 1], [0], 1, 1, 1, 64),
    ([1, 2, 3], [0, 3], [1], 1, 1, 8, 256),
    ([33000 + 50 * i for i in range(32)], [0, 32], [32768], 8, 1, 4, 128),
    ([17000 + i for i in range(256)], [0, 256], [16383], 8, 1, 4, 128),
    ([3000 * (i % 7) for i in range(128)], [0, 5, 5, 90, 120], [1000, 77, 4096, 64], 4, 4, 16, 128),
    ([0] * 5, [0, 3], [0], 2, 1, 4, 128),
    ([0] * 5, [0, 3], [100], 2, 1, 4, 128),
    ([100, 50, 0], [0, 3], [80], 2, 2, 150, 128),  # 300 columns: two suffix items a head
    ([700] * 9, [2, 7], [640], 3, 1, 2, 192),  # sequences before and behind the group
    ([700] * 9, [5, 2, 30], [640, 100], 3, 1, 2, 64),  # bounds that fall and pass the batch
    ([900] * 6, [], [], 2, 1, 4, 128),  # no groups
    ([64] * 300, [0, 300], [63], 8, 1, 4, 128),
]


@pytest.mark.parametrize("case", CASES)
@pytest.mark.parametrize("workers", [1, 7, 256])
def test_every_tile_once(case, workers):
    ctx, indptr, prefix, hkv, ql, gqa, d = case
    check(ctx, indptr or [0], prefix, hkv, ql, gqa, d, 1 << 20, workers)


def test_random_plans():
    rng = np.random.default_rng(3)
    for _ in range(150):
        B = int(rng.integers(1, 40))
        G = int(rng.integers(0, min(B, 6) + 1))
        indptr = np.sort(rng.integers(0, B + 1, G + 1))
        top = int(10 ** rng.uniform(0, 4.5))
        check(rng.integers(0, top + 1, B).tolist(), indptr.tolist(), rng.integers(0, top + 1, G).tolist(),
              int(rng.integers(1, 9)), int(rng.integers(1, 5)), int(rng.choice([1, 2, 4, 7, 16, 40])),
              int(rng.choice([64, 128, 256])), int(rng.choice([512, 1 << 20])), int(rng.integers(1, 300)))


def test_lengths_are_held_to_a_table_row():
    p = check([10**9, 70], [0, 2], [10**8], 1, 1, 4, 128, 256, 16)
    assert p[:, 7].max() == 4


def test_shares_are_even():
    """On a long line no workgroup gets more than a tile and a piece's overhead
    beyond the mean."""
    pieces = check([17000 + i for i in range(256)], [0, 256], [16383], 8, 1, 4, 128, 1 << 20, 256)
    cost = np.zeros(256)
    for is_p, _, w, _, _, _, t0, t1 in pieces.tolist():
        cost[w if is_p else w // 4] += 160 + (t1 - t0) * 64 if is_p else 40 + (t1 - t0) * 22
    assert cost.max() <= cost.mean() + 64 + 160


def test_refusals():
    def code(*a):
        with pytest.raises(RuntimeError) as e:
            _lib.shared_prefix_workspace_bytes(*a)
        return str(e.value)

    assert "PA_ERR_HEAD_SIZE" in code(4, 1, 2, 1, 4, 96, 256)
    for bad in ((4097, 1, 2, 1, 4, 128, 256), (4, 1025, 2, 1, 4, 128, 256), (4, 1, 0, 1, 4, 128, 256),
                (4, 1, 2, 0, 4, 128, 256), (4, 1, 2, 1, 0, 128, 256), (4, 1, 2, 1, 4, 128, 0),
                (2049, 1, 2, 1, 4, 192, 256), (4, 513, 2, 1, 4, 192, 256), (513, 1, 2, 1, 4, 256, 256),
                (4, 129, 2, 1, 4, 256, 256)):
        assert "PA_ERR_SHAPE" in code(*bad)
