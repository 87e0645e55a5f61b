"""The page operators' launchers and C entries refuse bad calls on the CPU,
and the one-entry-at-a-time oracle keeps the pool's books."""

from __future__ import annotations

import ctypes
import os
import subprocess

import numpy as np
import pytest
import torch

from flydsl_amd import (_lib, compact_cache_pages, copy_cache_pages, extend_cache_pages, fork_cache_pages,
                        free_cache_pages)
from oracle import cache_pages as oracle
from tests._page_cases import make_pool

i32 = lambda *x: torch.tensor(x, dtype=torch.int32)


def holders(tables, lengths, pages, bs):
    refs = np.zeros(pages, np.int32)
    for r, n in enumerate(lengths):
        np.add.at(refs, tables[r, : -(-int(n) // bs)], 1)
    return refs


@pytest.mark.parametrize("seed", range(6))
def test_oracle_keeps_the_books(seed):
    """After any run of operators a page's count is the number of rows that
    hold it, and a row's tokens are where they were."""
    bs, pages = 16, 48
    rng = np.random.default_rng(seed)
    t, n, refs = make_pool(rows=10, width=8, pages=pages, bs=bs, seed=seed, empty=4)
    assert (refs == holders(t, n, pages, bs)).all()
    cache = rng.integers(0, 1 << 30, (pages, bs))
    read = lambda: [cache[t[r, np.arange(k) // bs], np.arange(k) % bs] for r, k in enumerate(n)]
    for _ in range(12):
        before, was = read(), n.copy()
        op = rng.integers(4)
        rows = rng.permutation(10)[:4]
        if op == 0:
            oracle.fork(t, n, refs, rows[:2], rows[2:], bs)
        elif op == 1:
            oracle.extend([cache], t, n, refs, rows, n[rows] + rng.integers(0, 20, 4), bs)
        elif op == 2:
            oracle.free(t, n, refs, rows[:2], bs, (n[rows[:2]] * rng.random(2)).astype(int))
        else:
            t, refs, _, live = oracle.compact([cache], t, n, refs, bs)
            assert (refs[:live] > 0).all() and not refs[live:].any()
        assert (refs == holders(t, n, pages, bs)).all()
        for r, row in enumerate(read()):
            k = min(len(row), was[r])
            assert (row[:k] == before[r][:k]).all()


def state(rows=4, width=3, pages=8):
    return torch.zeros(rows, width, dtype=torch.int32), torch.zeros(rows, dtype=torch.int32), torch.zeros(pages, dtype=torch.int32)


def test_refusals():
    t, n, r = state()
    cache = torch.zeros(8, 2, 16)

    def bad(match, fn, *a, err=ValueError, **kw):
        with pytest.raises(err, match=match):
            fn(*a, **kw)

    bad("on a GPU", fork_cache_pages, t, n, r, i32(0), i32(1), 16, err=RuntimeError)
    bad("on a GPU", copy_cache_pages, [cache], i32(0), i32(1), err=RuntimeError)
    bad("on a GPU", compact_cache_pages, [cache], t, n, r, 16, err=RuntimeError)
    bad("must be int32", fork_cache_pages, t.long(), n, r, i32(0), i32(1), 16)
    bad("2 dimensions", fork_cache_pages, t[0], n, r, i32(0), i32(1), 16)
    bad("one entry a table row", fork_cache_pages, t, n[:3], r, i32(0), i32(1), 16)
    bad("block_size", fork_cache_pages, t, n, r, i32(0), i32(1), 24)
    bad("block_size", fork_cache_pages, t, n, r, i32(0), i32(1), 0)
    bad("must have 1 entries", fork_cache_pages, t, n, r, i32(0), i32(1, 2), 16)
    bad("must be int32", fork_cache_pages, t, n, r, i32(0), i32(1).long(), 16)
    bad("must be contiguous", fork_cache_pages, t, n, r, i32(0, 1, 2, 3)[::2], i32(1, 2), 16)
    bad("last dimension", fork_cache_pages, t.t().contiguous().t(), n, r, i32(0), i32(1), 16)
    bad("must not overlap", fork_cache_pages, torch.zeros(1, 3, dtype=torch.int32).expand(4, 3), n, r, i32(0), i32(1), 16)
    bad("must have 2 entries", free_cache_pages, t, n, r, i32(0, 1), 16, new_lengths=i32(0))
    bad("8 pages", extend_cache_pages, [cache, cache[:4]], t, n, r, i32(0), i32(1), 16)
    bad("contiguous within a page", extend_cache_pages, [cache.transpose(1, 2)], t, n, r, i32(0), i32(1), 16)
    bad("must not overlap", copy_cache_pages, [cache[:1].expand(8, 2, 16)], i32(0), i32(1))
    bad("page dimension", copy_cache_pages, [torch.zeros(())], i32(0), i32(1))
    bad("at least one cache", copy_cache_pages, [], i32(0), i32(1))
    many = torch.zeros(5000, dtype=torch.int32)
    bad("at most 4096", extend_cache_pages, [cache], t, n, r, many, many, 16, err=NotImplementedError)
    bad("at most 65536", copy_cache_pages, [cache], many.repeat(14), many.repeat(14), err=NotImplementedError)
    bad("at most 4194304", free_cache_pages, t, n, torch.zeros((4 << 20) + 1, dtype=torch.int32), i32(0), 16,
        err=NotImplementedError)


def test_c_entries_refuse_before_any_launch():
    lib = _lib.load()
    P = 4096  # an aligned stand-in that nothing here reads
    t = _lib.PageTableArgs()
    fork = lambda n=1: lib.pa_fp8_fork_pages(t, P, P, n, P, None)
    assert lib.pa_fp8_fork_pages(None, P, P, 1, P, None) == -1
    t.abi_version = 99
    assert fork() == -8
    t.abi_version = _lib.ABI_VERSION
    t.block_tables = t.context_lengths = t.ref_counts = P
    t.stride_bt_seq, t.num_rows, t.max_blocks_per_seq, t.num_blocks, t.block_size = 3, 4, 3, 8, 16
    assert fork(0) == 0 and fork(65537) == -6 and fork(-1) == -6
    for f, v, code in (("block_size", 24, -3), ("block_size", 0, -3), ("num_blocks", (4 << 20) + 1, -6),
                       ("num_rows", -1, -6), ("ref_counts", None, -1), ("context_lengths", None, -1)):
        old = getattr(t, f)
        setattr(t, f, v)
        assert fork() == code, f
        assert lib.pa_fp8_free_pages(t, P, None, 1, P, None) == code
        assert lib.pa_fp8_extend_pages(t, None, 0, P, P, 1, P, P, 1 << 30, None) == code
        assert lib.pa_fp8_compact_pages(t, None, 0, P, 3, P, P, P, P, 1 << 30, None) == code
        setattr(t, f, old)
    c = (_lib.PageCache * 1)()
    c[0].data, c[0].stride_bytes, c[0].page_bytes = P, 64, 128
    assert lib.pa_fp8_copy_pages(c, 1, 8, P, P, 1, P, P, 1 << 20, None) == -6  # pages overlap
    c[0].stride_bytes, c[0].data = 128, None
    assert lib.pa_fp8_copy_pages(c, 1, 8, P, P, 1, P, P, 1 << 20, None) == -1
    c[0].data = P
    assert lib.pa_fp8_copy_pages(c, 1, 8, P, P, 0, P, P, 0, None) == 0
    assert lib.pa_fp8_copy_pages(c, 1, 8, P, P, 65, P, P, 8, None) == -9
    assert lib.pa_fp8_copy_pages(c, 1, 8, P, P, 65, P, None, 0, None) == -1
    assert lib.pa_fp8_extend_pages(t, c, 1, P, P, 4097, P, P, 1 << 30, None) == -6
    assert lib.pa_fp8_extend_pages(t, c, 1, P, P, 1, P, P, 16, None) == -9
    assert lib.pa_fp8_compact_pages(t, c, 1, P, 3, P, P, P, P, 16, None) == -9
    assert lib.pa_fp8_compact_pages(t, c, 1, P, 3, P, P, None, P, 1 << 30, None) == -1
    assert lib.pa_fp8_pages_workspace_bytes(7, 8, 1) == -6


@pytest.mark.parametrize("struct,cname", [(_lib.PageTableArgs, "pa_fp8_page_table_args"),
                                          (_lib.PageCache, "pa_fp8_page_cache"),
                                          (_lib.SharedPrefixArgs, "pa_fp8_shared_prefix_args")])
def test_struct_layout_matches_header(tmp_path, struct, cname):
    header = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "pa_fp8.h")
    fields = [f for f, _ in struct._fields_]
    c = tmp_path / "layout.c"
    c.write_text("\n".join(["#include <stdio.h>", "#include <stddef.h>", f'#include "{header}"', "int main(void){",
                            f'printf("%zu\\n", sizeof({cname}));']
                           + [f'printf("%zu\\n", offsetof({cname}, {f}));' for f in fields] + ["return 0;}"]))
    subprocess.run(["gcc", str(c), "-o", str(tmp_path / "layout")], check=True)
    out = subprocess.run([str(tmp_path / "layout")], capture_output=True, text=True, check=True).stdout
    assert [int(x) for x in out.split()] == [ctypes.sizeof(struct)] + [getattr(struct, f).offset for f in fields]
