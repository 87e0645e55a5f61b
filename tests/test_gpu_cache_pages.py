"""The page operators against the one-entry-at-a-time oracle: whole numbers
and moved bytes have to be equal."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from flydsl_amd import (_lib, compact_cache_pages, copy_cache_pages, extend_cache_pages, fork_cache_pages,
                        free_cache_pages)
from oracle import cache_pages as oracle
from tests._page_cases import make_caches, make_pool
from tests.test_gpu_checked import checked  # noqa: F401 (a fixture)
from tests.test_gpu_native import both

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
FP8 = torch.float8_e4m3fn
# one unit and a part of one, bytes that no 16 divides, a scale a token
SHAPES = [(FP8, 2, 8, 16, 16), (torch.uint8, 5000, 4), (torch.bfloat16, 3, 7), (torch.float32, 2, 16, 1)]


def dev(x):
    return torch.tensor(np.ascontiguousarray(x), dtype=torch.int32, device=DEV)


class State:
    """The same state on the host (numpy) and on the device."""

    def __init__(self, t, n, refs, bs, shapes=SHAPES, seed=0, spare=3):
        self.bs, self.t, self.n, self.refs = bs, t, n, refs
        self.caches = make_caches(len(refs), shapes, seed)
        self.host = [c.view(torch.uint8).flatten(1).numpy().copy() for c in self.caches]
        self.dc = [c.to(DEV) for c in self.caches]
        wide = torch.full((t.shape[0], t.shape[1] + spare), -7, dtype=torch.int32, device=DEV)
        self.dt = wide[:, : t.shape[1]]  # rows further apart than they are wide
        self.dt.copy_(dev(t))
        self.wide = wide
        self.dn, self.dr = dev(n), dev(refs)

    def same(self):
        assert (self.dt.cpu().numpy() == self.t).all()
        assert (self.wide[:, self.t.shape[1]:] == -7).all()
        assert (self.dn.cpu().numpy() == self.n).all()
        assert (self.dr.cpu().numpy() == self.refs).all()
        for d, h in zip(self.dc, self.host):
            assert (d.view(torch.uint8).flatten(1).cpu().numpy() == h).all()

    def fork(self, parents, children):
        got = fork_cache_pages(self.dt, self.dn, self.dr, dev(parents), dev(children), self.bs)
        assert got.tolist() == oracle.fork(self.t, self.n, self.refs, parents, children, self.bs)
        self.same()
        return got.tolist()

    def free(self, seqs, new=None):
        got = free_cache_pages(self.dt, self.dn, self.dr, dev(seqs), self.bs,
                               new_lengths=None if new is None else dev(new))
        assert got.tolist() == oracle.free(self.t, self.n, self.refs, seqs, self.bs, new)
        self.same()
        return got.tolist()

    def extend(self, seqs, new):
        got = extend_cache_pages(self.dc, self.dt, self.dn, self.dr, dev(seqs), dev(new), self.bs)
        assert got.tolist() == oracle.extend(self.host, self.t, self.n, self.refs, seqs, new, self.bs)
        self.same()
        return got.tolist()

    def compact(self):
        old = [x.clone() for x in (self.dt, self.dn, self.dr)]
        out = compact_cache_pages(self.dc, self.dt, self.dn, self.dr, self.bs)
        want = oracle.compact(self.host, self.t, self.n, self.refs, self.bs)
        for g, w in zip(out, want):
            assert (g.cpu().numpy() == w).all()
        assert all(torch.equal(a, b) for a, b in zip(old, (self.dt, self.dn, self.dr)))
        self.same()
        self.t, self.refs = want[0], want[1]
        self.dt.copy_(out[0])
        self.dr.copy_(out[1])
        return want


def test_random_runs():
    """Runs of operators on pools of many sizes, lists with rows out of range,
    rows named twice and lengths that do not fit."""
    rng = np.random.default_rng(0)
    for k in range(24):
        rows, width = int(rng.integers(2, 40)), int(rng.integers(1, 12))
        pages, bs = int(rng.choice([3, 17, 40, 300, 20000])), int(rng.choice([1, 16, 64]))
        print(f"[pages] run {k}: rows {rows} width {width} pages {pages} page size {bs}", flush=True)
        s = State(*make_pool(rows, width, pages, bs, fill=width, seed=k, empty=rows // 2), bs,
                  shapes=SHAPES if pages < 1000 else SHAPES[2:])
        for _ in range(6):
            m = int(rng.integers(1, rows + 3))
            a, b = (rng.integers(-1, rows + 1, m).tolist() for _ in range(2))
            near = [int(s.n[min(max(x, 0), rows - 1)]) for x in a]
            s.fork(a, b)
            s.extend(a, [max(0, x + int(rng.integers(-2, 2 * bs + 2))) for x in near])
            s.free(b, [int(s.n[min(max(x, 0), rows - 1)] * rng.random()) for x in b])
            if rng.random() < 0.5:
                s.compact()
            if rng.random() < 0.3:
                s.free(a)


def test_extend_copies_shared_pages_until_the_last_holder():
    t = np.zeros((4, 3), np.int32)
    t[0, :2] = [5, 2]
    n, refs = np.array([20, 0, 0, 0], np.int32), np.zeros(8, np.int32)
    refs[[5, 2]] = 1
    s = State(t, n, refs, 16)
    assert s.fork([0, 0, 0], [1, 2, 3]) == [1, 1, 1]
    assert s.extend([3, 0, 2], [21, 40, 20]) == [1, 1, 1]  # row 2 asks for nothing
    assert s.t[2, 1] == 2 and s.refs[2] == 2
    assert s.extend([2, 1], [33, 21]) == [1, 1]  # row 2 copies, row 1 is the last holder
    assert s.t[1, 1] == 2 and s.refs[2] == 1
    s.free([0, 1, 2, 3])
    assert not s.refs.any()


def test_extend_stops_where_the_pool_ends():
    t, n, refs = np.zeros((5, 4), np.int32), np.zeros(5, np.int32), np.zeros(6, np.int32)
    s = State(t, n, refs, 16)
    assert s.extend([0, 1, 2, 3, 4], [33, 0, 17, 40, 0]) == [1, 1, 1, 0, 0]
    assert s.refs.sum() == 5
    assert s.extend([3, 4], [16, 0]) == [1, 1]
    assert s.extend([3], [17]) == [0]


def test_a_shared_page_is_safe_where_the_pool_ends():
    """The last holder may only keep the page when those before it got their
    copies."""
    t = np.zeros((3, 2), np.int32)
    refs = np.zeros(1, np.int32)
    refs[0] = 1
    s = State(t, np.array([5, 0, 0], np.int32), refs, 16)
    s.fork([0], [1])
    assert s.extend([0, 1], [6, 6]) == [0, 0]


def test_freeing_more_than_is_held():
    t = np.zeros((3, 2), np.int32)  # two rows claim page 0, which counts one holder
    s = State(t, np.array([5, 5, 0], np.int32), np.array([1, 0], np.int32), 16)
    s.free([0, 1])
    assert not s.refs.any()


@pytest.mark.parametrize("n", [1, 5, 64, 65, 700, 2051])
def test_copies(n):
    rng = np.random.default_rng(n)
    pages = 2 * n + 5
    s = State(np.zeros((1, 1), np.int32), np.zeros(1, np.int32), np.zeros(pages, np.int32), 16)
    p = rng.permutation(pages)
    for src, dst in (
        (p[:n], p[n:2 * n]),  # apart
        (rng.integers(-2, pages + 2, n), rng.integers(-2, pages + 2, n)),  # anything, chains and repeats among it
        (np.zeros(n, int), p[:n]),  # one page to many, itself perhaps
        (p[:n], np.full(n, p[-1])),  # many onto one: the last counts
    ):
        got = copy_cache_pages(s.dc, dev(src), dev(dst))
        assert got.tolist() == oracle.copy(s.host, src.tolist(), dst.tolist())
        s.same()


def test_copies_of_unaligned_and_interleaved_caches():
    """Pages whose bytes are apart (keys and values of a page side by side),
    begin off 16-byte lines, or do not fill them; more caches than one launch
    takes."""
    pages = 20
    base = torch.randint(0, 256, (pages, 3, 1003), dtype=torch.uint8, device=DEV)
    many = [torch.randint(0, 256, (pages, 48), dtype=torch.uint8, device=DEV) for _ in range(200)]
    caches = [base[:, 0], base[:, 2, 5:900], base[:, 1, :1000]] + many
    want = [c.clone() for c in caches]
    src, dst = dev([3, 4, 5]), dev([10, 11, 0])
    for w in want:
        w[dst.long()] = w[src.long()]
    copy_cache_pages(caches, src, dst)
    assert all(torch.equal(a, b) for a, b in zip(caches, want))
    copy_cache_pages(tuple(caches), dst, src)  # a tuple, and back: equal pages


def test_offsets_past_32_bits():
    """A cache of more than 4 GiB: the copy of its last pages."""
    pages = 5 * 2**10
    c = torch.empty((pages, 2**20), dtype=torch.uint8, device=DEV)
    c[-1], c[-2], c[3] = 7, 9, 11
    copy_cache_pages([c], dev([pages - 1, 3]), dev([0, pages - 2]))
    assert (c[0] == 7).all() and (c[pages - 2] == 11).all()


def test_large_pool():
    """Several counting workgroups: pages far apart, all but a few held."""
    pages, bs = 50000, 16
    rng = np.random.default_rng(5)
    refs = np.ones(pages, np.int32)
    free = np.sort(rng.choice(pages, 30, replace=False))
    refs[free] = 0
    t = np.zeros((6, 8), np.int32)
    s = State(t, np.zeros(6, np.int32), refs, bs, shapes=[(torch.int32, 8)])
    assert s.extend([0, 1, 2, 3, 4], [100, 128, 1, 0, 96]) == [1, 1, 1, 1, 1]
    assert sorted(s.t[0, :7].tolist() + s.t[1].tolist() + [s.t[2, 0]]) == free[:16].tolist()
    s.compact()
    refs[:] = 0
    refs[-3:] = 1
    t[0, :3] = [pages - 1, pages - 2, pages - 3]
    s = State(t, np.array([48, 0, 0, 0, 0, 0], np.int32), refs, bs, shapes=[(torch.int32, 8)])
    assert s.compact()[3] == 3
    s = State(t, np.zeros(6, np.int32), np.zeros(pages, np.int32), bs, shapes=[(torch.int32, 8)])
    assert s.compact()[3] == 0


def test_long_lists():
    """As many sequences as an extend takes, every one in need of a copy."""
    rows, bs = 4097, 16
    t = np.zeros((rows, 2), np.int32)
    n, refs = np.zeros(rows, np.int32), np.zeros(5000, np.int32)
    n[0], refs[0] = 3, 1
    s = State(t, n, refs, bs, shapes=[(torch.int32, 4)])
    s.fork([0] * 4096, list(range(1, 4097)))
    s.extend(list(range(1, 4097)), [4] * 4096)
    s.free(list(range(4097)))
    assert not s.refs.any()


def test_no_caches_and_empty_lists():
    s = State(np.zeros((3, 2), np.int32), np.zeros(3, np.int32), np.zeros(4, np.int32), 16)
    s.dc, s.host = [], []
    assert s.extend([0, 1], [20, 3]) == [1, 1]
    s.compact()
    e = torch.zeros(0, dtype=torch.int32, device=DEV)
    for st in (fork_cache_pages(s.dt, s.dn, s.dr, e, e, 16), free_cache_pages(s.dt, s.dn, s.dr, e, 16),
               extend_cache_pages([], s.dt, s.dn, s.dr, e, e, 16),
               copy_cache_pages([torch.zeros(4, 2, device=DEV)], e, e)):
        assert st.shape == (0,)
    z = torch.zeros(4, 0, device=DEV)  # nothing to copy; the entries are judged all the same
    assert copy_cache_pages([z], dev([0, 9]), dev([1, 2])).tolist() == [1, 0]
    s.same()


def test_streams_and_graphs():
    """On a stream of its own, and captured: a fork, an extend and a free
    replayed with eager work between give the state that eager calls give."""
    bs = 16
    make = lambda: State(*make_pool(12, 8, 60, bs, seed=3, empty=6), bs)
    a, b = make(), make()
    parents, children = dev([0, 1, 0]), dev([6, 7, 8])
    grown = dev([int(a.n[p]) + 5 for p in (0, 1, 0)])

    def step(s, **kw):
        fork_cache_pages(s.dt, s.dn, s.dr, parents, children, bs, **kw)
        return extend_cache_pages(s.dc, s.dt, s.dn, s.dr, children, grown, bs, **kw)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    st = step(b, stream=side)
    side.synchronize()
    step(a)
    assert st.tolist() == [1, 1, 1]
    agree = lambda: all(torch.equal(x.view(torch.uint8), y.view(torch.uint8))  # bytes: a NaN equals itself
                        for x, y in zip([a.dt, a.dn, a.dr] + a.dc, [b.dt, b.dn, b.dr] + b.dc))
    assert agree()
    for s in (a, b):
        free_cache_pages(s.dt, s.dn, s.dr, children, bs)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step(b)
        moved = compact_cache_pages(b.dc, b.dt, b.dn, b.dr, bs)
        free_cache_pages(b.dt, b.dn, b.dr, children, bs, new_lengths=grown - grown)
    for _ in range(3):
        g.replay()
        step(a)
        want = compact_cache_pages(a.dc, a.dt, a.dn, a.dr, bs)
        free_cache_pages(a.dt, a.dn, a.dr, children, bs)
        assert all(torch.equal(x, y) for x, y in zip(moved, want))
        assert agree()
        free_cache_pages(a.dt, a.dn, a.dr, dev([2]), bs, new_lengths=dev([0]))
        free_cache_pages(b.dt, b.dn, b.dr, dev([2]), bs, new_lengths=dev([0]))


def test_native_path_gives_the_same_bits(monkeypatch):
    bs = 16
    s = State(*make_pool(12, 8, 60, bs, seed=8, empty=6), bs)
    old = [x.clone() for x in (s.dt, s.dn, s.dr, *s.dc)]

    def run_all():
        for x, o in zip((s.dt, s.dn, s.dr, *s.dc), old):
            x.copy_(o)
        a = fork_cache_pages(s.dt, s.dn, s.dr, dev([0, 1, 99]), dev([6, 7, 8]), bs)
        b = extend_cache_pages(s.dc, s.dt, s.dn, s.dr, dev([6, 7]), s.dn[[0, 1]] + 9, bs)
        c = copy_cache_pages(s.dc, dev([0, 1]), dev([58, 59]))
        d = free_cache_pages(s.dt, s.dn, s.dr, dev([0, 2]), bs, new_lengths=s.dn[[0, 2]] // 2)
        e = free_cache_pages(s.dt, s.dn, s.dr, dev([3]), bs)
        f = compact_cache_pages(s.dc, s.dt, s.dn, s.dr, bs)
        return [x.clone() for x in (a, b, c, d, e, *f, s.dt, s.dn, s.dr)] + [x.view(torch.uint8).clone() for x in s.dc]

    both(monkeypatch, run_all)


def test_checked_build(checked):
    """Table entries outside the cache are passed over and noted."""
    t, n, refs = make_pool(8, 6, 64, 16, seed=9, empty=3)
    s = State(t, n, refs, 16)
    s.fork([0, 1], [5, 6])
    s.extend([5, 6], [int(n[0]) + 3, int(n[1]) + 20])
    s.compact()
    assert _lib.debug_violations(checked) == 0
    t, n = np.array([[3, 99, 5], [7, -2, 0], [0, 0, 0]], np.int32), np.array([40, 20, 0], np.int32)
    refs = np.zeros(9, np.int32)
    refs[[3, 5, 7]] = 1
    s = State(t, n, refs, 16)
    s.fork([0], [2])
    assert _lib.debug_violations(checked) == _lib.VIOLATION_PAGE
    s.extend([1, 2], [30, 41])
    assert _lib.debug_violations(checked) == _lib.VIOLATION_PAGE
    s.compact()
    assert _lib.debug_violations(checked) == _lib.VIOLATION_PAGE
    s.free([0, 1, 2])
    assert _lib.debug_violations(checked) == _lib.VIOLATION_PAGE
    assert not s.refs.any()


@pytest.mark.parametrize("rows,width,pages", [(0, 3, 5), (3, 0, 5), (3, 2, 0)])
def test_empty_states(rows, width, pages):
    """No rows, no columns, no pages: every entry is left out, but for rows that
    stay empty."""
    z = lambda *s: torch.zeros(s, dtype=torch.int32, device=DEV)
    t, n, r, cache = z(rows, width), z(rows), z(pages), z(pages, 4)
    assert copy_cache_pages([cache], dev([0, 1]), dev([1, 7])).tolist() == [int(pages > 1), 0]
    ok = int(rows > 0)
    assert fork_cache_pages(t, n, r, dev([0]), dev([1]), 16).tolist() == [ok]
    assert extend_cache_pages([cache], t, n, r, dev([0]), dev([5]), 16).tolist() == [int(rows * width * pages > 0)]
    assert extend_cache_pages([cache], t, n, r, dev([1]), dev([0]), 16).tolist() == [ok]
    assert free_cache_pages(t, n, r, dev([0, 9]), 16).tolist() == [ok, 0]
    out = compact_cache_pages([cache], t, n, r, 16)
    assert out[0].shape == t.shape and out[1].shape == r.shape and int(out[3]) == 0
