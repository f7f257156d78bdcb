"""StateCache against a plain cache of Python lists, bit for bit: pages, tables, lengths and counts after each call."""
import ctypes

import numpy as np
import pytest
import torch

from yggdrasil_b200 import _native


def cache_class():
    from yggdrasil_b200 import StateCache
    return StateCache


class Plain:
    """The definition: a list of page contents, tables, and counts; new pages are the lowest free ones in order."""

    def __init__(self, pages, streams, per_stream):
        self.pages = pages.cpu().numpy().copy()
        self.table, self.m = [[] for _ in range(streams)], per_stream
        self.bad = self.full = False

    def refs(self):
        r = [0] * len(self.pages)
        for row in self.table:
            for p in row:
                r[p] += 1
        return r

    def free_pages(self):
        return [p for p, r in enumerate(self.refs()) if r == 0]

    def known(self, *streams):
        if any(s < 0 for s in streams):
            return False
        if any(s >= len(self.table) for s in streams):
            self.bad = True
            return False
        return True

    def fork(self, parents, children, depth=None):
        before, spare, taken = [list(r) for r in self.table], self.free_pages(), set()
        for i, (p, c) in enumerate(zip(parents, children)):
            if not self.known(p, c):
                continue
            row = before[p] if depth is None else before[p][:max(0, depth[i])]
            if not row:
                continue
            if before[c] or c in taken:
                self.bad = True
                continue
            taken.add(c)
            if not spare:
                self.full = True
                continue
            new = spare.pop(0)
            self.pages[new] = self.pages[row[-1]]
            self.table[c] = row[:-1] + [new]

    def grow(self, streams):
        before, spare, taken = [list(r) for r in self.table], self.free_pages(), set()
        for s in streams:
            if not self.known(s):
                continue
            if len(before[s]) >= self.m:
                self.full = True
                continue
            if s in taken:
                self.bad = True
                continue
            taken.add(s)
            if not spare:
                self.full = True
                continue
            new = spare.pop(0)
            self.pages[new] = self.pages[before[s][-1]] if before[s] else 0
            self.table[s] = before[s] + [new]

    def free(self, streams):
        for s in streams:
            if self.known(s):
                self.table[s] = []

    def compact(self):
        r = self.refs()
        n = sum(v > 0 for v in r)
        high = [p for p in range(n, len(r)) if r[p] > 0]
        new = dict(zip(high, [p for p in range(n) if r[p] == 0]))
        for p, q in new.items():
            self.pages[q] = self.pages[p]
        self.table = [[new.get(p, p) for p in row] for row in self.table]
        return n

    def read(self, streams):
        rows = [self.table[s] if self.known(s) else [] for s in streams]
        return np.stack([self.pages[r[-1]] if r else np.zeros_like(self.pages[0]) for r in rows])

    def write(self, streams, batch):
        for s, b in zip(streams, batch):
            if self.known(s) and self.table[s]:
                self.pages[self.table[s][-1]] = b


def pair(pages, streams, per_stream, shape=(4, 8), dtype=torch.int8, seed=0):
    cache = cache_class().empty(pages, streams, per_stream, shape=shape, dtype=dtype, device="cuda")
    g = torch.Generator().manual_seed(seed)
    data = torch.randint(-100, 100, (pages, *shape), generator=g).to(dtype)
    cache.pages.copy_(data)
    return cache, Plain(data, streams, per_stream)


def same(cache, plain):
    want = torch.full((len(plain.table), plain.m), -1, dtype=torch.int32)
    for s, row in enumerate(plain.table):
        want[s, :len(row)] = torch.tensor(row, dtype=torch.int32)
    assert torch.equal(cache.table.cpu(), want)
    assert cache.length.tolist() == [len(r) for r in plain.table]
    assert cache.refs.tolist() == plain.refs()
    assert np.array_equal(cache.pages.cpu().numpy(), plain.pages)
    raised = None
    try:
        cache.status()
    except (ValueError, RuntimeError) as e:
        raised = e
    assert isinstance(raised, ValueError) == plain.bad
    assert isinstance(raised, RuntimeError) == (plain.full and not plain.bad)
    plain.bad = plain.full = False


SHAPES = [((4, 128), torch.int8), ((5, 256), torch.float32), ((3, 96), torch.bfloat16), ((1, 1), torch.int8),
          ((3, 7), torch.int8), ((5, 3), torch.float16), ((1, 5), torch.float32), ((2, 64), torch.float64)]


@pytest.mark.gpu
@pytest.mark.parametrize("shape,dtype", SHAPES)
@pytest.mark.parametrize("streams,per_stream,pages", [(1, 1, 1), (3, 2, 5), (40, 3, 70), (1500, 2, 2500)])
def test_random_calls(streams, per_stream, pages, shape, dtype):
    cache, plain = pair(pages, streams, per_stream, shape, dtype)
    rng = np.random.default_rng(streams)
    some = lambda: rng.integers(-1, streams, rng.integers(0, streams + 2)).tolist()  # noqa: E731 (repeats among them)
    for step in range(14):
        what = ["grow", "fork", "deep", "free", "compact", "write", "read"][step % 7 if step < 7 else rng.integers(0, 7)]
        a = some()
        if what == "grow":
            cache.grow(a), plain.grow(a)
        elif what in ("fork", "deep"):
            b = rng.integers(-1, streams, len(a)).tolist()
            d = rng.integers(0, per_stream + 2, len(a)).tolist() if what == "deep" else None
            cache.fork(a, b, d), plain.fork(a, b, d)
        elif what == "free":
            a = a[:len(a) // 2]
            cache.free(a), plain.free(a)
        elif what == "compact":
            live = plain.compact()
            assert int(cache.compact()) == live
            assert not any(plain.refs()[live:]) and all(plain.refs()[:live])
        elif what == "write":
            a = list(dict.fromkeys(s for s in a if s >= 0))
            batch = torch.randint(-50, 50, (len(a), *shape)).to(dtype)
            cache.write(a, batch.cuda()), plain.write(a, batch.float().numpy() if dtype == torch.bfloat16 else
                                                      batch.numpy())
        else:
            got = cache.read(a).cpu()
            if a:
                assert np.array_equal(_np(got), plain.read(a))
        same_any(cache, plain)


def _np(t):
    return t.float().numpy() if t.dtype == torch.bfloat16 else t.numpy()


def same_any(cache, plain):
    if cache.pages.dtype == torch.bfloat16:
        view = type("View", (), dict(table=cache.table, length=cache.length, refs=cache.refs, pages=cache.pages.float(),
                                     status=cache.status))
        return same(view, plain)
    return same(cache, plain)


@pytest.fixture(autouse=True)
def _bfloat16_as_float(monkeypatch):
    keep = Plain.__init__

    def init(self, pages, streams, per_stream):
        keep(self, pages.float() if pages.dtype == torch.bfloat16 else pages, streams, per_stream)
    monkeypatch.setattr(Plain, "__init__", init)


@pytest.mark.gpu
@pytest.mark.parametrize("streams", [8, 1023, 1025, 5000])
def test_fork_shares_the_snapshots_and_copies_the_last_page(streams):
    cache, plain = pair(streams * 4, streams * 2, 3, seed=2)
    a = list(range(streams))
    for c in (cache, plain):
        c.grow(a)
        c.grow(a[::2])
        c.grow(a[::4])
        c.fork([x % 7 for x in a], [streams + x for x in a])
    same(cache, plain)
    for c in (cache, plain):
        c.free(a[1::2] + [0, 0, 1])
    same(cache, plain)
    assert int(cache.compact()) == plain.compact()
    same(cache, plain)


@pytest.mark.gpu
def test_a_pool_without_room_serves_the_first_and_reports():
    cache, plain = pair(6, 10, 1)
    for c in (cache, plain):
        c.grow([0, 1, 2, 3])
        c.fork([0, 1, 2, 3, 0], [4, 5, 6, 7, 8])
    same(cache, plain)
    assert cache.length.tolist() == [1] * 6 + [0] * 4
    for c in (cache, plain):
        c.grow([0, 7])
    same(cache, plain)


@pytest.mark.gpu
def test_what_cannot_be_done_is_left_undone():
    cache, plain = pair(20, 6, 2)
    for c in (cache, plain):
        c.grow([0, 1])
    same(cache, plain)
    dev = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    for parents, children in (([0, 1], [1, 2]), ([0, 1], [3, 3]), ([0, 4], [4, 5]), ([7, 0], [4, 6]), ([-1, 0], [5, -3])):
        cache.fork(dev(parents), dev(children))
        plain.fork(parents, children)
        same(cache, plain)
    cache.free(dev([9, -1, 2, 2])), plain.free([9, -1, 2, 2])
    same(cache, plain)
    cache.grow(dev([0, 0, 6])), plain.grow([0, 0, 6])
    same(cache, plain)
    assert np.array_equal(cache.read(dev([6, 0, -1])).cpu().numpy(), plain.read([6, 0, -1]))
    same(cache, plain)


@pytest.mark.gpu
def test_copy_of_pages():
    cache, plain = pair(50, 1, 1, shape=(3, 5))
    cache.copy([0, 1, 2, -1, 5], [10, 11, 12, 13, -1])
    for a, b in ((0, 10), (1, 11), (2, 12)):
        plain.pages[b] = plain.pages[a]
    same(cache, plain)
    cache.copy(torch.tensor([3, 60], device="cuda"), torch.tensor([14, 15], device="cuda"))
    plain.pages[14] = plain.pages[3]
    plain.bad = True
    same(cache, plain)


@pytest.mark.gpu
def test_compact_of_none_all_and_the_far_end():
    cache, plain = pair(3000, 3000, 1)
    assert int(cache.compact()) == plain.compact() == 0
    same(cache, plain)
    for c in (cache, plain):
        c.grow(list(range(3000)))
    assert int(cache.compact()) == plain.compact() == 3000
    same(cache, plain)
    for c in (cache, plain):
        c.free(list(range(2999)))
    assert int(cache.compact()) == plain.compact() == 1
    same(cache, plain)


@pytest.mark.gpu
def test_pages_beyond_32_bits_of_bytes():
    """A pool of 5 GB: the copies go beyond byte 2^32."""
    shape, pages = (1024, 1280), 4096
    cache = cache_class().empty(pages, 4100, 1, shape=shape, dtype=torch.int8, device="cuda")
    cache.grow(np.arange(pages - 1))
    cache.write([pages - 2], torch.full((1, *shape), 7, dtype=torch.int8, device="cuda"))
    cache.fork([pages - 2], [4099])
    assert cache.table[4099].item() == pages - 1 and bool((cache.pages[pages - 1] == 7).all())
    cache.free(np.arange(pages - 1))
    assert int(cache.compact()) == 1 and bool((cache.pages[0] == 7).all()) and cache.table[4099].item() == 0
    cache.status()


@pytest.mark.gpu
def test_around_tensors_on_another_stream_and_in_a_graph():
    cls = cache_class()
    made = cls.empty(400, 300, 2, shape=(4, 128), dtype=torch.int8, device="cuda")
    made.pages.random_(-100, 100)
    made.grow(np.arange(100))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        cache = cls(made.pages, made.table, made.length, made.refs)
        cache.fork(np.arange(100), np.arange(100, 200))
        cache.status()
    assert torch.equal(cache.read(np.arange(100)), cache.read(np.arange(100, 200)))
    # a graph of a step's housekeeping, replayed: fork, free, compact
    parents = torch.arange(50, dtype=torch.int32, device="cuda")
    children = parents + 200
    cache.fork(parents, children)
    cache.free(children)
    cache.compact()
    keep = [t.clone() for t in (cache.table, cache.length, cache.refs)]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.fork(parents, children)
        cache.free(children)
        live = cache.compact()
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    assert int(live) == 200
    for a, b in zip(keep, (cache.table, cache.length, cache.refs)):
        assert torch.equal(a, b)
    cache.status()


@pytest.mark.gpu
def test_refusals():
    cls = cache_class()
    ints = lambda *s: torch.zeros(s, dtype=torch.int32, device="cuda")  # noqa: E731
    pages = torch.zeros(8, 4, 16, dtype=torch.int8, device="cuda")
    cls(pages, ints(3, 2), ints(3), ints(8))
    for bad in ((pages.cpu(), ints(3, 2), ints(3), ints(8)), (pages[:, :, 1:], ints(3, 2), ints(3), ints(8)),
                (pages, ints(3), ints(3), ints(8)), (pages, ints(3, 2).long(), ints(3), ints(8)),
                (pages, ints(3, 2), ints(4), ints(8)), (pages, ints(3, 2), ints(3), ints(7)),
                (pages, ints(2, 3).T, ints(3), ints(8)), (pages, ints(3, 2), ints(3), ints(8).cpu())):
        with pytest.raises(ValueError):
            cls(*bad)
    with pytest.raises(ValueError):
        cls.empty(0, 3, shape=(2,), device="cuda")
    with pytest.raises(ValueError):
        cls.empty(4, 3, shape=(2,), device="cpu")
    cache = cls.empty(8, 4, 1, shape=(2, 3), dtype=torch.int8, device="cuda")
    for call in (lambda: cache.fork([0], [1, 2]), lambda: cache.fork([0], [4]), lambda: cache.grow([4]),
                 lambda: cache.grow([[0]]), lambda: cache.free([0.5]), lambda: cache.free(torch.zeros(2, device="cuda")),
                 lambda: cache.write([0], torch.zeros(1, 2, 4, dtype=torch.int8, device="cuda")),
                 lambda: cache.write([0], torch.zeros(1, 2, 3, device="cuda")), lambda: cache.copy([0], [8]),
                 lambda: cache.copy([0, 1], [2])):
        with pytest.raises(ValueError):
            call()


def test_c_entry_refuses_bad_arguments():
    """Checked before any CUDA call."""
    lib, E, p = _native.ops(), _native, 4096
    good = lambda: _native.YggCache(p, 8, 16, p, 4, 2, p, p, p, p)  # noqa: E731
    size = lib.ygg_cache_workspace(ctypes.byref(good()), 5)
    assert size > 0 and lib.ygg_cache_workspace(None, 5) == 0 and lib.ygg_cache_workspace(ctypes.byref(good()), -1) == 0
    assert lib.ygg_cache_fork(0, None, 1, p, p, None, p, size, None) == E.YGG_E_ARG
    for field, value in (("pages", None), ("page_count", 0), ("page_count", 1 << 31), ("page_bytes", 0), ("table", None),
                         ("streams", 0), ("per_stream", 0), ("length", None), ("refs", None), ("status", None),
                         ("sync", None)):
        c = good()
        setattr(c, field, value)
        assert lib.ygg_cache_free(0, ctypes.byref(c), 1, p, None) == E.YGG_E_ARG
        assert lib.ygg_cache_compact(0, ctypes.byref(c), p, p, 1 << 20, None) == E.YGG_E_ARG
    c = ctypes.byref(good())
    assert lib.ygg_cache_fork(0, c, -1, p, p, None, p, size, None) == E.YGG_E_ARG
    assert lib.ygg_cache_fork(0, c, 1, None, p, None, p, size, None) == E.YGG_E_ARG
    assert lib.ygg_cache_fork(0, c, 1, p, p, None, None, size, None) == E.YGG_E_ARG
    assert lib.ygg_cache_fork(0, c, 5, p, p, None, p, 8, None) == E.YGG_E_ARG
    assert lib.ygg_cache_fork(0, c, 0, None, None, None, None, 0, None) == E.YGG_OK
    assert lib.ygg_cache_free(0, c, 1, None, None) == E.YGG_E_ARG
    assert lib.ygg_cache_compact(0, c, None, p, size, None) == E.YGG_E_ARG
    assert lib.ygg_cache_read(0, c, 1, None, p, None) == E.YGG_E_ARG
    assert lib.ygg_cache_write(0, c, 1, p, None, None) == E.YGG_E_ARG
    assert lib.ygg_cache_copy(0, c, 1, p, None, None) == E.YGG_E_ARG


@pytest.mark.gpu
@pytest.mark.parametrize("pages", [20, 6000])
def test_tables_that_do_not_fit_their_counts_are_reported(pages):
    """A cache around tensors of the caller's: entries of pages beyond the pool, and of pages that nothing counts, at or
    beyond the number of live pages. compact moves what is counted, leaves those entries and reports them."""
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    data = torch.arange(pages, dtype=torch.int32, device="cuda")[:, None].repeat(1, 3) + 1
    refs = torch.zeros(pages, dtype=torch.int32, device="cuda")
    refs[pages - 2] = 1
    table = ints([[pages - 2, -1], [pages - 1, -1], [pages, -1], [2 ** 31 - 1, -1], [5, -1]])
    cache = cache_class()(data, table, ints([1] * 5), refs)
    assert int(cache.compact()) == 1
    assert cache.table[:, 0].tolist() == [0, pages - 1, pages, 2 ** 31 - 1, 5]
    assert refs[0].item() == 1 and int(refs.sum()) == 1 and data[0].tolist() == [pages - 1] * 3
    with pytest.raises(ValueError):
        cache.status()
    assert cache.read([0, 2, 3]).tolist() == [[pages - 1] * 3, [0] * 3, [0] * 3]
    with pytest.raises(ValueError):
        cache.status()
    keep = data.clone()
    cache.write([2, 3], torch.ones(2, 3, dtype=torch.int32, device="cuda"))
    assert torch.equal(data, keep)
    with pytest.raises(ValueError):
        cache.status()
    cache.grow([0, 2])
    assert cache.table[0].tolist() == [0, 1] and cache.table[2].tolist() == [pages, 2]
    assert data[1].tolist() == [pages - 1] * 3 and data[2].tolist() == [0] * 3
    with pytest.raises(ValueError):
        cache.status()


def words_by_two(monkeypatch):
    """Words of caches two at a time, and whatever a first call of each kind waits for behind us."""
    from yggdrasil_b200 import cache as module
    monkeypatch.setattr(module, "_SLOTS", 2)
    monkeypatch.setattr(module, "_pools", {})
    made = [cache_class().empty(4, 4, shape=(4,), dtype=torch.int8, device="cuda") for _ in range(30)]
    made[0].grow([0, 1])
    torch.cuda._sleep(100)
    torch.cuda.synchronize()
    del made
    module._pools.clear()


@pytest.mark.gpu
def test_words_of_a_cache_that_is_gone_serve_no_other_before_its_calls_are_done(monkeypatch):
    """A call that will report waits on a stream of its own, its cache goes, and others are made: none gets the report."""
    words_by_two(monkeypatch)
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    held = torch.zeros(1, 4, dtype=torch.int8, device="cuda"), ints([[-1], [-1]]), ints([0, 0]), ints([0])
    ids = ints([0, 1])
    first, cache = cache_class()(*held), cache_class()(*held)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(1_000_000_000)
        cache.grow(ids)   # one page for two streams
    assert not side.query()
    del first, cache
    made = [cache_class().empty(4, 4, shape=(4,), dtype=torch.int8, device="cuda") for _ in range(8)]
    torch.cuda.synchronize()
    assert held[2].sum().item() == 1
    for c in made:
        c.status()
    assert len({c._status[c._at].data_ptr() for c in made}) == len({c._sync[c._at].data_ptr() for c in made}) == 8


@pytest.mark.gpu
def test_words_are_used_again_and_a_cache_can_be_made_in_a_capture(monkeypatch):
    from yggdrasil_b200 import cache as module
    words_by_two(monkeypatch)
    make = lambda: cache_class().empty(4, 4, shape=(4,), dtype=torch.int8, device="cuda")  # noqa: E731
    seen = set()
    for _ in range(100):
        c = make()
        seen.add(c._status[c._at].data_ptr())
    assert len(seen) <= 8   # memory does not grow with the caches that were
    module._pools.clear()
    kept = [make(), make()]   # the second: half are out, the next two are got ready
    kept[0].grow([0])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        inside = cache_class()(kept[0].pages, kept[0].table, kept[0].length, kept[0].refs)
        inside.fork(kept[0].refs[:1] * 0, kept[0].refs[:1] * 0 + 1)
    graph.replay()
    inside.status()
    assert kept[0].length.tolist() == [1, 1, 0, 0]


@pytest.mark.gpu
def test_a_cache_whose_barrier_gave_up_stays_unusable():
    """What a wait that ran out leaves behind (the barrier's top bit and the status word): later calls give up at their first
    barrier, nothing is handed out or moved, and status() says so each time, cleared or not."""
    cache = cache_class().empty(6000, 6000, shape=(4,), dtype=torch.int8, device="cuda")
    cache.pages.fill_(3)
    cache.grow(np.arange(0, 6000, 2))
    cache.status()
    cache._sync[cache._at] |= -2 ** 63
    cache.grow(np.arange(1, 6000, 2))
    for _ in range(2):
        with pytest.raises(_native.YggError) as e:
            cache.status()
        assert e.value.code == _native.YGG_E_TIMEOUT
    assert cache.length[1::2].sum().item() == 0 and cache.refs.sum().item() == 3000
    cache._status[cache._at].zero_()
    cache.free(np.arange(1000))
    cache.compact()
    assert cache.refs.sum().item() == 2500 and int(cache.refs[2500:].sum()) > 0
    for _ in range(2):
        with pytest.raises(_native.YggError):
            cache.status(clear=False)


FAR = [-2 ** 32 + 5, 2, -2 ** 31 - 1, -2 ** 63, -7]   # low 32 bits: 5, 2, 2^31 - 1, 0, -7


@pytest.mark.parametrize("kind", [list, np.array, torch.tensor])
def test_host_indices_far_below_zero_are_padding(kind):
    from types import SimpleNamespace
    ids = cache_class()._ids(SimpleNamespace(device=torch.device("cpu")), kind(FAR), "streams", 8)
    assert ids.dtype == torch.int32 and ids.tolist() == [-1, 2, -1, -1, -1]
    for unsigned in (np.uint8, np.uint64):
        assert cache_class()._ids(SimpleNamespace(device=torch.device("cpu")), np.array([3, 7], unsigned), "x", 8).tolist() == [3, 7]
    with pytest.raises(ValueError):
        cache_class()._ids(SimpleNamespace(device=torch.device("cpu")), np.array([2 ** 64 - 1], np.uint64), "streams", 8)


@pytest.mark.gpu
def test_indices_far_below_zero_on_the_host_and_on_the_device():
    for ids in (FAR, torch.tensor(FAR, device="cuda")):
        cache, plain = pair(8, 8, 1)
        cache.grow(list(range(8))), plain.grow(list(range(8)))
        cache.free(ids), plain.free(FAR)
        same(cache, plain)
        assert cache.length.tolist() == [1, 1, 0, 1, 1, 1, 1, 1]


@pytest.mark.gpu
def test_derivatives_are_refused():
    import torch.autograd.forward_ad as fw
    ints = lambda *s: torch.zeros(s, dtype=torch.int32, device="cuda")  # noqa: E731
    make = lambda pages: cache_class()(pages, ints(2, 1) - 1, ints(2), ints(4))  # noqa: E731
    pages = torch.zeros(4, 3, device="cuda")
    cache, batch = make(pages), torch.ones(1, 3, device="cuda")
    cache.grow([0])
    leaf = batch.clone().requires_grad_()
    for b in (leaf, leaf.T.contiguous().T, leaf * 2):
        with pytest.raises(NotImplementedError):
            cache.write([0], b)
    with pytest.raises(NotImplementedError):
        make(pages.clone().requires_grad_())
    with fw.dual_level():
        with pytest.raises(NotImplementedError):
            cache.write([0], fw.make_dual(batch, batch))
    assert not bool(pages.any())
    with torch.no_grad():
        cache.write([0], leaf)
    assert torch.equal(cache.read([0]), batch)


@pytest.mark.gpu
def test_a_full_pool_says_so():
    cache = cache_class().empty(1, 2, shape=(4,), dtype=torch.int8, device="cuda")
    cache.grow([0, 1])
    with pytest.raises(_native.YggError) as e:
        cache.status()
    assert e.value.code == _native.YGG_E_CAPACITY and str(e.value) == "StateCache: no free page, or a full table row (-10)"


@pytest.mark.gpu
def test_fork_and_free_report_pages_beyond_the_pool():
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    data = torch.ones(8, 3, dtype=torch.int32, device="cuda")
    table, refs = ints([[9, 0], [-1, -1], [1, -1], [-1, -1]]), ints([1, 1, 0, 0, 0, 0, 0, 0])
    cache = cache_class()(data, table, ints([2, 0, 1, 0]), refs)
    cache.fork([2], [3])
    cache.status()
    cache.fork([0], [1])   # shares a page 9 of 8
    assert table[1].tolist() == [9, 3] and refs.tolist() == [1, 1, 1, 1, 0, 0, 0, 0]
    with pytest.raises(ValueError):
        cache.status()
    cache.free([3])
    cache.status()
    cache.free([0])
    assert table[0].tolist() == [-1, -1] and refs.tolist() == [0, 1, 0, 1, 0, 0, 0, 0]
    with pytest.raises(ValueError):
        cache.status()
