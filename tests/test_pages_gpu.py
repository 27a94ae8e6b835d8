"""The book of a paged cache's pages against plain Python, entry by entry, and the pages' bytes in the pools of all layers."""
import numpy as np
import pytest
import torch

import paged_oracle as po
import pages_oracle
from miinfer_b200 import kv, paged

pytestmark = pytest.mark.gpu


@pytest.fixture
def status():
    word = torch.zeros(1, dtype=torch.int32, device="cuda")
    kv.set_status_word(word)
    yield word
    kv.set_status_word(None)


class Both:
    """A book on the host and on the device, and pools that hold a number of its own in every page."""

    def __init__(self, pages, page, slots, max_pages, *, layers=2, mode=3, heads=2, d=128, qblock=32, seed=0):
        self.rng, self.host = np.random.default_rng(seed), pages_oracle.Book(pages, page, slots, max_pages)
        g = torch.Generator("cuda").manual_seed(seed)
        shape = (pages, heads, page)
        side = lambda q8: ([torch.randint(-128, 128, (*shape, d), generator=g, dtype=torch.int8, device="cuda"), torch.rand(*shape, d // qblock, generator=g, dtype=torch.float16, device="cuda")]
                           if q8 else [torch.rand(*shape, d, generator=g, dtype=torch.float16, device="cuda"), None])
        self.pools = [side(mode in (1, 3)) + side(mode in (2, 3)) for _ in range(layers)]
        self.views = [paged.PagedView.of(*planes, kv.KvCacheQuantMode(mode)) for planes in self.pools]
        self.want = [[None if t is None else t.clone() for t in planes] for planes in self.pools]
        self.upload()

    def upload(self):
        self.refs, self.tables, self.lengths = (torch.from_numpy(a.copy()).cuda() for a in (self.host.refs, self.host.tables, self.host.lengths))
        self.book = paged.PageBook(self.refs, self.tables, self.lengths, page_size=self.host.page)
        self.workspace = paged.pages_workspace(self.book)
        self.moved = torch.full((len(self.host.refs),), -9, dtype=torch.int32, device="cuda")

    def copy(self, source, target):
        for planes in self.want:
            for t in planes:
                if t is not None:
                    t[target] = t[source]

    def fill(self, lengths):
        """Sequences of these lengths, their pages drawn from all over the pool."""
        order = self.rng.permutation(len(self.host.refs))
        at = 0
        for s, n in enumerate(lengths):
            k = self.host.held(n)
            self.host.tables[s, :k] = order[at:at + k]
            self.host.refs[order[at:at + k]] = 1
            self.host.lengths[s] = n
            at += k
        self.upload()

    def grow(self, slots, add):
        paged.launch_pages_grow(self.book, po.ints(slots), po.ints(add), workspace=self.workspace)
        self.host.grow(slots, add)

    def fork(self, parents, children, at=None):
        paged.launch_pages_fork(self.book, self.views, po.ints(parents), po.ints(children), at=None if at is None else po.ints(at), workspace=self.workspace)
        self.host.fork(parents, children, at, self.copy)

    def free(self, slots):
        paged.launch_pages_free(self.book, po.ints(slots))
        self.host.free(slots)

    def compact(self):
        paged.launch_pages_compact(self.book, self.views, self.moved, workspace=self.workspace)
        assert np.array_equal(self.host.compact(self.copy), self.moved.cpu().numpy())

    def check(self, word=None):
        h = self.host
        assert np.array_equal(self.refs.cpu().numpy(), h.refs) and np.array_equal(self.lengths.cpu().numpy(), h.lengths)
        got = self.tables.cpu().numpy()
        for s, n in enumerate(h.lengths):
            assert np.array_equal(got[s, :h.held(n)], h.tables[s, :h.held(n)]), s
        for planes, want in zip(self.pools, self.want):
            for t, w in zip(planes, want):
                assert t is None or torch.equal(t.view(torch.uint8), w.view(torch.uint8))
        if word is not None:
            assert int(word) == h.status
            word.zero_()
            h.status = 0


@pytest.mark.parametrize("mode,qblock,d,heads,page", [(3, 32, 128, 2, 16), (3, 256, 256, 1, 16), (0, 128, 128, 3, 32), (1, 32, 256, 4, 64), (2, 128, 128, 5, 256)])
def test_a_server_s_life(cuda, status, mode, qblock, d, heads, page):
    """Rounds of growth, forks, ends and compactions, sizes drawn; the book and every byte of the pools after each."""
    b = Both(61, page, 12, 9, layers=3, mode=mode, heads=heads, d=d, qblock=qblock, seed=page + mode)
    rng = b.rng
    for step in range(12):
        slots = rng.permutation(12)[:rng.integers(1, 9)].tolist()
        b.grow(slots, rng.integers(0, 3 * page, len(slots)).tolist())
        b.check(status)
        empty = np.flatnonzero(b.host.lengths == 0).tolist()
        if empty:
            parents = rng.integers(0, 12, len(empty)).tolist()
            b.fork(parents, empty, rng.integers(0, 9 * page, len(empty)).tolist() if step % 2 else None)
            b.check(status)
        b.free(rng.permutation(12)[:rng.integers(1, 6)].tolist())
        b.check(status)
        b.compact()
        b.check(status)
        live = int((b.host.refs > 0).sum())
        assert (b.host.refs[:live] > 0).all()


@pytest.mark.parametrize("pages", [1, 3, 4, 37, 4095, 4096, 4097, 20001])
def test_pools_of_any_size(cuda, status, pages):
    """Scans over counts that end inside a thread's four, inside a block's or behind several."""
    b = Both(pages, 16, 300, max(1, pages // 7 + 1), layers=1, heads=1, seed=pages)
    lengths = b.rng.integers(0, 16 * max(1, pages // 90) + 1, 300).tolist() if pages > 4 else [1]
    while sum(b.host.held(n) for n in lengths) > pages:
        lengths.pop()
    b.fill(lengths)
    b.compact()
    b.check(status)
    b.free(b.rng.permutation(300)[:150].tolist())
    b.compact()
    b.check(status)
    b.compact()                                      # nothing is left to move
    b.check(status)
    slots = b.rng.permutation(300).tolist()
    b.grow(slots, b.rng.integers(0, 40, 300).tolist())
    b.check(status)


def test_all_pages_held_and_none(cuda, status):
    b = Both(40, 16, 4, 40, seed=4)
    b.compact()
    b.check(status)
    b.grow([2], [640])
    b.check(status)
    b.compact()
    b.check(status)
    b.grow([0], [1])                                 # no page is left
    assert b.host.status == pages_oracle.NO_PAGE
    b.check(status)
    b.free([2, 2, 0])
    b.check(status)
    assert int(b.refs.sum()) == 0


def test_entries_in_order_until_the_pages_run_out(cuda, status):
    """An entry gets all its pages or none; none behind it gets any, but for those that need none."""
    b = Both(23, 16, 9, 20, seed=5)
    b.fill([5, 0, 0, 16, 0, 0, 0, 0, 0])
    b.grow([0, 1, 2, 3, 4], [3, 200, 130, 1, 16])
    assert b.host.lengths.tolist()[:5] == [8, 200, 0, 16, 0]
    b.check(status)
    b.grow([0, 4, 2], [8, 100, 17])
    b.check(status)
    b.fork([1, 1, 1, 0, 3, 1], [5, 6, 7, 8, 2, 2])
    b.check(status)


def test_entries_that_are_refused(cuda, status):
    b = Both(50, 16, 8, 4, seed=6)
    b.fill([20, 33, 64, 0, 0, 0, 1, 0])
    b.grow([0, -1, 8, 0, 2, 1, 3, 4, 1000000], [5, 7, 1, 5, 1, -3, 65, 64, 2])
    assert b.host.lengths.tolist() == [25, 33, 64, 0, 64, 0, 1, 0] and b.host.status == pages_oracle.BAD_SLOT | pages_oracle.BAD_BOUND
    b.check(status)
    b.fork([1, 1, 5, 9, -1, 0, 0], [3, 3, 5, 7, 7, 1, -1])          # named twice; empty and its own parent; parents there are not (named twice as well); a child that is not empty; left out
    assert b.host.status == pages_oracle.BAD_SLOT
    b.check(status)
    b.fork([7, 3], [5, 7])                                          # 7 is empty before the call and a child in it: 5 gets what it held before
    b.check(status)
    assert b.host.lengths.tolist()[5] == 0
    b.free([-5, 3, 99, 3, 3])
    b.check(status)


def test_lengths_to_fork_at(cuda, status):
    b = Both(60, 32, 10, 5, mode=0, seed=7)
    b.fill([100, 64])
    b.fork([0, 0, 0, 0, 0, 1, 1, 1], [2, 3, 4, 5, 6, 7, 8, 9], [0, 1, 31, 32, 1000, 64, 33, -7])
    assert b.host.lengths.tolist() == [100, 64, 0, 1, 31, 32, 100, 64, 33, 0]
    b.check(status)
    b.free([0, 1, 6])
    b.compact()
    b.check(status)
    b.free(list(range(10)))
    b.check(status)
    assert int(b.refs.abs().sum()) == 0


def test_counts_that_others_add_to(cuda, status):
    """A prefix index holds pages of its own; they stay when the sequence ends, move with the others, and the map says where to."""
    b = Both(30, 16, 3, 10, seed=8)
    b.fill([70, 50, 90])
    own = b.host.tables[1, :2].copy()
    b.host.refs[own] += 1
    b.refs += torch.from_numpy(np.bincount(own, minlength=30).astype(np.int32)).cuda()
    bytes_of = [b.pools[0][0][int(p)].clone() for p in own]
    b.free([1, 0])
    b.check(status)
    assert (b.host.refs[own] == 1).all()
    b.compact()
    b.check(status)
    now = b.moved.cpu().numpy()[own]
    assert (now >= 0).all() and all(torch.equal(b.pools[0][0][int(p)], x) for p, x in zip(now, bytes_of))


def test_pages_outside_the_pool_are_not_followed(cuda, status):
    b = Both(30, 16, 5, 6, seed=9)
    b.fill([40, 33, 20, 0, 0])
    b.tables[0, 1], b.tables[1, 2] = 30, -4
    before = b.refs.clone()
    paged.launch_pages_fork(b.book, b.views, po.ints([1]), po.ints([3]), workspace=b.workspace)      # its last page is to be copied
    assert int(status) == pages_oracle.BAD_PAGE
    status.zero_()
    before[b.host.tables[1, :2]] += 1
    before[int(b.tables[3, 2])] += 1
    assert torch.equal(b.refs, before)
    paged.launch_pages_free(b.book, po.ints([0, 3]))
    assert int(status) == pages_oracle.BAD_PAGE
    assert int(b.refs.min()) == 0 and b.lengths.tolist() == [0, 33, 20, 0, 0]
    status.zero_()
    paged.launch_pages_compact(b.book, b.views, b.moved, workspace=b.workspace)
    assert int(status) == pages_oracle.BAD_PAGE and int(b.tables[1, 2]) == -4
    held = b.tables[1, :2].tolist() + b.tables[2, :2].tolist()      # and the two pages whose entries were written over are held still
    assert len(set(held)) == 4 and max(held) < 6 and (b.refs > 0).tolist() == [True] * 6 + [False] * 24
    status.zero_()
    # a page that is given back more often than it is held
    b.tables[4, 0] = 20
    b.lengths[4] = 5
    paged.launch_pages_free(b.book, po.ints([4]))
    assert int(status) == pages_oracle.BAD_PAGE and int(b.refs[20]) == 0


@pytest.mark.parametrize("layers,mode,page,heads,d", [(1, 3, 16, 1, 128), (3, 0, 64, 4, 256), (17, 3, 32, 3, 128), (128, 2, 16, 1, 256)])
def test_copies_between_pools(cuda, status, layers, mode, page, heads, d):
    a, b = (Both(n, page, 1, 1, layers=layers, mode=mode, heads=heads, d=d, qblock=d if layers == 3 else 32, seed=n) for n in (41, 29))
    sources, targets = a.rng.permutation(41)[:20], b.rng.permutation(29)[:20]
    sources[3], targets[5], sources[7] = 41, -1, -2
    paged.launch_pages_copy(a.views, b.views, po.ints(sources), po.ints(targets))
    for s, t in zip(sources, targets):
        if 0 <= s < 41 and t >= 0:
            for x, y in zip(a.want, b.want):
                for u, v in zip(x, y):
                    if u is not None:
                        v[int(t)] = u[int(s)]
    a.check()
    b.check()
    assert int(status) == pages_oracle.BAD_PAGE
    status.zero_()
    paged.launch_pages_copy(b.views, b.views, po.ints([28, 0]), po.ints([1, 29]))       # within a pool; a target outside it
    b.copy(28, 1)
    b.check()
    assert int(status) == pages_oracle.BAD_PAGE


def test_nothing_to_do(cuda, status):
    b = Both(8, 16, 2, 3, seed=1)
    none = po.ints([])
    b.grow([], [])
    b.free([])
    b.fork([], [])
    paged.launch_pages_copy(b.views, b.views, none, none)
    b.check(status)


def test_most_slots(cuda, status):
    """8192 slots, all of them entries: the search's arrays at their largest."""
    b = Both(9000, 16, 8192, 2, layers=1, heads=1, seed=3)
    slots = b.rng.permutation(8192).tolist()
    b.grow(slots, b.rng.integers(0, 20, 8192).tolist())
    b.check(status)
    b.free(slots[:5000])
    b.check(status)
    b.compact()
    b.check(status)


def test_a_captured_step_replays_with_what_the_arrays_hold(cuda, status):
    """Ends, forks, growth and a compaction in one graph, replayed over other entries; a second graph over the same workspace."""
    b = Both(64, 16, 8, 7, seed=11)
    b.fill([50, 20, 33, 0, 0, 0, 0, 0])
    ending, parents, children, slots, add = (po.ints(x) for x in ([1, -1], [0, 2], [1, 3], [0, 1, 2], [1, 1, 20]))

    def step():
        paged.launch_pages_free(b.book, ending)
        paged.launch_pages_fork(b.book, b.views, parents, children, workspace=b.workspace)
        paged.launch_pages_grow(b.book, slots, add, workspace=b.workspace)
        paged.launch_pages_compact(b.book, b.views, b.moved, workspace=b.workspace)

    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step()
        graphs.append(graph)
    b.check()                                        # a capture runs nothing
    for i, arrays in enumerate([([1, -1], [0, 2], [1, 3], [0, 1, 2], [1, 1, 20]), ([3, 0], [2, 1], [4, 0], [4, 2, 9], [40, 2, 1]), ([4, 2], [1, 1], [5, 6], [5, 6, -1], [3, 0, 0])]):
        for t, x in zip((ending, parents, children, slots, add), arrays):
            t.copy_(po.ints(x))
        graphs[i % 2].replay()
        h = b.host
        h.free(arrays[0])
        h.fork(arrays[1], arrays[2], copy=b.copy)
        h.grow(arrays[3], arrays[4])
        moved = h.compact(b.copy)
        assert np.array_equal(moved, b.moved.cpu().numpy())
        b.check(status)


def test_a_stream_of_its_own(cuda, status):
    b = Both(64, 16, 8, 7, seed=12)
    b.fill([50, 20, 33])
    stream = torch.cuda.Stream()
    slots, add = po.ints([0, 3]), po.ints([30, 9])
    parents, children = po.ints([0]), po.ints([4])
    stream.wait_stream(torch.cuda.current_stream())
    paged.launch_pages_grow(b.book, slots, add, workspace=b.workspace, stream=stream)
    paged.launch_pages_fork(b.book, b.views, parents, children, workspace=b.workspace, stream=stream)
    paged.launch_pages_free(b.book, slots, stream=stream)
    paged.launch_pages_compact(b.book, b.views, b.moved, workspace=b.workspace, stream=stream)
    stream.synchronize()
    b.host.grow([0, 3], [30, 9])
    b.host.fork([0], [4], copy=b.copy)
    b.host.free([0, 3])
    b.host.compact(b.copy)
    b.check(status)


def test_tensors_that_are_refused(cuda):
    b = Both(16, 16, 4, 4, seed=2)
    long, short, host = torch.zeros(3, dtype=torch.int64, device="cuda"), po.ints([1]), torch.zeros(3, dtype=torch.int32)
    three = po.ints([0, 1, 2])
    for args in ((long, three), (three, long), (three, short), (host, three), (three, torch.zeros(6, dtype=torch.int32, device="cuda")[::2])):
        with pytest.raises(ValueError):
            paged.launch_pages_grow(b.book, *args, workspace=b.workspace)
    with pytest.raises(TypeError):
        paged.launch_pages_grow(b.views[0], three, three, workspace=b.workspace)
    with pytest.raises(TypeError):
        paged.launch_pages_compact(b.book, b.views[0], b.moved, workspace=b.workspace)
    with pytest.raises(TypeError):
        paged.launch_pages_compact(b.book, [b.book], b.moved, workspace=b.workspace)
    with pytest.raises(ValueError):
        paged.launch_pages_compact(b.book, b.views, b.moved[:-1], workspace=b.workspace)
    with pytest.raises(ValueError):
        paged.launch_pages_copy(b.views, b.views[:1], three, three)
    with pytest.raises(paged._lib.B200KvError):
        paged.launch_pages_compact(b.book, b.views, b.moved, workspace=b.workspace[:100])
    with pytest.raises(paged._lib.B200KvError):
        paged.launch_pages_compact(b.book, [], b.moved, workspace=b.workspace)
    with pytest.raises(ValueError):
        paged.PageBook(b.refs, b.tables, b.lengths[:2], page_size=16)
    with pytest.raises(ValueError):
        paged.PageBook(b.refs.long(), b.tables, b.lengths, page_size=16)
    b.check()


def test_store_and_attend_over_the_book_s_tables(cuda, status):
    """As they are used together: prompts grow and are stored, forks go on with tokens of their own, the pages are moved together, and attention sees the same before and after."""
    rng = np.random.default_rng(13)
    hq, heads, d, page = 8, 2, 128, 16
    caches = [paged.PagedKvCache(40, page, kv.KvCacheQuantMode.kQ8Q8, kv_heads=heads, head_dim=d, qblock=32) for _ in range(2)]
    views = [c.view() for c in caches]
    book = paged.PageBook.empty(40, page, 6, 8)
    ws = paged.pages_workspace(book)
    rows = lambda n: torch.from_numpy(rng.standard_normal((n, heads * d), dtype=np.float32)).cuda().half()

    def batch_of(tokens):
        starts = np.concatenate([[0], np.cumsum(tokens)])
        return paged.PagedBatch(book.tables_tensor, po.ints(starts), book.lengths_tensor, total_tokens=int(starts[-1]), max_tokens=max(tokens), max_length=8 * page)

    def store(tokens):
        paged.launch_pages_grow(book, po.ints(range(6)), po.ints(tokens), workspace=ws)
        kvs = [(rows(sum(tokens)), rows(sum(tokens))) for _ in views]
        for view, (k, v) in zip(views, kvs):
            paged.launch_paged_store(view, batch_of(tokens), k, v, None)
        return kvs

    first = store([50, 30, 0, 0, 0, 0])
    paged.launch_pages_fork(book, views, po.ints([0, 0, 1]), po.ints([2, 3, 4]), workspace=ws)
    second = store([1, 1, 1, 1, 1, 0])
    assert book.lengths_tensor.tolist() == [51, 31, 51, 51, 31, 0]
    refs = book.refs_tensor.cpu().numpy()
    assert refs[book.tables_tensor[0, :3].cpu().numpy()].tolist() == [3, 3, 3] and refs.sum() == 4 + 2 + 4 + 4 + 2
    q = torch.from_numpy(rng.standard_normal((5, hq, d), dtype=np.float32)).cuda().half()

    def attend():
        got = []
        for view in views:
            batch = batch_of([1, 1, 1, 1, 1, 0])
            out = torch.zeros(5, hq, d, dtype=torch.float16, device="cuda")
            paged.launch_paged_attention(view, batch, q, out, query_heads=hq, scale=0.09, workspace=paged.paged_workspace(view, batch, hq))
            got.append(out)
        return got

    before = attend()
    # what a fork holds is its parent's prompt and its own token
    for layer, cache in enumerate(caches):
        for slot, parent, row in ((0, 0, 0), (2, 0, 2), (3, 0, 3), (1, 1, 1), (4, 1, 4)):
            n = (50, 30)[parent]
            own = paged.PagedKvCache(8, page, kv.KvCacheQuantMode.kQ8Q8, kv_heads=heads, head_dim=d, qblock=32)
            batch = paged.PagedBatch(torch.arange(8, dtype=torch.int32, device="cuda")[None].contiguous(), po.ints([0, n + 1]), po.ints([n + 1]), total_tokens=n + 1, max_tokens=n + 1,
                                     max_length=n + 1)
            k, v = (torch.cat((a[(0, 50)[parent]:(50, 80)[parent]], b[row:row + 1])) for a, b in zip(first[layer], second[layer]))
            paged.launch_paged_store(own.view(), batch, k, v, None)
            pages = book.tables_tensor[slot, :-(-(n + 1) // page)].long()
            got = cache.key[pages].transpose(1, 2).flatten(0, 1)[:n + 1]
            assert torch.equal(got, own.key[:len(pages)].transpose(1, 2).flatten(0, 1)[:n + 1])
    paged.launch_pages_free(book, po.ints([0, 1]))
    moved = torch.zeros(40, dtype=torch.int32, device="cuda")
    paged.launch_pages_compact(book, views, moved, workspace=ws)
    assert int((book.refs_tensor > 0).sum()) == int(book.tables_tensor[[2, 3, 4]].max()) + 1
    batch = paged.PagedBatch(book.tables_tensor, po.ints([0, 0, 0, 1, 2, 3, 3]), book.lengths_tensor, total_tokens=3, max_tokens=1, max_length=8 * page)
    for view, want in zip(views, before):
        out = torch.zeros(3, hq, d, dtype=torch.float16, device="cuda")
        paged.launch_paged_attention(view, batch, q[2:].contiguous(), out, query_heads=hq, scale=0.09, workspace=paged.paged_workspace(view, batch, hq))
        assert torch.equal(out, want[2:])
    assert int(status) == 0
