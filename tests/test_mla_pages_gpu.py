"""Page management of the latent cache on a GPU: copy, extend, fork, free, compact, against Python lists, bit for bit."""
import random

import pytest
import torch

import paged_reference as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ext(cuda_device):
    import cuda_agent_b200
    return cuda_agent_b200.load_extension()


def ints(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


class State:
    """A pool on the GPU and the same in lists."""

    def __init__(self, dev, slots, max_pages, pool, page, layers=2, row=8, dtype=torch.bfloat16):
        self.dev, self.page = dev, page
        self.table = torch.full((slots, max_pages), -1, dtype=torch.int32, device=dev)
        self.length = torch.zeros(slots, dtype=torch.int32, device=dev)
        self.refcount = torch.zeros(pool, dtype=torch.int32, device=dev)
        g = torch.Generator(device=dev).manual_seed(pool)
        self.pages = torch.randint(-100, 100, (layers, pool, page, row), generator=g, device=dev).to(dtype)
        self.reset()

    def reset(self):
        self.want = ref.Pool(self.table, self.length, self.refcount, self.page)
        self.want_pages = self.pages.clone()

    def check(self):
        for a, b in self.want.copies:
            self.want_pages[:, b] = self.want_pages[:, a]
        self.want.copies = []
        assert self.table.tolist() == self.want.table
        assert self.length.tolist() == self.want.length
        assert self.refcount.tolist() == self.want.count
        assert torch.equal(self.pages, self.want_pages)

    def held(self):
        return sum(n > 0 for n in self.want.count)


@pytest.mark.parametrize("page,pool,seed", [(1, 300, 0), (4, 200, 1), (16, 5000, 2), (64, 40, 3), (3, 9000, 4)])
def test_a_long_history_of_calls(ext, cuda_device, page, pool, seed):
    """Random extends, forks, frees and compactions, each checked whole; the pool fills up and empties."""
    rng = random.Random(seed)
    slots, max_pages = 24, max(4, pool // 8)
    s = State(cuda_device, slots, max_pages, pool, page)
    for _ in range(60):
        live = [i for i, n in enumerate(s.want.length) if n]
        empty = [i for i, n in enumerate(s.want.length) if not n]
        room = pool - s.held()
        what = rng.choice(["extend", "extend", "fork", "free", "compact"])
        if what == "extend":
            seqs = rng.sample(range(slots), rng.randint(1, slots))
            new = [min(max_pages * page, s.want.length[i] + rng.choice([0, 1, 2, page, rng.randint(0, 3 * page)])) for i in seqs]
            need = sum(max(0, -(-n // page) - -(-s.want.length[i] // page)) for i, n in zip(seqs, new))
            if need > room:
                with pytest.raises(RuntimeError, match="free pages"):
                    ext.mla_pages_extend(s.table, s.length, s.refcount, ints(seqs, s.dev), ints(new, s.dev), page, True)
            else:
                s.want.extend(seqs, new)
                ext.mla_pages_extend(s.table, s.length, s.refcount, ints(seqs, s.dev), ints(new, s.dev), page, True)
        elif what == "fork" and live and empty:
            dst = rng.sample(empty, rng.randint(1, len(empty)))
            src = [rng.choice(live) for _ in dst]
            need = sum(s.want.length[a] % page != 0 for a in src)
            if need > room:
                with pytest.raises(RuntimeError, match="free pages"):
                    ext.mla_pages_fork(s.pages, s.table, s.length, s.refcount, ints(src, s.dev), ints(dst, s.dev), True)
            else:
                s.want.fork(src, dst)
                ext.mla_pages_fork(s.pages, s.table, s.length, s.refcount, ints(src, s.dev), ints(dst, s.dev), True)
        elif what == "free" and live:
            seqs = rng.sample(live, rng.randint(1, len(live)))
            s.want.free(seqs)
            ext.mla_pages_free(s.table, s.length, s.refcount, ints(seqs + seqs[:1], s.dev), page, True)   # one twice
        elif what == "compact":
            s.want.compact()
            ext.mla_pages_compact(s.pages, s.table, s.length, s.refcount, True)
        s.check()


@pytest.mark.parametrize("dtype,row", [(torch.bfloat16, 576), (torch.bfloat16, 6), (torch.int8, 7), (torch.float32, 1)])
@pytest.mark.parametrize("layers,strided", [(1, False), (3, False), (3, True)])
def test_copy(ext, cuda_device, dtype, row, layers, strided):
    """Every access width; layers that are views of a wider store."""
    g = torch.Generator(device=cuda_device).manual_seed(row)
    store = torch.randint(-9, 9, (layers, 2, 50, 5, row), generator=g, device=cuda_device).to(dtype)
    pages = store[:, 1] if strided else store[:, 1].contiguous()
    before = store.clone()
    want = pages.clone()
    src, dst = [3, 3, 7, -1, 49, 8, 9], [10, 0, 48, 5, 1, -1, 9]        # a page twice as source, skipped pairs, onto itself
    for a, b in zip(src, dst):
        if a >= 0 and b >= 0:
            want[:, b] = pages[:, a]
    got = ext.mla_pages_copy(pages, ints(src, cuda_device), ints(dst, cuda_device), True)
    assert got.data_ptr() == pages.data_ptr() and torch.equal(pages, want)
    assert torch.equal(store[:, 0], before[:, 0])


def test_copy_refuses_pairs_that_depend_on_their_order(ext, cuda_device):
    pages = torch.arange(20, device=cuda_device, dtype=torch.float32)[None, :, None, None].repeat(2, 1, 3, 4).contiguous()
    before = pages.clone()
    for src, dst, fine in (([1, 2, 5], [9, 9, 10], [(5, 10)]),            # a page written twice
                           ([1, 9, 5], [9, 11, 10], [(5, 10)]),           # a page written and read
                           ([1, 20, 5], [9, 11, 20], [(1, 9)]),           # beyond the pool
                           ([1, 2 ** 31 - 1, 4], [12, 3, 13], [(1, 12), (4, 13)])):
        pages.copy_(before)
        with pytest.raises(RuntimeError, match="out of range or listed twice"):
            ext.mla_pages_copy(pages, ints(src, cuda_device), ints(dst, cuda_device), True)
        want = before.clone()
        for a, b in fine:
            want[:, b] = before[:, a]
        assert torch.equal(pages, want)


def test_copy_of_many_pages_and_of_none(ext, cuda_device):
    g = torch.Generator(device=cuda_device).manual_seed(0)
    pages = torch.randn(1, 6000, 16, 64, generator=g, device=cuda_device)
    order = torch.randperm(6000, generator=g, device=cuda_device).to(torch.int32)
    want = pages.clone()
    want[:, order[3000:].long()] = pages[:, order[:3000].long()]
    ext.mla_pages_copy(pages, order[:3000], order[3000:], True)
    assert torch.equal(pages, want)
    ext.mla_pages_copy(pages, order[:0], order[:0], True)
    ext.mla_pages_copy(pages[:0], order[:10], order[10:20], True)
    assert torch.equal(pages, want)


def test_extend_and_fork_change_everything_or_nothing(ext, cuda_device):
    s = State(cuda_device, 6, 8, 20, 4)
    call = lambda seqs, new: ext.mla_pages_extend(s.table, s.length, s.refcount, ints(seqs, s.dev), ints(new, s.dev), 4, True)
    s.want.extend([0, 3], [10, 4])
    call([0, 3], [10, 4])
    s.check()
    for seqs, new, text in (([0, 1, 0], [12, 3, 14], "listed twice"), ([1, 6], [3, 3], "out of range"), ([1, -1], [3, 3], "out of range"),
                            ([1, 2], [3, 33], "free pages"), ([1, 2], [3, 2 ** 31 - 1], "free pages"),
                            ([1, 2, 4], [32, 32, 5], "free pages")):
        with pytest.raises(RuntimeError, match=text):
            call(seqs, new)
        s.check()
    call([0, 1], [-5, 0])                            # nothing to do
    call([], [])
    s.check()
    fork = lambda src, dst: ext.mla_pages_fork(s.pages, s.table, s.length, s.refcount, ints(src, s.dev), ints(dst, s.dev), True)
    for src, dst, text in (([0, 0], [1, 1], "listed twice"), ([0, 6], [1, 2], "out of range"), ([0, 0], [1, -1], "out of range"),
                           ([0, 0], [1, 3], "in use"), ([0], [0], "in use")):
        with pytest.raises(RuntimeError, match=text):
            fork(src, dst)
        s.check()
    s.want.extend([4], [32])
    call([4], [32])
    s.want.extend([5], [32])
    call([5], [32])                                  # 20 pages are taken
    s.check()
    with pytest.raises(RuntimeError, match="free pages"):
        fork([0], [1])
    s.check()
    s.want.fork([3, 4], [1, 2])
    fork([3, 4], [1, 2])                             # full pages only: shared without a free one
    s.check()
    fork([], [])
    with pytest.raises(RuntimeError, match="out of range"):
        ext.mla_pages_free(s.table, s.length, s.refcount, ints([6], s.dev), 4, True)
    s.check()


def test_chains_of_empty_parents(ext, cuda_device):
    """An empty parent gives an empty child, also when it is another pair's child."""
    s = State(cuda_device, 5, 4, 9, 4)
    ext.mla_pages_fork(s.pages, s.table, s.length, s.refcount, ints([1, 2, 3], s.dev), ints([2, 3, 4], s.dev), True)
    s.check()


def test_large_lists(ext, cuda_device):
    """More sequences than one pass of the deciding CTA takes, and pools of more than one scan step."""
    s = State(cuda_device, 3001, 6, 20000, 2, layers=1, row=2)
    seqs = list(range(3000))
    random.Random(0).shuffle(seqs)
    new = [1 + i % 11 for i in range(3000)]
    s.want.extend(seqs, new)
    ext.mla_pages_extend(s.table, s.length, s.refcount, ints(seqs, s.dev), ints(new, s.dev), 2, True)
    s.check()
    s.want.free(seqs[::2])
    ext.mla_pages_free(s.table, s.length, s.refcount, ints(seqs[::2], s.dev), 2, True)
    src = [seqs[1 + 2 * (i % 1500)] for i in range(1500)]
    s.want.fork(src, seqs[::2])
    ext.mla_pages_fork(s.pages, s.table, s.length, s.refcount, ints(src, s.dev), ints(seqs[::2], s.dev), True)
    s.check()
    s.want.free(seqs[1::4])
    ext.mla_pages_free(s.table, s.length, s.refcount, ints(seqs[1::4], s.dev), 2, True)
    s.want.compact()
    ext.mla_pages_compact(s.pages, s.table, s.length, s.refcount, True)
    s.check()
    s.want.compact()                                  # nothing left to move
    ext.mla_pages_compact(s.pages, s.table, s.length, s.refcount, True)
    s.check()


def test_tables_that_disagree_with_the_counts(ext, cuda_device):
    """Entries outside the pool, and pages that count as free, are reported; nothing outside the arrays is touched."""
    s = State(cuda_device, 4, 4, 12, 4)
    ext.mla_pages_extend(s.table, s.length, s.refcount, ints([0, 1], s.dev), ints([16, 9], s.dev), 4, True)
    for bad in (-1, 12, 2 ** 31 - 1, 11):             # 11 is free
        table, length, count = s.table.clone(), s.length.clone(), s.refcount.clone()
        table[0, 2] = bad
        with pytest.raises(RuntimeError, match="page table"):
            ext.mla_pages_free(table, length, count, ints([0], s.dev), 4, True)
        assert count.tolist() == [0, 0, 1, 0, 1, 1, 1] + [0] * 5
        table = s.table.clone()
        table[1, 0] = bad
        keep = table.clone()
        with pytest.raises(RuntimeError, match="page table"):
            ext.mla_pages_compact(s.pages, table, s.length, s.refcount.clone(), True)
        assert torch.equal(table, keep)               # seven pages in use, the seven lowest: nothing moves
    table = s.table.clone()
    table[1, 2] = 12
    with pytest.raises(RuntimeError, match="page table"):
        ext.mla_pages_fork(s.pages, table, s.length, s.refcount, ints([1], s.dev), ints([2], s.dev), True)
    s.reset()
    s.check()


def test_in_a_graph_and_on_a_stream(ext, cuda_device):
    s = State(cuda_device, 8, 8, 40, 4)
    seqs, new, dst = ints([0, 1, 2], s.dev), ints([9, 4, 17], s.dev), ints([5, 6, 7], s.dev)

    def step():
        ext.mla_pages_extend(s.table, s.length, s.refcount, seqs, new, 4)
        ext.mla_pages_fork(s.pages, s.table, s.length, s.refcount, seqs, dst)
        ext.mla_pages_free(s.table, s.length, s.refcount, seqs, 4)
        ext.mla_pages_compact(s.pages, s.table, s.length, s.refcount)

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    stream = torch.cuda.Stream()
    for replay in range(3):
        s.want.extend(seqs.tolist(), new.tolist())
        s.want.fork(seqs.tolist(), dst.tolist())
        for a, b in s.want.copies:
            s.want_pages[:, b] = s.want_pages[:, a]
        s.want.copies = []
        s.want.free(seqs.tolist())
        s.want.compact()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            graph.replay() if replay else step()
        stream.synchronize()
        s.check()
        s.want.free(dst.tolist())
        ext.mla_pages_free(s.table, s.length, s.refcount, dst, 4, True)
        s.check()


def test_pages_refusals(ext, cuda_device):
    s = State(cuda_device, 4, 4, 12, 4)
    one = ints([0], s.dev)
    for bad in (lambda: ext.mla_pages_copy(s.pages.transpose(1, 2), one, one), lambda: ext.mla_pages_copy(s.pages, one, ints([0, 1], s.dev)),
                lambda: ext.mla_pages_copy(s.pages, one.long(), one), lambda: ext.mla_pages_copy(s.pages.cpu(), one, one),
                lambda: ext.mla_pages_copy(s.pages[0, 0], one, one), lambda: ext.mla_pages_copy(s.pages[:1].expand(3, 12, 4, 8), one, one),
                lambda: ext.mla_pages_extend(s.table, s.length, s.refcount, one, one, 0),
                lambda: ext.mla_pages_extend(s.table, s.length[:3], s.refcount, one, one, 4),
                lambda: ext.mla_pages_extend(s.table, s.length, s.refcount, one, ints([1, 2], s.dev), 4),
                lambda: ext.mla_pages_extend(s.table, s.length, s.refcount, one.cpu(), one, 4),
                lambda: ext.mla_pages_extend(s.table, s.length, s.refcount, ints([0, 1, 2, 3], s.dev), s.length, 4),
                lambda: ext.mla_pages_fork(s.pages, s.table, s.length, s.refcount[:5], one, one),
                lambda: ext.mla_pages_fork(s.pages, s.table.t(), s.length, s.refcount, one, one),
                lambda: ext.mla_pages_free(s.table, s.length, s.refcount, one, -4),
                lambda: ext.mla_pages_compact(s.pages[:, :5], s.table, s.length, s.refcount)):
        with pytest.raises(RuntimeError):
            bad()
    s.check()


def test_lists_inside_the_pool_are_refused_and_one_buffer_is_not(ext, cuda_device):
    """A list that is read again after the table or the lengths changed would no longer say what was checked."""
    store = torch.zeros(16 + 4 + 12 + 8, dtype=torch.int32, device=cuda_device)
    table, length, refcount, lists = store[:16].view(4, 4), store[16:20], store[20:32], store[32:]
    table.fill_(-1)
    pages = torch.zeros(2, 12, 4, 8, dtype=torch.int32, device=cuda_device)
    one = ints([0], cuda_device)
    inside = pages[0, 0, 0]
    for bad in (lambda: ext.mla_pages_extend(table, length, refcount, length, ints([1, 1, 1, 1], cuda_device), 4),
                lambda: ext.mla_pages_extend(table, length, refcount, refcount[:1], one, 4),
                lambda: ext.mla_pages_extend(table, length, refcount, one, table[3, 3:], 4),
                lambda: ext.mla_pages_extend(table, store[15:19], refcount, one, one, 4),
                lambda: ext.mla_pages_extend(table, length, store[19:31], one, one, 4),
                lambda: ext.mla_pages_fork(pages, table, length, refcount, length[:1], one),
                lambda: ext.mla_pages_fork(pages, table, length, refcount, one, inside[:1]),
                lambda: ext.mla_pages_copy(pages, one, inside[:1]),
                lambda: ext.mla_pages_free(table, length, refcount, table[0], 4)):
        with pytest.raises(RuntimeError, match="overlap"):
            bad()
    assert (table == -1).all() and not length.any() and not refcount.any()
    lists[:2] = ints([2, 7], cuda_device)
    ext.mla_pages_extend(table, length, refcount, lists[:1], lists[1:2], 4, True)
    assert table[2].tolist() == [0, 1, -1, -1] and length.tolist() == [0, 0, 7, 0] and refcount[:3].tolist() == [1, 1, 0]


@pytest.mark.parametrize("at", [0, 1, 2, 4])
def test_fork_with_a_bad_entry_changes_nothing(ext, cuda_device, at):
    """Any needed entry of the parent (full pages 0 to 3, the partly filled fifth): outside the pool, or a page that counts as
    free and could be the child's fresh one. Sound pairs of the same call are not carried out either."""
    s = State(cuda_device, 6, 6, 14, 4)
    ext.mla_pages_extend(s.table, s.length, s.refcount, ints([0, 1], s.dev), ints([18, 9], s.dev), 4, True)
    s.reset()
    for bad in (-1, 14, 2 ** 31 - 1, 8):              # eight pages are in use, 8 is the lowest free one
        table = s.table.clone()
        table[0, at] = bad
        keep = table.clone()
        with pytest.raises(RuntimeError, match="page table"):
            ext.mla_pages_fork(s.pages, table, s.length, s.refcount, ints([1, 0, 0, 1], s.dev), ints([2, 3, 4, 5], s.dev), True)
        assert torch.equal(table, keep)
        s.check()                                     # lengths, counts and pages as they were
    broken = s.table.clone()
    broken[1, 2] = 13
    broken[0, 5] = 99                                 # behind the parent's last page: not needed
    ext.mla_pages_fork(s.pages, broken, s.length, s.refcount, ints([0, 0], s.dev), ints([2, 3], s.dev), True)
    s.table.copy_(broken)
    s.want.table = broken.tolist()
    for row in (2, 3):
        s.want.table[row] = [-1] * 6
    s.want.fork([0, 0], [2, 3])
    s.check()


def test_compact_reports_an_entry_at_a_free_page(ext, cuda_device):
    """A row that names a free page, which the compaction fills with another sequence's data, whether the page lies among
    those that stay or above them."""
    s = State(cuda_device, 5, 4, 12, 4)
    ext.mla_pages_extend(s.table, s.length, s.refcount, ints([0, 1, 2], s.dev), ints([8, 8, 8], s.dev), 4, True)
    ext.mla_pages_free(s.table, s.length, s.refcount, ints([1], s.dev), 4, True)
    assert s.refcount.tolist()[:6] == [1, 1, 0, 0, 1, 1]
    for bad in (3, 11):
        table, length, count = s.table.clone(), s.length.clone(), s.refcount.clone()
        table[0, 1] = bad
        with pytest.raises(RuntimeError, match="page table"):
            ext.mla_pages_compact(s.pages.clone(), table, length, count, True)


def test_tables_inside_the_pages_are_refused(ext, cuda_device):
    pages = torch.zeros(2, 12, 4, 8, dtype=torch.int32, device=cuda_device)
    s = State(cuda_device, 4, 4, 12, 4)
    one, two = ints([0], s.dev), ints([1], s.dev)
    table, length, refcount = pages[0, 0, :2].view(4, 4), pages[1, 11, 3, 4:], pages.view(-1)[100:112]
    for t, n, r in ((table, s.length, s.refcount), (s.table, length, s.refcount), (s.table, s.length, refcount)):
        with pytest.raises(RuntimeError, match="overlap"):
            ext.mla_pages_fork(pages, t, n, r, one, two)
        with pytest.raises(RuntimeError, match="overlap"):
            ext.mla_pages_compact(pages, t, n, r)
    assert not pages.any()
    # the tables in gaps between the layers are elsewhere
    store = torch.zeros(2, 12 * 4 * 8 + 64, dtype=torch.int32, device=cuda_device)
    pages = store[:, :12 * 4 * 8].view(2, 12, 4, 8)
    s.refcount = store[0, 12 * 4 * 8:][:12]
    s.pages = pages
    s.reset()
    s.want.extend([0], [6])
    ext.mla_pages_extend(s.table, s.length, s.refcount, one, ints([6], s.dev), 4, True)
    s.want.fork([0], [1])
    ext.mla_pages_fork(pages, s.table, s.length, s.refcount, one, two, True)
    s.check()


def test_empty_lists_anywhere(ext, cuda_device):
    """A list without elements shares nothing, wherever it points."""
    s = State(cuda_device, 6, 6, 14, 4, dtype=torch.int32)
    none = (s.length[2:2], s.table[1, 3:3], s.refcount[5:5], s.pages.view(-1)[40:40])
    for a in none:
        ext.mla_pages_extend(s.table, s.length, s.refcount, a, a, 4, True)
        ext.mla_pages_fork(s.pages, s.table, s.length, s.refcount, a, a, True)
        ext.mla_pages_free(s.table, s.length, s.refcount, a, 4, True)
        ext.mla_pages_copy(s.pages, a, a, True)
    s.check()
