"""Page operations against the Python oracle: whole numbers and bytes, all equal."""

import numpy as np
import pytest

import oracle

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
from tensorsmith_b200 import engine  # noqa: E402


class Pages:
    def __init__(self, lens, pages, page, *, layers=2, words=8, slots=None, seed=0, pins=0):
        rng = np.random.default_rng(seed)
        self.page = page
        lens = np.asarray(lens, np.int32)
        need = -(-lens // page)
        slots = int(need.max(initial=0)) + 2 if slots is None else slots
        table = np.full((len(lens), slots), -1, np.int32)
        order = rng.permutation(pages)
        at = 0
        for r, n in enumerate(need):
            table[r, :n] = order[at:at + n]
            at += n
        refs = np.zeros(pages, np.int32)
        refs[table[table >= 0]] += 1
        refs[order[at:at + pins]] += 1  # held by the caller alone
        pool = rng.integers(0, 2**62, (layers, pages, 2, words))
        self.oracle = oracle.PagesOracle(table, lens, refs, pool, page)
        self.table, self.lens, self.refs, self.pool = (torch.from_numpy(x.copy()).cuda() for x in (table, lens, refs, pool))
        self.counters = torch.tensor([int((refs == 0).sum()), 0, 0, 0], dtype=torch.int32, device="cuda")

    def fork(self, index):
        idx = torch.tensor(index, dtype=torch.int32, device="cuda")
        self.table, self.lens = engine.kv_pages_fork(self.table, self.lens, idx, self.refs, self.counters,
                                                     page_size=self.page)
        self.oracle.fork(index)

    def reserve(self, steps):
        rows = len(self.oracle.lens)
        given = steps if isinstance(steps, int) else torch.tensor(steps, dtype=torch.int32, device="cuda")
        engine.kv_pages_reserve(self.pool, self.table, self.lens, given, self.refs, self.counters, page_size=self.page)
        return self.oracle.reserve([steps] * rows if isinstance(steps, int) else steps)

    def advance(self, steps):
        self.lens += torch.tensor(steps, dtype=torch.int32, device="cuda")
        self.oracle.lens = self.oracle.lens + np.asarray(steps, np.int32)

    def check(self, error=0):
        o = self.oracle
        np.testing.assert_array_equal(self.table.cpu().numpy(), o.table)
        np.testing.assert_array_equal(self.lens.cpu().numpy(), o.lens)
        np.testing.assert_array_equal(self.refs.cpu().numpy(), o.refs)
        np.testing.assert_array_equal(self.pool.cpu().numpy(), o.pool)
        free, low, err, _ = self.counters.tolist()
        assert free == (o.refs == 0).sum() and err == error
        assert not (o.refs[:low] == 0).any()


@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("lens", [[0], [1], [16], [17, 64], [100, 0, 63, 64, 65, 5, 130, 1]])
def test_reserve_of_unshared_rows(page, lens):
    p = Pages(lens, 60, page, seed=len(lens))
    for steps in (1, 0, page, 2 * page - 1):
        if p.reserve(steps):
            p.check()
            p.advance([steps] * len(lens))


@pytest.mark.parametrize("seed", range(6))
def test_random_histories(seed):
    """Forks, frees, reorders, reserves and compactions in a row, shared partial pages among them."""
    rng = np.random.default_rng(seed)
    page, rows = int(rng.choice([16, 32])), int(rng.integers(2, 40))
    p = Pages(rng.integers(0, 5 * page, rows), 900, page, seed=seed, slots=12, words=int(rng.choice([2, 8, 2600])),
              layers=int(rng.integers(1, 4)), pins=5)
    for _ in range(8):
        n = len(p.oracle.lens)
        kind = rng.integers(0, 4)
        if kind == 0:
            p.fork(rng.integers(-1, n, int(rng.integers(1, 40))).tolist())
        elif kind == 1:
            engine.kv_pages_compact(p.pool, p.table, p.refs, p.counters)
            p.oracle.compact()
        else:
            room = 12 * page - p.oracle.lens
            steps = np.minimum(rng.integers(0, 2 * page, n), room).astype(np.int32)
            assert p.reserve(steps.tolist())
            p.check()
            p.advance(steps)
        # pool contents past a compaction's live pages are free pages' leftovers, equal on both sides
        p.check()


def test_many_rows_share_one_page():
    """1500 rows (more than a block's threads) fork one prompt and all write to its last page."""
    p = Pages([21], 2000, 16, layers=1)
    p.fork([0] * 1500)
    p.check()
    assert p.reserve(1)
    p.check()
    assert p.refs.max() == 1500  # the full first page stays shared


def test_a_pinned_partial_page_is_copied_by_every_writer():
    p = Pages([5, 5], 10, 16)
    held = int(p.oracle.table[0, 0])
    p.refs[held] += 1
    p.oracle.refs[held] += 1
    assert p.reserve(1)
    p.check()
    assert int(p.refs[held]) == 1


def test_free_returns_pages():
    p = Pages([40, 17, 3], 8, 16)
    p.fork([-1, 1, -1])
    p.check()
    p.fork([-1])
    p.check()
    assert p.counters[0] == 8


def test_shortage_changes_nothing():
    p = Pages([16, 16], 3, 16)
    p.fork([0, 1])
    assert not p.reserve(1)  # two pages wanted, one free
    p.check(error=engine.PAGES_SHORT)
    p = Pages([16, 16], 30, 16, slots=2)
    assert not p.reserve(17)  # a third slot
    p.check(error=engine.PAGES_NO_SLOT)
    p = Pages([16], 3, 16)
    idx = torch.tensor([1], dtype=torch.int32, device="cuda")
    table, lens = engine.kv_pages_fork(p.table, p.lens, idx, p.refs, p.counters, page_size=16)
    assert (table == -1).all() and lens.tolist() == [0] and p.counters[2] == engine.PAGES_BAD_INDEX


@pytest.mark.parametrize("pages, live", [(1, 0), (1, 1), (5, 3), (4096, 1000), (4097, 4097), (20000, 7777)])
def test_compact_sizes(pages, live):
    """Around the 4096 pages that a block ranks, nothing to do and everything free included."""
    rng = np.random.default_rng(pages + live)
    table = np.full((1, max(1, live)), -1, np.int32)
    table[0, :live] = rng.permutation(pages)[:live]
    refs = np.zeros(pages, np.int32)
    refs[table[0, :live]] = rng.integers(1, 4, live)
    pool = rng.integers(0, 2**62, (1, pages, 1, 2))
    o = oracle.PagesOracle(table, [0], refs, pool, 16)
    o.compact()
    counters = torch.tensor([pages - live, 0, 0, 0], dtype=torch.int32, device="cuda")
    dev = [torch.from_numpy(x.copy()).cuda() for x in (table, refs, pool)]
    outs = torch.full_like(dev[0], 77), torch.full_like(dev[1], 77)
    pool_before = dev[2].clone()
    got = engine.kv_pages_compact(dev[2], dev[0], dev[1], counters, table_out=outs[0], refs_out=outs[1])
    assert got[0] is outs[0] and got[1] is outs[1]
    np.testing.assert_array_equal(outs[0].cpu().numpy(), o.table)
    np.testing.assert_array_equal(outs[1].cpu().numpy(), o.refs)
    np.testing.assert_array_equal(dev[2].cpu().numpy(), o.pool)
    np.testing.assert_array_equal(dev[0].cpu().numpy(), table)  # inputs untouched
    assert counters.tolist()[:3] == [pages - live, live, 0]
    engine.kv_pages_compact(pool_before, dev[0], dev[1], counters)  # in place
    np.testing.assert_array_equal(dev[0].cpu().numpy(), o.table)
    np.testing.assert_array_equal(dev[1].cpu().numpy(), o.refs)


def test_copy_between_pools():
    a = torch.randint(0, 2**62, (3, 9, 2, 500), device="cuda")
    b = torch.zeros(3, 20, 2, 500, dtype=torch.int64, device="cuda")
    src = torch.tensor([8, -1, 0, 3, 9], dtype=torch.int32, device="cuda")
    dst = torch.tensor([19, 2, -1, 0, 5], dtype=torch.int32, device="cuda")
    engine.kv_pages_copy(a, src, b, dst)
    want = torch.zeros_like(b)
    want[:, 19], want[:, 0] = a[:, 8], a[:, 3]
    assert torch.equal(b, want)
    none = torch.empty(0, dtype=torch.int32, device="cuda")
    engine.kv_pages_copy(a, none, b, none)


def test_refusals():
    p = Pages([5, 5], 10, 16)
    idx = torch.tensor([0, 1], dtype=torch.int32, device="cuda")
    kw = dict(page_size=16)
    for bad in (lambda: engine.kv_pages_fork(p.table, p.lens, idx.long(), p.refs, p.counters, **kw),
                lambda: engine.kv_pages_fork(p.table, p.lens[:1], idx, p.refs, p.counters, **kw),
                lambda: engine.kv_pages_fork(p.table, p.lens, idx[:0], p.refs, p.counters, **kw),
                lambda: engine.kv_pages_fork(p.table, p.lens, idx, p.refs, p.counters[:3], **kw),
                lambda: engine.kv_pages_reserve(p.pool, p.table, p.lens, -1, p.refs, p.counters, **kw),
                lambda: engine.kv_pages_reserve(p.pool, p.table, p.lens, 1, p.refs[:9], p.counters, **kw),
                lambda: engine.kv_pages_reserve(p.pool.transpose(2, 3), p.table, p.lens, 1, p.refs, p.counters, **kw),
                lambda: engine.kv_pages_reserve(p.pool, p.table, p.lens, idx.long(), p.refs, p.counters, **kw),
                lambda: engine.kv_pages_compact(p.pool, p.table, p.refs, p.counters, table_out=p.table[:1]),
                lambda: engine.kv_pages_copy(p.pool, idx, p.pool[:1], idx),
                lambda: engine.kv_pages_copy(p.pool, idx.long(), p.pool, idx),
                lambda: engine.kv_pages_copy(p.pool.cpu(), idx, p.pool, idx)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(engine._lib.EngineError):  # the new table must not be the old one
        engine.kv_pages_fork(p.table, p.lens, idx, p.refs, p.counters, table_out=p.table, **kw)
    p.check()
