"""Block tables, slots and positions (``kernels/paged.py``) against a plain
walk over the requests; every output is an integer and has to be equal."""
import random

import pytest
import torch

from kernels.paged import PagedStep, PagedTables, paged_release, paged_step

pytestmark = pytest.mark.gpu


def _i32(a, dev):
    return torch.tensor(a, dtype=torch.int32, device=dev).reshape(len(a))


class Walk:
    """The same state on the host, request by request."""

    def __init__(self, requests, width, pages, page):
        self.tables = [[] for _ in range(requests)]
        self.lengths = [0] * requests
        self.free = list(range(pages - 1, -1, -1))
        self.width, self.page = width, page

    def step(self, new, total):
        starts, slots, positions, failed = [0], [-1] * total, [-1] * total, []
        asked, available = 0, len(self.free)
        for b, m in enumerate(new):
            first, end = sum(max(0, x) for x in new[:b]), sum(max(0, x) for x in new[:b + 1])
            starts.append(min(end, total))
            n = self.lengths[b]
            fits = m >= 0 and n + m <= self.width * self.page and end <= total
            need = -(-(n + m) // self.page) - -(-n // self.page) if fits else 0
            asked += need
            ok = fits and (need == 0 or asked <= available)
            failed.append(0 if ok else 1)
            if not ok:
                continue
            for i in range(m):
                p = n + i
                if p // self.page == len(self.tables[b]):
                    self.tables[b].append(self.free.pop())
                slots[first + i] = self.tables[b][p // self.page] * self.page + p % self.page
                positions[first + i] = p
            self.lengths[b] += m
        return starts, slots, positions, failed

    def release(self, keep):
        for b, k in enumerate(keep):
            k = min(max(k, 0), self.lengths[b])
            held = -(-k // self.page)
            self.free += self.tables[b][held:]
            del self.tables[b][held:]
            self.lengths[b] = k


def _same(tables, walk):
    state = tables.state.tolist()
    assert state[:-1] == walk.lengths and state[-1] == len(walk.free)
    assert tables.free_pages[:state[-1]].tolist() == walk.free
    for row, pages in zip(tables.block_tables.tolist(), walk.tables):
        assert row[:len(pages)] == pages


def _step(tables, walk, new, total, dev, out=None):
    old = tables.state.clone()
    r = paged_step(tables, _i32(new, dev), total, out=out)
    assert torch.equal(tables.state, old), "a step changes the state only when it is committed"
    starts, slots, positions, failed = walk.step(new, total)
    assert r.query_start.tolist() == starts and r.failed.tolist() == failed
    assert r.slots.tolist() == slots and r.positions.tolist() == positions
    tables.commit(r)
    _same(tables, walk)
    return r


@pytest.mark.parametrize("requests,page", [(1, 16), (7, 64), (64, 16), (255, 32), (256, 128), (257, 16), (1000, 256)])
def test_steps_and_releases(gpu, requests, page):
    rng = random.Random(requests)
    width = 12
    pages = requests * 7 + 3
    tables, walk = PagedTables(requests, width, pages, page, gpu), Walk(requests, width, pages, page)
    for step in range(6):
        if step % 2 == 0:       # prompts and single tokens, some requests idle
            new = [rng.choice([0, 1, 1, 1, page - 1, page, page + 1, rng.randint(0, 3 * page)]) for _ in range(requests)]
        else:
            new = [1] * requests
        _step(tables, walk, new, sum(new) + rng.choice([0, 0, 5]), gpu)
        if step in (2, 4):
            keep = [rng.choice([0, n, n, max(0, n - 1), n + 9, -3, n // 2]) for n in walk.lengths]
            paged_release(tables, _i32(keep, gpu))
            walk.release(keep)
            _same(tables, walk)


def test_free_pages_that_are_part_of_a_cache(gpu):
    """A stack of a few pages with large numbers: numbers are not bounded by the stack's length."""
    free = _i32([7, 2**26 - 1, 9000], gpu)
    tables = PagedTables.of(torch.full((2, 4), -1, dtype=torch.int32, device=gpu), _i32([0, 0, 3], gpu), free, 16)
    r = paged_step(tables, _i32([17, 1], gpu), 18)
    assert r.slots.tolist() == [9000 * 16 + i for i in range(16)] + [(2**26 - 1) * 16, 7 * 16]
    assert r.state.tolist() == [17, 1, 0] and tables.block_tables[:, :2].tolist() == [[9000, 2**26 - 1], [7, -1]]


def test_refused_requests(gpu):
    """Too few pages, rows past the batch, tokens past the table, a negative number."""
    tables, walk = PagedTables(6, 4, 9, 16, gpu), Walk(6, 4, 9, 16)
    _step(tables, walk, [16, 15, 40, 65, 0, 3], 139, gpu)                 # 65 pass the table
    _step(tables, walk, [0, 1, 16, -1, 2, 1], 20, gpu)                    # nothing is left for one that needs two
    _step(tables, walk, [1, 0, 0, 40, 16, 1], 58, gpu)                    # not enough pages from the fourth on
    _step(tables, walk, [0, 3, 2, 0, 0, 2], 6, gpu)                       # the last one's rows pass the batch
    _step(tables, walk, [0, 0, 0, 0, 0, 0], 3, gpu)
    _step(tables, walk, [0, 0, 0, 0, 0, 0], 0, gpu)
    _step(tables, walk, [2**31 - 1] * 5 + [1], 7, gpu)


def test_most_requests_and_many_rows(gpu):
    rng = random.Random(2)
    tables, walk = PagedTables(4096, 3, 9000, 16, gpu), Walk(4096, 3, 9000, 16)
    new = [rng.randint(0, 20) for _ in range(4096)]
    _step(tables, walk, new, sum(new), gpu)
    tables, walk = PagedTables(3, 4000, 9000, 16, gpu), Walk(3, 4000, 9000, 16)
    _step(tables, walk, [50001, 0, 20003], 70004, gpu)
    paged_release(tables, _i32([17, 0, 0], gpu))
    walk.release([17, 0, 0])
    _same(tables, walk)


def test_step_can_be_given_up_and_repeated(gpu):
    tables = PagedTables(3, 8, 10, 16, gpu)
    new = _i32([20, 1, 40], gpu)
    a, b = paged_step(tables, new, 61), paged_step(tables, new, 61)
    for x, y in zip(vars(a).values(), vars(b).values()):
        assert torch.equal(x, y)
    assert tables.lengths.tolist() == [0, 0, 0] and tables.free_count.item() == 10


def test_step_into_given_tensors_and_in_a_graph(gpu):
    """Two steps in turn write each other's state: captured once, replayed."""
    tables, walk = PagedTables(5, 40, 150, 16, gpu), Walk(5, 40, 150, 16)
    _step(tables, walk, [3, 17, 1, 30, 9], 60, gpu)
    state = tables.state
    one = torch.ones(5, dtype=torch.int32, device=gpu)
    r = PagedStep.empty(5, 5, gpu)

    def step():
        paged_step(tables, one, 5, out=r)
        state.copy_(r.state)

    side = torch.cuda.Stream(gpu)
    side.wait_stream(torch.cuda.current_stream(gpu))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step()
    torch.cuda.current_stream(gpu).wait_stream(side)
    for _ in range(40):
        graph.replay()
        torch.cuda.synchronize()
        starts, slots, positions, failed = walk.step([1] * 5, 5)
        assert r.slots.tolist() == slots and r.positions.tolist() == positions and r.failed.tolist() == failed
        _same(tables, walk)


def test_refusals(gpu):
    tables = PagedTables(3, 4, 5, 16, gpu)
    new = _i32([1, 1, 1], gpu)
    for bad in (lambda: paged_step(tables, new.long(), 3),
                lambda: paged_step(tables, new[:2], 3),
                lambda: paged_step(tables, new.cpu(), 3),
                lambda: paged_step(tables, new, -1),
                lambda: paged_step(tables, new, 3, out=PagedStep.empty(3, 4, gpu)),
                lambda: paged_release(tables, new.long()),
                lambda: PagedTables(3, 4, 5, 24, gpu),
                lambda: PagedTables(4097, 4, 5, 16, gpu),
                lambda: PagedTables.of(tables.block_tables, tables.state[:-1], tables.free_pages, 16),
                lambda: tables.commit(PagedStep.empty(4, 3, gpu))):
        with pytest.raises(ValueError):
            bad()
    r = paged_step(tables, new, 3)
    tables.commit(r)
    with pytest.raises(ValueError):
        paged_step(tables, new, 3, out=r)
