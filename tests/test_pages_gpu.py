"""The pages of a paged cache on the device against the same bookkeeping in Python: handing out,
sharing, giving back, moving and copying, down to the order of pages; what cannot be done is
reported and left undone; long random histories, and replays of captured calls."""
import random

import pytest
import torch

from __graft_entry__ import load_package

pkg = load_package()
capi = pkg.capi
pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = capi.Context(0)
    yield c
    c.close()


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


class Model:
    """The pool in Python.  Every token of a sequence has a number of its own in each plane."""

    def __init__(self, pages, page, slots, table_len):
        self.pages, self.page, self.slots, self.table_len = pages, page, slots, table_len
        self.refs = [0] * pages
        self.held = [[] for _ in range(slots)]
        self.length = [0] * slots

    def free_pages(self):
        return [i for i, r in enumerate(self.refs) if r == 0]

    def extend(self, slots, counts):
        """What of it cannot be done: the codes."""
        wrong, seen, free, full = set(), set(), self.free_pages(), False
        for s, c in zip(slots, counts):
            if s == -1:
                continue
            if not 0 <= s < self.slots or s in seen or c < 0 or \
                    self.length[s] + c > self.table_len * self.page:
                seen.add(s)
                wrong.add("outside")
                continue
            seen.add(s)
            need = -(-(self.length[s] + c) // self.page) - len(self.held[s])
            if need > 0 and (full or need > len(free)):
                full = True  # pages go out in order
                wrong.add("out of pages")
                continue
            for _ in range(need):
                p = free.pop(0)
                self.refs[p] = 1
                self.held[s].append(p)
            self.length[s] += c
        return wrong

    def fork(self, parents, children):
        wrong, seen, free, copies = set(), set(), self.free_pages(), []
        before = list(self.length)
        for p, c in zip(parents, children):
            if -1 in (p, c):
                seen.add(c)
                continue
            if not (0 <= p < self.slots and 0 <= c < self.slots) or c in seen or before[c] != 0:
                seen.add(c)
                wrong.add("outside")
                continue
            seen.add(c)
            length = before[p]
            full = length // self.page
            if length % self.page and not free:
                wrong.add("out of pages")
                continue
            self.held[c] = self.held[p][:full]
            for q in self.held[c]:
                self.refs[q] += 1
            if length % self.page:
                q = free.pop(0)
                self.refs[q] = 1
                copies.append((self.held[p][full], q))
                self.held[c].append(q)
            self.length[c] = length
        return wrong, copies

    def free(self, slots):
        wrong = set()
        for s in slots:
            if s == -1:
                continue
            if not 0 <= s < self.slots:
                wrong.add("outside")
                continue
            for p in self.held[s]:
                self.refs[p] -= 1
            self.held[s], self.length[s] = [], 0
        return wrong

    def compact(self):
        used = sum(r != 0 for r in self.refs)
        movers = [p for p in range(used, self.pages) if self.refs[p]]
        holes = [p for p in range(used) if not self.refs[p]]
        to = dict(zip(movers, holes))
        for a, b in to.items():
            self.refs[b], self.refs[a] = self.refs[a], 0
        self.held = [[to.get(p, p) for p in h] for h in self.held]
        return used, list(to.items())


class Device:
    def __init__(self, ctx, m, planes=3, page_bytes=48, seed=0):
        self.ctx, self.m = ctx, m
        z = lambda *s: torch.zeros(s, dtype=torch.int32, device="cuda")  # noqa: E731
        self.refs, self.tables, self.lengths = z(m.pages), z(m.slots, m.table_len), z(m.slots)
        self.pool = capi.PagePool(self.refs, self.tables, self.lengths, m.page)
        g = torch.Generator().manual_seed(seed)
        self.want = torch.randint(0, 256, (planes, m.pages, page_bytes), dtype=torch.uint8,
                                  generator=g)
        self.data = [p.clone().cuda() for p in self.want]
        self.planes = capi.PagePlanes(self.data)
        self.work, self.used = z(m.pages), z(1)

    def sync(self, wrong=()):
        torch.cuda.synchronize()
        try:
            self.ctx.sync()
            said = None
        except capi.B200W4Error as e:
            said = str(e)
        if not wrong:
            assert said is None, said
        else:
            assert said and any(w in said for w in wrong), (said, wrong)

    def copied(self, pairs):
        for a, b in pairs:
            self.want[:, b] = self.want[:, a]

    def check(self):
        m = self.m
        assert self.refs.cpu().tolist() == m.refs
        assert self.lengths.cpu().tolist() == m.length
        tables = self.tables.cpu().tolist()
        for s in range(m.slots):
            assert tables[s][:len(m.held[s])] == m.held[s], s
        for p, want in zip(self.data, self.want):
            assert torch.equal(p.cpu(), want)


@pytest.mark.parametrize("pages,page,slots,table_len,page_bytes,seed", [
    (40, 4, 6, 12, 16, 1), (5, 1, 4, 5, 48, 2), (300, 16, 9, 40, 8192 * 5 + 16, 3),
    (20000, 3, 30, 900, 16, 4), (64, 7, 12, 9, 32784, 5)])
def test_random_histories(ctx, pages, page, slots, table_len, page_bytes, seed):
    rng = random.Random(seed)
    m = Model(pages, page, slots, table_len)
    d = Device(ctx, m, 2 if page_bytes > 9999 else 3, page_bytes, seed)
    for step in range(60):
        what = rng.choice(["extend", "extend", "extend", "fork", "free", "compact"])
        if what == "extend":
            some = rng.sample(range(slots), rng.randint(1, slots))
            counts = [rng.choice([0, 1, page, rng.randint(0, 3 * page * table_len // 8)])
                      for _ in some]
            if rng.random() < 0.2:
                some[-1] = rng.choice([-1, slots, some[0]])
            granted = ints([-9] * (len(some) + 1))
            before = list(m.length)
            d.ctx.pages_extend(d.pool, ints(some), ints(counts), granted)
            wrong = m.extend(some, counts)
            for i, (s, c) in enumerate(zip(some, counts)):
                if s in some[:i] or not 0 <= s < slots:
                    assert granted[i] == -1
                elif c:
                    assert granted[i] == (s if m.length[s] != before[s] else -1)
            assert granted[-1] == -9
        elif what == "fork":
            parents = [rng.randrange(slots) for _ in range(rng.randint(1, slots))]
            children = [rng.randrange(-1, slots) for _ in parents]
            parents[0] = rng.choice([parents[0], -1])
            d.ctx.pages_fork(d.pool, d.planes, ints(parents), ints(children))
            wrong, copies = m.fork(parents, children)
            d.copied(copies)
        elif what == "free":
            some = [rng.randrange(slots) for _ in range(rng.randint(1, slots // 2))]
            if rng.random() < 0.2:
                some.append(rng.choice([slots, -1]))
            d.ctx.pages_free(d.pool, ints(some))
            wrong = m.free(some)
        else:
            d.ctx.pages_compact(d.pool, d.planes, d.work, d.used)
            used, moves = m.compact()
            wrong = set()
            d.copied(moves)
            assert int(d.used) == used
        d.sync(wrong)
        d.check()


def test_every_slot_by_default(ctx):
    m = Model(30, 4, 5, 6)
    d = Device(ctx, m)
    for _ in range(6):
        d.ctx.pages_extend(d.pool)
        m.extend(range(5), [1] * 5)
    d.ctx.pages_extend(d.pool, counts=ints([0, 3, 0]))
    m.extend(range(3), [0, 3, 0])
    d.sync()
    d.check()
    d.ctx.pages_free(d.pool)
    m.free(range(5))
    d.sync()
    d.check()


def test_a_thousand_sequences(ctx):
    m = Model(9000, 2, 1100, 8)
    d = Device(ctx, m)
    rng = random.Random(3)
    slots, counts = rng.sample(range(1100), 512), [rng.randint(0, 15) for _ in range(512)]
    d.ctx.pages_extend(d.pool, ints(slots), ints(counts))
    assert not m.extend(slots, counts)
    rest = [s for s in range(1100) if m.length[s] == 0][:1024]
    parents = [rng.choice(slots) for _ in rest]
    d.ctx.pages_fork(d.pool, d.planes, ints(parents), ints(rest))
    wrong, copies = m.fork(parents, rest)
    assert not wrong
    d.copied(copies)
    d.sync()
    d.check()
    d.ctx.pages_free(d.pool, ints(slots + slots))  # the same slot twice
    m.free(slots)
    d.ctx.pages_compact(d.pool, d.planes, d.work)
    _, moves = m.compact()
    d.copied(moves)
    d.sync()
    d.check()


def test_three_hundred_planes_and_odd_pages(ctx):
    """More planes than a launch takes, pages that end inside a block's piece."""
    m = Model(9, 4, 3, 4)
    d = Device(ctx, m, planes=300, page_bytes=16 * 2048 + 16)
    d.ctx.pages_extend(d.pool, ints([0]), ints([13]))
    m.extend([0], [13])
    d.ctx.pages_fork(d.pool, d.planes, ints([0, 0]), ints([2, 1]))
    d.copied(m.fork([0, 0], [2, 1])[1])
    d.ctx.pages_free(d.pool, ints([0]))
    m.free([0])
    d.ctx.pages_copy(d.planes, ints([8, 5, 5]), ints([7, 6, 5]))
    d.copied([(8, 7), (5, 6)])
    d.ctx.pages_compact(d.pool, d.planes, d.work, d.used)
    d.copied(m.compact()[1])
    d.sync()
    d.check()


def test_bad_pages_of_a_copy_are_left_out(ctx):
    m = Model(6, 4, 2, 2)
    d = Device(ctx, m)
    d.ctx.pages_copy(d.planes, ints([0, 6, 1, -1]), ints([3, 4, 1 << 30, 5]))
    d.copied([(0, 3)])
    d.sync({"outside"})
    d.check()


def test_steps_are_replayed_across_page_borders(ctx):
    m = Model(50, 4, 5, 10)
    d = Device(ctx, m)
    d.ctx.pages_extend(d.pool, ints([0, 2, 4]), ints([3, 9, 4]))
    m.extend([0, 2, 4], [3, 9, 4])
    live = ints([1, 0, 1, 0, 1])
    d.ctx.pages_extend(d.pool, counts=live)  # the kernel is loaded outside the capture
    m.extend(range(5), [1, 0, 1, 0, 1])
    torch.cuda.synchronize()
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        ctx.set_stream(side.cuda_stream)
        with torch.cuda.graph(graph, stream=side):
            d.ctx.pages_extend(d.pool, counts=live)
    ctx.set_stream(0)
    for _ in range(11):
        graph.replay()
        m.extend(range(5), [1, 0, 1, 0, 1])
    d.sync()
    d.check()


def test_refusals(ctx):
    m = Model(6, 4, 3, 2)
    d = Device(ctx, m)
    launches = ctx.launches
    few = [p[:3] for p in d.data]
    for call in (lambda: ctx.pages_extend(d.pool, ints([0] * 1025)),
                 lambda: ctx.pages_extend(d.pool, counts=ints([0] * 4)),
                 lambda: ctx.pages_fork(d.pool, d.planes, ints([0] * 1025), ints([1] * 1025)),
                 lambda: ctx.pages_fork(d.pool, capi.PagePlanes(few), ints([0]), ints([1])),
                 lambda: ctx.pages_free(d.pool, ints([])),
                 lambda: ctx.pages_compact(d.pool, capi.PagePlanes(few), d.work),
                 lambda: ctx.pages_copy(capi.PagePlanes([p[:, :8].contiguous() for p in d.data]),
                                        ints([0]), ints([1])),
                 lambda: ctx.pages_copy(d.planes, ints([]), ints([]))):
        with pytest.raises(capi.B200W4Error):
            call()
    for call in (lambda: ctx.pages_compact(d.pool, d.planes, d.work[:5]),
                 lambda: ctx.pages_fork(d.pool, d.planes, ints([0, 1]), ints([1])),
                 lambda: ctx.pages_extend(d.pool, ints([0, 1]), ints([1]))):
        with pytest.raises(ValueError):
            call()
    assert ctx.launches == launches
    d.check()


def test_demands_whose_sum_passes_32_bits(ctx):
    """1024 sequences that ask for 2^21 + 1 pages each of a pool of 16: none gets one."""
    each = 2 ** 21 + 1
    pool = capi.PagePool(ints([0] * 16), torch.empty((1024, each), dtype=torch.int32, device="cuda"),
                         ints([0] * 1024), 1)
    granted = ints([7] * 1024)
    ctx.pages_extend(pool, counts=ints([0] + [each] * 1022 + [1]), granted=granted)
    with pytest.raises(capi.B200W4Error, match="out of pages"):
        ctx.sync()
    refs, _, lengths = pool.keep
    assert granted.tolist() == [0] + [-1] * 1023
    assert int(lengths.abs().sum()) == 0 and int(refs.abs().sum()) == 0


def test_a_pool_of_too_many_pages_is_refused(ctx):
    one = ints([0])
    pool = capi.PagePool(one, one.view(1, 1), one, 1)
    pool.pages = 2 ** 30
    with pytest.raises(capi.B200W4Error, match="2.30"):
        ctx.pages_free(pool)
