"""The page cache on the GPU against the same operations on lists."""
import random

import pytest
import torch

import thrust_amd
from lm_util import get, put

pytestmark = pytest.mark.gpu


class Lists:
    """The definitions: one request after the other, one page after the other."""

    def __init__(self, pools, page_size, tables, lengths, refs):
        self.size, self.most = page_size, tables.shape[1]
        self.pools = [p.clone() for p in pools]
        self.tables = tables.tolist()
        self.lengths, self.refs = lengths.tolist(), refs.tolist()

    def held(self, n):
        return -(-n // self.size)

    def copy(self, pairs):
        for pool in self.pools:
            old = pool.clone()
            for a, b in pairs:
                pool[b] = old[a]

    def valid(self, s):
        return 0 <= s < len(self.lengths)

    def free(self, sequences):
        self.resize(sequences, [0] * len(sequences), free_only=True)

    def resize(self, sequences, lengths, free_only=False):
        n = len(sequences)
        ok = [self.valid(s) and 0 <= want <= self.most * self.size and s not in sequences[:i] for i, (s, want) in enumerate(zip(sequences, lengths))]
        for i in range(n):
            s = sequences[i]
            if ok[i] and lengths[i] < self.lengths[s]:
                for j in range(self.held(lengths[i]), self.held(self.lengths[s])):
                    if 0 <= self.tables[s][j] < len(self.refs):
                        self.refs[self.tables[s][j]] -= 1
                    self.tables[s][j] = -1
                self.lengths[s] = lengths[i]
        if free_only:
            return ok
        free = [p for p, r in enumerate(self.refs) if r == 0]
        at, copies, refs = 0, [], list(self.refs)
        for i in range(n):
            if not ok[i]:
                continue
            s, want = sequences[i], lengths[i]
            had, have = self.held(self.lengths[s]), self.held(want)
            if want <= self.lengths[s]:
                continue
            last = self.tables[s][self.lengths[s] // self.size] if self.lengths[s] % self.size else -1
            own = 0 <= last < len(refs) and refs[last] > 1
            need = have - had + own
            mine = free[at:at + need]
            at += need
            if len(mine) < need:
                ok[i] = False
                continue
            if own:
                copies.append((last, mine[0]))
                self.refs[last] -= 1
                self.refs[mine[0]] = 1
                self.tables[s][self.lengths[s] // self.size] = mine[0]
                mine = mine[1:]
            for j, p in enumerate(mine):
                self.tables[s][had + j] = p
                self.refs[p] = 1
            self.lengths[s] = want
        self.copy(copies)
        return ok

    def fork(self, parents, children, share):
        free = [p for p, r in enumerate(self.refs) if r == 0]
        at, copies, ok, before = 0, [], [], list(self.lengths)
        for i, (p, c) in enumerate(zip(parents, children)):
            good = self.valid(p) and self.valid(c) and before[c] == 0 and c not in children[:i] and c not in parents
            if good:
                n = self.lengths[p]
                held = self.held(n)
                need = (1 if n % self.size else 0) if share else held
                mine = free[at:at + need]
                at += need
                good = len(mine) == need
                if good:
                    for j in range(held):
                        q = self.tables[p][j]
                        if j < held - need:
                            if 0 <= q < len(self.refs):
                                self.refs[q] += 1
                        else:
                            new = mine[j - held + need]
                            if 0 <= q < len(self.refs):
                                copies.append((q, new))
                            q = new
                            self.refs[q] = 1
                        self.tables[c][j] = q
                    self.lengths[c] = n
            ok.append(good)
        self.copy(copies)
        return ok

    def compact(self):
        live = sum(r > 0 for r in self.refs)
        holes = [p for p in range(live) if self.refs[p] == 0]
        high = [p for p in range(len(self.refs) - 1, live - 1, -1) if self.refs[p] > 0]
        self.copy(list(zip(high, holes)))
        names = dict(zip(high, holes))
        for a, b in names.items():
            self.refs[b], self.refs[a] = self.refs[a], 0
        self.tables = [[names.get(q, q) if 0 <= q < len(self.refs) else -1 for q in row] for row in self.tables]
        return live


def ints(v):
    return put(torch.tensor(v, dtype=torch.int32))


def make(pages, shapes, page_size, sequences, most, seed=1, unaligned=False):
    g = torch.Generator().manual_seed(seed)
    pools = []
    for shape, dtype in shapes:
        v = torch.randint(-100, 100, (pages,) + shape, generator=g).to(dtype)
        pools.append(v)
    on = [put(torch.cat([v.flatten()[:1], v.flatten()]))[1:].view(v.shape) if unaligned else put(v) for v in pools]
    cache = thrust_amd.PageCache(on, page_size, sequences, most)
    return cache, Lists(pools, page_size, get(cache.tables), get(cache.lengths), get(cache.refs))


def same(cache, ref):
    assert get(cache.tables).tolist() == ref.tables
    assert get(cache.lengths).tolist() == ref.lengths
    assert get(cache.refs).tolist() == ref.refs
    for a, b in zip(cache.pools, ref.pools):
        assert torch.equal(get(a), b)


POOLS = {
    "states": [((5,), torch.float32)] * 3,
    "keys and values": [((4, 2, 8), torch.bfloat16)] * 4,
    "odd bytes": [((13,), torch.int8)] * 2,
    "one byte": [((1,), torch.uint8)],
    "over a copy unit": [((4100, 1), torch.float32), ((2, 2050), torch.int32)],
    "no bytes": [((0,), torch.float32)],
}


@pytest.mark.parametrize("pools", list(POOLS), ids=str)
@pytest.mark.parametrize("page_size,most,unaligned", [(16, 6, False), (1, 9, True), (1 << 20, 1, False), (7, 4, True)])
def test_life_of_a_cache(pools, page_size, most, unaligned):
    """Random requests, valid and not, until pages have run out and come back many times."""
    rng = random.Random(len(pools) * 100 + page_size)
    pages, sequences = (23, 11) if pools == "over a copy unit" else (70, 25)
    cache, ref = make(pages, POOLS[pools], page_size, sequences, most, unaligned=unaligned)
    cap, refused, copied = page_size * most, 0, 0
    for turn in range(8 if pools == "over a copy unit" else 30):
        n = rng.choice([1, 2, 5, 9])
        ids = [rng.randrange(sequences) for _ in range(n)]
        if rng.random() < 0.5:
            ids[0] = rng.choice([-1, sequences, 2 ** 31 - 1, -2 ** 31, ids[-1]])
        what = rng.choice(["resize", "resize", "resize", "fork", "fork", "copy", "free", "compact"])
        if what == "resize":
            lengths = [rng.choice([rng.randint(0, cap), min(cap, ref.lengths[s] + 1) if 0 <= s < sequences else 3]) for s in ids]
            if rng.random() < 0.2:
                lengths[-1] = rng.choice([-1, cap + 1, -2 ** 31, 2 ** 31 - 1])
            done = get(cache.resize(ints(ids), ints(lengths))).tolist()
            assert done == ref.resize(ids, lengths)
            refused += not all(done)
        elif what in ("fork", "copy"):
            empty = [s for s in range(sequences) if ref.lengths[s] == 0]
            rng.shuffle(empty)
            children = (empty + ids)[:n]
            used = [s for s in range(sequences) if ref.lengths[s]] or [0]
            parents = [rng.choice(used + [rng.randrange(-1, sequences + 1)]) for _ in range(n)]
            done = get(cache.fork(ints(parents), ints(children), share=what == "fork")).tolist()
            assert done == ref.fork(parents, children, what == "fork")
            copied += any(done)
        elif what == "free":
            cache.free(ints(ids))
            ref.free(ids)
        else:
            assert get(cache.compact()).tolist() == [ref.compact()]
        same(cache, ref)
    assert sum(r > 0 for r in ref.refs) == len({q for row in ref.tables for q in row if q >= 0})


def test_fork_shares_full_pages_and_growth_copies_a_shared_one():
    cache, ref = make(20, [((16, 2), torch.float32)], 16, 6, 4)
    for c in (cache, ref):
        c.resize(*((ints(v) if c is cache else v) for v in ([0], [40])))
    assert get(cache.tables)[0].tolist() == [0, 1, 2, -1]
    cache.fork(ints([0, 0]), ints([1, 2]))
    ref.fork([0, 0], [1, 2], True)
    same(cache, ref)
    assert get(cache.refs)[:5].tolist() == [3, 3, 1, 1, 1]
    # cut back into a shared page: it is copied when the sequences grow again, in the order of the requests
    for ids, lengths in (([0, 1, 2], [20, 20, 20]), ([1, 0], [21, 33])):
        assert get(cache.resize(ints(ids), ints(lengths))).tolist() == ref.resize(ids, lengths) == [True] * len(ids)
        same(cache, ref)
    assert get(cache.tables)[:3, :2].tolist() == [[0, 3], [0, 2], [0, 1]] and get(cache.refs)[1] == 1


def test_requests_are_served_in_order_and_whole():
    cache, ref = make(10, [((3,), torch.float32)], 4, 5, 8)
    ids, lengths = [3, 1, 0, 4], [13, 30, 9, 8]  # 4, 8, 3, 2 pages: what all requests up to one want counts
    done = get(cache.resize(ints(ids), ints(lengths))).tolist()
    assert done == ref.resize(ids, lengths) == [True, False, False, False]
    same(cache, ref)
    assert get(cache.resize(ints([1, 3]), ints([24, 0]))).tolist() == [True, True]  # pages given up in the call count
    assert get(cache.tables)[1].tolist() == [0, 1, 2, 3, 4, 5, -1, -1]
    assert get(cache.fork(ints([1, 1]), ints([0, 1]), share=False)).tolist() == [False, False]  # 4 pages for 6; not empty
    assert get(cache.refs).tolist() == [1] * 6 + [0] * 4


def test_tables_that_name_no_page():
    tables = torch.tensor([[5, 99, -7, 2], [-1, -1, -1, -1], [1, 2 ** 31 - 1, -2 ** 31, 9]], dtype=torch.int32)
    lengths = torch.tensor([15, 0, 13], dtype=torch.int32)
    refs = torch.tensor([0, 1, 1, 0, 0, 1, 0, 0, 0, 1, 0, 0], dtype=torch.int32)
    for op in range(4):
        pools = [torch.arange(36.0).view(12, 3)]
        cache = thrust_amd.PageCache([put(pools[0])], 4, 3, 4, tables=put(tables), lengths=put(lengths), refs=put(refs))
        ref = Lists(pools, 4, tables, lengths, refs)
        if op < 2:
            assert get(cache.fork(ints([0]), ints([1]), share=op == 0)).tolist() == ref.fork([0], [1], op == 0)
        elif op == 2:
            assert get(cache.resize(ints([2, 0]), ints([14, 2]))).tolist() == ref.resize([2, 0], [14, 2])
        else:
            assert get(cache.compact()).tolist() == [ref.compact()]
        same(cache, ref)


def test_lengths_out_of_range_are_taken_as_the_nearest():
    pools = [torch.arange(24.0).view(8, 3)]
    tables = torch.tensor([[0, 1], [2, -1], [-1, -1]], dtype=torch.int32)
    refs = torch.tensor([1, 1, 1, 0, 0, 0, 0, 0], dtype=torch.int32)
    cache = thrust_amd.PageCache([put(pools[0])], 4, 3, 2, tables=put(tables), lengths=ints([2 ** 31 - 1, -5, 0]), refs=put(refs))
    assert get(cache.fork(ints([0, 1]), ints([2, 1]))).tolist() == [True, False]  # -5 is not empty, as a child
    assert get(cache.tables).tolist() == [[0, 1], [2, -1], [0, 1]] and get(cache.lengths).tolist() == [2 ** 31 - 1, -5, 8]
    cache.free(ints([0]))
    assert get(cache.refs).tolist() == [1, 1, 1, 0, 0, 0, 0, 0]


@pytest.mark.parametrize("pages", [1, 2047, 2048, 2049, 10000])
@pytest.mark.parametrize("live", [0.0, 0.3, 0.97, 1.0])
def test_compact_many_pages(pages, live):
    g = torch.Generator().manual_seed(pages)
    refs = (torch.rand(pages, generator=g) < live).int() * torch.randint(1, 4, (pages,), generator=g).int()
    used = refs.nonzero().flatten().int()
    sequences, most = 37, 50
    tables = torch.full((sequences, most), -1, dtype=torch.int32)
    if len(used):
        tables = used[torch.randint(0, len(used), (sequences, most), generator=g)]
    lengths = torch.full((sequences,), most, dtype=torch.int32)
    pool = torch.arange(pages * 2).view(pages, 2)
    ref = Lists([pool], 1, tables, lengths, refs)
    n = ref.compact()
    apart = thrust_amd.PageCache([put(pool)], 1, sequences, most, tables=put(tables), lengths=put(lengths), refs=put(refs))
    new_tables, new_refs = put(torch.zeros_like(tables)), put(torch.full_like(refs, 77))
    assert get(apart.compact(tables=new_tables, refs=new_refs)).tolist() == [n]
    assert get(new_tables).tolist() == ref.tables and get(new_refs).tolist() == ref.refs and torch.equal(get(apart.pools[0]), ref.pools[0])
    assert torch.equal(get(apart.tables), tables) and torch.equal(get(apart.refs), refs)  # the old ones stand ...
    old = pool[tables.long().clamp(min=0)]
    moved = torch.isin(tables, torch.arange(n, dtype=torch.int32), invert=True)
    assert torch.equal(get(apart.pools[0])[tables.long().clamp(min=0)][moved], old[moved])  # ... and so does what they name
    here = thrust_amd.PageCache([put(pool)], 1, sequences, most, tables=put(tables), lengths=put(lengths), refs=put(refs))
    assert get(here.compact()).tolist() == [n]
    same(here, ref)


@pytest.mark.parametrize("requests", [300, 1100])
def test_fork_and_resize_many_requests(requests):
    sequences = 2 * requests
    cache, ref = make(3 * requests + 50, [((1,), torch.int32)], 4, sequences, 3)
    rng = random.Random(requests)
    ids = list(range(sequences))
    rng.shuffle(ids)
    lengths = [rng.randint(0, 12) for _ in range(requests)]
    first, second = ids[:requests], ids[requests:]
    for call in range(3):
        if call == 0:
            a, b = get(cache.resize(ints(first), ints(lengths))).tolist(), ref.resize(first, lengths)
        elif call == 1:
            a, b = get(cache.fork(ints(first), ints(second))).tolist(), ref.fork(first, second, True)
        else:
            a, b = get(cache.resize(ints(ids), ints([2] * sequences))).tolist(), ref.resize(ids, [2] * sequences)
        assert a == b
        same(cache, ref)


def test_nothing_to_do():
    cache, ref = make(0, [((3,), torch.float32)], 4, 3, 2)
    assert get(cache.resize(ints([0, 1]), ints([0, 1]))).tolist() == [True, False]
    assert get(cache.fork(ints([0]), ints([1]))).tolist() == [True]
    assert get(cache.compact()).tolist() == [0]
    cache, ref = make(5, [((3,), torch.float32)], 4, 3, 2)
    none = put(torch.zeros(0, dtype=torch.int32))
    assert get(cache.resize(none, none)).tolist() == [] and get(cache.fork(none, none)).tolist() == []
    cache.free(none)
    assert get(cache.compact()).tolist() == [0]
    same(cache, ref)
    cache, ref = make(5, [((3,), torch.float32)], 4, 0, 0)
    assert get(cache.resize(ints([0]), ints([1]))).tolist() == [False]
    assert get(cache.compact()).tolist() == [0]


def test_states_of_a_recurrence_in_a_cache():
    """Prompts are scanned, their last states kept in pages, sequences forked and continued token by token, closed up in between: the
    outputs are those of one scan over each whole sequence."""
    channels, prompts, tokens = 132, [5, 1, 70], 6
    g = torch.Generator().manual_seed(5)
    pool = put(torch.zeros(9, channels))
    cache = thrust_amd.PageCache([pool], 1 << 20, 5, 1)

    def rows(n):
        return torch.rand(n, channels, generator=g).bfloat16(), torch.randn(n, channels, generator=g).bfloat16()
    gate, x = rows(sum(prompts))
    offsets = torch.tensor([0] + prompts).cumsum(0).int()
    # a page that is given back leaves a hole for the compaction
    assert get(cache.resize(ints([4, 0, 1, 2]), ints([1] + prompts))).all()
    cache.free(ints([4]))
    out, final = thrust_amd.linear_scan(put(gate), put(x), offsets=put(offsets))
    pool[cache.tables[:3, 0].long()] = final
    histories = [[gate[a:b], x[a:b]] for a, b in zip(offsets[:-1].tolist(), offsets[1:].tolist())]
    assert get(cache.fork(ints([2, 2]), ints([3, 4]))).all()
    histories += [[v.clone() for v in histories[2]] for _ in range(2)]
    got = [[] for _ in range(5)]
    for t in range(tokens):
        if t == 3:
            assert get(cache.compact()).tolist() == [5]
        gate, x = rows(5)
        slots = cache.tables[:, 0].contiguous()
        assert t < 3 or sorted(get(slots).tolist()) == list(range(5))
        step = get(thrust_amd.linear_scan_step(put(gate), put(x), pool, slots=slots))
        for s in range(5):
            histories[s] = [torch.cat([a, b[s:s + 1]]) for a, b in zip(histories[s], (gate, x))]
            got[s].append(step[s])
    for s in range(5):
        want, final = thrust_amd.linear_scan(put(histories[s][0][None]), put(histories[s][1][None]))
        tail = get(want)[0, -tokens:].float()
        # both are within the bound of a 32-bit sum of the exact value, then rounded: at most one step apart, relative to the
        # largest value that the sum of at most 76 terms below 5 can have met (1e-3 absolute covers 2 * 80 roundings of 2^-24 * 100)
        assert ((torch.stack(got[s]).float() - tail).abs() <= torch.finfo(torch.bfloat16).eps * tail.abs() + 1e-3).all()


@pytest.mark.needs_device
def test_requests_in_a_graph():
    cache, ref = make(400, [((64,), torch.float32)] * 2, 4, 40, 12)
    ids, lengths = put(torch.arange(10).int()), put(torch.full((10,), 9).int())
    parents, children = put(torch.zeros(5).int()), put(torch.arange(20, 25).int())

    def one():
        cache.free(children)
        done = cache.resize(ids, lengths)
        forked = cache.fork(parents, children)
        return done, forked, cache.compact()
    one()
    cache.free(put(torch.arange(40).int()))
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        outs = one()
    ref.pools = [get(p) for p in cache.pools]
    rng = random.Random(2)
    for r in range(5):
        a = rng.sample(range(20), 10)
        b = [rng.randint(0, 48) for _ in range(10)]
        p = [rng.choice(a) for _ in range(5)]
        ids.copy_(torch.tensor(a).int())
        lengths.copy_(torch.tensor(b).int())
        parents.copy_(torch.tensor(p).int())
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        ref.free(list(range(20, 25)))
        want = ref.resize(a, b), ref.fork(p, list(range(20, 25)), True), [ref.compact()]
        assert [get(o).tolist() for o in outs] == list(want)
        same(cache, ref)


@pytest.mark.needs_device
def test_two_caches_on_two_streams():
    pairs = [make(9000 if k else 300, [((64,), torch.float32)] * 3, 4, 200, 10, seed=k) for k in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    ids, lengths = list(range(100)), [(7 * i) % 41 for i in range(100)]
    parents, children = list(range(0, 60, 3)), list(range(100, 120))
    t = [ints(v) for v in (ids, lengths, parents, children, ids[:50])]
    torch.cuda.synchronize()
    for _ in range(3):
        for (cache, _), stream in zip(pairs, streams):
            with torch.cuda.stream(stream):
                cache.resize(t[0], t[1])
                cache.fork(t[2], t[3])
                cache.free(t[4])
                cache.compact()
    torch.cuda.synchronize()
    for cache, ref in pairs:
        for _ in range(3):
            ref.resize(ids, lengths)
            ref.fork(parents, children, True)
            ref.free(ids[:50])
            ref.compact()
        same(cache, ref)


@pytest.mark.needs_device
def test_pools_past_4_gib():
    pages, width = 70000, 20000  # 5.6 GB of float32
    pool = torch.zeros((pages, width), device="cuda")
    refs = torch.zeros(pages, dtype=torch.int32, device="cuda")
    cache = thrust_amd.PageCache([pool], 1 << 20, 4, 1, refs=refs)
    refs[: pages - 1] = 1  # of no table: only the last page is free
    assert get(cache.resize(ints([0]), ints([3]))).all()
    assert get(cache.tables)[0, 0] == pages - 1
    pool[pages - 1] = torch.arange(width, device="cuda").float()
    refs[5:pages - 1] = 0
    assert get(cache.fork(ints([0]), ints([1]))).all() and get(cache.tables)[1, 0] == 5
    assert get(cache.compact()).tolist() == [7]
    assert get(cache.tables)[:2, 0].tolist() == [6, 5]
    want = torch.arange(width).float()
    assert torch.equal(get(pool[5]), want) and torch.equal(get(pool[6]), want)


# ---------------------------------------------------------------------------------------
# Growth into pages that are shared, request after request
# ---------------------------------------------------------------------------------------
class InOrder(Lists):
    """As Lists, with the counts as the requests before left them: who is alone with its page when its turn comes keeps it."""

    def resize(self, sequences, lengths, free_only=False):
        ok = super().resize(sequences, [min(a, self.lengths[s]) if self.valid(s) and a >= 0 else a for s, a in zip(sequences, lengths)], free_only)
        if free_only:
            return ok
        free, at, copies = [p for p, r in enumerate(self.refs) if r == 0], 0, []
        for i, (s, want) in enumerate(zip(sequences, lengths)):
            ok[i] = ok[i] and want <= self.most * self.size
            if not ok[i] or want <= self.lengths[s]:
                continue
            had, part = self.held(self.lengths[s]), self.lengths[s] % self.size
            last = self.tables[s][had - 1] if part else -1
            own = 0 <= last < len(self.refs) and self.refs[last] > 1
            need = self.held(want) - had + own
            mine = free[at:at + need]
            at += need
            if len(mine) < need:
                ok[i] = False
                continue
            if own:
                copies.append((last, mine[0]))
                self.refs[last] -= 1
                self.refs[mine[0]] = 1
                self.tables[s][had - 1] = mine.pop(0)
            for j, p in enumerate(mine):
                self.tables[s][had + j], self.refs[p] = p, 1
            self.lengths[s] = want
        self.copy(copies)
        return ok


def shared(pages, sequences, page_size, most, groups, unused=0):
    """A cache in which the sequences of a group share the first pages of its first one, cut back into the last of them."""
    cache, ref = make(pages, [((page_size, 3), torch.float32), ((page_size, 3), torch.int32)], page_size, sequences, most)
    ref.__class__ = InOrder
    for members, full, keep in groups:
        for c, v in ((cache, ints), (ref, lambda x: x)):
            c.resize(v(members[:1]), v([full * page_size]))
            for k in range(1, len(members)):
                if c is cache:
                    c.fork(v(members[:1]), v(members[k:k + 1]))
                else:
                    c.fork(members[:1], members[k:k + 1], True)
            c.resize(v(members), v([keep] * len(members)))
    same(cache, ref)
    return cache, ref


def test_the_last_of_those_that_grow_keeps_the_page():
    cache, ref = shared(3, 2, 4, 2, [([0, 1], 2, 6)])
    assert get(cache.resize(ints([0, 1]), ints([7, 7]))).tolist() == [True, True] == ref.resize([0, 1], [7, 7])
    assert get(cache.tables).tolist() == [[0, 2], [0, 1]] and get(cache.refs).tolist() == [2, 1, 1]
    same(cache, ref)
    # one that does not grow keeps it too; of three that grow two are given copies
    cache, ref = shared(9, 4, 4, 4, [([2, 0, 3, 1], 1, 3)])
    assert get(cache.resize(ints([3, 0, 1]), ints([4, 9, 1]))).tolist() == [True] * 3 == ref.resize([3, 0, 1], [4, 9, 1])
    same(cache, ref)
    assert get(cache.refs).tolist() == [2, 1, 1, 1, 1, 0, 0, 0, 0]
    assert get(cache.resize(ints([1, 2]), ints([5, 4]))).tolist() == [True] * 2 == ref.resize([1, 2], [5, 4])
    same(cache, ref)


def test_a_page_is_not_kept_where_one_before_was_refused():
    # sequence 0 would leave the page but finds no copy: sequence 1 still shares it and is refused too, 4 is served
    groups = [([0, 1], 1, 2), ([2], 2, 8), ([3], 1, 4), ([4], 1, 1)]
    cache, ref = shared(5, 5, 4, 4, groups)
    assert get(cache.resize(ints([0, 1, 4]), ints([3, 3, 2]))).tolist() == [False, False, True] == ref.resize([0, 1, 4], [3, 3, 2])
    same(cache, ref)
    # an unrelated request between them is refused: the second of the two keeps the page all the same
    cache, ref = shared(6, 5, 4, 4, groups)
    for c, v in ((cache, ints), (ref, list)):
        done = c.resize(v([0, 3, 1, 4, 2]), v([3, 9, 3, 4, 8]))
        assert (get(done).tolist() if c is cache else done) == [True, False, True, True, True]
    same(cache, ref)
    # it wants pages besides: refused with the rest
    cache, ref = shared(7, 5, 4, 4, groups)
    for c, v in ((cache, ints), (ref, list)):
        done = c.resize(v([0, 1, 3]), v([3, 16, 5]))
        assert (get(done).tolist() if c is cache else done) == [True, False, False]
    same(cache, ref)


@pytest.mark.parametrize("pages,sequences,requests", [(60, 24, 20), (400, 150, 64), (400, 150, 65), (700, 300, 290), (9000, 60, 50)], ids=str)
def test_many_that_grow_into_shared_pages(pages, sequences, requests):
    rng = random.Random(requests)
    size, most = 4, 6
    for turn in range(4):
        ids, groups = list(range(sequences)), []
        rng.shuffle(ids)
        room = pages // 2
        while ids and room >= 5:
            members = [ids.pop() for _ in range(min(len(ids), rng.choice([1, 2, 3, 9, 40])))]
            full = rng.randint(1, 4)
            groups.append((members, full, rng.randint(1, full * size)))
            room -= full
        cache, ref = shared(pages, sequences, size, most, groups)
        if turn % 2:  # few pages are left
            spare = ref.refs.count(0) - rng.randint(0, sequences // 2)
            for c in (cache.refs, None):
                held = [p for p, r in enumerate(ref.refs) if r == 0][:spare]
                if c is not None:
                    c[put(torch.tensor(held, dtype=torch.int64))] = 1
            for p in held:
                ref.refs[p] = 1
        names = rng.sample(range(sequences), min(requests, sequences))
        names[0], names[-1] = names[-1], names[1]  # one twice
        lengths = [max(0, min(size * most + 1, ref.lengths[s] + rng.choice([0, 1, 1, 1, 1, 2, 7, -3]))) for s in names]
        done = get(cache.resize(ints(names), ints(lengths))).tolist()
        assert done == ref.resize(names, lengths)
        same(cache, ref)


def test_torch_is_told_what_is_written():
    cache, _ = make(9, POOLS["keys and values"], 4, 5, 3)
    own = [cache.tables, cache.lengths, cache.refs]

    def written(call, tensors, kept=()):
        was = [t._version for t in tensors], [t._version for t in kept]
        call()
        assert all(t._version > a for t, a in zip(tensors, was[0])) and [t._version for t in kept] == was[1]
    written(lambda: cache.resize(ints([0, 1]), ints([5, 6])), own + cache.pools)
    written(lambda: cache.fork(ints([0]), ints([2])), own + cache.pools)
    written(lambda: cache.free(ints([1])), own, cache.pools)
    written(lambda: cache.compact(), [cache.tables, cache.refs] + cache.pools, [cache.lengths])
    apart = [put(torch.zeros_like(get(t))) for t in (cache.tables, cache.refs)]
    written(lambda: cache.compact(*apart), apart + cache.pools, own)
    with torch.inference_mode():  # tensors without a version
        cache, _ = make(9, POOLS["keys and values"], 4, 5, 3)
    cache.resize(ints([0, 1]), ints([5, 6]))


@pytest.mark.needs_device
def test_a_cache_that_is_dropped_under_a_pending_call():
    """The addresses of its pools are in memory of its own, which no other tensor gets before the call has read it."""
    stream, tables = torch.cuda.Stream(), []
    for _ in range(3):
        cache, ref = make(40, [((64,), torch.float32)] * 3, 4, 8, 5)
        pools, rows, a, b, ids, lengths = cache.pools, cache.tables, ints([0]), ints([1]), ints([0]), ints([7])
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            torch.cuda._sleep(50_000_000)  # tens of milliseconds
            cache.resize(ids, lengths)
            cache.fork(a, b, share=False)
        where = cache._pointers.tensor.data_ptr()
        keep = [cache.lengths, cache.refs]
        del cache
        others = [torch.zeros(3, dtype=torch.int64, device="cuda") for _ in range(64)]
        assert not stream.query()
        assert all(t.data_ptr() != where for t in others)
        torch.cuda.synchronize()
        ref.resize([0], [7])
        ref.fork([0], [1], False)
        assert get(rows).tolist() == ref.tables and get(keep[0]).tolist() == ref.lengths and get(keep[1]).tolist() == ref.refs
        assert all(torch.equal(get(p), q) for p, q in zip(pools, ref.pools))


@pytest.mark.needs_device
def test_a_graph_outlives_the_cache_that_it_was_captured_with():
    cache, ref = make(40, [((64,), torch.float32)] * 3, 4, 8, 5)
    own, ids, lengths, a, b = (cache.tables, cache.lengths, cache.refs, cache.pools), ints([0]), ints([7]), ints([0]), ints([1])
    cache.resize(ids, lengths)
    cache.fork(a, b)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.free(b)
        done = cache.fork(a, b, share=False)
    where = cache._pointers.tensor.data_ptr()
    del cache
    others = [torch.zeros(3, dtype=torch.int64, device="cuda") for _ in range(64)]
    assert all(t.data_ptr() != where for t in others)
    ref.resize([0], [7])
    ref.fork([0], [1], True)
    for r in range(3):
        graph.replay()
        torch.cuda.synchronize()
        ref.free([1])
        assert get(done).tolist() == [True] == ref.fork([0], [1], False)
        assert get(own[0]).tolist() == ref.tables and get(own[1]).tolist() == ref.lengths and get(own[2]).tolist() == ref.refs
        assert all(torch.equal(get(p), q) for p, q in zip(own[3], ref.pools))


def test_compact_into_an_empty_view_of_something_else():
    """A table without entries meets nothing, wherever it points."""
    counts = ints([0, 2, 0, 1, 0])
    pool = put(torch.arange(10.0).view(5, 2))
    cache = thrust_amd.PageCache([pool], 4, 3, 0, refs=counts)
    new = ints([7] * 5)
    assert get(cache.compact(tables=counts[2:2].view(3, 0), refs=new)).tolist() == [2]
    assert get(new).tolist() == [1, 2, 0, 0, 0] and get(counts).tolist() == [0, 2, 0, 1, 0]
    assert get(pool)[:2].tolist() == [[6.0, 7.0], [2.0, 3.0]]
