"""PagedKVCache's own operators against a model of them on the CPU that holds the
pools, tables and counts as the contract says, entry by entry."""
import math
import random

import pytest
import torch

from memory_efficient_attn_layer_amd import PagedKVCache

pytestmark = pytest.mark.gpu


class Model:
    """The cache's contract, one entry at a time."""

    def __init__(self, cache):
        self.page, self.M = cache.page, cache.table.shape[1]
        self.pools = [cache.k.cpu().clone(), cache.v.cpu().clone()]
        self.table, self.lengths = cache.table.cpu().clone(), cache.lengths.cpu().clone()
        self.refs, self.status = cache.refs.cpu().clone(), 0

    def held(self, rows):
        return -(-rows // self.page)

    def free(self):
        return [p for p in range(len(self.refs)) if self.refs[p] <= 0]

    def place(self, s, r):
        return int(self.table[s, r // self.page]), r % self.page

    def give_back(self, s, first, last):
        for j in range(first, last):
            self.refs[self.table[s, j]] -= 1
            self.table[s, j] = -1

    def append(self, k, v, counts):
        """k, v (total, H, N), counts[s] rows each."""
        free, used, t0 = self.free(), 0, 0
        refs0 = self.refs.clone()
        todo = []
        for s, n in enumerate(counts):
            old, rows = int(self.lengths[s]), slice(t0, t0 + n)
            t0 += n
            if n == 0:
                continue
            if old + n > self.M * self.page:
                self.status |= 2
                continue
            shared = old % self.page > 0 and refs0[self.table[s, old // self.page]] > 1
            need = self.held(old + n) - self.held(old) + shared
            mine = free[used:used + need]
            used += need
            if len(mine) < need:
                self.status |= 1
                continue
            todo.append((s, old, n, rows, shared, mine))
        for s, old, n, rows, shared, mine in todo:
            if shared:
                page, j = mine[0], old // self.page
                for pool in self.pools:
                    pool[page, :, :old % self.page] = pool[self.table[s, j], :, :old % self.page]
                self.refs[self.table[s, j]] -= 1
                self.table[s, j] = page
                mine, taken = mine[1:], [page]
            else:
                taken = []
            for j, page in enumerate(mine):
                self.table[s, self.held(old) + j] = page
            for page in taken + mine:
                self.refs[page] = 1
            for i in range(n):
                page, row = self.place(s, old + i)
                self.pools[0][page, :, row] = k[rows][i]
                self.pools[1][page, :, row] = v[rows][i]
            self.lengths[s] = old + n

    def accept(self, n, path, counts):
        free, used, refs0 = self.free(), 0, self.refs.clone()
        back = []
        for s in range(len(self.lengths)):
            old = int(self.lengths[s])
            base = max(old - n, 0)
            count = min(max(int(counts[s]), 0), len(path[s]), old - base)
            shared = [j for j in range(base // self.page, self.held(base + count)) if refs0[self.table[s, j]] > 1] if count else []
            mine = free[used:used + len(shared)]
            used += len(shared)
            if len(mine) < len(shared):
                self.status |= 1
                continue
            rows = [self.place(s, base + min(max(int(path[s][i]), 0), old - base - 1)) for i in range(count)]
            moved = [[pool[page, :, row].clone() for page, row in rows] for pool in self.pools]
            for j, page in zip(shared, mine):
                if j == base // self.page:
                    for pool in self.pools:
                        pool[page, :, :base % self.page] = pool[self.table[s, j], :, :base % self.page]
                self.refs[self.table[s, j]] -= 1
                self.table[s, j] = page
                self.refs[page] = 1
            for pool, values in zip(self.pools, moved):
                for i, x in enumerate(values):
                    page, row = self.place(s, base + i)
                    pool[page, :, row] = x
            back.append((s, base + count, old))
        for s, new, old in back:
            self.give_back(s, self.held(new), self.held(old))
            self.lengths[s] = new

    def truncate(self, lengths):
        for s, new in enumerate(lengths):
            old = int(self.lengths[s])
            new = min(max(int(new), 0), old)
            self.give_back(s, self.held(new), self.held(old))
            self.lengths[s] = new

    def fork(self, parents):
        table, lengths = self.table.clone(), self.lengths.clone()
        for s, p in enumerate(parents):
            live = 0 <= p < len(lengths)
            for j in range(self.M):
                if self.table[s, j] >= 0:
                    self.refs[self.table[s, j]] -= 1
            self.table[s] = table[p] if live else -1
            self.lengths[s] = lengths[p] if live else 0
            for j in range(self.M):
                if self.table[s, j] >= 0:
                    self.refs[self.table[s, j]] += 1

    def compact(self):
        live = int((self.refs > 0).sum())
        source = [p for p in range(live, len(self.refs)) if self.refs[p] > 0]
        target = [p for p in range(live) if self.refs[p] <= 0]
        for a, b in zip(source, target):
            for pool in self.pools:
                pool[b] = pool[a]
            self.table[self.table == a] = b
            self.refs[b], self.refs[a] = int(self.refs[a]), 0

    def same(self, cache):
        assert torch.equal(cache.lengths.cpu(), self.lengths)
        assert torch.equal(cache.table.cpu(), self.table)
        assert torch.equal(cache.refs.cpu(), self.refs)
        assert int(cache.status) == self.status
        for a, b in zip((cache.k, cache.v), self.pools):
            assert torch.equal(a.cpu().view(torch.int16), b.view(torch.int16))


def _cache(S, H, N, pages, page, max_pages, dtype=torch.bfloat16, seed=0):
    c = PagedKVCache.empty(S, H, N, pages, "cuda", page=page, max_pages=max_pages, dtype=dtype)
    g = torch.Generator("cuda").manual_seed(seed)
    c.k.copy_(torch.randn(c.k.shape, device="cuda", generator=g))
    c.v.copy_(torch.randn(c.v.shape, device="cuda", generator=g))
    return c


def _rows(n, H, N, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(n, H, N, generator=g).to(dtype), torch.randn(n, H, N, generator=g).to(dtype)


@pytest.mark.parametrize("S,H,N,page,pages,max_pages,dtype", [
    (5, 2, 64, 16, 60, 9, torch.bfloat16), (7, 1, 32, 32, 40, 5, torch.float16), (3, 3, 128, 64, 20, 4, torch.bfloat16),
    (4, 2, 256, 16, 50, 20, torch.float16), (70, 1, 32, 16, 150, 4, torch.bfloat16),
], ids=["page16", "page32-fp16", "page64", "wide-fp16", "many"])
@pytest.mark.parametrize("seed", [0, 1])
def test_any_order_of_calls(S, H, N, page, pages, max_pages, dtype, seed):
    """Calls in a drawn order, with pools that run out and sequences that fill up."""
    rng = random.Random(seed)
    c = _cache(S, H, N, pages, page, max_pages, dtype)
    m = Model(c)
    for it in range(30):
        what = rng.choice(("append", "append", "append", "packed", "tree", "fork", "truncate", "free", "compact"))
        if what == "append":
            n = rng.choice((1, 1, 3, page, 2 * page + 1))
            k, v = _rows(S * n, H, N, dtype, it)
            c.append(k.view(S, n, H, N).cuda(), v.view(S, n, H, N).cuda())
            m.append(k, v, [n] * S)
        elif what == "packed":
            counts = [rng.choice((0, 0, 1, page - 1, page, 3 * page)) for _ in range(S)]
            if sum(counts) == 0:
                continue
            k, v = _rows(sum(counts), H, N, dtype, it)
            cu = torch.tensor([0] + torch.tensor(counts).cumsum(0).tolist(), dtype=torch.int32)
            c.append(k.cuda(), v.cuda(), cu.cuda() if it % 2 else cu)
            m.append(k, v, counts)
        elif what == "tree":
            n = rng.choice((1, 4, page, page + 7))
            most = rng.randint(1, n)
            path = [[rng.randint(-1, n) for _ in range(most)] for _ in range(S)]
            counts = [rng.randint(-1, most + 1) for _ in range(S)]
            c.accept(n, path, counts)
            m.accept(n, path, counts)
        elif what == "fork":
            parents = [rng.choice((s, s, rng.randrange(S), -1, S)) for s in range(S)]
            c.fork(parents)
            m.fork(parents)
        elif what == "truncate":
            new = [rng.choice((1 << 20, int(x) - 1, int(x) // 2, page, -3)) for x in m.lengths]
            c.truncate(new)
            m.truncate(new)
        elif what == "free":
            gone = [s for s in range(S) if rng.random() < 0.3]
            c.free(gone)
            m.truncate([0 if s in gone else 1 << 20 for s in range(S)])
        else:
            c.compact()
            m.compact()
        m.same(c)


def test_large_tables():
    """More sequences than a plan has threads, a table that is forked in two launches."""
    S, H, N, page = 1100, 1, 32, 16
    c = _cache(S, H, N, 2600, page, 12)
    m = Model(c)
    for it, n in enumerate((9, 10, 1)):
        k, v = _rows(S * n, H, N, torch.bfloat16, it)
        c.append(k.view(S, n, H, N).cuda(), v.view(S, n, H, N).cuda()), m.append(k, v, [n] * S)
        m.same(c)
        parents = [(s * 31 + it) % S if s % 3 else s for s in range(S)]
        c.fork(parents), m.fork(parents)
        m.same(c)
        path, counts = [[2, 0]] * S, [s % 3 for s in range(S)]
        c.accept(4, path, counts), m.accept(4, path, counts)
        m.same(c)
    c.compact(), m.compact()
    m.same(c)


@pytest.mark.parametrize("pages,held", [(4099, 1), (4096, 4096), (9001, 3000), (9001, 8200), (8193, 0)])
def test_pools_of_many_pages_are_compacted(pages, held):
    """More pages than one pass of the plan takes; none to move, none free, most of both."""
    c = _cache(4, 1, 32, pages, 16, pages // 4 + 1)
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(held))[:held].to(torch.int32)
    for s in range(4):
        mine = order[s::4]
        c.table[s, : len(mine)] = mine.cuda()
        c.lengths[s] = 16 * len(mine)
    c.refs[order.long().cuda()] = 1
    m = Model(c)
    c.compact()
    m.compact()
    m.same(c)


def test_shared_pages_are_copied_by_every_writer():
    """Three sequences on one prompt; two of them write, one into the middle of the
    tree of the others."""
    c = _cache(3, 2, 64, 20, 16, 6)
    m = Model(c)
    k, v = _rows(40, 2, 64, torch.bfloat16, 1)
    for call in (lambda x: x.append(*(t.cuda() if x is c else t for t in (k, v)), [0, 40, 40, 40] if x is c else [40, 0, 0]),
                 lambda x: x.fork([0, 0, 0])):
        call(c), call(m)
        m.same(c)
    assert c.refs[:3].tolist() == [3, 3, 3]
    # A tree of 20 rows, all of it in shared pages, taken apart by two of them.
    path, counts = [[19, 0, 19, 7], [3, 2, 1, 0], [0, 0, 0, 0]], [4, 3, 0]
    c.accept(20, path, counts), m.accept(20, path, counts)
    m.same(c)
    k, v = _rows(3, 2, 64, torch.bfloat16, 2)
    c.append(k[:, None].cuda(), v[:, None].cuda()), m.append(k, v, [1, 1, 1])
    m.same(c)


def test_full_pool_and_full_sequences_are_reported():
    c = _cache(2, 1, 32, 3, 16, 2)
    k, v = _rows(2 * 16, 1, 32, torch.bfloat16, 0)
    c.append(k.view(2, 16, 1, 32).cuda(), v.view(2, 16, 1, 32).cuda())
    c.verify()
    c.append(k.view(2, 16, 1, 32).cuda(), v.view(2, 16, 1, 32).cuda())
    assert c.lengths.tolist() == [32, 16]
    with pytest.raises(RuntimeError, match="pages"):
        c.verify()
    c.verify()  # reported once
    c.append(k[:1].view(1, 1, 1, 32).expand(2, 1, 1, 32).cuda(), v[:1].view(1, 1, 1, 32).expand(2, 1, 1, 32).cuda())
    assert c.lengths.tolist() == [32, 16]
    with pytest.raises(RuntimeError, match="pages and a sequence would pass 32 rows"):
        c.verify()


def test_rows_with_strides_of_their_own():
    """From a (sequences, heads, rows, N) cache, and from a slice of a joint projection."""
    c = _cache(2, 2, 64, 20, 16, 8)
    m = Model(c)
    old = torch.randn(2, 2, 50, 64, device="cuda").bfloat16()
    joint = torch.randn(2, 3, 4, 64, device="cuda").bfloat16()
    for k, v in ((old.transpose(1, 2), old.flip(0).transpose(1, 2)), (joint[:, :, :2], joint[:, :, 2:]),
                 (joint[:, :, :2, :].float().bfloat16()[..., torch.randperm(64, device="cuda")], joint[:, :, 2:])):
        c.append(k, v)
        m.append(k.flatten(0, 1).cpu(), v.flatten(0, 1).cpu(), [k.shape[1]] * 2)
        m.same(c)


def test_refusals_on_the_gpu():
    c = _cache(2, 2, 64, 8, 16, 4)
    k = torch.zeros(2, 3, 2, 64, device="cuda", dtype=torch.bfloat16)
    for bad in (k[:1], k[:, :, :1], k[..., :32], k[0]):
        with pytest.raises(ValueError):
            c.append(bad, bad)
    with pytest.raises(ValueError):
        c.append(k, k[:, :2])
    with pytest.raises(TypeError):
        c.append(k.half(), k.half())
    for cu in ([0, 3], [0, 1, 2], [0, 4, 3], torch.tensor([0, 1, 3], device="cuda")):
        with pytest.raises(ValueError):
            c.append(k[0], k[0], cu)
    with pytest.raises(ValueError):
        c.accept(0, [[0], [0]], [1, 1])
    with pytest.raises(ValueError):
        c.accept(2, [[0, 1, 2]] * 2, [1, 1])
    with pytest.raises(ValueError):
        c.accept(2, [[0]], [1, 1])
    for call in (lambda: c.truncate([0, 1 << 40]), lambda: c.truncate([0.0, 1.0]), lambda: c.accept(2, [[0.5], [1]], [1, 1]),
                 lambda: c.truncate([1]), lambda: c.fork(torch.zeros(2, device="cuda")), lambda: c.free([2]),
                 lambda: c.accept(2, [[0], [1]], [1])):
        with pytest.raises(ValueError):
            call()
    c.append(k[:, :0], k[:, :0])  # nothing to write
    assert c.lengths.tolist() == [0, 0] and int(c.status) == 0


def test_entries_outside_the_pool_are_skipped():
    """A table from elsewhere with entries that name no page."""
    c = _cache(2, 1, 32, 4, 16, 3)
    c.lengths.copy_(torch.tensor([20, 10]))
    c.table.copy_(torch.tensor([[0, 99, -1], [-7, -1, -1]]))
    c.refs.copy_(torch.tensor([1, 0, 0, 0]))
    pools = c.k.clone(), c.v.clone()
    k, v = _rows(4, 1, 32, torch.bfloat16, 3)
    c.append(k.view(2, 2, 1, 32).cuda(), v.view(2, 2, 1, 32).cuda())  # rows 20, 21 and 10, 11: no page takes them
    c.accept(2, [[1], [1]], [1, 1])
    c.compact()
    c.fork([1, 0])
    c.truncate([0, 0])
    assert torch.equal(c.k, pools[0]) and torch.equal(c.v, pools[1])
    assert c.lengths.tolist() == [0, 0] and c.refs.tolist() == [0, 0, 0, 0]


def test_captured_and_replayed():
    """A step of beam search in a graph (fork, append, set back), eager calls between."""
    S, H, N, page = 6, 2, 64, 16
    c = _cache(S, H, N, 80, page, 6)
    m = Model(c)
    k, v = _rows(S * 21, H, N, torch.bfloat16, 0)
    c.append(k.view(S, 21, H, N).cuda(), v.view(S, 21, H, N).cuda()), m.append(k, v, [21] * S)
    parents = torch.arange(S, dtype=torch.int32, device="cuda")
    rows = [torch.zeros(S, 1, H, N, device="cuda", dtype=torch.bfloat16) for _ in range(2)]
    back = torch.full((S,), 1 << 20, dtype=torch.int32, device="cuda")

    def step():
        c.fork(parents)
        c.append(*rows)
        c.truncate(back)

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):  # (recorded, not run)
        step()
    for it in range(6):
        new = [(s + it) % S // 2 * 2 for s in range(S)]
        x, y = _rows(S, H, N, torch.bfloat16, 10 + it)
        parents.copy_(torch.tensor(new))
        rows[0].copy_(x[:, None])
        rows[1].copy_(y[:, None])
        keep = [1 << 20] * S if it % 3 else [20] * S
        back.copy_(torch.tensor(keep))
        graph.replay()
        m.fork(new), m.append(x, y, [1] * S), m.truncate(keep)
        m.same(c)
        if it == 2:
            c.compact(), m.compact()
            m.same(c)


def test_offsets_past_32_bits():
    """Pages whose element offset passes 2^32."""
    H, N, page, pages = 8, 256, 256, 8400  # 524288 elements a page
    c = PagedKVCache.empty(2, H, N, pages, "cuda", page=page, max_pages=8)
    assert c.k.numel() > 1 << 32
    c.refs[: pages - 6] = 1  # others hold the front
    k = torch.randn(2, 600, H, N, device="cuda").bfloat16()
    v = torch.randn(2, 600, H, N, device="cuda").bfloat16()
    c.append(k, v)
    assert c.table[:, :3].flatten().tolist() == list(range(pages - 6, pages))
    c.accept(100, [[99, 50]] * 2, [2, 2])
    for pool, x in ((c.k, k), (c.v, v)):
        for s in range(2):
            ids = c.table[s, :2].long()
            got = pool[ids].transpose(1, 2).reshape(-1, H, N)[:502]
            assert torch.equal(got, torch.cat((x[s, :500], x[s, 599:600], x[s, 550:551])))
    c.refs[: pages - 6] = 0
    c.compact()
    assert sorted(c.table[:, :2].flatten().tolist()) == [0, 1, 2, 3] and c.refs[:5].tolist() == [1, 1, 1, 1, 0]
    got = c.v[c.table[1, :2].long()].transpose(1, 2).reshape(-1, H, N)[:500]
    assert torch.equal(got, v[1, :500])
