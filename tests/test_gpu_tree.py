"""tree_attn against 64-bit attention over the rows of each sequence, and the
operators together, as a decoding loop uses them."""
import math
import random

import pytest
import torch

from memory_efficient_attn_layer_amd import KVCache, PagedKVCache, grouped_attn_varlen, tree_attn
from tests import grouped_util as gu

pytestmark = pytest.mark.gpu

bf16, fp16 = torch.bfloat16, torch.float16


def _cache(lens, H, N, page, dtype, seed=0, room=0, fill=math.nan):
    """A cache with rows of normal values; the rest of the pool holds ``fill``."""
    pages = sum(-(-L // page) for L in lens) + 5
    g = torch.Generator("cuda").manual_seed(seed)
    c = PagedKVCache.empty(len(lens), H, N, pages, "cuda", page=page, max_pages=-(-max(max(lens) + room, 1) // page),
                           dtype=dtype)
    c.k.fill_(fill)
    c.v.fill_(fill)
    total = sum(lens)
    # Rows written in two parts, so that the pages of a sequence are not consecutive.
    k, v = (torch.randn(total, H, N, device="cuda", generator=g).to(dtype) for _ in range(2))
    first = [L // 2 for L in lens]
    starts = [sum(lens[:i]) for i in range(len(lens))]
    for part in (0, 1):
        ids = [torch.arange(a + (0 if part == 0 else f), a + (f if part == 0 else L))
               for a, f, L in zip(starts, first, lens)]
        cu = [0] + torch.tensor([len(i) for i in ids]).cumsum(0).tolist()
        ids = torch.cat(ids).cuda()
        c.append(k[ids], v[ids], cu)
    c.verify()
    assert c.lengths.tolist() == list(lens)
    return c


def _tree(S, n, seed):
    """Masks of drafted trees: every token hangs on the sequence or on an earlier token."""
    rng = random.Random(seed)
    mask = torch.zeros(S, n, n, dtype=torch.bool)
    for s in range(S):
        for i in range(n):
            up = rng.randint(-1, i - 1)
            if up >= 0:
                mask[s, i] = mask[s, up]
            mask[s, i, i] = True
    return mask.cuda()


def _check(c, Hq, n, mask, seed=1, scale=None, spread=1.0):
    g = torch.Generator("cuda").manual_seed(seed)
    N = c.k.shape[3]
    q = (torch.randn(c.sequences, n, Hq, N, device="cuda", generator=g) * spread).to(c.k.dtype)
    got = tree_attn(q, c, mask, scale)
    gu.assert_within("o", got.cpu(), gu.step(q, c, mask, N ** -0.5 if scale is None else scale))
    return q, got


@pytest.mark.parametrize("dtype", [bf16, fp16])
@pytest.mark.parametrize("N,page", [(32, 16), (64, 64), (128, 16), (128, 256), (256, 32)])
@pytest.mark.parametrize("Hq,Hkv,n", [(1, 1, 1), (8, 2, 1), (40, 1, 1), (4, 2, 7), (6, 2, 33), (3, 3, 64), (2, 1, 256)])
def test_step_and_tree(Hq, Hkv, n, N, page, dtype):
    """One block of query rows, two, four, more; lengths at and around tiles and
    pages; sequences with fewer rows than new tokens, and with none."""
    lens = [n + 300, 0, n, max(n - 3, 1), n + 128, n + 127, n + 1]
    c = _cache(lens, Hkv, N, page, dtype, seed=n)
    _check(c, Hq, n, None if n % 2 == 0 or n == 1 else _tree(len(lens), n, n))


@pytest.mark.parametrize("Hq,Hkv,n,page,L", [(8, 2, 1, 64, 20000), (4, 4, 16, 16, 9000), (8, 1, 20, 32, 33000)])
def test_long_contexts_are_split(Hq, Hkv, n, page, L):
    c = _cache([L, 5 + n, L // 3], Hkv, 128, page, bf16)
    _check(c, Hq, n, _tree(3, n, 0) if n > 1 else None)


@pytest.mark.parametrize("S,H,most", [(40, 8, 2500), (65, 1, 3000), (300, 1, 700), (700, 2, 100), (4097, 1, 40)])
def test_many_sequences(S, H, most):
    """More sequences than run at one time, than a wave has lanes, than are counted."""
    lens = [(s * 7919) % most for s in range(S)]
    lens[S // 2] = 9000 if S in (65, 4097) else most
    c = _cache(lens, H, 32, 16, bf16)
    _check(c, H, 1, None)


@pytest.mark.parametrize("one", [False, True], ids=["each", "shared"])
@pytest.mark.parametrize("Hq,Hkv,N", [(1, 1, 128), (3, 1, 32), (10, 2, 64)])
@pytest.mark.parametrize("n", [2, 31, 32, 33, 64, 65, 129, 200, 256])
def test_any_mask(n, Hq, Hkv, N, one):
    """Masks of no shape at all, tokens that see later ones among them, the new rows
    at any place of a tile, of a page, of a chunk."""
    lens = [n, n + 31, n + 97, n // 2, n + 1000, 1, n + 4096 - 13]
    c = _cache(lens, Hkv, N, 32, bf16, seed=n)
    g = torch.Generator("cuda").manual_seed(n)
    shape = (n, n) if one else (len(lens), n, n)
    _check(c, Hq, n, torch.rand(shape, device="cuda", generator=g) < 0.3)


def test_capacities_whose_rows_pass_32_bits():
    """Tables so long that the sequences could have 2^35 rows."""
    S, M = 33, (1 << 22) - 1
    lens = [9000] + [(7 * s) % 90 for s in range(1, S)]
    small = _cache(lens, 1, 32, 256, bf16)
    table = torch.full((S, M), -1, device="cuda", dtype=torch.int32)
    table[:, : small.table.shape[1]] = small.table
    c = PagedKVCache(small.k, small.v, table, small.lengths, small.refs, small.status)
    q, got = _check(small, 1, 1, None)
    gu.assert_within("o", tree_attn(q, c).cpu(), gu.step(q, small, None, 32 ** -0.5))


@pytest.mark.parametrize("n,Hq", [(5, 4), (40, 4), (70, 4)])
@pytest.mark.parametrize("lens", [[0, 0, 200], [2000, 3, 90]], ids=["short", "split"])
def test_tokens_that_see_nothing_get_zeros(lens, n, Hq):
    """Masks without an entry: over no rows in front, nothing is left."""
    c = _cache(lens, 2, 64, 16, bf16, room=n)
    mask = _tree(3, n, 3)
    mask[:, 2] = False
    _, got = _check(c, Hq, n, mask)
    assert not bool(got[1, :n - lens[1]].any())
    if lens[1] <= n:
        assert not bool(got[1, 2].any())
    _check(c, Hq, n, torch.zeros(n, n, dtype=torch.bool, device="cuda"))
    _check(c, Hq, n, torch.ones(n, n, dtype=torch.bool, device="cuda"))


@pytest.mark.parametrize("N", [32, 64, 128, 256])
@pytest.mark.parametrize("n", [4, 40, 70])
def test_infinities_in_hidden_rows(n, N):
    """A NaN or infinity in a row reaches the tokens that see the row only."""
    c = _cache([n + 50, n + 700], 1, N, 32, bf16)
    mask = _tree(2, n, 1)
    mask[:, :, 1] = False
    mask[:, 3, 1] = True
    q, clean = _check(c, 2, n, mask)
    for s, L in enumerate((n + 50, n + 700)):
        row = L - n + 1
        page = int(c.table[s, row // 32])
        c.v[page, 0, row % 32, 5], c.v[page, 0, row % 32, 6] = math.nan, -math.inf
        c.k[page, 0, row % 32] = c.k[page, 0, row % 32].float().abs().to(bf16)
    got = tree_attn(q, c, mask)
    others = [i for i in range(n) if i != 3]
    assert torch.equal(got[:, others], clean[:, others])
    assert bool(torch.isnan(got[:, 3, :, 5]).all()) and bool((got[:, 3, :, 6] == -math.inf).all())
    assert bool(torch.isfinite(got[:, 3][..., 7:]).all())
    c.k[int(c.table[0, (51) // 32]), 0, 51 % 32] = math.nan  # row 51 of sequence 0: token 1
    got = tree_attn(q, c, mask)
    assert torch.equal(got[:, others], clean[:, others]) and bool(torch.isnan(got[0, 3]).all())


def test_large_logits_and_layouts():
    c = _cache([1000, 77], 2, 64, 16, fp16)
    for scale in (3.0, 1e-20):
        _check(c, 4, 3, None, scale=scale)
    g = torch.Generator("cuda").manual_seed(0)
    wide = torch.randn(2, 4, 9, 64 * 2, device="cuda", generator=g).half()
    q = wide.transpose(1, 2)[..., 64:]  # (2, 9, 4, 64), heads outermost
    want = gu.step(q, c, None, 0.125)
    gu.assert_within("strided", tree_attn(q, c).cpu(), want)
    gu.assert_within("unaligned", tree_attn(torch.cat((q, q), -1)[..., 1:65], c).cpu(),
                     gu.step(torch.cat((q, q), -1)[..., 1:65], c, None, 0.125))
    one = tree_attn(q[:, 0], c)
    assert one.shape == (2, 4, 64) and torch.equal(one, tree_attn(q[:, :1], c)[:, 0])
    m = torch.rand(9, 9, device="cuda") < 0.5
    assert torch.equal(tree_attn(q, c, m), tree_attn(q, c, m.expand(2, 9, 9)))
    assert torch.equal(tree_attn(q, c, m.T), tree_attn(q, c, m.T.contiguous()))


def test_pages_outside_the_pool_are_hidden():
    c = _cache([100, 300], 2, 64, 16, bf16)
    q = torch.randn(2, 1, 4, 64, device="cuda").bfloat16()
    c.table[0, 2], c.table[1, 0], c.table[1, 5] = 1 << 20, -5, -1
    got = tree_attn(q, c)
    for s, gone in ((0, (2,)), (1, (0, 5))):
        L = int(c.lengths[s])
        keep = [r for r in range(L) if r // 16 not in gone]
        ids = c.table[s, : -(-L // 16)].long().clamp(0, c.refs.shape[0] - 1)
        k, v = (p[ids].transpose(1, 2).reshape(-1, 2, 64)[keep].double() for p in (c.k, c.v))
        for h in range(4):
            o, _, mag = gu.attend(q[s, :, h].double(), k[:, h // 2], v[:, h // 2],
                                  torch.ones(1, len(keep), dtype=torch.bool, device="cuda"), 0.125)
            gu.assert_within("o", got[s, :, h], (o, 2.0 ** -8 * (2 * o.abs() + mag) + gu.SLACK * mag))


def test_pools_past_32_bits():
    H, N, page, pages = 8, 128, 64, 66000
    c = PagedKVCache.empty(1, H, N, pages, "cuda", page=page, max_pages=16)
    assert c.k.numel() > 1 << 32
    c.refs[: pages - 12] = 1
    k, v = (torch.randn(1, 700, H, N, device="cuda").bfloat16() for _ in range(2))
    c.append(k, v)
    assert int(c.table[0, 0]) == pages - 12
    _check(c, 16, 3, None)


@pytest.mark.parametrize("Hq,Hkv,N,page,dtype", [(8, 2, 64, 16, bf16), (4, 4, 128, 32, fp16)])
def test_together_speculative_decoding(Hq, Hkv, N, page, dtype):
    """Prompts read and cached, beams shared from them, drafted trees checked, the
    accepted path kept, one token more, a sequence ended, the pool compacted: at
    every step the attention equals the one over the rows that should be there."""
    g = torch.Generator("cuda").manual_seed(6)
    lens, n, S = [50, 1, 130, 33], 12, 6

    def rows(*shape):
        return torch.randn(*shape, N, device="cuda", generator=g).to(dtype)

    total = sum(lens)
    q, k, v = rows(total, Hq), rows(total, Hkv), rows(total, Hkv)
    cu = [0] + torch.tensor(lens).cumsum(0).tolist()
    gu.assert_within("prompt", grouped_attn_varlen(q, k, v, cu), gu.packed(q, k, v, lens, N ** -0.5)["o"])
    c = PagedKVCache.empty(S, Hkv, N, 80, "cuda", page=page, max_pages=400 // page, dtype=dtype)
    c.append(k, v, cu + [total, total])
    text = [(k[a:b], v[a:b]) for a, b in zip(cu[:-1], cu[1:])] + [(k[:0], v[:0])] * 2
    parents = [0, 1, 2, 3, 0, 2]
    c.fork(parents)
    text = [text[p] for p in parents]
    for it in range(3):
        mask, dk, dv = _tree(S, n, it), rows(S, n, Hkv), rows(S, n, Hkv)
        c.append(dk, dv)
        text = [(torch.cat((a, x)), torch.cat((b, y))) for (a, b), x, y in zip(text, dk, dv)]
        tq = rows(S, n, Hq)
        got, want = tree_attn(tq, c, mask), gu.step(tq, c, mask, N ** -0.5)
        gu.assert_within("tree", got.cpu(), want)
        path = torch.stack([torch.randperm(n, generator=g, device="cuda")[:4].sort().values for _ in range(S)]).int()
        counts = torch.tensor([(it + s) % 5 for s in range(S)], dtype=torch.int32, device="cuda")
        c.accept(n, path, counts)
        for s in range(S):
            keep = torch.cat((torch.arange(len(text[s][0]) - n, device="cuda"),
                              len(text[s][0]) - n + path[s, : int(counts[s])].long()))
            text[s] = tuple(t[keep] for t in text[s])
        dk, dv = rows(S, 1, Hkv), rows(S, 1, Hkv)
        c.append(dk, dv)
        text = [(torch.cat((a, x)), torch.cat((b, y))) for (a, b), x, y in zip(text, dk, dv)]
        if it == 1:
            c.free([1])
            c.compact()
            c.fork([0, 3, 2, 3, 4, 5])
            text[1] = text[3]
        for s in range(S):
            assert torch.equal(gu.cache_rows(c, s, c.k), text[s][0]) and torch.equal(gu.cache_rows(c, s, c.v), text[s][1])
        _check(c, Hq, 1, None, seed=it)
    c.verify()


def test_together_captured():
    """append, tree_attn and accept in one graph, replayed on growing sequences."""
    S, H, N, n = 3, 2, 64, 5
    c = _cache([20, 60, 7], H, N, 16, bf16, room=200, fill=0.0)
    twin = PagedKVCache(*(t.clone() for t in (c.k, c.v, c.table, c.lengths, c.refs, c.status)))
    k, v = (torch.zeros(S, n, H, N, device="cuda", dtype=bf16) for _ in range(2))
    q, mask = torch.zeros(S, n, 4, N, device="cuda", dtype=bf16), torch.zeros(S, n, n, device="cuda", dtype=torch.bool)
    path, counts = (torch.zeros(S, *m, device="cuda", dtype=torch.int32) for m in ((n,), ()))

    def step(cache):
        cache.append(k, v)
        o = tree_attn(q, cache, mask)
        cache.accept(n, path, counts)
        return o

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(c)
    g = torch.Generator("cuda").manual_seed(1)
    for it in range(5):
        for t in (k, v, q):
            t.copy_(torch.randn(t.shape, device="cuda", generator=g))
        mask.copy_(_tree(S, n, it))
        path.copy_(torch.arange(n).expand(S, n))
        counts.copy_(torch.tensor([it % 3, 5, 1]))
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        assert torch.equal(got, step(twin))
        for a, b in ((c.k, twin.k), (c.v, twin.v), (c.table, twin.table), (c.lengths, twin.lengths), (c.refs, twin.refs)):
            assert torch.equal(a, b)
    c.verify()


def test_rows_of_a_kv_cache_move_over():
    """A prompt's rows of the contiguous cache, appended as they lie there."""
    old = KVCache.empty(2, 4, 64, 100, "cuda")
    old.k.normal_()
    old.v.normal_()
    c = PagedKVCache.empty(2, 4, 64, 20, "cuda", page=32)
    c.append(old.k[:, :, :70].transpose(1, 2), old.v[:, :, :70].transpose(1, 2))
    for s in range(2):
        assert torch.equal(gu.cache_rows(c, s, c.k), old.k[s, :, :70].transpose(0, 1))
    _check(c, 4, 1, None)
