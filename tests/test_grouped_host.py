"""Refusals of the grouped and paged entry points, before anything is launched
(no GPU needed), and the references of their tests."""
import ctypes
import math

import pytest
import torch

from memory_efficient_attn_layer_amd import PagedKVCache, _lib, grouped_attn_varlen, tree_attn
from tests import grouped_util as gu

bf16 = torch.bfloat16


def _qkv(total=8, Hq=4, Hkv=2, N=64, dtype=bf16):
    return (torch.zeros(total, h, N, dtype=dtype) for h in (Hq, Hkv, Hkv))


@pytest.mark.parametrize("shape,exc", [
    (dict(Hq=4, Hkv=3), ValueError), (dict(N=48), ValueError), (dict(N=16), ValueError), (dict(total=0), ValueError),
    (dict(dtype=torch.float32), TypeError), (dict(), RuntimeError),
], ids=["heads", "width-48", "width-16", "empty", "fp32", "cpu"])
def test_grouped_refuses(shape, exc):
    with pytest.raises(exc):
        grouped_attn_varlen(*_qkv(**shape), [0, 8])


def test_grouped_refuses_operands_that_do_not_match():
    q, k, v = _qkv()
    for bad in ((q[0], k, v), (q, k[:7], v[:7]), (q, k, v[..., :32]), (q, k[:, :0], v[:, :0]), (q, k, v[:, :1])):
        with pytest.raises(ValueError):
            grouped_attn_varlen(*bad, [0, 8])
    with pytest.raises(TypeError):
        grouped_attn_varlen(q, k.half(), v, [0, 8])


def _desc(**kw):
    d = dict(total=8, nseq=1, Hq=4, Hkv=2, N=64, q_tok=256, q_head=64, k_tok=128, k_head=64, v_tok=128, v_head=64,
             scale=0.125, dtype=0)
    d.update(kw)
    return _lib.MeaGrouped(*d.values())


@pytest.mark.parametrize("kw,code", [
    (dict(N=16), -3), (dict(total=0), -2), (dict(nseq=0), -2), (dict(total=1 << 30), -2), (dict(Hkv=3), -12),
    (dict(dtype=2), -14), (dict(q_tok=252), -15), (dict(k_tok=1 << 25), -15), (dict(v_head=-8), -15), (dict(scale=0.0), -16),
    (dict(scale=math.inf), -16), (dict(scale=math.nan), -16),
])
def test_grouped_descriptor_codes(kw, code):
    lib, P = _lib.load(), 4096  # (never touched)
    assert lib.mea_grouped_fwd(_desc(**kw), P, P, P, P, P, None, None, None) == code
    assert lib.mea_grouped_bwd(_desc(**kw), P, P, P, P, P, P, P, P, P, P, P, P, 1 << 20, None) == code
    assert lib.mea_grouped_workspace_bytes(_desc(**kw)) == 0
    assert _lib.strerror(code) != "unknown status"


def test_grouped_pointer_codes():
    lib, P = _lib.load(), 4096
    assert lib.mea_grouped_fwd(_desc(), None, P, P, P, P, None, None, None) == -1
    assert lib.mea_grouped_fwd(_desc(), P, P, P, P + 2, P, None, None, None) == -6
    assert lib.mea_grouped_fwd(_desc(), P, P, P, P, P, P, None, None) == -1  # o_rest without lse
    assert lib.mea_grouped_fwd(_desc(dtype=1), P, P, P, P, P, P, P, None) == -14  # nothing is saved in fp16
    assert lib.mea_grouped_bwd(_desc(dtype=1), P, P, P, P, P, P, P, P, P, P, P, P, 1 << 20, None) == -14
    need = lib.mea_grouped_workspace_bytes(_desc())
    assert need >= 8 * 4 * 4
    assert lib.mea_grouped_bwd(_desc(), P, P, P, P, P, P, P, P, P, P, P, P, need - 1, None) == -5


def _cache(S=2, H=2, N=64, pages=4, **kw):
    return PagedKVCache.empty(S, H, N, pages, "cpu", **kw)


@pytest.mark.parametrize("kw,exc", [
    (dict(N=16), ValueError), (dict(page=48), ValueError), (dict(page=8), ValueError), (dict(page=512), ValueError),
    (dict(dtype=torch.float32), TypeError), (dict(S=0), ValueError), (dict(pages=0), ValueError), (dict(H=0), ValueError),
])
def test_cache_refuses(kw, exc):
    with pytest.raises(exc):
        _cache(**kw)


def test_cache_refuses_tensors_that_do_not_match():
    c = _cache()
    parts = dict(k=c.k, v=c.v, table=c.table, lengths=c.lengths, refs=c.refs, status=c.status)
    for name, t in (("v", c.v[..., :32].contiguous()), ("v", c.v.half()), ("lengths", c.lengths[:1]), ("refs", c.refs[:3]),
                    ("status", torch.zeros(2, dtype=torch.int32)), ("k", c.k.transpose(1, 2)), ("table", c.table[0])):
        with pytest.raises(ValueError):
            PagedKVCache(**{**parts, name: t})
    with pytest.raises(TypeError):
        PagedKVCache(**{**parts, "table": c.table.long()})
    assert c.capacity == 256 and c.sequences == 2 and c.page == 64


def test_cache_calls_refuse_the_cpu():
    c = _cache()
    k = torch.zeros(2, 1, 2, 64, dtype=bf16)
    for call in (lambda: c.append(k, k), lambda: c.accept(1, [[0], [0]], [1, 1]), lambda: c.truncate([0, 0]),
                 lambda: c.free([0]), lambda: c.fork([0, 1]), c.compact, lambda: tree_attn(k, c)):
        with pytest.raises(RuntimeError):
            call()


@pytest.mark.parametrize("q,mask,exc", [
    (torch.zeros(2, 3, 4, 64, dtype=torch.half), None, TypeError),
    (torch.zeros(3, 1, 4, 64, dtype=bf16), None, ValueError),
    (torch.zeros(2, 1, 4, 32, dtype=bf16), None, ValueError),
    (torch.zeros(2, 1, 3, 64, dtype=bf16), None, ValueError),
    (torch.zeros(2, 0, 4, 64, dtype=bf16), None, ValueError),
    (torch.zeros(2, 257, 4, 64, dtype=bf16), None, ValueError),
    (torch.zeros(2, 64, dtype=bf16), None, ValueError),
    (torch.zeros(2, 3, 4, 64, dtype=bf16), torch.ones(3, 3), ValueError),
    (torch.zeros(2, 3, 4, 64, dtype=bf16), torch.ones(2, 3, 2, dtype=torch.bool), ValueError),
    (torch.zeros(2, 3, 4, 64, dtype=bf16), torch.ones(1, 3, 3, dtype=torch.bool), ValueError),
])
def test_tree_attn_refuses(q, mask, exc):
    with pytest.raises(exc):
        tree_attn(q, _cache(), mask)


def _c_cache(**kw):
    d = dict(k=4096, v=4096, table=4096, lengths=4096, refs=4096, status=4096, seqs=2, pages=4, Hkv=2, page=64, N=64,
             max_pages=4, dtype=0)
    d.update(kw)
    return _lib.MeaPaged(*d.values())


@pytest.mark.parametrize("kw,code", [
    (dict(k=None), -1), (dict(table=None), -1), (dict(v=4098), -6), (dict(refs=4097), -6), (dict(N=40), -3),
    (dict(page=24), -13), (dict(page=8), -13), (dict(seqs=0), -2), (dict(max_pages=1 << 26), -2), (dict(pages=1 << 31), -2),
    (dict(dtype=7), -14),
])
def test_paged_codes(kw, code):
    lib, P, big = _lib.load(), 4096, 1 << 30
    c, st = _c_cache(**kw), (ctypes.c_int64 * 6)(*[64] * 6)
    assert lib.mea_paged_workspace_bytes(c) == 0
    assert lib.mea_paged_append(c, P, P, st, None, 1, 2, P, big, None) == code
    assert lib.mea_paged_accept(c, 2, P, 1, P, P, big, None) == code
    assert lib.mea_paged_truncate(c, P, None) == code
    assert lib.mea_paged_fork(c, P, P, big, None) == code
    assert lib.mea_paged_compact(c, P, big, None) == code
    assert lib.mea_tree_attn(c, 1, 4, 1.0, P, st, None, 0, P, P, big, None) == code


def test_paged_call_codes():
    lib, P, big = _lib.load(), 4096, 1 << 30
    c, st = _c_cache(), (ctypes.c_int64 * 6)(*[64] * 6)
    need = lib.mea_paged_workspace_bytes(c)
    assert need > 0
    assert lib.mea_paged_append(c, P, P, st, None, 1, 2, P, need - 1, None) == -5
    assert lib.mea_paged_append(c, P, P, st, None, 0, 0, P, big, None) == -2
    assert lib.mea_paged_append(c, P, None, st, None, 1, 2, P, big, None) == -1
    assert lib.mea_paged_append(c, P, P, (ctypes.c_int64 * 6)(*[60] * 6), None, 1, 2, P, big, None) == -15
    for n, most in ((0, 1), (257, 1), (4, 5), (4, 0)):
        assert lib.mea_paged_accept(c, n, P, most, P, P, big, None) == -2
    assert lib.mea_tree_attn(c, 1, 3, 1.0, P, st, None, 0, P, P, big, None) == -12
    assert lib.mea_tree_attn(c, 257, 4, 1.0, P, st, None, 0, P, P, big, None) == -2
    assert lib.mea_tree_attn(c, 1, 4, -1.0, P, st, None, 0, P, P, big, None) == -16
    assert lib.mea_tree_attn(c, 1, 4, 1.0, P, st, None, -1, P, P, big, None) == -15


def test_reference_gradients_are_those_of_autograd():
    """The tests' own formulas against torch's derivatives in 64 bits."""
    g = torch.Generator().manual_seed(3)
    q, k, v, do = (torch.randn(9, h, 32, generator=g, dtype=torch.float64) for h in (4, 2, 2, 4))
    for t in (q, k, v):
        t.requires_grad_(True)
    seen = torch.block_diag(*[torch.tril(torch.ones(n, n)) for n in (5, 4)]).bool()
    a = torch.einsum("ihd,jhd->hij", q, k.repeat_interleave(2, 1)) * 0.3
    o = torch.einsum("hij,jhd->ihd", torch.softmax(a.masked_fill(~seen, -math.inf), -1), v.repeat_interleave(2, 1))
    grads = torch.autograd.grad(o, (q, k, v), do)
    gu_half, gu.half_step = gu.half_step, lambda dtype: 2.0 ** -8
    try:
        ref = gu.packed(q, k, v, [5, 4], 0.3, do)
    finally:
        gu.half_step = gu_half
    for name, t in zip(("o", "dq", "dk", "dv"), (o, *grads)):
        assert torch.allclose(ref[name][0], t, rtol=1e-12, atol=1e-12), name
