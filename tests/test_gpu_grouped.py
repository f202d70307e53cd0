"""grouped_attn_varlen against 64-bit attention, sequence by sequence, with
elementwise error bounds (tests/grouped_util.py)."""
import math

import pytest
import torch

from memory_efficient_attn_layer_amd import grouped_attn_varlen
from tests import grouped_util as gu

pytestmark = pytest.mark.gpu

bf16, fp16 = torch.bfloat16, torch.float16


def _inputs(lens, Hq, Hkv, N, dtype, seed=0, spread=1.0, behind=0):
    g = torch.Generator("cuda").manual_seed(seed)
    total = sum(lens) + behind

    def normal(H):
        return (torch.randn(total, H, N, device="cuda", generator=g) * spread).to(dtype)

    return normal(Hq), normal(Hkv), normal(Hkv), normal(Hq)


def _offsets(lens):
    return torch.tensor([0] + torch.tensor(lens).cumsum(0).tolist(), dtype=torch.int32, device="cuda")


LENS = {"one": [1], "short": [0, 5, 0, 1, 33, 2], "edges": [127, 128, 129, 31, 32, 64], "long": [300, 7, 1025],
        "many": [1 + (7 * i) % 40 for i in range(150)]}


def _check(lens, q, k, v, do, scale=None, backward=True, cu=None):
    sc = 1 / math.sqrt(q.shape[2]) if scale is None else scale
    n = sum(lens)
    if backward:
        q, k, v = (t.detach().requires_grad_(True) for t in (q, k, v))
    o = grouped_attn_varlen(q, k, v, _offsets(lens) if cu is None else cu, scale)
    ref = gu.packed(q[:n], k[:n], v[:n], lens, sc, do[:n] if backward else None)
    gu.assert_within("o", o[:n].detach(), ref["o"])
    assert not bool(o[n:].any())  # tokens of no sequence
    if backward:
        for name, t in zip(("dq", "dk", "dv"), torch.autograd.grad(o, (q, k, v), do)):
            gu.assert_within(name, t[:n], ref[name])
            assert not bool(t[n:].any())


@pytest.mark.parametrize("N", [32, 64, 128, 256])
@pytest.mark.parametrize("Hq,Hkv", [(1, 1), (4, 2), (6, 2), (8, 1), (5, 1), (16, 8)])
@pytest.mark.parametrize("lens", ["one", "short", "edges", "long"])
def test_forward_and_gradients(lens, Hq, Hkv, N):
    _check(LENS[lens], *_inputs(LENS[lens], Hq, Hkv, N, bf16, seed=Hq + N))


@pytest.mark.parametrize("N", [32, 64, 128, 256])
@pytest.mark.parametrize("Hq,Hkv,lens", [(4, 2, "edges"), (3, 3, "long"), (8, 1, "short"), (2, 1, "many")])
def test_forward_fp16(Hq, Hkv, lens, N):
    _check(LENS[lens], *_inputs(LENS[lens], Hq, Hkv, N, fp16, seed=N), backward=False)


@pytest.mark.parametrize("nseq", [61, 62, 63, 64, 150])
def test_as_many_sequences_as_lanes_and_more(nseq):
    lens = LENS["many"][:nseq]
    _check(lens, *_inputs(lens, 4, 2, 64, bf16))


@pytest.mark.parametrize("lens,Hq,Hkv,N", [([2500], 4, 1, 128), ([4100, 60], 2, 1, 64), ([1500, 1400], 8, 1, 256), ([700], 8, 1, 32)])
def test_key_blocks_in_parts(lens, Hq, Hkv, N):
    """Few key blocks with many query tiles: the gradients' sums are joined from parts."""
    _check(lens, *_inputs(lens, Hq, Hkv, N, bf16, behind=70))


def test_no_second_derivative():
    leaves = [t.requires_grad_(True) for t in _inputs([20], 2, 1, 32, bf16)[:3]]
    o = grouped_attn_varlen(*leaves, [0, 20])
    with pytest.raises(RuntimeError, match="second"):
        torch.autograd.grad(o.float().square().sum(), leaves[0], create_graph=True)


def test_tokens_of_no_sequence_get_zeros():
    lens = [70, 0, 130]
    q, k, v, do = _inputs(lens, 4, 2, 64, bf16, behind=300)
    for t in (q, k, v):
        t[sum(lens):] = math.nan
    _check(lens, q, k, v, do)
    # In front of the first sequence too.
    cu = torch.tensor([90, 200], dtype=torch.int32, device="cuda")
    q, k, v, _ = _inputs([400], 4, 2, 64, bf16)
    o = grouped_attn_varlen(q, k, v, cu)
    ref = gu.packed(q[90:200], k[90:200], v[90:200], [110], 0.125)
    gu.assert_within("o", o[90:200], ref["o"])
    assert not bool(o[:90].any()) and not bool(o[200:].any())


@pytest.mark.parametrize("dtype", [bf16, fp16])
@pytest.mark.parametrize("kind", ["rising", "falling", "far-apart", "equal", "tiny-scale"])
def test_logits_of_any_size(kind, dtype):
    """Rows whose maximum keeps moving, logits hundreds apart, all the same."""
    L, N = 500, 64
    q, k, v, do = _inputs([L], 4, 2, N, dtype, seed=5)
    scale = 0.125
    if kind in ("rising", "falling"):
        ramp = torch.linspace(0, 4, L, device="cuda") if kind == "rising" else torch.linspace(4, 0, L, device="cuda")
        k = (ramp[:, None, None] * torch.ones_like(k, dtype=torch.float32)).to(dtype)
        q = torch.ones_like(q)
        scale = 0.5  # logits up to 128, a rise of a quarter per key
    elif kind == "far-apart":
        scale = 3.0
    elif kind == "equal":
        q = torch.zeros_like(q)
    else:
        scale = 1e-30
    _check([L], q, k, v, do, scale, backward=dtype == bf16)


def test_rows_with_strides_of_their_own():
    """q, k and v as slices of one joint projection, heads not next to each other,
    and a key shared by every head through a stride of 0."""
    lens, N = [70, 1, 200], 64
    g = torch.Generator("cuda").manual_seed(2)
    joint = torch.randn(sum(lens), 8 + 2 + 2, N, device="cuda", generator=g).bfloat16()
    do = torch.randn(sum(lens), 8, N, device="cuda", generator=g).bfloat16()
    q, k, v = joint[:, :8], joint[:, 8:10], joint[:, 10:]
    _check(lens, q, k, v, do)
    head_major = joint.transpose(0, 1).contiguous().transpose(0, 1)
    _check(lens, head_major[:, :8], head_major[:, 8:10], head_major[:, 10:], do)
    odd = torch.randn(sum(lens), 12, N + 1, device="cuda", generator=g).bfloat16()[..., 1:]  # not 16-byte rows
    _check(lens, odd[:, :8], odd[:, 8:10], odd[:, 10:], do)
    one = joint[:, 8:9].detach().clone().requires_grad_(True)
    q2 = q.detach().clone().requires_grad_(True)
    o = grouped_attn_varlen(q2, one.expand(-1, 4, -1), one.expand(-1, 4, -1), _offsets(lens))
    ref = gu.packed(q2, one, one, lens, 0.125, do)
    gu.assert_within("o", o.detach(), ref["o"])
    (dk,) = torch.autograd.grad(o, one, do)
    # Autograd adds the gradients of the eight expanded heads in bf16: each is
    # rounded, and so is every partial sum.
    want = ref["dk"][0] + ref["dv"][0]
    mag = gu.packed(q2.abs(), one.abs(), one.abs(), lens, 0.125, do.abs())
    tol = ref["dk"][1] + ref["dv"][1] + 2.0 ** -8 * 8 * (mag["dv"][0].abs() + ref["dk"][1] * 2 ** 8)
    gu.assert_within("broadcast", dk, (want, tol))


def test_gradient_against_differences():
    """The kernel's gradients against differences of the 64-bit loss."""
    lens, N, h = [40, 3, 65], 32, 1e-4
    q, k, v, do = _inputs(lens, 4, 2, N, bf16, seed=8)
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    grads = torch.autograd.grad(grouped_attn_varlen(*leaves, _offsets(lens)), leaves, do)
    ref = gu.packed(q, k, v, lens, N ** -0.5, do)
    g = torch.Generator("cuda").manual_seed(1)
    real, gu.half_step = gu.half_step, lambda dtype: 0.0
    try:
        for i, name in enumerate(("dq", "dk", "dv")):
            way = torch.randn(leaves[i].shape, device="cuda", generator=g, dtype=torch.float64)
            loss = []
            for s in (h, -h):
                x = [t.detach().double() for t in leaves]
                x[i] = x[i] + s * way
                loss.append((gu.packed(*x, lens, N ** -0.5)["o"][0] * do.double()).sum())
            slope = float(loss[0] - loss[1]) / (2 * h)
            got = float((grads[i].double() * way).sum())
            tol = float((ref[name][1] * way.abs()).sum()) + 1e-5 * abs(slope)
            assert abs(got - slope) <= tol, name
            # The bound above is far wider than the error: it is a sum of random signs.
            assert abs(got - slope) <= 6 * float((ref[name][1] * way).square().sum().sqrt()) + 1e-5 * abs(slope), name
    finally:
        gu.half_step = real


@pytest.mark.parametrize("N", [32, 64, 128, 256])
@pytest.mark.parametrize("Hq,Hkv", [(4, 1), (2, 1), (1, 1)])
def test_infinities_reach_only_the_rows_that_see_them(Hq, Hkv, N):
    lens = [75, 140]
    q, k, v, _ = _inputs(lens, Hq, Hkv, N, bf16)
    clean = grouped_attn_varlen(q, k, v, _offsets(lens))
    v[75 + 40, 0, 3], v[75 + 99, 0, N - 1], v[75 + 40, 0, 9] = math.nan, math.inf, -math.inf
    k[75 + 120, 0, 0] = math.nan
    got = grouped_attn_varlen(q, k, v, _offsets(lens))
    assert torch.equal(got[:75 + 40], clean[:75 + 40])  # the other sequence, and the rows in front
    rows = got[75:]
    assert bool(torch.isnan(rows[40:, :, 3]).all()) and bool((rows[40:120, :, 9] == -math.inf).all())
    assert bool((rows[99:120, :, N - 1] == math.inf).all()) and bool(torch.isfinite(rows[40:99, :, N - 1]).all())
    assert bool(torch.isnan(rows[120:]).all())  # a NaN score
    rest = [d for d in range(N) if d not in (3, 9, N - 1)]
    assert bool(torch.isfinite(rows[40:120][..., rest]).all())


def test_gradients_of_one_sequence_do_not_reach_another():
    lens = [64, 100, 30]
    q, k, v, do = _inputs(lens, 4, 2, 64, bf16)
    cu = _offsets(lens)

    def grads():
        leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
        return torch.autograd.grad(grouped_attn_varlen(*leaves, cu), leaves, do)

    clean = grads()
    for t in (q, k, v, do):
        t[64:164] = math.nan
    for a, b in zip(grads(), clean):
        assert torch.equal(a[:64], b[:64]) and torch.equal(a[164:], b[164:])


def test_same_bits_every_time_and_without_saving():
    lens = [333, 90]
    q, k, v, do = _inputs(lens, 8, 2, 128, bf16)
    runs = []
    for _ in range(2):
        leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
        o = grouped_attn_varlen(*leaves, _offsets(lens))
        runs.append((o.detach(), *torch.autograd.grad(o, leaves, do)))
    assert all(torch.equal(a, b) for a, b in zip(*runs))
    assert torch.equal(runs[0][0], grouped_attn_varlen(q, k, v, _offsets(lens)))
    assert torch.equal(runs[0][0], grouped_attn_varlen(q, k, v, [0, 333, 423]))


def test_offsets_on_the_host_are_checked():
    q, k, v, _ = _inputs([20], 2, 1, 32, bf16)
    for cu in ([0], [0, 19], [1, 20], [0, 15, 10, 20], torch.tensor([0, 21])):
        with pytest.raises(ValueError):
            grouped_attn_varlen(q, k, v, cu)
    for cu in (torch.tensor([0, 20], device="cuda"), torch.tensor([[0, 20]], dtype=torch.int32, device="cuda")):
        with pytest.raises(ValueError):
            grouped_attn_varlen(q, k, v, cu)
    with pytest.raises(ValueError):
        grouped_attn_varlen(q, k, v, [0, 20], scale=0.0)
    with pytest.raises(TypeError):
        grouped_attn_varlen(q.half().requires_grad_(True), k.half(), v.half(), [0, 20])
    with torch.no_grad():
        assert grouped_attn_varlen(q.half().requires_grad_(True), k.half(), v.half(), [0, 20]).grad_fn is None


def test_another_stream():
    lens = [200, 31]
    q, k, v, _ = _inputs(lens, 4, 2, 64, bf16)
    want = grouped_attn_varlen(q, k, v, _offsets(lens))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = grouped_attn_varlen(q, k, v, _offsets(lens))
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)


def test_captured_and_replayed():
    """Forward and gradients in a graph, new inputs and lengths between replays."""
    lens = [100, 60, 40]
    q, k, v, do = _inputs(lens, 4, 2, 64, bf16)
    cu = _offsets(lens)
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]

    def run():
        o = grouped_attn_varlen(*leaves, cu)
        return (o, *torch.autograd.grad(o, leaves, do))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    for i, new in enumerate(([100, 60, 40], [1, 199, 0], [64, 64, 72], [200, 0, 0])):
        fresh = _inputs(new, 4, 2, 64, bf16, seed=20 + i)
        with torch.no_grad():
            for t, x in zip((*leaves, do), fresh):
                t.copy_(x)
        cu.copy_(_offsets(new))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.detach().clone() for t in out]
        for a, b in zip(got, run()):
            assert torch.equal(a, b.detach())


def test_offsets_past_32_bits():
    """Rows whose element offset passes 2^31 (and 2^32 bytes)."""
    L, n, Hq, N = 64, 1040, 256, 128  # 66560 tokens x 256 heads x 128
    g = torch.Generator("cuda").manual_seed(4)
    q = torch.empty(n * L, Hq, N, device="cuda", dtype=bf16).normal_(generator=g)
    assert q.numel() > 1 << 31
    k, v = (torch.randn(n * L, 2, N, device="cuda", generator=g).to(bf16) for _ in range(2))
    q.requires_grad_(True)
    o = grouped_attn_varlen(q, k, v, _offsets([L] * n))
    do = torch.randn(n * L, 1, N, device="cuda", generator=g).to(bf16).expand(-1, Hq, -1)
    (dq,) = torch.autograd.grad(o, q, do)
    for r in (slice(0, L), slice((n - 1) * L, n * L)):
        for h in (0, Hq - 1):
            kv = slice(h // 128, h // 128 + 1)
            ref = gu.packed(q[r, h:h + 1], k[r, kv], v[r, kv], [L], N ** -0.5, do[r, h:h + 1])
            gu.assert_within("o", o[r, h:h + 1].detach(), ref["o"])
            gu.assert_within("dq", dq[r, h:h + 1], ref["dq"])
