"""The operators of grouped attention and of the paged cache, as calls to measure.

Each case is one pass that a program makes:

  kind  "prompt"   attention over packed prompts (no gradient)
        "train"    the same, forward and the gradients of q, k and v
        "step"     n new tokens per sequence over a paged cache (n = 1: one
                   token; more: a drafted tree with its mask)
        "verify"   a drafted tree's rows written to the cache, the accepted
                   path kept, and the sequences set back to where they began
        "beams"    beams taken over from their parents, one row written to
                   each (the shared last pages are copied), and set back
        "refill"   half of the sequences end, the pages in use move together,
                   new prompts are written into the ended slots
  B, T        sequences, and the longest (the others follow from these two)
  Hq, Hkv, N  query heads, key/value heads, head width
  n           new tokens per sequence
  page        rows of a page
  dtype       "bf16" or "fp16"

With ``own`` false the operators run in plain torch operations in 32 bits,
with ``own`` true through this package.
"""
from __future__ import annotations

import math

import torch

own = False

DEVICE = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def _case(name, kind, B, T, Hq, Hkv, N, n=0, page=0, dtype="bf16"):
    c = dict(kind=kind, B=B, T=T, Hq=Hq, Hkv=Hkv, N=N, n=n, page=page, dtype=dtype)
    if name is not None:
        c["name"] = name
    return c


def listed():
    return [
        # One short prompt of a small model: launches and host work.
        _case("prompt-smallest", "prompt", 1, 256, 4, 2, 64),
        # A serving batch of chat prompts of many lengths, fp16.
        _case("prompt-batch-fp16", "prompt", 12, 2001, 16, 4, 128, dtype="fp16"),
        # One long document read at once.
        _case("prompt-long", "prompt", 1, 16384, 16, 2, 128),
        # Training on documents packed back to back.
        _case("train-packed", "train", 24, 2000, 8, 4, 64),
        # Training on long sequences with wide heads.
        _case("train-long", "train", 2, 8192, 16, 4, 128),
        # One user's next token.
        _case("step-one", "step", 1, 4096, 16, 4, 128, n=1, page=64),
        # The next token of a batch of users at positions of their own.
        _case("step-batch", "step", 64, 8192, 16, 2, 128, n=1, page=64),
        # Drafted trees of a batch, fp16, small pages.
        _case("tree-batch-fp16", "step", 16, 4096, 16, 4, 128, n=32, page=16, dtype="fp16"),
        # A large tree over one very long context.
        _case("tree-long", "step", 1, 131072, 16, 8, 128, n=64, page=128),
        # The cache's share of a speculative step: tree in, path kept.
        _case("cache-verify", "verify", 16, 4096, 8, 4, 128, n=32, page=64),
        # A step of beam search, eight beams to a prompt.
        _case("cache-beams", "beams", 64, 4096, 8, 2, 128, n=1, page=64),
        # Sequences end, the pool is compacted, new prompts come.
        _case("cache-refill", "refill", 32, 8192, 8, 8, 128, page=64),
    ]


def _log_uniform(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)) - 1e-9)))))


def draw(rng):
    """One more case: sizes log-uniform over what the listed ones stand for, mostly odd."""
    kind = rng.choice(("prompt", "train", "step", "step", "verify", "beams", "refill"))
    N = rng.choice((32, 64, 64, 128, 128, 128, 256))
    Hkv, G = rng.choice((1, 2, 3, 4, 8)), rng.choice((1, 2, 3, 4, 5, 8))
    dtype = "bf16" if kind == "train" else rng.choice(("bf16", "fp16"))
    page = rng.choice((16, 32, 64, 128, 256))
    if kind in ("prompt", "train"):
        Hq = Hkv * G
        scores, products = (1 << 31) // Hq, (1 << 38) // (Hq * N)  # B T^2 at most: memory of the plain form, work
        T = _log_uniform(rng, 1, min(8192, math.isqrt(min(scores, products))))
        B = _log_uniform(rng, 1, max(1, min(32, 32768 // T, min(scores, products) // (T * T))))
        return _case(None, kind, B, T, Hq, Hkv, N, dtype=dtype)
    if kind == "step":
        n = 1 if rng.random() < 0.4 else _log_uniform(rng, 2, 64)
        T = _log_uniform(rng, n, 65536)
        B = _log_uniform(rng, 1, max(1, min(64, (1 << 27) // (T * Hkv * N), (1 << 30) // (T * Hkv * G * n))))
        return _case(None, kind, B, T, Hkv * G, Hkv, N, n=n, page=page, dtype=dtype)
    n = {"verify": _log_uniform(rng, 2, 64), "beams": 1, "refill": 0}[kind]
    T = _log_uniform(rng, 64 + n, 8192)
    B = _log_uniform(rng, 2, max(2, min(64, (1 << 26) // (T * Hkv * N))))
    return _case(None, kind, B, T, Hkv * G, Hkv, N, n=n, page=page, dtype=dtype)


def _lengths(c):
    """Sequence lengths of a case: the longest first, then spread over [least, T]; of eight or more, one of length 1
    and (without new tokens to hold) one of length 0."""
    B, T, least = c["B"], c["T"], max(c["n"], 1)
    lens = [T] + [max(least, int(T * (0.15 + 0.85 * ((0.618034 * i) % 1.0)))) for i in range(1, B)]
    if B >= 8 and c["kind"] in ("prompt", "train"):
        lens[3], lens[5] = 1, 0
    return lens


def _max_pages(c):
    return -(-(c["T"] + c["n"]) // c["page"])


def _held(c):
    return [-(-t // c["page"]) for t in _lengths(c)]


def _pool(c):
    """Pages of the pool: what the sequences hold, and room for a step's new and copied pages."""
    held = sum(_held(c))
    return held + held // 4 + c["B"] * (2 + c["n"] // c["page"]) + 1


def _accepted(c, s):
    """How many drafted tokens of sequence s are kept."""
    return (5 * s + 3) % min(c["n"] + 1, 8)


def prepare(case, seed):
    c, dt = case, DTYPES[case["dtype"]]
    g = torch.Generator(DEVICE).manual_seed(int(seed))

    def normal(*shape):
        return torch.randn(*shape, device=DEVICE, generator=g, dtype=torch.float32).to(dt)

    B, Hq, Hkv, N, n, page = c["B"], c["Hq"], c["Hkv"], c["N"], c["n"], c["page"]
    lens = _lengths(c)
    s = {"case": c}
    if c["kind"] in ("prompt", "train"):
        total = sum(lens)
        offsets = torch.zeros(B + 1, dtype=torch.int64)
        offsets[1:] = torch.tensor(lens).cumsum(0)
        s["cu"] = offsets.to(device=DEVICE, dtype=torch.int32)
        s["q"], s["k"], s["v"] = normal(total, Hq, N), normal(total, Hkv, N), normal(total, Hkv, N)
        if c["kind"] == "train":
            s["do"] = normal(total, Hq, N)
            for name in ("q", "k", "v"):
                s[name].requires_grad_(True)
        return s
    # A cache whose pages lie in the pool as serving leaves them: in no order.
    P, M, held = _pool(c), _max_pages(c), torch.tensor(_held(c), device=DEVICE)
    order = torch.randperm(P, device=DEVICE, generator=g)
    slot = torch.arange(M, device=DEVICE)[None, :]
    first = (held.cumsum(0) - held)[:, None]
    s["table"] = torch.where(slot < held[:, None], order[(first + slot).clamp(max=P - 1)], -1).to(torch.int32)
    s["refs"] = torch.zeros(P, dtype=torch.int32, device=DEVICE)
    s["refs"][order[: int(sum(_held(c)))]] = 1
    s["lengths"] = torch.tensor(lens, dtype=torch.int32, device=DEVICE)
    s["status"] = torch.zeros(1, dtype=torch.int32, device=DEVICE)
    s["pool_k"], s["pool_v"] = normal(P, Hkv, page, N), normal(P, Hkv, page, N)
    s["back"] = s["lengths"].clone()
    if n > 1:
        # A drafted tree: every token hangs on the sequence or on an earlier token.
        at = torch.arange(n, device=DEVICE)
        up = (torch.rand(B, n, device=DEVICE, generator=g) * (at + 1)).long().clamp(max=n) - 1
        mask = torch.zeros(B, n, n, dtype=torch.bool, device=DEVICE)
        node = at.expand(B, n)
        for _ in range(n):
            mask |= (at[None, None, :] == node[:, :, None]) & (node >= 0)[:, :, None]
            node = torch.where(node >= 0, up.gather(1, node.clamp(min=0)), -1)
        s["mask"] = mask
    if c["kind"] == "step":
        s["q"] = normal(B, n, Hq, N)
    if c["kind"] == "verify":
        s["k"], s["v"] = normal(B, n, Hkv, N), normal(B, n, Hkv, N)
        most = min(n, 8)
        s["counts"] = torch.tensor([_accepted(c, b) for b in range(B)], dtype=torch.int32, device=DEVICE)
        s["path"] = torch.rand(B, n, device=DEVICE, generator=g).argsort(1)[:, :most].sort(1).values.to(torch.int32)
    if c["kind"] == "beams":
        s["k"], s["v"] = normal(B, n, Hkv, N), normal(B, n, Hkv, N)
        lo = torch.arange(B, device=DEVICE) // 8 * 8
        width = torch.minimum(torch.full_like(lo, 8), B - lo)
        s["parents"] = (lo + (torch.rand(B, device=DEVICE, generator=g) * width).long().clamp(max=7)).to(torch.int32)
        s["lengths"].copy_(s["lengths"][lo])  # the beams of a prompt are equally long ...
        s["back"].copy_(s["lengths"])
        fill = torch.randperm(P, device=DEVICE, generator=g)  # ... and share its whole pages
        full = (s["lengths"] // page)[:, None]
        rest = (s["lengths"][:, None] % page > 0) & (slot == full)
        s["table"] = torch.where(slot < full, s["table"][lo], torch.where(rest, -2, -1).to(torch.int32))
        s["refs"].zero_()
        used = s["table"][s["table"] >= 0].long()
        s["refs"].index_add_(0, used, torch.ones_like(used, dtype=torch.int32))
        spare = fill[s["refs"][fill] == 0]
        s["table"][s["table"] == -2] = spare[: int(rest.sum())].to(torch.int32)
        s["refs"][spare[: int(rest.sum())]] = 1
    if c["kind"] == "refill":
        even = torch.arange(B, device=DEVICE) % 2
        s["turn"] = 0
        s["keep"], s["cu"], s["k"], s["v"] = [], [], [], []
        for part in (0, 1):
            new = torch.where(even == part, s["lengths"], 0)
            s["keep"].append(torch.where(even == part, 0, s["lengths"]).to(torch.int32))
            offsets = torch.zeros(B + 1, dtype=torch.int32, device=DEVICE)
            offsets[1:] = new.cumsum(0)
            s["cu"].append(offsets)
            total = sum(t for i, t in enumerate(lens) if i % 2 == part)
            s["k"].append(normal(total, Hkv, N))
            s["v"].append(normal(total, Hkv, N))
    if own:
        s["cache"] = _package().PagedKVCache(s["pool_k"], s["pool_v"], s["table"], s["lengths"], s["refs"], s["status"])
    return s


def _package():
    import memory_efficient_attn_layer_amd

    return memory_efficient_attn_layer_amd


def run(state):
    kind = state["case"]["kind"]
    if own:
        ops = _package()
        if kind == "prompt":
            return ops.grouped_attn_varlen(state["q"], state["k"], state["v"], state["cu"])
        if kind == "train":
            o = ops.grouped_attn_varlen(state["q"], state["k"], state["v"], state["cu"])
            return (o.detach(), *torch.autograd.grad(o, (state["q"], state["k"], state["v"]), state["do"]))
        cache = state["cache"]
        if kind == "step":
            return ops.tree_attn(state["q"], cache, state.get("mask"))
        if kind == "verify":
            cache.append(state["k"], state["v"])
            cache.accept(state["case"]["n"], state["path"], state["counts"])
            cache.truncate(state["back"])
        elif kind == "beams":
            cache.fork(state["parents"])
            cache.append(state["k"], state["v"])
            cache.truncate(state["back"])
        else:
            part = state["turn"]
            state["turn"] = 1 - part
            cache.truncate(state["keep"][part])
            cache.compact()
            cache.append(state["k"][part], state["v"][part], state["cu"][part])
        return [cache.k, cache.v, cache.table, cache.lengths, cache.refs, cache.status]
    if kind == "prompt":
        return _attention(state, state["q"], state["k"], state["v"])
    if kind == "train":
        o = _attention(state, state["q"], state["k"], state["v"])
        return (o.detach(), *torch.autograd.grad(o, (state["q"], state["k"], state["v"]), state["do"]))
    if kind == "step":
        return _step(state)
    if kind == "verify":
        _append(state, state["k"].flatten(0, 1), state["v"].flatten(0, 1), None)
        _accept(state, state["path"], state["counts"])
        _truncate(state, state["back"])
    elif kind == "beams":
        _fork(state, state["parents"])
        _append(state, state["k"].flatten(0, 1), state["v"].flatten(0, 1), None)
        _truncate(state, state["back"])
    else:
        part = state["turn"]
        state["turn"] = 1 - part
        _truncate(state, state["keep"][part])
        _compact(state)
        _append(state, state["k"][part], state["v"][part], state["cu"][part])
    return [state["pool_k"], state["pool_v"], state["table"], state["lengths"], state["refs"], state["status"]]


# ---- plain forms -----------------------------------------------------------


def _attention(s, q, k, v):
    """Causal attention of packed sequences as one padded batch, query heads grouped under their key head."""
    c = s["case"]
    B, T, Hkv, N, G = c["B"], c["T"], c["Hkv"], c["N"], c["Hq"] // c["Hkv"]
    cu = s["cu"].long()
    pos = torch.arange(T, device=DEVICE)
    tok = torch.minimum(cu[:-1, None] + pos[None, :], cu[-1] - 1)
    qp = q.float()[tok].reshape(B, T, Hkv, G, N).permute(0, 2, 3, 1, 4).reshape(B, Hkv, G * T, N)
    kp = k.float()[tok].permute(0, 2, 1, 3)
    vp = v.float()[tok].permute(0, 2, 1, 3)
    a = torch.matmul(qp, kp.transpose(2, 3)).view(B, Hkv, G, T, T) * (1.0 / math.sqrt(N))
    a = a.masked_fill(pos[None, :] > pos[:, None], float("-inf"))
    p = torch.exp(a - a.amax(-1, keepdim=True).detach())
    p = p / p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(B, Hkv, G * T, T), vp).view(B, Hkv, G, T, N).permute(0, 3, 1, 2, 4)
    at = torch.arange(q.shape[0], device=DEVICE)
    b = torch.searchsorted(cu[1:], at, right=True)
    return o.reshape(B, T, Hkv * G, N)[b, at - cu[b]].to(q.dtype)


def _step(s):
    """Attention of the last n rows' queries over the pages of their sequences."""
    c = s["case"]
    B, n, Hkv, N, page, G = c["B"], c["n"], c["Hkv"], c["N"], c["page"], c["Hq"] // c["Hkv"]
    L = s["table"].shape[1] * page
    pages = s["table"].long().clamp(min=0)
    k = s["pool_k"][pages].permute(0, 2, 1, 3, 4).reshape(B, Hkv, L, N).float()
    v = s["pool_v"][pages].permute(0, 2, 1, 3, 4).reshape(B, Hkv, L, N).float()
    q = s["q"].float().reshape(B, n, Hkv, G, N).permute(0, 2, 3, 1, 4).reshape(B, Hkv, G * n, N)
    a = torch.matmul(q, k.transpose(2, 3)).view(B, Hkv, G, n, L) * (1.0 / math.sqrt(N))
    rel = torch.arange(L, device=DEVICE)[None, :] - (s["lengths"].long() - n)[:, None]  # row among the new ones
    seen = (rel < 0)[:, None, :].expand(B, n, L)
    new = rel.clamp(0, n - 1)[:, None, :].expand(B, n, L)
    tree = s["mask"].gather(2, new) if "mask" in s else torch.ones_like(seen)
    seen = seen | (tree & ((rel >= 0) & (rel < n))[:, None, :])
    a = a.masked_fill(~seen[:, None, None], float("-inf"))
    top = a.amax(-1, keepdim=True)
    p = torch.exp(a - torch.where(top == float("-inf"), 0.0, top))
    den = p.sum(-1, keepdim=True)
    p = p / torch.where(den == 0, 1.0, den)
    v = torch.where((rel < n)[:, None, :, None], v, 0.0)
    o = torch.matmul(p.view(B, Hkv, G * n, L), v).view(B, Hkv, G, n, N)
    return o.permute(0, 3, 1, 2, 4).reshape(B, n, Hkv * G, N).to(s["q"].dtype)


def _free_pages(s):
    """Pages without a holder first, in order; and how many there are."""
    taken = s["refs"] > 0
    return torch.argsort(taken.to(torch.int8), stable=True), (~taken).sum()


def _drop(s, gone):
    """The table's entries at ``gone`` (B, M) leave their pages."""
    page = s["table"].long().clamp(min=0)
    s["refs"].index_add_(0, page.flatten(), -gone.flatten().to(torch.int32))
    s["table"].masked_fill_(gone, -1)


def _write(pool, page, row, rows, ok):
    """pool[page, :, row] = rows where ok; elsewhere the pool stays."""
    first = ok.to(torch.int8).argmax()  # the others repeat one that is written; with none, what is there is written back
    page, row = torch.where(ok, page, page[first]), torch.where(ok, row, row[first])
    rows = torch.where(ok[:, None, None], rows, rows[first])
    pool[page, :, row] = torch.where(ok.any(), rows, pool[page, :, row])


def _append(s, k, v, cu):
    c = s["case"]
    B, n, page = c["B"], c["n"], c["page"]
    M = s["table"].shape[1]
    old = s["lengths"].long()
    more = (cu[1:] - cu[:-1]).long() if cu is not None else torch.full_like(old, n)
    fits = old + more <= M * page
    held, last = (old + page - 1) // page, (old + more + page - 1) // page
    tail = s["table"].long().gather(1, (old // page).clamp(max=M - 1)[:, None])[:, 0].clamp(min=0)
    copy = (old % page > 0) & (more > 0) & (s["refs"][tail] > 1)
    need = torch.where(fits, last - held + copy, 0)
    done = need.cumsum(0)
    free, count = _free_pages(s)
    room = (done <= count) | (need == 0)
    ok = fits & room & (more > 0)
    s["status"] |= ((~room).any().to(torch.int32) + 2 * (~fits).any().to(torch.int32)).to(torch.int32)
    slot = torch.arange(M, device=DEVICE)[None, :]
    taken = ok[:, None] & ((copy[:, None] & (slot == held[:, None] - 1)) | ((slot >= held[:, None]) & (slot < last[:, None])))
    rank = (done - need)[:, None] + taken.cumsum(1) - 1
    given = free[rank.clamp(0, free.shape[0] - 1)]
    copy = copy & ok
    s["refs"].index_add_(0, tail, -copy.to(torch.int32))
    s["refs"].index_add_(0, torch.where(taken, given, 0).flatten(), taken.flatten().to(torch.int32))
    s["table"].copy_(torch.where(taken, given.to(torch.int32), s["table"]))
    # Rows of the copied last pages, then the new rows.
    fresh = s["table"].long().gather(1, (old // page).clamp(max=M - 1)[:, None])[:, 0].clamp(min=0)
    row = torch.arange(page, device=DEVICE)
    part = (copy[:, None] & (row[None, :] < (old % page)[:, None])).flatten()
    at_new, at_old = fresh.repeat_interleave(page, output_size=B * page), tail.repeat_interleave(page, output_size=B * page)
    rows = row.repeat(B)
    if c["kind"] == "beams":  # (no page is shared in the other cases)
        _write(s["pool_k"], at_new, rows, s["pool_k"][at_old, :, rows], part)
        _write(s["pool_v"], at_new, rows, s["pool_v"][at_old, :, rows], part)
    tok = torch.arange(k.shape[0], device=DEVICE)
    if cu is not None:
        b = torch.searchsorted(cu[1:].contiguous(), tok.to(torch.int32), right=True)
        into = old[b] + tok - cu[b]
    else:
        b = tok // n
        into = old[b] + tok % n
    at = s["table"].long()[b, (into // page).clamp(max=M - 1)].clamp(min=0)
    _write(s["pool_k"], at, into % page, k, ok[b])
    _write(s["pool_v"], at, into % page, v, ok[b])
    s["lengths"] += torch.where(ok, more, 0).to(torch.int32)


def _accept(s, path, counts):
    """Rows of the accepted path move to the front of the tree; the pages behind are left (none is shared here)."""
    c = s["case"]
    B, n, page = c["B"], c["n"], c["page"]
    M, most = s["table"].shape[1], path.shape[1]
    old = s["lengths"].long()
    base = (old - n).clamp(min=0)
    count = torch.minimum(counts.long().clamp(0, most), old - base)
    i = torch.arange(most, device=DEVICE)[None, :].expand(B, most)
    source = base[:, None] + torch.minimum(path.long().clamp(min=0), (old - base - 1).clamp(min=0)[:, None])
    target = base[:, None] + i
    table = s["table"].long().clamp(min=0)
    from_page = table.gather(1, (source // page).clamp(max=M - 1)).flatten()
    to_page = table.gather(1, (target // page).clamp(max=M - 1)).flatten()
    ok = (i < count[:, None]).flatten()
    from_row, to_row = (source % page).flatten(), (target % page).flatten()
    k, v = s["pool_k"][from_page, :, from_row], s["pool_v"][from_page, :, from_row]
    _write(s["pool_k"], to_page, to_row, k, ok)
    _write(s["pool_v"], to_page, to_row, v, ok)
    _truncate(s, (base + count).to(torch.int32))


def _truncate(s, lengths):
    page = s["case"]["page"]
    old = s["lengths"].long()
    new = torch.minimum(lengths.long().clamp(min=0), old)
    slot = torch.arange(s["table"].shape[1], device=DEVICE)[None, :]
    _drop(s, (slot >= ((new + page - 1) // page)[:, None]) & (slot < ((old + page - 1) // page)[:, None]))
    s["lengths"].copy_(new.to(torch.int32))


def _fork(s, parents):
    p = parents.long()
    live = (p >= 0) & (p < p.shape[0])
    p = torch.where(live, p, 0)
    table = torch.where(live[:, None], s["table"][p], -1)
    entries = torch.cat((table.flatten(), s["table"].flatten()))
    by = torch.cat((torch.ones_like(table).flatten(), -torch.ones_like(table).flatten()))
    s["refs"].index_add_(0, entries.long().clamp(min=0), torch.where(entries >= 0, by, 0))
    s["lengths"].copy_(torch.where(live, s["lengths"][p], 0))
    s["table"].copy_(table)


def _compact(s):
    """The pages in use move to the front of the pool: the k-th one behind the front to the k-th free one in it."""
    P = s["refs"].shape[0]
    used = s["refs"] > 0
    live = used.sum()
    at = torch.arange(P, device=DEVICE)
    moves, holes = used & (at >= live), ~used & (at < live)
    source = torch.argsort((~moves).to(torch.int8), stable=True)
    target = torch.argsort((~holes).to(torch.int8), stable=True)
    moved = at < moves.sum()
    came, went = torch.arange(P + 1, device=DEVICE), torch.arange(P + 1, device=DEVICE)  # (entry P: not moved)
    came[torch.where(moved, target, P)] = source
    went[torch.where(moved, source, P)] = target
    came, went = came[:P], went[:P]
    s["pool_k"].copy_(s["pool_k"][came])
    s["pool_v"].copy_(s["pool_v"][came])
    s["table"].copy_(torch.where(s["table"] >= 0, went[s["table"].long().clamp(min=0)].to(torch.int32), s["table"]))
    s["refs"].copy_(torch.where(moves, 0, s["refs"][came]))


# ---- work and definition ---------------------------------------------------


def work(case):
    c = case
    lens, N, Hq, Hkv, n = _lengths(c), c["N"], c["Hq"], c["Hkv"], c["n"]
    if c["kind"] in ("prompt", "train"):
        total, pairs = sum(lens), sum(t * (t + 1) // 2 for t in lens)
        rows = 2 * total * N
        moved, flops = rows * (2 * Hq + 2 * Hkv), 4 * Hq * N * pairs
        if c["kind"] == "train":
            moved, flops = rows * (4 * Hq + 4 * Hkv), int(3.5 * flops)
        return {"bytes": moved, "flops": flops}
    if c["kind"] == "step":
        return {"bytes": 4 * sum(lens) * Hkv * N + 4 * c["B"] * n * Hq * N + (c["B"] * n * n if n > 1 else 0),
                "flops": 4 * n * Hq * N * sum(lens)}
    row, page = 4 * Hkv * N, c["page"]  # one row of k and v
    if c["kind"] == "verify":
        kept = sum(_accepted(c, b) for b in range(c["B"]))
        return {"bytes": 2 * row * (c["B"] * n + kept), "flops": 0}
    if c["kind"] == "beams":
        tails = sum(lens[b // 8 * 8] % page for b in range(c["B"]))
        return {"bytes": 2 * row * (c["B"] + tails) + 8 * sum(_held(c)), "flops": 0}
    held = _held(c)
    moved, new = min(sum(held[::2]), sum(held[1::2])), sum(lens) // 2  # two passes take turns
    return {"bytes": 2 * row * (moved * page + new), "flops": 0}


def exact(case, seed):
    """Attention in 64 bits, sequence by sequence and head by head. The other cases move rows and compute nothing."""
    c = case
    if c["kind"] not in ("prompt", "train", "step"):
        return None
    s = prepare(case, seed)
    G, sl, lens = c["Hq"] // c["Hkv"], c["N"] ** -0.5, _lengths(c)
    if c["kind"] == "step":
        out = torch.zeros(c["B"], c["n"], c["Hq"], c["N"], dtype=torch.float64, device=DEVICE)
        for b, L in enumerate(lens):
            ids = s["table"][b, : -(-L // c["page"])].long()
            ctx = L - c["n"]
            for h in range(c["Hkv"]):
                k = s["pool_k"][ids, h].reshape(-1, c["N"])[:L].double()
                v = s["pool_v"][ids, h].reshape(-1, c["N"])[:L].double()
                for i in range(c["n"]):
                    seen = torch.ones(L, dtype=torch.bool, device=DEVICE)
                    if "mask" in s:
                        seen[ctx:] = s["mask"][b, i]
                    w = torch.softmax((s["q"][b, i, h * G:(h + 1) * G].double() @ k[seen].T) * sl, dim=-1)
                    out[b, i, h * G:(h + 1) * G] = w @ v[seen]
        return out
    q, k, v = (s[x].detach().double() for x in ("q", "k", "v"))
    out = torch.zeros_like(q)
    grads = [torch.zeros_like(x) for x in (q, k, v)]
    t0 = 0
    for L in lens:
        rows = slice(t0, t0 + L)
        later = torch.triu(torch.ones(L, L, dtype=torch.bool, device=DEVICE), 1)
        for h in range(c["Hq"] if L else 0):
            kv = h // G
            a = (q[rows, h] @ k[rows, kv].T) * sl
            a[later] = float("-inf")
            w = torch.softmax(a, dim=-1)
            out[rows, h] = w @ v[rows, kv]
            if c["kind"] == "train":
                d = s["do"][rows, h].double()
                dw = d @ v[rows, kv].T
                da = w * (dw - (w * dw).sum(-1, keepdim=True))
                grads[0][rows, h] = sl * (da @ k[rows, kv])
                grads[1][rows, kv] += sl * (da.T @ q[rows, h])
                grads[2][rows, kv] += w.T @ d
        t0 += L
    return out if c["kind"] == "prompt" else (out, *grads)
