"""A key/value cache of pages that sequences share and give back, and the
attention of new tokens over it.

``KVCache`` holds one block of rows per sequence, as long as the longest may
get. ``PagedKVCache`` holds a pool of pages and a table of the pages of each
sequence, so that memory follows the rows that are there, beams and samples
share their prompt, and a finished sequence's pages serve the next one:

    cache = PagedKVCache.empty(sequences, Hkv, N, pages, "cuda")
    cache.append(k, v)                    # (sequences, n, Hkv, N), or packed with offsets
    o = tree_attn(q, cache)               # (sequences, n, Hq, N): the n new tokens' rows
    cache.append(k, v); o = tree_attn(q, cache, mask)      # a drafted tree ...
    cache.accept(n, path, counts)                          # ... and what is kept of it
    cache.fork(parents); cache.truncate(lengths); cache.free([3, 5]); cache.compact()

All of it runs in libmea.so on the current stream. The tables live on the GPU and
change there in stream order: no call waits for the GPU (but ``verify`` and the
hand-over of lists), and all of them can be captured into a graph. A cache is
used by one stream at a time (its calls share a workspace). ``tree_attn`` takes no gradient, like
``decode_step``.
"""
from __future__ import annotations

from dataclasses import dataclass, field

import torch

from . import _lib
from .grouped import SUPPORTED_WIDTHS, _check_scale, _rows

PAGE_SIZES = (16, 32, 64, 128, 256)
MAX_TREE = 256  # new tokens per sequence

@dataclass(frozen=True, eq=False)
class PagedKVCache:
    """``k`` and ``v`` (pages, Hkv, page, N), bfloat16 or float16; ``table``
    (sequences, max_pages), ``lengths`` (sequences,), ``refs`` (pages,) and
    ``status`` (1,), int32. Row r of sequence s is row r % page of page
    ``table[s, r // page]``; entries past the sequence are -1; ``refs`` counts the
    entries that hold a page. ``PagedKVCache.empty`` makes one; the tensors may
    also come from elsewhere (a saved cache), and are then taken as they are."""

    k: torch.Tensor
    v: torch.Tensor
    table: torch.Tensor
    lengths: torch.Tensor
    refs: torch.Tensor
    status: torch.Tensor
    _c: _lib.MeaPaged = field(init=False, repr=False)
    _ws: torch.Tensor = field(init=False, repr=False)  # of the cache's own calls, which come one after the other
    _tree_ws: dict = field(init=False, repr=False)  # (n, Hq) -> workspace bytes of tree_attn

    @classmethod
    def empty(cls, sequences: int, H: int, N: int, pages: int, device, page: int = 64, max_pages: int | None = None,
              dtype=torch.bfloat16) -> "PagedKVCache":
        """A cache without rows for ``sequences`` sequences of up to
        ``max_pages`` (all ``pages`` by default) pages of ``page`` rows each, H
        key/value heads of N dimensions."""
        max_pages = pages if max_pages is None else max_pages

        def ints(*shape, value=0):
            return torch.full(shape, value, device=device, dtype=torch.int32)

        pool = (pages, H, page, N)
        return cls(torch.zeros(pool, device=device, dtype=dtype), torch.zeros(pool, device=device, dtype=dtype),
                   ints(sequences, max_pages, value=-1), ints(sequences), ints(pages), ints(1))

    def __post_init__(self):
        for name in ("k", "v", "table", "lengths", "refs", "status"):
            t = getattr(self, name)
            if not isinstance(t, torch.Tensor) or not t.is_contiguous():
                raise ValueError(f"cache.{name} must be a contiguous tensor")
            if t.device != self.k.device:
                raise ValueError(f"cache.{name} is on {t.device}, cache.k is on {self.k.device}")
            if name in ("k", "v"):
                if t.dim() != 4 or t.shape != self.k.shape or t.dtype != self.k.dtype or t.data_ptr() % 16 != 0:
                    raise ValueError("cache.k and cache.v must be (pages, Hkv, page, N) tensors of one type")
            elif t.dtype != torch.int32:
                raise TypeError(f"cache.{name} must be int32, got {t.dtype}")
        if self.k.dtype not in _lib.MEA_DTYPES:
            raise TypeError(f"the cache must be bfloat16 or float16, got {self.k.dtype}")
        pages, H, page, N = self.k.shape
        if N not in SUPPORTED_WIDTHS:
            raise ValueError(f"head width N={N} not supported (supported: {SUPPORTED_WIDTHS})")
        if page not in PAGE_SIZES:
            raise ValueError(f"page={page} rows not supported (supported: {PAGE_SIZES})")
        if self.table.dim() != 2 or min(self.table.shape) < 1 or pages < 1 or H < 1:
            raise ValueError("cache.table must be (sequences, max_pages), the pool not empty")
        S, M = self.table.shape
        for name, n in (("lengths", S), ("refs", pages), ("status", 1)):
            if getattr(self, name).shape != (n,):
                raise ValueError(f"cache.{name} has shape {tuple(getattr(self, name).shape)}, expected ({n},)")
        c = _lib.MeaPaged(self.k.data_ptr(), self.v.data_ptr(), self.table.data_ptr(), self.lengths.data_ptr(),
                          self.refs.data_ptr(), self.status.data_ptr(), S, pages, H, page, N, M,
                          _lib.MEA_DTYPES[self.k.dtype])
        object.__setattr__(self, "_c", c)
        ws_bytes = _lib.load().mea_paged_workspace_bytes(c)
        if ws_bytes == 0:
            raise ValueError(f"cache of {S} sequences, {pages} pages and {M} pages a sequence is out of range")
        object.__setattr__(self, "_ws", torch.empty(ws_bytes, device=self.k.device, dtype=torch.uint8))
        object.__setattr__(self, "_tree_ws", {})

    @property
    def sequences(self) -> int:
        return self.table.shape[0]

    @property
    def page(self) -> int:
        return self.k.shape[2]

    @property
    def capacity(self) -> int:
        """Rows a sequence can have."""
        return self.table.shape[1] * self.page

    def append(self, k, v, cu_seqlens=None) -> None:
        """Writes new rows behind the sequences and makes them longer: k and v
        (sequences, n, Hkv, N), n for each, or (total, Hkv, N) with the
        sequences + 1 offsets ``cu_seqlens``, cu[s+1] - cu[s] for sequence s (a
        list or CPU tensor is checked, an int32 device tensor trusted). Pages
        are taken as needed, the lowest free ones first, sequence by sequence; a
        page that other sequences hold too is copied before rows are written
        into it. A sequence for which there are too few pages, or that would
        pass the capacity, stays as it is; see ``verify``. k and v must not be
        parts of the pool."""
        self._on_gpu()
        S, (_, H, _, N) = self.sequences, self.k.shape
        packed = cu_seqlens is not None
        for name, t in (("k", k), ("v", v)):
            if not isinstance(t, torch.Tensor) or t.shape != (
                    (k.shape[0], H, N) if packed else (S, k.shape[1] if k.dim() > 1 else 0, H, N)):
                shape = tuple(t.shape) if isinstance(t, torch.Tensor) else type(t).__name__
                raise ValueError(f"{name} must be ({'total' if packed else f'{S}, n'}, {H}, {N}), got {shape}")
            if t.dtype != self.k.dtype or t.device != self.k.device:
                raise TypeError(f"{name} is {t.dtype} on {t.device}, the cache {self.k.dtype} on {self.k.device}")
        total = k.shape[0] if packed else S * k.shape[1]
        if packed:
            cu_seqlens = self._ints("cu_seqlens", cu_seqlens, S + 1, offsets=total)
        if total == 0:
            return
        k, v = _rows(k), _rows(v)
        st = _lib.strides(0, *k.stride()[:2], 0, *v.stride()[:2]) if packed else _lib.strides(*k.stride()[:3], *v.stride()[:3])
        with _lib.on_device(k.device):
            rc = _lib.load().mea_paged_append(self._c, k.data_ptr(), v.data_ptr(), st, _lib.ptr(cu_seqlens),
                                              0 if packed else k.shape[1], total, self._ws.data_ptr(), self._ws.shape[0],
                                              _lib.stream_of(k.device))
        _lib.check(rc, "mea_paged_append")

    def accept(self, n: int, path, counts) -> None:
        """Keeps the accepted part of a drafted tree, the last ``n`` rows of each
        sequence: row i of the tree becomes its row ``path[s, i]`` for
        i < ``counts[s]``, the other rows go. ``path`` (sequences, most <= n) and
        ``counts`` (sequences,): int32 device tensors or lists. Values are
        clamped to the tree."""
        self._on_gpu()
        n = int(n)
        if not 1 <= n <= MAX_TREE:
            raise ValueError(f"n={n} must be in [1, {MAX_TREE}]")
        if not isinstance(path, torch.Tensor):
            path = torch.tensor(path)
            if path.dtype != torch.int64 or int(path.abs().max()) >= 1 << 31:
                raise ValueError("path must hold 32-bit ints")
            path = path.to(device=self.k.device, dtype=torch.int32)
        if (path.dim() != 2 or path.shape[0] != self.sequences or not 1 <= path.shape[1] <= n
                or path.dtype != torch.int32 or path.device != self.k.device):
            raise ValueError(f"path must be an int32 tensor ({self.sequences}, 1 .. {n}) on {self.k.device}")
        path, counts = path.contiguous(), self._ints("counts", counts, self.sequences)
        with _lib.on_device(path.device):
            rc = _lib.load().mea_paged_accept(self._c, n, path.data_ptr(), path.shape[1], counts.data_ptr(),
                                              self._ws.data_ptr(), self._ws.shape[0], _lib.stream_of(path.device))
        _lib.check(rc, "mea_paged_accept")

    def truncate(self, lengths) -> None:
        """Sequence s keeps its first ``lengths[s]`` rows (at most those it has)
        and gives back the pages behind them. ``lengths``: (sequences,), an int32
        device tensor or a list."""
        self._on_gpu()
        lengths = self._ints("lengths", lengths, self.sequences)
        with _lib.on_device(lengths.device):
            rc = _lib.load().mea_paged_truncate(self._c, lengths.data_ptr(), _lib.stream_of(lengths.device))
        _lib.check(rc, "mea_paged_truncate")

    def free(self, sequences) -> None:
        """The listed sequences (ints) end: no rows, their pages given back."""
        keep = [self.capacity] * self.sequences
        for s in sequences:
            if not 0 <= int(s) < self.sequences:
                raise ValueError(f"sequence {s} is not in [0, {self.sequences})")
            keep[int(s)] = 0
        self.truncate(keep)

    def fork(self, parents) -> None:
        """Sequence s goes on as what sequence ``parents[s]`` is now, sharing its
        pages (each writes into pages of its own from then on); -1 (or any other
        value outside the sequences): it ends. ``parents``: (sequences,), an int32
        device tensor or a list."""
        self._on_gpu()
        parents = self._ints("parents", parents, self.sequences)
        with _lib.on_device(parents.device):
            rc = _lib.load().mea_paged_fork(self._c, parents.data_ptr(), self._ws.data_ptr(), self._ws.shape[0],
                                            _lib.stream_of(parents.device))
        _lib.check(rc, "mea_paged_fork")

    def compact(self) -> None:
        """Moves the pages in use to the front of the pool: afterwards they are
        pages 0 .. (how many there are) - 1."""
        self._on_gpu()
        dev = self.k.device
        with _lib.on_device(dev):
            rc = _lib.load().mea_paged_compact(self._c, self._ws.data_ptr(), self._ws.shape[0], _lib.stream_of(dev))
        _lib.check(rc, "mea_paged_compact")

    def verify(self) -> None:
        """Waits for the GPU and raises RuntimeError if an earlier call found too
        few pages or rows for a sequence (and left it as it was)."""
        status = int(self.status.item())
        if status != 0:
            self.status.zero_()
            what = [text for bit, text in ((_lib.MEA_PAGED_NO_PAGES, "the pool ran out of pages"),
                                           (_lib.MEA_PAGED_NO_ROWS, f"a sequence would pass {self.capacity} rows"))
                    if status & bit]
            raise RuntimeError("PagedKVCache: " + " and ".join(what))

    def _on_gpu(self) -> None:
        if not self.k.is_cuda:
            raise RuntimeError("PagedKVCache runs only on a ROCm GPU device (there is no CPU path)")

    def _ints(self, name: str, values, n: int, offsets: int | None = None) -> torch.Tensor:
        """``values`` as an int32 device tensor of n entries (``offsets``: the
        tokens that n offsets on the host must cover)."""
        dev = self.k.device
        if not isinstance(values, torch.Tensor) or (offsets is not None and values.device.type == "cpu"):
            values = torch.as_tensor(values)
            if values.dim() != 1 or values.numel() != n or values.dtype.is_floating_point or values.dtype == torch.bool:
                raise ValueError(f"{name} must have {n} entries, all ints")
            if int(values.min()) < -(1 << 31) or int(values.max()) >= 1 << 31:
                raise ValueError(f"{name} must hold 32-bit ints")
            if offsets is not None:
                from .attention import check_offsets

                check_offsets([int(x) for x in values.tolist()], offsets)
            return values.to(device=dev, dtype=torch.int32)
        if values.shape != (n,) or values.dtype != torch.int32 or values.device != dev:
            raise ValueError(f"{name} must be an int32 tensor of shape ({n},) on {dev}")
        return values.contiguous()


def tree_attn(q, cache: PagedKVCache, mask=None, scale=None) -> torch.Tensor:
    """Attention of the n newest tokens of every sequence over its rows of the
    cache, their own among them (``append`` their k and v first): q
    (sequences, n, Hq, N), n <= 256, or (sequences, Hq, N) for one token each;
    returns the shape of q. Every token sees all rows in front of the n newest;
    of those, token i sees token j where ``mask[..., i, j]``, a bool tensor
    (sequences, n, n) or (n, n) (a drafted tree: its ancestors and itself), or,
    without a mask, where j <= i. A token that sees no row gets zeros. Hq is a
    multiple of the cache's heads; ``scale`` defaults to 1 / sqrt(N)."""
    if not isinstance(q, torch.Tensor) or q.dim() not in (3, 4):
        raise ValueError("q must be a (sequences, n, Hq, N) or (sequences, Hq, N) tensor")
    q4 = q.unsqueeze(1) if q.dim() == 3 else q
    S, n, Hq, N = q4.shape
    pages, H, _, Nc = cache.k.shape
    if q.dtype != cache.k.dtype:
        raise TypeError(f"q is {q.dtype}, the cache is {cache.k.dtype}")
    if q.device != cache.k.device:
        raise ValueError(f"q is on {q.device}, the cache is on {cache.k.device}")
    if S != cache.sequences or N != Nc:
        raise ValueError(f"q must be ({cache.sequences}, n, Hq, {Nc}), got {tuple(q.shape)}")
    if not 1 <= n <= MAX_TREE:
        raise ValueError(f"n={n} new tokens must be in [1, {MAX_TREE}]")
    if Hq < 1 or Hq % H != 0:
        raise ValueError(f"{Hq} query heads are no multiple of the cache's {H}")
    scale = _check_scale(scale, N)
    mask_seq = 0
    if mask is not None:
        if not isinstance(mask, torch.Tensor) or mask.dtype != torch.bool or mask.shape not in ((n, n), (S, n, n)):
            raise ValueError(f"mask must be a bool tensor of shape ({n}, {n}) or ({S}, {n}, {n})")
        if mask.device != q.device:
            raise ValueError(f"mask is on {mask.device}, q is on {q.device}")
        mask = mask.contiguous()
        mask_seq = n * n if mask.dim() == 3 else 0
    cache._on_gpu()
    lib = _lib.load()
    dev = q.device
    q4 = _rows(q4)
    o = torch.empty((S, n, Hq, N), device=dev, dtype=q.dtype)
    ws_bytes = cache._tree_ws.get((n, Hq))
    if ws_bytes is None:
        ws_bytes = cache._tree_ws[(n, Hq)] = lib.mea_tree_workspace_bytes(cache._c, n, Hq)
    ws = torch.empty(ws_bytes, device=dev, dtype=torch.uint8) if ws_bytes else None
    with _lib.on_device(dev):
        rc = lib.mea_tree_attn(cache._c, n, Hq, scale, q4.data_ptr(), _lib.strides(*q4.stride()[:3]), _lib.ptr(mask), mask_seq,
                               o.data_ptr(), _lib.ptr(ws), ws_bytes, _lib.stream_of(dev))
    _lib.check(rc, "mea_tree_attn")
    return o if q.dim() == 4 else o[:, 0]


__all__ = ["PagedKVCache", "tree_attn", "PAGE_SIZES", "MAX_TREE"]
