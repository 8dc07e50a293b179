"""Paged KV cache: keys and values in pages of a pool that sequences take, share and give back.

The contiguous cache (:mod:`.kv_cache`) grows by moving, and holds one batch.  Here a pool holds
pages of ``page`` slots, ``k_pages`` / ``v_pages`` ``[P, H, page, D]`` (head-major in a page, as the
contiguous cache is), and every row of a batch names its pages in ``tables`` ``[B, W]``: slot ``j``
of row ``b`` is place ``j % page`` of page ``tables[b, j // page]``.  The operators

* :func:`paged_kv_append` - rotary of the new keys, then keys and values into their slots,
* :func:`paged_attention` / :func:`paged_attention_with_lse` - attention over a row's slots, one new
  token or a chunk of them, by the masking rule and with the ``(out, lse)`` convention of
  :mod:`.attention`,
* :func:`paged_tree_attention` / :func:`paged_tree_attention_with_lse` - the same for a tree of drafted
  tokens in the row's last slots (:func:`tree_masks` from the nodes' parents),
* :func:`paged_kv_keep` - the accepted nodes' rows moved into line, in all layers' pools,
* :func:`paged_kv_read` - a row's slots as contiguous keys and values,
* :func:`copy_pages` - copies of whole pages through all layers' pools,

read tables and lengths on the device, so nothing waits for the host and a captured graph follows
what its tensors hold.  A page index outside the pool is a page that holds nothing.  The kernels read them
more than once, so nothing may write to them (from another stream, say) before the call's work is done.

Pages of ``torch.float8_e4m3fn`` take half the memory, and half the reads of a decode step.  With them go
``k_scales`` / ``v_scales`` ``[P, H, page]`` (uint8): the numbers ``q`` of a slot and head stand for
``q * 2^(s - 127)``, ``s`` its scale byte, 1 to 254.  The append chooses it per row: ``s - 127`` is the smallest
whole number ``e >= -117`` with ``max |x| <= 448 * 2^e``.  Values keep 4 significant bits (half a step is
``2^-4`` of a value); infinities and NaN become NaN.

:class:`PageBook` keeps which sequence holds which pages (sharing, copy on write, compaction) on the
host, and :class:`PagedKVCache` is the pools of a model's layers with their book.
"""

from __future__ import annotations

import heapq
import math
import operator
from typing import Dict, List, Optional, Sequence, Tuple, Union

import torch

from . import _native as nat
from .attention import KVMap, _check_heads, _kv_map_list


def paged_kv_append(k_pages: torch.Tensor, v_pages: torch.Tensor, tables: torch.Tensor,
                    offsets: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *,
                    cos: Optional[torch.Tensor] = None, sin: Optional[torch.Tensor] = None,
                    counts: Optional[torch.Tensor] = None,
                    pos_pages: Optional[torch.Tensor] = None,
                    pos: Optional[torch.Tensor] = None,
                    k_scales: Optional[torch.Tensor] = None,
                    v_scales: Optional[torch.Tensor] = None) -> None:
    """Writes ``k`` (rotated with ``cos``/``sin`` ``[B, n, D]`` when given) and ``v`` ``[B, n, H, D]``
    into row ``b``'s slots ``offsets[b] .. offsets[b] + counts[b] - 1``, in place.

    ``counts`` ``[B]`` says how many of a row's ``n`` tokens there are (all without it); ``pos``
    ``[B, n]`` goes into ``pos_pages`` ``[P, page]`` where the cache keeps positions.  The rotation
    is that of :func:`~.layers.apply_rotary`, rounded once at its end (``apply_rotary`` rounds its
    products too).  A slot is written by one token: pages that rows share are full ones, or copied
    before (:func:`copy_pages`).  Tokens of slots that a row has no page for are dropped.

    Into 8-bit pages (with both scales) go rows of bf16, f16 or f32; keys are rotated in f32 and rounded to
    e4m3 alone.
    """
    if (cos is None) != (sin is None):
        raise ValueError("give both rotary tables or neither")
    if (pos is None) != (pos_pages is None):
        raise ValueError("give both pos and pos_pages or neither")
    if v.dtype != k.dtype:
        raise ValueError("k and v must share one dtype")
    _check_pages(k.dtype, k_pages, v_pages, k_scales, v_scales, "k, v")
    nat.ops().paged_kv_append(k_pages, v_pages, pos_pages, tables, offsets, counts, k, v, pos, cos,
                              sin, k_scales, v_scales)


def _check_pages(dtype, k_pages, v_pages, k_scales, v_scales, what):
    if k_scales is None and v_scales is None:
        if k_pages.dtype != dtype or v_pages.dtype != dtype:
            raise ValueError(f"{what}, k_pages and v_pages must share a dtype, got {dtype}, "
                             f"{k_pages.dtype}, {v_pages.dtype} (8-bit pages need their scales)")
    elif k_scales is None or v_scales is None:
        raise ValueError("give both scales or neither")
    elif k_pages.dtype != torch.float8_e4m3fn or v_pages.dtype != torch.float8_e4m3fn:
        raise ValueError(f"scales go with float8_e4m3fn pages, got {k_pages.dtype}, {v_pages.dtype}")


def _check_attention(q, k_pages, v_pages, k_scales, v_scales, scale, kv_map):
    if q.dim() != 4 or k_pages.dim() != 4:
        raise ValueError("q must be [B, S, H, D] and k_pages [P, H, page, D]")
    _check_pages(q.dtype, k_pages, v_pages, k_scales, v_scales, "q")
    mapping = _kv_map_list(kv_map)
    _check_heads(q.shape[2], k_pages.shape[1], mapping)
    return 1.0 / math.sqrt(q.shape[-1]) if scale is None else float(scale), mapping


def _attend(q, k_pages, v_pages, tables, lengths, q_pos, pos_pages, causal, scale, kv_map, with_lse,
            k_scales, v_scales):
    scale, mapping = _check_attention(q, k_pages, v_pages, k_scales, v_scales, scale, kv_map)
    return nat.ops().paged_attention(q, k_pages, v_pages, pos_pages, tables, lengths, q_pos,
                                     bool(causal), scale, mapping, with_lse, k_scales, v_scales)


def paged_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                    tables: torch.Tensor, lengths: torch.Tensor, q_pos: torch.Tensor, *,
                    pos_pages: Optional[torch.Tensor] = None, causal: bool = True,
                    scale: Optional[float] = None, kv_map: KVMap = None,
                    k_scales: Optional[torch.Tensor] = None,
                    v_scales: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of ``q`` ``[B, S, H, D]`` over slots ``0 .. lengths[b]-1`` of each row's pages;
    returns ``[B, S, H, D]`` in ``q.dtype``.

    The position of slot ``j`` is ``j``, or what ``pos_pages`` ``[P, page]`` holds there when given
    (a rank's share of a sequence, unused slots as -1); a key is visible as in
    :func:`~.attention.attention`.  Queries with position -1 are padding under the causal rule; rows
    without a visible key are 0.  The new tokens are appended first, and ``lengths`` counts them.
    What hidden slots hold does not reach a result, infinities and NaN included.

    Probabilities keep f32's bits for single and few tokens (up to 16 query rows of a KV head); those of
    bf16 and f16 chunks on the matrix cores are rounded to the type once before they weigh the values, so
    a row's result may differ by such a rounding with the number of tokens in the call.
    :func:`paged_attention_with_lse` keeps them in every form.

    8-bit pages (with both scales) are attended as the values that they stand for, by queries of bf16, f16
    or f32; f16 ones meet values that f16 holds (f16 rows leave no others in the pages).
    """
    return _attend(q, k_pages, v_pages, tables, lengths, q_pos, pos_pages, causal, scale, kv_map,
                   False, k_scales, v_scales)[0]


def paged_attention_with_lse(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                             tables: torch.Tensor, lengths: torch.Tensor, q_pos: torch.Tensor, *,
                             pos_pages: Optional[torch.Tensor] = None, causal: bool = True,
                             scale: Optional[float] = None, kv_map: KVMap = None,
                             k_scales: Optional[torch.Tensor] = None,
                             v_scales: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """:func:`paged_attention` returning ``(out, lse)`` in accumulation precision, for the exact
    merges of partial results (:func:`~.attention.merge_attention`); empty rows give ``(0, -inf)``."""
    out, lse = _attend(q, k_pages, v_pages, tables, lengths, q_pos, pos_pages, causal, scale, kv_map,
                       True, k_scales, v_scales)
    return out, lse


def tree_masks(parents: torch.Tensor, counts: Optional[torch.Tensor] = None
               ) -> Tuple[torch.Tensor, torch.Tensor]:
    """``(masks, depths)`` of trees of up to 512 drafted tokens, on the device.

    ``parents`` ``[B, T]`` names each node's parent, an earlier node; anything else (-1) makes a node
    follow the sequence itself.  ``masks`` ``[B, T, ceil(T / 64)]`` (int64) has bit ``j % 64`` of word ``j //
    64`` set in node ``i``'s row where ``j`` is ``i`` or one of its ancestors; ``depths`` ``[B, T]`` counts a
    node's ancestors, so its position is that of the first new slot plus its depth.  Nodes from
    ``counts[b]`` on have no bits and depth 0.
    """
    masks, depths = nat.ops().tree_masks(parents, counts)
    return masks, depths


def _tree(q, k_pages, v_pages, tables, lengths, counts, masks, scale, kv_map, with_lse, k_scales, v_scales):
    scale, mapping = _check_attention(q, k_pages, v_pages, k_scales, v_scales, scale, kv_map)
    if masks.dim() == 3 and masks.shape[0] == 1 and q.shape[0] != 1:
        masks = masks.expand(q.shape[0], -1, -1)
    return nat.ops().paged_tree_attention(q, k_pages, v_pages, k_scales, v_scales, tables, lengths, counts,
                                          masks, scale, mapping, with_lse)


def paged_tree_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                         tables: torch.Tensor, lengths: torch.Tensor, counts: torch.Tensor,
                         masks: torch.Tensor, *, scale: Optional[float] = None, kv_map: KVMap = None,
                         k_scales: Optional[torch.Tensor] = None,
                         v_scales: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of ``q`` ``[B, T, H, D]``, the nodes of a tree of drafted tokens in the last ``counts[b]``
    of each row's ``lengths[b]`` slots; returns ``[B, T, H, D]`` in ``q.dtype``.

    Node ``i`` is in slot ``lengths[b] - counts[b] + i``, appended like any token.  It sees every slot
    before the tree, and the slots of the nodes ``j`` whose bit is set in ``masks`` ``[B, T, ceil(T / 64)]``
    (int64, bit ``j % 64`` of word ``j // 64``; a first dimension of 1 is every row's): those of
    :func:`tree_masks`, or any other.  Nodes from ``counts[b]`` on are padding, and 0, as is a node that
    sees nothing.  ``T`` is up to 512.  Precision, 8-bit pages and what hidden slots may hold are
    :func:`paged_attention`'s.
    """
    return _tree(q, k_pages, v_pages, tables, lengths, counts, masks, scale, kv_map, False, k_scales,
                 v_scales)[0]


def paged_tree_attention_with_lse(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                                  tables: torch.Tensor, lengths: torch.Tensor, counts: torch.Tensor,
                                  masks: torch.Tensor, *, scale: Optional[float] = None,
                                  kv_map: KVMap = None, k_scales: Optional[torch.Tensor] = None,
                                  v_scales: Optional[torch.Tensor] = None
                                  ) -> Tuple[torch.Tensor, torch.Tensor]:
    """:func:`paged_tree_attention` returning ``(out, lse)`` in accumulation precision (for a rank that
    holds the tree and a share of the sequence; the other ranks' shares by :func:`paged_attention_with_lse`)."""
    out, lse = _tree(q, k_pages, v_pages, tables, lengths, counts, masks, scale, kv_map, True, k_scales,
                     v_scales)
    return out, lse


def paged_kv_keep(kv: torch.Tensor, tables: torch.Tensor, offsets: torch.Tensor, path: torch.Tensor, *,
                  counts: Optional[torch.Tensor] = None, scales: Optional[torch.Tensor] = None) -> None:
    """Moves the accepted nodes of a tree into line, in place: slot ``offsets[b] + i`` of row ``b`` takes
    what slot ``offsets[b] + path[b, i]`` held, in every pool of ``kv`` ``[..., P, H, page, D]`` (all
    layers' keys and values; what precedes the pages collapses into one dimension, and a head's slots of a page are
    contiguous, so pools of ``[P, page, H, D]`` seen as these are refused) and of ``scales`` ``[..., P, H, page]``,
    which 8-bit pages have.

    ``path`` ``[B, n]`` names the accepted nodes in order, on the device, padded with -1.  A node is never
    before its place in line, so entries below their index move nothing, nor do those from ``counts[b]`` on,
    the row's nodes, where ``counts`` ``[B]`` is given.
    """
    nat.ops().paged_kv_keep(kv, scales, tables, offsets, counts, path)


def paged_kv_read(k_pages: torch.Tensor, v_pages: torch.Tensor, tables: torch.Tensor,
                  offsets: torch.Tensor, n: int, *, counts: Optional[torch.Tensor] = None,
                  dtype: Optional[torch.dtype] = None, k_scales: Optional[torch.Tensor] = None,
                  v_scales: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """``(k, v)`` ``[B, n, H, D]``: what row ``b``'s slots ``offsets[b] .. offsets[b] + counts[b] - 1`` hold
    (``n`` of them without ``counts``, and at most), and 0 from there on and where a row has no page.

    8-bit pages are read as ``dtype``: bf16 (the default), f16 or f32, which hold their values as they are (but
    for magnitudes outside f16's normal numbers, which are rounded); others as their own.
    """
    if dtype is None:
        dtype = torch.bfloat16 if k_pages.dtype == torch.float8_e4m3fn else k_pages.dtype
    if k_scales is None and v_scales is None:
        _check_pages(dtype, k_pages, v_pages, None, None, "dtype")
    else:
        _check_pages(None, k_pages, v_pages, k_scales, v_scales, "dtype")
    k, v = nat.ops().paged_kv_read(k_pages, v_pages, k_scales, v_scales, tables, offsets, counts,
                                   operator.index(n), dtype)
    return k, v


def _page_list(pages: Union[torch.Tensor, Sequence[int]]) -> torch.Tensor:
    if isinstance(pages, torch.Tensor):
        return pages
    try:
        return torch.tensor([operator.index(p) for p in pages], dtype=torch.int64)
    except TypeError:
        raise ValueError("page indices must be whole numbers") from None


def copy_pages(pools: Union[torch.Tensor, Sequence[torch.Tensor]],
               src: Union[torch.Tensor, Sequence[int]], dst: Union[torch.Tensor, Sequence[int]], *,
               dim: int = 0) -> None:
    """Copies page ``src[i]`` to page ``dst[i]`` in every pool, in place.

    ``pools`` is a tensor or up to 16 of them, with the pages along ``dim``: what follows it is
    contiguous, and what precedes it (layers, keys and values) holds more pools of the same pages.
    ``src`` and ``dst`` are host lists (the pages are handed out on the host): they go with the
    launch, without a transfer, and a captured call copies the same pages on every replay.
    ``ValueError`` if a page is written twice, or both read and written, or does not exist, and for
    indices that are not whole numbers.
    """
    pools = [pools] if isinstance(pools, torch.Tensor) else list(pools)
    nat.ops().copy_pages(pools, int(dim), _page_list(src), _page_list(dst))


class PageBook:
    """Which sequence holds which pages of a pool, on the host.

    A page is held by one sequence, or by several that share a prefix (:meth:`fork`); a sequence
    gets a page of its own before it writes into one that others hold.  The lowest free page is
    handed out first.  A call that fails changes nothing.
    """

    def __init__(self, pages: int, page: int) -> None:
        if pages < 1 or page < 1:
            raise ValueError("a pool needs at least one page of at least one slot")
        self.pages, self.page = int(pages), int(page)
        self._free: List[int] = list(range(self.pages))  # a heap
        self._holders: List[int] = [0] * self.pages
        self._tables: Dict[int, List[int]] = {}
        self._lengths: Dict[int, int] = {}
        self._next = 0

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def length(self, seq: int) -> int:
        return self._lengths[self._known(seq)]

    def table(self, seq: int) -> List[int]:
        return list(self._tables[self._known(seq)])

    def sequences(self) -> List[int]:
        return list(self._tables)

    def _known(self, seq: int) -> int:
        if seq not in self._tables:
            raise ValueError(f"no sequence {seq}")
        return seq

    def new(self) -> int:
        """A new sequence without tokens."""
        seq, self._next = self._next, self._next + 1
        self._tables[seq], self._lengths[seq] = [], 0
        return seq

    def fork(self, seq: int) -> int:
        """A new sequence with the tokens of ``seq``, on the same pages."""
        pages, length = self._tables[self._known(seq)], self._lengths[seq]
        child = self.new()
        self._tables[child], self._lengths[child] = list(pages), length
        for p in pages:
            self._holders[p] += 1
        return child

    def _give_back(self, page: int) -> None:
        self._holders[page] -= 1
        if self._holders[page] == 0:
            heapq.heappush(self._free, page)

    def free(self, seq: int) -> None:
        """Ends a sequence; the pages that nobody else holds are free."""
        for p in self._tables.pop(self._known(seq)):
            self._give_back(p)
        del self._lengths[seq]

    def truncate(self, seq: int, length: int) -> None:
        """Drops the tokens of ``seq`` from ``length`` on (rejected drafts)."""
        if not 0 <= length <= self.length(seq):
            raise ValueError(f"sequence {seq} has {self._lengths[seq]} tokens, not {length}")
        keep = -(-length // self.page)
        for p in self._tables[seq][keep:]:
            self._give_back(p)
        del self._tables[seq][keep:]
        self._lengths[seq] = length

    def extend(self, seqs: Sequence[int], counts: Sequence[int]) -> List[Tuple[int, int]]:
        """Adds ``counts[i]`` tokens to ``seqs[i]``, with the pages they need; returns the page copies
        ``(from, to)`` that have to be done before they are written.  ``RuntimeError`` when the pool
        has too few free pages."""
        if len(seqs) != len(counts) or len(set(seqs)) != len(seqs):
            raise ValueError("need distinct sequences with a count each")
        counts = [operator.index(n) for n in counts]
        if any(n < 0 for n in counts):
            raise ValueError("counts must not be negative")
        need, left = 0, {}
        for seq, n in zip(seqs, counts):
            table, length = self._tables[self._known(seq)], self._lengths[seq]
            need += max(0, -(-(length + n) // self.page) - len(table))
            if n and length % self.page:
                last = table[-1]
                holders = left.get(last, self._holders[last])
                if holders > 1:
                    need += 1
                    left[last] = holders - 1
        if need > len(self._free):
            raise RuntimeError(f"the cache is full: {need} pages needed, {len(self._free)} free")
        copies = []
        for seq, n in zip(seqs, counts):
            table = self._tables[seq]
            if n and self._lengths[seq] % self.page and self._holders[table[-1]] > 1:
                page = self._take()
                copies.append((table[-1], page))
                self._holders[table[-1]] -= 1
                table[-1] = page
            self._lengths[seq] += n
            while len(table) * self.page < self._lengths[seq]:
                table.append(self._take())
        return copies

    def _retract(self, seqs: Sequence[int], lengths: Sequence[int],
                 copies: List[Tuple[int, int]]) -> None:
        """Takes the last :meth:`extend` back, given the lengths before it and what it returned."""
        came_from = {b: a for a, b in copies}
        for seq, length in zip(seqs, lengths):
            self.truncate(seq, length)
            table = self._tables[seq]
            if table and table[-1] in came_from:
                own, table[-1] = table[-1], came_from[table[-1]]
                self._holders[table[-1]] += 1
                self._give_back(own)

    def _take(self) -> int:
        page = heapq.heappop(self._free)
        self._holders[page] = 1
        return page

    def compact(self) -> List[Tuple[int, int]]:
        """Renames the held pages to the lowest indices; returns the page copies ``(from, to)`` that
        have to be done before the tables are used."""
        moves = self._moves()
        self._rename(moves)
        return moves

    def _moves(self) -> List[Tuple[int, int]]:
        held = [p for p in range(self.pages) if self._holders[p]]
        holes = [p for p in range(len(held)) if not self._holders[p]]
        return list(zip((p for p in reversed(held) if p >= len(held)), holes))

    def _rename(self, moves: List[Tuple[int, int]]) -> None:
        to = dict(moves)
        for table in self._tables.values():
            table[:] = [to.get(p, p) for p in table]
        for a, b in moves:
            self._holders[b], self._holders[a] = self._holders[a], 0
        self._free = [p for p in range(self.pages) if not self._holders[p]]


class PagedStep:
    """The device side of one step of :class:`PagedKVCache`: ``tables`` ``[B, W]``, ``offsets``,
    ``counts`` and ``lengths`` ``[B]`` (int64), the views of one buffer."""

    def __init__(self, rows: int, width: int, device) -> None:
        self.buffer = torch.empty(rows * (width + 3), dtype=torch.int64, device=device)
        self.tables = self.buffer[3 * rows:].view(rows, width)
        self.offsets, self.counts, self.lengths = self.buffer[:3 * rows].view(3, rows)
        self.cache, self.epoch = None, -1
        self.most = 0  # new tokens of a row at most
        self.seqs: List[int] = []  # the rows' sequences, and their lengths before the step and with it
        self.starts: List[int] = []
        self.ends: List[int] = []


class PagedKVCache:
    """The paged key/value cache of a model's layers on one device.

    One allocation ``[layers, 2, P, H, page, D]`` for keys and values, shared page tables for all
    layers, and with ``positions`` a pool of the slots' positions (for a rank that holds a share of
    each sequence; otherwise slot ``j`` is position ``j``).  A model's step is::

        step = cache.extend(seqs, counts)              # pages for the new tokens, copies on write
        for layer in range(layers):
            cache.append(layer, step, k, v, cos=cos, sin=sin)
            out = cache.attention(layer, step, q, q_pos)

    With a tree of drafted tokens in each row::

        step = cache.extend(seqs, nodes)
        masks, depths = tree_masks(parents)
        for layer in range(layers):                    # tables of position offset + depth
            cache.append(layer, step, k, v, cos=cos, sin=sin)
            out = cache.tree_attention(layer, step, q, masks)
        cache.keep(step, path, kept)                   # the accepted nodes, the others are dropped

    With ``dtype=torch.float8_e4m3fn`` keys and values are held in 8 bits, with their scale bytes.

    A step made before :meth:`fork`, :meth:`free`, :meth:`truncate` or :meth:`compact` is refused
    after it: its pages may be another's (a fork shares tokens, so they are written before it).
    Everything runs on the current stream.  A captured graph holds appends and attention; ``extend``
    and ``compact`` come between its replays, and are refused in a capture, which would not run them.
    One thread at a time calls a cache.
    """

    def __init__(self, layers: int, pages: int, page: int, heads: int, head_dim: int, *,
                 dtype: torch.dtype = torch.bfloat16, device="cuda", positions: bool = False) -> None:
        self.book = PageBook(pages, page)
        self.kv = torch.empty(layers, 2, pages, heads, page, head_dim, dtype=dtype, device=device)
        self.scales = (torch.empty(layers, 2, pages, heads, page, dtype=torch.uint8, device=device)
                       if dtype == torch.float8_e4m3fn else None)
        self.pos_pages = (torch.full((pages, page), -1, dtype=torch.int64, device=device)
                          if positions else None)
        self._epoch = 0

    def pages(self, layer: int) -> Tuple[torch.Tensor, torch.Tensor]:
        """``(k_pages, v_pages)`` of a layer."""
        return self.kv[layer, 0], self.kv[layer, 1]

    def _scales(self, layer: int) -> Dict[str, torch.Tensor]:
        """The arguments that 8-bit pages add to a call."""
        if self.scales is None:
            return {}
        return {"k_scales": self.scales[layer, 0], "v_scales": self.scales[layer, 1]}

    @property
    def free_pages(self) -> int:
        return self.book.free_pages

    def length(self, seq: int) -> int:
        return self.book.length(seq)

    def new(self) -> int:
        """A new sequence without tokens."""
        return self.book.new()

    def fork(self, seq: int) -> int:
        """A new sequence that shares the tokens of ``seq``; the page that both would write next is
        copied when one of them is extended."""
        child = self.book.fork(seq)
        self._epoch += 1
        return child

    def free(self, seq: int) -> None:
        """Ends a sequence and gives its pages back."""
        self.book.free(seq)
        self._epoch += 1

    def truncate(self, seq: int, length: int) -> None:
        """Drops the tokens of ``seq`` from ``length`` on."""
        self.book.truncate(seq, length)
        self._epoch += 1

    def _copy(self, moves: List[Tuple[int, int]]) -> None:
        if not moves:
            return
        src, dst = zip(*moves)
        pools = [self.kv.flatten(0, 1)]
        if self.scales is not None:
            pools.append(self.scales.flatten(0, 1))
        if self.pos_pages is not None:
            pools.append(self.pos_pages.unsqueeze(0))
        copy_pages(pools, src, dst, dim=1)

    def _outside_capture(self, what: str) -> None:
        if self.kv.is_cuda and torch.cuda.is_current_stream_capturing():
            raise RuntimeError(f"{what} belongs before a graph's replay, not into its capture")

    def compact(self) -> int:
        """Moves the held pages to the lowest indices; returns how many moved."""
        self._outside_capture("compact")
        moves = self.book._moves()
        self._copy(moves)  # (into free pages: a copy that fails changes no table)
        self.book._rename(moves)
        self._epoch += 1
        return len(moves)

    def extend(self, seqs: Sequence[int], counts: Union[int, Sequence[int]],
               into: Optional[PagedStep] = None) -> PagedStep:
        """Room for ``counts[i]`` new tokens of ``seqs[i]`` (0: the sequence is only read) and the
        step's tensors.  With ``into`` a step of the same number of rows is filled in place, its
        width allowing, for a captured graph that reads it (its appends write as many tokens a row as
        they were captured with, so ``counts`` stays within those).  A call that fails adds no tokens."""
        self._outside_capture("extend")
        seqs = list(seqs)
        counts = [int(counts)] * len(seqs) if isinstance(counts, int) else [operator.index(n) for n in counts]
        if into is not None:
            if into.tables.shape[0] != len(seqs):
                raise ValueError(f"the step has {into.tables.shape[0]} rows, not {len(seqs)}")
            if len(counts) == len(seqs):
                page = self.book.page
                widest = max((-(-(self.length(s) + max(n, 0)) // page) for s, n in zip(seqs, counts)),
                             default=0)
                if widest > into.tables.shape[1]:
                    raise ValueError(f"the step is {into.tables.shape[1]} pages wide, {widest} needed")
        offsets = [self.length(s) for s in seqs]
        copies = self.book.extend(seqs, counts)
        try:
            self._copy(copies)
            tables = [self.book.table(s) for s in seqs]
            step = into
            if step is None:
                step = PagedStep(len(seqs), max(map(len, tables), default=0), self.kv.device)
            width = step.tables.shape[1]
            host = offsets + counts + [self.length(s) for s in seqs]
            for t in tables:
                host += t + [-1] * (width - len(t))
            staged = torch.tensor(host, dtype=torch.int64, pin_memory=self.kv.is_cuda)
            step.buffer.copy_(staged, non_blocking=True)
        except BaseException:  # (no memory for the step, a copy refused: without a step nothing is added)
            self.book._retract(seqs, offsets, copies)
            raise
        step.cache, step.epoch, step.most = self, self._epoch, max(counts, default=0)
        step.seqs, step.starts, step.ends = seqs, offsets, host[2 * len(seqs):3 * len(seqs)]
        return step

    def _check(self, step: PagedStep) -> None:
        if step.cache is not self:
            raise RuntimeError("the step is not this cache's")
        if step.epoch != self._epoch:
            raise RuntimeError("the step is older than the last fork, free, truncate or compact")

    def append(self, layer: int, step: PagedStep, k: torch.Tensor, v: torch.Tensor, *,
               cos: Optional[torch.Tensor] = None, sin: Optional[torch.Tensor] = None,
               pos: Optional[torch.Tensor] = None) -> None:
        """Writes a layer's new keys and values (:func:`paged_kv_append`); rows with fewer new tokens
        than ``k`` and ``v`` hold are padded."""
        self._check(step)
        if k.dim() == 4 and k.shape[1] < step.most:
            raise ValueError(f"the step adds up to {step.most} tokens to a row, k holds {k.shape[1]}")
        k_pages, v_pages = self.pages(layer)
        paged_kv_append(k_pages, v_pages, step.tables, step.offsets, k, v, cos=cos, sin=sin,
                        counts=step.counts, pos_pages=self.pos_pages, pos=pos, **self._scales(layer))

    def attention(self, layer: int, step: PagedStep, q: torch.Tensor, q_pos: torch.Tensor, *,
                  causal: bool = True, scale: Optional[float] = None, kv_map: KVMap = None
                  ) -> torch.Tensor:
        """A layer's attention over the step's sequences (:func:`paged_attention`)."""
        self._check(step)
        return paged_attention(q, *self.pages(layer), step.tables, step.lengths, q_pos,
                               pos_pages=self.pos_pages, causal=causal, scale=scale, kv_map=kv_map,
                               **self._scales(layer))

    def attention_with_lse(self, layer: int, step: PagedStep, q: torch.Tensor, q_pos: torch.Tensor,
                           *, causal: bool = True, scale: Optional[float] = None,
                           kv_map: KVMap = None) -> Tuple[torch.Tensor, torch.Tensor]:
        """The same with the log-sum-exp (:func:`paged_attention_with_lse`)."""
        self._check(step)
        return paged_attention_with_lse(q, *self.pages(layer), step.tables, step.lengths, q_pos,
                                        pos_pages=self.pos_pages, causal=causal, scale=scale,
                                        kv_map=kv_map, **self._scales(layer))

    def tree_attention(self, layer: int, step: PagedStep, q: torch.Tensor, masks: torch.Tensor, *,
                       scale: Optional[float] = None, kv_map: KVMap = None) -> torch.Tensor:
        """A layer's attention of the step's new tokens as trees (:func:`paged_tree_attention`)."""
        self._check_tree(step)
        if q.dim() == 4 and q.shape[1] < step.most:
            raise ValueError(f"the step adds up to {step.most} tokens to a row, q holds {q.shape[1]}")
        return paged_tree_attention(q, *self.pages(layer), step.tables, step.lengths, step.counts, masks,
                                    scale=scale, kv_map=kv_map, **self._scales(layer))

    def _check_tree(self, step: PagedStep) -> None:
        self._check(step)
        if self.pos_pages is not None:
            raise NotImplementedError("trees take a cache without positions of its own")

    def keep(self, step: PagedStep, path: torch.Tensor, kept: Sequence[int]) -> None:
        """Keeps the accepted nodes of the step's trees as the sequences' next tokens and drops the others:
        row ``b`` keeps ``kept[b]`` nodes, the first of ``path[b]`` ``[B, n]`` (indices in order, on the
        device).  ``kept`` is on the host, as the lengths are; the step is used up."""
        self._check_tree(step)
        self._outside_capture("keep")
        kept = [operator.index(n) for n in kept]
        if path.dim() != 2 or path.shape[0] != len(step.seqs) or len(kept) != len(step.seqs):
            raise ValueError(f"path must be [{len(step.seqs)}, n], with a count each")
        for seq, start, end, n in zip(step.seqs, step.starts, step.ends, kept):
            if self.length(seq) != end:
                raise RuntimeError(f"sequence {seq} was extended after the step")
            if not 0 <= n <= min(end - start, path.shape[1]):
                raise ValueError(f"sequence {seq} cannot keep {n} of {end - start} nodes, "
                                 f"{path.shape[1]} in the path")
        paged_kv_keep(self.kv, step.tables, step.offsets, path, counts=step.counts, scales=self.scales)
        for seq, start, n in zip(step.seqs, step.starts, kept):
            self.book.truncate(seq, start + n)
        self._epoch += 1

    def read(self, layer: int, step: PagedStep, n: int, *, dtype: Optional[torch.dtype] = None
             ) -> Tuple[torch.Tensor, torch.Tensor]:
        """The first ``n`` slots of the step's sequences in a layer as ``(k, v)`` ``[B, n, H, D]``, 0 behind
        a sequence's end (:func:`paged_kv_read`)."""
        self._check(step)
        return paged_kv_read(*self.pages(layer), step.tables, torch.zeros_like(step.lengths), n,
                             counts=step.lengths, dtype=dtype, **self._scales(layer))


__all__ = [
    "PageBook",
    "PagedKVCache",
    "PagedStep",
    "copy_pages",
    "paged_attention",
    "paged_attention_with_lse",
    "paged_kv_append",
    "paged_kv_keep",
    "paged_kv_read",
    "paged_tree_attention",
    "paged_tree_attention_with_lse",
    "tree_masks",
]
