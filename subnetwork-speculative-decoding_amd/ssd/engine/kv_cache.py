"""Shared KV cache for target and draft (reference ssd/engine/kv_cache.py).

One arena per cache in HBM, keyed by *base* layer index like the reference's slots:
``k`` and ``vt`` are each [layers, kv_heads, max_len * head_dim] bf16, max_len a multiple of 64,
in the 64-slot block layout of csrc/common.h (k_off / v_off): every 64-slot block of K is stored
as the tree-attention kernel's S = K Q^T operand tiles and every block of V as its O = V^T P^T
operand tiles, each tile in lane order, so the kernel reads a block as contiguous 1 KiB loads.
``read`` / ``ops.kv_untile`` give the plain [kv_heads, slots, head_dim] view.

Writes happen inside the fused q/k/v + RoPE GEMM epilogue; ``keep_positions`` (the
accepted-path compaction) is one kernel launch over every layer. ``seq_len`` bookkeeping,
``advance``/``crop``/``reset`` and the overflow ``RuntimeError`` follow the reference
(kv_cache.py:21-73). Batch size is 1, as in the reference's speculative decoding.
"""

from __future__ import annotations

from typing import Optional

import torch

from ssd import _lib, ops


class KVCache:
    def __init__(self, num_slots: int, max_length: int, kv_heads: Optional[int] = None,
                 head_dim: Optional[int] = None, device=None):
        self.num_slots = num_slots
        self.max_length = max_length
        # Slot capacity in whole 64-slot blocks (the block layout's unit).
        self.capacity = (max_length + 63) // 64 * 64
        self.seq_len = 0
        self.kv_heads, self.head_dim, self.device = kv_heads, head_dim, device
        self.k: Optional[torch.Tensor] = None
        self.vt: Optional[torch.Tensor] = None
        if kv_heads is not None and head_dim is not None and device is not None:
            self._alloc()

    def _alloc(self) -> None:
        shape = (self.num_slots, self.kv_heads, self.capacity * self.head_dim)
        self.k = torch.zeros(shape, dtype=torch.bfloat16, device=self.device)
        self.vt = torch.zeros(shape, dtype=torch.bfloat16, device=self.device)

    def ensure(self, kv_heads: int, head_dim: int, device) -> None:
        if self.k is None:
            self.kv_heads, self.head_dim, self.device = kv_heads, head_dim, torch.device(device)
            self._alloc()

    def get_seq_length(self) -> int:
        return self.seq_len

    def check_room(self, end: int) -> None:
        if end > self.max_length:
            raise RuntimeError(f"KVCache overflow: {end} > max_length={self.max_length}")

    def layer(self, i: int) -> tuple[torch.Tensor, torch.Tensor]:
        return self.k[i], self.vt[i]

    def update(self, slot: int, k: torch.Tensor, v: torch.Tensor):
        """Write k/v [1, kv_heads, q, hd] at [seq_len, seq_len+q) of base layer ``slot`` and return
        plain copies [1, kv_heads, seq_len+q, hd] of K and V (API form of the reference's update;
        decoding writes in-kernel)."""
        q = k.shape[2]
        end = self.seq_len + q
        self.check_room(end)
        self.ensure(k.shape[1], k.shape[3], k.device)
        k_idx, v_idx = ops.kv_block_index(self.capacity, self.head_dim, self.k.device)
        self.k[slot][:, k_idx[self.seq_len:end]] = k[0].to(torch.bfloat16)
        self.vt[slot][:, v_idx[self.seq_len:end]] = v[0].to(torch.bfloat16)
        kk, vv = self.read(slot, end)
        return kk[None], vv[None]

    def read(self, slot: int, end: int) -> tuple[torch.Tensor, torch.Tensor]:
        """Plain copies K, V [kv_heads, end, head_dim] of slots [0, end) of base layer ``slot``."""
        k_idx, v_idx = ops.kv_block_index(self.capacity, self.head_dim, self.k.device)
        return self.k[slot][:, k_idx[:end]], self.vt[slot][:, v_idx[:end]]

    def advance(self, n: int) -> None:
        self.seq_len += n

    def crop(self, length: int) -> None:
        if length > self.seq_len:
            raise ValueError(f"cannot crop to {length} > current length {self.seq_len}")
        self.seq_len = length

    def keep_positions(self, start: int, positions) -> None:
        """Move entries ``positions`` (absolute, >= start) to [start, start+n) in every layer
        with one kernel launch; sources are all read before any destination is written."""
        pos = positions.tolist() if isinstance(positions, torch.Tensor) else list(positions)
        n = len(pos)
        if n == 0 or pos == list(range(start, start + n)) or self.k is None:
            self.seq_len = start + n
            return
        if min(pos) < start or max(pos) >= self.capacity:
            raise ValueError("keep_positions: positions out of range")
        src = torch.tensor(pos, dtype=torch.int32).to(self.device)
        n_dev = torch.tensor([n], dtype=torch.int32).to(self.device)
        ops.kv_compact(self.k, self.vt, self.num_slots, self.kv_heads, self.head_dim, self.capacity, start, src,
                       n_dev, n)
        self.seq_len = start + n

    def compact_device(self, start: int, src: torch.Tensor, n_dev: torch.Tensor, n_max: int,
                       pos_base: Optional[torch.Tensor] = None) -> None:
        """Compaction with sources and count already on the device (the engine's path: no host sync);
        with ``pos_base`` the destination start is relative to that device word."""
        ops.kv_compact(self.k, self.vt, self.num_slots, self.kv_heads, self.head_dim, self.capacity, start, src,
                       n_dev, n_max, pos_base)

    def reset(self) -> None:
        self.seq_len = 0


class KVCacheQ8:
    """KV caches of ``sequences`` sequences in 8 bits: e4m3 codes and one power-of-two exponent per (slot, kv head) of
    K and of V, 2 * (head_dim + 1) bytes a slot and head against the bf16 cache's 4 * head_dim. Arrays
    [layers, sequences, kv_heads, capacity * head_dim] (codes) and [..., capacity] (exponents), in the operand order
    documented at SsdKvQ8 in the C header. head_dim 64 or 128. ``capacity`` is max_length rounded up to a multiple of 64, and
    the bound of every call: a sequence has slots [0, capacity), places outside them are outside the cache.

    Rows are quantised as they are written (``write``, K rotated in the same launch), every stored value is a bf16
    value, so ``read`` returns exactly what ``attend`` uses. Lengths are the caller's: rows name their sequence and slot.
    ``span`` (keys per record of the attention, a multiple of 64) is part of the arithmetic: rows of two caches agree
    bit for bit when their keys, queries and spans do. None: ``default_span``."""

    def __init__(self, num_slots: int, max_length: int, kv_heads: int, head_dim: int, device, sequences: int = 1,
                 span: Optional[int] = None):
        if head_dim not in (64, 128):
            raise ValueError(f"KVCacheQ8: head_dim {head_dim} unsupported (64, 128)")
        if min(num_slots, max_length, kv_heads, sequences) < 1:
            raise ValueError("KVCacheQ8: layers, max_length, kv_heads and sequences must be positive")
        if span is not None and (not 64 <= span <= 1 << 20 or span % 64):
            raise ValueError(f"KVCacheQ8: span {span} must be a multiple of 64 up to 2^20")
        self.num_slots, self.max_length = num_slots, max_length
        self.kv_heads, self.head_dim, self.sequences = kv_heads, head_dim, sequences
        self.capacity = (max_length + 63) // 64 * 64
        self.span = self.default_span(self.capacity) if span is None else span
        lead = (num_slots, sequences, kv_heads)
        codes = dict(dtype=torch.uint8, device=device)
        self.k = torch.zeros(*lead, self.capacity * head_dim, **codes)
        self.v = torch.zeros_like(self.k)
        self.k_exp = torch.full((*lead, self.capacity), 127, **codes)
        self.v_exp = torch.full_like(self.k_exp, 127)
        self.device = self.k.device
        self._layers = [_lib.SsdKvQ8(self.k[i].data_ptr(), self.v[i].data_ptr(), self.k_exp[i].data_ptr(),
                                     self.v_exp[i].data_ptr(), sequences, kv_heads, head_dim, self.capacity)
                        for i in range(num_slots)]
        for i, d in enumerate(self._layers):  # a descriptor keeps its arrays, and knows how many layers they hold from its own on
            # (no reference of ctypes to itself: such a cycle is never collected, nor are the arrays on it)
            d.arrays, d.layers, d.device_index = (self.k, self.v, self.k_exp, self.v_exp), num_slots - i, self.k.get_device()

    @staticmethod
    def default_span(capacity: int) -> int:
        """Keys of a span (one wave's work in turn; four spans leave one record): short ones for latency, long ones for
        fewer records. us at 64 / 128 / 256 / 512 / 1024 keys, 32 heads on 8 kv heads of 128, one row: 4096 keys 7.9 / 8.9 /
        10.3 / 18.5 / 20.7, 8100 10.3 / 10.4 / 12.0 / 16.5 / 32, 16384 11.6 / 10.3 / 12.4 / 17.0 / 27, 33000 25 / 24 / 20.4 / 19.9 /
        29; 25 rows: 19.6 / 15.6 / 16.1 / 19.0 / 24, 25 / 21.5 / 19.3 / 27 / 37, 38 / 30 / 27 / 24 / 33, 62 / 46 / 40 / 37 / 37. Caches that end
        with a few blocks: 13 trees of 9 rows at 98 keys 10.3 / 12.3 at 64 / 128."""
        return 64 if capacity <= 256 else 128 if capacity < 6144 else 256 if capacity < 16384 else 512

    def layer(self, i: int) -> _lib.SsdKvQ8:
        """The descriptor of layer ``i`` for the ops that take a cache."""
        return self._layers[i]

    def write(self, i: int, k: torch.Tensor, v: torch.Tensor, seq: torch.Tensor, slot: torch.Tensor, rope=None, pos=None,
              interleaved: bool = False, q: Optional[torch.Tensor] = None,
              q_out: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
        """Rows k, v [M, kv_heads * head_dim] (any row stride) into layer ``i`` at (seq[m], slot[m]) (int32 on the device,
        all places different; rows at slots outside [0, capacity) or of no sequence are not written). ``rope``: (cos, sin)
        tables of ``models.llama.rope_tables_f32``, K rotated to ``pos`` before it is quantised; with ``q``
        [M, heads * head_dim] its rows are rotated too and returned (in ``q_out`` if given, which may be ``q``)."""
        heads = 0 if q is None else self._heads(q)
        return ops.kv_q8_write(self._layers[i], k, v, k.shape[0], seq, slot, rope, pos, interleaved, q, heads, q_out)

    def _heads(self, q: torch.Tensor) -> int:
        heads, rest = divmod(q.shape[-1], self.head_dim)
        if rest:
            raise ValueError(f"q has {q.shape[-1]} columns, not a multiple of head_dim {self.head_dim}")
        return heads

    def load(self, i: int, cache: KVCache, length: int, seq: int = 0, start: int = 0) -> None:
        """Slots [start, length) of a bf16 cache's layer ``i`` (a prompt's, after its prefill) into sequence ``seq``."""
        if not 0 <= start <= length <= self.capacity or not 0 <= seq < self.sequences:
            raise ValueError(f"KVCacheQ8.load: slots [{start}, {length}) or sequence {seq} outside the cache")
        if (cache.kv_heads, cache.head_dim) != (self.kv_heads, self.head_dim) or length > cache.max_length:
            raise ValueError(f"KVCacheQ8.load: {length} slots of {self.kv_heads} heads of {self.head_dim} from a cache with "
                             f"{cache.max_length} of {cache.kv_heads} of {cache.head_dim}")
        k, v = (x[:, start:].transpose(0, 1).flatten(1) for x in cache.read(i, length))
        slot = torch.arange(start, length, dtype=torch.int32, device=self.device)
        self.write(i, k, v, torch.full_like(slot, seq), slot)

    def read(self, i: int, seq: torch.Tensor, slot: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
        """K, V [M, kv_heads * head_dim] bf16 of layer ``i`` at (seq[m], slot[m]); zeros for slots outside [0, capacity) and
        for no sequence."""
        return ops.kv_q8_read(self._layers[i], seq.numel(), seq, slot)

    def attend_floats(self, m: int, heads: int, l_max: int) -> int:
        """Workspace floats of ``attend`` for ``m`` rows."""
        return ops.attn_q8_ws_floats(m, heads, self.head_dim, l_max, self.span)

    def attend(self, i: int, q: torch.Tensor, row_begin: torch.Tensor, prefix: torch.Tensor, depth: torch.Tensor,
               anc: torch.Tensor, rows_max: int, l_max: int, out: Optional[torch.Tensor] = None,
               ws: Optional[torch.Tensor] = None, scale: Optional[float] = None) -> torch.Tensor:
        """Tree attention of q [M, heads * head_dim] over layer ``i``: sequence s owns rows row_begin[s] ..
        row_begin[s + 1] (at most rows_max <= 64), row t attends slots [0, prefix[t]) then anc[t, :depth[t]] of anc [M, 32]
        (a depth above 32 counts as 32); zeros for rows that attend nothing; rows of no sequence are left as ``out`` has
        them (unset without ``out``). l_max <= capacity bounds prefix + depth. ``ws``: fp32, attend_floats(M, heads, l_max)
        (None: allocated here)."""
        return ops.tree_attention_q8(self._layers[i], q, q.shape[0], self._heads(q), row_begin, prefix, depth, anc, rows_max,
                                     l_max, self.span, ws, out, scale)

    def compact_device(self, start: torch.Tensor, src: torch.Tensor, n: torch.Tensor) -> None:
        """In every layer, sequence s's slots src[s, :n[s]] move to [start[s], start[s] + n[s]) (int32 on the device; src
        [sequences, n_max <= 64]): the accepted paths of a verified batch, one launch. Moves from or to slots outside
        [0, capacity) are skipped."""
        if src.dim() != 2 or src.shape[0] != self.sequences:
            raise ValueError(f"src must be [{self.sequences}, n_max], got {tuple(src.shape)}")
        ops.kv_q8_compact(self._layers[0], self.num_slots, start, src, n, src.shape[1])


class PagedBatch:
    """The sequences of a call on a paged cache, on its device (all int32): ``table`` [S, columns] (unit column stride), the page
    of slots 64 p .. 64 p + 63 of sequence s at [s, p]; ``lengths`` [S], slots in use, new rows included; ``row_begin`` [S + 1],
    sequence s's packed rows being row_begin[s] .. row_begin[s + 1] (increasing, at most ``rows_max`` each; None: one row a
    sequence). Row i of a sequence's n sits at slot lengths[s] - n + i. The tensors are read when a call runs: they may be
    updated in place between calls and between replays of a graph, and the object keeps them. ``capacity``: slots the table
    can hold."""

    def __init__(self, table: torch.Tensor, lengths: torch.Tensor, row_begin: Optional[torch.Tensor] = None, rows_max: int = 1):
        for t, name in ((table, "table"), (lengths, "lengths"), (row_begin, "row_begin")):
            if t is not None and (not isinstance(t, torch.Tensor) or t.dtype is not torch.int32 or t.device.type != "cuda"
                                  or t.device != table.device):
                got = f"{t.dtype} on {t.device}" if isinstance(t, torch.Tensor) else type(t).__name__
                raise ValueError(f"PagedBatch: {name} must be an int32 tensor on the cache's device, got {got}")
        if table.dim() != 2 or table.shape[1] < 1 or table.shape[1] > 1 and table.stride(1) != 1:
            raise ValueError(f"PagedBatch: table must be [S, >= 1] with unit column stride, got {tuple(table.shape)}, strides "
                             f"{table.stride()}")
        n, cols = table.shape
        if lengths.shape != (n,) or not lengths.is_contiguous():
            raise ValueError(f"PagedBatch: lengths must be [{n}] and contiguous, got {tuple(lengths.shape)}")
        if row_begin is not None and (row_begin.shape != (n + 1,) or not row_begin.is_contiguous()):
            raise ValueError(f"PagedBatch: row_begin must be [{n + 1}] and contiguous, got {tuple(row_begin.shape)}")
        if rows_max < 0 or row_begin is None and rows_max > 1:
            raise ValueError(f"PagedBatch: rows_max {rows_max} " + ("needs row_begin" if rows_max > 1 else "must not be negative"))
        ld = table.stride(0) if n > 1 else cols
        if ld < cols:
            raise ValueError(f"PagedBatch: the rows of table overlap (strides {table.stride()})")
        self.table, self.lengths, self.row_begin, self.rows_max = table, lengths, row_begin, rows_max
        self.n_seq, self.capacity, self.device_index = n, cols * PagedKVCache.PAGE, table.get_device()
        self.desc = _lib.SsdPagedBatch(table.data_ptr(), ld, cols, n, None if row_begin is None else row_begin.data_ptr(),
                                       lengths.data_ptr(), rows_max)


class PagedKVCache:
    """KV caches of a batch of sequences in pages of 64 slots, bf16: per layer a pool of ``pages`` pages, each with every kv head's K and
    V of its slots. A page is the same number in every layer. Which page holds what is the caller's (``PagedBatch``);
    ``alloc`` and ``free`` keep count of the unused ones. Arrays k, v [layers, pages, kv_heads, 64 * head_dim], 64 slots of a
    head in the block layout of csrc/common.h; head_dim 64 or 128. Calls that write (``write``, ``evict``) need pages that
    belong to one sequence; reads and attention may share pages (a common prefix).

    ``span``: slots of a wave's share of a group in ``attend`` (four a group; a multiple of 64 up to 4096), part of its arithmetic: rows agree bit
    for bit between calls of the same span, whatever their batch. None: by the table's width (``default_span``)."""

    PAGE = 64

    def __init__(self, num_slots: int, pages: int, kv_heads: int, head_dim: int, device, span: Optional[int] = None):
        if head_dim not in (64, 128):
            raise ValueError(f"PagedKVCache: head_dim {head_dim} unsupported (64, 128)")
        if min(num_slots, pages, kv_heads) < 1:
            raise ValueError("PagedKVCache: layers, pages and kv_heads must be positive")
        if span is not None and (not 64 <= span <= 4096 or span % 64):
            raise ValueError(f"PagedKVCache: span {span} must be a multiple of 64 up to 4096")
        self.num_slots, self.pages, self.kv_heads, self.head_dim, self.span = num_slots, pages, kv_heads, head_dim, span
        shape = (num_slots, pages, kv_heads, self.PAGE * head_dim)
        self.k = torch.zeros(shape, dtype=torch.bfloat16, device=device)
        self.v = torch.zeros_like(self.k)
        self.device = self.k.device
        self._free = list(range(pages - 1, -1, -1))
        self._layers = [_lib.SsdPagedKv(self.k[i].data_ptr(), self.v[i].data_ptr(), pages, kv_heads, head_dim)
                        for i in range(num_slots)]
        for i, d in enumerate(self._layers):  # as KVCacheQ8's
            d.arrays, d.layers, d.device_index = (self.k, self.v), num_slots - i, self.k.get_device()

    @staticmethod
    def default_span(capacity: int) -> int:
        """Slots of a wave's share for tables of ``capacity`` slots: one launch while four shares hold them all, then short ones for
        latency, long ones for fewer records. us of one row at 64 / 128 / 256 / 512 / 1024, 32 heads on 8 kv heads of 128: 500 keys
        10.4 / 8.0, 1000 10.2 / 11.2 / 9.7, 4000 10.5 / 11.0 / 12.6 / 16.2 / 20, 16000 18.6 / 18.4 / 17.9 / 19.9 / 28, 40000 35 / 35 /
        36 / 32 / 32, 131000 120 / 113 / 116 / 106 / 102; of 32 sequences of one row of up to 4000 keys 83 / 79 / 77 / 79 / 78, of six
        of 16 rows 50 / 42 / 42 / 45 / 45."""
        for most, span in ((256, 64), (512, 128), (1024, 256), (12288, 128), (32768, 256), (65536, 512)):
            if capacity <= most:
                return span
        return 1024

    # ------------------------------------------------------------------ pages
    @classmethod
    def pages_for(cls, length: int) -> int:
        """Pages that ``length`` slots take."""
        return (length + cls.PAGE - 1) // cls.PAGE

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def alloc(self, n: int) -> list:
        """``n`` unused pages; RuntimeError if there are not as many."""
        if n < 0:
            raise ValueError(f"PagedKVCache: cannot allocate {n} pages")
        if n > len(self._free):
            raise RuntimeError(f"PagedKVCache overflow: {n} pages wanted, {len(self._free)} of {self.pages} unused")
        return [self._free.pop() for _ in range(n)]

    def free(self, pages) -> None:
        """Takes pages back; work already enqueued on them on this stream runs before what reuses them."""
        pages = [int(p) for p in pages]
        if any(not 0 <= p < self.pages for p in pages) or len(set(pages)) != len(pages) or not set(pages).isdisjoint(self._free):
            raise ValueError(f"PagedKVCache: pages {pages} are not all in use")
        self._free.extend(reversed(pages))

    # ------------------------------------------------------------------ operators
    def layer(self, i: int) -> _lib.SsdPagedKv:
        """The descriptor of layer ``i`` for the ops that take a cache."""
        return self._layers[i]

    def _heads(self, q: torch.Tensor) -> int:
        heads, rest = divmod(q.shape[-1], self.head_dim)
        if rest or heads % self.kv_heads or not heads:
            raise ValueError(f"q has {q.shape[-1]} columns, not heads of {self.head_dim} in a multiple of {self.kv_heads}")
        return heads

    def _span(self, batch: PagedBatch) -> int:
        return self.default_span(batch.capacity) if self.span is None else self.span

    def write(self, i: int, k: torch.Tensor, v: torch.Tensor, batch: PagedBatch) -> None:
        """Rows k, v [M, kv_heads * head_dim] (any row stride) into layer ``i`` at their sequences' slots; K as it is to be attended
        (rotated: ``ops.rope``). Rows without a slot are not written."""
        ops.paged_write(self._layers[i], batch, k, v)

    def read(self, i: int, batch: PagedBatch, m: int, k_out: Optional[torch.Tensor] = None,
             v_out: Optional[torch.Tensor] = None) -> tuple[torch.Tensor, torch.Tensor]:
        """K, V [m, kv_heads * head_dim] of layer ``i``: the rows that ``write`` would write; zeros for rows without a slot."""
        return ops.paged_read(self._layers[i], batch, m, k_out, v_out)

    def attend_floats(self, m: int, heads: int, batch: PagedBatch, l_max: Optional[int] = None, weights: bool = False) -> int:
        """Workspace floats of ``attend`` for up to ``m`` rows."""
        pairs = max(min(batch.rows_max, m) * heads // self.kv_heads, 1) if weights else 0
        return ops.paged_attn_ws_floats(m, heads, self.head_dim, batch.capacity if l_max is None else l_max, self._span(batch), pairs)

    def attend(self, i: int, q: torch.Tensor, batch: PagedBatch, l_max: Optional[int] = None, out: Optional[torch.Tensor] = None,
               ws: Optional[torch.Tensor] = None, scale: Optional[float] = None, weights: Optional[torch.Tensor] = None,
               decay: float = 1.0) -> torch.Tensor:
        """Attention of q [M, heads * head_dim], few rows a sequence (a decode step, a drafted chain, the last rows of a prompt), over
        layer ``i``: every row attends its sequence's slots up to its own. Zeros for rows that attend nothing. ``l_max`` (None: the
        table's capacity) bounds the lengths: slots from there on are not attended, and a close bound saves empty
        workgroups. ``weights`` fp32 [S, kv_heads, >= l_max]: decay * weights + the softmax weights each slot in use received from the
        call's rows, summed over rows and a kv head's query heads (decay 0: set); sequences without rows keep theirs. ``ws``: fp32, attend_floats(...).
        Rows of no sequence, and those past ``rows_max``, are left as they were; in an ``out`` made here they are unset. ``out`` may be ``q``, but not with
        weights of more than 16 (row, query head) pairs a kv head."""
        return ops.paged_attention(self._layers[i], batch, q, self._heads(q), l_max, self._span(batch), ws, out, scale, weights, decay)

    def prompt_floats(self, m: int, heads: int, batch: PagedBatch, l_max: Optional[int] = None) -> int:
        """Workspace floats of ``attend_prompt`` for ``m`` rows."""
        return ops.paged_prompt_ws_floats(m, heads, self.kv_heads, self.head_dim, batch.n_seq, batch.capacity if l_max is None else l_max)

    def attend_prompt(self, i: int, q: torch.Tensor, batch: PagedBatch, l_max: Optional[int] = None,
                      out: Optional[torch.Tensor] = None, ws: Optional[torch.Tensor] = None, scale: Optional[float] = None) -> torch.Tensor:
        """The same for many rows a sequence: whole prompts or further pieces of them, packed, whose K and V have been written; from about
        64 (row, query head) pairs a kv head on it is the faster one (us of attend / attend_prompt, 4 heads a kv head: 6 sequences of 8 rows
        after 2500 to 4000 keys 24 / 27, of 16 rows 33 / 29, of 32 rows 49 / 32; 24 of 16 rows after 2000 keys 62 / 41; one of 16 rows after
        4000 12 / 19). Each softmax weight is rounded to one bf16 number here, to two in ``attend``: error of the output 0.0018 and 0.0017 of its
        norm. ``ws``: fp32, prompt_floats(...). Rows of no sequence as in ``attend``; ``out`` may be ``q``."""
        return ops.paged_prompt(self._layers[i], batch, q, self._heads(q), l_max, ws, out, scale)

    def evict(self, batch: PagedBatch, after: PagedBatch, weights: torch.Tensor, keep: int, recent: int = 0, first: int = 0,
              out_weights: Optional[torch.Tensor] = None, kept: Optional[torch.Tensor] = None) -> tuple[torch.Tensor, torch.Tensor]:
        """Cuts every sequence of ``batch`` to ``keep`` slots, in all layers, each layer and kv head by its own ``weights`` fp32
        [layers, S, kv_heads, >= lengths]: the ``first`` and the ``recent`` last slots stay, and those of the largest weight between
        (equal ones: the lowest). What stays moves to the pages of ``after``, which must not be pages of ``batch``, and
        after.lengths becomes min(lengths, keep); if ``keep`` is more than the sequences have, all stay. A slot is not a position any more: K
        that stays was rotated to the position it was written at, so later rows are rotated to positions that the caller counts on. Returns
        (kept [layers, S, kv_heads, keep] int32: the slots it came from, then -1; the weights that moved along, then zeros)."""
        return ops.paged_evict(self._layers[0], self.num_slots, self.k.stride(0), batch, after, weights, keep, recent, first, out_weights,
                               kept)
