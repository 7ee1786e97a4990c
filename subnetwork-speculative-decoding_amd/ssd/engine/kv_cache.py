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
