"""Decode attention for batches in which groups of sequences share a long prefix.

Sequences forked from one another (or behind one system prompt) name the same pages for their first
keys. ``PrefixGroups`` holds which sequences share how many keys; ``attn_shared_prefix`` reads each
group's shared pages once for all of its sequences instead of once per sequence.
"""
from __future__ import annotations

from typing import Optional, Sequence, Tuple

import numpy as np
import torch

_HDR = 8      # header ints of the device table, [0] = number of prefix items
_ITEM = 8     # ints per prefix item
_ROWS = 64    # query rows of a sequence: new tokens x heads of a KV group
_TILE = 256   # query rows per prefix item
_OWN = 8      # query rows per worker on a sequence's own keys
_WORKERS = 12  # such workers per SM
_MAX_BATCH = 1024
_KEYS = 64    # key ranges of prefix items are multiples of this


class PrefixGroups:
    """Which sequences of a decode batch share a prefix, and the attention's work list and workspace.

    ``batch`` sequences (slots) bring ``q_len`` new tokens each; ``hq`` / ``hkv`` query and KV heads of
    ``head_dim``. Nothing is shared until ``set``. A call that is being captured into a CUDA graph uses the
    largest launch this object can need, so replays follow later ``set`` calls, block tables and lengths.
    All memory is allocated here: use one object per stream (two calls on two streams, or two graphs that may
    replay at the same time, need one each)."""

    def __init__(self, batch: int, hq: int, hkv: int, head_dim: int, q_len: int = 1, device=None):
        if not 1 <= batch <= _MAX_BATCH or q_len < 1:
            raise ValueError(f"PrefixGroups serves 1 to {_MAX_BATCH} sequences and at least one new token each, got {batch} x {q_len}")
        if hkv < 1 or hq % hkv or head_dim not in (64, 128):
            raise ValueError(f"{hq} query heads over {hkv} KV heads of {head_dim}: need hq % hkv == 0 and head_dim 64 or 128")
        self.group = hq // hkv
        if q_len * self.group > _ROWS:
            raise ValueError(f"{q_len} new tokens x {self.group} heads per KV head exceed {_ROWS} query rows")
        self.batch, self.hq, self.hkv, self.head_dim, self.q_len = batch, hq, hkv, head_dim, q_len
        self.device = torch.device(device if device is not None else "cuda")
        if self.device.type == "cuda" and self.device.index is None:
            self.device = torch.device("cuda", torch.cuda.current_device())
        sms = torch.cuda.get_device_properties(self.device).multi_processor_count if self.device.type == "cuda" else 148
        self._sms = sms
        rows = batch * q_len
        # one wave of prefix items, or one for each tile of rows where there are more of those
        self.item_cap = sms + hkv * (-(-rows * self.group // _TILE) + batch)
        self._items_at = _HDR + (5 * batch + 2 + 3) // 4 * 4
        # partial rows: of the prefix items (full ones, and one more wave for tiles that are not), then of the pieces
        # that the keys behind the prefixes are cut into
        self._own_at = _TILE * sms + rows * hq
        own_rows = q_len * self.group
        slots = self._own_at + (_WORKERS * sms + batch * hkv * -(-own_rows // _OWN)) * min(_OWN, own_rows)
        self._po = torch.empty(slots * head_dim, dtype=torch.float32, device=self.device)
        self._pml = torch.empty(slots * 2, dtype=torch.float32, device=self.device)
        self._meta = torch.zeros(self._items_at + _ITEM * self.item_cap, dtype=torch.int32, device=self.device)
        from . import scratch
        self._err = scratch(self.device).err if self.device.type == "cuda" else None
        self.n_items = 0
        self.set([])

    def set(self, groups: Sequence[Tuple[Sequence[int], int]]) -> "PrefixGroups":
        """``groups``: (sequences, shared keys) pairs. The first ``shared`` keys of every sequence of a group
        must be the same tokens; they are read through the block table of the group's first sequence, which has to
        hold them all, and what the others' tables hold for them is not used. A sequence may be in one group at
        most; one in none attends its own pages alone. Not inside a capture: the list comes from the host."""
        if self.device.type == "cuda" and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("PrefixGroups.set copies from host memory: call it before the capture, or between replays")
        B, T, G = self.batch, self.q_len, self.group
        seen = set()
        for seqs, shared in groups:
            if shared < 0:
                raise ValueError(f"a shared prefix of {shared} keys")
            for b in seqs:
                if not 0 <= int(b) < B:
                    raise ValueError(f"sequence {b} outside a batch of {B}")
                if int(b) in seen:
                    raise ValueError(f"sequence {b} is in two prefix groups")
                seen.add(int(b))
        groups = [([int(b) for b in seqs], int(n)) for seqs, n in groups if len(seqs) and n > 0]
        meta = np.zeros(self._meta.shape[0], dtype=np.int32)
        prefix, base, slots, member = (meta[_HDR + i * B:_HDR + (i + 1) * B] for i in range(4))
        tiles = [-(-len(seqs) * T * G // _TILE) for seqs, _ in groups]
        # Every item takes the same number of 64-key blocks, the fewest with which the items make one wave: a
        # block costs the same whether it serves 256 rows (tensor cores) or few (memory).
        blocks = [-(-n // _KEYS) for _, n in groups]
        per = max(1, -(-sum(t * self.hkv * k for t, k in zip(tiles, blocks)) // self._sms))
        while per < max(blocks, default=1) and sum(t * self.hkv * -(-k // per) for t, k in zip(tiles, blocks)) > self._sms:
            per += 1
        per *= _KEYS
        items, off = [], 0
        for t, (seqs, n) in zip(tiles, groups):
            splits = -(-n // per)
            size = -(-(-(-n // splits)) // _KEYS) * _KEYS
            splits = -(-n // size)
            member[off:off + len(seqs)] = seqs
            prefix[seqs], slots[seqs] = n, splits
            rows = len(seqs) * T * G
            h, i, s = np.meshgrid(np.arange(self.hkv), np.arange(t), np.arange(splits), indexing="ij")
            one = np.zeros((h.size, _ITEM), dtype=np.int32)
            one[:, 0], one[:, 1] = seqs[0], off
            one[:, 2] = i.reshape(-1) * _TILE
            one[:, 3] = np.minimum(_TILE, rows - one[:, 2])
            one[:, 4], one[:, 5] = h.reshape(-1), s.reshape(-1) * size
            one[:, 6], one[:, 7] = np.minimum(n, one[:, 5] + size), s.reshape(-1)
            items.append(one)
            off += len(seqs)
        per_seq = slots.astype(np.int64) * (T * self.hq)
        base[:] = np.concatenate([[0], np.cumsum(per_seq)[:-1]])
        n_items = sum(len(x) for x in items)
        assert n_items <= self.item_cap and int(per_seq.sum()) <= self._own_at, "prefix work list exceeds its workspace"
        if items:
            meta[self._items_at:self._items_at + _ITEM * n_items] = np.concatenate(items).reshape(-1)
        meta[0] = n_items
        host = torch.from_numpy(meta)
        if self.device.type == "cuda":
            with torch.cuda.device(self.device):
                self._meta.copy_(host.pin_memory(), non_blocking=True)
        else:
            self._meta.copy_(host)
        self.n_items = n_items
        return self


def attn_shared_prefix(q: torch.Tensor, kcache: torch.Tensor, vcache: torch.Tensor, block_tables: torch.Tensor,
                       seq_lens: torch.Tensor, groups: PrefixGroups, out: torch.Tensor, scale: float,
                       window: int = 0) -> torch.Tensor:
    """Causal paged GQA attention of the ``q_len`` newest tokens of every sequence, the shared prefixes of
    ``groups`` read once per group. q, out [B * q_len, hq * D] bf16 (the tokens of a sequence together);
    kcache, vcache [pages, hkv, page, D] bf16 (pages of a multiple of 16 tokens); block_tables [B, pages] and
    seq_lens [B] int32 as in ``attn_decode``, lengths including the new tokens. A token without any key gives
    zeros, one that meets NaN gives NaN. ``window``: attend the last ``window`` keys only. ``scale`` must be
    positive: the largest score is looked for before it is applied. Softmax sums and outputs are held in fp32, the
    weights are rounded to bf16 for the product."""
    from . import _count, ext
    if not 1e-30 <= scale <= 1e30:
        raise ValueError(f"a scale of {scale}: must be positive and finite")
    B, T = groups.batch, groups.q_len
    if seq_lens.shape[0] != B or q.shape[0] != B * T or q.shape[1] != groups.hq * groups.head_dim:
        raise ValueError(f"q {tuple(q.shape)} and {seq_lens.shape[0]} lengths do not fit groups of {B} sequences x {T} "
                         f"tokens x {groups.hq} heads of {groups.head_dim}")
    if kcache.shape[1] != groups.hkv or kcache.shape[3] != groups.head_dim:
        raise ValueError(f"cache {tuple(kcache.shape)} does not fit groups of {groups.hkv} KV heads of {groups.head_dim}")
    if groups.device != q.device:
        raise ValueError(f"groups on {groups.device}, q on {q.device}")
    _count(ext().attn_shared(q, kcache, vcache, block_tables, seq_lens, groups._meta, groups._po, groups._pml, out,
                             groups._err, groups.n_items, groups.item_cap, groups._own_at, scale, window))
    return out
