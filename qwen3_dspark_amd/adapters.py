"""Low-rank adapters of many requests beside the shared q/k/v projection: token t of
a request with adapter a projects with W + scaling[a] B_a A_a in place of W (its
attention's q_proj, k_proj and v_proj), each request of a batch with its own adapter
or none, in the launch that projects the batch.

    adapters = [QKVAdapters(a_q, b_q, a_k, b_k, a_v, b_v, scaling=...) for each layer]
    batch = AdapterBatch(device, lengths=[7] * 64, ids=[...])      # once per round, for every layer
    q = store.stage_projected(tx, layer, hidden, prologue, adapters=adapters[layer], batch=batch)

The shared weights are read once for the whole batch, as without adapters.  Adapters of
different ranks share one QKVAdapters by zero rows of A (or columns of B).  A key or value
cached under an adapter belongs to it: requests that share a prompt's rows
(PersistentTargetKV.share_prefix) are ones whose adapter is the same.
"""
import math
from numbers import Real

import torch

from ._device import Prepared, require_gfx950, upload
from .kernels import HEAD_DIM, KV_HEADS, Q_HEADS

TILE_TOKENS = (16, 32)       # tokens of one adapter per shrinking workgroup, of small and of large calls
SMALL_PAIRS = 256            # (tile, 16 ranks) pairs of small calls (measured at the kernel's launch)
MAX_RANK = 256


class AdapterBatch:
    """Which adapter each request of a packed batch has: lengths, tokens per request;
    ids, its adapter or -1.  Built once per batch shape, uploaded once, and read by the
    prologue of every layer (also under graph capture, with these lengths and ids)."""

    def __init__(self, device, lengths, ids):
        lengths, ids = list(lengths), list(ids)
        if (not lengths or len(lengths) != len(ids) or any(type(n) is not int or n < 1 for n in lengths)
                or any(type(a) is not int or not -1 <= a < 2 ** 31 for a in ids)):
            raise ValueError('One positive length and one adapter (or -1) per request required')
        self.tokens, self.largest = sum(lengths), max(ids)
        if self.tokens >= 2 ** 31:
            raise ValueError('At most 2^31 - 1 tokens per batch')
        tiles, at, run = [], 0, None                 # neighbours of one adapter share tiles
        for n, a in zip(lengths, ids):
            if run is not None and run[1] == a:
                run[2] += n
            else:
                run = [at, a, n]
                tiles.append(run)
            at += n
        tiles = [[(t, min(size, t0 + n - t), a, 0) for t0, a, n in tiles if a >= 0 for t in range(t0, t0 + n, size)]
                 for size in TILE_TOKENS]
        self.device = require_gfx950(device)
        self.token_adapter = upload(self.device, [a for n, a in zip(lengths, ids) for _ in range(n)])
        self.tiles = upload(self.device, [x for size in tiles for t in size for x in t])
        self._lists = tuple(zip(TILE_TOKENS, map(len, tiles), (self.tiles.data_ptr(),
                                                               self.tiles.data_ptr() + 16 * len(tiles[0]))))
        self.any = bool(tiles[0])
        self._ready = Prepared(self.device, self.token_adapter, self.tiles)

    def tile_list(self, rank):
        """(address, tiles, tokens per tile at most) of the list for adapters of a rank."""
        (small, n_small, at_small), (large, n_large, at_large) = self._lists
        if n_small * (rank // 16) <= SMALL_PAIRS:
            return at_small, n_small, small
        return at_large, n_large, large


class QKVAdapters:
    """The q/k/v adapters of one layer: a_* [n, rank, hidden], b_q [n, 2048, rank], b_k and b_v
    [n, 1024, rank], bf16 on a gfx950 GPU; scaling: a number, or one per adapter.  The
    weights are laid out once, here."""

    def __init__(self, a_q, b_q, a_k, b_k, a_v, b_v, *, scaling=1.0):
        given = (a_q, b_q, a_k, b_k, a_v, b_v)
        if any(not isinstance(t, torch.Tensor) or t.ndim != 3 or t.dtype != torch.bfloat16 or t.device != a_q.device
               for t in given):
            raise ValueError('Adapters must be bf16 [n, rank, hidden] and [n, outputs, rank] on one device')
        n, rank, hidden = a_q.shape
        q, kv = Q_HEADS * HEAD_DIM, KV_HEADS * HEAD_DIM
        if (n < 1 or any(t.shape != a_q.shape for t in (a_k, a_v)) or b_q.shape != (n, q, rank)
                or any(t.shape != (n, kv, rank) for t in (b_k, b_v))):
            raise ValueError('Adapters must be a [n, rank, hidden], b_q [n, 2048, rank], b_k and b_v [n, 1024, rank]')
        if not 1 <= rank <= MAX_RANK or hidden < 128 or hidden % 128:
            raise ValueError(f'Rank must be in [1, {MAX_RANK}] and hidden a positive multiple of 128')
        scaling = [scaling] * n if isinstance(scaling, Real) else list(scaling)
        if len(scaling) != n or any(isinstance(x, bool) or not isinstance(x, Real) or not math.isfinite(x)
                                    for x in scaling):
            raise ValueError('scaling must be a finite number, or one per adapter')
        self.device = require_gfx950(a_q.device)
        self.count, self.rank, self.hidden = n, rank, hidden
        self.padded_rank = 16 if rank <= 16 else 32 if rank <= 32 else -(-rank // 64) * 64      # what the kernels take
        self.a = torch.zeros((n, 3, self.padded_rank, hidden), dtype=torch.bfloat16, device=self.device)
        self.b = torch.zeros((n, q + 2 * kv, self.padded_rank), dtype=torch.bfloat16, device=self.device)
        for i, t in enumerate((a_q, a_k, a_v)):
            self.a[:, i, :rank] = t.detach()
        for at, t in ((0, b_q), (q, b_k), (q + kv, b_v)):
            self.b[:, at:at + t.shape[1], :rank] = t.detach()
        self.scaling = upload(self.device, [float(x) for x in scaling], torch.float32)
        self._ready = Prepared(self.device, self.a, self.b, self.scaling)
        self.pointers = (self.a.data_ptr(), self.b.data_ptr(), self.scaling.data_ptr(), n, self.padded_rank, rank)

    def check(self, batch, tokens, hidden, device):
        """Refuse a batch or prologue that these adapters do not fit."""
        if not isinstance(batch, AdapterBatch) or batch.tokens != tokens or batch.device != device:
            raise ValueError(f'batch must be an AdapterBatch of {tokens} tokens on the prologue device')
        if self.device != device or self.hidden != hidden:
            raise ValueError('Adapters must have the prologue\'s hidden size and device')
        if batch.largest >= self.count:
            raise ValueError(f'The batch names adapter {batch.largest} of {self.count}')

    def ready(self, batch, stream):
        """Before the launches on the stream of this handle."""
        self._ready.on(self.device, stream)
        batch._ready.on(self.device, stream)

    def scratch(self, tokens):
        """Elements of the scaled A x of a batch, two bf16 numbers each."""
        return 3 * tokens * 2 * self.padded_rank
