"""Serving form of the sparse-attention models: an 8-bit block cache of keys
and values, and the single-token (or few-token) step over it.

`SparseAttention`'s LSH graph is a function of the whole key set (bucket
tables, first-C members, a plane count that follows the length), so it is not
carried forward by a token; the reference has no serving form either. A step
takes its neighbours from the cache instead: the blocks whose bound of q.k (q
in 8 bits) is highest stand in for the LSH candidates, beside the window's and
the global tokens' blocks, or -- without a block budget -- the whole sequence.

A `BlockCache` holds the buffers of `num_layers` layers that share one block
table. Pages are handed out on the GPU (`reserve`), so a decoding step makes no
host decision and can be captured as a CUDA graph.
"""
from __future__ import annotations

from typing import Optional, Tuple, Union

import torch

from . import ops


class BlockCache:
    """Keys and values of `batch` sequences in 8 bits, one range (amax) for each
    block of `block_size` tokens, kv head and K / V.

    max_tokens: the longest a sequence may grow (the block table's width).
    num_blocks: pages of each layer's pool; by default enough for every
        sequence to reach max_tokens.
    top_blocks: blocks a step attends for each token and kv head (the `top`
        of `select`); None: every block of the sequence.

    One step is `reserve` (once), then for each layer `append` and `attend`
    (with `select` between them for a block budget) -- what
    `SparseAttention.step` does. start / lens (batch,) are the lengths before
    and after the current step. Tokens are not taken back: a completed block no
    longer has its tokens as they came.
    """

    def __init__(self, batch: int, num_kv_heads: int, head_dim: int, max_tokens: int, *, num_layers: int = 1,
                 block_size: int = 64, num_blocks: Optional[int] = None, top_blocks: Optional[int] = None,
                 dtype: torch.dtype = torch.bfloat16, device: Union[str, torch.device] = "cuda"):
        if min(batch, num_kv_heads, head_dim, max_tokens, num_layers) < 1:
            raise ValueError("BlockCache: batch, num_kv_heads, head_dim, max_tokens and num_layers must be >= 1")
        if block_size not in (16, 32, 64):
            raise NotImplementedError(f"BlockCache: block_size must be 16, 32 or 64 (got {block_size})")
        if head_dim not in (32, 64, 96, 128):
            raise NotImplementedError(f"BlockCache: head_dim must be 32, 64, 96 or 128 (got {head_dim})")
        if dtype not in (torch.float32, torch.bfloat16):
            raise NotImplementedError(f"BlockCache: dtype must be float32 or bfloat16 (got {dtype})")
        if top_blocks is not None and top_blocks < 1:
            raise ValueError(f"BlockCache: top_blocks must be >= 1 (got {top_blocks})")
        device = torch.device(device)
        if device.type != "cuda":
            raise RuntimeError(f"ssa_b200 runs on CUDA tensors only (there is no CPU path); got device {device}")
        self.batch, self.num_kv_heads, self.head_dim = batch, num_kv_heads, head_dim
        self.block_size, self.top_blocks, self.num_layers = block_size, top_blocks, num_layers
        self.max_blocks = -(-max_tokens // block_size)
        P = batch * self.max_blocks if num_blocks is None else num_blocks
        if P < 1:
            raise ValueError(f"BlockCache: num_blocks must be >= 1 (got {num_blocks})")
        self.num_blocks = P
        L, n_kv, bs, d = num_layers, num_kv_heads, block_size, head_dim
        self.k_codes = torch.zeros(L, P, n_kv, bs, d, dtype=torch.int8, device=device)
        self.v_codes = torch.zeros(L, P, n_kv, bs, d, dtype=torch.int8, device=device)
        self.amax = torch.zeros(L, P, n_kv, 2, device=device)
        self.bounds = torch.zeros(L, P, n_kv, 2, d, dtype=torch.int8, device=device)
        self.tail = torch.zeros(L, batch, n_kv, 2, bs, d, dtype=dtype, device=device)
        self.table = torch.full((batch, self.max_blocks), -1, dtype=torch.int32, device=device)
        self.start = torch.zeros(batch, dtype=torch.int32, device=device)
        self.lens = torch.zeros(batch, dtype=torch.int32, device=device)
        self.free = torch.arange(P - 1, -1, -1, dtype=torch.int32, device=device)
        self.state = torch.tensor([P, 0], dtype=torch.int32, device=device)
        self.ragged = False  # the present step's lengths may differ
        self.rows: Optional[int] = None  # the most tokens a sequence has in it, where the host knows
        # the layers' tensors, sliced once: a slice costs as much as a launch
        self._layers = [(self.k_codes[i], self.v_codes[i], self.amax[i], self.bounds[i], self.tail[i]) for i in range(L)]

    # -- lengths and pages ---------------------------------------------------
    def reserve(self, new_lens: Union[int, torch.Tensor], prompt: bool = False, limit: Optional[int] = None) -> None:
        """Begins a step of new_lens more tokens (an int for all sequences, or
        (batch,) int32 on the device): start becomes the present lengths, lens
        the new ones, and the blocks they open get pages. A sequence for which
        the table or the pool has no room keeps its length -- its tokens of
        this step are not stored and their attention is 0 -- and is counted in
        `refused()`. With `prompt` the same holds for a sequence that has
        tokens already and is given more. limit: the rows that the step's
        tensors have; greater entries of a tensor new_lens are cut to it (without
        it they must not be greater: a token that is counted and never appended
        stands for whatever its page held before)."""
        self.ragged = torch.is_tensor(new_lens)
        self.rows = limit if self.ragged else new_lens
        if not self.ragged:
            if limit is not None and new_lens > limit:
                raise ValueError(f"BlockCache.reserve: {new_lens} new tokens, but {limit} rows")
            new_lens = torch.full_like(self.lens, new_lens)
        elif new_lens.shape != self.lens.shape or new_lens.dtype != torch.int32 or new_lens.device != self.lens.device:
            raise ValueError(f"BlockCache.reserve: new_lens must be a ({self.batch},) int32 tensor on {self.lens.device}, got "
                             f"{new_lens.dtype} {tuple(new_lens.shape)} on {new_lens.device}")
        elif limit is not None:
            new_lens = new_lens.clamp(max=limit)
        if prompt:
            late = (self.lens > 0) & (new_lens > 0)
            new_lens = new_lens.masked_fill(late, 0)
            self.state[1] += late.sum()
        ops.cache_reserve(self.lens, new_lens, self.table, self.free, self.state, self.block_size,
                          out=(self.start, self.lens, self.state))

    def release(self, rows: torch.Tensor) -> None:
        """Empties the sequences of `rows` (a (batch,) bool mask): their pages
        go back to the pool, their lengths to 0. Waits for the GPU."""
        rows = rows.to(device=self.table.device, dtype=torch.bool)
        if rows.shape != (self.batch,):
            raise ValueError(f"BlockCache.release: a ({self.batch},) mask expected, got {tuple(rows.shape)}")
        held = (self.lens + self.block_size - 1) // self.block_size
        col = torch.arange(self.max_blocks, device=self.table.device)
        pages = self.table[rows[:, None] & (col < held[:, None])]
        n = int(self.state[0])
        self.free[n:n + pages.numel()] = pages
        self.state[0] += pages.numel()
        self.lens[rows] = 0
        self.start[rows] = 0
        self.table[rows] = -1

    def refused(self) -> int:
        """Sequences `reserve` had no room for so far (waits for the GPU)."""
        return int(self.state[1])

    # -- one layer -----------------------------------------------------------
    def append(self, k: torch.Tensor, v: torch.Tensor, layer: int = 0, want_values: bool = False):
        """Stores the step's k, v (batch, n_kv, n, d) (ops.cache_append), n at
        least what `reserve` was given."""
        if self.rows is not None and k.dim() == 4 and k.shape[2] < self.rows:
            raise ValueError(f"BlockCache.append: {k.shape[2]} rows, but up to {self.rows} new tokens were reserved")
        kc, vc, am, bd, tail = self._layers[layer]
        return ops.cache_append(k, v, kc, vc, am, bd, tail, self.table, self.start, self.lens, want_values)

    def select(self, q: torch.Tensor, layer: int = 0, top: Optional[int] = None, sink: int = 1, local: int = 1) -> torch.Tensor:
        """The blocks to attend for the step's q (ops.cache_select); top
        defaults to top_blocks. Call it behind the layer's append."""
        _, _, am, bd, _ = self._layers[layer]
        top = self.top_blocks if top is None else top
        if top is None:
            raise ValueError("BlockCache.select: no block budget (top, or top_blocks of the cache)")
        return ops.cache_select(q, bd, am, self.table, self.start, self.lens, top, self.block_size, sink, local)

    def attend(self, q: torch.Tensor, scale: float, layer: int = 0, blocks: Optional[torch.Tensor] = None,
               causal: bool = True, want_lse: bool = False):
        """Attention of the step's q over the layer's cache (ops.cache_attention)."""
        kc, vc, am, _, _ = self._layers[layer]
        return ops.cache_attention(q, kc, vc, am, self.table, self.start, self.lens, scale, blocks, causal, want_lse)

    def values(self, layer: int = 0) -> Tuple[torch.Tensor, torch.Tensor]:
        """k, v (batch, n_kv, max_blocks * block_size, d) fp32 as the cache
        holds them, 0 behind each sequence's length (for inspection)."""
        kc, vc, am, _, _ = self._layers[layer]
        page = self.table.clamp(min=0).long()
        pos = torch.arange(self.max_blocks * self.block_size, device=self.table.device)
        real = (pos < self.lens[:, None])[:, None, :, None]
        out = []
        for i, codes in enumerate((kc, vc)):
            x = codes[page].float() * (am[page][..., i] / 127)[..., None, None]
            out.append(torch.where(real, x.transpose(1, 2).flatten(2, 3), 0.0))
        return out[0], out[1]
