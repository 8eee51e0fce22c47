"""The paged key-value cache of the attention layers and their rotary positions.

    rope = Rope(64, base=1e7)                                  # a quarter of a 256-value head
    cache = KVCache(layers=10, rows=2, tokens_per_row=4096, kv_heads=2, head_dim=256, quantised=True)
    cache.reserve(row, tokens)                                 # host: pages for a row's tokens
    q = cache.write(layer, k, v, positions, rows=rows, q=q, rope=rope)   # prompt chunk or frame
    k, v = cache.read(layer, lengths, max_length)              # dense bf16, for a prompt's attention
    out, lse = cache.attend(layer, q, lengths)                 # one new token a row

`write`, `read` and `attend` launch one or two kernels on the current stream, read lengths, positions and the
page table from device memory and never synchronise, so a decode frame of them is captured into a CUDA
graph; `reserve` and `release` are called between replays (they rewrite the table in place).
"""

from __future__ import annotations

import math
from typing import Optional, Tuple

import torch
from torch import Tensor

from . import ops


def rope_frequencies(rotary_dim: int, base: float = 10000.0, scaling: Optional[str] = None, stretch: float = 1.0,
                     trained_length: int = 0) -> Tuple[Tensor, float]:
    """(float64 [rotary_dim / 2] angle of one position for each pair, factor on the rotated values).

    scaling None: base ** (-2i / rotary_dim). "linear": positions compressed by stretch. "ntk": base
    enlarged so that the slowest pair is slowed by stretch and the fastest stays. "yarn": pairs that turn more
    than 32 times over trained_length stay, those that turn less than once are slowed by stretch, a linear
    ramp in the number of turns between, and the rotated values grow by 0.1 ln(stretch) + 1. Checkpoints are also
    trained and served with a ramp that is linear in the pair's index between those two, with other bounds, or
    with another factor; frequencies in between then differ by tens of percent. Such a model's own frequencies
    and factor go into a `Rope` as they are."""
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError("rotary_dim must be even and at least 2")
    if base <= 0 or stretch < 1:
        raise ValueError("base must be positive and stretch at least 1")
    if scaling not in (None, "linear", "ntk", "yarn"):
        raise ValueError(f"unknown scaling {scaling!r}: None, 'linear', 'ntk' or 'yarn'")
    if scaling == "ntk":
        base = base * stretch ** (rotary_dim / (rotary_dim - 2) if rotary_dim > 2 else 1.0)
    f = float(base) ** (-torch.arange(0, rotary_dim, 2, dtype=torch.float64) / rotary_dim)
    factor = 1.0
    if scaling == "linear":
        f = f / stretch
    elif scaling == "yarn":
        if trained_length < 1:
            raise ValueError("'yarn' needs the trained length")
        keep = ((trained_length * f / (2 * math.pi) - 1) / 31).clamp(0, 1)
        f = f * keep + f / stretch * (1 - keep)
        factor = 0.1 * math.log(stretch) + 1
    return f, factor


class Rope:
    """Rotary positions of one kind of head: `rope(x, positions)` turns bf16 [T, heads, dim].

    inv_freq (float64 [rotary_dim / 2] on the device) and factor are plain attributes: a model whose frequencies
    none of the scalings gives sets them after construction."""

    def __init__(self, rotary_dim: int, base: float = 10000.0, interleaved: bool = False, scaling: Optional[str] = None,
                 stretch: float = 1.0, trained_length: int = 0, device="cuda"):
        f, self.factor = rope_frequencies(rotary_dim, base, scaling, stretch, trained_length)
        self.inv_freq = f.to(device)
        self.interleaved = bool(interleaved)

    def __call__(self, x: Tensor, positions: Tensor) -> Tensor:
        return ops.rope(x, positions, self.inv_freq, self.interleaved, self.factor)


class KVCache:
    """Pages of keys and values for `layers` attention layers, with one page table for all of them.

    k, v [layers, pages, kv_heads, page_size, head_dim] bf16, or float8_e4m3fn with one power-of-two exponent a
    token and head in k_exp, v_exp (int8 [layers, pages, kv_heads, page_size]): half the memory and traffic.
    table int32 [rows, pages_per_row] on the device, -1 where a row has no page. status: one device word that
    collects tokens which the kernels skipped because their page or place does not exist (4), and waits that
    ran out (1); `check` reads it."""

    def __init__(self, layers: int, rows: int, tokens_per_row: int, kv_heads: int, head_dim: int, page_size: int = 64,
                 pages: Optional[int] = None, quantised: bool = False, device="cuda"):
        if min(layers, rows, tokens_per_row, kv_heads) < 1:
            raise ValueError("layers, rows, tokens_per_row and kv_heads must be at least 1")
        if page_size < 16 or page_size % 16:
            raise ValueError("page_size must be a multiple of 16")
        if head_dim not in (64, 128, 192, 256):
            raise ValueError("head_dim must be 64, 128, 192 or 256")
        self.page_size, self.pages_per_row = page_size, -(-tokens_per_row // page_size)
        pages = rows * self.pages_per_row if pages is None else pages
        if pages < 1:
            raise ValueError("pages must be at least 1")
        shape = (layers, pages, kv_heads, page_size, head_dim)
        dtype = torch.float8_e4m3fn if quantised else torch.bfloat16
        held = [torch.zeros(shape, dtype=dtype, device=device) for _ in range(2)]
        exps = [torch.zeros(shape[:-1], dtype=torch.int8, device=device) if quantised else None for _ in range(2)]
        self._buffers = (*held, *exps)
        self._views = [tuple(None if b is None else b[i] for b in self._buffers) for i in range(layers)]
        self.table = torch.full((rows, self.pages_per_row), -1, dtype=torch.int32, device=device)
        self.status = torch.zeros(1, dtype=torch.int32, device=device)
        self._free = list(range(pages - 1, -1, -1))
        self._held = [[] for _ in range(rows)]

    # the buffers are not replaced: `layer` hands out views that were made once (four of them cost 8 us a call)
    k = property(lambda self: self._buffers[0])
    v = property(lambda self: self._buffers[1])
    k_exp = property(lambda self: self._buffers[2])
    v_exp = property(lambda self: self._buffers[3])

    def layer(self, layer: int) -> Tuple[Tensor, Tensor, Optional[Tensor], Optional[Tensor]]:
        """(k, v, k_exp, v_exp) of one layer, as the ops take them."""
        return self._views[layer]

    def reserve(self, row: int, tokens: int) -> None:
        """Gives a row pages for its first `tokens` tokens (those it has stay). Raises, changing nothing, when
        the row's table or the cache has no room."""
        have = self._held[row]
        need = -(-tokens // self.page_size) - len(have)
        if need <= 0:
            return
        if len(have) + need > self.pages_per_row:
            raise RuntimeError(f"row {row}: {tokens} tokens need more than its {self.pages_per_row} pages")
        if need > len(self._free):
            raise RuntimeError(f"row {row}: {need} pages needed, {len(self._free)} free")
        new = [self._free.pop() for _ in range(need)]
        self.table[row, len(have):len(have) + need] = torch.tensor(new, dtype=torch.int32).to(self.table.device)
        have.extend(new)

    def release(self, row: int) -> None:
        """Takes a row's pages back; calls already on the stream still see them."""
        self._free.extend(reversed(self._held[row]))
        self._held[row] = []
        self.table[row].fill_(-1)

    def write(self, layer: int, k: Tensor, v: Tensor, positions: Tensor, rows: Optional[Tensor] = None,
              q: Optional[Tensor] = None, rope: Optional[Rope] = None) -> Tensor:
        """Caches T tokens' keys and values at (rows[t], positions[t]) and returns q (see `ops.kv_write`); with
        rope, keys and queries are rotated in the same launch."""
        if rope is None:
            q_out = ops.kv_write(k, v, positions, self.table, *self.layer(layer), self.status, rows, q)
        else:
            q_out = ops.kv_write(k, v, positions, self.table, *self.layer(layer), self.status, rows, q, rope.inv_freq,
                                 rope.interleaved, rope.factor)
        return q_out

    def read(self, layer: int, lengths: Tensor, max_length: int) -> Tuple[Tensor, Tensor]:
        """Dense bf16 keys and values [rows, kv_heads, max_length, head_dim] (see `ops.kv_read`)."""
        return ops.kv_read(*self.layer(layer), self.table, lengths, max_length, self.status)

    def attend(self, layer: int, q: Tensor, lengths: Tensor, scale: Optional[float] = None, window: int = 0,
               max_tokens: Optional[int] = None) -> Tuple[Tensor, Tensor]:
        """One new token's attention a row: (out, lse), see `ops.paged_attention`. max_tokens: no row is longer
        (one of a few bucket sizes, as the engine's graphs have, engine.py:412-415)."""
        if max_tokens is not None and max_tokens < 0:
            raise ValueError("max_tokens must not be negative")
        table = self.table if max_tokens is None else self.table[:, :-(-max_tokens // self.page_size)]
        return ops.paged_attention(q, *self.layer(layer), table, lengths, self.status, scale, window)

    def check(self) -> int:
        """Reads and clears the status word (synchronises). 0: nothing was skipped."""
        word = int(self.status.item())
        if word:
            self.status.zero_()
        return word
