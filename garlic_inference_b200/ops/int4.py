"""Weights and cache rows in 4 bits: what holds them, and the entry points that make, read and use them.

A number q of 0 .. 15 stands for step * q + low, both bfloat16: one pair for 128 inputs of an output of a weight
(`Int4Weight`), one for 64 numbers of a head in the cache (`Int4Rows`).  Two numbers lie in a byte, the first in its low half.
A group with a number that is not finite stands for NaN.

  weights   `quantize_weight`, `dequantize_weight`; `linear` and its kin (linear.py) take an `Int4Weight` for their weight
  cache     `append` writes a step's keys and values, `read` gives back what the pages hold of given tokens,
            `attention_decode` and `attention_prompt` read them

Products and attention compute with the numbers that the codes stand for, not with these rounded again, save where
`attention_prompt` and `linear` say so.  Upstream has neither.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional

import torch

from . import kernels
from .kernels import BF16, _dense, _ptr, _stream, code
from .library import KernelError, check, require_gpu

GROUP_WEIGHT = 128          # inputs that share a step
GROUP_ROWS = 64             # numbers of a head that share a step
TILE_BYTES = 1088           # 16 outputs x 128 inputs: 1,024 bytes of codes, then (step, low) of the 16 outputs
LINEAR_MAX_ROWS = 16        # rows of x that the kernel reading a weight's codes takes


@dataclass
class Int4Weight:
    """A weight [n, k] in 4 bits.  `tiles` uint8 [ceil(n / 16), ceil(k / 128), 1088]: per tile two pieces of 512 bytes (outputs
    0-7 and 8-15), in each 8 outputs x 4 quarters of 32 inputs x 16 bytes, then step and low value (bfloat16) of each of the 16
    outputs.  What a tile holds beyond the weight's sizes is not used."""
    tiles: torch.Tensor
    n: int
    k: int

    def __post_init__(self):
        want = (-(-self.n // 16), -(-self.k // GROUP_WEIGHT), TILE_BYTES)
        if self.n < 1 or self.k < 1 or self.tiles.dtype != torch.uint8 or tuple(self.tiles.shape) != want or \
                not self.tiles.is_contiguous():
            raise KernelError(f"tiles {tuple(self.tiles.shape)} of {self.tiles.dtype} for a weight of {self.n} x {self.k} in 4 "
                              f"bits: dense uint8 {want} holds it")

    @property
    def shape(self) -> tuple:
        return (self.n, self.k)

    @property
    def device(self):
        return self.tiles.device

    def numel(self) -> int:
        return self.n * self.k

    def bytes(self) -> int:
        return self.tiles.numel()


@dataclass
class Int4Rows:
    """Pages of a cache in 4 bits: `codes` uint8 [pages, heads, page size, d / 2], `meta` bfloat16 [pages, heads, page size,
    d / 64, 2] (step, low)."""
    codes: torch.Tensor
    meta: torch.Tensor

    def __post_init__(self):
        c, m = self.codes, self.meta
        if c.dim() != 4 or c.dtype != torch.uint8 or c.shape[3] < 32 or c.shape[3] % 32 or m.dtype != torch.bfloat16 or \
                tuple(m.shape) != (*c.shape[:3], c.shape[3] // 32, 2) or not (c.is_contiguous() and m.is_contiguous()):
            raise KernelError(f"codes {tuple(c.shape)} of {c.dtype} and steps {tuple(m.shape)} of {m.dtype} are no pages in 4 bits: "
                              "dense uint8 [pages, heads, page size, d / 2] and bfloat16 [pages, heads, page size, d / 64, 2], "
                              "d a multiple of 64")

    @property
    def head_dim(self) -> int:
        return self.codes.shape[3] * 2

    @property
    def shape(self) -> tuple:
        """[pages, heads, page size, d], as a pool of numbers would have it"""
        return (*self.codes.shape[:3], self.head_dim)

    @staticmethod
    def zeros(pages: int, heads: int, page_size: int, head_dim: int, device) -> "Int4Rows":
        if head_dim < GROUP_ROWS or head_dim % GROUP_ROWS:
            raise KernelError(f"rows in 4 bits want heads that are a multiple of {GROUP_ROWS} numbers, not {head_dim}")
        return Int4Rows(torch.zeros((pages, heads, page_size, head_dim // 2), dtype=torch.uint8, device=device),
                        torch.zeros((pages, heads, page_size, head_dim // GROUP_ROWS, 2), dtype=torch.bfloat16, device=device))


# ------------------------------------------------------------------------------------------------------------ weights
def _on_gpu(t: torch.Tensor, name: str) -> None:
    if not t.is_cuda:
        raise KernelError(f"{name} is on {t.device}; the kernels run on the GPU only")


def quantize_weight(w: torch.Tensor) -> Int4Weight:
    """The weight [n, k] (bfloat16 or float32, rows may lie apart) in 4 bits: low = the group's smallest number, step =
    (largest - smallest) / 15, both rounded to bfloat16 so that the range covers the group; every number the nearest of the 16."""
    l = require_gpu()
    kernels._rows(w, "w")
    n, k = w.shape
    if n < 1 or k < 1:
        raise KernelError(f"a weight of {n} x {k} has nothing to hold")
    tiles = torch.empty((-(-n // 16), -(-k // GROUP_WEIGHT), TILE_BYTES), dtype=torch.uint8, device=w.device)
    check(l.gi_int4_quantize_weight(_ptr(w), code(w.dtype), w.stride(0) if n > 1 else k, _ptr(tiles), n, k, _stream()), l)
    return Int4Weight(tiles, n, k)


def dequantize_weight(w: Int4Weight, dtype: torch.dtype = torch.bfloat16, first: int = 0, rows: Optional[int] = None,
                      out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Outputs first .. first + rows - 1 of the weight as [rows, k] in `dtype` (rounded once)."""
    l = require_gpu()
    _on_gpu(w.tiles, "w")
    rows = w.n - first if rows is None else rows
    if not 0 <= first <= first + rows <= w.n or rows < 1:
        raise KernelError(f"outputs {first} .. {first + rows - 1} of a weight of {w.n}")
    if out is None:
        out = torch.empty((rows, w.k), dtype=dtype, device=w.device)
    if _dense(out, "out", dtype).shape != (rows, w.k):
        raise KernelError(f"out {tuple(out.shape)} for {rows} outputs of {w.k} inputs")
    check(l.gi_int4_dequantize_weight(_ptr(w.tiles), _ptr(out), code(dtype), first, rows, w.n, w.k, _stream()), l)
    return out


def linear_rows(x: torch.Tensor, w: Int4Weight, out_dtype: torch.dtype = torch.bfloat16, unit: Optional[tuple] = None,
                out: Optional[torch.Tensor] = None, ranks: int = 0, parts: int = 0) -> torch.Tensor:
    """x W^T for 1 to 16 rows of bfloat16 x, reading the weight's codes once; with `unit` (a `kernels.glu_shape` tuple) the gated
    unit of the weight's first half of outputs (a multiple of 16) and its last.  `out` may be columns of a wider matrix.
    `ranks`, `parts`: blocks that share the inputs, and parts of a block's share that its warps take (0: chosen by the entry point)."""
    l = require_gpu()
    _dense(x, "x", torch.bfloat16), _on_gpu(w.tiles, "w")
    if x.dim() != 2 or x.shape[1] != w.k:
        raise KernelError(f"x {tuple(x.shape)} does not fit a weight {w.shape} ([out, in])")
    m, n = x.shape[0], w.n // 2 if unit is not None else w.n
    if out is None:
        out = torch.empty((m, n), dtype=out_dtype, device=x.device)
    kernels._rows(out, "out", out_dtype)
    if out.shape != (m, n):
        raise KernelError(f"out {tuple(out.shape)} for a result of {(m, n)}")
    ld = out.stride(0) if m > 1 else max(n, out.stride(0))
    check(l.gi_int4_linear(_ptr(x), _ptr(w.tiles), _ptr(out), code(out_dtype), ld, m, w.n, w.k, int(unit is not None),
                           *(unit or (0, 1.0, float("inf"), float("inf"), 0.0)), int(ranks), int(parts), _ptr(kernels.tcgen05_error_flag(x.device)), _stream()), l)
    return out


# -------------------------------------------------------------------------------------------------------------- cache
def _pools(k_rows: Int4Rows, v_rows: Int4Rows) -> tuple:
    for r, name in ((k_rows, "k_rows"), (v_rows, "v_rows")):
        if not isinstance(r, Int4Rows):
            raise KernelError(f"{name} is a {type(r).__name__}; pages in 4 bits are an Int4Rows")
        _on_gpu(r.codes, name)
    if k_rows.shape != v_rows.shape:
        raise KernelError(f"pages of keys {k_rows.shape} and of values {v_rows.shape} differ")
    return k_rows.shape


def _ints(**named) -> None:
    for name, t in named.items():
        _dense(t, name, torch.int32)


def _tokens(n: int, tok_pos: torch.Tensor, tok_slot: torch.Tensor) -> None:
    if tok_pos.numel() < n or tok_slot.numel() < n:
        raise KernelError("tok_pos / tok_slot are shorter than the token rows")


def _table(block_table: torch.Tensor) -> tuple:
    if block_table.dim() != 2:
        raise KernelError(f"a block table is [slots, pages], not {tuple(block_table.shape)}")
    return tuple(block_table.shape)


def append(k: torch.Tensor, v: torch.Tensor, k_rows: Int4Rows, v_rows: Int4Rows, block_table: torch.Tensor, tok_pos: torch.Tensor,
           tok_slot: torch.Tensor, status: torch.Tensor) -> None:
    """Keys and values [n, heads, d] (bfloat16 or float32; tokens and heads may lie apart, numbers of a head may not) of the step's
    tokens into their pages.  Tokens with slot -1 are padding; a place outside the cache is reported in `status` and not
    written.  The tokens' places are distinct."""
    l = require_gpu()
    n_pages, heads, page_size, d = _pools(k_rows, v_rows)
    for t, name in ((k, "k"), (v, "v")):
        _on_gpu(t, name)
        if t.dim() != 3 or tuple(t.shape[1:]) != (heads, d) or t.stride(2) != 1 or t.dtype != k.dtype or t.shape != k.shape:
            raise KernelError(f"{name} {tuple(t.shape)} of {t.dtype} (strides {t.stride()}) is no [n, {heads}, {d}] with dense heads")
    _ints(block_table=block_table, tok_pos=tok_pos, tok_slot=tok_slot, status=status)
    n = k.shape[0]
    _tokens(n, tok_pos, tok_slot)
    n_slots, width = _table(block_table)
    check(l.gi_int4_append(_ptr(k), k.stride(0), k.stride(1), _ptr(v), v.stride(0), v.stride(1), code(k.dtype), _ptr(k_rows.codes),
                           _ptr(k_rows.meta), _ptr(v_rows.codes), _ptr(v_rows.meta), _ptr(block_table), _ptr(tok_pos), _ptr(tok_slot),
                           n, heads, d, n_slots, width, page_size, n_pages, _ptr(status), _stream()), l)


def read(rows: Int4Rows, block_table: torch.Tensor, tok_pos: torch.Tensor, tok_slot: torch.Tensor, status: torch.Tensor,
         dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """What the pages hold of the listed tokens, [n, heads, d] in `dtype`; zeros for slot -1 and where nothing is mapped (which
    `status` reports)."""
    l = require_gpu()
    n_pages, heads, page_size, d = _pools(rows, rows)
    _ints(block_table=block_table, tok_pos=tok_pos, tok_slot=tok_slot, status=status)
    n = tok_pos.numel()
    _tokens(n, tok_pos, tok_slot)
    n_slots, width = _table(block_table)
    out = torch.empty((n, heads, d), dtype=dtype, device=rows.codes.device)
    check(l.gi_int4_read(_ptr(rows.codes), _ptr(rows.meta), _ptr(out), code(dtype), _ptr(block_table), _ptr(tok_pos), _ptr(tok_slot),
                         n, heads, d, n_slots, width, page_size, n_pages, _ptr(status), _stream()), l)
    return out


def attention_takes(dtype: torch.dtype, head_dim: int) -> bool:
    """Whether attention over a cache in 4 bits takes this activation type and head size."""
    return dtype == torch.bfloat16 and head_dim in (64, 128)


def _queries(q: torch.Tensor, shape: tuple) -> tuple:
    _dense(q, "q", torch.bfloat16)
    if q.dim() != 3 or q.shape[2] != shape[3] or q.shape[2] not in (64, 128) or q.shape[1] % shape[1] or q.shape[1] < 1:
        raise KernelError(f"queries {tuple(q.shape)} over pages of {shape[1]} heads of {shape[3]}: [n, a multiple of the heads, 64 or 128]")
    return tuple(q.shape)


def _few(q, k_rows, v_rows, block_table, runs, n_runs, most_rows, tok_pos, tok_slot, scale, window, status, out, n_splits) -> None:
    l = require_gpu()
    n_pages, heads, page_size, d = k_rows.shape
    n, n_q, _ = q.shape
    part_o = part_ml = None
    if n_splits > 1:
        part_o = torch.empty((n * n_q * n_splits * d,), dtype=torch.float32, device=q.device)
        part_ml = torch.empty((n * n_q * n_splits * 2,), dtype=torch.float32, device=q.device)
    check(l.gi_int4_attention(_ptr(q), _ptr(k_rows.codes), _ptr(k_rows.meta), _ptr(v_rows.codes), _ptr(v_rows.meta), _ptr(block_table),
                              _ptr(runs), n_runs, most_rows, _ptr(tok_pos), _ptr(tok_slot), _ptr(out), _ptr(part_o), _ptr(part_ml),
                              n_q, heads, d, block_table.shape[0], block_table.shape[1], page_size, n_pages, int(window or 0),
                              float(scale), n_splits, _ptr(status), _stream()), l)
    if n_splits > 1:
        check(l.gi_attention_decode_combine(_ptr(part_o), _ptr(part_ml), _ptr(out), n * n_q, d, n_splits, _stream()), l)


def decode_splits(n_runs: int, heads: int) -> int:
    """Slices of the keys per (run, key/value head, block of columns)."""
    return max(1, min(64, -(-888 // max(1, n_runs * heads))))


def attention_decode(q: torch.Tensor, k_rows: Int4Rows, v_rows: Int4Rows, block_table: torch.Tensor, tok_pos: torch.Tensor,
                     tok_slot: torch.Tensor, scale: float, window: int, status: torch.Tensor,
                     n_splits: Optional[int] = None) -> torch.Tensor:
    """Attention of one token per sequence, q [n, n_q, d] bfloat16 at positions `tok_pos` (their own keys are in the cache), over
    what the cache holds of their sequences; `window` > 0: the last `window` keys.  Returns [n, n_q * d]; rows of slot
    -1 are zeros.  d is 64 or 128."""
    shape = _pools(k_rows, v_rows)
    n, n_q, d = _queries(q, shape)
    _ints(block_table=block_table, tok_pos=tok_pos, tok_slot=tok_slot, status=status)
    _tokens(n, tok_pos, tok_slot)
    _table(block_table)
    out = torch.empty((n, n_q * d), dtype=q.dtype, device=q.device)
    _few(q, k_rows, v_rows, block_table, None, n, 1, tok_pos, tok_slot, scale, window, status, out, n_splits or decode_splits(n, shape[1]))
    return out


def attention_prompt(q: torch.Tensor, k_rows: Int4Rows, v_rows: Int4Rows, block_table: torch.Tensor, runs: torch.Tensor,
                     blocks: torch.Tensor, scale: float, window: int, status: torch.Tensor) -> torch.Tensor:
    """Attention of prompts, or portions of prompts, q [n, n_q, d] bfloat16, over the cache (the tokens' own keys are in it).  `runs`
    int32 [n_runs, 4] cuts the rows into runs of at most 128 consecutive tokens of one sequence: {slot, first row, rows, position
    of the first row}; rows in no run are zeros.  `blocks` int32 [n_blocks, 2] lists, each once, the blocks of 64 positions
    that any of them sees: {slot, position / 64}.  The blocks' keys and values are rounded to bfloat16 pages for the tensor-memory
    kernel.  Returns [n, n_q * d]."""
    l = require_gpu()
    shape = _pools(k_rows, v_rows)
    n_pages, heads, page_size, d = shape
    n, n_q, _ = _queries(q, shape)
    _ints(block_table=block_table, runs=runs, blocks=blocks, status=status)
    if runs.dim() != 2 or runs.shape[1] != 4 or blocks.dim() != 2 or blocks.shape[1] != 2:
        raise KernelError(f"runs {tuple(runs.shape)} and blocks {tuple(blocks.shape)} are no int32 [n_runs, 4] and [n_blocks, 2]")
    n_slots, width = _table(block_table)
    if runs.shape[0] == 0 or n == 0:
        return torch.zeros((n, n_q * d), dtype=q.dtype, device=q.device)
    n_blocks, max_blocks = blocks.shape[0], -(-width * page_size // 64)
    pages = torch.empty((2, n_blocks, heads, 64, d), dtype=q.dtype, device=q.device)
    table = torch.full((n_slots, max_blocks), -1, dtype=torch.int32, device=q.device)
    check(l.gi_int4_gather(_ptr(k_rows.codes), _ptr(k_rows.meta), _ptr(v_rows.codes), _ptr(v_rows.meta), _ptr(pages[0]), _ptr(pages[1]),
                           _ptr(table), _ptr(blocks), n_blocks, _ptr(block_table), heads, d, n_slots, width, max_blocks, page_size,
                           n_pages, _ptr(status), _stream()), l)
    return kernels.attention_prefill_tcgen05(q, pages[0], pages[1], table, runs, scale, window)
