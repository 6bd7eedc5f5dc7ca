"""Weights and cache rows in 4 bits: what holds them, and the entry points that make, read and use them.

A number q of 0 .. 15 stands for step * q + low, both bfloat16: one pair for 128 inputs of an output of a weight
(`Int4Weight`), one for 64 numbers of a head in the cache (`Int4Rows`).  Two numbers lie in a byte, the first in its low half.
A group with a number that is not finite stands for NaN.

  weights   `quantize_weight`, `dequantize_weight`; `linear` and its kin (linear.py) take an `Int4Weight` for their weight
  cache     `append` writes a step's keys and values (`qk_norm_rope_append`: out of the joined projection), `read` gives back what the pages hold of given tokens,
            `attention_decode` and `attention_prompt` read them

Products and attention compute with the numbers that the codes stand for, not with these rounded again, save where
`attention_prompt` and `linear` say so.  Upstream has neither.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional

import torch

from . import kernels
from .kernels import code
from .library import KernelError, check, require_gpu

GROUP_WEIGHT = 128          # inputs that share a step
GROUP_ROWS = 64             # numbers of a head that share a step
TILE_BYTES = 1088           # 16 outputs x 128 inputs: 1,024 bytes of codes, then (step, low) of the 16 outputs
_NO_UNIT = (0, 1.0, float("inf"), float("inf"), 0.0)
MAX_CLUSTER = 8             # slices of the keys that join themselves
PLACES, PLACES_WIDE = 592, 444      # blocks of the attention kernel that 148 SMs hold: for up to 8 columns, and for up to 16
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
        if self.n < 1 or self.k < 1 or self.tiles.dtype is not torch.uint8 or self.tiles.shape != want or not self.tiles.is_contiguous():
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
        shape = c.shape
        if len(shape) != 4 or c.dtype is not torch.uint8 or shape[3] < 32 or shape[3] % 32 or m.dtype is not torch.bfloat16 or \
                m.shape != (*shape[:3], shape[3] // 32, 2) or not (c.is_contiguous() and m.is_contiguous()):
            raise KernelError(f"codes {tuple(c.shape)} of {c.dtype} and steps {tuple(m.shape)} of {m.dtype} are no pages in 4 bits: "
                              "dense uint8 [pages, heads, page size, d / 2] and bfloat16 [pages, heads, page size, d / 64, 2], "
                              "d a multiple of 64")
        self.shape = (*shape[:3], shape[3] * 2)              # [pages, heads, page size, d], as a pool of numbers would have it
        self.index = c.get_device()                          # -1: not on a GPU
        if m.get_device() != self.index:
            raise KernelError(f"codes on {c.device} and steps on {m.device}")

    @property
    def head_dim(self) -> int:
        return self.shape[3]

    @staticmethod
    def zeros(pages: int, heads: int, page_size: int, head_dim: int, device) -> "Int4Rows":
        if head_dim < GROUP_ROWS or head_dim % GROUP_ROWS:
            raise KernelError(f"rows in 4 bits want heads that are a multiple of {GROUP_ROWS} numbers, not {head_dim}")
        return Int4Rows(torch.zeros((pages, heads, page_size, head_dim // 2), dtype=torch.uint8, device=device),
                        torch.zeros((pages, heads, page_size, head_dim // GROUP_ROWS, 2), dtype=torch.bfloat16, device=device))


# ------------------------------------------------------------------------------------------------------------ weights
def _stream(device: int) -> int:
    return torch._C._cuda_getCurrentRawStream(device)


def _check(device: int, t: torch.Tensor, name: str, dtype: Optional[torch.dtype] = None, dense: bool = True) -> int:
    """The tensor's address, after checking that it lies on the current device, `device` (the kernels are launched there)."""
    if t.get_device() != device:
        raise KernelError(f"{name} is on {t.device}; the kernels run on the current GPU, cuda:{device}")
    if dtype is not None and t.dtype is not dtype:
        raise KernelError(f"{name} is {t.dtype}, the kernel wants {dtype}")
    if dense and not t.is_contiguous():
        raise KernelError(f"{name} of shape {tuple(t.shape)} and strides {t.stride()} is not dense")
    return t.data_ptr()


def _start() -> tuple:
    return require_gpu(), torch._C._cuda_getDevice()


def quantize_weight(w: torch.Tensor) -> Int4Weight:
    """The weight [n, k] (bfloat16 or float32, rows may lie apart) in 4 bits: low = the group's smallest number, step =
    (largest - smallest) / 15, both rounded to bfloat16 so that the range covers the group; every number the nearest of the 16."""
    l, dev = _start()
    if w.dim() != 2 or w.shape[0] < 1 or w.shape[1] < 1 or w.stride(1) != 1:
        raise KernelError(f"a weight of shape {tuple(w.shape)} and strides {w.stride()}: [n, k] with dense rows, n and k at least 1")
    n, k = w.shape
    at = _check(dev, w, "w", dense=False)
    tiles = torch.empty((-(-n // 16), -(-k // GROUP_WEIGHT), TILE_BYTES), dtype=torch.uint8, device=w.device)
    check(l.gi_int4_quantize_weight(at, code(w.dtype), w.stride(0) if n > 1 else k, tiles.data_ptr(), n, k, _stream(dev)), l)
    return Int4Weight(tiles, n, k)


def dequantize_weight(w: Int4Weight, dtype: torch.dtype = torch.bfloat16, first: int = 0, rows: Optional[int] = None,
                      out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Outputs first .. first + rows - 1 of the weight as [rows, k] in `dtype` (rounded once)."""
    l, dev = _start()
    tiles = _check(dev, w.tiles, "w")
    rows = w.n - first if rows is None else rows
    if not 0 <= first <= first + rows <= w.n or rows < 1:
        raise KernelError(f"outputs {first} .. {first + rows - 1} of a weight of {w.n}")
    if out is None:
        out = torch.empty((rows, w.k), dtype=dtype, device=w.device)
    at = _check(dev, out, "out", dtype)
    if out.shape != (rows, w.k):
        raise KernelError(f"out {tuple(out.shape)} for {rows} outputs of {w.k} inputs")
    check(l.gi_int4_dequantize_weight(tiles, at, code(dtype), first, rows, w.n, w.k, _stream(dev)), l)
    return out


def linear_rows(x: torch.Tensor, w: Int4Weight, out_dtype: torch.dtype = torch.bfloat16, unit: Optional[tuple] = None,
                out: Optional[torch.Tensor] = None, ranks: int = 0, parts: int = 0) -> torch.Tensor:
    """x W^T for 1 to 16 rows of bfloat16 x, reading the weight's codes once; with `unit` (a `kernels.glu_shape` tuple) the gated
    unit of the weight's first half of outputs (a multiple of 16) and its last.  `out` may be columns of a wider matrix.
    `ranks`, `parts`: blocks that share the inputs, and parts of a block's share that its warps take (0: chosen by the entry point)."""
    l, at, tiles, to, m, ld, flag, dev, out = _product(x, w, out_dtype, unit, out, w.k)
    check(l.gi_int4_linear(at, tiles, to, code(out_dtype), ld, m, w.n, w.k, int(unit is not None), *(unit or _NO_UNIT), ranks, parts,
                           flag, _stream(dev)), l)
    return out


_rows_take: dict = {}


def linear_rows_takes(rows: int, w: Int4Weight, gated: bool) -> bool:
    """Whether `linear_rows` has room in shared memory for so many rows of x and their sums, which grow with the weight's inputs and
    outputs.  The answer is the same for 1 to 8 and for 9 to 16 rows, and is kept."""
    if not 1 <= rows <= LINEAR_MAX_ROWS:
        return False
    key = (rows > 8, w.n, w.k, gated, w.tiles.get_device())
    takes = _rows_take.get(key)
    if takes is None:
        takes = _rows_take[key] = bool(require_gpu().gi_int4_linear_takes(rows, w.n, w.k, int(gated)))
    return takes


def linear_wide(x: torch.Tensor, w: Int4Weight, out_dtype: torch.dtype = torch.bfloat16, unit: Optional[tuple] = None,
                out: Optional[torch.Tensor] = None, ranks: int = 0) -> torch.Tensor:
    """`linear_rows` for any number of rows (their length a multiple of 8, x on 16 bytes; for an odd inner size x has zeros behind it, up to
    the next multiple of 8): the numbers that the codes stand for are
    rounded to bfloat16 for the tensor cores, once for 32 or 64 rows.  `ranks`: blocks that share the inputs (0: chosen by the
    entry point)."""
    k = -(-w.k // 8) * 8
    l, at, tiles, to, m, ld, flag, dev, out = _product(x, w, out_dtype, unit, out, k)
    check(l.gi_int4_linear_tcgen05(at, tiles, to, code(out_dtype), ld, m, w.n, k, int(unit is not None), *(unit or _NO_UNIT), ranks,
                                   flag, _stream(dev)), l)
    return out


def _product(x, w, out_dtype, unit, out, k: int) -> tuple:
    l, dev = _start()
    at, tiles = _check(dev, x, "x", torch.bfloat16), _check(dev, w.tiles, "w")
    if x.dim() != 2 or x.shape[1] != k:
        raise KernelError(f"x {tuple(x.shape)} does not fit a weight {w.shape} ([out, in]): rows of {k}")
    m, n = x.shape[0], w.n // 2 if unit is not None else w.n
    if out is None:
        out = x.new_empty((m, n), dtype=out_dtype)
    elif out.shape != (m, n) or n > 1 and out.stride(1) != 1:
        raise KernelError(f"out {tuple(out.shape)} (strides {out.stride()}) for a result of {(m, n)} with dense rows")
    to = _check(dev, out, "out", out_dtype, dense=False)
    flag = kernels._tcgen05_flag.get(dev)
    if flag is None:
        flag = kernels.tcgen05_error_flag(x.device)
    return l, at, tiles, to, m, out.stride(0) if m > 1 else n, flag.data_ptr(), dev, out


# -------------------------------------------------------------------------------------------------------------- cache
def _pools(dev: int, k_rows: Int4Rows, v_rows: Int4Rows) -> tuple:
    """(shape, addresses of the keys' codes and steps, the values')"""
    if not isinstance(k_rows, Int4Rows) or not isinstance(v_rows, Int4Rows):
        raise KernelError(f"pages in 4 bits are an Int4Rows, not {type(k_rows).__name__} and {type(v_rows).__name__}")
    shape = k_rows.shape
    if shape != v_rows.shape:
        raise KernelError(f"pages of keys {shape} and of values {v_rows.shape} differ")
    if k_rows.index != dev or v_rows.index != dev:
        raise KernelError(f"pages on {k_rows.codes.device} and {v_rows.codes.device}; the kernels run on the current GPU, cuda:{dev}")
    return shape, (k_rows.codes.data_ptr(), k_rows.meta.data_ptr(), v_rows.codes.data_ptr(), v_rows.meta.data_ptr())


def _table(dev: int, block_table: torch.Tensor) -> tuple:
    if block_table.dim() != 2:
        raise KernelError(f"a block table is [slots, pages], not {tuple(block_table.shape)}")
    return _check(dev, block_table, "block_table", torch.int32), *block_table.shape


def _tokens(dev: int, n: int, tok_pos: torch.Tensor, tok_slot: torch.Tensor) -> tuple:
    if tok_pos.numel() < n or tok_slot.numel() < n:
        raise KernelError("tok_pos / tok_slot are shorter than the token rows")
    return _check(dev, tok_pos, "tok_pos", torch.int32), _check(dev, tok_slot, "tok_slot", torch.int32)


def _status(dev: int, status: torch.Tensor) -> int:
    if status.numel() < 1:
        raise KernelError("status is one int32")
    return _check(dev, status, "status", torch.int32)


def append(k: torch.Tensor, v: torch.Tensor, k_rows: Int4Rows, v_rows: Int4Rows, block_table: torch.Tensor, tok_pos: torch.Tensor,
           tok_slot: torch.Tensor, status: torch.Tensor) -> None:
    """Keys and values [n, heads, d] (bfloat16 or float32; tokens and heads may lie apart, numbers of a head may not) of the step's
    tokens into their pages.  Tokens with slot -1 are padding; a place outside the cache is reported in `status` and not
    written.  The tokens' places are distinct."""
    l, dev = _start()
    (n_pages, heads, page_size, d), pools = _pools(dev, k_rows, v_rows)
    n = k.shape[0]
    if k.shape != (n, heads, d) or v.shape != k.shape or v.dtype is not k.dtype or k.stride(2) != 1 or v.stride(2) != 1:
        raise KernelError(f"k {tuple(k.shape)} and v {tuple(v.shape)} of {k.dtype} and {v.dtype} (strides {k.stride()}, {v.stride()}) are no "
                          f"[n, {heads}, {d}] of one type with dense heads")
    table, n_slots, width = _table(dev, block_table)
    pos, slot = _tokens(dev, n, tok_pos, tok_slot)
    check(l.gi_int4_append(_check(dev, k, "k", dense=False), k.stride(0), k.stride(1), _check(dev, v, "v", dense=False), v.stride(0),
                           v.stride(1), code(k.dtype), *pools, table, pos, slot, n, heads, d, n_slots, width, page_size, n_pages,
                           _status(dev, status), _stream(dev)), l)


def qk_norm_rope_append(qkv: torch.Tensor, n_q: int, n_kv: int, head_dim: int, q_weight: Optional[torch.Tensor],
                        k_weight: Optional[torch.Tensor], eps: float, cos: torch.Tensor, sin: torch.Tensor, rotary_dim: int,
                        tok_pos: torch.Tensor, tok_slot: torch.Tensor, k_rows: Int4Rows, v_rows: Int4Rows, block_table: torch.Tensor,
                        status: torch.Tensor, append: bool = True) -> torch.Tensor:
    """`kernels.qk_norm_rope_append` over pages in 4 bits: norm and rotate q and k of packed projections [n, (n_q + 2 n_kv) d];
    returns q [n, n_q, d] and (with `append`) writes k (not rounded to bfloat16 before) and v of every token with a slot."""
    l, dev = _start()
    shape, pools = _pools(dev, k_rows, v_rows)
    n_pages, heads, page_size, d = shape
    at = _check(dev, qkv, "qkv", torch.bfloat16)
    if (heads, d) != (n_kv, head_dim) or qkv.dim() != 2 or qkv.shape[1] != (n_q + 2 * n_kv) * head_dim:
        raise KernelError(f"projections {tuple(qkv.shape)} and pages {shape} do not fit {n_q} query heads and {n_kv} key/value heads of "
                          f"{head_dim}")
    n = qkv.shape[0]
    if cos.dim() != 2 or cos.shape != sin.shape or cos.shape[1] * 2 != rotary_dim:
        raise KernelError(f"rotary tables {tuple(cos.shape)} and {tuple(sin.shape)} do not fit rotary_dim {rotary_dim}")
    q_w = k_w = None
    w_code = 0
    if (q_weight is None) != (k_weight is None):
        raise KernelError("q and k norm weights go together")
    if q_weight is not None:
        q_w, k_w, w_code = _check(dev, q_weight, "q_weight"), _check(dev, k_weight, "k_weight", q_weight.dtype), code(q_weight.dtype)
        if q_weight.numel() != head_dim or k_weight.numel() != head_dim:
            raise KernelError("q/k norm weights must have head_dim elements")
    table, n_slots, width = _table(dev, block_table)
    pos, slot = _tokens(dev, n, tok_pos, tok_slot)
    q = qkv.new_empty((n, n_q, head_dim))
    check(l.gi_int4_qk_norm_rope_append(at, q.data_ptr(), *pools, q_w, k_w, w_code, float(eps), _check(dev, cos, "cos", torch.float32),
                                        _check(dev, sin, "sin", torch.float32), rotary_dim, pos, slot, table, n, n_q, n_kv, head_dim,
                                        n_slots, width, page_size, n_pages, cos.shape[0], int(append), _status(dev, status),
                                        _stream(dev)), l)
    return q


def read(rows: Int4Rows, block_table: torch.Tensor, tok_pos: torch.Tensor, tok_slot: torch.Tensor, status: torch.Tensor,
         dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """What the pages hold of the listed tokens, [n, heads, d] in `dtype`; zeros for slot -1 and where nothing is mapped (which
    `status` reports)."""
    l, dev = _start()
    (n_pages, heads, page_size, d), pools = _pools(dev, rows, rows)
    n = tok_pos.numel()
    table, n_slots, width = _table(dev, block_table)
    pos, slot = _tokens(dev, n, tok_pos, tok_slot)
    out = rows.meta.new_empty((n, heads, d), dtype=dtype)
    check(l.gi_int4_read(pools[0], pools[1], out.data_ptr(), code(dtype), table, pos, slot, n, heads, d, n_slots, width, page_size,
                         n_pages, _status(dev, status), _stream(dev)), l)
    return out


def attention_takes(dtype: torch.dtype, head_dim: int) -> bool:
    """Whether attention over a cache in 4 bits takes this activation type and head size."""
    return dtype == torch.bfloat16 and head_dim in (64, 128)


def _queries(dev: int, q: torch.Tensor, shape: tuple) -> int:
    if q.dim() != 3 or q.shape[2] != shape[3] or q.shape[2] not in (64, 128) or q.shape[1] % shape[1] or q.shape[1] < 1:
        raise KernelError(f"queries {tuple(q.shape)} over pages of {shape[1]} heads of {shape[3]}: [n, a multiple of the heads, 64 or 128]")
    return _check(dev, q, "q", torch.bfloat16)


def _few(l, dev: int, q: torch.Tensor, at: int, shape: tuple, pools: tuple, table: tuple, runs, n_runs: int, pos, slot, scale: float,
         window: int, status: torch.Tensor, out: torch.Tensor, n_splits: int, blocks: int, places: int) -> torch.Tensor:
    """`blocks`: of the kernel, without slices; `places`: how many blocks of its kind run at once.  Up to 8 slices are a cluster and join
    themselves where all blocks have a place at once (8 runs of 2,048 keys, 6 slices: 12.7 us, 14.0 with a second kernel, part of the pages
    in L2); where they wait for places, a cluster waits for as many as it has blocks (64 runs of 500 keys, 4 slices: 35.7 against 24.3)."""
    n_pages, heads, page_size, d = shape
    n, n_q, _ = q.shape
    part_o = part_ml = None
    if n_splits > MAX_CLUSTER or n_splits > 1 and n_splits * blocks > places:      # one workspace: the slices' sums, then their maxima and weights
        room = q.new_empty((n * n_q * n_splits * (d + 2),), dtype=torch.float32)
        part_o = room.data_ptr()
        part_ml = part_o + n * n_q * n_splits * d * 4
        kernels.counters.launches += 1                       # the kernel that joins the slices
    check(l.gi_int4_attention(at, *pools, table[0], runs, n_runs, n, pos, slot, out.data_ptr(), part_o, part_ml, n_q, heads, d, table[1],
                              table[2], page_size, n_pages, window, scale, n_splits, _status(dev, status), _stream(dev)), l)
    return out


def _tiles(columns: int) -> tuple:
    """(blocks of a run's columns, how many such blocks run at once): 8 columns a block up to 8, 16 beyond.  Slices by these counts, by those of 8
    columns for all, in us: 8 runs of 2,048 keys, 8 heads of 128, groups of 16 17.5, 27.8; 20 of 2,000, 4 heads of 64, groups of 32 17.7,
    27.5; 1 of 131,000, 8 heads of 128, groups of 16 68.8, 86.9."""
    return (1, PLACES) if columns <= 8 else (-(-columns // 16), PLACES_WIDE)


def decode_splits(n_runs: int, heads: int, keys: int, places: int = PLACES, uneven: int = 1024) -> int:
    """Slices of the keys per (run, key/value head): as many as fill the 148 SMs with 4 blocks each (`places`), a run of many keys among
    others one for every `uneven` keys up to 8 (lengths may differ, and are not known here), none of fewer than 256 keys, 8
    instead of a few more (they join themselves).  `keys`: what the table's width or the window lets a run see, which is the cache's
    capacity rather than a length; runs far below it pay for slices that are empty.  Heads of 128, us by slices, nothing in L2:
      8 runs of 2,048 keys, 8 heads    1: 21.3   4: 12.8   6: 14.3   8: 14.8   14: 15.8   74: 23.5      (8 taken)
      1 run of 131,000 keys, 8 heads   37: 47.5   55: 44.6   74: 45.7   111: 53.0                       (74)
      1 run of 4,000 keys, 8 heads     1: 36.4   4: 14.6   8: 10.6   16: 10.3                           (16)
      48 runs of 1 .. 8,000, 8 heads   1: 87.0   4: 64.2   7: 61.2   9: 63.1   14: 68.9                 (7)
      64 runs of 500 keys, 8 heads     1: 18.3   2: 26.3   8: 29.8                                      (1; 8 in a table of 262,144)
      1 run of 100 keys, 8 heads       1: 5.9   4: 7.4   74: 11.3                                       (1; 74 in a table of 131,072)"""
    n = max(1, min(max(places // max(1, n_runs * heads), min(8, keys // uneven)), -(-keys // 256), 74))
    return 8 if 8 < n < 12 else n


# Up to how many columns (tokens x query heads of a key/value head) of a run, on average, `attention_prompt` reads the codes.  12 runs of
# 3,000 keys, 8 heads of 128, in us against 153 with wide pages: 20 columns 51, 64 columns 82, 96 columns 137, 128 columns 154; 40 runs
# of 1,000 keys against 163: 62, 96, 147, 185.
FEW_COLUMNS = 96
# Wide pages of a layer's step: up to so many bytes a step of short and long sequences is one call, beyond them two; and where more than one
# sequence would fill them, so many at a time.  8 key/value heads of 128, groups of 4, us and MB held, as one call / split:
#   4 x 1 behind 500, 300 new        59 (11) / 121 (3): launches            47 x 1 behind 6,000, 512 new       269 (22) / 138 (7)
#   8 x 1 behind 2,000, 200 of 2,200 202 (1) / 112 (10)                     40 x 1 behind 8,000, 2,048 new   1,116 (1,284) / 186 (24)
#   6 x 512 behind 30,000            1,890 (740) / 1,960 (262)              32 x 1 behind 8,000, 4,096 new   1,034 (1,056) / 300 (48)
TOGETHER_BYTES = 32 << 20
GATHER_BYTES = 256 << 20


def attention_decode(q: torch.Tensor, k_rows: Int4Rows, v_rows: Int4Rows, block_table: torch.Tensor, tok_pos: torch.Tensor,
                     tok_slot: torch.Tensor, scale: float, window: int, status: torch.Tensor,
                     n_splits: Optional[int] = None) -> torch.Tensor:
    """Attention of one token per sequence, q [n, n_q, d] bfloat16 at positions `tok_pos` (their own keys are in the cache), over
    what the cache holds of their sequences; `window` > 0: the last `window` keys.  Returns [n, n_q * d]; rows of slot
    -1 are zeros.  d is 64 or 128."""
    l, dev = _start()
    shape, pools = _pools(dev, k_rows, v_rows)
    at = _queries(dev, q, shape)
    n, n_q, d = q.shape
    pos, slot = _tokens(dev, n, tok_pos, tok_slot)
    table = _table(dev, block_table)
    window = int(window or 0)
    tiles, places = _tiles(n_q // shape[1])
    if not n_splits:
        keys = table[2] * shape[2]
        n_splits = decode_splits(n * tiles, shape[1], min(keys, window) if window else keys, places)
    return _few(l, dev, q, at, shape, pools, table, None, n, pos, slot, scale, window, status, q.new_empty((n, n_q * d)), n_splits,
                n * shape[1] * tiles, places)


def attention_prompt(q: torch.Tensor, k_rows: Int4Rows, v_rows: Int4Rows, block_table: torch.Tensor, runs: torch.Tensor,
                     blocks: torch.Tensor, scale: float, window: int, status: torch.Tensor,
                     out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of prompts, or portions of prompts, q [n, n_q, d] bfloat16, over the cache (the tokens' own keys are in it).  `runs`
    int32 [n_runs, 4] cuts the rows into runs of at most 128 consecutive tokens of one sequence: {slot, first row, rows, position
    of the first row}; rows in no run are zeros, no row is in two.  `blocks` int32 [n_blocks, 2] lists, each once, the blocks of 64
    positions that any of them sees: {slot, position / 64}.  Runs of a few tokens read the cache as single tokens do;
    for longer ones the blocks' keys and values are rounded to bfloat16 pages for the tensor-memory kernel.  One call has one way, by the
    mean length of its runs: short runs beside long ones are `attention_some`'s.  Returns [n, n_q * d]; `out` (dense): written there, rows
    in no run stay as they are (those of a run that names no slot, or what does not exist, stay or become zeros)."""
    return _prompt(q, k_rows, v_rows, block_table, runs, blocks, scale, window, status, out)


def attention_some(q: torch.Tensor, rows: torch.Tensor, k_rows: Int4Rows, v_rows: Int4Rows, block_table: torch.Tensor, runs: torch.Tensor,
                   blocks: torch.Tensor, scale: float, window: int, status: torch.Tensor, out: torch.Tensor) -> torch.Tensor:
    """`attention_prompt` for some rows of q: `rows` int32 names them, each once, and `runs` counts in that list.  Their results go into the
    same rows of `out` [n, n_q * d], which is returned; the others stay as they are.  A row that does not exist is reported in `status`.  A step of single tokens and long prompts is one
    call of each: the tokens' keys are read as codes, only the prompts' are gathered."""
    l, dev = _start()
    if rows.dim() != 1 or q.dim() != 3 or out.shape != (q.shape[0], q.shape[1] * q.shape[2]):
        raise KernelError(f"rows {tuple(rows.shape)} of queries {tuple(q.shape)} into {tuple(out.shape)}")
    n, n_q, d = q.shape
    some = q.new_empty((rows.shape[0], n_q, d))
    move = (_check(dev, rows, "rows", torch.int32), some.shape[0], n, n_q * d * 2)
    check(l.gi_int4_move_rows(_check(dev, q, "q", torch.bfloat16), some.data_ptr(), *move, 0, _status(dev, status), _stream(dev)), l)
    to = _check(dev, out, "out", torch.bfloat16)
    done = _prompt(some, k_rows, v_rows, block_table, runs, blocks, scale, window, status, None)
    check(l.gi_int4_move_rows(to, done.data_ptr(), *move, 1, _status(dev, status), _stream(dev)), l)
    return out


def _prompt(q, k_rows, v_rows, block_table, runs, blocks, scale: float, window: int, status, out) -> torch.Tensor:
    l, dev = _start()
    shape, pools = _pools(dev, k_rows, v_rows)
    n_pages, heads, page_size, d = shape
    at = _queries(dev, q, shape)
    n, n_q, _ = q.shape
    if runs.dim() != 2 or runs.shape[1] != 4 or blocks.dim() != 2 or blocks.shape[1] != 2:
        raise KernelError(f"runs {tuple(runs.shape)} and blocks {tuple(blocks.shape)} are no int32 [n_runs, 4] and [n_blocks, 2]")
    runs_at, blocks_at = _check(dev, runs, "runs", torch.int32), _check(dev, blocks, "blocks", torch.int32)
    table = _table(dev, block_table)
    _, n_slots, width = table
    window, n_runs, n_blocks = int(window or 0), runs.shape[0], blocks.shape[0]
    if out is not None and (out.shape != (n, n_q * d) or _check(dev, out, "out", torch.bfloat16) % 16):
        raise KernelError(f"out {tuple(out.shape)} for a result of {(n, n_q * d)} that starts on 16 bytes")
    if n_runs == 0 or n == 0:
        return q.new_zeros((n, n_q * d)) if out is None else out
    columns = -(-n * (n_q // heads) // n_runs)
    if columns <= FEW_COLUMNS:
        tiles, places = _tiles(columns)
        return _few(l, dev, q, at, shape, pools, table, runs_at, n_runs, None, None, scale, window, status,
                    q.new_zeros((n, n_q * d)) if out is None else out, decode_splits(n_runs * tiles, heads, 64 * n_blocks // n_runs, places, 2048), n_runs * heads * tiles, places)
    if n_blocks == 0:
        raise KernelError(f"{n_runs} runs that see no block of the cache")
    max_blocks = -(-width * page_size // 64)
    kept = torch.empty_like(runs)
    pages = q.new_empty((2, n_blocks, heads, 64, d))
    new_table = block_table.new_full((n_slots, max_blocks), -1)
    check(l.gi_int4_gather(*pools, pages[0].data_ptr(), pages[1].data_ptr(), new_table.data_ptr(), blocks_at, n_blocks, runs_at,
                           kept.data_ptr(), n_runs, n, table[0], heads, d, n_slots, width, max_blocks, page_size, n_pages, window,
                           _status(dev, status), _stream(dev)), l)
    return kernels.attention_prefill_tcgen05(q, pages[0], pages[1], new_table, kept, scale, window, out=out)
