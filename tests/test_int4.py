"""4 bits without a GPU: what the holders of weights and pages refuse, the cache's pages, the options of the entry points."""
import numpy as np
import pytest
import torch

from garlic_inference_b200.cache import CacheError, KVRequirement, PagedCache
from garlic_inference_b200.cli import build_parser
from garlic_inference_b200.engine import AutoModel
from garlic_inference_b200.ops import KernelError, int4
from garlic_inference_b200.parts import Runtime, StepShape, part_class
from garlic_inference_b200.parts.attention import key_blocks


def test_weights_are_held_in_whole_tiles():
    good = torch.zeros(3, 2, 1088, dtype=torch.uint8)
    w = int4.Int4Weight(good, 33, 129)
    assert w.shape == (33, 129) and w.numel() == 33 * 129 and w.bytes() == 6 * 1088
    for tiles, n, k in ((good, 49, 129), (good, 32, 129), (good, 33, 257), (good, 0, 129), (good, 33, 0), (good[:, :1], 33, 129),
                        (good.transpose(0, 1).contiguous().transpose(0, 1), 33, 129), (good.to(torch.int8), 33, 129),
                        (good.reshape(6, 1088), 33, 129)):
        with pytest.raises(KernelError, match="tiles"):
            int4.Int4Weight(tiles, n, k)


def test_pages_are_held_dense():
    codes, meta = torch.zeros(2, 3, 4, 64, dtype=torch.uint8), torch.zeros(2, 3, 4, 2, 2, dtype=torch.bfloat16)
    assert int4.Int4Rows(codes, meta).shape == (2, 3, 4, 128)
    for c, m in ((codes, meta[..., :1]), (codes, meta.float()), (codes.short(), meta), (codes[..., :48], meta), (codes[:1], meta),
                 (codes.transpose(1, 2), meta.transpose(1, 2)), (codes[..., ::2], meta[..., :1, :]), (codes[0], meta[0])):
        with pytest.raises(KernelError, match="no pages in 4 bits"):
            int4.Int4Rows(c, m)
    for d in (0, 32, 96):
        with pytest.raises(KernelError, match="multiple of 64"):
            int4.Int4Rows.zeros(1, 1, 4, d, "cpu")


def test_slices_of_the_keys():
    for n in (1, 2, 7, 64, 1000):
        for heads in (1, 2, 8, 40):
            for keys in (1, 64, 255, 257, 5000, 1 << 20):
                s = int4.decode_splits(n, heads, keys)
                assert 1 <= s <= 74 and (s - 1) * 256 < keys
    assert int4.decode_splits(1, 8, 131000) == 74 and int4.decode_splits(64, 8, 512) == 1


@pytest.mark.parametrize("window", [0, 1, 64, 65, 300])
def test_blocks_of_keys_that_a_step_sees(window):
    slots, lens, past = [4, 0, 2, 1], [3, 200, 1, 64], [0, 500, 127, 64]
    got = key_blocks(StepShape(slots, [0, 3, 203, 204], lens, past, False), window)
    want = {(s, j // 64) for s, n, p in zip(slots, lens, past) for i in range(p, p + n)
            for j in range(max(0, i - window + 1) if window else 0, i + 1)}
    assert got.dtype == np.int32 and len(got) == len(want) and {tuple(r) for r in got.tolist()} == want


def test_pages_of_the_cache():
    reqs = [KVRequirement(2, 128, bits=4), KVRequirement(2, 128), KVRequirement(2, 128, bits=4), KVRequirement(1, 64, window=40, bits=4)]
    cache = PagedCache(reqs, max_tokens=256, max_positions=256, dtype=torch.bfloat16, device="cpu", page_size=16)
    a, b, c, d = (cache.kv_view(i) for i in range(4))
    assert a.block_table is c.block_table and a.block_table is not b.block_table
    for v, shape in ((a, (16, 2, 16, 128)), (c, (16, 2, 16, 128)), (d, (16, 1, 16, 64))):
        assert isinstance(v.k_pool, int4.Int4Rows) and v.k_pool.shape == v.v_pool.shape == shape
    held = {t.data_ptr() for v in (a, c) for r in (v.k_pool, v.v_pool) for t in (r.codes, r.meta)}
    assert len(held) == 8 and isinstance(b.k_pool, torch.Tensor)
    # two numbers a byte and four bytes for 64 of them
    assert cache.bytes_per_token() == 2 * 2 * 2 * (64 + 8) + 2 * 2 * 128 * 2 + 2 * (32 + 4)
    for bad in (KVRequirement(2, 128, bits=8), KVRequirement(2, 128, planes=1, bits=4), KVRequirement(2, 128, value_dim=64, bits=4),
                KVRequirement(2, 128, window=64, mean_block=16, bits=4), KVRequirement(2, 128, window=64, keep_first=4, bits=4)):
        with pytest.raises(CacheError, match="bits"):
            PagedCache([bad], max_tokens=64, max_positions=64, dtype=torch.bfloat16, device="cpu", page_size=16)


class _Load:
    def __init__(self, shapes):
        self.shapes = shapes

    def dtype(self, *names):
        return torch.bfloat16

    def __call__(self, name, out=None):
        return torch.zeros(self.shapes[name].shape, dtype=torch.bfloat16) if out is None else out.zero_()


def test_attention_that_cannot_keep_its_keys_in_4_bits_says_so():
    cls = part_class("gqa_attention")
    for dtype, d in ((torch.float32, 128), (torch.bfloat16, 32), (torch.bfloat16, 96)):
        params = dict(hidden_size=64, n_heads=4, n_kv_heads=2, head_dim=d)
        with pytest.raises(ValueError, match="4 bits"):
            cls(params, _Load(cls.wanted(params)), Runtime(dtype, torch.device("cpu"), cache="int4"))
    params = dict(hidden_size=64, n_heads=4, n_kv_heads=2, head_dim=64)
    part = cls(params, _Load(cls.wanted(params)), Runtime(torch.bfloat16, torch.device("cpu"), cache="int4"))
    assert part.cache_requirement() == KVRequirement(2, 64, None, bits=4)


@pytest.mark.parametrize("name", ["weights", "cache"])
def test_options_of_the_entry_points(name, tmp_path):
    for make in (lambda **k: AutoModel.from_random(None, **k), lambda **k: AutoModel.from_pretrained(tmp_path, **k)):
        with pytest.raises(ValueError, match=f"{name} must be None or 'int4'"):
            make(**{name: "int8"})
    args = build_parser().parse_args(["folder", f"--{name}", "int4"])
    assert getattr(args, name) == "int4" and getattr(build_parser().parse_args(["folder"]), name) is None
    with pytest.raises(SystemExit):
        build_parser().parse_args(["folder", f"--{name}", "int2"])


def test_products_go_where_there_is_room(monkeypatch):
    """The choice of product against the capacity that the kernel for up to 16 rows states, over sizes on both sides of it."""
    from garlic_inference_b200.ops import lib, linear as entry, swiglu_product
    taken = []
    for name in ("linear_rows", "linear_wide"):
        monkeypatch.setattr(int4, name, lambda x, w, *a, name=name, **k: taken.append(name))
    monkeypatch.setattr(int4, "require_gpu", lib)
    monkeypatch.setattr(int4, "_rows_take", {})
    both = set()
    for k in (128, 1024, 4096, 8192, 16384, 28672, 32768, 120000):
        for n in (32, 2048, 8192, 57344, 106496, 152064):
            w = int4.Int4Weight(torch.empty(n // 16, -(-k // 128), 1088, dtype=torch.uint8, device="meta"), n, k)
            for m in (1, 8, 9, 12, 16, 17):
                x = torch.empty((m, k), dtype=torch.bfloat16, device="meta")
                for product, gated in ((entry, 0), (swiglu_product, 1)):
                    product(x, w)
                    takes = lib().gi_int4_linear_takes(m, n, k, gated)
                    both.add((takes, m <= 16))
                    assert taken.pop() == ("linear_rows" if takes else "linear_wide"), (m, n, k, gated)
    assert both == {(0, True), (1, True), (0, False)}


def test_gated_units_are_made_wide_in_bounded_pieces():
    from garlic_inference_b200.ops.linear import INT4_GATED_BYTES, _gated_columns
    for n in (16, 128, 4096, 12288, 57344, 700000):
        for k in (128, 4096, 8192, 120000, 2000000):
            c = _gated_columns(n, k)
            assert c == n if 4 * n * k <= INT4_GATED_BYTES // 2 else c == n or c < n and c % 128 == 0
            assert 4 * min(c, n) * k <= max(INT4_GATED_BYTES, 4 * 128 * k)
            assert -(-n // c) <= -(-4 * n * k // INT4_GATED_BYTES) * 2


def _layer(group, d=128, kv=2, window=None):
    cls = part_class("gqa_attention")
    params = dict(hidden_size=64, n_heads=kv * group, n_kv_heads=kv, head_dim=d, **({} if window is None else {"window": window}))
    return cls(params, _Load(cls.wanted(params)), Runtime(torch.bfloat16, torch.device("cpu"), cache="int4"))


@pytest.mark.parametrize("window", [None, 100])
@pytest.mark.parametrize("group", [1, 4, 7])
def test_steps_are_split_into_short_and_long_sequences(group, window, monkeypatch):
    """Over random steps: every row is in one run of one call, short sequences in the call that names its rows, every call's blocks are those
    that its own sequences see, and no list of long ones holds more than the limit unless it is one sequence."""
    import random
    rnd = random.Random(group)
    part = _layer(group, window=window)
    limit = 20
    monkeypatch.setattr(int4, "GATHER_BYTES", limit * 4 * 64 * part.n_kv * part.d)
    assert len(part._calls(StepShape([0, 1], [0, 1], [1, 300], [50, 0], False))[1]) == 1      # little to gather: one call
    monkeypatch.setattr(int4, "TOGETHER_BYTES", 0)
    kinds = set()
    for _ in range(60):
        n = rnd.randint(1, 9)
        lens = [rnd.choice([1, 1, 2, 20, 97, 130, 300]) for _ in range(n)]
        past = [rnd.choice([0, 5, 64, 500, 1500]) for _ in range(n)]
        slots = rnd.sample(range(20), n)
        starts = [sum(lens[:i]) for i in range(n)]
        shape = StepShape(slots, starts, lens, past, all(x == 1 for x in lens))
        if shape.all_single:
            continue
        arrays, calls = part._calls(shape)
        assert set(arrays) == {a for c in calls for a in c if a} and part.step_arrays(shape, None).keys() == arrays.keys()
        short = {i for i in range(n) if lens[i] * group <= int4.FEW_COLUMNS}
        covered = []
        for rows, runs, blocks in calls:
            of = np.arange(sum(lens)) if rows is None else arrays[rows]()
            seen, got, held = set(), arrays[runs](), arrays[blocks]()
            assert got.dtype == held.dtype == np.int32 and of.dtype in (np.int32, np.int64)
            who = set()
            for s, r, c, p in got.tolist():
                i = slots.index(s)
                who.add(i)
                assert 1 <= c <= 128 and [int(x) for x in of[r:r + c]] == list(range(starts[i] + p - past[i], starts[i] + p - past[i] + c))
                covered += [int(x) for x in of[r:r + c]]
                w = window or 1 << 30
                seen |= {(s, j // 64) for q in range(p, p + c) for j in (max(0, q - w + 1), q)}
                seen |= {(s, b) for b in range(max(0, p - w + 1) // 64, (p + c - 1) // 64 + 1)}
            assert {tuple(b) for b in held.tolist()} == seen and len(held) == len(seen)
            if len(calls) > 1:
                assert who <= short if rows else not who & short
                assert rows or len(who) == 1 or len(held) <= limit
        assert sorted(covered) == list(range(sum(lens)))
        kinds.add((len(calls) > 1, calls[-1][0] is not None))
    assert kinds >= {(False, False), (True, True)}


def test_slices_are_counted_with_the_blocks_that_run_at_once():
    """Groups of more than 8 have blocks of 16 columns, of which fewer run at once: whatever joins as clusters has a place, all at once."""
    assert int4._tiles(1) == int4._tiles(8) == (1, 592) and int4._tiles(9) == int4._tiles(16) == (1, 444) and int4._tiles(17) == (2, 444)
    for group in (1, 4, 8, 9, 12, 16, 24, 32, 48):
        tiles, places = int4._tiles(group)
        for n in (1, 3, 8, 20, 64, 300):
            for heads in (1, 4, 8):
                s = int4.decode_splits(n * tiles, heads, 2048, places)
                assert s <= 2 or s * n * tiles * heads <= places      # (2: runs of 2,048 keys may differ in length)
    assert int4.decode_splits(8, 8, 2048, 444) == 6
