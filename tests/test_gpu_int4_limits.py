"""4 bits at the limits of what the entry points take: float32 activations in recorded steps, sizes beyond one kernel's room, steps of unlike
runs, numbers far apart."""
import shutil

import pytest
import torch

import plain_int4 as plain
import tiny
from test_gpu_int4 import check_attention, gen, linear_bound, make_cache, random_weight, randn, runs_and_blocks, wide_bound
from test_gpu_int4_model import HELD, load

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(scope="module")
def ops():
    from garlic_inference_b200 import ops
    return ops


def held_folder(folder, to):
    """The model of `folder` with the numbers that its weights' codes stand for as float32 weights."""
    from garlic_inference_b200.ops import int4
    from garlic_inference_b200.weights import Checkpoint
    from garlic_inference_b200.weights.safetensors_io import write_safetensors
    ckpt = Checkpoint(folder)
    tensors = {}
    for n in ckpt.names():
        t = ckpt.tensor(n).clone()
        if any(f"{p}.weight" in n for p in HELD):
            t = int4.dequantize_weight(int4.quantize_weight(t.cuda()), torch.float32).cpu()
        tensors[n] = t
    shutil.copy(folder / "config.json", to / "config.json")
    write_safetensors(to / "model.safetensors", tensors)
    return to


# ------------------------------------------------------------------------------------------------ weights made wide
@pytest.mark.parametrize("name", ["D", "E"])
def test_float32_steps_recorded_and_eager(name, model_dirs, tmp_path):
    """Every layer's weight is made wide right in front of its product: recorded steps, whose kernels start early, give the bits
    of eager ones, and both the logits of the codes' numbers."""
    reqs = tiny.random_requests(tiny.TINY[name]["cfg"]["vocab_size"], [90, 41, 7], seed=6)
    want = tiny.plain_logits(held_folder(model_dirs(name), tmp_path), reqs)
    traces = (tiny.trace_tail_by_one(reqs, tail=24), tiny.trace_batched(reqs, [["r0", "r1", "r2"]], prompt_frac=0.5))
    for trace in traces:
        got = []
        for graphs in (True, False):
            model = load(model_dirs(name), max_tokens=384, dtype="float32", weights="int4", use_graphs=graphs)
            got.append(tiny.run_trace_in_process(model, trace))
            tiny.compare(got[-1], want, tiny.TOL["float32"], f"{name} graphs={graphs}")
        for rid in got[0]:
            for p in got[0][rid]:
                assert (got[0][rid][p] == got[1][rid][p]).all(), (rid, p)


@pytest.mark.parametrize("m,n,k", [(1, 256, 192), (3, 100, 384), (9, 64, 130), (1, 1024, 2048), (40, 2048, 1024)])
def test_products_right_behind_the_kernel_that_makes_their_weight(ops, m, n, k):
    """With launches that let the next kernel start early: weights of one size in turn, so that what the memory held before is another
    weight; float32 rows over 4-bit weights, and weights that are quantised in front of their product."""
    g = gen(m + n + k)
    ws = [randn(g, n, k) for _ in range(4)]
    held = [ops.int4.quantize_weight(w) for w in ws]
    x = randn(g, m, k)
    xb = x.to(torch.bfloat16)
    want = [(ops.linear(x, h), ops.linear(xb, h, torch.float32)) for h in held]
    torch.cuda.synchronize()
    from garlic_inference_b200.ops import kernels
    kernels.set_dependent_launch(True)
    try:
        for _ in range(5):
            got = []
            for w, h in zip(ws, held):
                a = ops.linear(x, h)
                fresh = ops.int4.quantize_weight(w)
                got.append((a, ops.linear(xb, fresh, torch.float32)))
                del fresh
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for p, q in zip(got, want) for a, b in zip(p, q))
    finally:
        kernels.set_dependent_launch(False)


# -------------------------------------------------------------------------------------------- sizes beyond a kernel's room
@pytest.mark.parametrize("m,n,k,gated", [(16, 2048, 32768, False), (9, 2048, 32768, False), (16, 32, 32768, True), (12, 152064, 4096, False),
                                         (10, 57344, 8192, True), (9, 8192, 28672, False), (1, 106496, 16384, True)])
def test_steps_of_few_rows_whose_sums_have_no_room_beside_them(ops, m, n, k, gated):
    g = gen(m + n + k)
    tile = torch.randint(0, 256, (n // 16, k // 128, 1088), dtype=torch.uint8, device=DEV, generator=g)
    tile[..., 1024:] = torch.tensor([0.01, -0.08], dtype=torch.bfloat16, device=DEV).view(torch.uint8).repeat(16)
    w = ops.int4.Int4Weight(tile, n, k)
    assert not ops.int4.linear_rows_takes(m, w, gated)
    x = randn(g, m, k).to(torch.bfloat16)
    got = ops.swiglu_product(x, w) if gated else ops.linear(x, w, torch.float32)
    half = n // 2 if gated else n
    assert got.shape == (m, half)
    # 16 outputs at either end (of both halves), each against 64 bits; bounds: test_gpu_int4.wide_bound, and a bfloat16 result of a unit
    for a in {0, half - 16}:
        parts = [ops.int4.Int4Weight(tile[i // 16:i // 16 + 1].clone(), 16, k) for i in ((a, half + a) if gated else (a,))]
        y = [x.double() @ plain.values(*plain.unpack_weight(p), 128).t() for p in parts]
        off = [wide_bound(x, p) for p in parts]
        if gated:
            want = y[0] * torch.sigmoid(y[0]) * y[1]
            bound = 2 ** -8 * want.abs() + 1.1 * off[0] * (y[1].abs() + off[1]) + y[0].abs() * off[1] + 2 ** -19 * (y[0] * y[1]).abs() + 2 ** -30
        else:
            want, bound = y[0], off[0] + 2 ** -24 * y[0].abs()
        assert float(((got[:, a:a + 16].double() - want).abs() / bound).max()) <= 1


def test_room_is_counted_with_the_clusters_that_the_device_holds(ops):
    """What the choice of product counts on is what the launch is made with: whatever is stated to fit runs, at the edges of the room."""
    l = ops.lib()
    held = [l.gi_int4_linear_held(r) for r in range(1, 9)]
    assert held[0] == torch.cuda.get_device_properties(0).multi_processor_count and all(0 < b * r <= held[0] for r, b in enumerate(held, 1))
    assert l.gi_int4_linear_held(0) == l.gi_int4_linear_held(9) == -1
    for m, k, gated in ((1, 16384, 1), (8, 16384, 1), (16, 4096, 0), (16, 8192, 1), (9, 28672, 0)):
        unit = 32
        low, high = 1, 8192                                  # outputs in units of 32: the last that fit, to within an eighth
        assert l.gi_int4_linear_takes(m, low * unit, k, gated) == 1
        while high - low > max(1, low // 8):
            mid = (low + high) // 2
            low, high = (mid, high) if l.gi_int4_linear_takes(m, mid * unit, k, gated) == 1 else (low, mid)
        n = low * unit
        tiles = torch.zeros(n // 16, k // 128, 1088, dtype=torch.uint8, device=DEV)
        tiles[..., 1024:] = torch.tensor([0.01, 0.5], dtype=torch.bfloat16, device=DEV).view(torch.uint8).repeat(16)
        w = ops.int4.Int4Weight(tiles, n, k)
        x = torch.ones((m, k), dtype=torch.bfloat16, device=DEV)
        unit_of = ops.kernels.glu_shape("silu") if gated else None
        got = ops.int4.linear_rows(x, w, torch.float32, unit_of)
        y = 0.5 * k                                          # every code is 0: sums of halves, exact in float32
        assert torch.equal(got, torch.full_like(got, y * y if gated else y))


@pytest.mark.parametrize("m", [1, 8, 11])
def test_large_inputs_and_steps_whose_product_is_no_number(ops, m):
    """x up to 2^115, steps up to 2^20: what an output's codes leave of them is finite, and zero where they all are.  Bound: the
    kernel's of test_gpu_int4.linear_bound, 8 roundings a group and the ends of sums whose numbers add up to A."""
    g = gen(m)
    n, k = 40, 300
    codes = torch.zeros(n, k, dtype=torch.long, device=DEV)
    codes[1::4, 3] = 1                                       # one input of one group
    codes[2::4, 200:210] = 15
    groups = 3
    step = torch.full((n, groups), 2.0 ** 20, device=DEV)
    step[2::4] = 2.0 ** 4
    low = torch.zeros(n, groups, device=DEV)
    low[3::4] = 1.0
    w = ops.int4.Int4Weight(plain.pack_weight(codes, step, low), n, k)
    x = torch.zeros(m, k, device=DEV)
    x[:, 100] = 2.0 ** 115                                   # meets codes of 0, or the low value 1
    x[:, 3] = randn(g, m) * 2.0 ** 100
    x[:, 200:210] = (1 + torch.rand(m, 10, generator=g, device=DEV)) * 2.0 ** 114
    x = x.to(torch.bfloat16)
    wide = plain.values(*plain.unpack_weight(w), 128)
    want = x.double() @ wide.t()
    assert bool((want[:, 0::4] == 0).all()) and bool((want.abs() < 2.0 ** 126).all())
    assert bool((want[:, 1::4] != 0).all()) and float(want[:, 2::4].abs().min()) > 2.0 ** 120
    got = ops.linear(x, w, torch.float32).double()
    assert bool(torch.isfinite(got).all()) and bool((got[:, 0::4] == 0).all())
    assert float(((got - want).abs() / (linear_bound(x, w) + 2 ** -24 * want.abs() + 2.0 ** -126)).max()) <= 1


# ------------------------------------------------------------------------------------------------ steps far apart
def far_apart(ops, heads, kv, d, page, lengths, seed, huge, where):
    """A filled cache whose values at the given (sequence, position) are `huge` times as large as the others."""
    g = gen(seed)
    k_rows, v_rows, table, status, k, v, pos, slot = make_cache(ops, g, lengths, kv, d, page)
    starts = [sum(lengths[:s]) for s in range(len(lengths))]
    for s, p in where:
        v[starts[s] + p] *= huge
    ops.int4.append(k, v, k_rows, v_rows, table, pos, slot, status)
    return g, k_rows, v_rows, table, status


@pytest.mark.parametrize("huge", [2.0 ** 20, 2.0 ** 40, 2.0 ** 100])
@pytest.mark.parametrize("heads,d,page", [(4, 128, 64), (2, 64, 64), (12, 128, 16)])
def test_large_values_behind_the_window_leave_no_trace(ops, heads, d, page, huge):
    """Keys in front of the window lie in the first chunk of keys that is read: whatever their values' size, a token's result is as exact as
    without them."""
    window, n = 70, 300
    first = n - window
    g, k_rows, v_rows, table, status = far_apart(ops, heads, 1, d, page, [n, n], 41, huge, [(0, p) for p in range(first - 20, first)])
    q = randn(g, 2, heads, d).to(torch.bfloat16)
    pos, slot = torch.full((2,), n - 1, dtype=torch.int32, device=DEV), torch.arange(2, dtype=torch.int32, device=DEV)
    for splits in (None, 1):
        got = ops.int4.attention_decode(q, k_rows, v_rows, table, pos, slot, d ** -0.5, window, status, n_splits=splits)
        check_attention(got, *plain.attention(q, k_rows, v_rows, table, [(0, 0, 1, n - 1), (1, 1, 1, n - 1)], d ** -0.5, window))


@pytest.mark.parametrize("huge", [2.0 ** 20, 2.0 ** 40, 2.0 ** 100])
@pytest.mark.parametrize("heads,kv,d,seqs", [(4, 1, 128, [(200, 4), (33, 2)]), (4, 2, 64, [(64, 3), (0, 5)]), (8, 1, 128, [(90, 6)])])
def test_large_values_of_later_tokens_leave_no_trace(ops, heads, kv, d, seqs, huge):
    """The tokens of a run in front of one with large values do not see it: their results are as exact as without it."""
    where = [(s, p + n - 2 if n > 2 else p + n - 1) for s, (p, n) in enumerate(seqs)]
    g, k_rows, v_rows, table, status = far_apart(ops, heads, kv, d, 64, [p + n for p, n in seqs], 43, huge, where)
    spans, row = [], 0
    for s, (p, n) in enumerate(seqs):
        spans.append((s, row, n, p))
        row += n
    q = randn(g, row, heads, d).to(torch.bfloat16)
    runs, blocks = runs_and_blocks(spans, 0)
    got = ops.int4.attention_prompt(q, k_rows, v_rows, table, runs, blocks, d ** -0.5, 0, status)
    check_attention(got, *plain.attention(q, k_rows, v_rows, table, spans, d ** -0.5, 0))


@pytest.mark.parametrize("ratio", [2.0 ** 12, 2.0 ** 30, 2.0 ** 60])
@pytest.mark.parametrize("heads,d,at", [(4, 128, 3), (2, 64, 40), (16, 128, 255)])
def test_a_large_value_with_hardly_any_weight_costs_the_others_nothing(ops, heads, d, at, ratio):
    """One key's probability is 2^-69 or so of the others' and its values are `ratio` times as large: the others keep their bits."""
    n = 256
    g = gen(47)
    k_rows, v_rows, table, status, k, v, pos, slot = make_cache(ops, g, [n], 1, d, 64)
    q = torch.ones(1, heads, d, device=DEV).to(torch.bfloat16)
    k *= 0.1
    k[at] = -48.0 / d ** 0.5                                 # its score is 48 below the others'
    v[at] *= ratio
    ops.int4.append(k, v, k_rows, v_rows, table, pos, slot, status)
    spans = [(0, 0, 1, n - 1)]
    for splits in (None, 1):
        got = ops.int4.attention_decode(q, k_rows, v_rows, table, pos[-1:], slot[:1], d ** -0.5, 0, status, n_splits=splits)
        check_attention(got, *plain.attention(q, k_rows, v_rows, table, spans, d ** -0.5, 0))


def test_values_of_all_sizes(ops):
    """Every token's values are a power of two of their own, up and down over 2^40, seen by single tokens, short runs and their heads."""
    heads, kv, d, n = 6, 2, 128, 400
    g = gen(53)
    k_rows, v_rows, table, status, k, v, pos, slot = make_cache(ops, g, [n, n], kv, d, 64)
    v *= torch.exp2(torch.randint(-20, 21, (2 * n, 1, 1), generator=g, device=DEV).float()).to(torch.bfloat16)
    ops.int4.append(k, v, k_rows, v_rows, table, pos, slot, status)
    q = randn(g, 7, heads, d).to(torch.bfloat16)
    spans = [(0, 0, 1, n - 1), (1, 1, 6, n - 6)]
    at = torch.tensor([n - 1], dtype=torch.int32, device=DEV)
    got = ops.int4.attention_decode(q[:1], k_rows, v_rows, table, at, slot[:1], d ** -0.5, 0, status)
    check_attention(got, *plain.attention(q[:1], k_rows, v_rows, table, spans[:1], d ** -0.5, 0))
    runs, blocks = runs_and_blocks(spans, 0)
    got = ops.int4.attention_prompt(q, k_rows, v_rows, table, runs, blocks, d ** -0.5, 0, status)
    check_attention(got, *plain.attention(q, k_rows, v_rows, table, spans, d ** -0.5, 0))
    assert int(status) == 0


# ------------------------------------------------------------------------------------------------ prompts, held tightly
def wide_attention(q, k_rows, v_rows, table, spans, scale, window):
    """What the gathered path computes: softmax over keys and values rounded to bfloat16, and how far it may be off.

    The bound, per number: 2^-8 of it (its own rounding); 2^-8 of sum p |v| / sum p (probabilities rounded to bfloat16); float32 sums
    over n keys, 2^-24 of sum p |v| / sum p for each of n / 16 products in turn and 64 at the ends; scores: d / 16 + 8 roundings of
    2^-24 of sum |q| |k| and 2^-22 of exp2, which the result sees twice."""
    n, n_q, d = q.shape
    out = torch.zeros(n, n_q * d, dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(out)
    for slot, row, count, past in spans:
        k, v = (plain.values(*plain.sequence(rows, table[slot], past + count), 64).to(torch.bfloat16).double() for rows in (k_rows, v_rows))
        i, j = torch.arange(past, past + count, device=q.device)[:, None], torch.arange(past + count, device=q.device)[None]
        hidden = (j > i) | ((j <= i - window) if window else torch.zeros_like(j > i))
        for h in range(n_q):
            e = h // (n_q // k.shape[0])
            x = q[row:row + count, h].double()
            p = torch.softmax((x @ k[e].t() * scale).masked_fill(hidden, -float("inf")), dim=1)
            cols = slice(h * d, (h + 1) * d)
            o, size = p @ v[e], p @ v[e].abs()
            off = ((d / 16 + 8) * 2 ** -24 * 1.4427 * scale * (x.abs() @ k[e].abs().t()).masked_fill(hidden, 0.0)).amax(1, keepdim=True) + 2 ** -22
            out[row:row + count, cols] = o
            bound[row:row + count, cols] = 2 ** -8 * o.abs() + (2 ** -8 + ((past + count) / 16 + 64) * 2 ** -24 + 2 * off) * size
    return out, bound


TIGHT = [
    # heads, kv heads, d, page, (cached, new), window
    (4, 2, 128, 64, [(0, 1)], 0),
    (4, 1, 64, 16, [(0, 5), (30, 1), (100, 3)], 0),
    (8, 2, 128, 64, [(500, 4), (64, 4), (0, 2)], 0),
    (5, 1, 128, 32, [(700, 5), (0, 17)], 40),
    (6, 2, 64, 7, [(90, 9), (333, 3), (5, 20)], 0),
    (16, 1, 128, 128, [(250, 5), (129, 2)], 100),
    (24, 2, 64, 64, [(1000, 3), (33, 8), (64, 1)], 64),
    (3, 1, 64, 1, [(70, 31)], 1),
    (32, 8, 128, 64, [(0, 300), (200, 130)], 0),
    (6, 3, 64, 64, [(0, 129), (1000, 64), (60, 70)], 0),
    (4, 2, 128, 16, [(300, 200), (0, 40)], 100),
    (16, 1, 64, 7, [(90, 33), (0, 64)], 0),
    (8, 1, 128, 64, [(127, 200), (64, 64)], 65),
    (4, 1, 64, 32, [(0, 128), (511, 140)], 300),
]


@pytest.mark.parametrize("heads,kv,d,page,seqs,window", TIGHT)
def test_prompts_are_held_to_their_own_path(ops, heads, kv, d, page, seqs, window):
    """Runs that read codes are held to the codes' numbers, gathered ones to these rounded to bfloat16; an oracle with a key too many, a
    key too few, queries one position early or a scale of 0.95 is told apart by the same bounds."""
    g = gen(heads + 3 * d + page + len(seqs))
    k_rows, v_rows, table, status, *_ = make_cache(ops, g, [p + n for p, n in seqs], kv, d, page)
    spans, row = [], 0
    for s, (p, n) in enumerate(seqs):
        spans.append((s, row, n, p))
        row += n
    q = (1.5 * randn(g, row, heads, d)).to(torch.bfloat16)
    runs, blocks = runs_and_blocks(spans, window)
    got = ops.int4.attention_prompt(q, k_rows, v_rows, table, runs, blocks, d ** -0.5, window, status).double()
    few = -(-row * (heads // kv) // len(runs)) <= ops.int4.FEW_COLUMNS
    oracle = plain.attention if few else wide_attention
    worst = lambda **other: float(((got - (w := oracle(**{**dict(q=q, k_rows=k_rows, v_rows=v_rows, table=table, spans=spans, scale=d ** -0.5,
                                                                 window=window), **other}))[0]).abs() / (w[1] + 1e-30)).max())
    assert int(status) == 0 and worst() <= 1
    if max(p + n for p, n in seqs) > 1:
        assert worst(scale=0.95 * d ** -0.5) > 1 or window == 1
        early = [(s, r, n, p - 1) for s, r, n, p in spans if p]
        if early:
            only = torch.zeros_like(got, dtype=torch.bool)
            for s, r, n, p in early:
                only[r:r + n] = True
            o, b = oracle(q, k_rows, v_rows, table, early, d ** -0.5, window)
            assert float(((got - o).abs() / (b + 1e-30))[only].max()) > 1
    if window:
        assert worst(window=window + 1) > 1 and (window == 1 or worst(window=window - 1) > 1)


@pytest.mark.parametrize("window", [0, 90])
def test_long_runs_report_pages_that_are_missing(ops, window):
    """Gathered prompts say what those that read codes say: a page missing that some row sees is reported; in front of the window and
    behind the end there need be none, and a run that goes beyond the table is left out."""
    g = gen(61)
    heads, kv, d, page, n = 8, 1, 64, 16, 40
    k_rows, v_rows, table, status, *_ = make_cache(ops, g, [230, 60], kv, d, page)
    q = randn(g, 2 * n, heads, d).to(torch.bfloat16)
    spans = [(0, 0, n, 190), (1, n, n, 20)]
    runs, blocks = runs_and_blocks(spans, window)
    call = lambda t, r=runs: ops.int4.attention_prompt(q, k_rows, v_rows, t, r, blocks, d ** -0.5, window, status)
    want = call(table)
    assert 2 * n * heads // 2 > ops.int4.FEW_COLUMNS and int(status) == 0
    unseen = table.clone()
    if window:
        unseen[0, :(190 - window + 1) // page] = -1
        assert torch.equal(call(unseen), want) and int(status) == 0
    first = (190 - window + 1) // page if window else 0
    for slot, p in ((0, first), (0, 229 // page), (0, 160 // page), (1, 0), (1, 59 // page)):
        for value in (-1, 100000):
            missing = unseen.clone()
            missing[slot, p] = value
            got = call(missing)
            assert int(status) == 5, (slot, p)
            status.zero_()
            rows = slice(n, 2 * n) if slot == 0 else slice(0, n)
            assert torch.equal(got[rows], want[rows])
    # a table of 15 pages of 16: position 240 lies beyond it, though in its last block of 64
    beyond = runs.clone()
    at = int((runs[:, 0] == 0).nonzero()[0])
    beyond[at, 3] = 240 - n + 1
    narrow = table[:, :15].contiguous()
    got = call(narrow, beyond)
    assert int(status) == 4 and not bool(got[:n].any()) and torch.equal(got[n:], want[n:])


# ------------------------------------------------------------------------------------------------ gated units of long prompts
def unit_bound(x, w, want, gate, up):
    """A unit of long prompts: the weight's numbers rounded to bfloat16 (wide_bound), the unit in float32 (|silu'| <= 1.1, silu within 2^-19 of
    itself), its result rounded to bfloat16.  No rounding of gate and up in between."""
    off, inter = wide_bound(x, w), gate.shape[1]
    return 2 ** -8 * want.abs() + 1.1 * off[:, :inter] * (up.abs() + off[:, inter:]) + gate.abs() * off[:, inter:] + 2 ** -19 * (gate * up).abs() + 2 ** -30


def test_gate_and_up_of_a_long_prompt_are_not_rounded(ops):
    """Weights of whole numbers, exact in bfloat16, and inputs of whole numbers: every product is exact, and the unit's result the bfloat16
    next to its 64-bit value (or one step off where float32 lies on the other side of a half)."""
    g = gen(71)
    m, inter, k = 400, 96, 256
    codes = torch.randint(0, 16, (2 * inter, k), generator=g, device=DEV)
    step, low = torch.ones(2 * inter, 2, device=DEV), torch.full((2 * inter, 2), -7.0, device=DEV)
    w = ops.int4.Int4Weight(plain.pack_weight(codes, step, low), 2 * inter, k)
    x = torch.randint(-15, 16, (m, k), generator=g, device=DEV).to(torch.bfloat16)
    y = x.double() @ plain.values(*plain.unpack_weight(w), 128).t()
    gate, up = y.chunk(2, 1)
    assert float((gate.to(torch.bfloat16).double() != gate).double().mean()) > 0 and float(y.abs().max()) < 2 ** 24
    want = gate * torch.sigmoid(gate) * up
    got = ops.swiglu_product(x, w).double()
    assert float(((got - want).abs() / (2 ** -8 * want.abs() * (1 + 2 ** -10) + 2 ** -30)).max()) <= 1
    # rounding both factors first would be told apart
    gate, up = (t.to(torch.bfloat16).double() for t in (gate, up))
    other = (gate * torch.sigmoid(gate) * up).to(torch.bfloat16).double()      # as such a kernel would give it
    assert float(((other - want).abs() / (2 ** -8 * want.abs() + 2 ** -30)).max()) > 1


@pytest.mark.parametrize("first,more", [(1, 5), (8, 0), (3, 13), (0, 7)])
@pytest.mark.parametrize("m", [5, 40, 385, 600])
def test_units_into_columns_that_start_anywhere(ops, m, first, more):
    """`out` may be any columns of a wider matrix, whatever the rows: the numbers of a result of its own, and nothing beside them."""
    g = gen(m + first)
    inter, k = 208, 256
    w = ops.int4.quantize_weight(randn(g, 2 * inter, k) * 0.06)
    x = randn(g, m, k).to(torch.bfloat16)
    wide = torch.full((m, first + inter + more), 7.0, dtype=torch.bfloat16, device=DEV)
    got = ops.glu_product(x, w, ops.kernels.glu_shape("silu"), out=wide[:, first:first + inter])
    assert got.data_ptr() == wide[:, first:].data_ptr() and torch.equal(got, ops.swiglu_product(x, w))
    assert bool((wide[:, :first] == 7).all()) and bool((wide[:, first + inter:] == 7).all())
    y = x.double() @ plain.values(*plain.unpack_weight(w), 128).t()
    gate, up = y.chunk(2, 1)
    want = gate * torch.sigmoid(gate) * up
    assert float(((got.double() - want).abs() / unit_bound(x, w, want, gate, up)).max()) <= 1


@pytest.mark.parametrize("m,inter,k", [(400, 6000, 4096), (700, 2064, 16384)])
def test_wide_units_of_long_prompts_take_a_bounded_work_space(ops, m, inter, k, monkeypatch):
    """Several pieces of the weight, the last a short one: the bits of the weight as a whole, results against 64 bits, and what the call holds
    beside its result."""
    import sys
    limit = 32 << 20
    monkeypatch.setattr(sys.modules["garlic_inference_b200.ops.linear"], "INT4_GATED_BYTES", limit)
    g = gen(m)
    w = random_weight(ops, g, 2 * inter, k)
    x = (randn(g, m, k) * 0.2).to(torch.bfloat16)
    assert 4 * inter * k > 2 * limit
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    got = ops.swiglu_product(x, w)
    torch.cuda.synchronize()
    assert torch.cuda.max_memory_allocated() - before <= limit + 2 * m * inter + (1 << 20)
    monkeypatch.undo()
    assert torch.equal(got, ops.swiglu_product(x, w))
    y = x.double() @ plain.values(*plain.unpack_weight(w), 128).t()
    gate, up = y.chunk(2, 1)
    want = gate * torch.sigmoid(gate) * up
    assert float(((got.double() - want).abs() / unit_bound(x, w, want, gate, up)).max()) <= 1


# ------------------------------------------------------------------------------------------------ steps of unlike sequences
MIXED = [
    # heads, kv heads, d, page, (cached, new), window
    (8, 2, 128, 64, [(300, 1), (64, 150), (900, 1), (0, 1), (10, 3)], 0),
    (4, 1, 64, 16, [(0, 200), (333, 1), (64, 24), (100, 25)], 0),
    (4, 2, 128, 64, [(500, 1), (200, 130), (0, 300), (90, 2)], 100),
    (6, 6, 64, 7, [(70, 97), (70, 96), (5, 1)], 0),
]


@pytest.mark.parametrize("limit", [256 << 20, 1])
@pytest.mark.parametrize("heads,kv,d,page,seqs,window", MIXED)
def test_a_layer_over_short_and_long_sequences(ops, heads, kv, d, page, seqs, window, limit, monkeypatch):
    """What a layer makes of such a step: rows of short sequences as exact as codes allow, those of long ones as the gathered path; all long
    ones gathered together, and one by one."""
    from garlic_inference_b200.cache.paged import KVView
    from garlic_inference_b200.parts import StepContext
    from test_int4 import _layer
    monkeypatch.setattr(ops.int4, "GATHER_BYTES", limit)
    monkeypatch.setattr(ops.int4, "TOGETHER_BYTES", 0)
    g = gen(heads + d + page)
    k_rows, v_rows, table, status, *_ = make_cache(ops, g, [p + n for p, n in seqs], kv, d, page)
    part = _layer(heads // kv, d, kv, window or None)
    lens, past = [n for _, n in seqs], [p for p, _ in seqs]
    starts = [sum(lens[:i]) for i in range(len(lens))]
    n = sum(lens)
    at = torch.zeros(n, dtype=torch.int32, device=DEV)
    ctx = StepContext(n, at, at, at, list(range(len(seqs))), starts, lens, past, False, status=status)
    kv_view = KVView(k_rows, v_rows, table, page, window or None)
    q = (1.5 * randn(g, n, heads, d)).to(torch.bfloat16)
    got = part.attend(q, kv_view, ctx)
    spans = [(s, starts[s], lens[s], past[s]) for s in range(len(seqs))]
    short = [t for t in spans if t[2] * (heads // kv) <= ops.int4.FEW_COLUMNS]
    long = [t for t in spans if t not in short]
    assert short and long and int(status) == 0
    for part_of, oracle in ((short, plain.attention), (long, wide_attention)):
        want, bound = oracle(q, k_rows, v_rows, table, part_of, part.scale, window)
        for _, r, c, _ in part_of:
            check_attention(got[r:r + c], want[r:r + c], bound[r:r + c])
    ctx.arrays.clear()
    assert torch.equal(got, part.attend(q, kv_view, ctx))


def test_single_tokens_beside_a_prompt_gather_nothing_of_theirs(ops):
    """40 single tokens behind 1,000 and a prompt of 300: what the layer holds meanwhile is the prompt's pages, not the others'."""
    from garlic_inference_b200.cache.paged import KVView
    from garlic_inference_b200.parts import StepContext
    from test_int4 import _layer
    heads, kv, d = 8, 2, 128
    seqs = [(1000, 1)] * 20 + [(0, 300)] + [(1000, 1)] * 20
    k_rows, v_rows, table, status, *_ = make_cache(ops, gen(3), [p + n for p, n in seqs], kv, d, 64)
    part = _layer(heads // kv, d, kv)
    lens, past = [n for _, n in seqs], [p for p, _ in seqs]
    starts = [sum(lens[:i]) for i in range(len(lens))]
    n = sum(lens)
    at = torch.zeros(n, dtype=torch.int32, device=DEV)
    ctx = StepContext(n, at, at, at, list(range(len(seqs))), starts, lens, past, False, status=status)
    kv_view = KVView(k_rows, v_rows, table, 64, None)
    q = randn(gen(4), n, heads, d).to(torch.bfloat16)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    part.attend(q, kv_view, ctx)
    torch.cuda.synchronize()
    pages = 5 * 2 * 64 * kv * d * 2                          # the prompt's five blocks, keys and values
    slices = 40 * heads * 8 * (d + 2) * 4
    assert torch.cuda.max_memory_allocated() - before <= pages + slices + 4 * n * heads * d * 2 + (1 << 20)
    assert 40 * 16 * 2 * 64 * kv * d * 2 > pages + slices + 4 * n * heads * d * 2 + (1 << 20)


def test_some_rows_of_a_step(ops):
    """Rows in any order; what no row names stays; rows that do not exist are reported and put nowhere; refusals."""
    g = gen(83)
    heads, kv, d = 4, 2, 64
    k_rows, v_rows, table, status, *_ = make_cache(ops, g, [50, 70, 9], kv, d, 16)
    q = randn(g, 9, heads, d).to(torch.bfloat16)
    rows = torch.tensor([7, 2, 0, 1], dtype=torch.int32, device=DEV)      # sequence 1 at 69, sequence 0 at 47, sequence 2 at 7 and 8
    runs, blocks = runs_and_blocks([(1, 0, 1, 69), (0, 1, 1, 47), (2, 2, 2, 7)], 0)
    fixed = (k_rows, v_rows, table, runs, blocks, d ** -0.5, 0, status)
    out = torch.full((9, heads * d), 5.0, dtype=torch.bfloat16, device=DEV)
    assert ops.int4.attention_some(q, rows, *fixed, out) is out
    want = ops.int4.attention_prompt(q[rows.long()].contiguous(), *fixed)
    assert int(status) == 0 and torch.equal(out[rows.long()], want) and bool((out[[3, 4, 5, 6, 8]] == 5).all())
    for bad in (-1, 9, 2147483647):
        some = rows.clone()
        some[1] = bad
        out.fill_(5.0)
        ops.int4.attention_some(q, some, *fixed, out)
        assert int(status) == 4 and torch.equal(out[[7, 0, 1]], want[[0, 2, 3]]) and bool((out[[2, 3, 4, 5, 6, 8]] == 5).all())
        status.zero_()
    for call in (lambda: ops.int4.attention_some(q, rows.long(), *fixed, out), lambda: ops.int4.attention_some(q, rows[None], *fixed, out),
                 lambda: ops.int4.attention_some(q, rows, *fixed, out[:8]), lambda: ops.int4.attention_some(q, rows, *fixed, out.float()),
                 lambda: ops.int4.attention_some(q, rows.cpu(), *fixed, out), lambda: ops.int4.attention_some(q[:, ::2], rows, *fixed, out[:, :heads * d // 2]),
                 lambda: ops.int4.attention_prompt(q, *fixed, out[:8]), lambda: ops.int4.attention_prompt(q, *fixed, out.float()),
                 lambda: ops.int4.attention_prompt(q, *fixed, out[:, ::2])):
        with pytest.raises(ops.KernelError):
            call()
    none = torch.zeros(0, dtype=torch.int32, device=DEV)
    out.fill_(5.0)
    ops.int4.attention_some(q, none, k_rows, v_rows, table, runs[:0], blocks, d ** -0.5, 0, status, out)
    assert int(status) == 0 and bool((out == 5).all())


# ------------------------------------------------------------------------------------------------ the largest numbers
MOST = 2.0 ** 127 * (2 - 2.0 ** -7)                          # the largest bfloat16


def largest_groups(dtype):
    """Groups of 64 numbers up to the ends of bfloat16, and of float32: [groups, 64]."""
    g = gen(89)
    r = torch.rand(8, 64, generator=g, device=DEV, dtype=torch.float64)
    x = torch.stack([r[0] * MOST, -r[1] * MOST, (2 * r[2] - 1) * MOST, MOST * (0.99 + 0.01 * r[3]), torch.full_like(r[4], MOST),
                     torch.full_like(r[5], -MOST), r[6] * 0.9 * MOST, (2 * r[7] - 1) * MOST])
    x[0, 3], x[1, 5], x[2, 7], x[2, 8], x[3, 1] = MOST, -MOST, MOST, -MOST, MOST
    x = x.clamp(-MOST, MOST)
    if dtype == torch.float32:
        top = torch.finfo(torch.float32).max
        x[7, 0], x[7, 1], x[0, 9], x[4, :] = top, -top, top, top
    return x.to(dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_the_largest_numbers_come_back_finite(ops, dtype):
    """Within half a step (2^-18 of a step for the quotient) of themselves, or of the largest bfloat16; in bfloat16 with its rounding, 2^-8."""
    x = largest_groups(dtype)
    want = x.double().clamp(-MOST, MOST)
    w = ops.int4.quantize_weight(torch.cat([x, x], 1))       # groups of 128
    codes, step, low = plain.unpack_weight(w)
    rows = [ops.int4.Int4Rows.zeros(1, 8, 16, 64, DEV) for _ in range(2)]
    table = torch.zeros(1, 1, dtype=torch.int32, device=DEV)
    pos, slot, status = torch.zeros(1, dtype=torch.int32, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV)
    ops.int4.append(x[None], x[None], *rows, table, pos, slot, status)
    steps = rows[0].meta[0, :, 0, 0, 0].double()
    for t in (torch.float32, torch.bfloat16):
        back = ops.int4.dequantize_weight(w, t)[:, :64].double()
        read = ops.int4.read(rows[0], table, pos, slot, status, t)[0].double()
        for got, s in ((back, step[:, 0]), (read, steps)):
            assert bool(torch.isfinite(got).all())
            bound = s[:, None] * (0.5 + 2 ** -18) + (2 ** -8 if t == torch.bfloat16 else 2 ** -24) * want.abs()
            assert float(((got - want).abs() / bound).max()) <= 1
    y = torch.zeros(20, 128, dtype=torch.bfloat16, device=DEV)
    y[:, 5] = 2.0 ** -100
    for rows_of in (8, 20):                                  # a number that is finite stays one on its way to the tensor cores
        assert bool(torch.isfinite(ops.linear(y[:rows_of], w, torch.float32)).all())


# ------------------------------------------------------------------------------------------------ inputs of very unlike sizes
def lined_up(x, w):
    """What lining products up cuts off (int4.cuh): 17 times 2^-14 of the largest |x| of the 16 inputs that an instruction takes, times the step.
    Instruction (j, h) of a group takes inputs 32 t + 8 j + 2 h + {0, 1, 4, 5}, t = 0 .. 3."""
    of = torch.tensor([[32 * t + 8 * j + 2 * h + e for t in range(4) for e in (0, 1, 4, 5)] for j in range(4) for h in range(2)], device=DEV)
    groups = torch.nn.functional.pad(x.double().abs(), (0, -w.k % 128)).unflatten(1, (-1, 128))
    return 17 * 2 ** -14 * groups[:, :, of].amax(-1).sum(-1) @ plain.unpack_weight(w)[1].t()


@pytest.mark.parametrize("spread", [1.0, 2.0, 4.0])
@pytest.mark.parametrize("m,n,k", [(1, 777, 65), (8, 33, 128), (7, 32, 1024), (16, 64, 4096)])
def test_inputs_of_very_unlike_sizes(ops, m, n, k, spread):
    """Inputs that span up to 2^30, and some 300 times as large as their neighbours."""
    for seed in range(6):
        g = gen(seed + k)
        w = random_weight(ops, g, n, k)
        x = (randn(g, m, k) * torch.exp(spread * randn(g, k))).to(torch.bfloat16)
        if seed % 2:
            x[:, seed % k] *= 300
        want = x.double() @ plain.values(*plain.unpack_weight(w), 128).t()
        got = ops.linear(x, w, torch.float32).double()
        assert float(((got - want).abs() / (linear_bound(x, w) + lined_up(x, w) + 2 ** -24 * want.abs())).max()) <= 1


def attention_lined_up(q, k_rows, v_rows, table, spans, scale, window):
    """What lining products up (int4.cuh) can cut off of `plain.attention`'s results: 17 times 2^-14 of the largest |q| of every 16 numbers of a
    head, times a key's step, in its score, which a result sees twice; and of the largest p step of every 16 keys."""
    of = torch.tensor([[32 * h + 8 * t + 2 * i + e for t in range(4) for e in (0, 1, 4, 5)] for h in range(2) for i in range(2)], device=DEV)
    n, n_q, d = q.shape
    out = torch.zeros(n, n_q * d, dtype=torch.float64, device=DEV)
    for slot, row, count, past in spans:
        (kc, ks, kl), (vc, vs, vl) = (plain.sequence(r, table[slot], past + count) for r in (k_rows, v_rows))
        k, v = plain.values(kc, ks, kl, 64), plain.values(vc, vs, vl, 64)
        i, j = torch.arange(past, past + count, device=DEV)[:, None], torch.arange(past + count, device=DEV)[None]
        hidden = (j > i) | ((j <= i - window) if window else torch.zeros_like(j > i))
        for h in range(n_q):
            e, x = h // (n_q // k.shape[0]), q[row:row + count, h].double()
            p = torch.softmax((x @ k[e].t() * scale).masked_fill(hidden, -float("inf")), dim=1)
            most = x.abs().unflatten(1, (-1, 64))[:, :, of].amax(-1).sum(-1)
            off = (17 * 2 ** -14 * 1.4427 * scale * (most @ ks[e].t())).masked_fill(hidden, 0.0).amax(1, keepdim=True)
            steps = torch.nn.functional.pad(p[:, :, None] * vs[e][None], (0, 0, 0, -(past + count) % 16)).unflatten(1, (-1, 16)).amax(2).sum(1)
            out[row:row + count, h * d:(h + 1) * d] = 2 * off * (p @ v[e].abs()) + 17 * 2 ** -14 * steps.repeat_interleave(64, -1)
    return out


@pytest.mark.parametrize("down", [0, 14, 20])
@pytest.mark.parametrize("at", [0, 20, 150])
@pytest.mark.parametrize("heads,d,new", [(4, 128, 1), (2, 64, 1), (4, 64, 7), (16, 128, 1)])
def test_one_small_value_with_nearly_all_the_weight(ops, heads, d, new, at, down):
    """A key with nearly all the probability whose values are 2^-`down` of the others': these, far more of them and each of hardly any weight,
    are to be as exact as the sum of all asks, in front of that key and behind it, and for tokens that do not see the largest."""
    n = 200 + new
    g = gen(97 + at)
    k_rows, v_rows, table, status, k, v, pos, slot = make_cache(ops, g, [n], 1, d, 64)
    k *= 0.05
    k[at] = 20.0 / d ** 0.5                                  # its score lies about 20 above the others'
    v[at] *= 2.0 ** -down
    v[-1] *= 2.0 ** 12
    ops.int4.append(k, v, k_rows, v_rows, table, pos, slot, status)
    q = (1 + 0.1 * randn(g, new, heads, d)).to(torch.bfloat16)
    spans = [(0, 0, new, n - new)]
    args = (q, k_rows, v_rows, table, spans, d ** -0.5, 0)
    want, bound = plain.attention(*args)
    if new == 1:
        got = [ops.int4.attention_decode(q, k_rows, v_rows, table, pos[-1:], slot[:1], d ** -0.5, 0, status, n_splits=s) for s in (None, 1)]
    else:
        got = [ops.int4.attention_prompt(q, k_rows, v_rows, table, *runs_and_blocks(spans, 0), d ** -0.5, 0, status)]
    for t in got:
        check_attention(t, want, bound + attention_lined_up(*args))
