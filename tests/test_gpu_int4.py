"""Weights and cache rows in 4 bits on the GPU: every entry point against the formulas in 64 bits (plain_int4.py)."""
import random

import pytest
import torch

import plain_int4 as plain

pytestmark = pytest.mark.gpu
DEV = "cuda"
NAN, INF = float("nan"), float("inf")


@pytest.fixture(scope="module")
def ops():
    from garlic_inference_b200 import ops
    return ops


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def randn(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV)


# ------------------------------------------------------------------------------------------------------------ weights
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n,k", [(16, 128), (1, 1), (37, 300), (128, 4096), (5, 127)])
def test_weights_are_quantised_by_the_formula(ops, n, k, dtype):
    w = (randn(gen(n + k), n, k) * 0.02 + 0.003).to(dtype)
    w[0, :min(k, 128)] = 0.25                                # a group of equal numbers has step 0
    got = ops.int4.quantize_weight(w)
    codes, step, low = plain.unpack_weight(got)
    want = plain.quantise(w, 128)
    assert torch.equal(step, want[1]) and torch.equal(low, want[2])
    # float32 quotients may round to the other side of a half; half a step either way then
    differ = codes != want[0]
    assert int((codes - want[0]).abs().max()) <= 1
    if bool(differ.any()):
        x = ((w.double() - low.repeat_interleave(128, -1)[:, :k]) / step.repeat_interleave(128, -1)[:, :k])[differ]
        assert float((x - x.floor() - 0.5).abs().max()) < 2 ** -18
    back = plain.values(codes, step, low, 128)
    assert float((back - w.double()).abs().sub(step.repeat_interleave(128, -1)[:, :k] * (0.5 + 2 ** -18)).max()) <= 0
    for t in (torch.bfloat16, torch.float32):
        assert torch.equal(ops.int4.dequantize_weight(got, t), back.float().to(t))
    if n > 3:
        assert torch.equal(ops.int4.dequantize_weight(got, torch.float32, 2, n - 3), back.float()[2:n - 1])


def test_weights_whose_numbers_are_not_finite(ops):
    w = randn(gen(3), 20, 256).to(torch.bfloat16)
    w[2, 5], w[3, 200], w[4, 0] = NAN, INF, -INF
    w[5, :128] = 3.3e38
    w[5, :64] = -3.3e38
    codes, step, low = plain.unpack_weight(ops.int4.quantize_weight(w))
    bad = torch.zeros(20, 2, dtype=torch.bool, device=DEV)
    bad[2, 0] = bad[3, 1] = bad[4, 0] = True
    assert torch.equal(torch.isnan(step), bad) and torch.equal(torch.isnan(low), bad)
    assert codes[5, :128].unique().tolist() == [0, 15]


def linear_bound(x, w):
    """How far the kernel that reads codes may be off: the result's rounding is the caller's.  Float32 roundings of sums whose numbers
    add up to A = sum step code |x| + |low| |x|: 8 in a group, 2 a group, 8 blocks and 16 of the ends; and what f16 leaves of
    a scaled x, 2^-36 of the row's largest number."""
    codes, step, low = plain.unpack_weight(w)
    zero = torch.zeros_like(low)
    sq, lo = plain.values(codes, step, zero, 128), plain.values(torch.zeros_like(codes), zero, low.abs(), 128)
    a = x.double().abs() @ (sq + lo).t()
    return (32 + 2 * step.shape[1]) * 2 ** -24 * a + 2 ** -36 * x.double().abs().amax(1, keepdim=True) * sq.sum(1)[None]


def wide_bound(x, w):
    """What rounding each number of the weight to bfloat16 (2^-8 of it) and float32 sums of k products (2^-24 each) leave."""
    a = x.double().abs() @ plain.values(*plain.unpack_weight(w), 128).abs().t()
    return a * (2 ** -8 + (w.k + 16) * 2 ** -24)


def random_weight(ops, g, n, k):
    codes = torch.randint(0, 16, (n, k), generator=g, device=DEV)
    groups = -(-k // 128)
    step = (0.2 + torch.rand(n, groups, generator=g, device=DEV)) * 0.01
    low = -step * (6 + 3 * torch.rand(n, groups, generator=g, device=DEV))
    return ops.int4.Int4Weight(plain.pack_weight(codes, step, low), n, k)


SHAPES = [(1, 16, 128), (1, 6144, 4096), (2, 1, 1), (3, 777, 1347), (5, 48, 640), (8, 4096, 1024), (8, 33, 9000), (9, 256, 256), (13, 100, 4100),
          (16, 512, 12288), (17, 64, 384), (40, 130, 1000)]


@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_linear(ops, m, n, k, out_dtype):
    g = gen(m * 1000 + n + k)
    w = random_weight(ops, g, n, k)
    x = (randn(g, m, k) * torch.exp(randn(g, k))).to(torch.bfloat16)
    got = ops.linear(x, w, out_dtype)
    assert got.shape == (m, n) and got.dtype == out_dtype
    want = x.double() @ plain.values(*plain.unpack_weight(w), 128).t()
    bound = linear_bound(x, w) * 1.0 + (2 ** -8 if out_dtype == torch.bfloat16 else 2 ** -24) * want.abs()
    if m > 16:                                               # the weight's numbers may be rounded to bfloat16: see wide_bound
        bound += wide_bound(x, w)
    worst = ((got.double() - want).abs() / bound).max()
    assert float(worst) <= 1, float(worst)
    assert torch.equal(got, ops.linear(x, w, out_dtype))


@pytest.mark.parametrize("m,n,k", [(7, 1500, 1152), (16, 300, 700), (8, 20000, 640)])
@pytest.mark.parametrize("ranks", range(1, 9))
def test_linear_cut_in_any_way(ops, ranks, m, n, k):
    g = gen(ranks + n)
    w = random_weight(ops, g, n, k)                          # 9, 6 and 5 groups: uneven shares, and none for some
    x = randn(g, m, k).to(torch.bfloat16)
    want = x.double() @ plain.values(*plain.unpack_weight(w), 128).t()
    for parts in (1, 2, 4, 8, 16) if ranks <= -(-k // 128) else []:
        if parts > -(-(-(-k // 128)) // ranks):
            continue
        got = ops.int4.linear_rows(x, w, torch.float32, ranks=ranks, parts=parts)
        assert float(((got.double() - want).abs() / (linear_bound(x, w) + 2 ** -24 * want.abs())).max()) <= 1


@pytest.mark.parametrize("m", [1, 7, 16, 33])
@pytest.mark.parametrize("inter,k", [(16, 128), (768, 1024), (40, 200), (2000, 640)])
def test_gated_units(ops, m, inter, k):
    from garlic_inference_b200.ops import kernels
    g = gen(m + inter + k)
    w = random_weight(ops, g, 2 * inter, k)
    x = randn(g, m, k).to(torch.bfloat16)
    y = x.double() @ plain.values(*plain.unpack_weight(w), 128).t()
    off = linear_bound(x, w) + (wide_bound(x, w) if m > 16 else 0)
    gate, up = y[:, :inter], y[:, inter:]
    # |silu'| <= 1.1, |gelu'| <= 1.13
    for unit, act in ((kernels.glu_shape("silu"), lambda z: z * torch.sigmoid(z)),
                      (kernels.glu_shape("gelu_tanh", gate_max=1.0, up_limit=0.5, up_shift=1.0),
                       lambda z: torch.nn.functional.gelu(z, approximate="tanh"))):
        gg, uu = (gate, up) if unit[0] == 0 else (gate.clamp(max=1.0), up.clamp(-0.5, 0.5) + 1.0)
        want = act(gg) * uu
        got = ops.swiglu_product(x, w) if unit[0] == 0 else ops.glu_product(x, w, unit)
        # the function of a float32 is within 2^-20 of itself
        bound = 2 ** -8 * want.abs() + 1.13 * off[:, :inter] * uu.abs() + act(gg).abs() * off[:, inter:] + 2 ** -19 * (gg * uu).abs() + 2 ** -30
        assert got.dtype == torch.bfloat16 and got.shape == (m, inter)
        assert float(((got.double() - want).abs() / bound).max()) <= 1
    wide = torch.full((m, inter + 24), 7.0, dtype=torch.bfloat16, device=DEV)
    ops.glu_product(x, w, kernels.glu_shape("silu"), out=wide[:, 8:8 + inter])
    assert torch.equal(wide[:, 8:8 + inter], ops.swiglu_product(x, w))
    assert bool((wide[:, :8] == 7).all()) and bool((wide[:, 8 + inter:] == 7).all())


@pytest.mark.parametrize("m,n,k", [(70, 96, 256), (130, 700, 1024), (100, 40, 333), (257, 512, 640)])
def test_linear_of_many_rows_and_of_float32(ops, m, n, k):
    g = gen(m + n + k)
    w = random_weight(ops, g, n, k)
    x = randn(g, m, k)
    wide = plain.values(*plain.unpack_weight(w), 128)
    # float32: numbers of the weight rounded once, then a float32 product of k numbers
    want = x.double() @ wide.t()
    a = x.double().abs() @ wide.abs().t()
    assert float(((ops.linear(x, w).double() - want).abs() / (a * (k + 4) * 2 ** -24)).max()) <= 1
    # bfloat16: numbers of the weight rounded to bfloat16 where the weight is made wide
    xb = x.to(torch.bfloat16)
    want = xb.double() @ wide.t()
    a = xb.double().abs() @ wide.abs().t()
    bound = a * (2 ** -8 + (k + 4) * 2 ** -24) + linear_bound(xb, w) + 2 ** -8 * want.abs()
    assert float(((ops.linear(xb, w).double() - want).abs() / bound).max()) <= 1
    if n % 2 == 0:
        got = ops.swiglu_product(xb, w).double()
        gate, up = want.chunk(2, 1)
        off = bound
        silu = gate * torch.sigmoid(gate)
        # both factors rounded to bfloat16 first where the activation is the product's last step
        tol = 2 ** -8 * (silu * up).abs() + (1.1 * (off[:, :n // 2] + 2 ** -8 * gate.abs())) * (up.abs() + off[:, n // 2:]) \
            + (silu.abs() + 2 ** -8 * gate.abs()) * (off[:, n // 2:] + 2 ** -8 * up.abs()) + 2 ** -18 * (gate * up).abs() + 2 ** -30
        assert float(((got - silu * up).abs() / tol).max()) <= 1


@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("m,n,k", [(1, 1, 8), (17, 128, 128), (32, 129, 136), (33, 16, 2000), (64, 300, 1024), (65, 777, 904), (128, 1000, 640), (200, 48, 512),
                                   (385, 260, 256)])
def test_products_on_tensor_memory(ops, m, n, k, out_dtype):
    g = gen(m + n + k)
    w = random_weight(ops, g, n, k)
    x = (randn(g, m, k) * torch.exp(randn(g, k))).to(torch.bfloat16)
    want = x.double() @ plain.values(*plain.unpack_weight(w), 128).t()
    bound = wide_bound(x, w) + (2 ** -8 if out_dtype == torch.bfloat16 else 2 ** -24) * want.abs()
    for ranks in range(0, min(8, -(-k // 128)) + 1):
        out = torch.full((m, n + 5), 9.0, dtype=out_dtype, device=DEV)
        got = ops.int4.linear_wide(x, w, out_dtype, out=out[:, 2:2 + n], ranks=ranks)
        assert float(((got.double() - want).abs() / bound).max()) <= 1, ranks
        assert torch.equal(got, ops.int4.linear_wide(x, w, out_dtype, ranks=ranks))
        assert bool((out[:, :2] == 9).all()) and bool((out[:, 2 + n:] == 9).all())


@pytest.mark.parametrize("m,n,k", [(17, 40, 65), (111, 78, 65), (400, 32, 333), (30, 300, 1021)])
def test_rows_of_odd_lengths_and_starts(ops, m, n, k):
    g = gen(m + n + k)
    w = random_weight(ops, g, n, k)
    filled = plain.pack_weight(torch.nn.functional.pad(plain.unpack_weight(w)[0], (0, -k % 128), value=15.0), *plain.unpack_weight(w)[1:])
    w = ops.int4.Int4Weight(filled, n, k)                    # beyond k the codes are not zeros
    x = randn(g, m, k).to(torch.bfloat16)
    want = x.double() @ plain.values(*plain.unpack_weight(w), 128).t()
    bound = wide_bound(x, w) + 2 ** -24 * want.abs()
    got = ops.linear(x, w, torch.float32)
    assert float(((got.double() - want).abs() / bound).max()) <= 1
    flat = torch.zeros(m * 128 + 3, dtype=torch.bfloat16, device=DEV)
    odd = flat[3:].view(m, 128)                              # even rows that start on 6 bytes
    odd.copy_(randn(g, m, 128))
    v = random_weight(ops, g, n, 128)
    assert torch.equal(ops.linear(odd, v, torch.float32), ops.linear(odd.clone(), v, torch.float32))
    assert torch.equal(ops.linear(odd[:11], v, torch.float32), ops.linear(odd[:11].clone(), v, torch.float32))


@pytest.mark.parametrize("m,inter,k", [(20, 16, 128), (40, 48, 520), (100, 208, 1024), (150, 64, 384), (64, 1000, 256)])
def test_gated_units_on_tensor_memory(ops, m, inter, k):
    from garlic_inference_b200.ops import kernels
    g = gen(m + inter + k)
    w = random_weight(ops, g, 2 * inter, k)
    x = randn(g, m, k).to(torch.bfloat16)
    y = x.double() @ plain.values(*plain.unpack_weight(w), 128).t()
    off = wide_bound(x, w)
    gate, up = y[:, :inter], y[:, inter:]
    for unit, act in ((kernels.glu_shape("silu"), lambda z: z * torch.sigmoid(z)),
                      (kernels.glu_shape("gelu_tanh", gate_max=1.0, up_limit=0.5, up_shift=1.0),
                       lambda z: torch.nn.functional.gelu(z, approximate="tanh"))):
        gg, uu = (gate, up) if unit[0] == 0 else (gate.clamp(max=1.0), up.clamp(-0.5, 0.5) + 1.0)
        want = act(gg) * uu
        bound = 2 ** -24 * want.abs() + 1.13 * off[:, :inter] * (uu.abs() + off[:, inter:]) + act(gg).abs() * off[:, inter:] + 2 ** -19 * (gg * uu).abs() + 2 ** -30
        if inter % 16:                                       # halves that end inside a tile: `linear`'s business
            with pytest.raises(ops.KernelError):
                ops.int4.linear_wide(x, w, torch.float32, unit)
            continue
        for ranks in range(0, min(4, -(-k // 128)) + 1):
            got = ops.int4.linear_wide(x, w, torch.float32, unit, ranks=ranks)
            assert float(((got.double() - want).abs() / bound).max()) <= 1


def test_rows_that_are_not_finite_stay_alone_on_tensor_memory(ops):
    g = gen(19)
    w = random_weight(ops, g, 150, 704)
    x = randn(g, 40, 704).to(torch.bfloat16)
    clean = ops.int4.linear_wide(x, w, torch.float32)
    x[3, 5], x[20, 700], x[39, 0] = NAN, INF, -INF
    got = ops.int4.linear_wide(x, w, torch.float32)
    rest = [i for i in range(40) if i not in (3, 20, 39)]
    assert torch.equal(got[rest], clean[rest]) and bool(torch.isnan(got[3]).all()) and not bool(torch.isfinite(got[[20, 39]]).any())
    w.tiles[2, 1, 1024 + 4 * 5:1024 + 4 * 5 + 4] = torch.tensor([0xC0, 0x7F, 0xC0, 0x7F], dtype=torch.uint8, device=DEV)      # output 37, NaN group
    got = ops.int4.linear_wide(clean.new_zeros(40, 704).to(torch.bfloat16) + 1, w, torch.float32)
    assert bool(torch.isnan(got[:, 37]).all()) and int(torch.isnan(got).sum()) == 40


def test_weights_with_more_inputs_than_16_rows_have_room_for(ops):
    g = gen(23)
    for k, m in ((120000, 16), (120001, 16), (120000, 20)):
        w = random_weight(ops, g, 32, k)
        x = randn(g, m, k).to(torch.bfloat16)
        want = x.double() @ plain.values(*plain.unpack_weight(w), 128).t()
        bound = wide_bound(x, w) + 2 ** -24 * want.abs()
        assert float(((ops.linear(x, w, torch.float32).double() - want).abs() / bound).max()) <= 1
        assert ops.swiglu_product(x, w).shape == (m, 16)


def test_rows_of_x_that_are_not_finite_or_huge_or_tiny(ops):
    g = gen(11)
    w = random_weight(ops, g, 70, 700)
    x = randn(g, 8, 700).to(torch.bfloat16)
    x[1, 3], x[2, 300], x[3, 10], x[3, 11] = NAN, INF, INF, -INF
    x[4] *= 1e36
    x[5] *= 1e-37
    x[6] = 0
    x[7, 5] = 1e4                                            # one large number among ordinary ones
    wide = plain.values(*plain.unpack_weight(w), 128)
    want = x.double() @ wide.t()
    got = ops.linear(x, w, torch.float32).double()
    assert bool(torch.isnan(got[1]).all()) and bool(torch.isnan(got[3]).sum() == torch.isnan(want[3]).sum())
    assert torch.equal(torch.isinf(got[2]), torch.isinf(want[2])) and torch.equal(got[2] > 0, want[2] > 0)
    for r in (0, 4, 5, 6, 7):
        bound = linear_bound(x[r:r + 1], w)[0] * 1.0 + (700 * 2 ** -24) * (x[r].double().abs() @ wide.abs().t()) + 2 ** -140
        assert float(((got[r] - want[r]).abs() / bound).max()) <= 1, r
    clean = x.clone()
    clean[1:4] = 1.0
    assert torch.equal(ops.linear(clean, w, torch.float32)[[0, 5, 6, 7]].double(), got[[0, 5, 6, 7]])      # neighbours see nothing of it


# -------------------------------------------------------------------------------------------------------------- cache
def make_cache(ops, g, sequences, heads, d, page, spare=2, scale=1.0):
    """Pages of sequences of the given lengths, in random order, filled by `append`; (k_rows, v_rows, table, status, k, v)."""
    need = [-(-n // page) for n in sequences]
    n_pages, width = sum(need) + spare, max(need) + 1
    order = torch.randperm(n_pages, generator=torch.Generator().manual_seed(7)).tolist()
    table = torch.full((len(sequences), width), -1, dtype=torch.int32)
    at = 0
    for s, c in enumerate(need):
        table[s, :c] = torch.tensor(order[at:at + c], dtype=torch.int32)
        at += c
    table = table.to(DEV)
    rows = [ops.int4.Int4Rows.zeros(n_pages, heads, page, d, DEV) for _ in range(2)]
    for r in rows:                                           # what pages held before is garbage, NaN among it
        r.codes.fill_(0xA5)
        r.meta.fill_(NAN)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    pos = torch.cat([torch.arange(n) for n in sequences]).to(torch.int32).to(DEV)
    slot = torch.cat([torch.full((n,), s) for s, n in enumerate(sequences)]).to(torch.int32).to(DEV)
    k = (randn(g, len(pos), heads, d) * scale + 0.5 * randn(g, heads, d)).to(torch.bfloat16)
    v = (randn(g, len(pos), heads, d) + 0.3).to(torch.bfloat16)
    ops.int4.append(k, v, *rows, table, pos, slot, status)
    assert int(status) == 0
    return rows[0], rows[1], table, status, k, v, pos, slot


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads,d,page", [(1, 64, 16), (3, 128, 64), (8, 128, 32), (2, 256, 7), (5, 64, 1)])
def test_append_and_read(ops, heads, d, page, dtype):
    g = gen(heads * d + page)
    tokens, slots = 45, 3
    rows = [ops.int4.Int4Rows.zeros(60, heads, page, d, DEV) for _ in range(2)]
    before = [(r.codes.clone(), r.meta.clone()) for r in rows]
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    width = -(-20 // page)
    table = torch.randperm(60, generator=torch.Generator().manual_seed(1))[:slots * width].reshape(slots, width).to(torch.int32).to(DEV)
    pos = torch.tensor([i % 15 for i in range(tokens)], dtype=torch.int32, device=DEV)
    slot = torch.tensor([i // 15 for i in range(tokens)], dtype=torch.int32, device=DEV)
    slot[4] = -1
    wide = (randn(g, tokens, 2 * heads + 1, d + 3) * torch.exp(randn(g, d + 3))).to(dtype)        # strides of their own, odd starts
    k, v = wide[:, :heads, 3:], wide[:, heads + 1:, :d]
    k[7, 0, :64] = 0.5
    ops.int4.append(k, v, *rows, table, pos, slot, status)
    for r, x, b in zip(rows, (k, v), before):
        codes, step, low = plain.quantise(x, 64)
        want = plain.values(codes, step, low, 64)
        want[4] = 0
        got = ops.int4.read(r, table, pos, slot, status, torch.float32)
        flip = (got.double() != want.float().double())
        if bool(flip.any()):                                 # a quotient next to a half, in float32
            st = step.repeat_interleave(64, -1)
            u = ((x.double() - low.repeat_interleave(64, -1)) / st)[flip]
            assert float((u - u.floor() - 0.5).abs().max()) < 2 ** -18
        assert torch.equal(ops.int4.read(r, table, pos, slot, status), got.to(torch.bfloat16))
        # nothing but the tokens' rows was written
        touched = torch.zeros(60, page, dtype=torch.bool, device=DEV)
        live = slot >= 0
        touched[table[slot[live].long(), (pos[live] // page).long()].long(), (pos[live] % page).long()] = True
        assert torch.equal(r.codes.transpose(1, 2)[~touched], b[0].transpose(1, 2)[~touched])
        assert torch.equal(r.meta.transpose(1, 2)[~touched], b[1].transpose(1, 2)[~touched])
    assert int(status) == 0


def test_rows_whose_numbers_are_not_finite_or_far_apart(ops):
    k = randn(gen(5), 6, 1, 128).to(torch.bfloat16)
    k[0, 0, 3], k[1, 0, 100], k[2, 0, 0] = NAN, INF, -INF
    k[3, 0, :64], k[3, 0, :32] = 3.3e38, -3.3e38
    k[4, 0, :64] = 1e-40
    k[4, 0, 0] = 0
    rows = [ops.int4.Int4Rows.zeros(1, 1, 8, 128, DEV) for _ in range(2)]
    table = torch.zeros(1, 1, dtype=torch.int32, device=DEV)
    pos, slot = torch.arange(6, dtype=torch.int32, device=DEV), torch.zeros(6, dtype=torch.int32, device=DEV)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    ops.int4.append(k, k, *rows, table, pos, slot, status)
    got = ops.int4.read(rows[0], table, pos, slot, status, torch.float32)[:, 0]
    nan = torch.isnan(got.unflatten(1, (2, 64)))
    assert bool(nan[0, 0].all()) and bool(nan[1, 1].all()) and bool(nan[2, 0].all())
    assert int(nan.sum()) == 3 * 64
    # the step is rounded up by at most 2^-7 of itself, and the largest number is 15 steps, twice its own size, above the lowest
    assert float((got[3, :64].double() / k[3, 0, :64].double() - 1).abs().max()) <= 2 * 2 ** -7
    assert float((got[4, :64].double() - k[4, 0, :64].double()).abs().max()) <= 1e-40 / 15


def test_places_outside_the_cache_are_reported_and_not_written(ops):
    rows = [ops.int4.Int4Rows.zeros(2, 1, 4, 64, DEV) for _ in range(2)]
    table = torch.tensor([[0, 1, -1], [5, -1, -1]], dtype=torch.int32, device=DEV)
    x = randn(gen(1), 1, 1, 64).to(torch.bfloat16)
    q = randn(gen(2), 1, 2, 64).to(torch.bfloat16)
    for pos, slot, codes in ((12, 0, (1, 1, 4)), (-1, 0, (1, 1, 4)), (8, 0, (2, 2, 5)), (0, 1, (2, 2, 5)), (0, 2, (1, 1, 4))):
        p, s = (torch.tensor([t], dtype=torch.int32, device=DEV) for t in (pos, slot))
        status = torch.zeros(1, dtype=torch.int32, device=DEV)
        ops.int4.append(x, x, *rows, table, p, s, status)
        assert int(status) == codes[0]
        assert not bool(rows[0].codes.any()) and not bool(rows[1].meta.any())
        status.zero_()
        assert not bool(ops.int4.read(rows[0], table, p, s, status).any()) and int(status) == codes[1]
        status.zero_()
        assert not bool(ops.int4.attention_decode(q, *rows, table, p, s, 0.125, 0, status).any()) and int(status) == codes[2]


def check_attention(got, want, bound):
    bad = torch.isnan(want)
    assert torch.equal(torch.isnan(got), bad)
    worst = ((got.double() - want).abs() / (bound + 1e-30))[~bad].max()
    assert float(worst) <= 1, float(worst)


DECODE = [
    # heads, kv heads, d, page, lengths, window
    (1, 1, 64, 16, [1], 0),
    (4, 1, 128, 64, [1, 2, 31, 32, 33, 64, 65, 127, 128, 129], 0),
    (32, 8, 128, 64, [2048, 5, 700], 0),
    (16, 2, 64, 32, [300, 1000, 17], 0),
    (15, 3, 128, 7, [100, 250, 6], 0),
    (24, 2, 64, 128, [129, 511], 0),
    (48, 2, 128, 64, [400, 90], 0),
    (8, 4, 128, 64, [1000, 40, 200], 64),
    (8, 1, 64, 16, [1000, 40, 333], 37),
    (3, 1, 128, 64, [500], 1),
]


@pytest.mark.parametrize("splits", [None, 1, 3])
@pytest.mark.parametrize("heads,kv,d,page,lengths,window", DECODE)
def test_decode(ops, heads, kv, d, page, lengths, window, splits):
    g = gen(heads + d + page + len(lengths))
    k_rows, v_rows, table, status, *_ = make_cache(ops, g, lengths, kv, d, page)
    order = list(range(len(lengths)))
    random.Random(3).shuffle(order)
    slots = order[:1] + [-1] + order[1:]                     # an idle row between
    q = (1.5 * randn(g, len(slots), heads, d)).to(torch.bfloat16)
    pos = torch.tensor([lengths[s] - 1 if s >= 0 else 0 for s in slots], dtype=torch.int32, device=DEV)
    slot = torch.tensor(slots, dtype=torch.int32, device=DEV)
    got = ops.int4.attention_decode(q, k_rows, v_rows, table, pos, slot, d ** -0.5, window, status, n_splits=splits)
    spans = [(s, i, 1, lengths[s] - 1) for i, s in enumerate(slots) if s >= 0]
    check_attention(got, *plain.attention(q, k_rows, v_rows, table, spans, d ** -0.5, window))
    assert int(status) == 0 and not bool(got[1].any())
    assert torch.equal(got, ops.int4.attention_decode(q, k_rows, v_rows, table, pos, slot, d ** -0.5, window, status, n_splits=splits))


@pytest.mark.parametrize("splits", [2, 5, 8, 9, 12, 74, 256])
@pytest.mark.parametrize("heads,kv,d,n,least,most", [(4, 1, 128, 5, 1, 700), (16, 8, 64, 60, 1, 400), (6, 6, 128, 3, 800, 1000)])
def test_slices_join_in_either_way(ops, heads, kv, d, n, least, most, splits):
    """Few blocks join in clusters, many (60 sequences of 8 heads) and more than 8 slices by a second kernel; most slices are empty."""
    rnd = random.Random(n)
    lengths = [rnd.randint(least, most) for _ in range(n)]
    g = gen(n + splits)
    k_rows, v_rows, table, status, *_ = make_cache(ops, g, lengths, kv, d, 64)
    q = randn(g, n, heads, d).to(torch.bfloat16)
    pos, slot = torch.tensor(lengths, dtype=torch.int32, device=DEV) - 1, torch.arange(n, dtype=torch.int32, device=DEV)
    slot[n // 2] = -1
    got = ops.int4.attention_decode(q, k_rows, v_rows, table, pos, slot, d ** -0.5, 0, status, n_splits=splits)
    spans = [(i, i, 1, lengths[i] - 1) for i in range(n) if i != n // 2]
    check_attention(got, *plain.attention(q, k_rows, v_rows, table, spans, d ** -0.5, 0))
    assert int(status) == 0 and not bool(got[n // 2].any())


def runs_and_blocks(spans, window):
    runs = sorted(((s, r + a, min(128, n - a), p + a) for s, r, n, p in spans for a in range(0, n, 128)), key=lambda t: -(t[2] + t[3]))
    blocks = [(s, b) for s, r, n, p in spans for b in range((max(0, p - window + 1) if window else 0) // 64, -(-(p + n) // 64))]
    return torch.tensor(runs, dtype=torch.int32, device=DEV), torch.tensor(blocks, dtype=torch.int32, device=DEV)


PROMPT = [
    # heads, kv heads, d, page, (cached, new), window
    (4, 2, 128, 64, [(0, 1)], 0),
    (4, 1, 64, 16, [(0, 5), (30, 1), (100, 3)], 0),
    (8, 2, 128, 64, [(500, 4), (64, 4), (0, 2)], 0),
    (5, 1, 128, 32, [(700, 5), (0, 17)], 40),
    (32, 8, 128, 64, [(0, 300), (200, 130)], 0),
    (6, 3, 64, 64, [(0, 129), (1000, 64), (60, 70)], 0),
    (4, 2, 128, 16, [(300, 200), (0, 40)], 100),
    (16, 1, 64, 7, [(90, 33), (0, 64)], 0),
]


@pytest.mark.parametrize("heads,kv,d,page,seqs,window", PROMPT)
def test_prompt(ops, heads, kv, d, page, seqs, window):
    g = gen(heads + d + page + len(seqs))
    k_rows, v_rows, table, status, *_ = make_cache(ops, g, [p + n for p, n in seqs], kv, d, page)
    spans, row = [], 0
    for s, (p, n) in enumerate(seqs):
        spans.append((s, row, n, p))
        row += n
    q = (1.5 * randn(g, row + 2, heads, d)).to(torch.bfloat16)        # two rows in no run
    runs, blocks = runs_and_blocks(spans, window)
    got = ops.int4.attention_prompt(q, k_rows, v_rows, table, runs, blocks, d ** -0.5, window, status)
    want, bound = plain.attention(q, k_rows, v_rows, table, spans, d ** -0.5, window)
    # where keys and values are made wide, each of their numbers is rounded to bfloat16, and so are the probabilities
    wide_bound = bound.clone()
    for s, r, n, p in spans:
        kc, ks, kl = plain.sequence(k_rows, table[s], p + n)
        vc, vs, vl = plain.sequence(v_rows, table[s], p + n)
        k, v = plain.values(kc, ks, kl, 64), plain.values(vc, vs, vl, 64)
        for h in range(heads):
            e = h // (heads // kv)
            off = 2 ** -8 * (q[r:r + n, h].double().abs() @ k[e].abs().t()).amax(1, keepdim=True) * d ** -0.5
            wide_bound[r:r + n, h * d:(h + 1) * d] += (2 * off + 2 ** -7) * v[e].abs().amax(0)[None]
    check_attention(got, want, wide_bound)
    assert int(status) == 0 and not bool(got[row:].any())


def test_values_that_are_not_finite_reach_only_the_tokens_that_see_them(ops):
    g = gen(9)
    heads, kv, d, n = 4, 2, 128, 100
    k_rows, v_rows, table, status, k, v, pos, slot = make_cache(ops, g, [n, n], kv, d, 64)
    v[50, 0, 70] = NAN                                       # sequence 0, position 50, the second group of key/value head 0
    ops.int4.append(k, v, k_rows, v_rows, table, pos, slot, status)
    q = randn(g, 4, heads, d).to(torch.bfloat16)
    at = torch.tensor([49, 50, 99, 99], dtype=torch.int32, device=DEV)
    of = torch.tensor([0, 0, 0, 1], dtype=torch.int32, device=DEV)
    for splits in (1, 2):
        got = ops.int4.attention_decode(q, k_rows, v_rows, table, at, of, 0.1, 0, status, n_splits=splits)
        bad = torch.isnan(got).reshape(4, heads, 2, 64)
        want = torch.zeros_like(bad)
        want[1:3, :2, 1] = True
        assert torch.equal(bad, want)
        q2 = q.clone()
        q2[2, 3, 5] = INF
        bad = torch.isnan(ops.int4.attention_decode(q2, k_rows, v_rows, table, at, of, 0.1, 0, status, n_splits=splits)).reshape(4, heads, d)
        assert bool(bad[2, 3].all()) and not bool(bad[3].any()) and not bool(bad[2, 2].any())
    k[30, 1, 0] = INF                                        # a key of key/value head 1: every later query of its heads
    ops.int4.append(k, v, k_rows, v_rows, table, pos, slot, status)
    bad = torch.isnan(ops.int4.attention_decode(q, k_rows, v_rows, table, at, of, 0.1, 0, status)).reshape(4, heads, d)
    assert bool(bad[:3, 2:].all()) and not bool(bad[3].any()) and not bool(bad[0, :2].any())


# -------------------------------------------------------------------------------------------- a layer's step, as it is used
def rotary(count, half, g):
    angle = torch.arange(count, device=DEV)[:, None] * torch.exp(-3 * torch.rand(half, generator=g, device=DEV))[None]
    return torch.cos(angle), torch.sin(angle)


@pytest.mark.parametrize("heads,kv,d,rot,norm,page", [(4, 2, 128, 128, torch.bfloat16, 64), (3, 1, 64, 64, None, 16), (6, 2, 64, 32, torch.float32, 7),
                                                      (5, 5, 128, 0, torch.bfloat16, 64), (2, 1, 128, 34, None, 32), (32, 8, 128, 128, torch.float32, 64)])
def test_projections_are_normed_rotated_and_appended(ops, heads, kv, d, rot, norm, page):
    """Bounds: q is rounded to bfloat16 (2^-8); float32 before that: the sum of d squares, its root, two products and a sum, 32
    roundings of 2^-24 of |a cos| + |b sin| at most.  k stays within half a step of its group (2^-18 of a step for the quotient)."""
    g = gen(heads * d + rot)
    lengths = [40, 3, 90]
    rows = [ops.int4.Int4Rows.zeros(60, kv, page, d, DEV) for _ in range(2)]
    width = -(-128 // page)
    table = torch.randperm(60, generator=torch.Generator().manual_seed(2))[:3 * width].reshape(3, width).to(torch.int32).to(DEV)
    pos = torch.tensor([0, 39, 17, 2, 89, 64, 5], dtype=torch.int32, device=DEV)
    slot = torch.tensor([0, 0, -1, 1, 2, 2, 2], dtype=torch.int32, device=DEV)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    qkv = (randn(g, 7, (heads + 2 * kv) * d) * torch.exp(randn(g, (heads + 2 * kv) * d))).to(torch.bfloat16)
    wq, wk = (None, None) if norm is None else ((1 + 0.3 * randn(g, d)).to(norm) for _ in range(2))
    cos, sin = rotary(100, rot // 2, g)
    args = (qkv, heads, kv, d, wq, wk, 1e-6, cos, sin, rot, pos, slot, *rows, table, status)
    before = [r.codes.clone() for r in rows]
    assert torch.equal(ops.int4.qk_norm_rope_append(*args, append=False), ops.int4.qk_norm_rope_append(*args))
    got = ops.int4.qk_norm_rope_append(*args)
    assert int(status) == 0 and not torch.equal(before[0], rows[0].codes)

    def made(x, w):
        x = x.double().unflatten(1, (-1, d))
        if w is not None:
            x = x * torch.rsqrt(x.square().mean(2, keepdim=True) + 1e-6) * w.double()
        y, size, h = x.clone(), x.abs(), rot // 2
        if rot:
            c, s = (t.double()[pos.long()][:, None] for t in (cos, sin))
            a, b = x[..., :h], x[..., h:rot]
            y[..., :h], y[..., h:rot] = a * c - b * s, b * c + a * s
            size = size.clone()
            size[..., :h], size[..., h:rot] = (a * c).abs() + (b * s).abs(), (b * c).abs() + (a * s).abs()
        return y, size * 32 * 2 ** -24

    want, off = made(qkv[:, :heads * d], wq)
    assert bool(((got.double() - want).abs() <= want.abs() * 2 ** -8 + off + 1e-38).all())
    live = slot >= 0
    k = ops.int4.read(rows[0], table, pos, slot, status, torch.float32)
    want, off = made(qkv[:, heads * d:(heads + kv) * d], wk)
    at = (table[slot[live].long(), (pos[live] // page).long()].long(), slice(None), (pos[live] % page).long())
    step = rows[0].meta[at][..., 0].double().repeat_interleave(64, -1)
    assert bool(((k.double() - want).abs()[live] <= step * (0.5 + 2 ** -18) + off[live] + want.abs()[live] * 2 ** -23).all())
    assert not bool(k[~live].any())
    # values, and keys without norm and rotation, as `append` writes them
    other = [ops.int4.Int4Rows.zeros(60, kv, page, d, DEV) for _ in range(2)]
    plain_k, plain_v = (qkv[:, a * d:(a + kv) * d].unflatten(1, (kv, d)) for a in (heads, heads + kv))
    ops.int4.append(plain_k, plain_v, *other, table, pos, slot, status)
    for i in range(1 if norm is not None or rot else 0, 2):
        assert torch.equal(rows[i].codes, other[i].codes) and torch.equal(rows[i].meta, other[i].meta)


def test_a_step_on_another_stream_and_from_two_graphs(ops):
    """Projection, append, attention and output projection: on a stream of their own, and recorded twice and replayed in
    turn, give the bits of the eager run on the default stream."""
    g = gen(11)
    heads, kv, d, hidden, lengths = 8, 2, 128, 256, [900, 30, 257]
    k_rows, v_rows, table, status, *_ = make_cache(ops, g, [n + 1 for n in lengths], kv, d, 64)
    w_qkv = ops.int4.quantize_weight(0.05 * randn(g, (heads + 2 * kv) * d, hidden))
    w_o = ops.int4.quantize_weight(0.05 * randn(g, hidden, heads * d))
    pos, slot = torch.tensor(lengths, dtype=torch.int32, device=DEV), torch.arange(3, dtype=torch.int32, device=DEV)
    cos, sin = rotary(1000, d // 2, g)
    xs = [randn(g, 3, hidden).to(torch.bfloat16) for _ in range(2)]

    def step(x):
        qkv = ops.linear(x, w_qkv)
        q = ops.int4.qk_norm_rope_append(qkv, heads, kv, d, None, None, 1e-6, cos, sin, d, pos, slot, k_rows, v_rows, table, status)
        return ops.linear(ops.int4.attention_decode(q, k_rows, v_rows, table, pos, slot, d ** -0.5, 0, status, n_splits=3), w_o)

    want = [step(x) for x in xs]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = [step(x) for x in xs]
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graphs, outs = [], []
    for x in xs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step(x))
        graphs.append(graph)
    for _ in range(3):
        for graph, out, w in zip(graphs, outs, want):
            out.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, w)
    assert int(status) == 0


def test_prompts_of_few_and_of_many_tokens_agree_where_they_meet(ops):
    """The two ways through the cache give the same result within what each may be off."""
    g = gen(13)
    heads, kv, d = 8, 2, 128
    seqs = [(200, 12), (64, 12), (0, 12)]
    k_rows, v_rows, table, status, *_ = make_cache(ops, g, [p + n for p, n in seqs], kv, d, 64)
    spans = [(s, 12 * s, 12, p) for s, (p, n) in enumerate(seqs)]
    q = randn(g, 36, heads, d).to(torch.bfloat16)
    runs, blocks = runs_and_blocks(spans, 0)
    few = ops.int4.attention_prompt(q, k_rows, v_rows, table, runs, blocks, d ** -0.5, 0, status)
    check_attention(few, *plain.attention(q, k_rows, v_rows, table, spans, d ** -0.5, 0))
    empty = torch.cat([runs[:1].clone(), runs])              # a run without rows, and one of a slot that is idle
    empty[0, 2] = 0
    idle = torch.cat([runs, runs[:1]])
    idle[0, 0] = -1
    assert torch.equal(ops.int4.attention_prompt(q, k_rows, v_rows, table, empty, blocks, d ** -0.5, 0, status), few)
    part = ops.int4.attention_prompt(q, k_rows, v_rows, table, idle[:-1], blocks, d ** -0.5, 0, status)
    rows = slice(int(idle[0, 1]), int(idle[0, 1]) + 12)
    assert int(status) == 0 and not bool(part[rows].any())
    for bad in ([0, -1, 4, 0], [0, 30, 12, 0], [0, 0, 12, 1000], [9, 0, 12, 0]):
        status.zero_()
        bad = torch.tensor([bad], dtype=torch.int32, device=DEV)
        assert not bool(ops.int4.attention_prompt(q[:12], k_rows, v_rows, table, bad, blocks, d ** -0.5, 0, status).any()) and int(status) == 4


def test_long_runs_that_do_not_exist_are_left_out(ops):
    """Runs of more columns than are read as single tokens: a slot, rows or positions that do not exist are reported, the others stay right."""
    g = gen(29)
    heads, kv, d, n = 8, 1, 64, 40
    k_rows, v_rows, table, status, *_ = make_cache(ops, g, [100, 60], kv, d, 16)
    q = randn(g, 2 * n, heads, d).to(torch.bfloat16)
    runs, blocks = runs_and_blocks([(0, 0, n, 60), (1, n, n, 20)], 0)
    assert 2 * n * heads > ops.int4.FEW_COLUMNS * 2
    want = ops.int4.attention_prompt(q, k_rows, v_rows, table, runs, blocks, 0.125, 0, status)
    assert int(status) == 0 and torch.equal(runs[0].cpu(), torch.tensor([0, 0, n, 60], dtype=torch.int32))
    for bad, code in (([-1, 0, n, 60], 0), ([0, 0, 0, 60], 0), ([2, 0, n, 60], 4), ([0, -1, n, 60], 4), ([0, n + 1, n, 60], 4), ([0, 0, n, -1], 4),
                      ([0, 0, n, 100000], 4), ([0, 0, 129, 0], 4), ([0, 0, n, 2147483647], 4)):
        status.zero_()
        some = runs.clone()
        some[0] = torch.tensor(bad, dtype=torch.int32)
        got = ops.int4.attention_prompt(q, k_rows, v_rows, table, some, blocks, 0.125, 0, status)
        assert int(status) == code and torch.equal(got[n:], want[n:]) and not bool(got[:n].any()), bad
    with pytest.raises(ops.KernelError):
        ops.int4.attention_prompt(q, k_rows, v_rows, table, runs, blocks[:0], 0.125, 0, status)


def test_pages_given_back_behind_the_window_are_not_missed(ops):
    g = gen(17)
    heads, kv, d, n, window = 4, 1, 64, 300, 50
    k_rows, v_rows, table, status, *_ = make_cache(ops, g, [n], kv, d, 16)
    q = randn(g, 3, heads, d).to(torch.bfloat16)
    pos, slot = torch.tensor([n - 1], dtype=torch.int32, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV)
    runs, blocks = runs_and_blocks([(0, 0, 3, n - 3)], window)
    want = ops.int4.attention_decode(q[:1], k_rows, v_rows, table, pos, slot, 0.125, window, status)
    want_runs = ops.int4.attention_prompt(q, k_rows, v_rows, table, runs, blocks, 0.125, window, status)
    table[0, :(n - 3 - window + 1) // 16] = -1
    assert torch.equal(ops.int4.attention_decode(q[:1], k_rows, v_rows, table, pos, slot, 0.125, window, status), want)
    assert torch.equal(ops.int4.attention_prompt(q, k_rows, v_rows, table, runs, blocks, 0.125, window, status), want_runs)
    assert int(status) == 0
    table[0, (n - 10) // 16] = -1                            # one that the window holds is
    ops.int4.attention_decode(q[:1], k_rows, v_rows, table, pos, slot, 0.125, window, status)
    assert int(status) == 5


def test_pages_and_tiles_beyond_32_bits(ops):
    """Codes that lie further than 2^32 bytes into their tensors."""
    g = gen(31)
    heads, kv, d, page = 4, 8, 128, 64
    n_pages = (1 << 32) // (kv * page * d // 2) + 40
    k_rows, v_rows = (ops.int4.Int4Rows.zeros(n_pages, kv, page, d, DEV) for _ in range(2))
    table = torch.tensor([[n_pages - 1, n_pages - 7, 3, n_pages - 30]], dtype=torch.int32, device=DEV)
    near = torch.tensor([[3, 2, 0, 1]], dtype=torch.int32, device=DEV)
    small = [ops.int4.Int4Rows.zeros(4, kv, page, d, DEV) for _ in range(2)]
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    pos, slot = torch.arange(240, dtype=torch.int32, device=DEV), torch.zeros(240, dtype=torch.int32, device=DEV)
    k, v = (randn(g, 240, kv, d).to(torch.bfloat16) for _ in range(2))
    q = randn(g, 240, 2 * kv, d).to(torch.bfloat16)
    runs, blocks = runs_and_blocks([(0, 0, 240, 0)], 0)
    out = []
    for rows, t in (((k_rows, v_rows), table), (small, near)):
        ops.int4.append(k, v, *rows, t, pos, slot, status)
        out.append([ops.int4.read(rows[0], t, pos, slot, status), ops.int4.attention_decode(q[:1], *rows, t, pos[239:], slot, 0.09, 0, status),
                    ops.int4.attention_prompt(q, *rows, t, runs, blocks, 0.09, 0, status),
                    ops.int4.attention_prompt(q[:3], *rows, t, torch.tensor([[0, 0, 3, 237]], dtype=torch.int32, device=DEV), blocks, 0.09, 0, status)])
    assert int(status) == 0 and all(torch.equal(a, b) for a, b in zip(*out)) and bool(out[0][0].any())
    del k_rows, v_rows, out
    n, ins = 140000, 65536                                   # 8,750 x 512 tiles, 4.9 GB
    tiles = torch.randint(0, 256, (n // 16, ins // 128, 1088), dtype=torch.uint8, device=DEV, generator=g)
    tiles[..., 1024:] = torch.tensor([0.01, -0.08], dtype=torch.bfloat16, device=DEV).view(torch.uint8).repeat(16)
    w, last = ops.int4.Int4Weight(tiles, n, ins), ops.int4.Int4Weight(tiles[-2:].clone(), 32, ins)
    for m in (2, 20):
        x = randn(g, m, ins).to(torch.bfloat16)
        want = x.double() @ plain.values(*plain.unpack_weight(last), 128).t()
        got = ops.linear(x, w, torch.float32)[:, -32:].double()
        assert float(((got - want).abs() / (wide_bound(x, last) + 2 ** -24 * want.abs())).max()) <= 1
    assert torch.equal(ops.int4.dequantize_weight(w, torch.float32, n - 32, 32), ops.int4.dequantize_weight(last, torch.float32))


def test_refusals(ops):
    KernelError = ops.KernelError
    i4 = ops.int4
    rows = [i4.Int4Rows.zeros(4, 2, 16, 64, DEV) for _ in range(2)]
    table = torch.zeros(2, 2, dtype=torch.int32, device=DEV)
    pos = slot = torch.zeros(3, dtype=torch.int32, device=DEV)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    x = torch.zeros(3, 2, 64, dtype=torch.bfloat16, device=DEV)
    q = torch.zeros(3, 4, 64, dtype=torch.bfloat16, device=DEV)
    w = i4.quantize_weight(torch.zeros(32, 128, device=DEV))
    y = torch.zeros(3, 128, dtype=torch.bfloat16, device=DEV)
    runs = torch.zeros(1, 4, dtype=torch.int32, device=DEV)
    blocks = torch.zeros(1, 2, dtype=torch.int32, device=DEV)
    other = i4.Int4Rows.zeros(4, 2, 16, 128, DEV)
    on_cpu = i4.Int4Rows.zeros(4, 2, 16, 64, "cpu")
    calls = [
        lambda: i4.quantize_weight(torch.zeros(4, 4)), lambda: i4.quantize_weight(torch.zeros(4, 4, device=DEV).t()[:, ::2]),
        lambda: i4.quantize_weight(torch.zeros(0, 4, device=DEV)), lambda: i4.quantize_weight(torch.zeros(4, 4, device=DEV, dtype=torch.float16)),
        lambda: i4.quantize_weight(torch.zeros(4, device=DEV)),
        lambda: i4.dequantize_weight(w, first=1, rows=32), lambda: i4.dequantize_weight(w, first=-1, rows=2), lambda: i4.dequantize_weight(w, torch.float16),
        lambda: i4.dequantize_weight(w, out=torch.zeros(31, 128, device=DEV, dtype=torch.bfloat16)),
        lambda: ops.linear(y[:, :64], w), lambda: ops.linear(y[0], w), lambda: ops.linear(y.to(torch.float16), w), lambda: ops.linear(y.cpu(), w),
        lambda: i4.linear_rows(y[:0], w), lambda: i4.linear_rows(torch.zeros(17, 128, dtype=torch.bfloat16, device=DEV), w), lambda: i4.linear_rows(y, w, torch.float16),
        lambda: i4.linear_rows(y, w, out=torch.zeros(3, 31, device=DEV, dtype=torch.bfloat16)),
        lambda: i4.linear_rows(y, w, out=torch.zeros(32, 3, device=DEV, dtype=torch.bfloat16).t()),
        lambda: i4.linear_wide(y[:0], w), lambda: i4.linear_wide(y[:, :120].contiguous(), i4.quantize_weight(torch.zeros(8, 121, device=DEV))),
        lambda: i4.linear_wide(torch.zeros(3, 136, dtype=torch.bfloat16, device=DEV), i4.quantize_weight(torch.zeros(8, 121, device=DEV))),
        lambda: i4.linear_wide(torch.zeros(3, 121, dtype=torch.bfloat16, device=DEV), i4.quantize_weight(torch.zeros(8, 121, device=DEV))),
        lambda: i4.linear_wide(y.flatten()[4:].as_strided((2, 128), (128, 1)), w), lambda: i4.linear_wide(y, w, ranks=2), lambda: i4.linear_wide(y, w, ranks=9),
        lambda: ops.swiglu_product(y, i4.quantize_weight(torch.zeros(33, 128, device=DEV))),
        lambda: i4.append(x, x[:, :1], *rows, table, pos, slot, status), lambda: i4.append(x, x.float(), *rows, table, pos, slot, status),
        lambda: i4.append(x.transpose(1, 2).contiguous().transpose(1, 2), x, *rows, table, pos, slot, status),
        lambda: i4.append(x, x, rows[0], other, table, pos, slot, status), lambda: i4.append(x, x, on_cpu, on_cpu, table, pos, slot, status),
        lambda: i4.append(x, x, rows[0].codes, rows[1], table, pos, slot, status), lambda: i4.append(x, x, *rows, table[0], pos, slot, status),
        lambda: i4.append(x, x, *rows, table, pos[:2], slot, status), lambda: i4.append(x, x, *rows, table, pos.long(), slot, status),
        lambda: i4.append(x, x, *rows, table, pos, slot.cpu(), status), lambda: i4.append(x, x, *rows, table.t(), pos, slot, status[:0]),
        lambda: i4.append(x.to(torch.float16), x.to(torch.float16), *rows, table, pos, slot, status),
        lambda: i4.read(rows[0], table, pos, slot, status, torch.float16), lambda: i4.read(rows[0], table.float(), pos, slot, status),
        lambda: i4.attention_decode(q.float(), *rows, table, pos, slot, 1.0, 0, status), lambda: i4.attention_decode(q[:, :3], *rows, table, pos, slot, 1.0, 0, status),
        lambda: i4.attention_decode(q[:, :, :32], *rows, table, pos, slot, 1.0, 0, status), lambda: i4.attention_decode(q[:, ::2], *rows, table, pos, slot, 1.0, 0, status),
        lambda: i4.attention_decode(q, *rows, table, pos, slot, 1.0, -1, status), lambda: i4.attention_decode(q, *rows, table, pos, slot, 1.0, 0, status, n_splits=257),
        lambda: i4.attention_decode(q, rows[0], other, table, pos, slot, 1.0, 0, status),
        lambda: i4.attention_prompt(q, *rows, table, runs[0], blocks, 1.0, 0, status), lambda: i4.attention_prompt(q, *rows, table, runs.long(), blocks, 1.0, 0, status),
        lambda: i4.attention_prompt(q, *rows, table, runs, blocks.cpu(), 1.0, 0, status),
    ]
    cos = torch.zeros(4, 32, device=DEV)
    qkv = torch.zeros(3, 8 * 64, dtype=torch.bfloat16, device=DEV)
    rope = lambda a=qkv, n_q=4, c=cos, s=cos, r=64, wq=None, wk=None: i4.qk_norm_rope_append(a, n_q, 2, 64, wq, wk, 1e-6, c, s, r, pos, slot, *rows, table, status)
    calls += [lambda: rope(a=qkv.float()), lambda: rope(a=qkv[:, :-64]), lambda: rope(n_q=5), lambda: rope(r=32), lambda: rope(s=cos[:2]),
              lambda: rope(wq=cos[0]), lambda: rope(wq=cos[0], wk=cos[0]), lambda: rope(c=cos.cpu(), s=cos.cpu())]
    for i, call in enumerate(calls):
        with pytest.raises(KernelError):
            call()
            raise AssertionError(f"call {i} was taken")
    assert rope().shape == (3, 4, 64)
    torch.cuda.synchronize()
    assert ops.linear(y[:0], w).shape == (0, 32)
    assert i4.attention_decode(q[:0], *rows, table, pos, slot, 1.0, 0, status).shape == (0, 256)
    i4.append(x[:0], x[:0], *rows, table, pos[:0], slot[:0], status)
    assert i4.read(rows[0], table, pos[:0], slot[:0], status).shape == (0, 2, 64)
