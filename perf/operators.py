"""The 4-bit operators that performance is followed on: products with weights in 4 bits, and a key/value cache in 4 bits
with the attention that reads it.

Four kinds of path:

  linear   y = x W^T, or silu(x Wg^T) * (x Wu^T), for a weight held in 4 bits with a step and a low value per output and
           128 inputs.
  append   new keys and values go into the cache's pages in 4 bits, with a step and a low value per 64 numbers, and what the
           pages then stand for is read back.
  decode   one new token per sequence attends to what the cache holds of its sequence.
  prompt   prompts, or portions of prompts behind cached tokens, attend to the cache, their own tokens included.

A number q of 0 .. 15 stands for step * q + low (both bfloat16).  Two numbers lie in a byte, the first in its low half.

A weight [out, in] lies in tiles of 16 outputs and 128 inputs, uint8 [ceil(out / 16), ceil(in / 128), 1088]: two pieces of
512 bytes (outputs 0-7 and 8-15 of the tile), in each 8 outputs x 4 parts of 32 inputs x 16 bytes, then for each of the 16
outputs its step and its low value.  What a tile holds beyond the weight's sizes is never used.

Pages of the cache are uint8 [pages, heads, page size, d / 2] and bfloat16 [pages, heads, page size, d / 64, 2] (step, low).
"""
import math
import random

import torch

own = False
DEV = "cuda"
GROUP_W, GROUP_KV, TILE = 128, 64, 1088


# ------------------------------------------------------------------------------------------------------------ cases
def _linear(name, rows, outs, ins, glu=False):
    c = dict(op="linear", rows=rows, outs=outs, ins=ins, glu=glu)
    return dict(c, name=name) if name else c


def _cache(name, op, heads, kv_heads, d, sequences, past, new=1, ragged=False, window=0, page=64, idle=0, lengths=1):
    c = dict(op=op, heads=heads, kv_heads=kv_heads, d=d, sequences=sequences, past=past, new=new, ragged=ragged, window=window,
             page=page, idle=idle, lengths=lengths)
    return dict(c, name=name) if name else c


def listed():
    return [
        # one user's token through the joined query, key and value projection of the benchmark's model: latency
        _linear("linear_one", 1, 6144, 4096),
        # the benchmark's batch of eight through its feed-forward's first half, the largest weight of a layer
        _linear("glu_eight", 8, 12288, 4096, glu=True),
        # a busy server's step through the second half of a wider model's feed-forward
        _linear("linear_21", 21, 5120, 17408),
        # sizes of nobody's layer: neither whole tiles of outputs nor whole groups of inputs
        _linear("linear_odd", 3, 777, 1347),
        # a whole prompt of the benchmark's length through the first half of the feed-forward: arithmetic
        _linear("glu_prompt", 2048, 12288, 4096, glu=True),
        # a decode step's eight tokens into the cache: the smallest call
        _cache("append_eight", "append", 32, 8, 128, 8, 2048),
        # portions of seven prompts into the cache, heads of 64
        _cache("append_ragged", "append", 16, 4, 64, 7, 2500, new=700, ragged=True),
        # the benchmark's batch: eight conversations of 2,048 tokens
        _cache("decode_eight", "decode", 32, 8, 128, 8, 2048),
        # one long document: few rows over a long axis
        _cache("decode_long", "decode", 32, 8, 128, 1, 131000),
        # a busy server: conversations of all lengths and two slots idle, five query heads to a key/value head
        _cache("decode_ragged_48", "decode", 40, 8, 128, 48, 8000, ragged=True, idle=2),
        # the last tokens of prompts that were brought in portions, and drafts that wait for their check: a few tokens each
        _cache("prompt_few", "prompt", 32, 8, 128, 12, 6000, new=5, ragged=True),
        # what a server's scheduler puts together: portions of seven prompts behind cached tokens, heads of 64, a window
        _cache("prompt_ragged", "prompt", 16, 4, 64, 7, 2500, new=700, ragged=True, window=1500),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["linear", "linear", "append", "decode", "decode", "prompt"])
    if op == "linear":
        rows, outs, ins = _spread(rng, 1, 2048) if rng.random() < 0.4 else _spread(rng, 1, 64), _spread(rng, 16, 17408), _spread(rng, 64, 17408)
        if rng.random() < 0.6:                                # most layers' sizes are whole
            outs, ins = -(-outs // 64) * 64, -(-ins // 128) * 128
        glu = rng.random() < 0.4
        while outs * ins * (2 if glu else 1) > 90e6 or rows * outs * ins * (2 if glu else 1) > 100e9:
            outs, rows = max(16, outs // 32 * 16), max(1, rows - rows // 4)
        return _linear(None, rows, outs, ins, glu)
    kv = rng.choice([1, 2, 4, 8])
    group = rng.choice([1, 2, 3, 4, 5, 7, 8, 16])
    d, page = rng.choice([64, 128, 128]), rng.choice([16, 32, 64, 64, 64, 128])
    ragged, window = rng.random() < 0.7, _spread(rng, 32, 4096) if rng.random() < 0.25 else 0
    sequences, lengths = _spread(rng, 1, 64), rng.randrange(1, 1 << 20)
    if op == "decode":
        past = _spread(rng, 1, min(131000, 3000000 // (sequences * kv)))
        return _cache(None, op, kv * group, kv, d, sequences, past, 1, ragged, window, page, rng.choice([0, 0, 1]), lengths)
    sequences = min(sequences, 16)
    new = _spread(rng, 1, 4000 // sequences)
    past = _spread(rng, 1, 6000) if rng.random() < 0.6 else 0
    return _cache(None, op, kv * group, kv, d, sequences, past, new, ragged, window, page, 0, lengths)


def _lengths(case):
    """(cached tokens, new tokens) of every sequence; ragged ones spread from a few up to the case's numbers."""
    r = random.Random(case["lengths"] * 7919 + case["sequences"])
    past, new = [], []
    for _ in range(case["sequences"]):
        past.append(int(case["past"] * r.random() ** 1.5) if case["ragged"] else case["past"])
        new.append(1 + int((case["new"] - 1) * r.random()) if case["ragged"] else case["new"])
    return past, new


# --------------------------------------------------------------------------------------------------------- inputs
def _up_bf16(x):
    """The smallest bfloat16 that is not below the positive float32 x."""
    return ((x.view(torch.int32) + 0xFFFF) & -0x10000).view(torch.float32).to(torch.bfloat16)


def _quantise(rows):
    """bfloat16 [..., d] -> numbers 0 .. 15 (uint8 [..., d]), steps and low values [..., d / 64, 2]."""
    x = rows.float().unflatten(-1, (-1, GROUP_KV))
    low, high = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    step = _up_bf16((high * 0.5 - low * 0.5) / torch.full((), 7.5, device=x.device)).float()
    q = torch.round((x * 0.5 - low * 0.5) / (step * 0.5)).clamp(0, 15)
    q = torch.where(step > 0, q, torch.zeros_like(q)).to(torch.uint8).flatten(-2)
    return q, torch.cat([step, low], -1).to(torch.bfloat16)


def _pack(q):
    return q[..., 0::2] | (q[..., 1::2] << 4)


def _randn(gen, *shape):
    return torch.randn(*shape, generator=gen, device=DEV)


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    if case["op"] == "linear":
        rows, ins = case["rows"], case["ins"]
        n = case["outs"] * (2 if case["glu"] else 1)
        tn, tk = -(-n // 16), -(-ins // GROUP_W)
        tiles = torch.empty(tn, tk, TILE, dtype=torch.uint8, device=DEV)
        q = (_randn(gen, tn, tk, 2048).mul_(2.6).add_(7.5).round_().clamp_(0, 15)).to(torch.uint8)
        tiles[:, :, :1024] = _pack(q)
        del q
        step = (0.4 + 0.6 * torch.rand(tn, tk, 16, generator=gen, device=DEV)) * (1.4 / (2.6 * math.sqrt(ins)))
        low = -step * (7.0 + torch.rand(tn, tk, 16, generator=gen, device=DEV))
        meta = torch.stack([step, low], -1).to(torch.bfloat16)
        tiles[:, :, 1024:] = meta.view(torch.uint8).reshape(tn, tk, 64)
        scale = torch.exp(0.6 * _randn(gen, ins))
        scale[torch.randint(ins, (max(1, ins // 500),), generator=gen, device=DEV)] *= 12      # a few large channels
        return dict(op="linear", x=(_randn(gen, rows, ins) * scale).to(torch.bfloat16), tiles=tiles, n=n, ins=ins, glu=case["glu"])
    past, new = _lengths(case)
    S, page, kv, d = case["sequences"], case["page"], case["kv_heads"], case["d"]
    total = [p + n for p, n in zip(past, new)]
    need = [-(-t // page) for t in total]
    n_pages, width = sum(need) + 3, max(need) + 2
    order = torch.randperm(n_pages, generator=torch.Generator().manual_seed(seed)).tolist()
    slots = list(range(S + case["idle"]))
    random.Random(seed).shuffle(slots)                        # a sequence's slot is not its place in the step
    table = torch.full((len(slots), width), -1, dtype=torch.int32)
    at = 0
    for s in range(S):
        table[slots[s], :need[s]] = torch.tensor(order[at:at + need[s]], dtype=torch.int32)
        at += need[s]
    state = dict(op=case["op"], table=table.to(DEV), scale=d ** -0.5, window=case["window"], page=page, heads=case["heads"],
                 status=torch.zeros(1, dtype=torch.int32, device=DEV), longest=max(total), most_new=max(new))
    pools = []
    for values in (False, True):
        rows = _randn(gen, n_pages * page, kv, d)
        if not values:                                        # keys: some channels are large and off centre
            rows = rows * torch.exp(0.5 * _randn(gen, kv, d)) + 2 * _randn(gen, kv, d) * (torch.rand(kv, d, generator=gen, device=DEV) < 0.1)
        q, meta = _quantise(rows.to(torch.bfloat16))
        pools.append((_pack(q).view(n_pages, page, kv, d // 2).transpose(1, 2).contiguous(),
                      meta.view(n_pages, page, kv, d // 64, 2).transpose(1, 2).contiguous()))
        del rows, q, meta
    state["k"], state["v"] = pools
    idle = case["idle"] if case["op"] == "decode" else 0
    pos = torch.cat([torch.arange(p, p + n) for p, n in zip(past, new)] + [torch.zeros(idle, dtype=torch.long)])
    slot = torch.cat([torch.full((n,), slots[s]) for s, n in enumerate(new)] + [torch.full((idle,), -1)])
    state["pos"], state["slot"] = pos.to(torch.int32).to(DEV), slot.to(torch.int32).to(DEV)
    tokens = len(pos)
    if case["op"] == "append":                                # columns of the joined projection's rows
        joined = _randn(gen, tokens, (case["heads"] + 2 * kv) * d) * torch.exp(0.5 * _randn(gen, (case["heads"] + 2 * kv) * d))
        joined = joined.to(torch.bfloat16)
        state["new_k"] = joined[:, case["heads"] * d:(case["heads"] + kv) * d].unflatten(1, (kv, d))
        state["new_v"] = joined[:, (case["heads"] + kv) * d:].unflatten(1, (kv, d))
        return state
    state["q"] = (1.5 * _randn(gen, tokens, case["heads"], d)).to(torch.bfloat16)
    # the sequences of the step: slot, first row, new tokens, cached tokens
    starts = [sum(new[:s]) for s in range(S)]
    state["spans"] = torch.tensor([[slots[s], starts[s], new[s], past[s]] for s in range(S)], device=DEV)
    if case["op"] == "prompt":
        # runs of at most 128 tokens of a sequence: slot, first row, rows, first position; the longest walks first
        runs = [(slots[s], starts[s] + r, min(128, new[s] - r), past[s] + r) for s in range(S) for r in range(0, new[s], 128)]
        runs.sort(key=lambda t: -(t[3] + t[2]))
        state["runs"] = torch.tensor(runs, dtype=torch.int32, device=DEV)
        # blocks of 64 positions that some token of the step sees: slot, number of the block
        first = [max(0, past[s] - case["window"] + 1) // 64 if case["window"] else 0 for s in range(S)]
        blocks = [(slots[s], b) for s in range(S) for b in range(first[s], -(-total[s] // 64))]
        state["blocks"] = torch.tensor(blocks, dtype=torch.int32, device=DEV)
    return state


# ------------------------------------------------------------------------------------------------------ plain forms
def _weight(tiles, n, ins):
    """The numbers that the tiles stand for, float32 [n, ins]."""
    tn, tk, _ = tiles.shape
    codes, meta = tiles[:, :, :1024], tiles[:, :, 1024:].contiguous().view(torch.bfloat16).float().view(tn, tk, 16, 2)
    q = torch.stack([codes & 15, codes >> 4], -1).float().view(tn, tk, 16, GROUP_W)          # two pieces of 8 outputs, 4 x 32 inputs
    w = meta[..., :1] * q + meta[..., 1:]
    return w.transpose(1, 2).reshape(tn * 16, tk * GROUP_W)[:n, :ins]


def _rows_of(pool, pages, offsets):
    """float32 values of the cache's rows at (page, offset within it), [..., heads, d]; pages below 0 give zeros."""
    codes, meta = pool
    here = pages.clamp(min=0).long()
    c, m = codes[here, :, offsets], meta[here, :, offsets].float()
    q = torch.stack([c & 15, c >> 4], -1).float().flatten(-2).unflatten(-1, (-1, GROUP_KV))
    rows = (m[..., :1] * q + m[..., 1:]).flatten(-2)
    return rows * (pages >= 0)[..., None, None]


def _plain_append(s):
    page = torch.where(s["slot"] >= 0, s["table"][s["slot"].clamp(min=0).long(), (s["pos"] // s["page"]).long()], -1)
    offset = (s["pos"] % s["page"]).long()
    out = []
    for pool, new in ((s["k"], s["new_k"]), (s["v"], s["new_v"])):
        q, meta = _quantise(new)
        pool[0][page.long(), :, offset] = _pack(q)
        pool[1][page.long(), :, offset] = meta
        out.append(_rows_of(pool, page, offset).to(torch.bfloat16))
    return out


def _plain_attention(s):
    q, spans, L = s["q"].float(), s["spans"], s["longest"]
    n, heads, d = q.shape
    slot, start, new, past = spans.unbind(1)
    at = torch.arange(L, device=q.device)
    table = s["table"][slot]                                                                  # [S, width]
    pages = torch.where(at < (past + new)[:, None], table[:, at // s["page"]], -1)
    offsets = (at % s["page"]).expand_as(pages)
    k, v = _rows_of(s["k"], pages, offsets), _rows_of(s["v"], pages, offsets)                # [S, L, kv, d]
    kv = k.shape[2]
    t = torch.arange(s["most_new"], device=q.device)
    rows = (start[:, None] + torch.minimum(t, new[:, None] - 1))                              # [S, T], the last again behind the end
    here = past[:, None] + t
    qs = q[rows].unflatten(2, (kv, heads // kv)).permute(0, 2, 1, 3, 4).flatten(2, 3)         # [S, kv, T * group, d]
    scores = (qs @ k.permute(0, 2, 3, 1)) * s["scale"]
    seen = at <= here[..., None]
    if s["window"]:
        seen = seen & (at > here[..., None] - s["window"])
    scores = scores.unflatten(2, (len(t), heads // kv)).masked_fill(~seen[:, None, :, None], -math.inf)
    p = torch.exp(scores - scores.amax(-1, keepdim=True))
    p = (p / p.sum(-1, keepdim=True)).flatten(2, 3)
    o = (p @ v.transpose(1, 2)).unflatten(2, (len(t), heads // kv)).permute(0, 2, 1, 3, 4).flatten(2)      # [S, T, heads * d]
    out = torch.zeros(n, heads * d, dtype=torch.bfloat16, device=q.device)
    there = t < new[:, None]
    out[rows[there]] = o[there].to(torch.bfloat16)
    return out


def run(state):
    s = state
    if own:
        from garlic_inference_b200.ops import int4, linear, swiglu_product
        if s["op"] == "linear":
            w = int4.Int4Weight(s["tiles"], s["n"], s["ins"])
            return swiglu_product(s["x"], w) if s["glu"] else linear(s["x"], w)
        k, v = int4.Int4Rows(*s["k"]), int4.Int4Rows(*s["v"])
        if s["op"] == "append":
            int4.append(s["new_k"], s["new_v"], k, v, s["table"], s["pos"], s["slot"], s["status"])
            return [int4.read(r, s["table"], s["pos"], s["slot"], s["status"]) for r in (k, v)]
        if s["op"] == "decode":
            return int4.attention_decode(s["q"], k, v, s["table"], s["pos"], s["slot"], s["scale"], s["window"], s["status"])
        return int4.attention_prompt(s["q"], k, v, s["table"], s["runs"], s["blocks"], s["scale"], s["window"], s["status"])
    if s["op"] == "linear":
        y = s["x"].float() @ _weight(s["tiles"], s["n"], s["ins"]).t()
        if s["glu"]:
            gate, up = y.chunk(2, dim=1)
            y = gate / (1 + torch.exp(-gate)) * up
        return y.to(torch.bfloat16)
    return _plain_append(s) if s["op"] == "append" else _plain_attention(s)


# ------------------------------------------------------------------------------------------------- floors and checks
def work(case):
    if case["op"] == "linear":
        n = case["outs"] * (2 if case["glu"] else 1)
        return {"bytes": n * case["ins"] * 4.25 / 8 + 2 * case["rows"] * (case["ins"] + case["outs"]),
                "flops": 2 * case["rows"] * n * case["ins"]}
    past, new = _lengths(case)
    kv, d, heads, window = case["kv_heads"], case["d"], case["heads"], case["window"]
    row = kv * (d / 2 + d / 16)                               # bytes of a token's keys (or values) in the cache
    if case["op"] == "append":                                # read in 16 bits, written, read again and given back in 16 bits
        return {"bytes": 2 * sum(new) * (2 * row + 4 * kv * d), "flops": 2 * sum(new) * kv * d * 4}
    seen = 0
    for p, n in zip(past, new):
        for i in range(p, p + n):
            seen += min(i + 1, window) if window else i + 1
    keys = sum(min(p + n, window + n - 1) if window else p + n for p, n in zip(past, new))
    return {"bytes": 2 * keys * row + 4 * sum(new) * heads * d, "flops": 4 * seen * heads * d}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "linear":
        tn, tk, _ = s["tiles"].shape
        meta = s["tiles"][:, :, 1024:].contiguous().view(torch.bfloat16).double().reshape(tn, tk, 16, 2)
        x = torch.zeros(case["rows"], tk * GROUP_W, dtype=torch.float64, device=DEV)
        x[:, :case["ins"]] = s["x"].double()
        y = torch.zeros(case["rows"], tn * 16, dtype=torch.float64, device=DEV)
        for g in range(tk):                                   # a group of inputs at a time
            codes = s["tiles"][:, g, :1024].reshape(tn * 16, 64).long()
            q = torch.empty(tn * 16, GROUP_W, dtype=torch.float64, device=DEV)
            q[:, 0::2], q[:, 1::2] = (codes % 16).double(), (codes // 16).double()
            part = x[:, g * GROUP_W:(g + 1) * GROUP_W]
            step, low = meta[:, g, :, 0].reshape(-1), meta[:, g, :, 1].reshape(-1)
            y += (part @ q.t()) * step + part.sum(1, keepdim=True) * low
        y = y[:, :s["n"]]
        if case["glu"]:
            gate, up = y[:, :case["outs"]], y[:, case["outs"]:]
            y = gate * torch.sigmoid(gate) * up
        return y

    def values(pool, slot, count):
        pages = s["table"][slot, :-(-count // s["page"])].long()
        codes, meta = pool[0][pages], pool[1][pages].double()
        q = torch.empty(*codes.shape[:-1], codes.shape[-1] * 2, dtype=torch.float64, device=DEV)
        q[..., 0::2], q[..., 1::2] = (codes % 16).double(), (codes // 16).double()
        step, low = (meta[..., i].repeat_interleave(GROUP_KV, -1) for i in (0, 1))
        return (q * step + low).permute(1, 0, 2, 3).reshape(q.shape[1], -1, q.shape[-1])[:, :count]

    if case["op"] == "append":
        out = []
        for new in (s["new_k"], s["new_v"]):
            x = new.double().reshape(*new.shape[:-1], -1, GROUP_KV)
            low = x.min(-1, keepdim=True).values
            least = (x.max(-1, keepdim=True).values - low) / 15
            step = least.to(torch.bfloat16)                   # to the next bfloat16 where rounding went below
            step = torch.where(step.double() < least, (step.view(torch.int16) + 1).view(torch.bfloat16), step).double()
            q = torch.nan_to_num((x - low) / step).round().clamp(0, 15)
            out.append((low + q * step).reshape(new.shape))
        return out
    q = s["q"].double()
    n, heads, d = q.shape
    out = torch.zeros(n, heads * d, dtype=torch.float64, device=DEV)
    for slot, start, new, past in s["spans"].tolist():
        k, v = values(s["k"], slot, past + new), values(s["v"], slot, past + new)
        for h in range(heads):
            j = h // (heads // k.shape[0])
            a = q[start:start + new, h] @ k[j].t() * s["scale"]
            i, c = torch.arange(past, past + new, device=DEV)[:, None], torch.arange(past + new, device=DEV)[None]
            a[(c > i) | ((c <= i - case["window"]) if case["window"] else torch.zeros_like(c > i))] = -math.inf
            out[start:start + new, h * d:(h + 1) * d] = torch.softmax(a, dim=1) @ v[j]
    return out
