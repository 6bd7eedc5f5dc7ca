"""4-bit weights and cache rows restated plainly, for the tests: numbers in 64 bits, one formula a function."""
import torch


def bf16_up(x):
    """The smallest bfloat16 not below x (float64, not negative)."""
    b = x.to(torch.bfloat16)
    return torch.where(b.double() < x, (b.view(torch.int16) + 1).view(torch.bfloat16), b).double()


def bf16_down(x):
    """The largest bfloat16 not above x (float32)."""
    u = x.float().view(torch.int32)
    return (torch.where(u < 0, u + 0xFFFF, u) & -0x10000).view(torch.float32).double()


def quantise(x, group):
    """x [..., n] in groups of `group` (the last may be short): codes [..., n], steps and low values [..., ceil(n / group)]."""
    n = x.shape[-1]
    pad = -n % group
    g = torch.cat([x, x[..., -1:].expand(*x.shape[:-1], pad)], -1).unflatten(-1, (-1, group))
    finite = torch.isfinite(g).all(-1, keepdim=True)
    g = torch.where(finite, g, torch.zeros_like(g))
    low = bf16_down(g.amin(-1, keepdim=True))
    step = bf16_up((g.amax(-1, keepdim=True).double() - low) / 15)
    codes = torch.where(step > 0, torch.round((g.double() - low) / step).clamp(0, 15), torch.zeros_like(step))
    nan = torch.full_like(step, float("nan"))
    step, low = torch.where(finite, step, nan), torch.where(finite, low, nan)
    return codes.flatten(-2)[..., :n], step[..., 0], low[..., 0]


def values(codes, step, low, group):
    """The numbers that codes [..., n] stand for."""
    n = codes.shape[-1]
    return codes.double() * step.repeat_interleave(group, -1)[..., :n] + low.repeat_interleave(group, -1)[..., :n]


def unpack_weight(w):
    """(codes [n, k], steps, low values [n, ceil(k / 128)]) of an `Int4Weight`, in 64 bits."""
    tn, tk, _ = w.tiles.shape
    t = w.tiles.reshape(tn, tk, 1088)
    body = t[..., :1024].reshape(tn, tk, 16, 64)
    codes = torch.stack([body & 15, body >> 4], -1).reshape(tn, tk, 16, 128)
    codes = codes.transpose(1, 2).reshape(tn * 16, tk * 128)[:w.n, :w.k]
    meta = t[..., 1024:].contiguous().view(torch.bfloat16).reshape(tn, tk, 16, 2).transpose(1, 2).reshape(tn * 16, tk, 2)[:w.n]
    return codes.double(), meta[..., 0].double(), meta[..., 1].double()


def pack_weight(codes, step, low):
    """Tiles of codes [n, k] (whole numbers), steps and low values [n, ceil(k / 128)]."""
    n, k = codes.shape
    tn, tk = -(-n // 16), -(-k // 128)
    c = torch.zeros(tn * 16, tk * 128, dtype=torch.uint8, device=codes.device)
    c[:n, :k] = codes.to(torch.uint8)
    c = c.reshape(tn, 16, tk, 64, 2).transpose(1, 2)
    meta = torch.zeros(tn * 16, tk, 2, dtype=torch.bfloat16, device=codes.device)
    meta[:n, :, 0], meta[:n, :, 1] = step.to(torch.bfloat16), low.to(torch.bfloat16)
    tiles = torch.empty(tn, tk, 1088, dtype=torch.uint8, device=codes.device)
    tiles[..., :1024] = (c[..., 0] | (c[..., 1] << 4)).reshape(tn, tk, 1024)
    tiles[..., 1024:] = meta.reshape(tn, 16, tk, 2).transpose(1, 2).contiguous().view(torch.uint8).reshape(tn, tk, 64)
    return tiles


def unpack_rows(rows):
    """(codes [pages, heads, page size, d], steps, low values [pages, heads, page size, d / 64]) of an `Int4Rows`, in 64 bits."""
    c = rows.codes
    return torch.stack([c & 15, c >> 4], -1).flatten(-2).double(), rows.meta[..., 0].double(), rows.meta[..., 1].double()


def sequence(rows, table_row, count):
    """codes, steps and low values of a sequence's first `count` positions: [heads, count, d] and [heads, count, d / 64]."""
    page = rows.codes.shape[2]
    pages = table_row[:-(-count // page)].long()
    return [t[pages].transpose(0, 1).flatten(1, 2)[:, :count] for t in unpack_rows(rows)]


def attention(q, k_rows, v_rows, table, spans, scale, window):
    """softmax(q k scale) v for spans {slot, first row, rows, first position}, and how far a kernel may be off.

    Returns (result [n, n_q * d], the bound).  The bound counts, per number of the result:
      2^-8 of it for its own rounding to bfloat16;
      2^-11 of sum p step code / sum p: p step is rounded to f16;
      float32 sums over the keys, 16 at a time, of numbers that add up to sum p (step code + |low|) / sum p: 2^-23 of that for
      every 16 keys and 64 more for the ends;
      and scores: 24 roundings of float32 (2^-24) in sums whose numbers add up to A = sum step code |q| + |low| |q|, what an f16
      leaves of q (2^-36 of the largest |q| times sum step code), exp2 within 2^-22 of itself, all of which a
      probability sees once, and the result twice (in its sum and in what it is divided by)."""
    n, n_q, d = q.shape
    out = torch.zeros(n, n_q * d, dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(out)
    for slot, row, count, past in spans:
        if slot < 0:
            continue
        kc, ks, kl = sequence(k_rows, table[slot], past + count)
        vc, vs, vl = sequence(v_rows, table[slot], past + count)
        k, v = values(kc, ks, kl, 64), values(vc, vs, vl, 64)
        spread = values(vc, vs, torch.zeros_like(vl), 64)
        heads = k.shape[0]
        i, j = torch.arange(past, past + count, device=q.device)[:, None], torch.arange(past + count, device=q.device)[None]
        hidden = (j > i) | ((j <= i - window) if window else torch.zeros_like(j > i))
        for h in range(n_q):
            e = h // (n_q // heads)
            x = q[row:row + count, h].double()
            s = (x @ k[e].t() * scale).masked_fill(hidden, -float("inf"))
            p = torch.exp(s - s.amax(1, keepdim=True))
            total = p.sum(1, keepdim=True)
            # a value that is not finite joins the rows that see it, and only these
            seen = lambda t: torch.where(torch.isfinite(t), t, torch.zeros_like(t))
            bad = ((~torch.isfinite(v[e])).double().t()[None] * (~hidden).double()[:, None]).sum(2) > 0 \
                if not bool(torch.isfinite(v[e]).all()) else None
            o = (p / total) @ seen(v[e])
            if bad is not None:
                o = torch.where(bad, torch.full_like(o, float("nan")), o)
            cols = slice(h * d, (h + 1) * d)
            out[row:row + count, cols] = o
            kq = values(kc[e], ks[e], torch.zeros_like(kl[e]), 64)
            a = (x.abs() @ (kq + (k[e] - kq).abs()).t()).masked_fill(hidden, 0.0) * scale
            most = x.abs().amax(1, keepdim=True)
            off = 24 * 2 ** -24 * 1.4427 * a + 2 ** -36 * most * (kq.sum(1)[None] * scale) + 2 ** -22 + 2 ** -23 * s.masked_fill(hidden, 0.0).abs()
            off = (off * (p > 0)).amax(1, keepdim=True)
            size = (p / total) @ seen(v[e].abs())
            parts = (p / total) @ seen(spread[e] + (v[e] - spread[e]).abs())
            bound[row:row + count, cols] = 2 ** -8 * o.abs() + 2 ** -11 * (p / total) @ seen(spread[e]) + 2 * off * size \
                + ((past + count) / 16 + 64) * 2 ** -23 * parts
    return out, bound
