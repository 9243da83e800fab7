"""The cache held in 4 bits in its plainest form, in 64 bits: what a block of coordinates is held as, the bytes of a page,
attention over held keys and values, the sums of attention weight, and which keys stay."""
import math

import torch

MAGNITUDES = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


def held(x):
    """(codes, exponents, values) of x [..., dim]: a block of 32 at a time, one number at a time."""
    x = x.double()
    dim, pad = x.shape[-1], -(-x.shape[-1] // 32) * 32
    flat = torch.nn.functional.pad(x, (0, pad - dim)).reshape(-1, 32)
    flat = torch.where(flat.isnan(), torch.zeros_like(flat), flat)
    codes, powers = torch.zeros(flat.shape, dtype=torch.uint8), torch.zeros(len(flat), dtype=torch.int64)
    for b, block in enumerate(flat):
        most = float(block.abs().max())
        s = -125
        while s < 125 and most > 7 * 2.0 ** s:
            s += 1
        powers[b] = s
        away = (block.abs()[:, None] / 2.0 ** s - MAGNITUDES).abs()
        away[block.abs().isinf()] = torch.tensor([1.0] * 7 + [0.0], dtype=torch.float64)
        best = away.min(1, keepdim=True).values
        for i in range(32):
            near = [j for j in range(8) if float(away[i, j]) == float(best[i])]
            codes[b, i] = (near[0] if len(near) == 1 else [j for j in near if j % 2 == 0][0]) + (8 if block[i] < 0 else 0)
    values = MAGNITUDES[(codes & 7).long()] * torch.where(codes > 7, -1.0, 1.0) * (2.0 ** powers.double())[:, None]
    shape = x.shape[:-1]
    return codes.reshape(*shape, pad), powers.reshape(*shape, pad // 32), values.reshape(*shape, pad)[..., :dim]


def quick_held(x):
    """The values of `held`, for larger inputs: finite numbers, by comparisons over all at once."""
    x = x.double()
    dim, pad = x.shape[-1], -(-x.shape[-1] // 32) * 32
    y = torch.nn.functional.pad(x, (0, pad - dim)).reshape(*x.shape[:-1], pad // 32, 32)
    most = y.abs().amax(-1, keepdim=True).clamp(min=2.0 ** -300)
    s = torch.ceil(torch.log2(most / 7)).clamp(-125, 125)
    z = y.abs() / 2.0 ** s
    code = sum((z > t) if even else (z >= t) for t, even in ((.25, 1), (.75, 0), (1.25, 1), (1.75, 0), (2.5, 1), (3.5, 0), (5.0, 1)))
    code = code | (8 * (y < 0))
    values = MAGNITUDES[code & 7] * y.sign() * 2.0 ** s
    return code.reshape(*x.shape[:-1], pad).to(torch.uint8), s.reshape(*x.shape[:-1], pad // 32).long(), values.reshape(*x.shape[:-1], pad)[..., :dim]


def put(page, t, value, codes, powers, P):
    """Writes one token's codes [pad] and exponents into a head's page (uint8 bytes), coordinate by coordinate."""
    pad = len(codes)
    cut = 128 if pad % 128 == 0 else 64 if pad % 64 == 0 else 32
    for d in range(0, pad, 2):
        byte = int(codes[d]) | int(codes[d + 1]) << 4
        if value:
            run = cut // 16                                     # coordinates of a sixteenth of a slice
            where = P * pad // 2 + (((t // 8) * (pad // cut) + d // cut) * 16 + d % cut // run) * 8 * run // 2 + (t % 8) * run // 2 + d % run // 2
        else:
            where = t * pad // 2 + d // 2
        page[where] = byte
    for b in range(pad // 32):
        page[P * pad + ((pad // 32 if value else 0) + b) * P + t] = int(powers[b]) + 127


def pages_of(keys, values, slots, n_pages, P, fill=None):
    """Pages uint8 [n_pages, heads, bytes] that hold keys and values [T, heads, dim] in token slots; `fill`: bytes elsewhere."""
    T, heads, dim = keys.shape
    pad = -(-dim // 32) * 32
    pages = torch.zeros(n_pages, heads, P * (pad + pad // 16), dtype=torch.uint8) if fill is None else fill.clone()
    kc, kp, _ = quick_held(keys)
    vc, vp, _ = quick_held(values)
    import numpy as np
    raw = pages.numpy()
    for i, slot in enumerate(slots):
        if slot < 0:
            continue
        for h in range(heads):
            page = raw[slot // P, h]
            put(page, slot % P, False, kc[i, h].numpy(), kp[i, h].numpy(), P)
            put(page, slot % P, True, vc[i, h].numpy(), vp[i, h].numpy(), P)
    return torch.from_numpy(np.ascontiguousarray(raw))


def attention(q, keys, values, cached, scale, window=0):
    """(out, |values| weighed likewise, weights [heads, rows, keys], scores) of rows q [n, heads, dim] behind `cached` keys; keys and
    values [heads of keys, cached + n, dim], a row that sees none gets zeros."""
    n, heads, _ = q.shape
    group = heads // keys.shape[0]
    total = keys.shape[1]
    row = torch.arange(n)[:, None] + cached
    index = torch.arange(total)[None]
    seen = (index <= row) & ((index > row - window) if window else torch.ones(1, 1, dtype=torch.bool))
    k, v = keys.double().repeat_interleave(group, 0), values.double().repeat_interleave(group, 0)
    s = torch.matmul(q.double().transpose(0, 1), k.transpose(1, 2)) * scale
    s = s.masked_fill(~seen, -math.inf)
    most = s.amax(-1, keepdim=True)
    w = torch.exp(s - torch.where(most.isinf(), torch.zeros_like(most), most))
    total = w.sum(-1, keepdim=True)
    w = torch.where(total > 0, w / total.clamp(min=1e-300), torch.zeros_like(w))
    return torch.matmul(w, v).transpose(0, 1), torch.matmul(w, v.abs()).transpose(0, 1), w, s


def score_error(q, keys, scale):
    """How far a score may be off, at most over the heads: products are exact, each of the sums of `dim` of them rounds in 32 bits, as does the
    scaling; in the exponent of 2, in units of the natural one."""
    group = q.shape[1] // keys.shape[0]
    k = keys.double().abs().repeat_interleave(group, 0)
    most = torch.matmul(q.double().abs().transpose(0, 1), k.transpose(1, 2)).amax() * scale
    return float(most) * (3 * q.shape[2] + 8) * 2.0 ** -24


def stays(w, n, keep, recent):
    """Indices, in order, of the keys of one head that stay."""
    if n <= keep:
        return list(range(n))
    old = max(0, n - recent)
    value = [float(x) for x in w[:old]]
    order = sorted(range(old), key=lambda i: (math.isnan(value[i]), 0.0 if math.isnan(value[i]) else -value[i], i))      # (a NaN is below every number)
    return sorted(order[:keep - (n - old)]) + list(range(old, n))
