"""What is measured of the cache held in 4 bits: writing keys and values into it, attention over it, the sums of every
key's attention weight, and the eviction of the keys with the least of it.

A page of a key/value head holds P tokens.  A token's key (and its value) is cut into blocks of 32 coordinates (the
last one filled up with zeros); a block is held as a power of two 2^s and 32 codes of 4 bits: a sign above the number of one
of the magnitudes 0, 0.5, 1, 1.5, 2, 3, 4, 6.  s is such that the block's largest magnitude lies in (3.5, 7] 2^s; a
coordinate becomes the nearest of the magnitudes, ties to the even number, above 6 to 6.  The bytes of a page of a head:
the keys, token by token, two coordinates a byte (the first in the low half); the values by 8 tokens, slices of 128 (64,
32) coordinates, sixteenths of a slice, and then token by token; a byte (s + 127) for every block and token of the keys;
the same of the values.
"""
import math
import random
from types import SimpleNamespace

import torch

own = False

GPU = "cuda:0"
PAGE = 16
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


# -- the cases --------------------------------------------------------------------------------------------------------

def _text(numbers):
    """Numbers a request, as a case holds them."""
    return " ".join(str(n) for n in numbers)


def _numbers(text):
    return [int(n) for n in text.split()]


def listed():
    return [
        # a decode step of eight requests at the smallest layer sizes: one launch whose latency counts
        {"name": "write 8 rows", "op": "write", "rows": 8, "heads": 9, "kv": 3, "dim": 64, "type": "bf16", "interleaved": False},
        # a prompt portion at the sizes of the largest preset
        {"name": "write 2048 rows", "op": "write", "rows": 2048, "heads": 32, "kv": 8, "dim": 128, "type": "bf16", "interleaved": False},
        # one short request decodes
        {"name": "decode 1 of 300", "op": "attend", "heads": 9, "kv": 3, "dim": 64, "type": "bf16", "window": 0, "cached": "300",
         "counts": "1", "weights": False},
        # eight requests behind their prompts, a key head for every query head
        {"name": "decode 8 of 4k", "op": "attend", "heads": 32, "kv": 32, "dim": 64, "type": "bf16", "window": 0,
         "cached": "2048 2501 4095 3333 2890 4000 3601 2222", "counts": _text([1] * 8), "weights": False},
        # many long contexts, what the narrow cache is for
        {"name": "decode 32 of 16k", "op": "attend", "heads": 32, "kv": 8, "dim": 128, "type": "bf16", "window": 0,
         "cached": _text(8192 + 263 * i for i in range(32)), "counts": _text([1] * 32), "weights": False},
        # the second portion of a long prompt
        {"name": "prompt 4000 after 1111", "op": "attend", "heads": 32, "kv": 8, "dim": 128, "type": "bf16", "window": 0, "cached": "1111",
         "counts": "4000", "weights": False},
        # portions of prompts beside decoded tokens, 32-bit activations, heads that fill no power of two, a window
        {"name": "mixed step f32", "op": "attend", "heads": 6, "kv": 2, "dim": 96, "type": "f32", "window": 500,
         "cached": "0 77 1500 900 0 2011", "counts": "333 1 1 200 17 1", "weights": False},
        # requests at their bound of keys decode, and every key's weight is summed
        {"name": "decode and sum 16 of 2k", "op": "attend", "heads": 32, "kv": 8, "dim": 128, "type": "bf16", "window": 0,
         "cached": _text(2049 + 7 * i for i in range(16)), "counts": _text([1] * 16), "weights": True},
        # a prompt whose keys' weights are summed
        {"name": "prompt and sum 2048", "op": "attend", "heads": 9, "kv": 3, "dim": 64, "type": "bf16", "window": 0, "cached": "0",
         "counts": "2048", "weights": True},
        # one decoding request passes its bound by 64 keys: all layers of the smallest preset
        {"name": "evict 2112 to 2048", "op": "evict", "sites": 30, "kv": 3, "dim": 64, "lengths": "2112", "keep": 2048, "recent": 512},
        # long prompts shrink to their bound: some layers of the largest preset
        {"name": "evict 16k to 1k", "op": "evict", "sites": 4, "kv": 8, "dim": 128, "lengths": "16384 9001 12345 1500", "keep": 1024,
         "recent": 256},
    ]


def _between(rng, low, high):
    """A whole number, its logarithm spread evenly."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    heads, kv, dim = rng.choice([(9, 3, 64), (32, 32, 64), (32, 8, 128), (6, 2, 96), (4, 1, 80), (8, 8, 32), (16, 2, 256), (5, 5, 16)])
    kind = rng.choice(["float32", "bfloat16", "bfloat16"])
    kind = "f32" if kind == "float32" else "bf16"
    op = rng.choice(["write", "decode", "decode", "prompt", "evict"])
    if op == "write":
        return {"op": "write", "rows": _between(rng, 1, 2048), "heads": heads, "kv": kv, "dim": dim, "type": kind,
                "interleaved": rng.random() < 0.3}
    if op == "evict":
        keep = _between(rng, 64, 2048)
        longest = min(16384, (1 << 16) // kv)
        lengths = [_between(rng, keep // 2 + 1, max(keep + 64, longest)) for _ in range(rng.randint(1, 3))]
        return {"op": "evict", "sites": rng.randint(1, 6), "kv": kv, "dim": dim, "lengths": _text(lengths), "keep": keep,
                "recent": rng.randint(0, keep)}
    window = 0 if rng.random() < 0.7 else _between(rng, 16, 2048)
    weights = rng.random() < 0.4
    if op == "decode":
        requests = _between(rng, 1, 32)
        top = min(16384, (1 << 20) // (requests * kv * dim // 128 + 1))
        cached = [_between(rng, 1, max(64, top)) - 1 for _ in range(requests)]
        counts = [1] * requests
    else:
        n = rng.randint(1, 4)
        cached = [rng.choice([0, _between(rng, 1, 3000)]) for _ in range(n)]
        counts = [_between(rng, 1, 2000 // n) for _ in range(n)]
    return {"op": "attend", "heads": heads, "kv": kv, "dim": dim, "type": kind, "window": window, "cached": _text(cached), "counts": _text(counts),
            "weights": weights}


def work(case):
    kv, dim = case["kv"], case["dim"]
    held = kv * (dim // 2 + -(-dim // 32))            # bytes of a token's keys (or values)
    if case["op"] == "evict":
        lengths = _numbers(case["lengths"])
        kept = sum(min(n, case["keep"]) for n in lengths) * case["sites"]
        seen = sum(lengths) * case["sites"]
        # weights read and the kept ones written, kept indices; the kept keys and values read, and written as 16-bit values
        return {"bytes": 4 * kv * (seen + 2 * kept) + 2 * kept * held + 4 * kept * kv * dim, "flops": 0}
    size = 2 if case["type"] == "bf16" else 4
    heads = case["heads"]
    if case["op"] == "write":
        rows = case["rows"]
        return {"bytes": rows * (size * (2 * heads + 2 * kv) * dim + 4 * kv * dim), "flops": 0}
    pairs, keys = 0, 0
    window = case["window"] or 1 << 30
    counts = _numbers(case["counts"])
    for n, c in zip(counts, _numbers(case["cached"])):
        pairs += sum(min(c + i + 1, window) for i in range(n))
        keys += min(c + n, window + n - 1)
    rows = sum(counts)
    bytes_, flops = 2 * rows * heads * dim * size + 2 * keys * held, 4 * pairs * heads * dim
    if case["weights"]:
        bytes_ += 8 * kv * keys
    return {"bytes": bytes_, "flops": flops}


# -- the format, by elementary operations -------------------------------------------------------------------------------

MAGNITUDES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _sizes(dim, page):
    """(coordinates with the zeros behind them, blocks, coordinates of a slice of the values, bytes of a page)."""
    pad = -(-dim // 32) * 32
    cut = 128 if pad % 128 == 0 else 64 if pad % 64 == 0 else 32
    return pad, pad // 32, cut, page * (pad + pad // 16)


def _codes(x):
    """Codes and exponents of float x [..., dim]: (uint8 [..., pad], int32 [..., blocks])."""
    dim = x.shape[-1]
    pad = -(-dim // 32) * 32
    x = torch.nn.functional.pad(x, (0, pad - dim)).unflatten(-1, (pad // 32, 32))
    m, e = torch.frexp(x.abs().amax(-1))              # the largest magnitude is m 2^e with m in [0.5, 1)
    s = torch.where(m > 0.875, e - 2, e - 3).clamp(-125, 125)
    y = torch.ldexp(x.abs(), -s.unsqueeze(-1))
    code = (y > 0.25).to(torch.uint8) + (y >= 0.75) + (y > 1.25) + (y >= 1.75) + (y > 2.5) + (y >= 3.5) + (y > 5)
    return (code | (x < 0).to(torch.uint8) << 3).flatten(-2), s


def _values(codes, s, dim):
    """Floats [..., dim] that codes [..., pad] and exponents [..., blocks] stand for."""
    table = torch.tensor(MAGNITUDES + tuple(-m for m in MAGNITUDES), device=codes.device)
    x = table[codes.int()].unflatten(-1, (-1, 32))
    return torch.ldexp(x, s.unsqueeze(-1)).flatten(-2)[..., :dim]


def _pages(keys, values, page):
    """uint8 pages [..., heads, bytes] of keys and values [..., heads, page, dim]."""
    _, blocks, cut, _ = _sizes(keys.shape[-1], page)
    (kc, ks), (vc, vs) = _codes(keys), _codes(values)
    kc, vc = (c[..., 0::2] | c[..., 1::2] << 4 for c in (kc, vc))
    vc = vc.unflatten(-1, (-1, 16, cut // 32)).unflatten(-4, (page // 8, 8)).movedim(-4, -2)
    scales = [(s + 127).to(torch.uint8).transpose(-1, -2).flatten(-2) for s in (ks, vs)]
    return torch.cat([kc.flatten(-2), vc.flatten(-5), *scales], -1)


def _held(pages, dim, page):
    """Keys and values, floats [..., heads, page, dim], that pages [..., heads, bytes] hold."""
    pad, blocks, cut, _ = _sizes(dim, page)
    half = page * pad // 2
    kc, vc = pages[..., :half].unflatten(-1, (page, -1)), pages[..., half:2 * half]
    vc = vc.unflatten(-1, (page // 8, pad // cut, 16, 8, cut // 32)).movedim(-2, -4).flatten(-3).flatten(-3, -2)
    scales = pages[..., 2 * half:].unflatten(-1, (2, blocks, page)).transpose(-1, -2).int() - 127
    return [_values(torch.stack([c & 15, c >> 4], -1).flatten(-2), scales[..., i, :, :], dim) for i, c in ((0, kc), (1, vc))]


# -- inputs -----------------------------------------------------------------------------------------------------------

def _filled(lengths, sites, kv, dim, g):
    """A pool of pages in no order that holds `lengths` tokens a request, and its block tables."""
    wide = max(-(-n // PAGE) for n in lengths)
    total = sum(-(-n // PAGE) for n in lengths)
    order = torch.randperm(total + 2, generator=g, device=GPU).int()
    tables = torch.full((len(lengths), wide), -1, dtype=torch.int32, device=GPU)
    pool = torch.zeros(sites, total + 2, kv, _sizes(dim, PAGE)[3], dtype=torch.uint8, device=GPU)
    spread = torch.exp(0.5 * torch.randn(2, kv, 1, dim, generator=g, device=GPU))     # some channels are wide, as trained ones are
    spread /= spread.square().mean(-1, keepdim=True).sqrt()
    at = 0
    for r, n in enumerate(lengths):
        pages = -(-n // PAGE)
        tables[r, :pages] = order[at:at + pages]
        for site in range(sites):
            k, v = torch.randn(2, pages, kv, PAGE, dim, generator=g, device=GPU) * spread.unsqueeze(1)
            pool[site, order[at:at + pages].long()] = _pages(k, v, PAGE)
        at += pages
    return pool, tables, order[at:]


def prepare(case, seed):
    g = torch.Generator(device=GPU).manual_seed(seed)
    kv, dim = case["kv"], case["dim"]
    s = SimpleNamespace(op=case["op"], kv=kv, dim=dim)
    if case["op"] == "write":
        rows, heads = case["rows"], case["heads"]
        dtype = TYPES[case["type"]]
        s.heads, s.interleaved = heads, case["interleaved"]
        s.qkv = torch.randn(rows, (heads + 2 * kv) * dim, generator=g, device=GPU).to(dtype)
        s.positions = torch.randint(0, 8192, (rows,), generator=g, device=GPU).int()
        pages = -(-rows // PAGE) + 3
        s.slots = torch.randperm(pages * PAGE, generator=g, device=GPU)[:rows].int()
        angle = torch.arange(8192, device=GPU).double()[:, None] * 1e4 ** (-torch.arange(dim // 2, device=GPU).double() / (dim // 2))
        s.cos, s.sin = angle.cos().float(), angle.sin().float()
        s.pool = torch.zeros(1, pages, kv, _sizes(dim, PAGE)[3], dtype=torch.uint8, device=GPU)
        s.q = torch.empty(rows, heads * dim, dtype=dtype, device=GPU)
        s.keys, s.values = (torch.empty(1, rows, kv, dim, dtype=torch.bfloat16, device=GPU) for _ in range(2))
        return s
    if case["op"] == "evict":
        s.keep, s.recent, s.sites = case["keep"], case["recent"], case["sites"]
        lengths = _numbers(case["lengths"])
        requests, longest = len(lengths), max(max(lengths), case["keep"])
        # the pages that the kept keys go to, in a row behind those that are held
        fresh = -(-case["keep"] // PAGE)
        pool, s.tables, _ = _filled(lengths, s.sites, kv, dim, g)
        held = pool.shape[1]
        s.pool = torch.cat([pool, torch.zeros(s.sites, requests * fresh, *pool.shape[2:], dtype=torch.uint8, device=GPU)], 1)
        s.new_tables = (held + torch.arange(requests * fresh, device=GPU)).int().view(requests, fresh)
        s.lengths = torch.tensor(lengths, dtype=torch.int32, device=GPU)
        s.slots = torch.arange(requests, dtype=torch.int32, device=GPU)
        s.new_slots = s.slots + requests
        # sums of attention weights: a few keys have most of it, many have hardly any and are alike
        w = torch.exp(2 * torch.randn(s.sites, 2 * requests, kv, longest, generator=g, device=GPU))
        s.weights = [t.contiguous() for t in torch.where(w < 0.5, (w * 64).round() / 64, w)]
        s.kept = torch.empty(s.sites, requests, kv, s.keep, dtype=torch.int32, device=GPU)
        shape = (requests * s.keep, kv, dim)
        s.place = (s.new_tables.long()[:, torch.arange(s.keep, device=GPU) // PAGE] * PAGE + torch.arange(s.keep, device=GPU) % PAGE).int().flatten()
        s.keys, s.values = (torch.empty(s.sites, *shape, dtype=torch.bfloat16, device=GPU) for _ in range(2))
        return s
    heads, counts, cached = case["heads"], _numbers(case["counts"]), _numbers(case["cached"])
    dtype = TYPES[case["type"]]
    s.heads, s.window, s.scale = heads, case["window"], dim ** -0.5
    s.pool, s.tables, _ = _filled([c + n for c, n in zip(cached, counts)], 1, kv, dim, g)
    rows, most, S = sum(counts), max(counts), len(counts)
    s.query = (1.5 * torch.randn(rows, heads * dim, generator=g, device=GPU)).to(dtype)
    s.out = torch.empty_like(s.query)
    firsts = [sum(counts[:i]) for i in range(S)]
    where = torch.tensor(firsts, device=GPU)[:, None] + torch.arange(most, device=GPU)
    s.there = torch.arange(most, device=GPU) < torch.tensor(counts, device=GPU)[:, None]      # which rows a request has
    s.where = torch.where(s.there, where, 0)
    s.last = torch.tensor(cached, device=GPU)[:, None] + torch.arange(most, device=GPU)       # the last key a row sees
    s.counts, s.cached = counts, cached
    s.sums = None
    if case["weights"]:
        capacity = s.tables.shape[1] * PAGE
        s.sums = torch.rand(S + 2, kv, capacity, generator=g, device=GPU)
        s.stats = torch.empty(rows, heads, device=GPU)
        s.slots = torch.randperm(S + 2, generator=g, device=GPU)[:S].int()
    if own:
        from runtime.kernels import cache4
        s.plan = cache4.plan(counts, cached, heads, kv, dim, window=s.window, device=GPU, dtype=dtype,
                             state_slots=s.slots.tolist() if s.sums is not None else None)
    return s


# -- one pass -----------------------------------------------------------------------------------------------------------

def run(s):
    if own:
        return _run_own(s)
    return {"write": _write, "attend": _attend, "evict": _evict}[s.op](s)


def _run_own(s):
    from runtime.kernels import cache4
    if s.op == "write":
        cache4.rope_write(s.qkv, s.positions, s.slots, s.cos, s.sin, s.pool[0], s.q, s.heads, s.kv, s.dim, PAGE, interleaved=s.interleaved)
        cache4.read(s.pool, s.slots, s.keys, s.values, s.kv, s.dim, PAGE)
        return {"q": s.q, "keys": s.keys[0], "values": s.values[0]}
    if s.op == "evict":
        cache4.evict(s.pool, s.weights, s.tables, s.new_tables, s.lengths, s.slots, s.new_slots, s.kv, s.dim, PAGE, s.keep, s.recent, s.kept)
        n, top = len(s.lengths), s.keep
        cache4.read(s.pool, s.place, s.keys, s.values, s.kv, s.dim, PAGE)
        return {"kept": s.kept, "weights": [w[n:, :, :top] for w in s.weights],
                "keys": s.keys.unflatten(1, (n, top)), "values": s.values.unflatten(1, (n, top))}
    cache4.attention(s.query, s.pool[0], s.tables, s.plan, s.out, s.heads, s.kv, s.dim, PAGE, s.scale, window=s.window,
                     stats=None if s.sums is None else s.stats)
    if s.sums is None:
        return {"out": s.out}
    cache4.add_weights(s.query, s.stats, s.pool[0], s.tables, s.plan, s.sums, s.heads, s.kv, s.dim, PAGE, s.scale, window=s.window)
    return {"out": s.out, "weights": s.sums}


def _turned(x, cos, sin, interleaved):
    """Floats x [rows, heads, dim] turned by the angles of their rows [rows, 1, dim / 2]."""
    half = x.shape[-1] // 2
    a, b = (x[..., 0::2], x[..., 1::2]) if interleaved else (x[..., :half], x[..., half:])
    a, b = a * cos - b * sin, b * cos + a * sin
    return torch.stack([a, b], -1).flatten(-2) if interleaved else torch.cat([a, b], -1)


def _write(s):
    rows = s.qkv.shape[0]
    at = s.positions.long()
    q, k, v = s.qkv.float().view(rows, -1, s.dim).split([s.heads, s.kv, s.kv], 1)
    cos, sin = s.cos[at][:, None], s.sin[at][:, None]
    q, k = _turned(q, cos, sin, s.interleaved), _turned(k, cos, sin, s.interleaved)
    held = [_values(*_codes(x), s.dim).to(torch.bfloat16) for x in (k, v)]
    return {"q": q.flatten(1).to(s.qkv.dtype), "keys": held[0], "values": held[1]}


def _attend(s):
    S, most = s.where.shape
    group = s.heads // s.kv
    keys, values = (x.movedim(2, 1).flatten(2, 3) for x in _held(s.pool[0][s.tables.clamp(min=0).long()], s.dim, PAGE))
    q = s.query.float()[s.where].view(S, most, s.kv, group, s.dim).permute(0, 2, 3, 1, 4).flatten(2, 3)
    index = torch.arange(keys.shape[2], device=GPU)
    seen = index <= s.last[..., None]
    if s.window:
        seen &= index > s.last[..., None] - s.window
    seen = (seen & s.there[..., None])[:, None, None]
    p = ((q @ keys.transpose(-1, -2)) * s.scale).unflatten(2, (group, most))
    p = torch.exp(p.masked_fill_(~seen, -math.inf) - p.amax(-1, keepdim=True).clamp(min=-3e38))
    p /= p.sum(-1, keepdim=True).clamp(min=1e-38)
    out = (p.flatten(2, 3) @ values).unflatten(2, (group, most)).permute(0, 3, 1, 2, 4).flatten(2)
    out = {"out": out[s.there].to(s.query.dtype)}
    if s.sums is not None:
        s.sums[s.slots.long()] += p.sum((2, 3))
        out["weights"] = s.sums
    return out


def _evict(s):
    n, top = s.lengths.long(), s.keep
    w = torch.stack([t[s.slots.long()] for t in s.weights])                   # [sites, requests, heads, keys]
    index = torch.arange(w.shape[-1], device=GPU)
    length = n[:, None, None]
    rank = torch.where(index < length, torch.where(index >= length - s.recent, math.inf, w), -math.inf)
    order = torch.sort(rank, dim=-1, descending=True, stable=True).indices[..., :top]
    there = torch.arange(top, device=GPU) < length
    chosen = torch.sort(torch.where(there, order, 1 << 40), dim=-1).values
    kept = torch.where(there, chosen, 0)
    page = torch.gather(s.tables.long()[None, :, None].expand(*kept.shape[:3], -1), -1, kept // PAGE)
    site, head = (torch.arange(d, device=GPU).view(shape) for d, shape in ((s.sites, (-1, 1, 1, 1)), (s.kv, (1, 1, -1, 1))))
    held = []
    for x in _held(s.pool, s.dim, PAGE):
        x = x[site, page, head, kept % PAGE]                                  # [sites, requests, heads, keep, dim]
        held.append(torch.where(there[..., None], x, 0).transpose(2, 3).to(torch.bfloat16))
    return {"kept": torch.where(there, kept, -1).int(), "weights": list(torch.where(there, torch.gather(w, -1, kept), 0)),
            "keys": held[0], "values": held[1]}


# -- the definition in 64 bits --------------------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    return {"write": _exact_write, "attend": _exact_attend, "evict": _exact_evict}[s.op](s)


def _exact_blocks(x):
    """What blocks of 32 of the last axis are held as, in 64 bits: the scale by logarithms, the magnitudes by distance."""
    rest = -x.shape[-1] % 32
    y = torch.cat([x, x.new_zeros(*x.shape[:-1], rest)], -1)
    y = y.reshape(*x.shape[:-1], -1, 32)
    most = y.abs().amax(-1, keepdim=True)
    step = 2.0 ** torch.ceil(torch.log2(most.clamp(min=2.0 ** -120) / 7))     # the largest magnitude in (3.5, 7] steps
    grid = torch.tensor([MAGNITUDES[i] for i in (0, 2, 4, 6, 1, 3, 5, 7)], dtype=torch.float64, device=x.device)
    near = ((y / step).abs()[..., None] - grid).abs().argmin(-1)              # of two as near the first: an even number
    return (grid[near] * torch.sign(y) * step).reshape(*x.shape[:-1], -1)[..., :x.shape[-1]]


def _exact_write(s):
    rows, dim = s.qkv.shape[0], s.dim
    x = s.qkv.double().reshape(rows, -1, dim)
    z = x[:, :s.heads + s.kv]
    z = torch.complex(z[..., 0::2], z[..., 1::2]) if s.interleaved else torch.complex(z[..., :dim // 2], z[..., dim // 2:])
    z = z * torch.complex(s.cos.double(), s.sin.double())[s.positions.long()][:, None]
    z = torch.view_as_real(z).reshape(rows, -1, dim) if s.interleaved else torch.cat([z.real, z.imag], -1)
    return {"q": z[:, :s.heads].reshape(rows, -1), "keys": _exact_blocks(z[:, s.heads:]), "values": _exact_blocks(x[:, s.heads + s.kv:])}


def _exact_tokens(s, site, request, length):
    """Keys and values [heads, length, dim] of a request in 64 bits."""
    pad, blocks, cut, _ = _sizes(s.dim, PAGE)
    b = s.pool[site][s.tables[request, :-(-length // PAGE)].long()].long()
    half = PAGE * pad // 2
    signed = torch.tensor([m * f for f in (1, -1) for m in MAGNITUDES], dtype=torch.float64, device=GPU)
    token, d = torch.arange(PAGE, device=GPU)[:, None], torch.arange(pad, device=GPU)[None]
    at_key = token * (pad // 2) + d // 2
    inner = d % cut
    at_value = half + (((token // 8 * (pad // cut) + d // cut) * 16 + inner * 16 // cut) * 8 + token % 8) * (cut // 32) + inner % (cut // 16) // 2
    found = []
    for at, scales in ((at_key, 2 * half), (at_value, 2 * half + blocks * PAGE)):
        code = (b[..., at] >> (4 * (d % 2))) & 15
        x = signed[code] * 2.0 ** (b[..., scales + d // 32 * PAGE + token] - 127).double()
        found.append(x.transpose(0, 1).reshape(s.kv, -1, pad)[:, :length, :s.dim])
    return found


def _exact_attend(s):
    group, first = s.heads // s.kv, 0
    out = torch.zeros(s.query.shape, dtype=torch.float64, device=GPU)
    sums = None if s.sums is None else s.sums.double()
    for r, (n, c) in enumerate(zip(s.counts, s.cached)):
        keys, values = _exact_tokens(s, 0, r, c + n)
        mask = torch.ones(n, c + n, dtype=torch.bool, device=GPU).tril(c)
        if s.window:
            mask = mask.triu(c - s.window + 1)
        q = s.query[first:first + n].double().view(n, s.heads, s.dim)
        for h in range(s.heads):
            p = torch.softmax((q[:, h] @ keys[h // group].T * s.scale).masked_fill(~mask, -math.inf), -1)
            out[first:first + n, h * s.dim:(h + 1) * s.dim] = p @ values[h // group]
            if sums is not None:
                sums[s.slots[r].item(), h // group, :c + n] += p.sum(0)
        first += n
    return {"out": out} if sums is None else {"out": out, "weights": sums}


def _exact_evict(s):
    requests, top = len(s.lengths), s.keep
    keys = torch.zeros(s.sites, requests, top, s.kv, s.dim, dtype=torch.float64, device=GPU)
    values, kept = torch.zeros_like(keys), torch.full((s.sites, requests, s.kv, top), -1, dtype=torch.int32, device=GPU)
    weights = [torch.zeros(requests, s.kv, top, dtype=torch.float64, device=GPU) for _ in range(s.sites)]
    for site in range(s.sites):
        for r, n in enumerate(s.lengths.tolist()):
            k, v = _exact_tokens(s, site, r, n)
            for h in range(s.kv):
                w = s.weights[site][s.slots[r].item(), h, :n].double()
                old = max(0, n - s.recent)
                # by weight, and of equal ones by index: a key is kept if fewer than top - recent stand before it
                order = sorted(range(old), key=w.tolist().__getitem__, reverse=True) if n > top else list(range(old))
                index = torch.tensor(sorted(order[:max(0, top - (n - old))]) + list(range(old, n)), device=GPU)[-top:]
                m = len(index)
                kept[site, r, h, :m] = index.int()
                weights[site][r, h, :m] = w[index]
                keys[site, r, :m, h], values[site, r, :m, h] = k[h, index], v[h, index]
    return {"kept": kept, "weights": weights, "keys": keys, "values": values}
