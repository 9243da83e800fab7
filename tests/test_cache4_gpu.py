"""The kernels of the cache held in 4 bits against a plain implementation in 64 bits."""
import math

import pytest
import torch

import plain_cache4 as plain

pytestmark = pytest.mark.gpu

GPU = "cuda:0"
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
HALF = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}     # half a step of a rounding


def cache4():
    from runtime.kernels import cache4 as c
    return c


def slots_of(table, n, P):
    return [table[i // P] * P + i % P for i in range(n)]


# -- writing -----------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dim,heads,kv,P", [(64, 9, 3, 16), (128, 8, 2, 16), (32, 2, 2, 8), (96, 6, 2, 16), (16, 5, 5, 16), (80, 4, 1, 32), (256, 2, 1, 8),
                                            (20, 3, 1, 16), (160, 2, 2, 16), (192, 2, 1, 16), (224, 1, 1, 64), (2, 2, 1, 8)])
@pytest.mark.parametrize("kind,interleaved", [("bf16", False), ("f32", False), ("bf16", True)])
def test_write_and_read(dim, heads, kv, P, kind, interleaved):
    c, g = cache4(), torch.Generator().manual_seed(dim + heads)
    rows, dtype = 21, TYPES[kind]
    rot = dim if dim < 40 else dim - 16                            # (some coordinates do not turn)
    qkv = (torch.randn(rows, (heads + 2 * kv) * dim, generator=g) * torch.exp(torch.randn(rows, 1, generator=g) * 2)).to(dtype)
    qkv[3] = 0.0
    positions = torch.randint(0, 500, (rows,), generator=g, dtype=torch.int32)
    n_pages = rows // P + 3
    slots = torch.randperm(n_pages * P, generator=g)[:rows].int()
    slots[7] = -1
    angle = torch.arange(500).double()[:, None] * 1e4 ** (-torch.arange(rot // 2).double() / (rot // 2))
    cos, sin = angle.cos().float(), angle.sin().float()
    pages = torch.full((n_pages, kv, c.record_bytes(dim, P)), 0xA5, dtype=torch.uint8)
    x = qkv.float().view(rows, -1, dim)
    turned = x.clone()
    a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if interleaved else (x[..., :rot // 2], x[..., rot // 2:rot])
    cs, sn = cos[positions.long()][:, None], sin[positions.long()][:, None]
    first, second = a * cs - b * sn, b * cs + a * sn                # (32 bits, product by product, as the format says)
    if interleaved:
        turned[..., 0:rot:2], turned[..., 1:rot:2] = first, second
    else:
        turned[..., :rot // 2], turned[..., rot // 2:rot] = first, second
    k, v = turned[:, heads:heads + kv], x[:, heads + kv:]
    expected = plain.pages_of(k, v, slots.tolist(), n_pages, P, fill=pages)
    gpu = [t.to(GPU) for t in (qkv, positions, slots, cos, sin, pages)]
    q = torch.empty(rows, heads * dim, dtype=dtype, device=GPU)
    c.rope_write(*gpu, q, heads, kv, dim, P, interleaved=interleaved)
    assert torch.equal(q.cpu(), turned[:, :heads].reshape(rows, -1).to(dtype))
    assert torch.equal(gpu[0].cpu(), qkv)
    assert torch.equal(gpu[5].cpu(), expected)                     # every byte, also those that no row writes
    keys, values = (torch.empty(1, rows, kv, dim, dtype=torch.bfloat16, device=GPU) for _ in range(2))
    c.read(gpu[5][None], gpu[2], keys, values, kv, dim, P)
    for got, x in ((keys, k), (values, v)):
        want = plain.quick_held(x)[2]
        want[7] = 0.0
        assert torch.equal(got[0].cpu().double(), want)


def test_what_is_held_is_finite():
    """Borders between two codes, numbers beyond every scale, zeros, infinities and NaN."""
    c = cache4()
    dim, P = 32, 8
    rows = [[0.0] * 32, [7.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0] * 2 + [-7.0, -0.25, -0.75, -1.25, -1.75, -2.5, -3.5, -5.0] * 2,
            [7.0 + 2.0 ** -20] + [0.5, 1.5, 2.5, 3.5, 5.0, 7.0, 10.0] * 4 + [0.0] * 3, [math.inf, -math.inf, 3.0] + [1.0] * 29, [math.nan, 3.0, -1.0] + [0.5] * 29,
            [3e38, -3e38] + [1e30] * 30, [1e-45, 1e-40, -1e-38] + [0.0] * 29, [2.0 ** -124, 2.0 ** -126, 2.0 ** -127] + [2.0 ** -128] * 29]
    x = torch.tensor(rows, dtype=torch.float32)
    n = len(rows)
    qkv = torch.stack([x, x, -x], 1).reshape(n, 96).to(GPU)
    cos, sin = torch.ones(1, 1, device=GPU), torch.zeros(1, 1, device=GPU)
    pages = torch.zeros(1, 1, c.record_bytes(dim, P), dtype=torch.uint8, device=GPU)
    slots = torch.arange(n, dtype=torch.int32, device=GPU)
    q = torch.empty(n, 32, device=GPU)
    # (coordinates 0 and 1 turn by nothing: NaN and infinities times zero would spread to the neighbour, so keys are checked where both are finite)
    c.rope_write(qkv, torch.zeros(n, dtype=torch.int32, device=GPU), slots, cos, sin, pages, q, 1, 1, dim, P)
    keys, values = (torch.empty(1, n, 1, dim, dtype=torch.bfloat16, device=GPU) for _ in range(2))
    c.read(pages[None], slots, keys, values, 1, dim, P)
    for got, y, where in ((keys, x, [0, 1, 2, 5, 6, 7]), (values, -x, range(n))):
        got = got[0, :, 0].cpu().double()
        assert got.isfinite().all()
        for i in where:
            assert torch.equal(got[i], plain.held(y[i])[2]), i


# -- attention ------------------------------------------------------------------------------------------------------

def a_step(counts, cached, heads, kv, dim, P, kind, seed=0, spread=1.5):
    g = torch.Generator().manual_seed(seed)
    S, rows = len(counts), sum(counts)
    lengths = [a + b for a, b in zip(counts, cached)]
    need = [-(-n // P) for n in lengths]
    n_pages = sum(need) + 3
    order = torch.randperm(n_pages, generator=g).tolist()
    width = max(need) + 1
    tables = torch.full((S, width), -1, dtype=torch.int32)
    # bytes that nobody wrote may be anything: scales of 255, codes of any kind
    pages = torch.randint(0, 256, (n_pages, kv, cache4().record_bytes(dim, P)), generator=g, dtype=torch.int32).to(torch.uint8)
    pages[..., P * plain_pad(dim):] = 255
    keys, values = [], []
    for s in range(S):
        own = [order.pop() for _ in range(need[s])]
        tables[s, :need[s]] = torch.tensor(own, dtype=torch.int32)
        k, v = torch.randn(2, lengths[s], kv, dim, generator=g)
        pages = plain.pages_of(k, v, slots_of(own, lengths[s], P), n_pages, P, fill=pages)
        keys.append(plain.quick_held(k)[2].transpose(0, 1))
        values.append(plain.quick_held(v)[2].transpose(0, 1))
    q = (spread * torch.randn(rows, heads * dim, generator=g)).to(TYPES[kind])
    return q, pages, tables, keys, values


def plain_pad(dim):
    return -(-dim // 32) * 32


def check_step(counts, cached, heads, kv, dim, P, kind, window=0, weights=False, force=None, seed=0):
    c = cache4()
    q, pages, tables, keys, values = a_step(counts, cached, heads, kv, dim, P, kind, seed)
    dtype, scale = TYPES[kind], dim ** -0.5
    S, rows = len(counts), sum(counts)
    plan = c.plan(counts, cached, heads, kv, dim, window=window, dtype=dtype, state_slots=[S - s for s in range(S)] if weights else None)
    if force is not None:
        plan = forced(c, plan, counts, cached, *force, window)
    out = torch.full((rows, heads * dim), math.nan, dtype=dtype, device=GPU)
    stats = torch.empty(rows, heads, device=GPU) if weights else None
    gq, gp, gt = q.to(GPU), pages.to(GPU), tables.to(GPU)
    c.attention(gq, gp, gt, plan, out, heads, kv, dim, P, scale, window=window, stats=stats)
    got, first = out.cpu().double().view(rows, heads, dim), 0
    sums = None
    if weights:
        before = torch.rand(S + 2, kv, max(a + b for a, b in zip(counts, cached)) + 5, generator=torch.Generator().manual_seed(seed))
        sums = before.to(GPU)
        c.add_weights(gq, stats, gp, gt, plan, sums, heads, kv, dim, P, scale, window=window)
        again = before.to(GPU)
        c.add_weights(gq, stats, gp, gt, plan, again, heads, kv, dim, P, scale, window=window)
        assert torch.equal(sums, again)
        sums, expected_sums, room = sums.cpu().double(), before.double(), torch.zeros(before.shape, dtype=torch.float64)
    for s in range(S):
        n = counts[s]
        rowsq = q[first:first + n].double().view(n, heads, dim)
        want, weighed, w, score = plain.attention(rowsq, keys[s], values[s], cached[s], scale, window)
        # A weight is off by twice what a score may be off (itself and the sum that it is divided by), by its exponential (2^-21, both) and, where it
        # goes to the instruction in bf16, by half a step; the sums over the keys round in 32 bits; the result rounds once
        off = 2 * plain.score_error(rowsq, keys[s], scale) + 2.0 ** -21 + (keys[s].shape[1] + 32) * 2.0 ** -24
        room_out = weighed * (off + (HALF[dtype] if kind == "bf16" else 2.0 ** -23)) + want.abs() * HALF[dtype]
        worst = ((got[first:first + n] - want).abs() - room_out * 1.01).max()
        assert worst <= 0, (s, float(worst), float((got[first:first + n] - want).abs().max()))
        if weights:
            part = w.view(kv, heads // kv, n, -1).sum((1, 2))
            expected_sums[S - s, :, :part.shape[1]] += part
            room[S - s, :, :part.shape[1]] += part * (off + (n * heads // kv + 16) * 2.0 ** -24) + expected_sums[S - s, :, :part.shape[1]] * 2.0 ** -23
        first += n
    if weights:
        assert ((sums - expected_sums).abs() <= room * 1.01).all()


def forced(c, plan, counts, cached, form, pieces, window):
    """The plan with another form and another number of pieces."""
    group = plan.heads // plan.kv_heads
    per_task = max(1, c.tile_of(form) // group)
    return c._plan(counts, cached, plan.heads, plan.kv_heads, plan.dim, window, torch.device(GPU), None, form, per_task, pieces)


HEADS = [(9, 3, 64), (4, 4, 64), (8, 2, 128), (6, 2, 96), (5, 5, 16), (4, 1, 80), (16, 2, 256), (3, 1, 20), (2, 1, 160), (2, 2, 192), (3, 1, 224), (40, 1, 64), (34, 2, 32)]


@pytest.mark.parametrize("heads,kv,dim", HEADS)
@pytest.mark.parametrize("kind", ["bf16", "f32"])
def test_decode(heads, kv, dim, kind):
    check_step([1] * 5, [0, 1, 31, 97, 200], heads, kv, dim, 16, kind, weights=True)


@pytest.mark.parametrize("heads,kv,dim", HEADS)
@pytest.mark.parametrize("kind", ["bf16", "f32"])
def test_prompts_beside_single_tokens(heads, kv, dim, kind):
    check_step([37, 1, 70, 5], [0, 63, 41, 9], heads, kv, dim, 16, kind, weights=True)


@pytest.mark.parametrize("P", [8, 16, 32, 128])
@pytest.mark.parametrize("window", [0, 1, 7, 40, 1000])
@pytest.mark.parametrize("counts,cached", [([1, 1, 1], [0, 50, 130]), ([45, 1, 90], [0, 70, 33])])
def test_windows_and_pages(P, window, counts, cached):
    check_step(counts, cached, 6, 2, 64, P, "bf16", window=window, weights=True)


@pytest.mark.parametrize("pieces", [1, 20])
@pytest.mark.parametrize("form,heads,kv,dim,kind", [(form, *h, kind) for form in range(3) for h in ((9, 3, 64), (8, 2, 128), (2, 1, 256), (6, 2, 96))
                                                    for kind in TYPES if form == 0 or (kind == "bf16" and h[2] <= 128)])
@pytest.mark.parametrize("window", [0, 50, 400])
def test_forms_and_pieces(form, pieces, heads, kv, dim, window, kind, monkeypatch):
    monkeypatch.setattr(cache4(), "LEAST_PIECE", 2)
    check_step([90, 1, 33], [10, 70, 500], heads, kv, dim, 16, kind, window=window, force=(form, pieces))


@pytest.mark.parametrize("shares", [0, 1, 2, 5])
@pytest.mark.parametrize("window", [0, 30])
@pytest.mark.parametrize("heads,kv,dim,kind", [(8, 2, 128, "bf16"), (9, 3, 64, "bf16"), (9, 3, 64, "f32"), (3, 1, 20, "bf16"), (2, 1, 256, "f32"), (40, 1, 32, "bf16")])
def test_shares_of_the_sums(shares, window, heads, kv, dim, kind, monkeypatch):
    monkeypatch.setattr(cache4(), "shares_of", lambda *a: shares)
    check_step([3, 1, 2], [40, 0, 300], heads, kv, dim, 16, kind, window=window, weights=True)
    check_step([150, 1, 40], [10, 70, 200], heads, kv, dim, 16, kind, window=window, weights=True)


# -- which keys stay ----------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dim,kv,P", [(64, 3, 16), (128, 2, 16), (96, 2, 8), (16, 1, 32), (256, 1, 16)])
@pytest.mark.parametrize("keep,recent", [(24, 8), (24, 0), (24, 24), (1, 0), (1, 1), (33, 5)])
@pytest.mark.parametrize("same_slot", [False, True])
def test_evict(dim, kv, P, keep, recent, same_slot):
    c, g = cache4(), torch.Generator().manual_seed(keep + recent)
    sites, lengths = 2, [100, 24, 7, 61, 0]
    R, capacity = len(lengths), 110
    need = [-(-n // P) for n in lengths]
    fresh = -(-keep // P)
    n_pages = sum(need) + R * fresh + 2
    order = torch.randperm(n_pages, generator=g).tolist()
    tables = torch.full((R, max(need)), -1, dtype=torch.int32)
    keys, values = torch.randn(2, sites, R, max(lengths), kv, dim, generator=g)
    storage = torch.randint(0, 256, (sites, n_pages, kv, c.record_bytes(dim, P)), generator=g, dtype=torch.int32).to(torch.uint8)
    for r in range(R):
        own = [order.pop() for _ in range(need[r])]
        tables[r, :need[r]] = torch.tensor(own, dtype=torch.int32)
        for site in range(sites):
            storage[site] = plain.pages_of(keys[site, r, :lengths[r]], values[site, r, :lengths[r]], slots_of(own, lengths[r], P), n_pages, P, fill=storage[site])
    new_tables = torch.tensor([[order.pop() for _ in range(fresh)] for _ in range(R)], dtype=torch.int32)
    slots = torch.tensor([3, 0, 5, 1, 2], dtype=torch.int32)
    new_slots = slots if same_slot else torch.tensor([7, 9, 6, 8, 4], dtype=torch.int32)
    sums = torch.exp(torch.randn(sites, 10, kv, capacity, generator=g))
    sums = torch.where(sums < 1, torch.zeros(()), sums)            # (many are alike)
    sums[0, 3, 0, :40] = torch.tensor([math.nan, math.inf, -0.0, 0.0, -1.0] * 8)
    gpu = [t.to(GPU) for t in sums]
    pool = storage.to(GPU)
    kept = torch.empty(sites, R, kv, keep, dtype=torch.int32, device=GPU)
    c.evict(pool, gpu, tables.to(GPU), new_tables.to(GPU), torch.tensor(lengths, dtype=torch.int32, device=GPU), slots.to(GPU), new_slots.to(GPU), kv, dim, P, keep,
            recent, kept)
    after = pool.cpu()
    kept = kept.cpu()
    want_sums = sums.clone()
    want_pool = storage.clone()
    for site in range(sites):
        for r in range(R):
            for h in range(kv):
                index = plain.stays(sums[site, slots[r], h], lengths[r], keep, recent)
                assert kept[site, r, h].tolist() == index + [-1] * (keep - len(index)), (site, r, h)
                row = torch.zeros(capacity)
                row[:len(index)] = sums[site, slots[r], h, index]
                want_sums[site, new_slots[r], h] = row
                if index:
                    sl = slots_of(new_tables[r].tolist(), len(index), P)
                    one = plain.pages_of(keys[site, r, index, h:h + 1], values[site, r, index, h:h + 1], sl, n_pages, P, fill=want_pool[site, :, h:h + 1])
                    want_pool[site, :, h:h + 1] = one
    if lengths[-1] == 0:                                            # (a request without keys: nothing of it is touched)
        want_sums[:, new_slots[-1]] = sums[:, new_slots[-1]]
    for site in range(sites):
        assert torch.equal(torch.nan_to_num(gpu[site].cpu(), nan=-5.0), torch.nan_to_num(want_sums[site], nan=-5.0))
    assert torch.equal(after, want_pool)


def test_evict_many_keys_and_sites():
    """Lengths past several turns of a block, more sites than one launch takes."""
    c, g = cache4(), torch.Generator(device=GPU).manual_seed(3)
    sites, kv, dim, P, n, keep, recent = 70, 1, 32, 16, 5003, 2100, 300
    pages = -(-n // P) + -(-keep // P)
    storage = torch.randint(0, 200, (sites, pages, kv, c.record_bytes(dim, P)), generator=g, device=GPU, dtype=torch.int32).to(torch.uint8)
    sums = [t.contiguous() for t in (torch.rand(sites, 1, kv, n, generator=g, device=GPU) * 50).round() / 50]
    tables = torch.arange(-(-n // P), device=GPU, dtype=torch.int32)[None]
    new_tables = torch.arange(-(-n // P), pages, device=GPU, dtype=torch.int32)[None]
    before = [t.cpu() for t in sums]
    kept = torch.empty(sites, 1, kv, keep, dtype=torch.int32, device=GPU)
    zero = torch.zeros(1, dtype=torch.int32, device=GPU)
    c.evict(storage, sums, tables, new_tables, zero + n, zero, zero, kv, dim, P, keep, recent, kept)
    place = torch.arange(keep, device=GPU, dtype=torch.int32) + int(new_tables[0, 0]) * P
    a, b, ka, vb = (torch.empty(sites, keep, kv, dim, dtype=torch.bfloat16, device=GPU) for _ in range(4))
    c.read(storage, place, a, b, kv, dim, P)
    for site in range(sites):
        index = plain.stays(before[site][0, 0].tolist(), n, keep, recent)
        assert kept[site, 0, 0].tolist() == index
        assert torch.equal(sums[site][0, 0, :keep].cpu(), before[site][0, 0, index]) and not sums[site][0, 0, keep:].any()
        c.read(storage[site:site + 1], torch.tensor(index, dtype=torch.int32, device=GPU), ka[:1], vb[:1], kv, dim, P)
        assert torch.equal(a[site], ka[0]) and torch.equal(b[site], vb[0])


@pytest.mark.parametrize("n,keep,recent", [(40000, 3000, 100), (40000, 39000, 0), (16385, 16384, 16000), (16384, 1, 0), (33000, 20000, 20000)])
@pytest.mark.parametrize("kind", ["spread", "ties", "alike", "narrow", "special"])
def test_which_keys_stay_of_long_rows(n, keep, recent, kind):
    """Rows past what a block holds in registers; sums that are all alike, differ in a few last bits, or are no numbers."""
    c, g = cache4(), torch.Generator().manual_seed(n + keep)
    w = torch.exp(4 * torch.randn(2, n, generator=g))
    if kind == "ties":
        w = (torch.rand(2, n, generator=g) * 5).round()
    elif kind == "alike":
        w = torch.full((2, n), 3.0)
    elif kind == "narrow":
        w = (torch.full((2, n), 1.0).view(torch.int32) + torch.randint(0, 5, (2, n), generator=g, dtype=torch.int32)).view(torch.float32)
    elif kind == "special":
        w = torch.tensor([math.nan, math.inf, -math.inf, 0.0, -0.0, 1e-45, -1.0, 3e38])[torch.randint(0, 8, (2, n), generator=g)]
    P, dim = 16, 32
    pages = -(-n // P) + -(-keep // P)
    storage = torch.zeros(1, pages, 2, c.record_bytes(dim, P), dtype=torch.uint8, device=GPU)
    sums = [w[None].clone().to(GPU)]
    tables = torch.arange(-(-n // P), device=GPU, dtype=torch.int32)[None]
    new_tables = torch.arange(-(-n // P), pages, device=GPU, dtype=torch.int32)[None]
    kept = torch.empty(1, 1, 2, keep, dtype=torch.int32, device=GPU)
    zero = torch.zeros(1, dtype=torch.int32, device=GPU)
    c.evict(storage, sums, tables, new_tables, zero + n, zero, zero, 2, dim, P, keep, recent, kept)
    for h in range(2):
        index = plain.stays(w[h].tolist(), n, keep, recent)
        assert kept[0, 0, h].tolist() == index
        want = torch.zeros(n)
        want[:keep] = w[h, index]
        assert torch.equal(torch.nan_to_num(sums[0][0, h].cpu(), nan=-5.0), torch.nan_to_num(want, nan=-5.0))
