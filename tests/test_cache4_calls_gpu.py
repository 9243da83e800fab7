"""The kernels of the cache held in 4 bits, called as a program may call them: in a captured graph, on other streams, with pages that are none,
with rows that are no numbers, at the ends of the sizes, past 32 bits; and calls that are refused."""
import dataclasses
import math

import pytest
import torch

import plain_cache4 as plain
from test_cache4_gpu import GPU, HALF, TYPES, a_step, cache4, check_step, forced, slots_of

pytestmark = pytest.mark.gpu


class Run:
    """A step as it is used: rows written, attention with the sums of its weights, keys given up, what is left read back."""

    def __init__(self, seed=0):
        c, g = cache4(), torch.Generator().manual_seed(seed)
        self.heads, self.kv, self.dim, self.P, self.keep, self.recent = 6, 2, 64, 16, 40, 8
        counts, cached = [5, 1, 70], [60, 100, 0]
        lengths = [a + b for a, b in zip(counts, cached)]
        need, fresh = [-(-n // self.P) for n in lengths], -(-self.keep // self.P)
        n_pages = sum(need) + 3 * fresh
        order = torch.randperm(n_pages, generator=g).tolist()
        tables = torch.full((3, max(need)), -1, dtype=torch.int32)
        slots, positions, rows = [], [], sum(counts)
        for r in range(3):
            own = [order.pop() for _ in range(need[r])]
            tables[r, :need[r]] = torch.tensor(own, dtype=torch.int32)
            slots += slots_of(own, lengths[r], self.P)[cached[r]:]
            positions += list(range(cached[r], lengths[r]))
        new_tables = torch.tensor([[order.pop() for _ in range(fresh)] for _ in range(3)], dtype=torch.int32)
        storage = torch.randint(0, 256, (1, n_pages, self.kv, c.record_bytes(self.dim, self.P)), generator=g, dtype=torch.int32).to(torch.uint8)
        storage[..., self.P * self.dim:] = torch.randint(120, 128, storage[..., self.P * self.dim:].shape, generator=g, dtype=torch.int32).to(torch.uint8)
        angle = torch.arange(200).double()[:, None] * 1e4 ** (-torch.arange(self.dim // 2).double() / (self.dim // 2))
        whole = lambda x: torch.tensor(x, dtype=torch.int32, device=GPU)          # noqa: E731
        self.tables, self.new_tables, self.first, self.sums_first = tables.to(GPU), new_tables.to(GPU), storage.to(GPU), torch.rand(1, 5, self.kv, 120, generator=g).to(GPU)
        self.positions, self.slots, self.lengths, self.old, self.new = whole(positions), whole(slots), whole(lengths), whole([2, 0, 1]), whole([2, 4, 3])
        self.cos, self.sin = angle.cos().float().to(GPU), angle.sin().float().to(GPU)
        self.place = whole([s for r in range(3) for s in slots_of(new_tables[r].tolist(), self.keep, self.P)])
        self.plan = c.plan(counts, cached, self.heads, self.kv, self.dim, state_slots=[2, 0, 1])
        self.storage, self.sums = self.first.clone(), self.sums_first.clone()
        empty = lambda *s, dtype=torch.bfloat16: torch.zeros(*s, dtype=dtype, device=GPU)      # noqa: E731
        self.qkv = empty(rows, (self.heads + 2 * self.kv) * self.dim)
        self.q, self.out, self.stats = empty(rows, self.heads * self.dim), empty(rows, self.heads * self.dim), empty(rows, self.heads, dtype=torch.float32)
        self.kept = empty(1, 3, self.kv, self.keep, dtype=torch.int32)
        self.keys, self.values = (empty(1, 3 * self.keep, self.kv, self.dim) for _ in range(2))

    def fresh(self, seed):
        self.qkv.copy_(torch.randn(self.qkv.shape, generator=torch.Generator().manual_seed(seed)))
        self.storage.copy_(self.first)
        self.sums.copy_(self.sums_first)

    def __call__(self):
        c, s = cache4(), self
        c.rope_write(s.qkv, s.positions, s.slots, s.cos, s.sin, s.storage[0], s.q, s.heads, s.kv, s.dim, s.P)
        c.attention(s.q, s.storage[0], s.tables, s.plan, s.out, s.heads, s.kv, s.dim, s.P, 0.125, stats=s.stats)
        c.add_weights(s.q, s.stats, s.storage[0], s.tables, s.plan, s.sums[0], s.heads, s.kv, s.dim, s.P, 0.125)
        c.evict(s.storage, [s.sums[0]], s.tables, s.new_tables, s.lengths, s.old, s.new, s.kv, s.dim, s.P, s.keep, s.recent, s.kept)
        c.read(s.storage, s.place, s.keys, s.values, s.kv, s.dim, s.P)

    def got(self):
        return {n: getattr(self, n).clone() for n in ("q", "out", "stats", "sums", "kept", "storage", "keys", "values")}


def same(a, b):
    for name in a:
        assert torch.equal(a[name], b[name]), name


def eager(seed, step):
    run = Run(seed)
    run.fresh(step)
    run()
    return run.got()


def test_a_run_against_64_bits():
    """What a step leaves: the kept keys are those with the largest sums that its own attention weights make, and hold what was written."""
    run = Run(1)
    run.fresh(5)
    run()
    got = {n: t.cpu() for n, t in run.got().items()}
    x = run.qkv.cpu().float().view(76, 10, 64)
    first = 0
    for r, (n, cached, slot, new) in enumerate([(5, 60, 2, 2), (1, 100, 0, 4), (70, 0, 1, 3)]):
        length = n + cached
        keys, values = (torch.empty(1, length, 2, 64, dtype=torch.bfloat16, device=GPU) for _ in range(2))
        own = torch.tensor(slots_of(run.tables[r].tolist(), length, 16), dtype=torch.int32, device=GPU)
        cache4().read(run.storage, own, keys, values, 2, 64, 16)     # (the pages of the old table are as they were before keys were given up)
        k, v = keys[0].cpu().double().transpose(0, 1), values[0].cpu().double().transpose(0, 1)
        assert torch.equal(v[:, cached:].transpose(0, 1), plain.quick_held(x[first:first + n, 8:])[2])
        q = got["q"][first:first + n].double().view(n, 6, 64)
        want, weighed, w, _ = plain.attention(q, k, v, cached, 0.125)
        # (as for every step: twice a score's error, the exponentials', the weights' half steps, the sum over keys in 32 bits, the result's rounding)
        off = 2 * plain.score_error(q, k, 0.125) + 2.0 ** -21 + (length + 32) * 2.0 ** -24
        assert ((got["out"][first:first + n].double().view(n, 6, 64) - want).abs() <= 1.01 * (weighed * (off + 2.0 ** -8) + want.abs() * 2.0 ** -8)).all()
        sums = run.sums_first[0, slot].cpu().double()
        sums[:, :length] += w.view(2, 3, n, -1).sum((1, 2))
        room = sums * (off + (3 * n + 16) * 2.0 ** -24) * 1.01
        for h in range(2):
            index = got["kept"][0, r, h]
            index = index[index >= 0].long()
            assert len(index) == 40 and (index[1:] > index[:-1]).all() and index[-8:].tolist() == list(range(length - 8, length))
            out = torch.ones(length - 8, dtype=torch.bool)
            out[index[:-8]] = False
            out = out.nonzero()[:, 0]
            assert (sums[h, index[:-8]] + room[h, index[:-8]]).min() >= (sums[h, out] - room[h, out]).max()
            assert ((got["sums"][0, new, h, :40].double() - sums[h, index]).abs() <= room[h, index]).all() and not got["sums"][0, new, h, 40:].any()
            at = torch.arange(40 * r, 40 * r + 40)
            assert torch.equal(got["keys"][0, at, h].double(), k[h, index]) and torch.equal(got["values"][0, at, h].double(), v[h, index])
        first += n


def test_a_captured_run_is_the_eager_one():
    run = Run(2)
    run.fresh(0)
    run()                                                          # (libraries are loaded before the capture)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    for step in (3, 4, 3, 5):
        run.fresh(step)
        graph.replay()
        torch.cuda.synchronize()
        same(run.got(), eager(2, step))


def test_two_graphs_with_plans_of_their_own():
    """Replayed at the same time on two streams."""
    runs = [Run(6), Run(7)]
    graphs, streams = [], [torch.cuda.Stream() for _ in runs]
    for run in runs:
        run.fresh(1)
        run()
        torch.cuda.synchronize()
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            run()
    for step in (1, 2, 3):
        for run in runs:
            run.fresh(step)
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for seed, run in zip((6, 7), runs):
            same(run.got(), eager(seed, step))


def test_another_stream_than_the_default():
    run, stream = Run(8), torch.cuda.Stream()
    run.fresh(2)
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        run()
    torch.cuda.current_stream().wait_stream(stream)
    same(run.got(), eager(8, 2))


def test_streams_at_the_same_time():
    counts, cached = [1] * 8, [700, 3, 0, 2000, 90, 1500, 31, 400]
    steps = []
    for seed in range(3):
        q, pages, tables, _, _ = a_step(counts, cached, 8, 2, 64, 16, "bf16", seed)
        plan = cache4().plan(counts, cached, 8, 2, 64, state_slots=list(range(8)))
        assert plan.merges is not None                             # (keys in pieces: the workspace is used)
        steps.append((q.to(GPU), pages.to(GPU), tables.to(GPU), plan, torch.cuda.Stream()))

    def go(s):
        q, pages, tables, plan, _ = s
        out, stats, sums = torch.empty_like(q), torch.empty(8, 8, device=GPU), torch.zeros(8, 2, 2001, device=GPU)
        for _ in range(10):
            cache4().attention(q, pages, tables, plan, out, 8, 2, 64, 16, 0.1, stats=stats)
            cache4().add_weights(q, stats, pages, tables, plan, sums, 8, 2, 64, 16, 0.1)
        return out, stats, sums
    alone = []
    for s in steps:
        alone.append(go(s))
        torch.cuda.synchronize()
    together = []
    for s in steps:
        with torch.cuda.stream(s[4]):
            together.append(go(s))
    torch.cuda.synchronize()
    for a, b in zip(alone, together):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("form,pieces,kind", [(0, 1, "bf16"), (0, 9, "bf16"), (0, 9, "f32"), (1, 1, "bf16"), (1, 9, "bf16"), (2, 1, "bf16"), (2, 9, "bf16")])
@pytest.mark.parametrize("P", [8, 16, 64])
def test_pages_that_are_none(form, pieces, kind, P, monkeypatch):
    """Keys in them are not seen, wherever they lie; a row that sees no key gets zeros, -inf and adds nothing."""
    monkeypatch.setattr(cache4(), "LEAST_PIECE", 2)
    c, heads, kv, dim, scale = cache4(), 6, 2, 64, 0.2
    counts, cached = [40, 1, 3, 130], [90, 200, 20, 10]
    q, pages, tables, keys, values = a_step(counts, cached, heads, kv, dim, P, kind, seed=P)
    none = [-1, len(pages), 2 ** 31 - 1, -2 ** 31]
    for s, gone in enumerate([[0], [1, 2], range(tables.shape[1]), [1]]):
        for i, page in enumerate(gone):
            if page < tables.shape[1]:
                tables[s, page] = none[(i + s) % 4]
    plan = forced(c, c.plan(counts, cached, heads, kv, dim, dtype=TYPES[kind]), counts, cached, form, pieces, 0)
    summed = c.plan(counts, cached, heads, kv, dim, dtype=TYPES[kind], state_slots=[0, 1, 2, 3])
    gq, gp, gt = q.to(GPU), pages.to(GPU), tables.to(GPU)
    out, stats = torch.full_like(gq, math.nan), torch.full((len(q), heads), math.nan, device=GPU)
    c.attention(gq, gp, gt, plan, out, heads, kv, dim, P, scale, stats=stats)
    sums = torch.zeros(4, kv, 220, device=GPU)
    c.add_weights(gq, stats, gp, gt, summed, sums, heads, kv, dim, P, scale)
    out, stats, sums, first = out.cpu().double().view(-1, heads, dim), stats.cpu(), sums.cpu().double(), 0
    for s, n in enumerate(counts):
        total = n + cached[s]
        held = torch.tensor([0 <= int(tables[s, t // P]) < len(pages) for t in range(total)])
        rows = q[first:first + n].double().view(n, heads, dim)
        seen = held[None] & (torch.arange(total)[None] <= torch.arange(n)[:, None] + cached[s])
        k, v = keys[s].repeat_interleave(3, 0), values[s].repeat_interleave(3, 0)
        score = (torch.matmul(rows.transpose(0, 1), k.transpose(1, 2)) * scale).masked_fill(~seen, -math.inf)
        lse = torch.logsumexp(score, -1)
        w = torch.where(seen.any(-1)[None, :, None], torch.exp(score - lse[..., None]), torch.zeros(()).double())
        want, weighed = torch.matmul(w, v).transpose(0, 1), torch.matmul(w, v.abs()).transpose(0, 1)
        # (as for every step: twice a score's error, the exponentials', the weights' half steps, the sum over keys in 32 bits, the result's rounding)
        off = 2 * plain.score_error(rows, keys[s], scale) + 2.0 ** -21 + (total + 32) * 2.0 ** -24
        room = weighed * (off + (HALF[TYPES[kind]] if kind == "bf16" else 2.0 ** -23)) + want.abs() * HALF[TYPES[kind]]
        assert ((out[first:first + n] - want).abs() <= 1.01 * room).all(), s
        empty = ~seen.any(-1)
        assert (stats[first:first + n][empty] == -math.inf).all() and stats[first:first + n][~empty].isfinite().all()
        part = w.view(kv, 3, n, total).sum((1, 2))
        assert ((sums[s, :, :total] - part).abs() <= 1.01 * part * (off + (3 * n + 16) * 2.0 ** -24 + 2.0 ** -23)).all() and not sums[s, :, total:].any()
        first += n


@pytest.mark.parametrize("form", [0, 1, 2])
def test_rows_that_are_no_numbers_stay_alone(form):
    """What a block's other rows get is what they get beside numbers, to a step's bounds (a block's rows raise their maxima together)."""
    counts, cached, heads, kv, dim = [60, 1, 9], [30, 100, 0], 4, 2, 128
    c = cache4()
    q, pages, tables, keys, values = a_step(counts, cached, heads, kv, dim, 16, "bf16")
    plan = forced(c, c.plan(counts, cached, heads, kv, dim), counts, cached, form, 1, 0)
    x = q.clone().view(-1, heads, dim)
    x[7, 1], x[20, 3, 5], x[60, 0, 100], x[65, 2] = math.nan, math.inf, -math.inf, math.nan
    clean = torch.ones(len(q), heads, dtype=torch.bool)
    clean[7, 1] = clean[20, 3] = clean[60, 0] = clean[65, 2] = False
    out, stats = torch.empty(len(q), heads * dim, dtype=torch.bfloat16, device=GPU), torch.empty(len(q), heads, device=GPU)
    c.attention(x.view(len(q), -1).to(GPU), pages.to(GPU), tables.to(GPU), plan, out, heads, kv, dim, 16, 0.1, stats=stats)
    out, first = out.cpu().double().view(-1, heads, dim), 0
    for s, n in enumerate(counts):
        rows = q[first:first + n].double().view(n, heads, dim)
        want, weighed, _, _ = plain.attention(rows, keys[s], values[s], cached[s], 0.1)
        # (as for every step: twice a score's error, the exponentials', the weights' half steps, the sum over keys in 32 bits, the result's rounding)
        off = 2 * plain.score_error(rows, keys[s], 0.1) + 2.0 ** -21 + (n + cached[s] + 32) * 2.0 ** -24
        good = clean[first:first + n]
        assert ((out[first:first + n] - want).abs() <= 1.01 * (weighed * (off + 2.0 ** -8) + want.abs() * 2.0 ** -8))[good].all(), s
        first += n
    assert out[7, 1].isnan().all() and out[65, 2].isnan().all() and stats.cpu()[clean].isfinite().all()


def test_rows_behind_the_last_segment_are_left_as_they_were():
    counts, cached = [20, 1], [5, 90]
    c = cache4()
    q, pages, tables, _, _ = a_step(counts, cached, 9, 3, 64, 16, "bf16")
    plan = c.plan(counts, cached, 9, 3, 64, state_slots=[0, 1])
    padded = dataclasses.replace(plan, rows=24, room=None)
    gp, gt = pages.to(GPU), tables.to(GPU)
    more = torch.cat([q, torch.full((3, 9 * 64), math.nan, dtype=q.dtype)]).to(GPU)
    out, stats, sums = torch.full_like(more, 7.0), torch.full((24, 9), 7.0, device=GPU), torch.zeros(2, 3, 91, device=GPU)
    c.attention(more, gp, gt, padded, out, 9, 3, 64, 16, 0.1, stats=stats)
    c.add_weights(more, stats, gp, gt, padded, sums, 9, 3, 64, 16, 0.1)
    want, ws, wsums = torch.empty_like(out[:21]), torch.empty(21, 9, device=GPU), torch.zeros(2, 3, 91, device=GPU)
    c.attention(q.to(GPU), gp, gt, plan, want, 9, 3, 64, 16, 0.1, stats=ws)
    c.add_weights(q.to(GPU), ws, gp, gt, plan, wsums, 9, 3, 64, 16, 0.1)
    assert torch.equal(out[:21], want) and torch.equal(stats[:21], ws) and torch.equal(sums, wsums)
    assert (out[21:] == 7).all() and (stats[21:] == 7).all()


@pytest.mark.parametrize("heads,kv,dim,P,kind", [(1, 1, 2, 8, "bf16"), (3, 1, 34, 16, "f32"), (2, 2, 66, 8, "bf16"), (2, 1, 130, 64, "bf16"), (4, 2, 254, 8, "f32"), (300, 1, 32, 16, "bf16"),
                                                 (2, 1, 64, 4096, "bf16"), (130, 130, 8, 8, "bf16")])
def test_the_ends_of_the_sizes(heads, kv, dim, P, kind):
    check_step([1, 1], [0, 77], heads, kv, dim, P, kind, weights=True)
    check_step([19, 1], [3, 40], heads, kv, dim, P, kind, weights=True)


def test_many_requests_of_few_keys():
    check_step([1] * 400, [i % 9 for i in range(400)], 4, 2, 64, 8, "bf16", weights=True)


def test_pools_past_32_bits():
    """Five gigabytes of pages: the last of them take part in every call as the first do in a small pool."""
    c, g = cache4(), torch.Generator().manual_seed(0)
    heads, kv, dim, P, rows = 4, 2, 256, 8, 21
    record = c.record_bytes(dim, P)
    n = (5 << 30) // (kv * record)
    small, large = torch.zeros(1, 9, kv, record, dtype=torch.uint8, device=GPU), torch.zeros(1, n, kv, record, dtype=torch.uint8, device=GPU)
    assert large.numel() > 1 << 32
    tables = torch.tensor([[4, 0, 2]], dtype=torch.int32)
    qkv = torch.randn(rows, (heads + 2 * kv) * dim, generator=g).to(torch.bfloat16).to(GPU)
    positions = torch.arange(rows, dtype=torch.int32, device=GPU)
    cos, sin = torch.rand(2, 40, dim // 2, generator=g).to(GPU)
    got = []
    for pool, shift in ((small, 0), (large, n - 9)):
        own = tables + shift
        slots = torch.tensor(slots_of(own[0].tolist(), rows, P), dtype=torch.int32, device=GPU)
        q = torch.empty(rows, heads * dim, dtype=torch.bfloat16, device=GPU)
        c.rope_write(qkv, positions, slots, cos, sin, pool[0], q, heads, kv, dim, P)
        results = [q]
        for counts, cached in (([rows], [0]), ([1], [rows - 1])):
            part = q[rows - counts[0]:].contiguous()
            out, stats, sums = torch.empty_like(part), torch.empty(counts[0], heads, device=GPU), torch.zeros(1, kv, rows, device=GPU)
            plan = c.plan(counts, cached, heads, kv, dim, state_slots=[0])
            c.attention(part, pool[0], own.to(GPU), plan, out, heads, kv, dim, P, 0.05, stats=stats)
            c.add_weights(part, stats, pool[0], own.to(GPU), plan, sums, heads, kv, dim, P, 0.05)
            results += [out, stats, sums]
        new = torch.tensor([[6, 8]], dtype=torch.int32) + shift
        zero, kept = torch.zeros(1, dtype=torch.int32, device=GPU), torch.empty(1, 1, kv, 12, dtype=torch.int32, device=GPU)
        c.evict(pool, [sums], own.to(GPU), new.to(GPU), zero + rows, zero, zero, kv, dim, P, 12, 4, kept)
        place = torch.tensor(slots_of(new[0].tolist(), 12, P), dtype=torch.int32, device=GPU)
        keys, values = (torch.empty(1, 12, kv, dim, dtype=torch.bfloat16, device=GPU) for _ in range(2))
        c.read(pool, place, keys, values, kv, dim, P)
        got.append(results + [kept, sums, keys, values])
    assert all(torch.equal(a, b) for a, b in zip(*got)) and got[0][-1].abs().max() > 0
    assert torch.equal(small[0], large[0, n - 9:]) and not large[0, :9].any()


def test_lengths_and_slots_out_of_range_when_keys_are_given_up():
    """More keys than the table or the sums have: those that there are.  Less than none, or sums that are nowhere: nothing happens to the request."""
    c, kv, dim, P, keep = cache4(), 2, 32, 8, 10
    storage = torch.randint(0, 128, (1, 20, kv, c.record_bytes(dim, P)), dtype=torch.int32).to(torch.uint8).to(GPU)
    sums = torch.rand(6, kv, 30, generator=torch.Generator().manual_seed(1)).to(GPU)
    tables = torch.tensor([[0, 1, 2, 3], [4, 5, 6, 7], [8, 9, 10, 11], [0, 1, 2, 3], [4, 5, 6, 7]], dtype=torch.int32, device=GPU)
    new_tables = torch.tensor([[12, 13], [14, 15], [16, 17], [18, 19], [-1, 99]], dtype=torch.int32, device=GPU)
    lengths = torch.tensor([2 ** 31 - 1, -5, 20, 20, 20], dtype=torch.int32, device=GPU)
    slots = torch.tensor([0, 1, 6, -1, 4], dtype=torch.int32, device=GPU)
    new_slots = torch.tensor([0, 1, 2, 3, 4], dtype=torch.int32, device=GPU)
    before, pool = sums.cpu(), storage.cpu()
    kept = torch.full((1, 5, kv, keep), 7, dtype=torch.int32, device=GPU)
    c.evict(storage, [sums], tables, new_tables, lengths, slots, new_slots, kv, dim, P, keep, 3, kept)
    kept, after, left = kept.cpu(), sums.cpu(), storage.cpu()
    for h in range(kv):
        assert kept[0, 0, h].tolist() == plain.stays(before[0, h].tolist(), 30, keep, 3)
        assert kept[0, 4, h].tolist() == plain.stays(before[4, h].tolist(), 20, keep, 3)
    assert (kept[0, 1:4] == -1).all()
    assert torch.equal(after[[1, 2, 3, 5]], before[[1, 2, 3, 5]])
    assert torch.equal(left[0, :12], pool[0, :12]) and torch.equal(left[0, 14:], pool[0, 14:])


def test_calls_that_are_refused():
    """Before anything is launched: nothing that the call was given changes."""
    from runtime.kernels.ops import KernelError
    run = Run(9)
    run.fresh(1)
    c, s = cache4(), run
    other = c.plan([76], [0], 6, 2, 64, state_slots=[0])
    unnamed = c.plan([5, 1, 70], [60, 100, 0], 6, 2, 64)
    windowed = c.plan([5, 1, 70], [60, 100, 0], 6, 2, 64, window=50, state_slots=[2, 0, 1])
    wide = torch.empty(76, 2 * 6 * 64, dtype=torch.bfloat16, device=GPU)
    shifted = torch.empty(76 * 6 * 64 + 8, dtype=torch.bfloat16, device=GPU)[1:76 * 6 * 64 + 1].view(76, 6 * 64)
    calls = {
        "write": (c.rope_write, [s.qkv, s.positions, s.slots, s.cos, s.sin, s.storage[0], s.q, 6, 2, 64, 16]),
        "read": (c.read, [s.storage, s.place, s.keys, s.values, 2, 64, 16]),
        "attention": (c.attention, [s.q, s.storage[0], s.tables, s.plan, s.out, 6, 2, 64, 16, 0.125]),
        "sums": (c.add_weights, [s.q, s.stats, s.storage[0], s.tables, s.plan, s.sums[0], 6, 2, 64, 16, 0.125]),
        "evict": (c.evict, [s.storage, [s.sums[0]], s.tables, s.new_tables, s.lengths, s.old, s.new, 2, 64, 16, 40, 8, s.kept]),
    }
    wrong = [("write", 0, s.qkv.t()), ("write", 0, s.qkv.half()), ("write", 1, s.positions.long()), ("write", 2, s.slots[:-1]), ("write", 3, s.cos[:, :16]), ("write", 4, s.sin.double()),
             ("write", 5, s.storage[0, :, :1]), ("write", 5, s.storage[0].cpu()), ("write", 6, wide[:, ::2]), ("write", 6, s.q.float()), ("write", 7, 5), ("write", 10, 32),
             ("read", 1, s.place[::2]), ("read", 2, s.keys.float()), ("read", 3, s.values[:, 1:]), ("read", 0, s.storage[:, :0]),
             ("attention", 0, wide[:, :384]), ("attention", 0, shifted), ("attention", 0, s.q.float()), ("attention", 0, s.q[1:]), ("attention", 1, s.storage[0, :, :, 16:]), ("attention", 2, s.tables[:2]),
             ("attention", 2, s.tables.long()), ("attention", 3, None), ("attention", 3, windowed), ("attention", 4, s.out.float()), ("attention", 9, math.inf), ("attention", 9, math.nan), ("attention", 5, 2),
             ("sums", 1, s.stats[:, :5]), ("sums", 1, s.stats.half()), ("sums", 3, s.tables.t()), ("sums", 4, unnamed), ("sums", 4, windowed), ("sums", 5, s.sums[0, :2]), ("sums", 5, s.sums[0, :, :, :100]),
             ("sums", 5, s.sums[0, :, :1]), ("sums", 5, s.sums[0].double()),
             ("evict", 1, []), ("evict", 1, [s.sums[0], s.sums[0]]), ("evict", 1, [s.sums[0].double()]), ("evict", 1, [s.sums[0, :, :, ::2]]), ("evict", 1, [s.sums[0].cpu()]), ("evict", 2, s.tables[:2]),
             ("evict", 3, s.new_tables[:, :2]), ("evict", 4, s.lengths.long()), ("evict", 5, s.old[:2]), ("evict", 10, 121), ("evict", 11, 41), ("evict", 12, s.kept[..., :39])]
    before = run.got()
    for name, at, value in wrong:
        call, args = calls[name]
        with pytest.raises((KernelError, TypeError)):
            call(*[value if i == at else a for i, a in enumerate(args)])
    with pytest.raises(KernelError):
        c.attention(s.q[:1].contiguous(), s.storage[0], s.tables, other, s.out, 6, 2, 64, 16, 0.125)
    with pytest.raises(KernelError):
        c.attention(s.q, s.storage[0], s.tables, s.plan, s.out, 6, 2, 64, 16, 0.125, window=50)
    with pytest.raises(KernelError):
        c.attention(s.q, s.storage[0], s.tables, s.plan, s.out, 6, 2, 64, 16, 0.125, stats=s.stats[:, :5])
    same(run.got(), before)


def test_a_request_whose_keys_could_not_be_moved_is_only_released(folders, monkeypatch):
    from conftest import TINY, random_tokens
    from test_cache4_engine_gpu import make_runner
    from runtime.engine.runner import StepEntry
    from runtime.kernels.ops import KernelError
    runner = make_runner(folders["a"], "float32", keep=16, recent=4, slack=8, portion=16)
    tokens = random_tokens(4, 40, TINY["a"]["vocab_size"])

    def fails(*args):
        raise KernelError("no")
    runner.create("x")
    runner.step([StepEntry("x", tokens[:16], [])])
    with monkeypatch.context() as m:
        m.setattr(cache4(), "evict", fails)
        with pytest.raises(KernelError):
            runner.step([StepEntry("x", tokens[16:32], [15])])
    with pytest.raises(Exception, match="x"):
        runner.step([StepEntry("x", tokens[32:33], [0])])
    runner.cache.check()
    runner.release("x")
    runner.create("x")
    runner.step([StepEntry("x", tokens[:16], [])])
    assert runner.step([StepEntry("x", tokens[16:32], [15])]).isfinite().all() and runner.cache.cached("x") == 16


@pytest.mark.parametrize("execution", ["eager", "graph"])
def test_a_layer_that_reads_another_layers_keys_in_4_bits(execution):
    """Logits of a portion and of single tokens behind it against 64 bits over what the two caches hold."""
    import numpy as np
    import plain_llama as P
    from conftest import assert_close
    from test_cache4_engine_gpu import held
    from test_norm_hand_over_gpu import EPS, THETA, model_of
    from runtime.engine import ModelRunner, StepEntry
    heads, kv, order = 4, 2, [(0, None), (1, 0), (0, None), (2, None)]
    model, w, _ = model_of(128, heads, kv, 256, [{}, {"own_kv": False}, {}], order)
    model.bind({name: torch.from_numpy(t).float().to(GPU) for name, t in w.items()}, torch.float32, torch.device(GPU))
    model.hold_cache(4)
    runner = ModelRunner(model, n_pages=8, page_size=16, max_requests=1, execution=execution)
    tokens = np.random.default_rng(3).integers(0, 96, size=45)
    runner.create("x")
    got = [runner.step([StepEntry("x", list(tokens[:40]), list(range(40)))]).cpu().numpy()]
    got += [runner.step([StepEntry("x", [int(t)], [0])]).cpu().numpy() for t in tokens[40:]]
    sites = [site for site in range(len(order)) if site in runner.cache.group_of_site]
    caches = {site: held(runner, "x", site, 45) for site in sites}
    assert len(sites) == 3
    x, pos = w["embed.weight"][tokens], np.arange(45)
    for site, (layer, reads) in enumerate(order):
        n = f"l{layer}"
        q = P.rope(P.linear(P.rmsnorm(x, w[n + ".n1.weight"], EPS), w[n + ".attn.q_proj.weight"]).reshape(45, heads, 64), pos, THETA)
        k, v = caches[site if reads is None else reads]
        x = x + P.linear(P.causal_attention(q, k, v).reshape(45, heads * 64), w[n + ".attn.o_proj.weight"])
        h = P.rmsnorm(x, w[n + ".n2.weight"], EPS)
        x = x + P.linear(P.swiglu(P.linear(h, w[n + ".mlp.gate_proj.weight"]), P.linear(h, w[n + ".mlp.up_proj.weight"])), w[n + ".mlp.down_proj.weight"])
    assert_close(np.concatenate(got), P.linear(P.rmsnorm(x, w["final.weight"], EPS), w["head.weight"]), "float32", execution)
