"""The cache in 4 bits on the host: how a step is cut into tasks and pieces, what the manager keeps, refusals."""
import random

import numpy as np
import pytest
import torch

import plain_cache4 as plain
from runtime.cache import CacheManager, FourBitNeed, KVNeed, OutOfPages
from runtime.cache.manager import pages_that_fit
from runtime.kernels import cache4
from runtime.kernels.ops import KernelError


def test_the_plain_forms_of_the_format_agree():
    g = torch.Generator().manual_seed(0)
    x = torch.randn(3, 2, 40, generator=g) * torch.exp(3 * torch.randn(3, 2, 1, generator=g))
    x[0, 0, :8] = torch.tensor([7.0, 0.25, 0.75, 1.25, -1.75, 2.5, -3.5, 5.0])
    for a, b in zip(plain.held(x), plain.quick_held(x)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("seed", range(30))
def test_tasks_cover_every_row_and_key_once(seed):
    rng = random.Random(seed)
    S = rng.randint(1, 9)
    counts = [rng.choice([1, 1, rng.randint(1, 300)]) for _ in range(S)]
    cached = [rng.choice([0, rng.randint(0, 40), rng.randint(0, 5000)]) for _ in range(S)]
    window = rng.choice([0, 0, 1, 33, 700])
    per_task, pieces = rng.choice([1, 4, 5, 32]), rng.choice([1, 7, 64, 500])
    rows = sum(counts)
    tasks, merges = (np.empty((n, k), dtype=np.int32) for n, k in zip(cache4.most_tasks(rows, S, per_task, pieces), (8, 4)))
    n, m = cache4.fill_pieces(tasks, merges, counts, cached, per_task, pieces, window)
    assert (tasks[n:] == -1).all() and (merges[m:] == -1).all()
    seen, parts, firsts = {}, {}, np.cumsum([0] + counts)
    for seg, row0, count, sees, begin, stop, piece, _ in tasks[:n].tolist():
        assert 0 <= seg < S and firsts[seg] <= row0 and row0 + count <= firsts[seg + 1] and 0 < count <= per_task and begin < stop
        assert sees == cached[seg] + (row0 - firsts[seg]) + 1
        seen.setdefault(row0, []).append((begin, stop, piece))
        assert piece not in parts or piece == -1
        parts[piece] = row0
    covered = sorted((row0, next(t[2] for t in tasks[:n].tolist() if t[1] == row0)) for row0 in seen)
    assert [r for r, c in covered for r in range(r, r + c)] == list(range(rows))
    split = {m[0]: m for m in merges[:m].tolist()}
    for row0, spans in seen.items():
        seg, count, sees = next((t[0], t[2], t[3]) for t in tasks[:n].tolist() if t[1] == row0)
        first = max(0, sees - window) // 32 if window else 0
        spans.sort()
        assert spans[0][0] == first and spans[-1][1] == -(-(sees + count - 1) // 32)
        assert all(a[1] == b[0] for a, b in zip(spans, spans[1:]))
        if len(spans) == 1:
            assert spans[0][2] == -1 and row0 not in split
        else:
            assert split[row0][1] == count and [s[2] for s in spans] == list(range(split[row0][2], split[row0][2] + split[row0][3]))
    assert sorted(p for p in parts if p >= 0) == list(range(len([p for p in parts if p >= 0])))


@pytest.mark.parametrize("counts,cached,kw", [([], [], {}), ([1], [0, 1], {}), ([0], [3], {}), ([1], [-1], {}), ([1, 1], [0, 0], {"state_slots": [3, 3]}),
                                              ([1], [0], {"state_slots": [-1]}), ([1], [0], {"window": -4}), ([1.5], [0], {}), ([1], [0], {"dtype": torch.float16}),
                                              ([1], [0], {"heads": 5, "kv": 2}), ([1], [0], {"dim": 258}), ([1], [0], {"dim": 33}), ([1], [0], {"dim": 0})])
def test_plans_refuse(counts, cached, kw):
    heads, kv, dim = kw.pop("heads", 4), kw.pop("kv", 2), kw.pop("dim", 64)
    with pytest.raises((KernelError, TypeError)):
        cache4.plan(counts, cached, heads, kv, dim, device="cpu", **kw)


def test_entry_points_refuse():
    """Everything that is wrong with a call is found before a launch, also where there is no GPU."""
    def z(*shape, dtype=torch.float32):
        return torch.zeros(*shape, dtype=dtype)
    pages = z(3, 2, cache4.record_bytes(64, 16), dtype=torch.uint8)
    i = lambda *s: z(*s, dtype=torch.int32)                        # noqa: E731
    write = (z(5, 8 * 64), i(5), i(5), z(9, 32), z(9, 32), pages, z(5, 4 * 64), 4, 2, 64, 16)
    read = (pages[None], i(5), z(1, 5, 2, 64, dtype=torch.bfloat16), z(1, 5, 2, 64, dtype=torch.bfloat16), 2, 64, 16)
    plan = cache4.plan([1, 4], [0, 20], 4, 2, 64, device="cpu", state_slots=[0, 1], dtype=torch.float32)
    attention = (z(5, 4 * 64), pages, i(2, 3), plan, z(5, 4 * 64), 4, 2, 64, 16, 0.1)
    add = (z(5, 4 * 64), z(5, 4), pages, i(2, 3), plan, z(2, 2, 40), 4, 2, 64, 16, 0.1)
    evict = (pages[None], [z(2, 2, 40)], i(1, 2), i(1, 1), i(1), i(1), i(1), 2, 64, 16, 8, 2, i(1, 1, 2, 8))
    for call, args in ((cache4.rope_write, write), (cache4.read, read), (cache4.attention, attention), (cache4.add_weights, add), (cache4.evict, evict)):
        with pytest.raises(KernelError, match="GPU"):              # (tensors of the host)
            call(*args)
    for call, args, at, wrong in [(cache4.rope_write, write, 9, 63), (cache4.rope_write, write, 10, 12), (cache4.rope_write, write, 10, 4), (cache4.rope_write, write, 7, 5),
                                  (cache4.read, read, 5, 300), (cache4.attention, attention, 8, 0), (cache4.evict, evict, 10, 0), (cache4.evict, evict, 11, 9)]:
        with pytest.raises(KernelError):
            call(*[wrong if k == at else a for k, a in enumerate(args)])


def bounded(pages=40, keep=16, slack=6, **kw):
    return CacheManager({0: FourBitNeed(2, 16, None, keep, slack), 1: FourBitNeed(2, 16, None, keep, slack)}, pages, 4, 8, **kw)


def test_a_request_gives_up_keys():
    m = bounded()
    m.create("a")
    m.append_many([("a", 22)])
    assert not m.overfull("a") and m.cached("a") == 22
    (d,) = m.append_many([("a", 1)])
    assert d.start == 22 and d.dropped == 0 and m.overfull("a")
    ((old, new),) = m.give_up("a")
    assert len(old) == 6 and len(new) == 4 and not set(old) & set(new) and m.table(0, "a") == new
    assert m.length("a") == 23 and m.cached("a") == 16 and not m.overfull("a")
    m.check()
    (d,) = m.append_many([("a", 1)])
    assert d.start == 23 and d.dropped == 7 and d.slots[0] == [m.table(0, "a")[4] * 4]
    (d,) = m.append_many([("a", 40)], commit=False)
    assert d.slots[0][0] == m.table(0, "a")[4] * 4 + 1 and len(m.table(0, "a")) == 15
    m.abandon([d])
    assert len(m.table(0, "a")) == 5
    m.check()
    m.release("a")
    m.create("a")
    assert m.cached("a") == 0 and m.free_pages() == [40]


def test_forks_after_keys_were_given_up():
    m = bounded()
    m.create("a")
    m.append_many([("a", 30)])
    m.give_up("a")
    m.append_many([("a", 1)])
    m.fork("a", "b")
    assert m.cached("b") == 17 and m.length("b") == 31
    m.append_many([("a", 1), ("b", 1)])
    assert m.table(0, "a")[4] != m.table(0, "b")[4] and m.table(0, "a")[:4] == m.table(0, "b")[:4]
    m.append_many([("b", 8)])
    shared = list(m.table(0, "a"))
    m.give_up("b")
    assert m.table(0, "a") == shared and not set(m.table(0, "b")) & set(shared)
    m.check()


@pytest.mark.parametrize("seed", range(10))
def test_random_orders_lose_no_page(seed):
    rng = random.Random(seed)
    m, live = bounded(pages=30), []
    for step in range(300):
        what = rng.random()
        if what < 0.1 and len(live) < 5:
            m.create(step)
            live.append(step)
        elif what < 0.17 and live and len(live) < 5:
            m.fork(rng.choice(live), step)
            live.append(step)
        elif what < 0.22 and live:
            m.release(live.pop(rng.randrange(len(live))))
        elif live:
            items = [(r, rng.choice([1, 1, rng.randint(1, 12)])) for r in rng.sample(live, rng.randint(1, len(live)))]
            one_each = rng.random() < 0.5
            try:
                m.append_many([(r, 1 if one_each else n) for r, n in items])
            except OutOfPages:
                pass
            for r, _ in items:
                if m.overfull(r):
                    before = (m.cached(r), list(m.table(0, r)))
                    try:
                        m.give_up(r)
                        assert m.cached(r) == 16
                    except OutOfPages:
                        assert (m.cached(r), m.table(0, r)) == before
        m.check()


def test_the_manager_keeps_one_bound_and_promises_what_is_left():
    with pytest.raises(ValueError, match="bound"):
        CacheManager({0: FourBitNeed(2, 16, None, 16, 4), 1: FourBitNeed(2, 16, None, 0, 0)}, 8, 4, 2)
    with pytest.raises(ValueError, match="windows"):
        CacheManager({0: FourBitNeed(2, 16, 8, 16, 4)}, 8, 4, 2)
    m = bounded(pages=40)
    assert m.capacity() == [36] and m.most_pages_held(1000, 8) == [8] and m.most_pages_held(5, 8) == [2]
    free = CacheManager({0: FourBitNeed(2, 16)}, 40, 4, 2)
    assert free.capacity() == [40] and free.most_pages_held(1000, 8) == [250]


def test_a_page_of_4_bits_takes_little():
    need = FourBitNeed(8, 128)
    assert need.storage_shape(3, 10, 16) == (3, 10, 8, cache4.record_bytes(128, 16)) and cache4.record_bytes(128, 16) == 16 * 136
    wide = pages_that_fit({0: KVNeed(8, 128)}, 16, 2, 1 << 30)
    assert 3.7 < pages_that_fit({0: need}, 16, 2, 1 << 30) / wide < 3.8


def test_models_that_cannot_hold_their_cache_in_4_bits_say_so():
    from runtime.config import preset
    from runtime.engine.loading import build_from_config_dict
    for name in ("novosun-tiny", "ditazen-tiny", "noresun-tiny", "guduzen-tiny"):
        model = build_from_config_dict(preset(name))[2]
        with pytest.raises(ValueError, match="4 bits|type only"):
            model.hold_cache(4)
    model = build_from_config_dict(preset("tiny-a"))[2]
    for wrong in (dict(bits=8), dict(keep=-1), dict(keep=8, recent=9), dict(keep=8, portion=0), dict(keep=8, slack=0)):
        with pytest.raises(ValueError):
            model.hold_cache(**wrong)
    assert model.kept_keys is None
    model.hold_cache(4, keep=8)
    assert model.kept_keys == (8, 2, 2048) and model.state_needs()[0].shape == (2, 8 + 64 + 2048)
