"""The engine's host side of a bounded number of keys in the cache of 4 bits: what a step leaves for the next while keys are given up, and what
is refused, without a GPU."""
import types

import pytest
import torch

from runtime.config import preset
from runtime.engine.loading import build_from_config_dict


class Event:
    def record(self):
        pass

    def synchronize(self):
        pass


@pytest.fixture
def host_runner(monkeypatch):
    """Makes ModelRunners whose memory lies on the host and whose kernels do nothing: logits are zeros, evictions are listed."""
    from runtime.engine import runner as module
    moved = []
    for name in ("empty", "zeros"):
        make = getattr(torch, name)
        monkeypatch.setattr(torch, name, lambda *a, make=make, pin_memory=False, **kw: make(*a, **kw))
    monkeypatch.setattr(torch.cuda, "is_available", lambda: True)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: "stream")
    monkeypatch.setattr(torch.cuda, "Event", Event)
    monkeypatch.setattr(module.ops, "prepare", lambda units: None)
    monkeypatch.setattr(module.ops, "move_states", lambda storages, source, slot: None)
    monkeypatch.setattr(module.cache4, "evict", lambda *a: moved.append([t.clone() if isinstance(t, torch.Tensor) else t for t in a[2:7]]))

    def make(pages, page_size=16, max_requests=8, **hold):
        model = build_from_config_dict(preset("tiny-a"))[2]
        model.hold_cache(4, **hold)
        model._max_positions = 8192
        runner = module.ModelRunner(model, n_pages=pages, page_size=page_size, max_requests=max_requests, device="cpu")
        runner._forward = lambda ctx, take: torch.zeros(ctx.logit_rows.shape[0], model.vocab_size)
        return runner, moved
    return make


@pytest.mark.parametrize("requests", [1, 3, 4, 5, 8])
def test_a_steps_logit_slots_outlive_the_evictions_behind_it(host_runner, requests):
    """Requests that decode side by side pass their bound in one step.  Tokens are picked afterwards, at the slots that the step's metadata names."""
    from runtime.engine.runner import StepEntry
    runner, moved = host_runner(pages=4096, keep=2048, recent=64, slack=64, portion=2112)
    for r in range(requests):
        runner.create(r)
    runner.step([StepEntry(r, [1] * 2112, []) for r in range(requests)])
    assert not moved
    runner.step([StepEntry(r, [1], [0]) for r in range(requests)])
    assert len(moved) == requests and all(runner.cache.cached(r) == 2048 for r in range(requests))
    wanted, slots, where = runner._last_wanted
    assert wanted == list(range(requests)) and where.tolist() == slots == [runner.cache.slots.slot_of(r) for r in range(requests)]
    # and each eviction was told of its own request: keys held, slots, pages
    for r, (tables, new_tables, lengths, slots, new_slots) in enumerate(moved):
        assert lengths.tolist() == [2113] and slots.tolist() == new_slots.tolist() == [runner.cache.slots.slot_of(r)]
        assert new_tables[0].tolist() == runner.cache.table(0, r) and tables.shape == (1, 133)
    runner.cache.check()


def test_nothing_is_picked_from_a_step_whose_kept_keys_could_not_be_moved(host_runner, monkeypatch):
    """The step raises, nobody has its logits: those of an earlier step must not be taken for them."""
    from runtime.engine import runner as module
    from runtime.engine.runner import StepEntry
    runner, _ = host_runner(pages=64, keep=32, recent=8, slack=16, portion=64)
    runner.create("x")
    logits = runner.step([StepEntry("x", [1] * 40, [39])])

    def fails(*args):
        raise module.ops.KernelError("no")
    monkeypatch.setattr(module.cache4, "evict", fails)
    with pytest.raises(module.ops.KernelError):
        runner.step([StepEntry("x", [1] * 20, [19])])

    class Sampler:
        def pick(self, logits, params, out, index):
            raise AssertionError("picked")
    with pytest.raises(ValueError, match="not those of the last step"):
        runner.pick(Sampler(), logits, [(0.0, 0, 0)])


@pytest.fixture
def sized(monkeypatch):
    """Engine.from_folder on the host: the number of pages that its runner is made with, the memory free for them being `free` bytes."""
    from runtime.engine import loading, runner as module
    from runtime.engine.scheduler import Engine

    class Asked(Exception):
        pass

    def asked(model, n_pages, **kw):
        raise Asked(n_pages)

    def make(free, positions=8192, name="tiny-a", **kw):
        model = build_from_config_dict(preset(name))[2]
        model._max_positions = positions
        monkeypatch.setattr(loading, "load_model", lambda folder, dtype, device: model)
        monkeypatch.setattr(torch.cuda, "mem_get_info", lambda device: (free, free))
        monkeypatch.setattr(module, "ModelRunner", asked)
        with pytest.raises(Asked) as got:
            Engine.from_folder("", pages=0, **kw)
        return got.value.args[0], model
    return make


def test_a_pool_as_large_as_fits_is_no_larger_than_bounded_requests_can_use(sized):
    """Eight requests of 512 + 64 + 32 keys, and the pages that the kept keys of one move to; all their tokens where nothing bounds them."""
    most, bounded = 1 << 40, dict(cache_bits=4, keep_keys=512, prefill_chunk=32)
    assert sized(most, **bounded)[0] == 8 * 38 + 32
    assert sized(most, page_size=8, max_active=20, **bounded)[0] == 20 * 76 + 64
    assert sized(most, positions=300, **bounded)[0] == 8 * 19 + 32         # (requests that never reach the bound)
    assert sized(most, cache_bits=4, prefill_chunk=32)[0] == 8 * 512
    assert sized(most, prefill_chunk=32)[0] == 8 * 512
    assert sized(1 << 20, cache_bits=4, prefill_chunk=32)[0] < 8 * 512


def test_a_pool_as_large_as_fits_leaves_room_for_the_sums(sized):
    """The sums of attention weights take memory beside the pages: both together are four fifths of what is free."""
    free = 1 << 20
    pages, model = sized(free, cache_bits=4, keep_keys=512, prefill_chunk=32, max_active=32)
    sums = 32 * sum(4 * need.shape[0] * need.shape[1] for need in model.state_needs().values())
    page = sum(need.bytes_per_token(2) * 16 for need in model.cache_needs().values())
    assert sums > free // 4 and pages == int(0.8 * free - sums) // page > 100


def test_a_pool_that_the_kept_keys_fill_is_refused_by_name(host_runner):
    """The pages that one request's kept keys move to are set aside: where that is the whole pool, no request could ever run."""
    from runtime.engine.scheduler import Engine, Request
    for pages in (100, 128):
        with pytest.raises(ValueError, match=f"{pages} pages of 16.*2048 keys.*128"):
            Engine(host_runner(pages=pages, keep=2048, portion=8)[0])
    engine = Engine(host_runner(pages=129, keep=2048, portion=8)[0])
    engine.submit(Request("short", [1] * 10, 6))                          # (15 tokens in the one page left)
    with pytest.raises(ValueError, match="128 more are set aside"):
        engine.submit(Request("longer", [1] * 10, 8))
    Engine(host_runner(pages=1)[0]).submit(Request("all keys", [1] * 10, 6))


def test_the_documented_command_takes_requests_of_any_length(sized):
    """The README's command with a bounded number of keys: its pool holds a request at its bound, whatever the requests' lengths."""
    import shlex
    from conftest import ROOT
    from runtime.cache import CacheManager
    lines = [line for line in (ROOT / "README.md").read_text().splitlines() if line.startswith("python") and "--keep-keys" in line]
    assert lines
    for line in lines:
        words = shlex.split(line)
        option = lambda name, default: int(words[words.index(name) + 1]) if name in words else default      # noqa: E731
        pages, size, chunk = option("--pages", 128), option("--page-size", 16), min(option("--prefill-chunk", 8), option("--token-budget", 32))
        auto, model = sized(200 << 30, positions=131072, page_size=size, prefill_chunk=chunk, cache_bits=option("--cache-bits", None), keep_keys=option("--keep-keys", 0))
        cache = CacheManager(model.cache_needs(), pages or auto, size, 8)
        assert all(most <= left for most, left in zip(cache.most_pages_held(131072, chunk), cache.capacity()))


def test_a_cache_is_held_otherwise_only_before_a_runner_has_it(host_runner):
    """A runner's pages are laid out when it is made; a model whose runners are gone may be told anew."""
    from runtime.engine import runner as module
    runner, _ = host_runner(pages=8)
    model = runner.model
    for again in (dict(), dict(keep=8)):
        with pytest.raises(ValueError, match="before a runner"):
            model.hold_cache(4, **again)
    assert model.kept_keys is None and all(layer.mixer.four_bits == (0, 64, 2048) for layer in model.layers)
    del runner
    model.hold_cache(4, keep=8)
    assert module.ModelRunner(model, n_pages=8, device="cpu").cache.keep == 8
    plain = build_from_config_dict(preset("tiny-a"))[2]
    plain.dtype = torch.float32
    one = module.ModelRunner(plain, n_pages=8, device="cpu")
    with pytest.raises(ValueError, match="before a runner"):
        plain.hold_cache(4)
    assert one.cache.pages_of_site(0)[1].dtype == torch.float32 and not plain.layers[0].mixer.four_bits


def test_a_refused_bound_leaves_the_cache_held_as_it_was():
    model = build_from_config_dict(preset("tiny-a"))[2]
    model.layers[-1].mixer.window = 8                                     # (holds its keys in 4 bits, but no bounded number of them)
    with pytest.raises(ValueError, match="without a window"):
        model.hold_cache(4, keep=8)
    assert all(layer.mixer.four_bits is None for layer in model.layers) and model.kept_keys is None
    model.hold_cache(4)
    with pytest.raises(ValueError, match="without a window"):
        model.hold_cache(4, keep=8)
    assert all(layer.mixer.four_bits == (0, 64, 2048) for layer in model.layers) and model.kept_keys is None


@pytest.mark.parametrize("wrong", [dict(keep_recent=4), dict(keep_recent=0), dict(keep_keys=8), dict(cache_bits=4, keep_recent=4)])
def test_options_of_a_bound_that_is_not_there_are_refused(monkeypatch, wrong):
    """`keep_recent` says which of a bounded number of keys stay: without the bound it says nothing."""
    from runtime.engine import loading, runner as module
    from runtime.engine.scheduler import Engine
    monkeypatch.setattr(loading, "load_model", lambda folder, dtype, device: build_from_config_dict(preset("tiny-a"))[2])
    monkeypatch.setattr(module, "ModelRunner", lambda *a, **kw: pytest.fail("a runner was made"))
    with pytest.raises(ValueError, match="keep|kept"):
        Engine.from_folder("", **wrong)


@pytest.mark.parametrize("kv_heads, dim, page_size, fits", [(8, 128, 1 << 21, True), (8, 128, 1 << 22, False), (1, 256, 1 << 22, True), (1, 256, 1 << 23, False),
                                                            (1, 2, 1 << 25, True), (1, 2, 1 << 26, False), (2, 32, 1 << 25, True), (4, 32, 1 << 25, False)])
def test_pages_past_32_bits_are_refused(kv_heads, dim, page_size, fits):
    """A head's page is reckoned in 31 bits and a page of all heads in 32: larger ones would be read from the wrong place.  (Found before anything
    else of the call, here that its tensors are not on a GPU.)"""
    from runtime.kernels import cache4
    from runtime.kernels.ops import KernelError
    bytes_of = kv_heads * cache4.record_bytes(dim, page_size)
    assert fits == (bytes_of < 1 << 32 and bytes_of // kv_heads < 1 << 31)
    none = torch.zeros(1, 1)
    plan = cache4.plan([1], [0], 2 * kv_heads, kv_heads, dim, device="cpu", state_slots=[0])
    calls = [(cache4.rope_write, (none, none, none, none, none, none, none, 2 * kv_heads, kv_heads, dim, page_size)),
             (cache4.read, (none, none, none, none, kv_heads, dim, page_size)),
             (cache4.attention, (none, none, none, plan, none, 2 * kv_heads, kv_heads, dim, page_size, 0.1)),
             (cache4.add_weights, (none, none, none, none, plan, none, 2 * kv_heads, kv_heads, dim, page_size, 0.1)),
             (cache4.evict, (none, [none], none, none, none, none, none, kv_heads, dim, page_size, 8, 2, none))]
    for call, args in calls:
        with pytest.raises(KernelError, match="GPU|plan" if fits else "32 bits"):
            call(*args)


@pytest.mark.parametrize("counts, cached", [([2048, 1], [0, 32767]), ([1024, 1], [0, 32767]), ([2048, 1], [0, 8191]), ([2048] + [1] * 8, [0] + [4095] * 8),
                                            ([64, 2048], [32768, 0]), ([512, 1600], [16384, 0]), ([300] * 40 + [1], [0] * 40 + [100000])])
@pytest.mark.parametrize("heads, kv_heads, dim", [(32, 8, 128), (9, 3, 64)])
def test_long_rows_beside_a_prompt_are_cut(counts, cached, heads, kv_heads, dim):
    """However many tiles a prompt makes, no task walks keys that would be many pieces: the step would wait for it."""
    from runtime.kernels import cache4
    plan = cache4.plan(counts, cached, heads, kv_heads, dim, device="cpu")
    steps = (plan.tasks[:, 5] - plan.tasks[:, 4]).tolist()
    pieces = cache4.pieces_for(kv_heads, heads // kv_heads, plan.rows_per_task, plan.form, False)
    assert max(steps) <= 2.5 * max(cache4.LEAST_PIECE, -(-sum(steps) // pieces)) < max(cached) / 32
    # and what a prompt brings by itself is not: its last rows have twice the keys of the average
    alone = cache4.plan([2048], [0], heads, kv_heads, dim, device="cpu")
    assert alone.merges is None and max((alone.tasks[:, 5] - alone.tasks[:, 4]).tolist()) == 64


@pytest.mark.parametrize("heads, kv_heads, dim, counts, cached", [(32, 8, 128, [480] + [1] * 31, 1920), (32, 32, 64, [2000] + [1] * 63, 2000), (9, 3, 64, [1, 300, 1, 5], 100),
                                                                  (32, 8, 128, [1024] + [1] * 32, 8191)])
def test_segments_are_summed_by_their_own_number_of_items(heads, kv_heads, dim, counts, cached):
    """A portion's items are shared by blocks however many single rows stand beside it, and those keep waves of their own."""
    from runtime.engine.context import Batch
    from runtime.kernels import cache4
    plan = cache4.plan(counts, [cached] * len(counts), heads, kv_heads, dim, device="cpu", state_slots=range(len(counts)))
    assert plan.shares >= 1 and plan.few and plan.many == 1
    for few in ([1] * 64, [16, 1, 3]):
        plan = cache4.plan(few, [cached] * len(few), heads, kv_heads, dim, device="cpu", state_slots=range(len(few)))
        assert plan.shares == 0 and plan.few and plan.many == 0
    plan = cache4.plan([300, 200], [0, 0], heads, kv_heads, dim, device="cpu", state_slots=[0, 1])
    assert plan.shares >= 1 and not plan.few and plan.many == 2
    plan = cache4.plan([3, 70, 1, 100], [5, 6, 7, 8], heads, kv_heads, dim, device="cpu", state_slots=[9, 4, 0, 2])
    assert plan.segments.tolist() == [[74, 100, 8, 2, 3], [3, 70, 6, 4, 1], [0, 3, 5, 9, 0], [73, 1, 7, 0, 2]]
    # what an engine's step says of it
    step = lambda counts: Batch(counts, [0] * len(counts), None, False, {})                        # noqa: E731
    group = heads // kv_heads
    _, _, rows, few, many = cache4.step_arrays(heads, kv_heads, dim, None, torch.zeros(1, dtype=torch.bfloat16), True)
    assert [rows.launch_value(step(c)) for c in (counts, [1, 1], [7])] == [max(counts), 1, 7]
    batches = [step(c) for c in (counts, [300, 200], [64 // group, 300], [64 // group + 1, 300], [1])]
    assert [few.launch_value(b) for b in batches] == [1, 0, 1, 0, 1] and [many.launch_value(b) for b in batches] == [1, 2, 1, 2, 0]


def test_a_step_tells_its_largest_position_apart_from_its_most_keys(host_runner):
    """Positions go on counting where keys are given up: what sizes launches over keys is not what positions reach."""
    from runtime.engine.runner import StepEntry
    runner, _ = host_runner(pages=64, keep=32, recent=8, slack=16, portion=64)
    seen = []
    runner._forward = lambda ctx, take: seen.append((ctx.max_context, ctx.span_hint, int(ctx.positions.max()) + 1))
    runner.create("x"), runner.create("y")
    runner.step([StepEntry("x", [1] * 60, []), StepEntry("y", [1] * 9, [])])
    runner.step([StepEntry("x", [1], []), StepEntry("y", [1], [])])
    runner.step([StepEntry("y", [1], [])])
    assert seen == [(60, 60, 60), (61, 33, 61), (11, 11, 11)]


@pytest.mark.parametrize("page_size", [4, 24, 1 << 26])
def test_pages_that_the_kernels_do_not_take_are_refused_with_the_runner(host_runner, page_size):
    """Not by every request's first step."""
    from runtime.kernels.ops import KernelError
    with pytest.raises(KernelError, match="pages of"):
        host_runner(pages=1, page_size=page_size)
