"""A bounded number of keys in the cache of 4 bits, as the scheduler runs it."""
import pytest

from conftest import TINY, random_tokens

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("execution", ["eager", "graph"])
def test_requests_of_equal_length_pass_their_bound_together(folders, execution, dtype):
    """Each step's tokens stay on the device until the next takes them: that keys are given up in between, of every request at once, changes none
    of them."""
    from runtime.engine.scheduler import Engine, Request
    prompts = [random_tokens(200 + i, 216, TINY["c"]["vocab_size"]) for i in range(6)]
    outputs = []
    for overlap in (False, True):
        e = Engine.from_folder(folders["c"], dtype=dtype, pages=400, page_size=8, execution=execution, token_budget=4000, prefill_chunk=16, overlap=overlap,
                               cache_bits=4, keep_keys=160)
        for i, p in enumerate(prompts):
            e.submit(Request(str(i), p, 100))
        e.run()
        assert e.runner.counters["evictions_of_keys"] == 2 * len(prompts)
        assert len({e.requests[str(i)].launched for i in range(len(prompts))}) == 1
        outputs.append([e.requests[str(i)].generated for i in range(len(prompts))])
    assert outputs[0] == outputs[1] and all(len(o) == 100 for o in outputs[0])


def test_the_command_line_names_a_pool_that_the_kept_keys_fill(folders):
    import json
    import os
    import subprocess
    import sys
    from conftest import ROOT
    env = dict(os.environ, PYTHONPATH=str(ROOT))
    base = [sys.executable, "-m", "runtime", "--checkpoint", str(folders["c"]), "--tokens", "1,2,3", "--max-new-tokens", "8", "--cache-bits", "4", "--keep-keys", "2048"]
    out = subprocess.run(base, capture_output=True, text=True, env=env, cwd=ROOT, timeout=100)
    assert out.returncode != 0 and "128 pages of 16 holds no request" in out.stderr
    out = subprocess.run(base + ["--pages", "0"], capture_output=True, text=True, env=env, cwd=ROOT, timeout=100)
    assert out.returncode == 0, out.stderr
    assert len(json.loads(out.stdout)["requests"][0]["generated"]) == 8


@pytest.mark.parametrize("form, heads, kv, dim, kind", [(0, 9, 3, 64, "bf16"), (0, 8, 2, 128, "f32"), (1, 8, 2, 128, "bf16"), (2, 8, 2, 128, "bf16"), (2, 9, 3, 64, "bf16"), (0, 2, 1, 256, "bf16")])
@pytest.mark.parametrize("window", [0, 400])
def test_long_rows_are_cut_beside_more_tiles_than_pieces(form, heads, kv, dim, kind, window, monkeypatch):
    """A row behind many keys, and a portion behind as many, beside a prompt whose tiles alone are as many as the pieces asked for."""
    import test_cache4_gpu as step
    monkeypatch.setattr(step.cache4(), "LEAST_PIECE", 2)
    made, plan = [], step.cache4()._plan
    monkeypatch.setattr(step.cache4(), "_plan", lambda *a: (made.append(plan(*a)), made[-1])[1])
    pieces = -(-300 // max(1, step.cache4().tile_of(form) // (heads // kv)))
    step.check_step([300, 1, 9], [0, 1500, 1400], heads, kv, dim, 16, kind, window=window, force=(form, pieces))
    counts = [(made[-1].tasks[:, 0] == seg).sum().item() for seg in range(3)]
    # (the prompt's tiles walk 5 steps on average, the row 47: over 8 to 75 pieces 17 steps at most a piece, so that the row makes three)
    assert counts[0] >= pieces and (window or (counts[1] > 2 and made[-1].merges is not None))


@pytest.mark.parametrize("counts, cached", [([150, 1, 40, 3, 1], [10, 70, 200, 0, 333]), ([1, 16, 17, 64, 65, 1], [5, 0, 90, 130, 31, 2]), ([100, 90], [0, 300])])
@pytest.mark.parametrize("heads, kv, dim, kind", [(8, 2, 128, "bf16"), (9, 3, 64, "f32"), (4, 4, 64, "bf16"), (3, 1, 20, "bf16"), (40, 1, 32, "bf16"), (2, 1, 256, "bf16")])
@pytest.mark.parametrize("window", [0, 60])
def test_sums_of_segments_of_few_and_of_many_items(counts, cached, heads, kv, dim, kind, window):
    """Either kernel takes its own segments, and together every one once."""
    from test_cache4_gpu import check_step
    check_step(counts, cached, heads, kv, dim, 16, kind, window=window, weights=True)


@pytest.mark.parametrize("chunk", [16, 20, 40])
def test_sums_of_mixed_steps_are_alike_however_they_run(folders, chunk):
    """Portions of 20 rows (60 items) are few, but their captured programs' 32 would be many; those of 40 are many beside decoding rows."""
    from runtime.engine.scheduler import Engine, Request
    prompts = [random_tokens(300 + i, n, TINY["c"]["vocab_size"]) for i, n in enumerate([1, 130, 60, 200, 40])]
    tokens, sums = [], []
    for execution in ("eager", "graph"):
        e = Engine.from_folder(folders["c"], dtype="float32", pages=400, page_size=8, execution=execution, policy="decode_first", token_budget=4000, prefill_chunk=chunk,
                               cache_bits=4, keep_keys=100)
        for i, p in enumerate(prompts):
            e.submit(Request(str(i), p, 60))
        seen = []
        while e.tick():
            seen.append({key: sum(e.runner.cache.state_storage[site][e.runner.cache.slots.slot_of(key)].double().sum() for site in (0, 1)).item() for key in e.runner.cache.lengths})
        tokens.append([e.requests[str(i)].generated for i in range(len(prompts))])
        sums.append(seen)
        assert e.runner.counters["evictions_of_keys"] > 0 and (execution == "eager" or e.runner.counters["replays"] > 0)
    assert tokens[0] == tokens[1] and sums[0] == sums[1]
