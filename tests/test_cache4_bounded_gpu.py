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
