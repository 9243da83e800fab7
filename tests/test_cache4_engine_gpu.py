"""The engine with a cache that holds keys and values in 4 bits, with all keys and with a bounded number of them."""
import json
import math
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

import plain_cache4 as plain
import plain_llama as P
from conftest import ROOT, TINY, assert_close, random_tokens

pytestmark = pytest.mark.gpu


def make_runner(folder, dtype, pages=64, page_size=16, execution="eager", **hold):
    from runtime.engine.loading import load_model
    from runtime.engine.runner import ModelRunner
    model = load_model(folder, dtype=dtype)
    model.hold_cache(4, **hold)
    return ModelRunner(model, n_pages=pages, page_size=page_size, max_requests=8, execution=execution)


def held(runner, request, site, n):
    """Keys and values [n, heads, dim] that the request's pages hold at a site, float64."""
    from runtime.kernels import cache4
    gid, index = runner.cache.group_of_site[site]
    group, need = runner.cache.groups[gid], runner.cache.groups[gid].need
    table, size = group.tables[request], group.page_size
    slots = torch.tensor([table[i // size] * size + i % size for i in range(n)], dtype=torch.int32, device="cuda")
    keys, values = (torch.empty(1, n, need.kv_heads, need.head_dim, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    cache4.read(group.storage[index:index + 1], slots, keys, values, need.kv_heads, need.head_dim, size)
    return keys[0].double().cpu().numpy(), values[0].double().cpu().numpy()


def plain_forward(cfg, w, tokens, caches, positions, first):
    """Logits of the rows `tokens` at `positions`; caches[layer] = held keys and values per key head ([n, heads, dim]) of everything
    up to and with these rows, which are the last; row i sees the first `first` + i of them."""
    c = cfg
    heads, kv, dim = c["num_attention_heads"], c["num_key_value_heads"], P.head_dim_of(c)
    x = np.asarray(w["model.embed_tokens.weight"], np.float64)[np.asarray(tokens)]
    made = []
    for layer in range(c["num_hidden_layers"]):
        p = f"model.layers.{layer}."
        h = P.rmsnorm(x, w[p + "input_layernorm.weight"], c["rms_norm_eps"])
        q = P.rope(P.linear(h, w[p + "self_attn.q_proj.weight"]).reshape(-1, heads, dim), positions, c["rope_theta"])
        k = P.rope(P.linear(h, w[p + "self_attn.k_proj.weight"]).reshape(-1, kv, dim), positions, c["rope_theta"])
        v = P.linear(h, w[p + "self_attn.v_proj.weight"]).reshape(-1, kv, dim)
        made.append((k, v))
        keys, values = caches[layer]
        out = np.stack([P.attention_one_query(q[t], keys[:first + t], values[:first + t]) for t in range(len(tokens))])
        x = x + P.linear(out.reshape(len(tokens), heads * dim), w[p + "self_attn.o_proj.weight"])
        h = P.rmsnorm(x, w[p + "post_attention_layernorm.weight"], c["rms_norm_eps"])
        x = x + P.linear(P.swiglu(P.linear(h, w[p + "mlp.gate_proj.weight"]), P.linear(h, w[p + "mlp.up_proj.weight"])), w[p + "mlp.down_proj.weight"])
    head = w["model.embed_tokens.weight"] if c.get("tie_word_embeddings", False) else w["lm_head.weight"]
    return P.linear(P.rmsnorm(x, w["model.norm.weight"], c["rms_norm_eps"]), head), made


def near(held_rows, rows, dtype):
    """Whether held numbers are the nearest of their block's: within half the widest gap (one step of the scale), plus what the
    activations of that type are off by."""
    pad = -rows.shape[-1] % 32
    blocks = np.abs(np.pad(rows, ((0, 0), (0, 0), (0, pad)))).reshape(*rows.shape[:2], -1, 32).max(-1)
    step = np.repeat(blocks / 3.5, 32, axis=-1)[..., :rows.shape[-1]]
    slack = 1e-3 if dtype == "float32" else 0.2
    return (np.abs(held_rows - rows) <= step * (1 + slack) + slack * np.abs(rows).max()).all()


@pytest.mark.parametrize("execution", ["eager", "graph"])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("name", ["a", "b", "c", "d"])
def test_logits_are_those_of_what_is_held(folders, name, dtype, execution):
    from runtime.engine.runner import StepEntry
    cfg, w = P.read_folder(folders[name])
    runner = make_runner(folders[name], dtype, execution=execution)
    tokens = random_tokens(7, 70, TINY[name]["vocab_size"])
    other = random_tokens(8, 40, TINY[name]["vocab_size"])
    got = []
    runner.create("r"), runner.create("s")
    for a, b in [(0, 33), (33, 60), *((i, i + 1) for i in range(60, 70))]:       # portions, then one by one beside another request
        entries = [StepEntry("r", tokens[a:b], list(range(b - a)))] + ([StepEntry("s", other[a:b], [])] if b <= 40 else [])
        got.append(runner.step(entries)[:b - a].double().cpu().numpy())
    caches = [held(runner, "r", site, 70) for site in range(cfg["num_hidden_layers"])]
    want, made = plain_forward(cfg, w, tokens, caches, np.arange(70), 1)
    assert_close(np.concatenate(got), want, dtype, "4 bits")
    for (k, v), (hk, hv) in zip(made, caches):
        assert near(hk, k, dtype) and near(hv, v, dtype)
    runner.cache.check()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("name", ["a", "c"])
def test_a_bounded_number_of_keys(folders, name, dtype):
    """A prompt in portions past the bound, then single tokens: the kept keys are those that the sums speak for, and the next logits are those
    of attention over them."""
    from runtime.engine.runner import StepEntry
    cfg, w = P.read_folder(folders[name])
    layers, kv = cfg["num_hidden_layers"], cfg["num_key_value_heads"]
    tokens = random_tokens(17, 150, TINY[name]["vocab_size"])
    keep, recent, slack = 40, 10, 12
    bound = dict(keep=keep, recent=recent, slack=slack, portion=60)
    runner = make_runner(folders[name], dtype, **bound)
    free = make_runner(folders[name], dtype, keep=400, recent=0, slack=64, portion=100)      # sums, and gives nothing up
    for r in (runner, free):
        r.create("r")
        r.step([StepEntry("r", tokens[:50], [])])
    assert runner.cache.cached("r") == 50 and not runner.cache.overfull("r")
    before = [held(free, "r", site, 50) for site in range(layers)]
    sums = [free.cache.state_storage[site][free.cache.slots.slot_of("r")].cpu() for site in range(layers)]
    for site in range(layers):                                                            # every row's weights come to one a head
        total = sums[site].double().sum().item()
        assert abs(total - 50 * cfg["num_attention_heads"]) < 1e-3 * total
    # the step that goes past keep + slack: 3 tokens beyond
    for r in (runner, free):
        r.step([StepEntry("r", tokens[50:53], [])])
    assert runner.cache.cached("r") == keep and runner.length("r") == 53 and free.cache.cached("r") == 53
    sums = [free.cache.state_storage[site][free.cache.slots.slot_of("r")].cpu() for site in range(layers)]
    for site in range(layers):
        all_keys, all_values = held(free, "r", site, 53)
        assert (all_keys[:50] == before[site][0]).all()
        kept_keys, kept_values = held(runner, "r", site, keep)
        left = runner.cache.state_storage[site][runner.cache.slots.slot_of("r")].cpu()
        for h in range(kv):
            index = plain.stays(sums[site][h], 53, keep, recent)
            assert (kept_keys[:, h] == all_keys[index, h]).all() and (kept_values[:, h] == all_values[index, h]).all()
            assert torch.equal(left[h, :keep], sums[site][h, index]) and not left[h, keep:].any()
    runner.cache.check()
    assert len(runner.cache.table(0, "r")) == -(-keep // 16)
    # decode past the bound again
    for i in range(53, 53 + 2 * slack + 5):
        kept_before = [held(runner, "r", site, runner.cache.cached("r")) for site in range(layers)]
        n = runner.cache.cached("r")
        logits = runner.step([StepEntry("r", [tokens[i]], [0])])[0].double().cpu().numpy()
        if runner.cache.cached("r") == n + 1:
            caches = [held(runner, "r", site, n + 1) for site in range(layers)]
            for (k, v), (k0, v0) in zip(caches, kept_before):
                assert (k[:n] == k0).all() and (v[:n] == v0).all()
            want, _ = plain_forward(cfg, w, [tokens[i]], caches, np.array([i]), n + 1)
            assert_close(logits[None], want, dtype, "bounded")
        else:
            assert n == keep + slack and runner.cache.cached("r") == keep
        assert runner.cache.cached("r") <= keep + slack and runner.length("r") == i + 1
        runner.cache.check()
    assert runner.counters["evictions_of_keys"] >= 3
    with pytest.raises(ValueError, match="at most"):
        runner.step([StepEntry("r", tokens[:100], [])])
    runner.release("r")
    assert runner.cache.free_pages() == [64]


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("keep", [0, 24])
def test_ways_of_running_agree(folders, dtype, keep):
    from runtime.engine.scheduler import Engine, Request
    V = TINY["c"]["vocab_size"]
    prompts = [random_tokens(140 + i, n, V) for i, n in enumerate([1, 70, 30, 140])]
    outputs = []
    # (the same portions of every prompt in all of them: what is given up goes by the sums at the end of a step)
    for policy, execution, overlap in [("serial", "eager", False), ("decode_first", "eager", False), ("decode_first", "graph", False), ("chunked", "graph", True)]:
        e = Engine.from_folder(folders["c"], dtype=dtype, pages=80, page_size=8, execution=execution, policy=policy, token_budget=4000, prefill_chunk=16,
                               overlap=overlap, cache_bits=4, keep_keys=keep)
        for i, p in enumerate(prompts):
            e.submit(Request(str(i), p, 90))
        assert all(r.status == "finished" and len(r.generated) == 90 for r in e.run())
        e.runner.cache.check()
        assert e.runner.cache.free_pages() == [80]
        assert (e.runner.counters.get("evictions_of_keys", 0) > 0) == bool(keep)
        outputs.append([e.requests[str(i)].generated for i in range(len(prompts))])
        if execution == "graph":
            assert any(p["graph"] is not None for p in e.runner.programs.values())
    if dtype == "float32":     # (in bfloat16 rows of another batch may round otherwise and part at a near tie)
        assert all(o == outputs[0] for o in outputs[1:])
    else:
        assert outputs[1] == outputs[2]


def test_forks_share_pages_and_keep_their_own_sums(folders):
    from runtime.engine.runner import StepEntry
    runner = make_runner(folders["a"], "float32", keep=32, recent=8, slack=16, portion=64)
    alone = make_runner(folders["a"], "float32", keep=32, recent=8, slack=16, portion=64)
    tokens = random_tokens(5, 120, TINY["a"]["vocab_size"])
    for r in (runner, alone):
        r.create("x")
        r.step([StepEntry("x", tokens[:40], [])])
    runner.fork("x", "y")
    for i in range(40, 100):       # the fork decodes past its bound; the source stays where it was
        a = runner.step([StepEntry("y", [tokens[i]], [0])])[0].clone()
        b = alone.step([StepEntry("x", [tokens[i]], [0])])[0]
        assert torch.equal(a, b)
        runner.cache.check()
    again = make_runner(folders["a"], "float32", keep=32, recent=8, slack=16, portion=64)
    again.create("x")
    again.step([StepEntry("x", tokens[:40], [])])
    for i in range(100, 118):
        assert torch.equal(runner.step([StepEntry("x", [tokens[i]], [0])])[0], again.step([StepEntry("x", [tokens[i]], [0])])[0])


def test_no_room_for_the_kept_keys_gives_up_nothing(folders):
    from runtime.engine.runner import StepEntry
    runner = make_runner(folders["a"], "float32", pages=4, keep=32, recent=8, slack=16, portion=16)     # (the kept keys would need two more pages)
    tokens = random_tokens(5, 64, TINY["a"]["vocab_size"])
    runner.create("x")
    for i in range(0, 64, 16):
        runner.step([StepEntry("x", tokens[i:i + 16], [])])
    assert runner.cache.cached("x") == 64 and runner.cache.free_pages() == [0]
    runner.cache.check()
    with pytest.raises(ValueError, match="at most 64"):
        runner.step([StepEntry("x", [1], [])])


def test_command_line(folders):
    env = dict(os.environ, PYTHONPATH=str(ROOT))
    base = [sys.executable, "-m", "runtime", "--checkpoint", str(folders["c"]), "--tokens", ",".join(map(str, random_tokens(1, 60, 1003))), "--max-new-tokens", "40",
            "--prefill-chunk", "16", "--token-budget", "16", "--report"]
    out = subprocess.run(base + ["--cache-bits", "4", "--keep-keys", "24"], capture_output=True, text=True, env=env, cwd=ROOT, timeout=300)
    assert out.returncode == 0, out.stderr
    report = json.loads(out.stdout)
    assert len(report["requests"][0]["generated"]) == 40 and report["runner"]["evictions_of_keys"] > 0
    out = subprocess.run(base + ["--keep-keys", "24"], capture_output=True, text=True, env=env, cwd=ROOT, timeout=300)
    assert out.returncode != 0 and "cache of 4 bits" in out.stderr
