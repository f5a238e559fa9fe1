"""An engine whose cache is held in 8 bits, end to end, and the scoring of tokens: against the plain model with keys and values that went
through the same codes, across cuts, batches, graphs and steps queued ahead; the command line."""
import math
import os
import subprocess
import sys

import pytest
import torch

from plain import cache_8bit_plain, qwen2_plain

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CONFIG = {"architectures": ["Qwen2ForCausalLM"], "num_hidden_layers": 2, "hidden_size": 128, "num_attention_heads": 4, "num_key_value_heads": 2,
          "head_dim": 64, "intermediate_size": 176, "vocab_size": 300, "rope_theta": 10000.0, "rms_norm_eps": 1e-6, "tie_word_embeddings": True,
          "max_position_embeddings": 512}


@pytest.fixture(scope="module")
def folder(tmp_path_factory):
    from aegean_tge_b200 import write_random_model
    path = str(tmp_path_factory.mktemp("model"))
    write_random_model(path, CONFIG, seed=5, dtype="float32")
    return path


def engine(folder, dtype="float32", **kw):
    from aegean_tge_b200 import Engine
    return Engine(folder, dtype=dtype, **{"context": 256, "max_tokens": 4096, "cache_dtype": "int8", "page_size": 16, **kw})


def prompt(n, seed=0):
    return torch.randint(0, CONFIG["vocab_size"], (n,), generator=torch.Generator().manual_seed(seed)).tolist()


def plain_logits(folder, tokens, monkeypatch):
    """The plain model in float64 whose keys and values stand for their codes, a scale per position and head."""
    raw, weights = qwen2_plain.read_model(folder)
    exact = qwen2_plain.attention

    def through_codes(x):
        scale = x.abs().amax(-1, keepdim=True)
        return torch.round(127 * x / scale) * scale / 127

    monkeypatch.setattr(qwen2_plain, "attention", lambda q, k, v, window=0: exact(q, through_codes(k), through_codes(v), window))
    return qwen2_plain.logits_of(raw, weights, tokens).double()


def run(eng, cuts, tokens, name="r"):
    from aegean_tge_b200.engine.batch import Portion
    rows, at = [], 0
    for n in cuts:
        rows.append(eng.runner.step([Portion(name, tokens[at:at + n], list(range(n)))]).double().cpu())
        at += n
    eng.runner.finish(name)
    return torch.cat(rows)


# A code at a tie may fall to either side in float32: 1/127 of a block's largest number, of which a logit sees a small part.
# bfloat16: the general bound of whole-model logits.
@pytest.mark.parametrize("dtype,tolerance", [("float32", 2e-3), ("bfloat16", 3.5e-2)])
@pytest.mark.parametrize("cuts", [[40], [1] * 40, [17, 1, 1, 20, 1]])
def test_logits(folder, monkeypatch, dtype, tolerance, cuts):
    tokens = prompt(40)
    want = plain_logits(folder, tokens, monkeypatch)
    got = run(engine(folder, dtype), cuts, tokens)
    assert float((got - want).abs().max()) < tolerance * float(want.abs().max())


def test_the_cache_is_what_moves_the_answers(folder):
    """Beside an engine with the cache in float32: near, and not the same."""
    tokens = prompt(60)
    a, b = run(engine(folder), [60], tokens), run(engine(folder, cache_dtype=None), [60], tokens)
    apart = float((a - b).abs().max()) / float(b.abs().max())
    assert 1e-6 < apart < 5e-2


@pytest.mark.parametrize("block,page", [(4, 16), (16, 16), (64, 64)])
def test_blocks_of_positions(folder, block, page):
    """Larger blocks: their entries depend on the cut; the answers stay near those of the cache in float32."""
    tokens = prompt(100)
    want = run(engine(folder, cache_dtype=None), [100], tokens)
    for cuts in ([100], [30, 1, 1, 1, 67]):
        got = run(engine(folder, cache_block=block, page_size=page), cuts, tokens)
        assert float((got - want).abs().max()) < 5e-2 * float(want.abs().max())


def test_a_row_does_not_depend_on_the_cut(folder):
    """Blocks of one: the cache is the same whatever the cut; float32 rows differ by the order of sums alone."""
    tokens = prompt(90)
    rows = [run(engine(folder), cuts, tokens) for cuts in ([90], [1] * 90, [64, 1, 25])]
    for other in rows[1:]:
        assert float((other - rows[0]).abs().max()) < 2e-3 * float(rows[0].abs().max())


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_graphs_and_steps_ahead_change_no_token(folder, dtype):
    """Requests of unlike lengths that come and go: the same tokens with and without graph replay and steps queued ahead."""
    batch = [prompt(n, seed=n) for n in (3, 40, 17, 90, 5, 64, 1)]
    want = engine(folder, dtype, use_graphs=False, run_ahead=False).generate(batch, n=24)
    assert engine(folder, dtype).generate(batch, n=24) == want
    if dtype == "float32":          # also when few pages force requests out and in again: blocks of one are recomputed as they were
        small = engine(folder, dtype, max_tokens=192)
        assert small.generate(batch[:3], n=24) == want[:3]


def test_a_mixed_step(folder):
    """Single tokens beside portions in one step: every row as on its own."""
    from aegean_tge_b200.engine.batch import Portion
    for dtype in ("float32", "bfloat16"):
        eng = engine(folder, dtype)
        first = {f"s{i}": prompt(10 + 7 * i, seed=i) for i in range(9)}
        for name, tokens in first.items():
            eng.runner.step([Portion(name, tokens, [])])
        step = [Portion(name, [int(name[1:]) + 5], [0]) for name in first] + [Portion("p", prompt(50, seed=77), [0, 49]), Portion("q", prompt(2, seed=78), [1])]
        together = eng.runner.step(step).double().cpu()
        alone = engine(folder, dtype)
        for name, tokens in first.items():
            alone.runner.step([Portion(name, tokens, [])])
        rows = torch.cat([alone.runner.step([portion]) for portion in step]).double().cpu()
        assert float((together - rows).abs().max()) < {"float32": 2e-3, "bfloat16": 2e-2}[dtype] * float(rows.abs().max())


def test_what_is_refused(folder):
    for kw in ({"cache_dtype": "int4"}, {"cache_block": 3}, {"cache_block": 32}, {"cache_block": 0}):
        with pytest.raises(ValueError):
            engine(folder, **kw)


# ---------------------------------------------------------------------------
@pytest.mark.parametrize("cache", [None, "int8"])
@pytest.mark.parametrize("budget", [2048, 16, 1])
def test_score(folder, cache, budget):
    """Engine.score against the logits it goes by, in one portion or many, with another request live; nothing of it stays."""
    eng = engine(folder, cache_dtype=cache, max_batch_tokens=budget)
    tokens = prompt(41)
    free = eng.cache.groups[0].pool.free_count
    from aegean_tge_b200.engine.batch import Portion
    eng.runner.step([Portion("other", [1], [])])
    scores = eng.score(tokens, top=6)
    eng.runner.finish("other")
    assert eng.cache.groups[0].pool.free_count == free
    rows = run(eng, [40], tokens[:40])
    assert scores.logprob.shape == (40,) and scores.top_ids.shape == (40, 6)
    for i in range(40):
        lp, entropy, rank, ids, lps = cache_8bit_plain.token_logprobs(rows[i].tolist(), tokens[i + 1], 6)
        # portions of other sizes add in another order: 1e-5 of logits of some units, a flipped code 2e-3
        assert abs(float(scores.logprob[i]) - lp) < 1e-2 and abs(float(scores.entropy[i]) - entropy) < 1e-2
        assert max(abs(a - b) for a, b in zip(scores.top_logprobs[i].tolist(), lps)) < 1e-2
        if budget == 2048:
            assert int(scores.rank[i]) == rank and scores.top_ids[i].tolist() == ids
    assert eng.generate(tokens[:5], n=4) == engine(folder, cache_dtype=cache).generate(tokens[:5], n=4)


def test_score_refuses(folder):
    eng = engine(folder)
    for tokens, top in (([1], 0), ([1, 300], 0), ([1, -1], 0), ([1, 2], 33), ([1, 2], -1), (prompt(258), 0)):
        with pytest.raises(ValueError):
            eng.score(tokens, top=top)
    assert eng.score(prompt(257)).logprob.shape == (256,) and not eng.cache.live_requests()


def test_command_line(folder):
    def tge(*args):
        done = subprocess.run([sys.executable, os.path.join(ROOT, "bin", "tge"), *args], capture_output=True, text=True, timeout=600)
        assert done.returncode == 0, done.stderr
        return done.stdout
    tokens = prompt(20)
    text = tge("score", "--model", folder, "--dtype", "float32", "--context", "64", "--tokens", " ".join(map(str, tokens)), "--top", "3", "--cache-dtype", "int8",
               "--cache-block", "4", "--compare", "--max-batch-tokens", "8")
    lines = [line for line in text.splitlines() if "entropy" in line and "rank" in line]
    assert [int(line.split(":")[0]) for line in lines] == tokens[1:]
    assert "score    : 19 tokens" in text and "compare  :" in text
    worst = float(text.split("worst ")[1].split(";")[0])
    assert 0 < worst < 0.5 and math.isfinite(worst)
    assert "ids      :" in tge("generate", "--model", folder, "--tokens", "1 2 3", "--n", "4", "--cache-dtype", "int8", "--print-ids", "--num-pages", "8")
    assert "over a cache of int8" in tge("fidelity", "--model", folder, "--tokens", "20", "--cache-dtype", "int8", "--num-pages", "8", "--context", "64")


def test_a_layer_that_reads_an_earlier_layers_cache(monkeypatch):
    """It rotates its queries and stores nothing; the cut changes nothing, and the codes move its logits by little."""
    import dataclasses

    from aegean_tge_b200 import Engine, registry
    from aegean_tge_b200.registry import Architecture, architecture_of, register_architecture
    base = architecture_of(CONFIG)

    def shared(config):
        spec = base.build_spec(config)
        return dataclasses.replace(spec, layers=(spec.layers[0], dataclasses.replace(spec.layers[1], cache_from=0)))

    monkeypatch.setattr(registry, "_ARCHITECTURES", dict(registry._ARCHITECTURES))
    register_architecture(Architecture("SharedCacheForCausalLM", base.parse_config, shared, base.random_plan))
    raw = dict(CONFIG, architectures=["SharedCacheForCausalLM"])
    tokens = prompt(90)

    def rows(cuts, cache_dtype):
        eng = Engine(random_config=raw, dtype="float32", context=256, max_tokens=4096, page_size=16, cache_dtype=cache_dtype)
        assert len(eng.cache.groups) == 1
        return run(eng, cuts, tokens)

    whole, exact = rows([90], "int8"), rows([90], None)
    assert float((rows([30, 1, 1, 58], "int8") - whole).abs().max()) < 2e-3 * float(whole.abs().max())
    moved = float((whole - exact).abs().max()) / float(exact.abs().max())
    assert 1e-6 < moved < 5e-2


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_layers_over_a_window_whose_pages_are_given_back(monkeypatch, dtype):
    """Pages behind the window are released as a request grows: cut prompts and single tokens go on without a fault."""
    import dataclasses

    from aegean_tge_b200 import Engine, ops, registry
    from aegean_tge_b200.registry import Architecture, architecture_of, register_architecture
    base = architecture_of(CONFIG)

    def windowed(config):
        spec = base.build_spec(config)
        narrow = [dataclasses.replace(layer, mixer=dataclasses.replace(layer.mixer, params=dict(layer.mixer.params, window=100))) for layer in spec.layers]
        return dataclasses.replace(spec, layers=tuple(narrow))

    monkeypatch.setattr(registry, "_ARCHITECTURES", dict(registry._ARCHITECTURES))
    register_architecture(Architecture("WindowedForCausalLM", base.parse_config, windowed, base.random_plan))
    raw = dict(CONFIG, architectures=["WindowedForCausalLM"])
    tokens = prompt(400)

    def rows(cuts, cache_dtype):
        eng = Engine(random_config=raw, dtype=dtype, context=512, max_tokens=4096, page_size=16, cache_dtype=cache_dtype)
        found = run(eng, cuts, tokens)
        ops.check_status()
        return found

    whole, exact = rows([400], "int8"), rows([400], None)
    cut = rows([130, 70, 90, 1, 50, 1, 1, 57], "int8")
    assert float((cut - whole).abs().max()) < {"float32": 2e-3, "bfloat16": 3.5e-2}[dtype] * float(whole.abs().max())
    assert float((whole - exact).abs().max()) < 5e-2 * float(exact.abs().max())
