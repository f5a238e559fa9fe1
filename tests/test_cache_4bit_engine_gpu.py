"""An engine whose cache is held in 4 bits, end to end: against the plain model with keys and values that went through the same codes, across cuts,
batches, graphs and steps queued ahead; layers with norms of queries and keys, and with rotations of neighbours; the command line."""
import dataclasses
import math
import os
import subprocess
import sys

import pytest
import torch

from plain import qwen2_plain

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
    return Engine(folder, dtype=dtype, **{"context": 256, "max_tokens": 4096, "cache_dtype": "uint4", "page_size": 16, **kw})


def prompt(n, seed=0):
    return torch.randint(0, CONFIG["vocab_size"], (n,), generator=torch.Generator().manual_seed(seed)).tolist()


def through_codes(x):
    """What an entry of x [..., dim] (float64) reads as."""
    y = x.unflatten(-1, (-1, 32))
    lo, hi = y.amin(-1, keepdim=True), y.amax(-1, keepdim=True)
    base = (lo + (hi - lo) * (8 / 15)).float().bfloat16().double()
    least = torch.maximum((hi - base) / 7, (base - lo) / 8)
    step = least.float().bfloat16()
    step = torch.where(step.double() < least, (step.view(torch.int16) + 1).view(torch.bfloat16), step).double()
    return (base + (torch.round((y - base) / step) + 0.0).clamp(-8, 7) * step).flatten(-2).to(x.dtype)


def run(eng, cuts, tokens, name="r"):
    from aegean_tge_b200.engine.batch import Portion
    rows, at = [], 0
    for n in cuts:
        rows.append(eng.runner.step([Portion(name, tokens[at:at + n], list(range(n)))]).double().cpu())
        at += n
    eng.runner.finish(name)
    return torch.cat(rows)


def moved(a, b):
    return float((a - b).abs().max()) / float(b.abs().max())


# A code at a tie may fall to either side in float32: a fifteenth of a group's span in one number of one entry, of which a logit sees a small part.
@pytest.mark.parametrize("cuts", [[40], [1] * 40, [17, 1, 1, 20, 1]])
def test_logits(folder, monkeypatch, cuts):
    tokens = prompt(40)
    raw, weights = qwen2_plain.read_model(folder)
    exact = qwen2_plain.attention
    monkeypatch.setattr(qwen2_plain, "attention", lambda q, k, v, window=0: exact(q, through_codes(k.double()).to(k.dtype), through_codes(v.double()).to(v.dtype), window))
    want = qwen2_plain.logits_of(raw, weights, tokens).double()
    assert moved(run(engine(folder), cuts, tokens), want) < 1e-2


def test_the_cache_is_what_moves_the_answers(folder):
    """Beside an engine with the cache in float32: near, and not the same; 8 bits move them by less."""
    tokens = prompt(60)
    four, eight, none = (run(engine(folder, cache_dtype=kind), [60], tokens) for kind in ("uint4", "int8", None))
    assert 1e-5 < moved(four, none) < 0.3 and moved(eight, none) < 0.25 * moved(four, none)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_a_row_does_not_depend_on_the_cut(folder, dtype):
    """Entries are a function of their rows: float32 rows differ by the order of sums, and what that moves across a border between codes; bfloat16 rows of
    other products round otherwise, some codes in every entry with them: less than the cache moves the answers."""
    tokens = prompt(90)
    rows = [run(engine(folder, dtype), cuts, tokens) for cuts in ([90], [1] * 90, [64, 1, 25])]
    bound = 1e-2 if dtype == "float32" else moved(rows[0], run(engine(folder, dtype, cache_dtype=None), [90], tokens)) + 3.5e-2
    for other in rows[1:]:
        assert moved(other, rows[0]) < bound


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_graphs_and_steps_ahead_change_no_token(folder, dtype):
    """Requests of unlike lengths that come and go: the same tokens with and without graph replay and steps queued ahead."""
    batch = [prompt(n, seed=n) for n in (3, 40, 17, 90, 5, 64, 1)]
    want = engine(folder, dtype, use_graphs=False, run_ahead=False).generate(batch, n=24)
    assert engine(folder, dtype).generate(batch, n=24) == want
    if dtype == "float32":          # also when few pages force requests out and in again: entries are recomputed as they were
        small = engine(folder, dtype, max_tokens=192)
        assert small.generate(batch[:3], n=24) == want[:3]


def test_a_mixed_step(folder):
    """Single tokens beside portions in one step: every row as on its own."""
    from aegean_tge_b200.engine.batch import Portion
    eng = engine(folder)
    first = {f"s{i}": prompt(10 + 7 * i, seed=i) for i in range(9)}
    for name, tokens in first.items():
        eng.runner.step([Portion(name, tokens, [])])
    step = [Portion(name, [int(name[1:]) + 5], [0]) for name in first] + [Portion("p", prompt(50, seed=77), [0, 49]), Portion("q", prompt(2, seed=78), [1])]
    together = eng.runner.step(step).double().cpu()
    alone = engine(folder)
    for name, tokens in first.items():
        alone.runner.step([Portion(name, tokens, [])])
    assert moved(together, torch.cat([alone.runner.step([portion]) for portion in step]).double().cpu()) < 1e-2


def test_score(folder):
    """A prompt's tokens scored over the cache: near the scores over one in float32, and what the logits say."""
    tokens = prompt(41)
    four, none = engine(folder).score(tokens, top=4), engine(folder, cache_dtype=None).score(tokens, top=4)
    assert 0 < float((four.logprob - none.logprob).abs().max()) < 0.5
    rows = torch.log_softmax(run(engine(folder), [40], tokens[:40]), -1)
    assert float((rows[torch.arange(40), torch.tensor(tokens[1:])] - four.logprob.double().cpu()).abs().max()) < 1e-2


def test_what_is_refused(folder):
    for kw in ({"cache_block": 4}, {"cache_dtype": "int4"}, {"cache_dtype": "uint8"}):
        with pytest.raises(ValueError):
            engine(folder, **kw)


def test_command_line(folder):
    def tge(*args):
        done = subprocess.run([sys.executable, os.path.join(ROOT, "bin", "tge"), *args], capture_output=True, text=True, timeout=600)
        assert done.returncode == 0, done.stderr
        return done.stdout
    tokens = prompt(20)
    text = tge("score", "--model", folder, "--dtype", "float32", "--context", "64", "--tokens", " ".join(map(str, tokens)), "--top", "3", "--cache-dtype", "uint4",
               "--compare", "--max-batch-tokens", "8")
    assert "score    : 19 tokens" in text and "compare  :" in text
    worst = float(text.split("worst ")[1].split(";")[0])
    assert 0 < worst < 1.0 and math.isfinite(worst)
    assert "ids      :" in tge("generate", "--model", folder, "--tokens", "1 2 3", "--n", "4", "--cache-dtype", "uint4", "--print-ids", "--num-pages", "8")
    assert "over a cache of uint4" in tge("fidelity", "--model", folder, "--tokens", "20", "--cache-dtype", "uint4", "--num-pages", "8", "--context", "64")


def registered(monkeypatch, name, change, extra=()):
    """An architecture like the base one whose layers `change` has been through."""
    from aegean_tge_b200 import registry
    from aegean_tge_b200.registry import Architecture, architecture_of, register_architecture
    base = architecture_of(CONFIG)

    def build(config):
        spec = base.build_spec(config)
        return dataclasses.replace(spec, layers=tuple(change(i, layer) for i, layer in enumerate(spec.layers)))

    def plan(config):
        yield from base.random_plan(config)
        yield from extra

    monkeypatch.setattr(registry, "_ARCHITECTURES", dict(registry._ARCHITECTURES))
    register_architecture(Architecture(name, base.parse_config, build, plan))
    return dict(CONFIG, architectures=[name])


def rows_of(raw, tokens, cuts, cache_dtype, dtype="float32"):
    from aegean_tge_b200 import Engine, ops
    eng = Engine(random_config=raw, dtype=dtype, context=512, max_tokens=4096, page_size=16, cache_dtype=cache_dtype)
    found = run(eng, cuts, tokens)
    ops.check_status()
    return found


@pytest.mark.parametrize("shared", [False, True])
@pytest.mark.parametrize("normed,position", [(True, "rope_neox"), (True, "rope_interleaved"), (False, "rope_interleaved"), (False, "rope_neox"), (True, "none")])
def test_layers_of_other_kinds(monkeypatch, normed, position, shared):
    """Norms of each head, rotations of neighbours, none; a layer that reads an earlier layer's cache and stores nothing: the cut changes
    nothing, and the codes move the logits by little."""
    from aegean_tge_b200.registry import architecture_of  # noqa: F401
    from aegean_tge_b200.config.model_spec import PartSpec
    from aegean_tge_b200.weights.random_init import uniform
    extra = [(f"model.layers.{n}.self_attn.{x}_norm.weight", (64,), "vector", uniform(0.5, 1.5)) for n in range(2) for x in "qk"] if normed else []

    def change(i, layer):
        params = dict(layer.mixer.params, position=PartSpec(position, {} if position == "none" else {"head_dim": 64, "theta": 10000.0}))
        weights = dict(layer.mixer.weights)
        if normed:
            params["qk_norm"] = {"scope": "head", "eps": 1e-6}
            weights.update({f"{x}_norm.weight": f"model.layers.{i}.self_attn.{x}_norm.weight" for x in "qk"})
        layer = dataclasses.replace(layer, mixer=dataclasses.replace(layer.mixer, params=params, weights=weights))
        return dataclasses.replace(layer, cache_from=0) if shared and i == 1 else layer

    raw = registered(monkeypatch, "OtherKindForCausalLM", change, extra)
    tokens = prompt(90)
    whole, exact = rows_of(raw, tokens, [90], "uint4"), rows_of(raw, tokens, [90], None)
    assert moved(rows_of(raw, tokens, [30, 1, 1, 58], "uint4"), whole) < 1e-2
    assert 1e-5 < moved(whole, exact) < 0.3


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_layers_over_a_window_whose_pages_are_given_back(monkeypatch, dtype):
    """Pages behind the window are released as a request grows: cut prompts and single tokens go on without a fault."""
    raw = registered(monkeypatch, "WindowedForCausalLM",
                     lambda i, layer: dataclasses.replace(layer, mixer=dataclasses.replace(layer.mixer, params=dict(layer.mixer.params, window=100))))
    tokens = prompt(400)
    whole, exact = (rows_of(raw, tokens, [400], kind, dtype) for kind in ("uint4", None))
    cut = rows_of(raw, tokens, [130, 70, 90, 1, 50, 1, 1, 57], "uint4", dtype)
    assert moved(cut, whole) < (1e-2 if dtype == "float32" else moved(whole, exact) + 3.5e-2)
    assert moved(whole, exact) < 0.3
