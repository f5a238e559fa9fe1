"""The 8-bit cache on the host: what a spec says of its entries, what the cache manager lays out, what is refused; the command line."""
import os
import subprocess
import sys

import pytest
import torch

from aegean_tge_b200.cache.manager import CacheManager
from aegean_tge_b200.config.model_spec import PartSpec
from aegean_tge_b200.models.decoder import DecoderModel
from aegean_tge_b200.parts.base import MIXERS, BuildEnv, PagedCacheSpec, build_part
from aegean_tge_b200.registry import architecture_of

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CONFIG = {"architectures": ["Qwen2ForCausalLM"], "num_hidden_layers": 2, "hidden_size": 64, "num_attention_heads": 4, "num_key_value_heads": 2,
          "head_dim": 16, "intermediate_size": 176, "vocab_size": 256, "rope_theta": 10000.0, "rms_norm_eps": 1e-6, "tie_word_embeddings": True,
          "max_position_embeddings": 256}


def env(block, page=16, dtype=torch.bfloat16):
    return BuildEnv(dtype=dtype, device=torch.device("cpu"), hidden_size=64, max_positions=64, page_size=page, ops=None, cache_block=block)


def attention(block, **options):
    position = PartSpec("rope_neox", {"head_dim": 16, "theta": 10000.0})
    return build_part(MIXERS, PartSpec("gqa_attention", {"hidden_size": 64, "heads": 4, "kv_heads": 2, "head_dim": 16, "position": position, **options}),
                      env(block))


@pytest.mark.parametrize("block,page", [(1, 16), (4, 16), (16, 16), (64, 64)])
def test_layout_and_bytes(block, page):
    spec = attention(block).cache_spec()
    per_token = 2 * 2 * (16 + 4 / block)
    assert spec.bytes_per_token(2) == per_token == spec.bytes_per_token(4)
    manager = CacheManager(page, 4)
    manager.add_layer(0, spec, None)
    manager.add_layer(1, spec, None)
    manager.add_layer(2, PagedCacheSpec((("k", (2, 16)), ("v", (2, 16)))), None)           # the same positions in the run dtype
    assert len(manager.groups) == 1 and manager.layer_variant == {0: 0, 1: 0, 2: 1}
    assert manager.groups[0].bytes_per_page(2) == round(page * (2 * per_token + 2 * 2 * 16 * 2))
    manager.set_pool_sizes([5])
    manager.allocate_storage(torch.bfloat16, torch.device("cpu"))
    held = manager.layer_cache(1).paged
    assert held["k"].dtype == held["v"].dtype == torch.int8 and held["k"].shape == (6, 2, page, 16)
    assert held["k_scale"].dtype == torch.float32 and held["k_scale"].shape == (6, 2, page // block, 1)
    assert held["k_scale"].squeeze(-1).is_contiguous()
    assert manager.layer_cache(2).paged["k"].dtype == torch.bfloat16


def test_entries_that_differ_in_type_alone_are_kept_apart():
    shapes = (("k", (2, 16)), ("v", (2, 16)))
    manager = CacheManager(16, 2)
    manager.add_layer(0, PagedCacheSpec(shapes), None)
    manager.add_layer(1, PagedCacheSpec(shapes, formats=(("k", torch.int8, 1), ("v", torch.int8, 1))), None)
    assert manager.layer_variant == {0: 0, 1: 1}
    with pytest.raises(ValueError):
        PagedCacheSpec(shapes).covering(PagedCacheSpec(shapes, formats=(("k", torch.int8, 1),)))
    wide = PagedCacheSpec(shapes, window=8, formats=(("k", torch.int8, 1),))
    assert wide.covering(PagedCacheSpec(shapes, window=16, formats=wide.formats)) == PagedCacheSpec(shapes, window=16, formats=wide.formats)


def test_a_block_that_does_not_divide_the_page_is_refused():
    manager = CacheManager(16, 2)
    manager.add_layer(0, PagedCacheSpec((("s", (2, 1)),), formats=(("s", torch.float32, 32),)), None)
    manager.set_pool_sizes([2])
    with pytest.raises(ValueError):
        manager.allocate_storage(torch.float32, torch.device("cpu"))


def test_a_model_says_what_its_cache_takes():
    arch = architecture_of(CONFIG)
    spec = arch.build_spec(arch.parse_config(CONFIG))
    assert DecoderModel(spec, env(None)).cache_bytes_per_token() == 2 * 2 * 2 * 16 * 2
    model = DecoderModel(spec, env(1))
    assert model.cache_bytes_per_token() == 2 * 2 * 2 * (16 + 4)
    assert model.decode_cache_bytes(100) == 100 * model.cache_bytes_per_token()


@pytest.mark.parametrize("options,holds", [({}, True), ({"window": 32}, True), ({"sinks": True}, True), ({"qk_norm": {"scope": "head", "eps": 1e-6}}, False),
                                           ({"value_dim": 8}, False), ({"short_conv": 3}, False), ({"output_gate": True}, False)])
def test_which_attention_can_hold_it(options, holds):
    assert attention(None, **options).holds_8bit is holds
    kept = attention(4, **options).cache_spec()
    assert bool(kept.formats) is holds


def test_a_model_that_cannot_refuses():
    from aegean_tge_b200.bench_tools import mozepel_config
    raw = mozepel_config(64, 4, 2, 16, 176, 4, 256, window=64, pool=16)
    arch = architecture_of(raw)
    spec = arch.build_spec(arch.parse_config(raw))
    DecoderModel(spec, BuildEnv(torch.bfloat16, torch.device("cpu"), spec.hidden_size, 64, 16, None))
    with pytest.raises(ValueError, match="8 bits"):
        DecoderModel(spec, BuildEnv(torch.bfloat16, torch.device("cpu"), spec.hidden_size, 64, 16, None, cache_block=1))


def test_command_line(tmp_path):
    def tge(*args):
        return subprocess.run([sys.executable, os.path.join(ROOT, "bin", "tge"), *args], capture_output=True, text=True, timeout=300)
    import json
    path = tmp_path / "config.json"
    path.write_text(json.dumps(CONFIG))
    plain = tge("plan", "--model", str(tmp_path))
    eight = tge("plan", "--model", str(tmp_path), "--cache-dtype", "int8")
    assert plain.returncode == eight.returncode == 0
    assert "256 bytes per token" in plain.stdout and "160 bytes per token" in eight.stdout
    for wrong in (["score", "--config", str(path)], ["score", "--config", str(path), "--tokens", "1 2", "--prompt-len", "5"],
                  ["score", "--config", str(path), "--tokens", "1 2", "--compare"], ["score", "--config", str(path), "--tokens", "1 2", "--top", "33"],
                  ["score", "--config", str(path), "--tokens", "1 2", "--cache-dtype", "int4"]):
        assert tge(*wrong).returncode == 2, wrong


@pytest.mark.parametrize("block", [0, -4, 3, 128])
def test_a_block_that_no_page_holds_is_refused_wherever_a_model_is_put_together(block, tmp_path):
    """By `tge plan` as by an engine."""
    import json
    arch = architecture_of(CONFIG)
    with pytest.raises(ValueError, match="cache_block"):
        DecoderModel(arch.build_spec(arch.parse_config(CONFIG)), env(block))
    (tmp_path / "config.json").write_text(json.dumps(CONFIG))
    done = subprocess.run([sys.executable, os.path.join(ROOT, "bin", "tge"), "plan", "--model", str(tmp_path), "--cache-dtype", "int8", "--cache-block", str(block)],
                          capture_output=True, text=True, timeout=300)
    assert done.returncode != 0 and "cache_block" in done.stderr
