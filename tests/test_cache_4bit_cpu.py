"""The 4-bit cache on the host: its definition's own properties, what a spec says of its entries, what the cache manager lays out, what is refused."""
import json
import math
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
from plain import cache_4bit_plain as plain

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CONFIG = {"architectures": ["Qwen2ForCausalLM"], "num_hidden_layers": 2, "hidden_size": 64, "num_attention_heads": 4, "num_key_value_heads": 2,
          "head_dim": 16, "intermediate_size": 176, "vocab_size": 256, "rope_theta": 10000.0, "rms_norm_eps": 1e-6, "tie_word_embeddings": True,
          "max_position_embeddings": 256}


def env(four=True, page=16, dtype=torch.bfloat16, block=None):
    return BuildEnv(dtype=dtype, device=torch.device("cpu"), hidden_size=64, max_positions=64, page_size=page, ops=None, cache_block=block, cache_4bit=four)


def attention(four=True, position="rope_neox", head_dim=16, **options):
    place = PartSpec(position, {"head_dim": head_dim, "theta": 10000.0} if position != "none" else {})
    return build_part(MIXERS, PartSpec("gqa_attention", {"hidden_size": 64, "heads": 4, "kv_heads": 2, "head_dim": head_dim, "position": place, **options}), env(four))


@pytest.mark.parametrize("size", [1e-40, 1e-3, 1.0, 1e20])
def test_an_entrys_values_lie_within_half_a_step(size):
    """The plain definition against itself: no number of a group lies outside its sixteen values, the step is no more than the span asks for."""
    gen = torch.Generator().manual_seed(1)
    for dim in (32, 64, 40, 7):
        for shift in (0.0, 30.0):
            x = ((torch.randn(dim, generator=gen) + shift) * size).float()
            codes, steps, bases = plain.entry(x)
            for j in range(-(-dim // 32)):
                part = x[32 * j:32 * j + 32].double()
                values = torch.tensor([bases[j] + (c - 8) * steps[j] for c in codes[32 * j:32 * j + 32]], dtype=torch.float64)
                assert float((values - part).abs().max()) <= steps[j] * (0.5 + 1e-6) + 2.0 ** -22 * float(part.abs().max()) + 1e-44
                # the base is known to 2^-9 of itself, the step to 2^-7 of itself
                span = float(part.max() - part.min())
                assert steps[j] <= (span / 15 + 2.0 ** -8 * abs(bases[j]) / 7) * (1 + 2.0 ** -6) + 1e-40
    assert plain.entry(torch.zeros(32)) == ([8] * 32, [0.0], [0.0])
    for bad in (math.nan, math.inf, 2.0 ** 96, -1e38):
        assert plain.entry(torch.tensor([0.5, bad]))[0] is None


def test_the_order_of_the_codes():
    """Number 32 j + 4 g + n of an entry of G groups is nibble n of the (g G + j)-th two bytes."""
    for dim in (16, 64, 80, 128):
        groups = -(-dim // 32)
        for d in range(dim):
            units = torch.zeros(16 * groups, dtype=torch.uint8)
            j, g, n = d // 32, d % 32 // 4, d % 4
            units[2 * (g * groups + j) + n // 2] = 9 << (4 * (n % 2))
            assert plain.unpack(units, dim).tolist() == [9 if i == d else 0 for i in range(dim)]


@pytest.mark.parametrize("head_dim,groups", [(16, 1), (32, 1), (64, 2), (80, 3), (128, 4)])
def test_layout_and_bytes(head_dim, groups):
    spec = attention(head_dim=head_dim).cache_spec()
    per_token = 2 * 2 * (16 * groups + 4 * groups)
    assert spec.bytes_per_token(2) == per_token == spec.bytes_per_token(4)
    manager = CacheManager(16, 4)
    manager.add_layer(0, spec, None)
    manager.add_layer(1, spec, None)
    manager.add_layer(2, PagedCacheSpec((("k", (2, 16)), ("v", (2, 16)))), None)           # the same positions in the run dtype
    assert len(manager.groups) == 1 and manager.layer_variant == {0: 0, 1: 0, 2: 1}
    manager.set_pool_sizes([5])
    manager.allocate_storage(torch.float32, torch.device("cpu"))
    held = manager.layer_cache(1).paged
    assert held["k"].dtype == held["v"].dtype == torch.uint8 and held["k"].shape == held["v"].shape == (6, 2, 16, 16 * groups)
    assert held["k_groups"].dtype == held["v_groups"].dtype == torch.bfloat16 and held["k_groups"].shape == (6, 2, 16, 2 * groups)
    assert all(t.is_contiguous() for t in held.values())


def test_a_model_says_what_its_cache_takes():
    arch = architecture_of(CONFIG)
    spec = arch.build_spec(arch.parse_config(CONFIG))
    model = DecoderModel(spec, env())
    assert model.cache_bytes_per_token() == 2 * 2 * 2 * (16 + 4)
    assert model.decode_cache_bytes(100) == 100 * model.cache_bytes_per_token()
    with pytest.raises(ValueError, match="8 bits or in 4"):
        DecoderModel(spec, env(block=1))


NORM = {"scope": "head", "eps": 1e-6}


@pytest.mark.parametrize("options,holds", [({}, True), ({"window": 32}, True), ({"sinks": True}, True), ({"qk_norm": NORM}, True), ({"qk_norm": NORM, "window": 8}, True),
                                           ({"position": "rope_interleaved"}, True), ({"position": "rope_interleaved", "qk_norm": NORM}, True), ({"position": "none"}, True),
                                           ({"qk_norm": {"scope": "projection", "eps": 1e-6}}, False), ({"value_dim": 8}, False), ({"short_conv": 3}, False),
                                           ({"output_gate": True}, False), ({"value_mix": "first"}, False), ({"qk_norm": dict(NORM, after_rotation=True)}, False)])
def test_which_attention_can_hold_it(options, holds):
    assert attention(False, **options).holds_4bit is holds
    kept = attention(True, **options).cache_spec()
    assert bool(kept.formats) is holds
    assert not attention(False, **options).cache_spec().formats


def test_a_model_that_cannot_refuses():
    from aegean_tge_b200.bench_tools import mozepel_config
    raw = mozepel_config(64, 4, 2, 16, 176, 4, 256, window=64, pool=16)
    arch = architecture_of(raw)
    spec = arch.build_spec(arch.parse_config(raw))
    with pytest.raises(ValueError, match="4 bits"):
        DecoderModel(spec, BuildEnv(torch.bfloat16, torch.device("cpu"), spec.hidden_size, 64, 16, None, cache_4bit=True))


def test_command_line(tmp_path):
    def tge(*args):
        return subprocess.run([sys.executable, os.path.join(ROOT, "bin", "tge"), *args], capture_output=True, text=True, timeout=300)
    (tmp_path / "config.json").write_text(json.dumps(CONFIG))
    four = tge("plan", "--model", str(tmp_path), "--cache-dtype", "uint4")
    assert four.returncode == 0 and "160 bytes per token" in four.stdout        # (heads of 16 take a group of 32 whole)
    wide = dict(CONFIG, head_dim=32)
    (tmp_path / "config.json").write_text(json.dumps(wide))
    assert "512 bytes per token" in tge("plan", "--model", str(tmp_path)).stdout
    assert "160 bytes per token" in tge("plan", "--model", str(tmp_path), "--cache-dtype", "uint4").stdout
    assert tge("plan", "--model", str(tmp_path), "--cache-dtype", "uint4", "--cache-block", "4").returncode == 2
    assert tge("plan", "--model", str(tmp_path), "--cache-dtype", "uint8").returncode == 2


def test_operators_refuse_what_is_not_on_a_device():
    """Before any kernel is built or loaded."""
    from aegean_tge_b200 import ops
    pages, pairs = torch.zeros(2, 1, 16, 32, dtype=torch.uint8), torch.zeros(2, 1, 16, 4).bfloat16()
    ints = torch.zeros(2, dtype=torch.int32)
    table = torch.zeros(1, 1, dtype=torch.int32)
    with pytest.raises(ops.KernelError, match="CUDA"):
        ops.norm_rope_kv_store_4bit(torch.zeros(1, 192), None, None, 0, ints[:1], ints[:1], 1, table, pages, pages, pairs, pairs, 1, 1, 64)
    with pytest.raises(ops.KernelError, match="CUDA"):
        ops.read_cache_4bit(pages, pages, pairs, pairs, table, ints, ints[:1], [1], 64, torch.float32)
    with pytest.raises(ops.KernelError, match="CUDA"):
        ops.attention_4bit(torch.zeros(1, 64), pages, pages, pairs, pairs, table, ints, ints[:1], ints[:1], ints[:1], 1, 1, 1, 1, 1, 64, 0.1)
