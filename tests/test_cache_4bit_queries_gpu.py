"""Queries of a layer that reads another layer's 4-bit cache: prepared as the owner's are, without a store."""
import dataclasses

import pytest
import torch

from helpers import batch_index
from test_cache_4bit_engine_gpu import prompt, registered, run
from test_cache_4bit_gpu import DEV, Cache, ops, tables  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dim,rotary", [(64, 64), (128, 128), (48, 24), (256, 0)])
@pytest.mark.parametrize("normed,pairs", [(False, False), (True, False), (True, True)])
def test_queries_without_a_store(ops, dtype, dim, rotary, normed, pairs):
    """A layer that reads another's cache: the queries of the call that stores, bit for bit, from rows that need hold nothing else; pages are not touched."""
    heads, kv, lens, starts = 5, 2, [1, 40, 7], [8, 0, 100]
    cache = Cache([a + b for a, b in zip(lens, starts)], kv, dim, 16)
    gen = torch.Generator().manual_seed(4)
    qkv = torch.randn(48, (heads + 2 * kv) * dim, generator=gen).to(dtype).to(DEV)
    weight = (1.0 + 0.3 * torch.randn(dim, generator=gen)).to(DEV)
    cos, sin = (t.to(DEV) for t in tables(200, rotary)) if rotary else (None, None)
    positions, seq, _, _ = batch_index(lens, starts, DEV)
    kw = {"pairs": pairs, **({"q_norm": weight, "k_norm": weight} if normed else {})}
    device, table = cache.device(), cache.table.to(DEV)
    want = ops.norm_rope_kv_store_4bit(qkv, cos, sin, rotary, positions, seq, 3, table, *device, heads, kv, dim, **kw)
    alone = {key: value for key, value in kw.items() if key != "k_norm"}
    for rows in (qkv, qkv[:, :heads * dim], qkv[:, :heads * dim].contiguous()):
        got = ops.norm_rope_kv_store_4bit(rows, cos, sin, rotary, positions, seq, 3, None, None, None, None, None, heads, kv, dim, **alone)
        assert torch.equal(got, want)
    ops.check_status()
    if rotary:                                               # positions that the tables do not have are reported as ever
        ops.norm_rope_kv_store_4bit(qkv, cos[:50], sin[:50], rotary, positions, seq, 3, None, None, None, None, None, heads, kv, dim, **alone)
        with pytest.raises(ops.DeviceStatusError):
            ops.check_status()
    for some in ((table, device[0], None, None, None), (None, *device), (table, None, device[1], None, None), (None, None, None, device[2], device[3])):
        with pytest.raises((ops.KernelError, AttributeError)):
            ops.norm_rope_kv_store_4bit(qkv, cos, sin, rotary, positions, seq, 3, *some, heads, kv, dim, **alone)
    with pytest.raises(ops.KernelError):
        ops.norm_rope_kv_store_4bit(qkv[:, :heads * dim - 1], cos, sin, rotary, positions, seq, 3, None, None, None, None, None, heads, kv, dim, **alone)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("normed,position", [(True, "rope_neox"), (True, "rope_interleaved"), (False, "rope_interleaved"), (False, "rope_neox"), (True, "none")])
def test_queries_of_a_layer_that_reads_anothers_cache(monkeypatch, dtype, normed, position):
    """The bits that the kernel that stores makes of the same product, with one rounding behind norm and rotation."""
    from aegean_tge_b200 import Engine, ops
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
        return dataclasses.replace(layer, cache_from=0) if i == 1 else layer

    eng = Engine(random_config=registered(monkeypatch, "SharedForCausalLM", change, extra), dtype=dtype, context=256, max_tokens=1024, page_size=16, cache_dtype="uint4",
                 use_graphs=False)
    linear, attention, last, seen = ops.linear, ops.attention_4bit, [], []

    def spy_linear(*args, **kw):
        out = linear(*args, **kw)
        last[:] = [out.clone() if isinstance(out, torch.Tensor) else None]
        return out

    def spy_attention(q, *args, **kw):
        seen.append((last[0], q.clone(), args))
        return attention(q, *args, **kw)

    monkeypatch.setattr(ops, "linear", spy_linear)
    monkeypatch.setattr(ops, "attention_4bit", spy_attention)
    run(eng, [40, 1, 9], prompt(50))
    assert len(seen) == 6
    for n, (qkv, q, args) in enumerate(seen):
        mixer = eng.model.blocks[n % 2].mixer
        held = [torch.zeros_like(t) for t in args[:4]]
        tables = mixer.position.rotary_tables()
        cos, sin, rotary = tables if tables is not None else mixer.position.pair_tables()
        want = ops.norm_rope_kv_store_4bit(qkv, cos, sin, rotary, args[7], args[8], args[9], args[4], *held, mixer.heads, mixer.kv_heads, mixer.head_dim,
                                           q_norm=mixer.q_norm_w, k_norm=mixer.k_norm_w, eps=1e-6, pairs=tables is None)
        assert torch.equal(q, want), n
    ops.check_status()
