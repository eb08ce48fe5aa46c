"""CPU tests of the host side around the rotating append and the decayed linear attention: registry, requirements, configurations,
the rotation's table, refusals."""

import math

import pytest
import torch

from easydel_amd.caching import DecayStateCache, DecayStateCacheConfig, DecayStateCacheView, DecayStateMetadata, RaggedPagesMetadata
from easydel_amd.operations import CacheType, MetadataField, OperationMetadata, OperationRegistry, Rotary


def test_registry_and_requirements():
    op = OperationRegistry.create("ragged_decay_linear_attention", OperationMetadata())
    req = type(op).get_requirements()
    assert req.cache.supported == CacheType.RECURRENT and req.cache.cache_view_class is DecayStateCacheView
    assert MetadataField.STATE_INDICES in req.metadata.required and MetadataField.PAGES_TABLES not in req.metadata.required


def test_state_pool():
    config = DecayStateCacheConfig.create(2, 4, 16, 32, num_slots=5)
    cache = DecayStateCache.init_cache(config, device="cpu")
    assert len(cache.views) == 2 and tuple(cache.views[1].state.shape) == (5, 4, 16, 32) and cache.views[1].layer_index == 1
    assert cache.views[0].state.dtype == torch.float32 and not cache.views[0].state.any()
    assert cache.views[0].concatenate_to_cache(None, None, None) is cache.views[0]
    sized = DecayStateCacheConfig.create(3, 4, 16, 32, free_hbm_bytes=1 << 30, hbm_utilization=0.5)
    assert sized.num_slots == (1 << 29) // (3 * 4 * 16 * 32 * 4)
    for bad in (dict(num_hidden_layers=0), dict(num_kv_heads=0), dict(k_headdim=0), dict(v_headdim=-1)):
        with pytest.raises(ValueError, match="must be positive"):
            DecayStateCacheConfig.create(**{**dict(num_hidden_layers=1, num_kv_heads=1, k_headdim=4, v_headdim=4, num_slots=1), **bad})
    with pytest.raises(ValueError, match="num_slots"):
        DecayStateCacheConfig.create(1, 1, 256, 256, free_hbm_bytes=1000)


def test_metadata_of_the_paged_layers():
    for version in ("v2", "v3"):
        meta = RaggedPagesMetadata.create_empty(8, 3, 2, page_size=16, version=version, device="cpu")
        meta.num_seqs[0] = 2
        if version == "v3":
            meta.request_distribution[2] = 2
        got = DecayStateMetadata.from_ragged(meta, torch.zeros(3, dtype=torch.int32))
        assert got.num_seqs.tolist() == [2] and got.query_start_loc is meta.query_start_loc and got.context_lens is meta.context_lens


def test_rotation_table():
    r = Rotary.create(8, 100_000, theta=500.0, is_neox_style=False, device="cpu")
    assert tuple(r.cos_sin.shape) == (100_000, 8) and r.cos_sin.dtype == torch.float32 and not r.is_neox_style
    for p in (0, 1, 99_999):
        for d in range(4):
            angle = p * 500.0 ** (-2 * d / 8)
            # half a float32 step of a value below one, and the angle's own 64-bit rounding
            assert abs(float(r.cos_sin[p, d]) - math.cos(angle)) <= 2.0 ** -25 + 1e-10
            assert abs(float(r.cos_sin[p, 4 + d]) - math.sin(angle)) <= 2.0 ** -25 + 1e-10
    for bad in ((7, 10), (0, 10), (8, 0)):
        with pytest.raises(ValueError):
            Rotary.create(*bad, device="cpu")


def test_reading_operations_refuse_a_rotation():
    r = Rotary.create(8, 4, device="cpu")
    q = torch.zeros(1, 1, 8)
    with pytest.raises(NotImplementedError, match="rope_concatenate_to_cache"):
        OperationRegistry.create("ragged_page_attention_v2", OperationMetadata())(q, q, q, None, None, rope=r)
    with pytest.raises(NotImplementedError, match="rope_concatenate_to_cache"):
        OperationRegistry.create("unified_attention", OperationMetadata())(q, None, None, rope=r)
    op = OperationRegistry.create("ragged_page_attention_v3", OperationMetadata())
    with pytest.raises(NotImplementedError, match="shard-local"):
        meta = RaggedPagesMetadata.create_empty(1, 1, 1, version="v3", device="cpu")
        op.forward_v3_dp_local_shard(q, q, q, torch.zeros(1, 16, 2, 8), meta, 0, 1, rope=r)
    with pytest.raises(NotImplementedError, match="shard-local"):
        pool = torch.zeros(1, 16, 1, 8)
        OperationRegistry.create("unified_attention", OperationMetadata()).forward_dp_local_shard(q, pool, pool, meta, 0, 1, rope=r)


def test_the_linear_layer_takes_parts_of_every_head(monkeypatch):
    """One projection reshaped to heads and split inside each head, with and without a batch axis; rows of a projection stay where they are."""
    from easydel_amd import kernels

    seen = []
    monkeypatch.setattr(kernels, "decay_linear_attention", lambda q, k, v, g, state, *a, **kw: (seen.append((q, k, v)) or q.new_zeros(*q.shape[:2], v.shape[2]), state))
    op = OperationRegistry.create("ragged_decay_linear_attention", OperationMetadata())
    view = DecayStateCacheView.init(DecayStateCacheConfig.create(1, 2, 16, 32, num_slots=3), device="cpu")
    i = torch.zeros(3, dtype=torch.int32)
    meta = DecayStateMetadata(query_start_loc=i, num_seqs=i[:1], state_indices=i[:2])
    heads = torch.arange(5 * 2 * 64.0).reshape(5, 2, 64)
    parts = heads.split((16, 16, 32), -1)
    for lead in ((), (1,)):
        out = op(*(x.reshape(*lead, *x.shape) for x in parts), view, meta, torch.zeros(2)).attention_outputs
        assert out.shape == (*lead, 5, 2, 32)
        for got, want in zip(seen.pop(), parts):
            assert torch.equal(got, want) and got[0].is_contiguous()
    rows = [x.unflatten(1, (2, -1)) for x in heads.flatten(1).split((32, 32, 64), 1)]
    op(*rows, view, meta, torch.zeros(2))
    assert [x.data_ptr() for x in seen.pop()] == [x.data_ptr() for x in rows]
