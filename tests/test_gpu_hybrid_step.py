"""GPU tests of the operators as a serving step uses them together: the rotating append behind the attention operations and the
cache views, and decayed linear attention layers on the same ragged metadata, over prefill, chunked prefill and decode."""

import numpy as np
import pytest
import torch

import test_gpu_decay_attention as decay
from easydel_amd import kernels
from easydel_amd.caching import (DecayStateCacheConfig, DecayStateCacheView, DecayStateMetadata, MLARaggedPagesCacheConfig, MLARaggedPagesCacheView,
                                 RaggedPagesCacheConfig, RaggedPagesCacheView, RaggedPagesMetadata, UnifiedAttentionCacheConfig,
                                 UnifiedAttentionCacheView, compute_ragged_batch_fields)
from easydel_amd.operations import OperationMetadata, OperationRegistry, Rotary
from rope_testlib import BF16, FP8, INT8, append_scaled, decode, encode, raw_of, rotate, table, token_positions

pytestmark = pytest.mark.gpu

STEPS = [[70, 3, 0, 1], [1, 40, 5, 0], [1, 1, 1, 33], [1, 1, 0, 1]]  # tokens scheduled for each of four requests


def _steps(page_size, version="v3", seed=0):
    """(fields, T, positions of the tokens) of every step; five rows, the last never used."""
    rng = np.random.default_rng(seed)
    pages = rng.permutation(np.arange(1, 41)).astype(np.int32).reshape(5, 8)
    done = np.zeros(5, np.int32)
    for scheduled in STEPS:
        sched = np.array(scheduled + [0], np.int32)
        fields = compute_ragged_batch_fields(scheduled_full=sched, active_mask_full=sched >= 0, num_computed_tokens=done, page_table=pages,
                                             version=version, max_num_reqs=5, page_size=page_size)
        T = int(sched.sum()) + 2
        yield fields, T, token_positions(fields["context_lens"], fields["query_start_loc"], int(fields["num_seqs"][0]), T)
        done = done + sched


def _draw(rng, gpu, *shape):
    raw = encode(rng.standard_normal(shape).astype(np.float32), BF16)
    return raw, torch.from_numpy(raw.view(np.int16)).to(gpu).view(torch.bfloat16)


def _turned(raw, pos, tab, neox, gpu):
    rows = tab[np.clip(pos, 0, len(tab) - 1)]
    out = encode(rotate(decode(raw, BF16), rows, tab.shape[1], neox), BF16)
    return torch.from_numpy(out.view(np.int16)).to(gpu).view(torch.bfloat16)


@pytest.mark.parametrize("neox", [True, False])
@pytest.mark.parametrize("Hq,Hkv,D,rope_dim,kvdtype", [(8, 2, 128, 128, torch.bfloat16), (6, 3, 64, 32, torch.bfloat16), (4, 2, 80, 80, torch.bfloat16),
                                                       (8, 2, 128, 64, torch.float8_e4m3fn)])
def test_v3_operation_with_rope_is_the_one_without_on_rotated_inputs(gpu, Hq, Hkv, D, rope_dim, kvdtype, neox):
    rng = np.random.default_rng(3)
    config = RaggedPagesCacheConfig.create(kvdtype, 1, Hkv, 256, kv_head_dim_size=D, page_size=32, num_pages=41)
    a, b = (RaggedPagesCacheView.init(config, device=gpu) for _ in range(2))
    op = OperationRegistry.create("ragged_page_attention_v3", OperationMetadata())
    rope = Rotary.create(rope_dim, 256, is_neox_style=neox, device=gpu)
    for fields, T, pos in _steps(32):
        meta = RaggedPagesMetadata.from_numpy(fields, version="v3", page_size=32, device=gpu)
        (q_raw, q), (k_raw, k), (_, v) = _draw(rng, gpu, T, Hq, D), _draw(rng, gpu, T, Hkv, D), _draw(rng, gpu, T, Hkv, D)
        tab = rope.cos_sin.cpu().numpy()
        got = op(q[None], k[None], v[None], a, meta, rope=rope).attention_outputs
        want = op(_turned(q_raw, pos, tab, neox, gpu), _turned(k_raw, pos, tab, neox, gpu), v, b, meta).attention_outputs
        torch.cuda.synchronize()
        assert got.shape == (1, T, Hq, D)
        if kvdtype == torch.bfloat16:
            assert torch.equal(a.kv_pages, b.kv_pages) and torch.equal(got[0], want)
        else:  # the rotating write casts the float32 keys, the other one keys rounded to bf16 before: one e4m3 step apart at most
            x, y = a.kv_pages.float(), b.kv_pages.float()
            assert ((x - y).abs() <= torch.maximum(x.abs(), y.abs()) * 2.0 ** -3 + 2.0 ** -9).all()
            again = kernels.ragged_paged_attention(_turned(q_raw, pos, tab, neox, gpu), a.kv_pages, meta.context_lens, meta.pages_tables.reshape(-1),
                                                   meta.query_start_loc, meta.request_distribution[2:3], num_kv_heads=Hkv)
            assert torch.equal(got[0], again)


@pytest.mark.parametrize("kv", [FP8, INT8])
def test_v3_operation_with_rope_over_scaled_pages(gpu, kv):
    rng = np.random.default_rng(4)
    Hq, Hkv, D, kvdtype = 8, 2, 128, torch.float8_e4m3fn if kv == FP8 else torch.int8
    config = RaggedPagesCacheConfig.create(kvdtype, 1, Hkv, 256, kv_head_dim_size=D, page_size=32, num_pages=41)
    view = RaggedPagesCacheView.init(config, device=gpu, scaled=True)
    op = OperationRegistry.create("ragged_page_attention_v3", OperationMetadata())
    rope = Rotary.create(D, 256, device=gpu)
    tab = rope.cos_sin.cpu().numpy()
    C = config.combined_heads_per_token
    codes, scales = np.zeros((41, 32, C, D), np.uint8), np.ones((41, C), np.float32)
    for fields, T, pos in _steps(32):
        meta = RaggedPagesMetadata.from_numpy(fields, version="v3", page_size=32, device=gpu)
        (q_raw, q), (k_raw, k), (v_raw, v) = _draw(rng, gpu, T, Hq, D), _draw(rng, gpu, T, Hkv, D), _draw(rng, gpu, T, Hkv, D)
        got = op(q, k, v, view, meta, rope=rope).attention_outputs
        k32 = rotate(decode(k_raw, BF16), tab[np.clip(pos, 0, 255)], D, True)
        codes, scales = append_scaled(k32, decode(v_raw, BF16), codes, scales, fields["context_lens"], fields["pages_tables"], fields["query_start_loc"],
                                      int(fields["request_distribution"][2]), kv)
        torch.cuda.synchronize()
        assert np.array_equal(view.kv_pages.view(torch.uint8).cpu().numpy().reshape(codes.shape), codes)
        assert np.array_equal(view.kv_scales.cpu().numpy(), scales)
        want = kernels.ragged_paged_attention(_turned(q_raw, pos, tab, True, gpu), view.kv_pages, meta.context_lens, meta.pages_tables.reshape(-1),
                                              meta.query_start_loc, meta.request_distribution[2:3], kv_scales=view.kv_scales, num_kv_heads=Hkv)
        assert torch.equal(got, want)


def test_unified_view_with_rope(gpu):
    rng = np.random.default_rng(5)
    Hq, Hkv, D = 8, 4, 64
    config = UnifiedAttentionCacheConfig.create(torch.bfloat16, 1, Hkv, 256, D, page_size=32, num_pages=41)
    a, b = (UnifiedAttentionCacheView.init(config, device=gpu) for _ in range(2))
    op = OperationRegistry.create("unified_attention", OperationMetadata())
    rope = Rotary.create(D, 256, device=gpu)
    tab = rope.cos_sin.cpu().numpy()
    for fields, T, pos in _steps(32, version="v2"):
        meta = RaggedPagesMetadata.from_numpy(fields, version="v2", page_size=32, device=gpu)
        (q_raw, q), (k_raw, k), (_, v) = _draw(rng, gpu, T, Hq, D), _draw(rng, gpu, T, Hkv, D), _draw(rng, gpu, T, Hkv, D)
        got = op(a.rope_concatenate_to_cache(q, k, v, meta, rope), a, meta).attention_outputs
        b.concatenate_to_cache(_turned(k_raw, pos, tab, True, gpu), v, meta)
        want = op(_turned(q_raw, pos, tab, True, gpu), b, meta).attention_outputs
        torch.cuda.synchronize()
        assert torch.equal(a.key_cache, b.key_cache) and torch.equal(a.value_cache, b.value_cache) and torch.equal(got, want)


def test_v2_view_with_rope(gpu):
    rng = np.random.default_rng(6)
    config = RaggedPagesCacheConfig.create(torch.bfloat16, 1, 2, 256, kv_head_dim_size=128, page_size=32, num_pages=41, version="v2")
    a, b = (RaggedPagesCacheView.init(config, device=gpu) for _ in range(2))
    rope = Rotary.create(128, 256, device=gpu)
    tab = rope.cos_sin.cpu().numpy()
    for fields, T, pos in _steps(32, version="v2"):
        meta = RaggedPagesMetadata.from_numpy(fields, version="v2", page_size=32, device=gpu)
        (_, q), (k_raw, k), (_, v) = _draw(rng, gpu, T, 4, 128), _draw(rng, gpu, T, 2, 128), _draw(rng, gpu, T, 2, 128)
        a.rope_concatenate_to_cache(q, k, v, meta, rope)
        b.concatenate_to_cache(_turned(k_raw, pos, tab, True, gpu), v, meta)
        torch.cuda.synchronize()
        assert torch.equal(a.kv_pages, b.kv_pages)


def test_multi_latent_operation_with_rope(gpu):
    rng = np.random.default_rng(7)
    config = MLARaggedPagesCacheConfig.create(torch.bfloat16, 1, 1, 256, kv_lora_rank=512, qk_rope_head_dim=64, page_size=32, num_pages=41)
    a, b = (MLARaggedPagesCacheView.init(config, device=gpu) for _ in range(2))
    op = OperationRegistry.create("multi_latent_ragged_page_attention_v2", OperationMetadata())
    rope = Rotary.create(64, 256, is_neox_style=False, device=gpu)
    tab = rope.cos_sin.cpu().numpy()
    for fields, T, pos in _steps(32):
        meta = RaggedPagesMetadata.from_numpy(fields, version="v3", page_size=32, device=gpu)
        (_, qn), (qp_raw, qp), (_, kv), (pe_raw, pe) = (_draw(rng, gpu, *s) for s in ((T, 16, 512), (T, 16, 64), (T, 512), (T, 1, 64)))
        got = op(qn, qp, kv, pe[:, 0], a, meta, softmax_scale=192 ** -0.5, rope=rope).attention_outputs
        want = op(qn, _turned(qp_raw, pos, tab, False, gpu), kv, _turned(pe_raw, pos, tab, False, gpu)[:, 0], b, meta, softmax_scale=192 ** -0.5).attention_outputs
        torch.cuda.synchronize()
        assert torch.equal(a.kv_pages, b.kv_pages) and torch.equal(got, want)


@pytest.mark.parametrize("tag", [BF16, decay.F32])
def test_hybrid_layers_over_a_request_s_life(gpu, tag):
    """A paged layer and a linear layer on one step's metadata; the linear layer's outputs and states over four steps against the
    recurrence in 64 bits from the states it was given, and a request that starts over in a slot someone left."""
    rng = np.random.default_rng(8)
    Hq, Hkv, Dk, Dv = 4, 2, 64, 64
    pages = RaggedPagesCacheConfig.create(torch.bfloat16, 1, 2, 256, kv_head_dim_size=64, page_size=32, num_pages=41)
    paged = RaggedPagesCacheView.init(pages, device=gpu)
    states = DecayStateCacheView.init(DecayStateCacheConfig.create(1, Hkv, Dk, Dv, num_slots=7), device=gpu)
    states.state.fill_(float("nan"))  # what an earlier owner left: fresh requests start from zero all the same
    attend, linear = (OperationRegistry.create(n, OperationMetadata()) for n in ("ragged_page_attention_v3", "ragged_decay_linear_attention"))
    rope = Rotary.create(64, 256, device=gpu)
    slots = np.array([4, 1, 6, 0, 2], np.int32)
    log_decay = np.array([-0.05, -0.7], np.float32)
    for fields, T, _ in _steps(32):
        meta = RaggedPagesMetadata.from_numpy(fields, version="v3", page_size=32, device=gpu)
        _, q = _draw(rng, gpu, T, 4, 64)
        _, k = _draw(rng, gpu, T, 2, 64)
        out = attend(q, k, k, paged, meta, rope=rope).attention_outputs
        assert torch.isfinite(out).all()
        c = decay.Case()
        c.Hq, c.Hkv, c.Dk, c.Dv, c.tag, c.n, c.S, c.N, c.T = Hq, Hkv, Dk, Dv, tag, int(fields["num_seqs"][0]), 5, 7, T
        c.qsl, c.ctx = fields["query_start_loc"], fields["context_lens"]
        c.q_lens = np.diff(c.qsl)[:c.n]
        c.past = (c.ctx[:c.n] - c.q_lens)
        c.slot_in = c.slot_out = slots
        c.log_decay, c.state = log_decay, states.state.cpu().numpy().copy()
        c.q, c.k, c.v = (encode(rng.standard_normal(s).astype(np.float32), tag) for s in ((T, Hq, Dk), (T, Hkv, Dk), (T, Hkv, Dv)))
        up = lambda x: decay.tl.to_torch(x, tag, gpu)[None]  # noqa: E731
        got = linear(up(c.q), up(c.k), up(c.v), states, DecayStateMetadata.from_ragged(meta, torch.from_numpy(slots).to(gpu)),
                     torch.from_numpy(log_decay).to(gpu))
        torch.cuda.synchronize()
        assert got.attention_outputs.shape == (1, T, Hq, Dv) and got.cache_view is states
        unowned = np.isnan(c.state)
        now = states.state.cpu().numpy()
        written = [int(slots[i]) for i in range(c.n) if c.q_lens[i] > 0]
        rest = [s for s in range(7) if s not in written]
        assert np.array_equal(now[rest], c.state[rest], equal_nan=True)
        assert np.isfinite(now[written]).all()
        c.state[unowned] = 0.0
        decay.check(c, got.attention_outputs[0], torch.from_numpy(np.where(np.isnan(now), 0.0, now)), in_place=True)
