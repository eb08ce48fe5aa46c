"""GPU tests of the operations with ``rope=`` on the operands that layers have in hand: parts of their projections, types that differ."""

import numpy as np
import pytest
import torch

from easydel_amd.caching import (DecayStateCacheConfig, DecayStateCacheView, DecayStateMetadata, MLARaggedPagesCacheConfig, MLARaggedPagesCacheView,
                                 RaggedPagesCacheConfig, RaggedPagesCacheView, RaggedPagesMetadata)
from easydel_amd.operations import OperationMetadata, OperationRegistry, Rotary
from rope_testlib import BF16, F32, decode, encode, rotate, tl
from test_gpu_hybrid_step import _steps

pytestmark = pytest.mark.gpu

TYPE = {BF16: torch.bfloat16, F32: torch.float32}


def _draw(rng, gpu, tag, *shape):
    raw = encode(rng.standard_normal(shape).astype(np.float32), tag)
    return decode(raw, tag), tl.to_torch(raw, tag, gpu)


def _turned(x, pos, tab, neox, gpu):
    """Rotated in float32, rounded once to bfloat16."""
    rows = tab[np.clip(pos, 0, len(tab) - 1)]
    return tl.to_torch(encode(rotate(x, rows, tab.shape[1], neox), BF16), BF16, gpu)


@pytest.mark.parametrize("neox", [True, False])
@pytest.mark.parametrize("q_tag,k_tag", [(BF16, BF16), (F32, BF16), (BF16, F32), (F32, F32)])
def test_multi_latent_operation_with_rope_on_parts_of_projections(gpu, q_tag, k_tag, neox):
    """Queries are the tail of every head of one projection, latent rows and rope keys the two ends of another's rows."""
    rng = np.random.default_rng(17)
    H, rank, nope, R = 16, 512, 128, 64
    config = MLARaggedPagesCacheConfig.create(torch.bfloat16, 1, 1, 256, kv_lora_rank=rank, qk_rope_head_dim=R, page_size=32, num_pages=41)
    a, b = (MLARaggedPagesCacheView.init(config, device=gpu) for _ in range(2))
    op = OperationRegistry.create("multi_latent_ragged_page_attention_v2", OperationMetadata())
    rope = Rotary.create(R, 256, is_neox_style=neox, device=gpu)
    tab = rope.cos_sin.cpu().numpy()
    for fields, T, pos in _steps(32):
        meta = RaggedPagesMetadata.from_numpy(fields, version="v3", page_size=32, device=gpu)
        (_, absorbed), (q32, q), (kv32, kv) = _draw(rng, gpu, BF16, T, H, rank), _draw(rng, gpu, q_tag, T, H, nope + R), _draw(rng, gpu, k_tag, T, rank + R)
        latent, pe = kv.split([rank, R], -1)
        got = op(absorbed, q[..., nope:], latent, pe, a, meta, softmax_scale=192 ** -0.5, rope=rope).attention_outputs
        want = op(absorbed, _turned(q32[..., nope:], pos, tab, neox, gpu), latent, _turned(kv32[:, None, rank:], pos, tab, neox, gpu)[:, 0], b, meta,
                  softmax_scale=192 ** -0.5).attention_outputs
        torch.cuda.synchronize()
        assert got.dtype == torch.bfloat16 and torch.equal(a.kv_pages, b.kv_pages) and torch.equal(got, want)


@pytest.mark.parametrize("q_tag,kv_tag", [(BF16, BF16), (BF16, F32), (F32, BF16)])
@pytest.mark.parametrize("kvdtype", [torch.bfloat16, torch.float32])
def test_v3_operation_with_rope_on_parts_of_heads_and_other_types(gpu, kvdtype, q_tag, kv_tag):
    """Heads of 64 that are the front of heads of 80 of one projection."""
    rng = np.random.default_rng(18)
    Hq, Hkv, D = 4, 2, 64
    config = RaggedPagesCacheConfig.create(kvdtype, 1, Hkv, 256, kv_head_dim_size=D, page_size=32, num_pages=41)
    a, b = (RaggedPagesCacheView.init(config, device=gpu) for _ in range(2))
    op = OperationRegistry.create("ragged_page_attention_v3", OperationMetadata())
    rope = Rotary.create(D, 256, device=gpu)
    tab = rope.cos_sin.cpu().numpy()
    for fields, T, pos in _steps(32):
        meta = RaggedPagesMetadata.from_numpy(fields, version="v3", page_size=32, device=gpu)
        (q32, q), (k32, k), (_, v) = _draw(rng, gpu, q_tag, T, Hq, 80), _draw(rng, gpu, kv_tag, T, Hkv, 80), _draw(rng, gpu, kv_tag, T, Hkv, 80)
        got = op(q[..., :D], k[..., :D], v[..., :D], a, meta, rope=rope).attention_outputs
        rows = tab[np.clip(pos, 0, len(tab) - 1)]
        turned = lambda x: torch.from_numpy(rotate(x[..., :D], rows, D, True)).to(gpu)  # noqa: E731
        want = op(turned(q32).to(TYPE[q_tag]), turned(k32), v[..., :D], b, meta).attention_outputs
        torch.cuda.synchronize()
        assert got.dtype == TYPE[q_tag] and torch.equal(a.kv_pages, b.kv_pages) and torch.equal(got, want)


@pytest.mark.parametrize("tag", [BF16, F32])
def test_linear_layer_on_parts_of_heads(gpu, tag):
    rng = np.random.default_rng(19)
    T, H, D = 70, 3, 64
    _, heads = _draw(rng, gpu, tag, T, H, 3 * D)
    parts = heads.split(D, -1)
    one = lambda *x: torch.tensor(x, dtype=torch.int32, device=gpu)  # noqa: E731
    meta = DecayStateMetadata(query_start_loc=one(0, 69, 70), num_seqs=one(2), state_indices=one(2, 0))
    decays = torch.tensor([-0.1, -1.0, -3.0], device=gpu)
    op = OperationRegistry.create("ragged_decay_linear_attention", OperationMetadata())
    views = [DecayStateCacheView.init(DecayStateCacheConfig.create(1, H, D, D, num_slots=3), device=gpu) for _ in range(2)]
    got = op(*parts, views[0], meta, decays).attention_outputs
    want = op(*(x.contiguous() for x in parts), views[1], meta, decays).attention_outputs
    torch.cuda.synchronize()
    assert torch.equal(got, want) and torch.equal(views[0].state, views[1].state) and torch.isfinite(got).all()
