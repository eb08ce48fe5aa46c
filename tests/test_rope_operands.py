"""CPU tests of what the operations hand to the rotating writes: the operands of the call without ``rope=`` are taken with it too."""

import pytest
import torch

from easydel_amd import kernels
from easydel_amd.caching import (MLARaggedPagesCacheConfig, MLARaggedPagesCacheView, RaggedPagesCacheConfig, RaggedPagesCacheView,
                                 RaggedPagesMetadata)
from easydel_amd.operations import OperationMetadata, OperationRegistry, Rotary

T = 5


def _meta():
    return RaggedPagesMetadata.create_empty(T, 2, 2, page_size=16, version="v3", device="cpu")


def _rows_in_place(t):
    return t[0].is_contiguous() and t.stride(0) >= t[0].numel()


@pytest.fixture
def latent(monkeypatch):
    """The multi-latent operation with its two kernel calls recorded."""
    seen = {}

    def write(queries_pe, keys_values, keys_pe, kv_pages, *a, **k):
        seen["write"] = (queries_pe, keys_values, keys_pe)
        return torch.empty_like(queries_pe).contiguous(), kv_pages

    def read(queries_nope, queries_pe, *a, **k):
        seen["read"] = (queries_nope, queries_pe)
        return torch.empty_like(queries_nope), None

    monkeypatch.setattr(kernels, "rope_mla_page_scatter", write)
    monkeypatch.setattr(kernels, "mla_ragged_paged_attention", read)
    op = OperationRegistry.create("multi_latent_ragged_page_attention_v2", OperationMetadata())
    config = MLARaggedPagesCacheConfig.create(torch.bfloat16, 1, 1, 64, kv_lora_rank=128, qk_rope_head_dim=64, page_size=16, num_pages=3)
    view = MLARaggedPagesCacheView.init(config, device="cpu")
    rope = Rotary.create(64, 64, device="cpu")

    def run(nope, pe, kv, kpe):
        op(nope, pe, kv, kpe, view, _meta(), rope=rope)
        return seen

    return run


def _latent_operands(dtype=torch.bfloat16):
    q = torch.zeros(T, 3, 96 + 64, dtype=dtype)  # heads of one projection: the part without a position, then the rope part
    kv = torch.zeros(T, 128 + 64, dtype=dtype)
    return torch.zeros(T, 3, 128, dtype=dtype), q.split([96, 64], -1)[1], *kv.split([128, 64], -1)


def test_multi_latent_takes_the_parts_of_its_projections(latent):
    nope, pe, kv, kpe = _latent_operands()
    assert not pe[0].is_contiguous()
    seen = latent(nope, pe, kv, kpe)
    assert all(_rows_in_place(t) for t in seen["write"]) and seen["write"][1].is_contiguous()
    assert seen["write"][2].data_ptr() == kpe.data_ptr()  # whole rows stay where they are


@pytest.mark.parametrize("pe_type,kpe_type", [(torch.float32, torch.bfloat16), (torch.bfloat16, torch.float32), (torch.float32, torch.float32),
                                              (torch.float16, torch.float16)])
def test_multi_latent_takes_types_that_differ(latent, pe_type, kpe_type):
    """Rotated in float32, and only the result in the type of ``queries_nope``."""
    nope, pe, kv, kpe = _latent_operands()
    seen = latent(nope, pe.to(pe_type), kv, kpe.to(kpe_type))
    assert seen["write"][0].dtype == seen["write"][2].dtype == torch.float32
    assert seen["read"][1].dtype == torch.bfloat16


@pytest.fixture
def v3(monkeypatch):
    """The v3 operation with its two kernel calls recorded."""
    seen = {}

    def write(query, key, value, kv_pages, *a, kv_scales=None, **k):
        seen["write"] = (query, key, value)
        out = torch.empty_like(query).contiguous()
        return (out, kv_pages) if kv_scales is None else (out, kv_pages, kv_scales)

    def read(query, *a, **k):
        seen["read"] = query
        return torch.empty_like(query)

    monkeypatch.setattr(kernels, "rope_page_scatter_ragged", write)
    monkeypatch.setattr(kernels, "ragged_paged_attention", read)
    op = OperationRegistry.create("ragged_page_attention_v3", OperationMetadata())
    rope = Rotary.create(64, 64, device="cpu")

    def run(q, k, v, kvdtype=torch.bfloat16, scaled=None):
        config = RaggedPagesCacheConfig.create(kvdtype, 1, 2, 64, kv_head_dim_size=64, page_size=16, num_pages=3)
        op(q, k, v, RaggedPagesCacheView.init(config, device="cpu", scaled=scaled), _meta(), rope=rope)
        return seen

    return run


def test_v3_takes_parts_of_every_head(v3):
    q, k, v = (torch.zeros(T, h, 80, dtype=torch.bfloat16)[..., :64] for h in (4, 2, 2))
    seen = v3(q, k, v)
    assert all(_rows_in_place(t) for t in seen["write"])
    assert all(_rows_in_place(t) for t in v3(*(torch.zeros(1, h, 64).expand(T, h, 64) for h in (4, 2, 2)))["write"])  # one row for all tokens
    qkv = torch.zeros(T, 8 * 64, dtype=torch.bfloat16)
    views = [x.unflatten(1, (-1, 64)) for x in qkv.split((256, 128, 128), 1)]
    seen = v3(*views)
    assert [t.data_ptr() for t in seen["write"]] == [t.data_ptr() for t in views]  # rows of a projection are read in place


@pytest.mark.parametrize("types", [(torch.bfloat16, torch.float32, torch.float32), (torch.float32, torch.bfloat16, torch.bfloat16),
                                   (torch.bfloat16, torch.bfloat16, torch.float32), (torch.bfloat16, torch.float16, torch.float16)])
def test_v3_takes_types_that_differ(v3, types):
    seen = v3(*(torch.zeros(T, h, 64, dtype=t) for h, t in zip((4, 2, 2), types)))
    assert {t.dtype for t in seen["write"]} == {torch.float32}
    assert seen["read"].dtype == types[0]


def test_narrowing_is_told_with_rope_as_without(latent, v3, caplog):
    """Rows of a wider type than the pages are cast with a warning; scaled pages are coded, which is no cast."""
    wide, narrow = torch.float32, torch.bfloat16
    ops = _latent_operands()
    for kv, kpe, told in ((narrow, narrow, False), (wide, narrow, True), (narrow, wide, True)):
        caplog.clear()
        latent(*ops[:2], ops[2].to(kv), ops[3].to(kpe))
        assert ("lower-precision KV cache dtype" in caplog.text) == told
    q, k = torch.zeros(T, 4, 64, dtype=narrow), torch.zeros(T, 2, 64, dtype=narrow)
    for key, value, kvdtype, scaled, told in ((k, k, narrow, None, False), (k.to(wide), k, narrow, None, True), (k, k.to(wide), narrow, None, True),
                                              (k, k, torch.float8_e4m3fn, None, True), (k, k, torch.float8_e4m3fn, True, False), (k, k, torch.int8, None, False)):
        caplog.clear()
        v3(q, key, value, kvdtype, scaled)
        assert ("lower-precision KV cache dtype" in caplog.text) == told


def test_token_rows_are_copied_only_where_they_must_be():
    from easydel_amd.operations.rotary import token_rows

    x = torch.arange(6 * 5 * 8.0).reshape(6, 5, 8)
    for t, stays in ((x, True), (x[:, 1:3], True), (x[::2], True), (x[:, 2], True), (x[:1, 1:], True), (x[:, :, :1], False), (x[:0, :, :4], True),
                     (x[:, :, :4], False), (x[:, ::2], False), (x.transpose(0, 1), False), (x[:1].expand(6, 5, 8), False), (x[:, :1, :4], True), (x[:1, :, :4], False),
                     (x[:, 0, ::2], False), (x[:, 0, :0], True)):
        got = token_rows(t)
        assert torch.equal(got, t) and (got is t) == stays, (t.shape, t.stride())
        assert got.shape[0] == 0 or got[0].is_contiguous()
